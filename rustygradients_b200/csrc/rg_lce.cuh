// Shared between the two forms of the linear cross entropy (rg_b200.h): few rows on the CUDA cores (rg_lce.cu) and many
// rows on the tensor cores (rg_lce_tc.cu).
#pragma once
#include "rg_train.cuh"

// What one call works on, and its scratch.
struct lce_call {
    int R, D, V;
    int dtype;
    const void *x, *w;     // [R][D], [D][V]
    const float* bias;     // V or NULL
    const int* tgt;        // R: target column, -1 for a row that is left out
    const float* lse;      // backward: R
    const float* scal;     // device: [0] rows with a target, [1] dloss / rows (0 when there is none)
    int* err;              // raised by a wait that gives up
    int ncounters;         // tile counters that the call needs
    int* ticket;           // words that start at 0
    unsigned* largest;     // f32 on the tensor cores: largest finite magnitude of w and of x, as bits
    int* counters;
    float2* parts;         // forward: (maximum, sum of exponentials) of row r over slice p at [p * R + r]
    float* tz;             // forward: logit of the target
    int nparts;
    void* dw;              // backward: [D][V] in dtype
    float* dbias;          // V or NULL
    void* dx;              // [R][D] in dtype
};

// Running maximum and sum of exponentials of a softmax row.  m = -inf, s = 0 is the empty row.
struct lce_ms {
    float m, s;
};
__device__ __forceinline__ lce_ms lce_merge(lce_ms a, lce_ms b) {
    const float m = fmaxf(a.m, b.m);
    const float ref = m == -INFINITY ? 0.f : m;  // rows of -inf only: exp(-inf - 0) = 0, the sum stays 0
    return {m, a.s * expf(a.m - ref) + b.s * expf(b.m - ref)};
}

// out[i] = scale * sum over p of parts[p][i] (dx, or dw; i < count, which may be 0), fixed order; and, where dbias is given,
// dbias[c] = scale * sum over p of dbparts[p][c], c < cols (rows dbpitch apart).  tgt (NULL for dw): the rows of D values without
// a target are 0 whatever the scale is.
void lce_finish_launch(rg_ctx* ctx, const float* parts, int nparts, size_t count, const float* scal, const int* tgt, int D, void* out, int dtype,
                          const float* dbparts, int dbrows, int dbpitch, int cols, float* dbias);

// The tensor-core form.
rg_status lce_tc_forward(rg_ctx* ctx, lce_call& c);
rg_status lce_tc_backward(rg_ctx* ctx, lce_call& c);
int lce_tc_nparts(rg_ctx* ctx, const lce_call& c);
int lce_tc_backward_launches(const lce_call& c);

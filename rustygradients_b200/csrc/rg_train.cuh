// What the training ops share on the host side.
#pragma once
#include "rg_internal.cuh"

// Outputs (and scratch) of an op while it is being enqueued: whatever has not been given to the caller is deleted, in
// stream order, when the op returns - on its error paths as on success.  The context's lock is held.
template <int N>
struct rg_outputs {
    rg_storage* p[N] = {};
    rg_storage*& operator[](int i) { return p[i]; }
    void give(std::initializer_list<rg_storage**> to) {
        int i = 0;
        for (rg_storage** t : to) *t = p[i], p[i] = nullptr, i++;
    }
    ~rg_outputs() {
        for (rg_storage* s : p) delete s;
    }
};

// These ops allocate from the stream-ordered pool and some of them wait for a check of their arguments, which a capture
// would turn into nodes of a graph or refuse in its middle.
static inline rg_status rg_not_capturing(rg_ctx* ctx, const char* op) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    const cudaError_t e = cudaStreamIsCapturing(ctx->stream, &cs);
    if (e == cudaSuccess && cs == cudaStreamCaptureStatusNone) return RG_OK;
    cudaGetLastError();
    return rg_fail(RG_ERR_UNSUPPORTED, "%s is not enqueued into a stream capture", op);
}

// out0[c] (c < split) and out1[c - split]: sums over the rows of parts [nparts][cols], in a fixed order.
void rg_colsum_launch(rg_ctx* ctx, const float* parts, int nparts, long long cols, float* out0, float* out1, long long split);

// Softmax cross entropy of a vocabulary projection without its logits (rg_b200.h: rg_linear_cross_entropy and its
// gradient): the entry points, the check of the targets, the final sums, and the form for few rows.
//
//   z = x w + bias,  lse_r = log sum_v exp z_rv,  loss = mean over rows with a target of (lse_r - z_{r,t})
//   dz = (exp(z - lse) - onehot) dloss / n,  dx = dz w^T,  dw = x^T dz,  dbias = sum_r dz
//
// The logits exist a tile at a time: the forward pass keeps (maximum, sum of exponentials) per row and slice of the
// vocabulary, the backward pass computes them once more from x, w and the saved lse.
#include "rg_lce.cuh"
#include "rg_lce_plan.h"

#include <algorithm>

// ---------------------------------------------------------------------------
// targets
// ---------------------------------------------------------------------------
// Ids are carried as f32 and truncated like the other index inputs.  One CTA: the rows with a target are counted, the number
// of bad ones goes to the host with the number of the call, and what the later kernels of the call need is set up.
__global__ void __launch_bounds__(1024) lce_check_kernel(const float* __restrict__ targets, int R, int V, long long ignore,
                                                         const float* __restrict__ dloss, int* __restrict__ tgt, float* __restrict__ tz,
                                                         float* __restrict__ scal, int* __restrict__ zero, int nzero,
                                                         volatile unsigned long long* host, unsigned call) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ int live_s, bad_s;
    if (threadIdx.x == 0) live_s = bad_s = 0;
    for (int i = threadIdx.x; i < nzero; i += 1024) zero[i] = 0;
    __syncthreads();
    int live = 0, bad = 0;
#pragma unroll 4
    for (int r = threadIdx.x; r < R; r += 1024) {
        const float f = targets[r];
        const bool number = fabsf(f) < 9e15f;  // not NaN, fits an integer
        const long long t = number ? (long long)f : -1;
        int v = -1;
        if (number && t == ignore) v = -1;
        else if (!number || f < 0.f || t >= V) bad++;
        else v = (int)t, live++;
        tgt[r] = v;
        if (tz) tz[r] = 0.f;
    }
    atomicAdd(&live_s, live);  // whole numbers: the order does not matter
    atomicAdd(&bad_s, bad);
    __syncthreads();
    if (threadIdx.x == 0) {
        scal[0] = (float)live_s;
        scal[1] = live_s ? (dloss ? dloss[0] : 1.f) / (float)live_s : 0.f;
        *host = (unsigned long long)call << 32 | (unsigned)bad_s;
    }
}

// lse of 8 rows per CTA: 32 threads share the slices of a row, lanes of 8 rows read 64 contiguous bytes.  The maximum of
// all slices comes first, so the sum is one exponential per slice with no chain between them.  Then the loss: the sum of a
// CTA's rows in f64; the last CTA to finish adds the CTAs in order and divides.
__global__ void __launch_bounds__(256) lce_loss_kernel(const float2* parts, int nparts, int R, const int* tgt, const float* tz,
                                                       const float* scal, int* ticket, double* sums, float* __restrict__ lse_out,
                                                       float* __restrict__ loss) {
    __shared__ float red[32][9];
    __shared__ double rows_s[8];
    __shared__ bool last;
    rg_pdl_sync();
    const int row = threadIdx.x & 7, slice = threadIdx.x >> 3;
    const int r = blockIdx.x * 8 + row;
    // the first 16 slices of a thread stay in registers (all of them up to a vocabulary of 65536)
    float2 v[16];
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++) {
        const int p = slice + 32 * k;
        v[k] = (r < R && p < nparts) ? parts[(size_t)p * R + r] : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int k = 0; k < 16; k++) m = fmaxf(m, v[k].x);
    if (r < R)
        for (int p = slice + 512; p < nparts; p += 32) m = fmaxf(m, parts[(size_t)p * R + r].x);
    red[slice][row] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; k++) m = fmaxf(m, red[k][row]);
    const float ref = m == -INFINITY ? 0.f : m;  // a row of -inf only: every term below is 0
#pragma unroll
    for (int k = 0; k < 16; k++) s += v[k].y * expf(v[k].x - ref);
    if (r < R)
        for (int p = slice + 512; p < nparts; p += 32) {
            const float2 q = parts[(size_t)p * R + r];
            s += q.y * expf(q.x - ref);
        }
    __syncthreads();
    red[slice][row] = s;
    __syncthreads();
    if (threadIdx.x < 8) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; k++) s += red[k][row];
        double off = 0.0;
        if (r < R) {
            const float lse = m + logf(s);
            lse_out[r] = lse;
            if (tgt[r] >= 0) off = (double)lse - (double)tz[r];
        }
        rows_s[row] = off;
        __syncwarp(0xff);
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int k = 0; k < 8; k++) t += rows_s[k];
            sums[blockIdx.x] = t;
            __threadfence();
            last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    __shared__ double tot[256];
    double t = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) t += __ldcg(sums + i);
    tot[threadIdx.x] = t;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) tot[threadIdx.x] += tot[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) loss[0] = scal[0] > 0.f ? (float)(tot[0] / (double)scal[0]) : 0.f;
}

// The final sums of the gradient: the first `xblocks` blocks those of dx (or dw), the others 32 columns of dbias each, eight
// warps sharing the partials.  (A launch of its own for dbias cost 3 us.)
template <typename T, int VEC>
__global__ void __launch_bounds__(256) lce_finish_kernel(const float* parts, int nparts, size_t count, const float* scal, const int* tgt, int D,
                                                         T* __restrict__ dx, int xblocks, const float* dbparts, int dbrows, int dbpitch,
                                                         int cols, float* __restrict__ dbias) {
    __shared__ float red[8][32];
    rg_pdl_sync();
    const float scale = scal[1];
    if ((int)blockIdx.x >= xblocks) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        const int c = ((int)blockIdx.x - xblocks) * 32 + lane;
        float s = 0.f;
        if (c < cols)
#pragma unroll 8
            for (int p = w; p < dbrows; p += 8) s += dbparts[(size_t)p * dbpitch + c];
        red[w][lane] = s;
        __syncthreads();
        if (w || c >= cols) return;
#pragma unroll
        for (int k = 1; k < 8; k++) s += red[k][lane];
        dbias[c] = s * scale;
        return;
    }
    // an upstream gradient that overflowed reaches the rows with a target only
    const bool rows = tgt && !(fabsf(scale) <= 3.4028235e38f);
    auto scaled = [&](float v, size_t at) { return rows && tgt[at / D] < 0 ? 0.f : v * scale; };
    const size_t stride = (size_t)xblocks * 256 * VEC;
    for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * VEC; i < count; i += stride) {
        if constexpr (VEC == 4) {
            float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int z = 0; z < nparts; z++) {
                const float4 q = *reinterpret_cast<const float4*>(parts + (size_t)z * count + i);
                t.x += q.x, t.y += q.y, t.z += q.z, t.w += q.w;
            }
            const float v[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int k = 0; k < 4; k++) dx[i + k] = rg_from_float<T>(scaled(v[k], i + k));
        } else {
            dx[i] = rg_from_float<T>(scaled(rg_sum_parts(parts + i, nparts, count), i));
        }
    }
}
template <typename T>
static void lce_finish_typed(rg_ctx* ctx, const float* parts, int nparts, size_t count, const float* scal, const int* tgt, int D, T* dx,
                             const float* dbparts,
                             int dbrows, int dbpitch, int cols, float* dbias) {
    // four values a thread where every partial starts on a 16-byte boundary and there are threads enough (768 values and 50
    // partials: 15 us against 6; 6.5 million values and one partial: 9 us against 26)
    const bool vec = count % 4 == 0 && count >= ((size_t)1 << 19);
    const int xblocks = (int)std::min<size_t>((count + (vec ? 1023 : 255)) / (vec ? 1024 : 256), (size_t)ctx->sm_count * 16);
    rg_launch(true, vec ? lce_finish_kernel<T, 4> : lce_finish_kernel<T, 1>, dim3((unsigned)(xblocks + (dbias ? rg_cdiv(cols, 32) : 0))), dim3(256),
              0, ctx->stream, parts, nparts, count, scal, tgt, D, dx, xblocks, dbparts, dbrows, dbpitch, cols, dbias);
    RG_LAUNCHED(ctx);
}
void lce_finish_launch(rg_ctx* ctx, const float* parts, int nparts, size_t count, const float* scal, const int* tgt, int D, void* out, int dtype,
                          const float* dbparts, int dbrows, int dbpitch, int cols, float* dbias) {
    if (dtype == RG_DTYPE_F32) lce_finish_typed(ctx, parts, nparts, count, scal, tgt, D, (float*)out, dbparts, dbrows, dbpitch, cols, dbias);
    else lce_finish_typed(ctx, parts, nparts, count, scal, tgt, D, (__nv_bfloat16*)out, dbparts, dbrows, dbpitch, cols, dbias);
}

// ---------------------------------------------------------------------------
// few rows: w is read once (twice in the gradient) by coalesced loads, the products are f32 FMAs
// ---------------------------------------------------------------------------
// Four values of a row of w are one load, although rows of an odd vocabulary start anywhere: warp q takes rows q, q + 8, ...,
// all of which start at the same offset from an aligned address, and shifts its columns by it.  A tile is 124 columns, so
// that the 128 a warp reads cover it for every shift; what it reads outside belongs to columns whose sums are not used.
template <typename T>
struct lce_four;
template <>
struct lce_four<float> { typedef float4 type; };
template <>
struct lce_four<__nv_bfloat16> { typedef uint2 type; };

// w[at .. at + 3], at a multiple of 4; zeros beyond the matrix
template <typename T>
__device__ __forceinline__ void lce_load4(const T* __restrict__ w, size_t at, size_t total, float (&v)[4]) {
    typedef typename lce_four<T>::type F;
    if (at + 4 <= total) {
        const F raw = *reinterpret_cast<const F*>(w + at);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = rg_to_float(e[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = at + k < total ? rg_to_float(w[at + k]) : 0.f;
    }
}

// RB values from shared memory, as wide as they are aligned
template <int RB>
__device__ __forceinline__ void lce_rows(const float* p, float (&v)[RB]) {
    if constexpr (RB >= 4) {
#pragma unroll
        for (int r = 0; r < RB; r += 4) {
            const float4 q = *reinterpret_cast<const float4*>(p + r);
            v[r] = q.x, v[r + 1] = q.y, v[r + 2] = q.z, v[r + 3] = q.w;
        }
    } else if constexpr (RB == 2) {
        const float2 q = *reinterpret_cast<const float2*>(p);
        v[0] = q.x, v[1] = q.y;
    } else {
        v[0] = *p;
    }
}

#define LCE_COLS 124
template <typename T, int RB>
struct lce_few {
    static constexpr int PAIRS = (RB + 1) / 2;
    static constexpr int DC = RB == 16 ? 512 : 1024;     // rows of w between two refills of x
    static constexpr int AHEAD = 32 / (int)sizeof(T);     // rows of w a warp has on their way: 4 KB
    static constexpr int RING = 8 * AHEAD * 128 * (int)sizeof(T), X = DC * RB * 4, SUMS = 8 * RB * 128 * 4;
    static constexpr size_t SMEM = RING + X > SUMS ? RING + X : SUMS;
};

// z[k][j]: logit of row warp + 8 k and column lane + 32 j of the tile (-inf outside).  The 8 warps share the D axis.  Each lane
// copies its four values of the warp's next rows of w asynchronously into a ring of its own in shared memory (kept in
// registers they left too few warps: 3.5 TB/s), and multiplies them with the RB values of x, which lie in shared memory as
// [d][row]: one or a few broadcast loads.  Rows of x are multiplied two at a time.  [8,768] x [768,50257] f32: 38 us, 4.0 TB/s, DRAM
// active 46 %.  Neither the bytes nor the strips of 512 of them bound it: a kernel that only adds up the same strips takes 24 to
// 26 us (6.0 to 6.4 TB/s).  What is left are the instructions of a row of w in each warp (16 paired multiplications, three shared
// loads, a copy, its commit and its wait); 16 rows: 64 us.
template <typename T, int RB>
__device__ __forceinline__ void lce_few_logits(const lce_call& c, unsigned char* sm, float (&z)[RB / 8 > 0 ? RB / 8 : 1][4]) {
    typedef lce_few<T, RB> F;
    typedef typename lce_four<T>::type V4;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c0 = blockIdx.x * LCE_COLS, shift = lce_few_shift(c.V, w);
    // lanes beyond the row read its last aligned place again: their sums are not used
    const int col0 = min(c0 - shift + 4 * lane, lce_few_last(c.V, shift));
    const size_t total = (size_t)c.D * c.V, step = (size_t)8 * c.V;
    const T* x = static_cast<const T*>(c.x);
    const T* wt = static_cast<const T*>(c.w);
    V4* ring = reinterpret_cast<V4*>(sm) + w * F::AHEAD * 32 + lane;
    float* xs = reinterpret_cast<float*>(sm + F::RING);
    float2 acc[F::PAIRS][4];  // rows 2 i and 2 i + 1 of column j
#pragma unroll
    for (int i = 0; i < F::PAIRS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = make_float2(0.f, 0.f);
    // this warp's rows of w: w, w + 8, ...; those at the end of the matrix are read with a guard
    const int rows = (c.D - w + 7) / 8, safe = lce_few_safe(c.D, c.V, w);
    const T* from = wt + (size_t)w * c.V + col0;
    auto copy = [&](int k) {
        if (k < safe) {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + (k % F::AHEAD) * 32);
            if constexpr (sizeof(V4) == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from + (size_t)k * step) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from + (size_t)k * step) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < F::AHEAD - 1; k++) copy(k);
    for (int d0 = 0; d0 < c.D; d0 += F::DC) {
        const int dn = min(F::DC, c.D - d0), k1 = min(rows, (d0 + F::DC) / 8);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll 2
            for (int d = threadIdx.x; d < dn; d += 256) xs[d * RB + r] = r < c.R ? rg_to_float(x[(size_t)r * c.D + d0 + d]) : 0.f;
        __syncthreads();
#pragma unroll 4
        for (int k = d0 / 8; k < k1; k++) {
            copy(k + F::AHEAD - 1);  // into the slot that was read in the turn before
            asm volatile("cp.async.wait_group %0;" ::"n"(F::AHEAD - 1) : "memory");
            float wv[4];
            if (k < safe) {
                const V4 raw = ring[(k % F::AHEAD) * 32];
                const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
                for (int j = 0; j < 4; j++) wv[j] = rg_to_float(e[j]);
            } else {
                lce_load4(wt, (size_t)(w + 8 * k) * c.V + col0, total, wv);
            }
            float xv[RB];
            lce_rows<RB>(xs + (w + 8 * k - d0) * RB, xv);
#pragma unroll
            for (int i = 0; i < F::PAIRS; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (RB == 1) acc[0][j].x = fmaf(xv[0], wv[j], acc[0][j].x);
                    else acc[i][j] = rg_fma2(make_float2(xv[2 * i], xv[2 * i + 1]), make_float2(wv[j], wv[j]), acc[i][j]);
                }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    float* sums = reinterpret_cast<float*>(sm);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int col = 4 * lane + j - shift;
            if (col >= 0 && c0 + col < c.V) sums[(w * RB + r) * 128 + col] = r % 2 ? acc[r / 2][j].y : acc[r / 2][j].x;
        }
    __syncthreads();
    // warp w takes rows w, w + 8, ...: the sum over the 8 slices of D, then the bias
#pragma unroll
    for (int k = 0; k < (RB / 8 > 0 ? RB / 8 : 1); k++) {
        const int r = w + 8 * k;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int col = lane + 32 * j;
            const bool in = col < LCE_COLS && c0 + col < c.V;
            float t = 0.f;
            if (r < RB && in)
#pragma unroll
                for (int q = 0; q < 8; q++) t += sums[(q * RB + r) * 128 + col];
            z[k][j] = in ? t + (c.bias ? c.bias[c0 + col] : 0.f) : -INFINITY;
        }
    }
}

template <typename T, int RB>
__global__ void __launch_bounds__(256, RB <= 4 ? 4 : RB <= 8 ? 3 : 2) lce_few_fwd_kernel(const lce_call c) {
    extern __shared__ __align__(16) unsigned char lce_sm[];
    float z[RB / 8 > 0 ? RB / 8 : 1][4];
    lce_few_logits<T, RB>(c, lce_sm, z);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the targets; x and w were there before
#pragma unroll
    for (int k = 0; k < (RB / 8 > 0 ? RB / 8 : 1); k++) {
        const int r = w + 8 * k;
        if (r >= c.R || r >= RB) continue;  // whole warps
        const int t = c.tgt[r] - (int)blockIdx.x * LCE_COLS;
        float m = fmaxf(fmaxf(z[k][0], z[k][1]), fmaxf(z[k][2], z[k][3]));
        m = rg_warp_max(m);
        const float ref = m == -INFINITY ? 0.f : m;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s += expf(z[k][j] - ref);
            if (t == lane + 32 * j && t < LCE_COLS) c.tz[r] = z[k][j];
        }
        s = rg_warp_sum(s);
        if (lane == 0) c.parts[(size_t)blockIdx.x * c.R + r] = make_float2(m, s);
    }
}

// dz (without the common factor dloss / n) of all rows, f32 [R][V], and the bias gradient
template <typename T, int RB>
__global__ void __launch_bounds__(256, RB <= 4 ? 4 : RB <= 8 ? 3 : 2) lce_few_dz_kernel(const lce_call c, float* __restrict__ dz) {
    extern __shared__ __align__(16) unsigned char lce_sm[];
    float z[RB / 8 > 0 ? RB / 8 : 1][4];
    lce_few_logits<T, RB>(c, lce_sm, z);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c0 = (int)blockIdx.x * LCE_COLS;
    float* sm = reinterpret_cast<float*>(lce_sm);
    float col[4] = {0.f, 0.f, 0.f, 0.f};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the targets; x and w were there before
    {
#pragma unroll
        for (int k = 0; k < (RB / 8 > 0 ? RB / 8 : 1); k++) {
            const int r = w + 8 * k;
            if (r >= c.R || r >= RB) continue;
            const int t = c.tgt[r];
            const float lse = c.lse[r];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int v = c0 + lane + 32 * j;
                if (lane + 32 * j < LCE_COLS && v < c.V) {
                    const float p = t < 0 ? 0.f : expf(z[k][j] - lse) - (v == t ? 1.f : 0.f);
                    dz[(size_t)r * c.V + v] = p;
                    col[j] += p;
                }
            }
        }
    }
    if (!c.dbias) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) sm[w * 128 + lane + 32 * j] = col[j];
    __syncthreads();
    if (threadIdx.x < LCE_COLS && c0 + (int)threadIdx.x < c.V) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; q++) s += sm[q * 128 + threadIdx.x];
        c.dbias[c0 + threadIdx.x] = s * c.scal[1];
    }
}

// dw and partial dx.  A warp has 128 columns (lane + 32 j), a CTA 1024, and walks LCE_DG rows of w: a thread holds dz of RB
// rows and 4 columns in registers, each value of w is one load, each of dw one store.  The RB products with dz are summed
// over the warp by halving exchanges (each adds two rows at once, so RB rows cost RB shuffles plus the steps left), over the
// 8 warps in shared memory.  (Four-value loads with shifted columns, as above, need their own dz per shift: slower.)  w in, dw
// out: 81 us for 8 rows of [768,50257] f32, 3.8 TB/s; 128 us for 16, bound by the exchanges.
#define LCE_DG 32
template <typename T, int RB>
__global__ void __launch_bounds__(256) lce_few_grad_kernel(const lce_call c, const float* dz, float* __restrict__ dxparts) {
    constexpr int PAIRS = (RB + 1) / 2;
    __shared__ __align__(16) float xs[LCE_DG][RB];
    __shared__ float dxs[8][LCE_DG][RB];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c0 = (int)blockIdx.x * 1024 + w * 128 + lane;
    const int d0 = (int)blockIdx.y * LCE_DG, dn = min(LCE_DG, c.D - d0);
    const T* x = static_cast<const T*>(c.x);
    const T* wt = static_cast<const T*>(c.w) + (size_t)d0 * c.V + c0;
    T* dw = static_cast<T*>(c.dw) + (size_t)d0 * c.V + c0;
    rg_pdl_sync();
    const float scale = c.scal[1];
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; j++) in[j] = c0 + 32 * j < c.V;
    for (int i = threadIdx.x; i < LCE_DG * RB; i += 256) {
        const int r = i / LCE_DG, d = i % LCE_DG;
        xs[d][r] = (r < c.R && d < dn) ? rg_to_float(x[(size_t)r * c.D + d0 + d]) : 0.f;
    }
    float2 g[PAIRS][4];
#pragma unroll
    for (int i = 0; i < PAIRS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            g[i][j].x = (2 * i < c.R && in[j]) ? dz[(size_t)(2 * i) * c.V + c0 + 32 * j] : 0.f;
            g[i][j].y = (2 * i + 1 < c.R && in[j]) ? dz[(size_t)(2 * i + 1) * c.V + c0 + 32 * j] : 0.f;
        }
    T next[4];
#pragma unroll
    for (int j = 0; j < 4; j++) next[j] = in[j] ? wt[32 * j] : rg_from_float<T>(0.f);
    __syncthreads();
#pragma unroll 2
    for (int d = 0; d < dn; d++, wt += c.V, dw += c.V) {
        float wv[4];
        float2 o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) wv[j] = rg_to_float(next[j]), o[j] = make_float2(0.f, 0.f);
        if (d + 1 < dn)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (in[j]) next[j] = wt[c.V + 32 * j];
        float xv[RB], q[2 * PAIRS];
        lce_rows<RB>(xs[d], xv);
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            const float2 xp = make_float2(xv[2 * i], RB > 1 ? xv[RB > 1 ? 2 * i + 1 : 0] : 0.f);
            float2 s = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[j] = rg_fma2(xp, g[i][j], o[j]);
                s = rg_fma2(g[i][j], make_float2(wv[j], wv[j]), s);
            }
            q[2 * i] = s.x, q[2 * i + 1] = s.y;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (in[j]) dw[32 * j] = rg_from_float<T>((o[j].x + o[j].y) * scale);
        // after the exchanges lane l holds row l / (32 / RB), summed over the lanes that share it
        int half = 16;
#pragma unroll
        for (int n = RB / 2; n >= 1; n >>= 1, half >>= 1) {
            const bool up = lane & half;
#pragma unroll
            for (int i = 0; i < n; i++) {
                const float keep = up ? q[i + n] : q[i], send = up ? q[i] : q[i + n];
                q[i] = keep + __shfl_xor_sync(RG_FULL_MASK, send, half);
            }
        }
        float s = q[0];
#pragma unroll
        for (int o2 = 16 / RB; o2 > 0; o2 >>= 1) s += __shfl_xor_sync(RG_FULL_MASK, s, o2);
        if (lane % (32 / RB) == 0) dxs[w][d][lane / (32 / RB)] = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < dn * RB; i += 256) {
        const int d = i % dn, r = i / dn;
        if (r >= c.R) continue;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) s += dxs[k][d][r];
        dxparts[((size_t)blockIdx.x * c.R + r) * c.D + d0 + d] = s;
    }
}

// The form for few rows, by what was measured at [R,768] x [768,50257] (us for the call; the other side for the same rows; no
// other width and vocabulary was measured, and with a few hundred classes this form has only as many CTAs as 124 go into them):
//   forward   f32  8 rows 46, the tensor cores 57;  9 rows 67 and 55
//             bf16 V aligned: 2 rows 34, the tensor cores 38; 3 rows 37 and 37
//             bf16 V odd: the tensor cores, 34 for 1 to 16 rows (34 for 1, 38 for 4, 47 for 8 rows here)
//   gradient  f32  16 rows 203, the tensor cores 227
//             bf16 V aligned: 4 rows 98, the tensor cores 107; 8 rows 121
//             bf16 V odd: 8 rows 120, the tensor cores 135; 9 rows 184
static bool lce_is_few(const lce_call& c, bool grad) {
    if (c.dtype == RG_DTYPE_F32) return c.R <= (grad ? 16 : 8);
    if (c.V % 8 == 0) return c.R <= (grad ? 4 : 2);
    return grad && c.R <= 8;
}

static int lce_few_tiles(int V) { return rg_cdiv(V, LCE_COLS); }
static int lce_few_parts(int V) { return rg_cdiv(V, 1024); }

template <typename T, int RB>
static void lce_few_fwd_launch(rg_ctx* ctx, const lce_call& c) {
    const size_t smem = lce_few<T, RB>::SMEM;
    if (smem > 48 * 1024) cudaFuncSetAttribute(lce_few_fwd_kernel<T, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    // starts while the check of the targets runs and waits for it before it uses them
    rg_launch(true, lce_few_fwd_kernel<T, RB>, dim3((unsigned)lce_few_tiles(c.V)), dim3(256), smem, ctx->stream, c);
    RG_LAUNCHED(ctx);
}
template <typename T, int RB>
static void lce_few_bwd_launch(rg_ctx* ctx, const lce_call& c, float* dz, float* dxparts) {
    const size_t smem = lce_few<T, RB>::SMEM;
    if (smem > 48 * 1024) cudaFuncSetAttribute(lce_few_dz_kernel<T, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    rg_launch(true, lce_few_dz_kernel<T, RB>, dim3((unsigned)lce_few_tiles(c.V)), dim3(256), smem, ctx->stream, c, dz);
    rg_launch(true, lce_few_grad_kernel<T, RB>, dim3((unsigned)lce_few_parts(c.V), (unsigned)rg_cdiv(c.D, LCE_DG)), dim3(256), 0, ctx->stream, c,
              (const float*)dz, dxparts);
    ctx->launches += 2;
}
// the rows of lce_is_few
static void lce_few_forward(rg_ctx* ctx, const lce_call& c) {
    if (c.dtype == RG_DTYPE_F32) {
        if (c.R <= 1) lce_few_fwd_launch<float, 1>(ctx, c);
        else if (c.R <= 2) lce_few_fwd_launch<float, 2>(ctx, c);
        else if (c.R <= 4) lce_few_fwd_launch<float, 4>(ctx, c);
        else lce_few_fwd_launch<float, 8>(ctx, c);
    } else {
        if (c.R <= 1) lce_few_fwd_launch<__nv_bfloat16, 1>(ctx, c);
        else lce_few_fwd_launch<__nv_bfloat16, 2>(ctx, c);
    }
}
static void lce_few_backward(rg_ctx* ctx, const lce_call& c, float* dz, float* dxparts) {
    if (c.dtype == RG_DTYPE_F32) {
        if (c.R <= 1) lce_few_bwd_launch<float, 1>(ctx, c, dz, dxparts);
        else if (c.R <= 2) lce_few_bwd_launch<float, 2>(ctx, c, dz, dxparts);
        else if (c.R <= 4) lce_few_bwd_launch<float, 4>(ctx, c, dz, dxparts);
        else if (c.R <= 8) lce_few_bwd_launch<float, 8>(ctx, c, dz, dxparts);
        else lce_few_bwd_launch<float, 16>(ctx, c, dz, dxparts);
    } else {
        if (c.R <= 1) lce_few_bwd_launch<__nv_bfloat16, 1>(ctx, c, dz, dxparts);
        else if (c.R <= 2) lce_few_bwd_launch<__nv_bfloat16, 2>(ctx, c, dz, dxparts);
        else if (c.R <= 4) lce_few_bwd_launch<__nv_bfloat16, 4>(ctx, c, dz, dxparts);
        else lce_few_bwd_launch<__nv_bfloat16, 8>(ctx, c, dz, dxparts);
    }
}

// ---------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------
static rg_status lce_args(const char* op, rg_ctx* ctx, const rg_storage* x, const rg_storage* w, const rg_storage* bias,
                          const rg_storage* targets, lce_call* c) {
    if (x->shape.size() != 2 || w->shape.size() != 2)
        return rg_fail(RG_ERR_DIMENSION, "%s: x and w are 2D, got %zuD and %zuD", op, x->shape.size(), w->shape.size());
    if (x->shape[1] != w->shape[0])
        return rg_fail(RG_ERR_SHAPE, "Incompatible shapes for 2D dot product: [%zu, %zu] and [%zu, %zu]", x->shape[0], x->shape[1],
                       w->shape[0], w->shape[1]);
    if (x->dtype != w->dtype) return rg_fail(RG_ERR_UNSUPPORTED, "%s: x and w have different types", op);
    const size_t R = x->shape[0], D = x->shape[1], V = w->shape[1];
    if (!D || !V) return rg_fail(RG_ERR_SHAPE, "%s: a projection of [%zu, %zu]", op, D, V);
    if (R > (1u << 24) || D > (1u << 20) || V > (1u << 24))  // ids above 2^24 are not exact in f32
        return rg_fail(RG_ERR_SHAPE, "%s: %zu rows, %zu columns, %zu classes are beyond the limits 2^24, 2^20, 2^24", op, R, D, V);
    if (targets->len != R) return rg_fail(RG_ERR_SHAPE, "targets hold %zu elements for %zu rows", targets->len, R);
    RG_TRY(rg_need_f32("targets and bias", targets, bias));
    if (bias && bias->len != V) return rg_fail(RG_ERR_SHAPE, "bias holds %zu elements for %zu classes", bias->len, V);
    RG_TRY(rg_not_capturing(ctx, op));
    memset(c, 0, sizeof(*c));
    c->err = ctx->d_flag + 1;
    c->R = (int)R, c->D = (int)D, c->V = (int)V, c->dtype = x->dtype;
    c->x = x->raw(), c->w = w->raw(), c->bias = bias ? bias->data() : nullptr;
    return RG_OK;
}

// Enqueues the check of the targets; lce_checked waits for its answer (not for what was enqueued after it).
static rg_status lce_check_launch(rg_ctx* ctx, lce_call& c, const rg_storage* targets, long long ignore, const rg_storage* dloss,
                                  rg_storage** scratch) {
    // tgt [R] | tz [R] | scal [2] | words that start at 0
    const int nzero = 3 + c.ncounters;
    const size_t words = 2 * (size_t)c.R + 2 + nzero;
    RG_TRY(rg_alloc_storage(ctx, &words, 1, scratch));
    float* base = (*scratch)->data();
    c.tgt = reinterpret_cast<int*>(base), c.tz = base + c.R, c.scal = base + 2 * (size_t)c.R;
    c.ticket = reinterpret_cast<int*>(base + 2 * (size_t)c.R + 2);
    c.largest = reinterpret_cast<unsigned*>(base + 2 * (size_t)c.R + 3);
    c.counters = reinterpret_cast<int*>(base + 2 * (size_t)c.R + 5);
    lce_check_kernel<<<1, 1024, 0, ctx->stream>>>(targets->data(), c.R, c.V, ignore, dloss ? dloss->data() : nullptr,
                                                  const_cast<int*>(c.tgt), c.tz, const_cast<float*>(c.scal), c.ticket, nzero, ctx->h_check,
                                                  ++ctx->check_no);
    RG_LAUNCHED(ctx);
    RG_CUDA(cudaGetLastError());
    return RG_OK;
}
static rg_status lce_checked(rg_ctx* ctx, const lce_call& c) {
    unsigned long long v;
    for (unsigned spins = 1; (unsigned)((v = *ctx->h_check) >> 32) != ctx->check_no; spins++) {
        if (spins % 65536) continue;
        const cudaError_t e = cudaStreamQuery(ctx->stream);  // a stream that failed never answers
        if (e == cudaErrorNotReady) continue;
        if (e == cudaSuccess && (unsigned)(*ctx->h_check >> 32) == ctx->check_no) continue;
        return rg_fail(RG_ERR_BACKEND, "linear_cross_entropy: %s", cudaGetErrorString(e));
    }
    if ((unsigned)v) return rg_fail(RG_ERR_SHAPE, "Target index out of bounds for %d classes", c.V);
    return RG_OK;
}

extern "C" rg_status rg_linear_cross_entropy(rg_ctx* ctx, const rg_storage* x, const rg_storage* w, const rg_storage* bias,
                                             const rg_storage* targets, int64_t ignore_index, rg_storage** loss, rg_storage** lse) {
    if (!ctx || !x || !w || !targets || !loss || !lse) return rg_fail(RG_ERR_INVALID_INPUT, "NULL argument");
    *loss = *lse = nullptr;
    RG_TRY(rg_same_ctx(ctx, {x, w, bias, targets}));
    rg_op_guard g(ctx);
    lce_call c;
    RG_TRY(lce_args("linear_cross_entropy", ctx, x, w, bias, targets, &c));
    const size_t one = 1, rows = (size_t)c.R;
    rg_outputs<5> o;  // loss, lse, scratch of the check, partials, sums
    RG_TRY(rg_alloc_storage(ctx, &one, 1, &o[0]));
    RG_TRY(rg_alloc_storage(ctx, &rows, 1, &o[1]));
    if (!c.R) {
        RG_CUDA(cudaMemsetAsync(o[0]->raw(), 0, 4, ctx->stream));
        o.give({loss, lse});
        return RG_OK;
    }
    const bool few = lce_is_few(c, false);
    c.ncounters = few ? 0 : 1;
    RG_TRY(lce_check_launch(ctx, c, targets, ignore_index, nullptr, &o[2]));
    c.nparts = few ? lce_few_tiles(c.V) : lce_tc_nparts(ctx, c);
    const size_t pwords = 2 * (size_t)c.nparts * rows, blocks = (size_t)rg_cdiv(c.R, 8), swords = 2 * blocks;
    RG_TRY(rg_alloc_storage(ctx, &pwords, 1, &o[3]));
    RG_TRY(rg_alloc_storage(ctx, &swords, 1, &o[4]));
    c.parts = static_cast<float2*>(o[3]->raw());
    if (few) lce_few_forward(ctx, c);
    else RG_TRY(lce_tc_forward(ctx, c));
    rg_launch(true, lce_loss_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, (const float2*)c.parts, c.nparts, c.R, c.tgt,
              (const float*)c.tz, c.scal, c.ticket, static_cast<double*>(o[4]->raw()), o[1]->data(), o[0]->data());
    RG_LAUNCHED(ctx);
    RG_CUDA(cudaGetLastError());
    RG_TRY(lce_checked(ctx, c));
    o.give({loss, lse});
    return RG_OK;
}

extern "C" rg_status rg_linear_cross_entropy_bwd(rg_ctx* ctx, const rg_storage* x, const rg_storage* w, const rg_storage* bias,
                                                 const rg_storage* targets, int64_t ignore_index, const rg_storage* lse,
                                                 const rg_storage* dloss, rg_storage** dx, rg_storage** dw, rg_storage** dbias) {
    if (!ctx || !x || !w || !targets || !lse || !dx || !dw || (bias && !dbias)) return rg_fail(RG_ERR_INVALID_INPUT, "NULL argument");
    *dx = *dw = nullptr;
    if (dbias) *dbias = nullptr;
    RG_TRY(rg_same_ctx(ctx, {x, w, bias, targets, lse, dloss}));
    rg_op_guard g(ctx);
    lce_call c;
    RG_TRY(lce_args("linear_cross_entropy_bwd", ctx, x, w, bias, targets, &c));
    RG_TRY(rg_need_f32("lse and dloss", lse, dloss));
    if (lse->len != (size_t)c.R) return rg_fail(RG_ERR_SHAPE, "lse holds %zu elements for %d rows", lse->len, c.R);
    if (dloss && dloss->len != 1) return rg_fail(RG_ERR_SHAPE, "dloss holds %zu elements instead of 1", dloss->len);
    rg_outputs<6> o;  // dx, dw, dbias, scratch of the check, dz, partial dx
    RG_TRY(rg_alloc_storage(ctx, x->shape.data(), 2, &o[0], x->dtype));
    RG_TRY(rg_alloc_storage(ctx, w->shape.data(), 2, &o[1], w->dtype));
    if (bias) RG_TRY(rg_alloc_storage(ctx, bias->shape.data(), (int)bias->shape.size(), &o[2]));
    c.lse = lse->data(), c.dx = o[0]->raw(), c.dw = o[1]->raw(), c.dbias = bias ? o[2]->data() : nullptr;
    if (!c.R) {
        RG_CUDA(cudaMemsetAsync(o[1]->raw(), 0, o[1]->len * rg_dtype_size(o[1]->dtype), ctx->stream));
        if (bias) RG_CUDA(cudaMemsetAsync(o[2]->raw(), 0, o[2]->len * 4, ctx->stream));
    } else {
        const bool few = lce_is_few(c, true);
        c.ncounters = few ? 0 : lce_tc_backward_launches(c);
        RG_TRY(lce_check_launch(ctx, c, targets, ignore_index, dloss, &o[3]));
        if (few) {
            const size_t zlen = (size_t)c.R * c.V, nparts = (size_t)lce_few_parts(c.V), plen = nparts * c.R * c.D;
            RG_TRY(rg_alloc_storage(ctx, &zlen, 1, &o[4]));
            RG_TRY(rg_alloc_storage(ctx, &plen, 1, &o[5]));
            lce_few_backward(ctx, c, o[4]->data(), o[5]->data());
            lce_finish_launch(ctx, o[5]->data(), (int)nparts, (size_t)c.R * c.D, c.scal, c.tgt, c.D, c.dx, c.dtype, nullptr, 0, 0, 0,
                              nullptr);
        } else {
            RG_TRY(lce_tc_backward(ctx, c));
        }
        RG_CUDA(cudaGetLastError());
        RG_TRY(lce_checked(ctx, c));
    }
    if (dbias) o.give({dx, dw, dbias});
    else o.give({dx, dw});
    return RG_OK;
}

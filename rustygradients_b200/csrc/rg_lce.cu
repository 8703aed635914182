// Softmax cross entropy of a vocabulary projection without its logits (rg_b200.h: rg_linear_cross_entropy and its
// gradient): the entry points, the check of the targets, the final sums, and the form for few rows.
//
//   z = x w + bias,  lse_r = log sum_v exp z_rv,  loss = mean over rows with a target of (lse_r - z_{r,t})
//   dz = (exp(z - lse) - onehot) dloss / n,  dx = dz w^T,  dw = x^T dz,  dbias = sum_r dz
//
// The logits exist a tile at a time: the forward pass keeps (maximum, sum of exponentials) per row and slice of the
// vocabulary, the backward pass computes them once more from x, w and the saved lse.
#include "rg_lce.cuh"

#include <algorithm>

// ---------------------------------------------------------------------------
// targets
// ---------------------------------------------------------------------------
// Ids are carried as f32 and truncated like the other index inputs.  One CTA: the rows with a target are counted, the bad
// ones reported in status[0], and what the later kernels of the call need is set up.
__global__ void __launch_bounds__(1024) lce_check_kernel(const float* __restrict__ targets, int R, int V, long long ignore,
                                                         const float* __restrict__ dloss, int* __restrict__ tgt, float* __restrict__ tz,
                                                         float* __restrict__ scal, int* __restrict__ status) {
    __shared__ int live_s, bad_s;
    if (threadIdx.x == 0) live_s = bad_s = 0;
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
        status[0] = bad_s;
        status[1] = 0;  // ticket of lce_loss_kernel
        status[2] = 0;  // largest magnitude of w
    }
}

// lse of 8 rows per CTA: 32 threads share the slices of a row, lanes of 8 rows read 64 contiguous bytes.  The maximum of
// all slices comes first, so the sum is one exponential per slice with no chain between them.  Then the loss: the sum of a
// CTA's rows in f64; the last CTA to finish adds the CTAs in order and divides.
__global__ void __launch_bounds__(256) lce_loss_kernel(const float2* __restrict__ parts, int nparts, int R, const int* __restrict__ tgt,
                                                       const float* __restrict__ tz, const float* __restrict__ scal,
                                                       int* __restrict__ ticket, double* __restrict__ sums, float* __restrict__ lse_out,
                                                       float* __restrict__ loss) {
    __shared__ float red[32][9];
    __shared__ double rows_s[8];
    __shared__ bool last;
    const int row = threadIdx.x & 7, slice = threadIdx.x >> 3;
    const int r = blockIdx.x * 8 + row;
    const float2* mine = parts + (size_t)slice * R + r;
    float m = -INFINITY, s = 0.f;
    if (r < R)
#pragma unroll 8
        for (int p = slice; p < nparts; p += 32) m = fmaxf(m, parts[(size_t)p * R + r].x);
    red[slice][row] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; k++) m = fmaxf(m, red[k][row]);
    const float ref = m == -INFINITY ? 0.f : m;  // a row of -inf only: every term below is 0
    if (r < R)
#pragma unroll 8
        for (int p = slice; p < nparts; p += 32, mine += (size_t)32 * R) {
            const float2 v = *mine;
            s += v.y * expf(v.x - ref);
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

template <typename T>
__global__ void __launch_bounds__(256) lce_dx_finish_kernel(const float* __restrict__ parts, int nparts, size_t count,
                                                            const float* __restrict__ scal, T* __restrict__ dx) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    dx[i] = rg_from_float<T>(rg_sum_parts(parts + i, nparts, count) * scal[1]);
}
void lce_dx_finish_launch(rg_ctx* ctx, const float* parts, int nparts, size_t count, const float* scal, void* dx, int dtype) {
    const unsigned grid = (unsigned)((count + 255) / 256);
    if (dtype == RG_DTYPE_F32) lce_dx_finish_kernel<float><<<grid, 256, 0, ctx->stream>>>(parts, nparts, count, scal, (float*)dx);
    else lce_dx_finish_kernel<__nv_bfloat16><<<grid, 256, 0, ctx->stream>>>(parts, nparts, count, scal, (__nv_bfloat16*)dx);
    RG_LAUNCHED(ctx);
}

__global__ void __launch_bounds__(1024) lce_dbias_finish_kernel(const float* __restrict__ parts, int nparts, int V,
                                                                const float* __restrict__ scal, float* __restrict__ out) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < V)
        for (int p = w; p < nparts; p += 32) s += parts[(size_t)p * V + c];
    red[w][lane] = s;
    __syncthreads();
    s = rg_warp_sum(red[lane][w]);
    const int o = blockIdx.x * 32 + w;
    if (lane == 0 && o < V) out[o] = s * scal[1];
}
void lce_dbias_finish_launch(rg_ctx* ctx, const float* parts, int nparts, int V, const float* scal, float* dbias) {
    lce_dbias_finish_kernel<<<rg_cdiv(V, 32), 1024, 0, ctx->stream>>>(parts, nparts, V, scal, dbias);
    RG_LAUNCHED(ctx);
}

// ---------------------------------------------------------------------------
// few rows: w is read once (twice in the gradient) by coalesced loads, the products are f32 FMAs
// ---------------------------------------------------------------------------
// A CTA owns 128 columns, a lane the columns lane + 32 j: no alignment of the rows of w is needed.  Its 8 warps share the D
// axis and add their sums through shared memory.  x lies in shared memory as [d][row], so the RB values of one d are one or
// a few broadcast loads.
#define LCE_DC 1024  // rows of w between two refills of x
template <int RB>
constexpr size_t lce_few_smem() {
    return sizeof(float) * (LCE_DC * RB > 8 * RB * 128 ? LCE_DC * RB : 8 * RB * 128);
}

template <typename T, int RB>
__device__ __forceinline__ void lce_few_logits(const lce_call& c, float* sm, float (&z)[RB / 8 > 0 ? RB / 8 : 1][4]) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c0 = blockIdx.x * 128 + lane;
    const T* x = static_cast<const T*>(c.x);
    const T* wt = static_cast<const T*>(c.w);
    float acc[RB][4];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[r][j] = 0.f;
    for (int d0 = 0; d0 < c.D; d0 += LCE_DC) {
        const int dn = min(LCE_DC, c.D - d0);
        __syncthreads();
        for (int i = threadIdx.x; i < LCE_DC * RB; i += 256) {
            const int r = i / LCE_DC, d = i % LCE_DC;
            sm[d * RB + r] = (r < c.R && d < dn) ? rg_to_float(x[(size_t)r * c.D + d0 + d]) : 0.f;
        }
        __syncthreads();
#pragma unroll 4
        for (int d = w; d < dn; d += 8) {
            const T* wr = wt + (size_t)(d0 + d) * c.V;
            float wv[4];
#pragma unroll
            for (int j = 0; j < 4; j++) wv[j] = c0 + 32 * j < c.V ? rg_to_float(wr[c0 + 32 * j]) : 0.f;
#pragma unroll
            for (int r = 0; r < RB; r++) {
                const float xv = sm[d * RB + r];
#pragma unroll
                for (int j = 0; j < 4; j++) acc[r][j] = fmaf(xv, wv[j], acc[r][j]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) sm[(w * RB + r) * 128 + lane + 32 * j] = acc[r][j];
    __syncthreads();
    // warp w takes rows w, w + 8, ...: the sum over the 8 slices of D, then the bias
#pragma unroll
    for (int k = 0; k < (RB / 8 > 0 ? RB / 8 : 1); k++) {
        const int r = w + 8 * k;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float s = 0.f;
            if (r < RB)
#pragma unroll
                for (int q = 0; q < 8; q++) s += sm[(q * RB + r) * 128 + lane + 32 * j];
            const int col = c0 + 32 * j;
            z[k][j] = col < c.V ? s + (c.bias ? c.bias[col] : 0.f) : -INFINITY;
        }
    }
}

template <typename T, int RB>
__global__ void __launch_bounds__(256) lce_few_fwd_kernel(const lce_call c) {
    extern __shared__ float sm[];
    float z[RB / 8 > 0 ? RB / 8 : 1][4];
    lce_few_logits<T, RB>(c, sm, z);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < (RB / 8 > 0 ? RB / 8 : 1); k++) {
        const int r = w + 8 * k;
        if (r >= c.R || r >= RB) continue;  // whole warps
        const int t = c.tgt[r];
        float m = fmaxf(fmaxf(z[k][0], z[k][1]), fmaxf(z[k][2], z[k][3]));
        m = rg_warp_max(m);
        const float ref = m == -INFINITY ? 0.f : m;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s += expf(z[k][j] - ref);
            if (t == (int)blockIdx.x * 128 + lane + 32 * j) c.tz[r] = z[k][j];
        }
        s = rg_warp_sum(s);
        if (lane == 0) c.parts[(size_t)blockIdx.x * c.R + r] = make_float2(m, s);
    }
}

// dz (without the common factor dloss / n) of all rows, f32 [R][V], and the bias gradient
template <typename T, int RB>
__global__ void __launch_bounds__(256) lce_few_dz_kernel(const lce_call c, float* __restrict__ dz) {
    extern __shared__ float sm[];
    float z[RB / 8 > 0 ? RB / 8 : 1][4];
    lce_few_logits<T, RB>(c, sm, z);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    float col[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < (RB / 8 > 0 ? RB / 8 : 1); k++) {
        const int r = w + 8 * k;
        if (r >= c.R || r >= RB) continue;
        const int t = c.tgt[r];
        const float lse = c.lse[r];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int v = (int)blockIdx.x * 128 + lane + 32 * j;
            if (v < c.V) {
                const float p = t < 0 ? 0.f : expf(z[k][j] - lse) - (v == t ? 1.f : 0.f);
                dz[(size_t)r * c.V + v] = p;
                col[j] += p;
            }
        }
    }
    if (!c.dbias) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; j++) sm[w * 128 + lane + 32 * j] = col[j];
    __syncthreads();
    if (threadIdx.x < 128) {
        const int v = (int)blockIdx.x * 128 + threadIdx.x;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 8; q++) s += sm[q * 128 + threadIdx.x];
        if (v < c.V) c.dbias[v] = s * c.scal[1];
    }
}

// dw and partial dx.  A thread holds dz of RB rows and 4 columns in registers and walks LCE_DG rows of w: one load of w
// and one store of dw per element; the RB products with dz are summed over the warp by halving exchanges (each exchange
// adds two rows at once, so RB rows cost RB shuffles plus the steps left), over the 8 warps in shared memory.
#define LCE_DG 32
template <typename T, int RB>
__global__ void __launch_bounds__(256) lce_few_grad_kernel(const lce_call c, const float* __restrict__ dz, float* __restrict__ dxparts) {
    __shared__ float xs[LCE_DG][RB];
    __shared__ float dxs[8][LCE_DG][RB];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c0 = (int)blockIdx.x * 1024 + w * 128 + lane;
    const int d0 = (int)blockIdx.y * LCE_DG, dn = min(LCE_DG, c.D - d0);
    const T* x = static_cast<const T*>(c.x);
    const T* wt = static_cast<const T*>(c.w);
    T* dw = static_cast<T*>(c.dw);
    const float scale = c.scal[1];
    for (int i = threadIdx.x; i < LCE_DG * RB; i += 256) {
        const int r = i / LCE_DG, d = i % LCE_DG;
        xs[d][r] = (r < c.R && d < dn) ? rg_to_float(x[(size_t)r * c.D + d0 + d]) : 0.f;
    }
    float g[RB][4];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) g[r][j] = (r < c.R && c0 + 32 * j < c.V) ? dz[(size_t)r * c.V + c0 + 32 * j] : 0.f;
    __syncthreads();
#pragma unroll 2
    for (int d = 0; d < dn; d++) {
        const size_t at = (size_t)(d0 + d) * c.V + c0;
        float wv[4], o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) wv[j] = c0 + 32 * j < c.V ? rg_to_float(wt[at + 32 * j]) : 0.f, o[j] = 0.f;
        float q[RB];
#pragma unroll
        for (int r = 0; r < RB; r++) {
            const float xv = xs[d][r];
            q[r] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[j] = fmaf(xv, g[r][j], o[j]);
                q[r] = fmaf(g[r][j], wv[j], q[r]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (c0 + 32 * j < c.V) dw[at + 32 * j] = rg_from_float<T>(o[j] * scale);
        // halving exchange: after it, lane l holds row (l / (32 / RB)) summed over the lanes that share it
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

#define LCE_FEW_ROWS 16

template <typename T, int RB>
static void lce_few_launch(rg_ctx* ctx, const lce_call& c, float* dz, float* dxparts) {
    const unsigned tiles = (unsigned)rg_cdiv(c.V, 128);
    const size_t smem = lce_few_smem<RB>();
    if (!dz) {
        if (smem > 48 * 1024) cudaFuncSetAttribute(lce_few_fwd_kernel<T, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        lce_few_fwd_kernel<T, RB><<<tiles, 256, smem, ctx->stream>>>(c);
        RG_LAUNCHED(ctx);
        return;
    }
    if (smem > 48 * 1024) cudaFuncSetAttribute(lce_few_dz_kernel<T, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    lce_few_dz_kernel<T, RB><<<tiles, 256, smem, ctx->stream>>>(c, dz);
    lce_few_grad_kernel<T, RB><<<dim3((unsigned)rg_cdiv(c.V, 1024), (unsigned)rg_cdiv(c.D, LCE_DG)), 256, 0, ctx->stream>>>(c, dz, dxparts);
    ctx->launches += 2;
}
template <typename T>
static void lce_few_rows(rg_ctx* ctx, const lce_call& c, float* dz, float* dxparts) {
    if (c.R <= 1) lce_few_launch<T, 1>(ctx, c, dz, dxparts);
    else if (c.R <= 2) lce_few_launch<T, 2>(ctx, c, dz, dxparts);
    else if (c.R <= 4) lce_few_launch<T, 4>(ctx, c, dz, dxparts);
    else if (c.R <= 8) lce_few_launch<T, 8>(ctx, c, dz, dxparts);
    else lce_few_launch<T, 16>(ctx, c, dz, dxparts);
}
static void lce_few(rg_ctx* ctx, const lce_call& c, float* dz, float* dxparts) {
    if (c.dtype == RG_DTYPE_F32) lce_few_rows<float>(ctx, c, dz, dxparts);
    else lce_few_rows<__nv_bfloat16>(ctx, c, dz, dxparts);
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
    c->R = (int)R, c->D = (int)D, c->V = (int)V, c->dtype = x->dtype;
    c->x = x->raw(), c->w = w->raw(), c->bias = bias ? bias->data() : nullptr;
    return RG_OK;
}

// Enqueues the check of the targets; lce_checked waits for it (not for what was enqueued after it).
static rg_status lce_check_launch(rg_ctx* ctx, lce_call& c, const rg_storage* targets, long long ignore, const rg_storage* dloss,
                                  rg_storage** scratch) {
    // tgt [R] | tz [R] | scal [2] | status [3]
    const size_t words = 2 * (size_t)c.R + 5;
    RG_TRY(rg_alloc_storage(ctx, &words, 1, scratch));
    float* base = (*scratch)->data();
    c.tgt = reinterpret_cast<int*>(base), c.tz = base + c.R, c.scal = base + 2 * (size_t)c.R;
    c.wmax = reinterpret_cast<unsigned*>(base + 2 * (size_t)c.R + 4);
    lce_check_kernel<<<1, 1024, 0, ctx->stream>>>(targets->data(), c.R, c.V, ignore, dloss ? dloss->data() : nullptr,
                                                  const_cast<int*>(c.tgt), c.tz, const_cast<float*>(c.scal),
                                                  reinterpret_cast<int*>(const_cast<float*>(c.scal)) + 2);
    RG_LAUNCHED(ctx);
    RG_CUDA(cudaGetLastError());
    RG_CUDA(cudaMemcpyAsync(ctx->h_flag, c.scal + 2, sizeof(int), cudaMemcpyDeviceToHost, ctx->stream));
    RG_CUDA(cudaEventRecord(ctx->check_ev, ctx->stream));
    return RG_OK;
}
static rg_status lce_checked(rg_ctx* ctx, const lce_call& c) {
    RG_CUDA(cudaEventSynchronize(ctx->check_ev));
    if (ctx->h_flag[0]) return rg_fail(RG_ERR_SHAPE, "Target index out of bounds for %d classes", c.V);
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
    RG_TRY(lce_check_launch(ctx, c, targets, ignore_index, nullptr, &o[2]));
    const bool few = c.R <= LCE_FEW_ROWS;
    c.nparts = few ? rg_cdiv(c.V, 128) : lce_tc_nparts(c.V);
    const size_t pwords = 2 * (size_t)c.nparts * rows, blocks = (size_t)rg_cdiv(c.R, 8), swords = 2 * blocks;
    RG_TRY(rg_alloc_storage(ctx, &pwords, 1, &o[3]));
    RG_TRY(rg_alloc_storage(ctx, &swords, 1, &o[4]));
    c.parts = static_cast<float2*>(o[3]->raw());
    if (few) lce_few(ctx, c, nullptr, nullptr);
    else RG_TRY(lce_tc_forward(ctx, c));
    lce_loss_kernel<<<(unsigned)blocks, 256, 0, ctx->stream>>>(c.parts, c.nparts, c.R, c.tgt, c.tz, c.scal,
                                                               reinterpret_cast<int*>(const_cast<float*>(c.scal)) + 3,
                                                               static_cast<double*>(o[4]->raw()), o[1]->data(), o[0]->data());
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
        RG_TRY(lce_check_launch(ctx, c, targets, ignore_index, dloss, &o[3]));
        if (c.R <= LCE_FEW_ROWS) {
            const size_t zlen = (size_t)c.R * c.V, nparts = (size_t)rg_cdiv(c.V, 1024), plen = nparts * c.R * c.D;
            RG_TRY(rg_alloc_storage(ctx, &zlen, 1, &o[4]));
            RG_TRY(rg_alloc_storage(ctx, &plen, 1, &o[5]));
            lce_few(ctx, c, o[4]->data(), o[5]->data());
            lce_dx_finish_launch(ctx, o[5]->data(), (int)nparts, (size_t)c.R * c.D, c.scal, c.dx, c.dtype);
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

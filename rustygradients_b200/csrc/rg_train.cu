// Training ops that are bound by memory traffic: LayerNorm with saved statistics, its gradient, and clipping by the global
// gradient norm (rg_b200.h, "training ops").  The loss of the vocabulary projection is in rg_lce.cu.
#include "rg_internal.cuh"
#include "rg_train.cuh"

#include <algorithm>

// ---------------------------------------------------------------------------
// rows in registers
// ---------------------------------------------------------------------------
// A row of n values belongs to a group of 32 * WPR threads; thread t of the group holds the PER vectors of VEC values that
// start at (t + j * group) * VEC, so every access of a warp is contiguous.  VEC values are 16 bytes when every row starts
// on a 16-byte boundary, else 4 bytes (two bf16) or one value.
template <typename T, int VEC>
struct ln_vec;
template <>
struct ln_vec<float, 4> { typedef float4 type; };
template <>
struct ln_vec<float, 1> { typedef float type; };
template <>
struct ln_vec<__nv_bfloat16, 8> { typedef uint4 type; };
template <>
struct ln_vec<__nv_bfloat16, 2> { typedef uint32_t type; };
template <>
struct ln_vec<__nv_bfloat16, 1> { typedef unsigned short type; };

template <typename T, int VEC>
__device__ __forceinline__ void ln_load(const T* __restrict__ p, float (&v)[VEC]) {
    typedef typename ln_vec<T, VEC>::type V;
    const V raw = __ldcs(reinterpret_cast<const V*>(p));
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = rg_to_float(e[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void ln_store(T* __restrict__ p, const float (&v)[VEC]) {
    typedef typename ln_vec<T, VEC>::type V;
    V raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; i++) e[i] = rg_from_float<T>(v[i]);
    *reinterpret_cast<V*>(p) = raw;
}

// VEC parameters (f32, storages start on 16-byte boundaries and c is a multiple of VEC)
template <int VEC>
__device__ __forceinline__ void ln_param(const float* __restrict__ p, float (&v)[VEC]) {
    if (VEC >= 4) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(p + i));
            v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
        }
    } else if (VEC == 2) {
        const float2 q = __ldg(reinterpret_cast<const float2*>(p));
        v[0] = q.x, v[VEC - 1] = q.y;
    } else {
        v[0] = __ldg(p);
    }
}

// Sums of two values over the WPR warps of a row group, in a fixed order; every thread of the group gets them.  red: two
// slots of WPR pairs for this group, used in turn, so that one barrier per call - of this group alone - is enough.
template <int WPR>
__device__ __forceinline__ float2 ln_group_sum(float a, float b, float2* red, int group, int gwarp) {
    a = rg_warp_sum(a), b = rg_warp_sum(b);
    if (WPR == 1) return make_float2(a, b);
    if ((threadIdx.x & 31) == 0) red[gwarp] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(32 * WPR) : "memory");
    float2 r = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WPR; w++) {
        const float2 p = red[w];
        r.x += p.x, r.y += p.y;
    }
    return r;
}

// y = (x - mean) rstd gamma + beta.  One read of x: the mean, then the squared deviations from it, are summed over the
// registers, so the variance does not cancel however far the row is from zero.  Memory bound: x in, y out.  A group walks
// rows with the next row's loads in flight behind the two sums of this one.  32768 x 768 f32: 31 us, 6.5 TB/s counting x and y
// once each; 43 of the 101 MB of y reach DRAM within the kernel, the rest leaves L2 behind it.
template <typename T, int VEC, int PER, int WPR, int THREADS>
__global__ void __launch_bounds__(THREADS) rg_ln_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                            const float* __restrict__ beta, T* __restrict__ y,
                                                            float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows,
                                                            int n, float eps) {
    constexpr int GROUPS = THREADS / 32 / WPR;
    typedef typename ln_vec<T, VEC>::type V;
    __shared__ float2 red[2][GROUPS][WPR];
    const int group = threadIdx.x / (32 * WPR), t = threadIdx.x % (32 * WPR), gwarp = t >> 5;
    const long long step = (long long)gridDim.x * GROUPS;
    V next[PER];
    long long row = (long long)blockIdx.x * GROUPS + group;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int c = (t + j * 32 * WPR) * VEC;
        if (row < rows && c < n) next[j] = __ldcs(reinterpret_cast<const V*>(x + row * n + c));
    }
    for (; row < rows; row += step) {  // the same number of turns for every thread of the group
        float v[PER][VEC];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int c = (t + j * 32 * WPR) * VEC;
            const T* e = reinterpret_cast<const T*>(&next[j]);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                v[j][i] = c < n ? rg_to_float(e[i]) : 0.f;
                s += v[j][i];
            }
            if (row + step < rows && c < n) next[j] = __ldcs(reinterpret_cast<const V*>(x + (row + step) * n + c));
        }
        const float mean = ln_group_sum<WPR>(s, 0.f, red[0][group], group, gwarp).x / (float)n;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < PER; j++)
            if ((t + j * 32 * WPR) * VEC < n)
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = v[j][i] - mean;
                    q += d * d;
                }
        const float var = ln_group_sum<WPR>(q, 0.f, red[1][group], group, gwarp).x / (float)n;
        const float rstd = 1.f / sqrtf(var + eps);
        if (t == 0) mean_out[row] = mean, rstd_out[row] = rstd;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int c = (t + j * 32 * WPR) * VEC;
            if (c < n) {
                float gm[VEC], bt[VEC];
                ln_param<VEC>(gamma + c, gm);
                ln_param<VEC>(beta + c, bt);
#pragma unroll
                for (int i = 0; i < VEC; i++) v[j][i] = (v[j][i] - mean) * rstd * gm[i] + bt[i];
                ln_store<T, VEC>(y + row * n + c, v[j]);
            }
        }
    }
}

// Rows too long for the registers: three passes, the last two from L2.
template <typename T>
__global__ void __launch_bounds__(512) rg_ln_fwd_long_kernel(const T* __restrict__ x, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, T* __restrict__ y,
                                                             float* __restrict__ mean_out, float* __restrict__ rstd_out, long long n,
                                                             float eps) {
    __shared__ float2 red[2][16];
    const T* xr = x + (long long)blockIdx.x * n;
    float s = 0.f, q = 0.f;
    for (long long c = threadIdx.x; c < n; c += 512) s += rg_to_float(xr[c]);
    const float mean = ln_group_sum<16>(s, 0.f, red[0], 0, threadIdx.x >> 5).x / (float)n;
    for (long long c = threadIdx.x; c < n; c += 512) {
        const float d = rg_to_float(xr[c]) - mean;
        q += d * d;
    }
    const float rstd = 1.f / sqrtf(ln_group_sum<16>(q, 0.f, red[1], 0, threadIdx.x >> 5).x / (float)n + eps);
    if (threadIdx.x == 0) mean_out[blockIdx.x] = mean, rstd_out[blockIdx.x] = rstd;
    for (long long c = threadIdx.x; c < n; c += 512)
        y[(long long)blockIdx.x * n + c] = rg_from_float<T>((rg_to_float(xr[c]) - mean) * rstd * gamma[c] + beta[c]);
}

__device__ __forceinline__ float ln_half(float2 v, int i) { return i & 1 ? v.y : v.x; }

// Resident CTAs per SM of the gradient: registers for 8 or 16 values a thread (two column sums, this row and the next one)
#define LN_BWD_CTAS(threads, values) ((threads) == 256 ? ((values) == 8 ? 3 : 2) : 1)

// dx = rstd (a - mean(a) - xh mean(a xh)), and the two column sums dgamma = sum dy xh, dbeta = sum dy.  One read of dy and
// x serves all three: a group walks rows, every thread always on the same columns, so the column sums stay in its registers
// until the end; then the CTA's groups are added and the CTA leaves one partial row of sums, which rg_colsum_kernel adds over
// the CTAs.  Memory bound: dy and x in, dx out; the next row's loads are in flight behind the sums of this one.  16384 x 1600
// bf16: 33 us, 4.8 TB/s, and 5.6 us for the sums; bound by the two sums of every row, which 16 warps an SM (their 32 column
// sums a thread fill the registers) do not hide: rows further ahead, through shared memory, gained nothing.
template <typename T, int VEC, int PER, int WPR, int THREADS>
__global__ void __launch_bounds__(THREADS, LN_BWD_CTAS(THREADS, PER * VEC)) rg_ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                            const float* __restrict__ gamma, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, T* __restrict__ dx,
                                                            float* __restrict__ parts, long long rows, int n) {
    constexpr int GROUPS = THREADS / 32 / WPR, COLS = 32 * WPR * PER * VEC;
    constexpr int PAIRS = PER * VEC / 2;     // value e of a thread (vector e / VEC) is half e % 2 of pair e / 2
    constexpr bool AHEAD = PER * VEC <= 16;  // room in the registers for the next row
    typedef typename ln_vec<T, VEC>::type V;
    __shared__ float2 red[2][GROUPS][WPR];
    __shared__ float comb[GROUPS > 1 ? GROUPS * COLS : 1];
    const int group = threadIdx.x / (32 * WPR), t = threadIdx.x % (32 * WPR), gwarp = t >> 5;
    const long long step = (long long)gridDim.x * GROUPS;
    float2 dg[PAIRS], db[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; i++) dg[i] = db[i] = make_float2(0.f, 0.f);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the sum over the CTAs waits for all of this kernel
    const float inv_n = 1.f / (float)n;
    long long row = (long long)blockIdx.x * GROUPS + group;
    V nx[PER], ng[PER];
    float nm = 0.f, nr = 0.f;
    auto fetch = [&](long long at) {
        if (at >= rows) return;
        nm = mean[at], nr = rstd[at];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int c = (t + j * 32 * WPR) * VEC;
            if (c < n) {
                nx[j] = __ldcs(reinterpret_cast<const V*>(x + at * n + c));
                ng[j] = __ldcs(reinterpret_cast<const V*>(dy + at * n + c));
            }
        }
    };
    if (AHEAD) fetch(row);
    for (int turn = 0; row < rows; row += step, turn ^= 1) {
        if (!AHEAD) fetch(row);
        float2 xv[PAIRS], gv[PAIRS];
        const float m = nm, r = nr;
#pragma unroll
        for (int e = 0; e < PER * VEC; e++) {
            const bool in = (t + e / VEC * 32 * WPR) * VEC < n;
            const float a = in ? rg_to_float(reinterpret_cast<const T*>(&nx[e / VEC])[e % VEC]) : m;
            const float b = in ? rg_to_float(reinterpret_cast<const T*>(&ng[e / VEC])[e % VEC]) : 0.f;
            if (e % 2) xv[e / 2].y = a, gv[e / 2].y = b;
            else xv[e / 2].x = a, gv[e / 2].x = b;
        }
        if (AHEAD) fetch(row + step);
        float gm[PER][VEC];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int c = (t + j * 32 * WPR) * VEC;
            ln_param<VEC>(gamma + (c < n ? c : 0), gm[j]);  // dy is 0 beyond the row
        }
        const float2 m2 = make_float2(-m, -m), r2 = make_float2(r, r);
        float2 s1 = make_float2(0.f, 0.f), s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            const float2 xh = rg_mul2(rg_add2(xv[i], m2), r2), g = gv[i];
            db[i] = rg_add2(db[i], g);
            dg[i] = rg_fma2(g, xh, dg[i]);
            const float2 a = rg_mul2(g, make_float2(gm[2 * i / VEC][2 * i % VEC], gm[(2 * i + 1) / VEC][(2 * i + 1) % VEC]));
            s1 = rg_add2(s1, a), s2 = rg_fma2(a, xh, s2);
            xv[i] = xh, gv[i] = a;
        }
        const float2 s = ln_group_sum<WPR>(s1.x + s1.y, s2.x + s2.y, red[turn][group], group, gwarp);
        const float2 k1 = make_float2(-s.x * inv_n, -s.x * inv_n), k2 = make_float2(-s.y * inv_n, -s.y * inv_n);
#pragma unroll
        for (int i = 0; i < PAIRS; i++) gv[i] = rg_mul2(r2, rg_fma2(xv[i], k2, rg_add2(gv[i], k1)));
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int c = (t + j * 32 * WPR) * VEC;
            if (c < n) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; i++) o[i] = ln_half(gv[(j * VEC + i) / 2], j * VEC + i);
                ln_store<T, VEC>(dx + row * n + c, o);
            }
        }
    }
    // the groups of the CTA, in order, then one partial row [dgamma | dbeta] of the CTA
    float* out = parts + (size_t)blockIdx.x * 2 * n;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        if (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; j++)
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    comb[group * COLS + (t + j * 32 * WPR) * VEC + i] = ln_half(which ? db[(j * VEC + i) / 2] : dg[(j * VEC + i) / 2], j * VEC + i);
            __syncthreads();
            for (int c = threadIdx.x; c < n; c += THREADS) {
                float s = 0.f;
#pragma unroll
                for (int g = 0; g < GROUPS; g++) s += comb[g * COLS + c];
                out[which * n + c] = s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int c = (t + j * 32 * WPR) * VEC;
                if (c < n)
#pragma unroll
                    for (int i = 0; i < VEC; i++)
                        out[which * n + c + i] = ln_half(which ? db[(j * VEC + i) / 2] : dg[(j * VEC + i) / 2], j * VEC + i);
            }
        }
    }
}

// Rows too long for the registers: dx row by row in two passes, and the column sums over a slice of the rows each.
template <typename T>
__global__ void __launch_bounds__(512) rg_ln_bwd_long_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                const float* __restrict__ gamma, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, T* __restrict__ dx, long long n) {
    __shared__ float2 red[16];
    const T *xr = x + (long long)blockIdx.x * n, *gr = dy + (long long)blockIdx.x * n;
    const float m = mean[blockIdx.x], r = rstd[blockIdx.x];
    float s1 = 0.f, s2 = 0.f;
    for (long long c = threadIdx.x; c < n; c += 512) {
        const float a = rg_to_float(gr[c]) * gamma[c];
        s1 += a, s2 += a * (rg_to_float(xr[c]) - m) * r;
    }
    const float2 s = ln_group_sum<16>(s1, s2, red, 0, threadIdx.x >> 5);
    s1 = s.x / (float)n, s2 = s.y / (float)n;
    for (long long c = threadIdx.x; c < n; c += 512)
        dx[(long long)blockIdx.x * n + c] =
            rg_from_float<T>(r * (rg_to_float(gr[c]) * gamma[c] - s1 - (rg_to_float(xr[c]) - m) * r * s2));
}
template <typename T>
__global__ void __launch_bounds__(256) rg_ln_bwd_long_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                  float* __restrict__ parts, long long rows, long long n) {
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float dg = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = rg_to_float(dy[row * n + c]);
        db += g, dg += g * (rg_to_float(x[row * n + c]) - mean[row]) * rstd[row];
    }
    parts[(size_t)blockIdx.y * 2 * n + c] = dg;
    parts[(size_t)blockIdx.y * 2 * n + n + c] = db;
}

// out[c] = sum over p of parts[p][c], c < cols, in a fixed order: a CTA takes 32 columns, its 32 warps every 32nd partial.
__global__ void __launch_bounds__(1024) rg_colsum_kernel(const float* parts, int nparts, long long cols,
                                                         float* __restrict__ out0, float* __restrict__ out1, long long split) {
    __shared__ float red[32][33];
    rg_pdl_sync();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < cols) {
        int p = w;
        for (; p + 96 < nparts; p += 128) {  // four loads in flight
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = parts[(size_t)(p + u * 32) * cols + c];
#pragma unroll
            for (int u = 0; u < 4; u++) s += v[u];
        }
        for (; p < nparts; p += 32) s += parts[(size_t)p * cols + c];
    }
    red[w][lane] = s;
    __syncthreads();
    s = rg_warp_sum(red[lane][w]);  // the 32 slices of column w of this CTA
    const long long o = (long long)blockIdx.x * 32 + w;
    if (lane == 0 && o < cols) {
        if (o < split) out0[o] = s;
        else out1[o - split] = s;
    }
}

void rg_colsum_launch(rg_ctx* ctx, const float* parts, int nparts, long long cols, float* out0, float* out1, long long split) {
    rg_launch(true, rg_colsum_kernel, dim3((unsigned)rg_cdiv(cols, 32)), dim3(1024), 0, ctx->stream, parts, nparts, cols, out0, out1, split);
    RG_LAUNCHED(ctx);
}

// ---------------------------------------------------------------------------
// host side of LayerNorm
// ---------------------------------------------------------------------------
struct ln_args {
    const void *x, *dy;
    const float *gamma, *beta, *mean, *rstd;
    void* out;
    float *mean_out, *rstd_out, *parts;
    long long rows;
    int n;
    float eps;
};

#define LN_MAX_N 16384   // 512 threads with 32 values each

template <bool BWD, typename T, int VEC, int PER, int WPR, int THREADS>
static void ln_launch_one(rg_ctx* ctx, const ln_args& a, int* nparts) {
    constexpr int GROUPS = THREADS / 32 / WPR;
    const long long groups = (a.rows + GROUPS - 1) / GROUPS;
    if constexpr (!BWD) {
        const int grid = (int)std::min<long long>(groups, (long long)ctx->sm_count * (2048 / THREADS));
        rg_ln_fwd_kernel<T, VEC, PER, WPR, THREADS><<<grid, THREADS, 0, ctx->stream>>>(
            (const T*)a.x, a.gamma, a.beta, (T*)a.out, a.mean_out, a.rstd_out, a.rows, a.n, a.eps);
    } else {
        *nparts = (int)std::min<long long>(groups, (long long)ctx->sm_count * LN_BWD_CTAS(THREADS, PER * VEC));
        if (!a.parts) return;  // the caller asks for the number of partial rows first
        rg_ln_bwd_kernel<T, VEC, PER, WPR, THREADS><<<*nparts, THREADS, 0, ctx->stream>>>((const T*)a.dy, (const T*)a.x, a.gamma, a.mean,
                                                                                         a.rstd, (T*)a.out, a.parts, a.rows, a.n);
    }
    RG_LAUNCHED(ctx);
}

// Values per thread of the gradient (16384 x 1600, us with the column sums): f32 8 64, 16 67; bf16 8 46, 16 40; rows that
// allow only single-value loads 8 (32000 x 767: 54 against 81).  Forward up to 32.  More only where a group is the whole CTA.
template <bool BWD, typename T, int VEC>
static void ln_launch_vec(rg_ctx* ctx, const ln_args& a, int* nparts) {
    constexpr int P = 8 / VEC;
    if constexpr (BWD) {
        constexpr int Q = sizeof(T) == 2 && VEC > 1 ? 2 : 1;  // 8 Q values, 256 Q columns a warp
        if (a.n <= 256) ln_launch_one<true, T, VEC, P, 1, 256>(ctx, a, nparts);
        else if (a.n <= 512) ln_launch_one<true, T, VEC, Q * P, 2 / Q, 256>(ctx, a, nparts);
        else if (a.n <= 1024) ln_launch_one<true, T, VEC, Q * P, 4 / Q, 256>(ctx, a, nparts);
        else if (a.n <= 2048) ln_launch_one<true, T, VEC, Q * P, 8 / Q, 256>(ctx, a, nparts);
        else if (a.n <= 4096) ln_launch_one<true, T, VEC, 2 * P, 8, 256>(ctx, a, nparts);
        else if (a.n <= 8192) ln_launch_one<true, T, VEC, 2 * P, 16, 512>(ctx, a, nparts);
        else ln_launch_one<true, T, VEC, 4 * P, 16, 512>(ctx, a, nparts);
    } else {
        if (a.n <= 256) ln_launch_one<false, T, VEC, P, 1, 256>(ctx, a, nparts);
        else if (a.n <= 512) ln_launch_one<false, T, VEC, 2 * P, 1, 256>(ctx, a, nparts);
        else if (a.n <= 1024) ln_launch_one<false, T, VEC, 4 * P, 1, 256>(ctx, a, nparts);
        else if (a.n <= 2048) ln_launch_one<false, T, VEC, 4 * P, 2, 256>(ctx, a, nparts);
        else if (a.n <= 4096) ln_launch_one<false, T, VEC, 4 * P, 4, 256>(ctx, a, nparts);
        else if (a.n <= 8192) ln_launch_one<false, T, VEC, 4 * P, 8, 256>(ctx, a, nparts);
        else ln_launch_one<false, T, VEC, 4 * P, 16, 512>(ctx, a, nparts);
    }
}

template <bool BWD>
static void ln_launch(rg_ctx* ctx, const ln_args& a, int dtype, int* nparts) {
    if (dtype == RG_DTYPE_F32) {
        if (a.n % 4 == 0) ln_launch_vec<BWD, float, 4>(ctx, a, nparts);
        else ln_launch_vec<BWD, float, 1>(ctx, a, nparts);
    } else {
        if (a.n % 8 == 0) ln_launch_vec<BWD, __nv_bfloat16, 8>(ctx, a, nparts);
        else if (a.n % 2 == 0) ln_launch_vec<BWD, __nv_bfloat16, 2>(ctx, a, nparts);
        else ln_launch_vec<BWD, __nv_bfloat16, 1>(ctx, a, nparts);
    }
}

static rg_status ln_check(const char* op, rg_ctx* ctx, const rg_storage* x, const rg_storage* gamma, size_t* rows) {
    if (x->shape.empty()) return rg_fail(RG_ERR_DIMENSION, "%s requires at least 1 dimension, got 0", op);
    const size_t n = x->shape.back();
    if (n == 0 || n > 0x7fffffff) return rg_fail(RG_ERR_SHAPE, "%s: rows of %zu values", op, n);
    RG_TRY(rg_need_f32("a LayerNorm parameter or statistic", gamma));
    if (gamma->len != n)
        return rg_fail(RG_ERR_SHAPE, "Invalid shape for gamma in LayerNorm: expected [1, %zu], got %zu elements", n, gamma->len);
    *rows = x->len / n;
    if (*rows > 0x7fffffff) return rg_fail(RG_ERR_SHAPE, "%s: %zu rows", op, *rows);
    return rg_not_capturing(ctx, op);
}

extern "C" rg_status rg_layer_norm_fwd(rg_ctx* ctx, const rg_storage* x, const rg_storage* gamma, const rg_storage* beta, float epsilon,
                                       rg_storage** y, rg_storage** mean, rg_storage** rstd) {
    if (!ctx || !x || !gamma || !beta || !y || !mean || !rstd) return rg_fail(RG_ERR_INVALID_INPUT, "NULL argument");
    *y = *mean = *rstd = nullptr;
    RG_TRY(rg_same_ctx(ctx, {x, gamma, beta}));
    rg_op_guard g(ctx);
    size_t rows = 0;
    RG_TRY(ln_check("layer_norm", ctx, x, gamma, &rows));
    const size_t n = x->shape.back();
    RG_TRY(rg_need_f32("a LayerNorm parameter or statistic", beta));
    if (beta->len != n)
        return rg_fail(RG_ERR_SHAPE, "Invalid shape for beta in LayerNorm: expected [1, %zu], got %zu elements", n, beta->len);
    rg_outputs<3> o;
    const int lead = (int)x->shape.size() - 1;
    RG_TRY(rg_alloc_storage(ctx, x->shape.data(), lead + 1, &o[0], x->dtype));
    RG_TRY(rg_alloc_storage(ctx, x->shape.data(), lead, &o[1]));
    RG_TRY(rg_alloc_storage(ctx, x->shape.data(), lead, &o[2]));
    if (rows) {
        if (n > LN_MAX_N) {
            if (x->dtype == RG_DTYPE_F32)
                rg_ln_fwd_long_kernel<float><<<(unsigned)rows, 512, 0, ctx->stream>>>(x->data(), gamma->data(), beta->data(), o[0]->data(),
                                                                                     o[1]->data(), o[2]->data(), (long long)n, epsilon);
            else
                rg_ln_fwd_long_kernel<__nv_bfloat16><<<(unsigned)rows, 512, 0, ctx->stream>>>(
                    (const __nv_bfloat16*)x->raw(), gamma->data(), beta->data(), (__nv_bfloat16*)o[0]->raw(), o[1]->data(), o[2]->data(),
                    (long long)n, epsilon);
            RG_LAUNCHED(ctx);
        } else {
            ln_args a;
            memset(&a, 0, sizeof(a));
            a.x = x->raw(), a.gamma = gamma->data(), a.beta = beta->data(), a.out = o[0]->raw();
            a.mean_out = o[1]->data(), a.rstd_out = o[2]->data(), a.rows = (long long)rows, a.n = (int)n, a.eps = epsilon;
            ln_launch<false>(ctx, a, x->dtype, nullptr);
        }
    }
    RG_CUDA(cudaGetLastError());
    o.give({y, mean, rstd});
    return RG_OK;
}

extern "C" rg_status rg_layer_norm_bwd(rg_ctx* ctx, const rg_storage* dy, const rg_storage* x, const rg_storage* gamma,
                                       const rg_storage* mean, const rg_storage* rstd, rg_storage** dx, rg_storage** dgamma,
                                       rg_storage** dbeta) {
    if (!ctx || !dy || !x || !gamma || !mean || !rstd || !dx || !dgamma || !dbeta) return rg_fail(RG_ERR_INVALID_INPUT, "NULL argument");
    *dx = *dgamma = *dbeta = nullptr;
    RG_TRY(rg_same_ctx(ctx, {dy, x, gamma, mean, rstd}));
    rg_op_guard g(ctx);
    size_t rows = 0;
    RG_TRY(ln_check("layer_norm_bwd", ctx, x, gamma, &rows));
    RG_TRY(rg_need_f32("a LayerNorm parameter or statistic", mean, rstd));
    const size_t n = x->shape.back();
    if (dy->shape != x->shape) return rg_fail(RG_ERR_SHAPE, "layer_norm_bwd: dy does not have the shape of x");
    if (dy->dtype != x->dtype) return rg_fail(RG_ERR_UNSUPPORTED, "layer_norm_bwd: dy and x have different types");
    if (mean->len != rows || rstd->len != rows)
        return rg_fail(RG_ERR_SHAPE, "layer_norm_bwd: %zu rows, %zu means, %zu deviations", rows, mean->len, rstd->len);
    rg_outputs<4> o;  // the last one: partial column sums
    RG_TRY(rg_alloc_storage(ctx, x->shape.data(), (int)x->shape.size(), &o[0], x->dtype));
    RG_TRY(rg_alloc_storage(ctx, gamma->shape.data(), (int)gamma->shape.size(), &o[1]));
    RG_TRY(rg_alloc_storage(ctx, gamma->shape.data(), (int)gamma->shape.size(), &o[2]));
    if (!rows) {
        RG_CUDA(cudaMemsetAsync(o[1]->raw(), 0, n * 4, ctx->stream));
        RG_CUDA(cudaMemsetAsync(o[2]->raw(), 0, n * 4, ctx->stream));
    } else {
        ln_args a;
        memset(&a, 0, sizeof(a));
        a.x = x->raw(), a.dy = dy->raw(), a.gamma = gamma->data(), a.mean = mean->data(), a.rstd = rstd->data(), a.out = o[0]->raw();
        a.rows = (long long)rows, a.n = (int)n;
        // long rows: slices of the rows until the blocks of 256 columns fill the GPU
        int nparts = (int)std::min<size_t>({rows, 64, std::max<size_t>(1, (size_t)ctx->sm_count * 8 * 256 / n)});
        if (n <= LN_MAX_N) ln_launch<true>(ctx, a, x->dtype, &nparts);  // a.parts is NULL: only counts
        const size_t pshape[2] = {(size_t)nparts, 2 * n};
        RG_TRY(rg_alloc_storage(ctx, pshape, 2, &o[3]));
        a.parts = o[3]->data();
        if (n <= LN_MAX_N) {
            ln_launch<true>(ctx, a, x->dtype, &nparts);
        } else {
            const dim3 cols((unsigned)((n + 255) / 256), (unsigned)nparts);
            if (x->dtype == RG_DTYPE_F32) {
                rg_ln_bwd_long_dx_kernel<float><<<(unsigned)rows, 512, 0, ctx->stream>>>(dy->data(), x->data(), a.gamma, a.mean, a.rstd,
                                                                                        o[0]->data(), (long long)n);
                rg_ln_bwd_long_cols_kernel<float><<<cols, 256, 0, ctx->stream>>>(dy->data(), x->data(), a.mean, a.rstd, a.parts, a.rows,
                                                                                (long long)n);
            } else {
                typedef __nv_bfloat16 H;
                rg_ln_bwd_long_dx_kernel<H><<<(unsigned)rows, 512, 0, ctx->stream>>>((const H*)a.dy, (const H*)a.x, a.gamma, a.mean, a.rstd,
                                                                                    (H*)a.out, (long long)n);
                rg_ln_bwd_long_cols_kernel<H><<<cols, 256, 0, ctx->stream>>>((const H*)a.dy, (const H*)a.x, a.mean, a.rstd, a.parts, a.rows,
                                                                            (long long)n);
            }
            ctx->launches += 2;
        }
        rg_colsum_launch(ctx, a.parts, nparts, 2 * (long long)n, o[1]->data(), o[2]->data(), (long long)n);
    }
    RG_CUDA(cudaGetLastError());
    o.give({dx, dgamma, dbeta});
    return RG_OK;
}

// ---------------------------------------------------------------------------
// clipping by the global norm
// ---------------------------------------------------------------------------
// Two passes over all tensors: the sum of squares, then the scaled copy (the scale depends on every value, so 2 reads and a
// write per value is what has to move; what the last-level cache still holds of the first pass is read from there, because
// a CTA walks its pieces backwards in the second one; 38 tensors of 445 MB in bf16: 79 and 143 us, 5.7 and 6.2 TB/s).  The
// tensors are one list of pieces of CLIP_PIECE values; the table of tensors travels as a kernel parameter, so no copy
// precedes the launch.
// The sum is held in f64: an f32 square overflows from 1.8e19 and vanishes below 1e-23, and the sum of hundreds of millions
// of terms would lose digits.
#define CLIP_PIECE 8192
#define CLIP_TENSORS 256
struct clip_entry {
    const void* in;
    void* out;
    long long len;
    int first;  // number of the first piece
    int bf16;
};
struct clip_table {
    clip_entry e[CLIP_TENSORS];
    int n, pieces;
};

__device__ __forceinline__ int clip_find(const clip_table& t, int piece) {
    int lo = 0, hi = t.n - 1;  // the last tensor whose first piece is not after `piece`
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first <= piece) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double clip_block_sum(double v, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(RG_FULL_MASK, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) s += red[w];
    return s;
}

// Eight squares are added in f32 as a tree (at most 4 roundings on the way of each) and their sum joins the f64 total:
// one conversion and one f64 addition for eight values (a conversion for each bounded the kernel at 3.7 TB/s).  Where the
// f32 sum is zero or anywhere near the ends of its range, the eight go through f64 one by one.
__device__ __forceinline__ void clip_add8(double& acc, const float (&v)[8]) {
    const float a = fmaf(v[1], v[1], v[0] * v[0]), b = fmaf(v[3], v[3], v[2] * v[2]);
    const float c = fmaf(v[5], v[5], v[4] * v[4]), d = fmaf(v[7], v[7], v[6] * v[6]);
    const float s = (a + b) + (c + d);
    if (s > 0x1p-90f && s < 0x1p120f) {
        acc += (double)s;
    } else {
#pragma unroll 1
        for (int k = 0; k < 8; k++) {
            const double w = v[k];
            acc = fma(w, w, acc);
        }
    }
}

__global__ void __launch_bounds__(256) rg_clip_sumsq_kernel(const __grid_constant__ clip_table t, double* __restrict__ parts) {
    __shared__ double red[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    double acc = 0.0;
    for (int p = blockIdx.x; p < t.pieces; p += gridDim.x) {
        const clip_entry& e = t.e[clip_find(t, p)];
        const long long at = (long long)(p - e.first) * CLIP_PIECE;
        const int len = (int)min((long long)CLIP_PIECE, e.len - at);
        if (e.bf16) {
            const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(e.in) + at;
            if (len == CLIP_PIECE) {
                uint4 raw[4];
#pragma unroll
                for (int k = 0; k < 4; k++) raw[k] = reinterpret_cast<const uint4*>(src)[threadIdx.x + k * 256];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 4; j++) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                    clip_add8(acc, v);
                }
            } else {
                for (int i = threadIdx.x; i < len; i += 256) {
                    const double w = __bfloat162float(src[i]);
                    acc = fma(w, w, acc);
                }
            }
        } else {
            const float* src = static_cast<const float*>(e.in) + at;
            if (len == CLIP_PIECE) {
                float4 raw[8];
#pragma unroll
                for (int k = 0; k < 8; k++) raw[k] = reinterpret_cast<const float4*>(src)[threadIdx.x + k * 256];
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const float v[8] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w, raw[k + 1].x, raw[k + 1].y, raw[k + 1].z, raw[k + 1].w};
                    clip_add8(acc, v);
                }
            } else {
                for (int i = threadIdx.x; i < len; i += 256) {
                    const double w = src[i];
                    acc = fma(w, w, acc);
                }
            }
        }
    }
    acc = clip_block_sum(acc, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(256) rg_clip_scale_kernel(const __grid_constant__ clip_table t, const double* parts,
                                                            int nparts, float max_norm, float* __restrict__ norm_out) {
    __shared__ double red[8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += parts[i];
    s = clip_block_sum(s, red);
    const double norm = sqrt(s);  // may be beyond f32 where every gradient is inside
    // min(1, max / norm); a NaN norm fails the comparisons and stays, an infinite maximum leaves everything as it is, infinities
    // too.  A factor near the smallest normal f32 would lose digits: it is applied in two steps, the second one an exact power of
    // two.
    const double ratio = norm <= (double)max_norm ? 1.0 : (double)max_norm / norm;
    const bool tiny = ratio < 0x1p-100;
    const float c = (float)(tiny ? ratio * 0x1p64 : ratio), c2 = tiny ? 0x1p-64f : 1.f;
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
    const int turns = (t.pieces - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    for (int k = turns - 1; k >= 0; k--) {
        const int p = blockIdx.x + k * gridDim.x;
        const clip_entry& e = t.e[clip_find(t, p)];
        const long long at = (long long)(p - e.first) * CLIP_PIECE;
        const int len = (int)min((long long)CLIP_PIECE, e.len - at);
        if (e.bf16) {
            const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(e.in) + at;
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(e.out) + at;
#pragma unroll 4
            for (int i = threadIdx.x * 8; i + 8 <= len; i += 256 * 8) {
                float v[8];
                ln_load<__nv_bfloat16, 8>(src + i, v);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = v[j] * c * c2;
                ln_store<__nv_bfloat16, 8>(dst + i, v);
            }
            for (int i = (len & ~7) + threadIdx.x; i < len; i += 256) dst[i] = __float2bfloat16_rn(__bfloat162float(src[i]) * c * c2);
        } else {
            const float* src = static_cast<const float*>(e.in) + at;
            float* dst = static_cast<float*>(e.out) + at;
#pragma unroll 8
            for (int i = threadIdx.x * 4; i + 4 <= len; i += 256 * 4) {
                float v[4];
                ln_load<float, 4>(src + i, v);
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = v[j] * c * c2;
                ln_store<float, 4>(dst + i, v);
            }
            for (int i = (len & ~3) + threadIdx.x; i < len; i += 256) dst[i] = src[i] * c * c2;
        }
    }
}

extern "C" rg_status rg_clip_grad_norm(rg_ctx* ctx, const rg_storage* const* grads, size_t n, float max_norm, rg_storage** out,
                                       rg_storage** norm) {
    if (!ctx || !norm || (n && (!grads || !out))) return rg_fail(RG_ERR_INVALID_INPUT, "NULL argument");
    *norm = nullptr;
    for (size_t i = 0; i < n; i++) out[i] = nullptr;
    if (!(max_norm > 0.f)) return rg_fail(RG_ERR_INVALID_INPUT, "clip_grad_norm: max_norm must be positive");
    for (size_t i = 0; i < n; i++) {
        if (!grads[i]) return rg_fail(RG_ERR_INVALID_INPUT, "NULL argument");
        RG_TRY(rg_same_ctx(ctx, {grads[i]}));
        if (grads[i]->len / CLIP_PIECE > 0x3fffffff) return rg_fail(RG_ERR_SHAPE, "clip_grad_norm: a gradient of %zu values", grads[i]->len);
    }
    rg_op_guard g(ctx);
    RG_TRY(rg_not_capturing(ctx, "clip_grad_norm"));
    return rg_no_throw([&]() -> rg_status {
        // launches of up to CLIP_TENSORS tensors and 2^30 pieces each; empty gradients take no entry
        std::vector<std::unique_ptr<rg_storage>> made(n);
        std::vector<clip_table> tables(1);
        memset(&tables[0], 0, sizeof(clip_table));
        for (size_t i = 0; i < n; i++) {
            rg_storage* st = nullptr;
            RG_TRY(rg_alloc_storage(ctx, grads[i]->shape.data(), (int)grads[i]->shape.size(), &st, grads[i]->dtype));
            made[i].reset(st);
            if (!st->len) continue;
            const int pieces = (int)((st->len + CLIP_PIECE - 1) / CLIP_PIECE);
            if (tables.back().n == CLIP_TENSORS || tables.back().pieces + pieces > (1 << 30)) {
                tables.emplace_back();
                memset(&tables.back(), 0, sizeof(clip_table));
            }
            clip_table& t = tables.back();
            t.e[t.n++] = {grads[i]->raw(), st->raw(), (long long)st->len, t.pieces, grads[i]->dtype == RG_DTYPE_BF16};
            t.pieces += pieces;
        }
        rg_outputs<2> o;
        const size_t one = 1;
        RG_TRY(rg_alloc_storage(ctx, &one, 1, &o[0]));
        std::vector<int> ctas;
        int nparts = 0;
        for (const clip_table& t : tables) {
            ctas.push_back(std::max(1, std::min(t.pieces, ctx->sm_count * 8)));
            nparts += ctas.back();
        }
        const size_t words = (size_t)nparts * 2;
        RG_TRY(rg_alloc_storage(ctx, &words, 1, &o[1]));
        double* parts = static_cast<double*>(o[1]->raw());
        int at = 0;
        for (size_t k = 0; k < tables.size(); k++) {
            rg_clip_sumsq_kernel<<<ctas[k], 256, 0, ctx->stream>>>(tables[k], parts + at);
            at += ctas[k];
        }
        for (size_t k = tables.size(); k-- > 0;)  // the first one follows the sums directly and may start early
            rg_launch(k + 1 == tables.size(), rg_clip_scale_kernel, dim3(ctas[k]), dim3(256), 0, ctx->stream, tables[k], (const double*)parts, nparts,
                      max_norm, k ? nullptr : o[0]->data());
        ctx->launches += 2 * tables.size();
        RG_CUDA(cudaGetLastError());
        for (size_t i = 0; i < n; i++) out[i] = made[i].release();
        o.give({norm});
        return RG_OK;
    });
}

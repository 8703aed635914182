// Linear cross entropy on the tensor cores (sm_100a): the three contractions of rg_lce.cuh for many rows (lce_tc_kernel), and
// the logits of a few row tiles straight from w (lce_mid_kernel).
//
//   logits  z[R,V]  = x[R,D] w[D,V]      -> (maximum, sum) per row and tile, or dz of a piece of the vocabulary
//   dx      [R,D]   = dz[R,V] w[D,V]^T
//   dw      [D,V]   = x[R,D]^T dz[R,V], computed as its transpose dz^T x: V fills whole row tiles of 256, and the column
//                     tiles of D can be narrow
//
// Every operand is used as it lies in memory: tcgen05 takes a shared-memory tile either with the contraction axis
// contiguous ("K-major") or with the other axis contiguous ("MN-major"), so no transposed copy of x, w or dz exists.  TMA
// brings 64-element wide boxes (128-byte swizzle) of three-dimensional arrays [plane][row][column]; what lies outside is
// filled with zeros, which handles every ragged edge of R, D and V.
//
// bf16 inputs are one plane and are multiplied as they are, with accumulators of 256 to 768 of K for the loss and one for all of
// K where the result is rounded to bf16 (lt_chain).  dz is one bf16 plane too: its rounding (half a step, at most 2^-8 of each
// value) costs dx and dw about half of what their own rounding to bf16 does (8e-4 of their norm at 4096x1600x50257); a second
// plane would double the products that are most of the gradient's time.  The form for few rows, where no product is bound by the
// tensor cores, keeps dz in f32.
// f32 inputs are split into planes of 16 bits whose products are accumulated in f32:
//  * logits: two f16 planes, x = 2^-a (x0 + x1) with a power of two per row of x and one for w that bring the largest
//    magnitude to 2^14..2^15.  x0 + x1 holds 22 bits, or what is above 2^-39 of that largest magnitude, whichever is less exact;
//    three of the four products are taken, the fourth is below 2^-22 of the magnitudes.  The scales leave in the epilogue.
//    A logit is then off by up to 2^-38 D max|x| max|w| beside the 2^-21 of its own products, and only its absolute error counts
//    in a softmax: pairs are used while that stays below 2^-16 (lt_wide; roundings that do not all go the same way leave some
//    2^-23).  A single huge value - in a class that a bias of -inf takes out, or a channel that the other side leaves at zero -
//    would cost all other logits their digits; where the largest magnitudes allow that, lce_mid_kernel multiplies triples of
//    bf16 instead, which have f32's range.  Both launches are enqueued and the device decides, so the host does not wait for
//    the maxima.
//  * dx, dw: the sums run over the vocabulary and over the rows, where dz spans many orders of magnitude (a rare word's
//    gradient is a sum of tiny ones), so f16's range is not enough: three bf16 planes hold all 24 bits (each the leading 8 bits
//    of what the planes before leave), and six of the nine products are taken; the others are below 2^-21.
// The tensor core truncates when it adds to its f32 accumulator, always towards zero, so a long chain loses about 2^-25 of the
// running sum per step (measured: a relative error of 7e-7 at K = 768 and 1.4e-5 at K = 50304 for random signs).  For f32
// inputs the chain is therefore cut after every k-block of 64 (lt_seg): in each the small products come first and that of the
// leading planes last, and the epilogue warps add the result to their f32 registers with rounding.  Errors of the norm against
// 64 bits, 600 rows, 128x300: dx 4.4e-7, dw 4.5e-7, dbias 2.2e-7, lse 7e-8 (f32 operations: 6.4e-7, 5.2e-7, 1.5e-7, 7e-8); cut
// after every two blocks 1.4e-6, 1.4e-6, 6.5e-7, 2.0e-7, at the same speed for the loss and 1 % faster for the gradient.
#include "rg_lce.cuh"

#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>

#define LT_BM 256  // rows of a tile: 128 in each CTA of a pair
#define LT_BK 64
// k-blocks of 64 per accumulator for logits of bf16 inputs, where it is cut (lt_chain): the loss, dz where dbias is summed from it,
// and both where there is no more than one tile for each pair of CTAs
#define LT_CHAIN_FWD 12
#define LT_CHAIN_DZ 6
#define LT_CHAIN_ONE 4
#define LT_SPIN_LIMIT (1u << 22)
#define LT_STAGE_ALL 196608   // bytes of the operand ring
#define LT_MAX_STAGES 6
#define LT_SMEM_BYTES (LT_STAGE_ALL + 8 * 32 * 33 * 4 + 1024 + 256)

// Two CTAs (two SMs) work on one tile of 256 x BN: each holds 128 rows of A, half of the columns of B, and the accumulator
// of its 128 rows.  A k-block then costs an SM 128 x 64 + BN/2 x 64 values from L2 instead of 128 x 64 + BN x 64, which
// bounded the one-SM form (12.5 TB/s from L2, 1.09 PFLOP/s in bf16).
// Measured (PFLOP/s of the products that are multiplied; a library product of bf16 reaches 1.6, 1.37 for seconds on end):
// logits of 4096x768x50257 f32 1.50 (634 us, tensor pipe active 79 %), of 8192x768x50257 bf16 1.26 (503 us, 64 %; 447 us when
// nothing is brought from L2, 487 when the epilogue does nothing); gradient of 2048x768x50257 f32: dz 1.00 (474 us, 47 %; 340
// without its planes and column sums), dx and dw 1.33 (1,430 us, 62 to 66 %); of 4096x1600x50257 bf16: dz 1.37, dx and dw 1.24.
// PLANES: 1 bf16 values, 2 pairs of f16, 3 triples of bf16.  CUT: the accumulator is cut along K and the pieces are added in
// registers (always for f32 inputs); else the epilogue works on the columns as they come from tensor memory.
enum { LT_FWD = 0, LT_DZ = 1, LT_GRAD = 2 };
template <int PLANES, int EPI = LT_GRAD, bool CUT = PLANES != 1>
struct lt_shape {
    static constexpr int BN = PLANES == 3 ? 128 : 256;
    static constexpr int A_BYTES = 128 * LT_BK * 2, B_BYTES = BN / 2 * LT_BK * 2;  // of one CTA
    static constexpr int STAGE_BYTES = PLANES * (A_BYTES + B_BYTES);
    static constexpr int STAGES = LT_STAGE_ALL / STAGE_BYTES;  // 6, 3 or 2
    static constexpr int BUFFERS = 512 / BN;  // accumulators in tensor memory
    // Warp 0 copies, warp 1 multiplies, FIRST.. the eight epilogue warps.  Where pieces of 256 columns are added, a thread holds
    // 128 of them in registers, more than 12 warps get at launch, so registers move between whole groups of four warps: 384
    // threads x 168 at launch = 128 x (56 + 224 + 224).
    static constexpr bool MOVE_REGS = CUT && BN == 256;
    static constexpr int FIRST = MOVE_REGS ? 4 : 2, THREADS = 32 * (FIRST + 8);
};

// One contraction of a launch: C[M,N] = sum over K of A[m,k] B[n,k]
struct lt_prob {
    int M, N, K;
    int tiles_m, tiles_n, splits, kb_per;  // the K axis is cut into `splits` runs of kb_per 64-wide blocks
    int a_mn, b_mn;                        // 1: the M (N) axis is the contiguous one
    int a_k0, b_k0, b_n0;                  // where the piece of the vocabulary starts in A or B
};

struct lt_args {
    lt_prob p[2];
    int nprobs;
    int* counter;  // tiles handed out beyond the first of each CTA
    int* err;
    int R, D, V;
    int v0, vn;    // piece of the vocabulary: first column, number of columns
    const float* bias;
    const float *xscale, *wscale;  // PLANES 2: the scale of each row of x and of w, to be taken out of the logits
    const unsigned* largest;       // PLANES 2: no tile is worked on where lt_wide() says so
    const int* tgt;
    float2* parts;            // LT_FWD
    float* tz;
    const float* lse;         // LT_DZ
    __nv_bfloat16* dz;        // [plane][R][dz_pitch]: 1 plane for bf16, 3 for f32 inputs
    long long dz_pitch;
    float* dbparts;           // [LT_BM / 32 * tiles_m][dz_pitch] or NULL
    float* dxparts;           // LT_GRAD: [splits][R][D]
    int dx_add;               // add to what the pieces before left there
    int dx_t;                 // the first problem computes dx^T
    void* dw;                 // [D][V]
    float* dwparts;           // [splits][D][V], or NULL: the second problem's K axis is not cut
    int dw_bf16;
    const float* scal;
    int chain;                // PLANES 1, CUT: k-blocks per accumulator, at most
};

// f32 logits: do the largest finite magnitudes of w and x ask for more range than a pair of f16 has?  (A product beyond f32 is
// infinite here, and wide.)
__device__ __forceinline__ bool lt_wide(const unsigned* largest, int D) {
    return __uint_as_float(largest[0]) * __uint_as_float(largest[1]) * (float)D > 0x1p22f;
}

__device__ __forceinline__ uint32_t lt_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void lt_bar_init(uint64_t* b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(lt_smem(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void lt_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(lt_smem(b)) : "memory");
}
// the same place in the shared memory of CTA 0 of the pair
__device__ __forceinline__ uint32_t lt_leader(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(lt_smem(p)));
    return a;
}
__device__ __forceinline__ uint32_t lt_peer(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(lt_smem(p)), "r"(rank));
    return a;
}
// For what has been read into registers already (tensor memory after its wait, a tile number that has been used): nothing in
// memory is published, so no cluster-wide release - it would wait for every store of this thread that is still on its way.
__device__ __forceinline__ void lt_arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// ordered after what this thread has read and written before
__device__ __forceinline__ void lt_publish_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// e^(v + less) of two values: two roundings of the argument (2^-24 of it each) and the 2 steps of the exponential instruction
__device__ __forceinline__ float2 lt_exp2(float2 v, float2 less) {
    const float2 t = rg_mul2(rg_add2(v, less), make_float2(1.44269504088896341f, 1.44269504088896341f));
    float2 r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(t.y));
    return r;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool lt_wait(uint64_t* bar, uint32_t parity, int* err) {
    uint32_t ok = 0, spins = 0;
    while (true) {
        if (CLUSTER)
            asm volatile(
                "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(lt_smem(bar)), "r"(parity)
                : "memory");
        else
            asm volatile(
                "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(ok)
                : "r"(lt_smem(bar)), "r"(parity)
                : "memory");
        if (ok) return true;
        if (++spins > LT_SPIN_LIMIT) {
            atomicExch(err, 1);
            return false;
        }
    }
}
// by a whole warp: all of its lanes go on, or none does
template <bool CLUSTER = false>
__device__ __forceinline__ bool lt_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
    return __all_sync(RG_FULL_MASK, lt_wait<CLUSTER>(bar, parity, err));
}
// into this CTA's shared memory; the bytes are counted on a barrier of CTA 0
__device__ __forceinline__ void lt_tma(const CUtensorMap* map, void* dst, uint32_t bar, int x, int y, int plane) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            lt_smem(dst)),
        "l"(map), "r"(x), "r"(y), "r"(plane), "r"(bar)
        : "memory");
}
// Shared-memory descriptors, 128-byte swizzle.  K-major: rows of 64 elements (128 bytes), groups of 8 rows 1024 bytes
// apart.  MN-major: rows of 64 M (N) elements, one per k; groups of 8 k 1024 bytes apart, the next 64 M (N) elements 64
// rows (8192 bytes) further.
__device__ __forceinline__ uint64_t lt_desc(uint32_t addr, int mn) {
    uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
    if (mn) d |= (uint64_t)(8192 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void lt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
        "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrives on the barrier at this place in both CTAs once the MMAs issued so far are done
__device__ __forceinline__ void lt_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(lt_smem(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void lt_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void lt_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The leading 8 bits of a finite value as bf16 (truncated, so it cannot overflow); what is left is exact in f32.  Infinity
// and NaN go to the first plane as they are and leave nothing.
__device__ __forceinline__ void lt_split3(float v, uint32_t& h0, uint32_t& h1, uint32_t& h2) {
    const uint32_t b0 = __float_as_uint(v) & 0xffff0000u;
    const bool fin = (b0 & 0x7f800000u) != 0x7f800000u;
    const float r1 = fin ? v - __uint_as_float(b0) : 0.f;
    const uint32_t b1 = __float_as_uint(r1) & 0xffff0000u;
    const float r2 = r1 - __uint_as_float(b1);
    // a NaN whose leading bits alone would read as infinity stays a NaN
    h0 = (v != v) ? 0x7fc0u : b0 >> 16, h1 = b1 >> 16, h2 = __float_as_uint(r2) >> 16;
}

struct lt_tile {
    int prob, m, n, split;
};
template <int EPI>
__device__ __forceinline__ lt_tile lt_decode(const lt_args& e, int t) {
    lt_tile r;
    const int n0 = e.p[0].tiles_m * e.p[0].tiles_n * e.p[0].splits;
    if (EPI == LT_GRAD && t < n0) {  // dx: the column tiles of one row tile together (they share dz), one run of K after the other
        r.prob = 0;
        r.n = t % e.p[0].tiles_n, t /= e.p[0].tiles_n;
        r.m = t % e.p[0].tiles_m, r.split = t / e.p[0].tiles_m;
        return r;
    }
    if (EPI == LT_GRAD) {  // dw: the column tiles of one row tile together (they share dz)
        r.prob = 1, t -= n0;
        r.n = t % e.p[1].tiles_n, t /= e.p[1].tiles_n;
        r.m = t % e.p[1].tiles_m, r.split = t / e.p[1].tiles_m;
        return r;
    }
    // logits: the row tiles of one column tile together (they share w)
    r.prob = 0, r.split = 0;
    r.m = t % e.p[0].tiles_m, r.n = t / e.p[0].tiles_m;
    return r;
}
// Columns of a tile that are multiplied: the last tile of a row is as narrow as the matrix allows.
template <int PLANES>
__device__ __forceinline__ int lt_width(const lt_prob& p, int n) {
    return min(lt_shape<PLANES>::BN, (p.N - n * lt_shape<PLANES>::BN + 31) & ~31);
}

// How the nkb k-blocks of a tile are cut into accumulators: their number, and the k-blocks of accumulator sg.  Pairs have two
// accumulators in tensor memory, and the epilogue of the tile before (3,500 cycles) lasts longer than the products of two k-blocks
// (1,536 each); so of 8 k-blocks and more the first two accumulators take two each: loss of 1024x768x50257 280 -> 266 us, of 4096
// rows 818 to 857 -> 752 to 781; dx 4.0e-7 -> 6.5e-7 at worst (2500x512x300; f32 operations 9.9e-7).
template <int PLANES, bool CUT>
__device__ __forceinline__ int lt_segs(const lt_args& e, int nkb) {
    if (!CUT) return 1;
    return PLANES == 3 ? nkb : PLANES == 2 ? nkb - (nkb >= 8 ? 2 : 0) : (nkb + e.chain - 1) / e.chain;
}
template <int PLANES, bool CUT>
__device__ __forceinline__ int lt_seg(int nkb, int segs, int sg) {
    if (!CUT) return nkb;
    if (PLANES != 1) return PLANES == 2 && nkb >= 8 && sg < 2 ? 2 : 1;
    const int chain = (nkb + segs - 1) / segs;  // about the same for all
    return min(chain, nkb - sg * chain);
}

// What a thread keeps of its row while the columns of a tile pass by.
struct lt_row {
    int row;        // row of C
    int group;      // number of the warp's 32 rows
    bool live;      // inside the matrix
    int tgt;
    float lse, scale;
    lce_ms ms;
};

// 32 consecutive columns of one row per thread (32 rows per warp), starting at column `col` of the tile's matrix.
template <int PLANES, int EPI>
__device__ __forceinline__ void lt_columns(const lt_args& e, const lt_tile& t, lt_row& w, float (&v)[32], int col, float* stage) {
    const int lane = threadIdx.x & 31;
    if (EPI == LT_FWD || EPI == LT_DZ) {
        const int c = e.v0 + col, left = e.v0 + e.vn - c;  // vocabulary column of v[0]; columns inside the piece
        if (left <= 0 && EPI == LT_FWD) return;
        if (PLANES == 2) {  // an exact power of two
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] *= w.scale;
        }
        if (e.bias) {
            if (left >= 32) {
                const float4* b = reinterpret_cast<const float4*>(e.bias + c);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float4 q = __ldg(b + j);
                    v[4 * j] += q.x, v[4 * j + 1] += q.y, v[4 * j + 2] += q.z, v[4 * j + 3] += q.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (j < left) v[j] += e.bias[c + j];
            }
        }
        const bool here = w.live && w.tgt >= c && w.tgt < c + 32;
        const bool any = __any_sync(RG_FULL_MASK, here);
        if (EPI == LT_FWD) {
            if (left < 32) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (j >= left) v[j] = -INFINITY;
            }
            if (any && here) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (w.tgt == c + j) e.tz[w.row] = v[j];
            }
            float mx[4] = {w.ms.m, v[1], v[2], v[3]};
            mx[0] = fmaxf(mx[0], v[0]);
#pragma unroll
            for (int j = 4; j < 32; j++) mx[j & 3] = fmaxf(mx[j & 3], v[j]);
            const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const float ref = m == -INFINITY ? 0.f : m;
            const float2 less = make_float2(-ref, -ref);
            float2 s[2] = {make_float2(w.ms.s * lt_exp2(make_float2(w.ms.m, w.ms.m), less).x, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int j = 0; j < 32; j += 2) s[(j >> 1) & 1] = rg_add2(s[(j >> 1) & 1], lt_exp2(make_float2(v[j], v[j + 1]), less));
            w.ms = {m, (s[0].x + s[0].y) + (s[1].x + s[1].y)};
        } else {
            const bool dead = !w.live || w.tgt < 0;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float2 p = lt_exp2(make_float2(v[j], v[j + 1]), make_float2(-w.lse, -w.lse));
                v[j] = (dead || j >= left) ? 0.f : p.x, v[j + 1] = (dead || j + 1 >= left) ? 0.f : p.y;
            }
            if (any && here) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (w.tgt == c + j) v[j] -= 1.f;
            }
            if (col < e.dz_pitch) {
                // A thread holds 64 bytes of a row of each plane.  Stored from here, a warp's instruction would touch 32 lines
                // with 16 bytes each; through shared memory four lanes store the 64 bytes of a row together.
                constexpr int ZP = PLANES == 1 ? 1 : 3;
                unsigned char* rows_s = reinterpret_cast<unsigned char*>(stage);  // 32 rows of 64 bytes, 80 apart
                const int row0 = w.row - lane, rows = e.R - row0;
                float rest[32];
#pragma unroll
                for (int j = 0; j < 32; j++) rest[j] = v[j];
#pragma unroll
                for (int p = 0; p < ZP; p++) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint32_t h[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float a = rest[j + 2 * k], b = rest[j + 2 * k + 1];
                            if (PLANES == 1) {
                                const __nv_bfloat162 q = __floats2bfloat162_rn(a, b);
                                h[k] = *reinterpret_cast<const uint32_t*>(&q);
                            } else {  // the leading 16 bits; what they leave is exact and goes to the next plane
                                h[k] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                                rest[j + 2 * k] = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
                                rest[j + 2 * k + 1] = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
                            }
                        }
                        *reinterpret_cast<uint4*>(rows_s + lane * 80 + j * 2) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                    __syncwarp();
                    __nv_bfloat16* o = e.dz + ((long long)p * e.R + row0) * e.dz_pitch + col + (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = i * 8 + (lane >> 2);
                        if (r < rows)
                            *reinterpret_cast<uint4*>(o + r * e.dz_pitch) = *reinterpret_cast<const uint4*>(rows_s + r * 80 + (lane & 3) * 16);
                    }
                    __syncwarp();
                }
            }
            if (e.dbparts) {
                // sums over the warp's 32 rows: 31 halving exchanges leave column `lane` in each lane
#pragma unroll
                for (int half = 16; half >= 1; half >>= 1) {
                    const bool up = lane & half;
#pragma unroll
                    for (int i = 0; i < half; i++) {
                        const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
                        v[i] = keep + __shfl_xor_sync(RG_FULL_MASK, send, half);
                    }
                }
                if (lane < left) e.dbparts[(size_t)w.group * e.dz_pitch + col + lane] = v[0];
            }
        }
        return;
    }
    const lt_prob& p = e.p[t.prob];
    const int cols = min(32, p.N - col);
    if (t.prob == 1) {
        // dw^T: the lanes are neighbouring columns of dw, a register is a row of it, so a warp's store is contiguous
        if (!w.live) return;
        const float scale = e.dwparts ? 1.f : e.scal[1];
        const size_t at = (size_t)col * e.V + e.v0 + w.row;
        if (e.dwparts) {
            float* o = e.dwparts + (size_t)t.split * e.D * e.V + at;
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (j < cols) o[(size_t)j * e.V] = v[j];
        } else if (e.dw_bf16) {
            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(e.dw) + at;
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (j < cols) o[(size_t)j * e.V] = __float2bfloat16_rn(v[j] * scale);
        } else {
            float* o = static_cast<float*>(e.dw) + at;
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (j < cols) o[(size_t)j * e.V] = v[j] * scale;
        }
        return;
    }
    if (cols <= 0) return;
    if (e.dx_t) {  // the lanes are neighbouring columns of dx
        if (!w.live) return;
        float* o = e.dxparts + ((size_t)t.split * e.R + col) * e.D + w.row;
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (j < cols) o[(size_t)j * e.D] = e.dx_add ? o[(size_t)j * e.D] + v[j] : v[j];
        return;
    }
    // partial dx: through shared memory, so that a warp stores 32 consecutive columns of one row at a time
#pragma unroll
    for (int j = 0; j < 32; j++) stage[lane * 33 + j] = v[j];
    __syncwarp();
    const int row0 = w.row - lane;
    const int rows = min(32, p.M - row0);
    if (lane < cols) {
        float* o = e.dxparts + ((size_t)t.split * e.R + row0) * e.D + col + lane;
#pragma unroll 8
        for (int r = 0; r < rows; r++) {
            float s = stage[r * 33 + lane];
            if (e.dx_add) s += o[(size_t)r * e.D];
            o[(size_t)r * e.D] = s;
        }
    }
    __syncwarp();
}

template <int PLANES, int EPI, bool CUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(lt_shape<PLANES, EPI, CUT>::THREADS, 1)
lce_tc_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmA1,
              const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ lt_args e) {
    typedef lt_shape<PLANES, EPI, CUT> S;
    extern __shared__ unsigned char lt_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(lt_raw) + 1023) & ~(uintptr_t)1023);
    float* stage_all = reinterpret_cast<float*>(ring + LT_STAGE_ALL);
    uint64_t* full = reinterpret_cast<uint64_t*>(stage_all + 8 * 32 * 33);  // used in CTA 0
    uint64_t* empty = full + LT_MAX_STAGES;
    uint64_t* acc_full = empty + LT_MAX_STAGES;  // [4]
    uint64_t* acc_empty = acc_full + 4;          // [4], used in CTA 0
    uint64_t* sched_full = acc_empty + 4;        // [2]
    uint64_t* sched_empty = sched_full + 2;      // [2], used in CTA 0
    uint64_t* drain = sched_empty + 2;
    volatile int* sched_tile = reinterpret_cast<volatile int*>(drain + 1);  // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    int total = 0;
    for (int i = 0; i < e.nprobs; i++) total += e.p[i].tiles_m * e.p[i].tiles_n * e.p[i].splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < LT_MAX_STAGES; s++) lt_bar_init(&full[s], 1), lt_bar_init(&empty[s], 1);
        for (int b = 0; b < S::BUFFERS; b++) lt_bar_init(&acc_full[b], 1), lt_bar_init(&acc_empty[b], 16);
        for (int b = 0; b < 2; b++) {
            lt_bar_init(&sched_full[b], 1), lt_bar_init(&sched_empty[b], 18);  // MMA thread and epilogue warps; copy thread and epilogue warps
        }
        lt_bar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(lt_smem(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // the barriers of both CTAs exist before either uses the other's
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    // everything above needs nothing from the kernels before; from here on they are complete
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (PLANES == 2 && lt_wide(e.largest, e.D)) total = 0;  // lce_mid_kernel does all of it

    if (warp < S::FIRST) {
    if (S::MOVE_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
        // ===== one thread of each CTA brings its operands; that of CTA 0 also hands out the tiles to both =====
        if (lane == 0) {
            uint32_t it = 0, ti = 0;
            bool ok = true;
            int tile = blockIdx.x >> 1;
            while (true) {
                const uint32_t slot = ti & 1u;
                int next = 0;
                if (rank == 0) {
                    ok = lt_wait(&sched_empty[slot], ((ti >> 1) & 1u) ^ 1u, e.err);
                    if (!ok) break;
                    sched_tile[slot] = tile;
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(lt_peer(const_cast<int*>(&sched_tile[slot]), 1)), "r"(tile) : "memory");
                    lt_arrive(&sched_full[slot]);
                    lt_publish_at(lt_peer(&sched_full[slot], 1));
                    if (tile < total) next = (int)(gridDim.x >> 1) + atomicAdd(e.counter, 1);  // arrives while this tile is loaded
                } else {
                    ok = lt_wait<true>(&sched_full[slot], (ti >> 1) & 1u, e.err);
                    if (!ok) break;
                    tile = sched_tile[slot];
                    lt_publish_at(lt_leader(&sched_empty[slot]));  // after the read
                }
                ti++;
                if (tile >= total) break;
                const lt_tile t = lt_decode<EPI>(e, tile);
                const lt_prob& p = e.p[t.prob];
                const CUtensorMap* ma = (EPI == LT_GRAD && t.prob) ? &tmA1 : &tmA0;
                const CUtensorMap* mb = (EPI == LT_GRAD && t.prob) ? &tmB1 : &tmB0;
                const int m0 = t.m * LT_BM + (int)rank * 128, n0 = t.n * S::BN + (int)rank * (lt_width<PLANES>(p, t.n) / 2);
                const int kb0 = t.split * p.kb_per, kb1 = min(kb0 + p.kb_per, (p.K + LT_BK - 1) / LT_BK);
                for (int kb = kb0; kb < kb1; kb++, it++) {
                    const int s = it % S::STAGES;
                    ok = lt_wait(&empty[s], ((it / S::STAGES) & 1u) ^ 1u, e.err);
                    if (!ok) break;
                    const uint32_t bar = lt_leader(&full[s]);
                    if (rank == 0)  // for the bytes of both CTAs (those of CTA 1 may already be arriving: the phase waits for this)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(lt_smem(&full[s])),
                                     "r"((uint32_t)(2 * S::STAGE_BYTES))
                                     : "memory");
                    unsigned char* a = ring + s * S::STAGE_BYTES;
                    unsigned char* b = a + PLANES * S::A_BYTES;
                    const int k = kb * LT_BK;
#pragma unroll
                    for (int pl = 0; pl < PLANES; pl++) {
                        if (p.a_mn) {
                            lt_tma(ma, a + pl * S::A_BYTES, bar, m0, k, pl);
                            lt_tma(ma, a + pl * S::A_BYTES + 8192, bar, m0 + 64, k, pl);
                        } else {
                            lt_tma(ma, a + pl * S::A_BYTES, bar, p.a_k0 + k, m0, pl);
                        }
                        if (p.b_mn) {
#pragma unroll
                            for (int j = 0; j < S::BN / 128; j++)
                                lt_tma(mb, b + pl * S::B_BYTES + j * 8192, bar, p.b_n0 + n0 + j * 64, k, pl);
                        } else {
                            lt_tma(mb, b + pl * S::B_BYTES, bar, p.b_k0 + k, n0, pl);
                        }
                    }
                }
                if (!ok) break;
                tile = next;
            }
            if (!ok)  // a wait gave up: the copies in flight land before the CTA's memory goes away
                for (uint32_t i = it > (uint32_t)S::STAGES ? it - S::STAGES : 0; i < it; i++)
                    lt_wait(&empty[i % S::STAGES], (i / S::STAGES) & 1u, e.err);
        }
    } else if (warp == 1) {
        // ===== one thread of CTA 0 issues the MMAs of the pair =====
        if (lane == 0 && rank == 0) {
            uint32_t it = 0, ti = 0, seg = 0;
            bool ok = true;
            while (true) {
                const uint32_t slot = ti & 1u;
                ok = lt_wait(&sched_full[slot], (ti >> 1) & 1u, e.err);
                if (!ok) break;
                const int tile = sched_tile[slot];
                lt_arrive(&sched_empty[slot]);
                ti++;
                if (tile >= total) break;
                const lt_tile t = lt_decode<EPI>(e, tile);
                const lt_prob& p = e.p[t.prob];
                const int kb0 = t.split * p.kb_per, nkb = min(p.kb_per, (p.K + LT_BK - 1) / LT_BK - kb0);
                // D f32, A and B bf16 (f16), their majors, N, M
                const uint32_t idesc = (1u << 4) | (PLANES == 2 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)p.a_mn << 15) | ((uint32_t)p.b_mn << 16) |
                                       ((uint32_t)(lt_width<PLANES>(p, t.n) >> 3) << 17) | ((uint32_t)(LT_BM >> 4) << 24);
                const uint32_t astep = p.a_mn ? 2048 : 32, bstep = p.b_mn ? 2048 : 32;  // 16 elements of K
                const int segs = lt_segs<PLANES, CUT>(e, nkb);
                for (int sg = 0; sg < segs && ok; sg++, seg++) {
                    const uint32_t buf = seg % S::BUFFERS;
                    ok = lt_wait(&acc_empty[buf], ((seg / S::BUFFERS) & 1u) ^ 1u, e.err);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t d = tmem + buf * S::BN;
                    const int blocks = lt_seg<PLANES, CUT>(nkb, segs, sg);
                    for (int kb = 0; kb < blocks; kb++, it++) {
                        const int s = it % S::STAGES;
                        ok = lt_wait(&full[s], (it / S::STAGES) & 1u, e.err);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t a = lt_smem(ring + s * S::STAGE_BYTES), b = a + PLANES * S::A_BYTES;
                        // pairs of planes, the smallest products first
                        constexpr int PRODUCTS = PLANES == 1 ? 1 : PLANES == 2 ? 3 : 6;
                        constexpr int pa[3][6] = {{0}, {0, 1, 0}, {0, 2, 1, 0, 1, 0}}, pb[3][6] = {{0}, {1, 0, 0}, {2, 0, 1, 1, 0, 0}};
#pragma unroll
                        for (int pr = 0; pr < PRODUCTS; pr++)
#pragma unroll
                            for (int k = 0; k < LT_BK / 16; k++)
                                lt_mma(d, lt_desc(a + pa[PLANES - 1][pr] * S::A_BYTES + k * astep, p.a_mn),
                                       lt_desc(b + pb[PLANES - 1][pr] * S::B_BYTES + k * bstep, p.b_mn), idesc, kb > 0 || pr > 0 || k > 0);
                        lt_commit(&empty[s]);
                    }
                    if (ok) lt_commit(&acc_full[buf]);
                }
                if (!ok) break;
            }
            if (!ok) {  // MMAs in flight finish before the tensor memory is given back
                lt_commit(drain);
                lt_wait(drain, 0, e.err);
            }
        }
    }
    } else {
        if (S::MOVE_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ===== epilogue warps: TMEM lane quarter = warp % 4, four for the left half of the columns, four for the right =====
        constexpr int HALF = S::BN / 2;
        const int q = warp & 3, half = warp < S::FIRST + 4 ? 0 : 1;
        float* stage = stage_all + (warp - S::FIRST) * 32 * 33;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + half * HALF;
        uint32_t ti = 0, seg = 0;
        bool ok = true;
        while (true) {
            const uint32_t slot = ti & 1u;
            ok = lt_wait_warp<true>(&sched_full[slot], (ti >> 1) & 1u, e.err);
            if (!ok) break;
            // lane 0's value goes to all lanes, so its read is complete before it hands the slot back (the arrival alone would not
            // wait for a read that is queued behind this warp's stores)
            const int tile = __shfl_sync(RG_FULL_MASK, lane == 0 ? sched_tile[slot] : 0, 0);
            if (lane == 0) lt_arrive_at(lt_leader(&sched_empty[slot]));
            ti++;
            if (tile >= total) break;
            const lt_tile t = lt_decode<EPI>(e, tile);
            const lt_prob& p = e.p[t.prob];
            lt_row w;
            w.group = t.m * (LT_BM / 32) + (int)rank * 4 + q;
            w.row = w.group * 32 + lane;
            w.live = w.row < p.M;
            w.ms = {-INFINITY, 0.f};
            w.tgt = (EPI != LT_GRAD && w.live) ? e.tgt[w.row] : -1;
            w.lse = (EPI == LT_DZ && w.live) ? e.lse[w.row] : 0.f;
            w.scale = (PLANES == 2 && w.live) ? e.xscale[w.row] * e.wscale[0] : 0.f;
            const int c0 = t.n * S::BN + half * HALF;
            const int kb0 = t.split * p.kb_per, nkb = min(p.kb_per, (p.K + LT_BK - 1) / LT_BK - kb0);
            const int segs = lt_segs<PLANES, CUT>(e, nkb);
            float acc[CUT ? HALF / 32 : 2][32];
            if (CUT)
#pragma unroll
                for (int c = 0; c < HALF / 32; c++)
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[c][j] = 0.f;
            for (int sg = 0; sg < segs; sg++, seg++) {
                const uint32_t buf = seg % S::BUFFERS;
                ok = lt_wait_warp(&acc_full[buf], (seg / S::BUFFERS) & 1u, e.err);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t ta = taddr + buf * S::BN;
                if constexpr (!CUT) {
                    // the next 32 columns are on their way while these are worked on
                    lt_ld32(ta, acc[0]);
#pragma unroll 1
                    for (int c = 0; c < HALF / 32; c += 2) {
                        lt_ld_wait();
                        lt_ld32(ta + (c + 1) * 32, acc[1]);
                        lt_columns<PLANES, EPI>(e, t, w, acc[0], c0 + c * 32, stage);
                        lt_ld_wait();
                        if (c + 2 < HALF / 32) {
                            lt_ld32(ta + (c + 2) * 32, acc[0]);
                        } else {  // the accumulator has been read: hand it back before the last columns are worked on
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) lt_arrive_at(lt_leader(&acc_empty[buf]));
                        }
                        lt_columns<PLANES, EPI>(e, t, w, acc[1], c0 + (c + 1) * 32, stage);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < HALF / 32; c += 2) {
                        float block[2][32];
                        lt_ld32(ta + c * 32, block[0]);
                        lt_ld32(ta + c * 32 + 32, block[1]);
                        lt_ld_wait();
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                const float2 t = rg_add2(make_float2(acc[c + h][j], acc[c + h][j + 1]), make_float2(block[h][j], block[h][j + 1]));
                                acc[c + h][j] = t.x, acc[c + h][j + 1] = t.y;
                            }
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) lt_arrive_at(lt_leader(&acc_empty[buf]));
                }
            }
            if (!ok) break;
            if constexpr (CUT) {
                // one copy of the epilogue's code: the next 32 columns move into its registers (four copies, 130 KB of
                // instructions, took a single tile from 14 to 26 us)
#pragma unroll 1
                for (int c = 0; c < HALF / 32; c++) {
                    lt_columns<PLANES, EPI>(e, t, w, acc[0], c0 + c * 32, stage);
#pragma unroll
                    for (int k = 1; k < HALF / 32; k++)
#pragma unroll
                        for (int j = 0; j < 32; j++) acc[k - 1][j] = acc[k][j];
                }
            }
            if (EPI == LT_FWD && w.live) e.parts[(size_t)(t.n * 2 + half) * e.R + w.row] = make_float2(w.ms.m, w.ms.s);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // neither CTA leaves (or gives back its tensor memory) while the other may still reach into it
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---------------------------------------------------------------------------
// some rows: logits from w as it lies in memory
// ---------------------------------------------------------------------------
// With few row tiles the kernel above waits for the planes of w: a pass for their scale, one that writes 4 bytes for every 4 it
// reads, and reading those.  Here sixteen warps read w once, with plain loads (a row of an odd vocabulary starts on any 2 or
// 4 bytes), split it in registers and store the planes to tensor memory, where it is the A operand; only x, which is small,
// is packed before.  The sides are swapped: z^T = w^T x^T, 128 columns of the vocabulary are the lanes of a tile and 64 (32)
// rows of x its columns, so a thread of the epilogue holds one column of the vocabulary.  f32 is split into bf16 triples (six
// products; no scale: what a value below 2^-117 has in its last bits is lost, bf16 has nothing smaller), the accumulator is
// cut every 128 of K and the sum taken in registers with rounding.
// Bound by the instructions of the split and by what one k-block ahead leaves in flight: 41 us for [17,768]x[768,50257], 3.8
// TB/s of w (bf16 26 us, 2.9 TB/s); dz of 64 rows 53 us.  Steps, us for f32 and bf16: w through shared memory 62, 40 (A was read from there for
// each product); through tensor memory 61, 37; the MMA warp's loops walked by all lanes, so that an MMA's operands are
// uniform values instead of 14 instructions each, 44, 36; k-blocks of 128 instead of 64, 41, 26.
// Four epilogue warps, sixteen that convert, one that copies x, one that multiplies, two that only give their registers away:
// 768 threads x 80 at launch = 128 x 152 + 512 x 64 + 128 x 72.
#define LM_THREADS 768
#define LM_BK 128

template <typename T>
struct lm_shape {
    static constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
    static constexpr int X_BYTES = 64 * LM_BK * 2, STAGE_BYTES = PLANES * X_BYTES;  // shared memory: x
    static constexpr int W_COLS = LM_BK / 2, STAGE_COLS = PLANES * W_COLS;  // tensor memory: w, two values to a column's word
    static constexpr int STAGES = PLANES == 3 ? 2 : 4;
    // accumulators of 64 columns: the tensor core goes on while the epilogue works on a tile's sums
    static constexpr int BUFFERS = (512 - STAGES * STAGE_COLS) / 64;
    static constexpr int CHAIN = PLANES == 3 ? 1 : LT_CHAIN_ONE * LT_BK / LM_BK;  // k-blocks per accumulator
    static constexpr int SMEM = STAGES * STAGE_BYTES + 2 * 4 * 64 * 8 + 1024 + 256;
};

struct lm_args {
    const void* w;   // [D][V]
    int R, D, V;
    int tile;        // columns of the vocabulary per tile, at most 128
    int tiles, groups;  // of columns; of 64 rows
    int v0, cols;    // columns that are covered: from v0, those of dz or of the partial sums
    const unsigned* largest;  // not NULL: only where lt_wide() says so, in place of lce_tc_kernel
    int* err;
    const float* bias;
    const int* tgt;
    float2* parts;   // LT_FWD
    float* tz;
    const float* lse;  // LT_DZ
    __nv_bfloat16* dz;  // [3][R][cols]
    float* dbparts;  // [groups * db_rows][cols] or NULL
    int db_rows;     // rows of dbparts for each group: the sums, then zeros
};

// A from tensor memory
__device__ __forceinline__ void lm_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
        "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void lm_st16(uint32_t taddr, const uint32_t (&h)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]), "r"(h[8]), "r"(h[9]), "r"(h[10]), "r"(h[11]),
        "r"(h[12]), "r"(h[13]), "r"(h[14]), "r"(h[15])
        : "memory");
}
__device__ __forceinline__ void lm_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(lt_smem(bar)) : "memory");
}
__device__ __forceinline__ void lm_tma(const CUtensorMap* map, void* dst, uint64_t* bar, int x, int y, int plane) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     lt_smem(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(plane), "r"(lt_smem(bar))
                 : "memory");
}
__device__ __forceinline__ uint32_t lm_bits(const float* p) { return __float_as_uint(__ldg(p)); }
__device__ __forceinline__ uint32_t lm_bits(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const unsigned short*>(p)); }

// sums over the warp of 32 values per lane: 31 halving exchanges leave that of value `lane` in each lane
__device__ __forceinline__ float lm_across(float (&v)[32], int lane) {
#pragma unroll
    for (int half = 16; half >= 1; half >>= 1) {
        const bool up = lane & half;
#pragma unroll
        for (int i = 0; i < half; i++) {
            const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(RG_FULL_MASK, send, half);
        }
    }
    return v[0];
}
__device__ __forceinline__ float lm_max(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

template <typename T, int EPI>
__global__ void __launch_bounds__(LM_THREADS, 1) lce_mid_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ lm_args e) {
    typedef lm_shape<T> S;
    extern __shared__ unsigned char lm_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(lm_raw) + 1023) & ~(uintptr_t)1023);
    float2* sums = reinterpret_cast<float2*>(ring + S::STAGES * S::STAGE_BYTES);  // [2][4][64]
    uint64_t* full_w = reinterpret_cast<uint64_t*>(sums + 2 * 4 * 64);
    uint64_t* full_x = full_w + S::STAGES;
    uint64_t* empty = full_x + S::STAGES;
    uint64_t* acc_full = empty + S::STAGES;  // [S::BUFFERS]
    uint64_t* acc_empty = acc_full + S::BUFFERS;
    uint64_t* merge = acc_empty + S::BUFFERS;
    uint64_t* drain = merge + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    // the same in all lanes, and known to be: what follows from it is computed once per warp
    const int warp = __shfl_sync(RG_FULL_MASK, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (e.largest) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (!lt_wide(e.largest, e.D)) return;
    }
    const int total = e.tiles * e.groups, nkb = (e.D + LM_BK - 1) / LM_BK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; s++) lt_bar_init(&full_w[s], 16), lt_bar_init(&full_x[s], 1), lt_bar_init(&empty[s], 1);
        for (int b = 0; b < S::BUFFERS; b++) lt_bar_init(&acc_full[b], 1), lt_bar_init(&acc_empty[b], 4);
        lt_bar_init(merge, 4);
        lt_bar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 21) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(lt_smem(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp >= 4 && warp < 20) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ===== w: a thread takes one column of the vocabulary (its lane of tensor memory) and 32 of the 128 rows of a k-block, so
        // 32 lanes read side by side.  The values of the next k-block are loaded into the registers that the conversion of this one
        // frees. =====
        const int row = ((warp - 4) >> 2) * 32;
        const T *w = static_cast<const T*>(e.w), *p = nullptr;
        int t = blockIdx.x, kb = 0;  // of the loads, a k-block ahead
        const uint32_t blocks = (uint32_t)((total - t + (int)gridDim.x - 1) / (int)gridDim.x) * nkb;
        auto place = [&]() {
            const int v0 = e.v0 + (t / e.groups) * e.tile;
            p = w + (size_t)row * e.V + min(v0 + (warp & 3) * 32 + lane, min(e.V, v0 + e.tile) - 1);
        };
        uint32_t raw[32];
        auto load = [&]() {
            const T* q = p + (size_t)(kb * LM_BK) * e.V;
            const int rows = t < total ? e.D - kb * LM_BK - row : 0;
            if (rows >= 32) {
#pragma unroll
                for (int j = 0; j < 32; j++) raw[j] = lm_bits(q + (size_t)j * e.V);
            } else {
#pragma unroll
                for (int j = 0; j < 32; j++) raw[j] = j < rows ? lm_bits(q + (size_t)j * e.V) : 0u;
            }
        };
        place();
        load();
        for (uint32_t it = 0; it < blocks; it++) {
            const int s = it % S::STAGES;
            if (++kb == nkb) {
                kb = 0, t += gridDim.x;
                if (t < total) place();
            }
            if (!lt_wait_warp(&empty[s], ((it / S::STAGES) & 1u) ^ 1u, e.err)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + s * S::STAGE_COLS + row / 2;
#pragma unroll
            for (int q = 0; q < S::PLANES; q++) {
                // f32: the leading 16 bits, and what they leave, which is exact (infinity leaves a NaN, NaN stays one)
                uint32_t h[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    uint32_t &a = raw[2 * j], &b = raw[2 * j + 1];
                    h[j] = __byte_perm(a, b, S::PLANES == 1 ? 0x5410 : 0x7632);
                    a = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xffff0000u));
                    b = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xffff0000u));
                }
                lm_st16(to + q * S::W_COLS, h);
            }
            load();
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) lt_arrive(&full_w[s]);
        }
    } else if (warp >= 20) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 20 && lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < total; t += gridDim.x)
                for (int kb = 0; kb < nkb; kb++, it++) {
                    const int s = it % S::STAGES;
                    ok = lt_wait(&empty[s], ((it / S::STAGES) & 1u) ^ 1u, e.err);
                    if (!ok) break;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(lt_smem(&full_x[s])),
                                 "r"((uint32_t)(S::PLANES * S::X_BYTES))
                                 : "memory");
                    unsigned char* x = ring + s * S::STAGE_BYTES;
#pragma unroll
                    for (int p = 0; p < 2 * S::PLANES; p++)  // 64 columns of a plane each; what lies outside x is filled with zeros
                        lm_tma(&tmX, x + p * (S::X_BYTES / 2), &full_x[s], kb * LM_BK + (p & 1) * 64, (t % e.groups) * 64, p >> 1);
                }
            // the copies have landed before the CTA's memory goes away, also where a wait gave up
            for (uint32_t i = it > (uint32_t)S::STAGES ? it - S::STAGES : 0; i < it; i++)
                lt_wait(&full_x[i % S::STAGES], (i / S::STAGES) & 1u, e.err);
        }
        if (warp == 21) {
            // The whole warp walks the loops and one lane issues: an MMA's operands then are uniform values.  (One thread in the
            // loops alone took 14 instructions, 30 ns, for each MMA to bring them there.)
            uint32_t it = 0, seg = 0, one;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
            bool ok = true;
            for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
                const int rows = min(64, e.R - (t % e.groups) * 64);
                // D f32, A and B bf16, N, M = 128
                const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(rows > 32 ? 8 : 4) << 17) | (8u << 24);
                for (int kb0 = 0; ok && kb0 < nkb; kb0 += S::CHAIN, seg++) {
                    const uint32_t buf = seg % S::BUFFERS;
                    ok = lt_wait_warp(&acc_empty[buf], ((seg / S::BUFFERS) & 1u) ^ 1u, e.err);
                    const uint32_t d = tmem + S::STAGES * S::STAGE_COLS + buf * 64;
                    const int end = min(S::CHAIN, nkb - kb0);
                    for (int kb = 0; ok && kb < end; kb++, it++) {
                        const int s = it % S::STAGES;
                        ok = lt_wait_warp(&full_x[s], (it / S::STAGES) & 1u, e.err) && lt_wait_warp(&full_w[s], (it / S::STAGES) & 1u, e.err);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t a = tmem + s * S::STAGE_COLS;
                        const uint64_t b = lt_desc(lt_smem(ring + s * S::STAGE_BYTES), 0);
                        constexpr int PRODUCTS = S::PLANES == 1 ? 1 : 6;
                        constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};  // the smallest products first
                        if (one) {
#pragma unroll
                            for (int pr = 0; pr < PRODUCTS; pr++)
#pragma unroll
                                for (int k = 0; k < LM_BK / 16; k++)
                                    lm_mma(d, a + (S::PLANES == 1 ? 0 : pa[pr]) * S::W_COLS + k * 8,
                                           b + ((S::PLANES == 1 ? 0 : pb[pr]) * S::X_BYTES + (k >> 2) * (S::X_BYTES / 2) + (k & 3) * 32) / 16,
                                           idesc, kb > 0 || pr > 0 || k > 0);
                            lm_commit(&empty[s]);
                            if (kb + 1 == end) lm_commit(&acc_full[buf]);
                        }
                    }
                }
            }
            if (one) lm_commit(drain);  // MMAs in flight finish before the tensor memory is given back
            lt_wait(drain, 0, e.err);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        // ===== epilogue: a thread holds one column of the vocabulary, 64 rows in two halves =====
        const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16) + S::STAGES * S::STAGE_COLS;
        const int place = warp * 32 + lane;
        uint32_t it = 0, nt = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x, nt++) {
            const int row0 = (t % e.groups) * 64, rows = min(64, e.R - row0), at = (t / e.groups) * e.tile, v0 = e.v0 + at;
            const int c = v0 + place;
            const bool mine = place < e.tile && at + place < e.cols, live = mine && c < e.V;
            const float bias = e.bias && live ? e.bias[c] : 0.f;
            float acc[2][32];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < 32; j++) acc[h][j] = 0.f;
            for (int kb = 0; kb < nkb; kb += S::CHAIN, it++) {
                const uint32_t buf = it % S::BUFFERS;
                ok = lt_wait_warp(&acc_full[buf], (it / S::BUFFERS) & 1u, e.err);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (h && rows <= 32) break;
                    float block[32];
                    lt_ld32(taddr + buf * 64 + h * 32, block);
                    lt_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 q = rg_add2(make_float2(acc[h][j], acc[h][j + 1]), make_float2(block[j], block[j + 1]));
                        acc[h][j] = q.x, acc[h][j + 1] = q.y;
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) lt_arrive(&acc_empty[buf]);
            }
            if (!ok) break;
            float db = 0.f;
            float2* mine_s = sums + ((nt & 1) * 4 + warp) * 64;
#pragma unroll 1
            for (int h = 0; h * 32 < rows; h++) {
                const int r0 = row0 + h * 32, left = min(32, e.R - r0);
                float(&v)[32] = acc[0];
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] += bias;
                const int tgt = lane < left ? e.tgt[r0 + lane] : -1;  // of row `lane`
                const bool hits = __any_sync(RG_FULL_MASK, tgt >= v0 && tgt < v0 + e.tile);  // a row has its target in the tile
                if (EPI == LT_FWD) {
                    if (hits) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (__shfl_sync(RG_FULL_MASK, tgt, j) == c && live) e.tz[r0 + j] = v[j];
                    }
                    float m = 0.f;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        v[j] = live ? v[j] : -INFINITY, v[j + 1] = live ? v[j + 1] : -INFINITY;
                        const float m0 = lm_max(v[j]), m1 = lm_max(v[j + 1]);
                        const float2 q = lt_exp2(make_float2(v[j], v[j + 1]), make_float2(m0 == -INFINITY ? 0.f : -m0, m1 == -INFINITY ? 0.f : -m1));
                        v[j] = q.x, v[j + 1] = q.y;
                        m = lane == j ? m0 : lane == j + 1 ? m1 : m;
                    }
                    mine_s[h * 32 + lane] = make_float2(m, lm_across(v, lane));
                } else {
                    const float lse = lane < left ? __ldg(e.lse + r0 + lane) : 0.f;
                    const unsigned dead = __ballot_sync(RG_FULL_MASK, tgt < 0);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 less = make_float2(-__shfl_sync(RG_FULL_MASK, lse, j), -__shfl_sync(RG_FULL_MASK, lse, j + 1));
                        const float2 q = lt_exp2(make_float2(v[j], v[j + 1]), less);
                        v[j] = (dead >> j & 1) || !live ? 0.f : q.x, v[j + 1] = (dead >> (j + 1) & 1) || !live ? 0.f : q.y;
                    }
                    if (hits) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (__shfl_sync(RG_FULL_MASK, tgt, j) == c && live) v[j] -= 1.f;
                    }
                    // Neighbouring lanes hold neighbouring columns: for each two rows they exchange halves, so an even lane stores
                    // two columns of the first row and an odd lane of the second (e.cols, e.tile and at are even).
                    const bool odd = lane & 1;
                    const size_t plane = (size_t)e.R * e.cols;
                    unsigned short* z = reinterpret_cast<unsigned short*>(e.dz + (size_t)(r0 + odd) * e.cols + (at + place - odd));
#pragma unroll
                    for (int j = 0; j < 32; j += 2, z += 2 * (size_t)e.cols) {
                        float d0 = v[j], d1 = v[j + 1];
                        db += d0, db += d1;
#pragma unroll
                        for (int p = 0; p < 3; p++) {
                            const uint32_t h = __byte_perm(__float_as_uint(d0), __float_as_uint(d1), 0x7632);  // rows j | j + 1
                            const uint32_t other = __shfl_xor_sync(RG_FULL_MASK, h, 1);
                            if (mine && j + odd < left)
                                *reinterpret_cast<uint32_t*>(z + p * plane) = odd ? __byte_perm(other, h, 0x7632) : __byte_perm(h, other, 0x5410);
                            d0 -= __uint_as_float(__float_as_uint(d0) & 0xffff0000u);
                            d1 -= __uint_as_float(__float_as_uint(d1) & 0xffff0000u);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 32; j++) acc[0][j] = acc[1][j];
            }
            if (EPI == LT_FWD) {  // the four warps' columns; the other half of `sums` is still being read for the tile before
                __syncwarp();
                if (lane == 0) lt_arrive(merge);
                ok = lt_wait_warp(merge, nt & 1u, e.err);
                if (!ok) break;
                const int r = threadIdx.x;
                if (r < rows) {
                    lce_ms a = {-INFINITY, 0.f};
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const float2 b = sums[((nt & 1) * 4 + q) * 64 + r];
                        a = lce_merge(a, {b.x, b.y});
                    }
                    e.parts[(size_t)(t / e.groups) * e.R + row0 + r] = make_float2(a.m, a.s);
                }
            } else if (e.dbparts && live) {
                float* o = e.dbparts + (size_t)(t % e.groups) * e.db_rows * e.cols + at + place;
                o[0] = db;
                for (int k = 1; k < e.db_rows; k++) o[(size_t)k * e.cols] = 0.f;
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 21) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------
// A bf16 matrix whose rows TMA cannot address (they do not start on 16-byte boundaries), copied to such rows (768 x 50257: 26
// us, 5.9 TB/s).
__global__ void __launch_bounds__(256) lt_align_kernel(const __nv_bfloat16* __restrict__ src, long long rows, int cols, int pitch,
                                                       __nv_bfloat16* __restrict__ dst) {
    rg_pdl_sync();
    const int groups = pitch / 8;
    const long long n = rows * groups, stride = (long long)gridDim.x * 256, total = rows * cols;
    const unsigned short* in = reinterpret_cast<const unsigned short*>(src);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
        const long long r = i / groups;
        const int c = (int)(i - r * groups) * 8;
        // eight values from two aligned loads (the second is a neighbour's first); what lies beyond the row is never read
        const long long at = r * cols + c, base = at & ~7ll;
        const int shift = (int)(at & 7);
        uint32_t h[4];
        if (base + 16 <= total) {
            const uint4 p = *reinterpret_cast<const uint4*>(in + base), q = *reinterpret_cast<const uint4*>(in + base + 8);
            const uint32_t w[9] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w, 0u};
            const int words = shift >> 1, bits = (shift & 1) * 16;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t lo = words == 0 ? w[k] : words == 1 ? w[k + 1] : words == 2 ? w[k + 2] : w[k + 3];
                const uint32_t hi = words == 0 ? w[k + 1] : words == 1 ? w[k + 2] : words == 2 ? w[k + 3] : w[k + 4];
                h[k] = __funnelshift_r(lo, hi, bits);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t a = at + 2 * k < total ? in[at + 2 * k] : 0u, b = at + 2 * k + 1 < total ? in[at + 2 * k + 1] : 0u;
                h[k] = a | (b << 16);
            }
        }
        *reinterpret_cast<uint4*>(dst + r * pitch + c) = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// The scale of a group of values with the largest finite magnitude m: 2^a with m 2^a in [2^14, 2^15), and 2^-a.  The exponent
// stays where both are normal numbers.
__device__ __forceinline__ float2 lt_scale(float m) {
    const int e = m > 0.f ? (int)(__float_as_uint(m) >> 23) - 127 : 14;  // subnormal: -127
    const int a = min(14 - e, 126);
    return make_float2(__int_as_float((a + 127) << 23), __int_as_float((127 - a) << 23));
}
__device__ __forceinline__ float lt_finite_abs(float v) {
    const float a = fabsf(v);
    return a <= 3.4028235e38f ? a : 0.f;  // infinity and NaN do not take part in the scale
}
// v 2^a as two f16: nearest, and nearest to what is left.  Infinity and NaN leave nothing.
__device__ __forceinline__ void lt_split2(float v, float scale, uint32_t& h0, uint32_t& h1) {
    const float s = v * scale;
    const __half a = __float2half_rn(s);
    const float r = s - __half2float(a);
    const __half b = __float2half_rn(fabsf(s) <= 65504.f ? r : 0.f);
    h0 = __half_as_ushort(a), h1 = __half_as_ushort(b);
}

// x as 16-bit planes [plane][rows][pitch]: pairs of f16 with a scale per row, triples of bf16, or both.
// A warp per row: the row is read for its largest magnitude and once more, from L1 or L2, to be written.
struct lt_rows {
    const float* src;
    int rows, cols, pitch;
    uint16_t *pair, *triple;
    float* scale;
};
__device__ __forceinline__ void lt_pack_row(const lt_rows& x, int r, bool pairs, bool triples) {
    const int lane = threadIdx.x & 31;
    if (r >= x.rows) return;
    const float* __restrict__ p = x.src + (size_t)r * x.cols;
    uint16_t* __restrict__ pair = pairs ? x.pair + (size_t)r * x.pitch : nullptr;
    uint16_t* __restrict__ triple = triples ? x.triple + (size_t)r * x.pitch : nullptr;
    float m = 0.f;
    if (pair)
#pragma unroll 8
        for (int c = lane; c < x.cols; c += 32) m = fmaxf(m, lt_finite_abs(__ldg(p + c)));
    const float2 sc = lt_scale(rg_warp_max(m));
    if (pair && lane == 0) x.scale[r] = sc.y;
    const size_t plane = (size_t)x.rows * x.pitch;
    for (int c0 = lane; c0 < x.cols; c0 += 128) {
        float v[4];  // loads first
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = c0 + 32 * k < x.cols ? __ldg(p + c0 + 32 * k) : 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int c = c0 + 32 * k;
            if (c >= x.cols) break;
            uint32_t h0, h1, h2;
            if (pair) {
                lt_split2(v[k], sc.x, h0, h1);
                pair[c] = (uint16_t)h0, pair[c + plane] = (uint16_t)h1;
            }
            if (triple) {
                lt_split3(v[k], h0, h1, h2);
                triple[c] = (uint16_t)h0, triple[c + plane] = (uint16_t)h1, triple[c + 2 * plane] = (uint16_t)h2;
            }
        }
    }
}
__global__ void __launch_bounds__(256) lt_pack_rows_kernel(const lt_rows x) {
    rg_pdl_sync();
    lt_pack_row(x, blockIdx.x * 8 + (threadIdx.x >> 5), false, true);
}

// Largest finite magnitudes of w (all blocks but the last `xblocks`) and of x (those), as bits - they order like the values -,
// into two words that lce_check_kernel has set to 0.
__global__ void __launch_bounds__(256) lt_max_kernel(const float* __restrict__ w, size_t wn, const float* __restrict__ x, size_t xn, int xblocks,
                                                     unsigned* __restrict__ out) {
    rg_pdl_sync();
    const int wblocks = (int)gridDim.x - xblocks;
    const bool of_x = (int)blockIdx.x >= wblocks;
    const float* __restrict__ src = of_x ? x : w;
    const size_t n = of_x ? xn : wn, block = of_x ? blockIdx.x - wblocks : blockIdx.x, stride = (size_t)(of_x ? xblocks : wblocks) * 256;
    const float4* v4 = reinterpret_cast<const float4*>(src);
    float m = 0.f;
#pragma unroll 4
    for (size_t i = block * 256 + threadIdx.x; i < n / 4; i += stride) {
        const float4 q = v4[i];
        m = fmaxf(m, fmaxf(fmaxf(lt_finite_abs(q.x), lt_finite_abs(q.y)), fmaxf(lt_finite_abs(q.z), lt_finite_abs(q.w))));
    }
    if (block == 0 && threadIdx.x < n % 4) m = fmaxf(m, lt_finite_abs(src[n - 1 - threadIdx.x]));
    m = rg_warp_max(m);
    if ((threadIdx.x & 31) == 0 && m > 0.f) atomicMax(out + of_x, __float_as_uint(m));  // a maximum: the order does not matter
}

// w as pairs of f16 with one scale for the whole matrix (not where lt_wide() says that they are not used), and triples of bf16,
// or one of them.  A thread takes 8
// neighbouring values of a row and writes 16 bytes of each plane.  The values are walked from the end: what the last-level
// cache still holds of lt_max_kernel's pass is read from there.  Memory bound: 4 bytes in, 4 (6, 10) out for pairs (triples,
// both); 768 x 50257: 52 (62, 89) us, 5.9 to 6.2 TB/s, and 30 us for the pass before.  The first blocks pack x, which took a
// launch of 4 to 8 us of its own.
template <bool PAIR, bool TRIPLE>
__global__ void __launch_bounds__(256) lt_pack_kernel(const float* __restrict__ src, int rows, int cols, int pitch,
                                                      const unsigned* largest, uint16_t* __restrict__ pair,
                                                      uint16_t* __restrict__ triple, float* __restrict__ scale_out, const lt_rows x) {
    rg_pdl_sync();
    const int xblocks = (x.rows + 7) / 8, block = (int)blockIdx.x - xblocks;
    const bool wide = PAIR && lt_wide(largest, rows);
    if (block < 0) {
        lt_pack_row(x, blockIdx.x * 8 + (threadIdx.x >> 5), PAIR && !wide, TRIPLE || wide);
        return;
    }
    if (wide && !TRIPLE) return;
    const float2 sc = PAIR ? lt_scale(__uint_as_float(*largest)) : make_float2(1.f, 1.f);
    if (PAIR && block == 0 && threadIdx.x == 0) *scale_out = sc.y;
    const int groups = pitch / 8;
    const long long n = (long long)rows * groups, stride = (long long)(gridDim.x - xblocks) * 256;
    const size_t plane = (size_t)rows * pitch;
    for (long long i = n - 1 - ((long long)block * 256 + threadIdx.x); i >= 0; i -= stride) {
        const long long r = i / groups;
        const int c = (int)(i - r * groups) * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = c + k < cols ? src[r * cols + c + k] : 0.f;
        const size_t at = (size_t)r * pitch + c;
        uint32_t h0[4], h1[4], h2[4];
        if (PAIR && !wide) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t a0, a1, b0, b1;
                lt_split2(v[2 * k], sc.x, a0, a1);
                lt_split2(v[2 * k + 1], sc.x, b0, b1);
                h0[k] = a0 | (b0 << 16), h1[k] = a1 | (b1 << 16);
            }
            *reinterpret_cast<uint4*>(pair + at) = make_uint4(h0[0], h0[1], h0[2], h0[3]);
            *reinterpret_cast<uint4*>(pair + plane + at) = make_uint4(h1[0], h1[1], h1[2], h1[3]);
        }
        if (TRIPLE) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t a0, a1, a2, b0, b1, b2;
                lt_split3(v[2 * k], a0, a1, a2);
                lt_split3(v[2 * k + 1], b0, b1, b2);
                h0[k] = a0 | (b0 << 16), h1[k] = a1 | (b1 << 16), h2[k] = a2 | (b2 << 16);
            }
            *reinterpret_cast<uint4*>(triple + at) = make_uint4(h0[0], h0[1], h0[2], h0[3]);
            *reinterpret_cast<uint4*>(triple + plane + at) = make_uint4(h1[0], h1[1], h1[2], h1[3]);
            *reinterpret_cast<uint4*>(triple + 2 * plane + at) = make_uint4(h2[0], h2[1], h2[2], h2[3]);
        }
    }
}

struct lt_operand {
    const void* base;
    int rows, cols, planes;
    long long pitch;  // elements
};

typedef CUresult (*lt_encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);

static rg_status lt_encoder(lt_encode_fn* fn) {
    static lt_encode_fn found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<lt_encode_fn>(f);
    }();
    if (!found) return rg_fail(RG_ERR_BACKEND, "cuTensorMapEncodeTiled is not available");
    *fn = found;
    return RG_OK;
}

static rg_status lt_map(CUtensorMap* map, const lt_operand& o, int box_rows) {
    lt_encode_fn encode = nullptr;
    RG_TRY(lt_encoder(&encode));
    const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
    const cuuint64_t strides[2] = {(cuuint64_t)o.pitch * 2, (cuuint64_t)o.pitch * 2 * o.rows};
    const cuuint32_t box[3] = {LT_BK, (cuuint32_t)box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return rg_fail(RG_ERR_BACKEND, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return RG_OK;
}

// x or w as TMA reads it.  bf16: the caller's matrix itself, or a copy with aligned rows; `logits` and `grads` are the same.
// f32: packed pairs for the logits and, where the call needs them, triples for the gradients.
struct lt_packed {
    lt_operand logits, grads;
    const float* scale;
    lt_rows rows;  // f32 x: what is still to be packed
    rg_outputs<3> mem;
};
// Allocates the planes of a matrix, or copies the rows of a bf16 one that TMA cannot address.
static rg_status lt_planes(rg_ctx* ctx, const void* src, int rows, int cols, int dtype, size_t scales, bool want_logits, bool want_grads,
                           lt_packed* o) {
    o->scale = nullptr;
    if (dtype == RG_DTYPE_BF16 && cols % 8 == 0) {
        o->logits = o->grads = {src, rows, cols, 1, cols};
        return RG_OK;
    }
    const int pitch = (cols + 7) / 8 * 8;
    const size_t plane = (size_t)rows * pitch, pair = 2 * plane, triple = 3 * plane;
    if (dtype == RG_DTYPE_BF16) {
        RG_TRY(rg_alloc_storage(ctx, &plane, 1, &o->mem[0], RG_DTYPE_BF16));
        const int grid = (int)std::min<long long>(((long long)rows * (pitch / 8) + 255) / 256, (long long)ctx->sm_count * 16);
        RG_CUDA(rg_launch(true, lt_align_kernel, dim3(grid), dim3(256), 0, ctx->stream, static_cast<const __nv_bfloat16*>(src),
                          (long long)rows, cols, pitch, static_cast<__nv_bfloat16*>(o->mem[0]->raw())));
        RG_LAUNCHED(ctx);
        o->logits = o->grads = {o->mem[0]->raw(), rows, cols, 1, pitch};
        return RG_OK;
    }
    if (want_logits) RG_TRY(rg_alloc_storage(ctx, &pair, 1, &o->mem[0], RG_DTYPE_BF16));
    if (want_logits) RG_TRY(rg_alloc_storage(ctx, &scales, 1, &o->mem[1]));
    if (want_grads) RG_TRY(rg_alloc_storage(ctx, &triple, 1, &o->mem[2], RG_DTYPE_BF16));
    uint16_t* two = want_logits ? static_cast<uint16_t*>(o->mem[0]->raw()) : nullptr;
    uint16_t* three = want_grads ? static_cast<uint16_t*>(o->mem[2]->raw()) : nullptr;
    float* scale = want_logits ? o->mem[1]->data() : nullptr;
    o->scale = scale;
    o->rows = {static_cast<const float*>(src), rows, cols, pitch, two, three, scale};
    o->logits = {two, rows, cols, 2, pitch};
    o->grads = {three, rows, cols, 3, pitch};
    return RG_OK;
}
// x and (w_too) w as the kernels read them.  A scale per row of x, one for w.  Where x has pairs it has room for triples too:
// lce_mid_kernel may have to take the call.
static rg_status lt_pack(rg_ctx* ctx, const lce_call& c, bool w_too, bool want_logits, bool want_grads, lt_packed* x, lt_packed* w) {
    RG_TRY(lt_planes(ctx, c.x, c.R, c.D, c.dtype, (size_t)c.R, want_logits, true, x));
    if (w_too) RG_TRY(lt_planes(ctx, c.w, c.D, c.V, c.dtype, 1, want_logits, want_grads, w));
    if (c.dtype == RG_DTYPE_BF16) return RG_OK;
    const int xblocks = rg_cdiv(c.R, 8);
    if (!w_too) {
        RG_CUDA(rg_launch(true, lt_pack_rows_kernel, dim3((unsigned)xblocks), dim3(256), 0, ctx->stream, x->rows));
    } else {
        const lt_rows& m = w->rows;
        if (want_logits) {
            const size_t n = (size_t)m.rows * m.cols, xn = (size_t)c.R * c.D;
            // one wave of blocks, shared by sizes (a wave each: 37 us instead of 30 for 4096x768x50257)
            const size_t wave = (size_t)ctx->sm_count * 8;
            auto blocks = [&](size_t k) { return std::max<size_t>(1, std::min((k / 4 + 255) / 256, wave * k / (n + xn))); };
            RG_CUDA(rg_launch(true, lt_max_kernel, dim3((unsigned)(blocks(n) + blocks(xn))), dim3(256), 0, ctx->stream, m.src, n, x->rows.src,
                              xn, (int)blocks(xn), c.largest));
            RG_LAUNCHED(ctx);
        }
        const unsigned grid = (unsigned)std::min<long long>(((long long)m.rows * (m.pitch / 8) + 255) / 256, (long long)ctx->sm_count * 16);
        RG_CUDA(rg_launch(true, !want_grads ? lt_pack_kernel<true, false> : want_logits ? lt_pack_kernel<true, true> : lt_pack_kernel<false, true>,
                          dim3(xblocks + grid), dim3(256), 0, ctx->stream, m.src, m.rows, m.cols, m.pitch, (const unsigned*)c.largest, m.pair,
                          m.triple, m.scale, x->rows));
    }
    RG_LAUNCHED(ctx);
    return RG_OK;
}

static_assert(lt_shape<1>::BN == lt_shape<2>::BN, "the logits have one width of column tiles");
#define LT_BN lt_shape<1>::BN

// The form of lce_mid_kernel, by what was measured at [R,768] x [768,50257], at no other width and vocabulary (us for the call,
// and with packed or copied operands):
// f32 forward 17 rows 53 (153), 128 rows 86 (152), 256 rows 139 (154); gradient 17 rows 229 (309), 192 rows 385 (402), 256
// rows 462 (434); bf16 with an odd vocabulary forward 17 rows 39 (65), 128 rows 56 (65), 192 rows 67 (66).  With an aligned
// one bf16 is read as it lies by TMA.
static bool lm_takes(const lce_call& c) { return c.dtype == RG_DTYPE_F32 ? c.R <= 192 : c.R <= 128 && c.V % 8; }

// Columns of a tile: as many tiles as whole rounds of the SMs hold.
static int lm_tile(rg_ctx* ctx, const lce_call& c, int cols) {
    const long long groups = rg_cdiv(c.R, 64), rounds = rg_cdiv(rg_cdiv(cols, 128) * groups, ctx->sm_count);
    const int tiles = (int)std::max<long long>(1, rounds * ctx->sm_count / groups);
    return std::min(128, std::max(64, (rg_cdiv(cols, tiles) + 3) / 4 * 4));
}
int lce_tc_nparts(rg_ctx* ctx, const lce_call& c) { return lm_takes(c) ? rg_cdiv(c.V, lm_tile(ctx, c, c.V)) : 2 * rg_cdiv(c.V, LT_BN); }

// `e` comes with the columns that are covered, and what the gradient stores.
template <typename T, int EPI>
static rg_status lm_launch(rg_ctx* ctx, const lce_call& c, const lt_packed& x, lm_args& e) {
    CUtensorMap map;
    RG_TRY(lt_map(&map, x.grads, 64));
    e.w = c.w, e.R = c.R, e.D = c.D, e.V = c.V;
    if (!e.groups) e.groups = rg_cdiv(c.R, 64);
    if (!e.tile) e.tile = lm_tile(ctx, c, e.cols);
    if (!e.db_rows) e.db_rows = 1;
    e.tiles = rg_cdiv(e.cols, e.tile);
    e.err = ctx->d_flag + 1;
    e.bias = c.bias, e.tgt = c.tgt, e.parts = c.parts, e.tz = c.tz, e.lse = c.lse;
    const long long total = (long long)e.tiles * e.groups;
    if (total > 0x7fffffff - 2 * ctx->sm_count) return rg_fail(RG_ERR_SHAPE, "linear_cross_entropy: too many tiles");
    const int grid = (int)std::min<long long>(total, ctx->sm_count);
    RG_CUDA(cudaFuncSetAttribute(lce_mid_kernel<T, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, lm_shape<T>::SMEM));
    RG_CUDA(rg_launch(true, lce_mid_kernel<T, EPI>, dim3(grid), dim3(LM_THREADS), lm_shape<T>::SMEM, ctx->stream, map, e));
    RG_LAUNCHED(ctx);
    return RG_OK;
}
// The same work as a launch of lce_tc_kernel<2, EPI> before it (x packed as triples too), done where that one leaves it: the
// same partial sums of 128 columns (FWD), the same dz, and rows of dbparts for 32 rows each (DZ).  Calls, us, with one weight of 1e10
// against ordinary weights: loss of 256 rows x768x50257 192 and 156, of 4096 2,180 and 770 to 850; gradient of 2048 3,020 and 2,210
// to 2,310.  Where it is not needed it costs 3 us.
template <int EPI>
static rg_status lm_launch_wide(rg_ctx* ctx, const lce_call& c, const lt_packed& x, int v0, int cols, __nv_bfloat16* dz, float* dbparts) {
    lm_args e;
    memset(&e, 0, sizeof(e));
    e.largest = c.largest;
    e.tile = LT_BN / 2, e.v0 = v0, e.cols = cols;
    if (EPI == LT_DZ) e.groups = LT_BM / 64 * rg_cdiv(c.R, LT_BM), e.db_rows = 2;
    e.dz = dz, e.dbparts = dbparts;
    return lm_launch<float, EPI>(ctx, c, x, e);
}

static lt_prob lt_problem(int M, int N, int K, int bn, int a_mn, int b_mn) {
    lt_prob p;
    memset(&p, 0, sizeof(p));
    p.M = M, p.N = N, p.K = K;
    p.tiles_m = rg_cdiv(M, LT_BM), p.tiles_n = rg_cdiv(N, bn), p.splits = 1, p.kb_per = rg_cdiv(K, LT_BK);
    p.a_mn = a_mn, p.b_mn = b_mn;
    return p;
}

template <int PLANES, int EPI, bool CUT>
static rg_status lt_launch(rg_ctx* ctx, const CUtensorMap* maps, lt_args& e) {
    RG_CUDA(cudaFuncSetAttribute(lce_tc_kernel<PLANES, EPI, CUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_SMEM_BYTES));
    long long total = 0;
    for (int i = 0; i < e.nprobs; i++) total += (long long)e.p[i].tiles_m * e.p[i].tiles_n * e.p[i].splits;
    if (total > 0x3fffffff) return rg_fail(RG_ERR_SHAPE, "linear_cross_entropy: too many tiles");
    const int grid = 2 * (int)std::min<long long>(total, ctx->sm_count / 2);
    RG_CUDA(rg_launch(true, lce_tc_kernel<PLANES, EPI, CUT>, dim3(grid), dim3(lt_shape<PLANES, EPI, CUT>::THREADS), LT_SMEM_BYTES, ctx->stream,
                      maps[0], maps[1], maps[2], maps[3], e));
    RG_LAUNCHED(ctx);
    e.counter++;  // each launch hands out its tiles from a counter of its own
    return RG_OK;
}
// bf16 logits in pieces along D: k-blocks per accumulator, 0 for one accumulator.  lse, the loss and dbias are f32, and a chain that
// truncates shows in them: off by up to 1.1e-6 (lse) and 4.4e-6 (dbias) of the norm at D = 1600, 5.7e-6 and 2e-5 at 9000, against
// 6.4e-7 with chains of 768, 1.3e-6 of 384 and 9e-7 of 256 for dbias.  dx and dw are rounded to bf16, so dz is only cut where
// dbias is asked for.  Cost of the long chains: loss of 4096x1600x50257 537 -> 553 us, gradients with a bias of 2048x768x50257 479
// -> 490 and of 4096x1600x50257 1,700 -> 1,765 (256 for all: 520 and 1,795); loss of 4096x192x50257 in pieces 221 instead of 160.
// With one tile for a pair of CTAs nothing waits for the epilogue, and 256 costs nothing (200x768x3000, 1000x768x4000: the same
// within 1 %).
template <int EPI>
static int lt_chain(rg_ctx* ctx, const lce_call& c, const lt_prob& p) {
    if (EPI == LT_DZ && !c.dbias) return 0;
    const bool one = (long long)p.tiles_m * p.tiles_n <= ctx->sm_count / 2;
    const int chain = one ? LT_CHAIN_ONE : EPI == LT_FWD ? LT_CHAIN_FWD : LT_CHAIN_DZ;
    return c.D > chain * LT_BK ? chain : 0;
}
template <int EPI>
static rg_status lt_run(rg_ctx* ctx, const lce_call& c, const CUtensorMap* maps, lt_args& e) {
    if (c.dtype == RG_DTYPE_F32) return lt_launch<EPI == LT_GRAD ? 3 : 2, EPI, true>(ctx, maps, e);
    if constexpr (EPI != LT_GRAD) {
        e.chain = lt_chain<EPI>(ctx, c, e.p[0]);
        if (e.chain) return lt_launch<1, EPI, true>(ctx, maps, e);
    }
    return lt_launch<1, EPI, false>(ctx, maps, e);
}

static void lt_common(rg_ctx* ctx, const lce_call& c, int* counter, lt_args* e) {
    memset(e, 0, sizeof(*e));
    e->counter = counter, e->err = ctx->d_flag + 1;
    e->R = c.R, e->D = c.D, e->V = c.V, e->v0 = 0, e->vn = c.V;
    e->bias = c.bias, e->tgt = c.tgt, e->lse = c.lse, e->scal = c.scal;
    e->parts = c.parts, e->tz = c.tz, e->largest = c.largest;
}

rg_status lce_tc_forward(rg_ctx* ctx, lce_call& c) {
    lt_packed x, w;
    if (lm_takes(c)) {
        RG_TRY(lt_pack(ctx, c, false, false, true, &x, nullptr));
        lm_args e;
        memset(&e, 0, sizeof(e));
        e.cols = c.V;
        return c.dtype == RG_DTYPE_F32 ? lm_launch<float, LT_FWD>(ctx, c, x, e) : lm_launch<__nv_bfloat16, LT_FWD>(ctx, c, x, e);
    }
    RG_TRY(lt_pack(ctx, c, true, true, false, &x, &w));
    CUtensorMap maps[4];
    RG_TRY(lt_map(&maps[0], x.logits, 128));
    RG_TRY(lt_map(&maps[1], w.logits, LT_BK));
    maps[2] = maps[0], maps[3] = maps[1];
    lt_args e;
    lt_common(ctx, c, c.counters, &e);
    e.xscale = x.scale, e.wscale = w.scale;
    e.nprobs = 1;
    e.p[0] = lt_problem(c.R, c.V, c.D, LT_BN, 0, 1);
    RG_TRY(lt_run<LT_FWD>(ctx, c, maps, e));
    if (c.dtype == RG_DTYPE_F32) RG_TRY(lm_launch_wide<LT_FWD>(ctx, c, x, 0, c.nparts * (LT_BN / 2), nullptr, nullptr));
    return RG_OK;
}

// The gradient goes over pieces of the vocabulary: dz of a piece is written as bf16 planes, then one launch multiplies it with w
// and with x.  A piece is as wide as LT_DZ_BYTES allow, but at least the 256 columns of a tile: beyond 1 Mi rows of bf16 (2^20)
// or 349,525 of f32 its dz grows with the rows, 512 or 1,536 bytes each (x itself holds 2 or 4 bytes for each of its columns).
// The partial sums of dbias are those of a piece too.
#define LT_DZ_BYTES ((size_t)512 << 20)

static int lt_piece(const lce_call& c) {
    const int planes = c.dtype == RG_DTYPE_F32 ? 3 : 1;
    const long long most = std::max<long long>(1, (long long)(LT_DZ_BYTES / ((size_t)planes * 2 * c.R)) / 256) * 256;
    const int pieces = (int)((c.V + most - 1) / most);
    return (int)std::min<long long>(most, (rg_cdiv(c.V, pieces) + 255) / 256 * 256);
}
int lce_tc_backward_launches(const lce_call& c) { return 2 * rg_cdiv(c.V, lt_piece(c)); }

rg_status lce_tc_backward(rg_ctx* ctx, lce_call& c) {
    rg_outputs<4> o;  // dz, partial dx, partial dbias, partial dw
    lt_packed x, w;
    const int planes = c.dtype == RG_DTYPE_F32 ? 3 : 1, bn = planes == 3 ? lt_shape<3>::BN : lt_shape<1>::BN;  // of the gradients
    const int clusters = ctx->sm_count / 2;
    const int piece = lt_piece(c), pieces = rg_cdiv(c.V, piece);
    const bool mid = c.dtype == RG_DTYPE_F32 && lm_takes(c) && pieces == 1;  // bf16: w is copied for dx all the same
    RG_TRY(lt_pack(ctx, c, true, !mid, true, &x, &w));

    const int width = std::min(piece, (c.V + 63) / 64 * 64);  // columns of dz that are stored
    const size_t zlen = (size_t)planes * c.R * width;
    RG_TRY(rg_alloc_storage(ctx, &zlen, 1, &o[0], RG_DTYPE_BF16));

    // dx or its transpose: whichever pads less (a row tile is 256, a column tile as narrow as 32)
    auto pad = [](long long m, long long n) { return (m + 255) / 256 * 256 * ((n + 31) / 32 * 32); };
    const bool dx_t = pad(c.D, c.R) < pad(c.R, c.D);
    const int first = std::min(piece, c.V);  // columns of the first piece; it writes every partial dx that is added in the end
    lt_prob pdx = dx_t ? lt_problem(c.D, c.R, first, bn, 0, 0) : lt_problem(c.R, c.D, first, bn, 0, 0);
    lt_prob pdw = lt_problem(piece, c.D, c.R, bn, 1, 1);
    // The K axes are cut where tiles are fewer or longer than makes an even load: runs of `run` k-blocks, none of them empty.  A
    // smaller last piece has fewer runs of dx and leaves the other sums alone; dw is only cut when there is one piece.
    const long long load = (long long)pdx.tiles_m * pdx.tiles_n * pdx.kb_per + (long long)pdw.tiles_m * pdw.tiles_n * pdw.kb_per;
    const int fair = (int)std::max<long long>(8, load / clusters / 2);
    auto cut = [&](lt_prob& p) {
        p.kb_per = rg_cdiv(p.kb_per, std::min(16, rg_cdiv(p.kb_per, fair)));
        return p.kb_per;
    };
    const int run = cut(pdx), splits = rg_cdiv(rg_cdiv(first, LT_BK), run);
    const bool cut_dw = pieces == 1 && pdw.tiles_m * pdw.tiles_n < clusters && pdw.kb_per > fair;
    const int run_w = cut_dw ? cut(pdw) : pdw.kb_per, splits_w = rg_cdiv(rg_cdiv(c.R, LT_BK), run_w);
    const size_t plen = (size_t)splits * c.R * c.D, wlen = (size_t)splits_w * c.D * c.V;
    RG_TRY(rg_alloc_storage(ctx, &plen, 1, &o[1]));
    if (cut_dw) RG_TRY(rg_alloc_storage(ctx, &wlen, 1, &o[3]));
    const int dbrows = mid ? rg_cdiv(c.R, 64) : LT_BM / 32 * rg_cdiv(c.R, LT_BM);
    if (c.dbias) {
        const size_t blen = (size_t)dbrows * width;
        RG_TRY(rg_alloc_storage(ctx, &blen, 1, &o[2]));
    }

    CUtensorMap mz[4] = {}, mg[4];
    lt_operand z = {o[0]->raw(), c.R, width, planes, width};
    if (!mid) RG_TRY(lt_map(&mz[0], x.logits, 128));
    if (!mid) RG_TRY(lt_map(&mz[1], w.logits, LT_BK));
    mz[2] = mz[0], mz[3] = mz[1];
    RG_TRY(lt_map(&mg[0], dx_t ? w.grads : z, 128));
    RG_TRY(lt_map(&mg[1], dx_t ? z : w.grads, bn / 2));
    RG_TRY(lt_map(&mg[2], z, LT_BK));
    RG_TRY(lt_map(&mg[3], x.grads, LT_BK));

    for (int i = 0; i < pieces; i++) {
        lt_args e;
        lt_common(ctx, c, c.counters + 2 * i, &e);
        e.xscale = x.scale, e.wscale = w.scale;
        e.v0 = i * piece, e.vn = std::min(piece, c.V - e.v0);
        e.dz = static_cast<__nv_bfloat16*>(o[0]->raw()), e.dz_pitch = width;
        e.dbparts = c.dbias ? o[2]->data() : nullptr;
        e.dxparts = o[1]->data(), e.dx_add = i > 0, e.dx_t = dx_t;
        e.dw = c.dw, e.dw_bf16 = c.dtype == RG_DTYPE_BF16;
        e.dwparts = cut_dw ? o[3]->data() : nullptr;
        e.nprobs = 1;
        e.p[0] = lt_problem(c.R, e.vn, c.D, LT_BN, 0, 1);
        e.p[0].b_n0 = e.v0;
        if (mid) {
            lm_args m;
            memset(&m, 0, sizeof(m));
            m.cols = width, m.dz = e.dz, m.dbparts = e.dbparts;
            RG_TRY((lm_launch<float, LT_DZ>(ctx, c, x, m)));
        } else {
            RG_TRY(lt_run<LT_DZ>(ctx, c, mz, e));
            if (c.dtype == RG_DTYPE_F32) RG_TRY(lm_launch_wide<LT_DZ>(ctx, c, x, e.v0, width, e.dz, e.dbparts));
        }
        e.nprobs = 2;
        e.p[0] = dx_t ? lt_problem(c.D, c.R, e.vn, bn, 0, 0) : lt_problem(c.R, c.D, e.vn, bn, 0, 0);
        e.p[0].splits = rg_cdiv(e.p[0].kb_per, run), e.p[0].kb_per = run;
        (dx_t ? e.p[0].a_k0 : e.p[0].b_k0) = e.v0;
        e.p[1] = lt_problem(e.vn, c.D, c.R, bn, 1, 1);
        e.p[1].splits = splits_w, e.p[1].kb_per = run_w;
        RG_TRY(lt_run<LT_GRAD>(ctx, c, mg, e));
        // the sums of dbias: with those of dx after the last piece, else in a launch of their own
        const bool last = i + 1 == pieces;
        if (last || c.dbias)
            lce_finish_launch(ctx, o[1]->data(), splits, last ? (size_t)c.R * c.D : 0, c.scal, c.tgt, c.D, c.dx, c.dtype, e.dbparts, dbrows,
                              width, e.vn, c.dbias ? c.dbias + e.v0 : nullptr);
    }
    if (cut_dw) lce_finish_launch(ctx, o[3]->data(), splits_w, (size_t)c.D * c.V, c.scal, nullptr, c.D, c.dw, c.dtype, nullptr, 0, 0, 0, nullptr);
    return RG_OK;
}

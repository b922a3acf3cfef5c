// Matrix products of the gated feed-forward block (included by gated_ffn.hip): out[m][j] = sum_k A(m, k) B(j, k) in fp32 / bf16 / fp16, sums in fp32.
//
// Each operand lies in memory with its reduction axis contiguous ("rows of k": x, weights in the forward) or across rows ("k-major": weights in the input
// gradients, both operands of the weight gradients); all four combinations run the same loop.  A workgroup owns a BM x BN tile; per step it stages 128
// bytes of k (64 sixteen-bit or 32 fp32 elements) of every row by global -> LDS DMA (16 bytes a lane, no registers) into one of two (four) buffers while the
// matrix instructions read the other; one barrier per step publishes the new buffer and frees the old one.
//
// Measured over 16 384 rows of 2048, n = 5632, bf16, each launch in a kernel trace (average of 12; the shortest are 4 - 10 % below): y 346 us (1.09 PFLOP/s), dx 623 us (1.21),
// the three weight gradients 965 us (1.18), the gate product with its epilogue 742 us (1.02), dh with its epilogue 543 us (0.70: 0.92 GB of g, u, dg and du pass through it); a
// large library product reaches 1.34 here.  fp32 (7 840 x 576 x 1 536): 75 - 109 TFLOP/s of 154, dh with its epilogue the least.  Steps of 64 bytes in 3 to 5 stages were
// 5 - 15 % slower, a second register set for all fragments spilled, and staggered starts of the workgroups changed nothing.
//
// LDS layouts, both without padding (DMA fills LDS linearly, so the SOURCE address carries the permutation):
//   rows of k:  row r of the tile = 128 bytes, its 16-byte chunk c at position c ^ ((r >> 1) & 7): the 16 lanes of one ds_read_b128 pass cover the 64 banks once
//   k-major:    row k of the tile = BM (BN) elements.  Sixteen bits: fragments come out of ds_read_b64_tr_b16 (a 16-lane group reads 4 rows of k x 16 columns
//               and returns them transposed), chunk c at c ^ (f << 1) with f = (k & 3) | ((k >> 3 & 1) << 2): the 8 rows that a pass touches lie in 8 different
//               32-byte slots.  fp32: 4-byte reads, chunk c at c ^ ((k >> 2 & 3) << 2): the 4 rows of a pass lie in 4 different 64-byte slots.
// Fragment order of k is the same for every layout (lane group g of 16 takes k = 8 g .. 8 g + 7 of 32, fp32: 4 g + e of 16), so results do not depend on it.
// The weights' side is the FIRST matrix operand: a lane then holds 4 consecutive output columns of one row, stored as one vector.

#include <atomic>
#include <type_traits>

namespace suhpe {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

enum { EPI_STORE = 0, EPI_GATE = 1, EPI_GATE_BWD = 2 };

// One product: A (M rows), B (N rows), out (M, N) with ldo columns from row to row
struct Product {
    const char *a[2], *b[2];                                           // by segment of the reduction, or (EPI_GATE's b) gate and up weights
    int64_t lda, ldb;                                                  // bytes from row to row
    int64_t M;
    int N, ldo;                                                        // EPI_GATE: columns of g, u, h; EPI_GATE_BWD: ldo >= N, zeros behind N
    void* out;                                                         // EPI_GATE: h; EPI_GATE_BWD: dg
    int tiles_m, tiles_n;
};

struct GemmArgs {
    Product pr[3];                                                     // independent products over the same k in one launch
    int64_t K;                                                         // reduction of ONE segment
    int nk, nseg;                                                      // steps of a segment; segments
    int tiles, whole, splits;                                          // all tiles; the first `whole` reduced by one workgroup each, the others by `splits` in equal parts
    const void *bias, *bias2;
    void* kept;                                                        // EPI_GATE: where g and u go, or null; EPI_GATE_BWD: where they come from
    void* uout;                                                        // EPI_GATE_BWD: du
    int act, accumulate;
    float* part;                                                       // [tile behind `whole`][split][BM][BN]
    float *cols, *cols2;                                               // EPI_GATE_BWD: column sums of dg and du, [row tile][N], or null
};

// tile number -> product, row tile, column tile: groups of 8 rows of tiles x all columns, so that neighbours in the order share operands in L2
__device__ __forceinline__ Product tile_of(const GemmArgs& p, int item, int* tile_m, int* tile_n) {
    Product pr = p.pr[0];
#pragma unroll
    for (int q = 1; q < 3; ++q) {
        const int before = pr.tiles_m * pr.tiles_n;
        if (item < before) break;
        item -= before;
        pr = p.pr[q];
    }
    constexpr int GROUP = 8;
    const int group = item / (GROUP * pr.tiles_n), first = group * GROUP, size = pr.tiles_m - first < GROUP ? pr.tiles_m - first : GROUP;
    item -= group * GROUP * pr.tiles_n;
    *tile_m = first + item % size;
    *tile_n = item / size;
    return pr;
}

// act and act' of 8 values, both from one exponential each.  One branch on the activation for all 8: chosen inside, per value, it cost the epilogues more vector time
// than the activation
__device__ __forceinline__ void act8(const float (&u)[8], int act, float (&a)[8]) {
    if (act == SUHPE_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = act_apply(u[e], SUHPE_ACT_SILU);
    } else if (act == SUHPE_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = act_apply(u[e], SUHPE_ACT_GELU);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = act_apply(u[e], act);
    }
}
__device__ __forceinline__ void act8_both(const float (&u)[8], int act, float (&a)[8], float (&da)[8]) {
    if (act == SUHPE_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float s = fast_sigmoid(u[e]);
            a[e] = u[e] * s;
            da[e] = s * (1.f + u[e] * (1.f - s));
        }
    } else if (act == SUHPE_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float x;
            const float cdf = 0.5f * (1.f + fast_erf(u[e] * 0.70710678118654752f, &x));
            a[e] = u[e] * cdf;
            da[e] = cdf + u[e] * 0.3989422804014327f * x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = act_apply(u[e], act);
            da[e] = act_grad(u[e], act);
        }
    }
}

template <typename T> struct Mfma;
template <> struct Mfma<bf16> {
    typedef bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(i32x4 a, i32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
};
template <> struct Mfma<f16> {
    typedef f16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 run(i32x4 a, i32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
    }
};
template <> struct Mfma<float> {
    static __device__ __forceinline__ f32x4 run(i32x4 a, i32x4 b, f32x4 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
};

// N pieces of 1 KiB at this lane's byte offsets from `base` into consecutive LDS pieces from `lds` on.  (s_nop 4: an SGPR operand may just have been
// written by a vector instruction; s_nop 2: m0 before its use.)
template <int N> __device__ __forceinline__ void dma(const unsigned (&off)[N], const char* base, unsigned lds) {
    // raw buffer descriptor of 2 GiB - 1 from `base` on: an offset of kOob reads as zero
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const i32x4 r = {__builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)), 0x7fffffff, 0x00020000};
    unsigned keep;
    if constexpr (N == 4)
        asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %1, %5, 0 offen lds\n\ts_add_u32 m0, m0, 1024\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %2, %5, 0 offen lds\n\ts_add_u32 m0, m0, 1024\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %3, %5, 0 offen lds\n\ts_add_u32 m0, m0, 1024\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %4, %5, 0 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(r), "s"(lds) : "memory", "scc");
    else if constexpr (N == 1)
        asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 2\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[0]), "s"(r), "s"(lds) : "memory");
    else {
        static_assert(N == 2, "one, two or four pieces");
        asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %1, %3, 0 offen lds\n\ts_add_u32 m0, m0, 1024\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[0]), "v"(off[1]), "s"(r), "s"(lds) : "memory", "scc");
    }
}

constexpr int kStep = 128;                                             // bytes of k a step

// LDS-side geometry of one operand: R rows of the tile, k contiguous or k-major
template <typename T, int R, bool KM> struct Side {
    static constexpr int ES = sizeof(T), BKE = kStep / ES, CH = 16 / ES, RB = R * ES, CPR = kStep / 16;
    static __device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }
    // tile row (or k) and global 16-byte chunk that lane `lane` of piece q fills
    static __device__ __forceinline__ void place(int q, int lane, int* row, int* chunk) {
        if constexpr (!KM) {
            const int r = q * (1024 / kStep) + lane / CPR;
            *row = r;
            *chunk = (lane % CPR) ^ swizzle(r);
        } else {
            const int at = q * 1024 + lane * 16, k = at / RB, c = (at % RB) >> 4;
            *row = k;
            *chunk = ES == 2 ? c ^ (((k & 3) | ((k >> 3 & 1) << 2)) << 1) : c ^ ((k >> 2 & 3) << 2);
        }
    }
    // byte offset of this lane's share of the fragment of rows 16 rb .. 16 rb + 15, k-group 0
    static __device__ __forceinline__ int lane_base(int lane) {
        const int g = lane >> 4, t = lane & 15;
        if constexpr (!KM) return t * kStep;
        else if constexpr (ES == 2) return (g * 8 + (t >> 2)) * RB + (t & 1) * 8;
        else return (g * 4) * RB + (t & 3) * 4;
    }
    static __device__ __forceinline__ i32x4 read(const char* tile, int base, int lane, int rb, int kk) {
        const int g = lane >> 4, t = lane & 15;
        if constexpr (!KM) {
            return *reinterpret_cast<const i32x4*>(tile + base + rb * 16 * kStep + (((kk * 4 + g) ^ swizzle(t)) << 4));
        } else if constexpr (ES == 2) {
            const int c = (rb * 2 + ((t & 3) >> 1)) ^ (((t >> 2) | ((g & 1) << 2)) << 1);
            const char* p = tile + base + kk * 32 * RB + (c << 4);
            typedef __attribute__((address_space(3))) s16x4* lp;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * RB));
            typedef int i32x2 __attribute__((ext_vector_type(2)));
            const i32x2 l = __builtin_bit_cast(i32x2, lo), h = __builtin_bit_cast(i32x2, hi);
            return i32x4{l[0], l[1], h[0], h[1]};
        } else {
            const int c = (rb * 4 + (t >> 2)) ^ (g << 2);
            const char* p = tile + base + kk * 16 * RB + (c << 4);
            i32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const int*>(p + e * RB);
            return v;
        }
    }
};

// blockIdx -> work item such that each of the 8 XCDs (workgroups are dealt to them in turn) takes one contiguous range: its L2 then sees neighbouring tiles
__device__ __forceinline__ int xcd_order(int bid, int total) {
    const int xcd = bid & 7, i = bid >> 3, per = total >> 3, extra = total & 7;
    return xcd * per + (xcd < extra ? xcd : extra) + i;
}

// at most `pending` of this wavefront's memory operations under way, none of its LDS reads; then the workgroup's barrier
template <int pending> __device__ __forceinline__ void wait_steps() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(pending) : "memory");
}

// 8 consecutive columns from / to memory (any element address); columns from `limit` on are zeros / left alone
template <typename T> __device__ __forceinline__ void load8(const T* p, int n, int limit, float (&v)[8]) {
    if (n + 8 <= limit) {
        T t[8];
        __builtin_memcpy(t, p, sizeof t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = n + e < limit ? (float)p[e] : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int n, int limit, const float (&v)[8]) {
    if (n + 8 <= limit) {
        T t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
        __builtin_memcpy(p, t, sizeof t);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < limit) p[e] = (T)v[e];
    }
}

// g and u between forward and backward.  fp32: as they are.  16-bit types: the upper 24 bits of their fp32 values (off by less than 2^-15), as [g: 16][u: 16][g: 8]
// [u: 8] bits.  Rounded to the tensors' type they would cost the gradients more than their own rounding does (31 360 x 384 x 1 024 bf16: dx, dWg and dWu off by
// 3.1e-3 of their norm, with 24 bits 2.3e-3, of which 1.7e-3 is the last rounding); 24 bits instead of 32 save a quarter of their way through memory.
inline int64_t kept_bytes(int es, int64_t m, int n) { return m * n * (es == 4 ? 8 : 6); }
template <typename T> __device__ __forceinline__ void keep8(void* kept, int64_t count, int which, int64_t at, int n, int limit, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        store8(static_cast<float*>(kept) + which * count + at, n, limit, v);
    } else {
        unsigned short* ph = static_cast<unsigned short*>(kept) + which * count + at;
        unsigned char* pl = static_cast<unsigned char*>(kept) + (4 + which) * count + at;
        if (n + 8 <= limit) {
            unsigned b[8], hi[4], lo[2];
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = __float_as_uint(v[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) hi[e] = __builtin_amdgcn_perm(b[2 * e + 1], b[2 * e], 0x07060302);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                lo[e] = __builtin_amdgcn_perm(b[4 * e + 1], b[4 * e], 0x0c0c0501) | __builtin_amdgcn_perm(b[4 * e + 3], b[4 * e + 2], 0x05010c0c);
            __builtin_memcpy(ph, hi, sizeof hi);
            __builtin_memcpy(pl, lo, sizeof lo);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < limit) {
                    ph[e] = (unsigned short)(__float_as_uint(v[e]) >> 16);
                    pl[e] = (unsigned char)(__float_as_uint(v[e]) >> 8);
                }
        }
    }
}
template <typename T> struct Kept8 {                                   // 8 values under way
    float f[sizeof(T) == 4 ? 8 : 1];
    unsigned hi[sizeof(T) == 4 ? 1 : 4], lo[sizeof(T) == 4 ? 1 : 2];
    __device__ __forceinline__ void load(const void* kept, int64_t count, int which, int64_t at, int n, int limit) {
        if constexpr (sizeof(T) == 4) {
            load8(static_cast<const float*>(kept) + which * count + at, n, limit, f);
        } else {
            const unsigned short* ph = static_cast<const unsigned short*>(kept) + which * count + at;
            const unsigned char* pl = static_cast<const unsigned char*>(kept) + (4 + which) * count + at;
            if (n + 8 <= limit) {
                __builtin_memcpy(hi, ph, sizeof hi);
                __builtin_memcpy(lo, pl, sizeof lo);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) hi[e] = 0;
                lo[0] = lo[1] = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + e < limit) {
                        hi[e / 2] |= (unsigned)ph[e] << (16 * (e & 1));
                        lo[e / 4] |= (unsigned)pl[e] << (8 * (e & 3));
                    }
            }
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return f[e];
        else return __uint_as_float((e & 1 ? hi[e / 2] & 0xffff0000u : hi[e / 2] << 16) | (lo[e / 4] >> (8 * (e & 3)) & 0xffu) << 8);
    }
};

template <typename T, typename O, int TM, int TN, int WM, int WN, int ST, bool AKM, bool BKM, int EPI>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_lowp(const GemmArgs p) {
    constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, NW = WM * WN, NT = 64 * NW;
    using SA = Side<T, BM, AKM>;
    using SB = Side<T, BN, BKM>;
    constexpr int BKE = SA::BKE, CH = SA::CH;                           // a step is two k-groups of 32 sixteen-bit or 16 fp32 elements each
    constexpr int PA = BM * kStep / 1024 / NW, PB = BN * kStep / 1024 / NW, STAGE = (BM + BN) * kStep;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int wm = wave / WN, wn = wave % WN;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int basea = SA::lane_base(lane), baseb = SB::lane_base(lane);
    // this workgroup's share: a whole tile, or one of the equal parts of a shared tile's steps (all tiles' first parts come first: workgroups side by side on an
    // XCD then read the same rows of k, and its L2 fetches them once)
    const int steps = p.nk * p.nseg;
    int item, split = 0;
    const bool complete = (int)blockIdx.x < p.whole;
    if (complete) {
        item = xcd_order(blockIdx.x, p.whole);
    } else {
        const int rest = p.tiles - p.whole;
        item = xcd_order(blockIdx.x - p.whole, rest * p.splits);
        split = item / rest;
        item += p.whole - split * rest;
    }
    const int s0 = complete ? 0 : (int)((int64_t)steps * split / p.splits), s1 = complete ? steps : (int)((int64_t)steps * (split + 1) / p.splits);
    int tile_m, tile_n;
    const Product pr = tile_of(p, item, &tile_m, &tile_n);
    const int64_t m0 = (int64_t)tile_m * BM;
    const int n0 = tile_n * (EPI == EPI_GATE ? BN / 2 : BN);
    {
        // this lane's pieces: byte offset within the step's source rows
        unsigned offa[PA], offb[PB];
#pragma unroll
        for (int i = 0; i < PA; ++i) {
            int row, chunk;
            SA::place(wave * PA + i, lane, &row, &chunk);
            if constexpr (!AKM) {
                const int64_t r = m0 + row < pr.M ? row : pr.M - 1 - m0;                // rows beyond the last repeat it: never stored
                offa[i] = (unsigned)(r * pr.lda + chunk * 16);
            } else {
                offa[i] = m0 + chunk * CH < pr.M ? (unsigned)(row * pr.lda + chunk * 16) : kOob;
            }
        }
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            int row, chunk;
            SB::place(wave * PB + i, lane, &row, &chunk);
            if constexpr (!BKM) {
                if constexpr (EPI == EPI_GATE) row = (row >> 5) * 16 + (row & 15);              // 16 gate rows, 16 up rows, ...
                const int64_t r = n0 + row < pr.N ? row : pr.N - 1 - n0;
                offb[i] = (unsigned)(r * pr.ldb + chunk * 16);
            } else {
                offb[i] = n0 + chunk * CH < pr.N ? (unsigned)(row * pr.ldb + chunk * 16) : kOob;
            }
        }
        auto send = [&](const unsigned (&oa)[PA], const unsigned (&ob)[PB], int which, int64_t k0, int stage) __attribute__((always_inline)) {
            const char* pa = (which ? pr.a[1] : pr.a[0]) + (AKM ? k0 * pr.lda + m0 * SA::ES : m0 * pr.lda + k0 * SA::ES);
            const unsigned la = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + wave * PA * 1024);
            const unsigned lb = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + BM * kStep + wave * PB * 1024);
            dma<PA>(oa, pa, la);
            if constexpr (EPI == EPI_GATE) {                           // a wavefront's pieces: 16 gate rows, then 16 up rows
                static_assert(PB * 1024 == 32 * kStep && !BKM, "a wavefront fills whole blocks of 16 gate and 16 up rows");
                const int64_t off = n0 * pr.ldb + k0 * SB::ES;
                unsigned g[PB / 2], u[PB / 2];
#pragma unroll
                for (int i = 0; i < PB / 2; ++i) { g[i] = ob[i]; u[i] = ob[PB / 2 + i]; }
                dma<PB / 2>(g, pr.b[0] + off, lb);
                dma<PB / 2>(u, pr.b[1] + off, lb + PB * 512);
            } else {
                const char* pb = (which ? pr.b[1] : pr.b[0]) + (BKM ? k0 * pr.ldb + (int64_t)n0 * SB::ES : n0 * pr.ldb + k0 * SB::ES);
                dma<PB>(ob, pb, lb);
            }
        };
        auto issue = [&](int s, int stage) __attribute__((always_inline)) {
            const int seg = s >= p.nk ? 1 : 0, kt = s - seg * p.nk;
            const int64_t k0 = (int64_t)kt * BKE;
            if (p.K - k0 >= BKE) {
                send(offa, offb, seg, k0, stage);
            } else {                                                    // the last step of a reduction that no whole steps make: what lies beyond reads as zero
                const int left = (int)(p.K - k0);
                unsigned oa[PA], ob[PB];
#pragma unroll
                for (int i = 0; i < PA; ++i) {
                    int row, chunk;
                    SA::place(wave * PA + i, lane, &row, &chunk);
                    oa[i] = (AKM ? row : chunk * CH) < left ? offa[i] : kOob;
                }
#pragma unroll
                for (int i = 0; i < PB; ++i) {
                    int row, chunk;
                    SB::place(wave * PB + i, lane, &row, &chunk);
                    ob[i] = (BKM ? row : chunk * CH) < left ? offb[i] : kOob;
                }
                send(oa, ob, seg, k0, stage);
            }
        };

        f32x4 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        issue(s0, 0);
        if (s0 + 1 < s1) issue(s0 + 1, 1);
        if constexpr (ST == 4) {
            if (s0 + 2 < s1) issue(s0 + 2, 2);
            if (s0 + 3 < s1) issue(s0 + 3, 3);
        }
        // Fragments of a k-group: the weights' side and the last two rows have two register sets in turn, the other rows one: row i's next fragment is read behind the
        // last matrix instruction that takes its present one (256 accumulator and fragment registers hold no second set of all of them).
        i32x4 fa[TM - 2], fz[2][2], fb[2][TN];
        // matrix instructions of the group in `set`, the next group's reads (from `stage`, k-group kk) between them; first: nothing to multiply yet
        auto advance = [&](auto set_, bool first, bool more, int stage, int kk) __attribute__((always_inline)) {
            constexpr int set = decltype(set_)::value;
            const char *ta = smem + stage * STAGE, *tb = ta + BM * kStep;
            if (more) {
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[set ^ 1][j] = SB::read(tb, baseb, lane, wn * TN + j, kk);
#pragma unroll
                for (int i = 0; i < 2; ++i) fz[set ^ 1][i] = SA::read(ta, basea, lane, wm * TM + TM - 2 + i, kk);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if (!first)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::run(fb[set][j], i < TM - 2 ? fa[i] : fz[set][i - (TM - 2)], acc[i][j]);
                if (more && i < TM - 2) fa[i] = SA::read(ta, basea, lane, wm * TM + i, kk);
            }
            if (!first) {
                constexpr int RA = AKM ? (sizeof(T) == 2 ? 2 : 4) : 1, RB = BKM ? (sizeof(T) == 2 ? 2 : 4) : 1, PER = sizeof(T) == 2 ? 1 : 4;
                __builtin_amdgcn_sched_group_barrier(0x100, RB * TN + 2 * RA, 0);               // LDS reads
#pragma unroll
                for (int i = 0; i < TM - 2; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, TN * PER, 0);                   // matrix instructions
                    __builtin_amdgcn_sched_group_barrier(0x100, RA, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * TN * PER, 0);
            }
        };
        // One barrier per step, between its two k-groups: it publishes the next step's buffer (every wavefront has waited for its own DMA) and frees this step's
        // (both groups' fragments are in registers), which the DMA of the step ST later then fills.  Fragments are read one group ahead throughout.
        static_assert(ST == 2 || ST == 4, "two or four buffers");
        if (s0 + ST - 1 < s1) wait_steps<(ST - 1) * (PA + PB)>();
        else wait_steps<0>();
        advance(std::integral_constant<int, 1>{}, true, true, 0, 0);
        for (int s = s0; s < s1; ++s) {
            const int stage = (s - s0) & (ST - 1);
            advance(std::integral_constant<int, 0>{}, false, true, stage, 1);
            if constexpr (ST == 2) wait_steps<0>();
            else if (s + ST - 1 < s1) wait_steps<(ST - 2) * (PA + PB)>();                         // (the ST - 2 steps behind the next one stay under way)
            else wait_steps<0>();
            if (s + ST < s1) issue(s + ST, stage);
            advance(std::integral_constant<int, 1>{}, false, true, (stage + 1) & (ST - 1), 0);    // (behind the last step: reads of a finished buffer, not used)
        }

        // ---- epilogue.  A lane holds 4 columns of a row (8 bytes of a 16-bit row): the sums go through LDS, some rows of each row of wavefronts at a time, and come
        // back as 8 columns of one row per thread, neighbouring threads side by side: whole 128-byte lines to memory.  16-byte chunk c of a staged row lies at
        // c ^ (row & 15): the 16 rows of a write pass and the 2 rows of a read pass cover the banks once.
        constexpr int PITCH = BN * 4, CI = 64 * WM * PITCH <= ST * STAGE ? 4 : 2, CHUNKS = TM / CI, ROWS = 16 * CI * WM;
        static_assert(TM % CI == 0 && ROWS * PITCH <= ST * STAGE, "a chunk fits the stages");
        const int t = lane & 15, g4 = lane >> 4;
        constexpr int WIDE = EPI == EPI_GATE ? BN / 2 : BN, LANES = WIDE / 8, RPP = NT / LANES, PASSES = ROWS / RPP;
        const int cg = threadIdx.x % LANES, r0 = threadIdx.x / LANES, n = n0 + cg * 8;
        const int rows_here = (int)(pr.M - m0 < BM ? pr.M - m0 : BM);
        const int part_tile = item - p.whole, limit = EPI == EPI_GATE_BWD ? pr.ldo : pr.N;
        float b1[8], b2[8], c1[8], c2[8];
        if constexpr (EPI == EPI_GATE_BWD) {
#pragma unroll
            for (int e = 0; e < 8; ++e) c1[e] = c2[e] = 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) b1[e] = b2[e] = 0.f;
            if (p.bias && n < limit) load8(static_cast<const T*>(p.bias) + n, n, limit, b1);
            if (EPI == EPI_GATE && p.bias2 && n < limit) load8(static_cast<const T*>(p.bias2) + n, n, limit, b2);
        }
        auto finish = [&](auto which_chunk) __attribute__((always_inline)) {
            constexpr int chunk = decltype(which_chunk)::value;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < CI; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const int c = (wn * TN + j) * 4 + g4;
                    *reinterpret_cast<f32x4*>(smem + ((wm * CI + i) * 16 + t) * PITCH + ((c ^ t) << 4)) = acc[chunk * CI + i][j];
                }
            __syncthreads();
            auto staged = [&](int r, int col, float (&v)[8]) __attribute__((always_inline)) {
                const char* row = smem + r * PITCH;
                const int c = col >> 2;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(row + ((c ^ (r & 15)) << 4)), hi = *reinterpret_cast<const f32x4*>(row + (((c + 1) ^ (r & 15)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = lo[e]; v[4 + e] = hi[e]; }
            };
            auto tile_row = [&](int r) { return r / (16 * CI) * (16 * TM) + chunk * (16 * CI) + r % (16 * CI); };
            // element offset of a row's columns: 32 bits from the tile's first row on
            auto at_row = [&](int r, int ld) { return m0 * ld + n + (unsigned)(tile_row(r) * ld); };
            if constexpr (EPI == EPI_GATE) {
#pragma unroll
                for (int q = 0; q < PASSES; ++q) {
                    const int r = r0 + q * RPP;
                    if (tile_row(r) >= rows_here || n >= limit) continue;
                    float gv[8], uv[8], hv[8];
                    const int col = (cg >> 1) * 32 + (cg & 1) * 8;     // 16 gate columns, 16 up columns, ...
                    staged(r, col, gv);
                    staged(r, col + 16, uv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        gv[e] += b1[e];
                        uv[e] += b2[e];
                    }
                    act8(gv, p.act, hv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) hv[e] *= uv[e];
                    const int64_t o = at_row(r, pr.ldo);
                    if (p.kept) {
                        keep8<T>(p.kept, pr.M * pr.N, 0, o, n, limit, gv);
                        keep8<T>(p.kept, pr.M * pr.N, 1, o, n, limit, uv);
                    }
                    store8(static_cast<T*>(pr.out) + o, n, limit, hv);
                }
            } else if constexpr (EPI == EPI_GATE_BWD) {
                constexpr int BATCH = sizeof(T) == 2 || TM == 4 ? 4 : 2;    // rows whose g and u are in flight together
                static_assert(PASSES % BATCH == 0, "");
#pragma unroll 1
                for (int q0 = 0; q0 < PASSES; q0 += BATCH) {
                    Kept8<T> gr[BATCH], ur[BATCH];
#pragma unroll
                    for (int q = 0; q < BATCH; ++q) {
                        const int r = r0 + (q0 + q) * RPP, lim = tile_row(r) < rows_here ? pr.N : 0;
                        const int64_t o = at_row(r, pr.N);
                        gr[q].load(p.kept, pr.M * pr.N, 0, o, n, lim);
                        ur[q].load(p.kept, pr.M * pr.N, 1, o, n, lim);
                    }
#pragma unroll
                    for (int q = 0; q < BATCH; ++q) {
                        const int r = r0 + (q0 + q) * RPP;
                        if (tile_row(r) >= rows_here || n >= limit) continue;
                        float dh[8], gv[8], a[8], da[8], dg[8], du[8];
                        staged(r, cg * 8, dh);
#pragma unroll
                        for (int e = 0; e < 8; ++e) gv[e] = gr[q].get(e);
                        act8_both(gv, p.act, a, da);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            dg[e] = dh[e] * ur[q].get(e) * da[e];
                            du[e] = dh[e] * a[e];
                        }
                        if (n + 8 > pr.N)                               // columns of padding are written as zeros
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (n + e >= pr.N) dg[e] = du[e] = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            c1[e] += dg[e];
                            c2[e] += du[e];
                        }
                        const int64_t o = at_row(r, pr.ldo);
                        store8(static_cast<T*>(pr.out) + o, n, limit, dg);
                        store8(static_cast<T*>(p.uout) + o, n, limit, du);
                    }
                }
            } else {
#pragma unroll 2
                for (int q = 0; q < PASSES; ++q) {
                    const int r = r0 + q * RPP;
                    float v[8];
                    staged(r, cg * 8, v);
                    if (!complete) {
                        float* o = p.part + (((int64_t)part_tile * p.splits + split) * BM + tile_row(r)) * BN + cg * 8;
                        __builtin_memcpy(o, v, sizeof v);
                        continue;
                    }
                    if (tile_row(r) >= rows_here || n >= limit) continue;
                    O* o = static_cast<O*>(pr.out) + at_row(r, pr.ldo);
                    float old[8];
                    if (p.accumulate) load8(o, n, limit, old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += p.accumulate ? old[e] : b1[e];
                    store8(o, n, limit, v);
                }
            }
        };
        finish(std::integral_constant<int, 0>{});
        if constexpr (CHUNKS > 1) finish(std::integral_constant<int, 1>{});
        if constexpr (CHUNKS > 2) {
            finish(std::integral_constant<int, 2>{});
            finish(std::integral_constant<int, 3>{});
        }
        static_assert(CHUNKS == 1 || CHUNKS == 2 || CHUNKS == 4, "");
        if constexpr (EPI == EPI_GATE_BWD)
            if (p.cols) {                                               // the tile's column sums of dg and du: RPP partial sums per column, in order
                float* red = reinterpret_cast<float*>(smem);
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    red[r0 * BN + cg * 8 + e] = c1[e];
                    red[(RPP + r0) * BN + cg * 8 + e] = c2[e];
                }
                __syncthreads();
                for (int i = threadIdx.x; i < 2 * BN; i += NT) {
                    const int which = i / BN, c = i - which * BN;
                    float sum = 0.f;
#pragma unroll
                    for (int r = 0; r < RPP; ++r) sum += red[(which * RPP + r) * BN + c];
                    if (n0 + c < pr.N) (which ? p.cols2 : p.cols)[(int64_t)tile_m * pr.N + n0 + c] = sum;
                }
            }
    }
}

// The shared tiles: out[m][n] = sum of the parts, in the order of k [+ bias[n]] [+ out].  Grid: (shared tiles, slices of a tile's rows)
template <typename T, typename O, int BM, int BN>
__global__ __launch_bounds__(256) void gemm_lowp_join(const GemmArgs p) {
    int tile_m, tile_n;
    const Product pr = tile_of(p, (int)blockIdx.x + p.whole, &tile_m, &tile_n);
    constexpr int LANES = BN / 8, RPP = 256 / LANES;
    const int64_t m0 = (int64_t)tile_m * BM;
    const int cg = threadIdx.x % LANES, n = tile_n * BN + cg * 8;
    if (n >= pr.N) return;
    const int rows = BM / gridDim.y;
    for (int r = blockIdx.y * rows + threadIdx.x / LANES; r < (int)(blockIdx.y + 1) * rows; r += RPP) {
        const int64_t m = m0 + r;
        if (m >= pr.M) return;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8];
        const float* part = p.part + ((int64_t)blockIdx.x * p.splits * BM + r) * BN + cg * 8;
#pragma unroll 4
        for (int z = 0; z < p.splits; ++z) {
            __builtin_memcpy(v, part + (int64_t)z * BM * BN, sizeof v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
        if (p.bias) {
            load8(static_cast<const T*>(p.bias) + n, n, pr.N, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
        O* o = static_cast<O*>(pr.out) + m * pr.ldo + n;
        if (p.accumulate) {
            load8(o, n, pr.N, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
        store8(o, n, pr.N, s);
    }
}

// rows of c elements copied to rows of cp >= c elements, zeros behind (operands whose rows are no multiple of 16 bytes)
template <typename T>
__global__ __launch_bounds__(256) void pad_rows(const T* __restrict__ src, int64_t rows, int c, int cp, T* __restrict__ dst) {
    constexpr int CH = 16 / sizeof(T);
    const int per = cp / CH;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int j = (int)(i - r * per) * CH;
        float v[CH];
#pragma unroll
        for (int e = 0; e < CH; ++e) v[e] = j + e < c ? (float)src[r * c + j + e] : 0.f;
        store_n<T, CH>(dst + r * cp + j, v);
    }
}

// ------------------------------------------------------------------------------------------ host side
struct Plan {
    int big = 0, tiles = 0, whole = 0, splits = 1, deep = 0;
    int grid() const { return whole + (tiles - whole) * splits; }
    int64_t part_bytes() const { return (int64_t)(tiles - whole) * splits * (big ? 256 * 256 : 128 * 128) * 4; }
};

// Tile: 256 x 256 (one workgroup of 8 wavefronts per CU) or 128 x 128 (4 wavefronts, two workgroups per CU).  A step of a large tile takes about 1.5 us on the
// full chip, a step of two small ones 1.0 us for half the work (fp32: 7.8 and 4.2 us); filling the pipeline and storing costs about 6 and 3 us.  Where no CU gets a second small
// workgroup, its LDS holds four buffers and three steps of loads stay under way: bf16 1000 x 768 x 2048 forward 42.2 -> 37.1 us, 2048 x 2048 x 5632 gradients 376 -> 340 us (fp32
// products wait for matrix instructions there: no gain, no loss).  Parts of a tile go down to 4 steps (fp32 500 x 384 x 1024 gradients with 8: 100 us, with 4: 90).  Whichever the sizes make cheaper by
// that count, padding of the last tiles and the last round of workgroups included, is taken.
// Shared tiles (products whose epilogue is linear): the tiles beyond the last full round are cut along k in equal parts, whose sums meet in a second launch in
// the order of k, where the parts' way through memory costs less than the idle CUs.
inline Plan plan_gemm(int count, const int64_t (*mn)[2], int64_t steps, int es, bool share) {
    Plan best;
    double best_us = 0.;
    for (int big = 0; big < 2; ++big) {
        const int64_t b = big ? 256 : 128, slots = big ? 256 : 512;
        int64_t tiles = 0;
        for (int i = 0; i < count; ++i) tiles += ceil_div(mn[i][0], b) * ceil_div(mn[i][1], b);
        if (tiles == 0) return best;
        const int64_t rest = tiles % slots;
        const double step = es == 2 ? (big ? 1.5 : 1.0) : (big ? 7.8 : 4.2), ends = big ? 6. : 3., full = (double)steps * step + ends;
        Plan q;
        q.big = big;
        q.tiles = q.whole = (int)tiles;
        // (a last round with one small workgroup per CU runs faster than one with two, with four buffers and 16-bit operands twice as fast)
        const double alone = es == 2 ? 0.5 : 0.6;
        double tail = rest == 0 ? 0. : (big || rest > slots / 2 ? full : (tiles <= 256 ? alone : 0.6) * full);
        if (share)
            for (int64_t z = 2; z <= 64 && rest > 0 && steps / z >= 4; ++z) {
                const double speed = !big && tiles < slots && rest * z <= 256 ? alone : 1.;
                const double us = (double)ceil_div(rest * z, slots) * ((double)ceil_div(steps, z) * step * speed + ends) + 6. + (double)(rest * z) * (big ? 0.262 : 0.0655) * 2 / 4.;
                if (us < tail) {
                    tail = us;
                    q.whole = (int)(tiles - rest);
                    q.splits = (int)z;
                }
            }
        const double us = (double)(tiles / slots) * full + tail;
        q.deep = !big && q.grid() <= 256;
        if (!big || us < best_us) {
            best = q;
            best_us = us;
        }
    }
    return best;
}
inline Plan plan_gemm(int64_t M, int64_t N, int64_t steps, int es, bool share) {
    const int64_t mn[1][2] = {{M, N}};
    return plan_gemm(1, mn, steps, es, share);
}

// more than 64 KB of LDS for a kernel: asked for once per device
template <auto kernel> int allow_lds(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return check_launch("gated_ffn: device");
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return SUHPE_OK;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return check_launch("gated_ffn: LDS size");
    done.fetch_or(bit, std::memory_order_relaxed);
    return SUHPE_OK;
}

template <typename T, typename O, bool AKM, bool BKM, int EPI>
int gemm_launch(GemmArgs a, int products, const Plan& q, hipStream_t st) {
    const int bm = q.big ? 256 : 128, bn = EPI == EPI_GATE ? bm / 2 : bm;
    for (int i = 0; i < products; ++i) {
        a.pr[i].tiles_m = (int)ceil_div(a.pr[i].M, bm);
        a.pr[i].tiles_n = (int)ceil_div(EPI == EPI_GATE_BWD ? a.pr[i].ldo : a.pr[i].N, bn);
    }
    a.tiles = q.tiles;
    a.whole = q.whole;
    a.splits = q.splits;
    a.nk = (int)ceil_div(a.K, kStep / (int)sizeof(T));
    const dim3 grid((unsigned)q.grid());
    const int lds = 2 * (bm + bm) * kStep;                             // two stages of either side's rows
    if (q.big) {
        constexpr auto k = gemm_lowp<T, O, 8, 4, 2, 4, 2, AKM, BKM, EPI>;
        if (int rc = allow_lds<k>(lds)) return rc;
        hipLaunchKernelGGL(k, grid, dim3(512), lds, st, a);
    } else {
        constexpr auto k = gemm_lowp<T, O, 4, 4, 2, 2, 2, AKM, BKM, EPI>;
        constexpr auto deep = gemm_lowp<T, O, 4, 4, 2, 2, 4, AKM, BKM, EPI>;
        if (q.deep) {
            if (int rc = allow_lds<deep>(2 * lds)) return rc;
            hipLaunchKernelGGL(deep, grid, dim3(256), 2 * lds, st, a);
        } else {
            hipLaunchKernelGGL(k, grid, dim3(256), lds, st, a);
        }
    }
    if constexpr (EPI == EPI_STORE)
        if (q.whole < q.tiles) {
            if (q.big) hipLaunchKernelGGL((gemm_lowp_join<T, O, 256, 256>), dim3(q.tiles - q.whole, 16), dim3(256), 0, st, a);
            else hipLaunchKernelGGL((gemm_lowp_join<T, O, 128, 128>), dim3(q.tiles - q.whole, 8), dim3(256), 0, st, a);
        }
    return check_launch("gated_ffn: product");
}

}  // namespace
}  // namespace suhpe

// Matrix products of the gated feed-forward block (included by gated_ffn.hip): out[m][j] = sum_k A(m, k) B(j, k) in fp32 / bf16 / fp16, sums in fp32.
//
// Each operand lies in memory with its reduction axis contiguous ("rows of k": x, weights in the forward) or across rows ("k-major": weights in the input
// gradients, both operands of the weight gradients); all four combinations run the same loop.  A workgroup owns a BM x BN tile; per step it stages 128
// bytes of k (64 sixteen-bit or 32 fp32 elements) of every row by global -> LDS DMA (16 bytes a lane, no registers) into one of two buffers while the
// matrix instructions read the other; one barrier per step publishes the new buffer and frees the old one.
//
// LDS layouts, both without padding (DMA fills LDS linearly, so the SOURCE address carries the permutation):
//   rows of k:  row r of the tile = 128 bytes, its 16-byte chunk c at position c ^ ((r >> 1) & 7): the 16 lanes of one ds_read_b128 pass cover the 64 banks once
//   k-major:    row k of the tile = BM (BN) elements.  Sixteen bits: fragments come out of ds_read_b64_tr_b16 (a 16-lane group reads 4 rows of k x 16 columns
//               and returns them transposed), chunk c at c ^ (f << 1) with f = (k & 3) | ((k >> 3 & 1) << 2): the 8 rows that a pass touches lie in 8 different
//               32-byte slots.  fp32: 4-byte reads, chunk c at c ^ ((k >> 2 & 3) << 2): the 4 rows of a pass lie in 4 different 64-byte slots.
// Fragment order of k is the same for every layout (lane group g of 16 takes k = 8 g .. 8 g + 7 of 32, fp32: 4 g + e of 16), so results do not depend on it.
// The weights' side is the FIRST matrix operand: a lane then holds 4 consecutive output columns of one row, stored as one vector.

#include <type_traits>

namespace suhpe {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

enum { EPI_STORE = 0, EPI_GATE = 1, EPI_GATE_BWD = 2 };

struct Operand {
    const char* p[2];                                                  // by segment / problem, or (EPI_GATE's B) gate and up weights
    int64_t ld;                                                        // bytes from row to row
    int64_t rows;                                                      // extent of the axis that is not k
};

struct GemmArgs {
    Operand a, b;
    int64_t M;                                                         // output rows
    int N;                                                             // output columns (EPI_GATE: of g, u, h)
    int64_t K;                                                         // reduction of ONE segment
    int nk, nseg, problems;                                            // steps of a segment; segments; independent products
    int tiles_m, tiles_n;
    int whole, streams;                                                // tiles that one workgroup reduces alone; workgroups that share the others' steps
    const void *bias, *bias2, *gin, *uin;
    void *out[2], *gout, *uout;                                        // EPI_GATE: out = h; EPI_GATE_BWD: gout = dg, uout = du
    int ldo;                                                           // columns from row to row of what is written (>= N; EPI_GATE_BWD: zeros behind N)
    int act, accumulate;
    float* part;                                                       // streams > 0: [2 streams][BM][BN]
    float *cols, *cols2;                                               // EPI_GATE_BWD: column sums of dg and du, [row tile][N], or null
};

// Steps first .. of the shared tiles that stream w takes (the shared tiles' steps, laid end to end, in equal parts)
__host__ __device__ __forceinline__ int64_t stream_start(int64_t total, int streams, int64_t w) { return total * w / streams; }

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
    else {
        static_assert(N == 2, "two or four pieces");
        asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %1, %3, 0 offen lds\n\ts_add_u32 m0, m0, 1024\n\ts_nop 2\n\t"
                     "buffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(off[0]), "v"(off[1]), "s"(r), "s"(lds) : "memory", "scc");
    }
}

// LDS-side geometry of one operand: R rows of the tile, k contiguous or k-major
template <typename T, int R, bool KM> struct Side {
    static constexpr int ES = sizeof(T), BKE = 128 / ES, CH = 16 / ES, RB = R * ES;
    // tile row (or k) and global 16-byte chunk that lane `lane` of piece q fills
    static __device__ __forceinline__ void place(int q, int lane, int* row, int* chunk) {
        if constexpr (!KM) {
            const int r = q * 8 + (lane >> 3);
            *row = r;
            *chunk = (lane & 7) ^ ((r >> 1) & 7);
        } else {
            const int at = q * 1024 + lane * 16, k = at / RB, c = (at % RB) >> 4;
            *row = k;
            *chunk = ES == 2 ? c ^ (((k & 3) | ((k >> 3 & 1) << 2)) << 1) : c ^ ((k >> 2 & 3) << 2);
        }
    }
    // byte offset of this lane's share of the fragment of rows 16 rb .. 16 rb + 15, k-group 0
    static __device__ __forceinline__ int lane_base(int lane) {
        const int g = lane >> 4, t = lane & 15;
        if constexpr (!KM) return t * 128;
        else if constexpr (ES == 2) return (g * 8 + (t >> 2)) * RB + (t & 1) * 8;
        else return (g * 4) * RB + (t & 3) * 4;
    }
    static __device__ __forceinline__ i32x4 read(const char* tile, int base, int lane, int rb, int kk) {
        const int g = lane >> 4, t = lane & 15;
        if constexpr (!KM) {
            return *reinterpret_cast<const i32x4*>(tile + base + rb * 2048 + (((kk * 4 + g) ^ ((t >> 1) & 7)) << 4));
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

template <typename T, typename O, int TM, int TN, int WM, int WN, bool AKM, bool BKM, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void gemm_lowp(const GemmArgs p) {
    constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, NW = WM * WN, NT = 64 * NW;
    using SA = Side<T, BM, AKM>;
    using SB = Side<T, BN, BKM>;
    constexpr int BKE = SA::BKE, CH = SA::CH, KG = 2;                   // k-groups of a step: 2 x 32 (fp32: 2 x 16)
    constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, STAGE = (BM + BN) * 128;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int wm = wave / WN, wn = wave % WN;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int basea = SA::lane_base(lane), baseb = SB::lane_base(lane);
    const int steps = p.nk * p.nseg, tiles = p.tiles_m * p.tiles_n;

    // this workgroup's share: one whole tile, or a range of the shared tiles' steps (pieces of at most two tiles and whole ones between them)
    int64_t at, end;
    int stream = -1;
    if ((int)blockIdx.x < p.whole) {
        at = (int64_t)xcd_order(blockIdx.x, p.whole) * steps;
        end = at + steps;
    } else {
        const int64_t total = ((int64_t)tiles * p.problems - p.whole) * steps;
        stream = xcd_order(blockIdx.x - p.whole, p.streams);
        at = (int64_t)p.whole * steps + stream_start(total, p.streams, stream);
        end = (int64_t)p.whole * steps + stream_start(total, p.streams, stream + 1);
    }
    for (int piece = 0; at < end; piece = 1) {
        int item = (int)(at / steps);
        const int s0 = (int)(at - (int64_t)item * steps), s1 = (int)(end - at < steps - s0 ? s0 + (end - at) : steps);
        at += s1 - s0;
        const bool complete = s0 == 0 && s1 == steps;
        const int prob = item / tiles;
        item -= prob * tiles;
        // tiles in groups of 8 rows of tiles x all columns: neighbours in the order share operands in L2
        constexpr int GROUP = 8;
        const int group = item / (GROUP * p.tiles_n), gm0 = group * GROUP, gsize = p.tiles_m - gm0 < GROUP ? p.tiles_m - gm0 : GROUP;
        item -= group * GROUP * p.tiles_n;
        const int tile_m = gm0 + item % gsize;
        const int64_t m0 = (int64_t)tile_m * BM;
        const int n0 = (item / gsize) * (EPI == EPI_GATE ? BN / 2 : BN);

        // this lane's pieces: byte offset within the step's source rows, and the first k of its chunk (k-major: its row of k) for the tail of the reduction
        unsigned offa[PA], offb[PB];
        int ka[PA], kb[PB];
#pragma unroll
        for (int i = 0; i < PA; ++i) {
            int row, chunk;
            SA::place(wave * PA + i, lane, &row, &chunk);
            if constexpr (!AKM) {
                const int64_t r = m0 + row < p.a.rows ? row : p.a.rows - 1 - m0;                // rows beyond the last repeat it: never stored
                offa[i] = (unsigned)(r * p.a.ld + chunk * 16);
                ka[i] = chunk * CH;
            } else {
                offa[i] = m0 + chunk * CH < p.a.rows ? (unsigned)(row * p.a.ld + chunk * 16) : kOob;
                ka[i] = row;
            }
        }
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            int row, chunk;
            SB::place(wave * PB + i, lane, &row, &chunk);
            if constexpr (!BKM) {
                if constexpr (EPI == EPI_GATE) row = (row >> 5) * 16 + (row & 15);              // 16 gate rows, 16 up rows, ...
                const int64_t r = n0 + row < p.b.rows ? row : p.b.rows - 1 - n0;
                offb[i] = (unsigned)(r * p.b.ld + chunk * 16);
                kb[i] = chunk * CH;
            } else {
                offb[i] = n0 + chunk * CH < p.b.rows ? (unsigned)(row * p.b.ld + chunk * 16) : kOob;
                kb[i] = row;
            }
        }
        auto issue = [&](int s, int stage) __attribute__((always_inline)) {
            const int seg = s >= p.nk ? 1 : 0, kt = s - seg * p.nk, which = seg + prob;
            const int64_t k0 = (int64_t)kt * BKE;
            const int left = (int)(p.K - k0 < BKE ? p.K - k0 : BKE);                            // elements of k in this step
            const char* pa = p.a.p[which] + (AKM ? k0 * p.a.ld + m0 * SA::ES : m0 * p.a.ld + k0 * SA::ES);
            unsigned oa[PA], ob[PB];
#pragma unroll
            for (int i = 0; i < PA; ++i) oa[i] = ka[i] < left ? offa[i] : kOob;
#pragma unroll
            for (int i = 0; i < PB; ++i) ob[i] = kb[i] < left ? offb[i] : kOob;
            const unsigned la = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + wave * PA * 1024);
            const unsigned lb = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + BM * 128 + wave * PB * 1024);
            dma<PA>(oa, pa, la);
            if constexpr (EPI == EPI_GATE) {                           // pieces 4 q, 4 q + 1: gate rows; 4 q + 2, 4 q + 3: up rows
                static_assert(PB == 4 && !BKM, "a wavefront fills whole blocks of 16 gate and 16 up rows");
                const int64_t off = n0 * p.b.ld + k0 * SB::ES;
                const unsigned g[2] = {ob[0], ob[1]}, u[2] = {ob[2], ob[3]};
                dma<2>(g, p.b.p[0] + off, lb);
                dma<2>(u, p.b.p[1] + off, lb + 2048);
            } else {
                const char* pb = p.b.p[which] + (BKM ? k0 * p.b.ld + (int64_t)n0 * SB::ES : n0 * p.b.ld + k0 * SB::ES);
                dma<PB>(ob, pb, lb);
            }
        };

        f32x4 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (piece) __syncthreads();                                    // the previous piece's results have left LDS
        issue(s0, 0);
        for (int s = s0; s < s1; ++s) {
            const int stage = (s - s0) & 1;
            // this wavefront's DMA of step s has landed and its reads of the other buffer are done; after the barrier that holds for all of them
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (s + 1 < s1) issue(s + 1, stage ^ 1);
            const char *ta = smem + stage * STAGE, *tb = ta + BM * 128;
#pragma unroll
            for (int kk = 0; kk < KG; ++kk) {
                i32x4 fa[TM], fb[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[j] = SB::read(tb, baseb, lane, wn * TN + j, kk);
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[i] = SA::read(ta, basea, lane, wm * TM + i, kk);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = Mfma<T>::run(fb[j], fa[i], acc[i][j]);
            }
        }

        // ---- epilogue.  A lane holds 4 columns of a row (8 bytes of a 16-bit row): the sums go through LDS, 64 rows of each row of wavefronts at a time, and come
        // back as 8 columns of one row per thread, neighbouring threads side by side: whole 128-byte lines to memory.  16-byte chunk c of a staged row lies at
        // c ^ (row & 15): the 16 rows of a write pass and the 2 rows of a read pass cover the banks once.
        constexpr int CHUNKS = TM / 4, ROWS = 64 * WM, PITCH = BN * 4;
        static_assert(TM % 4 == 0 && ROWS * PITCH <= 2 * STAGE, "a chunk fits the two stages");
        const int t = lane & 15, g4 = lane >> 4;
        constexpr int WIDE = EPI == EPI_GATE ? BN / 2 : BN, LANES = WIDE / 8, RPP = NT / LANES, PASSES = ROWS / RPP;
        const int cg = threadIdx.x % LANES, r0 = threadIdx.x / LANES, n = n0 + cg * 8;
        const int limit = EPI == EPI_GATE_BWD ? p.ldo : p.N;
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
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const int c = (wn * TN + j) * 4 + g4;
                    *reinterpret_cast<f32x4*>(smem + (wm * 64 + i * 16 + t) * PITCH + ((c ^ t) << 4)) = acc[chunk * 4 + i][j];
                }
            __syncthreads();
            auto staged = [&](int r, int col, float (&v)[8]) __attribute__((always_inline)) {
                const char* row = smem + r * PITCH;
                const int c = col >> 2;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(row + ((c ^ (r & 15)) << 4)), hi = *reinterpret_cast<const f32x4*>(row + (((c + 1) ^ (r & 15)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = lo[e]; v[4 + e] = hi[e]; }
            };
            auto row_of = [&](int r) { return m0 + (r >> 6) * (16 * TM) + chunk * 64 + (r & 63); };
            if constexpr (EPI == EPI_GATE) {
#pragma unroll
                for (int q = 0; q < PASSES; ++q) {
                    const int r = r0 + q * RPP;
                    const int64_t m = row_of(r);
                    if (m >= p.M || n >= limit) continue;
                    float gv[8], uv[8], hv[8];
                    const int col = (cg >> 1) * 32 + (cg & 1) * 8;     // 16 gate columns, 16 up columns, ...
                    staged(r, col, gv);
                    staged(r, col + 16, uv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        gv[e] += b1[e];
                        uv[e] += b2[e];
                        hv[e] = act_apply(gv[e], p.act) * uv[e];
                    }
                    const int64_t o = m * p.ldo + n;
                    if (p.gout) {
                        store8(static_cast<T*>(p.gout) + o, n, limit, gv);
                        store8(static_cast<T*>(p.uout) + o, n, limit, uv);
                    }
                    store8(static_cast<T*>(p.out[0]) + o, n, limit, hv);
                }
            } else if constexpr (EPI == EPI_GATE_BWD) {
                constexpr int BATCH = 16 / (int)sizeof(T) / 2;          // rows whose g and u are in flight together
                static_assert(PASSES % BATCH == 0, "");
#pragma unroll 1
                for (int q0 = 0; q0 < PASSES; q0 += BATCH) {
                    T gr[BATCH][8], ur[BATCH][8];
#pragma unroll
                    for (int q = 0; q < BATCH; ++q) {
                        const int64_t m = row_of(r0 + (q0 + q) * RPP), o = m * p.N + n;
                        const T *gi = static_cast<const T*>(p.gin) + o, *ui = static_cast<const T*>(p.uin) + o;
                        if (m < p.M && n + 8 <= p.N) {
                            __builtin_memcpy(gr[q], gi, sizeof gr[q]);
                            __builtin_memcpy(ur[q], ui, sizeof ur[q]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const bool ok = m < p.M && n + e < p.N;
                                gr[q][e] = ok ? gi[e] : (T)0.f;
                                ur[q][e] = ok ? ui[e] : (T)0.f;
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < BATCH; ++q) {
                        const int r = r0 + (q0 + q) * RPP;
                        const int64_t m = row_of(r);
                        if (m >= p.M || n >= limit) continue;
                        float dh[8], dg[8], du[8];
                        staged(r, cg * 8, dh);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float gv = (float)gr[q][e], uv = (float)ur[q][e];
                            const bool ok = n + e < p.N;               // (columns of padding are written as zeros)
                            dg[e] = ok ? dh[e] * uv * act_grad(gv, p.act) : 0.f;
                            du[e] = ok ? dh[e] * act_apply(gv, p.act) : 0.f;
                            c1[e] += dg[e];
                            c2[e] += du[e];
                        }
                        const int64_t o = m * p.ldo + n;
                        store8(static_cast<T*>(p.gout) + o, n, limit, dg);
                        store8(static_cast<T*>(p.uout) + o, n, limit, du);
                    }
                }
            } else {
#pragma unroll 2
                for (int q = 0; q < PASSES; ++q) {
                    const int r = r0 + q * RPP;
                    float v[8];
                    staged(r, cg * 8, v);
                    if (!complete) {                                    // a shared tile's piece: the first tile of the stream in slot 2 w, the last in 2 w + 1
                        float* o = p.part + ((int64_t)(2 * stream + piece) * BM + (r >> 6) * (16 * TM) + chunk * 64 + (r & 63)) * BN + cg * 8;
                        __builtin_memcpy(o, v, sizeof v);
                        continue;
                    }
                    const int64_t m = row_of(r);
                    if (m >= p.M || n >= limit) continue;
                    O* o = static_cast<O*>(p.out[prob]) + m * p.ldo + n;
                    float old[8];
                    if (p.accumulate) load8(o, n, limit, old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += p.accumulate ? old[e] : b1[e];
                    store8(o, n, limit, v);
                }
            }
        };
        finish(std::integral_constant<int, 0>{});
        if constexpr (CHUNKS == 2) finish(std::integral_constant<int, 1>{});
        static_assert(CHUNKS <= 2, "");
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
                    if (n0 + c < p.N) (which ? p.cols2 : p.cols)[(int64_t)tile_m * p.N + n0 + c] = sum;
                }
            }
    }
}

// The shared tiles: out[m][n] = sum of the pieces, in the order of k [+ bias[n]] [+ out].  Grid: (shared tiles, slices of a tile's rows)
template <typename T, typename O, int BM, int BN>
__global__ __launch_bounds__(256) void gemm_lowp_join(const GemmArgs p) {
    const int steps = p.nk * p.nseg, tiles = p.tiles_m * p.tiles_n;
    const int64_t total = ((int64_t)tiles * p.problems - p.whole) * steps, lo = (int64_t)blockIdx.x * steps, hi = lo + steps;
    int64_t w0 = lo * p.streams / total;                                // the stream that holds step lo
    while (w0 > 0 && stream_start(total, p.streams, w0) > lo) --w0;
    while (stream_start(total, p.streams, w0 + 1) <= lo) ++w0;
    if (stream_start(total, p.streams, w0) <= lo && stream_start(total, p.streams, w0 + 1) >= hi) return;      // one stream had it all
    int item = (int)blockIdx.x + p.whole;
    const int prob = item / tiles;
    item -= prob * tiles;
    constexpr int GROUP = 8, LANES = BN / 8, RPP = 256 / LANES;
    const int group = item / (GROUP * p.tiles_n), gm0 = group * GROUP, gsize = p.tiles_m - gm0 < GROUP ? p.tiles_m - gm0 : GROUP;
    item -= group * GROUP * p.tiles_n;
    const int64_t m0 = (int64_t)(gm0 + item % gsize) * BM;
    const int n0 = (item / gsize) * BN, cg = threadIdx.x % LANES, n = n0 + cg * 8;
    if (n >= p.N) return;
    const int rows = BM / gridDim.y;
    for (int r = blockIdx.y * rows + threadIdx.x / LANES; r < (int)(blockIdx.y + 1) * rows; r += RPP) {
        const int64_t m = m0 + r;
        if (m >= p.M) return;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8];
        for (int64_t w = w0; w < p.streams && stream_start(total, p.streams, w) < hi; ++w) {
            const bool first = stream_start(total, p.streams, w) / steps == (int64_t)blockIdx.x;
            __builtin_memcpy(v, p.part + ((2 * w + (first ? 0 : 1)) * BM + r) * BN + cg * 8, sizeof v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
        if (p.bias) {
            load8(static_cast<const T*>(p.bias) + n, n, p.N, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
        O* o = static_cast<O*>(p.out[prob]) + m * p.ldo + n;
        if (p.accumulate) {
            load8(o, n, p.N, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
        store8(o, n, p.N, s);
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
    int big, whole, streams;
    int64_t tiles_m, tiles_n;
    int64_t part_bytes() const { return streams ? (int64_t)2 * streams * (big ? 256 * 256 : 128 * 128) * 4 : 0; }
};

// Tile: 256 x 256 (one workgroup of 8 wavefronts per CU) or 128 x 128 (4 wavefronts, two workgroups per CU).  A step of a large tile takes about 1.9 us on the
// full chip, a step of two small ones 1.1 us for half the work; filling the pipeline and storing costs about 6 and 3 us.  Whichever the sizes make cheaper by
// that count, padding of the last tiles and the last round of workgroups included, is taken.
// Shared tiles (products whose epilogue is linear): the tiles beyond the last full round are cut along k, their steps laid end to end and dealt out evenly, at
// least 8 to a workgroup; the pieces are summed by a second launch in the order of k.  2 x 5632 x 2048 weight gradients over 16384 rows: 352 tiles take 2 rounds of
// 256 (31 % idle), shared 1.375.
inline Plan plan_gemm(int64_t M, int64_t N, int64_t steps, int problems, bool share) {
    Plan best{};
    if (M == 0) return best;
    double best_us = 0.;
    for (int big = 0; big < 2; ++big) {
        const int64_t b = big ? 256 : 128, slots = big ? 256 : 512;
        Plan q{big, 0, 0, ceil_div(M, b), ceil_div(N, b)};
        const int64_t tiles = q.tiles_m * q.tiles_n * problems, rounds = tiles / slots, rest = tiles - rounds * slots;
        const double step = big ? 1.9 : 1.1, ends = big ? 6. : 3.;
        double us = (double)rounds * ((double)steps * step + ends);
        // alone, the rest runs as long as a full round (the two small tiles of a CU at least share it); shared, its part plus the pieces' way through memory
        const double alone = (double)steps * step * (big || rest > slots / 2 ? 1. : 0.6) + ends;
        int64_t w = rest * steps / 8;
        if (w > slots) w = slots;
        const double shared = w > 0 ? (double)(rest * steps) / (double)w * step + 2 * ends + (double)w * 2 * (big ? 0.262 : 0.0655) * 2 / 4. : 1e30;
        if (rest == 0) q.whole = (int)tiles;
        else if (share && w > rest && shared < alone) { q.whole = (int)(rounds * slots); q.streams = (int)w; us += shared; }
        else { q.whole = (int)tiles; us += alone; }
        if (!big || us < best_us) { best = q; best_us = us; }
    }
    return best;
}

template <typename T, typename O, bool AKM, bool BKM, int EPI>
int gemm_launch(GemmArgs a, const Plan& q, hipStream_t st) {
    const int bm = q.big ? 256 : 128;
    a.tiles_m = (int)q.tiles_m;
    a.tiles_n = (int)q.tiles_n;
    a.whole = q.whole;
    a.streams = q.streams;
    a.nk = (int)ceil_div(a.K, 128 / (int)sizeof(T));
    SUHPE_REQUIRE(q.tiles_m * q.tiles_n * a.problems < 0x7fffffff, "gated_ffn: too many tiles");
    const int lds = 2 * (bm + bm) * 128;                               // two stages of 128 bytes per row of either side
    const dim3 grid((unsigned)(q.whole + q.streams));
    if (q.big) {
        auto k = gemm_lowp<T, O, 8, 4, 2, 4, AKM, BKM, EPI>;
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(k, grid, dim3(512), lds, st, a);
    } else {
        auto k = gemm_lowp<T, O, 4, 4, 2, 2, AKM, BKM, EPI>;
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(k, grid, dim3(256), lds, st, a);
    }
    if constexpr (EPI == EPI_STORE)
        if (q.streams) {
            const unsigned rest = (unsigned)(q.tiles_m * q.tiles_n * a.problems - q.whole);
            if (q.big) hipLaunchKernelGGL((gemm_lowp_join<T, O, 256, 256>), dim3(rest, 16), dim3(256), 0, st, a);
            else hipLaunchKernelGGL((gemm_lowp_join<T, O, 128, 128>), dim3(rest, 8), dim3(256), 0, st, a);
        }
    return check_launch("gated_ffn: product");
}

}  // namespace
}  // namespace suhpe

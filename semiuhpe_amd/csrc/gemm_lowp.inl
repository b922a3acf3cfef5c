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
    int nk, nseg, splits, problems;                                    // steps of a segment; segments; ways the steps are split; independent products
    int tiles_m, tiles_n;
    const void *bias, *bias2, *gin, *uin;
    void *out[2], *gout, *uout;                                        // EPI_GATE: out = h; EPI_GATE_BWD: gout = dg, uout = du
    int ldo;                                                           // columns from row to row of what is written (>= N; EPI_GATE_BWD: zeros behind N)
    int act, accumulate, vec;                                          // vec: rows and pointers allow 4-column vectors
    float* part;                                                       // splits > 1: [problem][split][M][N]
};

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

template <typename T, typename O, int TM, int TN, int WM, int WN, bool AKM, bool BKM, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void gemm_lowp(const GemmArgs p) {
    constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN, NW = WM * WN;
    using SA = Side<T, BM, AKM>;
    using SB = Side<T, BN, BKM>;
    constexpr int BKE = SA::BKE, CH = SA::CH, KG = 2;                   // k-groups of a step: 2 x 32 (fp32: 2 x 16)
    constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, STAGE = (BM + BN) * 128;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int wm = wave / WN, wn = wave % WN;

    // work item: [problem][split][tile group of 8 row tiles x all column tiles]
    int item = xcd_order(blockIdx.x, gridDim.x);
    const int tiles = p.tiles_m * p.tiles_n;
    const int prob = item / (tiles * p.splits);
    item -= prob * tiles * p.splits;
    const int split = item / tiles;
    item -= split * tiles;
    constexpr int GROUP = 8;
    const int group = item / (GROUP * p.tiles_n), gm0 = group * GROUP, gsize = p.tiles_m - gm0 < GROUP ? p.tiles_m - gm0 : GROUP;
    item -= group * GROUP * p.tiles_n;
    const int64_t m0 = (int64_t)(gm0 + item % gsize) * BM;
    const int n0 = (item / gsize) * (EPI == EPI_GATE ? BN / 2 : BN);
    const int steps = p.nk * p.nseg;
    const int s0 = (int)((int64_t)steps * split / p.splits), s1 = (int)((int64_t)steps * (split + 1) / p.splits);

    // this lane's pieces: byte offset within the step's source rows, and the first k of its chunk (k-major: its row of k) for the tail of the reduction
    unsigned offa[PA], offb[PB];
    int ka[PA], kb[PB];
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        int row, chunk;
        SA::place(wave * PA + i, lane, &row, &chunk);
        if constexpr (!AKM) {
            const int64_t r = m0 + row < p.a.rows ? row : p.a.rows - 1 - m0;                    // rows beyond the last repeat it: never stored
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
            if constexpr (EPI == EPI_GATE) row = (row >> 5) * 16 + (row & 15);                  // 16 gate rows, 16 up rows, ...
            const int64_t r = n0 + row < p.b.rows ? row : p.b.rows - 1 - n0;
            offb[i] = (unsigned)(r * p.b.ld + chunk * 16);
            kb[i] = chunk * CH;
        } else {
            offb[i] = n0 + chunk * CH < p.b.rows ? (unsigned)(row * p.b.ld + chunk * 16) : kOob;
            kb[i] = row;
        }
    }
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    auto issue = [&](int s, int stage) __attribute__((always_inline)) {
        const int seg = s >= p.nk ? 1 : 0, kt = s - seg * p.nk, which = seg + prob;
        const int64_t k0 = (int64_t)kt * BKE;
        const int left = (int)(p.K - k0 < BKE ? p.K - k0 : BKE);                                // elements of k in this step
        const char* pa = p.a.p[which] + (AKM ? k0 * p.a.ld + m0 * SA::ES : m0 * p.a.ld + k0 * SA::ES);
        unsigned oa[PA], ob[PB];
#pragma unroll
        for (int i = 0; i < PA; ++i) oa[i] = ka[i] < left ? offa[i] : kOob;
#pragma unroll
        for (int i = 0; i < PB; ++i) ob[i] = kb[i] < left ? offb[i] : kOob;
        const unsigned la = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + wave * PA * 1024);
        const unsigned lb = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + BM * 128 + wave * PB * 1024);
        dma<PA>(oa, pa, la);
        if constexpr (EPI == EPI_GATE) {                               // pieces 4 q, 4 q + 1: gate rows; 4 q + 2, 4 q + 3: up rows
            static_assert(PB == 4 && !BKM, "a wavefront fills whole blocks of 16 gate and 16 up rows");
            const int64_t at = n0 * p.b.ld + k0 * SB::ES;
            const unsigned g[2] = {ob[0], ob[1]}, u[2] = {ob[2], ob[3]};
            dma<2>(g, p.b.p[0] + at, lb);
            dma<2>(u, p.b.p[1] + at, lb + 2048);
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
    const int basea = SA::lane_base(lane), baseb = SB::lane_base(lane);
    if (s0 < s1) issue(s0, 0);
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

    // ---- epilogue: lane (t, g) holds columns 16 (wn TN + j) + 4 g .. + 3 of row 16 (wm TM + i) + t
    const int t = lane & 15, g4 = (lane >> 4) * 4;
    if constexpr (EPI == EPI_GATE) {
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
            const int n = n0 + (wn * TN + j) * 8 + g4;
            float bg[4], bu[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool ok = n + r < p.N;
                bg[r] = ok && p.bias ? (float)static_cast<const T*>(p.bias)[n + r] : 0.f;
                bu[r] = ok && p.bias2 ? (float)static_cast<const T*>(p.bias2)[n + r] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int64_t m = m0 + (wm * TM + i) * 16 + t;
                if (m >= p.M || n >= p.N) continue;
                float gv[4], uv[4], hv[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    gv[r] = acc[i][j][r] + bg[r];
                    uv[r] = acc[i][j + 1][r] + bu[r];
                    hv[r] = act_apply(gv[r], p.act) * uv[r];
                }
                const int64_t at = m * p.ldo + n;
                T *go = static_cast<T*>(p.gout), *uo = static_cast<T*>(p.uout), *ho = static_cast<T*>(p.out[0]);
                if (p.vec) {
                    if (go) { store_n<T, 4>(go + at, gv); store_n<T, 4>(uo + at, uv); }
                    store_n<T, 4>(ho + at, hv);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < p.N) {
                            if (go) { go[at + r] = (T)gv[r]; uo[at + r] = (T)uv[r]; }
                            ho[at + r] = (T)hv[r];
                        }
                }
            }
        }
    } else if constexpr (EPI == EPI_GATE_BWD) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = n0 + (wn * TN + j) * 16 + g4;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int64_t m = m0 + (wm * TM + i) * 16 + t;
                if (m >= p.M || n >= p.ldo) continue;
                float gv[4], uv[4], dg[4], du[4];
                const T *gi = static_cast<const T*>(p.gin) + m * p.N + n, *ui = static_cast<const T*>(p.uin) + m * p.N + n;
                if (p.vec) {
                    load_n<T, 4>(gi, gv);
                    load_n<T, 4>(ui, uv);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        gv[r] = n + r < p.N ? (float)gi[r] : 0.f;
                        uv[r] = n + r < p.N ? (float)ui[r] : 0.f;
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool ok = n + r < p.N;                       // (columns of padding are written as zeros)
                    dg[r] = ok ? acc[i][j][r] * uv[r] * act_grad(gv[r], p.act) : 0.f;
                    du[r] = ok ? acc[i][j][r] * act_apply(gv[r], p.act) : 0.f;
                }
                const int64_t at = m * p.ldo + n;                      // (ldo is a multiple of 4)
                store_n<T, 4>(static_cast<T*>(p.gout) + at, dg);
                store_n<T, 4>(static_cast<T*>(p.uout) + at, du);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = n0 + (wn * TN + j) * 16 + g4;
            float b[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) b[r] = p.bias && n + r < p.N ? (float)static_cast<const T*>(p.bias)[n + r] : 0.f;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int64_t m = m0 + (wm * TM + i) * 16 + t;
                if (m >= p.M || n >= p.N) continue;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r];
                if (p.splits > 1) {
                    float* o = p.part + (((int64_t)prob * p.splits + split) * p.M + m) * p.N + n;
                    if ((p.N & 3) == 0) store_n<float, 4>(o, v);
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n + r < p.N) o[r] = v[r];
                    continue;
                }
                O* o = static_cast<O*>(p.out[prob]) + m * p.ldo + n;
                if (p.vec) {
                    float old[4];
                    if (p.accumulate) load_n<O, 4>(o, old);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] += p.accumulate ? old[r] : b[r];
                    store_n<O, 4>(o, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < p.N) o[r] = (O)(p.accumulate ? (float)o[r] + v[r] : v[r] + b[r]);
                }
            }
        }
    }
}

// out[m][n] = sum over the splits, in order [+ bias[n]] [+ out]
template <typename T, typename O, int V>
__global__ __launch_bounds__(256) void gemm_lowp_join(const float* __restrict__ part, int splits, int64_t M, int N, const T* __restrict__ bias, O* out0, O* out1, int accumulate) {
    const int64_t total = M * N;
    const float* src = part + (int64_t)blockIdx.y * splits * total;
    O* out = blockIdx.y ? out1 : out0;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < total; i += (int64_t)gridDim.x * 256 * V) {
        float s[V], v[V];
        load_n<float, V>(src + i, s);
        for (int z = 1; z < splits; ++z) {
            load_n<float, V>(src + z * total + i, v);
#pragma unroll
            for (int r = 0; r < V; ++r) s[r] += v[r];
        }
        if (bias) {
            const int n = (int)(i % N);
#pragma unroll
            for (int r = 0; r < V; ++r) s[r] += (float)bias[n + r];
        }
        if (accumulate) {
            load_n<O, V>(out + i, v);
#pragma unroll
            for (int r = 0; r < V; ++r) s[r] = v[r] + s[r];
        }
        store_n<O, V>(out + i, s);
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
struct Plan { int big, splits; };                                      // tile 256 x 256 or 128 x 128; ways the reduction is split

// 256 x 256 tiles keep the matrix units fed from LDS best but leave one workgroup per CU: taken where there are enough of them for the 256 CUs and the
// reduction is long enough to pay for filling and draining one.  Few tiles: the reduction is split so that about two workgroups per CU run.
inline Plan plan_gemm(int64_t M, int64_t N, int64_t steps, int problems, bool splittable) {
    Plan q{0, 1};
    if (M == 0) return q;
    const int64_t big = ceil_div(M, 256) * ceil_div(N, 256) * problems;
    const int64_t small = ceil_div(M, 128) * ceil_div(N, 128) * problems;
    if (big >= 200 && steps >= 16) q.big = 1;
    else if (splittable && small < 384) {
        int64_t s = 512 / small;
        if (s > steps / 8) s = steps / 8;
        if (s > 64) s = 64;
        q.splits = s < 1 ? 1 : (int)s;
    }
    return q;
}

template <typename T, typename O, bool AKM, bool BKM, int EPI>
int gemm_launch(GemmArgs a, Plan q, hipStream_t st) {
    const int bm = q.big ? 256 : 128, bn = EPI == EPI_GATE ? bm / 2 : bm;
    a.tiles_m = (int)ceil_div(a.M, bm);
    a.tiles_n = (int)ceil_div(EPI == EPI_GATE_BWD ? a.ldo : a.N, bn);
    a.splits = q.splits;
    a.nk = (int)ceil_div(a.K, 128 / (int)sizeof(T));
    const int64_t grid = (int64_t)a.tiles_m * a.tiles_n * a.splits * a.problems;
    SUHPE_REQUIRE(grid < 0x7fffffff, "gated_ffn: too many tiles");
    const int lds = 2 * (bm + bm) * 128;                               // two stages of 128 bytes per row of either side
    if (q.big) {
        auto k = gemm_lowp<T, O, 8, 4, 2, 4, AKM, BKM, EPI>;
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(512), lds, st, a);
    } else {
        auto k = gemm_lowp<T, O, 4, 4, 2, 2, AKM, BKM, EPI>;
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(256), lds, st, a);
    }
    if (q.splits > 1) {
        const int64_t total = a.M * a.N;
        const bool v4 = (a.N & 3) == 0 && aligned(a.out[0], 4 * sizeof(O)) && aligned(a.out[1], 4 * sizeof(O));
        const dim3 g(grid_for(ceil_div(total, v4 ? 4 : 1), 256), a.problems);
        if (v4) hipLaunchKernelGGL((gemm_lowp_join<T, O, 4>), g, dim3(256), 0, st, a.part, q.splits, a.M, a.N, static_cast<const T*>(a.bias), static_cast<O*>(a.out[0]),
                                   static_cast<O*>(a.out[1]), a.accumulate);
        else hipLaunchKernelGGL((gemm_lowp_join<T, O, 1>), g, dim3(256), 0, st, a.part, q.splits, a.M, a.N, static_cast<const T*>(a.bias), static_cast<O*>(a.out[0]),
                                static_cast<O*>(a.out[1]), a.accumulate);
    }
    return check_launch("gated_ffn: product");
}

}  // namespace
}  // namespace suhpe

// Gated feed-forward block (forward and backward) in fp32 / bf16 / fp16:
//   g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u, y = h Wd^T + bd
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h, db = column sums
//
// Forward, two products: [g | u] with the activation and the product in the epilogue (a tile takes the SAME columns of Wg and Wu, so both factors of an
// output element meet in one lane's registers), then y.  Backward, four: dh whose epilogue turns it into dg and du at once (dh itself is never stored),
// dx as one product over two ranges of n, and the three weight gradients in one launch.  h, dg and du are rounded to the tensors' type once on their way to memory
// (they are operands of 16-bit matrix instructions next; few rows, where the weights are the traffic, multiply what h's rounding left as well), g and u keep 24 bits;
// every sum runs in fp32.
#include "lowp.h"
#include "gemm_lowp.inl"

namespace suhpe {
namespace {

// ------------------------------------------------------------------------------------------ few rows (serving)
// At most 32 rows: the weights are the traffic, each is read once, straight from memory into the matrix instructions' registers.  A workgroup takes 16 / P rows of
// the weights (GATE: of both); its W wavefronts split k and their sums meet in LDS in a fixed order.
// P > 1 (at most 16 / P rows of x): the 16 x 16 matrix instruction takes P stretches of k at once -- weight row r and x row m of stretch p in its rows and columns
// 16 / P * p + r, + m -- and the blocks on its diagonal are summed: P times as many workgroups, and P * 64 bytes of a weight row side by side in one load.
// 1 x 2048 x 5632 bf16 (69 MB of weights): 15.3 us = 4.5 TB/s with P = 4, 22 us with P = 1.
// TWO: x is h between the two products, in two parts, rounded and what the rounding left, and each weight fragment is multiplied with both: bf16 leaves out 2^-16 of h then
// (rounding alone 2^-8), fp16 2^-22 or 2^-25.  The parts of a chunk lie side by side ([row][chunk][part][CH], two_at), so that a fragment's rows are read in pieces of 128 bytes.
// 2048 x 5632 bf16, both products, in a captured graph: 1 row 16.6 -> 17.3 us, 8 rows 20.8 -> 23.1, 16 rows 33.0 -> 36.9.  From 17 rows on x's loads outnumber the weights' (32
// rows: 43.9 -> 51.4 us) and h is rounded, as it is in the tile kernels.
// Rows may start at any element (16-byte loads from any address); the last chunk of a row starts at K - CH, with what the chunk before it holds set to zero.
//
// A 16-byte load from an address that is not a multiple of 4 takes several times as long (13 x 1001 x 2727 fp16, the whole block: 22 us against 10 us for
// 13 x 1002 x 2726).  ODD: a chunk that starts on an odd element is read as the 16 bytes one element further (at a row's end: one element before) and the element
// that is missing there, and shifted into place.  A row of one chunk (last == 0) has no neighbour on either side and is read where it lies.
template <typename T> __device__ __forceinline__ bool shifted(const T* chunk, int last) { return last > 0 && (reinterpret_cast<uintptr_t>(chunk) & 2); }
struct Chunk { i32x4 d; unsigned short e; };
template <typename T, bool ODD> __device__ __forceinline__ Chunk load_k(const T* row, int k, int last) {
    Chunk c;
    const int at = k < last ? k : last;
    if constexpr (!ODD) {
        __builtin_memcpy(&c.d, row + at, 16);
        c.e = 0;
    } else {
        const bool odd = shifted(row + at, last);
        __builtin_memcpy(&c.d, row + at + (odd ? (at < last ? 1 : -1) : 0), 16);
        __builtin_memcpy(&c.e, row + at + (odd && at == last ? 7 : 0), 2);
    }
    return c;
}
template <typename T, bool ODD> __device__ __forceinline__ i32x4 chunk_of(const Chunk& c, const T* row, int k, int last) {
    if constexpr (!ODD) {
        return c.d;
    } else {
        const int at = k < last ? k : last;
        const bool odd = shifted(row + at, last), behind = at < last;
        const unsigned w[5] = {behind ? (unsigned)c.e << 16 : (unsigned)c.d[0], (unsigned)(behind ? c.d[0] : c.d[1]), (unsigned)(behind ? c.d[1] : c.d[2]),
                               (unsigned)(behind ? c.d[2] : c.d[3]), behind ? (unsigned)c.d[3] : (unsigned)c.e};
        i32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = odd ? (int)__builtin_amdgcn_alignbit(w[i + 1], w[i], 16) : c.d[i];
        return v;
    }
}
// zeroes the first `gone` elements of a chunk
template <typename T> __device__ __forceinline__ i32x4 drop_first(i32x4 v, int gone) {
    constexpr int CH = 16 / (int)sizeof(T);
    typename Vec<T, CH>::type e = __builtin_bit_cast(typename Vec<T, CH>::type, v);
#pragma unroll
    for (int i = 0; i < CH; ++i) e[i] = i < gone ? (T)0.f : e[i];
    return __builtin_bit_cast(i32x4, e);
}

inline int64_t two_chunks(int n, int ch) { return ceil_div(n, ch); }
// where the first part of element n of a row of N lies: the last chunk starts at N - CH, as the weights' does, and holds what the chunk before it holds once more
template <int CH> __device__ __forceinline__ int64_t two_at(int64_t row, int n, int N, bool last) {
    const int chunks = (N + CH - 1) / CH, c = last ? chunks - 1 : n / CH;
    return (row * chunks + c) * 2 * CH + (last ? n - (N - CH) : n % CH);
}

template <typename T, int P, int MT, int W, bool GATE, bool TWO, bool ODD>
__global__ __launch_bounds__(64 * W) void ffn_few_rows(const T* __restrict__ x, int M, int64_t K, const T* __restrict__ w, const T* __restrict__ w2, int N,
                                                       const T* __restrict__ bias, const T* __restrict__ bias2, int act, void* kept, T* __restrict__ out, T* __restrict__ two_out) {
    static_assert((P == 1 || MT == 1) && !(GATE && TWO), "");
    constexpr int CH = 16 / (int)sizeof(T), KE = 4 * CH * P, S = GATE ? 2 : 1, R = 16 / P;      // KE: k of one matrix step
    __shared__ float sums[W * P][S][MT][16 * R];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, t = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * R, part = t / R, rt = t % R, nr = n0 + rt < N ? n0 + rt : N - 1;
    const T *r1 = w + nr * K, *r2 = GATE ? w2 + nr * K : nullptr;
    constexpr int MX = TWO ? 2 * MT : MT;                                   // fragments of x: MT of its rows, then MT of what their rounding left
    const int chunks = (int)((K + CH - 1) / CH);
    const T* xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = x + (int64_t)(16 * i + rt < M ? 16 * i + rt : M - 1) * (TWO ? (int64_t)chunks * 2 * CH : K);
    const int steps = (int)((K + KE - 1) / KE), lo = steps * wave / W, hi = steps * (wave + 1) / W, last = (int)K - CH;
    f32x4 acc[S][MT];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[s][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = GATE || MX > 1 ? 4 : 8;                              // steps whose loads are in flight together
    for (int q = lo; q < hi; q += U) {
        Chunk ca[U][S], cb[U][MX];
#pragma unroll
        for (int v = 0; v < U; ++v) {
            if (q + v >= hi) break;
            const int k = (q + v) * KE + (part * 4 + g) * CH;
            ca[v][0] = load_k<T, ODD>(r1, k, last);
            if constexpr (GATE) ca[v][1] = load_k<T, ODD>(r2, k, last);
#pragma unroll
            for (int i = 0; i < MX; ++i) {
                if constexpr (TWO) cb[v][i].d = *reinterpret_cast<const i32x4*>(xr[i % MT] + ((k < last ? k / CH : chunks - 1) * 2 + i / MT) * CH);
                else cb[v][i] = load_k<T, ODD>(xr[i], k, last);
            }
        }
#pragma unroll
        for (int v = 0; v < U; ++v) {
            if (q + v >= hi) break;
            const int k = (q + v) * KE + (part * 4 + g) * CH;
            i32x4 a[S], b[MX];
            a[0] = chunk_of<T, ODD>(ca[v][0], r1, k, last);
            if constexpr (GATE) a[1] = chunk_of<T, ODD>(ca[v][1], r2, k, last);
#pragma unroll
            for (int i = 0; i < MX; ++i) {
                if constexpr (TWO) b[i] = cb[v][i].d;
                else b[i] = chunk_of<T, ODD>(cb[v][i], xr[i], k, last);
            }
            if ((q + v + 1) * KE > K) {                                // the row ends in this step
                const int over = k - last;
                const int gone = over < 0 ? 0 : over > CH ? CH : over;
#pragma unroll
                for (int s = 0; s < S; ++s) a[s] = drop_first<T>(a[s], gone);
#pragma unroll
                for (int i = 0; i < MX; ++i) b[i] = drop_first<T>(b[i], gone);
            }
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < MX; ++i) acc[s][i % MT] = Mfma<T>::run(a[s], b[i], acc[s][i % MT]);
        }
    }
    // lane (t, g) holds weight rows 4 g .. 4 g + 3, x row t of each product: kept where both lie in the same stretch
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if ((4 * g + r) / R == part) sums[wave * P + part][s][i][rt * R + (4 * g + r) % R] = acc[s][i][r];
    __syncthreads();
    // 16 R sums of W P terms each (MT = 2: twice), in order; Q lanes share one
    constexpr int OUT = MT * R * R, Q = OUT >= 64 * W ? 1 : OUT <= 64 ? 64 / OUT : 1;
    const int o = (int)threadIdx.x / Q, slice = (int)threadIdx.x % Q;
    if (o >= OUT) return;
    const int i = o / (R * R), at = o % (R * R);
    float total[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        total[s] = 0.f;
#pragma unroll
        for (int v = 0; v < W * P / Q; ++v) total[s] += sums[slice * (W * P / Q) + v][s][i][at];
#pragma unroll
        for (int d = 1; d < Q; d <<= 1) total[s] += __shfl_xor(total[s], d, 64);
    }
    const int m = 16 * i + at / R, n = n0 + at % R;
    if (slice || m >= M || n >= N) return;
    const int64_t to = (int64_t)m * N + n;
    const float v = total[0] + (bias ? (float)bias[n] : 0.f);
    if constexpr (GATE) {
        const float u = total[1] + (bias2 ? (float)bias2[n] : 0.f);
        if (kept) {                                                    // (one value at a time: the last of eight columns)
            const float gv[8] = {v}, uv[8] = {u};
            keep8<T>(kept, (int64_t)M * N, 0, to, 7, 8, gv);
            keep8<T>(kept, (int64_t)M * N, 1, to, 7, 8, uv);
        }
        const float h = act_apply(v, act) * u;
        const T rounded = (T)h;
        out[to] = rounded;
        if constexpr (sizeof(T) == 2 && MT == 1) {                     // both parts for the next product; the last chunk's columns may lie in the one before it too
            const T left = fabsf((float)rounded) < INFINITY ? (T)(h - (float)rounded) : (T)0.f;
            const bool behind = n >= N - CH;
            if (!behind || n / CH * CH + CH <= N) {
                T* at = two_out + two_at<CH>(m, n, N, false);
                at[0] = rounded; at[CH] = left;
            }
            if (behind) {
                T* at = two_out + two_at<CH>(m, n, N, true);
                at[0] = rounded; at[CH] = left;
            }
        }
    } else {
        out[to] = (T)v;
    }
}

constexpr int kFewRows = 32, kTwoRows = 16;

// two (16-bit types): GATE writes h there in two parts as well, the other product takes it as x
template <typename T, bool GATE>
void few_rows(const T* x, int M, int64_t K, const T* w, const T* w2, int N, const T* bias, const T* bias2, int act, void* kept, T* out, T* two, hipStream_t st) {
    constexpr bool TWO = !GATE && sizeof(T) == 2;
#define FEW_(P, MT, W, ODD)                                                                                                                                                 \
    hipLaunchKernelGGL((ffn_few_rows<T, P, MT, W, GATE, TWO && MT == 1, ODD>), dim3((unsigned)ceil_div(N, 16 / P)), dim3(64 * W), 0, st, TWO && MT == 1 ? two : x, M, K, w, w2, \
                       N, bias, bias2, act, kept, out, GATE ? two : nullptr)
#define FEW(P, MT, W)                                       \
    do {                                                    \
        if constexpr (sizeof(T) == 2) {                     \
            if (odd) { FEW_(P, MT, W, true); break; }       \
        }                                                   \
        FEW_(P, MT, W, false);                              \
    } while (0)
    const bool odd = K % 2 || (!(TWO && M <= kTwoRows) && !aligned(x, 4)) || !aligned(w, 4) || (w2 && !aligned(w2, 4));
    if (M <= 4) FEW(4, 1, 8);
    else if (M <= 8) FEW(2, 1, 8);
    else if (M <= 16) FEW(1, 1, 16);
    else FEW(1, 2, 16);
#undef FEW_
#undef FEW
}

// ------------------------------------------------------------------------------------------ column sums (bias gradients)
// dg's and du's come from the tiles of the product that makes them, dy's from a pass of its own: [row block][columns] each, finished in a fixed order
constexpr int kColBlocks = 256;

template <typename T>
__global__ __launch_bounds__(256) void column_sums(const T* __restrict__ x, int64_t rows, int c, int64_t rows_per_block, float* __restrict__ part) {
    __shared__ float lds[8][256];
    const int cg = threadIdx.x & 31, sub = threadIdx.x >> 5, n = blockIdx.y * 256 + cg * 8;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per_block, r1 = r0 + rows_per_block < rows ? r0 + rows_per_block : rows;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < c)
        for (int64_t r = r0 + sub; r < r1; r += 8) {
            float v[8];
            load8(x + r * c + n, n, c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
#pragma unroll
    for (int e = 0; e < 8; ++e) lds[sub][cg * 8 + e] = s[e];
    __syncthreads();
    const int j = blockIdx.y * 256 + threadIdx.x;
    if (j < c) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += lds[k][threadIdx.x];
        part[(int64_t)blockIdx.x * c + j] = t;
    }
}

struct ColumnJobs { const float* part[3]; int blocks[3], c[3]; void* out[3]; int jobs; };

template <typename O>
__global__ __launch_bounds__(1024) void column_sums_finish(const ColumnJobs q, int accumulate) {
    __shared__ float lds[64][17];
    const int job = blockIdx.z, c = q.c[job], blocks = q.blocks[job], col = threadIdx.x & 15, slice = threadIdx.x >> 4, j = blockIdx.x * 16 + col;
    if ((int)blockIdx.x * 16 >= c) return;
    float s = 0.f;
    if (j < c)
        for (int b = slice; b < blocks; b += 64) s += q.part[job][(int64_t)b * c + j];
    lds[slice][col] = s;
    __syncthreads();
    if (slice == 0 && j < c) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 64; ++k) t += lds[k][col];
        O* out = static_cast<O*>(q.out[job]);
        out[j] = (O)(accumulate ? (float)out[j] + t : t);
    }
}

// ------------------------------------------------------------------------------------------ workspaces
// Pieces of a call's workspace, laid out in one order by the size query and by the call
struct Space {
    char* base;
    int64_t used = 0;
    void* take(int64_t bytes) {
        void* p = base ? base + used : nullptr;
        used += ceil_div(bytes, 256) * 256;
        return p;
    }
};
struct Dims {
    int64_t m;
    int k, n, o, es;
    int ch() const { return 16 / es; }
    int pad(int c) const { return (int)ceil_div(c, ch()) * ch(); }
    bool odd(int c) const { return c % ch() != 0; }
    bool few() const { return m <= kFewRows && k >= ch() && n >= ch(); }      // (a row holds one chunk at least)
    int64_t two_bytes() const { return es == 2 && m <= kTwoRows ? m * two_chunks(n, ch()) * 32 : 0; }      // h in two parts
    int64_t steps(int64_t c) const { return ceil_div(c, 128 / es); }
    void* copy(Space& s, int64_t rows, int c) const { return odd(c) ? s.take(rows * pad(c) * es) : nullptr; }
};

struct FwdSpace {
    void *xp, *gp, *up, *hp, *dp;
    float* part;
    Plan gate, down;
    FwdSpace(const Dims& d, Space& s) : gate(plan_gemm(d.m, 2 * (int64_t)d.n, d.steps(d.k), d.es, false)), down(plan_gemm(d.m, d.o, d.steps(d.n), d.es, true)) {
        xp = d.copy(s, d.m, d.k); gp = d.copy(s, d.n, d.k); up = d.copy(s, d.n, d.k); hp = d.copy(s, d.m, d.n); dp = d.copy(s, d.o, d.n);
        part = static_cast<float*>(s.take(down.part_bytes()));
    }
};
struct BwdSpace {
    void *dg, *du, *xp, *gp, *up, *hp, *dp, *yp;
    float *part, *cols[3];
    Plan gate, dx, dw;
    int64_t gate_rows(const Dims& d) const { return ceil_div(d.m, gate.big ? 256 : 128); }
    BwdSpace(const Dims& d, Space& s) : gate(plan_gemm(d.m, d.pad(d.n), d.steps(d.o), d.es, false)), dx(plan_gemm(d.m, d.k, 2 * d.steps(d.n), d.es, true)) {
        const int64_t mn[3][2] = {{d.n, d.k}, {d.n, d.k}, {d.o, d.n}};
        dw = plan_gemm(3, mn, d.steps(d.m), d.es, true);
        dg = s.take(d.m * d.pad(d.n) * d.es);
        du = s.take(d.m * d.pad(d.n) * d.es);
        xp = d.copy(s, d.m, d.k); gp = d.copy(s, d.n, d.k); up = d.copy(s, d.n, d.k); hp = d.copy(s, d.m, d.n); dp = d.copy(s, d.o, d.n); yp = d.copy(s, d.m, d.o);
        part = static_cast<float*>(s.take(dx.part_bytes() > dw.part_bytes() ? dx.part_bytes() : dw.part_bytes()));
        for (int i = 0; i < 3; ++i) cols[i] = static_cast<float*>(s.take(i < 2 ? gate_rows(d) * d.n * 4 : (int64_t)kColBlocks * d.o * 4));
    }
};

// the operand itself, or its copy with rows of whole 16-byte chunks
template <typename T> const char* rows_of(const void* p, void* copy, int64_t rows, int c, const Dims& d, hipStream_t st) {
    if (!copy) return static_cast<const char*>(p);
    const int cp = d.pad(c);
    hipLaunchKernelGGL((pad_rows<T>), dim3(grid_for(rows * (cp / d.ch()), 256)), dim3(256), 0, st, static_cast<const T*>(p), rows, c, cp, static_cast<T*>(copy));
    return static_cast<const char*>(copy);
}

template <typename O> __global__ __launch_bounds__(256) void ffn_zero(O* p, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) p[i] = (O)0.f;
}

template <typename T>
int ffn_fwd(int act, const Dims& d, const void* x, const void* wg, const void* wu, const void* wd, const void* bg, const void* bu, const void* bd, void* kept, void* h,
            void* y, void* workspace, hipStream_t st) {
    auto c = [](const void* p) { return static_cast<const T*>(p); };
    auto w = [](void* p) { return static_cast<T*>(p); };
    if (d.few()) {
        T* two = d.two_bytes() ? w(workspace) : nullptr;
        few_rows<T, true>(c(x), (int)d.m, d.k, c(wg), c(wu), d.n, c(bg), c(bu), act, kept, w(h), two, st);
        few_rows<T, false>(c(h), (int)d.m, d.n, c(wd), nullptr, d.o, c(bd), nullptr, 0, nullptr, w(y), two, st);
        return check_launch("suhpe_gated_ffn_fwd");
    }
    Space space{static_cast<char*>(workspace)};
    const FwdSpace s(d, space);
    const int64_t kp = (int64_t)d.pad(d.k) * d.es, np = (int64_t)d.pad(d.n) * d.es;
    GemmArgs a{};
    a.pr[0] = {{rows_of<T>(x, s.xp, d.m, d.k, d, st), nullptr}, {rows_of<T>(wg, s.gp, d.n, d.k, d, st), rows_of<T>(wu, s.up, d.n, d.k, d, st)}, kp, kp, d.m, d.n, d.n, h, 0, 0};
    a.K = d.pad(d.k); a.nseg = 1;
    a.bias = bg; a.bias2 = bu; a.kept = kept; a.act = act;
    if (int rc = gemm_launch<T, T, false, false, EPI_GATE>(a, 1, s.gate, st)) return rc;
    a = GemmArgs{};
    a.pr[0] = {{rows_of<T>(h, s.hp, d.m, d.n, d, st), nullptr}, {rows_of<T>(wd, s.dp, d.o, d.n, d, st), nullptr}, np, np, d.m, d.o, d.o, y, 0, 0};
    a.K = d.pad(d.n); a.nseg = 1;
    a.bias = bd; a.part = s.part;
    return gemm_launch<T, T, false, false, EPI_STORE>(a, 1, s.down, st);
}

template <typename T, typename O>
int ffn_bwd(int act, const Dims& d, const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* kept, const void* h, void* dx, void* dwg,
            void* dwu, void* dwd, void* dbg, void* dbu, void* dbd, int accumulate, void* workspace, hipStream_t st) {
    Space space{static_cast<char*>(workspace)};
    const BwdSpace s(d, space);
    const int64_t np = (int64_t)d.pad(d.n) * d.es, kp = (int64_t)d.pad(d.k) * d.es, op = (int64_t)d.pad(d.o) * d.es;
    if (d.m > 0) {
        const char *dyr = rows_of<T>(dy, s.yp, d.m, d.o, d, st), *dg = static_cast<const char*>(s.dg), *du = static_cast<const char*>(s.du);
        GemmArgs a{};
        a.pr[0] = {{dyr, nullptr}, {rows_of<T>(wd, s.dp, d.o, d.n, d, st), nullptr}, op, np, d.m, d.n, d.pad(d.n), s.dg, 0, 0};
        a.K = d.o; a.nseg = 1;
        a.kept = const_cast<void*>(kept); a.uout = s.du; a.act = act;
        if (dbg || dbu) { a.cols = s.cols[0]; a.cols2 = s.cols[1]; }
        if (int rc = gemm_launch<T, T, false, true, EPI_GATE_BWD>(a, 1, s.gate, st)) return rc;
        if (dx) {
            a = GemmArgs{};
            a.pr[0] = {{dg, du}, {rows_of<T>(wg, s.gp, d.n, d.k, d, st), rows_of<T>(wu, s.up, d.n, d.k, d, st)}, np, kp, d.m, d.k, d.k, dx, 0, 0};
            a.K = d.n; a.nseg = 2; a.part = s.part;
            if (int rc = gemm_launch<T, T, false, true, EPI_STORE>(a, 1, s.dx, st)) return rc;
        }
        if (dwg) {
            a = GemmArgs{};
            const char* xr = rows_of<T>(x, s.xp, d.m, d.k, d, st);
            a.pr[0] = {{dg, nullptr}, {xr, nullptr}, np, kp, d.n, d.k, d.k, dwg, 0, 0};
            a.pr[1] = {{du, nullptr}, {xr, nullptr}, np, kp, d.n, d.k, d.k, dwu, 0, 0};
            a.pr[2] = {{dyr, nullptr}, {rows_of<T>(h, s.hp, d.m, d.n, d, st), nullptr}, op, np, d.o, d.n, d.n, dwd, 0, 0};
            a.K = d.m; a.nseg = 1; a.part = s.part; a.accumulate = accumulate;
            if (int rc = gemm_launch<T, O, true, true, EPI_STORE>(a, 3, s.dw, st)) return rc;
        }
    } else if (!accumulate) {                                          // no rows: the gradients are zero
        auto zero = [&](void* p, int64_t count) {
            if (p) hipLaunchKernelGGL((ffn_zero<O>), dim3(grid_for(count, 256)), dim3(256), 0, st, static_cast<O*>(p), count);
        };
        zero(dwg, (int64_t)d.n * d.k); zero(dwu, (int64_t)d.n * d.k); zero(dwd, (int64_t)d.o * d.n);
        zero(dbg, d.n); zero(dbu, d.n); zero(dbd, d.o);
    }
    if (d.m > 0 && (dbg || dbu || dbd)) {
        ColumnJobs q{};
        int widest = 0;
        auto add = [&](int c, void* out, const float* part, int blocks) {
            if (!out) return;
            q.c[q.jobs] = c; q.out[q.jobs] = out; q.part[q.jobs] = part; q.blocks[q.jobs++] = blocks;
            widest = c > widest ? c : widest;
        };
        add(d.n, dbg, s.cols[0], (int)s.gate_rows(d));
        add(d.n, dbu, s.cols[1], (int)s.gate_rows(d));
        if (dbd) {
            const int64_t per = ceil_div(d.m, ceil_div(d.m, 32) < kColBlocks ? ceil_div(d.m, 32) : kColBlocks);
            const int blocks = (int)ceil_div(d.m, per);
            hipLaunchKernelGGL((column_sums<T>), dim3(blocks, (unsigned)ceil_div(d.o, 256)), dim3(256), 0, st, static_cast<const T*>(dy), d.m, d.o, per, s.cols[2]);
            add(d.o, dbd, s.cols[2], blocks);
        }
        hipLaunchKernelGGL((column_sums_finish<O>), dim3((unsigned)ceil_div(widest, 16), 1, q.jobs), dim3(1024), 0, st, q, accumulate);
    }
    return check_launch("suhpe_gated_ffn_bwd");
}

int ffn_sizes(const char* who, int dtype, int act, int64_t m, int k, int n, int o) {
    SUHPE_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", who, dtype);
    SUHPE_REQUIRE(act >= SUHPE_ACT_NONE && act <= SUHPE_ACT_SIGMOID, "%s: unknown activation %d", who, act);
    SUHPE_REQUIRE(m >= 0 && m <= 0x7fffff00ll && k > 0 && n > 0 && o > 0, "%s: bad sizes m %lld k %d n %d o %d", who, (long long)m, k, n, o);
    SUHPE_REQUIRE(k <= (1 << 20) && n <= (1 << 20) && o <= (1 << 20), "%s: widths up to 2^20", who);
    return SUHPE_OK;
}
int space_short(const char* who, const void* workspace, int64_t have, int64_t need) {
    if (need == 0 || (workspace && have >= need && aligned(workspace, 256))) return SUHPE_OK;
    set_error("%s: workspace of %lld bytes at %p, needs %lld on a 256-byte boundary", who, (long long)have, workspace, (long long)need);
    return SUHPE_EWORKSPACE;
}

}  // namespace
}  // namespace suhpe

using namespace suhpe;

extern "C" {

int64_t suhpe_gated_ffn_kept_bytes(int dtype, int64_t m, int n) {
    SUHPE_REQUIRE(dtype_ok(dtype) && m >= 0 && n > 0, "suhpe_gated_ffn_kept_bytes: bad dtype or sizes");
    return kept_bytes(dtype_size(dtype), m, n);
}

int64_t suhpe_gated_ffn_fwd_workspace_bytes(int dtype, int64_t m, int k, int n, int o) {
    if (ffn_sizes("suhpe_gated_ffn_fwd_workspace_bytes", dtype, 0, m, k, n, o) || m == 0) return 0;
    const Dims d{m, k, n, o, dtype_size(dtype)};
    if (d.few()) return d.two_bytes();
    Space space{nullptr};
    const FwdSpace s(d, space);
    return space.used;
}

int suhpe_gated_ffn_fwd(int dtype, int act, int64_t m, int k, int n, int o, const void* x, const void* wg, const void* wu, const void* wd, const void* bg, const void* bu,
                        const void* bd, void* kept, void* h, void* y, void* workspace, int64_t workspace_bytes, suhpe_stream_t stream) {
    if (int rc = ffn_sizes("suhpe_gated_ffn_fwd", dtype, act, m, k, n, o)) return rc;
    if (m == 0) return SUHPE_OK;
    SUHPE_REQUIRE(x && wg && wu && wd && h && y, "suhpe_gated_ffn_fwd: null pointer");
    const Dims d{m, k, n, o, dtype_size(dtype)};
    if (!d.few())
        SUHPE_REQUIRE((d.odd(k) || (aligned(x, 16) && aligned(wg, 16) && aligned(wu, 16))) && (d.odd(n) || (aligned(h, 16) && aligned(wd, 16))),
                      "suhpe_gated_ffn_fwd: x, wg, wu, wd and h start on 16-byte boundaries");
    if (int rc = space_short("suhpe_gated_ffn_fwd", workspace, workspace_bytes, suhpe_gated_ffn_fwd_workspace_bytes(dtype, m, k, n, o))) return rc;
    // (y is written by the second product, which reads h, wd, bd and the workspace)
    const int64_t es = d.es, nk = (int64_t)n * k, on = (int64_t)o * n;
    const Range r[] = {{h, m * n * es}, {kept, kept_bytes(d.es, m, n)}, {workspace, suhpe_gated_ffn_fwd_workspace_bytes(dtype, m, k, n, o)}, {y, m * o * es},
                       {wd, on * es}, {bd, o * es}, {x, m * k * es}, {wg, nk * es}, {wu, nk * es}, {bg, n * es}, {bu, n * es}};
    SUHPE_REQUIRE(apart(r, 3, 11) && apart(r + 3, 1, 3), "suhpe_gated_ffn_fwd: h, kept and the workspace share no memory with each other, with y or with the inputs, nor y with wd or bd");
    hipStream_t st = as_stream(stream);
    if (dtype == SUHPE_F32) return ffn_fwd<float>(act, d, x, wg, wu, wd, bg, bu, bd, kept, h, y, workspace, st);
    if (dtype == SUHPE_BF16) return ffn_fwd<bf16>(act, d, x, wg, wu, wd, bg, bu, bd, kept, h, y, workspace, st);
    return ffn_fwd<f16>(act, d, x, wg, wu, wd, bg, bu, bd, kept, h, y, workspace, st);
}

int64_t suhpe_gated_ffn_bwd_workspace_bytes(int dtype, int64_t m, int k, int n, int o) {
    if (m == 0 || ffn_sizes("suhpe_gated_ffn_bwd_workspace_bytes", dtype, 0, m, k, n, o)) return 0;
    Space space{nullptr};
    const BwdSpace s(Dims{m, k, n, o, dtype_size(dtype)}, space);
    return space.used;
}

int suhpe_gated_ffn_bwd(int dtype, int act, int64_t m, int k, int n, int o, const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* kept,
                        const void* h, void* dx, void* dwg, void* dwu, void* dwd, void* dbg, void* dbu, void* dbd, int grad_dtype, int accumulate,
                        void* workspace, int64_t workspace_bytes, suhpe_stream_t stream) {
    if (int rc = ffn_sizes("suhpe_gated_ffn_bwd", dtype, act, m, k, n, o)) return rc;
    SUHPE_REQUIRE(grad_dtype == dtype || grad_dtype == SUHPE_F32, "suhpe_gated_ffn_bwd: gradients have the weights' type or fp32");
    SUHPE_REQUIRE((dwg != nullptr) == (dwu != nullptr) && (dwg != nullptr) == (dwd != nullptr), "suhpe_gated_ffn_bwd: the three weights' gradients are wanted together or not at all");
    SUHPE_REQUIRE(m == 0 || (dy && x && wg && wu && wd && kept && h), "suhpe_gated_ffn_bwd: null pointer");
    if (m == 0 && (accumulate || !(dwg || dbg || dbu || dbd))) return SUHPE_OK;      // nothing to write
    const Dims d{m, k, n, o, dtype_size(dtype)};
    if (m > 0)
        SUHPE_REQUIRE((d.odd(k) || (aligned(x, 16) && aligned(wg, 16) && aligned(wu, 16))) && (d.odd(n) || (aligned(h, 16) && aligned(wd, 16))) && (d.odd(o) || aligned(dy, 16)),
                      "suhpe_gated_ffn_bwd: dy, x, wg, wu, wd and h start on 16-byte boundaries");
    if (int rc = space_short("suhpe_gated_ffn_bwd", workspace, workspace_bytes, suhpe_gated_ffn_bwd_workspace_bytes(dtype, m, k, n, o))) return rc;
    const int64_t es = d.es, gs = dtype_size(grad_dtype), nk = (int64_t)n * k, on = (int64_t)o * n;
    const Range r[] = {{dx, m * k * es}, {dwg, nk * gs}, {dwu, nk * gs}, {dwd, on * gs}, {dbg, n * gs}, {dbu, n * gs}, {dbd, o * gs},
                       {dy, m * o * es}, {x, m * k * es}, {wg, nk * es}, {wu, nk * es}, {wd, on * es}, {kept, kept_bytes(d.es, m, n)}, {h, m * n * es}};
    SUHPE_REQUIRE(apart(r, 7, 14), "suhpe_gated_ffn_bwd: the gradients share no memory with each other or with the inputs");
    hipStream_t st = as_stream(stream);
#define FFN_BWD(T, O) ffn_bwd<T, O>(act, d, dy, x, wg, wu, wd, kept, h, dx, dwg, dwu, dwd, dbg, dbu, dbd, accumulate, workspace, st)
    if (dtype == SUHPE_F32) return FFN_BWD(float, float);
    if (dtype == SUHPE_BF16) return grad_dtype == SUHPE_F32 ? FFN_BWD(bf16, float) : FFN_BWD(bf16, bf16);
    return grad_dtype == SUHPE_F32 ? FFN_BWD(f16, float) : FFN_BWD(f16, f16);
#undef FFN_BWD
}

}  // extern "C"

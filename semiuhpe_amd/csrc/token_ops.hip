// Operators on token rows in fp32 / bf16 / fp16: rotary positions with several axes, dropout whose mask is never stored, 16-bit LayerNorm.
// All three are bound by memory: each element is read once and written once, in 16-byte vectors where sizes and addresses allow.
#include "lowp.h"

namespace suhpe {
namespace {

// ------------------------------------------------------------------------------------------ rotary positions
// Pair p of a head belongs to axis[p] and turns by pos[row][axis[p]] * freq[p] radians.  The angle is formed in 64 bits as REVOLUTIONS (freq holds
// radians / 2 pi): the whole turns are dropped exactly before the 32-bit sine and cosine, so a position of 10^6 is as exact as one of 10.
// A block takes R rows: it evaluates sine and cosine of each (row, pair) ONCE into LDS and then streams all heads of those rows past the table
// (q and k, every head: the evaluation is amortised over heads * rotated vectors).  Bound by memory: 31 360 rows of 12 heads x (q k v) x 32 fp32 out of place
// (289 MB) 55 us, 57 600 rows of 16 x 128 bf16 (473 MB) 92 us = 5.2 TB/s, what a large copy reaches.
template <typename P> __device__ __forceinline__ double pos_of(const P* pos, int64_t i) { return (double)pos[i]; }

struct RopeArgs {
    int64_t rows;
    int heads, parts, rotated, dh, naxes, pairs, halves, inverse, copy, rows_per_block;
    const double* freq;
    const int32_t* axis;
};

template <typename T, typename P, int V>
__global__ __launch_bounds__(256) void rope_axes_kernel(const T* x, T* y, const P* __restrict__ pos, const RopeArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 turn[];      // [row][pair] cos, sin
    const int64_t row0 = (int64_t)blockIdx.x * a.rows_per_block;
    const int nrows = (int)(a.rows - row0 < a.rows_per_block ? a.rows - row0 : a.rows_per_block);
    for (int i = threadIdx.x; i < nrows * a.pairs; i += 256) {
        const int r = i / a.pairs, p = i - r * a.pairs;
        const double rev = pos_of(pos, (row0 + r) * a.naxes + a.axis[p]) * a.freq[p];
        float s, c;
        sincospif(2.f * (float)(rev - rint(rev)), &s, &c);
        turn[i] = make_float2(c, a.inverse ? -s : s);
    }
    __syncthreads();
    // items of a head: rotated parts first -- `ir` vectors of pairs (halves: the first members, whose partners lie `pairs` further; adjacent: V / 2
    // pairs a vector; V == 1: one pair an item in both layouts) and `ip` vectors behind the rotated width -- then the parts that stay as they are
    const bool wide = V > 1 && !a.halves;
    const int ir = wide ? 2 * a.pairs / V : a.pairs / V, ip = a.copy ? (a.dh - 2 * a.pairs) / V : 0;
    const int irp = ir + ip, nrot = a.rotated * irp, nh = nrot + (a.copy ? (a.parts - a.rotated) * (a.dh / V) : 0);
    const int per_row = a.heads * nh, total = nrows * per_row;
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < total; i0 += 256 * U) {
        float v1[U][V], v2[U][V];
        int64_t at1[U];
        int at2[U], tab[U];                                            // tab: first pair's place in the table, -1: a plain copy
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u;
            at1[u] = -1;
            if (i >= total) continue;
            const int r = i / per_row, rem = i - r * per_row, h = rem / nh, j = rem - h * nh;
            const int64_t head = ((row0 + r) * a.heads + h) * a.parts * (int64_t)a.dh;
            at2[u] = -1;
            if (j < nrot) {
                const int part = j / irp, q = j - part * irp;
                if (q < ir) {
                    const int p = wide ? q * V / 2 : q * V;
                    tab[u] = r * a.pairs + p;
                    at1[u] = head + part * a.dh + (a.halves ? p : 2 * p);
                    if (!wide) at2[u] = a.halves ? a.pairs : 1;
                } else {
                    tab[u] = -1;
                    at1[u] = head + part * a.dh + 2 * a.pairs + (q - ir) * V;
                }
            } else {
                tab[u] = -1;
                at1[u] = head + a.rotated * a.dh + (int64_t)(j - nrot) * V;
            }
            load_n<T, V>(x + at1[u], v1[u]);
            if (at2[u] >= 0) load_n<T, V>(x + at1[u] + at2[u], v2[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at1[u] < 0) continue;
            if (tab[u] >= 0) {
                if (at2[u] >= 0) {
                    float o1[V], o2[V];
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float2 t = turn[tab[u] + k];
                        o1[k] = v1[u][k] * t.x - v2[u][k] * t.y;
                        o2[k] = v1[u][k] * t.y + v2[u][k] * t.x;
                    }
                    store_n<T, V>(y + at1[u], o1);
                    store_n<T, V>(y + at1[u] + at2[u], o2);
                } else if constexpr (V > 1) {
                    float o[V];
#pragma unroll
                    for (int k = 0; k < V; k += 2) {
                        const float2 t = turn[tab[u] + k / 2];
                        o[k] = v1[u][k] * t.x - v1[u][k + 1] * t.y;
                        o[k + 1] = v1[u][k] * t.y + v1[u][k + 1] * t.x;
                    }
                    store_n<T, V>(y + at1[u], o);
                }
            } else {
                store_n<T, V>(y + at1[u], v1[u]);
            }
        }
    }
}

template <typename T, typename P>
int rope_launch(const T* x, T* y, const P* pos, RopeArgs a, hipStream_t st) {
    constexpr int FULL = 16 / sizeof(T);
    const int step = a.halves ? a.pairs : 2 * a.pairs;                 // the widths that a vector must divide
    const auto fits = [&](int v) { return a.dh % v == 0 && step % v == 0 && aligned(x, v * sizeof(T)) && aligned(y, v * sizeof(T)); };
    // 4096 (fp32) or 8192 (16 bits) elements a workgroup: four 16-byte vectors a thread keep a few loads of each in flight; the table stays under 32 KB
    const int64_t width = (int64_t)a.heads * a.parts * a.dh;
    int64_t r = ceil_div(256 * 4 * FULL, width);
    if (r * a.pairs > 4096) r = 4096 / a.pairs;
    if (r < 1) r = 1;
    if (r > a.rows) r = a.rows;
    a.rows_per_block = (int)r;
    SUHPE_REQUIRE(ceil_div(a.rows, r) < (1 << 24), "suhpe_rope_axes: %lld rows of %lld elements are more than one launch holds", (long long)a.rows, (long long)width);
    const int64_t bytes = a.rows * width * (int64_t)sizeof(T);
    const Range ranges[] = {{y, bytes}, {a.copy ? x : nullptr, bytes}, {pos, a.rows * a.naxes * (int64_t)sizeof(P)}, {a.freq, a.pairs * 8}, {a.axis, a.pairs * 4}};
    SUHPE_REQUIRE(apart(ranges, 1, 5), "suhpe_rope_axes: y (unless it is x) shares no memory with the inputs");
    const dim3 grid((unsigned)ceil_div(a.rows, r));                    // (2^24 workgroups of 256: some 2^36 elements)
    const size_t lds = (size_t)r * a.pairs * sizeof(float2);
    if (fits(FULL)) hipLaunchKernelGGL((rope_axes_kernel<T, P, FULL>), grid, dim3(256), lds, st, x, y, pos, a);
    else if (fits(FULL / 2)) hipLaunchKernelGGL((rope_axes_kernel<T, P, FULL / 2>), grid, dim3(256), lds, st, x, y, pos, a);
    else hipLaunchKernelGGL((rope_axes_kernel<T, P, 1>), grid, dim3(256), lds, st, x, y, pos, a);
    return check_launch("suhpe_rope_axes");
}

template <typename T>
int rope_types(const void* x, void* y, const void* pos, int pos_type, const RopeArgs& a, hipStream_t st) {
    const T* xt = static_cast<const T*>(x);
    T* yt = static_cast<T*>(y);
    if (pos_type == SUHPE_POS_I32) return rope_launch<T, int32_t>(xt, yt, static_cast<const int32_t*>(pos), a, st);
    if (pos_type == SUHPE_POS_I64) return rope_launch<T, int64_t>(xt, yt, static_cast<const int64_t*>(pos), a, st);
    return rope_launch<T, float>(xt, yt, static_cast<const float*>(pos), a, st);
}

// ------------------------------------------------------------------------------------------ dropout without a stored mask
// y_i = [skip_i +] (r_i < keep ? x_i / keep : 0) with r_i the 24-bit number that suhpe_dropout_mask draws for element i at the same stream position:
// word i % 4 of Philox call counter[1] + position + i / 4.  The gradient is the same call on dy: nothing is kept between the two.
// A dropped element is 0 whatever x holds there (also infinities and NaN).  20 wide multiplies per 4 elements (one 32 x 32 -> 64 bit product gives both halves) hide
// behind the memory: 24 M bf16 elements, skip + dropout (145 MB) and the gradient (96 MB) 50 us = 4.8 TB/s.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void dropout_apply_kernel(const T* x, const T* skip, T* y, int64_t count, uint32_t bound, float scale,
                                                            const uint64_t* __restrict__ counter, uint64_t position) {
    constexpr int N = VECTOR ? 16 / sizeof(T) : 4;                      // elements of a thread's turn: one or two calls of the generator
    const uint64_t seed = counter[0], base = counter[1] + position;
    const int64_t turns = (count + N - 1) / N, stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < turns; i += stride) {
        const int64_t e0 = i * N;
        const int n = count - e0 < N ? (int)(count - e0) : N;
        float v[N], s[N];
        if (VECTOR && n == N) {
            load_n<T, N>(x + e0, v);
            if (skip) load_n<T, N>(skip + e0, s);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                v[k] = k < n ? (float)x[e0 + k] : 0.f;
                s[k] = k < n && skip ? (float)skip[e0 + k] : 0.f;
            }
        }
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            uint32_t w[4];
            philox_words(seed, base + (uint64_t)((e0 + q) >> 2), w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float d = (w[k] >> 8) < bound ? v[q + k] * scale : 0.f;
                v[q + k] = skip ? s[q + k] + d : d;
            }
        }
        if (VECTOR && n == N) {
            store_n<T, N>(y + e0, v);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k < n) y[e0 + k] = (T)v[k];
        }
    }
}

__global__ void dropout_advance_kernel(uint64_t* counter, uint64_t by) { counter[1] += by; }

template <typename T>
int dropout_launch(const void* x, const void* skip, void* y, int64_t count, uint32_t bound, float scale, const uint64_t* counter, uint64_t position, hipStream_t st) {
    const T *xt = static_cast<const T*>(x), *kt = static_cast<const T*>(skip);
    T* yt = static_cast<T*>(y);
    if (aligned(x, 16) && aligned(y, 16) && aligned(skip, 16))
        hipLaunchKernelGGL((dropout_apply_kernel<T, true>), dim3(grid_for(ceil_div(count, 16 / sizeof(T)), 256)), dim3(256), 0, st, xt, kt, yt, count, bound, scale, counter, position);
    else
        hipLaunchKernelGGL((dropout_apply_kernel<T, false>), dim3(grid_for(ceil_div(count, 4), 256)), dim3(256), 0, st, xt, kt, yt, count, bound, scale, counter, position);
    return check_launch("suhpe_dropout_apply");
}

// ------------------------------------------------------------------------------------------ LayerNorm of 16-bit rows
// y = (x - mean) rstd gamma + beta with the statistics, gamma, beta and the parameters' gradients in fp32: only x, y, dy, dx have 16 bits.
// LPR lanes share a row (8 .. 64, or the 256 of a block), each holding NV vectors of 8 elements in registers between the statistics and the result: one pass
// over memory.  Blocks are persistent: gamma and beta (8 bytes an element, twice what x and y take together) are loaded once per lane, not once per row, and
// the next row's loads are issued before this row's sums.  125 440 x 192 bf16: forward 17.5 us (5.5 TB/s), backward with the parameters' gradients 35 us
// (4.1 TB/s; 26 us without them: 48 more accumulators a lane leave two wavefronts per SIMD instead of three, and 512 partial rows are summed by a second launch).
//  Any width >= 8 runs on full vectors: a row's last vector starts at c - 8 and leaves out of the sums
// what the vector before it holds (both write the same bits there), and 16-byte accesses may start at any element.
template <typename T, int LPR, int NV> struct LnRow {
    typename Vec<T, 8>::type v[NV];
    __device__ __forceinline__ void load(const T* row, const int (&at)[NV]) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (at[k] >= 0) __builtin_memcpy(&v[k], row + at[k], 16);
    }
};

// sum over the LPR lanes of a row (lds: 2 x 4 floats, two places used in turn)
template <int LPR> __device__ __forceinline__ float row_sum(float v, float* lds, int& turn) {
    constexpr int S = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int o = S / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (LPR == 256) {
        float* at = lds + turn * 4;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (at[0] + at[1]) + (at[2] + at[3]);
        turn ^= 1;
    }
    return v;
}

// element offset of this lane's vectors in a row (-1: none), and how many leading elements of the last one the vector before it owns
template <int LPR, int NV> __device__ __forceinline__ void ln_places(int c, int (&at)[NV], int (&skip)[NV]) {
    const int sub = threadIdx.x % LPR;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int e = (sub + LPR * k) * 8;
        at[k] = e >= c ? -1 : e + 8 <= c ? e : c - 8;
        skip[k] = e >= c ? 8 : e - at[k];
    }
}

// this lane's columns of gamma or beta, in 16-byte loads (32 four-byte ones per lane took 20 us of a 27 us launch over 4 099 rows of 1 357)
template <int NV> __device__ __forceinline__ void ln_param(const float* p, const int (&at)[NV], float without, float (&v)[NV][8]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = without;
        if (p && at[k] >= 0) {
            float4 lo, hi;
            __builtin_memcpy(&lo, p + at[k], 16);
            __builtin_memcpy(&hi, p + at[k] + 4, 16);
            v[k][0] = lo.x; v[k][1] = lo.y; v[k][2] = lo.z; v[k][3] = lo.w;
            v[k][4] = hi.x; v[k][5] = hi.y; v[k][6] = hi.z; v[k][7] = hi.w;
        }
    }
}

template <typename T, int LPR, int NV>
__global__ __launch_bounds__(256) void layernorm16_fwd_kernel(const T* __restrict__ x, int64_t rows, int c, float eps, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float lds[8];
    int turn = 0;
    constexpr int RPB = 256 / LPR;
    int at[NV], skip[NV];
    ln_places<LPR, NV>(c, at, skip);
    float ga[NV][8], be[NV][8];
    ln_param<NV>(gamma, at, 1.f, ga);
    ln_param<NV>(beta, at, 0.f, be);
    const float inv = 1.f / c;
    const int64_t first = (int64_t)blockIdx.x * RPB, stride = (int64_t)gridDim.x * RPB;
    const int mine = threadIdx.x / LPR;
    LnRow<T, LPR, NV> cur, next;
    if (first + mine < rows) cur.load(x + (first + mine) * c, at);
    for (int64_t r0 = first; r0 < rows; r0 += stride) {
        const int64_t row = r0 + mine;
        if (row + stride < rows) next.load(x + (row + stride) * c, at);
        float v[NV][8], s = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[k][e] = (float)cur.v[k][e];
                s += e >= skip[k] ? v[k][e] : 0.f;
            }
        const float m = row_sum<LPR>(s, lds, turn) * inv;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[k][e] -= m;
                q += e >= skip[k] ? v[k][e] * v[k][e] : 0.f;
            }
        const float rs = 1.f / sqrtf(row_sum<LPR>(q, lds, turn) * inv + eps);
        if (row < rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (at[k] >= 0) {
                    typename Vec<T, 8>::type o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = (T)(v[k][e] * rs * ga[k][e] + be[k][e]);
                    __builtin_memcpy(y + row * c + at[k], &o, 16);
                }
            if (threadIdx.x % LPR == 0) { mean[row] = m; rstd[row] = rs; }
        }
        cur = next;
    }
}

// dx = rstd (g - mean(g) - xhat mean(g xhat)) [+ skip], g = dy gamma, and the block's column sums of dy xhat and dy: part[block][2][c].  x and dy are read once.
template <typename T, int LPR, int NV, bool COLS>
__global__ __launch_bounds__(256) void layernorm16_bwd_kernel(const T* __restrict__ x, const T* __restrict__ dy, int64_t rows, int c, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, const float* __restrict__ gamma, const T* __restrict__ bypass,
                                                              T* __restrict__ dx, float* __restrict__ part) {
    __shared__ float lds[8];
    extern __shared__ float cols[];                                    // [wavefront][2][c]
    int turn = 0;
    constexpr int RPB = 256 / LPR;
    int at[NV], skip[NV];
    ln_places<LPR, NV>(c, at, skip);
    float ga[NV][8], sg[NV][8], sb[NV][8];
    ln_param<NV>(gamma, at, 1.f, ga);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) sg[k][e] = sb[k][e] = 0.f;
    const float inv = 1.f / c;
    const int64_t first = (int64_t)blockIdx.x * RPB, stride = (int64_t)gridDim.x * RPB;
    const int mine = threadIdx.x / LPR;
    LnRow<T, LPR, NV> cx, cd, nx, nd;
    float m = 0.f, rs = 0.f, nm = 0.f, nrs = 0.f;
    if (first + mine < rows) {
        cx.load(x + (first + mine) * c, at);
        cd.load(dy + (first + mine) * c, at);
        m = mean[first + mine];
        rs = rstd[first + mine];
    }
    for (int64_t r0 = first; r0 < rows; r0 += stride) {
        const int64_t row = r0 + mine;
        if (row + stride < rows) {
            nx.load(x + (row + stride) * c, at);
            nd.load(dy + (row + stride) * c, at);
            nm = mean[row + stride];
            nrs = rstd[row + stride];
        }
        const bool live = row < rows;
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool own = live && e >= skip[k];
                const float d = (float)cd.v[k][e], xh = ((float)cx.v[k][e] - m) * rs, g = d * ga[k][e];
                s0 += own ? g : 0.f;
                s1 += own ? g * xh : 0.f;
                if constexpr (COLS) {
                    sg[k][e] += own ? d * xh : 0.f;
                    sb[k][e] += own ? d : 0.f;
                }
            }
        s0 = row_sum<LPR>(s0, lds, turn) * inv;
        s1 = row_sum<LPR>(s1, lds, turn) * inv;
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (at[k] >= 0) {
                    typename Vec<T, 8>::type o, b;
                    if (bypass) __builtin_memcpy(&b, bypass + row * c + at[k], 16);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {                      // (xhat and g again from the 16-bit rows: cheaper than the registers that would hold them)
                        const float xh = ((float)cx.v[k][e] - m) * rs, g = (float)cd.v[k][e] * ga[k][e];
                        const float d = rs * (g - s0 - xh * s1);
                        o[e] = (T)(bypass ? d + (float)b[e] : d);
                    }
                    __builtin_memcpy(dx + row * c + at[k], &o, 16);
                }
        }
        cx = nx; cd = nd; m = nm; rs = nrs;
    }
    if constexpr (COLS) {
        // rows of one wavefront first (lanes LPR, 2 LPR, ... apart), then the four wavefronts
        if constexpr (LPR < 64)
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int o = LPR; o < 64; o <<= 1) {
                        sg[k][e] += __shfl_xor(sg[k][e], o, 64);
                        sb[k][e] += __shfl_xor(sb[k][e], o, 64);
                    }
        float* const mine_part = part + (int64_t)blockIdx.x * 2 * c;
        if constexpr (LPR == 256) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e >= skip[k]) {                                // (one lane owns a column)
                        mine_part[at[k] + e] = sg[k][e];
                        mine_part[c + at[k] + e] = sb[k][e];
                    }
            return;
        }
        if ((int)(threadIdx.x & 63) < LPR) {
            float* at_wave = cols + (threadIdx.x >> 6) * 2 * c;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e >= skip[k]) {
                        at_wave[at[k] + e] = sg[k][e];
                        at_wave[c + at[k] + e] = sb[k][e];
                    }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * c; i += 256) mine_part[i] = (cols[i] + cols[2 * c + i]) + (cols[4 * c + i] + cols[6 * c + i]);
    }
}

// Widths under 8 and over 8192: one wavefront per row at a time, element by element (at most kAnyBlocks workgroups: a launch holds less than 2^32 threads)
constexpr int64_t kAnyBlocks = 1 << 20;
template <typename T>
__global__ __launch_bounds__(256) void layernorm16_fwd_any(const T* __restrict__ x, int64_t rows, int c, float eps, const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
        const T* xr = x + row * c;
        float s = 0.f;
        for (int j = lane; j < c; j += 64) s += (float)xr[j];
        const float m = wave_sum(s) / c;
        float q = 0.f;
        for (int j = lane; j < c; j += 64) { const float d = (float)xr[j] - m; q += d * d; }
        const float rs = 1.f / sqrtf(wave_sum(q) / c + eps);
        for (int j = lane; j < c; j += 64) y[row * c + j] = (T)(((float)xr[j] - m) * rs * (gamma ? gamma[j] : 1.f) + (beta ? beta[j] : 0.f));
        if (lane == 0) { mean[row] = m; rstd[row] = rs; }
    }
}

// dx = rstd (g - mean(g) - xhat mean(g xhat)) [+ skip], g = dy gamma
template <typename T>
__global__ __launch_bounds__(256) void layernorm16_bwd_dx_any(const T* __restrict__ x, const T* __restrict__ dy, int64_t rows, int c,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd, const float* __restrict__ gamma,
                                                              const T* __restrict__ skip, T* __restrict__ dx) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
        const float m = mean[row], rs = rstd[row];
        const int64_t at = row * c;
        float s0 = 0.f, s1 = 0.f;
        for (int j = lane; j < c; j += 64) {
            const float g = (float)dy[at + j] * (gamma ? gamma[j] : 1.f);
            s0 += g;
            s1 += g * (((float)x[at + j] - m) * rs);
        }
        s0 = wave_sum(s0) / c;
        s1 = wave_sum(s1) / c;
        for (int j = lane; j < c; j += 64) {
            const float g = (float)dy[at + j] * (gamma ? gamma[j] : 1.f), xh = ((float)x[at + j] - m) * rs;
            dx[at + j] = (T)(rs * (g - s0 - xh * s1) + (skip ? (float)skip[at + j] : 0.f));
        }
    }
}

// column sums of dy and dy * xhat over a block's rows: part[block][2][c]
template <typename T>
__global__ __launch_bounds__(256) void layernorm16_bwd_cols_any(const T* __restrict__ x, const T* __restrict__ dy, int64_t rows, int c, int64_t rows_per_block,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part) {
    __shared__ float lds[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.y * 64 + lane;
    const int64_t r0 = (int64_t)blockIdx.x * rows_per_block, r1 = r0 + rows_per_block < rows ? r0 + rows_per_block : rows;
    float sg = 0.f, sb = 0.f;
    if (j < c)
        for (int64_t r = r0 + wave; r < r1; r += 4) {
            const float d = (float)dy[r * c + j];
            sb += d;
            sg += d * (((float)x[r * c + j] - mean[r]) * rstd[r]);
        }
    lds[0][wave][lane] = sg;
    lds[1][wave][lane] = sb;
    __syncthreads();
    if (wave == 0 && j < c) {
        part[((int64_t)blockIdx.x * 2 + 0) * c + j] = (lds[0][0][lane] + lds[0][1][lane]) + (lds[0][2][lane] + lds[0][3][lane]);
        part[((int64_t)blockIdx.x * 2 + 1) * c + j] = (lds[1][0][lane] + lds[1][1][lane]) + (lds[1][2][lane] + lds[1][3][lane]);
    }
}

// the partial sums of `blocks` blocks in a fixed order: 16 columns x 64 slices per block, 8 loads of a thread in flight together
__global__ __launch_bounds__(1024) void layernorm16_bwd_finish(const float* __restrict__ part, int blocks, int c, float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                               int accumulate) {
    __shared__ float lds[64][17];
    const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, j = blockIdx.x * 16 + col, which = blockIdx.y;
    float s = 0.f;
    if (j < c)
        for (int b0 = slice; b0 < blocks; b0 += 512) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = b0 + 64 * u < blocks ? part[((int64_t)(b0 + 64 * u) * 2 + which) * c + j] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    lds[slice][col] = s;
    __syncthreads();
    float* out = which ? dbeta : dgamma;
    if (slice == 0 && j < c && out) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 64; ++k) t += lds[k][col];
        out[j] = accumulate ? out[j] + t : t;
    }
}

constexpr int kLnBlocks = 512;
inline unsigned any_blocks(int64_t rows) { return (unsigned)(ceil_div(rows, 4) < kAnyBlocks ? ceil_div(rows, 4) : kAnyBlocks); }

// lanes per row and vectors per lane for a width: as few lanes as hold the row in at most 3 vectors each (the sums cross few lanes and the parameters' registers
// stay few), then the whole block
#define LN16_WIDTHS(CALL)                                \
    const int nv = (c + 7) / 8;                          \
    if (nv <= 8) CALL(8, 1);                             \
    else if (nv <= 16) CALL(8, 2);                       \
    else if (nv <= 24) CALL(8, 3);                       \
    else if (nv <= 32) CALL(16, 2);                      \
    else if (nv <= 48) CALL(16, 3);                      \
    else if (nv <= 64) CALL(32, 2);                      \
    else if (nv <= 96) CALL(32, 3);                      \
    else if (nv <= 128) CALL(64, 2);                     \
    else if (nv <= 192) CALL(64, 3);                     \
    else if (nv <= 256) CALL(256, 1);                    \
    else if (nv <= 512) CALL(256, 2);                    \
    else CALL(256, 4);

template <typename T>
int ln16_fwd(const void* x, int64_t rows, int c, float eps, const float* gamma, const float* beta, void* y, float* mean, float* rstd, hipStream_t st) {
    const T* xt = static_cast<const T*>(x);
    T* yt = static_cast<T*>(y);
    if (c < 8 || c > 8192) {
        hipLaunchKernelGGL((layernorm16_fwd_any<T>), dim3(any_blocks(rows)), dim3(256), 0, st, xt, rows, c, eps, gamma, beta, yt, mean, rstd);
    } else {
#define LN16_FWD(L, V)                                                                                                                                           \
    do {                                                                                                                                                         \
        const int64_t need = ceil_div(rows, 256 / L);                                                                                                            \
        hipLaunchKernelGGL((layernorm16_fwd_kernel<T, L, V>), dim3((unsigned)(need < 2048 ? need : 2048)), dim3(256), 0, st, xt, rows, c, eps, gamma, beta, yt, mean, rstd); \
    } while (0)
        LN16_WIDTHS(LN16_FWD)
#undef LN16_FWD
    }
    return check_launch("suhpe_layernorm16_fwd");
}

template <typename T>
int ln16_bwd(const void* x, const void* dy, int64_t rows, int c, const float* mean, const float* rstd, const float* gamma, const void* skip, void* dx, float* dgamma,
             float* dbeta, int accumulate, float* part, hipStream_t st) {
    const T *xt = static_cast<const T*>(x), *dt = static_cast<const T*>(dy), *kt = static_cast<const T*>(skip);
    T* ot = static_cast<T*>(dx);
    const bool want = dgamma || dbeta;
    int blocks = 0;
    if (rows > 0 && (c < 8 || c > 8192)) {
        hipLaunchKernelGGL((layernorm16_bwd_dx_any<T>), dim3(any_blocks(rows)), dim3(256), 0, st, xt, dt, rows, c, mean, rstd, gamma, kt, ot);
        if (want) {
            blocks = (int)(ceil_div(rows, 16) < kLnBlocks ? ceil_div(rows, 16) : kLnBlocks);
            const int64_t per = ceil_div(rows, blocks);
            blocks = (int)ceil_div(rows, per);
            hipLaunchKernelGGL((layernorm16_bwd_cols_any<T>), dim3(blocks, (unsigned)ceil_div(c, 64)), dim3(256), 0, st, xt, dt, rows, c, per, mean, rstd, part);
        }
    } else if (rows > 0) {
    // Workgroups of the gradient with dgamma and dbeta: each leaves 2 c partial sums, which the second launch adds.  `need` counts groups of 256 / L rows: up to 256 one workgroup
    // each, below 1 024 one a CU, above a workgroup to every four groups, at most two a CU.  fp16, both launches, with 256 / the rule's / 512 workgroups: 31 360 x 384 27.3 /
    // 24.0 / 24.2 us, 125 440 x 192 52.8 / 40.2 / 40.3, 8 192 x 1024 20.8 / 19.0 / 19.0, 4 099 x 1357 19.5 / 19.5 / 20.0.  Where few groups are left to each, 512 would be up to
    // 1 us shorter: 6 000 x 1357 23.2 / 23.1 / 22.0, 7 840 x 576 17.4 / 17.5 / 16.4, 20 000 x 192 16.1 / 16.1 / 15.3.  The number decides the order of the sums, so it stays.
#define LN16_BWD(L, V)                                                                                                                                           \
    do {                                                                                                                                                         \
        const int64_t need = ceil_div(rows, 256 / L);                                                                                                            \
        blocks = (int)(need < 256 ? need : need < 1024 ? 256 : need < 2048 ? need / 4 : kLnBlocks);                                                              \
        if (want)                                                                                                                                                \
            hipLaunchKernelGGL((layernorm16_bwd_kernel<T, L, V, true>), dim3(blocks), dim3(256), L == 256 ? 0 : 8 * c * sizeof(float), st, xt, dt, rows, c, mean, rstd, gamma, kt, ot, part); \
        else                                                                                                                                                     \
            hipLaunchKernelGGL((layernorm16_bwd_kernel<T, L, V, false>), dim3((unsigned)(need < 2048 ? need : 2048)), dim3(256), 0, st, xt, dt, rows, c, mean, rstd, gamma, kt, ot, part); \
    } while (0)
        LN16_WIDTHS(LN16_BWD)
#undef LN16_BWD
    }
    if (want)
        hipLaunchKernelGGL(layernorm16_bwd_finish, dim3((unsigned)ceil_div(c, 16), 2), dim3(1024), 0, st, part, blocks, c, dgamma, dbeta, accumulate);
    return check_launch("suhpe_layernorm16_bwd");
}
#undef LN16_WIDTHS

}  // namespace
}  // namespace suhpe

using namespace suhpe;

extern "C" {

int suhpe_rope_axes(const void* x, int dtype, int64_t rows, int heads, int parts, int rotated, int dh, const void* pos, int pos_type, int naxes, const double* freq,
                    const int32_t* axis, int pairs, int halves, int inverse, void* y, suhpe_stream_t stream) {
    SUHPE_REQUIRE(dtype_ok(dtype), "suhpe_rope_axes: unknown dtype %d", dtype);
    SUHPE_REQUIRE(pos_type >= SUHPE_POS_I32 && pos_type <= SUHPE_POS_F32, "suhpe_rope_axes: unknown position type %d", pos_type);
    SUHPE_REQUIRE(rows >= 0 && heads > 0 && parts > 0 && rotated > 0 && rotated <= parts && dh > 1 && naxes > 0, "suhpe_rope_axes: bad sizes");
    SUHPE_REQUIRE(pairs > 0 && pairs <= 4096 && 2 * pairs <= dh, "suhpe_rope_axes: %d pairs do not fit heads of %d (at most 4096)", pairs, dh);
    SUHPE_REQUIRE((int64_t)heads * parts * dh <= (1 << 24), "suhpe_rope_axes: a row of %lld elements is too wide", (long long)heads * parts * dh);
    SUHPE_REQUIRE(rows <= 0x7fffffff, "suhpe_rope_axes: too many rows");
    if (rows == 0) return SUHPE_OK;
    SUHPE_REQUIRE(x && y && pos && freq && axis, "suhpe_rope_axes: null pointer");
    const RopeArgs a = {rows, heads, parts, rotated, dh, naxes, pairs, halves ? 1 : 0, inverse ? 1 : 0, x != y, 0, freq, axis};
    hipStream_t st = as_stream(stream);
    if (dtype == SUHPE_F32) return rope_types<float>(x, y, pos, pos_type, a, st);
    if (dtype == SUHPE_BF16) return rope_types<bf16>(x, y, pos, pos_type, a, st);
    return rope_types<f16>(x, y, pos, pos_type, a, st);
}

int suhpe_dropout_apply(const void* x, int dtype, int64_t count, float keep, const uint64_t* counter, uint64_t position, const void* skip, void* y, suhpe_stream_t stream) {
    SUHPE_REQUIRE(dtype_ok(dtype), "suhpe_dropout_apply: unknown dtype %d", dtype);
    SUHPE_REQUIRE(keep >= 0.f && keep <= 1.f, "suhpe_dropout_apply: keep %g outside [0, 1]", (double)keep);
    SUHPE_REQUIRE(count >= 0, "suhpe_dropout_apply: negative count");
    if (count == 0) return SUHPE_OK;
    SUHPE_REQUIRE(x && y && counter, "suhpe_dropout_apply: null pointer");
    const int64_t bytes = count * dtype_size(dtype);
    const Range ranges[] = {{y, bytes}, {x == y ? nullptr : x, bytes}, {skip == y ? nullptr : skip, bytes}, {counter, 16}};
    SUHPE_REQUIRE(apart(ranges, 1, 4), "suhpe_dropout_apply: y (unless it is x or skip) shares no memory with the inputs");
    // r < keep for r = k / 2^24, k a 24-bit integer  <=>  k < ceil(keep 2^24): the product is exact in double
    const double scaled = (double)keep * 16777216.0;
    uint32_t bound = (uint32_t)scaled;
    if ((double)bound < scaled) ++bound;
    const float scale = keep > 0.f ? 1.f / keep : 0.f;
    hipStream_t st = as_stream(stream);
    if (dtype == SUHPE_F32) return dropout_launch<float>(x, skip, y, count, bound, scale, counter, position, st);
    if (dtype == SUHPE_BF16) return dropout_launch<bf16>(x, skip, y, count, bound, scale, counter, position, st);
    return dropout_launch<f16>(x, skip, y, count, bound, scale, counter, position, st);
}

int suhpe_dropout_advance(uint64_t* counter, uint64_t by, suhpe_stream_t stream) {
    SUHPE_REQUIRE(counter, "suhpe_dropout_advance: null pointer");
    hipLaunchKernelGGL(dropout_advance_kernel, dim3(1), dim3(1), 0, as_stream(stream), counter, by);
    return check_launch("suhpe_dropout_advance");
}

int suhpe_layernorm16_fwd(const void* x, int dtype, int64_t rows, int c, float eps, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                          suhpe_stream_t stream) {
    SUHPE_REQUIRE(dtype == SUHPE_BF16 || dtype == SUHPE_F16, "suhpe_layernorm16_fwd: 16-bit rows only (fp32: suhpe_layernorm_fwd)");
    SUHPE_REQUIRE(rows >= 0 && c > 0 && rows <= 0x7fffffffll, "suhpe_layernorm16_fwd: bad sizes");
    if (rows == 0) return SUHPE_OK;
    SUHPE_REQUIRE(x && y && mean && rstd, "suhpe_layernorm16_fwd: null pointer");
    // (a wavefront holds its row in registers between reading and writing: y may be x itself)
    const int64_t row_bytes = rows * c * 2;
    const Range r[] = {{y, row_bytes}, {mean, rows * 4}, {rstd, rows * 4}, {x == y ? nullptr : x, row_bytes}, {gamma, (int64_t)c * 4}, {beta, (int64_t)c * 4}};
    SUHPE_REQUIRE(apart(r, 3, 6), "suhpe_layernorm16_fwd: y (unless it is x), mean and rstd share no memory with each other or with the inputs");
    if (dtype == SUHPE_BF16) return ln16_fwd<bf16>(x, rows, c, eps, gamma, beta, y, mean, rstd, as_stream(stream));
    return ln16_fwd<f16>(x, rows, c, eps, gamma, beta, y, mean, rstd, as_stream(stream));
}

int64_t suhpe_layernorm16_bwd_workspace_bytes(int c) { return (int64_t)kLnBlocks * 2 * c * (int64_t)sizeof(float); }

int suhpe_layernorm16_bwd(const void* x, const void* dy, int dtype, int64_t rows, int c, const float* mean, const float* rstd, const float* gamma, const void* skip, void* dx,
                          float* dgamma, float* dbeta, int accumulate, void* workspace, int64_t workspace_bytes, suhpe_stream_t stream) {
    SUHPE_REQUIRE(dtype == SUHPE_BF16 || dtype == SUHPE_F16, "suhpe_layernorm16_bwd: 16-bit rows only (fp32: suhpe_layernorm_bwd)");
    SUHPE_REQUIRE(rows >= 0 && c > 0 && rows <= 0x7fffffffll, "suhpe_layernorm16_bwd: bad sizes");
    SUHPE_REQUIRE(rows == 0 || (x && dy && dx && mean && rstd), "suhpe_layernorm16_bwd: null pointer");
    if (dgamma || dbeta) {
        SUHPE_REQUIRE(workspace, "suhpe_layernorm16_bwd: null workspace");
        if (workspace_bytes < suhpe_layernorm16_bwd_workspace_bytes(c)) {
            set_error("suhpe_layernorm16_bwd: workspace of %lld bytes, needs %lld", (long long)workspace_bytes, (long long)suhpe_layernorm16_bwd_workspace_bytes(c));
            return SUHPE_EWORKSPACE;
        }
    }
    const int64_t row_bytes = rows * c * 2;
    const Range r[] = {{rows ? dx : nullptr, row_bytes}, {dgamma, (int64_t)c * 4}, {dbeta, (int64_t)c * 4}, {dgamma || dbeta ? workspace : nullptr, suhpe_layernorm16_bwd_workspace_bytes(c)},
                       {x, row_bytes}, {dy, row_bytes}, {skip, row_bytes}, {mean, rows * 4}, {rstd, rows * 4}, {gamma, (int64_t)c * 4}};
    SUHPE_REQUIRE(apart(r, 4, 10), "suhpe_layernorm16_bwd: dx, dgamma, dbeta and the workspace share no memory with each other or with the inputs");
    float* part = static_cast<float*>(workspace);
    if (dtype == SUHPE_BF16) return ln16_bwd<bf16>(x, dy, rows, c, mean, rstd, gamma, skip, dx, dgamma, dbeta, accumulate, part, as_stream(stream));
    return ln16_bwd<f16>(x, dy, rows, c, mean, rstd, gamma, skip, dx, dgamma, dbeta, accumulate, part, as_stream(stream));
}

}  // extern "C"

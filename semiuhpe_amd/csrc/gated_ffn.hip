// Gated feed-forward block (forward and backward) in fp32 / bf16 / fp16:
//   g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u, y = h Wd^T + bd
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h, db = column sums
#include "lowp.h"

namespace suhpe {
namespace {

// One operand of a product over k: element (row, k) at p[row * rs + k * ks]
struct View { const void* p; int64_t rs, ks; };

// out[m][j] = sum_k A[m][k] B[j][k], 64 x 64 outputs per block, 4 x 4 per thread, sums in fp32
enum { EPI_STORE = 0, EPI_GATE = 1, EPI_GATE_BWD = 2 };
template <typename T, typename O, int EPI>
__global__ __launch_bounds__(256) void ffn_product_simple(View a, View b, View a2, View b2, int64_t M, int N, int64_t K, int64_t K2, const T* bias, const T* bias2, int act,
                                                          const T* gin, const T* uin, T* gout, T* uout, O* out, int accumulate) {
    __shared__ float As[16][65], Bs[16][65], Cs[EPI == EPI_GATE ? 16 : 1][65];
    const int t = threadIdx.x, tm = t & 15, tn = t >> 4;
    const int64_t m0 = (int64_t)blockIdx.x * 64;
    const int n0 = blockIdx.y * 64;
    float acc[4][4] = {}, acc2[4][4] = {};
    const int64_t kpad = (K + 15) / 16 * 16;
    for (int64_t k0 = 0; k0 < kpad + K2; k0 += 16) {
        const bool second = k0 >= kpad;
        const View& A = second ? a2 : a;
        const View& B = second ? b2 : b;
        const int64_t kb = second ? k0 - kpad : k0, ke = second ? K2 : K;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = t + 256 * i, kk = e & 15, r = e >> 4;
            const int64_t k = kb + kk;
            As[kk][r] = (m0 + r < M && k < ke) ? (float)static_cast<const T*>(A.p)[(m0 + r) * A.rs + k * A.ks] : 0.f;
            Bs[kk][r] = (n0 + r < N && k < ke) ? (float)static_cast<const T*>(B.p)[(n0 + r) * B.rs + k * B.ks] : 0.f;
            if (EPI == EPI_GATE) Cs[kk][r] = (n0 + r < N && k < ke) ? (float)static_cast<const T*>(b2.p)[(n0 + r) * b2.rs + k * b2.ks] : 0.f;
        }
        __syncthreads();
        for (int kk = 0; kk < 16; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] += As[kk][tm + 16 * i] * Bs[kk][tn + 16 * j];
                    if (EPI == EPI_GATE) acc2[i][j] += As[kk][tm + 16 * i] * Cs[kk][tn + 16 * j];
                }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + tm + 16 * i;
            const int n = n0 + tn + 16 * j;
            if (m >= M || n >= N) continue;
            const int64_t at = m * N + n;
            if constexpr (EPI == EPI_GATE) {
                const float g = acc[i][j] + (bias ? (float)bias[n] : 0.f), u = acc2[i][j] + (bias2 ? (float)bias2[n] : 0.f);
                if (gout) { gout[at] = (T)g; uout[at] = (T)u; }
                out[at] = (O)(act_apply(g, act) * u);
            } else if constexpr (EPI == EPI_GATE_BWD) {
                const float g = (float)gin[at], u = (float)uin[at];
                gout[at] = (T)(acc[i][j] * u * act_grad(g, act));
                uout[at] = (T)(acc[i][j] * act_apply(g, act));
            } else {
                float v = acc[i][j] + (bias ? (float)bias[n] : 0.f);
                if (accumulate) v += (float)out[at];
                out[at] = (O)v;
            }
        }
}

template <typename T, typename O>
__global__ __launch_bounds__(256) void ffn_column_sum_simple(const T* x, int64_t rows, int c, O* out, int accumulate) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= c) return;
    float s = 0.f;
    for (int64_t r = 0; r < rows; ++r) s += (float)x[r * c + j];
    out[j] = (O)(accumulate ? (float)out[j] + s : s);
}

inline dim3 tiles(int64_t M, int N) { return dim3((unsigned)ceil_div(M, 64), (unsigned)ceil_div(N, 64)); }

template <typename T>
int ffn_fwd(int act, int64_t m, int k, int n, int o, const void* x, const void* wg, const void* wu, const void* wd, const void* bg, const void* bu, const void* bd, void* g,
            void* u, void* h, void* y, hipStream_t st) {
    auto c = [](const void* p) { return static_cast<const T*>(p); };
    auto w = [](void* p) { return static_cast<T*>(p); };
    hipLaunchKernelGGL((ffn_product_simple<T, T, EPI_GATE>), tiles(m, n), dim3(256), 0, st, View{x, k, 1}, View{wg, k, 1}, View{}, View{wu, k, 1}, m, n, (int64_t)k, (int64_t)0,
                       c(bg), c(bu), act, nullptr, nullptr, w(g), w(u), w(h), 0);
    hipLaunchKernelGGL((ffn_product_simple<T, T, EPI_STORE>), tiles(m, o), dim3(256), 0, st, View{h, n, 1}, View{wd, n, 1}, View{}, View{}, m, o, (int64_t)n, (int64_t)0, c(bd),
                       nullptr, 0, nullptr, nullptr, nullptr, nullptr, w(y), 0);
    return check_launch("suhpe_gated_ffn_fwd");
}

template <typename T, typename O>
int ffn_bwd(int act, int64_t m, int k, int n, int o, const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* g, const void* u, const void* h,
            void* dx, void* dwg, void* dwu, void* dwd, void* dbg, void* dbu, void* dbd, int accumulate, void* dg, void* du, hipStream_t st) {
    auto c = [](const void* p) { return static_cast<const T*>(p); };
    auto w = [](void* p) { return static_cast<T*>(p); };
    auto q = [](void* p) { return static_cast<O*>(p); };
    if (m > 0) {
        hipLaunchKernelGGL((ffn_product_simple<T, T, EPI_GATE_BWD>), tiles(m, n), dim3(256), 0, st, View{dy, o, 1}, View{wd, 1, n}, View{}, View{}, m, n, (int64_t)o, (int64_t)0,
                           nullptr, nullptr, act, c(g), c(u), w(dg), w(du), static_cast<T*>(nullptr), 0);
        if (dx)
            hipLaunchKernelGGL((ffn_product_simple<T, T, EPI_STORE>), tiles(m, k), dim3(256), 0, st, View{dg, n, 1}, View{wg, 1, k}, View{du, n, 1}, View{wu, 1, k}, m, k,
                               (int64_t)n, (int64_t)n, nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, w(dx), 0);
    }
    auto weight = [&](const void* left, int rows, const void* right, int cols, void* out) {
        hipLaunchKernelGGL((ffn_product_simple<T, O, EPI_STORE>), tiles(rows, cols), dim3(256), 0, st, View{left, 1, rows}, View{right, 1, cols}, View{}, View{}, (int64_t)rows, cols, m,
                           (int64_t)0, nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, q(out), accumulate);
    };
    if (dwg) { weight(dg, n, x, k, dwg); weight(du, n, x, k, dwu); weight(dy, o, h, n, dwd); }
    auto bias = [&](const void* v, int cols, void* out) {
        if (out) hipLaunchKernelGGL((ffn_column_sum_simple<T, O>), dim3((unsigned)ceil_div(cols, 256)), dim3(256), 0, st, c(v), m, cols, q(out), accumulate);
    };
    bias(dg, n, dbg); bias(du, n, dbu); bias(dy, o, dbd);
    return check_launch("suhpe_gated_ffn_bwd");
}

int ffn_sizes(const char* who, int dtype, int act, int64_t m, int k, int n, int o) {
    SUHPE_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", who, dtype);
    SUHPE_REQUIRE(act >= SUHPE_ACT_NONE && act <= SUHPE_ACT_SIGMOID, "%s: unknown activation %d", who, act);
    SUHPE_REQUIRE(m >= 0 && m <= 0x7fffff00ll && k > 0 && n > 0 && o > 0, "%s: bad sizes m %lld k %d n %d o %d", who, (long long)m, k, n, o);
    SUHPE_REQUIRE(k <= (1 << 20) && n <= (1 << 20) && o <= (1 << 20), "%s: widths up to 2^20", who);
    return SUHPE_OK;
}

}  // namespace
}  // namespace suhpe

using namespace suhpe;

extern "C" {

int64_t suhpe_gated_ffn_fwd_workspace_bytes(int dtype, int64_t m, int k, int n, int o) { return 0; }

int suhpe_gated_ffn_fwd(int dtype, int act, int64_t m, int k, int n, int o, const void* x, const void* wg, const void* wu, const void* wd, const void* bg, const void* bu,
                        const void* bd, void* g, void* u, void* h, void* y, void* workspace, int64_t workspace_bytes, suhpe_stream_t stream) {
    if (int rc = ffn_sizes("suhpe_gated_ffn_fwd", dtype, act, m, k, n, o)) return rc;
    SUHPE_REQUIRE((g == nullptr) == (u == nullptr), "suhpe_gated_ffn_fwd: g and u are kept together or not at all");
    if (m == 0) return SUHPE_OK;
    SUHPE_REQUIRE(x && wg && wu && wd && h && y, "suhpe_gated_ffn_fwd: null pointer");
    hipStream_t st = as_stream(stream);
    if (dtype == SUHPE_F32) return ffn_fwd<float>(act, m, k, n, o, x, wg, wu, wd, bg, bu, bd, g, u, h, y, st);
    if (dtype == SUHPE_BF16) return ffn_fwd<bf16>(act, m, k, n, o, x, wg, wu, wd, bg, bu, bd, g, u, h, y, st);
    return ffn_fwd<f16>(act, m, k, n, o, x, wg, wu, wd, bg, bu, bd, g, u, h, y, st);
}

int64_t suhpe_gated_ffn_bwd_workspace_bytes(int dtype, int64_t m, int k, int n, int o) { return 2 * ceil_div(m * n * dtype_size(dtype), 256) * 256; }

int suhpe_gated_ffn_bwd(int dtype, int act, int64_t m, int k, int n, int o, const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* g,
                        const void* u, const void* h, void* dx, void* dwg, void* dwu, void* dwd, void* dbg, void* dbu, void* dbd, int grad_dtype, int accumulate,
                        void* workspace, int64_t workspace_bytes, suhpe_stream_t stream) {
    if (int rc = ffn_sizes("suhpe_gated_ffn_bwd", dtype, act, m, k, n, o)) return rc;
    SUHPE_REQUIRE(grad_dtype == dtype || grad_dtype == SUHPE_F32, "suhpe_gated_ffn_bwd: gradients have the weights' type or fp32");
    SUHPE_REQUIRE((dwg != nullptr) == (dwu != nullptr) && (dwg != nullptr) == (dwd != nullptr), "suhpe_gated_ffn_bwd: the three weights' gradients are wanted together or not at all");
    SUHPE_REQUIRE(m == 0 || (dy && x && wg && wu && wd && g && u && h), "suhpe_gated_ffn_bwd: null pointer");
    const int64_t need = suhpe_gated_ffn_bwd_workspace_bytes(dtype, m, k, n, o);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        set_error("suhpe_gated_ffn_bwd: workspace of %lld bytes, needs %lld", (long long)workspace_bytes, (long long)need);
        return SUHPE_EWORKSPACE;
    }
    void *dg = workspace, *du = static_cast<char*>(workspace) + need / 2;
    hipStream_t st = as_stream(stream);
#define FFN_BWD(T, O) ffn_bwd<T, O>(act, m, k, n, o, dy, x, wg, wu, wd, g, u, h, dx, dwg, dwu, dwd, dbg, dbu, dbd, accumulate, dg, du, st)
    if (dtype == SUHPE_F32) return FFN_BWD(float, float);
    if (dtype == SUHPE_BF16) return grad_dtype == SUHPE_F32 ? FFN_BWD(bf16, float) : FFN_BWD(bf16, bf16);
    return grad_dtype == SUHPE_F32 ? FFN_BWD(f16, float) : FFN_BWD(f16, f16);
#undef FFN_BWD
}

}  // extern "C"

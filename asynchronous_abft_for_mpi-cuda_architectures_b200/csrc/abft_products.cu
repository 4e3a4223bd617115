// Products of language models: rows quantised to 8-bit integers, the 8-bit
// product with a scale for each token and channel and an exact checksum test,
// and the gated feed-forward block with its gradients.
//
// Matrices are row-major, weights are N x K (a channel's weights are one row).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "abft_b200.h"
#include "abft_internal.h"

namespace abft {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ------------------------------------------------------------ activations ---
//
//   silu       a = g s,                s = 1 / (1 + e^-g)      a' = s (1 + g (1 - s))
//   gelu       a = g p,                p = erfc(-g/sqrt2) / 2    a' = p + g e^(-g^2/2) / sqrt(2 pi)
//   gelu_tanh  a = g t, t = s(2 c (g + b g^3)), c = sqrt(2/pi), b = 0.044715
//                                      a' = t + 2 c g t (1 - t) (1 + 3 b g^2)
//
// (1 + tanh z) / 2 = s(2 z), so both forms with a sigmoid share one
// exponential. Everything is evaluated in 32 bits; the sigmoid's fast division
// returns 0 for a divisor above 2^126, where the value is below 2^-126.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

constexpr float kTanhC2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;
constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

template <int ACT>
__device__ __forceinline__ float act(float g) {
    if constexpr (ACT == ABFT_ACT_SILU) return g * sigmoid(g);
    if constexpr (ACT == ABFT_ACT_GELU) return 0.5f * g * erfcf(-g * kSqrtHalf);
    return g * sigmoid(kTanhC2 * (g + kTanhB * g * g * g));
}

template <int ACT>
__device__ __forceinline__ void act_grad(float g, float& a, float& slope) {
    if constexpr (ACT == ABFT_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if constexpr (ACT == ABFT_ACT_GELU) {
        const float p = 0.5f * erfcf(-g * kSqrtHalf);
        a = g * p;
        slope = p + g * __expf(-0.5f * g * g) * kInvSqrt2Pi;
    } else {
        const float t = sigmoid(kTanhC2 * (g + kTanhB * g * g * g));
        a = g * t;
        // beyond 12 the second term is below the smallest number; the clamp keeps g^2 finite
        const float c = fminf(fmaxf(g, -12.0f), 12.0f);
        slope = t + kTanhC2 * c * t * (1.0f - t) * (1.0f + 3.0f * kTanhB * c * c);
    }
}

// -------------------------------------------------------- row quantisation ---
//
// scale = fl32(max |x| / 127), q = the real quotient x / scale rounded once to
// the nearest integer, ties to even. The first guess x * (1 / scale) is off by
// less than one step, and x - q scale is exact in 32 bits (both are multiples
// of the same power of two and the difference has at most 24 bits), so
// comparing twice it with the scale settles every tie.
__device__ __forceinline__ float round_quotient(float x, float scale, float inv) {
    float q = rintf(x * inv);
    const float r2 = 2.0f * fmaf(-q, scale, x);
    const float over = fabsf(r2) - scale;
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (over > 0.0f || (over == 0.0f && odd)) q += copysignf(1.0f, r2);
    return fminf(fmaxf(q, -127.0f), 127.0f);
}

template <typename T>
__global__ void __launch_bounds__(256) k_quantize_rows(const T* __restrict__ x, int64_t ldx, int K, int8_t* __restrict__ q,
                                                       int64_t ldq, float* __restrict__ scale,
                                                       const int32_t* __restrict__ checksum,
                                                       int64_t* __restrict__ expect) {
    __shared__ unsigned smax[8];
    __shared__ long long ssum[8];
    const int row = blockIdx.x;
    const T* xr = x + static_cast<int64_t>(row) * ldx;
    int8_t* qr = q + static_cast<int64_t>(row) * ldq;
    // largest magnitude by its bits: a NaN's are above infinity's, which are above every number's
    unsigned m = 0;
    for (int k = threadIdx.x; k < K; k += 256) m = max(m, __float_as_uint(to_f32(xr[k])) & 0x7fffffffu);
    m = __reduce_max_sync(~0u, m);
    if (threadIdx.x % 32 == 0) smax[threadIdx.x / 32] = m;
    __syncthreads();
    for (int w = 0; w < 8; ++w) m = max(m, smax[w]);
    const bool finite = m < 0x7f800000u;
    const float s = finite ? __fdiv_rn(__uint_as_float(m), 127.0f) : __uint_as_float(0x7fc00000u);
    // 2^100 keeps 1 / scale and the remainder clear of the subnormal range
    const float up = finite && s < 0x1p-100f ? 0x1p100f : 1.0f;
    const float su = s * up;
    const float inv = 1.0f / su;
    long long sum = 0;
    for (int k = threadIdx.x; k < K; k += 256) {
        const int v = finite && s > 0.0f ? static_cast<int>(round_quotient(to_f32(xr[k]) * up, su, inv)) : 0;
        qr[k] = static_cast<int8_t>(v);
        if (checksum) sum += static_cast<long long>(v) * checksum[k];
    }
    if (threadIdx.x == 0) scale[row] = s;
    if (checksum) {
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (threadIdx.x % 32 == 0) ssum[threadIdx.x / 32] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 8; ++w) sum += ssum[w];
            expect[row] = sum;
        }
    }
}

__global__ void __launch_bounds__(256) k_column_checksum(const int8_t* __restrict__ w, int64_t ldw, int N, int K,
                                                         int32_t* __restrict__ checksum) {
    const int k = blockIdx.x * 256 + threadIdx.x;
    if (k >= K) return;
    int sum = 0;
    for (int n = 0; n < N; ++n) sum += w[static_cast<int64_t>(n) * ldw + k];
    checksum[k] = sum;
}

// ---------------------------------------------------------------- products ---

constexpr int kTile = 64, kStep = 16;

// One 64 x 64 tile of A B^T per block, operands by element strides: A(m, k) at
// m * ar + k * ac, B(n, k) at n * br + k * bc.
template <typename T, typename Acc>
__device__ __forceinline__ void tile_product(const T* A, int64_t ar, int64_t ac, const T* B, int64_t br, int64_t bc,
                                             int M, int N, int K, int m0, int n0, Acc (&acc)[4][4]) {
    __shared__ Acc sa[kStep][kTile + 1], sb[kStep][kTile + 1];
    const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
    for (int k0 = 0; k0 < K; k0 += kStep) {
        for (int e = threadIdx.x; e < kTile * kStep; e += 256) {
            const int r = e / kStep, k = e % kStep;
            Acc a = 0, b = 0;
            if constexpr (sizeof(T) == 1) {
                if (m0 + r < M && k0 + k < K) a = A[(m0 + r) * ar + (k0 + k) * ac];
                if (n0 + r < N && k0 + k < K) b = B[(n0 + r) * br + (k0 + k) * bc];
            } else {
                if (m0 + r < M && k0 + k < K) a = to_f32(A[(m0 + r) * ar + (k0 + k) * ac]);
                if (n0 + r < N && k0 + k < K) b = to_f32(B[(n0 + r) * br + (k0 + k) * bc]);
            }
            sa[k][r] = a;
            sb[k][r] = b;
        }
        __syncthreads();
        for (int k = 0; k < kStep; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][tm * 4 + i] * sb[k][tn * 4 + j];
        __syncthreads();
    }
}

template <typename O>
__global__ void __launch_bounds__(256) k_int8_matmul(const int8_t* q, int64_t ldq, const float* q_scale,
                                                     const int8_t* w, int64_t ldw, const float* w_scale, int T, int N,
                                                     int K, O* y, int64_t ldy, unsigned long long* rowdiff) {
    int acc[4][4] = {};
    const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
    tile_product<int8_t, int>(q, ldq, 1, w, ldw, 1, T, N, K, m0, n0, acc);
    for (int i = 0; i < 4; ++i) {
        const int t = m0 + threadIdx.x / 16 * 4 + i;
        if (t >= T) continue;
        long long sum = 0;
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + threadIdx.x % 16 * 4 + j;
            if (n >= N) continue;
            sum += acc[i][j];
            y[t * ldy + n] = from_f32<O>(static_cast<float>(acc[i][j]) * q_scale[t] * w_scale[n]);
        }
        if (rowdiff) atomicAdd(rowdiff + t, static_cast<unsigned long long>(sum));
    }
}

__global__ void k_negate(const int64_t* __restrict__ in, int64_t* __restrict__ out, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = -in[i];
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_gated_ffn(const T* x, int64_t ldx, const T* wg, int64_t ldwg, const T* wu,
                                                   int64_t ldwu, int Tn, int N, int K, T* h, int64_t ldh, T* gs,
                                                   int64_t ldg, T* us, int64_t ldu) {
    float g[4][4] = {}, u[4][4] = {};
    const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
    tile_product<T, float>(x, ldx, 1, wg, ldwg, 1, Tn, N, K, m0, n0, g);
    tile_product<T, float>(x, ldx, 1, wu, ldwu, 1, Tn, N, K, m0, n0, u);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t t = m0 + threadIdx.x / 16 * 4 + i, n = n0 + threadIdx.x % 16 * 4 + j;
            if (t >= Tn || n >= N) continue;
            h[t * ldh + n] = from_f32<T>(act<ACT>(g[i][j]) * u[i][j]);
            if (gs) {
                gs[t * ldg + n] = from_f32<T>(g[i][j]);
                us[t * ldu + n] = from_f32<T>(u[i][j]);
            }
        }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_gate_grad(const T* dh, int64_t ldd, const T* g, int64_t ldg, const T* u,
                                                   int64_t ldu, int N, T* dg, T* du, int64_t ldo) {
    const int n = blockIdx.y * 256 + threadIdx.x;
    const int64_t t = blockIdx.x;
    if (n >= N) return;
    const float d = to_f32(dh[t * ldd + n]);
    float a, slope;
    act_grad<ACT>(to_f32(g[t * ldg + n]), a, slope);
    dg[t * ldo + n] = from_f32<T>(d * to_f32(u[t * ldu + n]) * slope);
    du[t * ldo + n] = from_f32<T>(d * a);
}

// C = A0 B0^T (+ A1 B1^T)
template <typename T>
__global__ void __launch_bounds__(256) k_product(const T* A0, const T* A1, int64_t ar, int64_t ac, const T* B0,
                                                 int64_t br0, int64_t bc0, const T* B1, int64_t br1, int64_t bc1,
                                                 int M, int N, int K, T* C, int64_t ldc) {
    float acc[4][4] = {};
    const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
    tile_product<T, float>(A0, ar, ac, B0, br0, bc0, M, N, K, m0, n0, acc);
    if (A1) tile_product<T, float>(A1, ar, ac, B1, br1, bc1, M, N, K, m0, n0, acc);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + threadIdx.x / 16 * 4 + i, n = n0 + threadIdx.x % 16 * 4 + j;
            if (m < M && n < N) C[m * ldc + n] = from_f32<T>(acc[i][j]);
        }
}

int cdiv(int a, int b) { return (a + b - 1) / b; }

int bad(const char* msg) {
    set_error(msg);
    return ABFT_ERR_ARG;
}

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? ABFT_OK : cuda_fail(e, what);
}

// dgate | dup, each T rows on a pitch of 16 bytes
int64_t grad_pitch(int N) { return (static_cast<int64_t>(N) + 7) / 8 * 8; }

template <typename F>
int with_type(int type, F&& f) {
    if (type == ABFT_TYPE_F16) return f(__half());
    return f(__nv_bfloat16());
}

template <typename F>
int with_act(int activation, F&& f) {
    if (activation == ABFT_ACT_SILU) return f(std::integral_constant<int, ABFT_ACT_SILU>());
    if (activation == ABFT_ACT_GELU) return f(std::integral_constant<int, ABFT_ACT_GELU>());
    return f(std::integral_constant<int, ABFT_ACT_GELU_TANH>());
}

}  // namespace
}  // namespace abft

using namespace abft;

extern "C" {

int abft_quantize_rows(const void* dX, int64_t ldx, int type, int T, int K, int8_t* dQ, int64_t ldq, float* dScale,
                       const int32_t* dChecksum, int64_t* dExpect, void* stream) {
    if (T < 0 || K < 1 || ldx < K || ldq < K || type < ABFT_TYPE_F32 || type > ABFT_TYPE_BF16)
        return bad("abft_quantize_rows: bad argument (need T >= 0, K >= 1, ldx >= K, ldq >= K and an element type)");
    if (T == 0) return ABFT_OK;
    if (!dX || !dQ || !dScale || (dChecksum != nullptr) != (dExpect != nullptr))
        return bad("abft_quantize_rows: bad argument (missing pointer, or one of dChecksum and dExpect alone)");
    auto go = [&](auto tag) {
        using E = decltype(tag);
        k_quantize_rows<E><<<T, 256, 0, (cudaStream_t)stream>>>((const E*)dX, ldx, K, dQ, ldq, dScale, dChecksum,
                                                                dExpect);
        return launched("abft_quantize_rows");
    };
    if (type == ABFT_TYPE_F32) return go(0.0f);
    return with_type(type, go);
}

int abft_column_checksum(const int8_t* dW, int64_t ldw, int N, int K, int32_t* dChecksum, void* stream) {
    if (!dW || !dChecksum || N < 1 || N > ABFT_INT8_MAX_ROWS || K < 1 || ldw < K)
        return bad("abft_column_checksum: bad argument (need pointers, 1 <= N <= 2^24, K >= 1, ldw >= K)");
    k_column_checksum<<<cdiv(K, 256), 256, 0, (cudaStream_t)stream>>>(dW, ldw, N, K, dChecksum);
    return launched("abft_column_checksum");
}

size_t abft_int8_matmul_ws_bytes(const int8_t* dQ, int64_t ldq, const int8_t* dW, int64_t ldw, int T, int N, int K) {
    return 0;
}

int abft_int8_matmul(const int8_t* dQ, int64_t ldq, const float* dQScale, const int8_t* dW, int64_t ldw,
                     const float* dWScale, int T, int N, int K, void* dY, int64_t ldy, int type,
                     const int64_t* dExpect, int64_t* dRowDiff, void* dWork, size_t work_bytes, void* stream) {
    if (T < 0 || N < 1 || K < 1 || K > ABFT_INT8_MAX_K || ldq < K || ldw < K || ldy < N || type < ABFT_TYPE_F32 ||
        type > ABFT_TYPE_BF16)
        return bad("abft_int8_matmul: bad argument (need T >= 0, N >= 1, 1 <= K <= 131071, ldq >= K, ldw >= K, "
                   "ldy >= N and an element type)");
    if (T == 0) return ABFT_OK;
    if (!dQ || !dQScale || !dW || !dWScale || !dY || (dExpect != nullptr) != (dRowDiff != nullptr))
        return bad("abft_int8_matmul: bad argument (missing pointer, or one of dExpect and dRowDiff alone)");
    if (work_bytes < abft_int8_matmul_ws_bytes(dQ, ldq, dW, ldw, T, N, K)) return bad("abft_int8_matmul: workspace too small");
    cudaStream_t s = (cudaStream_t)stream;
    if (dExpect) k_negate<<<cdiv(T, 256), 256, 0, s>>>(dExpect, dRowDiff, T);
    auto go = [&](auto tag) {
        using E = decltype(tag);
        k_int8_matmul<E><<<dim3(cdiv(N, kTile), cdiv(T, kTile)), 256, 0, s>>>(
            dQ, ldq, dQScale, dW, ldw, dWScale, T, N, K, (E*)dY, ldy, (unsigned long long*)dRowDiff);
        return launched("abft_int8_matmul");
    };
    if (type == ABFT_TYPE_F32) return go(0.0f);
    return with_type(type, go);
}

size_t abft_gated_ffn_ws_bytes(const void* dX, int64_t ldx, const void* dWGate, int64_t ldwg, const void* dWUp,
                               int64_t ldwu, int T, int N, int K) {
    return 0;
}

int abft_gated_ffn(const void* dX, int64_t ldx, const void* dWGate, int64_t ldwg, const void* dWUp, int64_t ldwu,
                   int T, int N, int K, int type, int activation, void* dH, int64_t ldh, void* dG, int64_t ldg,
                   void* dU, int64_t ldu, void* dWork, size_t work_bytes, void* stream) {
    if (T < 0 || N < 1 || K < 1 || ldx < K || ldwg < K || ldwu < K || ldh < N || (dG && ldg < N) || (dU && ldu < N) ||
        (type != ABFT_TYPE_F16 && type != ABFT_TYPE_BF16) || activation < ABFT_ACT_SILU ||
        activation > ABFT_ACT_GELU_TANH)
        return bad("abft_gated_ffn: bad argument (need T >= 0, N >= 1, K >= 1, pitches that hold a row, a 16-bit "
                   "element type and an activation)");
    if (T == 0) return ABFT_OK;
    if (!dX || !dWGate || !dWUp || !dH || (dG != nullptr) != (dU != nullptr))
        return bad("abft_gated_ffn: bad argument (missing pointer, or one of dG and dU alone)");
    if (work_bytes < abft_gated_ffn_ws_bytes(dX, ldx, dWGate, ldwg, dWUp, ldwu, T, N, K))
        return bad("abft_gated_ffn: workspace too small");
    return with_type(type, [&](auto tag) {
        using E = decltype(tag);
        return with_act(activation, [&](auto a) {
            k_gated_ffn<E, decltype(a)::value><<<dim3(cdiv(N, kTile), cdiv(T, kTile)), 256, 0, (cudaStream_t)stream>>>(
                (const E*)dX, ldx, (const E*)dWGate, ldwg, (const E*)dWUp, ldwu, T, N, K, (E*)dH, ldh, (E*)dG, ldg,
                (E*)dU, ldu);
            return launched("abft_gated_ffn");
        });
    });
}

size_t abft_gated_ffn_backward_ws_bytes(const void* dX, int64_t ldx, const void* dWGate, int64_t ldwg,
                                        const void* dWUp, int64_t ldwu, int T, int N, int K) {
    if (T < 1 || N < 1 || K < 1) return 0;
    return 4 * static_cast<size_t>(T) * grad_pitch(N);
}

int abft_gated_ffn_backward(const void* dDH, int64_t ldd, const void* dX, int64_t ldx, const void* dWGate,
                            int64_t ldwg, const void* dWUp, int64_t ldwu, const void* dG, int64_t ldg, const void* dU,
                            int64_t ldu, int T, int N, int K, int type, int activation, void* dDX, int64_t lddx,
                            void* dDWGate, int64_t lddwg, void* dDWUp, int64_t lddwu, void* dWork, size_t work_bytes,
                            void* stream) {
    if (T < 0 || N < 1 || K < 1 || ldd < N || ldx < K || ldwg < K || ldwu < K || ldg < N || ldu < N || lddx < K ||
        lddwg < K || lddwu < K || (type != ABFT_TYPE_F16 && type != ABFT_TYPE_BF16) || activation < ABFT_ACT_SILU ||
        activation > ABFT_ACT_GELU_TANH)
        return bad("abft_gated_ffn_backward: bad argument (need T >= 0, N >= 1, K >= 1, pitches that hold a row, a "
                   "16-bit element type and an activation)");
    if (!dDWGate || !dDWUp) return bad("abft_gated_ffn_backward: bad argument (missing pointer)");
    cudaStream_t s = (cudaStream_t)stream;
    if (T == 0) {  // no token: the weights' gradients are empty sums
        cudaError_t e = cudaMemset2DAsync(dDWGate, lddwg * 2, 0, static_cast<size_t>(K) * 2, N, s);
        if (e == cudaSuccess) e = cudaMemset2DAsync(dDWUp, lddwu * 2, 0, static_cast<size_t>(K) * 2, N, s);
        return e == cudaSuccess ? ABFT_OK : cuda_fail(e, "abft_gated_ffn_backward");
    }
    if (!dDH || !dX || !dWGate || !dWUp || !dG || !dU || !dDX)
        return bad("abft_gated_ffn_backward: bad argument (missing pointer)");
    if (!dWork || work_bytes < abft_gated_ffn_backward_ws_bytes(dX, ldx, dWGate, ldwg, dWUp, ldwu, T, N, K))
        return bad("abft_gated_ffn_backward: workspace too small");
    return with_type(type, [&](auto tag) {
        using E = decltype(tag);
        const int64_t p = grad_pitch(N);
        E* dg = (E*)dWork;
        E* du = dg + T * p;
        with_act(activation, [&](auto a) {
            k_gate_grad<E, decltype(a)::value><<<dim3(T, cdiv(N, 256)), 256, 0, s>>>(
                (const E*)dDH, ldd, (const E*)dG, ldg, (const E*)dU, ldu, N, dg, du, p);
            return 0;
        });
        k_product<E><<<dim3(cdiv(K, kTile), cdiv(T, kTile)), 256, 0, s>>>(
            dg, du, p, 1, (const E*)dWGate, 1, ldwg, (const E*)dWUp, 1, ldwu, T, K, N, (E*)dDX, lddx);
        k_product<E><<<dim3(cdiv(K, kTile), cdiv(N, kTile)), 256, 0, s>>>(
            dg, nullptr, 1, p, (const E*)dX, 1, ldx, nullptr, 0, 0, N, K, T, (E*)dDWGate, lddwg);
        k_product<E><<<dim3(cdiv(K, kTile), cdiv(N, kTile)), 256, 0, s>>>(
            du, nullptr, 1, p, (const E*)dX, 1, ldx, nullptr, 0, 0, N, K, T, (E*)dDWUp, lddwu);
        return launched("abft_gated_ffn_backward");
    });
}

}  // extern "C"

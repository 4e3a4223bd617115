// Products of language models: rows quantised to 8-bit integers, the 8-bit
// product with a scale for each token and channel and an exact checksum test,
// and the gated feed-forward block with its gradients.
//
// Matrices are row-major, weights are N x K (a channel's weights are one row).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "abft_b200.h"
#include "abft_internal.h"
#include "abft_tensor.h"

namespace abft {
namespace {

constexpr int kWaitLimit = 1 << 20;  // polls of the waits that follow one that ran out

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ------------------------------------------------------------ activations ---
//
//   silu       a = g s,                s = 1 / (1 + e^-g)      a' = s (1 + g (1 - s))
//   gelu       a = g p,                p = Phi(g) (below)      a' = p + g e^(-g^2/2) / sqrt(2 pi)
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

// The normal distribution function. With z = |g| / sqrt2 and t = 1 / (1 + 0.4 z) its
// tail is erfc(z) / 2 = t e^(f(t) - z^2) / 2, f(t) = ln(e^(z^2) erfc(z) / t); f is smooth
// on (0, 1], and a polynomial of degree 8 fitted to it (least squares at 4000
// Chebyshev nodes of 0 <= z <= 14, 64 bits) is off by 1.3e-7 with its coefficients as
// they stand; evaluated in 32 bits the tail is off by 4.4e-7 relative up to |g| = 1,
// 1.5e-6 up to 4 and 1.5e-5 up to 13 (the roundings of z and of the exponent, which grow
// with it), plus what the exponential loses of its argument.
// No branch and 18 instructions, where erfcf cost 3 to 4 us of results that are not
// hidden behind products (1000 x 1536 x 1024 block: 13.5 us, 11.5 so).
__device__ __forceinline__ float normal(float g) {
    const float z = fabsf(g) * kSqrtHalf;
    const float t = __fdividef(1.0f, fmaf(0.4f, z, 1.0f));
    float f = -0.21217621862888336f;
    f = fmaf(f, t, 0.9476717710494995f);
    f = fmaf(f, t, -1.5340924263000488f);
    f = fmaf(f, t, 1.0546685457229614f);
    f = fmaf(f, t, -0.48204973340034485f);
    f = fmaf(f, t, 0.3168873190879822f);
    f = fmaf(f, t, 0.39554527401924133f);
    f = fmaf(f, t, 1.0022913217544556f);
    f = fmaf(f, t, -1.488745927810669f);
    const float tail = 0.5f * t * __expf(fmaf(-z, z, f));
    return g < 0.0f ? tail : 1.0f - tail;
}

template <int ACT>
__device__ __forceinline__ float act(float g) {
    if constexpr (ACT == ABFT_ACT_SILU) return g * sigmoid(g);
    if constexpr (ACT == ABFT_ACT_GELU) return g * normal(g);
    return g * sigmoid(kTanhC2 * (g + kTanhB * g * g * g));
}

template <int ACT>
__device__ __forceinline__ void act_grad(float g, float& a, float& slope) {
    if constexpr (ACT == ABFT_ACT_SILU) {
        const float s = sigmoid(g);
        a = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if constexpr (ACT == ABFT_ACT_GELU) {
        const float p = normal(g);
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
// the nearest integer, ties to even. The first guess, x * (1 / scale) rounded,
// is off by at most one and only where the quotient lies within 2^-16 of a
// half; r = x - q scale is exact in 32 bits (both terms are multiples of the
// same power of two and the difference has at most 24 bits), so comparing |r|
// with scale / 2 settles it.
//
// Bound by reading x once: a row stays in registers between the search for its
// maximum and its rounding. 5 instructions for an element's integer: adding
// 1.5 * 2^23 rounds it and leaves it in the low byte, the remainder is only
// checked for the largest of 8.
constexpr float kRound = 12582912.0f;  // 1.5 * 2^23

// The guess t = kRound + q moved by one where the quotient's half was missed.
__device__ __forceinline__ float settle(float t, float x, float scale, float half) {
    const float r = fmaf(-(t - kRound), scale, x);
    const bool odd = (__float_as_int(t) & 1) != 0;
    if (fabsf(r) > half || (fabsf(r) == half && odd)) t += copysignf(1.0f, r);
    return t;
}

// Rows whose scale is near or below the smallest normal number: 2^100 times
// everything is exact and keeps 1 / scale and the remainder normal; the scale
// itself may have lost bits, so the quotient may pass 127.
__device__ __noinline__ int quantize_tiny(float x, float scale) {
    if (!(scale > 0.0f)) return 0;
    const float s = scale * 0x1p100f;
    x *= 0x1p100f;
    const float q = fminf(fmaxf(rintf(x / s), -200.0f), 200.0f);
    const float t = settle(q + kRound, fminf(fmaxf(x, -200.0f * s), 200.0f * s), s, 0.5f * s);
    return static_cast<int>(fminf(fmaxf(t - kRound, -127.0f), 127.0f));
}

// 16 bytes at any address inside [begin, end): two aligned loads and a shift, or,
// where those would leave the range, element by element.
template <typename T>
__device__ __forceinline__ uint4 load_any(const T* at, const void* begin, const void* end) {
    const char* p = reinterpret_cast<const char*>(at);
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    const char* low = p - off;
    if (off == 0) return __ldg(reinterpret_cast<const uint4*>(p));
    if (low < begin || low + 32 > end) {
        alignas(16) T e[16 / sizeof(T)];
#pragma unroll
        for (int i = 0; i < 16 / (int)sizeof(T); ++i) e[i] = at[i];
        return *reinterpret_cast<uint4*>(e);
    }
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(low)), b = __ldg(reinterpret_cast<const uint4*>(low) + 1);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (off & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int bits = (off & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

struct QuantArgs {
    bool aligned;    // rows of x and the checksum to 16 bytes, rows of q to 8
    const void* x;
    int64_t ldx;
    int T, K;
    int8_t* q;
    int64_t ldq;
    float* scale;
    const int32_t* checksum;
    int64_t* expect;
};

// Eight elements as they come from memory.
template <typename T>
struct Eight {
    uint4 v[sizeof(T) / 2];

    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void load_any(const T* p, const void* begin, const void* end) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = abft::load_any<T>(p + i * (16 / sizeof(T)), begin, end);
    }
    __device__ __forceinline__ void load(const T* p, int n) {  // n of them, zeros after
        alignas(16) T e[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) e[i] = p[i];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<uint4*>(e)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ float operator[](int i) const {
        const uint32_t w = word(i * (int)sizeof(T) / 4);
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
        else return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w & 0xffffu)));
    }
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& q = v[i / 4];
        return i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w;
    }
    // Largest magnitude by its bits (a NaN's are above infinity's, which are above every number's), as a packed pair for
    // the 16-bit types.
    __device__ __forceinline__ uint32_t largest(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) {
            if constexpr (sizeof(T) == 4) m = max(m, word(i) & 0x7fffffffu);
            else m = __vmaxu2(m, word(i) & 0x7fff7fffu);
        }
        return m;
    }
    // That largest as the bits of a 32-bit float.
    static __device__ __forceinline__ uint32_t magnitude(uint32_t m) {
        if constexpr (sizeof(T) == 4) return m;
        const uint32_t h = max(m & 0xffffu, m >> 16);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return h << 16;
        else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    }
};

__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float m;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// kRound + the integers of 8 elements; the low bytes are the integers.
template <typename T>
__device__ __forceinline__ void quantize_eight(const Eight<T>& e, float scale, float inv, float half, bool normal,
                                               float (&t)[8]) {
    if (normal) {
        float worst = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            t[i] = fmaf(e[i], inv, kRound);
            t[i + 1] = fmaf(e[i + 1], inv, kRound);
            worst = max_abs(worst, fmaf(-(t[i] - kRound), scale, e[i]), fmaf(-(t[i + 1] - kRound), scale, e[i + 1]));
        }
        if (worst >= half) {
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = settle(t[i], e[i], scale, half);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = kRound + static_cast<float>(quantize_tiny(e[i], scale));
    }
}

// Sum over a warp of 64-bit words that wrap: 27, 27 and 10 bits at a time, whose
// sums over 32 lanes fit 32 bits.
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
    const uint32_t a = __reduce_add_sync(~0u, (uint32_t)v & 0x7ffffffu);
    const uint32_t b = __reduce_add_sync(~0u, (uint32_t)(v >> 27) & 0x7ffffffu);
    const uint32_t c = __reduce_add_sync(~0u, (uint32_t)(v >> 54));
    return a + ((unsigned long long)b << 27) + ((unsigned long long)c << 54);
}

// Dot product of 4 signed and 4 unsigned bytes, added to c.
__device__ __forceinline__ int dot_su(uint32_t a, int b, int c) {
    int d;
    asm("dp4a.s32.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                       __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}

// One row per group of ROW threads, U pieces of 8 elements per thread, held in
// registers; U = 0: any number of pieces, read twice. Groups walk the rows, the
// next one loading while this one is rounded. With CHECK the checksum lies in
// shared memory as its four bytes, the top one signed, four elements' in a word:
// 4 of the 8-bit dot product instructions take 4 integers' share of the expected
// sum (64-bit multiply-adds cost 3 instructions an element; 16384 rows of 4096
// bfloat16: 55 us with them, 45 us so, 35 us without a checksum).
template <typename T, int ROW, int U, bool CHECK>
__global__ void __launch_bounds__(ROW < 128 ? 128 : ROW, 1024 / (ROW < 128 ? 128 : ROW))
    k_quantize_rows(const QuantArgs a) {
    constexpr int kHeld = U > 0 ? U : 1;
    constexpr int kBlock = ROW < 128 ? 128 : ROW, kGroups = kBlock / ROW, kWarps = ROW / 32;
    __shared__ uint32_t smax[2][kWarps];
    __shared__ unsigned long long ssum[2][kWarps];
    const int me = threadIdx.x % ROW;
    const int pieces = (a.K + 7) / 8;
    const T* x_end = reinterpret_cast<const T*>(a.x) + (a.T - 1) * a.ldx + a.K;
    auto load = [&](Eight<T>& e, const T* row, int p) {
        const int left = a.K - p * 8;
        if (left >= 8) {
            if (a.aligned) e.load(row + p * 8);
            else e.load_any(row + p * 8, a.x, x_end);
        } else if (left > 0) {
            e.load(row + p * 8, left);
        } else {
            e.zero();
        }
    };
    auto checks = [&](int (&c)[8], int p) {
        if (a.aligned && p * 8 + 8 <= a.K) {
            const int4 lo = __ldg(reinterpret_cast<const int4*>(a.checksum + p * 8));
            const int4 hi = __ldg(reinterpret_cast<const int4*>(a.checksum + p * 8) + 1);
            c[0] = lo.x, c[1] = lo.y, c[2] = lo.z, c[3] = lo.w;
            c[4] = hi.x, c[5] = hi.y, c[6] = hi.z, c[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = p * 8 + i < a.K ? a.checksum[p * 8 + i] : 0;
        }
    };
    tensor::wait_for_stream();
    tensor::let_next_start();
    const int64_t first = (int64_t)blockIdx.x * kGroups + threadIdx.x / ROW, stride = (int64_t)gridDim.x * kGroups;
    constexpr bool kAhead = U > 0 && sizeof(T) == 2;  // 32-bit rows would not fit the registers twice
    Eight<T> e[kHeld], next[kAhead ? kHeld : 1];
    auto fetch = [&](Eight<T>* to, int64_t row) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) load(to[u], reinterpret_cast<const T*>(a.x) + row * a.ldx, me + u * ROW);
    };
    if constexpr (kAhead)
        if (first < a.T) fetch(next, first);
    extern __shared__ int4 bytes[];  // of all pieces' first halves, then of the second ones
    if constexpr (CHECK && U > 0) {
        auto transpose = [](const int* k) {
            const uint32_t l01 = __byte_perm(k[0], k[1], 0x5140), h01 = __byte_perm(k[0], k[1], 0x7362);
            const uint32_t l23 = __byte_perm(k[2], k[3], 0x5140), h23 = __byte_perm(k[2], k[3], 0x7362);
            return make_int4(__byte_perm(l01, l23, 0x5410), __byte_perm(l01, l23, 0x7632),
                             __byte_perm(h01, h23, 0x5410), __byte_perm(h01, h23, 0x7632));
        };
        for (int p = threadIdx.x; p < pieces; p += kBlock) {
            int k[8];
            checks(k, p);
            bytes[p] = transpose(k);
            bytes[pieces + p] = transpose(k + 4);
        }
        __syncthreads();
    }
    int flip = 0;
    int64_t last = -1;  // the row whose warps' sums lie in shared memory
    auto finish = [&](int f) {
        if (me != 0 || last < 0) return;
        unsigned long long sum = 0;
        for (int w = 0; w < kWarps; ++w) sum += ssum[f][w];
        a.expect[last] = (int64_t)sum;
    };
    for (int64_t row = first; row < a.T; row += stride, flip ^= 1) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
        int8_t* q = a.q + row * a.ldq;
        uint32_t m = 0;
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if constexpr (kAhead) e[u] = next[u];
            if constexpr (kAhead) {
                if (row + stride < a.T) fetch(next, row + stride);
            } else {
                fetch(e, row);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) m = e[u].largest(m);
        } else {
#pragma unroll 4
            for (int p = me; p < pieces; p += ROW) {
                Eight<T> v;
                load(v, x, p);
                m = v.largest(m);
            }
        }
        m = __reduce_max_sync(~0u, Eight<T>::magnitude(m));
        if constexpr (kWarps > 1) {
            if (threadIdx.x % 32 == 0) smax[flip][threadIdx.x / 32] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = max(m, smax[flip][w]);
            if constexpr (CHECK) finish(flip ^ 1);  // of the row before, by this row's barrier
        }
        const bool finite = m < 0x7f800000u;
        const float s = finite ? __fdiv_rn(__uint_as_float(m), 127.0f) : __uint_as_float(0x7fc00000u);
        const bool normal = s >= 0x1p-100f;
        const float inv = __fdiv_rn(1.0f, s), half = 0.5f * s;
        int dot[4] = {};              // below 2^31: at most 32 integers of 127 times 255
        unsigned long long sum = 0;   // U = 0: K is not bounded
        auto write = [&](const Eight<T>& v, int p) {
            const int left = a.K - p * 8;
            if (left <= 0) return;
            float t[8];
            quantize_eight(v, s, inv, half, normal, t);
            const uint32_t lo = low_bytes(t[0], t[1], t[2], t[3]), hi = low_bytes(t[4], t[5], t[6], t[7]);
            if (a.aligned && left >= 8) {
                *reinterpret_cast<uint2*>(q + p * 8) = make_uint2(lo, hi);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < left) q[p * 8 + i] = static_cast<int8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
            }
            if constexpr (CHECK && U > 0) {
                const int4 first = bytes[p], second = bytes[pieces + p];
                dot[0] = dot_su(lo, first.x, dot_su(hi, second.x, dot[0]));
                dot[1] = dot_su(lo, first.y, dot_su(hi, second.y, dot[1]));
                dot[2] = dot_su(lo, first.z, dot_su(hi, second.z, dot[2]));
                dot[3] = __dp4a((int)lo, first.w, __dp4a((int)hi, second.w, dot[3]));
            } else if constexpr (CHECK) {
                int k[8];
                checks(k, p);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sum += (unsigned long long)((long long)static_cast<int8_t>(__float_as_int(t[i])) * k[i]);
            }
        };
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; ++u) write(e[u], me + u * ROW);
        } else {
#pragma unroll 2
            for (int p = me; p < pieces; p += ROW) {
                load(e[0], x, p);
                write(e[0], p);
            }
        }
        if (me == 0) a.scale[row] = s;
        if constexpr (CHECK) {
            if constexpr (U > 0) {
                for (int i = 3; i >= 0; --i)
                    sum = sum * 256 + (unsigned long long)(long long)__reduce_add_sync(~0u, dot[i]);
            } else {
                sum = warp_sum(sum);
            }
            if constexpr (kWarps > 1) {
                if (threadIdx.x % 32 == 0) ssum[flip][threadIdx.x / 32] = sum;
                last = row;
            } else if (me == 0) {
                a.expect[row] = (int64_t)sum;
            }
        }
    }
    if constexpr (CHECK && kWarps > 1) {
        __syncthreads();
        finish(flip ^ 1);
    }
}

// Column sums of an 8-bit weight: blocks of `rows` rows, their sums added as
// integers (the order does not matter). WIDE: 4 columns per load. A weight's checksum
// is taken once, when it is loaded; launched plainly, behind the memset of its sums.
// Bound by reading w where it is wide (131072 x 8192: 203 us, 81 % of the copy rate),
// else by a block's loads one after the other. Rows a block: 256 are best or as good
// for large weights (131072 x 8192: 240 us with 64, 201 with 128, 203 with 256, 210 with
// 1024; 8192 x 28672: 55 / 55 / 57 / 158); small ones would take fewer (4096 x 4096: 19
// / 25 / 43 / 154).
template <bool WIDE>
__global__ void __launch_bounds__(256) k_column_checksum(const int8_t* __restrict__ w, int64_t ldw, int N, int K,
                                                         int rows, int32_t* __restrict__ checksum) {
    constexpr int kC = WIDE ? 4 : 1;
    const int64_t k = ((int64_t)blockIdx.x * 256 + threadIdx.x) * kC;
    if (k >= K) return;
    const int first = (int)blockIdx.y * rows, last = min(N, first + rows);
    int sum[kC] = {};
    if (WIDE && k + kC <= K) {
#pragma unroll 8
        for (int n = first; n < last; ++n) {
            const int v = __ldg(reinterpret_cast<const int*>(w + n * ldw + k));
#pragma unroll
            for (int i = 0; i < kC; ++i) sum[i] += static_cast<int8_t>(v >> (8 * i));
        }
    } else {
        for (int n = first; n < last; ++n)
#pragma unroll
            for (int i = 0; i < kC; ++i)
                if (k + i < K) sum[i] += w[n * ldw + k + i];
    }
#pragma unroll
    for (int i = 0; i < kC; ++i)
        if (k + i < K) atomicAdd(checksum + k + i, sum[i]);
}

// ---------------------------------------------------------------- products ---
//
// One persistent kernel for all products, D = A B^T in tiles of 128 CG rows x
// BN columns of sums, on the tcgen05 tensor cores:
//
//   kInt8   q w^T, scaled                      A: q [T, K]       B: w [N, K]
//   kGate   act(x Wg^T) * (x Wu^T)             A: x [T, K]       B: Wg | Wu, BN / 2 rows each
//   kDx     dg Wg + du Wu                      A: dg, du [T, N]  B: Wg, Wu read along their rows (MN-major)
//   kDw     dg^T x and du^T x                  A: dg or du       B: x, both MN-major
//
// Warp 0 copies operand tiles to shared memory (TMA, 128-byte swizzle), one
// thread of warp 1 issues the matrix instructions, warps 4-11 take finished
// sums out of tensor memory; sums are double-buffered there, so the next
// tile's products run while this one is written. With CG = 2 two CTAs (two
// SMs) form one 256-row tile: each holds its 128 rows of A and half of B, and
// the matrix instruction of the leader reads both halves, which halves the
// copies of B per product.
//
// Finished sums go through a small piece of shared memory, so that a warp
// writes whole 64- or 128-byte runs of each output row, aligned or not.
//
// SPLIT: when there are too few tiles for the GPU, the CTAs of a cluster share
// one tile's K. Each sends its partial sums of a row to the CTA that writes that
// row (stores over the cluster; reading them there instead took 2 us more), which
// adds them up in a fixed order.
//
// Nothing is transposed in memory: an operand whose summed index runs along
// the pitch is MN-major, which the matrix instructions read directly. Rows and
// columns beyond a matrix are filled with zeros by the copies, so ragged sizes
// take the same path; sums along K of zeros change nothing.

enum { kInt8, kGate, kDx, kDw };

struct ProductArgs {
    int rows, cols;              // of one output
    int tiles_m, tiles_n;        // kDw: tiles_m counts both outputs' tiles
    int tiles_m1;                // of the first output
    int chunks;                  // of 128 bytes along K, one operand pair
    int split;                   // CTAs that share a tile's K
    int limit;                   // polls of a wait
    void* c[3];                  // outputs; kGate: h, g, u; kDw: dWg, dWu
    int64_t ld[3];
    bool wide[3];                // 16-byte stores are possible
    const float* row_scale;
    const float* col_scale;
    unsigned long long* rowdiff;  // holds minus what is expected
};

struct ProductMaps {
    CUtensorMap a[2], b[2];
};

// Waits that ran out in any product kernel of the device. It only grows: each host
// thread compares it with what it was told last, so none takes a fault from another.
__device__ unsigned g_faults;

constexpr int kProductThreads = 384;  // copies, matrix instructions, 2 idle warps (one holds tensor memory), 8 for results

template <int MODE, int CG, int BN, bool SPLIT, typename O>
struct Shape {
    static constexpr bool kTwoPairs = MODE == kDx;
    static constexpr bool kAMn = MODE == kDw;
    static constexpr bool kBMn = MODE == kDx || MODE == kDw;
    static constexpr int kCols = MODE == kGate ? BN / 2 : BN;  // of an output
    static constexpr int kABytes = 128 * 128, kBBytes = BN / CG * 128;  // of a stage, per CTA
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kOutBytes = 32 * (32 * (int)sizeof(O) + 16);  // 32 x 32 results on their way out, one warp
    // 227 KB of shared memory: alignment, barriers, 8 warps' results and channel scales; the rest are stages
    static constexpr int kOutRoom = SPLIT ? 0 : 8 * kOutBytes;
    static constexpr int kRoom = 227 * 1024 - 1024 - 512 - kOutRoom - 8 * 128 * 4;
    // SPLIT: pitch of partial sums, which overlay the stages (128 rows and at most 8 more, see share_rows)
    static constexpr int kPart = BN + 4;
    static constexpr int kStages = kRoom / kStageBytes < 8 ? kRoom / kStageBytes : 8;
    static constexpr int kOut = kStages * kStageBytes;
    static constexpr int kScales = kOut + kOutRoom;
    static constexpr int kBars = kScales + 8 * 128 * 4;
    static constexpr int kSmem = 1024 + kBars + 512;
    static constexpr int kTmemCols = 2 * BN;
};

// sum * row * column in this order: three roundings in 32 bits, 3.6e-8 of a float32
// result where one rounding of the 64-bit product leaves 2.5e-8, which would cost each
// result two conversions. Only sum * row could overflow where the result does not: a
// row's scale from 2^64 on is used 2^32 times smaller, which keeps that product (sum <
// 2^31) below 2^127 and above 2^32, and the result is taken back by 2^32 (the factor is
// 1 for others; 777 x 1531 x 1001: 8.4 us with it and without). The other end needs
// nothing: a whole number times a subnormal scale is rounded only to 24 bits.
struct RowScale {
    float scale, back;

    explicit __device__ __forceinline__ RowScale(float s)
        : scale(fabsf(s) >= 0x1p64f ? s * 0x1p-32f : s), back(fabsf(s) >= 0x1p64f ? 0x1p32f : 1.0f) {}
    __device__ __forceinline__ float times(int sum, float column) const {
        return static_cast<float>(sum) * scale * column * back;
    }
};

// SPLIT: rows of the largest share of a tile, at most.
__device__ __forceinline__ int share_rows(int split) { return 128 / split + (128 % split != 0); }

// A wait with a limit. `stop` is set for the whole CTA by the first that runs out.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, int limit, volatile int* stop) {
    for (int i = 0; i < limit; ++i) {
        if (tensor::bar_test(bar, parity)) return true;
        if ((i & 63) == 63 && *stop) return false;
    }
    if (!*stop) {
        *stop = 1;
        atomicAdd(&g_faults, 1u);
    }
    return false;
}

// Tile order: groups of 16 tile rows, columns inside a group, so that the CTAs
// at work at one time read few operand rows (L2 hits). 8192 x 16384 x 4096 block:
// 1477 us with groups of 8, 1469 of 16, 1481 of 24; 8-bit product of 16384 x 16384 x
// 4096: 732 / 717 / 717 (all three sides in runs of the same length; that product now
// takes 690 us in runs of 20 after a pause and 780 once the power cap has settled). The gradients sum over a long axis, along which all CTAs
// move together and nothing stays in L2, so there the two operands' shares should
// be alike: 3455 us with groups of 4, 3385 of 6, 3484 of 8, 3470 of 16.
template <int MODE>
__device__ __forceinline__ void tile_at(int i, int tiles_m, int tiles_n, int& m, int& n) {
    constexpr int kRows = MODE == kDx || MODE == kDw ? 6 : 16;
    const int group = kRows * tiles_n;
    const int g = i / group, r = i - g * group;
    const int h = min(kRows, tiles_m - g * kRows);
    n = r / h;
    m = g * kRows + r - n * h;
}

// A warp's 32 x 32 values (one row per lane) to a matrix at `to`, of which
// `rows` rows and `cols` columns exist; `wide`: 16-byte stores are possible.
template <typename O>
__device__ __forceinline__ void store_block(char* mine, O* to, int64_t ld, int rows, int cols, bool wide,
                                            const float (&v)[32]) {
    constexpr int kV = 16 / sizeof(O), kPieces = 32 / kV, kPitch = 32 * sizeof(O) + 16;
    const int lane = threadIdx.x % 32;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
        alignas(16) O pack[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) pack[i] = from_f32<O>(v[j * kV + i]);
        *reinterpret_cast<uint4*>(mine + lane * kPitch + j * 16) = *reinterpret_cast<uint4*>(pack);
    }
    __syncwarp();
    if (wide && cols >= 32) {
        const int r = lane / kPieces, piece = lane % kPieces;
        uint4 out[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            out[i] = *reinterpret_cast<const uint4*>(mine + (i * (32 / kPieces) + r) * kPitch + piece * 16);
        to += r * ld + piece * kV;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            if (i * (32 / kPieces) + r < rows) *reinterpret_cast<uint4*>(to + i * (32 / kPieces) * ld) = out[i];
    } else if (lane < cols) {
        to += lane;
        const char* from = mine + lane * sizeof(O);
#pragma unroll 1
        for (int i = 0; i < 32 && i < rows; i += 4) {
            O out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = *reinterpret_cast<const O*>(from + j * kPitch);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i + j < rows) *to = out[j];
                to += ld;
            }
            from += 4 * kPitch;
        }
    }
}

template <int MODE, int CG, int BN, bool SPLIT, typename O, int ACT>
__global__ void __launch_bounds__(kProductThreads, 1)
    k_product(const __grid_constant__ ProductMaps maps, const ProductArgs a) {
    using S = Shape<MODE, CG, BN, SPLIT, O>;
    static_assert(!SPLIT || (128 + 8) * S::kPart * 4 <= S::kOut, "the partial sums fit the stages");
    static_assert(!SPLIT || CG == 1, "a split tile is one CTA wide");
    extern __shared__ char raw[];
    char* smem = raw + (-tensor::smem_u32(raw) & 1023);
    const uint32_t base = tensor::smem_u32(smem);
    const uint32_t bars = base + S::kBars;
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (S::kStages + s); };
    auto sums_full = [&](int s) { return bars + 8 * (2 * S::kStages + s); };
    auto sums_empty = [&](int s) { return bars + 8 * (2 * S::kStages + 2 + s); };
    const uint32_t drained = bars + 8 * (2 * S::kStages + 4);
    volatile int* stop = reinterpret_cast<volatile int*>(smem + S::kBars + 8 * (2 * S::kStages + 5));
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(const_cast<int*>(stop) + 1);

    // the same in all lanes, and known to be
    const int warp = __shfl_sync(~0u, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t in_cluster = CG == 2 || SPLIT ? tensor::cluster_rank() : 0;
    const uint32_t rank = SPLIT ? 0 : in_cluster;  // in the pair
    const int tiles = a.tiles_m * a.tiles_n;
    const int first = SPLIT ? blockIdx.x / a.split : blockIdx.x / CG, step = SPLIT ? tiles : gridDim.x / CG;
    const int all = S::kTwoPairs ? 2 * a.chunks : a.chunks;
    // this CTA's part of K
    const int begin = SPLIT ? (int)((int64_t)all * in_cluster / a.split) : 0;
    const int end = SPLIT ? (int)((int64_t)all * (in_cluster + 1) / a.split) : all;
    constexpr int kElems = MODE == kInt8 ? 128 : 64;  // of 128 bytes along K

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            tensor::bar_init(full(s), 1);
            tensor::bar_init(empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            tensor::bar_init(sums_full(s), 1);
            tensor::bar_init(sums_empty(s), 8 * CG);
        }
        tensor::bar_init(drained, 1);
        *stop = 0;
        tensor::bar_init_fence();
    }
    if constexpr (CG == 2) {  // tensor memory of a pair is taken, and given back, only while both CTAs run
        __syncwarp();
        tensor::cluster_arrive_relaxed();
        tensor::cluster_wait();
    }
    if (warp == 2) tensor::tmem_alloc<CG>(tensor::smem_u32(const_cast<uint32_t*>(tmem_slot)), S::kTmemCols);
    tensor::tc_fence_before();
    __syncwarp();
    if constexpr (CG == 2) tensor::cluster_sync();
    else __syncthreads();
    if (SPLIT && warp < 4) tensor::cluster_arrive_relaxed();
    tensor::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    tensor::wait_for_stream();
    tensor::let_next_start();

    // The stages go round: `s` is the stage, `turn` the parity of its round. Both
    // loops below run in one elected thread and keep every address in a counter:
    // with divisions by the number of stages, and a vote of the warp per wait,
    // their own instructions took 0.21 us a chunk.
    if (warp == 0 && tensor::elect()) {
        // ------------------------------------------------ copies ---
        for (int i = 0; i < 2; ++i) {
            tensor::prefetch_map(&maps.a[i]);
            tensor::prefetch_map(&maps.b[i]);
        }
        const uint32_t done0 = CG == 2 ? tensor::in_leader(full(0)) : full(0);
        int s = 0, issued = 0;
        uint32_t turn = 0;
        bool ok = true;
        for (int tile = first; ok && tile < tiles; tile += step) {
            int mt, nt;
            tile_at<MODE>(tile, a.tiles_m, a.tiles_n, mt, nt);
            int pair = 0;
            if (MODE == kDw && mt >= a.tiles_m1) {
                mt -= a.tiles_m1;
                pair = 1;
            }
            const int m0 = (mt * CG + (int)rank) * 128;
            const int n0 = nt * S::kCols;
            for (int c = begin; c < end; ++c) {
                if (!wait_for(empty(s), turn ^ 1, a.limit, stop)) {
                    ok = false;
                    break;
                }
                if (rank == 0) tensor::bar_expect(full(s), CG * S::kStageBytes);
                const uint32_t done = done0 + 8 * s;
                const uint32_t sa = base + s * S::kStageBytes;
                int k = c;
                if constexpr (S::kTwoPairs) {
                    pair = c >= a.chunks;
                    k = pair ? c - a.chunks : c;
                }
                const CUtensorMap* am = &maps.a[pair];
                if constexpr (S::kAMn) {
                    tensor::tma_load<CG>(sa, am, m0, k * 64, done);
                    tensor::tma_load<CG>(sa + 8192, am, m0 + 64, k * 64, done);
                } else {
                    tensor::tma_load<CG>(sa, am, k * kElems, m0, done);
                }
                const uint32_t sb = sa + S::kABytes;
                if constexpr (S::kBMn) {
                    const CUtensorMap* bm = MODE == kDx ? &maps.b[pair] : &maps.b[0];
#pragma unroll
                    for (int j = 0; j < BN / CG / 64; ++j)
                        tensor::tma_load<CG>(sb + j * 8192, bm, n0 + (int)rank * (BN / CG) + j * 64, k * 64, done);
                } else if constexpr (MODE == kGate && CG == 2) {
                    tensor::tma_load<CG>(sb, &maps.b[rank], k * kElems, n0, done);
                } else if constexpr (MODE == kGate) {
                    tensor::tma_load<CG>(sb, &maps.b[0], k * kElems, n0, done);
                    tensor::tma_load<CG>(sb + S::kBBytes / 2, &maps.b[1], k * kElems, n0, done);
                } else {
                    tensor::tma_load<CG>(sb, &maps.b[0], k * kElems, n0 + (int)rank * (BN / CG), done);
                }
                issued = min(issued + 1, S::kStages);
                if (++s == S::kStages) {
                    s = 0;
                    turn ^= 1;
                }
            }
        }
        // The CTA stays until its last stages are read (the pair's leader signals both CTAs).
        auto last = [&](auto&& wait) {
            for (int j = 0, t = s, r = turn; j < issued; ++j) {
                if (--t < 0) {
                    t = S::kStages - 1;
                    r ^= 1;
                }
                wait(t, r);
            }
        };
        last([&](int t, int r) { ok = ok && wait_for(empty(t), r, a.limit, stop); });
        if (!ok) {  // after a wait that ran out the copies in flight land first
            if (rank == 0)
                last([&](int t, int r) {
                    for (int i = 0; i < kWaitLimit && !tensor::bar_test(full(t), r); ++i) {
                    }
                });
            else
                for (int i = 0; i < 1000 && issued > 0; ++i) __nanosleep(1000);
        }
    } else if (warp == 1 && tensor::elect()) {
        // ------------------------------------- matrix instructions ---
        constexpr uint32_t idesc = tensor::instruction(128 * CG, BN, MODE == kInt8, std::is_same<O, __nv_bfloat16>::value,
                                                       S::kAMn, S::kBMn);
        constexpr uint32_t a_step = S::kAMn ? 2048 >> 4 : 32 >> 4, b_step = S::kBMn ? 2048 >> 4 : 32 >> 4;
        const uint64_t a0 = tensor::operand(base, S::kAMn), b0 = tensor::operand(base + S::kABytes, S::kBMn);
        int s = 0, n = 0;
        uint32_t turn = 0;
        bool ok = true;
        for (int tile = first; rank == 0 && ok && tile < tiles; tile += step, ++n) {
            ok = wait_for(sums_empty(n & 1), ((n >> 1) + 1) & 1, a.limit, stop);
            const uint32_t d = tmem + (n & 1) * BN;
            for (int c = begin; ok && c < end; ++c) {
                ok = wait_for(full(s), turn, a.limit, stop);
                if (!ok) break;
                tensor::tc_fence_after();
                const uint64_t da = a0 + s * (S::kStageBytes >> 4), db = b0 + s * (S::kStageBytes >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    tensor::mma<CG, MODE == kInt8>(d, da + k * a_step, db + k * b_step, idesc, c > begin || k > 0);
                tensor::mma_commit<CG>(empty(s));
                if (++s == S::kStages) {
                    s = 0;
                    turn ^= 1;
                }
            }
            if (ok) tensor::mma_commit<CG>(sums_full(n & 1));
        }
        // instructions in flight still read shared and write tensor memory, in both CTAs of a pair
        if (rank == 0) tensor::mma_commit<CG>(drained);
        // (CTA 1 waits here from its start on: up to about a minute of kernel, unless a wait has run out)
        for (int i = 0; !tensor::bar_test(drained, 0) && (i < kWaitLimit || (i < 64 * kWaitLimit && !*stop)); ++i) {
        }
        // The other CTA's arrivals for the last sums travel behind its stores to global memory; they have to land before
        // this CTA goes, since the barrier at the end does not wait for them.
        for (int j = max(0, n - 2); CG == 2 && rank == 0 && ok && j < n; ++j)
            ok = wait_for(sums_empty(j & 1), (j >> 1) & 1, a.limit, stop);
    } else if (warp >= 4) {
        // -------------------------------------------------- results ---
        // warps w and w + 4 take the same 32 rows, each half of the columns
        const int w = warp % 4, half = warp / 8;
        constexpr int kBlocks = (SPLIT ? BN : S::kCols) / 32;
        const int j0 = half ? (kBlocks + 1) / 2 * 32 : 0, j1 = half ? kBlocks * 32 : (kBlocks + 1) / 2 * 32;
        const uint32_t lanes = tmem + ((uint32_t)w << 21);
        char* mine = smem + S::kOut + (warp - 4) * S::kOutBytes;
        // SPLIT: this lane's row belongs to CTA `owner`, from whose first row on it is row `in_share`
        const int owner = SPLIT ? ((w * 32 + lane + 1) * a.split - 1) / 128 : 0;
        const int in_share = w * 32 + lane - (SPLIT ? 128 * owner / a.split : 0);
        uint32_t part = 0;
        if constexpr (SPLIT)
            part = tensor::in_cta(base + ((int)in_cluster * share_rows(a.split) + in_share) * S::kPart * 4, owner);
        float* sc = reinterpret_cast<float*>(smem + S::kScales) + (warp - 4) * 128;
        int n = 0;
        for (int tile = first; tile < tiles; tile += step, ++n) {
            const int buf = n & 1;
            int mt, nt;
            tile_at<MODE>(tile, a.tiles_m, a.tiles_n, mt, nt);
            int out = 0;
            if (MODE == kDw && mt >= a.tiles_m1) {
                mt -= a.tiles_m1;
                out = 1;
            }
            const int m0 = (mt * CG + (int)rank) * 128 + w * 32;  // the warp's first row
            const int rows = a.rows - m0;
            const int n0 = nt * S::kCols;
            long long total = 0;
            RowScale rs(0.0f);
            if constexpr (MODE == kInt8 && !SPLIT) {
                if (lane < rows) rs = RowScale(a.row_scale[m0 + lane]);
                __syncwarp();
                for (int j = j0 + lane; j < j1; j += 32) sc[j - j0] = n0 + j < a.cols ? a.col_scale[n0 + j] : 0.0f;
                __syncwarp();
            }
            const bool ok = __all_sync(~0u, wait_for(sums_full(buf), (n >> 1) & 1, a.limit, stop));
            if constexpr (SPLIT) {  // no CTA's instructions read their stages any more
                tensor::cluster_arrive_relaxed();
                tensor::cluster_wait();
            }
            if (!ok) break;
            tensor::tc_fence_after();
            auto put = [&](int i, int j, const float(&v)[32]) {
                const int64_t ld = i == 0 ? a.ld[0] : i == 1 ? a.ld[1] : a.ld[2];
                void* c = i == 0 ? a.c[0] : i == 1 ? a.c[1] : a.c[2];
                const bool wide = i == 0 ? a.wide[0] : i == 1 ? a.wide[1] : a.wide[2];
                store_block<O>(mine, reinterpret_cast<O*>(c) + m0 * ld + n0 + j, ld, rows, a.cols - n0 - j, wide, v);
            };
            auto taken = [&] {  // the sums are out: the next tile may overwrite them
                tensor::tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    tensor::bar_arrive(CG == 2 ? tensor::in_leader(sums_empty(buf)) : sums_empty(buf));
            };
            if (!SPLIT && j0 == j1) taken();
#pragma unroll 1
            for (int j = j0; j < j1; j += 32) {
                uint32_t r[32], r2[32];
                __syncwarp();
                tensor::tmem_load32(lanes + buf * BN + j, r);
                if constexpr (MODE == kGate && !SPLIT) tensor::tmem_load32(lanes + buf * BN + S::kCols + j, r2);
                tensor::tmem_wait_load(r);
                if constexpr (MODE == kGate && !SPLIT) tensor::after_wait(r2);
                if (!SPLIT && j + 32 == j1) taken();
                float v[32];
                if constexpr (SPLIT) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        tensor::store_cluster(part + (j + i) * 4, r[i], r[i + 1], r[i + 2], r[i + 3]);
                } else if constexpr (MODE == kInt8) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 cs = *reinterpret_cast<const float4*>(sc + j - j0 + i);
                        const float scale[4] = {cs.x, cs.y, cs.z, cs.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int sum = static_cast<int>(r[i + k]);
                            total += sum;
                            v[i + k] = rs.times(sum, scale[k]);
                        }
                    }
                    put(0, j, v);
                } else if constexpr (MODE == kGate) {
                    float up[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        v[i] = __uint_as_float(r[i]);
                        up[i] = __uint_as_float(r2[i]);
                    }
                    if (a.c[1]) {
                        put(1, j, v);
                        put(2, j, up);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = act<ACT>(v[i]) * up[i];
                    put(0, j, v);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
                    put(out, j, v);
                }
            }
            // sums of columns and rows beyond the matrices are zeros
            if (MODE == kInt8 && !SPLIT && lane < rows && a.rowdiff)
                atomicAdd(a.rowdiff + m0 + lane, static_cast<unsigned long long>(total));
        }
    }
    __syncwarp();
    tensor::tc_fence_before();
    if constexpr (SPLIT) {
        if (warp < 4) tensor::cluster_wait();
        tensor::cluster_sync();  // the partial sums are there
    } else if constexpr (CG == 2) {
        // The leader's instructions use both CTAs' memory. All that one CTA sends the other has landed before the receiver
        // arrives here (its threads waited for it), so nobody waits for the stores to global memory.
        tensor::cluster_arrive_relaxed();
        tensor::cluster_wait();
    } else {
        __syncthreads();
    }
    tensor::tc_fence_after();
    if (warp == 2) tensor::tmem_free<CG>(tmem, S::kTmemCols);
    if constexpr (CG == 2) {
        tensor::cluster_arrive_relaxed();
        tensor::cluster_wait();
    }

    if constexpr (SPLIT) {
        // every CTA adds up its share of the tile's rows: a thread takes 4 columns of a row
        int mt, nt;
        tile_at<MODE>(first, a.tiles_m, a.tiles_n, mt, nt);
        int out = 0;
        if (MODE == kDw && mt >= a.tiles_m1) {
            mt -= a.tiles_m1;
            out = 1;
        }
        constexpr int kFours = S::kCols / 4;  // threads of a row, 32 at most
        const int n0 = nt * S::kCols;
        const int r0 = 128 * (int)in_cluster / a.split, r1 = 128 * ((int)in_cluster + 1) / a.split;
        const int rows = share_rows(a.split);
        auto sum = [&](int r, int c, auto(&v)[4]) {
            const char* at = smem + ((r - r0) * S::kPart + c) * 4;
#pragma unroll 4
            for (int p = 0; p < a.split; ++p) {
                const uint4 q = *reinterpret_cast<const uint4*>(at + p * rows * S::kPart * 4);
                if constexpr (MODE == kInt8) {
                    v[0] += (int)q.x, v[1] += (int)q.y, v[2] += (int)q.z, v[3] += (int)q.w;
                } else {
                    v[0] += __uint_as_float(q.x), v[1] += __uint_as_float(q.y);
                    v[2] += __uint_as_float(q.z), v[3] += __uint_as_float(q.w);
                }
            }
        };
        auto put = [&](int i, int64_t m, int c, const float(&v)[4]) {
            const int64_t ld = i == 0 ? a.ld[0] : i == 1 ? a.ld[1] : a.ld[2];
            void* all = i == 0 ? a.c[0] : i == 1 ? a.c[1] : a.c[2];
            const bool wide = i == 0 ? a.wide[0] : i == 1 ? a.wide[1] : a.wide[2];
            O* to = reinterpret_cast<O*>(all) + m * ld + n0 + c;
            if (wide && n0 + c + 4 <= a.cols) {
                alignas(16) O pack[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) pack[j] = from_f32<O>(v[j]);
                if constexpr (sizeof(O) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(pack);
                else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(pack);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n0 + c + j < a.cols) to[j] = from_f32<O>(v[j]);
            }
        };
        // whole warps go round together, the last with rows of the next share that it leaves alone
        for (int e = threadIdx.x; e < ((r1 - r0) * kFours + 31) / 32 * 32; e += kProductThreads) {
            const int r = min(r0 + e / kFours, r1 - 1), c = e % kFours * 4;
            const int64_t m = mt * 128 + r;
            const bool live = r0 + e / kFours < r1 && m < a.rows;
            if constexpr (MODE == kInt8) {
                int v[4] = {};
                sum(r, c, v);
                float y[4];
                const RowScale rs(live ? a.row_scale[m] : 0.0f);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = rs.times(v[i], n0 + c + i < a.cols ? a.col_scale[n0 + c + i] : 0.0f);
                if (live) put(0, m, c, y);
                if (a.rowdiff) {
                    long long total = (long long)v[0] + v[1] + v[2] + v[3];
#pragma unroll
                    for (int o = kFours / 2; o; o >>= 1) total += __shfl_down_sync(~0u, total, o, kFours);
                    if (c == 0 && live) atomicAdd(a.rowdiff + m, static_cast<unsigned long long>(total));
                }
            } else if constexpr (MODE == kGate) {
                float g[4] = {}, up[4] = {};
                sum(r, c, g);
                sum(r, c + S::kCols, up);
                if (live) {
                    if (a.c[1]) {
                        put(1, m, c, g);
                        put(2, m, c, up);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) g[i] = act<ACT>(g[i]) * up[i];
                    put(0, m, c, g);
                }
            } else {
                float v[4] = {};
                sum(r, c, v);
                if (live) put(out, m, c, v);
            }
        }
    }
}

// ------------------------------------------------------------ few tokens ---
//
// Products of few tokens are bound by reading the weight once. The
// 128-row tiles of the kernel above would leave most SMs without a tile and the
// rest waiting on few copies, so here a group of WK warps takes 16 weight rows
// (kGate: 8 of either weight) and shares their K: a warp reads runs of 64 bytes
// of 16 rows with 16-byte loads straight into the registers of the 16 x 8
// matrix instruction (weights are its 16 rows, tokens its 8 columns). The sum
// over K does not depend on the order of K, so lane t of a quad simply takes
// the quad's t-th 16 bytes of a row, and of a token, as its part of K. Tokens
// are re-read from L1. The warps' sums meet in shared memory, in a fixed order.

template <bool INT8, typename E>
__device__ __forceinline__ void few_mma(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
#define ABFT_FEW(shape, types)                                                                                  \
    asm volatile("mma.sync.aligned." shape ".row.col." types " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, " \
                 "{%0, %1, %2, %3};"                                                                            \
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])                                               \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if constexpr (INT8) ABFT_FEW("m16n8k32", "s32.s8.s8.s32");
    else if constexpr (std::is_same<E, __half>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        ABFT_FEW("m16n8k16", "f32.bf16.bf16.f32");
    }
#undef ABFT_FEW
}

struct FewArgs {
    const char* w[2];  // kGate: both weights; else the weight in w[0]
    int64_t ldw[2];    // bytes
    const char* x;
    int64_t ldx;       // bytes
    int T, N;
    int64_t kbytes;
    void* c[3];
    int64_t ld[3];
    const float* row_scale;
    const float* col_scale;
    unsigned long long* rowdiff;
};

// 16 bytes at byte `off` of a row of `n` bytes, zeros beyond it; weights pass L1 by.
template <bool STREAM>
__device__ __forceinline__ uint4 few_load(const char* row, int64_t off) {
    uint4 v;
    if constexpr (STREAM)
        asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(row + off));
    else
        v = __ldg(reinterpret_cast<const uint4*>(row + off));
    return v;
}

template <typename E>
__device__ __forceinline__ uint4 few_load_edge(const char* row, int64_t off, int64_t n) {
    if (off + 16 <= n) return __ldg(reinterpret_cast<const uint4*>(row + off));
    alignas(16) E e[16 / sizeof(E)] = {};
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(E); ++i)
        if (off + (i + 1) * (int)sizeof(E) <= n) e[i] = reinterpret_cast<const E*>(row + off)[i];
    return *reinterpret_cast<uint4*>(e);
}

template <bool GATE, typename E, int NT, int WK, typename O, int ACT>
__global__ void __launch_bounds__(256, 2) k_few(const FewArgs a) {
    constexpr bool kInt = sizeof(E) == 1;
    constexpr int kRows = GATE ? 8 : 16;   // weight rows (channels) of a group of WK warps
    constexpr int kU = NT == 4 ? 4 : 8;    // 64-byte pieces of K in flight per warp
    __shared__ uint32_t part[8][4 * NT][32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n0 = (blockIdx.x * (8 / WK) + warp / WK) * kRows;
    // rows and tokens beyond the last read the last one; their sums are not used
    const char* r0 = a.w[0] + (int64_t)min(n0 + g, a.N - 1) * a.ldw[0] + t * 16;
    const char* r1 = GATE ? a.w[1] + (int64_t)min(n0 + g, a.N - 1) * a.ldw[1] + t * 16
                          : a.w[0] + (int64_t)min(n0 + g + 8, a.N - 1) * a.ldw[0] + t * 16;
    const char* xr[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) xr[j] = a.x + (int64_t)min(j * 8 + g, a.T - 1) * a.ldx + t * 16;
    uint32_t c[NT][4] = {};
    auto multiply = [&](const uint4& w0, const uint4& w1, const uint4 (&x)[NT]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            few_mma<kInt, E>(c[j], w0.x, w1.x, w0.y, w1.y, x[j].x, x[j].y);
            few_mma<kInt, E>(c[j], w0.z, w1.z, w0.w, w1.w, x[j].z, x[j].w);
        }
    };
    tensor::wait_for_stream();
    tensor::let_next_start();
    int64_t k = (int64_t)(warp % WK) * kU * 64;
    for (; k + kU * 64 <= a.kbytes; k += WK * kU * 64) {
        uint4 w0[kU], w1[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            w0[u] = few_load<true>(r0, k + u * 64);
            w1[u] = few_load<true>(r1, k + u * 64);
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            uint4 x[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) x[j] = few_load<false>(xr[j], k + u * 64);
            multiply(w0[u], w1[u], x);
        }
    }
    for (; k < a.kbytes; k += 64) {  // the pieces of the run that ends inside: one warp of the group, once
        const int64_t left = a.kbytes - t * 16;
        const uint4 w0 = few_load_edge<E>(r0, k, left), w1 = few_load_edge<E>(r1, k, left);
        uint4 x[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j] = few_load_edge<E>(xr[j], k, left);
        multiply(w0, w1, x);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[warp][j * 4 + i][lane] = c[j][i];
    __syncthreads();
    // element (token, channel pair): c[0..1] of a quad are tokens 2 t, 2 t + 1 of row g, c[2..3] those of row g + 8
    for (int e = threadIdx.x; e < 64 * NT * (8 / WK); e += 256) {
        const int ch = e % 8, tok = e / 8 % (8 * NT), first = e / (64 * NT) * WK;
        const int from = ch * 4 + tok % 8 / 2, i = tok / 8 * 4 + tok % 2;
        const int n = (blockIdx.x * (8 / WK) + first / WK) * kRows + ch;
        if constexpr (kInt) {
            int s0 = 0, s1 = 0;
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                s0 += static_cast<int>(part[first + w][i][from]);
                s1 += static_cast<int>(part[first + w][i + 2][from]);
            }
            const bool in0 = tok < a.T && n < a.N, in1 = tok < a.T && n + 8 < a.N;
            const RowScale rs(tok < a.T ? a.row_scale[tok] : 0.0f);
            O* row = reinterpret_cast<O*>(a.c[0]) + tok * a.ld[0];
            if (in0) row[n] = from_f32<O>(rs.times(s0, a.col_scale[n]));
            if (in1) row[n + 8] = from_f32<O>(rs.times(s1, a.col_scale[n + 8]));
            if (a.rowdiff) {
                long long sum = (in0 ? (long long)s0 : 0) + (in1 ? (long long)s1 : 0);
                for (int o = 4; o; o >>= 1) sum += __shfl_down_sync(~0u, sum, o, 8);
                if (ch == 0 && tok < a.T) atomicAdd(a.rowdiff + tok, static_cast<unsigned long long>(sum));
            }
        } else {
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                gate += __uint_as_float(part[first + w][i][from]);
                up += __uint_as_float(part[first + w][i + 2][from]);
            }
            if (tok < a.T && n < a.N) {
                reinterpret_cast<O*>(a.c[0])[tok * a.ld[0] + n] = from_f32<O>(act<ACT>(gate) * up);
                if (a.c[1]) {
                    reinterpret_cast<O*>(a.c[1])[tok * a.ld[1] + n] = from_f32<O>(gate);
                    reinterpret_cast<O*>(a.c[2])[tok * a.ld[2] + n] = from_f32<O>(up);
                }
            }
        }
    }
}

// What the rows' sums are added to. A kernel that starts beside the one before it
// rather than a memset, which would end that: one quantised and verified token,
// 16384 x 4096, replayed from a graph on one weight: 12.4 us, 3.2 us less than with the
// memset (called eagerly, where the host's 27 us are the bound, the memset saves 1.5 us).
__global__ void __launch_bounds__(256) k_negate(const int64_t* __restrict__ in, int64_t* __restrict__ out, int n) {
    tensor::wait_for_stream();
    tensor::let_next_start();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = -in[i];
}

// Rows of up to three matrices onto another pitch, 16 bytes a thread.
struct PackArgs {
    const char* in[3];
    char* out[3];
    int64_t ld[3];       // bytes
    int64_t row[3];      // bytes of a row
    int64_t chunks[3];   // of 16 bytes of a row
    int64_t pitch[3];    // bytes of a row's copy
    int64_t end[3];      // chunks of this matrix and those before it
    int rows[3];
};

template <typename T>
__global__ void __launch_bounds__(256) k_pack(const PackArgs a) {
    tensor::wait_for_stream();
    tensor::let_next_start();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.end[2]; i += (int64_t)gridDim.x * 256) {
        const int m = i < a.end[0] ? 0 : i < a.end[1] ? 1 : 2;
        const int64_t e = i - (m == 0 ? 0 : a.end[m - 1]), r = e / a.chunks[m], c = (e - r * a.chunks[m]) * 16;
        const char* row = a.in[m] + r * a.ld[m];
        uint4 v;
        if (c + 16 <= a.row[m]) {
            v = load_any(reinterpret_cast<const T*>(row + c), a.in[m], a.in[m] + (a.rows[m] - 1) * a.ld[m] + a.row[m]);
        } else {
            alignas(16) T last[16 / sizeof(T)] = {};
            for (int j = 0; c + j * (int)sizeof(T) < a.row[m]; ++j) last[j] = reinterpret_cast<const T*>(row + c)[j];
            v = *reinterpret_cast<uint4*>(last);
        }
        *reinterpret_cast<uint4*>(a.out[m] + r * a.pitch[m] + c) = v;
    }
}

// dgate = dh u act'(g), dup = dh act(g). Bound by its five matrices; 8 elements
// per thread where every row is 16-byte aligned (VEC). Both are rounded once to the
// tensors' type: the matrix instructions that take them as operands have 16 bits, and
// it keeps the bytes that the two products read at half. A gradient is off by 2.35e-3
// of its size (bfloat16) instead of the 1.66e-3 of its own rounding, by 2.9e-4 instead
// of 2.1e-4 (float16). In float16 a dgate or dup above 65504 is infinite, as it is in
// any program that keeps it in that type, in one row of dx and one channel of a weight.
struct GradArgs {
    const void *dh, *g, *u;
    int64_t ldd, ldg, ldu;
    int T, N;
    void *dg, *du;
    int64_t ldo;
};

template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256) k_gate_grad(const GradArgs a) {
    tensor::wait_for_stream();
    tensor::let_next_start();
    const int pieces = (a.N + 7) / 8;
    const int64_t count = (int64_t)a.T * pieces;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / pieces;
        const int n = (int)(i - t * pieces) * 8;
        Eight<T> d, g, u;
        auto load = [&](Eight<T>& e, const void* p, int64_t ld) {
            const T* all = reinterpret_cast<const T*>(p);
            const T* row = all + t * ld + n;
            if (n + 8 > a.N) e.load(row, a.N - n);
            else if (VEC) e.load(row);
            else e.load_any(row, all, all + (a.T - 1) * ld + a.N);
        };
        load(d, a.dh, a.ldd);
        load(g, a.g, a.ldg);
        load(u, a.u, a.ldu);
        alignas(16) T og[8], ou[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v, slope;
            act_grad<ACT>(g[j], v, slope);
            og[j] = from_f32<T>(d[j] * u[j] * slope);
            ou[j] = from_f32<T>(d[j] * v);
        }
        // the pitch of dg and du holds whole pieces; what lies beyond N is not read by the products
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.dg) + t * a.ldo + n) = *reinterpret_cast<uint4*>(og);
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.du) + t * a.ldo + n) = *reinterpret_cast<uint4*>(ou);
    }
}

// -------------------------------------------------------------------- host ---

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

int bad(const char* msg) {
    set_error(msg);
    return ABFT_ERR_ARG;
}

// Sizes whose tiles' indexes stay inside 32 bits.
bool extents(int T, int N, int K) {
    constexpr int kMost = ABFT_PRODUCT_MAX;
    return T >= 0 && T <= kMost && N >= 1 && N <= kMost && K >= 1 && K <= kMost;
}

// Addresses of elements of `size` bytes; the kernels read and write them as such.
bool lie_on(int size, std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if ((uintptr_t)p & (size - 1)) return false;
    return true;
}

int size_of(int type) { return type == ABFT_TYPE_F32 ? 4 : 2; }

bool holds(const void* work, size_t bytes, size_t needed) {
    return needed == 0 || (work && bytes >= needed && ((uintptr_t)work & 15) == 0);
}

int status(cudaError_t e, const char* what) { return e == cudaSuccess ? ABFT_OK : cuda_fail(e, what); }

// Launches a kernel that may start up while the one before it ends.
template <typename... P, typename... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, int block, int smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A row-major operand of elements of `size` bytes. One that bulk tensor copies
// cannot read (base or pitch not a multiple of 16 bytes) is copied first.
struct Operand {
    const void* p;
    int64_t ld;
    int rows, cols, size;

    bool direct() const { return ((uintptr_t)p & 15) == 0 && (rows == 1 || (ld * size & 15) == 0); }
    // of the copy: whole lines, so that no copied row of 128 bytes crosses one (1000 x 1536 block with K = 1008: 13.5 us
    // on a pitch of 2016 bytes, 11.3 on 2048)
    int64_t packed_pitch() const { return cdiv((int64_t)cols * size, 128) * 128 / size; }
    size_t bytes() const { return direct() ? 0 : ((size_t)rows * packed_pitch() * size + 255) & ~(size_t)255; }
    bool same(const Operand& o) const {
        return p == o.p && ld == o.ld && rows == o.rows && cols == o.cols && size == o.size;
    }

    // Boxes of 128 bytes x box_rows.
    bool map(CUtensorMap* m, int box_rows) const {
        auto enc = encode_tiled();
        if (!enc) return false;
        const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
        const cuuint64_t strides[1] = {(cuuint64_t)(rows == 1 ? packed_pitch() : ld) * size};
        const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows};
        const cuuint32_t one[2] = {1, 1};
        return enc(m, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p),
                   dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
};

// Puts copies in `work` in place of the operands that are not direct; `work` moves on.
cudaError_t pack(std::initializer_list<Operand*> operands, char*& work, cudaStream_t s) {
    PackArgs a = {};
    int n = 0, size = 0;
    int64_t total = 0;
    for (Operand* o : operands) {
        if (o->direct()) continue;
        a.in[n] = (const char*)o->p;
        a.out[n] = work;
        a.ld[n] = o->ld * o->size;
        a.row[n] = (int64_t)o->cols * o->size;
        a.rows[n] = o->rows;
        a.chunks[n] = cdiv(a.row[n], 16);
        a.pitch[n] = o->packed_pitch() * o->size;
        total += a.rows[n] * a.chunks[n];
        for (int i = n; i < 3; ++i) a.end[i] = total;
        size = o->size;
        const size_t bytes = o->bytes();
        o->p = work;
        o->ld = o->packed_pitch();
        work += bytes;
        ++n;
    }
    if (n == 0) return cudaSuccess;
    const dim3 grid((unsigned)std::min<int64_t>(cdiv(total, 256), 148 * 32));
    return size == 1 ? launch_next(k_pack<int8_t>, grid, 256, 0, s, a) : launch_next(k_pack<uint16_t>, grid, 256, 0, s, a);
}

// Number of SMs of the current device.
int sm_count() {
    static std::atomic<int> cache[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev >= 0 && dev < 64 && cache[dev].load()) return cache[dev].load();
    int n = 148;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (dev >= 0 && dev < 64) cache[dev].store(n);
    return n;
}

// Threads per row and pieces held by each: the smallest that hold a row of K;
// a warp alone needs no barrier. Rows above 16384 do not fit a block's registers and
// are read twice: 4096 rows of 28672 bfloat16 take 113 us (153 with a checksum, whose
// 64-bit multiply-adds any K allows) where as many bytes in rows of 16384 take 62 (77).
template <typename T>
cudaError_t quantize(QuantArgs a, cudaStream_t s) {
    a.aligned = ((uintptr_t)a.x & 15) == 0 && (a.T == 1 || (a.ldx * (int64_t)sizeof(T) & 15) == 0) &&
                ((uintptr_t)a.q & 7) == 0 && (a.T == 1 || (a.ldq & 7) == 0) && ((uintptr_t)a.checksum & 15) == 0;
    using std::integral_constant;
    cudaError_t result = cudaSuccess;
    auto launch = [&](auto row, auto u, auto check) {
        constexpr int kRow = decltype(row)::value, kU = decltype(u)::value, kBlock = kRow < 128 ? 128 : kRow;
        const int smem = decltype(check)::value && kU > 0 ? (int)cdiv(a.K, 8) * 32 : 0;
        auto kernel = k_quantize_rows<T, kRow, kU, decltype(check)::value>;
        // a block has 48 KB unless more is asked for; the kernel's own variables (less than 1 KB) count too
        if (smem > 47 * 1024)
            result = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
        int64_t blocks = cdiv(a.T, kBlock / kRow);
        if (blocks > sm_count()) {  // as many as are resident at a time, each with the same number of rows
            int resident = 1;
            if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kBlock, smem) != cudaSuccess) {
                (void)cudaGetLastError();
                resident = 1;
            }
            blocks = std::min<int64_t>(blocks, (int64_t)sm_count() * std::max(resident, 1));
        }
        if (result == cudaSuccess) result = launch_next(kernel, dim3((unsigned)blocks), kBlock, smem, s, a);
    };
    const integral_constant<int, 32> warp;
    const integral_constant<int, 128> row128;
    const integral_constant<int, 256> row256;
    const integral_constant<int, 512> row512;
    const integral_constant<int, 0> walk;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    const bool few = a.T <= sm_count();  // an SM for every row: more threads to a row
    auto choose = [&](auto check) {
        if (a.K <= 256) launch(warp, one, check);
        else if (a.K <= 512) launch(warp, two, check);
        else if (a.K <= 1024) launch(warp, four, check);
        else if (few && a.K <= 4096) launch(row512, one, check);
        else if (a.K <= 2048) launch(row128, two, check);
        else if (a.K <= 4096) launch(row128, four, check);
        else if (!few && a.K <= 8192) launch(row256, four, check);
        else if (a.K <= 16384) launch(row512, four, check);
        else launch(row512, walk, check);
    };
    const std::true_type yes;
    const std::false_type no;
    a.checksum ? choose(yes) : choose(no);
    return result;
}

template <int MODE, int CG, int BN, bool SPLIT, typename O, int ACT>
int launch_product(const Operand (&a)[2], const Operand (&b)[2], ProductArgs args, const char* name, cudaStream_t s) {
    using S = Shape<MODE, CG, BN, SPLIT, O>;
    ProductMaps maps;
    const int b_box = S::kBMn ? 64 : MODE == kGate ? BN / 2 : BN / CG;
    const int a_box = S::kAMn ? 64 : 128;
    bool made = a[0].map(&maps.a[0], a_box) && b[0].map(&maps.b[0], b_box);
    maps.a[1] = maps.a[0];
    maps.b[1] = maps.b[0];
    if (made && !a[1].same(a[0])) made = a[1].map(&maps.a[1], a_box);
    if (made && !b[1].same(b[0])) made = b[1].map(&maps.b[1], b_box);
    if (!made) {
        set_error(std::string(name) + ": a tensor map could not be made");
        return ABFT_ERR_CUDA;
    }
    args.tiles_m1 = (int)cdiv(args.rows, 128 * CG);
    args.tiles_m = MODE == kDw ? 2 * args.tiles_m1 : args.tiles_m1;
    args.tiles_n = (int)cdiv(args.cols, S::kCols);
    args.limit = wait_limit();
    for (int i = 0; i < 3; ++i)
        args.wide[i] = ((uintptr_t)args.c[i] & 15) == 0 && (args.ld[i] * (int64_t)sizeof(O) & 15) == 0;
    auto kernel = k_product<MODE, CG, BN, SPLIT, O, ACT>;
    static std::atomic<uint64_t> ready{0};  // devices (of 64) on which the shared memory is allowed
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(ready.load() >> dev & 1))) {
        e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e == cudaSuccess && dev <= 63) ready.fetch_or(1ull << dev);
    }
    if (e != cudaSuccess) return cuda_fail(e, name);
    const int64_t tiles = (int64_t)args.tiles_m * args.tiles_n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(SPLIT ? tiles * args.split : std::min<int64_t>(tiles, sm_count() / CG) * CG));
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = SPLIT ? args.split : CG;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kernel, maps, args);
    return e == cudaSuccess ? ABFT_OK : cuda_fail(e, name);
}

// Whether k_few takes a product of T tokens with `bytes` of weights: always up to
// 16; up to 32 while the weights are small, since past that its own work shows
// (block of 16384 x 4096, 32 tokens: 65 us, 48 tokens by k_product 49 us; block of
// 1024 x 4096: 7.8 against 10.2 us). Operands off 16 bytes are copied before either
// kernel, at the same cost (block of 16384 x 4097: 145 us for one token, 153 for 13,
// by k_product 158 for 48), so the rule is theirs too.
bool few_tokens(int T, int64_t bytes) { return T <= 16 || (T <= 32 && bytes <= 32 << 20); }

template <bool GATE, typename E, typename O, int ACT = 0>
int few(const Operand& x, const Operand (&w)[2], const ProductArgs& p, const char* name, cudaStream_t s) {
    FewArgs a = {};
    for (int i = 0; i < 2; ++i) {
        a.w[i] = (const char*)w[i].p;
        a.ldw[i] = w[i].ld * w[i].size;
    }
    a.x = (const char*)x.p;
    a.ldx = x.ld * x.size;
    a.T = p.rows;
    a.N = p.cols;
    a.kbytes = (int64_t)x.cols * x.size;
    std::copy(p.c, p.c + 3, a.c);
    std::copy(p.ld, p.ld + 3, a.ld);
    a.row_scale = p.row_scale;
    a.col_scale = p.col_scale;
    a.rowdiff = p.rowdiff;
    // Warps that share a group's K: 8, so that a block streams whole rows, but none without a run of its own and 4 where
    // more tokens make the warps' work longer than their wait (block of 16384 x 4096, one token: 46.9 / 43.3 / 44.9 / 39.9
    // us with 1 / 2 / 4 / 8; 8-bit 8192 x 2048: 7.2 / 5.5 / 4.7 / 5.8; 16 tokens, block of 4096 x 4096: 28 / 17 / 14 / 16,
    // of 1024 x 4096: 27 / 14 / 8.4 / 6.0).
    const int64_t groups = cdiv(a.N, GATE ? 8 : 16);
    const int most = a.T > 8 && groups >= sm_count() * 2 ? 4 : 8;
    const int64_t run = a.T <= 16 ? 512 : 256;  // bytes of K that a warp takes at a time
    int wk = 1;
    while (wk < most && wk * run < a.kbytes) wk *= 2;
    using std::integral_constant;
    auto go = [&](auto nt, auto w) {
        constexpr int kWk = decltype(w)::value;
        return launch_next(k_few<GATE, E, decltype(nt)::value, kWk, O, ACT>, dim3((unsigned)cdiv(groups, 8 / kWk)), 256, 0,
                           s, a);
    };
    auto with_wk = [&](auto nt) {
        if (wk == 1) return go(nt, integral_constant<int, 1>());
        if (wk == 2) return go(nt, integral_constant<int, 2>());
        if (wk == 4) return go(nt, integral_constant<int, 4>());
        return go(nt, integral_constant<int, 8>());
    };
    if (a.T <= 8) return status(with_wk(integral_constant<int, 1>()), name);
    if (a.T <= 16) return status(with_wk(integral_constant<int, 2>()), name);
    return status(with_wk(integral_constant<int, 4>()), name);
}

// Clusters of `split` product CTAs (one an SM) that the GPU runs at a time; SMs
// come in groups that a cluster does not leave, so this is below SMs / split.
int clusters_at_once(int split) {
    static std::atomic<int> cache[64][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev > 63) return 0;
    int n = cache[dev][split].load();
    if (n) return n - 1;
    using S = Shape<kInt8, 1, 128, true, float>;
    auto kernel = k_product<kInt8, 1, 128, true, float, 0>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split);
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        return 0;
    }
    cache[dev][split].store(n + 1);
    return n;
}

// Tile and split by an estimate in us: a start and an end, and for every round of
// tiles its chunks of 128 bytes of K or its results on their way out, whichever
// is longer (kGate counts as if g or u were kept too, whether or not, so that h
// does not depend on it):
//
//                       start + end   a chunk (alone / all SMs busy)   32 x 32 results of a warp
//   pair of SMs, 256        5.2        0.30  (0.28 / 0.31)              4 x 0.45
//   one SM, 128 columns     4.0        0.20  (0.19 / 0.21)              2 x 0.45
//   one SM, 64 columns      4.0        0.185 (0.18 / 0.19)             1 x 0.45
//   split, 128 columns      7.3        0.20   all clusters at once only
//   split, 64 columns       5.8        0.18
//
// Examples, us measured (pair / 128 / 64 / best split): bf16 block of 8192 tokens,
// 16384 x 4096: 1540 / 2288 / - / -; 1000, 4096 x 4096: 45 / 58 / 88 / -; 1000, 1536 x
// 1024: 10.8 / 11.1 / 14.1 / -; 48, 1536 x 1024: 9.2 / 6.8 / 7.0 / 7.6; 48, 4096 x 4096:
// 23.2 / 16.6 / 16.3 / 13.3; 48, 512 x 16384: 76 / 52 / 50 / 14.
template <int MODE, typename O, int ACT = 0>
int product(const Operand (&a)[2], const Operand (&b)[2], ProductArgs args, const char* name, cudaStream_t s) {
    const int chunks = args.chunks * (MODE == kDx ? 2 : 1);
    auto tiles = [&](int rows, int columns) {
        return (MODE == kDw ? 2 : 1) * cdiv(args.rows, rows) * cdiv(args.cols, MODE == kGate ? columns / 2 : columns);
    };
    const int sms = sm_count();
    double best = 1e30;
    int which = 0;
    auto consider = [&](int i, int split, double ends, double chunk, int columns, int64_t rounds) {
        const double round = std::max(chunk * (double)cdiv(chunks, split), 0.45 / 64 * columns);
        const double us = ends + round * (double)rounds;
        if (us < best) {
            best = us;
            which = i;
            args.split = split;
        }
    };
    consider(0, 1, 5.2, 0.30, 256, cdiv(tiles(256, 256), std::max(sms / 2, 1)));
    consider(1, 1, 4.0, 0.20, 128, cdiv(tiles(128, 128), sms));
    consider(2, 1, 4.0, 0.185, 64, cdiv(tiles(128, 64), sms));
    for (int split = 2; split <= 8 && split <= chunks && tiles(128, 128) * split <= sms; ++split) {
        const int clusters = clusters_at_once(split);
        if (tiles(128, 128) <= clusters) consider(3, split, 7.3, 0.20, 0, 1);
        if (tiles(128, 64) <= clusters) consider(4, split, 5.8, 0.18, 0, 1);
    }
    switch (which) {
        case 0: return launch_product<MODE, 2, 256, false, O, ACT>(a, b, args, name, s);
        case 1: return launch_product<MODE, 1, 128, false, O, ACT>(a, b, args, name, s);
        case 2: return launch_product<MODE, 1, 64, false, O, ACT>(a, b, args, name, s);
        case 3: return launch_product<MODE, 1, 128, true, O, ACT>(a, b, args, name, s);
        default: return launch_product<MODE, 1, 64, true, O, ACT>(a, b, args, name, s);
    }
}

// dgate and dup, each T rows on a pitch of whole lines
int64_t grad_pitch(int N) { return cdiv(N, 64) * 64; }
size_t grad_bytes(int T, int N) { return (static_cast<size_t>(T) * grad_pitch(N) * 2 + 255) & ~(size_t)255; }

template <typename F>
auto with_type(int type, F&& f) {
    if (type == ABFT_TYPE_F16) return f(__half());
    return f(__nv_bfloat16());
}

template <typename F>
auto with_act(int activation, F&& f) {
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
    if (!extents(T, 1, K) || ldx < K || ldq < K || type < ABFT_TYPE_F32 || type > ABFT_TYPE_BF16)
        return bad("abft_quantize_rows: bad argument (need 0 <= T <= 2^30, 1 <= K <= 2^30, ldx >= K, ldq >= K and an "
                   "element type)");
    if (T == 0) return ABFT_OK;
    if (!dX || !dQ || !dScale || (dChecksum != nullptr) != (dExpect != nullptr))
        return bad("abft_quantize_rows: bad argument (missing pointer, or one of dChecksum and dExpect alone)");
    if (!lie_on(size_of(type), {dX}) || !lie_on(4, {dScale, dChecksum}) || !lie_on(8, {dExpect}))
        return bad("abft_quantize_rows: bad argument (a pointer not aligned to its elements)");
    const QuantArgs args{false, dX, ldx, T, K, dQ, ldq, dScale, dChecksum, dExpect};
    auto go = [&](auto tag) {
        return status(quantize<decltype(tag)>(args, (cudaStream_t)stream), "abft_quantize_rows");
    };
    if (type == ABFT_TYPE_F32) return go(0.0f);
    return with_type(type, go);
}

int abft_column_checksum(const int8_t* dW, int64_t ldw, int N, int K, int32_t* dChecksum, void* stream) {
    if (!dW || !dChecksum || N < 1 || N > ABFT_INT8_MAX_ROWS || !extents(0, N, K) || ldw < K || !lie_on(4, {dChecksum}))
        return bad("abft_column_checksum: bad argument (need pointers, dChecksum aligned to its elements, 1 <= N <= 2^24, "
                   "1 <= K <= 2^30, ldw >= K)");
    cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = cudaMemsetAsync(dChecksum, 0, sizeof(int32_t) * K, s);
    if (e != cudaSuccess) return cuda_fail(e, "abft_column_checksum");
    const int rows = std::max(256, (int)cdiv(N, 65535));  // a grid has 65535 blocks in y
    const unsigned chunks = (unsigned)cdiv(N, rows);
    if (((uintptr_t)dW & 3) == 0 && (ldw & 3) == 0)
        k_column_checksum<true><<<dim3((unsigned)cdiv(K, 1024), chunks), 256, 0, s>>>(dW, ldw, N, K, rows, dChecksum);
    else
        k_column_checksum<false><<<dim3((unsigned)cdiv(K, 256), chunks), 256, 0, s>>>(dW, ldw, N, K, rows, dChecksum);
    return status(cudaGetLastError(), "abft_column_checksum");
}

size_t abft_int8_matmul_ws_bytes(const int8_t* dQ, int64_t ldq, const int8_t* dW, int64_t ldw, int T, int N, int K) {
    if (T < 1 || !extents(T, N, K)) return 0;
    return Operand{dQ, ldq, T, K, 1}.bytes() + Operand{dW, ldw, N, K, 1}.bytes();
}

int abft_int8_matmul(const int8_t* dQ, int64_t ldq, const float* dQScale, const int8_t* dW, int64_t ldw,
                     const float* dWScale, int T, int N, int K, void* dY, int64_t ldy, int type,
                     const int64_t* dExpect, int64_t* dRowDiff, void* dWork, size_t work_bytes, void* stream) {
    if (!extents(T, N, K) || K > ABFT_INT8_MAX_K || ldq < K || ldw < K || ldy < N || type < ABFT_TYPE_F32 ||
        type > ABFT_TYPE_BF16)
        return bad("abft_int8_matmul: bad argument (need 0 <= T <= 2^30, 1 <= N <= 2^30, 1 <= K <= 131071, ldq >= K, "
                   "ldw >= K, ldy >= N and an element type)");
    if (T == 0) return ABFT_OK;
    if (!dQ || !dQScale || !dW || !dWScale || !dY || (dExpect != nullptr) != (dRowDiff != nullptr))
        return bad("abft_int8_matmul: bad argument (missing pointer, or one of dExpect and dRowDiff alone)");
    if (!lie_on(size_of(type), {dY}) || !lie_on(4, {dQScale, dWScale}) || !lie_on(8, {dExpect, dRowDiff}))
        return bad("abft_int8_matmul: bad argument (a pointer not aligned to its elements)");
    if (!holds(dWork, work_bytes, abft_int8_matmul_ws_bytes(dQ, ldq, dW, ldw, T, N, K)))
        return bad("abft_int8_matmul: workspace missing, too small or not 16-byte aligned");
    cudaStream_t s = (cudaStream_t)stream;
    if (dExpect) {
        const cudaError_t e = launch_next(k_negate, dim3((unsigned)cdiv(T, 256)), 256, 0, s, dExpect, dRowDiff, T);
        if (e != cudaSuccess) return cuda_fail(e, "abft_int8_matmul");
    }
    Operand q{dQ, ldq, T, K, 1}, w{dW, ldw, N, K, 1};
    char* work = (char*)dWork;
    const cudaError_t packed = pack({&q, &w}, work, s);
    if (packed != cudaSuccess) return cuda_fail(packed, "abft_int8_matmul");
    ProductArgs args = {};
    args.rows = T;
    args.cols = N;
    args.chunks = (int)cdiv(K, 128);
    args.c[0] = dY;
    args.ld[0] = ldy;
    args.row_scale = dQScale;
    args.col_scale = dWScale;
    args.rowdiff = (unsigned long long*)dRowDiff;
    auto go = [&](auto tag) {
        if (few_tokens(T, (int64_t)N * K)) return few<false, int8_t, decltype(tag)>(q, {w, w}, args, "abft_int8_matmul", s);
        return product<kInt8, decltype(tag)>({q, q}, {w, w}, args, "abft_int8_matmul", s);
    };
    if (type == ABFT_TYPE_F32) return go(0.0f);
    return with_type(type, go);
}

size_t abft_gated_ffn_ws_bytes(const void* dX, int64_t ldx, const void* dWGate, int64_t ldwg, const void* dWUp,
                               int64_t ldwu, int T, int N, int K) {
    if (T < 1 || !extents(T, N, K)) return 0;
    return Operand{dX, ldx, T, K, 2}.bytes() + Operand{dWGate, ldwg, N, K, 2}.bytes() +
           Operand{dWUp, ldwu, N, K, 2}.bytes();
}

int abft_gated_ffn(const void* dX, int64_t ldx, const void* dWGate, int64_t ldwg, const void* dWUp, int64_t ldwu,
                   int T, int N, int K, int type, int activation, void* dH, int64_t ldh, void* dG, int64_t ldg,
                   void* dU, int64_t ldu, void* dWork, size_t work_bytes, void* stream) {
    if (!extents(T, N, K) || ldx < K || ldwg < K || ldwu < K || ldh < N || (dG && ldg < N) || (dU && ldu < N) ||
        (type != ABFT_TYPE_F16 && type != ABFT_TYPE_BF16) || activation < ABFT_ACT_SILU ||
        activation > ABFT_ACT_GELU_TANH)
        return bad("abft_gated_ffn: bad argument (need 0 <= T <= 2^30, 1 <= N, K <= 2^30, pitches that hold a row, a "
                   "16-bit element type and an activation)");
    if (T == 0) return ABFT_OK;
    if (!dX || !dWGate || !dWUp || !dH || (dG != nullptr) != (dU != nullptr))
        return bad("abft_gated_ffn: bad argument (missing pointer, or one of dG and dU alone)");
    if (!lie_on(2, {dX, dWGate, dWUp, dH, dG, dU}))
        return bad("abft_gated_ffn: bad argument (a pointer not aligned to its elements)");
    if (!holds(dWork, work_bytes, abft_gated_ffn_ws_bytes(dX, ldx, dWGate, ldwg, dWUp, ldwu, T, N, K)))
        return bad("abft_gated_ffn: workspace missing, too small or not 16-byte aligned");
    cudaStream_t s = (cudaStream_t)stream;
    Operand x{dX, ldx, T, K, 2}, wg{dWGate, ldwg, N, K, 2}, wu{dWUp, ldwu, N, K, 2};
    char* work = (char*)dWork;
    const cudaError_t packed = pack({&x, &wg, &wu}, work, s);
    if (packed != cudaSuccess) return cuda_fail(packed, "abft_gated_ffn");
    ProductArgs args = {};
    args.rows = T;
    args.cols = N;
    args.chunks = (int)cdiv(K, 64);
    void* outs[3] = {dH, dG, dU};
    const int64_t pitches[3] = {ldh, ldg, ldu};
    std::copy(outs, outs + 3, args.c);
    std::copy(pitches, pitches + 3, args.ld);
    return with_type(type, [&](auto tag) {
        return with_act(activation, [&](auto a) {
            if (few_tokens(T, 4LL * N * K))
                return few<true, decltype(tag), decltype(tag), decltype(a)::value>(x, {wg, wu}, args, "abft_gated_ffn", s);
            return product<kGate, decltype(tag), decltype(a)::value>({x, x}, {wg, wu}, args, "abft_gated_ffn", s);
        });
    });
}

size_t abft_gated_ffn_backward_ws_bytes(const void* dX, int64_t ldx, const void* dWGate, int64_t ldwg,
                                        const void* dWUp, int64_t ldwu, int T, int N, int K) {
    if (T < 1 || !extents(T, N, K)) return 0;
    return 2 * grad_bytes(T, N) + abft_gated_ffn_ws_bytes(dX, ldx, dWGate, ldwg, dWUp, ldwu, T, N, K);
}

int abft_gated_ffn_backward(const void* dDH, int64_t ldd, const void* dX, int64_t ldx, const void* dWGate,
                            int64_t ldwg, const void* dWUp, int64_t ldwu, const void* dG, int64_t ldg, const void* dU,
                            int64_t ldu, int T, int N, int K, int type, int activation, void* dDX, int64_t lddx,
                            void* dDWGate, int64_t lddwg, void* dDWUp, int64_t lddwu, void* dWork, size_t work_bytes,
                            void* stream) {
    if (!extents(T, N, K) || ldd < N || ldx < K || ldwg < K || ldwu < K || ldg < N || ldu < N || lddx < K ||
        lddwg < K || lddwu < K || (type != ABFT_TYPE_F16 && type != ABFT_TYPE_BF16) || activation < ABFT_ACT_SILU ||
        activation > ABFT_ACT_GELU_TANH)
        return bad("abft_gated_ffn_backward: bad argument (need 0 <= T <= 2^30, 1 <= N, K <= 2^30, pitches that hold "
                   "a row, a 16-bit element type and an activation)");
    if (!dDWGate || !dDWUp) return bad("abft_gated_ffn_backward: bad argument (missing pointer)");
    if (!lie_on(2, {dDH, dX, dWGate, dWUp, dG, dU, dDX, dDWGate, dDWUp}))
        return bad("abft_gated_ffn_backward: bad argument (a pointer not aligned to its elements)");
    cudaStream_t s = (cudaStream_t)stream;
    if (T == 0) {  // no token: the weights' gradients are empty sums
        cudaError_t e = cudaMemset2DAsync(dDWGate, lddwg * 2, 0, static_cast<size_t>(K) * 2, N, s);
        if (e == cudaSuccess) e = cudaMemset2DAsync(dDWUp, lddwu * 2, 0, static_cast<size_t>(K) * 2, N, s);
        return e == cudaSuccess ? ABFT_OK : cuda_fail(e, "abft_gated_ffn_backward");
    }
    if (!dDH || !dX || !dWGate || !dWUp || !dG || !dU || !dDX)
        return bad("abft_gated_ffn_backward: bad argument (missing pointer)");
    if (!holds(dWork, work_bytes, abft_gated_ffn_backward_ws_bytes(dX, ldx, dWGate, ldwg, dWUp, ldwu, T, N, K)))
        return bad("abft_gated_ffn_backward: workspace missing, too small or not 16-byte aligned");
    const int64_t p = grad_pitch(N);
    char* work = (char*)dWork;
    const Operand dg{work, p, T, N, 2}, du{work + grad_bytes(T, N), p, T, N, 2};
    work += 2 * grad_bytes(T, N);
    Operand x{dX, ldx, T, K, 2}, wg{dWGate, ldwg, N, K, 2}, wu{dWUp, ldwu, N, K, 2};
    const cudaError_t packed = pack({&x, &wg, &wu}, work, s);
    if (packed != cudaSuccess) return cuda_fail(packed, "abft_gated_ffn_backward");
    return with_type(type, [&](auto tag) {
        using E = decltype(tag);
        const cudaError_t e = with_act(activation, [&](auto a) {
            const GradArgs ga{dDH, dG, dU, ldd, ldg, ldu, T, N, const_cast<void*>(dg.p), const_cast<void*>(du.p), p};
            const bool vec = Operand{dDH, ldd, T, N, 2}.direct() && Operand{dG, ldg, T, N, 2}.direct() &&
                             Operand{dU, ldu, T, N, 2}.direct();
            const unsigned grid = (unsigned)std::min<int64_t>(cdiv(T * cdiv(N, 8), 256), (int64_t)sm_count() * 64);
            return vec ? launch_next(k_gate_grad<E, decltype(a)::value, true>, dim3(grid), 256, 0, s, ga)
                       : launch_next(k_gate_grad<E, decltype(a)::value, false>, dim3(grid), 256, 0, s, ga);
        });
        if (e != cudaSuccess) return cuda_fail(e, "abft_gated_ffn_backward");
        ProductArgs args = {};
        args.rows = T;
        args.cols = K;
        args.chunks = (int)cdiv(N, 64);
        args.c[0] = dDX;
        args.ld[0] = lddx;
        if (int rc = product<kDx, E>({dg, du}, {wg, wu}, args, "abft_gated_ffn_backward", s)) return rc;
        args.rows = N;
        args.chunks = (int)cdiv(T, 64);
        args.c[0] = dDWGate;
        args.ld[0] = lddwg;
        args.c[1] = dDWUp;
        args.ld[1] = lddwu;
        return product<kDw, E>({dg, du}, {x, x}, args, "abft_gated_ffn_backward", s);
    });
}

int abft_products_status(int* fault) {
    if (!fault) return bad("abft_products_status: fault is NULL");
    static thread_local unsigned told[64];  // of each device
    int dev = 0;
    unsigned now = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // a copy alone does not wait for streams made not to wait for it
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&now, g_faults, sizeof(now));
    if (e != cudaSuccess) return cuda_fail(e, "abft_products_status");
    *fault = now != (dev < 64 ? told[dev] : 0);
    if (dev < 64) told[dev] = now;
    return ABFT_OK;
}

}  // extern "C"

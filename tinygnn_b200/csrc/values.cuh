// ============================================================================
//  values.cuh -- element types (fp32, bf16, fp16) and the 8-bit saved form of
//  a matrix, shared by the training operators' kernels.
//
//  Saved form of a rows x cols matrix: for each row and each block of 128
//  columns the least exponent e with max|x| <= 127 * 2^e, and one signed byte
//  round-to-even(x / 2^e) per value.  A power of two (rather than max|x| / 127)
//  costs up to one bit of resolution and buys an exact form: every value
//  code * 2^e has at most 7 significant bits, so bf16 holds it exactly and a
//  product on the tensor cores reads it with no second rounding; coding is a
//  multiplication by a power of two and one rounding, the same on every
//  machine.  The exponent is stored as the byte e + 127; kBad8 marks a block
//  that held an infinity or a NaN, whose every value restores as NaN.
// ============================================================================
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "launch.cuh"

namespace tg {

constexpr int kBlock8 = 128;   // columns that share an exponent
constexpr int kBad8 = 255;     // exponent byte of a block that held inf or NaN

inline size_t dtype_size(int dtype) { return dtype == TG_F32 ? 4 : 2; }

inline void check_dtype(const char* fn, const char* what, int dtype) {
    if (dtype != TG_F32 && dtype != TG_BF16 && dtype != TG_F16)
        invalid(std::string(fn) + ": " + what + " has no such type (" + std::to_string(dtype) + ")");
}

// Calls f with a value of the element type that `dtype` names.
template <class F>
void by_dtype(int dtype, F&& f) {
    if (dtype == TG_F32) f(float{});
    else if (dtype == TG_BF16) f(__nv_bfloat16{});
    else f(__half{});
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// V consecutive values at p (aligned to V * sizeof(T)) to and from fp32.
template <class T, int V>
struct alignas(V * sizeof(T)) Pack {
    T v[V];
};
template <class T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&x)[V]) {
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = to_f32(k.v[j]);
}
template <class T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&x)[V]) {
    Pack<T, V> k;
#pragma unroll
    for (int j = 0; j < V; ++j) k.v[j] = from_f32<T>(x[j]);
    *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// Magnitudes are compared as bit patterns: they order like the values, with
// infinity above every number and NaN above infinity (fmaxf would drop NaN).
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The exponent byte of a block whose largest magnitude has bits `m`.  127 is
// 1.984375 * 2^6, so e is the exponent of max|x| less 6, or one more when its
// mantissa is above 1.984375.
__device__ __forceinline__ int exponent8(uint32_t m, int emin) {
    if (m >= 0x7f800000u) return kBad8;
    const int e = static_cast<int>(m >> 23) - 133 + ((m & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return (e > emin ? e : emin) + 127;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// 2^-e, the factor from values to codes (0 for a bad block: its codes are 0).
__device__ __forceinline__ float encode8(int byte) { return byte == kBad8 ? 0.0f : pow2f(127 - byte); }
// 2^e, the factor from codes to values (NaN for a bad block).
__device__ __forceinline__ float decode8(int byte) {
    return byte == kBad8 ? __uint_as_float(0x7fffffffu) : pow2f(byte - 127);
}
// The code of x (inv = encode8(byte); an infinity or NaN times 0 is NaN, which
// converts to 0).  At the type's greatest exponent 64 * 2^e would overflow it.
__device__ __forceinline__ int8_t code8(float x, float inv, int byte, int top) {
    int c = __float2int_rn(__fmul_rn(x, inv));
    if (byte == top) c = c > 63 ? 63 : (c < -63 ? -63 : c);
    return static_cast<int8_t>(c);
}

// The least exponent of a block: 2^-126, or 2^-24 for fp16 matrices, whose
// values are multiples of it (so no value is lost, and each code * 2^e is an
// fp16 number too).
struct Range8 {
    int emin;  // least exponent
    int top;   // exponent byte of a block that holds the type's greatest values
};
inline Range8 range8(int dtype) { return dtype == TG_F16 ? Range8{-24, 10 + 127} : Range8{-126, 122 + 127}; }

template <class T, int W>
__device__ __forceinline__ T reduce_sum(T x) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) x = x + __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
template <int W>
__device__ __forceinline__ uint32_t reduce_max(uint32_t x) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// A matrix in the saved form, as the kernels take it (codes' rows start
// 16-byte aligned).
struct Saved8 {
    int8_t* codes;
    int64_t ld;
    uint8_t* exps;
    int64_t lde;
};

// ── Activations and their slopes ─────────────────────────────────────────
// The choice is made once for V values.  GELU's 1/2 (1 + tanh u) is computed
// as 1 / (1 + e^-2u), which equals it, does not cancel where tanh u is near
// -1, and costs one exponential and one reciprocal: with tanhf the 8-bit
// activation passes are bound by arithmetic instead of memory.
__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.0f, __fadd_rn(1.0f, expf(-x))); }

__device__ __forceinline__ float gelu_u(float x, float x2) {  // c (x + d x^3), c = sqrt(2 / pi)
    return __fmul_rn(0.7978845608f, fmaf(__fmul_rn(0.044715f, x2), x, x));
}

template <int V, class F>
__device__ __forceinline__ void map_v(float (&x)[V], F&& f) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = f(x[j]);
}

// x <- act(x)
template <int V>
__device__ __forceinline__ void act_forward(float (&x)[V], int act, float alpha) {
    switch (act) {
        case TG_ACT_RELU: map_v(x, [](float v) { return v < 0.0f ? 0.0f : v; }); break;  // NaN stays NaN
        case TG_ACT_LEAKY_RELU: map_v(x, [alpha](float v) { return v >= 0.0f ? v : __fmul_rn(alpha, v); }); break;
        case TG_ACT_ELU:
            map_v(x, [alpha](float v) { return v < 0.0f ? __fmul_rn(alpha, __fsub_rn(expf(v), 1.0f)) : v; });
            break;
        case TG_ACT_SIGMOID: map_v(x, [](float v) { return sigmoid_f(v); }); break;
        case TG_ACT_TANH: map_v(x, [](float v) { return tanhf(v); }); break;
        case TG_ACT_GELU:
            map_v(x, [](float v) {
                const float s = sigmoid_f(__fmul_rn(2.0f, gelu_u(v, __fmul_rn(v, v))));
                return s == 0.0f ? 0.0f : __fmul_rn(v, s);  // -inf: 0, not -inf * 0
            });
            break;
        default: break;
    }
}

// x <- act'(x)
template <int V>
__device__ __forceinline__ void act_slope(float (&x)[V], int act, float alpha) {
    switch (act) {
        case TG_ACT_RELU: map_v(x, [](float v) { return v > 0.0f ? 1.0f : (v <= 0.0f ? 0.0f : v); }); break;
        case TG_ACT_LEAKY_RELU:
            map_v(x, [alpha](float v) { return v >= 0.0f ? 1.0f : (v < 0.0f ? alpha : v); });
            break;
        case TG_ACT_ELU:
            map_v(x, [alpha](float v) { return v < 0.0f ? __fmul_rn(alpha, expf(v)) : (v >= 0.0f ? 1.0f : v); });
            break;
        case TG_ACT_SIGMOID:
            map_v(x, [](float v) {
                const float s = sigmoid_f(v);
                return __fmul_rn(s, __fsub_rn(1.0f, s));
            });
            break;
        case TG_ACT_TANH:
            map_v(x, [](float v) {
                const float t = tanhf(v);
                return fmaf(-t, t, 1.0f);
            });
            break;
        case TG_ACT_GELU:
            // s = 1 / (1 + e^-2u): act' = s + 2 x s (1 - s) u',  u' = c (1 + 3 d x^2).
            // Beyond |x| = 16 s is 0 or 1 in fp32, and u' may overflow.
            map_v(x, [](float v) {
                if (fabsf(v) > 16.0f) return v > 0.0f ? 1.0f : 0.0f;
                const float v2 = __fmul_rn(v, v);
                const float s = sigmoid_f(__fmul_rn(2.0f, gelu_u(v, v2)));
                const float du = __fmul_rn(0.7978845608f, fmaf(0.134145f, v2, 1.0f));
                return fmaf(__fmul_rn(__fmul_rn(2.0f, v), __fmul_rn(s, __fsub_rn(1.0f, s))), du, s);
            });
            break;
        default: map_v(x, [](float) { return 1.0f; }); break;
    }
}

// Whether rows starting at p with stride ld (elements of `size` bytes) are
// all 16-byte aligned.
inline bool rows_aligned16(const void* p, int64_t ld, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * static_cast<int64_t>(size) % 16 == 0;
}

inline void check_act(const char* fn, int act) {
    if (act < TG_ACT_NONE || act > TG_ACT_GELU)
        invalid(std::string(fn) + ": no such activation (" + std::to_string(act) + ")");
}

inline void check_rows_cols(const char* fn, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1 || rows > INT32_MAX || cols > INT32_MAX)
        invalid(std::string(fn) + ": a matrix of " + std::to_string(rows) + " rows and " + std::to_string(cols) +
                " columns is outside [0, 2^31) x [1, 2^31)");
}

inline void check_saved8(const char* fn, int64_t cols, const Saved8& s, bool needed) {
    check_ptr(fn, "codes", s.codes, needed);
    check_ptr(fn, "exponents", s.exps, needed);
    if (!s.codes) return;
    check_ld(fn, "codes", s.ld, cols);
    check_ld(fn, "exponents", s.lde, ceil_div(cols, kBlock8));
    if (!rows_aligned16(s.codes, s.ld, 1)) invalid(std::string(fn) + ": rows of codes must start 16-byte aligned");
}

}  // namespace tg

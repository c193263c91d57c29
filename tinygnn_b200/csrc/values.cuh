// ============================================================================
//  values.cuh -- element types (fp32, bf16, fp16) and the 8-bit saved form of
//  a matrix, shared by the training operators' kernels.
//
//  Saved form of a rows x cols matrix: for each row and each block of 128
//  columns the least exponent e with max|x| <= 127 * 2^e, and one signed byte
//  round-to-even(x / 2^e) per value (at the type's greatest exponent clamped to
//  63, since 64 * 2^e would overflow it).  A power of two (rather than max|x| / 127)
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

#include <type_traits>

#include "launch.cuh"

namespace tg {

constexpr int kBlock8 = 128;   // columns that share an exponent
constexpr int kBad8 = 255;     // exponent byte of a block that held inf or NaN

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

// V values as they lie in memory, in 32-bit words: where a kernel has a vector
// load and an elementwise one for edges, 16-bit values kept one by one would
// each take a register of their own (and an instruction to unpack).
template <class T, int V>
struct alignas(V * sizeof(T)) Raw {
    static constexpr int N = V * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[N];
};
__device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t bits(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
__device__ __forceinline__ uint32_t bits(__half x) { return __half_as_ushort(x); }

template <class T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {  // aligned to V * sizeof(T)
    return *reinterpret_cast<const Raw<T, V>*>(p);
}
template <class T, int V, class F>  // value j = f(j)
__device__ __forceinline__ Raw<T, V> gather_raw(F&& f) {
    Raw<T, V> k;
#pragma unroll
    for (int i = 0; i < Raw<T, V>::N; ++i) {
        if (sizeof(T) == 4) k.w[i] = bits(f(i));
        else k.w[i] = bits(f(2 * i)) | bits(f(2 * i + 1)) << 16;
    }
    return k;
}
template <int V>
__device__ __forceinline__ void widen(const Raw<float, V>& k, float* x) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = __uint_as_float(k.w[j]);
}
template <int V>
__device__ __forceinline__ void widen(const Raw<__nv_bfloat16, V>& k, float* x) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        x[j] = __uint_as_float(k.w[j / 2] << 16);
        x[j + 1] = __uint_as_float(k.w[j / 2] & 0xffff0000u);
    }
}
template <int V>
__device__ __forceinline__ void widen(const Raw<__half, V>& k, float* x) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&k.w[j / 2]));
        x[j] = t.x;
        x[j + 1] = t.y;
    }
}
// Rounded to T, two values an instruction where T has 16 bits.
template <int V>
__device__ __forceinline__ void narrow(const float* x, Raw<float, V>& k) {
#pragma unroll
    for (int j = 0; j < V; ++j) k.w[j] = __float_as_uint(x[j]);
}
template <int V>
__device__ __forceinline__ void narrow(const float* x, Raw<__nv_bfloat16, V>& k) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(x[j], x[j + 1]);
        k.w[j / 2] = *reinterpret_cast<const uint32_t*>(&t);
    }
}
template <int V>
__device__ __forceinline__ void narrow(const float* x, Raw<__half, V>& k) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        const __half2 t = __floats2half2_rn(x[j], x[j + 1]);
        k.w[j / 2] = *reinterpret_cast<const uint32_t*>(&t);
    }
}
template <class T, int V>
__device__ __forceinline__ void load_v(const T* p, float (&x)[V]) {
    widen(load_raw<T, V>(p), x);
}
template <class T, int V>
__device__ __forceinline__ void store_v(T* p, const float (&x)[V]) {
    Raw<T, V> k;
    narrow(x, k);
    *reinterpret_cast<Raw<T, V>*>(p) = k;
}

// V values as they were fetched from rows of any alignment (ALIGNED: from
// aligned ones).  16-bit values are fetched in whole words; where p is odd they
// start half a word in, and are shifted into place when they are widened, not
// when they are fetched: a kernel can ask for many before it waits for one.
template <class T, int V, bool ALIGNED>
struct Held {
    static constexpr bool kShift = !ALIGNED && sizeof(T) == 2;
    uint32_t w[V * static_cast<int>(sizeof(T)) / 4 + kShift];

    static __device__ __forceinline__ bool odd(const T* p) { return kShift && (reinterpret_cast<uintptr_t>(p) & 2); }
    // All V values are there.  (The first and the last word then reach one
    // value past the V, in words that hold one of them.)
    __device__ __forceinline__ void fetch(const T* p) {
        if constexpr (ALIGNED) {
            const Raw<T, V> k = load_raw<T, V>(p);
#pragma unroll
            for (int j = 0; j < Raw<T, V>::N; ++j) w[j] = k.w[j];
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = bits(p[j]);
        } else {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
#pragma unroll
            for (int j = 0; j < V / 2; ++j) w[j] = q[j];
            w[V / 2] = odd(p) ? q[V / 2] : 0u;
        }
    }
    // The first n values (all, for more; none, for n <= 0) are there.  Whole
    // words that hold one of them are read and kept as they are: values() with
    // n clears the rest, since an instruction on a word here would wait for it
    // (a layer norm's gradient that picked a row's last values out as it asked
    // for the next rows took 92 us for 65,536 x 511, and 76 without).
    __device__ __forceinline__ void fetch(const T* p, int n) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = j < n ? bits(p[j]) : 0u;
        } else {
            const int shift = odd(p);
            const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
#pragma unroll
            for (int j = 0; j < V / 2 + kShift; ++j) w[j] = n > 0 && 2 * j < (n < V ? n : V) + shift ? q[j] : 0u;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < V * static_cast<int>(sizeof(T)) / 4 + kShift; ++j) w[j] = 0u;
    }
    // odd: of the pointer they were fetched from.  n: zeros after the first n.
    __device__ __forceinline__ void values(bool odd, float* x, int n = V) const {
        Raw<T, V> k;
#pragma unroll
        for (int j = 0; j < Raw<T, V>::N; ++j) {
            if constexpr (kShift) k.w[j] = odd ? __byte_perm(w[j], w[j + 1], 0x5432) : w[j];
            else k.w[j] = w[j];
            if (sizeof(T) == 2 && 2 * j + 2 > n) k.w[j] = 2 * j + 1 == n ? k.w[j] & 0xffffu : 0u;
        }
        widen(k, x);
    }
};
// V values to p of any alignment (of T's), as they lie in memory.
template <class T, int V>
__device__ __forceinline__ void store_words(T* p, const Raw<T, V>& k) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = __uint_as_float(k.w[j]);
    } else if (reinterpret_cast<uintptr_t>(p) & 2) {
        uint16_t* q = reinterpret_cast<uint16_t*>(p);
        q[0] = static_cast<uint16_t>(k.w[0]);
#pragma unroll
        for (int j = 0; j + 1 < V / 2; ++j)
            *reinterpret_cast<uint32_t*>(q + 1 + 2 * j) = __byte_perm(k.w[j], k.w[j + 1], 0x5432);
        q[V - 1] = static_cast<uint16_t>(k.w[V / 2 - 1] >> 16);
    } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) reinterpret_cast<uint32_t*>(p)[j] = k.w[j];
    }
}
template <class T, int V>
__device__ __forceinline__ void store_any(T* p, const float (&x)[V]) {
    Raw<T, V> k;
    narrow(x, k);
    store_words(p, k);
}

// The first n of V values (all, for more; none, for n <= 0).
template <class T, int V>
__device__ __forceinline__ void store_some(T* p, const float (&x)[V], int n) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) p[j] = x[j];
    } else {
        Raw<T, V> k;
        narrow(x, k);
        n = n < V ? n : V;
        const int shift = (reinterpret_cast<uintptr_t>(p) >> 1) & 1;
        uint16_t* q = reinterpret_cast<uint16_t*>(p);
        if (shift && n > 0) q[0] = static_cast<uint16_t>(k.w[0]);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const uint32_t u = shift && j + 1 < V / 2 ? __byte_perm(k.w[j], k.w[j + 1 < V / 2 ? j + 1 : j], 0x5432) : k.w[j];
            if (2 * j + 1 + shift < n) *reinterpret_cast<uint32_t*>(q + 2 * j + shift) = u;
        }
        if (n > shift && (n - shift) % 2) {  // the last value is alone in its word
            uint32_t u = k.w[0];
#pragma unroll
            for (int j = 1; j < V / 2; ++j) u = (n - 1) / 2 == j ? k.w[j] : u;
            q[n - 1] = static_cast<uint16_t>((n - 1) % 2 ? u >> 16 : u);
        }
    }
}

// Two floats an instruction.
struct Pair {
    uint64_t v;
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Pair(uint64_t x) : v(x) {}
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
    return Pair(r);
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
    return Pair(r);
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.v), "l"(b.v), "l"(c.v));
    return Pair(r);
}

// max(a, |b|) that keeps a NaN (fmaxf drops it).
__device__ __forceinline__ float max_mag(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The exponent byte of a block whose largest magnitude is `most`.  127 is
// 1.984375 * 2^6, so e is the exponent of max|x| less 6, or one more when its
// mantissa is above 1.984375.
__device__ __forceinline__ int exponent8(float most, int emin) {
    const uint32_t m = __float_as_uint(most);
    if (m >= 0x7f800000u) return kBad8;
    const int e = static_cast<int>(m >> 23) - 133 + ((m & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return (e > emin ? e : emin) + 127;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// 2^-e, the factor from values to codes (0 for a bad block: its finite values
// get the code 0, the others any; all of them restore as NaN).
__device__ __forceinline__ float encode8(int byte) { return byte == kBad8 ? 0.0f : pow2f(127 - byte); }
// 2^e, the factor from codes to values (NaN for a bad block).
__device__ __forceinline__ float decode8(int byte) {
    return byte == kBad8 ? __uint_as_float(0x7fffffffu) : pow2f(byte - 127);
}
// Four codes as one word (inv = encode8(byte)).  x * inv + 1.5 * 2^23 rounds
// x * inv to the nearest integer, ties to even, and leaves its two's
// complement in the low bits: one FMA a value where a conversion instruction
// runs at an eighth of that rate.  At the type's greatest exponent 64 * 2^e
// would overflow it.
__device__ __forceinline__ uint32_t codes4(float x0, float x1, float x2, float x3, float inv, int byte, int top) {
    constexpr float kMagic = 12582912.0f;
    float r[4] = {x0, x1, x2, x3};
    if (byte == top) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __fmul_rn(fminf(fmaxf(__fmul_rn(r[j], inv), -63.0f), 63.0f), pow2f(byte - 127));
    }
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = __float_as_uint(fmaf(r[j], inv, kMagic));
    return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
}
__device__ __forceinline__ int8_t code8(float x, float inv, int byte, int top) {
    return static_cast<int8_t>(codes4(x, x, x, x, inv, byte, top) & 0xff);
}
// The values of four codes: the byte b + 128 in the mantissa of 2^23, less
// 2^23 + 128, is b; the product with 2^e is exact, so one FMA does both
// (beyond 2^100 its addend would overflow).
__device__ __forceinline__ void values4(uint32_t codes, int byte, float* x) {
    const uint32_t u = codes ^ 0x80808080u;
    const float scale = decode8(byte);
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + j));
    if (byte <= 227) {
        const float off = __fmul_rn(-8388736.0f, scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fmaf(f[j], scale, off);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __fmul_rn(__fsub_rn(f[j], 8388736.0f), scale);
    }
}
// V codes at p, aligned to V bytes.
template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const float* x, float inv, int byte, int top) {
    Raw<int8_t, V> k;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) k.w[j] = codes4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3], inv, byte, top);
    *reinterpret_cast<Raw<int8_t, V>*>(p) = k;
}
// The first n of them.
template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const float* x, float inv, int byte, int top, int n) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        const uint32_t u = codes4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3], inv, byte, top);
        if (4 * j + 4 <= n) {
            *reinterpret_cast<uint32_t*>(p + 4 * j) = u;
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (4 * j + i < n) p[4 * j + i] = static_cast<int8_t>(u >> 8 * i & 0xff);
        }
    }
}
// The first n of V codes at p (all, for more); p is aligned to 4 bytes.  Whole
// words that hold one of them are read: what follows the n is any code.
template <int V>
__device__ __forceinline__ Raw<int8_t, V> load_codes(const int8_t* p, int n) {
    Raw<int8_t, V> k;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) k.w[j] = 4 * j < n ? reinterpret_cast<const uint32_t*>(p)[j] : 0u;
    return k;
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
__device__ __forceinline__ float reduce_max(float x) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
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

// y = the values of a saved matrix (save8.cu).
template <class T>
void restore8(int64_t rows, int64_t cols, const Saved8& s, T* y, int64_t ldy, cudaStream_t stream);

// ── Activations and their slopes ─────────────────────────────────────────
// The choice is made once for V values.  GELU's 1/2 (1 + tanh u) is computed
// as 1 / (1 + e^-2u), which equals it, does not cancel where tanh u is near
// -1, and costs one exponential and one reciprocal.  FAST (for results of 16
// bits) takes the hardware's exponential, whose error of 2^-19 or less here
// is lost in the result's rounding of 2^-8 or 2^-11 where nothing cancels (for
// ELU near zero see expm1_f); with tanhf the 8-bit activation passes were bound
// by arithmetic (131,072 x 1024 bf16, forward and backward: 0.52 ms, and 0.29
// with it).
__device__ __forceinline__ float exp2_hw(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));  // within 2^-22; 2^-inf = 0
    return r;
}
template <bool FAST>
__device__ __forceinline__ float exp_f(float x) { return FAST ? __expf(x) : expf(x); }
// e^x - 1 for x <= 0.  The difference loses what 1 has more bits than e^x - 1;
// where that would show the series is summed instead.  FAST: four terms above
// -1/16 (the fifth is below 2^-22 of the sum; below -1/16 the difference is
// within 2^-17).  fp32: nine terms above -1/2 (the tenth is below 2^-30 of the
// sum; below, the hardware's exponential is within 2^-22 and the difference
// within 2^-21).  131,072 x 1,024 fp32 with the 8-bit copy: 223 us, 270 with
// expm1f, and 240 by expf's difference alone.
template <bool FAST>
__device__ __forceinline__ float expm1_f(float x) {
    float q = FAST ? 1.0f / 24.0f : 1.0f / 362880.0f;
    if (!FAST) {
        q = fmaf(x, q, 1.0f / 40320.0f);
        q = fmaf(x, q, 1.0f / 5040.0f);
        q = fmaf(x, q, 1.0f / 720.0f);
        q = fmaf(x, q, 1.0f / 120.0f);
        q = fmaf(x, q, 1.0f / 24.0f);
    }
    q = fmaf(x, q, 1.0f / 6.0f);
    q = fmaf(x, q, 0.5f);
    q = fmaf(__fmul_rn(x, x), q, x);
    return x > (FAST ? -0.0625f : -0.5f) ? q : __fsub_rn(exp2_hw(__fmul_rn(x, 1.4426950409f)), 1.0f);
}
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));  // 1 ulp; 1 / inf = 0
    return r;
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_f(float x) { return reciprocal(__fadd_rn(1.0f, exp_f<FAST>(-x))); }

// 1 / (1 + e^-2u), 2u = 2 c (x + d x^3), c = sqrt(2 / pi), d = 0.044715; the
// fast form takes 2^(-2u log2 e) with the factor in the constants.
template <bool FAST>
__device__ __forceinline__ float gelu_s(float x, float x2) {
    if (FAST) {
        return reciprocal(__fadd_rn(1.0f, exp2_hw(__fmul_rn(x, fmaf(-0.102943239f, x2, -2.302208198f)))));
    }
    return sigmoid_f<false>(__fmul_rn(x, fmaf(0.0713548162726f, x2, 1.5957691216f)));
}

template <int V, class F>
__device__ __forceinline__ void map_v(float (&x)[V], F&& f) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = f(x[j]);
}

// x <- act(x)
// ACT is the activation where it is known at compile time, else -1.
template <bool FAST, int ACT = -1, int V>
__device__ __forceinline__ void act_forward(float (&x)[V], int act, float alpha) {
    switch (ACT >= 0 ? ACT : act) {
        case TG_ACT_RELU: map_v(x, [](float v) { return v < 0.0f ? 0.0f : v; }); break;  // NaN stays NaN
        case TG_ACT_LEAKY_RELU: map_v(x, [alpha](float v) { return v >= 0.0f ? v : __fmul_rn(alpha, v); }); break;
        case TG_ACT_ELU:
            // (without a branch: a warp's values have both signs)
            map_v(x, [alpha](float v) {
                const float e = __fmul_rn(alpha, expm1_f<FAST>(fminf(v, 0.0f)));
                return v < 0.0f ? e : v;
            });
            break;
        case TG_ACT_SIGMOID: map_v(x, [](float v) { return sigmoid_f<FAST>(v); }); break;
        case TG_ACT_TANH: map_v(x, [](float v) { return tanhf(v); }); break;
        case TG_ACT_GELU:
            // below -16 the product is 0 in fp32 (and -inf * 0 would not be)
            map_v(x, [](float v) {
                v = max_nan(v, -16.0f);
                return __fmul_rn(v, gelu_s<FAST>(v, __fmul_rn(v, v)));
            });
            break;
        default: break;
    }
}

// x <- act'(x)
template <bool FAST, int ACT = -1, int V>
__device__ __forceinline__ void act_slope(float (&x)[V], int act, float alpha) {
    switch (ACT >= 0 ? ACT : act) {
        case TG_ACT_RELU: map_v(x, [](float v) { return v > 0.0f ? 1.0f : (v <= 0.0f ? 0.0f : v); }); break;
        case TG_ACT_LEAKY_RELU:
            map_v(x, [alpha](float v) { return v >= 0.0f ? 1.0f : (v < 0.0f ? alpha : v); });
            break;
        case TG_ACT_ELU:
            map_v(x, [alpha](float v) { return v < 0.0f ? __fmul_rn(alpha, exp_f<FAST>(v)) : (v >= 0.0f ? 1.0f : v); });
            break;
        case TG_ACT_SIGMOID:
            map_v(x, [](float v) {
                // s (1 - s) = e / (1 + e)^2, e = e^-|v|: 1 - s would cancel
                const float e = exp_f<FAST>(-fabsf(v)), s = reciprocal(__fadd_rn(1.0f, e));
                return __fmul_rn(__fmul_rn(e, s), s);
            });
            break;
        case TG_ACT_TANH:
            map_v(x, [](float v) {
                // 1 - tanh^2 = 4 e / (1 + e)^2, e = e^-2|v|
                const float e = exp_f<FAST>(__fmul_rn(-2.0f, fabsf(v))), s = reciprocal(__fadd_rn(1.0f, e));
                return __fmul_rn(__fmul_rn(4.0f, e), __fmul_rn(s, s));
            });
            break;
        case TG_ACT_GELU:
            // s = 1 / (1 + e^-2u): act' = s + x s (1 - s) (2u)',  (2u)' = 2 c (1 + 3 d x^2).
            // Beyond |x| = 16 s is 0 or 1 in fp32, and (2u)' may overflow.
            map_v(x, [](float v) {
                v = min_nan(max_nan(v, -16.0f), 16.0f);
                const float v2 = __fmul_rn(v, v);
                const float s = gelu_s<FAST>(v, v2);
                const float du = fmaf(0.2140644488f, v2, 1.5957691216f);
                return fmaf(__fmul_rn(v, fmaf(-s, s, s)), du, s);
            });
            break;
        default: map_v(x, [](float) { return 1.0f; }); break;
    }
}

// Calls f with the activation as a compile-time constant.
template <class F>
void by_act(int act, F&& f) {
    using std::integral_constant;
    switch (act) {
        case TG_ACT_RELU: f(integral_constant<int, TG_ACT_RELU>{}); break;
        case TG_ACT_ELU: f(integral_constant<int, TG_ACT_ELU>{}); break;
        case TG_ACT_LEAKY_RELU: f(integral_constant<int, TG_ACT_LEAKY_RELU>{}); break;
        case TG_ACT_SIGMOID: f(integral_constant<int, TG_ACT_SIGMOID>{}); break;
        case TG_ACT_TANH: f(integral_constant<int, TG_ACT_TANH>{}); break;
        case TG_ACT_GELU: f(integral_constant<int, TG_ACT_GELU>{}); break;
        default: f(integral_constant<int, TG_ACT_NONE>{});
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

// Without codes (where they are not `needed`) nothing is saved; with them the
// exponents have to be there too.
inline void check_saved8(const char* fn, int64_t cols, const Saved8& s, bool needed) {
    check_ptr(fn, "codes", s.codes, needed);
    check_ptr(fn, "exponents", s.exps, needed || s.codes);
    if (!s.codes) return;
    check_ld(fn, "codes", s.ld, cols);
    check_ld(fn, "exponents", s.lde, ceil_div(cols, kBlock8));
    if (!rows_aligned16(s.codes, s.ld, 1)) invalid(std::string(fn) + ": rows of codes must start 16-byte aligned");
}

}  // namespace tg

// ============================================================================
//  save8.cu -- 8-bit saved activations: an activation that keeps its input in
//  8 bits, the values back, and the activation's backward pass from them.
//
//  All three read and write each value once (the form is in values.cuh) and
//  are bound by HBM.  A unit of work is one block of 128 columns of one row:
//  its exponent needs the largest of the 128 magnitudes, which one warp's (or,
//  at 8 values a lane, half a warp's) shuffles give, so values stay in
//  registers between the read and the two writes.
// ============================================================================
#include <algorithm>

#include "values.cuh"

namespace tg {

namespace {

// Lane mapping of one block: G lanes, V values each.  Aligned rows: 16 bytes
// a lane, contiguous.  Others: 32 lanes, 4 values each, 32 columns apart.
template <class T, bool ALIGNED>
struct Lanes {
    static constexpr int V = ALIGNED ? 16 / static_cast<int>(sizeof(T)) : 4;
    static constexpr int G = kBlock8 / V;
    static __device__ __forceinline__ int col(int lane, int j) { return ALIGNED ? lane * V + j : j * 32 + lane; }
    // The lane's values of the block starting at p, of which `left` columns exist.
    static __device__ __forceinline__ void load(const T* p, int lane, int64_t left, float (&x)[V]) {
        if (ALIGNED && (lane + 1) * V <= left) {
            load_v<T, V>(p + lane * V, x);
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = col(lane, j) < left ? to_f32(p[col(lane, j)]) : 0.0f;
    }
    static __device__ __forceinline__ void store(T* p, int lane, int64_t left, const float (&x)[V]) {
        if (ALIGNED && (lane + 1) * V <= left) {
            store_v<T, V>(p + lane * V, x);
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (col(lane, j) < left) p[col(lane, j)] = from_f32<T>(x[j]);
    }
    static __device__ __forceinline__ void store_codes(int8_t* p, int lane, int64_t left, const float (&x)[V],
                                                       float inv, int byte, int top) {
        Pack<int8_t, V> k;
#pragma unroll
        for (int j = 0; j < V; ++j) k.v[j] = code8(x[j], inv, byte, top);
        if (ALIGNED && (lane + 1) * V <= left) {
            *reinterpret_cast<Pack<int8_t, V>*>(p + lane * V) = k;
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (col(lane, j) < left) p[col(lane, j)] = k.v[j];
    }
    static __device__ __forceinline__ void load_codes(const int8_t* p, int lane, int64_t left, float scale,
                                                      float (&x)[V]) {
        Pack<int8_t, V> k;
        if (ALIGNED && (lane + 1) * V <= left) {
            k = *reinterpret_cast<const Pack<int8_t, V>*>(p + lane * V);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) k.v[j] = col(lane, j) < left ? p[col(lane, j)] : int8_t(0);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = __fmul_rn(static_cast<float>(k.v[j]), scale);
    }
};

struct ActArgs {
    int64_t rows, cols, nb;  // nb blocks a row
    int act;
    float alpha;
    Range8 r8;
};

// y = act(x) (y nullable), saved = x in 8 bits.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) save8_kernel(ActArgs a, const T* x, int64_t ldx, T* y, int64_t ldy, Saved8 o) {
    using L = Lanes<T, ALIGNED>;
    const int lane = threadIdx.x % L::G;
    const int64_t total = a.rows * a.nb, step = static_cast<int64_t>(gridDim.x) * (256 / L::G);
    // Every lane of a warp takes part in the shuffles: the bound is the warp's first unit.
    int64_t u = static_cast<int64_t>(blockIdx.x) * (256 / L::G) + threadIdx.x / L::G;
    const int64_t first = static_cast<int>(threadIdx.x / 32 * (32 / L::G)) - static_cast<int>(threadIdx.x / L::G);  // this warp's first unit, less u
    for (; u + first < total; u += step) {
        const bool live = u < total;
        const int64_t row = live ? u / a.nb : 0, b = live ? u - row * a.nb : 0;
        const int64_t c0 = b * kBlock8, left = live ? a.cols - c0 : 0;
        float v[L::V];
        L::load(x + row * ldx + c0, lane, left, v);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < L::V; ++j) m = max(m, mag_bits(v[j]));
        const int byte = exponent8(reduce_max<L::G>(m), a.r8.emin);
        L::store_codes(o.codes + row * o.ld + c0, lane, left, v, encode8(byte), byte, a.r8.top);
        if (live && lane == 0) o.exps[row * o.lde + b] = static_cast<uint8_t>(byte);
        if (y) {
            act_forward(v, a.act, a.alpha);
            L::store(y + row * ldy + c0, lane, left, v);
        }
    }
}

// y = the values of a saved matrix.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) restore8_kernel(ActArgs a, Saved8 s, T* y, int64_t ldy) {
    using L = Lanes<T, ALIGNED>;
    const int lane = threadIdx.x % L::G;
    const int64_t total = a.rows * a.nb, step = static_cast<int64_t>(gridDim.x) * (256 / L::G);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * (256 / L::G) + threadIdx.x / L::G; u < total; u += step) {
        const int64_t row = u / a.nb, b = u - row * a.nb, c0 = b * kBlock8;
        float v[L::V];
        L::load_codes(s.codes + row * s.ld + c0, lane, a.cols - c0, decode8(s.exps[row * s.lde + b]), v);
        L::store(y + row * ldy + c0, lane, a.cols - c0, v);
    }
}

// dx = dy * act'(x), x given as it was or in 8 bits.
template <class T, bool ALIGNED, bool SAVED>
__global__ void __launch_bounds__(256) act_grad_kernel(ActArgs a, const T* dy, int64_t lddy, const T* x, int64_t ldx,
                                                       Saved8 s, T* dx, int64_t lddx) {
    using L = Lanes<T, ALIGNED>;
    const int lane = threadIdx.x % L::G;
    const int64_t total = a.rows * a.nb, step = static_cast<int64_t>(gridDim.x) * (256 / L::G);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * (256 / L::G) + threadIdx.x / L::G; u < total; u += step) {
        const int64_t row = u / a.nb, b = u - row * a.nb, c0 = b * kBlock8, left = a.cols - c0;
        float v[L::V], g[L::V];
        if (SAVED) L::load_codes(s.codes + row * s.ld + c0, lane, left, decode8(s.exps[row * s.lde + b]), v);
        else L::load(x + row * ldx + c0, lane, left, v);
        L::load(dy + row * lddy + c0, lane, left, g);
        act_slope(v, a.act, a.alpha);
#pragma unroll
        for (int j = 0; j < L::V; ++j) g[j] = __fmul_rn(g[j], v[j]);
        L::store(dx + row * lddx + c0, lane, left, g);
    }
}

unsigned grid_for(int64_t units, int per_block) {
    const int64_t want = ceil_div(units, per_block);
    return static_cast<unsigned>(std::min<int64_t>(want, int64_t(num_sms()) * 8));
}

template <class T>
bool aligned(const void* p, int64_t ld) {
    return p == nullptr || rows_aligned16(p, ld, sizeof(T));
}

}  // namespace

}  // namespace tg

extern "C" {

TG_API tg_status tg_save8(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ldx, int32_t act,
                          float alpha, void* y, int64_t ldy, int8_t* codes, int64_t ld_codes, uint8_t* exponents,
                          int64_t ld_exponents, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "save8";
        check_rows_cols(fn, rows, cols);
        check_dtype(fn, "x", dtype);
        check_act(fn, act);
        check_ptr(fn, "x", x, rows > 0);
        check_ld(fn, "x", ldx, cols);
        if (y) check_ld(fn, "y", ldy, cols);
        const Saved8 o{codes, ld_codes, exponents, ld_exponents};
        check_saved8(fn, cols, o, rows > 0);
        const ActArgs a{rows, cols, ceil_div(cols, kBlock8), act, alpha, range8(dtype)};
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const T* xp = static_cast<const T*>(x);
            T* yp = static_cast<T*>(y);
            const bool al = aligned<T>(x, ldx) && aligned<T>(y, ldy);
            auto kern = al ? save8_kernel<T, true> : save8_kernel<T, false>;
            const int per = 256 / (al ? Lanes<T, true>::G : Lanes<T, false>::G);
            launch("save8", kern, dim3(grid_for(rows * a.nb, per)), dim3(256), 0, as_stream(stream), a, xp, ldx, yp,
                   ldy, o);
        });
    });
}

TG_API tg_status tg_restore8(int64_t rows, int64_t cols, const int8_t* codes, int64_t ld_codes,
                             const uint8_t* exponents, int64_t ld_exponents, int32_t dtype, void* y, int64_t ldy,
                             void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "restore8";
        check_rows_cols(fn, rows, cols);
        check_dtype(fn, "y", dtype);
        check_ptr(fn, "y", y, rows > 0);
        check_ld(fn, "y", ldy, cols);
        const Saved8 s{const_cast<int8_t*>(codes), ld_codes, const_cast<uint8_t*>(exponents), ld_exponents};
        check_saved8(fn, cols, s, rows > 0);
        const ActArgs a{rows, cols, ceil_div(cols, kBlock8), TG_ACT_NONE, 0.0f, range8(dtype)};
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const bool al = aligned<T>(y, ldy);
            auto kern = al ? restore8_kernel<T, true> : restore8_kernel<T, false>;
            const int per = 256 / (al ? Lanes<T, true>::G : Lanes<T, false>::G);
            launch("restore8", kern, dim3(grid_for(rows * a.nb, per)), dim3(256), 0, as_stream(stream), a, s,
                   static_cast<T*>(y), ldy);
        });
    });
}

TG_API tg_status tg_activation_grad(int64_t rows, int64_t cols, int32_t dtype, const void* dy, int64_t lddy,
                                    const void* x, int64_t ldx, const int8_t* codes, int64_t ld_codes,
                                    const uint8_t* exponents, int64_t ld_exponents, int32_t act, float alpha,
                                    void* dx, int64_t lddx, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "activation_grad";
        check_rows_cols(fn, rows, cols);
        check_dtype(fn, "dy", dtype);
        check_act(fn, act);
        check_ptr(fn, "dy", dy, rows > 0);
        check_ptr(fn, "dx", dx, rows > 0);
        check_ld(fn, "dy", lddy, cols);
        check_ld(fn, "dx", lddx, cols);
        if ((x != nullptr) == (codes != nullptr) && rows > 0)
            invalid(std::string(fn) + ": exactly one of x and codes is given");
        if (x) check_ld(fn, "x", ldx, cols);
        const Saved8 s{const_cast<int8_t*>(codes), ld_codes, const_cast<uint8_t*>(exponents), ld_exponents};
        check_saved8(fn, cols, s, codes != nullptr);
        const ActArgs a{rows, cols, ceil_div(cols, kBlock8), act, alpha, range8(dtype)};
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const T* dyp = static_cast<const T*>(dy);
            const T* xp = static_cast<const T*>(x);
            T* dxp = static_cast<T*>(dx);
            const bool al = aligned<T>(dy, lddy) && aligned<T>(x, ldx) && aligned<T>(dx, lddx);
            auto kern = codes ? (al ? act_grad_kernel<T, true, true> : act_grad_kernel<T, false, true>)
                              : (al ? act_grad_kernel<T, true, false> : act_grad_kernel<T, false, false>);
            const int per = 256 / (al ? Lanes<T, true>::G : Lanes<T, false>::G);
            launch("activation_grad", kern, dim3(grid_for(rows * a.nb, per)), dim3(256), 0, as_stream(stream), a, dyp,
                   lddy, xp, ldx, s, dxp, lddx);
        });
    });
}

}  // extern "C"

// ============================================================================
//  save8.cu -- 8-bit saved activations: an activation that keeps its input in
//  8 bits, the values back, and the activation's backward pass from them.
//
//  All three read and write each value once (the form is in values.cuh).
//  Aligned rows are bound by HBM and, with an exponential and the codes'
//  rounding, by issue slots (131,072 x 1,024 bf16 GELU: 132 us forward, 134
//  back, bytes 104 each; DRAM 56 %, issue 62-65 %).  Rows that are not 16-byte
//  aligned move 4 bytes at a time (131,072 x 1,023: 303 and 201 us).  A block of 128 columns of one row is the work of G lanes
//  (16 bytes a lane: half a warp for 16-bit values, a warp for fp32): the
//  block's exponent is a shuffle reduction over values that stay in registers
//  between the read and the two writes.  A group keeps its columns and walks
//  the rows R apart, U rows at a time: the loads of U rows are in flight
//  together, and no row costs a division.
// ============================================================================
#include <algorithm>

#include "values.cuh"

namespace tg {

namespace {

// Lane mapping of one block: G lanes, 16 bytes of neighbouring values each
// (ALIGNED: one access, and no row ends inside a lane's).
template <class T, bool ALIGNED>
struct Lanes {
    static constexpr int V = 16 / static_cast<int>(sizeof(T));
    static constexpr int G = kBlock8 / V;
    static constexpr int U = ALIGNED ? 4 : 2;  // rows in flight
    static constexpr int kResident = ALIGNED ? 3 : 4;  // blocks of 256 threads a SM
    int lane, left;   // of the block's columns, `left` exist
    bool full;        // the lane's values are all there

    __device__ __forceinline__ Lanes(int64_t columns_left) {
        lane = threadIdx.x % G;
        left = columns_left < kBlock8 ? static_cast<int>(columns_left) : kBlock8;
        full = (lane + 1) * V <= left;
    }
    // Of the row whose block starts at p.
    __device__ __forceinline__ void load(const T* p, bool live, Held<T, V, ALIGNED>& k) const {
        if (full && live) k.fetch(p + lane * V);
        else if (!ALIGNED) k.fetch(p + lane * V, live ? left - lane * V : 0);
        else k.zero();
    }
    __device__ __forceinline__ void values(const Held<T, V, ALIGNED>& k, const T* p, float (&x)[V]) const {
        if (ALIGNED) k.values(false, x);
        else k.values(k.odd(p + lane * V), x, left - lane * V);
    }
    __device__ __forceinline__ void store(T* p, const float (&x)[V]) const {
        if constexpr (ALIGNED) {
            if (full) store_v<T, V>(p + lane * V, x);
        } else if (full) {
            store_any<T, V>(p + lane * V, x);
        } else {
            store_some<T, V>(p + lane * V, x, left - lane * V);
        }
    }
    __device__ __forceinline__ void save(int8_t* p, const float (&x)[V], int byte, int top) const {
        const float inv = encode8(byte);
        if (full) store_codes<V>(p + lane * V, x, inv, byte, top);
        else if (!ALIGNED) store_codes<V>(p + lane * V, x, inv, byte, top, left - lane * V);
    }
    __device__ __forceinline__ Raw<int8_t, V> codes(const int8_t* p, bool live) const {
        if (full && live) return *reinterpret_cast<const Raw<int8_t, V>*>(p + lane * V);
        return load_codes<V>(p + lane * V, live && !ALIGNED ? left - lane * V : 0);
    }
    static __device__ __forceinline__ void values(const Raw<int8_t, V>& k, int byte, float (&x)[V]) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) values4(k.w[j], byte, x + 4 * j);
    }
};

// The block of columns that this thread's group keeps, and its rows: row0,
// row0 + step, ...  base: the least row0 of the warp (every lane of a warp
// takes part in the shuffles, so a warp's loop runs on base).
struct Walk {
    int64_t b, row0, base, step;
};
template <int G>
__device__ __forceinline__ Walk walk(int64_t rows, int64_t nb) {
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (256 / G);
    const int64_t id = static_cast<int64_t>(blockIdx.x) * (256 / G) + threadIdx.x / G;
    Walk w;
    w.step = groups / nb;
    w.row0 = id / nb;
    w.b = id - w.row0 * nb;
    w.base = __shfl_sync(0xffffffffu, w.row0, 0);
    if (w.row0 >= w.step) w.row0 = rows;  // a group left over: no rows
    return w;
}

struct ActArgs {
    int64_t rows, cols, nb;  // nb blocks a row
    int act;
    float alpha;
    Range8 r8;
};

// y = act(x) (y nullable), saved = x in 8 bits.  ACT: as in act_forward.
template <class T, bool ALIGNED, int ACT>
__global__ void __launch_bounds__(256, Lanes<T, ALIGNED>::kResident) save8_kernel(ActArgs a, const T* x, int64_t ldx, T* y,
                                                                     int64_t ldy, Saved8 o) {
    using L = Lanes<T, ALIGNED>;
    constexpr int V = L::V, U = L::U;
    wait_for_previous();
    const Walk w = walk<L::G>(a.rows, a.nb);
    const int64_t c0 = w.b * kBlock8;
    const L l(a.cols - c0);
    const bool forward = y != nullptr;
    // pointers to the group's rows, a step at a time (multiples of the steps
    // would be kept in registers)
    const int64_t first = w.row0 < a.rows ? w.row0 : 0;
    const T* px = x + first * ldx + c0;
    T* py = y + (forward ? first * ldy + c0 : 0);
    int8_t* pc = o.codes + first * o.ld + c0;
    uint8_t* pe = o.exps + first * o.lde + w.b;
    const int64_t dx = w.step * ldx, dy = w.step * ldy, dc = w.step * o.ld, de = w.step * o.lde;
    for (int64_t base = w.base, row = w.row0; base < a.rows; base += U * w.step, row += U * w.step) {
        Held<T, V, ALIGNED> k[U];
        const T* at = px;
#pragma unroll
        for (int u = 0; u < U; ++u, px += dx) l.load(px, row + u * w.step < a.rows, k[u]);
#pragma unroll
        for (int u = 0; u < U; ++u, at += dx, py += dy, pc += dc, pe += de) {
            float v[V];
            l.values(k[u], at, v);
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) m = max_mag(m, v[j]);
            const int byte = exponent8(reduce_max<L::G>(m), a.r8.emin);
            if (row + u * w.step < a.rows) {
                l.save(pc, v, byte, a.r8.top);
                if (l.lane == 0) *pe = static_cast<uint8_t>(byte);
                if (forward) {
                    act_forward<sizeof(T) == 2, ACT>(v, a.act, a.alpha);
                    l.store(py, v);
                }
            }
            __syncwarp();
        }
    }
}

// y = the values of a saved matrix.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) restore8_kernel(ActArgs a, Saved8 s, T* y, int64_t ldy) {
    using L = Lanes<T, ALIGNED>;
    wait_for_previous();
    const Walk w = walk<L::G>(a.rows, a.nb);
    const int64_t c0 = w.b * kBlock8;
    const L l(a.cols - c0);
    constexpr int U = L::U;
    for (int64_t row = w.row0; row < a.rows; row += U * w.step) {
        Raw<int8_t, L::V> c[U];
        int e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row + u * w.step;
            const bool live = r < a.rows;
            c[u] = l.codes(s.codes + (live ? r : row) * s.ld + c0, live);
            e[u] = live ? s.exps[r * s.lde + w.b] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row + u * w.step;
            if (r >= a.rows) break;
            float v[L::V];
            L::values(c[u], e[u], v);
            l.store(y + r * ldy + c0, v);
        }
    }
}

// dx = dy * act'(x), x given as it was or in 8 bits.
template <class T, bool ALIGNED, bool SAVED, int ACT>
__global__ void __launch_bounds__(256, Lanes<T, ALIGNED>::kResident) act_grad_kernel(ActArgs a, const T* dy, int64_t lddy,
                                                                        const T* x, int64_t ldx, Saved8 s, T* dx,
                                                                        int64_t lddx) {
    using L = Lanes<T, ALIGNED>;
    constexpr int V = L::V, U = L::U;
    wait_for_previous();
    const Walk w = walk<L::G>(a.rows, a.nb);
    const int64_t c0 = w.b * kBlock8;
    const L l(a.cols - c0);
    if (w.row0 >= a.rows) return;
    const T *pg = dy + w.row0 * lddy + c0, *px = SAVED ? nullptr : x + w.row0 * ldx + c0;
    const int8_t* pc = SAVED ? s.codes + w.row0 * s.ld + c0 : nullptr;
    const uint8_t* pe = SAVED ? s.exps + w.row0 * s.lde + w.b : nullptr;
    T* po = dx + w.row0 * lddx + c0;
    const int64_t dg = w.step * lddy, dX = w.step * ldx, dc = w.step * s.ld, de = w.step * s.lde, dout = w.step * lddx;
    for (int64_t row = w.row0; row < a.rows; row += U * w.step) {
        Held<T, V, ALIGNED> g[U], k[SAVED ? 1 : U];
        const T *at_g = pg, *at_x = px;
        Raw<int8_t, V> c[SAVED ? U : 1];
        int e[U];
#pragma unroll
        for (int u = 0; u < U; ++u, pg += dg) {
            const bool live = row + u * w.step < a.rows;
            l.load(pg, live, g[u]);
            if (SAVED) {
                c[SAVED ? u : 0] = l.codes(pc, live);
                e[u] = live ? *pe : 0;
                pc += dc;
                pe += de;
            } else {
                l.load(px, live, k[SAVED ? 0 : u]);
                px += dX;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u, po += dout, at_g += dg, at_x += dX) {
            if (row + u * w.step >= a.rows) break;
            float v[V], d[V];
            if (SAVED) L::values(c[SAVED ? u : 0], e[u], v);
            else l.values(k[SAVED ? 0 : u], at_x, v);
            act_slope<sizeof(T) == 2, ACT>(v, a.act, a.alpha);
            l.values(g[u], at_g, d);
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = __fmul_rn(d[j], v[j]);
            l.store(po, d);
        }
    }
}

// Blocks of 256 threads for rows x nb blocks of columns: a group each when all
// are resident at once, else as many as are (and one group for every block of
// columns).
template <class L>
unsigned grid_for(int64_t rows, int64_t nb) {
    const int per = 256 / L::G;
    const int64_t want = ceil_div(rows * nb, per),
                  most = std::max<int64_t>(ceil_div(nb, per), int64_t(num_sms()) * L::kResident);
    return static_cast<unsigned>(std::min(want, most));
}

// Rows that start, and end, at multiples of 16 bytes.
template <class T>
bool aligned(const void* p, int64_t ld, int64_t cols) {
    return p == nullptr || (cols * sizeof(T) % 16 == 0 && rows_aligned16(p, ld, sizeof(T)));
}

}  // namespace

template <class T>
void restore8(int64_t rows, int64_t cols, const Saved8& s, T* y, int64_t ldy, cudaStream_t stream) {
    const ActArgs a{rows, cols, ceil_div(cols, kBlock8), TG_ACT_NONE, 0.0f, Range8{}};
    const bool al = aligned<T>(y, ldy, cols);
    const unsigned grid = al ? grid_for<Lanes<T, true>>(rows, a.nb) : grid_for<Lanes<T, false>>(rows, a.nb);
    launch_dependent("restore8", al ? restore8_kernel<T, true> : restore8_kernel<T, false>,
                     dim3(grid), dim3(256), 0, stream, a, s, y, ldy);
}
template void restore8<float>(int64_t, int64_t, const Saved8&, float*, int64_t, cudaStream_t);
template void restore8<__nv_bfloat16>(int64_t, int64_t, const Saved8&, __nv_bfloat16*, int64_t, cudaStream_t);
template void restore8<__half>(int64_t, int64_t, const Saved8&, __half*, int64_t, cudaStream_t);

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
            const bool al = aligned<T>(x, ldx, cols) && aligned<T>(y, ldy, cols);
            auto kern = save8_kernel<T, false, -1>;
            if (al) by_act(act, [&](auto k) { kern = save8_kernel<T, true, decltype(k)::value>; });
            const unsigned grid = al ? grid_for<Lanes<T, true>>(rows, a.nb) : grid_for<Lanes<T, false>>(rows, a.nb);
            launch_dependent("save8", kern, dim3(grid), dim3(256), 0, as_stream(stream), a, xp, ldx, yp,
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
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            restore8<T>(rows, cols, s, static_cast<T*>(y), ldy, as_stream(stream));
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
            const bool al = aligned<T>(dy, lddy, cols) && aligned<T>(x, ldx, cols) && aligned<T>(dx, lddx, cols);
            auto kern = codes ? act_grad_kernel<T, false, true, -1> : act_grad_kernel<T, false, false, -1>;
            if (al)
                by_act(act, [&](auto k) {
                    constexpr int A = decltype(k)::value;
                    kern = codes ? act_grad_kernel<T, true, true, A> : act_grad_kernel<T, true, false, A>;
                });
            const unsigned grid = al ? grid_for<Lanes<T, true>>(rows, a.nb) : grid_for<Lanes<T, false>>(rows, a.nb);
            launch_dependent("activation_grad", kern, dim3(grid), dim3(256), 0, as_stream(stream), a, dyp,
                   lddy, xp, ldx, s, dxp, lddx);
        });
    });
}

}  // extern "C"

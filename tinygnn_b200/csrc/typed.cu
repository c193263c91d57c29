// ============================================================================
//  typed.cu -- rows sorted by type through their type's weight, and the
//  gradients (a typed, or grouped, linear map).
//
//      Y[r]  = act(X[r] . W[t(r)] + b[t(r)])        X: M x K, W: T x K x N
//      dX[r] = dY[r] . W[t(r)]^T
//      dW[t] = sum over its rows of X[r]^T dY[r],   db[t] = sum of dY[r]
//
//  Type t owns rows [offsets[t], offsets[t + 1]).  The offsets live on the
//  device and are never read back: blocks find their tile from them.  Any
//  offsets are safe to read through (each bound is clamped to [0, M]); rows
//  that no type owns are not written.
// ============================================================================
#include <algorithm>
#include <vector>

#include "typed.cuh"

namespace tg {

namespace {

// ── Products on the FP32 units ───────────────────────────────────────────
// Tiles of 64 rows and 128 columns, 256 threads of 4 rows x 8 columns, the
// inner dimension in steps of 16 through shared memory.  Thread (ty, tx)
// holds columns tx + 16 j: the 128 columns of a row, which share an exponent
// in the saved form, lie in the 16 lanes of half a warp.
constexpr int FM = 64, FN = 128, FK = 16;

template <class GetA, class GetB>
__device__ __forceinline__ void fma_tiles(float (&acc)[4][8], int64_t k0, int64_t k1, GetA&& a, GetB&& b) {
    __shared__ float As[FK][FM + 4], Bs[FK][FN];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int64_t k = k0; k < k1; k += FK) {
        for (int i = threadIdx.x; i < FM * FK; i += 256) {
            const int m = i / FK, kk = i % FK;
            As[kk][m] = k + kk < k1 ? a(m, k + kk) : 0.0f;
        }
        for (int i = threadIdx.x; i < FN * FK; i += 256) {
            const int kk = i / FN, n = i % FN;
            Bs[kk][n] = k + kk < k1 ? b(k + kk, n) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < FK; ++kk) {
            float av[4], bv[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) av[i] = As[kk][ty * 4 + i];
#pragma unroll
            for (int j = 0; j < 8; ++j) bv[j] = Bs[kk][tx + 16 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
}

// C rows [r0, r1) of one type = A . B (+ epilogue).  TRANS: B is W^T.
template <class T, bool TRANS>
__global__ void __launch_bounds__(256) typed_rows_kernel(RowsArgs<T> g) {
    __shared__ int sh_type, sh_begin, sh_end;
    if (threadIdx.x == 0) {
        int tile = blockIdx.x;
        sh_type = -1;
        for (int t = 0; t < g.types; ++t) {
            const int b = clamp_row(g.offsets[t], g.M), e = clamp_row(g.offsets[t + 1], g.M);
            const int n = e > b ? (e - b + FM - 1) / FM : 0;
            if (tile < n) {
                sh_type = t;
                sh_begin = b + tile * FM;
                sh_end = e;
                break;
            }
            tile -= n;
        }
    }
    __syncthreads();
    if (sh_type < 0) return;
    const int64_t r0 = sh_begin, r1 = sh_end, n0 = static_cast<int64_t>(blockIdx.y) * FN;
    const T* w = g.W + sh_type * g.stride_w;
    float acc[4][8] = {};
    fma_tiles(
        acc, 0, g.K, [&](int m, int64_t k) { return r0 + m < r1 ? to_f32(g.A[(r0 + m) * g.lda + k]) : 0.0f; },
        [&](int64_t k, int n) {
            if (n0 + n >= g.N) return 0.0f;
            return to_f32(TRANS ? w[(n0 + n) * g.ldw + k] : w[k * g.ldw + n0 + n]);
        });
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + ty * 4 + i;
        const bool live = r < r1;
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (g.bias && n < g.N) acc[i][j] += g.bias[sh_type * g.N + n];
            if (n < g.N) m = max(m, mag_bits(acc[i][j]));
        }
        if (g.saved.codes) {
            const int byte = exponent8(reduce_max<16>(m), g.r8.emin);
            const float inv = encode8(byte);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t n = n0 + tx + 16 * j;
                if (live && n < g.N) g.saved.codes[r * g.saved.ld + n] = code8(acc[i][j], inv, byte, g.r8.top);
            }
            if (live && tx == 0) g.saved.exps[r * g.saved.lde + blockIdx.y] = static_cast<uint8_t>(byte);
        }
        act_forward(acc[i], g.act, g.alpha);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (live && n < g.N) g.C[r * g.ldc + n] = from_f32<T>(acc[i][j]);
        }
    }
}

// dW of one type (blockIdx.z), 64 x 128 of it.
template <class T, class O, bool SAVED>
__global__ void __launch_bounds__(256) typed_weight_kernel(WeightArgs<T, O> g) {
    const int t = blockIdx.z;
    const int64_t b = clamp_row(g.offsets[t], g.M), e = clamp_row(g.offsets[t + 1], g.M);
    const int64_t k0 = static_cast<int64_t>(blockIdx.x) * FM, n0 = static_cast<int64_t>(blockIdx.y) * FN;
    float acc[4][8] = {};
    fma_tiles(
        acc, b, e,
        [&](int m, int64_t r) {
            const int64_t k = k0 + m;
            if (k >= g.K) return 0.0f;
            if (SAVED)
                return __fmul_rn(static_cast<float>(g.saved.codes[r * g.saved.ld + k]),
                                 decode8(g.saved.exps[r * g.saved.lde + k / kBlock8]));
            return to_f32(g.X[r * g.ldx + k]);
        },
        [&](int64_t r, int n) { return n0 + n < g.N ? to_f32(g.dY[r * g.lddy + n0 + n]) : 0.0f; });
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t k = k0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (k < g.K && n < g.N) g.dW[t * g.stride_dw + k * g.lddw + n] = from_f32<O>(acc[i][j]);
        }
}

// db of one type (blockIdx.y), 32 columns of it.
template <class T, class O>
__global__ void __launch_bounds__(256) typed_bias_kernel(WeightArgs<T, O> g) {
    __shared__ float sh[8][33];
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32, t = blockIdx.y;
    const int64_t b = clamp_row(g.offsets[t], g.M), e = clamp_row(g.offsets[t + 1], g.M);
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float sum = 0.0f;
    if (n < g.N)
        for (int64_t r = b + w; r < e; r += 8) sum += to_f32(g.dY[r * g.lddy + n]);
    sh[w][lane] = sum;
    __syncthreads();
    if (w == 0 && n < g.N) {
        sum = 0.0f;
        for (int q = 0; q < 8; ++q) sum += sh[q][lane];
        g.db[t * g.N + n] = sum;
    }
}

void check_typed(const char* fn, int64_t M, int64_t K, int64_t N, int64_t types, int dtype, const int32_t* offsets) {
    check_rows_cols(fn, M, K);
    check_rows_cols(fn, M, N);
    check_dtype(fn, "the rows", dtype);
    if (types < 1 || types > kMaxTypes)
        invalid(std::string(fn) + ": the number of types (" + std::to_string(types) + ") is outside [1, " +
                std::to_string(kMaxTypes) + "]");
    check_ptr(fn, "offsets", offsets, true);
}

void check_weight(const char* fn, const char* what, int64_t K, int64_t N, int64_t ld, int64_t stride) {
    check_ld(fn, what, ld, N);
    if (stride < (K - 1) * ld + N)
        invalid(std::string(fn) + ": the types of " + what + " overlap (stride " + std::to_string(stride) + ")");
}

}  // namespace

}  // namespace tg

extern "C" {

TG_API tg_status tg_typed_linear(int64_t rows, int64_t K, int64_t N, int64_t types, int32_t dtype, const void* X,
                                 int64_t ldx, const void* W, int64_t ldw, int64_t stride_w, const int32_t* offsets,
                                 const float* bias, int32_t act, float alpha, void* Y, int64_t ldy, int8_t* codes,
                                 int64_t ld_codes, uint8_t* exponents, int64_t ld_exponents, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "typed_linear";
        check_typed(fn, rows, K, N, types, dtype, offsets);
        check_act(fn, act);
        check_ptr(fn, "X", X, rows > 0);
        check_ptr(fn, "W", W, rows > 0);
        check_ptr(fn, "Y", Y, rows > 0);
        check_ld(fn, "X", ldx, K);
        check_ld(fn, "Y", ldy, N);
        check_weight(fn, "W", K, N, ldw, stride_w);
        const Saved8 s{codes, ld_codes, exponents, ld_exponents};
        check_saved8(fn, N, s, false);
        if (rows == 0) return;
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const RowsArgs<T> g{rows, K, N, static_cast<int>(types), static_cast<const T*>(X), ldx,
                                static_cast<const T*>(W), ldw, stride_w, offsets, bias, act, alpha,
                                static_cast<T*>(Y), ldy, s, range8(dtype)};
            launch("typed_linear", typed_rows_kernel<T, false>,
                   dim3(static_cast<unsigned>(ceil_div(rows, FM) + types), static_cast<unsigned>(ceil_div(N, FN))),
                   dim3(256), 0, as_stream(stream), g);
        });
    });
}

TG_API tg_status tg_typed_linear_grad_input(int64_t rows, int64_t K, int64_t N, int64_t types, int32_t dtype,
                                            const void* dY, int64_t lddy, const void* W, int64_t ldw, int64_t stride_w,
                                            const int32_t* offsets, void* dX, int64_t lddx, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "typed_linear_grad_input";
        check_typed(fn, rows, K, N, types, dtype, offsets);
        check_ptr(fn, "dY", dY, rows > 0);
        check_ptr(fn, "W", W, rows > 0);
        check_ptr(fn, "dX", dX, rows > 0);
        check_ld(fn, "dY", lddy, N);
        check_ld(fn, "dX", lddx, K);
        check_weight(fn, "W", K, N, ldw, stride_w);
        if (rows == 0) return;
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const RowsArgs<T> g{rows, N, K, static_cast<int>(types), static_cast<const T*>(dY), lddy,
                                static_cast<const T*>(W), ldw, stride_w, offsets, nullptr, TG_ACT_NONE, 0.0f,
                                static_cast<T*>(dX), lddx, Saved8{}, Range8{}};
            launch("typed_linear_grad_input", typed_rows_kernel<T, true>,
                   dim3(static_cast<unsigned>(ceil_div(rows, FM) + types), static_cast<unsigned>(ceil_div(K, FN))),
                   dim3(256), 0, as_stream(stream), g);
        });
    });
}

TG_API tg_status tg_typed_linear_grad_weight(int64_t rows, int64_t K, int64_t N, int64_t types, int32_t dtype,
                                             const void* X, int64_t ldx, const int8_t* codes, int64_t ld_codes,
                                             const uint8_t* exponents, int64_t ld_exponents, const void* dY,
                                             int64_t lddy, const int32_t* offsets, int32_t dw_dtype, void* dW,
                                             int64_t lddw, int64_t stride_dw, float* db, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "typed_linear_grad_weight";
        check_typed(fn, rows, K, N, types, dtype, offsets);
        if (dw_dtype != TG_F32 && dw_dtype != dtype)
            invalid(std::string(fn) + ": dW must be float32 or of the rows' type");
        check_ptr(fn, "dY", dY, rows > 0);
        check_ptr(fn, "dW", dW, true);
        check_ld(fn, "dY", lddy, N);
        check_weight(fn, "dW", K, N, lddw, stride_dw);
        if ((X != nullptr) == (codes != nullptr) && rows > 0)
            invalid(std::string(fn) + ": exactly one of X and codes is given");
        if (X) check_ld(fn, "X", ldx, K);
        const Saved8 s{const_cast<int8_t*>(codes), ld_codes, const_cast<uint8_t*>(exponents), ld_exponents};
        check_saved8(fn, K, s, codes != nullptr);
        const auto run = [&](auto t, auto o) {
            using T = decltype(t);
            using O = decltype(o);
            const WeightArgs<T, O> g{rows, K, N, static_cast<int>(types), static_cast<const T*>(X), ldx, s,
                                     static_cast<const T*>(dY), lddy, offsets, static_cast<O*>(dW), lddw, stride_dw,
                                     db};
            launch("typed_linear_grad_weight", codes ? typed_weight_kernel<T, O, true> : typed_weight_kernel<T, O, false>,
                   dim3(static_cast<unsigned>(ceil_div(K, FM)), static_cast<unsigned>(ceil_div(N, FN)),
                        static_cast<unsigned>(types)),
                   dim3(256), 0, as_stream(stream), g);
            if (db)
                launch("typed_linear_grad_bias", typed_bias_kernel<T, O>,
                       dim3(static_cast<unsigned>(ceil_div(N, 32)), static_cast<unsigned>(types)), dim3(256), 0,
                       as_stream(stream), g);
        };
        by_dtype(dtype, [&](auto t) {
            if (dw_dtype == TG_F32) run(t, float{});
            else run(t, t);
        });
    });
}

TG_API tg_status tg_typed_check_offsets(int64_t rows, int64_t types, const int32_t* offsets, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "typed_check_offsets";
        check_typed(fn, rows, 1, 1, types, TG_F32, offsets);
        std::vector<int32_t> h(static_cast<size_t>(types + 1));
        cudaStream_t s = as_stream(stream);
        TG_CUDA(cudaMemcpyAsync(h.data(), offsets, h.size() * sizeof(int32_t), cudaMemcpyDeviceToHost, s));
        TG_CUDA(cudaStreamSynchronize(s));
        if (h.front() != 0) invalid("typed_check_offsets: offsets[0] must be 0, got " + std::to_string(h.front()));
        for (int64_t t = 0; t < types; ++t)
            if (h[t + 1] < h[t])
                invalid("typed_check_offsets: offsets must be non-decreasing, but offsets[" + std::to_string(t) +
                        "] = " + std::to_string(h[t]) + " > offsets[" + std::to_string(t + 1) + "] = " +
                        std::to_string(h[t + 1]));
        if (h.back() != rows)
            invalid("typed_check_offsets: offsets[" + std::to_string(types) + "] must equal the row count " +
                    std::to_string(rows) + ", got " + std::to_string(h.back()));
    });
}

}  // extern "C"

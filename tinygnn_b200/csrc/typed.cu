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

// ── db ───────────────────────────────────────────────────────────────────
// Column sums of each type's rows, in two steps of fixed order: chunks of
// kBiasChunk rows of one type (8 warps, a row each; the warps joined through
// shared memory), then a type's chunks.  One read of dY: bound by HBM.

// One warp: prefix[t] = the chunks before type t, at most `chunks` of them in
// all; the rows of a chunk.
__device__ __forceinline__ int64_t scan_chunks(const int32_t* offsets, int types, int64_t M, int chunks, int* prefix) {
    scan_types(offsets, types, M, kBiasChunk, prefix);
    __syncwarp();
    if (prefix[types] <= chunks) return kBiasChunk;
    int64_t owned = 0;  // types overlap
    for (int t = threadIdx.x & 31; t < types; t += 32) owned += rows_of(offsets, t, M);
    owned = reduce_sum<int64_t, 32>(owned);
    const int64_t per = bias_chunk(owned, M);
    __syncwarp();
    scan_types(offsets, types, M, per, prefix);
    return per;
}

// Columns of a warp: 16 bytes a lane when rows are aligned, else 4 columns a
// lane, 32 apart.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(256) typed_bias_kernel(int64_t M, int64_t N, int types, const int32_t* offsets,
                                                         const T* dY, int64_t lddy, float* part, int chunks,
                                                         int64_t* chunk_rows) {
    constexpr int V = ALIGNED ? 16 / static_cast<int>(sizeof(T)) : 4;
    __shared__ int prefix[kMaxTypes + 1];
    __shared__ float sh[8][32 * V];
    __shared__ int64_t rows;
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
    wait_for_previous();
    if (w == 0) {
        const int64_t per = scan_chunks(offsets, types, M, chunks, prefix);
        if (lane == 0) {
            rows = per;
            if (blockIdx.x == 0) *chunk_rows = per;
        }
    }
    __syncthreads();
    const int p = blockIdx.x % chunks;  // (a grid's y is too short for the widest matrices)
    if (p >= prefix[types]) return;
    const int t = find_type(prefix, types, p);
    const int64_t r0 = clamp_row(offsets[t], M) + (p - prefix[t]) * rows;
    const int64_t e = clamp_row(offsets[t + 1], M), r1 = r0 + rows < e ? r0 + rows : e;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x / chunks) * 32 * V;
    float sum[V] = {};
    const auto col = [&](int j) { return n0 + (ALIGNED ? lane * V + j : j * 32 + lane); };
    if (ALIGNED && col(0) + V <= N) {
        const T* q = dY + col(0);
#pragma unroll 8
        for (int64_t r = r0 + w; r < r1; r += 8) {
            float x[V];
            load_v<T, V>(q + r * lddy, x);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += x[j];
        }
    } else {
#pragma unroll 4
        for (int64_t r = r0 + w; r < r1; r += 8)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (col(j) < N) sum[j] += to_f32(dY[r * lddy + col(j)]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sh[w][j * 32 + lane] = sum[j];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += 256) {
        float all = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) all += sh[q][c];
        const int64_t n = n0 + (ALIGNED ? c % 32 * V + c / 32 : c);
        if (n < N) part[p * N + n] = all;
    }
}

__global__ void __launch_bounds__(256) typed_bias_join_kernel(int64_t M, int64_t N, const int32_t* offsets,
                                                              const float* part, const int64_t* chunk_rows, float* db) {
    __shared__ int prefix[kMaxTypes + 1];
    __shared__ float sh[8][33];
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32, t = blockIdx.y;
    wait_for_previous();
    if (w == 0) {  // (a division by a constant where it can be one)
        const int64_t per = *chunk_rows;
        if (per == kBiasChunk) scan_types(offsets, t + 1, M, kBiasChunk, prefix);
        else scan_types(offsets, t + 1, M, per, prefix);
    }
    __syncthreads();
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float sum = 0.0f;
    if (n < N) {
#pragma unroll 4
        for (int p = prefix[t] + w; p < prefix[t + 1]; p += 8) sum += part[p * N + n];
    }
    sh[w][lane] = sum;
    __syncthreads();
    if (w == 0 && n < N) {
        sum = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += sh[q][lane];
        db[t * N + n] = sum;
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

template <class T>
void typed_bias(int64_t M, int64_t N, int types, const int32_t* offsets, const T* dY, int64_t lddy, float* db,
                cudaStream_t s) {
    const int64_t chunks = M / kBiasChunk + types;
    Scratch<float> scratch(static_cast<size_t>(2 + chunks * N), s);
    int64_t* const chunk_rows = reinterpret_cast<int64_t*>(scratch.p);
    float* const part = scratch.p + 2;
    const bool al = rows_aligned16(dY, lddy, sizeof(T));
    const int64_t tile = al ? 32 * (16 / static_cast<int64_t>(sizeof(T))) : 128;
    launch_dependent("typed_linear_grad_bias", al ? typed_bias_kernel<T, true> : typed_bias_kernel<T, false>,
           dim3(static_cast<unsigned>(chunks * ceil_div(N, tile))), dim3(256), 0, s, M, N, types,
           offsets, dY, lddy, part, static_cast<int>(chunks), chunk_rows);
    launch_dependent("typed_linear_grad_bias", typed_bias_join_kernel,
           dim3(static_cast<unsigned>(ceil_div(N, 32)), static_cast<unsigned>(types)), dim3(256), 0, s, M, N, offsets,
           part, chunk_rows, db);
}

template void typed_bias<__nv_bfloat16>(int64_t, int64_t, int, const int32_t*, const __nv_bfloat16*, int64_t, float*,
                                        cudaStream_t);
template void typed_bias<__half>(int64_t, int64_t, int, const int32_t*, const __half*, int64_t, float*, cudaStream_t);

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
            typed_rows<T, false>(g, as_stream(stream));
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
            typed_rows<T, true>(g, as_stream(stream));
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
            typed_weight<T, O>(g, as_stream(stream));
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

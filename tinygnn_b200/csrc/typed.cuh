// ============================================================================
//  typed.cuh -- arguments of the typed linear map's kernels.
// ============================================================================
#pragma once

#include "values.cuh"

namespace tg {

constexpr int kMaxTypes = 1024;  // a block holds the types' tile counts in shared memory

// Row offsets come from the caller's device memory: every one is clamped.
__device__ __forceinline__ int clamp_row(int r, int64_t M) {
    return r < 0 ? 0 : (r > M ? static_cast<int>(M) : r);
}

// prefix[t] = number of pieces of `per` rows in the types before t (one warp).
__device__ __forceinline__ void scan_types(const int32_t* offsets, int types, int64_t M, int64_t per, int* prefix) {
    const int lane = threadIdx.x & 31;
    int carry = 0;
    if (lane == 0) prefix[0] = 0;
    for (int t0 = 0; t0 < types; t0 += 32) {
        const int t = t0 + lane;
        int n = 0;
        if (t < types) {
            const int b = clamp_row(offsets[t], M), e = clamp_row(offsets[t + 1], M);
            n = e > b ? static_cast<int>((e - b + per - 1) / per) : 0;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) n += up;
        }
        if (t < types) prefix[t + 1] = carry + n;
        carry += __shfl_sync(0xffffffffu, n, 31);
    }
}

// The type that piece p belongs to: the last t with prefix[t] <= p.
__device__ __forceinline__ int find_type(const int* prefix, int types, int p) {
    int lo = 0, hi = types;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (prefix[mid] <= p) lo = mid;
        else hi = mid;
    }
    return lo;
}

// C[r] = act(A[r] . B[t(r)] + bias[t(r)]), rows of A are K wide; B is W[t]
// (K x N) in the forward pass and W[t]^T (W[t]: N x K) in the input gradient.
template <class T>
struct RowsArgs {
    int64_t M, K, N;
    int types;
    const T* A;
    int64_t lda;
    const T* W;
    int64_t ldw, stride_w;
    const int32_t* offsets;
    const float* bias;  // types x N, nullable
    int act;
    float alpha;
    T* C;
    int64_t ldc;
    Saved8 saved;  // of the pre-activation; codes nullable
    Range8 r8;
};

// dW[t] (K x N) = sum over the type's rows of X[r]^T dY[r]; X given as it was
// or in 8 bits.
template <class T, class O>
struct WeightArgs {
    int64_t M, K, N;
    int types;
    const T* X;
    int64_t ldx;
    Saved8 saved;
    const T* dY;
    int64_t lddy;
    const int32_t* offsets;
    O* dW;
    int64_t lddw, stride_dw;
    float* db;  // types x N, nullable
};

// How a weight gradient is cut up: pieces of at most `piece` rows of a type,
// each summed by one CTA per tile of dW; types of several pieces leave partial
// sums [piece][K][ldp] (and [piece][N] of db) that a second kernel adds up in
// their order.
struct WeightPlan {
    int BN;  // columns of a tile
    int tiles_k, tiles_n;
    int64_t piece, ldp, items;
    float *part, *db_part;
    bool dy_by_tma;  // typed_weight_any: dY by TMA, db not summed on the way
};

// TMA-fed kernels and the choice between them and the others (typed_tc.cu).
template <class T, bool TRANS>
void typed_rows(const RowsArgs<T>& a, cudaStream_t s);
template <class T, class O>
void typed_weight(const WeightArgs<T, O>& a, cudaStream_t s);
int typed_tc_take_error();

// Loader-fed kernels (typed_any.cu).
template <class T, bool TRANS>
void typed_rows_any(const RowsArgs<T>& a, cudaStream_t s);
template <class T, class O>
void typed_weight_any(const WeightArgs<T, O>& a, const WeightPlan& w, cudaStream_t s);
int typed_any_take_error();

// db alone (typed.cu).
template <class T>
void typed_bias(int64_t M, int64_t N, int types, const int32_t* offsets, const T* dY, int64_t lddy, float* db,
                cudaStream_t s);

}  // namespace tg

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

// On the tensor cores (typed_tc.cu).
template <class T, bool TRANS>
void typed_rows_tc(const RowsArgs<T>& a, cudaStream_t s);
template <class T, class O>
void typed_weight_tc(const WeightArgs<T, O>& a, cudaStream_t s);
int typed_take_error();

}  // namespace tg

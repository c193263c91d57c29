// ============================================================================
//  typed_few.cu -- the typed products of a few rows (serving: single tokens or
//  nodes, each through its type's weight).
//
//  With a few rows (see few_rows()) the products read the used weights (or write all
//  of dW) and do next to no arithmetic: they are bound by HBM and by latency,
//  and a 128-row tensor-core tile would be filled for a row or two.  These
//  kernels stream the weights through FP32 FMAs.  Each row looks for its type
//  among all of them (one a thread).  Rows of one type read its weight again,
//  from L2.
// ============================================================================
#include <algorithm>

#include "typed.cuh"

namespace tg {

namespace {

constexpr int kFewThreads = 512;
constexpr int kFewCols = 128;    // columns of a forward block (one exponent of the saved form)
constexpr int kFewChunk = 2048;  // inner indexes of a row held in shared memory at a time

// The type that owns row r (the last, of types that overlap), -1 if none does.
// Every thread calls it.
__device__ __forceinline__ int type_of_row(const int32_t* offsets, int types, int64_t M, int64_t r) {
    int n = -1;
    for (int t = threadIdx.x; t < types; t += blockDim.x)
        if (clamp_row(offsets[t], M) <= r && r < clamp_row(offsets[t + 1], M)) n = t;
    __shared__ int owner[kFewThreads / 32];
    n = __reduce_max_sync(0xffffffffu, n);
    if (threadIdx.x % 32 == 0) owner[threadIdx.x / 32] = n;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) n = owner[w] > n ? owner[w] : n;
    return n;
}

// Y[r] = act(X[r] . W[t(r)] + bias): block (columns, row).
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kFewThreads) few_forward_kernel(const RowsArgs<T> g) {
    constexpr int V = 16 / static_cast<int>(sizeof(T)), LANES = kFewCols / V, STEP = kFewThreads / LANES;
    __shared__ float xs[kFewChunk];
    __shared__ float sums[STEP][kFewCols];
    wait_for_previous();
    const int64_t r = blockIdx.y, n0 = static_cast<int64_t>(blockIdx.x) * kFewCols;
    const int t = type_of_row(g.offsets, g.types, g.M, r);
    if (t < 0) return;
    const int lane = threadIdx.x % LANES, k_first = threadIdx.x / LANES;
    const int64_t n = n0 + lane * V;
    const int left = n + V <= g.N ? V : (n < g.N ? static_cast<int>(g.N - n) : 0);
    const T* w = g.W + t * g.stride_w + n;
    float acc[V] = {};
    for (int64_t k0 = 0; k0 < g.K; k0 += kFewChunk) {
        const int len = g.K - k0 < kFewChunk ? static_cast<int>(g.K - k0) : kFewChunk;
        __syncthreads();  // the last chunk has been used
        for (int k = threadIdx.x; k < len; k += kFewThreads) xs[k] = to_f32(g.A[r * g.lda + k0 + k]);
        __syncthreads();
        const T* p = w + (k0 + k_first) * g.ldw;
        const int64_t step = STEP * g.ldw;
        constexpr int U = 8;  // rows of W in flight
        for (int k = k_first; k < len; k += U * STEP) {
            Held<T, V, ALIGNED> h[U];
            const T* q = p;
#pragma unroll
            for (int u = 0; u < U; ++u, q += step) {
                if (k + u * STEP >= len) h[u].zero();
                else if (left == V) h[u].fetch(q);
                else if (left > 0) h[u].fetch(q, left);
                else h[u].zero();
            }
#pragma unroll
            for (int u = 0; u < U; ++u, p += step) {
                float v[V];
                h[u].values(h[u].odd(p), v);
                const float x = k + u * STEP < len ? xs[k + u * STEP] : 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = fmaf(x, v[j], acc[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sums[k_first][lane * V + j] = acc[j];
    __syncthreads();
    if (threadIdx.x >= kFewCols) return;
    // one column a thread
    const int64_t c = n0 + threadIdx.x;
    float z[1] = {0.0f};
#pragma unroll 8
    for (int q = 0; q < STEP; ++q) z[0] += sums[q][threadIdx.x];
    if (g.bias && c < g.N) z[0] += g.bias[t * g.N + c];
    if (g.saved.codes) {
        __shared__ float most[kFewCols / 32];
        const float m = reduce_max<32>(c < g.N ? fabsf(z[0]) : 0.0f);
        if (threadIdx.x % 32 == 0) most[threadIdx.x / 32] = m;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int byte = exponent8(max_nan(max_nan(most[0], most[1]), max_nan(most[2], most[3])), g.r8.emin);
        if (c < g.N) g.saved.codes[r * g.saved.ld + c] = code8(z[0], encode8(byte), byte, g.r8.top);
        if (threadIdx.x == 0) g.saved.exps[r * g.saved.lde + blockIdx.x] = static_cast<uint8_t>(byte);
    }
    act_forward<sizeof(T) == 2>(z, g.act, g.alpha);
    if (c < g.N) g.C[r * g.ldc + c] = from_f32<T>(z[0]);
}

// dX[r] = dY[r] . W[t(r)]^T: a warp per element of dX (a row of W), block
// (elements, row).  Here A is dY, K its width, N the width of dX.
constexpr int kFewOut = 2 * kFewThreads / 32;  // elements of a block

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kFewThreads) few_grad_input_kernel(const RowsArgs<T> g) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    __shared__ float ys[kFewChunk];
    wait_for_previous();
    const int64_t r = blockIdx.y;
    const int t = type_of_row(g.offsets, g.types, g.M, r);
    if (t < 0) return;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t out0 = static_cast<int64_t>(blockIdx.x) * kFewOut + warp * 2;
    float acc[2] = {0.0f, 0.0f};
    for (int64_t k0 = 0; k0 < g.K; k0 += kFewChunk) {
        const int len = g.K - k0 < kFewChunk ? static_cast<int>(g.K - k0) : kFewChunk;
        __syncthreads();
        for (int k = threadIdx.x; k < len; k += kFewThreads) ys[k] = to_f32(g.A[r * g.lda + k0 + k]);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (out0 + e >= g.N) break;
            const T* p = g.W + t * g.stride_w + (out0 + e) * g.ldw + k0;
            constexpr int U = 4;
            for (int k = lane * V; k < len; k += U * 32 * V) {
                Held<T, V, ALIGNED> h[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int at = k + u * 32 * V;
                    if (at + V <= len) h[u].fetch(p + at);
                    else if (at < len) h[u].fetch(p + at, len - at);
                    else h[u].zero();
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int at = k + u * 32 * V;
                    float v[V];
                    h[u].values(h[u].odd(p + at), v);
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (at + j < len) acc[e] = fmaf(ys[at + j], v[j], acc[e]);
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float z = reduce_sum<float, 32>(acc[e]);
        if (lane == 0 && out0 + e < g.N) g.C[r * g.ldc + out0 + e] = from_f32<T>(z);
    }
}

// dW[t][k] = sum over the type's rows of X[r][k] dY[r], most of them none: block
// (rows of dW, type), a thread per 8 columns.
template <class T, class O, bool SAVED>
__global__ void __launch_bounds__(256) few_grad_weight_kernel(const WeightArgs<T, O> g, int wide, int rows_per_block,
                                                              int vec) {
    constexpr int V = 8;
    wait_for_previous();
    const int t = blockIdx.y;
    const int b = clamp_row(g.offsets[t], g.M), e = clamp_row(g.offsets[t + 1], g.M);
    const int rr = threadIdx.x / wide;
    if (rr >= rows_per_block) return;
    for (int64_t k = static_cast<int64_t>(blockIdx.x) * rows_per_block + rr; k < g.K;
         k += static_cast<int64_t>(gridDim.x) * rows_per_block)
        for (int64_t n = (threadIdx.x - rr * wide) * V; n < g.N; n += wide * V) {
            float acc[V] = {};
            for (int r = b; r < e; ++r) {
                const float x = SAVED ? __fmul_rn(static_cast<float>(g.saved.codes[r * g.saved.ld + k]),
                                                  decode8(g.saved.exps[r * g.saved.lde + k / kBlock8]))
                                      : to_f32(g.X[r * g.ldx + k]);
                const T* p = g.dY + r * g.lddy + n;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (n + j < g.N) acc[j] = fmaf(x, to_f32(p[j]), acc[j]);
            }
            O* o = g.dW + t * g.stride_dw + k * g.lddw + n;
            if (vec && n + V <= g.N) {
                constexpr int S = 16 / static_cast<int>(sizeof(O));
#pragma unroll
                for (int j = 0; j < V; j += S) {
                    float part[S];
#pragma unroll
                    for (int i = 0; i < S; ++i) part[i] = acc[j + i];
                    store_v<O, S>(o + j, part);
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (n + j < g.N) o[j] = from_f32<O>(acc[j]);
            }
        }
    if (g.db && blockIdx.x == 0 && rr == 0)
        for (int64_t n = threadIdx.x; n < g.N; n += wide) {
            float sum = 0.0f;
            for (int r = b; r < e; ++r) sum += to_f32(g.dY[r * g.lddy + n]);
            g.db[t * g.N + n] = sum;
        }
}

}  // namespace

template <class T, bool TRANS>
void typed_rows_few(const RowsArgs<T>& a, cudaStream_t s) {
    const bool al = rows_aligned16(a.W, a.ldw, sizeof(T)) && (a.types == 1 || a.stride_w * sizeof(T) % 16 == 0);
    if constexpr (TRANS)
        launch_dependent("typed_few", al ? few_grad_input_kernel<T, true> : few_grad_input_kernel<T, false>,
                         dim3(static_cast<unsigned>(ceil_div(a.N, kFewOut)), static_cast<unsigned>(a.M)),
                         dim3(kFewThreads), 0, s, a);
    else
        launch_dependent("typed_few", al ? few_forward_kernel<T, true> : few_forward_kernel<T, false>,
                         dim3(static_cast<unsigned>(ceil_div(a.N, kFewCols)), static_cast<unsigned>(a.M)),
                         dim3(kFewThreads), 0, s, a);
}

template <class T, class O>
void typed_weight_few(const WeightArgs<T, O>& a, cudaStream_t s) {
    const int wide = static_cast<int>(std::min<int64_t>(ceil_div(a.N, 8), 256)), rpb = 256 / wide;
    const int vec = reinterpret_cast<uintptr_t>(a.dW) % 16 == 0 && a.lddw * sizeof(O) % 16 == 0 &&
                    (a.types == 1 || a.stride_dw * sizeof(O) % 16 == 0);
    // Enough blocks for every SM several times over, each with a few rows of dW;
    // and 64 a type, since all rows may lie in one (256 rows, 1,024 types, 1,024
    // x 1,024 bf16: 858 us in one type, 395 spread; 4 blocks a type 6,505, 392).
    const int64_t want = ceil_div(a.K, rpb * 4), most = std::max<int64_t>(64, int64_t(num_sms()) * 32 / a.types);
    launch_dependent("typed_few_weight",
                     a.saved.codes ? few_grad_weight_kernel<T, O, true> : few_grad_weight_kernel<T, O, false>,
                     dim3(static_cast<unsigned>(std::min(want, most)), static_cast<unsigned>(a.types)), dim3(256), 0,
                     s, a, wide, rpb, vec);
}

#define TG_TYPED_FEW(T)                                                       \
    template void typed_rows_few<T, false>(const RowsArgs<T>&, cudaStream_t); \
    template void typed_rows_few<T, true>(const RowsArgs<T>&, cudaStream_t);  \
    template void typed_weight_few<T, T>(const WeightArgs<T, T>&, cudaStream_t);
TG_TYPED_FEW(float)
TG_TYPED_FEW(__nv_bfloat16)
TG_TYPED_FEW(__half)
template void typed_weight_few<__nv_bfloat16, float>(const WeightArgs<__nv_bfloat16, float>&, cudaStream_t);
template void typed_weight_few<__half, float>(const WeightArgs<__half, float>&, cudaStream_t);

}  // namespace tg

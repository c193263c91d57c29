// ============================================================================
//  typed.cuh -- arguments of the typed linear map's kernels.
// ============================================================================
#pragma once

#include <algorithm>
#include <climits>

#include "values.cuh"

namespace tg {

constexpr int kMaxTypes = 1024;  // a block holds the types' tile counts in shared memory

// Row offsets come from the caller's device memory: every one is clamped.
__device__ __forceinline__ int clamp_row(int r, int64_t M) {
    return r < 0 ? 0 : (r > M ? static_cast<int>(M) : r);
}

// Pieces so far and n more (n below 2^29), at most INT_MAX: types that overlap
// own more than M rows between them, and a count that wrapped around would
// lead a block out of its type.  Pieces past the limit are not worked on.
__host__ __device__ __forceinline__ int add_pieces(int so_far, int n) {
    return n > INT_MAX - so_far ? INT_MAX : so_far + n;
}

// prefix[t] = number of pieces of `per` rows (128 or more) in the types before
// t (one warp).  The offsets of 128 types are asked for at once: a warp that
// went 32 at a time would wait for memory four times.
__device__ __forceinline__ void scan_types(const int32_t* offsets, int types, int64_t M, int64_t per, int* prefix) {
    const int lane = threadIdx.x & 31;
    int carry = 0;
    if (lane == 0) prefix[0] = 0;
    for (int t0 = 0; t0 < types; t0 += 128) {
        int b[4], e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = t0 + i * 32 + lane;
            b[i] = t < types ? offsets[t] : 0;
            e[i] = t < types ? offsets[t + 1] : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t0 + i * 32 >= types) break;
            const int t = t0 + i * 32 + lane, rows = clamp_row(e[i], M) - clamp_row(b[i], M);
            int n = rows > 0 ? static_cast<int>((rows + per - 1) / per) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += up;
            }
            if (t < types) prefix[t + 1] = add_pieces(carry, n);
            carry = add_pieces(carry, __shfl_sync(0xffffffffu, n, 31));
        }
    }
}

// Rows of a chunk of the bias gradient's sums when the types own `owned` rows
// of M between them: more than kBiasChunk where they overlap, so that there are
// never more than M / kBiasChunk + types chunks.
constexpr int kBiasChunk = 256;
__host__ __device__ __forceinline__ int64_t bias_chunk(int64_t owned, int64_t M) {
    return kBiasChunk * (owned <= M ? 1 : (owned + M - 1) / M);
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

// ── How a weight gradient is cut up ──────────────────────────────────────
// Each tile of each type's dW is a sum over the type's rows, in steps of 64.
// An item is a tile and a piece of its type's rows, for one CTA.  A type is
// one piece unless it has more steps than 5/4 of an SM's share of all the
// steps (`slots` SMs, `per` tiles a type); then it is cut into the fewest equal
// pieces that have no more.  Items run longest first, dealt out to the CTAs
// back and forth, so the CTAs' totals come out nearly equal without a counter
// in memory, and few types are cut at all: a cut type's pieces leave partial
// sums [slot][K][ldp] (and [slot][N] of db) that a second kernel adds up in
// their order.  Slots count the cut types' pieces only (with one for every
// piece, 1,024 types of 1,024 x 1,024 took 4.3 GB of scratch, most of it for
// types that are not cut).
constexpr int kStep = 64;
constexpr int kSortTypes = 256;  // more types than this keep their order (many items even out anyway)

__device__ __forceinline__ int rows_of(const int32_t* offsets, int t, int64_t M) {
    const int b = clamp_row(offsets[t], M), e = clamp_row(offsets[t + 1], M);
    return e > b ? e - b : 0;
}
// Rows of the longest piece, from the sum of all types' steps.  `longest`: the
// steps that a sum may take (kernels that cannot add up parts of it themselves,
// where the result is fp32).  Offsets that leave rows out or own rows twice
// keep within the same bounds: a type of at most the limit for M / 64 steps is
// never cut, and there are at most max_pieces().
__host__ __device__ __forceinline__ int64_t piece_limit(int64_t steps, int64_t M, int types, int per, int slots,
                                                        int longest) {
    if (steps < M / kStep) steps = M / kStep;
    if (steps > M / kStep + types) longest = 1 << 30;
    const int64_t share = (steps * per * 5 + slots * 4 - 1) / (slots * 4);
    return (share < 2 ? 2 : (share < longest ? share : longest)) * kStep;
}
// A type of n rows has fewer than n / limit + 1 pieces, and a limit is at least
// 5/4 of slots / per equal shares of the rows, or `longest` steps.
inline int64_t max_pieces(int64_t M, int types, int64_t per, int slots, int longest) {
    return types + std::max<int64_t>(slots / per, (M / kStep + types) / longest + 1);
}
// A cut type has fewer than 2 n / limit pieces.
inline int64_t max_slots(int64_t M, int types, int64_t per, int slots, int longest) {
    return 2 * std::max<int64_t>(slots / per + 1, (M / kStep + types) / longest + 1);
}
__host__ __device__ __forceinline__ int piece_count(int n, int64_t limit) { return static_cast<int>((n + limit - 1) / limit); }
// Rows of each piece (the last may have fewer; none is empty, since this is at most `limit`).
__host__ __device__ __forceinline__ int piece_rows(int n, int count) {
    return count <= 1 ? n : ((n + count - 1) / count + kStep - 1) / kStep * kStep;
}
// Whether type u's pieces come before type t's.
__device__ __forceinline__ bool piece_before(int types, int rows_u, int u, int rows_t, int t) {
    return types > kSortTypes ? u < t : rows_u > rows_t || (rows_u == rows_t && u < t);
}

// One warp: order[i] = the i-th type, and above its 16 bits how many types
// before it are one piece; prefix[i] = the pieces before it.
__device__ __forceinline__ void plan_pieces(const int32_t* offsets, int types, int64_t M, int per, int slots,
                                            int longest, int* prefix, uint32_t* order) {
    const int lane = threadIdx.x & 31;
    int64_t steps = 0;
    for (int t = lane; t < types; t += 32) steps += (rows_of(offsets, t, M) + kStep - 1) / kStep;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) steps += __shfl_xor_sync(0xffffffffu, steps, o);
    const int64_t limit = piece_limit(steps, M, types, per, slots, longest);
    if (types > kSortTypes) {
        for (int t = lane; t < types; t += 32) order[t] = static_cast<uint32_t>(t);
    } else {
        for (int t = lane; t < types; t += 32) {
            const int n = rows_of(offsets, t, M);
            prefix[t] = piece_rows(n, piece_count(n, limit));
        }
        __syncwarp();
        for (int t = lane; t < types; t += 32) {
            const int key = prefix[t];
            int rank = 0;
            for (int u = 0; u < types; ++u) rank += piece_before(types, prefix[u], u, key, t);
            order[rank] = static_cast<uint32_t>(t);
        }
    }
    __syncwarp();
    int carry = 0, whole = 0;
    for (int i0 = 0; i0 < types; i0 += 32) {
        const int i = i0 + lane;
        int n = i < types ? piece_count(rows_of(offsets, order[i], M), limit) : 0;
        const uint32_t ones = __ballot_sync(0xffffffffu, n == 1);
        if (i < types) order[i] |= static_cast<uint32_t>(whole + __popc(ones & ((1u << lane) - 1))) << 16;
        whole += __popc(ones);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) n += up;
        }
        if (i < types) prefix[i + 1] = carry + n;
        carry += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) prefix[0] = 0;
}

// Item number `it` in the order above.
struct WeightItem {
    int t, p;        // type, slot (of a cut type's piece)
    int in;          // tile of the type
    int64_t r0, r1;  // rows
    bool whole;      // the type is one piece
};
__device__ __forceinline__ WeightItem weight_item(const int32_t* offsets, int types, int64_t M, int per,
                                                  const int* prefix, const uint32_t* order, int64_t it) {
    WeightItem m;
    const int p = static_cast<int>(it / per);
    m.in = static_cast<int>(it - static_cast<int64_t>(p) * per);
    const int i = find_type(prefix, types, p);
    m.t = order[i] & 0xffff;
    m.p = p - static_cast<int>(order[i] >> 16);
    const int b = clamp_row(offsets[m.t], M), e = clamp_row(offsets[m.t + 1], M);
    const int count = prefix[i + 1] - prefix[i], len = piece_rows(e - b, count);
    m.r0 = b + static_cast<int64_t>(p - prefix[i]) * len;
    m.r1 = m.r0 + len < e ? m.r0 + len : e;
    m.whole = count == 1;
    return m;
}
// The item that CTA `cta` of `ctas` takes in its round `r`: back and forth.
__device__ __forceinline__ int64_t dealt(int64_t r, int64_t cta, int64_t ctas) {
    return r * ctas + (r & 1 ? ctas - 1 - cta : cta);
}

struct WeightPlan {
    int BN;  // columns of a tile
    int tiles_k, tiles_n, slots, longest;
    int64_t ldp, items;
    float *part, *db_part;
};

// TMA-fed kernels and the choice between them and the others (typed_tc.cu).
template <class T, bool TRANS>
void typed_rows(const RowsArgs<T>& a, cudaStream_t s);
template <class T, class O>
void typed_weight(const WeightArgs<T, O>& a, cudaStream_t s);
int typed_tc_take_error();

// A batch of 16-bit matrices that TMA can read (rows and matrices 16-byte aligned).
template <class T>
struct TmaMatrix {
    const T* p;
    int64_t ld, stride;
};

// TMA-fed kernels on CTA pairs (typed_pair.cu).
template <class T, bool TRANS>
void typed_rows_pair(const RowsArgs<T>& a, const TmaMatrix<T>& A, const TmaMatrix<T>& W, cudaStream_t s);
int typed_pair_take_error();

// Loader-fed kernels (typed_any.cu): all products of fp32 rows, weight gradients
// of 16-bit ones.
template <bool TRANS>
void typed_rows_any(const RowsArgs<float>& a, cudaStream_t s);
template <class T, class O>
void typed_weight_any(const WeightArgs<T, O>& a, const WeightPlan& w, cudaStream_t s);
int typed_any_take_error();

// A few rows (typed_few.cu).
constexpr int64_t kFewRows = 32;
template <class T, bool TRANS>
void typed_rows_few(const RowsArgs<T>& a, cudaStream_t s);
template <class T, class O>
void typed_weight_few(const WeightArgs<T, O>& a, cudaStream_t s);

// db alone (typed.cu).
template <class T>
void typed_bias(int64_t M, int64_t N, int types, const int32_t* offsets, const T* dY, int64_t lddy, float* db,
                cudaStream_t s);

}  // namespace tg

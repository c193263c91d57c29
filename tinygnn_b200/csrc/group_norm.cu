// ============================================================================
//  group_norm.cu -- group norm with an activation over the rows of each graph,
//  channels last, and its backward pass.
//
//  A group is the rows of one graph (offsets[g] .. offsets[g + 1]) and
//  cols / groups neighbouring columns:
//      h = (x - mean) r,  r = 1 / sqrt(mean (x - mean)^2 + eps)
//      u = h gamma + beta,  y = act(u)
//      du = dy act'(u),  dgamma = sum du h,  dbeta = sum du  (over all rows)
//      dx = r (g - mean g - h mean(g h)),  g = gamma du
//
//  Graphs have any sizes, which only the device knows, so the work is cut by
//  rows: a block walks chunks of R rows, thread (tx, ty) the V columns of one
//  16-byte vector in every ty-th row of it, and splits a chunk where a graph ends.
//  The first pass leaves one partial result for each column, chunk and graph in
//  it; chunk c's part of graph g is slot c + g, which no other part has, and there
//  are at most chunks + graphs of them.  A second, small kernel joins a graph's
//  slots in their order (no atomics, the same bits every run), and a third applies
//  the statistics.  Where graphs are small (small_rows below) each is a block's
//  instead, in one kernel, and the three have the larger ones alone.
//
//  A part's mean and sum of squared deviations come from one pass: each thread
//  sums x - k and (x - k)^2 with k its first value of the column (one of the
//  values it is subtracted from: where it is far from the others, so is the part's
//  deviation, and each row costs 2^-24 of it at most), and parts are joined by their
//  means and deviations, not by sums of squares.
//
//  232,965 x 128 bf16 in one graph, 8 groups: forward 46 us, gradient 64; x and dy
//  are read twice, and the second reading of 60 or 120 MB comes from HBM again
//  (its floor is 9.3 us a matrix).  16 graphs of 4,096 x 320 fp16 in 32 groups,
//  GELU: 43 and 70, bound by issue slots (50 %) and by 15 warps an SM, since
//  vectors of columns of two groups keep the factors of each column.
//
//  What is applied to a value is linear in its distance from the mean, with
//  factors of its column (the mean is not folded into the addend: a constant
//  graph's y is beta):
//      u = A (x - mean) + beta,  A = r gamma
//      dx = A du - E (x - mean) - D,  E = r^2 mean(g h),  D = r mean g
// ============================================================================
#include <algorithm>

#include "typed.cuh"

namespace tg {

namespace {

struct GroupArgs {
    int64_t rows;
    int cols, groups, per, graphs;  // per: columns of a group
    const int32_t* offsets;  // nullable: one graph of all rows
    int act;
    float alpha, eps;
    // the cut
    int least;               // graphs of at most as many rows are a block's (0: none are)
    int* large;              // of the `blocks` blocks that have whole graphs: whether one met a larger graph (with least)
    int blocks;
    int R, chunks;           // rows of a chunk, number of chunks
    int nv, tx, ty;          // vectors of a row, of a block; row lanes of a block
};

__device__ __forceinline__ int begin_of(const GroupArgs& a, int g) {
    return a.offsets ? clamp_row(a.offsets[g], a.rows) : 0;
}
__device__ __forceinline__ int end_of(const GroupArgs& a, int g) {
    return a.offsets ? clamp_row(a.offsets[g + 1], a.rows) : static_cast<int>(a.rows);
}
// The first graph that ends after row r (a.graphs: none), found by a warp.
__device__ __forceinline__ int graph_at(const GroupArgs& a, int r) {
    int lo = 0, hi = a.graphs;
    const int lane = threadIdx.x & 31;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, g = lo + lane * step;
        const uint32_t past = __ballot_sync(0xffffffffu, g >= hi || end_of(a, g) > r);
        if (past == 0) {
            lo += 31 * step + 1;
        } else {
            const int f = __ffs(past) - 1;
            hi = min(hi, lo + f * step);
            if (f > 0) lo += (f - 1) * step + 1;
        }
    }
    return lo;
}
// Whether all graphs are a block's, so that the chunks' kernels have nothing to do.
__device__ __forceinline__ bool none_large(const GroupArgs& a) {
    if (a.least == 0) return false;
    int any = 0;
    for (int i = threadIdx.x; i < a.blocks; i += blockDim.x) any |= a.large[i];
    return !__syncthreads_or(any);
}
// The first graph from g on that the chunks' kernels have; one that begins at
// row `end` or later (or a.graphs) where there is none before that row.
__device__ __forceinline__ int next_graph(const GroupArgs& a, int g, int64_t end) {
    if (a.least == 0) return g;
    for (const int lane = threadIdx.x & 31;; g += 32) {
        const int i = g + lane;
        const uint32_t m = __ballot_sync(0xffffffffu, i >= a.graphs || begin_of(a, i) >= end || end_of(a, i) - begin_of(a, i) > a.least);
        if (m) return g + __ffs(m) - 1;
    }
}
// Calls f(g, first row, end, slot) for the graphs' parts of chunk c.  With a.least a
// chunk has no whole graph (R <= least), so at most two parts: slots 2 c, and
// 2 c + 1 for the graph that begins in it.
template <class F>
__device__ __forceinline__ void for_parts(const GroupArgs& a, int c, F&& f) {
    const int64_t c0 = static_cast<int64_t>(c) * a.R, c1 = c0 + a.R < a.rows ? c0 + a.R : a.rows;
    for (int g = next_graph(a, graph_at(a, static_cast<int>(c0)), c1); g < a.graphs; g = next_graph(a, g + 1, c1)) {
        const int b = begin_of(a, g), e = end_of(a, g);
        if (b >= c1) break;
        const int lo = b > c0 ? b : static_cast<int>(c0), hi = e < c1 ? e : static_cast<int>(c1);
        if (lo < hi) f(g, lo, hi, a.least ? 2 * static_cast<int64_t>(c) + (b >= c0) : static_cast<int64_t>(c) + g);
        if (e >= c1) break;
    }
}
// Slot of the i-th part of graph g, whose first is in chunk `first`.
__device__ __forceinline__ int64_t slot_of(const GroupArgs& a, int g, int first, int i) {
    return a.least ? 2 * static_cast<int64_t>(first + i) + (i == 0) : static_cast<int64_t>(first + i) + g;
}

constexpr int kMaxThreads = 256;
// Blocks of an SM of the kernels that walk chunks.
constexpr int kParts = 4, kGrad = 2;
template <bool SPLIT>
constexpr int kApply = SPLIT ? 2 : 3;
constexpr int kJoinThreads = 1024;  // that join a graph's group of many parts
template <int W>
constexpr int kJoinBlock = W == 32 ? 256 : W;
// Blocks that share the groups of a large graph among small ones.
__host__ __device__ constexpr int large_blocks(int groups) { return groups < 4 ? groups : 4; }

// A thread's place: V columns from `col` on, of which `n` are there (ALIGNED: all
// or none), in the rows ty, ty + a.ty, ... of a part.
template <class T, bool ALIGNED>
struct Place {
    static constexpr int V = 16 / static_cast<int>(sizeof(T));
    using Values = Held<T, V, ALIGNED>;
    int tx, ty, col, n;
    __device__ __forceinline__ explicit Place(const GroupArgs& a) {
        tx = threadIdx.x % a.tx;
        ty = threadIdx.x / a.tx;
        col = (blockIdx.y * a.tx + tx) * V;
        n = ty < a.ty ? min(V, a.cols - col) : 0;
    }
    __device__ __forceinline__ void fetch(Values& v, const T* row) const {
        if (ALIGNED) v.fetch(row + col);
        else v.fetch(row + col, n);
    }
    __device__ __forceinline__ void values(const Values& v, const T* row, float (&x)[V]) const {
        v.values(Values::odd(row + col), x, ALIGNED ? V : n);
    }
    __device__ __forceinline__ void store(T* row, const float (&x)[V]) const {
        if (ALIGNED) store_v<T, V>(row + col, x);
        else store_some<T, V>(row + col, x, n);
    }
    template <class P>
    __device__ __forceinline__ void params(const P* p, float (&x)[V]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = j < n ? to_f32(p[col + j]) : 0.0f;
    }
    // This thread's rows of [lo, hi).
    __device__ __forceinline__ int rows_of(const GroupArgs& a, int lo, int hi) const {
        return n > 0 && lo + ty < hi ? (hi - lo - ty + a.ty - 1) / a.ty : 0;
    }
    // Calls f(values, the row of `out`, u) for this thread's rows of [lo, hi); U
    // rows are asked for before the first (u = 0) is looked at.
    template <int U, class F>
    __device__ __forceinline__ void for_rows(const GroupArgs& a, int lo, int hi, const T* x, int64_t ldx, T* out, int64_t ldo,
                                             F&& f) const {
        const int64_t step = a.ty * ldx, step_out = a.ty * ldo;
        const T* row = x + static_cast<int64_t>(lo + ty) * ldx;
        T* to = out + static_cast<int64_t>(lo + ty) * ldo;
        for (int left = rows_of(a, lo, hi); left > 0; left -= U) {
            Values v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < left) fetch(v[u], row + u * step);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u >= left) break;
                float z[V];
                values(v[u], row + u * step, z);
                f(z, to, u);
                to += step_out;
            }
            row += U * step;
        }
    }
    // The same for two matrices.
    template <int U, class F>
    __device__ __forceinline__ void for_rows(const GroupArgs& a, int lo, int hi, const T* x, int64_t ldx, const T* y, int64_t ldy,
                                             T* out, int64_t ldo, F&& f) const {
        const int64_t step = a.ty * ldx, step_y = a.ty * ldy, step_out = a.ty * ldo;
        const T *row = x + static_cast<int64_t>(lo + ty) * ldx, *row_y = y + static_cast<int64_t>(lo + ty) * ldy;
        T* to = out + static_cast<int64_t>(lo + ty) * ldo;
        for (int left = rows_of(a, lo, hi); left > 0; left -= U) {
            Values v[U], w[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u < left) {
                    fetch(v[u], row + u * step);
                    fetch(w[u], row_y + u * step_y);
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u >= left) break;
                float z[V], d[V];
                values(v[u], row + u * step, z);
                values(w[u], row_y + u * step_y, d);
                f(z, d, to);
                to += step_out;
            }
            row += U * step;
            row_y += U * step_y;
        }
    }
};

// x <- f(x) for the pairs of V values.
template <int V, class F>
__device__ __forceinline__ void pairs(float (&x)[V], F&& f) {
#pragma unroll
    for (int j = 0; j < V; j += 2) f(j, Pair(x[j], x[j + 1])).get(x[j], x[j + 1]);
}

// Two sums of every column of a block's threads, before they are joined over
// the row lanes, in shared memory.  (One pair more a plane: neighbouring columns
// lie in other banks.)
template <class T>
struct Sums {
    static constexpr int V = 16 / static_cast<int>(sizeof(T));
    float2* at;
    static __host__ __device__ constexpr int pairs(int threads) { return V * (threads + 1); }
    __device__ __forceinline__ void set(int j, float2 v) const { at[j * (blockDim.x + 1) + threadIdx.x] = v; }
    // Column c of the block's in row lane y.
    __device__ __forceinline__ float2 get(const GroupArgs& a, int c, int y) const {
        return at[(c % V) * (blockDim.x + 1) + y * a.tx + c / V];
    }
};

// ── forward ──────────────────────────────────────────────────────────────
// This thread's columns' means and sums of squared deviations over its rows of
// [lo, hi), U of them at a time.
template <int U, class T, bool ALIGNED>
__device__ __forceinline__ void part_sums(const GroupArgs& a, const Place<T, ALIGNED>& p, const T* x, int64_t ldx, int lo, int hi,
                                          const Sums<T>& sh) {
    constexpr int V = Place<T, ALIGNED>::V;
    float k[V], s[V], q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) k[j] = s[j] = q[j] = 0.0f;
    const int n = p.rows_of(a, lo, hi);
    bool first = true;
    p.template for_rows<U>(a, lo, hi, x, ldx, static_cast<T*>(nullptr), 0, [&](float (&z)[V], T*, int u) {
        if (u == 0 && first) {
#pragma unroll
            for (int j = 0; j < V; ++j) k[j] = z[j];
            first = false;
        }
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const Pair d = add2(Pair(z[j], z[j + 1]), Pair(-k[j], -k[j + 1]));
            add2(Pair(s[j], s[j + 1]), d).get(s[j], s[j + 1]);
            fma2(d, d, Pair(q[j], q[j + 1])).get(q[j], q[j + 1]);
        }
    });
    // (a value that is not finite: x - x is a NaN, and so are the deviations)
    const float inv = n ? __fdiv_rn(1.0f, static_cast<float>(n)) : 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float bad = __fsub_rn(k[j], k[j]);
        sh.set(j, make_float2(fmaf(s[j], inv, k[j]), __fadd_rn(max_nan(fmaf(-s[j], __fmul_rn(s[j], inv), q[j]), 0.0f), bad)));
    }
}
// (mean, sum of squared deviations) of the block's column c over all row lanes of a part of `rows` rows.
template <class T>
__device__ __forceinline__ float2 join_lanes(const GroupArgs& a, const Sums<T>& sh, int c, int rows) {
    const auto lane_rows = [&](int y) { return static_cast<float>((rows - y + a.ty - 1) / a.ty); };
    const int lanes = rows < a.ty ? rows : a.ty;
    const float first = sh.get(a, c, 0).x;
    float sum = 0.0f, dev = 0.0f;
    for (int y = 1; y < lanes; ++y) sum = fmaf(__fsub_rn(sh.get(a, c, y).x, first), lane_rows(y), sum);
    const float mean = __fadd_rn(first, __fdiv_rn(sum, static_cast<float>(rows)));
    for (int y = 0; y < lanes; ++y) {
        const float2 o = sh.get(a, c, y);
        const float e = __fsub_rn(o.x, mean);
        dev = __fadd_rn(dev, fmaf(__fmul_rn(e, e), lane_rows(y), o.y));
    }
    return make_float2(mean, dev);
}
// Calls f(c, column) for the block's columns that this thread joins.
template <class T, class F>
__device__ __forceinline__ void for_columns(const GroupArgs& a, F&& f) {
    constexpr int V = Sums<T>::V;
    const int first = blockIdx.y * a.tx * V;
    for (int c = threadIdx.x; c < a.tx * V && first + c < a.cols; c += blockDim.x) f(c, first + c);
}

// part[slot * cols + column] = (mean, sum of squared deviations) of the part's values.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kMaxThreads, kParts) group_parts_kernel(const GroupArgs a, const T* x, int64_t ldx, float2* part) {
    extern __shared__ float2 room[];
    const Sums<T> sh{room};
    wait_for_previous();
    if (none_large(a)) return;
    const Place<T, ALIGNED> p(a);
    const int c = blockIdx.x;
    for_parts(a, c, [&](int g, int lo, int hi, int64_t slot) {
        part_sums<4>(a, p, x, ldx, lo, hi, sh);
        __syncthreads();
        for_columns<T>(a, [&](int i, int column) {
            part[slot * a.cols + column] = join_lanes(a, sh, i, hi - lo);
        });
        __syncthreads();
    });
}

// This thread's parts of a graph's group, one of W threads: those of its columns
// c0 + col for col = first_col, + wide, ... < per, of each the slots first_slot,
// + step, ...
template <int W>
struct Share {
    int first, slots, wide, step, first_col, first_slot;
    __device__ __forceinline__ Share(const GroupArgs& a, int b, int e) : first(b / a.R), slots((e - 1) / a.R - first + 1) {
        // (of narrow groups a thread has the same column of every W / per-th slot)
        wide = a.per < W ? a.per : W;
        step = W / wide;
        const int t = threadIdx.x % W;
        first_col = t < wide * step ? t % wide : a.per;
        first_slot = t / wide;
    }
    // Rows of a graph's (b .. e) part in slot i.
    __device__ __forceinline__ int rows(const GroupArgs& a, int b, int e, int i) const {
        // (the last chunk's end may pass 2^31)
        const int r0 = (first + i) * a.R, r1 = e - r0 < a.R ? e : r0 + a.R;
        return r1 - (b > r0 ? b : r0);
    }
};
// The sum over W threads (a warp, or the block).
template <int W>
__device__ __forceinline__ float sum_of(float v, float* sh) {
    v = reduce_sum<float, 32>(v);
    if (W == 32) return v;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < W / 32; ++w) v = __fadd_rn(v, sh[w]);
    return v;
}
// Two sums in 64 bits (both at a time: a double's addition takes long to come back).
template <int W>
__device__ __forceinline__ void sums_of(double& s, double& d, double2* sh) {
    s = reduce_sum<double, 32>(s);
    d = reduce_sum<double, 32>(d);
    if (W == 32) return;
    const int lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) sh[threadIdx.x >> 5] = make_double2(s, d);
    __syncthreads();
    const double2 v = lane < W / 32 ? sh[lane] : make_double2(0.0, 0.0);
    s = reduce_sum<double, 32>(v.x);
    d = reduce_sum<double, 32>(v.y);
}

// Calls f(g, group) for the graphs' groups that W threads join: one, blockIdx.x's
// W-th part's; of large graphs among small ones those of the graph that begins in
// chunk blockIdx.x.
template <int W, class F>
__device__ __forceinline__ void for_sets(const GroupArgs& a, int block, F&& f) {
    if (a.least == 0) {
        const int64_t i = static_cast<int64_t>(block) * (kJoinBlock<W> / W) + threadIdx.x / W;
        if (i < static_cast<int64_t>(a.graphs) * a.groups) f(static_cast<int>(i / a.groups), static_cast<int>(i % a.groups));
        return;
    }
    const int share = large_blocks(a.groups);
    for_parts(a, block / share, [&](int g, int, int, int64_t slot) {
        if (slot % 2)
            for (int i = block % share; i < a.groups; i += share) f(g, i);
    });
}

// stats[g * groups + group] = (mean, rstd), (0, 0) for a graph without rows.
template <int W>
__global__ void __launch_bounds__(kJoinBlock<W>) group_stats_kernel(const GroupArgs a, const float2* part, float2* stats) {
    __shared__ double2 sh[32];
    wait_for_previous();
    if (none_large(a)) return;
    for_sets<W>(a, blockIdx.x, [&](int g, int group) {
        const int c0 = group * a.per, b = begin_of(a, g), e = end_of(a, g);
        float2 r = make_float2(0.0f, 0.0f);
        if (b < e) {
            const double all = static_cast<double>(e - b) * a.per;
            const float inv = __frcp_rn(static_cast<float>(all));
            // The parts' means m about the first part's, k: k is one mean of a hundred
            // thousand, and where its column or its rows stand apart from the rest the
            // sum of n (m - k)^2 is that many times what is left of it less that of
            // their mean.  So U parts at a time are summed about the first of them in
            // 32 bits, and those sums about k in 64: with z = m_0 - k,
            //     sum n (m - k)^2 = sum n (m - m_0)^2 + 2 z sum n (m - m_0) + z^2 sum n.
            // (4,096 x 1,024 with a first column 1,000 deviations off: rstd within 1.1e-4
            // in 32 bits alone, 1e-7 so.  An SM converts 16 numbers a clock to 64 bits:
            // each part by itself took 9 us longer of 80,000 parts.)
            constexpr int U = 8;
            const double k = part[slot_of(a, g, b / a.R, 0) * a.cols + c0].x;
            double s = 0.0, d = 0.0;
            const Share<W> mine(a, b, e);
            for (int col = mine.first_col; col < a.per; col += mine.wide)
                for (int i = mine.first_slot; i < mine.slots; i += U * mine.step) {
                    float2 p[U];
                    int n[U], rows = 0;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        // (one that is not there: the last, without rows)
                        const int slot = min(i + u * mine.step, mine.slots - 1);
                        p[u] = part[slot_of(a, g, mine.first, slot) * a.cols + c0 + col];
                        n[u] = i + u * mine.step < mine.slots ? mine.rows(a, b, e, slot) : 0;
                        rows += n[u];
                    }
                    float t = 0.0f, q = p[0].y;
#pragma unroll
                    for (int u = 1; u < U; ++u) {
                        const float x = __fsub_rn(p[u].x, p[0].x), w = __fmul_rn(x, static_cast<float>(n[u]));
                        t = __fadd_rn(t, w);
                        q = __fadd_rn(q, fmaf(x, w, n[u] ? p[u].y : 0.0f));
                    }
                    const double z = p[0].x - k, all_t = t, w = z * rows;
                    s += w + all_t;
                    d += fma(z, fma(2.0, all_t, w), static_cast<double>(q));
                }
            sums_of<W>(s, d, sh);
            // (s / all by its quotient in 32 bits and that of the remainder: a division in
            // 64 bits takes 2 us)
            const double near = __fmul_rn(static_cast<float>(s), inv);
            const double shift = near + __fmul_rn(static_cast<float>(fma(-near, all, s)), inv);
            const float var = max_nan(__fmul_rn(static_cast<float>(fma(-s, shift, d)), inv), 0.0f);
            r = make_float2(static_cast<float>(k + shift), __frsqrt_rn(__fadd_rn(var, a.eps)));
        }
        if (threadIdx.x % W == 0) stats[static_cast<int64_t>(g) * a.groups + group] = r;
    });
}

// Each of V columns' (first, second) of its group: one pair where the V columns
// are one group's (SPLIT false).
template <int V, bool SPLIT>
struct OfGroup {
    static constexpr int N = SPLIT ? V : 1;
    float2 at[N];
    __device__ __forceinline__ OfGroup(const GroupArgs& a, const float2* groups, int col) {
#pragma unroll
        for (int j = 0; j < N; ++j) at[j] = groups[min(col + j, a.cols - 1) / a.per];
    }
    __device__ __forceinline__ const float2& operator[](int j) const { return at[SPLIT ? j : 0]; }
};

// A thread's gamma and beta.
template <int V>
struct Params {
    float gamma[V], beta[V];
    template <class T, bool ALIGNED, class P>
    __device__ __forceinline__ Params(const Place<T, ALIGNED>& p, const P* g, const P* b) {
        p.params(g, gamma);
        p.params(b, beta);
    }
};

// y of this thread's rows of [lo, hi), a part of the graph with the groups' statistics `stats`.
template <bool SPLIT, class T, bool ALIGNED, int V>
__device__ __forceinline__ void apply_part(const GroupArgs& a, const Place<T, ALIGNED>& p, const T* x, int64_t ldx,
                                           const Params<V>& k, const float2* stats, T* y, int64_t ldy, int lo, int hi) {
    if (p.n <= 0) return;
    const OfGroup<V, SPLIT> st(a, stats, p.col);
    float A[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = __fmul_rn(k.gamma[j], st[j].y);
    p.template for_rows<4>(a, lo, hi, x, ldx, y, ldy, [&](float (&z)[V], T* to, int) {
        pairs(z, [&](int j, Pair v) {
            return fma2(add2(v, Pair(-st[j].x, -st[j + 1].x)), Pair(A[j], A[j + 1]), Pair(k.beta[j], k.beta[j + 1]));
        });
        act_forward<sizeof(T) == 2>(z, a.act, a.alpha);
        p.store(to, z);
    });
}

template <class T, class P, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(kMaxThreads, kApply<SPLIT>) group_apply_kernel(const GroupArgs a, const T* x, int64_t ldx, const P* gamma,
                                                                  const P* beta, const float2* stats, T* y, int64_t ldy) {
    wait_for_previous();
    if (none_large(a)) return;
    const Place<T, ALIGNED> p(a);
    const int c = blockIdx.x;
    for_parts(a, c, [&](int g, int lo, int hi, int64_t slot) {
        const Params<Place<T, ALIGNED>::V> k(p, gamma, beta);
        apply_part<SPLIT>(a, p, x, ldx, k, stats + static_cast<int64_t>(g) * a.groups, y, ldy, lo, hi);
    });
}

// Adds f(column, group)'s pairs over the columns of each group with the lanes
// that suit a group's width; put(group, sum, lanes, lane) by all of them.
template <int LANES, class F, class G>
__device__ __forceinline__ void over_groups_by(const GroupArgs& a, F&& f, G&& put) {
    const int lane = threadIdx.x % LANES, step = blockDim.x / LANES, first = threadIdx.x / LANES;
    // (all lanes of a warp go round as often)
    for (int i = first; i - first < a.groups; i += step) {
        float2 s = make_float2(0.0f, 0.0f);
        if (i < a.groups)
            for (int c = i * a.per + lane; c < (i + 1) * a.per; c += LANES) {
                const float2 v = f(c, i);
                s.x = __fadd_rn(s.x, v.x);
                s.y = __fadd_rn(s.y, v.y);
            }
        s.x = reduce_sum<float, LANES>(s.x);
        s.y = reduce_sum<float, LANES>(s.y);
        put(i, s, std::integral_constant<int, LANES>{}, lane);
    }
}
template <class F, class G>
__device__ __forceinline__ void over_groups(const GroupArgs& a, F&& f, G&& put) {
    if (a.per <= 4) over_groups_by<1>(a, f, put);
    else if (a.per <= 32) over_groups_by<8>(a, f, put);
    else over_groups_by<32>(a, f, put);
}

constexpr int kSmallCols = 2048;  // most columns of a block that has whole graphs

// A block for each graph of at most a.least rows: its second reading of x comes
// from L1 or L2.
template <class T, class P, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(kMaxThreads, 2) group_small_kernel(const GroupArgs a, const T* x, int64_t ldx, const P* gamma,
                                                                  const P* beta, float2* stats, T* y, int64_t ldy) {
    extern __shared__ float2 room[];
    const Sums<T> sh{room};
    float2 *columns = room + Sums<T>::pairs(blockDim.x), *mine = columns + a.cols;  // the columns', the groups' statistics
    wait_for_previous();
    const Place<T, ALIGNED> p(a);
    const Params<Place<T, ALIGNED>::V> k(p, gamma, beta);
    int large = 0;
    for (int g = blockIdx.x; g < a.graphs; g += gridDim.x) {
        const int b = begin_of(a, g), e = end_of(a, g);
        if (e - b > a.least) {
            large = 1;
            continue;
        }
        float2* out = stats + static_cast<int64_t>(g) * a.groups;
        if (b >= e) {
            for (int i = threadIdx.x; i < a.groups; i += blockDim.x) out[i] = make_float2(0.0f, 0.0f);
            continue;
        }
        part_sums<8>(a, p, x, ldx, b, e, sh);
        __syncthreads();
        for_columns<T>(a, [&](int i, int column) { columns[column] = join_lanes(a, sh, i, e - b); });
        __syncthreads();
        // (the columns of a group have the same number of values)
        const float rows = static_cast<float>(e - b), per = static_cast<float>(a.per);
        over_groups(
            a, [&](int c, int i) { return make_float2(__fsub_rn(columns[c].x, columns[i * a.per].x), 0.0f); },
            [&](int i, float2 s, auto lanes, int lane) {
                constexpr int LANES = decltype(lanes)::value;
                const bool here = i < a.groups;
                const float mean = here ? __fadd_rn(columns[i * a.per].x, __fdiv_rn(s.x, per)) : 0.0f;
                float d = 0.0f;
                if (here)
                    for (int c = i * a.per + lane; c < (i + 1) * a.per; c += LANES) {
                        const float z = __fsub_rn(columns[c].x, mean);
                        d = __fadd_rn(d, fmaf(__fmul_rn(z, z), rows, columns[c].y));
                    }
                d = reduce_sum<float, LANES>(d);
                const float2 r = make_float2(mean, __frsqrt_rn(__fadd_rn(__fdiv_rn(d, __fmul_rn(rows, per)), a.eps)));
                if (here && lane == 0) mine[i] = out[i] = r;
            });
        __syncthreads();
        apply_part<SPLIT>(a, p, x, ldx, k, mine, y, ldy, b, e);
    }
    if (threadIdx.x == 0) a.large[blockIdx.x] = large;
}

// ── backward ─────────────────────────────────────────────────────────────
// What a column's du takes: u = A (x - mean) + beta.
template <int V, bool SPLIT>
struct Slopes {
    float A[V];
    const Params<V>& k;
    OfGroup<V, SPLIT> st;
    __device__ __forceinline__ Slopes(const GroupArgs& a, int col, const Params<V>& k_, const float2* stats) : k(k_), st(a, stats, col) {
#pragma unroll
        for (int j = 0; j < V; ++j) A[j] = __fmul_rn(k.gamma[j], st[j].y);
    }
    // x <- x - mean, dy <- du
    template <bool FAST>
    __device__ __forceinline__ void du(const GroupArgs& a, float (&x)[V], float (&dy)[V]) const {
        float u[V];
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const Pair z = add2(Pair(x[j], x[j + 1]), Pair(-st[j].x, -st[j + 1].x));
            z.get(x[j], x[j + 1]);
            fma2(z, Pair(A[j], A[j + 1]), Pair(k.beta[j], k.beta[j + 1])).get(u[j], u[j + 1]);
        }
        act_slope<FAST>(u, a.act, a.alpha);
        pairs(dy, [&](int j, Pair d) { return mul2(d, Pair(u[j], u[j + 1])); });
    }
};

// This thread's columns' (sum du, sum du h) over its rows of [lo, hi).
template <bool SPLIT, class T, bool ALIGNED, int V>
__device__ __forceinline__ void grad_sums(const GroupArgs& a, const Place<T, ALIGNED>& p, const T* dy, int64_t lddy, const T* x,
                                          int64_t ldx, const Params<V>& params, const float2* stats, int lo, int hi, const Sums<T>& sh) {
    float s[V], t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = t[j] = 0.0f;
    if (p.n > 0) {
        const Slopes<V, SPLIT> k(a, p.col, params, stats);
        p.template for_rows<SPLIT ? 2 : 4>(a, lo, hi, x, ldx, dy, lddy, static_cast<T*>(nullptr), 0, [&](float (&z)[V], float (&d)[V], T*) {
            k.template du<sizeof(T) == 2>(a, z, d);
            pairs(s, [&](int j, Pair v) { return add2(v, Pair(d[j], d[j + 1])); });
            pairs(t, [&](int j, Pair v) { return fma2(Pair(d[j], d[j + 1]), Pair(z[j], z[j + 1]), v); });  // (times r below)
        });
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = __fmul_rn(t[j], k.st[j].y);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sh.set(j, make_float2(s[j], t[j]));
}
template <class T>
__device__ __forceinline__ float2 add_lanes(const GroupArgs& a, const Sums<T>& sh, int c) {
    float2 s = sh.get(a, c, 0);
    for (int y = 1; y < a.ty; ++y) {
        const float2 o = sh.get(a, c, y);
        s.x = __fadd_rn(s.x, o.x);
        s.y = __fadd_rn(s.y, o.y);
    }
    return s;
}

// dx of this thread's rows of [lo, hi); means: the groups' (mean g, mean g h).
template <bool SPLIT, class T, bool ALIGNED, int V>
__device__ __forceinline__ void grad_part(const GroupArgs& a, const Place<T, ALIGNED>& p, const T* dy, int64_t lddy, const T* x,
                                          int64_t ldx, const Params<V>& params, const float2* stats, const float2* means, T* dx,
                                          int64_t lddx, int lo, int hi) {
    if (p.n <= 0) return;
    const Slopes<V, SPLIT> k(a, p.col, params, stats);
    OfGroup<V, SPLIT> de(a, means, p.col);
#pragma unroll
    for (int j = 0; j < de.N; ++j)
        de.at[j] = make_float2(-__fmul_rn(k.st[j].y, de.at[j].x), -__fmul_rn(__fmul_rn(k.st[j].y, k.st[j].y), de.at[j].y));
    p.template for_rows<SPLIT ? 2 : 4>(a, lo, hi, x, ldx, dy, lddy, dx, lddx, [&](float (&z)[V], float (&d)[V], T* to) {
        k.template du<sizeof(T) == 2>(a, z, d);
        pairs(d, [&](int j, Pair v) {
            return fma2(Pair(k.A[j], k.A[j + 1]), v,
                        fma2(Pair(de[j].y, de[j + 1].y), Pair(z[j], z[j + 1]), Pair(de[j].x, de[j + 1].x)));
        });
        p.store(to, d);
    });
}

// part[slot * cols + column] = (sum du, sum du h) of the part; sums[block][2][cols]
// = (sum du h, sum du) over the block's rows.
template <class T, class P, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(kMaxThreads, kGrad) group_grad_parts_kernel(const GroupArgs a, const T* dy, int64_t lddy, const T* x,
                                                                       int64_t ldx, const P* gamma, const P* beta,
                                                                       const float2* stats, float2* part, float* sums) {
    extern __shared__ float2 room[];
    const Sums<T> sh{room};
    float2* total = room + Sums<T>::pairs(blockDim.x);  // of the block's columns
    wait_for_previous();
    if (none_large(a)) return;  // (nor are this block's sums read)
    const Place<T, ALIGNED> p(a);
    for (int i = threadIdx.x; i < a.tx * Sums<T>::V; i += blockDim.x) total[i] = make_float2(0.0f, 0.0f);
    const int c = blockIdx.x;
    for_parts(a, c, [&](int g, int lo, int hi, int64_t slot) {
        const Params<Place<T, ALIGNED>::V> k(p, gamma, beta);
        grad_sums<SPLIT>(a, p, dy, lddy, x, ldx, k, stats + static_cast<int64_t>(g) * a.groups, lo, hi, sh);
        __syncthreads();
        for_columns<T>(a, [&](int i, int column) {
            const float2 s = add_lanes(a, sh, i);
            part[slot * a.cols + column] = s;
            total[i] = make_float2(__fadd_rn(total[i].x, s.x), __fadd_rn(total[i].y, s.y));
        });
        __syncthreads();
    });
    float* out = sums + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    for_columns<T>(a, [&](int i, int column) {
        out[column] = total[i].y;
        out[a.cols + column] = total[i].x;
    });
}

// dgamma and dbeta: the sums of the blocks' rows in their order, kJoinColumns
// columns a block.
constexpr int kJoinColumns = 8;
template <class P>
__device__ __forceinline__ void join_params(const GroupArgs& a, int block, const float* sums, int sum_rows, P* dgamma, P* dbeta,
                                            float* sh) {
    const int c = block * kJoinColumns + threadIdx.x % kJoinColumns, lane = threadIdx.x / kJoinColumns;
    const int lanes = blockDim.x / kJoinColumns;
    float s = 0.0f;
    if (c < 2 * a.cols) {
#pragma unroll 8
        for (int r = lane; r < sum_rows; r += lanes) s = __fadd_rn(s, sums[static_cast<int64_t>(r) * 2 * a.cols + c]);
    }
    // the lanes of a warp have the same columns four times over
    s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 8));
    s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 16));
    if (threadIdx.x % 32 < kJoinColumns) sh[threadIdx.x / 32 * kJoinColumns + threadIdx.x % 32] = s;
    __syncthreads();
    if (lane == 0 && c < 2 * a.cols) {
        s = 0.0f;
        for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) s = __fadd_rn(s, sh[w * kJoinColumns + threadIdx.x]);
        if (c < a.cols) dgamma[c] = from_f32<P>(s);
        else dbeta[c - a.cols] = from_f32<P>(s);
    }
}

// means[g * groups + group] = (mean g, mean g h), in the first `blocks` blocks;
// dgamma and dbeta in the others.
template <class P, int W>
__global__ void __launch_bounds__(kJoinBlock<W>) group_grad_join_kernel(const GroupArgs a, const float2* part, const P* gamma,
                                                                      const float* sums, int sum_rows, int blocks, float2* means,
                                                                      P* dgamma, P* dbeta) {
    __shared__ float sh[kJoinBlock<W> / 32 * kJoinColumns];
    wait_for_previous();
    const bool none = none_large(a);
    if (static_cast<int>(blockIdx.x) >= blocks) {
        join_params(a, static_cast<int>(blockIdx.x) - blocks, sums, none ? a.blocks : sum_rows, dgamma, dbeta, sh);
        return;
    }
    if (none) return;
    for_sets<W>(a, blockIdx.x, [&](int g, int group) {
        const int b = begin_of(a, g), e = end_of(a, g);
        if (b >= e) return;
        float s = 0.0f, t = 0.0f;
        const Share<W> mine(a, b, e);
        for (int col = mine.first_col; col < a.per; col += mine.wide)
#pragma unroll 4
            for (int i = mine.first_slot; i < mine.slots; i += mine.step) {
                const int column = group * a.per + col;
                const float2 p = part[slot_of(a, g, mine.first, i) * a.cols + column];
                const float w = to_f32(gamma[column]);
                s = fmaf(w, p.x, s);
                t = fmaf(w, p.y, t);
            }
        s = sum_of<W>(s, sh);
        t = sum_of<W>(t, sh);
        const float all = __fmul_rn(static_cast<float>(e - b), static_cast<float>(a.per));
        if (threadIdx.x % W == 0)
            means[static_cast<int64_t>(g) * a.groups + group] = make_float2(__fdiv_rn(s, all), __fdiv_rn(t, all));
    });
}

template <class P>
__global__ void __launch_bounds__(kJoinThreads) group_params_kernel(const GroupArgs a, const float* sums, int sum_rows, P* dgamma,
                                                                   P* dbeta) {
    __shared__ float sh[kJoinThreads / 32 * kJoinColumns];
    wait_for_previous();
    join_params(a, static_cast<int>(blockIdx.x), sums, sum_rows, dgamma, dbeta, sh);
}

template <class T, class P, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(kMaxThreads, kGrad) group_grad_apply_kernel(const GroupArgs a, const T* dy, int64_t lddy, const T* x,
                                                                       int64_t ldx, const P* gamma, const P* beta,
                                                                       const float2* stats, const float2* means, T* dx,
                                                                       int64_t lddx) {
    wait_for_previous();
    if (none_large(a)) return;
    const Place<T, ALIGNED> p(a);
    const int c = blockIdx.x;
    for_parts(a, c, [&](int g, int lo, int hi, int64_t slot) {
        const Params<Place<T, ALIGNED>::V> k(p, gamma, beta);
        const int64_t o = static_cast<int64_t>(g) * a.groups;
        grad_part<SPLIT>(a, p, dy, lddy, x, ldx, k, stats + o, means + o, dx, lddx, lo, hi);
    });
}

// A block for each graph of at most a.least rows.
template <class T, class P, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(kMaxThreads, 2) group_grad_small_kernel(const GroupArgs a, const T* dy, int64_t lddy, const T* x,
                                                                       int64_t ldx, const P* gamma, const P* beta,
                                                                       const float2* stats, T* dx, int64_t lddx, float* sums) {
    extern __shared__ float2 room[];
    const Sums<T> sh{room};
    // the columns' sums in a graph and in all, the groups' means
    float2 *columns = room + Sums<T>::pairs(blockDim.x), *total = columns + a.cols, *means = total + a.cols;
    wait_for_previous();
    const Place<T, ALIGNED> p(a);
    const Params<Place<T, ALIGNED>::V> k(p, gamma, beta);
    for (int i = threadIdx.x; i < a.cols; i += blockDim.x) total[i] = make_float2(0.0f, 0.0f);
    int large = 0;
    for (int g = blockIdx.x; g < a.graphs; g += gridDim.x) {
        const int b = begin_of(a, g), e = end_of(a, g);
        large |= e - b > a.least;
        if (b >= e || e - b > a.least) continue;
        const float2* st = stats + static_cast<int64_t>(g) * a.groups;
        grad_sums<SPLIT>(a, p, dy, lddy, x, ldx, k, st, b, e, sh);
        __syncthreads();
        for_columns<T>(a, [&](int i, int column) {
            const float2 s = add_lanes(a, sh, i);
            const float w = to_f32(gamma[column]);
            columns[column] = make_float2(__fmul_rn(w, s.x), __fmul_rn(w, s.y));
            total[column] = make_float2(__fadd_rn(total[column].x, s.x), __fadd_rn(total[column].y, s.y));
        });
        __syncthreads();
        const float all = __fmul_rn(static_cast<float>(e - b), static_cast<float>(a.per));
        over_groups(
            a, [&](int c, int) { return columns[c]; },
            [&](int i, float2 s, auto, int lane) {
                if (i < a.groups && lane == 0) means[i] = make_float2(__fdiv_rn(s.x, all), __fdiv_rn(s.y, all));
            });
        __syncthreads();
        grad_part<SPLIT>(a, p, dy, lddy, x, ldx, k, st, means, dx, lddx, b, e);
    }
    __syncthreads();
    float* out = sums + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
        out[i] = total[i].y;
        out[a.cols + i] = total[i].x;
    }
    if (threadIdx.x == 0) a.large[blockIdx.x] = large;
}

// ── host ─────────────────────────────────────────────────────────────────
// f(rows aligned, vectors of several groups)
template <class T, class F>
void by_layout(const GroupArgs& a, bool aligned, F&& f) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    using std::false_type;
    using std::true_type;
    if (!aligned || a.cols % V != 0) f(false_type{}, true_type{});
    else if (a.per % V != 0) f(true_type{}, true_type{});
    else f(true_type{}, false_type{});
}

// Blocks as wide as the row (or an even share of it), up to 256 threads and 32
// row lanes, and one chunk for each of the `resident` blocks of an SM: a kernel
// whose blocks run in one and a third waves takes as long as with two.
GroupArgs cut(GroupArgs a, int V, int resident) {
    a.nv = static_cast<int>(ceil_div(a.cols, V));
    const int blocks = static_cast<int>(ceil_div(a.nv, kMaxThreads));
    a.tx = static_cast<int>(ceil_div(a.nv, blocks));
    a.ty = std::min(std::max(1, kMaxThreads / a.tx), 32);
    const int threads = (a.tx * a.ty + 31) / 32 * 32;
    const int64_t each = std::max<int64_t>(1, int64_t(num_sms()) * resident * (kMaxThreads / threads) / blocks);
    a.R = a.ty * static_cast<int>(std::max<int64_t>(1, ceil_div(a.rows, each * a.ty)));
    a.chunks = static_cast<int>(ceil_div(a.rows, a.R));
    return a;
}
// Most rows of a graph that is a block's: 64 KB, or the rows of a chunk.  0 where
// graphs are larger than half of that on the average: then all are cut in chunks,
// since a block has no other graph to go on with.  64 columns fp32, forward and
// gradient, us with whole graphs / in chunks alone: 2,048 graphs of 25 rows 24 + 25
// / 33 + 31, 16,384 80 + 105 / 167 + 204, 2,047 of one row and one of 49,153 46 + 37 /
// 337 + 435.  (About 10 of each are the launches that find no larger graph: without
// them 11 + 16, and 1,944 + 3,599 where there is one.)
int small_rows(const GroupArgs& a, size_t size) {
    const int64_t row = a.cols * static_cast<int64_t>(size);
    if (a.nv > kMaxThreads || a.cols > kSmallCols || a.graphs == 0 || a.rows / a.graphs * row > 32 << 10) return 0;
    return static_cast<int>(std::max<int64_t>(std::max<int64_t>((64 << 10) / row, 1), a.R));
}
// The cut of such graphs: eight rows a lane, where there are blocks enough.
GroupArgs cut_small(GroupArgs a) {
    if (a.graphs < 4 * num_sms()) return a;
    const int64_t lanes = std::max<int64_t>(ceil_div(ceil_div(a.rows, a.graphs), 8), 1);
    a.ty = static_cast<int>(std::min<int64_t>(a.ty, std::max<int64_t>(lanes, ceil_div(32, a.tx))));
    return a;
}
dim3 block_of(const GroupArgs& a) { return dim3(static_cast<unsigned>((a.tx * a.ty + 31) / 32 * 32)); }
dim3 grid_of(const GroupArgs& a) { return dim3(static_cast<unsigned>(a.chunks), static_cast<unsigned>(ceil_div(a.nv, a.tx))); }
// Blocks with `room` bytes of shared memory that run at a time, at most one a graph (`threads` an SM).
int small_blocks(const GroupArgs& a, size_t room, int threads) {
    const int fit = std::min({16, threads / static_cast<int>(block_of(a).x), static_cast<int>(228 * 1024 / (room + 1024))});
    return static_cast<int>(std::min<int64_t>(a.graphs, int64_t(num_sms()) * std::max(1, fit)));
}
size_t slots_of(const GroupArgs& a) {
    return (a.least ? 2 * static_cast<size_t>(a.chunks) : static_cast<size_t>(a.chunks) + a.graphs) * a.cols;
}
template <int W>
unsigned join_blocks(const GroupArgs& a, int64_t sets) {
    return static_cast<unsigned>(a.least ? int64_t(a.chunks) * large_blocks(a.groups) : ceil_div(sets, kJoinBlock<W> / W));
}
// Calls f with the threads that join a graph's group: by its parts, were the
// graphs alike (256 for the large ones among small ones).
template <class F>
void by_parts(const GroupArgs& a, F&& f) {
    if (a.least) return f(std::integral_constant<int, 256>{});
    const int64_t parts = (a.rows / a.R / std::max(a.graphs, 1) + 1) * a.per;
    if (parts <= 256) f(std::integral_constant<int, 32>{});
    else if (parts <= 4096) f(std::integral_constant<int, 256>{});
    else f(std::integral_constant<int, kJoinThreads>{});
}

void check_group(const char* fn, int64_t rows, int64_t cols, int64_t groups, int64_t graphs, const int32_t* offsets, int dtype,
                 int param_dtype, int act) {
    check_dtype(fn, "x", dtype);
    if (param_dtype != TG_F32 && param_dtype != dtype)
        invalid(std::string(fn) + ": gamma and beta must be fp32 or of the rows' type");
    check_rows_cols(fn, rows, cols);
    if (rows > INT32_MAX - 1024) invalid(std::string(fn) + ": more than 2^31 - 1024 rows");  // (row lanes count past the last)
    if (groups < 1 || cols % groups != 0)
        invalid(std::string(fn) + ": " + std::to_string(cols) + " columns cannot be cut into " + std::to_string(groups) + " groups");
    if (graphs < 0 || graphs > (1 << 24)) invalid(std::string(fn) + ": " + std::to_string(graphs) + " graphs are outside [0, 2^24]");
    if (graphs * groups > INT32_MAX) invalid(std::string(fn) + ": more than 2^31 groups in all graphs");
    check_ptr(fn, "offsets", offsets, graphs != 1);
    check_act(fn, act);
}

template <class F>
void by_types(int dtype, int param_dtype, F&& f) {
    by_dtype(dtype, [&](auto t) {
        if (param_dtype == TG_F32) f(t, float{});
        else f(t, t);
    });
}

}  // namespace

}  // namespace tg

extern "C" {

TG_API tg_status tg_group_norm(int64_t rows, int64_t cols, int64_t groups, int64_t graphs, const int32_t* offsets,
                               int32_t dtype, const void* x, int64_t ldx, int32_t param_dtype, const void* gamma,
                               const void* beta, float eps, int32_t act, float alpha, void* y, int64_t ldy, float* stats,
                               void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "group_norm";
        check_group(fn, rows, cols, groups, graphs, offsets, dtype, param_dtype, act);
        check_ptr(fn, "x", x, rows > 0);
        check_ptr(fn, "y", y, rows > 0);
        check_ptr(fn, "gamma", gamma, true);
        check_ptr(fn, "beta", beta, true);
        check_ptr(fn, "stats", stats, graphs > 0);
        check_ld(fn, "x", ldx, cols);
        check_ld(fn, "y", ldy, cols);
        if (!(eps >= 0.0f)) invalid("group_norm: eps must not be negative");
        if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) invalid("group_norm: stats must be 8-byte aligned");
        if (graphs == 0) return;
        cudaStream_t s = as_stream(stream);
        const GroupArgs g{rows, static_cast<int>(cols), static_cast<int>(groups), static_cast<int>(cols / groups), static_cast<int>(graphs), offsets, act, alpha, eps};
        by_types(dtype, param_dtype, [&](auto t, auto pt) {
            using T = decltype(t);
            using P = decltype(pt);
            const T* xp = static_cast<const T*>(x);
            const P *ga = static_cast<const P*>(gamma), *be = static_cast<const P*>(beta);
            const bool aligned = rows_aligned16(x, ldx, sizeof(T)) && rows_aligned16(y, ldy, sizeof(T));
            GroupArgs a = cut(g, 16 / sizeof(T), kParts);
            a.least = small_rows(a, sizeof(T));
            float2* st = reinterpret_cast<float2*>(stats);
            by_layout<T>(a, aligned, [&](auto al, auto split) {
                constexpr bool ALIGNED = decltype(al)::value, SPLIT = decltype(split)::value;
                const GroupArgs small = cut_small(a);
                const size_t room = (Sums<T>::pairs(block_of(small).x) + cols + groups) * sizeof(float2);
                const bool chunks = a.least == 0 || rows > a.least;  // else there is no larger graph
                a.blocks = a.least ? small_blocks(small, room, 512) : 0;
                // (one allocation: each takes the host 2 us)
                Scratch<float2> part((chunks ? slots_of(a) : 0) + (a.blocks + 1) / 2, s);
                a.large = reinterpret_cast<int*>(part.p + (chunks ? slots_of(a) : 0));
                if (a.least) {
                    GroupArgs c = small;
                    c.blocks = a.blocks;
                    c.large = a.large;
                    auto kern = group_small_kernel<T, P, ALIGNED, SPLIT>;
                    if (room > 48 * 1024) allow_shared(kern, kMaxShared);
                    launch_dependent("group_norm", kern, dim3(static_cast<unsigned>(c.blocks)), block_of(c), room, s, c, xp, ldx,
                                     ga, be, st, static_cast<T*>(y), ldy);
                    if (!chunks) return;
                }
                launch_dependent("group_norm_parts", group_parts_kernel<T, ALIGNED>, grid_of(a), block_of(a),
                                 Sums<T>::pairs(block_of(a).x) * sizeof(float2), s, a, xp, ldx, part.p);
                const int64_t sets = graphs * groups;
                by_parts(a, [&](auto width) {
                    constexpr int W = decltype(width)::value;
                    launch_dependent("group_norm_stats", group_stats_kernel<W>, dim3(join_blocks<W>(a, sets)), dim3(kJoinBlock<W>), 0, s, a, part.p,
                                     st);
                });
                GroupArgs c = cut(g, 16 / sizeof(T), kApply<SPLIT>);
                c.least = a.least, c.large = a.large, c.blocks = a.blocks;
                launch_dependent("group_norm", group_apply_kernel<T, P, ALIGNED, SPLIT>, grid_of(c), block_of(c), 0, s, c, xp, ldx, ga,
                                 be, st, static_cast<T*>(y), ldy);
            });
        });
    });
}

TG_API tg_status tg_group_norm_grad(int64_t rows, int64_t cols, int64_t groups, int64_t graphs, const int32_t* offsets,
                                    int32_t dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                    const float* stats, int32_t param_dtype, const void* gamma, const void* beta,
                                    int32_t act, float alpha, void* dx, int64_t lddx, void* dgamma, void* dbeta,
                                    void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "group_norm_grad";
        check_group(fn, rows, cols, groups, graphs, offsets, dtype, param_dtype, act);
        check_ptr(fn, "dy", dy, rows > 0);
        check_ptr(fn, "x", x, rows > 0);
        check_ptr(fn, "dx", dx, rows > 0);
        check_ptr(fn, "gamma", gamma, true);
        check_ptr(fn, "beta", beta, true);
        check_ptr(fn, "dgamma", dgamma, true);
        check_ptr(fn, "dbeta", dbeta, true);
        check_ptr(fn, "stats", stats, graphs > 0);
        check_ld(fn, "dy", lddy, cols);
        check_ld(fn, "x", ldx, cols);
        check_ld(fn, "dx", lddx, cols);
        if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) invalid("group_norm_grad: stats must be 8-byte aligned");
        cudaStream_t s = as_stream(stream);
        const GroupArgs g{rows, static_cast<int>(cols), static_cast<int>(groups), static_cast<int>(cols / groups), static_cast<int>(graphs), offsets, act, alpha, 0.0f};
        by_types(dtype, param_dtype, [&](auto t, auto pt) {
            using T = decltype(t);
            using P = decltype(pt);
            const T *xp = static_cast<const T*>(x), *dyp = static_cast<const T*>(dy);
            const P *ga = static_cast<const P*>(gamma), *be = static_cast<const P*>(beta);
            const bool aligned = rows_aligned16(x, ldx, sizeof(T)) && rows_aligned16(dy, lddy, sizeof(T)) &&
                                 rows_aligned16(dx, lddx, sizeof(T));
            GroupArgs a = cut(g, 16 / sizeof(T), kGrad);
            a.least = small_rows(a, sizeof(T));
            const float2* st = reinterpret_cast<const float2*>(stats);
            const int col_blocks = static_cast<int>(ceil_div(2 * cols, kJoinColumns));
            P *dg = static_cast<P*>(dgamma), *db = static_cast<P*>(dbeta);
            by_layout<T>(a, aligned, [&](auto al, auto split) {
                constexpr bool ALIGNED = decltype(al)::value, SPLIT = decltype(split)::value;
                // dgamma's and dbeta's sums of the blocks that have whole graphs, then those of the chunks
                GroupArgs c = cut_small(a);
                const size_t room = (Sums<T>::pairs(block_of(c).x) + 2 * cols + groups) * sizeof(float2);
                const int small = a.least ? small_blocks(c, room, 512) : 0;
                a.blocks = c.blocks = small;
                const bool large = a.least == 0 || rows > a.least;
                const dim3 grid = grid_of(a);
                const int sum_rows = small + (large ? static_cast<int>(grid.x) : 0);
                const size_t sets = static_cast<size_t>(graphs) * groups;
                // the parts, the groups' means, the blocks' sums and whether they met a larger graph
                Scratch<float2> part((large ? slots_of(a) + sets : 0) + static_cast<size_t>(sum_rows) * cols + (small + 1) / 2, s);
                float2* means = part.p + slots_of(a);
                float* sums = reinterpret_cast<float*>(large ? means + sets : part.p);
                a.large = c.large = reinterpret_cast<int*>(sums + static_cast<size_t>(sum_rows) * 2 * cols);
                if (a.least) {
                    auto kern = group_grad_small_kernel<T, P, ALIGNED, SPLIT>;
                    if (room > 48 * 1024) allow_shared(kern, kMaxShared);
                    launch_dependent("group_norm_grad", kern, dim3(static_cast<unsigned>(small)), block_of(c), room, s, c, dyp, lddy, xp,
                                     ldx, ga, be, st, static_cast<T*>(dx), lddx, sums);
                    if (!large) {
                        launch_dependent("group_norm_grad_params", group_params_kernel<P>, dim3(static_cast<unsigned>(col_blocks)),
                                         dim3(kJoinThreads), 0, s, c, sums, sum_rows, dg, db);
                        return;
                    }
                }
                launch_dependent("group_norm_grad_parts", group_grad_parts_kernel<T, P, ALIGNED, SPLIT>, grid, block_of(a),
                                 (Sums<T>::pairs(block_of(a).x) + a.tx * (16 / sizeof(T))) * sizeof(float2), s, a, dyp, lddy, xp, ldx, ga,
                                 be, st, part.p, sums + static_cast<size_t>(small) * 2 * cols);
                by_parts(a, [&](auto width) {
                    constexpr int W = decltype(width)::value;
                    const int blocks = static_cast<int>(join_blocks<W>(a, sets));
                    launch_dependent("group_norm_grad_join", group_grad_join_kernel<P, W>,
                                     dim3(static_cast<unsigned>(blocks + col_blocks)), dim3(kJoinBlock<W>), 0, s, a, part.p, ga, sums,
                                     sum_rows, blocks, means, dg, db);
                });
                launch_dependent("group_norm_grad", group_grad_apply_kernel<T, P, ALIGNED, SPLIT>, grid, block_of(a), 0, s, a, dyp, lddy,
                                 xp, ldx, ga, be, st, means, static_cast<T*>(dx), lddx);
            });
        });
    });
}

}  // extern "C"

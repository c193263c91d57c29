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
//  vector in every TY-th row of it, and splits a chunk where a graph ends.  The
//  first pass leaves one partial result for each vector of columns, chunk and
//  graph in it; chunk c's part of graph g is slot c + g, which no other part
//  has, and there are at most chunks + graphs of them.  A second, small kernel
//  joins a graph's slots in their order (no atomics, the same bits every run),
//  and a third applies the statistics.
//
//  A part's mean and sum of squared deviations come from one pass: each thread
//  sums x - k and (x - k)^2 with k its own first value, which cannot lose the
//  deviations (k is one of the few values it is subtracted from), and parts are
//  joined by their means and deviations, not by sums of squares.
// ============================================================================
#include <algorithm>

#include "typed.cuh"

namespace tg {

namespace {

// V values (or one of any alignment) in loads of at most 16 bytes.
template <class T, int V>
__device__ __forceinline__ void load_cols(const T* p, float (&x)[V]) {
    constexpr int N = V * static_cast<int>(sizeof(T)) > 16 ? 16 / static_cast<int>(sizeof(T)) : V;
    if constexpr (V == 1) {
        x[0] = to_f32(*p);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += N) widen(load_raw<T, N>(p + i), x + i);
    }
}
template <class T, int V>
__device__ __forceinline__ void store_cols(T* p, const float (&x)[V]) {
    if constexpr (V == 1) *p = from_f32<T>(x[0]);
    else store_v<T, V>(p, x);
}

struct GroupArgs {
    int64_t rows;
    int cols, groups, graphs;
    const int32_t* offsets;  // nullable: one graph of all rows
    int act;
    float alpha, eps;
    // the cut
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
// Calls f(g, first row, end) for the graphs' parts of chunk c.
template <class F>
__device__ __forceinline__ void for_parts(const GroupArgs& a, int c, F&& f) {
    const int64_t c0 = static_cast<int64_t>(c) * a.R, c1 = c0 + a.R < a.rows ? c0 + a.R : a.rows;
    for (int g = graph_at(a, static_cast<int>(c0)); g < a.graphs; ++g) {
        const int b = begin_of(a, g), e = end_of(a, g);
        if (b >= c1) break;
        const int lo = b > c0 ? b : static_cast<int>(c0), hi = e < c1 ? e : static_cast<int>(c1);
        if (lo < hi) f(g, lo, hi);
        if (e >= c1) break;
    }
}

// A thread's place.
struct Place {
    int tx, ty, vec;
    bool here;  // it has columns
    __device__ __forceinline__ explicit Place(const GroupArgs& a) {
        tx = threadIdx.x % a.tx;
        ty = threadIdx.x / a.tx;
        vec = blockIdx.y * a.tx + tx;
        here = ty < a.ty && vec < a.nv;
    }
};

// The sum over the row lanes of a block of two values a thread, in those of the first.
__device__ __forceinline__ float2 over_lanes(const GroupArgs& a, const Place& p, float2 v, float2* sh) {
    __syncthreads();
    sh[threadIdx.x] = v;
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
    if (p.ty == 0)
        for (int y = 0; y < a.ty; ++y) {
            const float2 o = sh[y * a.tx + p.tx];
            s.x = __fadd_rn(s.x, o.x);
            s.y = __fadd_rn(s.y, o.y);
        }
    return s;
}

constexpr int kMaxThreads = 256;

// ── forward ──────────────────────────────────────────────────────────────
// part[slot * nv + vec] = (mean, sum of squared deviations) of the part's values.
template <class T, int V>
__global__ void __launch_bounds__(kMaxThreads) group_parts_kernel(const GroupArgs a, const T* x, int64_t ldx, float2* part) {
    __shared__ float2 sh[kMaxThreads];
    wait_for_previous();
    const Place p(a);
    for (int c = blockIdx.x; c < a.chunks; c += gridDim.x)
        for_parts(a, c, [&](int g, int lo, int hi) {
            float s = 0.0f, q = 0.0f, k = 0.0f;
            int n = 0;
            if (p.here) {
                const T* at = x + static_cast<int64_t>(p.vec) * V;
                constexpr int U = 4;
                if (lo + p.ty < hi) k = to_f32(at[(lo + p.ty) * ldx]);
                for (int r = lo + p.ty; r < hi; r += a.ty * U) {
                    float z[U][V];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (r + u * a.ty < hi) load_cols<T, V>(at + (r + u * a.ty) * ldx, z[u]);
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (r + u * a.ty < hi) {
                            ++n;
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                const float d = __fsub_rn(z[u][j], k);
                                s = __fadd_rn(s, d);
                                q = fmaf(d, d, q);
                            }
                        }
                }
            }
            const float cnt = static_cast<float>(n * V), inv = n ? __fdiv_rn(1.0f, cnt) : 0.0f;
            const float m = fmaf(s, inv, k), d = max_nan(fmaf(-s, __fmul_rn(s, inv), q), 0.0f);
            // the row lanes' parts: lane y has the rows lo + y, + ty, ...
            __syncthreads();
            sh[threadIdx.x] = make_float2(m, d);
            __syncthreads();
            if (p.ty == 0 && p.here) {
                float sum = 0.0f, dev = 0.0f;
                const int rows = hi - lo;
                const auto lane_rows = [&](int y) { return static_cast<float>((rows - y + a.ty - 1) / a.ty); };
                const int lanes = rows < a.ty ? rows : a.ty;
                for (int y = 0; y < lanes; ++y) sum = fmaf(__fsub_rn(sh[y * a.tx + p.tx].x, m), lane_rows(y), sum);
                const float mean = __fadd_rn(m, __fdiv_rn(sum, static_cast<float>(rows)));
                for (int y = 0; y < lanes; ++y) {
                    const float2 o = sh[y * a.tx + p.tx];
                    const float e = __fsub_rn(o.x, mean);
                    dev = __fadd_rn(dev, fmaf(__fmul_rn(e, e), __fmul_rn(lane_rows(y), V), o.y));
                }
                part[static_cast<int64_t>(c + g) * a.nv + p.vec] = make_float2(mean, dev);
            }
        });
}

// Calls f(part, rows of it) for this thread's parts of a graph's group, one of
// W threads; w vectors of the group from v0 on.
template <int W, class F>
__device__ __forceinline__ void for_slots(const GroupArgs& a, int g, int b, int e, int v0, int w, const float2* part, F&& f) {
    const int c0 = b / a.R, c1 = (e - 1) / a.R;
    const int64_t items = static_cast<int64_t>(c1 - c0 + 1) * w;
    for (int64_t i = threadIdx.x % W; i < items; i += W) {
        const int c = c0 + static_cast<int>(i / w), v = v0 + static_cast<int>(i % w);
        const int64_t r0 = static_cast<int64_t>(c) * a.R, r1 = r0 + a.R;
        f(part[static_cast<int64_t>(c + g) * a.nv + v], static_cast<int>((e < r1 ? e : r1) - (b > r0 ? b : r0)));
    }
}
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

// stats[g * groups + group] = (mean, rstd), (0, 0) for a graph without rows.
template <int V, int W>
__global__ void __launch_bounds__(kMaxThreads) group_stats_kernel(const GroupArgs a, const float2* part, float2* stats) {
    __shared__ float sh[8];
    wait_for_previous();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (kMaxThreads / W) + threadIdx.x / W;
    if (i >= static_cast<int64_t>(a.graphs) * a.groups) return;
    const int g = static_cast<int>(i / a.groups), per = a.nv / a.groups, v0 = static_cast<int>(i % a.groups) * per;
    const int b = begin_of(a, g), e = end_of(a, g);
    float2 r = make_float2(0.0f, 0.0f);
    if (b < e) {
        const float rows = static_cast<float>(e - b), all = __fmul_rn(rows, static_cast<float>(per * V));
        // (about the first part's mean, so that the sum does not lose the differences)
        const float k = part[static_cast<int64_t>(b / a.R + g) * a.nv + v0].x;
        float s = 0.0f, d = 0.0f;
        for_slots<W>(a, g, b, e, v0, per, part, [&](float2 p, int n) { s = fmaf(__fsub_rn(p.x, k), static_cast<float>(n), s); });
        const float mean = __fadd_rn(k, __fdiv_rn(sum_of<W>(s, sh), __fmul_rn(rows, static_cast<float>(per))));
        for_slots<W>(a, g, b, e, v0, per, part, [&](float2 p, int n) {
            const float x = __fsub_rn(p.x, mean);
            d = __fadd_rn(d, fmaf(__fmul_rn(x, x), __fmul_rn(static_cast<float>(n), V), p.y));
        });
        const float var = __fdiv_rn(sum_of<W>(d, sh), all);
        r = make_float2(mean, __frsqrt_rn(__fadd_rn(var, a.eps)));
    }
    if (threadIdx.x % W == 0) stats[i] = r;
}

template <class T, class P, int V>
__global__ void __launch_bounds__(kMaxThreads) group_apply_kernel(const GroupArgs a, const T* x, int64_t ldx, const P* gamma,
                                                                  const P* beta, const float2* stats, T* y, int64_t ldy) {
    wait_for_previous();
    const Place p(a);
    const int64_t col = static_cast<int64_t>(p.vec) * V;
    float ga[V], be[V];
    if (p.here) {
        load_cols<P, V>(gamma + col, ga);
        load_cols<P, V>(beta + col, be);
    }
    const int group = p.here ? p.vec / (a.nv / a.groups) : 0;
    for (int c = blockIdx.x; c < a.chunks; c += gridDim.x)
        for_parts(a, c, [&](int g, int lo, int hi) {
            if (!p.here) return;
            const float2 st = stats[static_cast<int64_t>(g) * a.groups + group];
            const T* at = x + col;
            T* to = y + col;
            constexpr int U = 4;
            for (int r = lo + p.ty; r < hi; r += a.ty * U) {
                float z[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + u * a.ty < hi) load_cols<T, V>(at + (r + u * a.ty) * ldx, z[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + u * a.ty < hi) {
#pragma unroll
                        for (int j = 0; j < V; ++j) z[u][j] = fmaf(__fmul_rn(__fsub_rn(z[u][j], st.x), st.y), ga[j], be[j]);
                        act_forward<sizeof(T) == 2>(z[u], a.act, a.alpha);
                        store_cols<T, V>(to + (r + u * a.ty) * ldy, z[u]);
                    }
            }
        });
}

// ── backward ─────────────────────────────────────────────────────────────
// h and du of V values.
template <class T, int V>
__device__ __forceinline__ void slopes(const GroupArgs& a, float (&x)[V], float (&dy)[V], const float (&ga)[V],
                                       const float (&be)[V], float2 st) {
    float u[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        x[j] = __fmul_rn(__fsub_rn(x[j], st.x), st.y);
        u[j] = fmaf(x[j], ga[j], be[j]);
    }
    act_slope<sizeof(T) == 2>(u, a.act, a.alpha);
#pragma unroll
    for (int j = 0; j < V; ++j) dy[j] = __fmul_rn(dy[j], u[j]);
}

// part[slot * nv + vec] = (sum g, sum g h) of the part; sums[block][2][cols] =
// (sum du h, sum du) over the block's rows.
template <class T, class P, int V>
__global__ void __launch_bounds__(kMaxThreads) group_grad_parts_kernel(const GroupArgs a, const T* dy, int64_t lddy, const T* x,
                                                                       int64_t ldx, const P* gamma, const P* beta,
                                                                       const float2* stats, float2* part, float* sums) {
    __shared__ float2 sh[kMaxThreads];
    wait_for_previous();
    const Place p(a);
    const int64_t col = static_cast<int64_t>(p.vec) * V;
    float ga[V], be[V], dg[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) ga[j] = be[j] = dg[j] = db[j] = 0.0f;
    if (p.here) {
        load_cols<P, V>(gamma + col, ga);
        load_cols<P, V>(beta + col, be);
    }
    const int group = p.here ? p.vec / (a.nv / a.groups) : 0;
    for (int c = blockIdx.x; c < a.chunks; c += gridDim.x)
        for_parts(a, c, [&](int g, int lo, int hi) {
            float2 sum = make_float2(0.0f, 0.0f);
            if (p.here) {
                const float2 st = stats[static_cast<int64_t>(g) * a.groups + group];
                float s[V], sh_[V];
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] = sh_[j] = 0.0f;
                constexpr int U = 2;
                for (int r = lo + p.ty; r < hi; r += a.ty * U) {
                    float z[U][V], d[U][V];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (r + u * a.ty < hi) {
                            load_cols<T, V>(x + col + (r + u * a.ty) * ldx, z[u]);
                            load_cols<T, V>(dy + col + (r + u * a.ty) * lddy, d[u]);
                        }
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (r + u * a.ty < hi) {
                            slopes<T, V>(a, z[u], d[u], ga, be, st);
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                s[j] = __fadd_rn(s[j], d[u][j]);
                                sh_[j] = fmaf(d[u][j], z[u][j], sh_[j]);
                            }
                        }
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sum.x = fmaf(ga[j], s[j], sum.x);
                    sum.y = fmaf(ga[j], sh_[j], sum.y);
                    db[j] = __fadd_rn(db[j], s[j]);
                    dg[j] = __fadd_rn(dg[j], sh_[j]);
                }
            }
            sum = over_lanes(a, p, sum, sh);
            if (p.ty == 0 && p.here) part[static_cast<int64_t>(c + g) * a.nv + p.vec] = sum;
        });
    float* out = sums + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll 1
    for (int j = 0; j < V; ++j) {
        float2 v = make_float2(dg[0], db[0]);
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (i == j) v = make_float2(dg[i], db[i]);
        v = over_lanes(a, p, v, sh);
        if (p.ty == 0 && p.here) {
            out[col + j] = v.x;
            out[a.cols + col + j] = v.y;
        }
    }
}

// coef[g * groups + group] = (mean g, mean g h), in the first `blocks` blocks;
// dgamma and dbeta, the sums of the blocks' rows in their order, in the others.
template <class P, int V, int W>
__global__ void __launch_bounds__(kMaxThreads) group_grad_join_kernel(const GroupArgs a, const float2* part, const float* sums,
                                                                      int sum_rows, int blocks, float2* coef, P* dgamma,
                                                                      P* dbeta) {
    __shared__ float sh[kMaxThreads];
    wait_for_previous();
    if (static_cast<int>(blockIdx.x) < blocks) {
        const int64_t i = static_cast<int64_t>(blockIdx.x) * (kMaxThreads / W) + threadIdx.x / W;
        if (i >= static_cast<int64_t>(a.graphs) * a.groups) return;
        const int g = static_cast<int>(i / a.groups), per = a.nv / a.groups, v0 = static_cast<int>(i % a.groups) * per;
        const int b = begin_of(a, g), e = end_of(a, g);
        if (b >= e) return;
        float s = 0.0f, t = 0.0f;
        for_slots<W>(a, g, b, e, v0, per, part, [&](float2 p, int) {
            s = __fadd_rn(s, p.x);
            t = __fadd_rn(t, p.y);
        });
        s = sum_of<W>(s, sh);
        t = sum_of<W>(t, sh);
        const float all = __fmul_rn(static_cast<float>(e - b), static_cast<float>(per * V));
        if (threadIdx.x % W == 0) coef[i] = make_float2(__fdiv_rn(s, all), __fdiv_rn(t, all));
        return;
    }
    const int c = (blockIdx.x - blocks) * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < 2 * a.cols)
        for (int r = lane; r < sum_rows; r += kMaxThreads / 32) s = __fadd_rn(s, sums[static_cast<int64_t>(r) * 2 * a.cols + c]);
    sh[threadIdx.x] = s;
    __syncthreads();
    if (lane == 0 && c < 2 * a.cols) {
        s = 0.0f;
        for (int w = 0; w < kMaxThreads / 32; ++w) s = __fadd_rn(s, sh[w * 32 + threadIdx.x]);
        if (c < a.cols) dgamma[c] = from_f32<P>(s);
        else dbeta[c - a.cols] = from_f32<P>(s);
    }
}

template <class T, class P, int V>
__global__ void __launch_bounds__(kMaxThreads) group_grad_apply_kernel(const GroupArgs a, const T* dy, int64_t lddy, const T* x,
                                                                       int64_t ldx, const P* gamma, const P* beta,
                                                                       const float2* stats, const float2* coef, T* dx,
                                                                       int64_t lddx) {
    wait_for_previous();
    const Place p(a);
    const int64_t col = static_cast<int64_t>(p.vec) * V;
    float ga[V], be[V];
    if (p.here) {
        load_cols<P, V>(gamma + col, ga);
        load_cols<P, V>(beta + col, be);
    }
    const int group = p.here ? p.vec / (a.nv / a.groups) : 0;
    for (int c = blockIdx.x; c < a.chunks; c += gridDim.x)
        for_parts(a, c, [&](int g, int lo, int hi) {
            if (!p.here) return;
            const float2 st = stats[static_cast<int64_t>(g) * a.groups + group];
            const float2 co = coef[static_cast<int64_t>(g) * a.groups + group];
            constexpr int U = 2;
            for (int r = lo + p.ty; r < hi; r += a.ty * U) {
                float z[U][V], d[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + u * a.ty < hi) {
                        load_cols<T, V>(x + col + (r + u * a.ty) * ldx, z[u]);
                        load_cols<T, V>(dy + col + (r + u * a.ty) * lddy, d[u]);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + u * a.ty < hi) {
                        slopes<T, V>(a, z[u], d[u], ga, be, st);
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            d[u][j] = __fmul_rn(st.y, fmaf(-z[u][j], co.y, fmaf(ga[j], d[u][j], -co.x)));
                        store_cols<T, V>(dx + col + (r + u * a.ty) * lddx, d[u]);
                    }
            }
        });
}

// ── host ─────────────────────────────────────────────────────────────────
template <class T, class P, class F>
void by_vector(int64_t cols, int64_t groups, bool aligned, F&& f) {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const int64_t per = cols / groups;
    if (aligned && per % V == 0) f(std::integral_constant<int, V>{});
    else if (aligned && per % (V / 2) == 0 && cols % V == 0) f(std::integral_constant<int, V / 2>{});
    else f(std::integral_constant<int, 1>{});
}

// Blocks as wide as the row (or an even share of it), up to 256 threads and 32
// row lanes, and chunks of 8 rows a lane where that leaves four blocks an SM.
GroupArgs cut(GroupArgs a, int V) {
    a.nv = a.cols / V;
    const int blocks = static_cast<int>(ceil_div(a.nv, kMaxThreads));
    a.tx = static_cast<int>(ceil_div(a.nv, blocks));
    a.ty = std::min(std::max(1, kMaxThreads / a.tx), 32);
    const int64_t share = ceil_div(a.rows * blocks, int64_t(num_sms()) * 4 * a.ty);
    a.R = a.ty * static_cast<int>(std::min<int64_t>(std::max<int64_t>(share, 1), 8));
    a.chunks = static_cast<int>(ceil_div(a.rows, a.R));
    return a;
}
dim3 block_of(const GroupArgs& a) { return dim3(static_cast<unsigned>((a.tx * a.ty + 31) / 32 * 32)); }
dim3 grid_of(const GroupArgs& a) {
    const int64_t y = ceil_div(a.nv, a.tx);
    return dim3(static_cast<unsigned>(std::min<int64_t>(a.chunks, std::max<int64_t>(1, int64_t(num_sms()) * 8 / y))),
                static_cast<unsigned>(y));
}
size_t slots_of(const GroupArgs& a) { return (static_cast<size_t>(a.chunks) + a.graphs) * a.nv; }
// Whether a graph's group has so many parts (were the graphs alike) that a
// block joins them, not a warp.
bool many_parts(const GroupArgs& a) {
    return a.graphs > 0 && (a.rows / a.R / a.graphs + 1) * (a.nv / a.groups) > 256;
}

void check_group(const char* fn, int64_t rows, int64_t cols, int64_t groups, int64_t graphs, const int32_t* offsets, int dtype,
                 int param_dtype, int act) {
    check_dtype(fn, "x", dtype);
    if (param_dtype != TG_F32 && param_dtype != dtype)
        invalid(std::string(fn) + ": gamma and beta must be fp32 or of the rows' type");
    check_rows_cols(fn, rows, cols);
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
        const GroupArgs g{rows, static_cast<int>(cols), static_cast<int>(groups), static_cast<int>(graphs), offsets, act, alpha, eps};
        by_types(dtype, param_dtype, [&](auto t, auto pt) {
            using T = decltype(t);
            using P = decltype(pt);
            const T* xp = static_cast<const T*>(x);
            const P *ga = static_cast<const P*>(gamma), *be = static_cast<const P*>(beta);
            const bool aligned = rows_aligned16(x, ldx, sizeof(T)) && rows_aligned16(y, ldy, sizeof(T)) &&
                                 rows_aligned16(gamma, 0, 1) && rows_aligned16(beta, 0, 1);
            by_vector<T, P>(cols, groups, aligned, [&](auto vec) {
                constexpr int V = decltype(vec)::value;
                const GroupArgs a = cut(g, V);
                Scratch<float2> part(slots_of(a), s);
                launch_dependent("group_norm_parts", group_parts_kernel<T, V>, grid_of(a), block_of(a), 0, s, a, xp, ldx, part.p);
                const int64_t sets = graphs * groups;
                float2* st = reinterpret_cast<float2*>(stats);
                if (many_parts(a))
                    launch_dependent("group_norm_stats", group_stats_kernel<V, kMaxThreads>, dim3(static_cast<unsigned>(sets)),
                                     dim3(kMaxThreads), 0, s, a, part.p, st);
                else
                    launch_dependent("group_norm_stats", group_stats_kernel<V, 32>, dim3(static_cast<unsigned>(ceil_div(sets, 8))),
                                     dim3(kMaxThreads), 0, s, a, part.p, st);
                launch_dependent("group_norm", group_apply_kernel<T, P, V>, grid_of(a), block_of(a), 0, s, a, xp, ldx, ga, be,
                                 st, static_cast<T*>(y), ldy);
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
        const GroupArgs g{rows, static_cast<int>(cols), static_cast<int>(groups), static_cast<int>(graphs), offsets, act, alpha, 0.0f};
        by_types(dtype, param_dtype, [&](auto t, auto pt) {
            using T = decltype(t);
            using P = decltype(pt);
            const T *xp = static_cast<const T*>(x), *dyp = static_cast<const T*>(dy);
            const P *ga = static_cast<const P*>(gamma), *be = static_cast<const P*>(beta);
            const bool aligned = rows_aligned16(x, ldx, sizeof(T)) && rows_aligned16(dy, lddy, sizeof(T)) &&
                                 rows_aligned16(dx, lddx, sizeof(T)) && rows_aligned16(gamma, 0, 1) && rows_aligned16(beta, 0, 1);
            by_vector<T, P>(cols, groups, aligned, [&](auto vec) {
                constexpr int V = decltype(vec)::value;
                const GroupArgs a = cut(g, V);
                const dim3 grid = grid_of(a);
                const int sum_rows = static_cast<int>(grid.x);
                const size_t sets = static_cast<size_t>(graphs) * groups;
                Scratch<float2> part(slots_of(a) + sets, s);
                Scratch<float> sums(static_cast<size_t>(sum_rows) * 2 * cols, s);
                float2* coef = part.p + slots_of(a);
                const float2* st = reinterpret_cast<const float2*>(stats);
                launch_dependent("group_norm_grad_parts", group_grad_parts_kernel<T, P, V>, grid, block_of(a), 0, s, a, dyp, lddy,
                                 xp, ldx, ga, be, st, part.p, sums.p);
                const int col_blocks = static_cast<int>(ceil_div(2 * cols, 32));
                const auto join = [&](auto width) {
                    constexpr int W = decltype(width)::value;
                    const int blocks = static_cast<int>(ceil_div(sets, kMaxThreads / W));
                    launch_dependent("group_norm_grad_join", group_grad_join_kernel<P, V, W>,
                                     dim3(static_cast<unsigned>(blocks + col_blocks)), dim3(kMaxThreads), 0, s, a, part.p, sums.p,
                                     sum_rows, blocks, coef, static_cast<P*>(dgamma), static_cast<P*>(dbeta));
                };
                if (many_parts(a)) join(std::integral_constant<int, kMaxThreads>{});
                else join(std::integral_constant<int, 32>{});
                launch_dependent("group_norm_grad", group_grad_apply_kernel<T, P, V>, grid, block_of(a), 0, s, a, dyp, lddy, xp, ldx,
                                 ga, be, st, coef, static_cast<T*>(dx), lddx);
            });
        });
    });
}

}  // extern "C"

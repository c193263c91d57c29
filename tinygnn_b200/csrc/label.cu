// ============================================================================
//  label.cu -- log probabilities of each row's label, with the row's entropy
//  and its best classes, and the gradient of the first two.
//
//      log p_j = d_j - log s,  d_j = z_j - max z,  s = sum e^d_j
//      H = log s - (sum d_j e^d_j) / s
//      dz_j = a ([j = label] - p_j) - b p_j (log p_j + H),
//      a, b the gradients of log p_label and of H
//
//  The forward pass reads the scores once.  The best classes of wide rows come
//  from that pass too: the k-th greatest of the threads' maxima is not above the
//  k-th greatest score, so only the threads whose maximum reaches it can hold
//  one of the k, and only their scores (about k / threads of the row, from L2)
//  are read again.  The scores above that bound are ranked by (score descending,
//  class ascending) against each other; those equal to it fill up what is left
//  in the order of their classes, so that results do not depend on the order of
//  atomics.  Rows of at most 1,024 classes find the k-th rank itself.
//
//  8,192 x 131,072 bf16: 369 us forward (HBM's 336 at 6,399 GB/s; 5.8 TB/s), 645
//  the gradient (671: its read and write run above the copy's rate).  Forward and
//  gradient share nothing on chip: the gradients of the losses are known only
//  after the first.  The rows of 41 classes are bound by issue slots: 22 us of 6
//  without best classes, 48 with five.
// ============================================================================
#include <algorithm>

#include <cooperative_groups.h>

#include "logits.cuh"

namespace tg {

namespace {

using namespace logits;
namespace cg = cooperative_groups;

struct LabelArgs {
    int64_t rows;
    int n;             // classes
    const void* labels;
    bool wide_labels;  // of 8 bytes
    int top;
    float *log_probs, *entropy;
    float2* stats;     // (max, log s)
    float* top_log_probs;
    int32_t* top_classes;
};

struct RowResult {
    float m, log_s, entropy;
};
template <bool FAST>
__device__ __forceinline__ RowResult finish_row(const Soft& a) {
    if (a.m == -INFINITY) return {a.m, 0.0f, 0.0f};  // no class is left
    const float log_s = logf(a.s);
    return {a.m, log_s, __fsub_rn(log_s, __fmul_rn(kUnit<FAST>, __fdiv_rn(a.t, a.s)))};
}
__device__ __forceinline__ float log_prob(float z, const RowResult& r) {
    return __fsub_rn(__fsub_rn(z, r.m), r.log_s);  // (NaN where no class is left)
}
// What a row's first thread writes.  z: the score of its label.
__device__ __forceinline__ void write_row(const LabelArgs& a, int64_t row, bool labelled, float z, const RowResult& r) {
    a.log_probs[row] = labelled ? log_prob(z, r) : 0.0f;
    a.entropy[row] = r.entropy;
    a.stats[row] = make_float2(r.m, r.log_s);
}

// A score and its class as one number: greater for a greater score, and among
// equal scores for a lower class.  0: none.
__device__ __forceinline__ uint64_t entry(uint32_t rank, int column) {
    return static_cast<uint64_t>(rank) << 32 | (0xffffffffu - static_cast<uint32_t>(column));
}
__device__ __forceinline__ uint32_t entry_rank(uint64_t e) { return static_cast<uint32_t>(e >> 32); }
__device__ __forceinline__ int entry_column(uint64_t e) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(e)); }

// How many of the first n entries are greater than e.
__device__ __forceinline__ int place_of(const uint64_t* entries, int n, uint64_t e) {
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) place += entries[j] > e;
    return place;
}

// The lowest bits that the ranks of a type's scores share: zeros, ones for
// negative scores.
template <class T>
constexpr int kLow = sizeof(T) == 4 ? 0 : (std::is_same<T, __half>::value ? 13 : 16);
template <class T>
__device__ __forceinline__ uint32_t with_low_bits(uint32_t bound) {
    return bound >> 31 == 0 ? bound | ((1u << kLow<T>) - 1) : bound;
}

// ── narrow rows ──────────────────────────────────────────────────────────
template <int LPR>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    if constexpr (LPR == 32) {
        return __reduce_max_sync(0xffffffffu, x);
    } else {
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
        return x;
    }
}
template <int LPR>
__device__ __forceinline__ int lanes_min(int x) {
    if constexpr (LPR == 32) {
        return __reduce_min_sync(0xffffffffu, x);
    } else {
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) x = min(x, __shfl_xor_sync(0xffffffffu, x, o));
        return x;
    }
}

// The row's k best of a warp's E ranks a lane (0: none), class lane + 32 i, into
// list: the k-th greatest rank bit by bit, the ranks above it, and of those
// equal to it the first.
template <class T, int E>
__device__ __forceinline__ void warp_top(const uint32_t (&rank)[E], int k, uint64_t* list) {
    const int lane = threadIdx.x & 31;
    uint32_t bound = 0;
    for (int bit = 31; bit >= kLow<T>; --bit) {
        const uint32_t next = bound | 1u << bit;
        int reached = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) reached += rank[i] >= next;
        reached = __reduce_add_sync(0xffffffffu, reached);
        if (reached >= k) bound = next;
        if (reached == k) break;
    }
    bound = with_low_bits<T>(bound);
    int taken = 0;
    const auto take = [&](int i, bool x) {
        const uint32_t m = __ballot_sync(0xffffffffu, x);
        const int at = taken + __popc(m & ((1u << lane) - 1));
        if (x && at < k) list[at] = entry(rank[i], lane + i * 32);
        taken += __popc(m);
    };
#pragma unroll
    for (int i = 0; i < E; ++i) take(i, rank[i] > bound);
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (taken < k) take(i, rank[i] == bound);
    __syncwarp();
}

// How a row's best classes are found: one after the other, which takes longer
// for each, or by the rank of the last (warp_top), which gives a row 32 lanes
// whatever its classes.  us for 8, 12 and 20 classes, rounds / select: 200,000 x 41
// fp32 53, 69, 100 / 126, 129, 129; x 80 bf16 121, 163, 250 / 154, 159, 168;
// 80,000 x 168 fp16 85, 113, 168 / 90, 93, 98.
enum Top { kNone, kRounds, kSelect };

template <class T, int LPR, int E, Top TOP>
__global__ void __launch_bounds__(kNarrowThreads) label_narrow_kernel(const LabelArgs a, const T* x, int64_t ldx, int turns) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr float C = FAST ? kLog2e : 1.0f;
    constexpr int RPB = kNarrowThreads / LPR;
    extern __shared__ __align__(16) uint8_t sh[];
    __shared__ int labels[kNarrowThreads];
    __shared__ uint64_t lists[TOP == kSelect ? RPB : 1][TOP == kSelect ? kMaxTop : 1];
    wait_for_previous();
    const int lane = threadIdx.x % LPR, per = RPB * turns;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * per; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * per) {
        const int rows = a.rows - r0 < per ? static_cast<int>(a.rows - r0) : per;
        if (threadIdx.x < rows) labels[threadIdx.x] = class_at(a.labels, r0 + threadIdx.x, a.wide_labels);
        const T* st = stage_in(sh, x, ldx, r0, rows, a.n);
        __syncthreads();
        for (int sub = threadIdx.x / LPR; sub - static_cast<int>(threadIdx.x) / LPR < rows; sub += RPB) {
            float z[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int j = lane + i * LPR;
                z[i] = sub < rows && j < a.n ? to_f32(st[sub * a.n + j]) : -INFINITY;
            }
            Soft s;
            add_scores<FAST, true>(s, z, C);
            lanes_soft<FAST, true, LPR>(s, C);
            const RowResult r = finish_row<FAST>(s);
            const int64_t row = r0 + sub;
            if (lane == 0 && sub < rows) {
                const int label = labels[sub];
                const bool labelled = label >= 0 && label < a.n;
                write_row(a, row, labelled, labelled ? to_f32(st[sub * a.n + label]) : 0.0f, r);
            }
            if constexpr (TOP != kNone) {
                uint32_t rank[E];
#pragma unroll
                for (int i = 0; i < E; ++i) rank[i] = lane + i * LPR < a.n ? rank_of(z[i]) : 0u;
                if constexpr (TOP == kSelect) {
                    uint64_t* list = lists[threadIdx.x / LPR];
                    warp_top<T>(rank, a.top, list);
                    for (int i = lane; i < a.top && sub < rows; i += 32) {
                        const uint64_t e = list[i];
                        const int64_t o = row * a.top + place_of(list, a.top, e);
                        a.top_log_probs[o] = log_prob(score_of(entry_rank(e)), r);
                        a.top_classes[o] = entry_column(e);
                    }
                    __syncwarp();
                    continue;
                }
                uint32_t kept = 0;
                int kept_class = 0;
                for (int k = 0; k < a.top; ++k) {
                    // the row's greatest, then the first of its classes
                    uint32_t best = rank[0];
#pragma unroll
                    for (int i = 1; i < E; ++i) best = max(best, rank[i]);
                    best = lanes_max<LPR>(best);
                    int j = INT_MAX;
#pragma unroll
                    for (int i = E - 1; i >= 0; --i) j = rank[i] == best ? lane + i * LPR : j;
                    j = lanes_min<LPR>(j);
#pragma unroll
                    for (int i = 0; i < E; ++i) rank[i] = lane + i * LPR == j ? 0u : rank[i];
                    if (lane == k % LPR) kept = best, kept_class = j;
                    if (k % LPR == LPR - 1 || k == a.top - 1) {
                        const int64_t o = row * a.top + k - k % LPR + lane;
                        if (lane <= k % LPR && sub < rows) {
                            a.top_log_probs[o] = log_prob(score_of(kept), r);
                            a.top_classes[o] = kept_class;
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
}

// ── wide rows ────────────────────────────────────────────────────────────
// Scores above the bound, and equal to it, that a team ranks at a time.
template <int NT>
constexpr int kCandidates = NT == 32 ? 256 : 512;
template <int NT>
constexpr int kEquals = NT == 32 ? 64 : 256;

template <int NT>
struct TopShared {
    uint64_t best[kMaxTop];  // this CTA's best, in order
    uint64_t above[NT == 32 ? kCandidates<NT> : 8 * kMaxTop];  // candidates; then the best of all CTAs of the row
    int equal[kEquals<NT>];
    int n_above, n_equal, n_threads;
    int threads[NT == 32 ? 1 : NT];
    int sums[NT / 32];
    uint32_t bound;
};

// The `k` best scores of the part into sh.best, 0 where it has fewer.  `most`:
// the rank of this thread's greatest score among its vectors (0 without one).
template <class T, int NT>
__device__ __forceinline__ void part_top(TopShared<NT>& sh, const Part<T>& p, uint32_t most, int k) {
    constexpr int V = kVec<T>;
    using Team = logits::Team<NT>;
    const int tid = Team::thread(), warp = tid >> 5, lane = tid & 31;
    if (tid < k) sh.best[tid] = 0;
    // The greatest bound that k maxima reach, bit by bit (any that not many more
    // reach will do).
    uint32_t bound = 0;
    if (Team::count(most != 0) >= k) {
        for (int bit = 31; bit >= kLow<T>; --bit) {
            const uint32_t next = bound | 1u << bit;
            const int reached = Team::count(most >= next);
            if (reached >= k) bound = next;
            if (reached >= k && reached <= k + NT / 16) break;
        }
        bound = with_low_bits<T>(bound);
    }
    int above;
    for (;;) {
        if (tid == 0) sh.n_above = sh.n_equal = sh.n_threads = 0;
        if (NT == 32) __syncwarp();  // (a block's count is a barrier, a warp's ballot orders no memory)
        // Where many threads reach the bound its score is a common one: then
        // only those above it are looked at, and the equal ones found below.
        const bool common = Team::count(most != 0 && most >= bound) > (NT == 32 ? NT : 2 * k + 32);
        const bool mine = most != 0 && (common ? most > bound : most >= bound);
        if (NT > 32 && mine) sh.threads[atomicAdd(&sh.n_threads, 1)] = tid;
        if (common && tid == 0) sh.n_equal = kEquals<NT> + 1;
        const volatile int *above_now = &sh.n_above, *equal_now = &sh.n_equal;
        const auto look = [&](float z, int column) {
            const uint32_t r = rank_of(z);
            // (once there are too many, no more are counted: a row of equal
            // scores would queue up at the counter)
            if (r > bound) {
                if (*above_now <= kCandidates<NT>) {
                    const int i = atomicAdd(&sh.n_above, 1);
                    if (i < kCandidates<NT>) sh.above[i] = entry(r, column);
                }
            } else if (r == bound) {
                if (*equal_now <= kEquals<NT>) {
                    const int i = atomicAdd(&sh.n_equal, 1);
                    if (i < kEquals<NT>) sh.equal[i] = column;
                }
            }
        };
        if (tid < p.extra) look(to_f32(p.row[p.extra_column(tid)]), p.extra_column(tid));
        Team::sync();
        const auto look_at = [&](int v) {
            float z[V];
            widen(p.load(v), z);
#pragma unroll
            for (int j = 0; j < V; ++j) look(z[j], p.column(v) + j);
        };
        if (NT == 32) {
            if (mine)
                for (int v = p.v0 + tid; v < p.v1; v += 32) look_at(v);
        } else {
            // Those threads' vectors, dealt out to all.
            const int each = (p.v1 - p.v0 + NT - 1) / NT;
            const int64_t items = static_cast<int64_t>(sh.n_threads) * each;
            for (int64_t i = tid; i < items; i += NT) {
                const int t = static_cast<int>(i / each), v = p.v0 + sh.threads[t] + static_cast<int>(i - int64_t(t) * each) * NT;
                if (v < p.v1) look_at(v);
            }
        }
        Team::sync();
        above = sh.n_above;
        const int held = above < kCandidates<NT> ? above : kCandidates<NT>;
        // The rank of each among them is its place.
        for (int i = tid; i < held; i += NT) {
            const uint64_t e = sh.above[i];
            const int place = place_of(sh.above, held, e);
            if (place < k) sh.best[place] = e;
            if (place == k - 1) sh.bound = entry_rank(e);
        }
        Team::sync();
        if (above <= kCandidates<NT>) break;
        // Too many, as where a row's greatest scores lie with few threads: k of
        // those that were kept reach a greater bound.
        bound = sh.bound;
        Team::sync();
    }
    const int missing = k - above;
    if (missing <= 0 || bound == 0) return;
    const int equal = sh.n_equal;
    if (equal <= kEquals<NT>) {
        for (int i = tid; i < equal; i += NT) {
            const int column = sh.equal[i];
            int place = 0;
            for (int j = 0; j < equal; ++j) place += sh.equal[j] < column;
            if (place < missing) sh.best[above + place] = entry(bound, column);
        }
    } else {
        // Many equal scores: the first of them in the order of the columns.
        int found = 0;
        const auto step = [&](int count, auto&& put) {  // count: this thread's; put(i): its i-th
            int before = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += x;
            }
            if (lane == 31) sh.sums[warp] = before;
            Team::sync();
            int total = 0;
            before -= count;
            for (int w = 0; w < NT / 32; ++w) {
                if (w < warp) before += sh.sums[w];
                total += sh.sums[w];
            }
            for (int i = 0; i < count && found + before + i < missing; ++i)
                sh.best[above + found + before + i] = entry(bound, put(i));
            found += total;
            Team::sync();
        };
        const auto is = [&](int column) { return rank_of(to_f32(p.row[column])) == bound; };
        if (p.extra) step(tid < p.head && is(tid), [&](int) { return tid; });
        for (int v = p.v0 + tid; v - tid < p.v1 && found < missing; v += NT) {
            uint32_t mask = 0;
            if (v < p.v1) {
                float z[V];
                widen(p.load(v), z);
#pragma unroll
                for (int j = 0; j < V; ++j) mask |= (rank_of(z[j]) == bound ? 1u : 0u) << j;
            }
            step(__popc(mask), [&](int i) { return p.column(v) + static_cast<int>(__fns(mask, 0, i + 1)); });
        }
        if (p.extra && found < missing)
            step(tid < p.extra - p.head && is(p.tail + tid), [&](int) { return p.tail + tid; });
    }
}

template <int NT, bool TOP>
struct LabelShared {
    SoftShared soft;
    SoftCell mine[2];  // this CTA's state, of even and odd rounds
    TopShared<NT> top;
};
template <int NT>
struct LabelShared<NT, false> {
    SoftShared soft;
    SoftCell mine[2];
};

constexpr int kAhead = 4;  // slots of the ring: 32 KB of a block of 256 threads

template <class T, int NT, int TEAMS, bool TOP>
__global__ void __launch_bounds__(NT * TEAMS, 1024 / (NT * TEAMS)) label_wide_kernel(const LabelArgs a, const T* x, int64_t ldx) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr float C = FAST ? kLog2e : 1.0f;
    using Team = logits::Team<NT>;
    __shared__ LabelShared<NT, TOP> shared[TEAMS];
    extern __shared__ __align__(16) uint8_t room[];
    wait_for_previous();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks()), log_ranks = __ffs(ranks) - 1;
    const int team = TEAMS > 1 ? threadIdx.x / NT : 0, tid = Team::thread();
    const int64_t step = static_cast<int64_t>(gridDim.x / ranks) * TEAMS, first = static_cast<int64_t>(blockIdx.x / ranks) * TEAMS + team;
    LabelShared<NT, TOP>& sh = shared[team];
    Stream<T, NT> in(x, ldx, a.rows, a.n, first, step, rank, log_ranks, room + team * kAhead * Stream<T, NT>::kSlot, kAhead, false);
    // (a row's label is asked for a row ahead, its score at the row's start)
    int label = first < a.rows ? class_at(a.labels, first, a.wide_labels) : -1;
    int round = 0;
    for (int64_t row = first; row < a.rows; row += step, ++round) {
        const Part<T> p(x + row * ldx, a.n, rank, log_ranks);
        const bool labelled = label >= 0 && label < a.n;
        T at_label{}, beside{};
        if (rank == 0) {
            if (labelled && tid == 0) at_label = p.row[label];
            if (tid < p.extra) beside = p.row[p.extra_column(tid)];
            label = row + step < a.rows ? class_at(a.labels, row + step, a.wide_labels) : -1;
        }
        Soft s;
        const int steps = in.steps_of(p);
        for (int i = 0, have = p.v1 - p.v0; i < steps; ++i, have -= NT * in.W) {
            in.template wait<kAhead - 1>();
            in.template add<true>(s, in.from, have, C);
            in.from = in.next(in.from);
            in.ask();
        }
        const float most = s.m;
        if (tid < p.extra) {
            const float z[1] = {to_f32(beside)};
            add_scores<FAST, true>(s, z, C);
        }
        team_soft<FAST, true, NT>(s, C, sh.soft);
        if (ranks > 1 && tid == 0) sh.mine[round & 1].set(s);
        if constexpr (TOP) part_top<T, NT>(sh.top, p, p.v0 + tid < p.v1 ? rank_of(most) : 0u, a.top);
        if (ranks > 1) {
            cluster.sync();
            if (rank == 0) {
                s = Soft{};
                if (threadIdx.x % 32 < ranks) s = cluster.map_shared_rank(&sh.mine[round & 1], threadIdx.x % 32)->get();
                lanes_soft<FAST, true, 32>(s, C);
            }
        }
        if (rank == 0) {
            const RowResult r = finish_row<FAST>(s);
            if (tid == 0) write_row(a, row, labelled, to_f32(at_label), r);
            if constexpr (TOP) {
                Team::sync();
                const auto put = [&](int i, uint64_t e) {
                    a.top_log_probs[row * a.top + i] = log_prob(score_of(entry_rank(e)), r);
                    a.top_classes[row * a.top + i] = entry_column(e);
                };
                if (ranks == 1) {
                    for (int i = tid; i < a.top; i += NT) put(i, sh.top.best[i]);
                } else {
                    // (the candidates' room is free by now)
                    const int all = ranks * a.top;
                    for (int i = tid; i < all; i += NT) sh.top.above[i] = cluster.map_shared_rank(sh.top.best, i / a.top)[i % a.top];
                    Team::sync();
                    for (int i = tid; i < all; i += NT) {
                        const uint64_t e = sh.top.above[i];
                        const int place = place_of(sh.top.above, all, e);
                        if (place < a.top && e) put(place, e);
                    }
                }
            }
        }
        if (TOP && ranks > 1) cluster.sync();  // the CTAs' best have been read
        Team::sync();
    }
    if (ranks > 1) cluster.sync();  // no CTA leaves while its state may be read
}

// ── gradient ─────────────────────────────────────────────────────────────
struct GradArgs {
    int64_t rows;
    int n;
    const void* labels;
    bool wide_labels;
    const float2* stats;
    const float *dlog, *dentropy, *entropy;  // dentropy nullable, then entropy is not read
};
// dz_j = a [j = label] - p_j (c0 + c1 d_j), d_j = log p_j in units.
struct RowGrad {
    float m, log_s, a, c0, c1;
    int label;
};
template <bool FAST>
__device__ __forceinline__ RowGrad row_grad(const GradArgs& g, int64_t row) {
    const float2 s = g.stats[row];
    RowGrad r{s.x, __fmul_rn(s.y, FAST ? kLog2e : 1.0f), 0.0f, 0.0f, 0.0f, class_at(g.labels, row, g.wide_labels)};
    if (r.label >= g.n) r.label = -1;
    if (s.x == -INFINITY) {  // no class is left, no gradient
        r.m = 0.0f;
        r.label = -1;
        return r;
    }
    r.a = r.label >= 0 ? g.dlog[row] : 0.0f;
    r.c0 = r.a;
    if (g.dentropy) {
        const float b = g.dentropy[row];
        r.c0 = fmaf(b, g.entropy[row], r.a);
        r.c1 = __fmul_rn(b, kUnit<FAST>);
    }
    return r;
}
template <bool FAST>
__device__ __forceinline__ float grad_of(float z, const RowGrad& r) {
    const float d = max_nan(__fsub_rn(__fmul_rn(__fsub_rn(z, r.m), FAST ? kLog2e : 1.0f), r.log_s), -200.0f);
    return __fmul_rn(-expo<FAST>(d), fmaf(r.c1, d, r.c0));
}

template <class T, int LPR, int E>
__global__ void __launch_bounds__(kNarrowThreads) label_grad_narrow_kernel(const GradArgs g, const T* x, int64_t ldx, T* dx,
                                                                           int64_t lddx, int turns) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int RPB = kNarrowThreads / LPR;
    extern __shared__ __align__(16) uint8_t sh[];
    __shared__ RowGrad grads[kNarrowThreads];
    wait_for_previous();
    const int lane = threadIdx.x % LPR, per = RPB * turns;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * per; r0 < g.rows; r0 += static_cast<int64_t>(gridDim.x) * per) {
        const int rows = g.rows - r0 < per ? static_cast<int>(g.rows - r0) : per;
        if (threadIdx.x < rows) grads[threadIdx.x] = row_grad<FAST>(g, r0 + threadIdx.x);
        T* st = stage_in(sh, x, ldx, r0, rows, g.n);
        __syncthreads();
        for (int sub = threadIdx.x / LPR; sub < rows; sub += RPB) {
            const RowGrad r = grads[sub];
            T* p = st + sub * g.n;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int j = lane + i * LPR;
                if (j < g.n) {
                    float y = grad_of<FAST>(to_f32(p[j]), r);
                    if (j == r.label) y = __fadd_rn(y, r.a);
                    p[j] = from_f32<T>(y);
                }
            }
        }
        __syncthreads();
        stage_out(st, dx, lddx, r0, rows, g.n);
        __syncthreads();
    }
}

// A warp has U vectors a lane of one row.
template <class T, int U>
__global__ void __launch_bounds__(256) label_grad_wide_kernel(const GradArgs g, const T* x, int64_t ldx, T* dx, int64_t lddx,
                                                              int64_t items, int parts) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int V = kVec<T>;
    wait_for_previous();
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), row = item / parts;
    if (item >= items) return;
    const int lane = threadIdx.x & 31;
    const Part<T> p = Part<T>::of_size(x + row * ldx, g.n, static_cast<int>(item - row * parts), 32 * U);
    Raw<T, V> raw[U];
    T beside{};
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (p.v0 + lane + u * 32 < p.v1) raw[u] = p.load(p.v0 + lane + u * 32);
    if (lane < p.extra) beside = p.row[p.extra_column(lane)];
    T* out = dx + row * lddx;
    const RowGrad r = row_grad<FAST>(g, row);
    const bool aligned = (reinterpret_cast<uintptr_t>(out + p.head) & 15) == 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = p.v0 + lane + u * 32, first = p.column(v);
        if (v >= p.v1) break;
        float z[V];
        widen(raw[u], z);
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = grad_of<FAST>(z[j], r);
        if (static_cast<unsigned>(r.label - first) < V) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (first + j == r.label) z[j] = __fadd_rn(z[j], r.a);
        }
        if (aligned) store_v<T, V>(out + first, z);
        else store_any<T, V>(out + first, z);
    }
    if (lane < p.extra) {
        const int j = p.extra_column(lane);
        float y = grad_of<FAST>(to_f32(beside), r);
        if (j == r.label) y = __fadd_rn(y, r.a);
        out[j] = from_f32<T>(y);
    }
}

size_t staged_bytes(int rows, int64_t n, size_t size) { return static_cast<size_t>(rows * n) * size + 32; }

}  // namespace

}  // namespace tg

extern "C" {

TG_API tg_status tg_label_log_probs(int64_t rows, int64_t classes, int32_t dtype, const void* logits, int64_t ldz,
                                    const void* labels, int32_t label_bytes, int64_t top, float* log_probs,
                                    float* entropy, float* stats, float* top_log_probs, int32_t* top_classes,
                                    void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "label_log_probs";
        logits::check_row_args(fn, rows, classes, dtype, logits, ldz);
        logits::check_int_bytes(fn, "labels", label_bytes);
        check_ptr(fn, "labels", labels, rows > 0);
        check_ptr(fn, "log_probs", log_probs, rows > 0);
        check_ptr(fn, "entropy", entropy, rows > 0);
        check_ptr(fn, "stats", stats, rows > 0);
        if (top < 0 || top > logits::kMaxTop || top > classes)
            invalid(std::string(fn) + ": top = " + std::to_string(top) + " is outside [0, min(" +
                    std::to_string(logits::kMaxTop) + ", classes)]");
        check_ptr(fn, "top_log_probs", top_log_probs, rows > 0 && top > 0);
        check_ptr(fn, "top_classes", top_classes, rows > 0 && top > 0);
        if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) invalid(std::string(fn) + ": stats must be 8-byte aligned");
        const LabelArgs a{rows, static_cast<int>(classes), labels, label_bytes == 8, static_cast<int>(top), log_probs,
                          entropy, reinterpret_cast<float2*>(stats), top_log_probs, top_classes};
        cudaStream_t s = as_stream(stream);
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const T* x = static_cast<const T*>(logits);
            const auto narrow = [&](auto lpr, auto e, auto top_by) {
                constexpr int LPR = decltype(lpr)::value, E = decltype(e)::value, RPB = logits::kNarrowThreads / LPR;
                const int turns = logits::narrow_turns(RPB, classes, sizeof(T), rows);
                launch_dependent("label_log_probs", label_narrow_kernel<T, LPR, E, decltype(top_by)::value>,
                                 dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(rows, RPB * turns), num_sms() * 8))),
                                 dim3(logits::kNarrowThreads), staged_bytes(RPB * turns, classes, sizeof(T)), s, a, x, ldz, turns);
            };
            using std::integral_constant;
            const int rounds = classes <= 48 ? 24 : (classes <= 128 ? 12 : (classes <= logits::kNarrow ? 8 : 0));
            if (top > rounds && classes <= 1024) {
                const integral_constant<Top, kSelect> select;
                const integral_constant<int, 32> lanes;
                if (classes <= 64) narrow(lanes, integral_constant<int, 2>{}, select);
                else if (classes <= 128) narrow(lanes, integral_constant<int, 4>{}, select);
                else if (classes <= 256) narrow(lanes, integral_constant<int, 8>{}, select);
                else if (classes <= 512) narrow(lanes, integral_constant<int, 16>{}, select);
                else narrow(lanes, integral_constant<int, 32>{}, select);
                return;
            }
            if (classes <= logits::kNarrow) {
                logits::by_narrow(classes, [&](auto lpr, auto e) {
                    if (top) narrow(lpr, e, integral_constant<Top, kRounds>{});
                    else narrow(lpr, e, integral_constant<Top, kNone>{});
                });
                return;
            }
            const int ranks = logits::row_ranks(rows, classes, 4096);
            const auto go = [&](auto nt, auto teams) {
                constexpr int NT = decltype(nt)::value, TEAMS = decltype(teams)::value;
                auto kern = top ? label_wide_kernel<T, NT, TEAMS, true> : label_wide_kernel<T, NT, TEAMS, false>;
                const int room = TEAMS * kAhead * logits::Stream<T, NT>::kSlot;
                const int fixed = TEAMS * static_cast<int>(top ? sizeof(LabelShared<NT, true>) : sizeof(LabelShared<NT, false>));
                logits::launch_rows("label_log_probs", kern, ceil_div(rows, TEAMS), NT == 32 ? 1 : ranks,
                                    std::min(1024 / (NT * TEAMS), logits::kSharedSm / (room + fixed + 1024)), NT * TEAMS, room, s, a,
                                    x, ldz);
            };
            // A warp a row where there are rows for all warps, or a block: us by warp
            // / block, bf16: 16,000 x 1,500 16 / 38, x 4,096 30 / 48; 8,000 x 8,000
            // 32 / 36, 4,000 x 16,000 30 / 37.  With best classes: of 5, 16,000 x
            // 4,096 87 / 91, 8,000 x 8,000 82 / 62; of 32, 16,000 x 1,500 359 / 98
            // (its 32 maxima bound few of them well).
            const bool many = rows > 16 * num_sms();
            if (top == 0 ? classes <= (many ? 16384 : logits::kWarp) && rows > num_sms()
                         : classes <= logits::kWarp && rows > num_sms() && top <= 16) go(integral_constant<int, 32>{}, integral_constant<int, 4>{});
            else if (classes / ranks <= 8192) go(integral_constant<int, 128>{}, integral_constant<int, 1>{});
            else go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
        });
    });
}

TG_API tg_status tg_label_log_probs_grad(int64_t rows, int64_t classes, int32_t dtype, const float* dlog_probs,
                                         const float* dentropy, const void* logits, int64_t ldz, const void* labels,
                                         int32_t label_bytes, const float* stats, const float* entropy, void* dlogits,
                                         int64_t lddz, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "label_log_probs_grad";
        logits::check_row_args(fn, rows, classes, dtype, logits, ldz);
        logits::check_int_bytes(fn, "labels", label_bytes);
        check_ptr(fn, "labels", labels, rows > 0);
        check_ptr(fn, "dlog_probs", dlog_probs, rows > 0);
        check_ptr(fn, "stats", stats, rows > 0);
        check_ptr(fn, "entropy", entropy, rows > 0 && dentropy);
        check_ptr(fn, "dlogits", dlogits, rows > 0);
        check_ld(fn, "dlogits", lddz, classes);
        if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) invalid(std::string(fn) + ": stats must be 8-byte aligned");
        const GradArgs g{rows, static_cast<int>(classes), labels, label_bytes == 8,
                         reinterpret_cast<const float2*>(stats), dlog_probs, dentropy, entropy};
        cudaStream_t s = as_stream(stream);
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const T* x = static_cast<const T*>(logits);
            T* dx = static_cast<T*>(dlogits);
            if (classes <= logits::kNarrow) {
                logits::by_narrow(classes, [&](auto lpr, auto e) {
                    constexpr int LPR = decltype(lpr)::value, E = decltype(e)::value, RPB = logits::kNarrowThreads / LPR;
                    const int turns = logits::narrow_turns(RPB, classes, sizeof(T), rows);
                    launch_dependent("label_log_probs_grad", label_grad_narrow_kernel<T, LPR, E>,
                                     dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(rows, RPB * turns), num_sms() * 8))),
                                     dim3(logits::kNarrowThreads), staged_bytes(RPB * turns, classes, sizeof(T)), s, g, x, ldz, dx,
                                     lddz, turns);
                });
                return;
            }
            constexpr int U = 4;
            const int64_t parts = ceil_div(classes, int64_t(32) * U * logits::kVec<T>), items = rows * parts;
            if (ceil_div(items, 8) > INT32_MAX) invalid(std::string(fn) + ": more than 2^31 blocks of the gradient");
            launch_dependent("label_log_probs_grad", label_grad_wide_kernel<T, U>,
                             dim3(static_cast<unsigned>(ceil_div(items, 8))), dim3(256), 0, s, g, x, ldz, dx, lddz, items,
                             static_cast<int>(parts));
        });
    });
}

}  // extern "C"

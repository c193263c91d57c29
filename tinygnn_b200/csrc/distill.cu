// ============================================================================
//  distill.cu -- the distillation loss against a teacher's best logits of each
//  row, and its gradient, in one call.
//
//      q = softmax(t / T) over the teacher's k classes c_i of the row
//      p = softmax(z / T) over all classes
//      loss = T^2 sum_i q_i (log q_i - log p_{c_i})
//           = T (T sum_i q_i log q_i - sum_i q_i ((z_{c_i} - max z) - T log s))
//      dz_j = w T (p_j - sum over i with c_i = j of q_i)
//
//  (A factor T < 1 goes into the loss's terms: of scores at the type's lowest value
//  the sum may pass fp32's range where the loss does not.)
//
//  The gradient needs the row's sum before its first value, and the row's
//  scores twice: the second time they come from shared memory, so HBM sees them
//  once (269 MB read of 1,024 x 131,072 bf16; 386 when the second reading went to
//  L2).  The teacher's classes are put right after the row's p: each is computed
//  again from its score, less its q.
//
//  What bounds wide 16-bit rows: two exponentials a score on the SM's 16 a clock
//  (8.2 k of the about 18 k clocks that a row of 131,072 takes two SMs), the
//  sums and barriers between the two passes (1.6 k for each CTA's part), and
//  HBM (11.5 k): 8,192 rows 1,020 us, HBM's floor 671.
// ============================================================================
#include <algorithm>

#include <cooperative_groups.h>

#include "logits.cuh"

namespace tg {

namespace {

using namespace logits;
namespace cg = cooperative_groups;

struct DistillArgs {
    int64_t rows;
    int n, k;
    const void* classes;  // rows x k
    bool wide_classes;    // of 8 bytes
    int64_t ldc;
    const void* teacher;  // rows x k
    int64_t ldt;
    float temperature, inverse;  // inverse: 1 / temperature
    const float* weights;  // nullable
    float* loss;
};

constexpr int kAhead = 4;  // slots of a ring that holds no row

// One row's teacher in shared memory, 16-byte aligned.
struct Teacher {
    int* c;        // the classes, -1 for none
    float* q;      // their probabilities, 0 for none
    float* z;      // the student's scores of the classes
    float* scale;  // the row's weight times the temperature; 0 for a row without entries

    // Room for k entries and the scale, and where they lie in it.
    static __host__ __device__ constexpr int floats(int k) { return (3 * k + 4) / 4 * 4; }
    static __device__ __forceinline__ Teacher in(float* room, int k) {
        return {reinterpret_cast<int*>(room), room + k, room + 2 * k, room + 3 * k};
    }
};

// A lane's entries lane, lane + W, ... of a row as they were read.  They are
// kept as they lie in memory: an instruction on them would wait for them.
template <class T, class U, int N_>
struct Entries {
    static constexpr int W = 32, N = N_;
    uint2 c[N];
    U v[N];
    T z[N];  // the student's scores of the classes
    float weight;

    __device__ __forceinline__ void fetch(const DistillArgs& a, int64_t row, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + i * W;
            c[i] = make_uint2(0xffffffffu, 0xffffffffu);
            if (e >= a.k) continue;
            if (a.wide_classes) c[i] = static_cast<const uint2*>(a.classes)[row * a.ldc + e];
            else c[i].x = static_cast<const uint32_t*>(a.classes)[row * a.ldc + e];
            v[i] = static_cast<const U*>(a.teacher)[row * a.ldt + e];
        }
        weight = a.weights ? a.weights[row] : 1.0f;
    }
    // Entry i's class; one outside the row is none (-1).
    __device__ __forceinline__ int class_of(const DistillArgs& a, int i) const {
        const int j = static_cast<int>(c[i].x);
        return j >= 0 && j < a.n && (!a.wide_classes || c[i].y == 0) ? j : -1;
    }
    __device__ __forceinline__ void fetch_scores(const DistillArgs& a, const T* row) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (class_of(a, i) >= 0) z[i] = row[class_of(a, i)];
    }
};

// From a row's classes and logits in t.c and t.q (-inf for none), W lanes set
// their probabilities and the row's scale; each lane's part of T sum q log q, times
// min(T, 1), is returned.  (A lane reads what it wrote, and t.c of all lanes.)
template <int W>
__device__ __forceinline__ float finish_teacher(const DistillArgs& a, int lane, const Teacher& t, float weight) {
    const float c = a.inverse;
    float most = -INFINITY;
    for (int i = lane; i < a.k; i += W) most = max_nan(most, t.q[i]);
    most = reduce_max<W>(most);
    float s = 0.0f;
    for (int i = lane; i < a.k; i += W) s = __fadd_rn(s, t.c[i] >= 0 ? expf(distance(t.q[i], most, c)) : 0.0f);
    s = reduce_sum<float, W>(s);
    const float log_s = logf(s);
    float entropy = 0.0f;
    bool twice = false;
    for (int i = lane; i < a.k; i += W) {
        float q = 0.0f;
        const int j = t.c[i];
        if (j >= 0) {
            const float l = __fsub_rn(distance(t.q[i], most, c), log_s);
            q = expf(l);
            if (q != 0.0f) entropy = fmaf(q, l, entropy);
        }
        t.q[i] = q;
    }
    __syncwarp();
    // Classes that occur more than once: the first entry takes all their probabilities.
    for (int i = lane; i < a.k; i += W) {
        const int j = t.c[i];
        int same = 0;
        int o = 0;
        for (; o + 4 <= a.k; o += 4) {
            const int4 c4 = *reinterpret_cast<const int4*>(t.c + o);
            same += (c4.x == j) + (c4.y == j) + (c4.z == j) + (c4.w == j);
        }
        for (; o < a.k; ++o) same += t.c[o] == j;
        twice |= j >= 0 && same > 1;
    }
    if (__any_sync(0xffffffffu, twice)) {
        // First the later ones are marked (-2 - class: lanes still read classes), then the first adds theirs up.
        const auto class_in = [&](int e) { return t.c[e] < -1 ? -2 - t.c[e] : t.c[e]; };
        for (int i = lane; i < a.k; i += W) {
            const int j = class_in(i);
            bool later = false;
            for (int o = 0; o < i; ++o) later |= class_in(o) == j;
            if (j >= 0 && later) t.c[i] = -2 - j;
        }
        __syncwarp();
        for (int i = lane; i < a.k; i += W)
            if (t.c[i] >= 0)
                for (int o = i + 1; o < a.k; ++o)
                    if (t.c[o] == -2 - t.c[i]) t.q[i] = __fadd_rn(t.q[i], t.q[o]);
        __syncwarp();
        for (int i = lane; i < a.k; i += W)
            if (t.c[i] < 0) t.c[i] = -1, t.q[i] = 0.0f;
    }
    if (lane == 0) *t.scale = most == -INFINITY ? 0.0f : __fmul_rn(a.temperature, weight);
    __syncwarp();
    return __fmul_rn(__fmul_rn(a.temperature, fminf(a.temperature, 1.0f)), entropy);
}

// Fills `t` from a warp's entries; returned as above.
template <class T, class U, int N>
__device__ __forceinline__ float read_teacher(const DistillArgs& a, const Entries<T, U, N>& in, int lane, const Teacher& t) {
#pragma unroll
    for (int i = 0; i < in.N; ++i) {
        const int e = lane + i * 32, j = in.class_of(a, i);
        if (e >= a.k) continue;
        const float v = j >= 0 ? to_f32(in.v[i]) : -INFINITY;
        t.z[e] = j >= 0 ? to_f32(in.z[i]) : 0.0f;
        t.c[e] = v == -INFINITY ? -1 : j;
        t.q[e] = v;
    }
    return finish_teacher<32>(a, lane, t, in.weight);
}

// What a row's gradient takes from its softmax.  c: the exponential's units in
// 1 / T.
template <bool FAST>
struct RowScale {
    Origin o;
    float c, log_s;  // log of the sum, in the exponential's units
    float shift;     // T log p = (z - max) - shift: T times the sum's log, of the exact origin
    float inner;     // min(T, 1)
    float w;         // w T; 0 for a row without gradient
    // Where fp32 holds them well the origin, the sum and the weight go into one
    // addend: w p = +-2^(z c - K).  (|M| <= 64 and a weight above 2^-64 keep |K|
    // below 256, and its rounding, 2^-17 at most, far below a 16-bit result's 2^-12.)
    float K;
    bool quick;
    uint32_t sign;  // of two 16-bit results

    __device__ __forceinline__ RowScale(const Soft& s, float c_, float temperature, float scale) : o(s.m, c_), c(c_) {
        const float natural = logf(s.s);
        log_s = __fmul_rn(natural, FAST ? kLog2e : 1.0f);
        // (a folded row's sum has the rounding of M)
        inner = fminf(temperature, 1.0f);
        shift = __fmul_rn(temperature, FAST && !o.far ? fmaf(-kLn2, fmaf(o.m, c, -o.M), natural) : natural);
        w = s.m == -INFINITY ? 0.0f : scale;  // (no class is left, no gradient)
        quick = FAST && fabsf(o.M) <= 64.0f && fabsf(w) > 5.421e-20f;
        K = __fsub_rn(__fadd_rn(o.M, log_s), __log2f(fabsf(w)));
        sign = w < 0.0f ? 0x80008000u : 0u;
    }
    // T log p min(T, 1) of a score; NaN in a row without any score above -inf.
    // (Without T the quotient of a finite difference could pass fp32's range.)
    __device__ __forceinline__ float t_log_p(float z) const { return __fmul_rn(inner, __fsub_rn(__fsub_rn(z, o.m), shift)); }
    __device__ __forceinline__ float prob(float z) const {
        const float d = FAST ? o.d(z, c) : __fmul_rn(__fsub_rn(z, o.m), c);
        return expo<FAST>(max_nan(__fsub_rn(d, log_s), -200.0f));
    }
};
// The gradient at a class that the teacher does not name.
template <bool FAST>
__device__ __forceinline__ float grad_of(float z, const RowScale<FAST>& r) {
    return r.w == 0.0f ? 0.0f : __fmul_rn(r.w, r.prob(z));
}
// The gradient at the teacher's entry i.
template <bool FAST>
__device__ __forceinline__ float entry_grad(const Teacher& t, int i, const RowScale<FAST>& r) {
    return __fmul_rn(r.w, __fsub_rn(r.prob(t.z[i]), t.q[i]));
}
// The same for this thread's vectors of a row in the ring, of which slot `at` is
// the first and which has `have` vectors; each slot is asked into again.
// Returns the slot after the last.
template <bool FAST, class T, int NT>
__device__ __forceinline__ int write_grad(Stream<T, NT>& in, int at, int steps, int have, const RowScale<FAST>& r, T* to, bool aligned,
                                          bool wait = false) {
    constexpr int V = kVec<T>, W = Stream<T, NT>::W;
    const Pair c(r.c, r.c), k(-r.K, -r.K);
    for (int i = 0; i < steps; ++i, have -= NT * W) {
        if (wait) in.template wait<kAhead - 1>();
        uint32_t raw[4 * W];
        float z[W * V];
        in.read(at, have, raw);
        in.scores(raw, z);
        if (r.quick) {
#pragma unroll
            for (int j = 0; j < W * V; j += 2) {
                float x, y;
                fma2(Pair(z[j], z[j + 1]), c, k).get(x, y);
                z[j] = expo<FAST>(x), z[j + 1] = expo<FAST>(y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < W * V; ++j) z[j] = grad_of<FAST>(z[j], r);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            float y[V];
            Raw<T, V> out;
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = z[w * V + j];
            narrow(y, out);
            if (sizeof(T) == 2 && r.quick) {
#pragma unroll
                for (int j = 0; j < out.N; ++j) out.w[j] ^= r.sign;
            }
            if (have <= w * NT + Team<NT>::thread()) continue;
            if (aligned) *reinterpret_cast<Raw<T, V>*>(to + w * NT * V) = out;
            else store_words(to + w * NT * V, out);
        }
        to += NT * W * V;
        at = in.next(at);
        in.ask();
    }
    return at;
}

// ── narrow rows ──────────────────────────────────────────────────────────
template <class T, class U, int LPR, int E, bool GRAD>
__global__ void __launch_bounds__(kNarrowThreads) distill_narrow_kernel(const DistillArgs a, const T* x, int64_t ldx, T* dx,
                                                                        int64_t lddx, int turns, int stage) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int RPB = kNarrowThreads / LPR;
    extern __shared__ __align__(16) uint8_t sh[];
    wait_for_previous();
    const int lane = threadIdx.x % LPR, place = threadIdx.x / LPR, per = RPB * turns, room = Teacher::floats(a.k);
    float* teachers = reinterpret_cast<float*>(sh + stage);  // of all rows
    const float c = FAST ? __fmul_rn(kLog2e, a.inverse) : a.inverse;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * per; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * per) {
        const int rows = a.rows - r0 < per ? static_cast<int>(a.rows - r0) : per;
        for (int i = threadIdx.x; i < rows * a.k; i += kNarrowThreads) {
            const int r = i / a.k, e = i - r * a.k;
            const int j = class_at(a.classes, (r0 + r) * a.ldc + e, a.wide_classes);
            const float v = to_f32(static_cast<const U*>(a.teacher)[(r0 + r) * a.ldt + e]);
            const Teacher t = Teacher::in(teachers + r * room, a.k);
            const bool in = j >= 0 && j < a.n && v != -INFINITY;
            t.c[e] = in ? j : -1;
            t.q[e] = in ? v : -INFINITY;
        }
        if (threadIdx.x < rows) *Teacher::in(teachers + threadIdx.x * room, a.k).scale = a.weights ? a.weights[r0 + threadIdx.x] : 1.0f;
        T* st = stage_in(sh, x, ldx, r0, rows, a.n);
        __syncthreads();
        for (int first = 0; first < rows; first += RPB) {
            // (lanes without a row have masked scores and no teacher, and write nothing: any
            // row's scores may be written over by its own lanes)
            const bool here = first + place < rows;
            const int sub = here ? first + place : first;
            const int64_t row = r0 + sub;
            T* p = st + sub * a.n;
            const Teacher t = Teacher::in(teachers + (here ? sub : rows + place) * room, a.k);
            if (!here) {
                for (int i = lane; i < a.k; i += LPR) t.c[i] = -1, t.q[i] = -INFINITY;
                if (lane == 0) *t.scale = 0.0f;
            }
            for (int i = lane; i < a.k; i += LPR) t.z[i] = t.c[i] >= 0 ? to_f32(p[t.c[i]]) : 0.0f;
            float z[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int j = lane + i * LPR;
                z[i] = here && j < a.n ? to_f32(p[j]) : -INFINITY;
            }
            __syncwarp();  // (before the row's first lanes write over its scores)
            float loss = finish_teacher<LPR>(a, lane, t, *t.scale);
            Soft s;
            add_scores<FAST, false>(s, z, c);
            lanes_soft<FAST, false, LPR>(s, c);
            const RowScale<FAST> r(s, c, a.temperature, *t.scale);
            for (int i = lane; i < a.k; i += LPR)
                if (t.q[i] != 0.0f) loss = fmaf(-t.q[i], r.t_log_p(t.z[i]), loss);
            loss = reduce_sum<float, LPR>(loss);
            if (lane == 0 && here) a.loss[row] = __fmul_rn(fmaxf(a.temperature, 1.0f), loss);
            if constexpr (GRAD) {
                if (here) {
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const int j = lane + i * LPR;
                        if (j < a.n) p[j] = from_f32<T>(grad_of<FAST>(z[i], r));
                    }
                }
                __syncwarp();
                if (here && r.w != 0.0f)
                    for (int i = lane; i < a.k; i += LPR)
                        if (t.c[i] >= 0) p[t.c[i]] = from_f32<T>(entry_grad<FAST>(t, i, r));
            }
            __syncwarp();  // (before the next row's entries)
        }
        __syncthreads();
        if constexpr (GRAD) {
            stage_out(st, dx, lddx, r0, rows, a.n);
            __syncthreads();
        }
    }
}

// ── rows of a warp ───────────────────────────────────────────────────────
// As the wide rows' kernel below, with a warp in the place of the block: the ring
// has a row and kAhead slots of the next ones; without a gradient no row is held,
// and it has kAhead slots in all.
constexpr int kTeams = 4;

template <class T, class U, int N, bool GRAD>
__global__ void __launch_bounds__(32 * kTeams, 5) distill_warp_kernel(const DistillArgs a, const T* x, int64_t ldx, T* dx,
                                                                      int64_t lddx, int slots) {
    constexpr bool FAST = sizeof(T) == 2;
    extern __shared__ __align__(16) uint8_t room[];
    wait_for_previous();
    const int lane = threadIdx.x & 31, team = threadIdx.x >> 5;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kTeams, first = static_cast<int64_t>(blockIdx.x) * kTeams + team;
    const float c = FAST ? __fmul_rn(kLog2e, a.inverse) : a.inverse;
    Stream<T, 32> in(x, ldx, a.rows, a.n, first, step, 0, 0, room + team * slots * Stream<T, 32>::kSlot, slots, false);
    const Teacher t = Teacher::in(
        reinterpret_cast<float*>(room + kTeams * slots * Stream<T, 32>::kSlot) + team * Teacher::floats(a.k), a.k);
    // (a row's entries are asked for a row ahead, the scores of their classes at its start)
    Entries<T, U, N> entries;
    if (first < a.rows) entries.fetch(a, first, lane);
    for (int64_t row = first; row < a.rows; row += step) {
        const Part<T> p(x + row * ldx, a.n, 0, 0);
        T beside{};
        if (lane < p.extra) beside = p.row[p.extra_column(lane)];
        entries.fetch_scores(a, p.row);
        Soft s;
        const int steps = in.steps_of(p), mine_first = in.from, count = p.v1 - p.v0;
        if (GRAD) in.template wait<kAhead>();  // the row is there
        for (int i = 0, have = count; i < steps; ++i, have -= 32 * in.W) {
            if (!GRAD) in.template wait<kAhead - 1>();  // its next slot is
            in.template add<false>(s, in.from, have, c);
            in.from = in.next(in.from);
            if (!GRAD) in.ask();
        }
        if (lane < p.extra) {
            const float z[1] = {to_f32(beside)};
            add_scores<FAST, false>(s, z, c);
        }
        lanes_soft<FAST, false, 32>(s, c);
        float loss = read_teacher(a, entries, lane, t);
        if (row + step < a.rows) entries.fetch(a, row + step, lane);
        const RowScale<FAST> r(s, c, a.temperature, *t.scale);
        for (int i = lane; i < a.k; i += 32)
            if (t.q[i] != 0.0f) loss = fmaf(-t.q[i], r.t_log_p(t.z[i]), loss);
        loss = reduce_sum<float, 32>(loss);
        if (lane == 0) a.loss[row] = __fmul_rn(fmaxf(a.temperature, 1.0f), loss);
        if constexpr (GRAD) {
            T* out = dx + row * lddx;
            write_grad<FAST, T, 32>(in, mine_first, steps, count, r, out + p.column(p.v0 + lane),
                                    (reinterpret_cast<uintptr_t>(out + p.head) & 15) == 0);
            if (lane < p.extra) out[p.extra_column(lane)] = from_f32<T>(grad_of<FAST>(to_f32(beside), r));
            __syncwarp();
            if (r.w != 0.0f)
                for (int i = lane; i < a.k; i += 32)
                    if (t.c[i] >= 0) out[t.c[i]] = from_f32<T>(entry_grad<FAST>(t, i, r));
        }
        __syncwarp();  // (before the next row's entries)
    }
}

// ── wide rows ────────────────────────────────────────────────────────────
// NT threads read the row (Stream), and one warp more has the teacher: it sets
// the entries' gradients right once the row's p are written, and reads the next
// row's entries, while the others read the next row.
//
// With `hold` a CTA's part of the row fills the ring and stays there until its p
// are written, slot by slot the next row's after that; the other CTAs of the SM
// keep it busy meanwhile (three of 256 threads: 1,004 us for 8,192 x 131,072 bf16;
// two with four slots for the next row 1,147, one of 512 threads 1,286).  Without
// it (parts that do not fit) the row is read twice.

struct alignas(16) TeacherShared {
    int c[2][kMaxTop];
    float q[2][kMaxTop], z[2][kMaxTop], scale[2];
};

template <class T, class U, int NT, bool GRAD>
__global__ void __launch_bounds__(NT + 32, 768 / NT) distill_wide_kernel(const DistillArgs a, const T* x, int64_t ldx, T* dx, int64_t lddx,
                                                               int slots, bool hold) {
    constexpr bool FAST = sizeof(T) == 2;
    __shared__ SoftShared soft;
    __shared__ SoftCell mine[2];  // this CTA's state, of even and odd rounds
    __shared__ TeacherShared teacher;
    extern __shared__ __align__(16) uint8_t room[];
    wait_for_previous();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks()), log_ranks = __ffs(ranks) - 1;
    const int64_t clusters = gridDim.x / ranks, first = blockIdx.x / ranks;
    const float c = FAST ? __fmul_rn(kLog2e, a.inverse) : a.inverse;
    const auto meet = [] { asm volatile("bar.sync 2, %0;" ::"n"(NT + 32) : "memory"); };
    const auto all = [&] {  // the CTAs' states are there
        if (ranks > 1) cluster.sync();
        else meet();
    };
    const auto joined = [&](int b) {
        Soft s;
        const int lane = threadIdx.x % 32;
        if (ranks == 1) return mine[b].get();
        if (lane < ranks) s = cluster.map_shared_rank(&mine[b], lane)->get();
        lanes_soft<FAST, false, 32>(s, c);
        return s;
    };
    int round = 0;
    if (threadIdx.x < NT) {
        Stream<T, NT> in(x, ldx, a.rows, a.n, first, clusters, rank, log_ranks, room, slots, GRAD && !hold);
        for (int64_t row = first; row < a.rows; row += clusters, ++round) {
            const int b = round & 1;
            const Part<T> p(x + row * ldx, a.n, rank, log_ranks);
            T beside{};
            if (threadIdx.x < p.extra) beside = p.row[p.extra_column(threadIdx.x)];
            Soft s;
            const int steps = in.steps_of(p), mine_first = in.from;
            const int count = p.v1 - p.v0;
            if (GRAD && hold) in.template wait<0>();
            for (int i = 0, have = count; i < steps; ++i, have -= NT * in.W) {
                if (!(GRAD && hold)) in.template wait<kAhead - 1>();
                in.template add<false>(s, in.from, have, c);
                in.from = in.next(in.from);
                if (!(GRAD && hold)) in.ask();
            }
            if (threadIdx.x < p.extra) {
                const float z[1] = {to_f32(beside)};
                add_scores<FAST, false>(s, z, c);
            }
            team_soft<FAST, false, NT>(s, c, soft);
            if (threadIdx.x == 0) mine[b].set(s);
            all();
            if constexpr (GRAD) {
                s = joined(b);
                const RowScale<FAST> r(s, c, a.temperature, teacher.scale[b]);
                T* out = dx + row * lddx;
                const int end = write_grad<FAST, T, NT>(in, hold ? mine_first : in.from, steps, count, r,
                                                        out + p.column(p.v0 + threadIdx.x),
                                                        (reinterpret_cast<uintptr_t>(out + p.head) & 15) == 0, !hold);
                if (!hold) in.from = end;
                if (threadIdx.x < p.extra) out[p.extra_column(threadIdx.x)] = from_f32<T>(grad_of<FAST>(to_f32(beside), r));
            }
            meet();  // the row's p are written
        }
    } else {
        const int lane = threadIdx.x - NT;
        const auto entries = [&](int b) { return Teacher{teacher.c[b], teacher.q[b], teacher.z[b], &teacher.scale[b]}; };
        // A row's entries are asked for two rows ahead, the scores of their classes
        // while the row before is read, and put into shared memory after it.
        Entries<T, U, kMaxTop / 32> next;
        float own = 0.0f;
        if (first < a.rows) {
            next.fetch(a, first, lane);
            next.fetch_scores(a, x + first * ldx);
            own = read_teacher(a, next, lane, entries(0));
        }
        if (first + clusters < a.rows) next.fetch(a, first + clusters, lane);
        for (int64_t row = first; row < a.rows; row += clusters, ++round) {
            const int b = round & 1;
            const Teacher t = entries(b);
            if (row + clusters < a.rows) next.fetch_scores(a, x + (row + clusters) * ldx);
            all();
            const Soft s = joined(b);
            const RowScale<FAST> r(s, c, a.temperature, *t.scale);
            float loss = own;
            if (rank == 0) {
                for (int i = lane; i < a.k; i += 32)
                    if (t.q[i] != 0.0f) loss = fmaf(-t.q[i], r.t_log_p(t.z[i]), loss);
                loss = reduce_sum<float, 32>(loss);
                if (lane == 0) a.loss[row] = __fmul_rn(fmaxf(a.temperature, 1.0f), loss);
            }
            meet();
            if constexpr (GRAD) {
                const Part<T> p(x + row * ldx, a.n, rank, log_ranks);
                for (int e = lane; e < a.k; e += 32)
                    if (t.c[e] >= 0 && r.w != 0.0f && p.has(t.c[e])) dx[row * lddx + t.c[e]] = from_f32<T>(entry_grad<FAST>(t, e, r));
            }
            if (row + clusters < a.rows) own = read_teacher(a, next, lane, entries(b ^ 1));
            if (row + 2 * clusters < a.rows) next.fetch(a, row + 2 * clusters, lane);
        }
    }
    if (ranks > 1) cluster.sync();  // no CTA leaves while its state may be read
}

template <class T, class U>
void distill(const DistillArgs& a, const T* x, int64_t ldx, T* dx, int64_t lddx, cudaStream_t s) {
    if (a.n <= kNarrow) {
        by_narrow(a.n, [&](auto lpr, auto e) {
            constexpr int LPR = decltype(lpr)::value, E = decltype(e)::value, RPB = kNarrowThreads / LPR;
            auto kern = dx ? distill_narrow_kernel<T, U, LPR, E, true> : distill_narrow_kernel<T, U, LPR, E, false>;
            const int turns = narrow_turns(RPB, a.n + Teacher::floats(a.k) * 4 / static_cast<int>(sizeof(T)), sizeof(T), a.rows);
            const int stage = static_cast<int>((RPB * turns * a.n * sizeof(T) + 32 + 15) / 16 * 16);
            // (and a teacher for each of a turn's lanes that may have no row)
            const size_t bytes = stage + (RPB * turns + RPB) * Teacher::floats(a.k) * sizeof(float);
            if (bytes > 48 * 1024) allow_shared(kern, kMaxShared);
            launch_dependent("distill_loss", kern,
                             dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(a.rows, RPB * turns), num_sms() * 8))),
                             dim3(kNarrowThreads), bytes, s, a, x, ldx, dx, lddx, turns, stage);
        });
        return;
    }
    if (a.n <= kWarp && a.rows > num_sms()) {
        using In = Stream<T, 32>;
        const int slots = (dx ? static_cast<int>(ceil_div(a.n / kVec<T>, 32 * In::W)) : 0) + kAhead;
        const int bytes = kTeams * (slots * In::kSlot + Teacher::floats(a.k) * 4);
        auto kern = a.k <= 32 ? (dx ? distill_warp_kernel<T, U, 1, true> : distill_warp_kernel<T, U, 1, false>)
                              : (dx ? distill_warp_kernel<T, U, kMaxTop / 32, true> : distill_warp_kernel<T, U, kMaxTop / 32, false>);
        launch_rows("distill_loss", kern, ceil_div(a.rows, kTeams), 1, std::min(5, kSharedSm / (bytes + 1024)), 32 * kTeams, bytes, s, a, x, ldx, dx,
                    lddx, slots);
        return;
    }
    const auto go = [&](auto nt) {
        constexpr int NT = decltype(nt)::value, kSlot = Stream<T, NT>::kSlot;
        constexpr int kMost = 212 * 1024 * NT / 768 / kSlot;  // slots, with 768 reading threads an SM
        // Enough CTAs a row for the SMs to be busy, and for each to hold its part.
        int ranks = row_ranks(a.rows, a.n, 4096);
        const auto steps = [&] {
            return static_cast<int>(ceil_div(ceil_div(a.n / kVec<T>, ranks), NT * Stream<T, NT>::W));
        };
        while (dx && ranks < 8 && steps() > kMost) ranks *= 2;
        const bool hold = dx && steps() <= kMost;
        const int slots = hold ? steps() : kAhead;
        // (by registers, and by shared memory)
        const int resident = std::max(1, std::min(dx ? 768 / NT : 1024 / (NT + 32), kSharedSm / (slots * kSlot + 4608)));
        auto kern = dx ? distill_wide_kernel<T, U, NT, true> : distill_wide_kernel<T, U, NT, false>;
        launch_rows("distill_loss", kern, a.rows, ranks, resident, NT + 32, slots * kSlot, s, a, x, ldx, dx, lddx, slots, hold);
    };
    if (!dx) {
        if (a.n / row_ranks(a.rows, a.n, 4096) <= 8192) go(std::integral_constant<int, 128>{});
        else go(std::integral_constant<int, 256>{});
        return;
    }
    if (a.n * sizeof(T) <= 32 * 1024) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
}

}  // namespace

}  // namespace tg

extern "C" {

TG_API tg_status tg_distill_loss(int64_t rows, int64_t classes, int32_t dtype, const void* logits, int64_t ldz, int64_t k,
                                 const void* top_classes, int32_t class_bytes, int64_t ld_classes,
                                 int32_t teacher_dtype, const void* top_logits, int64_t ld_logits, float temperature,
                                 const float* weights, float* loss, void* dlogits, int64_t lddz, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "distill_loss";
        logits::check_row_args(fn, rows, classes, dtype, logits, ldz);
        logits::check_int_bytes(fn, "top_classes", class_bytes);
        if (k < 1 || k > logits::kMaxTop)
            invalid(std::string(fn) + ": " + std::to_string(k) + " classes a row are outside [1, " +
                    std::to_string(logits::kMaxTop) + "]");
        if (teacher_dtype != TG_F32 && teacher_dtype != dtype)
            invalid(std::string(fn) + ": top_logits must be fp32 or of the logits' type");
        check_ptr(fn, "top_classes", top_classes, rows > 0);
        check_ptr(fn, "top_logits", top_logits, rows > 0);
        check_ptr(fn, "loss", loss, rows > 0);
        check_ld(fn, "top_classes", ld_classes, k);
        check_ld(fn, "top_logits", ld_logits, k);
        if (dlogits) check_ld(fn, "dlogits", lddz, classes);
        if (!(temperature >= 1e-30f && temperature <= 1e30f))
            invalid(std::string(fn) + ": temperature must be positive and finite (1e-30 to 1e30)");
        const DistillArgs a{rows, static_cast<int>(classes), static_cast<int>(k), top_classes, class_bytes == 8, ld_classes,
                            top_logits, ld_logits, temperature, 1.0f / temperature, weights, loss};
        by_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            const T* x = static_cast<const T*>(logits);
            T* dx = static_cast<T*>(dlogits);
            if (teacher_dtype == TG_F32) distill<T, float>(a, x, ldz, dx, lddz, as_stream(stream));
            else distill<T, T>(a, x, ldz, dx, lddz, as_stream(stream));
        });
    });
}

}  // extern "C"

// ============================================================================
//  logits.cuh -- what the kernels on rows of class scores share (label.cu,
//  distill.cu): the running softmax of a row, its reduction over the threads
//  and CTAs that share the row, and how rows are read.
//
//  A row's softmax is kept as (m, s, t): the maximum so far, s = sum e^d and
//  t = sum d e^d with d = (z - m) c, so that one pass over the scores gives
//  log p = d - log s and the entropy log s - t / s.  A new maximum m' scales s
//  and t by e^((m - m') c).
//
//  Rows of at most kNarrow classes go through shared memory, many rows of
//  contiguous memory at a time (rows of 41 floats begin anywhere, and
//  16-byte loads of the whole block do not mind), and a row is then shared by
//  LPR lanes that keep E scores each in registers.  Wider rows are read in
//  16-byte vectors by a team: a warp up to kWarp classes (a row's sums then need
//  no barrier, and the SM has 16 to 32 rows under way), a block or the blocks of
//  a cluster beyond.  The few scores before the first and after the last aligned
//  vector are read one by one.
// ============================================================================
#pragma once

#include <algorithm>

#include "values.cuh"

namespace tg {
namespace logits {

constexpr int kNarrow = 256;    // widest row that goes through shared memory with others
constexpr int kWarp = 4096;     // widest row that a warp has alone
constexpr int kMaxTop = 128;    // most alternatives of a row
constexpr int kNarrowThreads = 256;
constexpr int kSharedSm = 228 * 1024;  // shared memory of an SM; each block takes 1 KB of it for itself

constexpr float kLn2 = 0.6931471806f, kLog2e = 1.4426950409f;

// 16-bit scores take the hardware's 2^x (within 2^-22), d in units of ln 2;
// fp32 scores expf, d in natural units.
template <bool FAST>
__device__ __forceinline__ float expo(float d) { return FAST ? exp2_hw(d) : expf(d); }
template <bool FAST>
constexpr float kUnit = FAST ? kLn2 : 1.0f;  // natural units of one unit of d

// d = (z - m) c, at least -200 (whose exponential is 0): a masked class's -inf
// would make d e^d a NaN.  A NaN stays one.
__device__ __forceinline__ float distance(float z, float m, float c) {
    return max_nan(__fmul_rn(__fsub_rn(z, m), c), -200.0f);
}
// The maximum as the scores' origin: a row without any score above -inf has
// the origin 0, and its exponentials are all 0.
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.0f : m; }

struct Soft {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
};

// 16-bit scores whose entropy is not asked for (FUSED): d = z c - M with M = m c
// rounded once, one instruction a score.  M's rounding r = m c - M shifts all of
// a row's d alike and falls out of log p = d - log s; it is at most 2^-15 while
// |M| <= 1024.  A maximum beyond that (`far`: a mask of a large finite number, a
// small temperature), where r could leave the exponential's range, takes
// (z - m) c, which is 0 at the maximum.  A row's state is always that of its own
// maximum's form; `between` takes r along where the two differ.  (With the entropy,
// whose log p of a sure label is to be 0, all rows take (z - m) c.)
template <bool FAST, bool ENTROPY>
constexpr bool kFused = FAST && !ENTROPY;
struct Origin {
    float m, M;
    bool far;
    __device__ __forceinline__ Origin(float most, float c) : m(origin(most)) {
        M = __fmul_rn(m, c);
        far = !(fabsf(M) <= 1024.0f);  // (or NaN)
    }
    // At least -inf: its exponential is 0.
    __device__ __forceinline__ float d(float z, float c) const {
        return far ? __fmul_rn(__fsub_rn(z, m), c) : fmaf(z, c, -M);
    }
};
// d of the maximum `from` as seen from the maximum `to`: what scales a state of
// the one to the other.
template <bool FUSED>
__device__ __forceinline__ float between(float from, float to, float c) {
    if (FUSED && from != -INFINITY) {
        const Origin a(from, c), b(to, c);
        if (!a.far) return b.far ? -fmaf(to, c, -a.M) : __fsub_rn(a.M, b.M);
        if (!b.far) return fmaf(from, c, -b.M);
    }
    return distance(from, to, c);
}
// A CTA's state where the other CTAs of its cluster read it.
struct SoftCell {
    float m, s, t;
    __device__ __forceinline__ void set(const Soft& a) { m = a.m, s = a.s, t = a.t; }
    __device__ __forceinline__ Soft get() const {
        Soft a;
        a.m = m, a.s = s, a.t = t;
        return a;
    }
};

// The greatest of N words' scores (a NaN, if there is one).
template <class T, int N>
__device__ __forceinline__ float top_of(const uint32_t (&w)[N]) {
    uint32_t top = w[0];
#pragma unroll
    for (int i = 1; i < N; ++i) {
        if (std::is_same<T, float>::value) top = __float_as_uint(max_nan(__uint_as_float(top), __uint_as_float(w[i])));
        else if (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(top) : "r"(w[i]));
        else asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(w[i]));
    }
    if (sizeof(T) == 4) return __uint_as_float(top);
    Raw<T, 2> r;
    r.w[0] = top;
    float z[2];
    widen(r, z);
    return max_nan(z[0], z[1]);
}

// The state with the maximum `top`, if that is not below its own.
template <bool FAST, bool ENTROPY>
__device__ __forceinline__ void see_top(Soft& a, float top, float c) {
    if (!(top <= a.m)) {
        top = max_nan(top, a.m);  // (a NaN stays the maximum)
        const float d = between<kFused<FAST, ENTROPY>>(a.m, top, c), f = expo<FAST>(d);
        if (ENTROPY) a.t = __fmul_rn(f, fmaf(d, a.s, a.t));
        a.s = __fmul_rn(a.s, f);
        a.m = top;
    }
}

// Adds V scores, of which `top` is the greatest (those that are not there are -inf).
template <bool FAST, bool ENTROPY, int V>
__device__ __forceinline__ void add_scores(Soft& a, const float (&z)[V], float top, float c) {
    see_top<FAST, ENTROPY>(a, top, c);
    Pair s(0.0f, 0.0f), t(0.0f, 0.0f);
    float x, y;
    const Origin o(a.m, c);
    if (kFused<FAST, ENTROPY> && !o.far) {
        const Pair k(-o.M, -o.M), cc(c, c);
#pragma unroll
        for (int j = 0; j + 1 < V; j += 2) {
            fma2(Pair(z[j], z[j + 1]), cc, k).get(x, y);
            s = add2(s, Pair(expo<FAST>(x), expo<FAST>(y)));
        }
        if (V % 2) s = add2(s, Pair(expo<FAST>(fmaf(z[V - 1], c, -o.M)), 0.0f));
    } else {
        const Pair k(-o.m, -o.m), cc(c, c);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            mul2(add2(Pair(z[j], z[j + 1 < V ? j + 1 : j]), k), cc).get(x, y);
            x = max_nan(x, -200.0f), y = max_nan(y, -200.0f);
            const Pair e(expo<FAST>(x), j + 1 < V ? expo<FAST>(y) : 0.0f);
            s = add2(s, e);
            if (ENTROPY) t = fma2(Pair(x, y), e, t);
        }
    }
    s.get(x, y);
    a.s = __fadd_rn(a.s, __fadd_rn(x, y));
    if (ENTROPY) {
        t.get(x, y);
        a.t = __fadd_rn(a.t, __fadd_rn(x, y));
    }
}
template <bool FAST, bool ENTROPY, int V>
__device__ __forceinline__ void add_scores(Soft& a, const float (&z)[V], float c) {
    float top = z[0];
#pragma unroll
    for (int j = 1; j < V; ++j) top = max_nan(top, z[j]);
    add_scores<FAST, ENTROPY, V>(a, z, top, c);
}

// The state with the maximum m, which is at least its own.
template <bool FAST, bool ENTROPY>
__device__ __forceinline__ void raise_to(Soft& a, float m, float c) {
    if (a.m == m) return;
    const float d = between<kFused<FAST, ENTROPY>>(a.m, m, c), f = expo<FAST>(d);
    if (ENTROPY) a.t = __fmul_rn(f, fmaf(d, a.s, a.t));
    a.s = __fmul_rn(a.s, f);
    a.m = m;
}

// The state of W neighbouring lanes, in each of them.
template <bool FAST, bool ENTROPY, int W>
__device__ __forceinline__ void lanes_soft(Soft& a, float c) {
    raise_to<FAST, ENTROPY>(a, reduce_max<W>(a.m), c);
    a.s = reduce_sum<float, W>(a.s);
    if (ENTROPY) a.t = reduce_sum<float, W>(a.t);
}

// The threads that share a row within a block: a warp (NT = 32; a block then has
// several teams), or the block's first NT threads.
template <int NT>
struct Team {
    static __device__ __forceinline__ int thread() { return NT == 32 ? threadIdx.x & 31 : threadIdx.x; }
    static __device__ __forceinline__ void sync() {
        if (NT == 32) __syncwarp();
        else asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
    }
    // How many of them; and a block's sync (a warp's ballot orders no memory).
    static __device__ __forceinline__ int count(bool x) {
        if (NT == 32) return __popc(__ballot_sync(0xffffffffu, x));
        int n;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %1, 0;\n\t"
            "bar.red.popc.u32 %0, 1, %2, p;\n\t}"
            : "=r"(n)
            : "r"(static_cast<uint32_t>(x)), "n"(NT)
            : "memory");
        return n;
    }
};

struct SoftShared {
    float m[32], s[32], t[32];
};
// The state of a team, in each of its threads.
template <bool FAST, bool ENTROPY, int NT>
__device__ __forceinline__ void team_soft(Soft& a, float c, SoftShared& sh) {
    constexpr int W = NT / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    lanes_soft<FAST, ENTROPY, 32>(a, c);
    if (NT == 32) return;
    if (lane == 0) {
        sh.m[warp] = a.m;
        sh.s[warp] = a.s;
        if (ENTROPY) sh.t[warp] = a.t;
    }
    Team<NT>::sync();
    a = Soft{};
    if (lane < W) {
        a.m = sh.m[lane];
        a.s = sh.s[lane];
        if (ENTROPY) a.t = sh.t[lane];
    }
    lanes_soft<FAST, ENTROPY, 32>(a, c);
}

// ── ranks of scores ──────────────────────────────────────────────────────
// A score as an integer of the same order (-0 counts as 0, a NaN of any sign
// as the greatest); 0 stands for no score.
__device__ __forceinline__ uint32_t rank_of(float z) {
    const uint32_t u = __float_as_uint(__fadd_rn(z, 0.0f));
    if (z != z) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t r) {
    return __uint_as_float(r & 0x80000000u ? r ^ 0x80000000u : ~r);  // (a NaN for 0xffffffff)
}

// ── rows ─────────────────────────────────────────────────────────────────
template <class T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <class T>
__device__ __forceinline__ uint32_t masked_word() {  // -inf, as it lies in memory
    if (sizeof(T) == 4) return 0xff800000u;
    return std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
}

// One CTA's part of a row: vectors [v0, v1) from `body` on, which is 16-byte
// aligned and starts at column `head`; `extra` scores beside the vectors (the
// first CTA's): columns 0 .. head, and from `tail` on.
template <class T>
struct Part {
    const T *row, *body;
    int head, tail, extra;
    int v0, v1;

    // Part `rank` of 2^log_ranks alike.
    __device__ __forceinline__ Part(const T* p, int n, int rank, int log_ranks) : row(p) {
        const int64_t nv = vectors(n, rank);
        v0 = static_cast<int>(nv * rank >> log_ranks);
        v1 = static_cast<int>(nv * (rank + 1) >> log_ranks);
    }
    // Part `rank` of those of `per` vectors.
    static __device__ __forceinline__ Part of_size(const T* p, int n, int rank, int per) {
        Part r(p);
        const int nv = r.vectors(n, rank);
        r.v0 = rank * per < nv ? rank * per : nv;
        r.v1 = nv - r.v0 < per ? nv : r.v0 + per;
        return r;
    }
    __device__ __forceinline__ bool has(int column) const {
        if (column < head || column >= tail) return extra > 0;
        const int v = (column - head) / kVec<T>;
        return v >= v0 && v < v1;
    }
    __device__ __forceinline__ int extra_column(int i) const { return i < head ? i : tail + i - head; }
    __device__ __forceinline__ int column(int v) const { return head + v * kVec<T>; }
    __device__ __forceinline__ Raw<T, kVec<T>> load(int v) const {
        return load_raw<T, kVec<T>>(body + static_cast<int64_t>(v) * kVec<T>);
    }

  private:
    __device__ __forceinline__ explicit Part(const T* p) : row(p) {}
    __device__ __forceinline__ int vectors(int n, int rank) {
        const int lead = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
        head = lead < n ? lead : n;
        body = row + head;
        const int nv = (n - head) / kVec<T>;
        tail = head + nv * kVec<T>;
        extra = rank == 0 ? head + n - tail : 0;
        return nv;
    }
};

// The parts of rows first, first + step, ... that one team has, read through a
// ring in shared memory by asynchronous copies, across the rows' ends: while a
// row's statistics are joined the next row's scores are on their way.  Each
// thread copies and reads the vectors part.v0 + thread, + NT, ..., two a slot of
// the ring, so that nobody waits for another thread's copies; one group of
// copies (empty after the last row) is committed a slot.
template <class T, int NT>
struct Stream {
    static constexpr int W = 2;                       // vectors of a slot
    static constexpr int kSlot = NT * W * 16;         // bytes
    const T* x;
    int64_t ldx, rows, step;
    int n, rank, log_ranks, slots;
    bool twice;      // each row is read twice
    uint32_t base;   // of this thread's vector in the first slot
    // what is asked for next
    int64_t row;
    const T* at;
    int left, steps, again, slot;
    // the slot that is read next
    int from;

    __device__ __forceinline__ Stream(const T* x_, int64_t ldx_, int64_t rows_, int n_, int64_t first, int64_t step_, int rank_,
                                      int log_ranks_, uint8_t* room, int slots_, bool twice_)
        : x(x_), ldx(ldx_), rows(rows_), step(step_), n(n_), rank(rank_), log_ranks(log_ranks_), slots(slots_), twice(twice_),
          base(static_cast<uint32_t>(__cvta_generic_to_shared(room)) + Team<NT>::thread() * 16), row(first), at(nullptr), left(0),
          steps(0), again(twice_ ? 2 : 1), slot(0), from(0) {
        open();
        for (int i = 0; i < slots; ++i) ask();
    }
    static __device__ __forceinline__ int steps_of(const Part<T>& p) {
        return (p.v1 - p.v0 + NT * W - 1) / (NT * W);
    }
    __device__ __forceinline__ void open() {
        while (row < rows) {
            const Part<T> p(x + row * ldx, n, rank, log_ranks);
            steps = steps_of(p);
            if (steps > 0) {
                at = p.body + (static_cast<int64_t>(p.v0) + Team<NT>::thread()) * kVec<T>;
                left = p.v1 - p.v0 - Team<NT>::thread() - (steps - 1) * NT * W;  // (of the last step's)
                return;
            }
            row += step;
        }
    }
    __device__ __forceinline__ uint32_t address(int s, int w) const { return base + (s * W + w) * (NT * 16); }
    // Asks for the next vectors, into the oldest slot (whose vectors have been used).
    __device__ __forceinline__ void ask() {
        if (steps > 0) {
            const uint32_t to = address(slot, 0);
            if (steps > 1) {
#pragma unroll
                for (int w = 0; w < W; ++w) copy(to + w * NT * 16, at + w * NT * kVec<T>);
            } else {
#pragma unroll
                for (int w = 0; w < W; ++w)
                    if (left > w * NT) copy(to + w * NT * 16, at + w * NT * kVec<T>);
            }
            at += W * NT * kVec<T>;
            if (--steps == 0) {
                if (--again == 0) {
                    again = twice ? 2 : 1;
                    row += step;
                }
                open();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot = next(slot);
    }
    static __device__ __forceinline__ void copy(uint32_t to, const T* from) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    }
    // Waits until at most N of the groups asked for are on their way.
    template <int N>
    __device__ __forceinline__ void wait() const {
        asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    }
    // Slot s as it lies in memory; vectors from `have` threads on are masked.
    __device__ __forceinline__ void read(int s, int have, uint32_t (&r)[4 * W]) const {
#pragma unroll
        for (int w = 0; w < W; ++w)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r[4 * w]), "=r"(r[4 * w + 1]), "=r"(r[4 * w + 2]), "=r"(r[4 * w + 3])
                         : "r"(address(s, w))
                         : "memory");
        if (have < NT * W) {  // (the last slot of a row)
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (have <= w * NT + Team<NT>::thread()) r[4 * w] = r[4 * w + 1] = r[4 * w + 2] = r[4 * w + 3] = masked_word<T>();
        }
    }
    static __device__ __forceinline__ void scores(const uint32_t (&r)[4 * W], float (&z)[W * kVec<T>]) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            Raw<T, kVec<T>> x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x.w[j] = r[4 * w + j];
            widen(x, z + w * kVec<T>);
        }
    }
    // Adds slot s to the running softmax.
    template <bool ENTROPY>
    __device__ __forceinline__ void add(Soft& a, int s, int have, float c) const {
        uint32_t r[4 * W];
        float z[W * kVec<T>];
        read(s, have, r);
        scores(r, z);
        add_scores<sizeof(T) == 2, ENTROPY>(a, z, top_of<T>(r), c);
    }
    __device__ __forceinline__ int next(int s) const { return s + 1 == slots ? 0 : s + 1; }
};

// Copies `rows` rows of n classes from row r0 on into shared memory (of n rows,
// and 16 bytes): returns the address of the first, the others follow n apart.
template <class T>
__device__ __forceinline__ T* stage_in(uint8_t* sh, const T* x, int64_t ldx, int64_t r0, int rows, int n) {
    const T* src = x + r0 * ldx;
    if (ldx != n) {
        T* to = reinterpret_cast<T*>(sh);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int r = warp; r < rows; r += kNarrowThreads / 32)
            for (int j = lane; j < n; j += 32) to[r * n + j] = src[r * ldx + j];
        return to;
    }
    constexpr int V = kVec<T>;
    const int phase = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15), count = rows * n;
    T* to = reinterpret_cast<T*>(sh + phase);
    const int lead = ((16 - phase) & 15) / static_cast<int>(sizeof(T)), head = lead < count ? lead : count;
    const int nv = (count - head) / V, tail = head + nv * V;
    if (threadIdx.x < head) to[threadIdx.x] = src[threadIdx.x];
    if (threadIdx.x < count - tail) to[tail + threadIdx.x] = src[tail + threadIdx.x];
    constexpr int U = 4;
    for (int v = threadIdx.x; v < nv; v += kNarrowThreads * U) {
        Raw<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * kNarrowThreads < nv) r[u] = load_raw<T, V>(src + head + (v + u * kNarrowThreads) * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * kNarrowThreads < nv) *reinterpret_cast<Raw<T, V>*>(to + head + (v + u * kNarrowThreads) * V) = r[u];
    }
    return to;
}
// The same way out again.
template <class T>
__device__ __forceinline__ void stage_out(const T* from, T* y, int64_t ldy, int64_t r0, int rows, int n) {
    T* dst = y + r0 * ldy;
    const int phase = static_cast<int>(reinterpret_cast<uintptr_t>(dst) & 15);
    if (ldy != n || phase != static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15)) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int r = warp; r < rows; r += kNarrowThreads / 32)
            for (int j = lane; j < n; j += 32) dst[r * ldy + j] = from[r * n + j];
        return;
    }
    constexpr int V = kVec<T>;
    const int count = rows * n;
    const int lead = ((16 - phase) & 15) / static_cast<int>(sizeof(T)), head = lead < count ? lead : count;
    const int nv = (count - head) / V, tail = head + nv * V;
    if (threadIdx.x < head) dst[threadIdx.x] = from[threadIdx.x];
    if (threadIdx.x < count - tail) dst[tail + threadIdx.x] = from[tail + threadIdx.x];
    for (int v = threadIdx.x; v < nv; v += kNarrowThreads)
        *reinterpret_cast<Raw<T, V>*>(dst + head + v * V) = load_raw<T, V>(from + head + v * V);
}

// Calls f with the lanes of a row and the scores a lane keeps, for n classes.
template <class F>
void by_narrow(int64_t n, F&& f) {
    using std::integral_constant;
    if (n <= 16) f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    else if (n <= 48) f(integral_constant<int, 8>{}, integral_constant<int, 6>{});
    else if (n <= 64) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (n <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
}
// How often RPB rows of n classes, taken together, make up about 16 KB; at most
// as many rows as threads.
inline int narrow_turns(int rpb, int64_t n, size_t size, int64_t rows) {
    const int64_t fit = std::min<int64_t>(16384 / (rpb * n * static_cast<int64_t>(size)), kNarrowThreads / rpb);
    return static_cast<int>(std::max<int64_t>(1, std::min(fit, ceil_div(rows, int64_t(rpb) * num_sms() * 4))));
}

// An integer of 4 or 8 bytes; what does not fit an int is none (-1).
__device__ __forceinline__ int class_at(const void* p, int64_t i, bool wide) {
    if (!wide) return static_cast<const int32_t*>(p)[i];
    const int64_t v = static_cast<const int64_t*>(p)[i];
    return v < 0 || v > INT32_MAX ? -1 : static_cast<int>(v);
}

constexpr int kFixed = 5 * 1024;  // more than the static shared memory of a kernel that takes over 32 KB beside it

// Launches clusters of `ranks` blocks for `rows` rows, at most as many as run at
// a time (`resident` blocks an SM: each cluster walks rows, and one that had to
// wait for another to end would come last), dependent on the previous kernel
// (wait_for_previous).
template <class K, class... A>
void launch_rows(const char* name, K kernel, int64_t rows, int ranks, int resident, int block, size_t smem, cudaStream_t s,
                 A... args) {
    if (rows == 0) return;
    if (smem > 32 * 1024) allow_shared(kernel, kMaxShared - kFixed);
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = static_cast<unsigned>(ranks);
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = ranks > 1 ? 2 : 1;
    int64_t clusters = std::max<int64_t>(1, int64_t(num_sms()) * resident / ranks);
    if (ranks > 1 && rows > clusters / 2) {
        // (not every SM finds partners)
        int most = 0;
        cfg.gridDim = dim3(static_cast<unsigned>(ranks));
        cuda_check(cudaOccupancyMaxActiveClusters(&most, kernel, &cfg), name);
        clusters = std::max(1, most);
    }
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(rows, clusters) * ranks));
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), name);
    count_launch(name);
}

// How many CTAs share a row of n classes: as many as fill the SMs (two CTAs
// each), up to 8, while each still has `least` classes.
inline int row_ranks(int64_t rows, int64_t n, int64_t least) {
    int ranks = 1;
    while (ranks < 8 && rows * ranks < num_sms() && n / (2 * ranks) >= least) ranks *= 2;
    return ranks;
}

inline void check_row_args(const char* fn, int64_t rows, int64_t classes, int dtype, const void* z, int64_t ldz) {
    check_dtype(fn, "logits", dtype);
    check_rows_cols(fn, rows, classes);
    check_ptr(fn, "logits", z, rows > 0);
    check_ld(fn, "logits", ldz, classes);
}

inline void check_int_bytes(const char* fn, const char* what, int bytes) {
    if (bytes != 4 && bytes != 8)
        invalid(std::string(fn) + ": " + what + " are integers of 4 or 8 bytes, not " + std::to_string(bytes));
}

}  // namespace logits
}  // namespace tg

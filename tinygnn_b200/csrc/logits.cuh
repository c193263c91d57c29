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
//  Rows of at most kNarrow classes go through shared memory, several rows of
//  contiguous memory at a time (rows of 41 floats begin anywhere, and
//  16-byte loads of the whole block do not mind), and a row is then shared by
//  LPR lanes that keep E scores each in registers.  Wider rows are shared by
//  the CTAs of a cluster, which read them in 16-byte vectors: the few scores
//  before the first and after the last aligned vector are the first CTA's.
// ============================================================================
#pragma once

#include "values.cuh"

namespace tg {
namespace logits {

constexpr int kNarrow = 1024;   // widest row that a warp keeps in registers
constexpr int kMaxTop = 128;    // most alternatives of a row
constexpr int kNarrowThreads = 256;

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

// Adds V scores (those that are not there are -inf).
template <bool FAST, bool ENTROPY, int V>
__device__ __forceinline__ void add_scores(Soft& a, const float (&z)[V], float c) {
    float top = z[0];
#pragma unroll
    for (int j = 1; j < V; ++j) top = max_nan(top, z[j]);
    if (!(top <= a.m)) {
        top = max_nan(top, a.m);  // (a NaN stays the maximum)
        const float d = distance(a.m, top, c), f = expo<FAST>(d);
        if (ENTROPY) a.t = __fmul_rn(f, fmaf(d, a.s, a.t));
        a.s = __fmul_rn(a.s, f);
        a.m = top;
    }
    const float m = origin(a.m);
    float s[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float d = distance(z[j], m, c), e = expo<FAST>(d);
        s[j & 1] = __fadd_rn(s[j & 1], e);
        if (ENTROPY) t[j & 1] = fmaf(d, e, t[j & 1]);
    }
    a.s = __fadd_rn(a.s, __fadd_rn(s[0], s[1]));
    if (ENTROPY) a.t = __fadd_rn(a.t, __fadd_rn(t[0], t[1]));
}

// The state with the maximum m, which is at least its own.
template <bool FAST, bool ENTROPY>
__device__ __forceinline__ void raise_to(Soft& a, float m, float c) {
    if (a.m == m) return;
    const float d = distance(a.m, m, c), f = expo<FAST>(d);
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

struct SoftShared {
    float m[32], s[32], t[32];
};
// The state of a block of NT threads, in each of them.
template <bool FAST, bool ENTROPY, int NT>
__device__ __forceinline__ void block_soft(Soft& a, float c, SoftShared& sh) {
    constexpr int W = NT / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    lanes_soft<FAST, ENTROPY, 32>(a, c);
    if (lane == 0) {
        sh.m[warp] = a.m;
        sh.s[warp] = a.s;
        if (ENTROPY) sh.t[warp] = a.t;
    }
    __syncthreads();
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
    int64_t v0, v1;

    __device__ __forceinline__ Part(const T* p, int64_t n, int rank, int ranks) : row(p) {
        const int lead = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
        head = lead < n ? lead : static_cast<int>(n);
        body = p + head;
        const int64_t nv = (n - head) / kVec<T>;
        tail = static_cast<int>(head + nv * kVec<T>);
        extra = rank == 0 ? head + static_cast<int>(n - tail) : 0;
        v0 = nv * rank / ranks;
        v1 = nv * (rank + 1) / ranks;
    }
    __device__ __forceinline__ int extra_column(int i) const { return i < head ? i : tail + i - head; }
    __device__ __forceinline__ int column(int64_t v) const { return head + static_cast<int>(v) * kVec<T>; }
    __device__ __forceinline__ Raw<T, kVec<T>> load(int64_t v) const { return load_raw<T, kVec<T>>(body + v * kVec<T>); }
};

// Calls f(v, V scores) for this thread's vectors, v0 + thread, + NT, ...; U are
// asked for before the first is looked at.
template <class T, int NT, int U, class F>
__device__ __forceinline__ void for_vectors(const Part<T>& p, F&& f) {
    constexpr int V = kVec<T>;
    for (int64_t v = p.v0 + threadIdx.x; v < p.v1; v += NT * U) {
        Raw<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * NT < p.v1) r[u] = p.load(v + u * NT);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + u * NT < p.v1) {
                float z[V];
                widen(r[u], z);
                f(v + u * NT, z);
            }
    }
}

// This thread's running softmax over its part (and, for the first threads of
// the first CTA, of one of the scores beside the vectors).
template <class T, int NT, int U, bool ENTROPY>
__device__ __forceinline__ Soft scan_part(const Part<T>& p, float c) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int V = kVec<T>;
    Soft a;
    for (int64_t v = p.v0 + threadIdx.x; v < p.v1; v += NT * U) {
        Raw<T, V> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (v + u * NT < p.v1) {
                r[u] = p.load(v + u * NT);
            } else {
#pragma unroll
                for (int j = 0; j < Raw<T, V>::N; ++j) r[u].w[j] = masked_word<T>();
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float z[V];
            widen(r[u], z);
            add_scores<FAST, ENTROPY>(a, z, c);
        }
    }
    return a;
}

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
    else if (n <= 64) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (n <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}

// An integer of 4 or 8 bytes; what does not fit an int is none (-1).
__device__ __forceinline__ int class_at(const void* p, int64_t i, bool wide) {
    if (!wide) return static_cast<const int32_t*>(p)[i];
    const int64_t v = static_cast<const int64_t*>(p)[i];
    return v < 0 || v > INT32_MAX ? -1 : static_cast<int>(v);
}

// Launches clusters of `ranks` blocks, `clusters` of them, dependent on the
// previous kernel (wait_for_previous).
template <class K, class... A>
void launch_clusters(const char* name, K kernel, int64_t clusters, int ranks, int block, size_t smem, cudaStream_t s,
                     A... args) {
    if (clusters == 0) return;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * ranks));
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

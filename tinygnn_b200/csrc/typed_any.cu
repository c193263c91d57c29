// ============================================================================
//  typed_any.cu -- the typed products on the tensor cores for operands that are
//  converted on their way into shared memory.
//
//  TMA copies values as they are.  Here eight loader warps read the operands
//  with plain loads and write the MMA's 16-bit tiles themselves, so one launch
//  takes
//   fp32       each value split into three bf16 parts (24 bits, exactly):
//              x0 = x's upper half, x1 = bf16(x - x0), x2 = bf16(x - x0 - x1);
//              a product is the six part products x_i y_j with i + j <= 2
//              (what is left out is below 2^-23 of it and of random sign), in
//              parts of 768 inner indexes that are added up in fp32, rounded
//              to nearest (see stage_mmas).  An infinity in an fp32 operand
//              gives NaN;
//   bf16, fp16 (weight gradients of moderate size: db is added up on the way);
//   8 bits     code * 2^e as one bf16 or fp16 value, exactly;
//  and rows past a type's end and columns past the matrix are zeros.  Where
//  dY passes through the loaders, they add up db on the way.
//
//    warps 0-7    loaders: the next stage's values are in registers (in
//                 flight) while this stage's are converted and written;
//    warp 8       the MMAs (one thread);
//    warps 12-15  the epilogue of one of two TMEM accumulators while the next
//                 tile is multiplied (warps 9-11 only take part in the set-up:
//                 a warp reads the TMEM lanes of its number modulo 4).
//
//  fp32: 232,965 x 602 x 128 forward takes 334-343 us, 0.11 PFLOP/s of fp32
//  products and six times that of MMAs (the tensor cores' measured rate would
//  allow 126 us).  The MMAs of a 128 x 128 tile read shared memory at its full
//  rate and are active 36 % of the time; the loaders' loads and stores take
//  another 23 % of shared memory's cycles and, of all load/store wavefronts, 52 %,
//  and issue slots are 40 % busy.  Nothing is full: with room for two stages of
//  96 KB, converting one stage and multiplying the other wait for each other.
// ============================================================================
#include <type_traits>

#include "typed_mma.cuh"

namespace tg {

namespace {

using namespace typed;

enum Op { kForward, kGradInput, kGradWeight };

constexpr int kLoaders = 256, kThreads = 512;

template <class T>
struct AnyArgs {
    int64_t M, K, N;  // rows; inner length (weight: rows of dW); output columns
    int types, tiles_m, tiles_n;  // tiles_m: of dW's rows (weight only)
    const int32_t* offsets;
    const T* A;
    int64_t lda;
    Saved8 a8;  // the first operand in 8 bits (weight only)
    const T* B;
    int64_t ldb, stride_b;
    bool a_pair, b_pair;  // rows aligned to two values, not to 16 bytes (fp32)
    // weight
    int slots;
    int64_t stride_c, ldp;
    float* part;
    int out_f32;
    float *db, *db_part;
};

// A tile's source: rows of 8-value chunks.
template <class T>
struct Source {
    const T* p;
    int64_t ld;
    int rows, cols;  // of the tile, how many exist
};

// Chunk c of row r of a plane: 128-byte rows, 16-byte chunks swizzled.  Tiles
// of more than 64 columns are chunks of 8 KB.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return static_cast<uint32_t>(c >> 3) * tc::kChunkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}
// (plain stores: the compiler may mix the conversions of many values, which
// volatile ones would run one chain after the other)
__device__ __forceinline__ void store_chunk(uint8_t* at, const uint32_t (&w)[4]) {
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
}
// N fp32 values (as words) to three bf16 parts, packed by twos: parts[q][N / 2].
template <int N>
__device__ __forceinline__ void split3(const uint32_t* w, uint32_t (&parts)[3][N / 2]) {
    float x[N];
    Raw<__nv_bfloat16, N> h;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __fsub_rn(__uint_as_float(w[j]), __uint_as_float(w[j] & 0xffff0000u));
#pragma unroll
    for (int j = 0; j < N / 2; ++j) parts[0][j] = __byte_perm(w[2 * j], w[2 * j + 1], 0x7632);
    narrow(x, h);
    float y[N];
    widen(h, y);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) parts[1][j] = h.w[j];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __fsub_rn(x[j], y[j]);
    narrow(x, h);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) parts[2][j] = h.w[j];
}
// 16 bytes of values into one plane (16-bit types: 16 bytes of it) or three
// (fp32: 8 bytes of each), `plane` bytes apart.
template <class T>
__device__ __forceinline__ void put16(uint8_t* at, uint32_t plane, const uint32_t* w) {
    if constexpr (sizeof(T) == 2) {
        store_chunk(at, {w[0], w[1], w[2], w[3]});
    } else {
        uint32_t k[3][2];
        split3<4>(w, k);
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<uint2*>(at + q * plane) = make_uint2(k[q][0], k[q][1]);
    }
}
// Two fp32 values into three planes.
__device__ __forceinline__ void put2(uint8_t* at, uint32_t plane, const uint32_t* w) {
    uint32_t k[3][1];
    split3<2>(w, k);
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint32_t*>(at + q * plane) = k[q][0];
}
template <class T>
__device__ __forceinline__ float value_of(const uint32_t* w, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    T v[2];
    *reinterpret_cast<uint32_t*>(v) = w[j / 2];
    return to_f32(v[j % 2]);
}

// The part of a tile of ROWS memory rows x COLS columns that one of THREADS
// loader threads moves.  Rows 16-byte aligned: VAL neighbouring columns (16
// bytes; 8 of an 8-bit copy) of every STEP-th row.  fp32 rows aligned to two
// values (602 columns; a copy would cost as much as the product): a warp takes
// 64 columns of a row at a time, two neighbouring ones a lane, so that its
// loads cover whole lines; halves of 128 columns belong to warps of one parity,
// so a lane keeps its columns.  No access is partly past a row's end (other
// matrices are copied first).
template <int ROWS, int COLS, int THREADS, int VAL>
struct Part {
    static constexpr int LANES = COLS / VAL, STEP = THREADS / LANES, N = ROWS / STEP;
    static constexpr int HALVES = COLS / 64, WARPS = THREADS / 32, PAIRS = ROWS * HALVES / WARPS;
    static constexpr int PAIR_STEP = WARPS / HALVES, kVal = VAL;
    static_assert(2 * PAIRS == VAL * N && 8 % PAIR_STEP == 0, "both forms hold as many values");
    static __device__ __forceinline__ constexpr int rows() { return ROWS; }
    static __device__ __forceinline__ constexpr int cols() { return COLS; }
    static __device__ __forceinline__ int col() { return threadIdx.x % LANES * VAL; }
    static __device__ __forceinline__ int row(int i) { return threadIdx.x % THREADS / LANES + i * STEP; }
    static __device__ __forceinline__ int warp() { return threadIdx.x % THREADS / 32; }
    static __device__ __forceinline__ int pair_col() { return warp() % HALVES * 64 + threadIdx.x % 32 * 2; }
    static __device__ __forceinline__ int pair_row(int i) { return warp() / HALVES + i * PAIR_STEP; }
};
// Words that one thread's values take.
template <class P, class T>
constexpr int words() { return P::N * P::kVal * static_cast<int>(sizeof(T)) / 4; }

// pair: rows aligned to two values (fp32 only).
template <class P, class T>
__device__ __forceinline__ void fetch_tile(const Source<T>& s, bool pair, uint32_t (&w)[words<P, T>()]) {
    if (sizeof(T) == 2 || !pair) {
        const T* p = s.p + P::row(0) * s.ld + P::col();
        const int64_t step = P::STEP * s.ld;
        const bool there = P::col() < s.cols;
#pragma unroll
        for (int i = 0; i < P::N; ++i, p += step) {
            const uint4 q = there && P::row(i) < s.rows ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
            w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
        }
    } else {
        const T* p = s.p + P::pair_row(0) * s.ld + P::pair_col();
        const int64_t step = P::PAIR_STEP * s.ld;
        const bool there = P::pair_col() < s.cols;
#pragma unroll
        for (int i = 0; i < words<P, T>() / 2; ++i, p += step) {
            const uint2 q = there && P::pair_row(i) < s.rows ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
            w[2 * i] = q.x, w[2 * i + 1] = q.y;
        }
    }
}
// The fetched values into the planes at `tile`; add: their column sums on top
// of `sum`.  A row's place in the swizzle repeats every 8 rows, so the
// addresses are a few and constant steps from them.
template <class P, class T>
__device__ __forceinline__ void put_tile(uint8_t* tile, uint32_t plane, bool pair,
                                         const uint32_t (&w)[words<P, T>()], bool add, float (&sum)[8]) {
    if (sizeof(T) == 2 || !pair) {
        static_assert(P::STEP % 8 == 0, "whole swizzle periods");
        uint8_t* at = tile + chunk_at(P::row(0), P::col() / 8) + P::col() % 8 * 2;
#pragma unroll
        for (int i = 0; i < P::N; ++i) put16<T>(at + i * P::STEP * 128, plane, w + i * 4);
        if (add) {
#pragma unroll
            for (int i = 0; i < P::N; ++i)
#pragma unroll
                for (int j = 0; j < P::kVal; ++j) sum[j] += value_of<T>(w + i * 4, j);
        }
    } else {
        constexpr int PERIOD = 8 / P::PAIR_STEP;
        const int c = P::pair_col();
        uint8_t* at[PERIOD];
#pragma unroll
        for (int i = 0; i < PERIOD; ++i) at[i] = tile + chunk_at(P::pair_row(i), c >> 3) + (c & 7) * 2;
#pragma unroll
        for (int i = 0; i < words<P, T>() / 2; ++i) put2(at[i % PERIOD] + i / PERIOD * 1024, plane, w + i * 2);
        if (add) {
#pragma unroll
            for (int i = 0; i < words<P, T>() / 2; ++i) {
                sum[0] += value_of<T>(w + i * 2, 0);
                sum[1] += value_of<T>(w + i * 2, 1);
            }
        }
    }
}
template <class P>
__device__ __forceinline__ void fetch_tile8(const Saved8& s, int64_t row0, int64_t col0, int rows, int cols,
                                            Raw<int8_t, 8> (&k)[P::N], int (&e)[P::N]) {
    const int c = P::col();
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
        const bool live = P::row(i) < rows && c < cols;
        const int64_t r = row0 + P::row(i);
        if (live) k[i] = *reinterpret_cast<const Raw<int8_t, 8>*>(s.codes + r * s.ld + col0 + c);
        else k[i].w[0] = k[i].w[1] = 0u;
        e[i] = live ? s.exps[r * s.lde + col0 / kBlock8] : 127;
    }
}

// What a step of the loop over (tile, inner block) is.
struct Item {
    int t, p;
    int64_t m0, n0;   // first row (rows products) or first row of dW; first column
    int64_t r0, r1;   // the type's rows from the tile's (piece's) first to the end
    int steps;
    bool whole;       // weight: the type has this one piece
};

template <class T, int OP>
__device__ __forceinline__ Item item_at(const AnyArgs<T>& g, const Shared& s, int64_t it, int BN) {
    Item m;
    if (OP == kGradWeight) {
        const WeightItem w = weight_item(g.offsets, g.types, g.M, g.tiles_m * g.tiles_n, s.prefix, s.order, it);
        m.t = w.t, m.p = w.p, m.r0 = w.r0, m.r1 = w.r1, m.whole = w.whole;
        m.m0 = static_cast<int64_t>(w.in / g.tiles_n) * BM;
        m.n0 = static_cast<int64_t>(w.in % g.tiles_n) * BN;
        m.steps = static_cast<int>((m.r1 - m.r0 + tc::kInner - 1) / tc::kInner);
        return m;
    }
    m.p = static_cast<int>(it / g.tiles_n);
    m.t = find_type(s.prefix, g.types, m.p);
    const int64_t b = clamp_row(g.offsets[m.t], g.M), e = clamp_row(g.offsets[m.t + 1], g.M);
    m.m0 = m.r0 = b + static_cast<int64_t>(m.p - s.prefix[m.t]) * BM;
    m.r1 = m.r0 + BM < e ? m.r0 + BM : e;
    m.n0 = (it - static_cast<int64_t>(m.p) * g.tiles_n) * BN;
    m.steps = static_cast<int>((g.K + tc::kInner - 1) / tc::kInner);
    m.whole = true;
    return m;
}

__device__ __forceinline__ int clip(int64_t n, int most) { return n < 0 ? 0 : (n < most ? static_cast<int>(n) : most); }

// The two operands' sources for inner block kb.
template <class T, int OP>
__device__ __forceinline__ Source<T> source_a(const AnyArgs<T>& g, const Item& m, int kb, int) {
    const int64_t k = static_cast<int64_t>(kb) * tc::kInner;
    if (OP == kGradWeight)
        return {g.A + (m.r0 + k) * g.lda + m.m0, g.lda, clip(m.r1 - m.r0 - k, tc::kInner), clip(g.K - m.m0, BM)};
    return {g.A + m.m0 * g.lda + k, g.lda, clip(m.r1 - m.r0, BM), clip(g.K - k, tc::kInner)};
}
template <class T, int OP>
__device__ __forceinline__ Source<T> source_b(const AnyArgs<T>& g, const Item& m, int kb, int BN) {
    const int64_t k = static_cast<int64_t>(kb) * tc::kInner;
    if (OP == kGradWeight)
        return {g.B + (m.r0 + k) * g.ldb + m.n0, g.ldb, clip(m.r1 - m.r0 - k, tc::kInner), clip(g.N - m.n0, BN)};
    const T* w = g.B + m.t * g.stride_b;
    if (OP == kForward) return {w + k * g.ldb + m.n0, g.ldb, clip(g.K - k, tc::kInner), clip(g.N - m.n0, BN)};
    return {w + m.n0 * g.ldb + k, g.ldb, clip(g.N - m.n0, BN), clip(g.K - k, tc::kInner)};
}

// SAVED: the first operand in 8 bits.
template <class T, int OP, int BN, bool SAVED>
__global__ void __launch_bounds__(kThreads, 1) typed_any_kernel(const AnyArgs<T> g, const RowsOut<T> out) {
    using H = typename Half<T>::type;
    constexpr int PA = SAVED ? 1 : Half<T>::planes, PB = Half<T>::planes;
    using S = Plan<PA, PB, BN>;
    constexpr int STAGES = S::kStages;
    constexpr bool W = OP == kGradWeight, A_OUTER = W, B_OUTER = OP != kGradInput, SPLIT = PB > 1;
    // Steps that one accumulator takes; sums of more are added up in the output.
    const int part = SPLIT ? 12 : (W && g.out_f32 ? 32 : 1 << 30);
    constexpr int ACC = SPLIT ? 2 * BN : BN;  // TMEM columns of a buffer
    constexpr uint32_t ID = tc::idesc(is_bf16<H>(), A_OUTER, B_OUTER, BM, BN);
    // 16-bit values: the loaders are two groups that take the stages in turn, so
    // that one group's loads are in flight while the other's arrive (fp32
    // values would need twice the registers, and take six times as long to
    // multiply).
    constexpr int GROUPS = sizeof(T) == 2 ? 2 : 1, THREADS = kLoaders / GROUPS;
    constexpr int VAL = 16 / static_cast<int>(sizeof(T));
    using PartA = Part<A_OUTER ? 64 : BM, A_OUTER ? BM : 64, THREADS, SAVED ? 8 : VAL>;
    using PartB = Part<B_OUTER ? 64 : BN, B_OUTER ? BN : 64, THREADS, VAL>;

    extern __shared__ uint8_t raw[];
    __shared__ Shared s;
    __shared__ float stage_out[4][(stage_bytes<float>() + 3) / 4];
    __shared__ float db_rows[W ? kLoaders * 8 : 1];
    const uint32_t ring = (mb::smem_u32(raw) + 1023) & ~1023u;
    uint8_t* const ring_p = raw + (ring - mb::smem_u32(raw));
    const uint32_t tmem = set_up<STAGES, BN, SPLIT>(s, 8 / GROUPS, 128, [&] {
        if (W) plan_pieces(g.offsets, g.types, g.M, g.tiles_m * g.tiles_n, g.slots, 1 << 30, s.prefix, s.order);
        else scan_types(g.offsets, g.types, g.M, BM, s.prefix);
    });
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t items = static_cast<int64_t>(s.prefix[g.types]) * (W ? g.tiles_m * g.tiles_n : g.tiles_n);

    // Round r's item of this CTA (rows products: equal items, in order).
    const auto item_of = [&](int64_t r) {
        return W ? dealt(r, blockIdx.x, gridDim.x) : blockIdx.x + r * gridDim.x;
    };

    if (warp < 8) {
        // ── loaders ──
        int64_t round = 0, it = item_of(0);
        bool ok = true;
        uint32_t ka[words<PartA, T>()], kb[words<PartB, T>()];
        Raw<int8_t, 8> k8[SAVED ? PartA::N : 1];
        int e8[SAVED ? PartA::N : 1];
        const auto fetch_a = [&](const Item& m, int step) {
            if constexpr (SAVED) {
                const int64_t k = static_cast<int64_t>(step) * tc::kInner;
                fetch_tile8<PartA>(g.a8, m.r0 + k, m.m0, clip(m.r1 - m.r0 - k, tc::kInner), clip(g.K - m.m0, BM), k8,
                                   e8);
            } else {
                fetch_tile<PartA, T>(source_a<T, OP>(g, m, step, BN), g.a_pair, ka);
            }
        };
        const auto fetch_b = [&](const Item& m, int step) {
            fetch_tile<PartB, T>(source_b<T, OP>(g, m, step, BN), g.b_pair, kb);
        };
        const int group = threadIdx.x / THREADS;
        // This group's first step of an item whose first stage is number i0.
        const auto first = [&](int64_t i0) { return GROUPS == 1 ? 0 : static_cast<int>((group + GROUPS - i0 % GROUPS) % GROUPS); };
        // `now` is the step whose values the registers hold, `next` the one
        // that is asked for while they are converted.  Values leave their
        // registers into the stage, and the next step's are asked for as soon
        // as they have: A's are on their way while B is converted, B's while
        // this thread waits for the next stage and converts A.  (One place
        // that fetches and one that converts: small products are bound by
        // instructions being fetched for the first time.)
        Item now{}, next{};
        int step = 0, next_step = 0;
        int64_t base = 0, next_base = 0;  // numbers of the items' first stages
        bool have = false, more = it < items;
        if (more) {
            next = item_at<T, OP>(g, s, it, BN);
            next_step = first(0);
        }
        float sum[8];
        const auto clear = [&] {
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
        };
        clear();
        // Adds the item's column sums of dY up (every loader thread calls it).
        const auto finish_sums = [&](const Item& m) {
            if constexpr (W) {
                if (g.db == nullptr || m.m0 != 0) return;
                // threads that share a column, as rows of db_rows
                const bool vec = sizeof(T) == 2 || !g.b_pair;
                const int G = vec ? kLoaders / PartB::LANES : 8 / PartB::HALVES;
                if (vec) {
#pragma unroll
                    for (int j = 0; j < VAL; ++j) db_rows[threadIdx.x / PartB::LANES * BN + PartB::col() + j] = sum[j];
                } else {
                    float* r = db_rows + threadIdx.x / 32 / PartB::HALVES * BN + PartB::pair_col();
                    r[0] = sum[0];
                    r[1] = sum[1];
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (ok && threadIdx.x < BN && m.n0 + threadIdx.x < g.N) {
                    float all = 0.0f;
#pragma unroll 4
                    for (int q = 0; q < G; ++q) all += db_rows[q * BN + threadIdx.x];
                    (m.whole ? g.db + m.t * g.N : g.db_part + m.p * g.N)[m.n0 + threadIdx.x] = all;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                clear();
            }
        };
        while (have || more) {
            // A group may have no step in an item (two groups, one step).
            const bool fetch_next = more && next_step < next.steps;
            uint8_t* const a = ring_p + static_cast<int>((base + step) % STAGES) * S::kStage;
            const int64_t n = base + step;
            if (have) {
                // (after a wait that ran out the loop goes on without waiting: the
                // loaders meet at barriers)
                if (ok && n >= STAGES) ok = mb::wait(&s.empty[n % STAGES], (n / STAGES - 1) & 1, &g_error, 41);
                ok = __all_sync(0xffffffffu, ok);
                if constexpr (SAVED) {
#pragma unroll
                    for (int u = 0; u < PartA::N; ++u) {
                        float x[8];
                        values4(k8[u].w[0], e8[u], x);
                        values4(k8[u].w[1], e8[u], x + 4);
                        Raw<H, 8> h;
                        narrow(x, h);
                        store_chunk(a + chunk_at(PartA::row(u), PartA::col() / 8), h.w);
                    }
                } else {
                    put_tile<PartA, T>(a, S::kA, g.a_pair, ka, false, sum);
                }
            }
            if (fetch_next) fetch_a(next, next_step);
            if (have) put_tile<PartB, T>(a + PA * S::kA, S::kB, g.b_pair, kb, W && g.db != nullptr && now.m0 == 0, sum);
            if (fetch_next) fetch_b(next, next_step);
            if (have) {
                // (the MMA's thread passes the writes on to the tensor cores: a
                // proxy fence here would wait for the loads just issued)
                __syncwarp();
                if (lane == 0 && ok) mb::arrive(&s.full[n % STAGES]);
            }
            // the sums of every item that `next` is about to leave behind are
            // complete once its last step has been converted
            if (have && (!more || next_base != base)) finish_sums(now);
            have = fetch_next;
            if (fetch_next || more) {
                if (fetch_next) {
                    now = next;
                    step = next_step;
                    base = next_base;
                }
                next_step += GROUPS;
                if (next_step >= next.steps) {
                    if (!fetch_next) finish_sums(next);  // nothing of this item was this group's
                    next_base += next.steps;
                    it = item_of(++round);
                    more = it < items;
                    if (more) {
                        next = item_at<T, OP>(g, s, it, BN);
                        next_step = first(next_base);
                    }
                }
            }
        }
    } else if (warp == 8) {
        // ── MMA issuer ──
        int64_t i = 0;
        int local = 0;  // accumulators filled
        bool ok = true;
        for (int64_t round = 0, it; (it = item_of(round)) < items && ok; ++round) {
            const Item m = item_at<T, OP>(g, s, it, BN);
            for (int k = 0; k < m.steps; ++k, ++i) {
                const int acc = local & 1;
                if (k % part == 0) {
                    if (local >= 2) ok = mb::wait(&s.acc_empty[acc], (local / 2 - 1) & 1, &g_error, 42);
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                    tc::fence_after();
                }
                const int st = static_cast<int>(i % STAGES);
                ok = mb::wait(&s.full[st], (i / STAGES) & 1, &g_error, 43);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc::fence_after();
                const bool done = k + 1 == m.steps || (k + 1) % part == 0;
                if (lane == 0) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the loaders' writes -> MMA reads
                    stage_mmas<PA, PB, BN, A_OUTER, B_OUTER>(ring + st * S::kStage, tmem + acc * ACC, ID, k % part == 0);
                    tc::commit(&s.empty[st]);
                    if (done) tc::commit(&s.acc_full[acc]);
                }
                local += done;
                __syncwarp();
            }
        }
    } else if (warp >= 12) {
        // ── epilogue ──
        const int q = warp & 3;
        T* buf = reinterpret_cast<T*>(stage_out[q]);
        float* buf32 = stage_out[q];
        int local = 0;
        bool ok = true;
        for (int64_t round = 0, it; (it = item_of(round)) < items && ok; ++round) {
            const Item m = item_at<T, OP>(g, s, it, BN);
            if (!W) prefetch_bias<T, BN>(out, m.t, m.n0);
            const int64_t r = m.m0 + q * 32;
            for (int k = 0; k < m.steps; k += part, ++local) {
                const bool first = k == 0, last = k + part >= m.steps;
                const int acc = local & 1;
                ok = mb::wait(&s.acc_full[acc], (local / 2) & 1, &g_error, 46);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc::fence_after();
                const uint32_t addr = tmem + acc * ACC + (static_cast<uint32_t>(q * 32) << 16);
                if constexpr (!W) {
                    finish_rows<T, BN, false, SPLIT>(addr, out, m.t, r, clip(m.r1 - r, 32), m.n0, buf, first,
                                                              last);
                } else {
                    const int rows = clip(g.K - r, 32);
#pragma unroll 1
                    for (int c0 = 0; c0 < BN && m.n0 + c0 < g.N; c0 += 32) {
                        float v[32];
                        load_acc<BN, SPLIT>(addr + c0, v);
                        const int64_t n = m.n0 + c0, left = g.N - n;
                        if (!m.whole) {
                            store_rows(g.part + (m.p * g.K + r) * g.ldp + n, g.ldp, rows, g.ldp - n, v, 2, buf32, !first);
                        } else if (sizeof(T) == 2 && g.out_f32) {
                            store_rows(reinterpret_cast<float*>(out.C) + m.t * g.stride_c + r * out.ldc + n, out.ldc,
                                       rows, left, v, out.mode, buf32, !first);
                        } else {
                            store_rows(out.C + m.t * g.stride_c + r * out.ldc + n, out.ldc, rows, left, v, out.mode, buf,
                                       !first);
                        }
                    }
                }
                tc::fence_before();
                mb::arrive(&s.acc_empty[acc]);
            }
        }
        if constexpr (W) {
            const int e = threadIdx.x - 384;
            if (sizeof(T) == 2 && g.out_f32)
                zero_empty_types(g.offsets, g.types, g.M, g.K, g.N, reinterpret_cast<float*>(out.C), out.ldc, g.stride_c,
                                 out.mode, e, 128);
            else zero_empty_types(g.offsets, g.types, g.M, g.K, g.N, out.C, out.ldc, g.stride_c, out.mode, e, 128);
            if (g.db)
                for (int t = blockIdx.x; t < g.types; t += gridDim.x)
                    if (rows_of(g.offsets, t, g.M) == 0)
                        for (int64_t n = e; n < g.N; n += 128) g.db[t * g.N + n] = 0.0f;
        }
    }
    tear_down<BN, SPLIT>(s, tmem, 8);
}

// The least alignment of fp32 rows that the loaders take, in bytes.
constexpr int64_t kLeast = 8;

template <class T, int OP, int BN, bool SAVED>
void go(const AnyArgs<T>& g, const RowsOut<T>& out, int64_t items, cudaStream_t s) {
    constexpr int PA = SAVED ? 1 : Half<T>::planes;
    run("typed_any", typed_any_kernel<T, OP, BN, SAVED>, kThreads, Plan<PA, Half<T>::planes, BN>::kBytes, items, s, g,
        out);
}

}  // namespace

template <bool TRANS>
void typed_rows_any(const RowsArgs<float>& a, cudaStream_t s) {
    using T = float;
    constexpr int OP = TRANS ? kGradInput : kForward;
    AnyArgs<T> g{};
    g.M = a.M, g.K = a.K, g.N = a.N, g.types = a.types, g.offsets = a.offsets;
    // W[t] is K x N in the forward pass, N x K in the input gradient.
    const int64_t wr = TRANS ? a.N : a.K, wc = TRANS ? a.K : a.N;
    const Operand<T> A(1, a.M, a.K, a.A, a.lda, 0, s, kLeast),
        W(a.types, wr, wc, a.W, a.ldw, a.stride_w, s, kLeast);
    g.A = A.p, g.lda = A.ld, g.B = W.p, g.ldb = W.ld, g.stride_b = W.stride;
    g.a_pair = !in_place(1, A.own ? A.ld : a.K, A.p, A.ld, 0);
    g.b_pair = !in_place(a.types, W.own ? W.ld : wc, W.p, W.ld, W.stride);
    const RowsOut<T> out{a.N, a.bias, a.act, a.alpha, a.C, a.ldc, store_mode(a.C, a.ldc * sizeof(T)), a.saved, a.r8};
    const int64_t pieces = a.M / BM + std::min<int64_t>(a.types, a.M);
    const int BN = tile_width(pieces, a.N, 128, a.saved.codes != nullptr);
    g.tiles_m = 1;
    g.tiles_n = static_cast<int>(ceil_div(a.N, BN));
    if (BN == 64) go<T, OP, 64, false>(g, out, pieces * g.tiles_n, s);
    else go<T, OP, 128, false>(g, out, pieces * g.tiles_n, s);
}

template <class T, class O>
void typed_weight_any(const WeightArgs<T, O>& a, const WeightPlan& w, cudaStream_t s) {
    AnyArgs<T> g{};
    g.M = a.M, g.K = a.K, g.N = a.N, g.types = a.types, g.offsets = a.offsets;
    g.tiles_m = w.tiles_k, g.tiles_n = w.tiles_n;
    g.a8 = a.saved;
    g.slots = w.slots, g.part = w.part, g.ldp = w.ldp, g.stride_c = a.stride_dw;
    g.out_f32 = sizeof(O) == 4;
    RowsOut<T> out{};
    out.N = a.N;
    out.C = reinterpret_cast<T*>(a.dW);
    out.ldc = a.lddw;
    out.mode = store_mode(a.dW, a.lddw * sizeof(O), a.stride_dw * sizeof(O));
    g.db = a.db, g.db_part = w.db_part;
    const auto by_width = [&](auto saved) {
        constexpr bool SAVED = decltype(saved)::value;
        if (w.BN == 64) go<T, kGradWeight, 64, SAVED>(g, out, w.items, s);
        else go<T, kGradWeight, 128, SAVED>(g, out, w.items, s);
    };
    const auto by_source = [&] {
        if (a.saved.codes) by_width(std::true_type{});
        else by_width(std::false_type{});
    };
    if constexpr (sizeof(T) == 2) {  // (rows that the loaders cannot read where they lie go by TMA)
        g.A = a.X, g.lda = a.ldx, g.B = a.dY, g.ldb = a.lddy;
        by_source();
    } else {
        const Operand<T> Y(1, a.M, a.N, a.dY, a.lddy, 0, s, kLeast);
        g.B = Y.p, g.ldb = Y.ld;
        g.b_pair = !in_place(1, Y.own ? Y.ld : a.N, Y.p, Y.ld, 0);
        if (a.saved.codes) {
            by_source();
            return;
        }
        const Operand<T> X(1, a.M, a.K, a.X, a.ldx, 0, s, kLeast);
        g.A = X.p, g.lda = X.ld;
        g.a_pair = !in_place(1, X.own ? X.ld : a.K, X.p, X.ld, 0);
        by_source();
    }
}

template void typed_rows_any<false>(const RowsArgs<float>&, cudaStream_t);
template void typed_rows_any<true>(const RowsArgs<float>&, cudaStream_t);
template void typed_weight_any<float, float>(const WeightArgs<float, float>&, const WeightPlan&, cudaStream_t);
template void typed_weight_any<__nv_bfloat16, __nv_bfloat16>(const WeightArgs<__nv_bfloat16, __nv_bfloat16>&,
                                                             const WeightPlan&, cudaStream_t);
template void typed_weight_any<__half, __half>(const WeightArgs<__half, __half>&, const WeightPlan&, cudaStream_t);
template void typed_weight_any<__nv_bfloat16, float>(const WeightArgs<__nv_bfloat16, float>&, const WeightPlan&,
                                                     cudaStream_t);
template void typed_weight_any<__half, float>(const WeightArgs<__half, float>&, const WeightPlan&, cudaStream_t);

int typed_any_take_error() { return take_error(); }

}  // namespace tg

// ============================================================================
//  norm.cu -- layer norm over the columns of each row, and its backward pass.
//
//      mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) r
//      y  = h gamma + beta
//      dx = r (g - mean g - h mean(g h)),  g = gamma dy
//      dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
//  The forward pass keeps (mu, r) of each row in fp32 and, if asked, h in 8
//  bits (values.cuh); the backward pass takes x or that copy.  Both read each
//  operand once and write each result once: a row stays in the registers of
//  the TPR threads that share it (4 threads for 32 columns up to 256 for 8192,
//  512 in the gradient), so the variance is a second pass over registers, not memory.
//  Rows of at most 512 columns are bound by HBM (232,965 x 128 bf16: 20 us, its
//  bytes 18.5).  Wider ones are not: a row's threads meet at barriers for its
//  sums with few other rows on the SM (12-16 warps, issue slots 43-51 %, DRAM
//  26-28 % for 4,104 columns fp16), and rows that are not 16-byte aligned are
//  read 4 bytes at a time (twice the load requests for 4,099 columns).  Rows
//  wider than 8192 columns are walked three times by one block each (the second
//  and third walk come from L2), value by value: 8,192 x 12,000 fp16 176 us,
//  its gradient from x 336, from the copy 762.
//
//  dgamma and dbeta are sums over all rows: each thread adds up its columns
//  over the rows it walks, a block joins its row groups through shared memory
//  and writes one partial row, and a second kernel adds the blocks' partial
//  rows in a fixed order -- no atomics, the same bits every run.
// ============================================================================
#include <algorithm>

#include "values.cuh"

namespace tg {

namespace {

struct NormArgs {
    int64_t rows, cols;
    float eps;
    Range8 r8;
};

// The part of a row that one of TPR threads holds: N slots of V neighbouring
// values, 16 bytes (ALIGNED: one access, and no row ends inside a slot).  A block of 128
// columns lies in one slot of 128 / V neighbouring lanes, so its largest
// magnitude is a shuffle reduction (ROW_IS_BLOCK: the TPR lanes of a row of at
// most 128 columns, and all their slots).
template <class T, bool ALIGNED, int TPR, int VPT>
struct RowPart {
    static constexpr int V = 16 / static_cast<int>(sizeof(T));
    static constexpr int N = VPT / V;
    static constexpr bool kAligned = ALIGNED;
    static constexpr int W = TPR < 32 ? TPR : 32;
    static constexpr bool ROW_IS_BLOCK = TPR * V < kBlock8;
    static constexpr int G = ROW_IS_BLOCK ? TPR : kBlock8 / V;
    static_assert(!ROW_IS_BLOCK || TPR * VPT <= kBlock8, "a row of several slots within a block");

    int t, cols;  // thread of the row, the row's columns
    __device__ __forceinline__ RowPart(int64_t columns) : t(threadIdx.x % TPR), cols(static_cast<int>(columns)) {}
    __device__ __forceinline__ int col(int i, int j) const { return (i * TPR + t) * V + j; }
    __device__ __forceinline__ bool has(int i, int j) const { return col(i, j) < cols; }
    // Slot i exists for some thread of the warp (the same answer for all of them).
    __device__ __forceinline__ bool any(int i) const { return (i * TPR + t / W * W) * V < cols; }
    // Slot i is all there for every thread of the warp's rows (the same answer
    // for all of them: a warp does not do both the whole and the ragged form).
    __device__ __forceinline__ bool whole(int i) const { return (i * TPR + t / W * W + W) * V <= cols; }
    // How many values of slot i the row has (may be more than V, or negative).
    __device__ __forceinline__ int left(int i) const { return cols - col(i, 0); }

    // The row's slots (zeros where there is nothing; `live` false: all zeros).
    using Slot = Held<T, V, ALIGNED>;
    __device__ __forceinline__ void fetch(const T* p, bool live, Slot (&k)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (live && (ALIGNED ? has(i, 0) : whole(i))) k[i].fetch(p + col(i, 0));
            else if (!ALIGNED && live && any(i)) k[i].fetch(p + col(i, 0), left(i));
            else k[i].zero();
        }
    }
    // Slot i of row p, fetched: zeros past the row's end.
    __device__ __forceinline__ void values(const Slot& k, const T* p, int i, float (&x)[V]) const {
        if (ALIGNED || whole(i)) k.values(Slot::odd(p), x);
        else k.values(Slot::odd(p), x, left(i));
    }
    // A slot of gamma or beta.
    template <class P>
    __device__ __forceinline__ void load(const P* p, int i, float (&x)[V]) const {
        if (ALIGNED ? has(i, 0) : whole(i) && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
            if constexpr (V * sizeof(P) <= 16) {
                load_v<P, V>(p + col(i, 0), x);
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(p + col(i, j));
                    x[j] = q.x, x[j + 1] = q.y, x[j + 2] = q.z, x[j + 3] = q.w;
                }
            }
        } else if (ALIGNED) {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = 0.0f;
        } else {
            Held<P, V, false> k;
            k.fetch(p + col(i, 0), left(i));
            k.values(k.odd(p), x, left(i));
        }
    }
    __device__ __forceinline__ void store(T* p, int i, const float (&x)[V]) const {
        if constexpr (ALIGNED) {
            if (has(i, 0)) store_v<T, V>(p + col(i, 0), x);
        } else if (whole(i)) {
            store_any<T, V>(p + col(i, 0), x);
        } else {
            store_some<T, V>(p + col(i, 0), x, left(i));
        }
    }
};

// Sums of S values over the TPR threads of a row; every thread gets them.
// `red`: S floats per warp of the block (rows of several warps; the whole
// block takes part).
template <int TPR, int S>
__device__ __forceinline__ void row_sum(float (&x)[S], float* red) {
#pragma unroll
    for (int k = 0; k < S; ++k) x[k] = reduce_sum<float, (TPR < 32 ? TPR : 32)>(x[k]);
    if constexpr (TPR > 32) {
        constexpr int NW = TPR / 32;
        const int lane = threadIdx.x % 32;
        __syncthreads();  // the previous sum has been read
        if (lane < S) red[threadIdx.x / 32 * S + lane] = S == 1 || lane == 0 ? x[0] : x[S - 1];
        __syncthreads();
        // each warp adds up the row's warps, one a lane
        const float* mine = red + threadIdx.x / TPR * NW * S;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            constexpr int P = NW <= 2 ? 2 : (NW <= 4 ? 4 : (NW <= 8 ? 8 : 16));
            x[k] = reduce_sum<float, P>(lane % P < NW ? mine[lane % P * S + k] : 0.0f);
        }
    }
}

// Threads of a block: whole rows.
template <int TPR>
constexpr int block_threads() { return TPR < 128 && 128 % TPR == 0 ? 128 : TPR; }

// Blocks a SM: the kernels are compiled and launched for as many.
template <int TPR, int VPT>
constexpr int resident() { return VPT > 16 ? 512 / block_threads<TPR>() : (TPR >= 256 ? 1024 / TPR : (VPT > 8 ? 5 : 8)); }
template <int TPR, int VPT>
constexpr int resident_grad() { return TPR >= 384 ? 1 : (TPR >= 256 ? 2 : (VPT > 8 ? 4 : 5)); }

// How many of its next rows a group of threads has asked for: as many as keep
// about 16 KB of loads in flight a SM (one row at a time left HBM at 45 %).
template <class T, int TPR, int VPT>
constexpr int rows_ahead() { return TPR >= 256 ? 1 : VPT * sizeof(T) <= 16 ? 4 : (VPT * sizeof(T) <= 32 ? 2 : 1); }

// gamma and beta as they lie in memory, kept in registers where they are few.
template <class R, class T, class P>
struct Params {
    static constexpr bool kKeep = R::N * R::V * sizeof(P) <= 32;
    Raw<P, R::V> k[kKeep ? R::N : 1];
    const P* p;
    __device__ __forceinline__ Params(const R& part, const P* q) : p(q) {
        if (kKeep) {
#pragma unroll
            for (int i = 0; i < R::N; ++i)
                k[kKeep ? i : 0] = gather_raw<P, R::V>(
                    [&](int j) { return part.has(i, j) ? p[part.col(i, j)] : from_f32<P>(0.0f); });
        }
    }
    __device__ __forceinline__ void get(const R& part, int i, float (&x)[R::V]) const {
        if (kKeep) widen(k[kKeep ? i : 0], x);
        else part.load(p, i, x);
    }
};

template <class T, class P, bool ALIGNED, int TPR, int VPT>
__global__ void __launch_bounds__(block_threads<TPR>(), resident<TPR, VPT>()) norm_kernel(NormArgs a, const T* x, int64_t ldx, const P* gamma,
                                                                    const P* beta, T* y, int64_t ldy, float2* stats,
                                                                    Saved8 s) {
    using R = RowPart<T, ALIGNED, TPR, VPT>;
    constexpr int V = R::V, N = R::N, D = rows_ahead<T, TPR, VPT>();
    __shared__ float red[32];
    constexpr int RPB = block_threads<TPR>() / TPR;
    wait_for_previous();
    const R part(a.cols);
    const float inv_n = __fdiv_rn(1.0f, static_cast<float>(a.cols));
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
    const Params<R, T, P> g(part, gamma), b(part, beta);
    // every thread takes part in the reductions: the loop runs on the block's first row
    int64_t base = static_cast<int64_t>(blockIdx.x) * RPB, row = base + threadIdx.x / TPR;
    typename R::Slot ring[D][N];
#pragma unroll
    for (int d = 0; d < D; ++d) {
        const int64_t r = row + d * step;
        part.fetch(x + (r < a.rows ? r * ldx : 0), r < a.rows, ring[d]);
    }
    while (base < a.rows) {
#pragma unroll
        for (int d = 0; d < D; ++d, base += step, row += step) {
            if (base >= a.rows) break;
            const bool live = row < a.rows;
            float v[N][V];
            float sum[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
                part.values(ring[d][i], x + row * ldx, i, v[i]);
#pragma unroll
                for (int j = 0; j < V; ++j) sum[0] += v[i][j];
            }
            const int64_t next = row + D * step;
            part.fetch(x + (next < a.rows ? next * ldx : 0), next < a.rows, ring[d]);
            row_sum<TPR>(sum, red);
            const float mean = __fmul_rn(sum[0], inv_n);
            float sq[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = __fsub_rn(v[i][j], mean);
                if (!part.whole(i)) {
#pragma unroll
                    for (int j = 0; j < V; ++j) v[i][j] = part.has(i, j) ? v[i][j] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) sq[0] = fmaf(v[i][j], v[i][j], sq[0]);
            }
            row_sum<TPR>(sq, red);
            const float rstd = rsqrtf(fmaf(sq[0], inv_n, a.eps));  // 2 ulp
            if (live && part.t == 0) stats[row] = make_float2(mean, rstd);
            float row_max = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
                map_v(v[i], [rstd](float u) { return __fmul_rn(u, rstd); });
                if (R::ROW_IS_BLOCK) {
#pragma unroll
                    for (int j = 0; j < V; ++j) row_max = max_mag(row_max, v[i][j]);
                }
            }
            const int64_t at = live ? row : 0;
            T* yr = y + at * ldy;
            int8_t* codes = s.codes + at * s.ld;
            uint8_t* exps = s.exps + at * s.lde;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
                if (s.codes) {
                    float m = row_max;
                    if (!R::ROW_IS_BLOCK) {
#pragma unroll
                        for (int j = 0; j < V; ++j) m = max_mag(m, v[i][j]);
                    }
                    const int byte = exponent8(reduce_max<R::G>(m), a.r8.emin);
                    const float inv = encode8(byte);
                    if (!live) {
                    } else if (ALIGNED ? part.has(i, 0) : part.whole(i)) {
                        store_codes<V>(codes + part.col(i, 0), v[i], inv, byte, a.r8.top);
                    } else if (!ALIGNED) {
                        store_codes<V>(codes + part.col(i, 0), v[i], inv, byte, a.r8.top, part.left(i));
                    }
                    // the first lane of the group that holds the block writes its exponent
                    if (live && part.t % R::G == 0 && (i == 0 || !R::ROW_IS_BLOCK) && part.has(i, 0))
                        exps[part.col(i, 0) / kBlock8] = static_cast<uint8_t>(byte);
                }
                float w[V], c[V];
                g.get(part, i, w);
                b.get(part, i, c);
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = fmaf(v[i][j], w[j], c[j]);
                if (live) part.store(yr, i, w);
            }
        }
    }
}

// The saved copy's part of a row, and its blocks' exponents.
template <class R>
__device__ __forceinline__ void fetch_codes(const R& part, const int8_t* codes, const uint8_t* exps, bool live,
                                            Raw<int8_t, R::V> (&k)[R::N], int (&e)[R::N]) {
#pragma unroll
    for (int i = 0; i < R::N; ++i) {
        e[i] = live && part.has(i, 0) ? exps[part.col(i, 0) / kBlock8] : 127;
        if (live && (R::kAligned ? part.has(i, 0) : part.whole(i)))
            k[i] = *reinterpret_cast<const Raw<int8_t, R::V>*>(codes + part.col(i, 0));
        else k[i] = load_codes<R::V>(codes + part.col(i, 0), live && !R::kAligned ? part.left(i) : 0);
    }
}

// dx, and this block's partial sums of dgamma and dbeta: part[block][2][cols].
template <class T, class P, bool ALIGNED, int TPR, int VPT, bool SAVED>
__global__ void __launch_bounds__(block_threads<TPR>(), resident_grad<TPR, VPT>()) norm_grad_kernel(NormArgs a, const T* dy, int64_t lddy,
                                                                         const T* x, int64_t ldx, Saved8 s,
                                                                         const float2* stats, const P* gamma, T* dx,
                                                                         int64_t lddx, float* partial) {
    using R = RowPart<T, ALIGNED, TPR, VPT>;
    constexpr int V = R::V, N = R::N, RPB = block_threads<TPR>() / TPR, D = (rows_ahead<T, TPR, VPT>() + 1) / 2;
    __shared__ float red[32];
    __shared__ float join[RPB > 1 ? RPB * TPR * VPT : 1];
    wait_for_previous();
    const R part(a.cols);
    const float inv_n = __fdiv_rn(1.0f, static_cast<float>(a.cols));
    const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
    const Params<R, T, P> w8(part, gamma);
    float ag[N][V], ab[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) ag[i][j] = ab[i][j] = 0.0f;
    typename R::Slot kd[D][N], kx[SAVED ? 1 : D][N];
    Raw<int8_t, V> kc[SAVED ? D : 1][N];
    int ke[SAVED ? D : 1][N];
    float2 st[D];
    const auto fetch = [&](int d, int64_t r) {
        const bool live = r < a.rows;
        const int64_t at = live ? r : 0;
        // (of a row that is not there h is 0, not what row 0's statistics make
        // of zeros: an infinity times its zero gradient would be NaN)
        st[d] = live ? stats[at] : make_float2(0.0f, 0.0f);
        part.fetch(dy + at * lddy, live, kd[d]);
        if constexpr (SAVED) fetch_codes(part, s.codes + at * s.ld, s.exps + at * s.lde, live, kc[SAVED ? d : 0], ke[SAVED ? d : 0]);
        else part.fetch(x + at * ldx, live, kx[SAVED ? 0 : d]);
    };
    int64_t base = static_cast<int64_t>(blockIdx.x) * RPB, row = base + threadIdx.x / TPR;
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(d, row + d * step);
    while (base < a.rows) {
#pragma unroll
        for (int d = 0; d < D; ++d, base += step, row += step) {
            if (base >= a.rows) break;
            const bool live = row < a.rows;
            const float mean = st[d].x, rstd = st[d].y;
            float h[N][V], g[N][V];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
                if constexpr (SAVED) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) values4(kc[SAVED ? d : 0][i].w[j / 4], ke[SAVED ? d : 0][i], &h[i][j]);
                } else {
                    part.values(kx[SAVED ? 0 : d][i], x + row * ldx, i, h[i]);
#pragma unroll
                    for (int j = 0; j < V; ++j) h[i][j] = __fmul_rn(__fsub_rn(h[i][j], mean), rstd);
                    if (!part.whole(i)) {
#pragma unroll
                        for (int j = 0; j < V; ++j) h[i][j] = part.has(i, j) ? h[i][j] : 0.0f;
                    }
                }
                part.values(kd[d][i], dy + row * lddy, i, g[i]);
            }
            fetch(d, row + D * step);
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
                float w[V];
                w8.get(part, i, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    ag[i][j] = fmaf(g[i][j], h[i][j], ag[i][j]);
                    ab[i][j] += g[i][j];
                    g[i][j] = __fmul_rn(g[i][j], w[j]);
                    sum[0] += g[i][j];
                    sum[1] = fmaf(g[i][j], h[i][j], sum[1]);
                }
            }
            row_sum<TPR>(sum, red);
            const float m1 = __fmul_rn(sum[0], inv_n), m2 = __fmul_rn(sum[1], inv_n);
            T* out = dx + (live ? row * lddx : 0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (!part.any(i)) break;
#pragma unroll
                for (int j = 0; j < V; ++j) g[i][j] = __fmul_rn(rstd, fmaf(-h[i][j], m2, __fsub_rn(g[i][j], m1)));
                if (live) part.store(out, i, g[i]);
            }
        }
    }
    float* sums = partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (part.has(i, j)) {
                    sums[part.col(i, j)] = ag[i][j];
                    sums[a.cols + part.col(i, j)] = ab[i][j];
                }
    } else {
        // The block's row groups, joined through shared memory: value k of
        // thread t of group q at (q * VPT + k) * TPR + t.
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    join[(threadIdx.x / TPR * VPT + i * V + j) * TPR + part.t] = half ? ab[i][j] : ag[i][j];
            __syncthreads();
            for (int q = threadIdx.x; q < TPR * VPT; q += block_threads<TPR>()) {
                float sum = 0.0f;
#pragma unroll 4
                for (int r = 0; r < RPB; ++r) sum += join[r * VPT * TPR + q];
                const int t = q % TPR, i = q / TPR / V, j = q / TPR % V;
                const int c = (i * TPR + t) * V + j;
                if (c < a.cols) sums[half * a.cols + c] = sum;
            }
        }
    }
}

// Rows wider than the register forms hold: one block walks a row.
template <class T, class P>
__global__ void __launch_bounds__(512) norm_wide_kernel(NormArgs a, const T* x, int64_t ldx, const P* gamma,
                                                        const P* beta, T* y, int64_t ldy, float2* stats, Saved8 s) {
    __shared__ float red[32];
    wait_for_previous();
    const float inv_n = __fdiv_rn(1.0f, static_cast<float>(a.cols));
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* xr = x + row * ldx;
        float sum[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < a.cols; c += 512) sum[0] += to_f32(xr[c]);
        row_sum<512>(sum, red);
        const float mean = __fmul_rn(sum[0], inv_n);
        float sq[1] = {0.0f};
        for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
            const float d = __fsub_rn(to_f32(xr[c]), mean);
            sq[0] = fmaf(d, d, sq[0]);
        }
        row_sum<512>(sq, red);
        const float rstd = rsqrtf(fmaf(sq[0], inv_n, a.eps));
        if (threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
        // one warp per block of 128 columns
        for (int64_t b = warp; b * kBlock8 < a.cols; b += 16) {
            float h[4];
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t c = b * kBlock8 + j * 32 + lane;
                h[j] = c < a.cols ? __fmul_rn(__fsub_rn(to_f32(xr[c]), mean), rstd) : 0.0f;
                m = max_mag(m, h[j]);
                if (c < a.cols) y[row * ldy + c] = from_f32<T>(fmaf(h[j], to_f32(gamma[c]), to_f32(beta[c])));
            }
            if (s.codes) {
                const int byte = exponent8(reduce_max<32>(m), a.r8.emin);
                const float inv = encode8(byte);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t c = b * kBlock8 + j * 32 + lane;
                    if (c < a.cols) s.codes[row * s.ld + c] = code8(h[j], inv, byte, a.r8.top);
                }
                if (lane == 0) s.exps[row * s.lde + b] = static_cast<uint8_t>(byte);
            }
        }
    }
}

template <class T, bool SAVED>
__device__ __forceinline__ float wide_h(const T* x, int64_t ldx, const Saved8& s, float2 st, int64_t row, int64_t c) {
    if (SAVED)
        return __fmul_rn(static_cast<float>(s.codes[row * s.ld + c]), decode8(s.exps[row * s.lde + c / kBlock8]));
    return __fmul_rn(__fsub_rn(to_f32(x[row * ldx + c]), st.x), st.y);
}

template <class T, class P, bool SAVED>
__global__ void __launch_bounds__(512) norm_wide_grad_kernel(NormArgs a, const T* dy, int64_t lddy, const T* x,
                                                             int64_t ldx, Saved8 s, const float2* stats, const P* gamma,
                                                             T* dx, int64_t lddx) {
    __shared__ float red[32];
    wait_for_previous();
    const float inv_n = __fdiv_rn(1.0f, static_cast<float>(a.cols));
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float2 st = stats[row];
        float sum[2] = {0.0f, 0.0f};
        for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
            const float g = __fmul_rn(to_f32(dy[row * lddy + c]), to_f32(gamma[c]));
            sum[0] += g;
            sum[1] = fmaf(g, wide_h<T, SAVED>(x, ldx, s, st, row, c), sum[1]);
        }
        row_sum<512>(sum, red);
        const float m1 = __fmul_rn(sum[0], inv_n), m2 = __fmul_rn(sum[1], inv_n);
        for (int64_t c = threadIdx.x; c < a.cols; c += 512) {
            const float g = __fmul_rn(to_f32(dy[row * lddy + c]), to_f32(gamma[c]));
            const float h = wide_h<T, SAVED>(x, ldx, s, st, row, c);
            dx[row * lddx + c] = from_f32<T>(__fmul_rn(st.y, fmaf(-h, m2, __fsub_rn(g, m1))));
        }
    }
}

// Partial sums of dgamma and dbeta for wide rows: a thread per column, the
// rows split over blockIdx.y.
template <class T, bool SAVED>
__global__ void __launch_bounds__(256) norm_wide_sums_kernel(NormArgs a, const T* dy, int64_t lddy, const T* x,
                                                             int64_t ldx, Saved8 s, const float2* stats, float* part) {
    wait_for_previous();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= a.cols) return;
    float sg = 0.0f, sb = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = to_f32(dy[row * lddy + c]);
        sg = fmaf(g, wide_h<T, SAVED>(x, ldx, s, stats[row], row, c), sg);
        sb += g;
    }
    float* out = part + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
    out[c] = sg;
    out[a.cols + c] = sb;
}

// dgamma / dbeta = the sum of `parts` partial rows [2][cols], in their order
// within each of 32 interleaved chains, which are joined in order.
template <class P>
__global__ void __launch_bounds__(1024) norm_join_kernel(const float* part, int parts, int64_t cols, P* dgamma, P* dbeta) {
    __shared__ float sh[32][33];
    wait_for_previous();
    const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;  // of 2 * cols
    float sum = 0.0f;
    if (c < 2 * cols) {
#pragma unroll 8
        for (int p = w; p < parts; p += 32) sum += part[static_cast<int64_t>(p) * 2 * cols + c];
    }
    sh[w][lane] = sum;
    __syncthreads();
    sum = reduce_sum<float, 32>(sh[lane][w]);  // warp w: column w's 32 chains
    const int64_t d = static_cast<int64_t>(blockIdx.x) * 32 + w;
    if (lane == 0 && d < 2 * cols) {
        if (d < cols) dgamma[d] = from_f32<P>(sum);
        else dbeta[d - cols] = from_f32<P>(sum);
    }
}

constexpr int64_t kRegisterCols = 8192;

// Calls f(TPR, VPT) with the row split for `cols` columns.
template <class F>
void by_width_narrow(int64_t cols, F&& f) {
    using std::integral_constant;
    if (cols <= 32) f(integral_constant<int, 4>{}, integral_constant<int, 8>{});
    else if (cols <= 64) f(integral_constant<int, 4>{}, integral_constant<int, 16>{});
    else if (cols <= 128) f(integral_constant<int, 8>{}, integral_constant<int, 16>{});
    else if (cols <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
}

// Above 4,096 columns, where one block has an SM to itself, 384 threads as far
// as they reach: with 512 a thread has 128 registers for a row's values and its
// sums.  33.5 million values, from x / from the 8-bit copy, us by 384 and 512
// threads: fp16, 4,104 columns 68, 76 / 69, 80;  6,144: 59, 65 / 59, 67;  4,099:
// 116, 136 / 134, 142;  5,121: 109, 121 / 122, 125;  half as many in fp32, 4,104:
// 48, 62 / 46, 47;  4,099: 82, 87 / 79, 79.  (Two blocks of 320: fp16, 4,104: 87 /
// 80;  4,099: 126 / 133;  fp32, 4,099: 75 / 69.  Three of 192 for 2,049: 136 / 140
// where 256 take 122 / 128.)
template <class F>
void by_width_grad(int64_t cols, F&& f) {
    using std::integral_constant;
    if (cols <= 512) by_width_narrow(cols, f);
    else if (cols <= 64 * 16) f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
    else if (cols <= 128 * 16) f(integral_constant<int, 128>{}, integral_constant<int, 16>{});
    else if (cols <= 256 * 16) f(integral_constant<int, 256>{}, integral_constant<int, 16>{});
    else if (cols <= 384 * 16) f(integral_constant<int, 384>{}, integral_constant<int, 16>{});
    else f(integral_constant<int, 512>{}, integral_constant<int, 16>{});
}

// The forward pass holds half as much a value: twice the values a thread, half
// the warps that a row's sums have to cross.  An SM holds 512 such threads; the
// steps are the multiples of 32 threads whose blocks fill at least 15/16 of
// them (96 by five, 160 by three; not 192 and 224).  33.5 million fp16 values
// without / with the 8-bit copy, us by that step and by the next power of two:
// 2,049 columns by 96 71 / 89, by 128 98 / 124;  2,056: 33 / 48, 36 / 55;  4,099
// by 160 73 / 95, by 256 102 / 127;  4,104: 33 / 49, 38 / 57;  5,120: 29 / 42, 33 /
// 47;  5,128 by 192 36 / 55, by 224 34 / 50, by 256 34 / 49;  6,144 by 224 33 / 49,
// by 256 31 / 44.
template <class F>
void by_width_forward(int64_t cols, F&& f) {
    using std::integral_constant;
    if (cols <= 512) by_width_narrow(cols, f);
    else if (cols <= 32 * 32) f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
    else if (cols <= 64 * 32) f(integral_constant<int, 64>{}, integral_constant<int, 32>{});
    else if (cols <= 96 * 32) f(integral_constant<int, 96>{}, integral_constant<int, 32>{});
    else if (cols <= 128 * 32) f(integral_constant<int, 128>{}, integral_constant<int, 32>{});
    else if (cols <= 160 * 32) f(integral_constant<int, 160>{}, integral_constant<int, 32>{});
    else f(integral_constant<int, 256>{}, integral_constant<int, 32>{});
}

// gamma and beta are fp32 or of the rows' own type.
template <class F>
void by_types(int dtype, int param_dtype, F&& f) {
    by_dtype(dtype, [&](auto t) {
        if (param_dtype == TG_F32) f(t, float{});
        else f(t, t);
    });
}

void check_norm(const char* fn, int64_t rows, int64_t cols, int dtype, int param_dtype) {
    check_rows_cols(fn, rows, cols);
    check_dtype(fn, "x", dtype);
    if (param_dtype != TG_F32 && param_dtype != dtype)
        invalid(std::string(fn) + ": gamma and beta must be float32 or of the rows' type");
}

void check_stats(const char* fn, const float* stats) {
    if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) invalid(std::string(fn) + ": stats must be 8-byte aligned");
}

}  // namespace

}  // namespace tg

extern "C" {

TG_API tg_status tg_layer_norm(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ldx,
                               int32_t param_dtype, const void* gamma, const void* beta, float eps, void* y,
                               int64_t ldy, float* stats, int8_t* codes, int64_t ld_codes, uint8_t* exponents,
                               int64_t ld_exponents, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "layer_norm";
        check_norm(fn, rows, cols, dtype, param_dtype);
        check_ptr(fn, "x", x, rows > 0);
        check_ptr(fn, "y", y, rows > 0);
        check_ptr(fn, "stats", stats, rows > 0);
        check_ptr(fn, "gamma", gamma, true);
        check_ptr(fn, "beta", beta, true);
        check_ld(fn, "x", ldx, cols);
        check_ld(fn, "y", ldy, cols);
        if (!(eps >= 0.0f)) invalid("layer_norm: eps must not be negative");
        check_stats(fn, stats);
        const Saved8 s{codes, ld_codes, exponents, ld_exponents};
        check_saved8(fn, cols, s, false);
        const NormArgs a{rows, cols, eps, range8(dtype)};
        float2* st = reinterpret_cast<float2*>(stats);
        by_types(dtype, param_dtype, [&](auto t, auto p) {
            using T = decltype(t);
            using P = decltype(p);
            const T* xp = static_cast<const T*>(x);
            T* yp = static_cast<T*>(y);
            const P *gp = static_cast<const P*>(gamma), *bp = static_cast<const P*>(beta);
            if (cols > kRegisterCols) {
                launch_dependent("layer_norm", norm_wide_kernel<T, P>, dim3(static_cast<unsigned>(std::min<int64_t>(rows, num_sms() * 4))),
                       dim3(512), 0, as_stream(stream), a, xp, ldx, gp, bp, yp, ldy, st, s);
                return;
            }
            // (8,191 x 4,096 fp16 with the 8-bit copy: 43 us; 59 with code for
            // rows that end inside a slot, 69 where the rows are not aligned)
            const bool al = cols * sizeof(T) % 16 == 0 && rows_aligned16(x, ldx, sizeof(T)) &&
                            rows_aligned16(y, ldy, sizeof(T)) &&
                            rows_aligned16(gamma, 0, 1) && rows_aligned16(beta, 0, 1);
            by_width_forward(cols, [&](auto tpr, auto vpt) {
                constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
                const int64_t blocks = std::min<int64_t>(ceil_div(rows, block_threads<TPR>() / TPR),
                                                         int64_t(num_sms()) * resident<TPR, VPT>());
                auto kern = al ? norm_kernel<T, P, true, TPR, VPT> : norm_kernel<T, P, false, TPR, VPT>;
                launch_dependent("layer_norm", kern, dim3(static_cast<unsigned>(blocks)),
                       dim3(block_threads<TPR>()), 0, as_stream(stream), a, xp, ldx, gp, bp, yp, ldy, st, s);
            });
        });
    });
}

TG_API tg_status tg_layer_norm_grad(int64_t rows, int64_t cols, int32_t dtype, const void* dy, int64_t lddy,
                                    const void* x, int64_t ldx, const int8_t* codes, int64_t ld_codes,
                                    const uint8_t* exponents, int64_t ld_exponents, const float* stats,
                                    int32_t param_dtype, const void* gamma, void* dx, int64_t lddx, void* dgamma,
                                    void* dbeta, void* stream) {
    return tg::guard([&] {
        tg::require_device();
        using namespace tg;
        const char* fn = "layer_norm_grad";
        check_norm(fn, rows, cols, dtype, param_dtype);
        check_ptr(fn, "dy", dy, rows > 0);
        check_ptr(fn, "dx", dx, rows > 0);
        check_ptr(fn, "stats", stats, rows > 0);
        check_ptr(fn, "gamma", gamma, true);
        check_ptr(fn, "dgamma", dgamma, true);
        check_ptr(fn, "dbeta", dbeta, true);
        check_ld(fn, "dy", lddy, cols);
        check_ld(fn, "dx", lddx, cols);
        if ((x != nullptr) == (codes != nullptr) && rows > 0)
            invalid(std::string(fn) + ": exactly one of x and codes is given");
        if (x) check_ld(fn, "x", ldx, cols);
        const Saved8 s{const_cast<int8_t*>(codes), ld_codes, const_cast<uint8_t*>(exponents), ld_exponents};
        check_saved8(fn, cols, s, codes != nullptr);
        check_stats(fn, stats);
        const NormArgs a{rows, cols, 0.0f, range8(dtype)};
        const float2* st = reinterpret_cast<const float2*>(stats);
        cudaStream_t str = as_stream(stream);
        by_types(dtype, param_dtype, [&](auto t, auto p) {
            using T = decltype(t);
            using P = decltype(p);
            const T *dyp = static_cast<const T*>(dy), *xp = static_cast<const T*>(x);
            T* dxp = static_cast<T*>(dx);
            const P* gp = static_cast<const P*>(gamma);
            int64_t parts = 0;
            const auto join = [&](const float* part) {
                launch_dependent("layer_norm_join", norm_join_kernel<P>, dim3(static_cast<unsigned>(ceil_div(2 * cols, 32))),
                       dim3(1024), 0, str, part, static_cast<int>(parts), cols, static_cast<P*>(dgamma),
                       static_cast<P*>(dbeta));
            };
            if (cols > kRegisterCols) {
                parts = std::min<int64_t>(std::max<int64_t>(ceil_div(rows, 16), 0), 64);
                Scratch<float> part(static_cast<size_t>(parts * 2 * cols), str);
                auto kern = codes ? norm_wide_grad_kernel<T, P, true> : norm_wide_grad_kernel<T, P, false>;
                launch_dependent("layer_norm_grad", kern, dim3(static_cast<unsigned>(std::min<int64_t>(rows, num_sms() * 4))),
                       dim3(512), 0, str, a, dyp, lddy, xp, ldx, s, st, gp, dxp, lddx);
                auto sums = codes ? norm_wide_sums_kernel<T, true> : norm_wide_sums_kernel<T, false>;
                launch_dependent("layer_norm_sums", sums,
                       dim3(static_cast<unsigned>(ceil_div(cols, 256)), static_cast<unsigned>(parts)), dim3(256), 0,
                       str, a, dyp, lddy, xp, ldx, s, st, part.p);
                join(part.p);
                return;
            }
            const bool al = cols * sizeof(T) % 16 == 0 && rows_aligned16(dy, lddy, sizeof(T)) &&
                            (codes || rows_aligned16(x, ldx, sizeof(T))) &&
                            rows_aligned16(dx, lddx, sizeof(T)) && rows_aligned16(gamma, 0, 1);
            by_width_grad(cols, [&](auto tpr, auto vpt) {
                constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
                constexpr int BT = block_threads<TPR>(), RPB = BT / TPR;
                auto kern = codes ? (al ? norm_grad_kernel<T, P, true, TPR, VPT, true>
                                        : norm_grad_kernel<T, P, false, TPR, VPT, true>)
                                  : (al ? norm_grad_kernel<T, P, true, TPR, VPT, false>
                                        : norm_grad_kernel<T, P, false, TPR, VPT, false>);
                parts = std::min<int64_t>(ceil_div(rows, RPB), int64_t(num_sms()) * resident_grad<TPR, VPT>());
                Scratch<float> part(static_cast<size_t>(parts * 2 * cols), str);
                launch_dependent("layer_norm_grad", kern, dim3(static_cast<unsigned>(parts)), dim3(BT), 0, str, a, dyp, lddy, xp,
                       ldx, s, st, gp, dxp, lddx, part.p);
                join(part.p);
            });
        });
    });
}

}  // extern "C"

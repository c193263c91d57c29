// ============================================================================
//  typed_mma.cuh -- what the typed products' tensor-core kernels share: the
//  shared-memory plan, set-up and tear-down, the MMAs of a stage, output
//  stores and the epilogue of the rows products.
// ============================================================================
#pragma once

#include <algorithm>

#include "tcgen05.cuh"
#include "typed.cuh"

namespace tg {
namespace typed {

constexpr int BM = 128;

// The error word of the including file's kernels: the first timeout code seen
// (0 = none).
namespace {
__device__ int g_error = 0;
}

// Ring of stages (1024-byte aligned): PA planes of the A tile, PB of the B tile.
template <int PA, int PB, int BN>
struct Plan {
    static constexpr uint32_t kA = BM * 128, kB = BN * 128;  // one plane's tile
    static constexpr uint32_t kStage = PA * kA + PB * kB;
    static constexpr int kStages = (192 * 1024) / kStage > 8 ? 8 : (192 * 1024) / kStage;
    static constexpr uint32_t kBytes = kStages * kStage + 1024;
    static_assert(kStages >= 2, "two stages");
};

struct Shared {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int prefix[kMaxTypes + 1];
    uint32_t order[kMaxTypes];  // weight gradients only
};

// TMEM columns: two buffers of an accumulator (SPLIT: of two, see stage_mmas).
template <int BN, bool SPLIT = false>
constexpr uint32_t tmem_cols() { return 2 * BN * (SPLIT ? 2 : 1); }

// Barriers, TMEM (warp 2) and the plan of the work (warp 3: plan(), over the
// types' offsets); every thread returns with them in place.
template <int STAGES, int BN, bool SPLIT = false, class F>
__device__ __forceinline__ uint32_t set_up(Shared& s, int full_arrivals, int acc_arrivals, F&& plan) {
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mb::init(&s.full[i], full_arrivals);
            mb::init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mb::init(&s.acc_full[i], 1);
            mb::init(&s.acc_empty[i], acc_arrivals);
        }
        mb::init(&s.drain, 1);
        mb::fence_init();
    }
    if (warp == 2) tc::alloc(&s.tmem, tmem_cols<BN, SPLIT>());
    wait_for_previous();
    if (warp == 3) plan();
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    return s.tmem;
}

// Every copy has landed; once every MMA of the issuing warp has retired, TMEM
// goes back.
template <int BN, bool SPLIT = false>
__device__ __forceinline__ void tear_down(Shared& s, uint32_t tmem, int mma_warp) {
    tc::fence_before();
    __syncthreads();
    const int warp = threadIdx.x >> 5;
    if (warp == mma_warp && (threadIdx.x & 31) == 0) {
        tc::commit(&s.drain);
        mb::wait(&s.drain, 0, &g_error, 26);
    }
    __syncthreads();
    tc::fence_after();
    if (warp == 2) tc::dealloc(tmem, tmem_cols<BN, SPLIT>());
}

// One warp: rows [valid, 64) of the 64-row chunks in `bytes` of shared memory
// become zero, and the tensor cores see it.
__device__ __forceinline__ void zero_rows(uint32_t base, uint32_t bytes, int valid) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t chunk = 0; chunk < bytes; chunk += tc::kChunkBytes)
        for (uint32_t o = valid * 128 + lane * 16; o < tc::kChunkBytes; o += 512)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + chunk + o), "r"(0u) : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// The MMAs of one stage: every plane product i + j <= 2.  An MMA truncates as
// it adds to the accumulator: about 2^-25 of it is lost each time, always
// towards zero.  So with several planes the products x_0 y_0 have an
// accumulator of their own and all the small ones another (BN columns on),
// where the same loss is 2^-8 as large; one accumulator for all six was ten
// times less exact (4e-6 of the result for 602 inner indexes).
template <int PA, int PB, int BN, bool A_OUTER, bool B_OUTER>
__device__ __forceinline__ void stage_mmas(uint32_t stage, uint32_t acc, uint32_t id, bool first) {
    using S = Plan<PA, PB, BN>;
    bool add = !first;
#pragma unroll
    for (int order = PA + PB - 2 < 2 ? PA + PB - 2 : 2; order >= 0; --order) {
        if (order == 0) add = !first;
#pragma unroll
        for (int i = PA - 1; i >= 0; --i) {
            const int j = order - i;
            if (j < 0 || j >= PB) continue;
            const uint32_t a = stage + i * S::kA, b = stage + PA * S::kA + j * S::kB;
#pragma unroll
            for (int s = 0; s < tc::kInner / 16; ++s) {
                tc::mma(acc + (order > 0 ? BN : 0), A_OUTER ? tc::desc_outer(a, s) : tc::desc_inner(a, s),
                        B_OUTER ? tc::desc_outer(b, s) : tc::desc_inner(b, s), id, add);
                add = true;
            }
        }
    }
}

// 32 columns of an accumulator (SPLIT: of the two).
template <int BN, bool SPLIT>
__device__ __forceinline__ void load_acc(uint32_t addr, float (&v)[32]) {
    tc::load32(addr, v);
    if constexpr (SPLIT) {
        float u[32];
        tc::load32(addr + BN, u);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], u[j]);
    }
}

// How an output's rows are aligned: 2 = 32 bytes, 1 = 16 bytes, 0 = neither
// (-1, for store_rows: neither, and there is no buffer to stage them in).
inline int store_mode(const void* p, int64_t row_bytes, int64_t matrix_bytes = 0) {
    const uint64_t b = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(row_bytes) |
                       static_cast<uint64_t>(matrix_bytes);
    return b % 32 == 0 ? 2 : (b % 16 == 0 ? 1 : 0);
}

// Bytes of a warp's staging buffer for outputs whose rows are not aligned: 32
// rows of 32 values, rows an odd number of words apart.
template <class O>
constexpr int stage_row() { return sizeof(O) == 4 ? 33 : 34; }
template <class O>
constexpr int stage_bytes() { return 32 * stage_row<O>() * static_cast<int>(sizeof(O)); }

// A warp's 32 rows x 32 columns: lane l holds row l of `v`; rows [0, rows) and
// columns [0, left) are stored at p + row * ld + column.  Aligned rows: each
// lane stores its own, 32 bytes (whole sectors) or 16 at a time.  Others:
// through `buf`, so that a warp's store covers 32 neighbouring columns of one
// row (lane-per-row stores would send one sector for every 2 or 4 bytes).
// add (fp32 only): on top of what this warp stored there before.
template <class O>
__device__ __forceinline__ void store_rows(O* p, int64_t ld, int rows, int64_t left, float (&v)[32], int mode, O* buf,
                                           bool add = false) {
    constexpr int W = 32 / sizeof(O);  // values per 32 bytes
    const int lane = threadIdx.x & 31;
    if (mode != 0) {
        if (lane >= rows) return;
        p += lane * ld;
        if constexpr (sizeof(O) == 4) {
            if (add) {
#pragma unroll
                for (int c = 0; c < 32; c += 4) {
                    if (mode > 0 && c + 4 <= left) {
                        const float4 q = *reinterpret_cast<const float4*>(p + c);
                        v[c] += q.x, v[c + 1] += q.y, v[c + 2] += q.z, v[c + 3] += q.w;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + j < left) v[c + j] += p[c + j];
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 32; c += W) {
            if (mode > 0 && c + W <= left) {
                Raw<O, W> k;
                narrow(v + c, k);
                const uint32_t* r = k.w;
                if (mode == 2) {
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + c), "r"(r[0]),
                                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                                 : "memory");
                } else {
                    uint4* q = reinterpret_cast<uint4*>(p + c);
                    q[0] = make_uint4(r[0], r[1], r[2], r[3]);
                    q[1] = make_uint4(r[4], r[5], r[6], r[7]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (c + j < left) p[c + j] = from_f32<O>(v[c + j]);
            }
        }
        return;
    }
    constexpr int S = stage_row<O>();
    __syncwarp();  // the previous chunk has been read
#pragma unroll
    for (int j = 0; j < 32; ++j) buf[lane * S + j] = from_f32<O>(v[j]);
    __syncwarp();
    if (lane < left) {
        if constexpr (sizeof(O) == 4) {
            if (add) {
#pragma unroll 8
                for (int r = 0; r < rows; ++r) p[r * ld + lane] += buf[r * S + lane];
                return;
            }
        }
#pragma unroll 8
        for (int r = 0; r < rows; ++r) p[r * ld + lane] = buf[r * S + lane];
    }
}

// dW of the types without rows is zero: every CTA's threads (id < n) write
// their share of all of them.
template <class O>
__device__ __forceinline__ void zero_empty_types(const int32_t* offsets, int types, int64_t M, int64_t K, int64_t N,
                                                 O* dW, int64_t ld, int64_t stride, int mode, int id, int n) {
    for (int t = 0; t < types; ++t) {
        if (rows_of(offsets, t, M) > 0) continue;
        for (int64_t k = blockIdx.x; k < K; k += gridDim.x) {
            O* row = dW + t * stride + k * ld;
            constexpr int W = 16 / static_cast<int>(sizeof(O));
            int64_t c = 0;
            if (mode > 0) {
                c = N / W * W;
                for (int64_t i = id * W; i < c; i += n * W) *reinterpret_cast<uint4*>(row + i) = make_uint4(0, 0, 0, 0);
            }
            for (int64_t i = c + id; i < N; i += n) row[i] = from_f32<O>(0.0f);
        }
    }
}

// ── epilogue of the rows products ────────────────────────────────────────
template <class O>
struct RowsOut {
    int64_t N;
    const float* bias;
    int act;
    float alpha;
    O* C;
    int64_t ldc;
    int mode;
    Saved8 saved;
    Range8 r8;
};

// 32 accumulator columns from n, and what `before` (this lane's row of C, if
// not null) holds of the sum so far; bias added; columns past N are zero.
template <class O, int BN, bool SPLIT>
__device__ __forceinline__ void load_biased(uint32_t addr, const RowsOut<O>& g, int type, int64_t n, const O* before,
                                            float (&v)[32]) {
    load_acc<BN, SPLIT>(addr, v);
    if constexpr (SPLIT) {
        if (before) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (n + j < g.N) v[j] = __fadd_rn(v[j], before[n + j]);
        }
    }
    if (!g.bias) return;
    const float* b = g.bias + type * g.N + n;
    if (n + 32 <= g.N && g.N % 4 == 0 && reinterpret_cast<uintptr_t>(g.bias) % 16 == 0) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(b + j));
            v[j] = __fadd_rn(v[j], q.x);
            v[j + 1] = __fadd_rn(v[j + 1], q.y);
            v[j + 2] = __fadd_rn(v[j + 2], q.z);
            v[j + 3] = __fadd_rn(v[j + 3], q.w);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (n + j < g.N) v[j] = __fadd_rn(v[j], __ldg(b + j));
    }
}

// Asks for a tile's bias while its products are still being summed (a warp).
template <class O, int BN>
__device__ __forceinline__ void prefetch_bias(const RowsOut<O>& g, int type, int64_t n0) {
    const int64_t n = n0 + (threadIdx.x & 31) * 32;
    if (g.bias && n < n0 + BN && n < g.N)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(g.bias + type * g.N + n));
}

// One warp's 32 rows (row0 .. row0 + rows) and BN columns (from n0) of a tile.
// FAST: act_forward's.  SPLIT (fp32): the accumulators hold part of the inner
// indexes; parts but the last (`last` false) only add to C, and `first` tells
// that C holds nothing yet.
template <class O, int BN, bool FAST, bool SPLIT = false>
__device__ __forceinline__ void finish_rows(uint32_t addr, const RowsOut<O>& g, int type, int64_t row0, int rows,
                                            int64_t n0, O* buf, bool first = true, bool last = true) {
    const int lane = threadIdx.x & 31;
    const bool live = lane < rows;
    const int64_t row = live ? row0 + lane : 0;
    if constexpr (SPLIT) {
        if (!last) {
#pragma unroll 1
            for (int c0 = 0; c0 < BN && n0 + c0 < g.N; c0 += 32) {
                float v[32];
                load_acc<BN, SPLIT>(addr + c0, v);
                store_rows(g.C + row0 * g.ldc + n0 + c0, g.ldc, rows, g.N - n0 - c0, v, g.mode, buf, !first);
            }
            return;
        }
        __syncwarp();  // C's rows may have been stored by other lanes
    }
    const O* before = SPLIT && !first && live ? g.C + row * g.ldc : nullptr;
    constexpr int W = BN < kBlock8 ? BN : kBlock8;
#pragma unroll 1
    for (int b0 = 0; b0 < BN && n0 + b0 < g.N; b0 += kBlock8) {
        int byte = 0;
        float inv = 0.0f;
        // An exponent's 128 columns may lie in two tiles of 64: then N <= 64
        // and there is one tile (the callers see to it).
        if (g.saved.codes) {  // the block's exponent needs all its columns first
            float m = 0.0f;
#pragma unroll 1
            for (int c0 = b0; c0 < b0 + W; c0 += 32) {
                float v[32];
                load_biased<O, BN, SPLIT>(addr + c0, g, type, n0 + c0, before, v);
#pragma unroll
                for (int j = 0; j < 32; ++j) m = max_mag(m, v[j]);
            }
            byte = exponent8(m, g.r8.emin);
            inv = encode8(byte);
            if (live) g.saved.exps[row * g.saved.lde + (n0 + b0) / kBlock8] = static_cast<uint8_t>(byte);
        }
#pragma unroll 1
        for (int c0 = b0; c0 < b0 + W; c0 += 32) {
            const int64_t left = g.N - n0 - c0;
            if (left <= 0) break;
            float v[32];
            load_biased<O, BN, SPLIT>(addr + c0, g, type, n0 + c0, before, v);
            if (g.saved.codes && live) {
                int8_t* o = g.saved.codes + row * g.saved.ld + n0 + c0;
#pragma unroll
                for (int h = 0; h < 32; h += 16) {
                    if (h + 16 <= left) {
                        store_codes<16>(o + h, v + h, inv, byte, g.r8.top);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (h + j < left) o[h + j] = code8(v[h + j], inv, byte, g.r8.top);
                    }
                }
            }
            act_forward<FAST>(v, g.act, g.alpha);
            store_rows(g.C + row0 * g.ldc + n0 + c0, g.ldc, rows, left, v, g.mode, buf);
        }
    }
}

template <class T> struct Half { using type = T; static constexpr int planes = 1; };
template <> struct Half<float> { using type = __nv_bfloat16; static constexpr int planes = 3; };
template <class H>
constexpr bool is_bf16() { return std::is_same<H, __nv_bfloat16>::value; }

// Boxes of 64 columns x box_rows rows of a batch of matrices.
template <class T>
CUtensorMap tma_map(const TmaMatrix<T>& m, int64_t batch, int64_t rows, int64_t cols, int box_rows) {
    const int64_t dims[3] = {cols, rows, batch}, strides[2] = {m.ld, m.stride};
    const int box[3] = {64, box_rows, 1};
    return tc::map16<3>(m.p, is_bf16<T>(), dims, strides, box);
}

// ── operands ─────────────────────────────────────────────────────────────
// Whether the kernels read a batch of matrices where they lie: rows and
// matrices 16-byte aligned, and no row that ends inside 16 bytes (fp32 rows
// for the loaders may be aligned to, and end at, two values).
template <class T>
bool in_place(int64_t batch, int64_t cols, const T* p, int64_t ld, int64_t stride, int64_t bytes = 16) {
    const uint64_t b = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(ld * sizeof(T)) |
                       static_cast<uint64_t>(cols * sizeof(T)) |
                       (batch > 1 ? static_cast<uint64_t>(stride * sizeof(T)) : 0);
    return b % bytes == 0;
}

// A copy with 16-byte aligned rows (zeros to their end) of a batch of matrices
// whose row r lies at (r / inner) * stride + (r % inner) * lds.  A warp a row.
template <class T>
__global__ void __launch_bounds__(256) align_kernel(int64_t rows, int64_t cols, const T* src, int64_t inner,
                                                    int64_t stride, int64_t lds, T* dst, int64_t ld) {
    constexpr int V = 16 / static_cast<int>(sizeof(T)), U = 4;
    wait_for_previous();
    const int lane = threadIdx.x % 32;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; r < rows; r += warps) {
        const T* p = src + r / inner * stride + r % inner * lds;
        const bool odd = Held<T, V, false>::odd(p);
        for (int64_t c0 = lane * V; c0 < ld; c0 += U * 32 * V) {
            Held<T, V, false> h[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + u * 32 * V;
                if (c + V <= cols) h[u].fetch(p + c);
                else h[u].fetch(p + c, c < cols ? static_cast<int>(cols - c) : 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + u * 32 * V;
                if (c >= ld) break;
                float x[V];
                h[u].values(odd, x, c < cols ? static_cast<int>(cols - c < V ? cols - c : V) : 0);
                store_v<T, V>(dst + r * ld + c, x);
            }
        }
    }
}

// A matrix (or a batch) in place, or an aligned copy of it in scratch.
template <class T>
struct Operand {
    const T* p = nullptr;
    int64_t ld = 0, stride = 0;  // elements
    T* own = nullptr;
    cudaStream_t s = nullptr;

    // least: the alignment in bytes that the kernel can do with.
    Operand(int64_t batch, int64_t rows, int64_t cols, const T* src, int64_t lds, int64_t src_stride, cudaStream_t st,
            int64_t least = 16)
        : s(st) {
        take(batch, rows, cols, src, lds, src_stride, least);
    }
    // A matrix given as it is or in 8 bits.
    Operand(int64_t rows, int64_t cols, const T* src, int64_t lds, const Saved8& saved, cudaStream_t st) : s(st) {
        if (!saved.codes) {
            take(1, rows, cols, src, lds, 0, 16);
            return;
        }
        make(1, rows, cols);
        restore8<T>(rows, cols, saved, own, ld, s);
    }
    ~Operand() {
        if (own) scratch_free(own, s);
    }
    Operand(const Operand&) = delete;
    Operand& operator=(const Operand&) = delete;
    TmaMatrix<T> matrix() const { return {p, ld, stride}; }

  private:
    void make(int64_t batch, int64_t rows, int64_t cols) {
        constexpr int64_t V = 16 / sizeof(T);
        ld = (cols + V - 1) / V * V;
        stride = rows * ld;
        own = static_cast<T*>(scratch_alloc(static_cast<size_t>(batch * stride) * sizeof(T), s));
        p = own;
    }
    void take(int64_t batch, int64_t rows, int64_t cols, const T* src, int64_t lds, int64_t src_stride, int64_t least) {
        // (TMA zero-fills past a row's end itself)
        const bool there = sizeof(T) == 2 ? rows_aligned16(src, lds, 2) && (batch == 1 || src_stride % 8 == 0)
                                          : in_place(batch, cols, src, lds, src_stride, least);
        if (there) {
            p = src;
            ld = lds;
            stride = batch == 1 ? rows * lds : src_stride;
            return;
        }
        make(batch, rows, cols);
        launch_dependent("typed_align", align_kernel<T>,
                         dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(batch * rows, 8), num_sms() * 8))),
                         dim3(256), 0, s, batch * rows, cols, src, rows, src_stride, lds, own, ld);
    }
};

// Reads and clears the error word (the stream is idle).
static int take_error() {
    int h = 0;
    TG_CUDA(cudaMemcpyFromSymbol(&h, g_error, sizeof(int)));
    if (h) {
        const int zero = 0;
        TG_CUDA(cudaMemcpyToSymbol(g_error, &zero, sizeof(int)));
    }
    return h;
}

// Tile width of a product with N columns and `pieces` row tiles (or dW tiles):
// the widest (it reads the rows fewest times) that still gives four of five
// SMs a tile, else the narrowest.  Forward, 4 types, us for widths 64 / 128 /
// 256 (tiles): bf16, K = N = 512: 4,096 rows 14.3 (288), 12.3 (144), 14.4 (72);
// 8,192 rows 18.4, 16.4 (272), 14.3 (136); fp32: 2,048 rows 22.5 (160), 26.6
// (80); 4,096 rows 34.8, 28.6 (144).  An exponent of a saved result needs its
// 128 columns in one tile.
inline int tile_width(int64_t pieces, int64_t N, int widest, bool saved) {
    const int least = saved && N > 64 ? 128 : 64;
    for (int w = widest; w > least; w /= 2)
        if (N > w / 2 && 5 * pieces * ceil_div(N, w) >= 4 * num_sms()) return w;
    return least;
}

// A persistent grid of at most one CTA per SM.
template <class K, class... A>
void run(const char* name, K kern, int threads, uint32_t smem, int64_t items, cudaStream_t s, A... args) {
    TG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    launch_dependent(name, kern, dim3(static_cast<unsigned>(std::min<int64_t>(items, num_sms()))), dim3(threads), smem, s,
           args...);
}

}  // namespace typed
}  // namespace tg

// ============================================================================
//  typed_tc.cu -- the typed linear map's products on the tensor cores.
//
//  rows kernel    C[r] = act(A[r] . B[t(r)] + bias[t(r)]): the forward pass
//                 (B = W[t], its columns contiguous) and the input gradient
//                 (B = W[t]^T).
//  weight kernel  dW[t] = sum over the type's rows of X[r]^T dY[r]; both
//                 operands have their outer index contiguous.
//
//  Operands are 16-bit.  bf16 and fp16 matrices are read where they lie when
//  their rows start 16-byte aligned (TMA's rule), from an aligned copy
//  otherwise.  An fp32 matrix is split into three bf16 planes,
//      x = x0 + x1 + x2,   x0 = bf16(x), x1 = bf16(x - x0), x2 = bf16(x - x0 - x1),
//  which holds its 24 bits exactly, and a product takes the six plane products
//  x_i y_j with i + j <= 2 (the others are below 2^-24 of it), smallest first.
//  A matrix saved in 8 bits is one bf16 (or fp16) plane, exactly.
//
//  Both kernels are persistent: CTAs walk tiles blockIdx.x, + gridDim.x, ...
//    warp 0       TMA loads into a ring of stages (64 inner indexes each);
//    warp 1       the MMAs (one thread), into one of two TMEM accumulators;
//    warp 2       TMEM allocation;
//    warps 4-11   the epilogue: warps 4-7 empty accumulator 0, warps 8-11
//                 accumulator 1, each while the next tile is multiplied.
//  The tiles come from the types' offsets, which stay on the device: each CTA
//  scans the types' tile counts into shared memory and finds a tile's type by
//  bisection.  Rows past a type's end that a tile reads are another type's:
//  the rows kernel computes and drops them, the weight kernel, where they
//  would enter the sum, zeroes them in shared memory before the MMA.
//  Every wait is bounded; one that runs out records a code in a device error
//  word (tg_take_device_error), and the CTA drains its copies and returns.
// ============================================================================
#include <algorithm>

#include "tcgen05.cuh"
#include "typed.cuh"

namespace tg {

namespace {

__device__ int g_typed_error = 0;  // first timeout code seen (0 = none)

constexpr int BM = 128;
constexpr int kThreads = 384;

// Shared-memory plan: ring of stages (1024-byte aligned), then the rest.
template <int PA, int PB, int BN>
struct Plan {
    static constexpr uint32_t kA = BM * 128, kB = BN * 128;  // one plane's tile
    static constexpr uint32_t kStage = PA * kA + PB * kB;
    static constexpr int kStages = (200 * 1024) / kStage > 8 ? 8 : (200 * 1024) / kStage;
    static constexpr uint32_t kBytes = kStages * kStage + 1024;
    static_assert(kStages >= 2, "two stages");
};

struct Shared {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int prefix[kMaxTypes + 1];
};

// The MMAs of one stage: every plane product i + j <= 2, smallest first.
template <int PA, int PB, int BN, bool A_OUTER, bool B_OUTER>
__device__ __forceinline__ void stage_mmas(uint32_t stage, uint32_t acc, uint32_t id, bool first) {
    using S = Plan<PA, PB, BN>;
    bool add = !first;
#pragma unroll
    for (int order = PA + PB - 2 < 2 ? PA + PB - 2 : 2; order >= 0; --order)
#pragma unroll
        for (int i = PA - 1; i >= 0; --i) {
            const int j = order - i;
            if (j < 0 || j >= PB) continue;
            const uint32_t a = stage + i * S::kA, b = stage + PA * S::kA + j * S::kB;
#pragma unroll
            for (int s = 0; s < tc::kInner / 16; ++s) {
                tc::mma(acc, A_OUTER ? tc::desc_outer(a, s) : tc::desc_inner(a, s),
                        B_OUTER ? tc::desc_outer(b, s) : tc::desc_inner(b, s), id, add);
                add = true;
            }
        }
}

// 32 consecutive columns of one row, of which `left` exist.  mode: 2 = every
// row 32-byte aligned, 1 = 16-byte, 0 = neither.
template <class O>
__device__ __forceinline__ void store32(O* p, const float (&v)[32], int64_t left, int mode) {
    constexpr int W = 32 / sizeof(O);  // values per 32 bytes
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
}

template <class O>
int store_mode(const O* p, int64_t ld) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(ld * sizeof(O));
    return bits % 32 == 0 ? 2 : (bits % 16 == 0 ? 1 : 0);
}

template <int BN>
constexpr uint32_t tmem_cols() { return 2 * BN < 64 ? 64 : 2 * BN; }

// Barriers, TMEM and the scan; every thread returns with them in place.
template <int STAGES, int BN>
__device__ __forceinline__ uint32_t set_up(Shared& s, const int32_t* offsets, int types, int64_t M, int64_t per) {
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mb::init(&s.full[i], 1);
            mb::init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mb::init(&s.acc_full[i], 1);
            mb::init(&s.acc_empty[i], 128);
        }
        mb::init(&s.drain, 1);
        mb::fence_init();
    }
    if (warp == 2) tc::alloc(&s.tmem, tmem_cols<BN>());
    if (warp == 3) scan_types(offsets, types, M, per, s.prefix);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    return s.tmem;
}

// Every MMA has retired and every copy has landed: TMEM goes back.
template <int BN>
__device__ __forceinline__ void tear_down(Shared& s, uint32_t tmem) {
    tc::fence_before();
    __syncthreads();
    const int warp = threadIdx.x >> 5;
    if (warp == 1 && (threadIdx.x & 31) == 0) {
        tc::commit(&s.drain);
        mb::wait(&s.drain, 0, &g_typed_error, 26);
    }
    __syncthreads();
    tc::fence_after();
    if (warp == 2) tc::dealloc(tmem, tmem_cols<BN>());
}

// ── rows kernel ──────────────────────────────────────────────────────────
template <class O>
struct RowsTc {
    int64_t M, K, N;
    int types, tiles_n;
    const int32_t* offsets;
    const float* bias;
    int act;
    float alpha;
    O* C;
    int64_t ldc;
    int mode;
    Saved8 saved;
    Range8 r8;
};

// 32 accumulator columns from n (bias added; columns past N are zero).
template <class O>
__device__ __forceinline__ void load_biased(uint32_t addr, const RowsTc<O>& g, int type, int64_t n, float (&v)[32]) {
    tc::load32(addr, v);
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

template <class O, int P, int BN, bool TRANS, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) typed_rows_tc_kernel(const __grid_constant__ CUtensorMap ma,
                                                                    const __grid_constant__ CUtensorMap mw,
                                                                    const RowsTc<O> g) {
    using S = Plan<P, P, BN>;
    constexpr int STAGES = S::kStages;
    constexpr uint32_t ID = tc::idesc(BF16, false, !TRANS, BM, BN);
    extern __shared__ uint8_t raw[];
    __shared__ Shared s;
    const uint32_t ring = (mb::smem_u32(raw) + 1023) & ~1023u;
    const uint32_t tmem = set_up<STAGES, BN>(s, g.offsets, g.types, g.M, BM);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tiles = static_cast<int64_t>(s.prefix[g.types]) * g.tiles_n;
    const int KB = static_cast<int>((g.K + tc::kInner - 1) / tc::kInner);

    if (warp == 0) {
        if (lane == 0) {
            int64_t i = 0;
            bool ok = true;
            for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int p = static_cast<int>(tile / g.tiles_n), n0 = static_cast<int>(tile % g.tiles_n) * BN;
                const int t = find_type(s.prefix, g.types, p);
                const int row0 = clamp_row(g.offsets[t], g.M) + (p - s.prefix[t]) * BM;
                for (int kb = 0; kb < KB; ++kb, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (i >= STAGES && !(ok = mb::wait(&s.empty[st], (i / STAGES - 1) & 1, &g_typed_error, 21))) break;
                    const uint32_t a = ring + st * S::kStage, b = a + P * S::kA;
                    mb::arrive_expect_tx(&s.full[st], S::kStage);
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        tc::tma3(a + q * S::kA, &ma, kb * tc::kInner, row0, q, &s.full[st]);
                        if (TRANS) {
                            tc::tma4(b + q * S::kB, &mw, kb * tc::kInner, n0, t, q, &s.full[st]);
                        } else {
#pragma unroll
                            for (int c = 0; c < BN / 64; ++c)
                                tc::tma4(b + q * S::kB + c * tc::kChunkBytes, &mw, n0 + c * 64, kb * tc::kInner, t, q,
                                         &s.full[st]);
                        }
                    }
                }
            }
            // Every copy issued must have landed before the CTA may exit.
            for (int64_t j = i > STAGES ? i - STAGES : 0; j < i; ++j)
                mb::wait(&s.full[j % STAGES], (j / STAGES) & 1, &g_typed_error, 22);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int64_t i = 0;
            int local = 0;
            bool ok = true;
            for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++local) {
                const int acc = local & 1;
                if (local >= 2 && !(ok = mb::wait(&s.acc_empty[acc], (local / 2 - 1) & 1, &g_typed_error, 23))) break;
                tc::fence_after();
                for (int kb = 0; kb < KB; ++kb, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (!(ok = mb::wait(&s.full[st], (i / STAGES) & 1, &g_typed_error, 24))) break;
                    tc::fence_after();
                    stage_mmas<P, P, BN, false, !TRANS>(ring + st * S::kStage, tmem + acc * BN, ID, kb == 0);
                    tc::commit(&s.empty[st]);
                }
                if (ok) tc::commit(&s.acc_full[acc]);
            }
        }
    } else if (warp >= 4) {
        const int acc = (warp - 4) >> 2, q = warp & 3;
        int local = acc;
        for (int64_t tile = blockIdx.x + acc * static_cast<int64_t>(gridDim.x); tile < tiles;
             tile += 2 * static_cast<int64_t>(gridDim.x), local += 2) {
            const int p = static_cast<int>(tile / g.tiles_n);
            const int64_t n0 = tile % g.tiles_n * BN;
            const int t = find_type(s.prefix, g.types, p);
            const int64_t row = clamp_row(g.offsets[t], g.M) + static_cast<int64_t>(p - s.prefix[t]) * BM + q * 32 + lane;
            const bool live = row < clamp_row(g.offsets[t + 1], g.M);
            if (!mb::wait(&s.acc_full[acc], (local / 2) & 1, &g_typed_error, 25)) break;
            tc::fence_after();
            const uint32_t addr = tmem + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
            O* c = g.C + (live ? row * g.ldc : 0) + n0;
#pragma unroll 1
            for (int b0 = 0; b0 < BN && n0 + b0 < g.N; b0 += kBlock8) {
                constexpr int W = BN < kBlock8 ? BN : kBlock8;
                int byte = 0;
                float inv = 0.0f;
                if (g.saved.codes) {  // the block's exponent needs all its columns first
                    float m = 0.0f;
#pragma unroll 1
                    for (int c0 = b0; c0 < b0 + W; c0 += 32) {
                        float v[32];
                        load_biased(addr + c0, g, t, n0 + c0, v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) m = max_mag(m, v[j]);
                    }
                    byte = exponent8(m, g.r8.emin);
                    inv = encode8(byte);
                    if (live) g.saved.exps[row * g.saved.lde + (n0 + b0) / kBlock8] = static_cast<uint8_t>(byte);
                }
#pragma unroll 1
                for (int c0 = b0; c0 < b0 + W; c0 += 32) {
                    float v[32];
                    load_biased(addr + c0, g, t, n0 + c0, v);
                    const int64_t left = live ? g.N - n0 - c0 : 0;
                    if (g.saved.codes && left > 0) {
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
                    act_forward<(P == 1)>(v, g.act, g.alpha);
                    store32(c + c0, v, left, g.mode);
                }
            }
            tc::fence_before();
            mb::arrive(&s.acc_empty[acc]);
        }
    }
    tear_down<BN>(s, tmem);
}

// ── weight kernel ────────────────────────────────────────────────────────
template <class O>
struct WeightTc {
    int64_t M, K, N;
    int types, tiles_k, tiles_n;
    const int32_t* offsets;
    int64_t piece;  // rows of a type that one sum takes
    O* dW;
    int64_t lddw, stride_dw;
    int mode;
    float* part;  // sums of types with several pieces: [piece][K][ldp]
    int64_t ldp;
};

template <class O, int PA, int PB, int BN, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) typed_weight_tc_kernel(const __grid_constant__ CUtensorMap mx,
                                                                      const __grid_constant__ CUtensorMap my,
                                                                      const WeightTc<O> g) {
    using S = Plan<PA, PB, BN>;
    constexpr int STAGES = S::kStages;
    constexpr uint32_t ID = tc::idesc(BF16, true, true, BM, BN);
    extern __shared__ uint8_t raw[];
    __shared__ Shared s;
    const uint32_t shift = (1024 - (mb::smem_u32(raw) & 1023)) & 1023;
    const uint32_t ring = mb::smem_u32(raw) + shift;
    const uint32_t tmem = set_up<STAGES, BN>(s, g.offsets, g.types, g.M, g.piece);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = g.tiles_k * g.tiles_n;
    const int64_t items = static_cast<int64_t>(s.prefix[g.types]) * per;

    // Item -> type, piece, tile, rows.
    struct Item {
        int t, p, k0, n0, row0, row1;
        bool whole;
    };
    const auto item_at = [&](int64_t it) {
        Item r;
        r.p = static_cast<int>(it / per);
        const int in = static_cast<int>(it % per);
        r.k0 = in / g.tiles_n * BM;
        r.n0 = in % g.tiles_n * BN;
        r.t = find_type(s.prefix, g.types, r.p);
        const int b = clamp_row(g.offsets[r.t], g.M), e = clamp_row(g.offsets[r.t + 1], g.M);
        r.row0 = b + static_cast<int>((r.p - s.prefix[r.t]) * g.piece);
        r.row1 = static_cast<int>(r.row0 + g.piece < e ? r.row0 + g.piece : e);
        r.whole = s.prefix[r.t + 1] - s.prefix[r.t] == 1;
        return r;
    };

    if (warp == 0) {
        if (lane == 0) {
            int64_t i = 0;
            bool ok = true;
            for (int64_t it = blockIdx.x; it < items && ok; it += gridDim.x) {
                const Item m = item_at(it);
                for (int r = m.row0; r < m.row1; r += tc::kInner, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (i >= STAGES && !(ok = mb::wait(&s.empty[st], (i / STAGES - 1) & 1, &g_typed_error, 31))) break;
                    const uint32_t a = ring + st * S::kStage, b = a + PA * S::kA;
                    mb::arrive_expect_tx(&s.full[st], S::kStage);
#pragma unroll
                    for (int q = 0; q < PA; ++q)
#pragma unroll
                        for (int c = 0; c < BM / 64; ++c)
                            tc::tma3(a + q * S::kA + c * tc::kChunkBytes, &mx, m.k0 + c * 64, r, q, &s.full[st]);
#pragma unroll
                    for (int q = 0; q < PB; ++q)
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c)
                            tc::tma3(b + q * S::kB + c * tc::kChunkBytes, &my, m.n0 + c * 64, r, q, &s.full[st]);
                }
            }
            for (int64_t j = i > STAGES ? i - STAGES : 0; j < i; ++j)
                mb::wait(&s.full[j % STAGES], (j / STAGES) & 1, &g_typed_error, 32);
        }
    } else if (warp == 1) {
        int64_t i = 0;
        int local = 0;
        bool ok = true;
        for (int64_t it = blockIdx.x; it < items && ok; it += gridDim.x, ++local) {
            const Item m = item_at(it);
            const int acc = local & 1;
            if (local >= 2) ok = mb::wait(&s.acc_empty[acc], (local / 2 - 1) & 1, &g_typed_error, 33);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc::fence_after();
            for (int r = m.row0; r < m.row1; r += tc::kInner, ++i) {
                const int st = static_cast<int>(i % STAGES);
                ok = mb::wait(&s.full[st], (i / STAGES) & 1, &g_typed_error, 34);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc::fence_after();
                const int valid = m.row1 - r;
                if (valid < tc::kInner) {
                    // Rows of the next type (or piece): zero in both operands (0 x NaN would not do).
                    uint8_t* base = raw + shift + st * S::kStage;
                    for (uint32_t o = valid * 128 + lane * 16; o < S::kStage; o += 512) {
                        // row o / 128 of its 64-row chunk; skip to the next chunk's first invalid row
                        const uint32_t in = o % tc::kChunkBytes;
                        if (in >= static_cast<uint32_t>(valid) * 128)
                            *reinterpret_cast<uint4*>(base + o) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (lane == 0) {
                    stage_mmas<PA, PB, BN, true, true>(ring + st * S::kStage, tmem + acc * BN, ID, r == m.row0);
                    tc::commit(&s.empty[st]);
                }
                __syncwarp();
            }
            if (ok && lane == 0) tc::commit(&s.acc_full[acc]);
        }
    } else if (warp >= 4) {
        const int acc = (warp - 4) >> 2, q = warp & 3;
        int local = acc;
        for (int64_t it = blockIdx.x + acc * static_cast<int64_t>(gridDim.x); it < items;
             it += 2 * static_cast<int64_t>(gridDim.x), local += 2) {
            const Item m = item_at(it);
            if (!mb::wait(&s.acc_full[acc], (local / 2) & 1, &g_typed_error, 35)) break;
            tc::fence_after();
            const uint32_t addr = tmem + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
            const int64_t k = m.k0 + q * 32 + lane;
            const bool live = k < g.K;
#pragma unroll 1
            for (int c0 = 0; c0 < BN && m.n0 + c0 < g.N; c0 += 32) {
                float v[32];
                tc::load32(addr + c0, v);
                const int64_t n = m.n0 + c0;
                if (!live) continue;
                if (m.whole) store32(g.dW + m.t * g.stride_dw + k * g.lddw + n, v, g.N - n, g.mode);
                else store32(g.part + (m.p * g.K + k) * g.ldp + n, v, g.ldp - n, 2);
            }
            tc::fence_before();
            mb::arrive(&s.acc_empty[acc]);
        }
    }
    tear_down<BN>(s, tmem);
}

// dW of the types that the weight kernel did not finish: the sum of a type's
// pieces in their order, zero for a type without rows.
template <class O>
__global__ void __launch_bounds__(256) typed_weight_join_kernel(const WeightTc<O> g) {
    __shared__ int prefix[kMaxTypes + 1];
    const int t = blockIdx.y;
    const int b = clamp_row(g.offsets[t], g.M), e = clamp_row(g.offsets[t + 1], g.M);
    const int64_t n = e > b ? (e - b + g.piece - 1) / g.piece : 0;
    if (n == 1) return;
    if (n > 1 && threadIdx.x < 32) scan_types(g.offsets, t, g.M, g.piece, prefix);
    __syncthreads();
    const float* part = n > 1 ? g.part + static_cast<int64_t>(prefix[t]) * g.K * g.ldp : nullptr;
    const int64_t vecs = g.ldp / 4, total = g.K * vecs;
    for (int64_t v = blockIdx.x * 256 + threadIdx.x; v < total; v += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t k = v / vecs, c = (v - k * vecs) * 4;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int64_t q = 0; q < n; ++q) {
            const float4 x = *reinterpret_cast<const float4*>(part + (q * g.K + k) * g.ldp + c);
            sum.x += x.x;
            sum.y += x.y;
            sum.z += x.z;
            sum.w += x.w;
        }
        O* o = g.dW + t * g.stride_dw + k * g.lddw + c;
        const float y[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < g.N) o[j] = from_f32<O>(y[j]);
    }
}

// ── operands ─────────────────────────────────────────────────────────────
// P 16-bit planes [P][rows][ld] of a matrix whose row r lies at
// (r / inner) * stride + (r % inner) * lds.
template <class T, class H, int P>
__global__ void __launch_bounds__(256) planes_kernel(int64_t rows, int64_t cols, const T* src, int64_t inner,
                                                     int64_t stride, int64_t lds, H* dst, int64_t ld) {
    const int64_t vecs = ld / 8, total = rows * vecs;
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; v < total;
         v += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = v / vecs, c = (v - r * vecs) * 8;
        const T* p = src + r / inner * stride + r % inner * lds + c;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c + j < cols ? to_f32(p[j]) : 0.0f;
#pragma unroll
        for (int q = 0; q < P; ++q) {
            Raw<H, 8> k;
            narrow(x, k);
            if (P > 1) {
                float top[8];
                widen(k, top);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // a finite value above bf16's greatest rounds to infinity: take the greatest
                    if (isinf(top[j]) && !isinf(x[j])) top[j] = copysignf(3.3895314e38f, x[j]);
                    x[j] = __fsub_rn(x[j], top[j]);
                }
                narrow(top, k);
            }
            *reinterpret_cast<Raw<H, 8>*>(dst + (q * rows + r) * ld + c) = k;
        }
    }
}

// One 16-bit plane of a saved matrix, exactly.
template <class H>
__global__ void __launch_bounds__(256) saved_plane_kernel(int64_t rows, int64_t cols, Saved8 s, H* dst, int64_t ld) {
    const int64_t vecs = ld / 8, total = rows * vecs;
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; v < total;
         v += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = v / vecs, c = (v - r * vecs) * 8;
        const int byte = s.exps[r * s.lde + c / kBlock8];
        const uint2 in = *reinterpret_cast<const uint2*>(s.codes + r * s.ld + c);
        float x[8];
        values4(in.x, byte, x);
        values4(in.y, byte, x + 4);
        store_v<H, 8>(dst + r * ld + c, x);
    }
}

template <class T> struct Half { using type = T; static constexpr int planes = 1; };
template <> struct Half<float> { using type = __nv_bfloat16; static constexpr int planes = 3; };

// A matrix (or `types` of them) as 16-bit planes: in place, or in scratch.
template <class H>
struct Operand {
    const H* p = nullptr;
    int64_t ld = 0, stride = 0, plane = 0;  // elements
    H* own = nullptr;
    cudaStream_t s = nullptr;
    ~Operand() {
        if (own) scratch_free(own, s);
    }
    Operand() = default;
    Operand(const Operand&) = delete;
    Operand& operator=(const Operand&) = delete;

    void make(int64_t rows, int64_t cols, int planes, cudaStream_t st) {
        s = st;
        ld = (cols + 7) / 8 * 8;
        plane = rows * ld;
        own = static_cast<H*>(scratch_alloc(static_cast<size_t>(planes * plane) * 2, st));
        p = own;
    }
};

unsigned prep_grid(int64_t rows, int64_t ld) {
    return static_cast<unsigned>(std::min<int64_t>(ceil_div(rows * (ld / 8), 256), int64_t(num_sms()) * 8));
}

// `batch` matrices of rows x cols, ld and stride apart.
template <class T>
void make_operand(Operand<typename Half<T>::type>& o, int64_t batch, int64_t rows, int64_t cols, const T* src,
                  int64_t ld, int64_t stride, cudaStream_t s) {
    using H = typename Half<T>::type;
    constexpr int P = Half<T>::planes;
    if constexpr (P == 1) {
        if (rows_aligned16(src, ld, 2) && (batch == 1 || stride % 8 == 0) && rows * ld * 2 < (int64_t(1) << 39) &&
            stride * 2 < (int64_t(1) << 39)) {
            o.p = src;
            o.ld = ld;
            o.stride = batch == 1 ? rows * ld : stride;
            o.plane = batch * o.stride;
            return;
        }
    }
    o.make(batch * rows, cols, P, s);
    o.stride = rows * o.ld;
    launch("typed_operand", planes_kernel<T, H, P>, dim3(prep_grid(batch * rows, o.ld)), dim3(256), 0, s, batch * rows,
           cols, src, rows, stride, ld, o.own, o.ld);
}

template <class H>
void make_saved_operand(Operand<H>& o, int64_t rows, int64_t cols, const Saved8& saved, cudaStream_t s) {
    o.make(rows, cols, 1, s);
    o.stride = rows * o.ld;
    launch("typed_operand", saved_plane_kernel<H>, dim3(prep_grid(rows, o.ld)), dim3(256), 0, s, rows, cols, saved,
           o.own, o.ld);
}

template <class H>
constexpr bool is_bf16() { return std::is_same<H, __nv_bfloat16>::value; }

template <class H>
CUtensorMap rows_map(const Operand<H>& o, int64_t rows, int64_t cols, int planes, int box_rows) {
    const int64_t dims[3] = {cols, rows, planes}, strides[2] = {o.ld, std::max<int64_t>(o.plane, 8)};
    const int box[3] = {64, box_rows, 1};
    return tc::map16<3>(o.p, is_bf16<H>(), dims, strides, box);
}

template <class K, class... A>
void run_tc(const char* name, K kern, uint32_t smem, int64_t tiles, cudaStream_t s, A... args) {
    TG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    launch(name, kern, dim3(static_cast<unsigned>(std::min<int64_t>(tiles, num_sms()))), dim3(kThreads), smem, s,
           args...);
}

template <class O>
void join_pieces(const WeightTc<O>& g, int types, cudaStream_t s) {
    launch("typed_weight_join", typed_weight_join_kernel<O>,
           dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(g.K * g.ldp / 4, 256), std::max(8, 16384 / types))),
                static_cast<unsigned>(types)),
           dim3(256), 0, s, g);
}

// Tile width.  Columns that no output has cost tensor time, and a wide tile
// reads the rows fewer times.
int tile_width(int64_t N, int widest) { return N <= 64 ? 64 : (N <= 128 || widest == 128 ? 128 : 256); }

}  // namespace

template <class T, bool TRANS>
void typed_rows_tc(const RowsArgs<T>& a, cudaStream_t s) {
    using H = typename Half<T>::type;
    constexpr int P = Half<T>::planes;
    Operand<H> A, W;
    make_operand<T>(A, 1, a.M, a.K, a.A, a.lda, 0, s);
    // W[t] is K x N in the forward pass, N x K in the input gradient.
    const int64_t wr = TRANS ? a.N : a.K, wc = TRANS ? a.K : a.N;
    make_operand<T>(W, a.types, wr, wc, a.W, a.ldw, a.stride_w, s);
    const CUtensorMap ma = rows_map(A, a.M, a.K, P, BM);
    const auto go = [&](auto bn) {
        constexpr int BN = decltype(bn)::value;
        const int64_t dims[4] = {wc, wr, a.types, P}, strides[3] = {W.ld, W.stride, W.plane};
        const int box[4] = {64, TRANS ? BN : 64, 1, 1};
        const CUtensorMap mw = tc::map16<4>(W.p, is_bf16<H>(), dims, strides, box);
        RowsTc<T> g{a.M, a.K, a.N, a.types, static_cast<int>(ceil_div(a.N, BN)), a.offsets, a.bias, a.act, a.alpha,
                    a.C, a.ldc, store_mode(a.C, a.ldc), a.saved, a.r8};
        run_tc("typed_rows", typed_rows_tc_kernel<T, P, BN, TRANS, is_bf16<H>()>, Plan<P, P, BN>::kBytes,
               (a.M / BM + a.types) * g.tiles_n, s, ma, mw, g);
    };
    switch (tile_width(a.N, P == 1 ? 256 : 128)) {
        case 64: go(std::integral_constant<int, 64>{}); break;
        case 128: go(std::integral_constant<int, 128>{}); break;
        default:
            if constexpr (P == 1) go(std::integral_constant<int, 256>{});
    }
}

template <class T, class O>
void typed_weight_tc(const WeightArgs<T, O>& a, cudaStream_t s) {
    using H = typename Half<T>::type;
    constexpr int PB = Half<T>::planes;
    Operand<H> X, Y;
    const bool saved = a.saved.codes != nullptr;
    if (a.M == 0) {  // no rows: dW is zero
        WeightTc<O> g{};
        g.K = a.K;
        g.N = a.N;
        g.offsets = a.offsets;
        g.piece = 1;
        g.dW = a.dW;
        g.lddw = a.lddw;
        g.stride_dw = a.stride_dw;
        g.ldp = (a.N + 7) / 8 * 8;
        join_pieces(g, a.types, s);
        return;
    }
    if (saved) make_saved_operand<H>(X, a.M, a.K, a.saved, s);
    else make_operand<T>(X, 1, a.M, a.K, a.X, a.ldx, 0, s);
    make_operand<T>(Y, 1, a.M, a.N, a.dY, a.lddy, 0, s);
    const CUtensorMap my = rows_map(Y, a.M, a.N, PB, 64);
    const auto go = [&](auto bn, auto pa) {
        constexpr int BN = decltype(bn)::value, PA = decltype(pa)::value;
        const CUtensorMap mx = rows_map(X, a.M, a.K, PA, 64);
        WeightTc<O> g{a.M, a.K, a.N, a.types, static_cast<int>(ceil_div(a.K, BM)), static_cast<int>(ceil_div(a.N, BN)),
                      a.offsets, 0, a.dW, a.lddw, a.stride_dw, store_mode(a.dW, a.lddw) , nullptr, (a.N + 7) / 8 * 8};
        if (a.stride_dw * sizeof(O) % 32 != 0) g.mode = a.stride_dw * sizeof(O) % 16 == 0 ? std::min(g.mode, 1) : 0;
        const int64_t per = int64_t(g.tiles_k) * g.tiles_n;
        // About 2.5 sums per SM: enough to even out types of unequal sizes,
        // few enough that the partial sums' traffic stays small.
        g.piece = std::max<int64_t>(128, ceil_div(a.M * per * 2, int64_t(num_sms()) * 5 * 64) * 64);
        const int64_t pieces = a.M / g.piece + std::min<int64_t>(a.types, a.M);
        Scratch<float> part(a.M > g.piece ? static_cast<size_t>(pieces * a.K * g.ldp) : 1, s);
        g.part = part.p;
        run_tc("typed_weight", typed_weight_tc_kernel<O, PA, PB, BN, is_bf16<H>()>, Plan<PA, PB, BN>::kBytes,
               pieces * per, s, mx, my, g);
        join_pieces(g, a.types, s);
    };
    const auto with_planes = [&](auto bn) {
        if constexpr (PB == 1) go(bn, std::integral_constant<int, 1>{});
        else if (saved) go(bn, std::integral_constant<int, 1>{});
        else go(bn, std::integral_constant<int, PB>{});
    };
    switch (tile_width(a.N, PB == 1 ? 256 : 128)) {
        case 64: with_planes(std::integral_constant<int, 64>{}); break;
        case 128: with_planes(std::integral_constant<int, 128>{}); break;
        default:
            if constexpr (PB == 1) with_planes(std::integral_constant<int, 256>{});
    }
}

#define TG_TYPED(T)                                                  \
    template void typed_rows_tc<T, false>(const RowsArgs<T>&, cudaStream_t); \
    template void typed_rows_tc<T, true>(const RowsArgs<T>&, cudaStream_t);  \
    template void typed_weight_tc<T, T>(const WeightArgs<T, T>&, cudaStream_t);
TG_TYPED(float)
TG_TYPED(__nv_bfloat16)
TG_TYPED(__half)
template void typed_weight_tc<__nv_bfloat16, float>(const WeightArgs<__nv_bfloat16, float>&, cudaStream_t);
template void typed_weight_tc<__half, float>(const WeightArgs<__half, float>&, cudaStream_t);

// Reads and clears the typed kernels' error word (the stream is idle).
int typed_take_error() {
    int h = 0;
    TG_CUDA(cudaMemcpyFromSymbol(&h, g_typed_error, sizeof(int)));
    if (h) {
        const int zero = 0;
        TG_CUDA(cudaMemcpyToSymbol(g_typed_error, &zero, sizeof(int)));
    }
    return h;
}

}  // namespace tg

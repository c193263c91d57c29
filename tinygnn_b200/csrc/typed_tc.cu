// ============================================================================
//  typed_tc.cu -- the typed linear map's products on the tensor cores, operands
//  by TMA, and the choice of kernel for every product.
//
//  rows kernel    C[r] = act(A[r] . B[t(r)] + bias[t(r)]): the forward pass
//                 (B = W[t], its columns contiguous) and the input gradient
//                 (B = W[t]^T).
//  weight kernel  dW[t] = sum over the type's rows of X[r]^T dY[r]; both
//                 operands have their outer index contiguous.
//
//  Operands are bf16 or fp16 with 16-byte aligned rows (TMA's rule); the other
//  forms are typed_any.cu's.  Both kernels are persistent: CTAs walk tiles
//  blockIdx.x, + gridDim.x, ...
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
#include "typed_mma.cuh"

namespace tg {

namespace {

using namespace typed;

constexpr int kThreads = 384;

// ── rows kernel ──────────────────────────────────────────────────────────
struct RowsTc {
    int64_t M, K;
    int types, tiles_n;
    const int32_t* offsets;
};

template <class T, int BN, bool TRANS>
__global__ void __launch_bounds__(kThreads, 1) typed_rows_tc_kernel(const __grid_constant__ CUtensorMap ma,
                                                                    const __grid_constant__ CUtensorMap mw,
                                                                    const RowsTc g, const RowsOut<T> out) {
    using S = Plan<1, 1, BN>;
    constexpr int STAGES = S::kStages;
    constexpr uint32_t ID = tc::idesc(is_bf16<T>(), false, !TRANS, BM, BN);
    extern __shared__ uint8_t raw[];
    __shared__ Shared s;
    __shared__ T stage_out[8][stage_bytes<T>() / sizeof(T)];
    const uint32_t ring = (mb::smem_u32(raw) + 1023) & ~1023u;
    if (threadIdx.x == 0) {
        tc::prefetch_map(&ma);
        tc::prefetch_map(&mw);
    }
    const uint32_t tmem = set_up<STAGES, BN>(s, 1, BN == 256 ? 256 : 128, [&] { scan_types(g.offsets, g.types, g.M, BM, s.prefix); });
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
                    if (i >= STAGES && !(ok = mb::wait(&s.empty[st], (i / STAGES - 1) & 1, &g_error, 21))) break;
                    const uint32_t a = ring + st * S::kStage, b = a + S::kA;
                    mb::arrive_expect_tx(&s.full[st], S::kStage);
                    tc::tma3(a, &ma, kb * tc::kInner, row0, 0, &s.full[st]);
                    if (TRANS) {
                        tc::tma3(b, &mw, kb * tc::kInner, n0, t, &s.full[st]);
                    } else {
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c)
                            tc::tma3(b + c * tc::kChunkBytes, &mw, n0 + c * 64, kb * tc::kInner, t, &s.full[st]);
                    }
                }
            }
            // Every copy issued must have landed before the CTA may exit.
            for (int64_t j = i > STAGES ? i - STAGES : 0; j < i; ++j)
                mb::wait(&s.full[j % STAGES], (j / STAGES) & 1, &g_error, 22);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int64_t i = 0;
            int local = 0;
            bool ok = true;
            for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++local) {
                const int acc = local & 1;
                if (local >= 2 && !(ok = mb::wait(&s.acc_empty[acc], (local / 2 - 1) & 1, &g_error, 23))) break;
                tc::fence_after();
                for (int kb = 0; kb < KB; ++kb, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (!(ok = mb::wait(&s.full[st], (i / STAGES) & 1, &g_error, 24))) break;
                    tc::fence_after();
                    stage_mmas<1, 1, BN, false, !TRANS>(ring + st * S::kStage, tmem + acc * BN, ID, kb == 0);
                    tc::commit(&s.empty[st]);
                }
                if (ok) tc::commit(&s.acc_full[acc]);
            }
        }
    } else if (warp >= 4) {
        // 256 columns: every tile is split between the two groups of four warps
        // (a lone tile's results leave in half the time); fewer: in turn.
        constexpr bool SHARE = BN == 256;
        constexpr int WIDTH = SHARE ? BN / 2 : BN;
        const int group = (warp - 4) >> 2, q = warp & 3, c0 = SHARE ? group * WIDTH : 0;
        int local = SHARE ? 0 : group;
        for (int64_t tile = blockIdx.x + local * static_cast<int64_t>(gridDim.x); tile < tiles;
             tile += (SHARE ? 1 : 2) * static_cast<int64_t>(gridDim.x), local += SHARE ? 1 : 2) {
            const int acc = local & 1;
            const int p = static_cast<int>(tile / g.tiles_n);
            const int t = find_type(s.prefix, g.types, p);
            const int64_t row0 = clamp_row(g.offsets[t], g.M) + static_cast<int64_t>(p - s.prefix[t]) * BM + q * 32;
            const int64_t left = clamp_row(g.offsets[t + 1], g.M) - row0, n0 = tile % g.tiles_n * BN + c0;
            prefetch_bias<T, WIDTH>(out, t, n0);
            const bool ok = mb::wait(&s.acc_full[acc], (local / 2) & 1, &g_error, 25);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::fence_after();
            finish_rows<T, WIDTH, true>(tmem + acc * BN + c0 + (static_cast<uint32_t>(q * 32) << 16), out, t, row0,
                                        left < 0 ? 0 : (left < 32 ? static_cast<int>(left) : 32), n0,
                                        stage_out[warp - 4]);
            tc::fence_before();
            mb::arrive(&s.acc_empty[acc]);
        }
    }
    tear_down<BN>(s, tmem, 1);
}

// ── weight kernel ────────────────────────────────────────────────────────
template <class O>
struct WeightTc {
    int64_t M, K, N;
    int types, tiles_k, tiles_n, slots, longest;
    const int32_t* offsets;
    O* dW;
    int64_t lddw, stride_dw;
    int mode;
    float* part;
    int64_t ldp;
};

template <class T, class O, int BN>
__global__ void __launch_bounds__(kThreads, 1) typed_weight_tc_kernel(const __grid_constant__ CUtensorMap mx,
                                                                      const __grid_constant__ CUtensorMap my,
                                                                      const WeightTc<O> g) {
    using S = Plan<1, 1, BN>;
    constexpr int STAGES = S::kStages;
    constexpr uint32_t ID = tc::idesc(is_bf16<T>(), true, true, BM, BN);
    extern __shared__ uint8_t raw[];
    __shared__ Shared s;
    __shared__ T stage_out[8][stage_bytes<T>() / sizeof(T)];
    const uint32_t ring = (mb::smem_u32(raw) + 1023) & ~1023u;
    const uint32_t tmem = set_up<STAGES, BN>(s, 1, 128, [&] {
        plan_pieces(g.offsets, g.types, g.M, g.tiles_k * g.tiles_n, g.slots, g.longest, s.prefix, s.order);
    });
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = g.tiles_k * g.tiles_n;
    const int64_t items = static_cast<int64_t>(s.prefix[g.types]) * per;

    struct Item {
        int t, p, k0, n0, row0, row1;
        bool whole;
    };
    const auto item_at = [&](int64_t it) {
        const WeightItem w = weight_item(g.offsets, g.types, g.M, per, s.prefix, s.order, it);
        return Item{w.t, w.p, w.in / g.tiles_n * BM, w.in % g.tiles_n * BN, static_cast<int>(w.r0),
                    static_cast<int>(w.r1), w.whole};
    };
    // Round r's item of this CTA.
    const auto dealt_item = [&](int64_t r) { return dealt(r, blockIdx.x, gridDim.x); };

    if (warp == 0) {
        if (lane == 0) {
            int64_t i = 0;
            bool ok = true;
            for (int64_t round = 0, it; (it = dealt_item(round)) < items && ok; ++round) {
                const Item m = item_at(it);
                for (int r = m.row0; r < m.row1; r += tc::kInner, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (i >= STAGES && !(ok = mb::wait(&s.empty[st], (i / STAGES - 1) & 1, &g_error, 31))) break;
                    const uint32_t a = ring + st * S::kStage, b = a + S::kA;
                    mb::arrive_expect_tx(&s.full[st], S::kStage);
#pragma unroll
                    for (int c = 0; c < BM / 64; ++c)
                        tc::tma3(a + c * tc::kChunkBytes, &mx, m.k0 + c * 64, r, 0, &s.full[st]);
#pragma unroll
                    for (int c = 0; c < BN / 64; ++c)
                        tc::tma3(b + c * tc::kChunkBytes, &my, m.n0 + c * 64, r, 0, &s.full[st]);
                }
            }
            for (int64_t j = i > STAGES ? i - STAGES : 0; j < i; ++j)
                mb::wait(&s.full[j % STAGES], (j / STAGES) & 1, &g_error, 32);
        }
    } else if (warp == 1) {
        int64_t i = 0;
        int local = 0;
        bool ok = true;
        for (int64_t it; (it = dealt_item(local)) < items && ok; ++local) {
            const Item m = item_at(it);
            const int acc = local & 1;
            if (local >= 2) ok = mb::wait(&s.acc_empty[acc], (local / 2 - 1) & 1, &g_error, 33);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc::fence_after();
            for (int r = m.row0; r < m.row1; r += tc::kInner, ++i) {
                const int st = static_cast<int>(i % STAGES);
                ok = mb::wait(&s.full[st], (i / STAGES) & 1, &g_error, 34);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
                tc::fence_after();
                // Rows of the next type (or piece): zero in both operands (0 x NaN would not do).
                if (m.row1 - r < tc::kInner) zero_rows(ring + st * S::kStage, S::kStage, m.row1 - r);
                if (lane == 0) {
                    stage_mmas<1, 1, BN, true, true>(ring + st * S::kStage, tmem + acc * BN, ID, r == m.row0);
                    tc::commit(&s.empty[st]);
                }
                __syncwarp();
            }
            if (ok && lane == 0) tc::commit(&s.acc_full[acc]);
        }
    } else if (warp >= 4) {
        const int acc = (warp - 4) >> 2, q = warp & 3;
        int local = acc;
        for (int64_t it; (it = dealt_item(local)) < items; local += 2) {
            const Item m = item_at(it);
            const bool ok = mb::wait(&s.acc_full[acc], (local / 2) & 1, &g_error, 35);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::fence_after();
            const uint32_t addr = tmem + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
            const int64_t k = m.k0 + q * 32, left_k = g.K - k;
            const int rows = left_k < 0 ? 0 : (left_k < 32 ? static_cast<int>(left_k) : 32);
#pragma unroll 1
            for (int c0 = 0; c0 < BN && m.n0 + c0 < g.N; c0 += 32) {
                float v[32];
                tc::load32(addr + c0, v);
                const int64_t n = m.n0 + c0;
                if (m.whole) {
                    O* o = g.dW + m.t * g.stride_dw + k * g.lddw + n;
                    // shared memory has room to stage rows of T, not of fp32
                    if constexpr (sizeof(O) == sizeof(T)) store_rows(o, g.lddw, rows, g.N - n, v, g.mode, stage_out[warp - 4]);
                    else store_rows(o, g.lddw, rows, g.N - n, v, g.mode == 0 ? -1 : g.mode, static_cast<O*>(nullptr));
                } else {
                    store_rows(g.part + (m.p * g.K + k) * g.ldp + n, g.ldp, rows, g.ldp - n, v, 2,
                               static_cast<float*>(nullptr));
                }
            }
            tc::fence_before();
            mb::arrive(&s.acc_empty[acc]);
        }
        zero_empty_types(g.offsets, g.types, g.M, g.K, g.N, g.dW, g.lddw, g.stride_dw, g.mode, threadIdx.x - 128, 256);
    }
    tear_down<BN>(s, tmem, 1);
}

// dW and db of the types with several pieces: the sum of the pieces in their order.
template <class O>
struct JoinArgs {
    int64_t M, K, N, ldp;
    int types, per, slots, longest;
    int64_t least;  // no type of at most as many rows is cut (the limit when no step is ragged)
    const int32_t* offsets;
    const float *part, *db_part;
    O* dW;
    int64_t lddw, stride_dw;
    float* db;  // nullable
};

template <class O>
__global__ void __launch_bounds__(256) typed_weight_join_kernel(const JoinArgs<O> g) {
    __shared__ int64_t sums[8];
    __shared__ int first[8];
    wait_for_previous();
    const int t = blockIdx.y, rows = rows_of(g.offsets, t, g.M);
    if (rows <= g.least) return;
    const auto block_sum = [&](auto x, auto* sh) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = x;
        __syncthreads();
        x = 0;
        for (int w = 0; w < 8; ++w) x += sh[w];
        return x;
    };
    int64_t steps = 0;
    for (int u = threadIdx.x; u < g.types; u += 256) steps += (rows_of(g.offsets, u, g.M) + kStep - 1) / kStep;
    const int64_t limit = piece_limit(block_sum(steps, sums), g.M, g.types, g.per, g.slots, g.longest);
    const int n = piece_count(rows, limit);
    if (n <= 1) return;  // the weight kernel wrote it
    // this type's first slot
    const int len = piece_rows(rows, n);
    int before = 0;
    for (int u = threadIdx.x; u < g.types; u += 256) {
        const int ru = rows_of(g.offsets, u, g.M), nu = piece_count(ru, limit);
        if (nu > 1 && piece_before(g.types, piece_rows(ru, nu), u, len, t)) before += nu;
    }
    const int64_t p = block_sum(before, first);
    const float* part = g.part + p * g.K * g.ldp;
    // four columns a thread; a block takes as many rows of dW at a time as it has threads for
    const int vecs = static_cast<int>(g.ldp / 4), wide = vecs < 256 ? vecs : 256, rpb = 256 / wide;
    const int64_t next = g.K * g.ldp;
    const int r = threadIdx.x / wide;
    for (int64_t k = blockIdx.x * rpb + r; r < rpb && k < g.K; k += static_cast<int64_t>(gridDim.x) * rpb)
        for (int64_t c = (threadIdx.x - r * wide) * 4; c < g.N; c += wide * 4) {
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float* q = part + k * g.ldp + c;
#pragma unroll 8
            for (int i = 0; i < n; ++i, q += next) {
                const float4 x = *reinterpret_cast<const float4*>(q);
                sum.x += x.x;
                sum.y += x.y;
                sum.z += x.z;
                sum.w += x.w;
            }
            O* o = g.dW + t * g.stride_dw + k * g.lddw + c;
            const float y[4] = {sum.x, sum.y, sum.z, sum.w};
            if (c + 4 <= g.N && (reinterpret_cast<uintptr_t>(o) % (4 * sizeof(O))) == 0) {
                store_v<O, 4>(o, y);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < g.N) o[j] = from_f32<O>(y[j]);
            }
        }
    if (g.db)
        for (int64_t c = blockIdx.x * 256 + threadIdx.x; c < g.N; c += static_cast<int64_t>(gridDim.x) * 256) {
            float sum = 0.0f;
#pragma unroll 8
            for (int i = 0; i < n; ++i) sum += g.db_part[(p + i) * g.N + c];
            g.db[t * g.N + c] = sum;
        }
}

template <class T, bool TRANS>
void typed_rows_tma(const RowsArgs<T>& a, cudaStream_t s) {
    const Operand<T> A(1, a.M, a.K, a.A, a.lda, 0, s);
    // W[t] is K x N in the forward pass, N x K in the input gradient.
    const int64_t wr = TRANS ? a.N : a.K, wc = TRANS ? a.K : a.N;
    const Operand<T> W(a.types, wr, wc, a.W, a.ldw, a.stride_w, s);
    // Pairs of CTAs for long sums, where 256-row tiles of 256 columns are enough
    // for all of them and the types long enough not to leave much of a tile
    // empty.  Measured, back to back, pairs against single CTAs: 65,536 x 2,048
    // x 2,048 437-459 against 481-485 us, 65,536 x 1,024 x 1,024 128 against
    // 140, 16,384 x 1,024 x 1,024 38.5 against 39.0, 65,536 x 512 x 512 47.2
    // both, 100,000 x 256 x 256 28.8 against 28.0.  (Weight gradients gained
    // nothing: 149 against 139 us for 65,536 x 1,024 x 1,024.)
    if (a.K > 512 && a.N > 128 && a.M / 512 >= a.types && (a.M / 256) * ceil_div(a.N, 256) >= num_sms()) {
        typed_rows_pair<T, TRANS>(a, A.matrix(), W.matrix(), s);
        return;
    }
    const CUtensorMap ma = tma_map(A.matrix(), 1, a.M, a.K, BM);
    const int64_t pieces = a.M / BM + std::min<int64_t>(a.types, a.M);
    const RowsOut<T> out{a.N, a.bias, a.act, a.alpha, a.C, a.ldc, store_mode(a.C, a.ldc * 2), a.saved, a.r8};
    const auto go = [&](auto bn) {
        constexpr int BN = decltype(bn)::value;
        const CUtensorMap mw = tma_map(W.matrix(), a.types, wr, wc, TRANS ? BN : 64);
        const RowsTc g{a.M, a.K, a.types, static_cast<int>(ceil_div(a.N, BN)), a.offsets};
        run("typed_rows", typed_rows_tc_kernel<T, BN, TRANS>, kThreads, Plan<1, 1, BN>::kBytes, pieces * g.tiles_n, s,
            ma, mw, g, out);
    };
    switch (tile_width(pieces, a.N, 256, a.saved.codes != nullptr)) {
        case 64: go(std::integral_constant<int, 64>{}); break;
        case 128: go(std::integral_constant<int, 128>{}); break;
        default: go(std::integral_constant<int, 256>{});
    }
}

template <class T, class O>
void typed_weight_tma(const WeightArgs<T, O>& a, const WeightPlan& w, cudaStream_t s) {
    // X in 8 bits: its values as a 16-bit matrix, exactly (33 us for 65,536 x
    // 1,024 at HBM rate; a kernel whose loaders decoded the codes into shared
    // memory for every tile of columns took 60 us longer than this and TMA).
    const Operand<T> X(a.M, a.K, a.X, a.ldx, a.saved, s), Y(1, a.M, a.N, a.dY, a.lddy, 0, s);
    const CUtensorMap mx = tma_map(X.matrix(), 1, a.M, a.K, 64), my = tma_map(Y.matrix(), 1, a.M, a.N, 64);
    const WeightTc<O> g{a.M, a.K, a.N, a.types, w.tiles_k, w.tiles_n, w.slots, w.longest, a.offsets, a.dW, a.lddw, a.stride_dw,
                        store_mode(a.dW, a.lddw * sizeof(O), a.stride_dw * sizeof(O)), w.part, w.ldp};
    const auto go = [&](auto bn) {
        constexpr int BN = decltype(bn)::value;
        run("typed_weight", typed_weight_tc_kernel<T, O, BN>, kThreads, Plan<1, 1, BN>::kBytes, w.items, s, mx, my, g);
    };
    switch (w.BN) {
        case 64: go(std::integral_constant<int, 64>{}); break;
        case 128: go(std::integral_constant<int, 128>{}); break;
        default: go(std::integral_constant<int, 256>{});
    }
}

// 2 M K N above which dW's 16-bit operands go by TMA, and db in kernels of its
// own: 16,384 x 512 x 512 bf16 without db, 26.9 by TMA and 29.7 us by loaders;
// 8,192 x 512 x 512 23.9 and 20.8 (and db's two kernels take 8 us more).
constexpr double kLargeFlops = 1e10;

}  // namespace

// Which products of a few rows stream the weights (typed_few.cu): those kernels
// read a row's weight from L2 or HBM for every row, so they lose to a tile when
// rows share a large weight; where rows have weights of their own the tiles are
// mostly empty.  The host does not see how the rows lie (unless there is one
// type), so each limit is where the worse of the two loses least.  us by few
// rows / by tiles, rows of one type | each in a type of its own (K = N = 2,048
// unless given; other weights in between, not in L2):
//   forward, 16 bits  8 rows 14.5 / 13.6 | 13.9 / 21.4;  16 rows 15.5 / 13.8 |
//                     24 / 30;  32 rows 28 / 13.5 | 45 / 44;  1,024: 32 rows
//                     9.3 / 8.9 | 13.9 / 17.7;  4,096: 4 rows 27 / 26 | 31 / 41,
//                     32 rows 93 / 23 | 165 / 160
//   forward, fp32     32 rows 36 / 55 | 81 / 235;  8,192: 8 rows 136 / 191 |
//                     300 / 899, 32 rows 445 / 193 | 663 / 1,897
//   dX, 16 bits       1 row 13.2 / 13.7 | 12.3 / 13.9;  4 rows 30 / 13.5 | 30 /
//                     19.5;  1,024: 4 rows 9.8 / 8.9 | 9.5 / 10.0, 8 rows 16.8 /
//                     8.8 | 16.8 / 12.5;  256: 16 rows 5.0 / 5.9 | 5.5 / 6.2, 32
//                     rows 8.3 / 5.9 | 8.4 / 6.8
//   dX, fp32          8 rows 26 / 53 | 28 / 69;  32 rows 82 / 54 | 86 / 234;
//                     1,024: 32 rows 24 / 29 | 27 / 70;  4,096 x 512: 32 rows
//                     55 / 16.5 | 56 / 111
bool few_rows(int64_t M, int64_t K, int64_t N, int types, size_t size, bool trans) {
    const double work = static_cast<double>(M) * K * N;
    if (M > kFewRows) return false;
    if (size == 2) return trans ? work <= (M <= 4 ? 1 << 22 : 1 << 20) : M <= 4 || work <= 1 << 25;
    return trans ? M <= 4 || work <= 1 << 25 : types > 1 || work <= 1 << 29;
}
// The weight gradients that go there: 8 rows, or no more rows than types (most
// of dW is zeros, and a tile kernel's CTAs walk all types for them).
// Measured as above, rows each in a type of its own | all in one: bf16, 1,024 x
// 1,024: 64 rows 47 / 78 | 143 / 94, 256 rows 172 / 320 | 716 / 648, 1,024 rows
// 667 / 1,250 | 2,886 / 2,474;  128 x 128: 64 rows 5.6 / 16 | 51 / 27, 1,024 rows
// 16 / 140 | 915 / 329;  fp32, 1,024 x 1,024: 1,024 rows 1,416 / 1,910 | 4,386 /
// 2,421.
bool few_weight_rows(int64_t M, int types) { return M <= 8 || M <= types; }

template <class T, bool TRANS>
void typed_rows(const RowsArgs<T>& a, cudaStream_t s) {
    if (few_rows(a.M, a.K, a.N, a.types, sizeof(T), TRANS)) typed_rows_few<T, TRANS>(a, s);
    else if constexpr (sizeof(T) == 2) typed_rows_tma<T, TRANS>(a, s);
    else typed_rows_any<TRANS>(a, s);
}

template <class T, class O>
void typed_weight(const WeightArgs<T, O>& a, cudaStream_t s) {
    if (few_weight_rows(a.M, a.types)) {  // no rows: dW and db are zero
        typed_weight_few<T, O>(a, s);
        return;
    }
    // by TMA; the rows that only a copy makes readable are worth it at any size
    // (8,192 x 511 x 513 bf16: 43 us, and 257 by loaders that take any alignment)
    const bool by_tma = sizeof(T) == 2 && (2.0 * a.M * a.K * a.N > kLargeFlops ||
                                           !(a.saved.codes || in_place(1, a.K, a.X, a.ldx, 0)) ||
                                           !in_place(1, a.N, a.dY, a.lddy, 0));
    WeightPlan w{};
    const int widest = by_tma ? 256 : 128;
    w.BN = a.N <= 64 ? 64 : (a.N <= 128 || widest == 128 ? 128 : 256);
    w.tiles_k = static_cast<int>(ceil_div(a.K, BM));
    w.tiles_n = static_cast<int>(ceil_div(a.N, w.BN));
    const int64_t per = int64_t(w.tiles_k) * w.tiles_n;
    w.slots = num_sms();
    w.longest = by_tma && sizeof(O) == 4 ? 64 : 1 << 30;
    const int64_t pieces = max_pieces(a.M, a.types, per, w.slots, w.longest);
    w.items = std::max<int64_t>(pieces * per, std::min(a.types, num_sms()));
    w.ldp = (a.N + 7) / 8 * 8;
    // None is, if even all the rows in one type are an SM's share or two steps.
    const bool joined = a.M > 2 * kStep && (per < w.slots || a.M > int64_t(w.longest) * kStep);
    const int64_t slots = joined ? max_slots(a.M, a.types, per, w.slots, w.longest) : 0;
    Scratch<float> part(static_cast<size_t>(slots * (a.K * w.ldp + a.N)), s);
    w.part = part.p;
    w.db_part = part.p + slots * a.K * w.ldp;
    bool done = false;
    if constexpr (sizeof(T) == 2) {
        if (by_tma) {
            if (a.db) typed_bias<T>(a.M, a.N, a.types, a.offsets, a.dY, a.lddy, a.db, s);
            typed_weight_tma<T, O>(a, w, s);
            done = true;
        }
    }
    if (!done) typed_weight_any<T, O>(a, w, s);
    if (joined) {
        const JoinArgs<O> j{a.M, a.K, a.N, w.ldp, a.types, static_cast<int>(per), w.slots, w.longest,
                            piece_limit(a.M / kStep, a.M, a.types, static_cast<int>(per), w.slots, w.longest), a.offsets, w.part,
                            w.db_part, a.dW, a.lddw, a.stride_dw, by_tma ? nullptr : a.db};
        const int64_t want = ceil_div(a.K * std::min<int64_t>(w.ldp / 4, 256), 256);
        launch_dependent("typed_weight_join", typed_weight_join_kernel<O>,
                         dim3(static_cast<unsigned>(std::min<int64_t>(want, std::max(1, 8 * num_sms() / a.types))),
                              static_cast<unsigned>(a.types)),
                         dim3(256), 0, s, j);
    }
}

#define TG_TYPED(T)                                                       \
    template void typed_rows<T, false>(const RowsArgs<T>&, cudaStream_t); \
    template void typed_rows<T, true>(const RowsArgs<T>&, cudaStream_t);  \
    template void typed_weight<T, T>(const WeightArgs<T, T>&, cudaStream_t);
TG_TYPED(float)
TG_TYPED(__nv_bfloat16)
TG_TYPED(__half)
template void typed_weight<__nv_bfloat16, float>(const WeightArgs<__nv_bfloat16, float>&, cudaStream_t);
template void typed_weight<__half, float>(const WeightArgs<__half, float>&, cudaStream_t);

int typed_tc_take_error() { return take_error(); }

}  // namespace tg

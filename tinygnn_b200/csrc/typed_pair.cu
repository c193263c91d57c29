// ============================================================================
//  typed_pair.cu -- the large typed products (forward pass, input gradient) on
//  pairs of CTAs: tiles of 256 rows x 256 columns, 16-bit operands by TMA.
//
//  A lone CTA's 128 x 256 tile takes 12 KB of operands per MMA of 16 inner
//  indexes (128 cycles); in a pair each CTA holds 128 rows and 128 of the 256
//  columns and takes 8 KB.  A step of 64 inner indexes takes 615 cycles (512 at
//  the tensor cores' peak), at the 1.29 GHz that the power cap leaves: 65,536 x
//  2,048 x 2,048 bf16 in 437-459 us, 1.2 PFLOP/s, where single CTAs take
//  481-485 (fewer bytes moved is less power and a higher clock).  For seconds on
//  end it takes 465 us at 1.28 GHz, with bias, GELU and the 8-bit copy 564.
//
//  The structure is typed_tc.cu's: warp 0 loads, warp 1 of rank 0 issues the
//  MMAs for both CTAs, warps 4-11 empty the two accumulators.
// ============================================================================
#include "typed_mma.cuh"

namespace tg {

namespace {

using namespace typed;

constexpr int kThreads = 384;
constexpr int BN = 256, HN = 128;  // columns of a tile, and of it in one CTA
constexpr int kRows = 2 * BM;      // rows of a tile

struct PairPlan {
    static constexpr uint32_t kA = BM * 128, kB = HN * 128, kStage = kA + kB;
    static constexpr int kStages = 6;
    static constexpr uint32_t kBytes = kStages * kStage + 1024;
};
constexpr int STAGES = PairPlan::kStages;

struct PairShared {
    uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int prefix[kMaxTypes + 1];
};

template <class F>
__device__ __forceinline__ uint32_t set_up_pair(PairShared& s, F&& plan) {
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mb::init(&s.full[i], 1);
            mb::init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mb::init(&s.acc_full[i], 1);
            mb::init(&s.acc_empty[i], 8);  // both CTAs' four epilogue warps
        }
        mb::init(&s.drain, 1);
        mb::fence_init();
    }
    if (warp == 2) tc::alloc_pair(&s.tmem, 2 * BN);
    wait_for_previous();
    if (warp == 3) plan();
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();  // the other CTA's barriers are there too
    tc::fence_after();
    return s.tmem;
}

// Both CTAs' copies have landed and rank 0's MMAs retired: TMEM goes back, and
// neither CTA leaves while the other may still signal it.
__device__ __forceinline__ void tear_down_pair(PairShared& s, uint32_t tmem, uint32_t rank) {
    tc::fence_before();
    __syncthreads();
    const int warp = threadIdx.x >> 5;
    if (rank == 0 && warp == 1 && (threadIdx.x & 31) == 0) tc::commit_pair(&s.drain);
    if (warp == 1 && (threadIdx.x & 31) == 0) mb::wait(&s.drain, 0, &g_error, 56);
    __syncthreads();
    tc::cluster_sync();
    tc::fence_after();
    if (warp == 2) tc::dealloc_pair(tmem, 2 * BN);
    tc::cluster_sync();
}

template <bool A_OUTER, bool B_OUTER>
__device__ __forceinline__ void stage_mmas_pair(uint32_t stage, uint32_t acc, uint32_t id, bool first) {
#pragma unroll
    for (int k = 0; k < tc::kInner / 16; ++k)
        tc::mma_pair(acc, A_OUTER ? tc::desc_outer(stage, k) : tc::desc_inner(stage, k),
                     B_OUTER ? tc::desc_outer(stage + PairPlan::kA, k) : tc::desc_inner(stage + PairPlan::kA, k), id,
                     !first || k > 0);
}

// ── rows kernel ──────────────────────────────────────────────────────────
struct RowsPair {
    int64_t M, K;
    int types, tiles_n;
    const int32_t* offsets;
};

template <class T, bool TRANS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    typed_rows_pair_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mw,
                           const RowsPair g, const RowsOut<T> out) {
    constexpr uint32_t ID = tc::idesc(is_bf16<T>(), false, !TRANS, kRows, BN);
    extern __shared__ uint8_t raw[];
    __shared__ PairShared s;
    __shared__ T stage_out[8][stage_bytes<T>() / sizeof(T)];
    const uint32_t ring = (mb::smem_u32(raw) + 1023) & ~1023u;
    const uint32_t rank = tc::cluster_rank();
    const uint32_t tmem = set_up_pair(s, [&] { scan_types(g.offsets, g.types, g.M, kRows, s.prefix); });
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tiles = static_cast<int64_t>(s.prefix[g.types]) * g.tiles_n;
    const int64_t first = blockIdx.x / 2, step = gridDim.x / 2;
    const int KB = static_cast<int>((g.K + tc::kInner - 1) / tc::kInner);

    if (warp == 0) {
        if (lane == 0) {
            int64_t i = 0;
            bool ok = true;
            for (int64_t tile = first; tile < tiles && ok; tile += step) {
                const int p = static_cast<int>(tile / g.tiles_n);
                const int n0 = static_cast<int>(tile % g.tiles_n) * BN + static_cast<int>(rank) * HN;
                const int t = find_type(s.prefix, g.types, p);
                const int row0 = clamp_row(g.offsets[t], g.M) + (p - s.prefix[t]) * kRows + static_cast<int>(rank) * BM;
                for (int kb = 0; kb < KB; ++kb, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (i >= STAGES && !(ok = mb::wait(&s.empty[st], (i / STAGES - 1) & 1, &g_error, 51))) break;
                    const uint32_t a = ring + st * PairPlan::kStage, b = a + PairPlan::kA;
                    // rank 0 expects both CTAs' bytes (a remote arrival would wait
                    // for this thread's earlier operations: 0.6 us a stage)
                    const uint32_t bar = tc::in_rank(&s.full[st], 0);
                    if (rank == 0) mb::arrive_expect_tx(&s.full[st], 2 * PairPlan::kStage);
                    tc::tma3_pair(a, &ma, kb * tc::kInner, row0, 0, bar);
                    if (TRANS) {
                        tc::tma3_pair(b, &mw, kb * tc::kInner, n0, t, bar);
                    } else {
#pragma unroll
                        for (int c = 0; c < HN / 64; ++c)
                            tc::tma3_pair(b + c * tc::kChunkBytes, &mw, n0 + c * 64, kb * tc::kInner, t, bar);
                    }
                }
            }
            // Every copy issued must have landed before the CTA may exit: the
            // MMAs that read a stage free it.  (After a wait that ran out too:
            // each of these is bounded by itself.)
            for (int64_t j = i > STAGES ? i - STAGES : 0; j < i; ++j)
                mb::wait(&s.empty[j % STAGES], (j / STAGES) & 1, &g_error, 52);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int64_t i = 0;
            int local = 0;
            bool ok = true;
            for (int64_t tile = first; tile < tiles && ok; tile += step, ++local) {
                const int acc = local & 1;
                if (local >= 2 && !(ok = tc::wait_cluster(&s.acc_empty[acc], (local / 2 - 1) & 1, &g_error, 53))) break;
                tc::fence_after();
                for (int kb = 0; kb < KB; ++kb, ++i) {
                    const int st = static_cast<int>(i % STAGES);
                    if (!(ok = tc::wait_cluster(&s.full[st], (i / STAGES) & 1, &g_error, 54))) break;
                    tc::fence_after();
                    stage_mmas_pair<false, !TRANS>(ring + st * PairPlan::kStage, tmem + acc * BN, ID, kb == 0);
                    tc::commit_pair(&s.empty[st]);
                }
                if (ok) tc::commit_pair(&s.acc_full[acc]);
            }
        }
    } else if (warp >= 4) {
        const int acc = (warp - 4) >> 2, q = warp & 3;
        const uint32_t freed = tc::in_rank(&s.acc_empty[acc], 0);
        int local = acc;
        for (int64_t tile = first + acc * step; tile < tiles; tile += 2 * step, local += 2) {
            const int p = static_cast<int>(tile / g.tiles_n);
            const int t = find_type(s.prefix, g.types, p);
            const int64_t row0 = clamp_row(g.offsets[t], g.M) + static_cast<int64_t>(p - s.prefix[t]) * kRows +
                                 rank * BM + q * 32;
            const int64_t left = clamp_row(g.offsets[t + 1], g.M) - row0;
            const bool ok = mb::wait(&s.acc_full[acc], (local / 2) & 1, &g_error, 55);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::fence_after();
            finish_rows<T, BN, true>(tmem + acc * BN + (static_cast<uint32_t>(q * 32) << 16), out, t, row0,
                                     left < 0 ? 0 : (left < 32 ? static_cast<int>(left) : 32), tile % g.tiles_n * BN,
                                     stage_out[warp - 4]);
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::arrive_at(freed);
        }
    }
    tear_down_pair(s, tmem, rank);
}

// A grid of pairs, at most one CTA per SM.
unsigned pair_grid(int64_t items) {
    return static_cast<unsigned>(2 * std::min<int64_t>(items, num_sms() / 2));
}

template <class K, class... A>
void run_pairs(const char* name, K kern, int64_t items, cudaStream_t s, A... args) {
    TG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(PairPlan::kBytes)));
    launch_dependent(name, kern, dim3(pair_grid(items)), dim3(kThreads), PairPlan::kBytes, s, args...);
}

}  // namespace

template <class T, bool TRANS>
void typed_rows_pair(const RowsArgs<T>& a, const TmaMatrix<T>& A, const TmaMatrix<T>& W, cudaStream_t s) {
    const int64_t wr = TRANS ? a.N : a.K, wc = TRANS ? a.K : a.N;
    const CUtensorMap ma = tma_map(A, 1, a.M, a.K, BM), mw = tma_map(W, a.types, wr, wc, TRANS ? HN : 64);
    const RowsOut<T> out{a.N, a.bias, a.act, a.alpha, a.C, a.ldc, store_mode(a.C, a.ldc * 2), a.saved, a.r8};
    const RowsPair g{a.M, a.K, a.types, static_cast<int>(ceil_div(a.N, BN)), a.offsets};
    run_pairs("typed_rows_pair", typed_rows_pair_kernel<T, TRANS>,
              (a.M / kRows + std::min<int64_t>(a.types, a.M)) * g.tiles_n, s, ma, mw, g, out);
}

#define TG_TYPED_PAIR(T)                                                                                  \
    template void typed_rows_pair<T, false>(const RowsArgs<T>&, const TmaMatrix<T>&, const TmaMatrix<T>&, \
                                            cudaStream_t);                                                \
    template void typed_rows_pair<T, true>(const RowsArgs<T>&, const TmaMatrix<T>&, const TmaMatrix<T>&,  \
                                           cudaStream_t);
TG_TYPED_PAIR(__nv_bfloat16)
TG_TYPED_PAIR(__half)

int typed_pair_take_error() { return take_error(); }

}  // namespace tg

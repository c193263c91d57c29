// ============================================================================
//  distill.cu -- the distillation loss against a teacher's best logits of each
//  row, and its gradient, in one call.
//
//      q = softmax(t / T) over the teacher's k classes c_i of the row
//      p = softmax(z / T) over all classes
//      loss = T^2 sum_i q_i (log q_i - log p_{c_i})
//      dz_j = w T (p_j - sum over i with c_i = j of q_i)
//
//  The gradient needs the row's sum before its first value, and the row's
//  scores twice: the second time they come from shared memory (narrow rows) or
//  L2 (wide ones), so HBM sees them once.  The teacher's classes are put right
//  after the row's p: each is computed again from its score, less its q.
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
    float temperature;
    const float* weights;  // nullable
    float* loss;
};

// The teacher's entry i of a row: a class outside the row is none (-1).
template <class U>
__device__ __forceinline__ int teacher_class(const DistillArgs& a, int64_t row, int i) {
    const int c = class_at(a.classes, row * a.ldc + i, a.wide_classes);
    return c < a.n ? c : -1;
}
template <class U>
__device__ __forceinline__ float teacher_logit(const DistillArgs& a, int64_t row, int i) {
    return to_f32(static_cast<const U*>(a.teacher)[row * a.ldt + i]);
}

// One row's teacher in shared memory.
struct Teacher {
    int* c;      // the classes, -1 for none
    float* q;    // their probabilities, 0 for none
    float* sum;  // of the probabilities: 1, or 0 without any
};

// Fills `t` with W lanes; each lane's part of sum q (log q) is returned.
template <class U, int W>
__device__ __forceinline__ float read_teacher(const DistillArgs& a, int64_t row, int lane, const Teacher& t) {
    const float c = __fdiv_rn(1.0f, a.temperature);
    float most = -INFINITY;
    for (int i = lane; i < a.k; i += W) {
        const int j = teacher_class<U>(a, row, i);
        const float v = j >= 0 ? teacher_logit<U>(a, row, i) : -INFINITY;
        t.c[i] = v == -INFINITY ? -1 : j;
        t.q[i] = v;
        most = max_nan(most, v);
    }
    most = reduce_max<W>(most);
    float s = 0.0f;
    for (int i = lane; i < a.k; i += W) s = __fadd_rn(s, t.c[i] >= 0 ? expf(distance(t.q[i], most, c)) : 0.0f);
    s = reduce_sum<float, W>(s);
    const float log_s = logf(s);
    float entropy = 0.0f;
    for (int i = lane; i < a.k; i += W) {
        float q = 0.0f;
        if (t.c[i] >= 0) {
            const float l = __fsub_rn(distance(t.q[i], most, c), log_s);
            q = expf(l);
            if (q != 0.0f) entropy = fmaf(q, l, entropy);
        }
        t.q[i] = q;
    }
    if (lane == 0) *t.sum = most == -INFINITY ? 0.0f : 1.0f;
    return entropy;
}

// log p of a score in natural units (the row's maximum m, log of its sum);
// NaN in a row without any score above -inf.
__device__ __forceinline__ float log_p(float z, float m, float log_s, float c) {
    return __fsub_rn(__fmul_rn(__fsub_rn(z, m), c), log_s);
}

struct RowScale {
    float m, c, log_s, w;  // origin, factor and log of the sum in the exponential's units; w T, 0 for rows without gradient
};
template <bool FAST>
__device__ __forceinline__ RowScale row_scale(const DistillArgs& a, int64_t row, const Soft& s, float sum_q) {
    RowScale r;
    r.m = origin(s.m);
    r.c = __fdiv_rn(FAST ? kLog2e : 1.0f, a.temperature);
    r.log_s = s.m == -INFINITY ? 0.0f : __fmul_rn(logf(s.s), FAST ? kLog2e : 1.0f);
    r.w = sum_q == 0.0f || s.m == -INFINITY ? 0.0f : __fmul_rn(a.temperature, a.weights ? a.weights[row] : 1.0f);
    return r;
}
template <bool FAST>
__device__ __forceinline__ float prob(float z, const RowScale& r) {
    return expo<FAST>(max_nan(__fsub_rn(__fmul_rn(__fsub_rn(z, r.m), r.c), r.log_s), -200.0f));
}
// The gradient at the teacher's entry i, whose score is z: where the class
// occurs more than once the first entry answers for all (false for the others).
template <bool FAST>
__device__ __forceinline__ bool entry_grad(const Teacher& t, int i, float z, const RowScale& r, int k, float& y) {
    const int c = t.c[i];
    for (int j = 0; j < i; ++j)
        if (t.c[j] == c) return false;
    float q = t.q[i];
    for (int j = i + 1; j < k; ++j)
        if (t.c[j] == c) q = __fadd_rn(q, t.q[j]);
    y = __fmul_rn(r.w, __fsub_rn(prob<FAST>(z, r), q));
    return true;
}

// ── narrow rows ──────────────────────────────────────────────────────────
template <class T, class U, int LPR, int E, bool GRAD>
__global__ void __launch_bounds__(kNarrowThreads) distill_narrow_kernel(const DistillArgs a, const T* x, int64_t ldx, T* dx,
                                                                        int64_t lddx, int stage) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int RPB = kNarrowThreads / LPR;
    extern __shared__ __align__(16) uint8_t sh[];
    wait_for_previous();
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    int* room = reinterpret_cast<int*>(sh + stage) + sub * (2 * a.k + 1);
    const Teacher t{room, reinterpret_cast<float*>(room + a.k), reinterpret_cast<float*>(room + 2 * a.k)};
    const float cn = __fdiv_rn(1.0f, a.temperature), c = __fdiv_rn(FAST ? kLog2e : 1.0f, a.temperature);
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * RPB; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * RPB) {
        const int rows = a.rows - r0 < RPB ? static_cast<int>(a.rows - r0) : RPB;
        const int64_t row = r0 + (sub < rows ? sub : 0);
        T* st = stage_in(sh, x, ldx, r0, rows, a.n);
        float loss = read_teacher<U, LPR>(a, row, lane, t);
        __syncthreads();
        T* p = st + (sub < rows ? sub : 0) * a.n;
        float z[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = lane + i * LPR;
            z[i] = j < a.n ? to_f32(p[j]) : -INFINITY;
        }
        Soft s;
        add_scores<FAST, false>(s, z, c);
        lanes_soft<FAST, false, LPR>(s, c);
        const float log_s = logf(s.s);
        for (int i = lane; i < a.k; i += LPR)
            if (t.q[i] != 0.0f) loss = fmaf(-t.q[i], log_p(to_f32(p[t.c[i]]), s.m, log_s, cn), loss);
        loss = reduce_sum<float, LPR>(loss);
        if (lane == 0 && sub < rows) a.loss[row] = __fmul_rn(__fmul_rn(a.temperature, a.temperature), loss);
        if constexpr (GRAD) {
            const RowScale r = row_scale<FAST>(a, row, s, *t.sum);
            __syncwarp();
            if (sub < rows) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const int j = lane + i * LPR;
                    if (j < a.n) p[j] = from_f32<T>(r.w == 0.0f ? 0.0f : __fmul_rn(r.w, prob<FAST>(z[i], r)));
                }
            }
            __syncwarp();
            if (sub < rows && r.w != 0.0f) {
                const T* from = x + row * ldx;
                float y;
                for (int i = lane; i < a.k; i += LPR)
                    if (t.c[i] >= 0 && entry_grad<FAST>(t, i, to_f32(from[t.c[i]]), r, a.k, y)) p[t.c[i]] = from_f32<T>(y);
            }
            __syncthreads();
            stage_out(st, dx, lddx, r0, rows, a.n);
        }
        __syncthreads();
    }
}

// ── wide rows ────────────────────────────────────────────────────────────
template <class T, class U, int NT, bool GRAD>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_wide_kernel(const DistillArgs a, const T* x, int64_t ldx, T* dx,
                                                                     int64_t lddx) {
    constexpr bool FAST = sizeof(T) == 2;
    constexpr int V = kVec<T>;
    __shared__ SoftShared soft;
    __shared__ SoftCell mine[2];  // this CTA's state, of even and odd rounds
    __shared__ int tc[kMaxTop];
    __shared__ float tq[kMaxTop];
    __shared__ float tsum;
    const Teacher t{tc, tq, &tsum};
    wait_for_previous();
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks());
    const int64_t clusters = gridDim.x / ranks;
    const float cn = __fdiv_rn(1.0f, a.temperature), c = __fdiv_rn(FAST ? kLog2e : 1.0f, a.temperature);
    int round = 0;
    for (int64_t row = blockIdx.x / ranks; row < a.rows; row += clusters, ++round) {
        float loss = 0.0f;
        if (threadIdx.x < 32) loss = read_teacher<U, 32>(a, row, threadIdx.x, t);
        const Part<T> p(x + row * ldx, a.n, rank, ranks);
        Soft s = scan_part<T, NT, 4, false>(p, c);
        if (threadIdx.x < p.extra) {
            const float z[1] = {to_f32(p.row[p.extra_column(threadIdx.x)])};
            add_scores<FAST, false>(s, z, c);
        }
        block_soft<FAST, false, NT>(s, c, soft);
        if (ranks > 1) {
            if (threadIdx.x == 0) mine[round & 1].set(s);
            cluster.sync();
            s = Soft{};
            if (threadIdx.x % 32 < ranks) s = cluster.map_shared_rank(&mine[round & 1], threadIdx.x % 32)->get();
            lanes_soft<FAST, false, 32>(s, c);
        }
        if (rank == 0 && threadIdx.x < 32) {
            const float log_s = logf(s.s);
            for (int i = threadIdx.x; i < a.k; i += 32)
                if (t.q[i] != 0.0f) loss = fmaf(-t.q[i], log_p(to_f32(p.row[t.c[i]]), s.m, log_s, cn), loss);
            loss = reduce_sum<float, 32>(loss);
            if (threadIdx.x == 0) a.loss[row] = __fmul_rn(__fmul_rn(a.temperature, a.temperature), loss);
        }
        if constexpr (GRAD) {
            T* out = dx + row * lddx;
            const RowScale r = row_scale<FAST>(a, row, s, *t.sum);
            const bool aligned = (reinterpret_cast<uintptr_t>(out + p.head) & 15) == 0;
            const auto grad = [&](float z) { return r.w == 0.0f ? 0.0f : __fmul_rn(r.w, prob<FAST>(z, r)); };
            for_vectors<T, NT, 4>(p, [&](int64_t v, float (&z)[V]) {
#pragma unroll
                for (int j = 0; j < V; ++j) z[j] = grad(z[j]);
                if (aligned) store_v<T, V>(out + p.column(v), z);
                else store_any<T, V>(out + p.column(v), z);
            });
            if (threadIdx.x < p.extra) {
                const int j = p.extra_column(threadIdx.x);
                out[j] = from_f32<T>(grad(to_f32(p.row[j])));
            }
            __syncthreads();  // the block's p are written
            if (threadIdx.x < a.k && r.w != 0.0f) {
                const int j = t.c[threadIdx.x];
                const bool here = j >= 0 && (j < p.head || j >= p.tail
                                                 ? rank == 0
                                                 : (j - p.head) / V >= p.v0 && (j - p.head) / V < p.v1);
                float y;
                if (here && entry_grad<FAST>(t, threadIdx.x, to_f32(p.row[j]), r, a.k, y)) out[j] = from_f32<T>(y);
            }
        }
        __syncthreads();
    }
    if (ranks > 1) cluster.sync();  // no CTA leaves while its state may be read
}

template <class T, class U>
void distill(const DistillArgs& a, const T* x, int64_t ldx, T* dx, int64_t lddx, cudaStream_t s) {
    if (a.n <= kNarrow) {
        by_narrow(a.n, [&](auto lpr, auto e) {
            constexpr int LPR = decltype(lpr)::value, E = decltype(e)::value, RPB = kNarrowThreads / LPR;
            auto kern = dx ? distill_narrow_kernel<T, U, LPR, E, true> : distill_narrow_kernel<T, U, LPR, E, false>;
            const int stage = static_cast<int>((RPB * a.n * sizeof(T) + 32 + 15) / 16 * 16);
            const size_t bytes = stage + RPB * (2 * a.k + 1) * sizeof(float);
            if (bytes > 48 * 1024) TG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
            launch_dependent("distill_loss", kern,
                             dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(a.rows, RPB), num_sms() * 16))),
                             dim3(kNarrowThreads), bytes, s, a, x, ldx, dx, lddx, stage);
        });
        return;
    }
    const int ranks = row_ranks(a.rows, a.n, 4096);
    const auto go = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        const int64_t clusters = std::min<int64_t>(a.rows, std::max<int64_t>(1, int64_t(num_sms()) * (1024 / NT) / ranks));
        auto kern = dx ? distill_wide_kernel<T, U, NT, true> : distill_wide_kernel<T, U, NT, false>;
        launch_clusters("distill_loss", kern, clusters, ranks, NT, 0, s, a, x, ldx, dx, lddx);
    };
    if (a.n / ranks <= 8192) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 512>{});
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
        if (!(temperature > 0.0f && temperature <= 3.0e38f))
            invalid(std::string(fn) + ": temperature must be positive and finite");
        const DistillArgs a{rows, static_cast<int>(classes), static_cast<int>(k), top_classes, class_bytes == 8, ld_classes,
                            top_logits, ld_logits, temperature, weights, loss};
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

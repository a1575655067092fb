// Distillation from a teacher's top logits: the loss of each row and the gradient
// of the student's logits, from one reading of the row.
//
// A row has V student logits z, K teacher entries (id, u), a weight w and the
// temperature tau:
//   p = softmax(u / tau) over the valid entries,  q = softmax(z / tau) over V,
//   loss = w tau^2 sum_k p_k (log p_k - log q[id_k]),
//   dz_v = w tau (q_v - P_v),  P_v = sum of p_k with id_k = v.
// Exponentials are 2^((z - max) log2(e) / tau): the difference first, so that their error
// stays that of the difference however large the logits are; sums are float32.  A NaN or
// +inf logit makes its row NaN through the sum; a row of -inf alone has q = 0.  Repeated
// ids: every entry forms the whole P of its id, so that all of them write the same value.
#include "train_common.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace cresso {

struct DistillArgs {
    const void *ids, *teacher;
    const float* weight;
    int64_t vocab, stride;
    int id_bytes, teacher_dtype, k;
    float tau;
};

// The teacher's side of a row in shared memory.
struct TopList {
    int id[CRESSO_TRAIN_MAX_TOP];   // -1: not valid
    float p[CRESSO_TRAIN_MAX_TOP];  // teacher probability
    float z[CRESSO_TRAIN_MAX_TOP];  // student logit at the id
    float entropy;                  // sum of p log p
    int any;                        // a valid entry exists
};

constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {  // relative error 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Fills the list with one warp; the block sees it after its next barrier.
template <typename T>
__device__ __forceinline__ void load_teacher(const DistillArgs& a, int64_t t, const T* row, TopList& top) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int k = lane; k < a.k; k += 32) {
        const int64_t id = load_id(a.ids, a.id_bytes, t * a.k + k);
        const float u = load_any(a.teacher, a.teacher_dtype, t * a.k + k);
        const bool valid = id >= 0 && id < a.vocab && u != -INFINITY;
        top.id[k] = valid ? (int)id : -1;
        top.p[k] = u;
        top.z[k] = valid ? to_float(row[id]) : 0.0f;
        if (valid) m = fmaxf(m, u);
    }
    m = warp_max(m);
    const float inv_tau = 1.0f / a.tau;
    float s = 0.0f;
    bool valid_here = false;
    for (int k = lane; k < a.k; k += 32) {
        if (top.id[k] < 0) continue;
        valid_here = true;
        s += expf((top.p[k] - m) * inv_tau);
    }
    const bool any = __any_sync(0xffffffffu, valid_here);
    s = warp_sum(s);
    const float log_s = logf(s);
    float entropy = 0.0f;
    for (int k = lane; k < a.k; k += 32) {
        const float lp = (top.p[k] - m) * inv_tau - log_s;
        const float p = top.id[k] >= 0 ? expf(lp) : 0.0f;
        if (p != 0.0f) entropy += p * lp;
        top.p[k] = p;
    }
    entropy = warp_sum(entropy);
    if (lane == 0) {
        top.entropy = entropy;
        top.any = any;
    }
    __syncwarp();
}

// Joins (maximum, sum of exponentials relative to it) over a warp.
__device__ __forceinline__ void join_warp(float& m, float& s, float c2) {
    const float top = warp_max(m);
    // a part without a finite maximum holds 0 or NaN and keeps it
    s = warp_sum(s * (m == top ? 1.0f : exp2_fast((m - top) * c2)));
    m = top;
}

// Loss of the row from its maximum and sum, and the entries' own gradients; one warp for the
// loss, `threads` threads for the gradients of the ids in [v0, v1).
__device__ __forceinline__ float row_loss(const DistillArgs& a, const TopList& top, float w, float m, float s) {
    const float inv_tau = 1.0f / a.tau, log_s = s == 0.0f ? 0.0f : logf(s);
    float cross = 0.0f;
    for (int k = threadIdx.x & 31; k < a.k; k += 32)
        if (top.p[k] != 0.0f) cross += top.p[k] * ((top.z[k] - m) * inv_tau - log_s);
    return w * a.tau * a.tau * (top.entropy - warp_sum(cross));
}
template <typename T>
__device__ __forceinline__ void top_gradients(const DistillArgs& a, const TopList& top, T* out, int64_t v0, int64_t v1,
                                              float c, float c2, float m, float inv_s) {
    for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
        const int id = top.id[k];
        if (id < v0 || id >= v1) continue;
        float p = 0.0f;
        for (int j = 0; j < a.k; ++j) p += top.id[j] == id ? top.p[j] : 0.0f;
        out[id] = from_float<T>(c * (exp2_fast((top.z[k] - m) * c2) * inv_s - p));
    }
}

// ------------------------------------------------------- rows in registers ---
//
// A row is cut into the 16-byte words of its memory and lies in the registers of a block, NV
// words a thread, or of a cluster of blocks: read once, written once.  Each thread takes the maximum of its logits and the sum
// relative to it, which are joined over warps, block and cluster in one exchange.
constexpr int kDistillThreads = 512;
constexpr int kDistillVecs = 8;

template <typename T>
constexpr int kWordLogits = 16 / (int)sizeof(T);

// Maximum of the logits of a word; NaN is left out.
template <typename T>
__device__ __forceinline__ float word_max(const uint32_t (&w)[4]) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])),
                     fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
    } else {
        using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
        auto as2 = [&](int i) { return *reinterpret_cast<const T2*>(&w[i]); };
        const T2 v = __hmax2(__hmax2(as2(0), as2(1)), __hmax2(as2(2), as2(3)));
        const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(&v));
        return fmaxf(f.x, f.y);
    }
}

// f(i, pair): the logits of a word two at a time.
template <typename T, typename F>
__device__ __forceinline__ void word_pairs(const uint32_t (&w)[4], F f) {
    if constexpr (sizeof(T) == 4) {
        f(0, make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])));
        f(1, make_float2(__uint_as_float(w[2]), __uint_as_float(w[3])));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f(i, unpack2<T>(w[i]));
    }
}

template <typename T, int NV>
__global__ void __launch_bounds__(NV == kDistillVecs ? 1024 : kDistillThreads)
    distill_kernel(DistillArgs a, const T* z, float* __restrict__ loss, T* grad, int cluster) {
    constexpr int N = kWordLogits<T>;
    __shared__ TopList top;
    __shared__ float2 warp_part[32], block_part;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    const int64_t t = blockIdx.x / cluster;
    const int rank = (int)(blockIdx.x % cluster);
    const T* row = z + t * a.stride;
    T* out = grad != nullptr ? grad + t * a.vocab : nullptr;
    const float w = a.weight != nullptr ? a.weight[t] : 1.0f;
    // the whole words of the row, this block's share of them; up to N - 1 logits before them and
    // behind them are left to single threads of the first and the last block
    const int vocab = (int)a.vocab;
    const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / sizeof(T)));
    const int words = (vocab - head) / N, share = (words + cluster - 1) / cluster;
    const int first = min(words, rank * share), count = min(words - first, share);
    const int tail = head + words * N;
    int edge = -1;
    if (rank == 0 && tid < head) edge = tid;
    if (rank == cluster - 1 && tid >= N && tid - N < vocab - tail) edge = tail + tid - N;
    const T* body = row + head + first * N;
    const bool live = w != 0.0f;
    uint32_t x[NV][4];
    float edge_x = -INFINITY;
    if (live) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
            const int i = v * threads + tid;
            const uint4 q = i < count ? reinterpret_cast<const uint4*>(body)[i] : make_uint4(kNone, kNone, kNone, kNone);
            x[v][0] = q.x;
            x[v][1] = q.y;
            x[v][2] = q.z;
            x[v][3] = q.w;
        }
        if (edge >= 0) edge_x = to_float(row[edge]);
        if (warp == 0) load_teacher<T>(a, t, row, top);
    }
    const float c2 = kLog2E / a.tau;
    float m = -INFINITY, s = 0.0f;
    if (live) {
#pragma unroll
        for (int v = 0; v < NV; ++v) m = fmaxf(m, word_max<T>(x[v]));
        m = fmaxf(m, edge_x);
        const float base = m == -INFINITY ? 0.0f : -m;
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            word_pairs<T>(x[v], [&](int, float2 f) {
                f = mul2(add2(f, make_float2(base, base)), make_float2(c2, c2));
                sum = add2(sum, make_float2(exp2_fast(f.x), exp2_fast(f.y)));
            });
        s = sum.x + sum.y + exp2_fast((edge_x + base) * c2);
        join_warp(m, s, c2);
    }
    if (lane == 0) warp_part[warp] = make_float2(m, s);
    __syncthreads();
    m = lane < warps ? warp_part[lane].x : -INFINITY;
    s = lane < warps ? warp_part[lane].y : 0.0f;
    join_warp(m, s, c2);
    if (cluster > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group group = cg::this_cluster();
        if (tid == 0) block_part = make_float2(m, s);
        group.sync();
        const float2 part = lane < cluster ? *group.map_shared_rank(&block_part, lane) : make_float2(-INFINITY, 0.0f);
        m = part.x;
        s = part.y;
        join_warp(m, s, c2);
    }
    const bool any = live && top.any;
    if (m == -INFINITY) m = 0.0f;
    if (rank == 0 && warp == 0) {
        const float l = any ? row_loss(a, top, w, m, s) : 0.0f;
        if (lane == 0) loss[t] = l;
    }
    if (out != nullptr) {
        const float inv_s = s == 0.0f ? 0.0f : 1.0f / s, c = any ? w * a.tau : 0.0f, ci = c * inv_s;
        T* out_body = out + head + first * N;
        const bool aligned = (reinterpret_cast<uintptr_t>(out_body) & 15) == 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = v * threads + tid;
            if (i >= count) break;
            uint32_t y[4] = {0, 0, 0, 0};
            if (any)
                word_pairs<T>(x[v], [&](int j, float2 f) {
                    f = mul2(add2(f, make_float2(-m, -m)), make_float2(c2, c2));
                    f = mul2(make_float2(exp2_fast(f.x), exp2_fast(f.y)), make_float2(ci, ci));
                    if constexpr (sizeof(T) == 4) {
                        y[2 * j] = __float_as_uint(f.x);
                        y[2 * j + 1] = __float_as_uint(f.y);
                    } else {
                        y[j] = pack2<T>(f.x, f.y);
                    }
                });
            if (aligned) {
                reinterpret_cast<uint4*>(out_body)[i] = make_uint4(y[0], y[1], y[2], y[3]);
            } else {  // rows of logits that lie further apart than those of the gradient
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if constexpr (sizeof(T) == 4)
                        reinterpret_cast<uint32_t*>(out_body)[i * N + j] = y[j];
                    else
                        reinterpret_cast<uint16_t*>(out_body)[i * N + j] = (uint16_t)(y[j / 2] >> (16 * (j & 1)));
            }
        }
        if (edge >= 0) out[edge] = from_float<T>(any ? ci * exp2_fast((edge_x - m) * c2) : 0.0f);
        if (any) {
            __syncthreads();
            const int v0 = rank == 0 ? 0 : head + first * N, v1 = rank == cluster - 1 ? vocab : head + (first + count) * N;
            top_gradients<T>(a, top, out, v0, v1, c, c2, m, inv_s);
        }
    }
    if (cluster > 1) cooperative_groups::this_cluster().sync();  // a peer may still read this block's part
}

// ------------------------------------------------------------- longer rows ---
//
// A row beyond the registers of a cluster of eight blocks: one block reads it three times.
template <typename T>
__global__ void __launch_bounds__(1024) distill_long_kernel(DistillArgs a, const T* z, float* __restrict__ loss,
                                                            T* grad) {
    __shared__ TopList top;
    __shared__ float sh[32];
    const int64_t t = blockIdx.x;
    const T* row = z + t * a.stride;
    T* out = grad != nullptr ? grad + t * a.vocab : nullptr;
    const float w = a.weight != nullptr ? a.weight[t] : 1.0f;
    if (w != 0.0f && threadIdx.x < 32) load_teacher<T>(a, t, row, top);
    __syncthreads();
    if (w == 0.0f || !top.any) {
        if (out != nullptr)
            for (int64_t v = threadIdx.x; v < a.vocab; v += blockDim.x) out[v] = from_float<T>(0.0f);
        if (threadIdx.x == 0) loss[t] = 0.0f;
        return;
    }
    const float c2 = kLog2E / a.tau;
    float m = -INFINITY;
    for (int64_t v = threadIdx.x; v < a.vocab; v += blockDim.x) m = fmaxf(m, to_float(row[v]));
    m = block_max(m, sh);
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f;
    for (int64_t v = threadIdx.x; v < a.vocab; v += blockDim.x) s += exp2_fast((to_float(row[v]) - m) * c2);
    s = block_sum(s, sh);
    if (threadIdx.x < 32) {
        const float l = row_loss(a, top, w, m, s);
        if (threadIdx.x == 0) loss[t] = l;
    }
    if (out == nullptr) return;
    const float inv_s = s == 0.0f ? 0.0f : 1.0f / s, c = w * a.tau;
    for (int64_t v = threadIdx.x; v < a.vocab; v += blockDim.x)
        out[v] = from_float<T>(c * inv_s * exp2_fast((to_float(row[v]) - m) * c2));
    __syncthreads();
    top_gradients<T>(a, top, out, 0, a.vocab, c, c2, m, inv_s);
}

// Threads and words of a thread for a block's share of a row.
struct DistillPlan {
    int cluster, threads, vecs;  // cluster 0: the kernel for longer rows
};
static DistillPlan distill_plan(int64_t n, int64_t words) {
    DistillPlan p{1, kDistillThreads, 1};
    while (p.cluster < 8 && words > (int64_t)p.cluster * kDistillThreads * kDistillVecs) p.cluster *= 2;
    if (words > (int64_t)p.cluster * kDistillThreads * kDistillVecs) {
        p.threads = 1024;
        if (words > (int64_t)p.cluster * p.threads * kDistillVecs) p.cluster = 0;
        p.vecs = kDistillVecs;
        return p;
    }
    // few rows: more blocks a row, as long as each of their threads has a word
    while (p.cluster < 8 && n * p.cluster < 2 * 148 && words >= 2 * p.cluster * kDistillThreads) p.cluster *= 2;
    const int64_t share = ceil_div(words, p.cluster);
    while (p.threads > 64 && share <= p.threads / 2) p.threads /= 2;
    while ((int64_t)p.vecs * p.threads < share) p.vecs *= 2;
    return p;
}

}  // namespace cresso

using namespace cresso;

extern "C" {

int cresso_distill(const void* logits, int64_t dtype, int64_t n, int64_t vocab, int64_t logits_stride, const void* ids,
                   int64_t id_bytes, const void* teacher, int64_t teacher_dtype, int64_t k, const float* weight,
                   double temperature, float* loss, void* grad, cresso_stream_t stream) {
    CRESSO_REQUIRE(train_dtype_ok(dtype) && train_dtype_ok(teacher_dtype), CRESSO_EUNSUPPORTED,
                   "distill: element types are float32, float16 and bfloat16");
    CRESSO_REQUIRE(id_bytes == 4 || id_bytes == 8, CRESSO_EINVAL, "distill: ids are int32 or int64");
    CRESSO_REQUIRE(n >= 0 && vocab >= 1 && logits_stride >= vocab && k >= 0, CRESSO_EINVAL,
                   "distill: negative size, an empty vocabulary, or row stride below the vocabulary");
    CRESSO_REQUIRE(n <= CRESSO_TRAIN_MAX_ROWS && vocab <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED,
                   "distill: more than 2^31 - 256 rows or logits of a row");
    CRESSO_REQUIRE(k <= CRESSO_TRAIN_MAX_TOP, CRESSO_EUNSUPPORTED, "distill: more than %d teacher entries",
                   (int)CRESSO_TRAIN_MAX_TOP);
    const float tau = (float)temperature;
    CRESSO_REQUIRE(temperature >= 1e-6 && temperature <= 1e6, CRESSO_EINVAL,
                   "distill: temperature must be in [1e-6, 1e6]");
    if (n == 0) return CRESSO_OK;
    CRESSO_REQUIRE(logits != nullptr && loss != nullptr && (k == 0 || (ids != nullptr && teacher != nullptr)),
                   CRESSO_EINVAL, "distill: NULL pointer");
    CRESSO_REQUIRE(grad != logits || logits_stride == vocab, CRESSO_EINVAL,
                   "distill: a gradient in place of the logits needs contiguous rows");
    NvtxRange range("distill n=%lld", (long long)n);
    const DistillArgs a{ids, teacher, weight, vocab, logits_stride, (int)id_bytes, (int)teacher_dtype, (int)k, tau};
    return with_dtype(dtype, [&](auto tz) {
        using T = decltype(tz);
        constexpr int N = kWordLogits<T>;
        const T* z = static_cast<const T*>(logits);
        T* g = static_cast<T*>(grad);
        const cudaStream_t s = (cudaStream_t)stream;
        const DistillPlan p = distill_plan(n, vocab / N);
        if (p.cluster == 0) {
            distill_long_kernel<T><<<(unsigned)n, 1024, 0, s>>>(a, z, loss, g);
            CRESSO_LAUNCHED("distill_long_kernel");
            return (int)CRESSO_OK;
        }
        CRESSO_REQUIRE(n * p.cluster <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED, "distill: too many rows");
        auto launch = [&](auto kernel) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((unsigned)(n * p.cluster));
            cfg.blockDim = dim3((unsigned)p.threads);
            cfg.stream = s;
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = (unsigned)p.cluster;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = p.cluster > 1 ? 1 : 0;
            CRESSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, z, loss, g, p.cluster));
            CRESSO_LAUNCHED("distill_kernel");
            return (int)CRESSO_OK;
        };
        switch (p.vecs) {
            case 1: return launch(distill_kernel<T, 1>);
            case 2: return launch(distill_kernel<T, 2>);
            case 4: return launch(distill_kernel<T, 4>);
            default: return launch(distill_kernel<T, kDistillVecs>);
        }
    });
}

}  // extern "C"

// Distillation from a teacher's top logits: the loss of each row and the gradient
// of the student's logits, from one reading of the row from DRAM.
//
// A row has V student logits z, K teacher entries (id, u), a weight w and the
// temperature tau:
//   p = softmax(u / tau) over the valid entries,  q = softmax(z / tau) over V,
//   loss = w tau^2 sum_k p_k (log p_k - log q[id_k]),
//   dz_v = w tau (q_v - P_v),  P_v = sum of p_k with id_k = v.
// Exponentials are 2^(z c - B) with c = log2(e) / tau and one B for the whole row: a fused
// operation, whose error is that of its result, because the same rounded B stands in the sum,
// in the gradient and in the loss.  B needs no maximum over the row, only a reference near it:
// every warp takes the largest of the first logits it reads, sums relative to that, and the
// parts are joined relative to the largest reference.  The sum is then at least 1; a row whose
// sum leaves (0.5, 1e18) (a later logit about 40 tau above its warp's reference, a row far from
// zero, or a warp without finite logits at first), or whose weight is tiny, is computed again from its
// maximum.  Sums are
// float32; an exponential below 2^-126 counts as zero.  A NaN or +inf logit makes its row NaN
// through the sum; a row of -inf alone has q = 0.  Repeated ids: every entry
// holds the whole P of its id, so that all of them write the same value.
#include "train_common.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace cresso {

struct DistillArgs {
    const void *ids, *teacher;
    const float* weight;
    int64_t vocab, stride;
    int id_bytes, teacher_dtype, k;
    float tau;
};

// The teacher's side of a row in shared memory: k ids (-1: not valid), teacher probabilities,
// their sums over equal ids and student logits at the ids, then the sum of p log p and whether
// a valid entry exists.
struct TopList {
    int* id;
    float *p, *same, *z, *entropy;
    int* any;
    __device__ __forceinline__ TopList(unsigned char* at, int k)
        : id(reinterpret_cast<int*>(at)), p(reinterpret_cast<float*>(at) + k), same(p + k), z(same + k), entropy(z + k),
          any(reinterpret_cast<int*>(entropy + 1)) {}
};
__host__ __device__ constexpr int top_bytes(int k) { return (16 * k + 8 + 15) / 16 * 16; }

// One warp's set of bits that finds ids that may occur twice, and the list of those.
constexpr int kSeenBits = 16384;
struct Seen {
    uint32_t bits[kSeenBits / 32];
    int count, id[CRESSO_TRAIN_MAX_TOP];
};

constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {  // relative error 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Fills the list with one warp; the block sees it after its next barrier.  First the loads, four
// entries a lane in flight together.
template <typename T>
__device__ __forceinline__ void load_teacher(const DistillArgs& a, int64_t t, const T* row, const TopList& top, Seen& seen) {
    const int lane = threadIdx.x & 31;
    const int64_t at = t * a.k;
    float m = -INFINITY;
    for (int i = lane; i < kSeenBits / 32; i += 32) seen.bits[i] = 0;
    if (lane == 0) seen.count = 0;
    for (int k0 = 0; k0 < a.k; k0 += 128) {
        int64_t id[4];
        float u[4], z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = min(k0 + 32 * j + lane, a.k - 1);
            id[j] = load_id(a.ids, a.id_bytes, at + k);
            u[j] = load_any(a.teacher, a.teacher_dtype, at + k);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!(id[j] >= 0 && id[j] < a.vocab && u[j] != -INFINITY)) id[j] = -1;
            z[j] = to_float(row[max(id[j], (int64_t)0)]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + 32 * j + lane;
            if (k >= a.k) break;
            top.id[k] = (int)id[j];
            top.p[k] = u[j];
            top.z[k] = z[j];
            if (id[j] >= 0) m = fmaxf(m, u[j]);
        }
    }
    __syncwarp();
    m = warp_max(m);
    const float inv_tau = 1.0f / a.tau;
    float s = 0.0f;
    bool valid_here = false;
    for (int k = lane; k < a.k; k += 32) {
        const int id = top.id[k];
        if (id < 0) continue;
        valid_here = true;
        s += expf((top.p[k] - m) * inv_tau);
        const uint32_t h = ((uint32_t)id * 2654435769u) >> 18;  // multiplicative hash to kSeenBits
        if (atomicOr(&seen.bits[h >> 5], 1u << (h & 31)) >> (h & 31) & 1u) seen.id[atomicAdd(&seen.count, 1)] = id;
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
        top.same[k] = p;
    }
    entropy = warp_sum(entropy);
    if (lane == 0) {
        *top.entropy = entropy;
        *top.any = any;
    }
    __syncwarp();
    // an id that occurs twice is in seen.id, whatever the order of the insertions was
    const int count = seen.count;
    if (count == 0) return;
    for (int k = lane; k < a.k; k += 32) {
        const int id = top.id[k];
        bool twice = false;
        for (int j = 0; j < count && !twice; ++j) twice = seen.id[j] == id;
        if (id < 0 || !twice) continue;
        float p = 0.0f;
        for (int j = 0; j < a.k; ++j) p += top.id[j] == id ? top.p[j] : 0.0f;
        top.same[k] = p;
    }
    __syncwarp();
}

// Joins (reference, sum relative to it) over the first WIDTH lanes of a warp; all lanes get it.
// The sums are relative to the rounded B of their references, or (FAR) to the maxima themselves,
// whose B may overflow.
template <int WIDTH, bool FAR = false>
__device__ __forceinline__ void join_warp(float& m, float& s, float c2) {
    float top = m;
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // a part without a finite reference holds 0 or NaN and keeps it
    s *= m == top ? 1.0f : exp2_fast(FAR ? (m - top) * c2 : __fmul_rn(m, c2) - __fmul_rn(top, c2));
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    m = __shfl_sync(0xffffffffu, top, 0);
    s = __shfl_sync(0xffffffffu, s, 0);
}

// B's rounding shifts all exponents of a row by up to 2^-24 |B|, which cancels as long as it
// is small.
constexpr float kFar = 16777216.0f;
constexpr float kLargeSum = 1e18f;
// The gradient's factor c / sum is a normal number for |c| from here on; a smaller one would lose
// digits that the large exponentials it meets bring back.
constexpr float kSmallFactor = 1.2e-20f;  // kLargeSum 2^-126

// Loss of the row from its reference m and sum by one warp, and the gradients of the entries' ids in
// [v0, v1) by `threads` threads.
__device__ __forceinline__ float row_loss(const DistillArgs& a, const TopList& top, float w, float c2, float m, float s) {
    // tau log q = z - m - tau log of the sum relative to m, which is s but for the rounding of B; in the
    // logits' units, halved, where a masked logit of the type's lowest value is finite at every
    // temperature, and times w tau, the gradient's factor, which loses nothing beside them
    const float log_s = (s == 0.0f ? 0.0f : logf(s)) - fmaf(m, c2, -__fmul_rn(m, c2)) * kLn2;
    const float half_m = 0.5f * m, half_tau = 0.5f * a.tau;
    float cross = 0.0f;
#pragma unroll 1  // 40 registers for the kernel; unrolled, the float32 form took 56
    for (int k = threadIdx.x & 31; k < a.k; k += 32)
        if (top.p[k] != 0.0f) cross += top.p[k] * (0.5f * top.z[k] - half_m - half_tau * log_s);
    return 2.0f * w * a.tau * (half_tau * *top.entropy - warp_sum(cross));
}
template <typename T>
__device__ __forceinline__ void top_gradients(const DistillArgs& a, const TopList& top, T* out, int threads, int v0, int v1,
                                              float c, float c2, float base, float inv_s) {
    for (int k = threadIdx.x; k < a.k; k += threads) {
        const int id = top.id[k];
        if (id >= v0 && id < v1)
            out[id] = from_float<T>(c * (exp2_fast(fmaf(top.z[k], c2, base)) * inv_s - top.same[k]));
    }
}

// ------------------------------------------------------------------ the rows ---
//
// A row belongs to a block, or to a cluster of blocks that hold a part of it each.  It is cut
// into the 16-byte words of its memory and read twice: once for the sum, from DRAM, and once for
// the gradient, while it is still in L2 (the rows at work at a time are a third of it).  No
// storage on the SM means many blocks an SM, in different phases: their loads overlap the others'
// exponentials, barriers and teacher lists.  One further warp prepares the teacher's list.
// Bound by the concurrency of loads and stores: 4096 rows of 32000 bfloat16 with their gradient take
// 88 us, 495 MB at 5.6 TB/s.  Rows in registers (125 us) or in shared memory with the next row on
// its way (100 us) leave fewer blocks; without any exponential the latter still took 93 us.  Six
// blocks an SM instead of five let rows fall out of L2 (105 us, 94 with five), and four take 76 us
// instead of 71 for 301 rows of 128259 float32.  Five follow from 40 registers a thread, which the
// compiler chooses by itself (-Xptxas -v shows them): asked for by a launch bound of five blocks it
// spilled (73 us), and the form of 64 threads got 72.
constexpr int kDistillThreads = 256;         // without the teacher's warp
// Bytes of a row that a block is given at least.  With the gradient, more of them are in L2 for
// longer and fewer blocks are better: 64 KB.  The loss alone is bound by what a block does before
// and after its part: 128 KB (1023 rows of 100003 float16: 41 us, 49 with 64 KB).
constexpr int64_t kDistillShare = 64 * 1024, kDistillLossShare = 128 * 1024;
constexpr int kDistillCluster = 8;

template <typename T>
constexpr int kWordLogits = 16 / (int)sizeof(T);

// Running maximum of the logits of words; NaN is left out.
template <typename T>
struct WordMax {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 m;
    __device__ __forceinline__ WordMax() {
        const uint32_t none = std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;  // -inf
        m = *reinterpret_cast<const T2*>(&none);
    }
    __device__ __forceinline__ void add(const uint4& w) {
        auto two = [](const uint32_t& v) { return *reinterpret_cast<const T2*>(&v); };
        m = __hmax2(__hmax2(m, __hmax2(two(w.x), two(w.y))), __hmax2(two(w.z), two(w.w)));
    }
    __device__ __forceinline__ float get() const {
        const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(&m));
        return fmaxf(f.x, f.y);
    }
};
template <>
struct WordMax<float> {
    float m = -INFINITY;
    __device__ __forceinline__ void add(const uint4& w) {
        m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(w.x), __uint_as_float(w.y))),
                  fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    }
    __device__ __forceinline__ float get() const { return m; }
};

// f(i, pair): the logits of a word two at a time.
template <typename T, typename F>
__device__ __forceinline__ void word_pairs(const uint4& w, F f) {
    if constexpr (sizeof(T) == 4) {
        f(0, make_float2(__uint_as_float(w.x), __uint_as_float(w.y)));
        f(1, make_float2(__uint_as_float(w.z), __uint_as_float(w.w)));
    } else {
        f(0, unpack2<T>(w.x));
        f(1, unpack2<T>(w.y));
        f(2, unpack2<T>(w.z));
        f(3, unpack2<T>(w.w));
    }
}

// A row's whole words and a block's share of them; up to N - 1 logits before the words and
// behind them are left to single threads of the first and the last block.
struct RowShare {
    int first, count;  // words
    int head, edge;    // logits before the words; the thread's single logit or -1
};
template <typename T>
__device__ __forceinline__ RowShare row_share(const T* row, int vocab, int rank, int log_cluster, int tid) {
    constexpr int N = kWordLogits<T>;
    const int cluster = 1 << log_cluster;
    RowShare r;
    r.head = min(vocab, (int)(((16u - ((uint32_t)reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / sizeof(T)));
    const int words = (vocab - r.head) / N, share = (words + cluster - 1) >> log_cluster, tail = r.head + words * N;
    r.first = min(words, rank * share);
    r.count = min(words - r.first, share);
    r.edge = -1;
    if (rank == 0 && tid < r.head) r.edge = tid;
    if (rank == cluster - 1 && tid >= N && tid - N < vocab - tail) r.edge = tail + tid - N;
    return r;
}

// f(i, get(i)) for the words i, i + THREADS, ... below count; U of them are fetched before
// the first is used.
template <int THREADS, int U, typename G, typename F>
__device__ __forceinline__ void each_word(int i, int count, G get, F f) {
    for (; i + (U - 1) * THREADS < count; i += U * THREADS) {
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = get(i + u * THREADS);
#pragma unroll
        for (int u = 0; u < U; ++u) f(i + u * THREADS, x[u]);
    }
    for (; i < count; i += THREADS) f(i, get(i));
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS + 32)
    distill_kernel(DistillArgs a, const T* z, float* __restrict__ loss, T* grad, int log_cluster) {
    constexpr int N = kWordLogits<T>, warps = THREADS / 32;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float2 warp_part[warps], block_part;
    __shared__ Seen seen;
    const TopList top(smem, a.k);
    const int cluster = 1 << log_cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = (int)a.vocab;
    const bool is_teacher = warp == warps;
    const int rank = (int)blockIdx.x & (cluster - 1);
    const int64_t t = blockIdx.x >> log_cluster;
    const T* row = z + t * a.stride;
    const RowShare r = row_share<T>(row, vocab, rank, log_cluster, tid);
    const uint4* words = reinterpret_cast<const uint4*>(row + r.head + r.first * N);
    T* out = grad != nullptr ? grad + t * a.vocab : nullptr;
    T* body = out + r.head + r.first * N;
    const bool aligned = (reinterpret_cast<uintptr_t>(body) & 15) == 0;
    const float w = a.weight != nullptr ? a.weight[t] : 1.0f;
    const float c2 = kLog2E / a.tau;
    constexpr int U = 4;
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;  // -inf
    uint4 x[U];  // the first words, on their way before the weight is known
    float edge = -INFINITY;
    if (!is_teacher) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            x[u] = tid + u * THREADS < r.count ? words[tid + u * THREADS] : make_uint4(kNone, kNone, kNone, kNone);
        if (r.edge >= 0) edge = to_float(row[r.edge]);
    }
    bool any = false;
    float m = 0.0f, s = 0.0f, far = 0.0f;
    if (w != 0.0f) {
        // with the gradient, the rest of the block's part is sent for at once (94 -> 89 us); the loss
        // alone has more of its part in flight anyway and loses by it
        if (out != nullptr && tid == 0 && r.count > U * THREADS)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(words + U * THREADS),
                         "r"((r.count - U * THREADS) * 16)
                         : "memory");
        if (is_teacher) {
            load_teacher<T>(a, t, row, top, seen);
        } else {
            WordMax<T> first;
#pragma unroll
            for (int u = 0; u < U; ++u) first.add(x[u]);
            m = warp_max(fmaxf(first.get(), edge));
            if (!(fabsf(m * c2) <= kFar)) m = 0.0f;
            const float base = -__fmul_rn(m, c2);
            float2 sum = make_float2(exp2_fast(fmaf(edge, c2, base)), 0.0f);
            auto add = [&](int, const uint4& y) {
                word_pairs<T>(y, [&](int, float2 f) {
                    f = __ffma2_rn(f, make_float2(c2, c2), make_float2(base, base));
                    sum = __fadd2_rn(sum, make_float2(exp2_fast(f.x), exp2_fast(f.y)));
                });
            };
#pragma unroll
            for (int u = 0; u < U; ++u) add(0, x[u]);
            each_word<THREADS, U>(tid + U * THREADS, r.count, [&](int i) { return words[i]; }, add);
            s = warp_sum(sum.x + sum.y);
            if (lane == 0) warp_part[warp] = make_float2(m, s);
        }
        __syncthreads();
        m = lane < warps ? warp_part[lane].x : -INFINITY;
        s = lane < warps ? warp_part[lane].y : 0.0f;
        join_warp<8>(m, s, c2);
        if (cluster > 1) {
            cg::cluster_group group = cg::this_cluster();
            if (tid == 0) block_part = make_float2(m, s);
            group.sync();
            const float2 p = lane < cluster ? *group.map_shared_rank(&block_part, lane) : make_float2(-INFINITY, 0.0f);
            m = p.x;
            s = p.y;
            join_warp<8>(m, s, c2);
        }
        any = *top.any;
        if (any && !(s < kLargeSum && s > 0.5f && (out == nullptr || fabsf(w * a.tau) >= kSmallFactor))) {
            // no usable reference, or a factor that needs the largest exponential to be 1: from the row's
            // maximum
            const T* part = reinterpret_cast<const T*>(words);
            m = -INFINITY;
            s = 0.0f;
            if (!is_teacher) {
                m = edge;
                for (int i = tid; i < r.count * N; i += THREADS) m = fmaxf(m, to_float(part[i]));
                const float from = m == -INFINITY ? 0.0f : m;
                s = exp2_fast((edge - from) * c2);
                for (int i = tid; i < r.count * N; i += THREADS) s += exp2_fast((to_float(part[i]) - from) * c2);
                join_warp<32, true>(m, s, c2);
            }
            __syncthreads();  // the parts of the first exchange have been read
            if (!is_teacher && lane == 0) warp_part[warp] = make_float2(m, s);
            __syncthreads();
            m = lane < warps ? warp_part[lane].x : -INFINITY;
            s = lane < warps ? warp_part[lane].y : 0.0f;
            join_warp<8, true>(m, s, c2);
            if (cluster > 1) {
                cg::cluster_group group = cg::this_cluster();
                group.sync();
                if (tid == 0) block_part = make_float2(m, s);
                group.sync();
                const float2 p = lane < cluster ? *group.map_shared_rank(&block_part, lane) : make_float2(-INFINITY, 0.0f);
                m = p.x;
                s = p.y;
                join_warp<8, true>(m, s, c2);
            }
            if (m == INFINITY) s = NAN;
            far = m == -INFINITY ? 0.0f : m;
            m = 0.0f;
            edge -= far;
            if (is_teacher)
                for (int k = lane; k < a.k; k += 32) top.z[k] -= far;
            __syncthreads();
        }
    }
    const float base = -__fmul_rn(m, c2);
    if (is_teacher) {
        if (rank == 0) {
            const float v = any ? row_loss(a, top, w, c2, m, s) : 0.0f;
            if (lane == 0) loss[t] = v;
        }
    } else if (out != nullptr) {
        const float c = w * a.tau, inv_s = s == 0.0f ? 0.0f : 1.0f / s, ci = c * inv_s;
        if (any && far == 0.0f && aligned) {
            each_word<THREADS, 2>(tid, r.count, [&](int i) { return words[i]; }, [&](int i, const uint4& x) {
                uint32_t o[4];
                word_pairs<T>(x, [&](int j, float2 f) {
                    f = __ffma2_rn(f, make_float2(c2, c2), make_float2(base, base));
                    f = __fmul2_rn(make_float2(exp2_fast(f.x), exp2_fast(f.y)), make_float2(ci, ci));
                    if constexpr (sizeof(T) == 4) {
                        o[2 * j] = __float_as_uint(f.x);
                        o[2 * j + 1] = __float_as_uint(f.y);
                    } else {
                        o[j] = pack2<T>(f.x, f.y);
                    }
                });
                __stcs(reinterpret_cast<uint4*>(body) + i, make_uint4(o[0], o[1], o[2], o[3]));
            });
        } else if (!any && aligned) {
            for (int i = tid; i < r.count; i += THREADS) __stcs(reinterpret_cast<uint4*>(body) + i, make_uint4(0, 0, 0, 0));
        } else {  // rows of logits that lie further apart than those of the gradient, or far ones
            const T* part = reinterpret_cast<const T*>(words);
            for (int i = tid; i < r.count * N; i += THREADS)
                body[i] = from_float<T>(any ? ci * exp2_fast(fmaf(to_float(part[i]) - far, c2, base)) : 0.0f);
        }
        if (r.edge >= 0) out[r.edge] = from_float<T>(any ? ci * exp2_fast(fmaf(edge, c2, base)) : 0.0f);
        if (any) {
            asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");  // the row is written
            const int v0 = rank == 0 ? 0 : r.head + r.first * N;
            const int v1 = rank == cluster - 1 ? vocab : r.head + (r.first + r.count) * N;
            top_gradients<T>(a, top, out, THREADS, v0, v1, c, c2, base, inv_s);
        }
    }
    if (cluster > 1) cg::this_cluster().sync();  // a peer may still read this block's part
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
        // blocks of a row: as many as its length asks for, and more where there are few rows
        const int64_t words = vocab / N;
        int log_cluster = 0;
        while ((1 << log_cluster) < kDistillCluster &&
               (words * 16 > ((g != nullptr ? kDistillShare : kDistillLossShare) << log_cluster) ||
                ((n << log_cluster) < 2 * 148 && words >= (int64_t)(2 << log_cluster) * kDistillThreads)))
            ++log_cluster;
        CRESSO_REQUIRE((n << log_cluster) <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED, "distill: too many rows");
        const bool small = (words >> log_cluster) <= kDistillThreads / 4;
        const auto kernel = small ? distill_kernel<T, kDistillThreads / 4> : distill_kernel<T, kDistillThreads>;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(n << log_cluster));
        cfg.blockDim = dim3((unsigned)(small ? kDistillThreads / 4 : kDistillThreads) + 32);
        cfg.dynamicSmemBytes = (size_t)top_bytes(a.k);
        cfg.stream = s;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 1u << log_cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = log_cluster > 0 ? 1 : 0;
        CRESSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, z, loss, g, log_cluster));
        CRESSO_LAUNCHED("distill_kernel");
        return (int)CRESSO_OK;
    });
}

}  // extern "C"

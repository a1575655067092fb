// Distillation from a teacher's top logits: the loss of each row and the gradient
// of the student's logits, from one reading of the row.
//
// A row has V student logits z, K teacher entries (id, u), a weight w and the
// temperature tau:
//   p = softmax(u / tau) over the valid entries,  q = softmax(z / tau) over V,
//   loss = w tau^2 sum_k p_k (log p_k - log q[id_k]),
//   dz_v = w tau (q_v - P_v),  P_v = sum of p_k with id_k = v.
// Exponentials are 2^(z c - B) with c = log2(e) / tau and one B for the whole row: a fused
// operation, whose error is that of its result, because the same rounded B stands in the sum,
// in the gradient and in the loss.  B needs no maximum over the row: it is r c for the largest
// student logit r at the teacher's ids, so the sum is at least 1, and only a row with a logit
// about 40 tau above r (or far from zero, or without a finite r) overflows; such a row is
// computed again from its maximum.  Sums are float32.  A NaN or +inf logit makes its row NaN
// through the sum; a row of -inf alone has q = 0.  Repeated ids: every entry holds the whole P
// of its id, so that all of them write the same value.
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
// their sums over equal ids and student logits at the ids, then the sum of p log p, whether a
// valid entry exists, and the largest of the logits.
struct TopList {
    int* id;
    float *p, *same, *z, *entropy;
    int* any;
    float* reference;
    __device__ __forceinline__ TopList(unsigned char* at, int k)
        : id(reinterpret_cast<int*>(at)), p(reinterpret_cast<float*>(at) + k), same(p + k), z(same + k), entropy(z + k),
          any(reinterpret_cast<int*>(entropy + 1)), reference(entropy + 2) {}
};
__host__ __device__ constexpr int top_bytes(int k) { return (16 * k + 12 + 15) / 16 * 16; }

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
// entries a lane in flight together, and the reference; returns the largest teacher logit.
template <typename T>
__device__ __forceinline__ float load_teacher(const DistillArgs& a, int64_t t, const T* row, const TopList& top) {
    const int lane = threadIdx.x & 31;
    const int64_t at = t * a.k;
    float m = -INFINITY, r = -INFINITY;
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
            if (id[j] >= 0) {
                m = fmaxf(m, u[j]);
                r = fmaxf(r, z[j]);
            }
        }
    }
    r = warp_max(r);
    if (lane == 0) *top.reference = r;
    __syncwarp();
    return warp_max(m);
}
// Then the probabilities.
__device__ __forceinline__ void finish_teacher(const DistillArgs& a, const TopList& top, float m, Seen& seen) {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < kSeenBits / 32; i += 32) seen.bits[i] = 0;
    if (lane == 0) seen.count = 0;
    __syncwarp();
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

// Joins (maximum, sum relative to it) over the first WIDTH lanes of a warp; all lanes get it.
template <int WIDTH>
__device__ __forceinline__ void join_warp(float& m, float& s, float c2) {
    float top = m;
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // a part without a finite maximum holds 0 or NaN and keeps it
    s *= m == top ? 1.0f : exp2_fast((m - top) * c2);
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    m = __shfl_sync(0xffffffffu, top, 0);
    s = __shfl_sync(0xffffffffu, s, 0);
}

// B's rounding shifts all exponents of a row by up to 2^-24 |B|, which cancels as long as it
// is small.
constexpr float kFar = 16777216.0f;
constexpr float kLargeSum = 1e18f;  // its reciprocal, times a small weight, stays a normal number

// Loss of the row from its base = -B and sum by one warp, and the gradients of the entries' ids in
// [v0, v1) by `threads` threads.
__device__ __forceinline__ float row_loss(const DistillArgs& a, const TopList& top, float w, float c2, float base, float s) {
    const float log_s = s == 0.0f ? 0.0f : logf(s);
    float cross = 0.0f;
    for (int k = threadIdx.x & 31; k < a.k; k += 32)
        if (top.p[k] != 0.0f) cross += top.p[k] * (fmaf(top.z[k], c2, base) * kLn2 - log_s);
    return w * a.tau * a.tau * (*top.entropy - warp_sum(cross));
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

// ----------------------------------------------------- rows in shared memory ---
//
// A row is cut into the 16-byte words of its memory and lies in the shared memory of a block,
// or of a cluster of blocks: read once, written once.  Each thread copies and reads the same
// words.  The blocks stay for many rows: a word of the next row takes the place of a word
// whose gradient is formed, and one further warp prepares the teacher lists two rows ahead,
// whose chain of dependent loads is about as long as a row takes.
constexpr int kDistillThreads = 256;          // the teacher's warp among them
constexpr int kDistillShare = 64 * 1024;      // bytes of a row in a block, three blocks an SM
constexpr int kDistillLongShare = 128 * 1024; // the same for the longest rows, one block an SM

template <typename T>
constexpr int kWordLogits = 16 / (int)sizeof(T);

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

// f(i) for the words i = tid, tid + THREADS, ... below count, U at a time.
template <int THREADS, int U, typename F>
__device__ __forceinline__ void each_word(int tid, int count, F f) {
    int i = tid;
    for (; i + (U - 1) * THREADS < count; i += U * THREADS)
#pragma unroll
        for (int u = 0; u < U; ++u) f(i + u * THREADS);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
        if (i + u * THREADS < count) f(i + u * THREADS);
}

template <typename T, int BLOCK>
__global__ void __launch_bounds__(BLOCK, 3 * kDistillThreads / BLOCK)
    distill_kernel(DistillArgs a, int64_t rows, const T* z, float* __restrict__ loss, T* grad, int log_cluster,
                   unsigned long long* tickets) {
    constexpr int N = kWordLogits<T>, threads = BLOCK - 32, warps = threads / 32;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float2 warp_part[2][warps], block_part[2];
    __shared__ Seen seen;
    __shared__ int64_t ticket[2];
    uint4* stage = reinterpret_cast<uint4*>(smem + 3 * top_bytes(a.k));
    auto list = [&](int i) { return TopList(smem + i * top_bytes(a.k), a.k); };
    const int cluster = 1 << log_cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = (int)a.vocab;
    const bool is_teacher = warp == warps;
    const int rank = (int)blockIdx.x & (cluster - 1);
    const int64_t workers = gridDim.x >> log_cluster;
    const float c2 = kLog2E / a.tau;
    auto weight = [&](int64_t t) { return t >= rows ? 0.0f : a.weight != nullptr ? a.weight[t] : 1.0f; };
    // The first two rows of a block (cluster) are its own, the others come by ticket, since masked
    // rows take no time.  The ticket of a row is taken two rows ahead.
    int64_t t = blockIdx.x >> log_cluster, t1 = t + workers, pending = rows;
    auto take = [&](bool more) {
        if (is_teacher && lane == 0 && rank == 0) pending = more ? 2 * workers + (int64_t)atomicAdd(tickets, 1ull) : rows;
    };
    take(t1 < rows);
    float w = weight(t), w1 = weight(t1);
    const T* row = z + t * a.stride;
    RowShare r = row_share<T>(row, vocab, rank, log_cluster, tid);
    float edge_x = -INFINITY;
    float teacher_top = -INFINITY;
    if (w != 0.0f) {
        if (is_teacher) {
            teacher_top = load_teacher<T>(a, t, row, list(0));
        } else {
            const T* body = row + r.head + r.first * N;
            each_word<threads, 4>(tid, r.count, [&](int i) { copy_vec<T, N>(reinterpret_cast<T*>(stage + i), body + i * N); });
            if (r.edge >= 0) edge_x = to_float(row[r.edge]);
        }
    }
    copy_commit();
    __syncthreads();  // the reference of the first row
    if (is_teacher) {
        if (w != 0.0f) finish_teacher(a, list(0), teacher_top, seen);
        if (w1 != 0.0f) finish_teacher(a, list(1), load_teacher<T>(a, t1, z + t1 * a.stride, list(1)), seen);
    }
    for (int b = 0, l = 0; t < rows; b ^= 1, l = l == 2 ? 0 : l + 1) {
        const bool live = w != 0.0f;
        const TopList top = list(l);
        const T* row_next = z + t1 * a.stride;
        const T* body_now = row + r.head + r.first * N;
        if (is_teacher && lane == 0) ticket[b] = pending;
        const float reference = live ? *top.reference : 0.0f;
        float base = -__fmul_rn(reference, c2), s = 0.0f;
        if (!is_teacher) {
            copy_wait<0>();
            if (live) {
                float2 sum = make_float2(exp2_fast(fmaf(edge_x, c2, base)), 0.0f);
                each_word<threads, 2>(tid, r.count, [&](int i) {
                    word_pairs<T>(stage[i], [&](int, float2 f) {
                        f = __ffma2_rn(f, make_float2(c2, c2), make_float2(base, base));
                        sum = __fadd2_rn(sum, make_float2(exp2_fast(f.x), exp2_fast(f.y)));
                    });
                });
                s = warp_sum(sum.x + sum.y);
            }
            if (lane == 0) warp_part[b][warp] = make_float2(0.0f, s);
        }
        // the next row
        const RowShare n = row_share<T>(row_next, vocab, rank, log_cluster, tid);
        const int fetched = w1 != 0.0f && !is_teacher ? n.count : 0;
        const T* body_next = row_next + n.head + n.first * N;
        auto fetch = [&](int i) { copy_vec<T, N>(reinterpret_cast<T*>(stage + i), body_next + i * N); };
        float edge_now = edge_x;
        if (!is_teacher) edge_x = w1 != 0.0f && n.edge >= 0 ? to_float(row_next[n.edge]) : -INFINITY;
        if (grad == nullptr) each_word<threads, 4>(tid, fetched, fetch);
        __syncthreads();
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < warps; ++i) s += warp_part[b][i].y;
        int64_t t2 = ticket[b];
        if (cluster > 1) {
            cg::cluster_group group = cg::this_cluster();
            if (tid == 0) block_part[b] = make_float2(0.0f, s);
            group.sync();
            s = 0.0f;
            for (int i = 0; i < cluster; ++i) s += group.map_shared_rank(&block_part[b], i)->y;
            t2 = *group.map_shared_rank(&ticket[b], 0);
        }
        const bool any = live && *top.any;
        const float w2 = weight(t2);
        float far = 0.0f;
        if (any && !(s < kLargeSum && fabsf(base) <= kFar)) {
            // no usable reference: from the row's maximum, over the logits in memory
            float m = -INFINITY;
            s = 0.0f;
            if (!is_teacher) {
                m = edge_now;
                for (int i = tid; i < r.count * N; i += threads) m = fmaxf(m, to_float(body_now[i]));
                const float from = m == -INFINITY ? 0.0f : m;
                s = exp2_fast((edge_now - from) * c2);
                for (int i = tid; i < r.count * N; i += threads) s += exp2_fast((to_float(body_now[i]) - from) * c2);
                join_warp<32>(m, s, c2);
            }
            __syncthreads();  // the parts of the first exchange have been read
            if (!is_teacher && lane == 0) warp_part[b][warp] = make_float2(m, s);
            __syncthreads();
            m = lane < warps ? warp_part[b][lane].x : -INFINITY;
            s = lane < warps ? warp_part[b][lane].y : 0.0f;
            join_warp<8>(m, s, c2);
            if (cluster > 1) {
                cg::cluster_group group = cg::this_cluster();
                group.sync();
                if (tid == 0) block_part[b] = make_float2(m, s);
                group.sync();
                const float2 part = lane < cluster ? *group.map_shared_rank(&block_part[b], lane) : make_float2(-INFINITY, 0.0f);
                m = part.x;
                s = part.y;
                join_warp<8>(m, s, c2);
            }
            if (m == INFINITY) s = NAN;
            far = m == -INFINITY ? 0.0f : m;
            base = 0.0f;
            edge_now -= far;
            if (is_teacher)
                for (int k = lane; k < a.k; k += 32) top.z[k] -= far;
            __syncthreads();
        }
        if (is_teacher) {
            if (rank == 0) {
                const float v = any ? row_loss(a, top, w, c2, base, s) : 0.0f;
                if (lane == 0) loss[t] = v;
            }
            take(t2 < rows);
            if (w2 != 0.0f) {
                const TopList ahead = list(l == 0 ? 2 : l - 1);
                finish_teacher(a, ahead, load_teacher<T>(a, t2, z + t2 * a.stride, ahead), seen);
            }
        } else {
            if (grad != nullptr) {
                T* out = grad + t * a.vocab;
                T* body = out + r.head + r.first * N;
                const bool aligned = (reinterpret_cast<uintptr_t>(body) & 15) == 0;
                const float c = w * a.tau, inv_s = s == 0.0f ? 0.0f : 1.0f / s, ci = c * inv_s;
                if (any && far == 0.0f && aligned) {
                    each_word<threads, 2>(tid, r.count, [&](int i) {
                        uint32_t o[4];
                        word_pairs<T>(stage[i], [&](int j, float2 f) {
                            f = __ffma2_rn(f, make_float2(c2, c2), make_float2(base, base));
                            f = __fmul2_rn(make_float2(exp2_fast(f.x), exp2_fast(f.y)), make_float2(ci, ci));
                            if constexpr (sizeof(T) == 4) {
                                o[2 * j] = __float_as_uint(f.x);
                                o[2 * j + 1] = __float_as_uint(f.y);
                            } else {
                                o[j] = pack2<T>(f.x, f.y);
                            }
                        });
                        reinterpret_cast<uint4*>(body)[i] = make_uint4(o[0], o[1], o[2], o[3]);
                        if (i < fetched) fetch(i);
                    });
                    // the next row may begin at another alignment and have one word more
                    if (r.count < fetched && (fetched - 1) % threads == tid) fetch(fetched - 1);
                } else if (!any && aligned) {
                    each_word<threads, 4>(tid, r.count, [&](int i) {
                        reinterpret_cast<uint4*>(body)[i] = make_uint4(0, 0, 0, 0);
                    });
                    each_word<threads, 4>(tid, fetched, fetch);
                } else {  // rows of logits that lie further apart than those of the gradient, or far ones
                    each_word<threads, 1>(tid, r.count, [&](int i) {
                        T e[N];
                        *reinterpret_cast<uint4*>(e) = stage[i];
#pragma unroll
                        for (int j = 0; j < N; ++j)
                            body[i * N + j] =
                                from_float<T>(any ? ci * exp2_fast(fmaf(to_float(e[j]) - far, c2, base)) : 0.0f);
                    });
                    each_word<threads, 4>(tid, fetched, fetch);
                }
                if (r.edge >= 0) out[r.edge] = from_float<T>(any ? ci * exp2_fast(fmaf(edge_now, c2, base)) : 0.0f);
                if (any) {
                    asm volatile("bar.sync 1, %0;" ::"n"(threads) : "memory");  // the row is written
                    const int v0 = rank == 0 ? 0 : r.head + r.first * N;
                    const int v1 = rank == cluster - 1 ? vocab : r.head + (r.first + r.count) * N;
                    top_gradients<T>(a, top, out, threads, v0, v1, c, c2, base, inv_s);
                }
            }
            copy_commit();
        }
        r = n;
        t = t1;
        t1 = t2;
        row = row_next;
        w = w1;
        w1 = w2;
    }
    if (cluster > 1) cg::this_cluster().sync();  // a peer may still read this block's part
}

// ------------------------------------------------------------- longer rows ---
//
// A row beyond the registers of a cluster of eight blocks: one block reads it three times.
template <typename T>
__global__ void __launch_bounds__(1024) distill_long_kernel(DistillArgs a, const T* z, float* __restrict__ loss,
                                                            T* grad) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float sh[32];
    __shared__ Seen seen;
    const TopList top(smem, a.k);
    const int64_t t = blockIdx.x;
    const T* row = z + t * a.stride;
    T* out = grad != nullptr ? grad + t * a.vocab : nullptr;
    const float w = a.weight != nullptr ? a.weight[t] : 1.0f;
    if (w != 0.0f && threadIdx.x < 32) finish_teacher(a, top, load_teacher<T>(a, t, row, top), seen);
    __syncthreads();
    if (w == 0.0f || !*top.any) {
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
    // the difference first: no B that could overflow
    auto term = [&](float x) { return exp2_fast((x - m) * c2); };
    float s = 0.0f;
    for (int64_t v = threadIdx.x; v < a.vocab; v += blockDim.x) s += term(to_float(row[v]));
    s = block_sum(s, sh);
    if (threadIdx.x < 32) {
        for (int k = threadIdx.x; k < a.k; k += 32) top.z[k] -= m;
        __syncwarp();
        const float l = row_loss(a, top, w, c2, 0.0f, s);
        if (threadIdx.x == 0) loss[t] = l;
    }
    if (out == nullptr) return;
    const float inv_s = s == 0.0f ? 0.0f : 1.0f / s, c = w * a.tau;
    for (int64_t v = threadIdx.x; v < a.vocab; v += blockDim.x) out[v] = from_float<T>(c * inv_s * term(to_float(row[v])));
    __syncthreads();
    top_gradients<T>(a, top, out, (int)blockDim.x, 0, (int)a.vocab, c, c2, 0.0f, inv_s);
}

constexpr int64_t kDistillScratch = 32;  // the ticket counter

// Blocks of a row and their threads.
struct DistillPlan {
    int cluster, threads;  // cluster 0: the kernel for longer rows
    int64_t share;         // words of a block
};
static DistillPlan distill_plan(int64_t n, int64_t words) {
    DistillPlan p{1, kDistillThreads, 0};
    while (p.cluster < 8 && words * 16 > (int64_t)p.cluster * kDistillShare) p.cluster *= 2;
    if (words * 16 > (int64_t)p.cluster * kDistillLongShare) p.cluster = 0;
    if (p.cluster == 0) return p;
    // few rows: more blocks a row, as long as each of their threads has a word
    while (p.cluster < 8 && n * p.cluster < 2 * 148 && words >= 2 * p.cluster * kDistillThreads) p.cluster *= 2;
    p.share = ceil_div(words, p.cluster);
    while (p.threads > kDistillThreads / 4 && p.share <= p.threads / 2) p.threads /= 2;
    return p;
}

}  // namespace cresso

using namespace cresso;

extern "C" {

int cresso_distill_scratch_bytes(int64_t n, int64_t vocab, int64_t* bytes) {
    CRESSO_REQUIRE(bytes != nullptr, CRESSO_EINVAL, "distill_scratch_bytes: NULL result");
    CRESSO_REQUIRE(n >= 0 && vocab >= 1, CRESSO_EINVAL, "distill: negative size, or an empty vocabulary");
    *bytes = kDistillScratch;
    return CRESSO_OK;
}

int cresso_distill(const void* logits, int64_t dtype, int64_t n, int64_t vocab, int64_t logits_stride, const void* ids,
                   int64_t id_bytes, const void* teacher, int64_t teacher_dtype, int64_t k, const float* weight,
                   double temperature, float* loss, void* grad, void* scratch, int64_t scratch_bytes,
                   cresso_stream_t stream) {
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
    CRESSO_REQUIRE(scratch != nullptr && scratch_bytes >= kDistillScratch, CRESSO_ESCRATCH,
                   "distill: scratch has %lld bytes, %lld are needed", (long long)scratch_bytes,
                   (long long)kDistillScratch);
    CRESSO_REQUIRE(aligned_to(scratch, 32), CRESSO_EINVAL, "distill: scratch is not 32-byte aligned");
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
            distill_long_kernel<T><<<(unsigned)n, 1024, top_bytes(a.k), s>>>(a, z, loss, g);
            CRESSO_LAUNCHED("distill_long_kernel");
            return (int)CRESSO_OK;
        }
        const int smem = (int)p.share * 16 + 3 * top_bytes(a.k);
        const auto kernel = p.threads == kDistillThreads       ? distill_kernel<T, kDistillThreads>
                            : p.threads == kDistillThreads / 2 ? distill_kernel<T, kDistillThreads / 2>
                                                               : distill_kernel<T, kDistillThreads / 4>;
        if (smem > 48 * 1024)
            CRESSO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kDistillLongShare + 3 * top_bytes(CRESSO_TRAIN_MAX_TOP)));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)p.cluster);
        cfg.blockDim = dim3((unsigned)p.threads);
        cfg.dynamicSmemBytes = (size_t)smem;
        cfg.stream = s;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)p.cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = p.cluster > 1 ? 1 : 0;
        int64_t workers = n;  // as many as stay on the GPU together
        if (n * p.cluster > 148) {
            int fit = 0;
            if (p.cluster > 1) {
                CRESSO_CUDA(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
            } else {
                CRESSO_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, p.threads, (size_t)smem));
                fit *= 148;
            }
            workers = std::min<int64_t>(n, std::max(1, fit));
        }
        cfg.gridDim = dim3((unsigned)(workers * p.cluster));
        int log_cluster = 0;
        while ((1 << log_cluster) < p.cluster) ++log_cluster;
        unsigned long long* tickets = static_cast<unsigned long long*>(scratch);
        if (n > workers) CRESSO_CUDA(cudaMemsetAsync(tickets, 0, 8, s));
        CRESSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, n, z, loss, g, log_cluster, tickets));
        CRESSO_LAUNCHED("distill_kernel");
        return (int)CRESSO_OK;
    });
}

}  // extern "C"

// Distillation from a teacher's top logits: the loss of each row and the gradient
// of the student's logits, from one reading of the row where the gradient is wanted.
//
// A row has V student logits z, K teacher entries (id, u), a weight w and the
// temperature tau:
//   p = softmax(u / tau) over the valid entries,  q = softmax(z / tau) over V,
//   loss = w tau^2 sum_k p_k (log p_k - log q[id_k]),
//   dz_v = w tau (q_v - P_v),  P_v = sum of p_k with id_k = v.
// Exponentials are taken relative to the row's maximum and summed in float32.  A
// NaN or +inf logit makes its row NaN through the sum; a row of -inf alone has
// q = 0.  Repeated ids: every entry forms the whole P of its id, so that all of
// them write the same value.
#include "train_common.cuh"

namespace cresso {

struct DistillArgs {
    const void *ids, *teacher;
    const float* weight;
    int64_t vocab, stride;
    int id_bytes, teacher_dtype, k;
    float tau;
};

constexpr int kDistillThreads = 512;

// The teacher's side of a row in shared memory.
struct TopList {
    int id[CRESSO_TRAIN_MAX_TOP];   // -1: not valid
    float p[CRESSO_TRAIN_MAX_TOP];  // teacher probability
    float z[CRESSO_TRAIN_MAX_TOP];  // student logit / tau at the id
};

// Fills ids and probabilities; returns sum_k p_k log p_k in every thread, and in
// `any` whether a valid entry exists.
__device__ __forceinline__ float load_teacher(const DistillArgs& a, int64_t t, TopList& top, float* sh, bool& any) {
    float m = -INFINITY;
    bool valid_here = false;
    for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
        const int64_t id = load_id(a.ids, a.id_bytes, t * a.k + k);
        const float u = load_any(a.teacher, a.teacher_dtype, t * a.k + k) / a.tau;
        const bool valid = id >= 0 && id < a.vocab && u != -INFINITY;
        top.id[k] = valid ? (int)id : -1;
        top.p[k] = u;
        if (valid) {
            m = fmaxf(m, u);
            valid_here = true;
        }
    }
    any = __syncthreads_or(valid_here);
    m = block_max(m, sh);
    float s = 0.0f;
    for (int k = threadIdx.x; k < a.k; k += blockDim.x)
        if (top.id[k] >= 0) s += expf(top.p[k] - m);
    s = block_sum(s, sh);
    const float log_s = logf(s);
    float ent = 0.0f;
    for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
        const float lp = top.p[k] - m - log_s;
        const float p = top.id[k] >= 0 ? expf(lp) : 0.0f;
        if (top.id[k] >= 0 && p != 0.0f) ent += p * lp;
        top.p[k] = p;
    }
    return block_sum(ent, sh);  // ends with a barrier: the list is complete
}

template <typename T>
__global__ void __launch_bounds__(kDistillThreads) distill_kernel(DistillArgs a, const T* z, float* __restrict__ loss,
                                                                  T* grad) {
    __shared__ TopList top;
    __shared__ float sh[32];
    const int64_t t = blockIdx.x;
    const T* row = z + t * a.stride;
    T* out = grad != nullptr ? grad + t * a.vocab : nullptr;
    const float w = a.weight != nullptr ? a.weight[t] : 1.0f;
    bool any = false;
    float ent = 0.0f;
    if (w != 0.0f) ent = load_teacher(a, t, top, sh, any);
    if (!any) {
        if (out != nullptr)
            for (int64_t v = threadIdx.x; v < a.vocab; v += kDistillThreads) out[v] = from_float<T>(0.0f);
        if (threadIdx.x == 0) loss[t] = 0.0f;
        return;
    }
    const float inv_tau = 1.0f / a.tau;
    float m = -INFINITY;
    for (int64_t v = threadIdx.x; v < a.vocab; v += kDistillThreads) m = fmaxf(m, to_float(row[v]) * inv_tau);
    m = block_max(m, sh);
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f;
    for (int64_t v = threadIdx.x; v < a.vocab; v += kDistillThreads) s += expf(to_float(row[v]) * inv_tau - m);
    s = block_sum(s, sh);
    const float log_s = s == 0.0f ? 0.0f : logf(s), inv_s = s == 0.0f ? 0.0f : 1.0f / s;
    float cross = 0.0f;
    for (int k = threadIdx.x; k < a.k; k += kDistillThreads) {
        if (top.id[k] < 0) continue;
        const float zk = to_float(row[top.id[k]]) * inv_tau;
        top.z[k] = zk;
        if (top.p[k] != 0.0f) cross += top.p[k] * (zk - m - log_s);
    }
    cross = block_sum(cross, sh);  // the barrier also ends the reads of z before grad may overwrite them
    if (threadIdx.x == 0) loss[t] = w * a.tau * a.tau * (ent - cross);
    if (out == nullptr) return;
    const float c = w * a.tau;
    for (int64_t v = threadIdx.x; v < a.vocab; v += kDistillThreads)
        out[v] = from_float<T>(c * (expf(to_float(row[v]) * inv_tau - m) * inv_s));
    __syncthreads();
    for (int k = threadIdx.x; k < a.k; k += kDistillThreads) {
        if (top.id[k] < 0) continue;
        float p = 0.0f;
        for (int j = 0; j < a.k; ++j) p += top.id[j] == top.id[k] ? top.p[j] : 0.0f;
        out[top.id[k]] = from_float<T>(c * (expf(top.z[k] - m) * inv_s - p));
    }
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
        distill_kernel<T><<<(unsigned)n, kDistillThreads, 0, (cudaStream_t)stream>>>(a, static_cast<const T*>(logits),
                                                                                   loss, static_cast<T*>(grad));
        CRESSO_LAUNCHED("distill_kernel");
        return (int)CRESSO_OK;
    });
}

}  // extern "C"

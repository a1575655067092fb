// The norms before and after a block, fused with the block's gate and residual
// scale, forward and backward.
//
// Forward, for a row of D elements (R = (mean v^2 + eps)^-1/2):
//   p = x Rx w_post,  h = residual + scale gate p,  y = h Rh w_pre.
// Backward, from h and x (both R are formed again, so nothing is saved), with
// n = h Rh and q = x Rx:
//   dn = d_y w_pre,            e = d_h + Rh (dn - n mean(dn n)),  d_residual = e
//   dp = scale gate e,         dq = dp w_post,  d_x = Rx (dq - q mean(dq q))
//   d_pre = sum_t d_y n,       d_post = sum_t dp q,  d_gate = scale sum e p.
#include "train_common.cuh"

#include <algorithm>

namespace cresso {

struct NormArgs {
    const void *post_w, *pre_w, *gate;
    int64_t n, width, rows_per_gate;  // rows_per_gate: consecutive rows that share a gate row
    int w_dtype, gate_dtype;
    float scale, eps;
};

template <typename TR, typename TX>
__global__ void __launch_bounds__(kThreads) norm_kernel(NormArgs a, const TR* __restrict__ res,
                                                        const TX* __restrict__ x, TR* __restrict__ h,
                                                        TX* __restrict__ y) {
    __shared__ float sh[32];
    const int64_t t = blockIdx.x, d = a.width;
    const int64_t g0 = a.gate != nullptr ? t / a.rows_per_gate * d : 0;
    const float inv_d = 1.0f / (float)d;
    float rx = 1.0f;
    if (x != nullptr && a.post_w != nullptr) {
        float s = 0.0f;
        for (int64_t c = threadIdx.x; c < d; c += kThreads) {
            const float v = to_float(x[t * d + c]);
            s += v * v;
        }
        rx = rsqrtf(block_sum(s, sh) * inv_d + a.eps);
    }
    auto value = [&](int64_t c) {
        float v = to_float(res[t * d + c]);
        if (x != nullptr) {
            float p = to_float(x[t * d + c]) * rx;
            if (a.post_w != nullptr) p *= load_any(a.post_w, a.w_dtype, c);
            if (a.gate != nullptr) p *= load_any(a.gate, a.gate_dtype, g0 + c);
            v += a.scale * p;
        }
        return v;
    };
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < d; c += kThreads) {
        const float v = value(c);
        s += v * v;
        if (x != nullptr) h[t * d + c] = from_float<TR>(v);
    }
    if (y == nullptr) return;
    const float rh = rsqrtf(block_sum(s, sh) * inv_d + a.eps);
    for (int64_t c = threadIdx.x; c < d; c += kThreads)
        y[t * d + c] = from_float<TX>(value(c) * rh * load_any(a.pre_w, a.w_dtype, c));
}

struct RowStats {
    float rx, rh, mean_dn_n, mean_dq_q;
};

// Row-wise gradients; leaves the row's statistics for the column sums.
template <typename TR, typename TX>
__global__ void __launch_bounds__(kThreads) norm_grad_kernel(NormArgs a, const TR* __restrict__ h,
                                                             const TX* __restrict__ x, const TR* __restrict__ dh,
                                                             const TX* __restrict__ dy, TR* __restrict__ dres,
                                                             TX* __restrict__ dx, RowStats* __restrict__ stats) {
    __shared__ float sh[32];
    const int64_t t = blockIdx.x, d = a.width;
    const int64_t g0 = a.gate != nullptr ? t / a.rows_per_gate * d : 0;
    const float inv_d = 1.0f / (float)d;
    float sh2 = 0.0f, sx2 = 0.0f, sdn = 0.0f;
    for (int64_t c = threadIdx.x; c < d; c += kThreads) {
        const float hv = to_float(h[t * d + c]);
        sh2 += hv * hv;
        if (x != nullptr) {
            const float xv = to_float(x[t * d + c]);
            sx2 += xv * xv;
        }
        if (dy != nullptr) sdn += to_float(dy[t * d + c]) * load_any(a.pre_w, a.w_dtype, c) * hv;
    }
    RowStats r;
    r.rh = rsqrtf(block_sum(sh2, sh) * inv_d + a.eps);
    r.rx = a.post_w != nullptr ? rsqrtf(block_sum(sx2, sh) * inv_d + a.eps) : 1.0f;
    r.mean_dn_n = block_sum(sdn, sh) * inv_d * r.rh;
    auto grad_h = [&](int64_t c) {
        float e = dh != nullptr ? to_float(dh[t * d + c]) : 0.0f;
        if (dy != nullptr) {
            const float dn = to_float(dy[t * d + c]) * load_any(a.pre_w, a.w_dtype, c);
            e += r.rh * (dn - to_float(h[t * d + c]) * r.rh * r.mean_dn_n);
        }
        return e;
    };
    auto grad_q = [&](int64_t c, float e) {
        float v = a.scale * e;
        if (a.gate != nullptr) v *= load_any(a.gate, a.gate_dtype, g0 + c);
        if (a.post_w != nullptr) v *= load_any(a.post_w, a.w_dtype, c);
        return v;
    };
    float sdq = 0.0f;
    for (int64_t c = threadIdx.x; c < d; c += kThreads) {
        const float e = grad_h(c);
        if (x != nullptr && a.post_w != nullptr) sdq += grad_q(c, e) * to_float(x[t * d + c]);
    }
    r.mean_dq_q = block_sum(sdq, sh) * inv_d * r.rx;
    for (int64_t c = threadIdx.x; c < d; c += kThreads) {
        const float e = grad_h(c);
        dres[t * d + c] = from_float<TR>(e);
        if (x != nullptr) {
            const float dq = grad_q(c, e);
            dx[t * d + c] = from_float<TX>(
                a.post_w != nullptr ? r.rx * (dq - to_float(x[t * d + c]) * r.rx * r.mean_dq_q) : dq);
        }
    }
    if (threadIdx.x == 0) stats[t] = r;
}

// Column sums of the weight gradients and the gate gradient over the rows
// [blockIdx.y * span, + span); one thread a column.  which: 0 post, 1 pre, 2 gate.
template <typename TR, typename TX>
__global__ void __launch_bounds__(kThreads) norm_columns_kernel(NormArgs a, int which, int64_t span,
                                                                const TR* __restrict__ h, const TX* __restrict__ x,
                                                                const TR* __restrict__ dh, const TX* __restrict__ dy,
                                                                const RowStats* __restrict__ stats, void* out,
                                                                int out_dtype) {
    const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x, d = a.width;
    if (c >= d) return;
    const float pre = dy != nullptr ? load_any(a.pre_w, a.w_dtype, c) : 0.0f;
    const float post = a.post_w != nullptr ? load_any(a.post_w, a.w_dtype, c) : 1.0f;
    for (int64_t b = blockIdx.y; b * span < a.n; b += gridDim.y) {
        float sum = 0.0f;
        for (int64_t t = b * span; t < min(a.n, (b + 1) * span); ++t) {
            const RowStats r = stats[t];
            const float n = to_float(h[t * d + c]) * r.rh;
            const float dyv = dy != nullptr ? to_float(dy[t * d + c]) : 0.0f;
            if (which == 1) {
                sum += dyv * n;
                continue;
            }
            const float e = (dh != nullptr ? to_float(dh[t * d + c]) : 0.0f) + r.rh * (dyv * pre - n * r.mean_dn_n);
            const float q = to_float(x[t * d + c]) * r.rx;
            if (which == 2)
                sum += a.scale * e * q * post;
            else
                sum += a.scale * e * q *
                       (a.gate != nullptr ? load_any(a.gate, a.gate_dtype, t / a.rows_per_gate * d + c) : 1.0f);
        }
        store_any(out, out_dtype, b * d + c, sum);
    }
}

static int norm_check(const char* who, int64_t n, int64_t width, int64_t gate_rows, bool has_gate, int64_t res_dtype,
                      int64_t act_dtype, int64_t weight_dtype, int64_t gate_dtype, double eps) {
    CRESSO_REQUIRE(train_dtype_ok(res_dtype) && train_dtype_ok(act_dtype) &&
                       (res_dtype == act_dtype || res_dtype == CRESSO_DTYPE_F32),
                   CRESSO_EUNSUPPORTED, "%s: x has the residual's type, or 16 bits beside a float32 residual", who);
    CRESSO_REQUIRE(train_dtype_ok(weight_dtype) && train_dtype_ok(gate_dtype), CRESSO_EUNSUPPORTED,
                   "%s: weights and gate are float32, float16 or bfloat16", who);
    CRESSO_REQUIRE(n >= 0 && width >= 0, CRESSO_EINVAL, "%s: negative size", who);
    CRESSO_REQUIRE(n <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED, "%s: more than 2^31 - 256 rows", who);
    CRESSO_REQUIRE(!has_gate || n == 0 || (gate_rows > 0 && n % gate_rows == 0), CRESSO_EINVAL,
                   "%s: the number of rows is not a multiple of the gate's rows", who);
    CRESSO_REQUIRE(eps >= 0.0, CRESSO_EINVAL, "%s: eps must be >= 0", who);
    return CRESSO_OK;
}

// f(TR(), TX()) for the type pairs that norm_check admits.
template <typename F>
int with_norm_types(int64_t res, int64_t act, F f) {
    if (res == act) return with_dtype(res, [&](auto t) { return f(t, t); });
    return act == CRESSO_DTYPE_F16 ? f(float(), __half()) : f(float(), __nv_bfloat16());
}

}  // namespace cresso

using namespace cresso;

extern "C" {

int cresso_block_norm(const void* residual, const void* x, const void* post_weight, const void* pre_weight,
                      const void* gate, int64_t n, int64_t width, int64_t gate_rows, int64_t res_dtype,
                      int64_t act_dtype, int64_t weight_dtype, int64_t gate_dtype, double scale, double eps, void* h,
                      void* y, cresso_stream_t stream) {
    const int st = norm_check("block_norm", n, width, gate_rows, gate != nullptr, res_dtype, act_dtype, weight_dtype,
                              gate_dtype, eps);
    if (st != CRESSO_OK) return st;
    CRESSO_REQUIRE(x != nullptr || (post_weight == nullptr && gate == nullptr) || n == 0 || width == 0, CRESSO_EINVAL,
                   "block_norm: a post weight or a gate needs x");
    if (n == 0 || width == 0) return CRESSO_OK;
    CRESSO_REQUIRE(residual != nullptr && (x == nullptr || h != nullptr) && (pre_weight == nullptr) == (y == nullptr) &&
                       (x != nullptr || y != nullptr),
                   CRESSO_EINVAL, "block_norm: NULL pointer, or y without pre_weight");
    NvtxRange range("block_norm n=%lld", (long long)n);
    const NormArgs a{post_weight, pre_weight, gate, n, width, gate != nullptr ? n / gate_rows : n,
                     (int)weight_dtype, (int)gate_dtype, (float)scale, (float)eps};
    return with_norm_types(res_dtype, act_dtype, [&](auto tr, auto tx) {
        using TR = decltype(tr);
        using TX = decltype(tx);
        norm_kernel<TR, TX><<<(unsigned)n, kThreads, 0, (cudaStream_t)stream>>>(
            a, static_cast<const TR*>(residual), static_cast<const TX*>(x), static_cast<TR*>(h), static_cast<TX*>(y));
        CRESSO_LAUNCHED("norm_kernel");
        return (int)CRESSO_OK;
    });
}

int cresso_block_norm_grad_scratch_bytes(int64_t n, int64_t width, int64_t gate_rows, int64_t* bytes) {
    CRESSO_REQUIRE(bytes != nullptr, CRESSO_EINVAL, "block_norm_grad_scratch_bytes: NULL result");
    CRESSO_REQUIRE(n >= 0 && width >= 0 && gate_rows >= 0, CRESSO_EINVAL, "block_norm_grad: negative size");
    *bytes = align_up(n * (int64_t)sizeof(RowStats), 256);
    return CRESSO_OK;
}

int cresso_block_norm_grad(const void* h, const void* x, const void* d_h, const void* d_y, const void* post_weight,
                           const void* pre_weight, const void* gate, int64_t n, int64_t width, int64_t gate_rows,
                           int64_t res_dtype, int64_t act_dtype, int64_t weight_dtype, int64_t gate_dtype,
                           double scale, double eps, void* d_residual, void* d_x, void* d_post_weight,
                           void* d_pre_weight, void* d_gate, void* scratch, int64_t scratch_bytes,
                           cresso_stream_t stream) {
    const int st = norm_check("block_norm_grad", n, width, gate_rows, gate != nullptr, res_dtype, act_dtype,
                              weight_dtype, gate_dtype, eps);
    if (st != CRESSO_OK) return st;
    if (width == 0) return CRESSO_OK;
    const cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {  // no rows: the sums over them are zero
        if (d_post_weight != nullptr)
            CRESSO_CUDA(cudaMemsetAsync(d_post_weight, 0, (size_t)(width * dtype_bytes(weight_dtype)), s));
        if (d_pre_weight != nullptr)
            CRESSO_CUDA(cudaMemsetAsync(d_pre_weight, 0, (size_t)(width * dtype_bytes(weight_dtype)), s));
        if (d_gate != nullptr && gate_rows > 0)
            CRESSO_CUDA(cudaMemsetAsync(d_gate, 0, (size_t)(gate_rows * width * dtype_bytes(gate_dtype)), s));
        return CRESSO_OK;
    }
    CRESSO_REQUIRE(x != nullptr || (post_weight == nullptr && gate == nullptr), CRESSO_EINVAL,
                   "block_norm_grad: a post weight or a gate needs x");
    CRESSO_REQUIRE(h != nullptr && d_residual != nullptr && (d_h != nullptr || d_y != nullptr) &&
                       (d_y == nullptr || pre_weight != nullptr),
                   CRESSO_EINVAL, "block_norm_grad: NULL pointer, or d_y without pre_weight");
    CRESSO_REQUIRE((x != nullptr) == (d_x != nullptr) && (post_weight != nullptr) == (d_post_weight != nullptr) &&
                       (d_y != nullptr) == (d_pre_weight != nullptr) && (gate != nullptr) == (d_gate != nullptr),
                   CRESSO_EINVAL, "block_norm_grad: an input without its gradient, or a gradient without its input");
    int64_t need = 0;
    const int sb = cresso_block_norm_grad_scratch_bytes(n, width, gate_rows, &need);
    if (sb != CRESSO_OK) return sb;
    CRESSO_REQUIRE(scratch != nullptr && scratch_bytes >= need, CRESSO_ESCRATCH,
                   "block_norm_grad: scratch has %lld bytes, %lld are needed", (long long)scratch_bytes, (long long)need);
    NvtxRange range("block_norm_grad n=%lld", (long long)n);
    const NormArgs a{post_weight, pre_weight, gate, n, width, gate != nullptr ? n / gate_rows : n,
                     (int)weight_dtype, (int)gate_dtype, (float)scale, (float)eps};
    RowStats* stats = static_cast<RowStats*>(scratch);
    return with_norm_types(res_dtype, act_dtype, [&](auto tr, auto tx) {
        using TR = decltype(tr);
        using TX = decltype(tx);
        const TR *ph = static_cast<const TR*>(h), *pdh = static_cast<const TR*>(d_h);
        const TX *px = static_cast<const TX*>(x), *pdy = static_cast<const TX*>(d_y);
        norm_grad_kernel<TR, TX><<<(unsigned)n, kThreads, 0, s>>>(a, ph, px, pdh, pdy, static_cast<TR*>(d_residual),
                                                                 static_cast<TX*>(d_x), stats);
        CRESSO_LAUNCHED("norm_grad_kernel");
        for (int which = 0; which < 3; ++which) {
            void* out = which == 0 ? d_post_weight : which == 1 ? d_pre_weight : d_gate;
            if (out == nullptr) continue;
            const int64_t span = which == 2 ? a.rows_per_gate : n;
            const dim3 grid((unsigned)ceil_div(width, kThreads), (unsigned)std::min<int64_t>(65535, n / span));
            norm_columns_kernel<TR, TX><<<grid, kThreads, 0, s>>>(a, which, span, ph, px, pdh, pdy, stats, out,
                                                                 (int)(which == 2 ? gate_dtype : weight_dtype));
            CRESSO_LAUNCHED("norm_columns_kernel");
        }
        return (int)CRESSO_OK;
    });
}

}  // extern "C"

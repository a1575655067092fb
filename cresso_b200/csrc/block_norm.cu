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

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace cresso {

struct NormArgs {
    const void *post_w, *pre_w, *gate;
    int64_t n, width, rows_per_gate;  // rows_per_gate: consecutive rows that share a gate row
    int w_dtype, gate_dtype;
    float scale, eps;
};

constexpr int kNormMaxWidth = CRESSO_TRAIN_MAX_NORM_WIDTH;
constexpr int kNormStageBytes = 220 * 1024;  // shared memory of a backward block's stages at most

// Columns of a thread (EL, 16 or 8), threads and blocks of a row: a row of more than 512 EL
// columns is cut over a cluster of 2 to 8 blocks, which add their sums through distributed
// shared memory.
struct NormShape {
    int elems, threads, cluster, block_width;
};
static NormShape norm_shape(int64_t width, int elems) {
    NormShape p{};
    p.elems = width > 512 * 8 ? 16 : elems;
    p.cluster = pow2_ceil(ceil_div(width, 512 * p.elems));
    p.block_width = (int)(p.cluster > 1 ? align_up(ceil_div(width, p.cluster), 8) : width);
    p.threads = (int)align_up(ceil_div(p.block_width, p.elems), 32);
    return p;
}
// Few rows, no more than there are SMs, are a matter of latency, for which 8 columns a thread are
// better in the forward pass: one row of 4096 takes 4.2 us instead of 6.2, and 300 rows 8.2 us
// instead of 6.2.
constexpr int64_t kNormFewRows = 149;

// Accesses first, first + 1, .. of a thread to p[0, d): VEC columns each, the accesses of a row
// blockDim.x VEC apart; zeros behind the row.  No access waits for another one.
template <typename T, int VEC, int N>
__device__ __forceinline__ void load_columns(const T* p, int d, int first, float (&v)[N][VEC]) {
    const int stride = blockDim.x * VEC, c = threadIdx.x * VEC + first * stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        Raw<T, VEC> u;
#pragma unroll
        for (int j = 0; j < (int)(sizeof(u.w) / 4); ++j) u.w[j] = 0;
        if (c + i * stride < d) u.load_global(p + c + i * stride);
        u.to(v[i]);
    }
}

// ----------------------------------------------------------------- forward ---
//
// A row lies in the registers of a block (of a warp up to 512 columns, four rows a block): x and
// residual are read once, h and y written once, two reductions between.  Weights and gate come from
// L1 for every row.  Many small blocks an SM, each at another point of its row, keep the memory busy
// without any staging; a loop that leaves at the row's end held up the loads behind it.  Bound by
// memory: 16384 rows of 4096, float32 beside bfloat16, take 125 us, 805 MB at 6.4 TB/s (139 us with
// such loops); three blocks of 512 threads an SM instead of two spill (218 us).
template <typename TR, typename TX, int VEC, int EL>
__global__ void __launch_bounds__(512, 2) norm_kernel(NormArgs a, const TR* __restrict__ res,
                                                      const TX* __restrict__ x, TR* __restrict__ h,
                                                      TX* __restrict__ y, int cluster, int block_width) {
    constexpr int NV = EL / VEC;
    namespace cg = cooperative_groups;
    __shared__ float red[2][32], peer[2];
    const int64_t width = a.width;
    const int rank = cluster > 1 ? (int)(blockIdx.x % cluster) : 0;
    const int64_t col0 = (int64_t)rank * block_width;
    const int d = (int)min((int64_t)block_width, width - col0);
    const int T = blockDim.x, tid = threadIdx.x, warps = T >> 5;  // blockDim.y rows, one warp each, when T is 32
    const int64_t t = (int64_t)(blockIdx.x / cluster) * blockDim.y + threadIdx.y;
    if (t >= a.n) return;  // a whole warp of the last block
    const float inv_d = 1.0f / (float)width;
    auto row_sum = [&](float v, int k) {
        v = warp_sum(v);
        if (warps > 1) {
            if ((tid & 31) == 0) red[k][tid >> 5] = v;
            __syncthreads();
            v = warp_sum((tid & 31) < warps ? red[k][tid & 31] : 0.0f);
        }
        if (cluster > 1) {
            cg::cluster_group group = cg::this_cluster();
            if (tid == 0) peer[k] = v;
            group.sync();
            v = 0.0f;
            for (int i = 0; i < cluster; ++i) v += *group.map_shared_rank(&peer[k], i);
        }
        return v;
    };
    float hv[NV][VEC], xv[NV][VEC];
    const int64_t at = t * width + col0;
    if (x != nullptr) load_columns(x + at, d, 0, xv);
    load_columns(res + at, d, 0, hv);
    // v *= an array's values at the thread's columns
    auto multiply = [&](float (&v)[NV][VEC], const void* p, int dtype, int64_t from) {
        with_any(p, dtype, [&](auto* w) {
            // all 16 single columns at once would spill more than the 16 to 48 bytes of this form
            constexpr int N = VEC == 1 ? 4 : NV;
#pragma unroll
            for (int first = 0; first < NV; first += N) {
                float f[N][VEC];
                load_columns(w + from, d, first, f);
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[first + i][j] *= f[i][j];
            }
        });
    };
    if (x != nullptr) {
        float rx = a.scale;
        if (a.post_w != nullptr) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s += xv[v][j] * xv[v][j];
            multiply(xv, a.post_w, a.w_dtype, col0);  // on the way while the sum is formed
            rx *= rsqrtf(row_sum(s, 0) * inv_d + a.eps);
        }
        if (a.gate != nullptr) multiply(xv, a.gate, a.gate_dtype, t / a.rows_per_gate * width + col0);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T + tid) * VEC;
            if (c >= d) break;
#pragma unroll
            for (int j = 0; j < VEC; ++j) hv[v][j] += rx * xv[v][j];
            store_global<TR, VEC>(h + at + c, hv[v]);
        }
    }
    if (y != nullptr) {
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += hv[v][j] * hv[v][j];
        multiply(hv, a.pre_w, a.w_dtype, col0);
        const float rh = rsqrtf(row_sum(s, 1) * inv_d + a.eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * T + tid) * VEC;
            if (c >= d) break;
#pragma unroll
            for (int j = 0; j < VEC; ++j) hv[v][j] *= rh;
            store_global<TX, VEC>(y + at + c, hv[v]);
        }
    }
    if (cluster > 1) cg::this_cluster().sync();  // a peer may still read this block's sums
}

// ---------------------------------------------------------------- backward ---
//
// One pass over the rows.  A thread owns fixed columns, so the factors of a column
// (pre = w_pre, A = scale gate w_post) and its sums over rows stay in registers.
// Per row: six sums over the row in one reduction (the second mean is expanded,
//   sum A x e = sum A x dh + Rh (sum A x dn - Rh m1 sum A x h),  m1 = mean(dn n)),
// then e, d_x and the column sums B = sum e q and sum d_y n.  Both remaining
// gradients follow from B, since the gate is constant over the rows of a unit:
//   d_gate = scale w_post B,  d_post = scale gate B
// (a gate with a row of its own for each row: d_gate per row, B over e q gate).
// Rows come through `stages` stages of shared memory that cp.async fills ahead.  A thread copies
// and reads the same columns, 2 or 8 at an access; rows of odd width or address (VEC 1) come as the
// 16-byte pieces that hold them, each shifted by its own offset.  Absent arrays and columns behind
// the row are zeros there, so that nothing but the stores is guarded: 12000 float16 rows of 2051
// take 191 us instead of 541, 16384 bfloat16 rows of 1030 80 us instead of 107.  The widest forms with a
// gate row for each row (VEC 1 or 2, EL 16) spill up to 392 bytes.
// Bound by memory, then by instructions: 16384 bfloat16 rows of 4096 take 132 us and 140 us with the
// column sums, 805 MB at 5.8 TB/s; scalar float32 arithmetic and bounds checks on every access took
// 182 us.
struct NormGrad {
    NormArgs a;
    const void *h, *x, *dh, *dy;
    void *dres, *dx, *dgate;  // dgate: only with a gate row for each row
    float *part_b, *part_pre;
    int64_t units, units_per_gate;
    int stages, cluster, block_width;
};

// Sums of 8 values over the block; every thread gets all of them, in the same order.
// One barrier; `red` [warps][8] is used again two calls later at the earliest.
__device__ __forceinline__ void sum8(float (&v)[8], float* red, int warps) {
    const int lane = threadIdx.x & 31;
    // a lane keeps half of its values in each of three exchanges, then sums the last one over 4 lanes
    float w4[4], w2[2], w1;
    const bool b4 = lane & 16, b3 = lane & 8, b2 = lane & 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w4[i] = (b4 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, b4 ? v[i] : v[4 + i], 16);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w2[i] = (b3 ? w4[2 + i] : w4[i]) + __shfl_xor_sync(0xffffffffu, b3 ? w4[i] : w4[2 + i], 8);
    w1 = (b2 ? w2[1] : w2[0]) + __shfl_xor_sync(0xffffffffu, b2 ? w2[0] : w2[1], 4);
    w1 += __shfl_xor_sync(0xffffffffu, w1, 2);
    w1 += __shfl_xor_sync(0xffffffffu, w1, 1);
    // lanes 4 i .. 4 i + 3 hold value i = 4 (lane bit 4) + 2 (lane bit 3) + (lane bit 2)
    if (warps == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __shfl_sync(0xffffffffu, w1, 4 * i);
        __syncwarp();
        return;
    }
    if ((lane & 3) == 0) red[(threadIdx.x >> 5) * 8 + (lane >> 2)] = w1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    for (int w = 0; w < warps; ++w) {
        const float4 lo = reinterpret_cast<const float4*>(red)[2 * w], hi = reinterpret_cast<const float4*>(red)[2 * w + 1];
        v[0] += lo.x;
        v[1] += lo.y;
        v[2] += lo.z;
        v[3] += lo.w;
        v[4] += hi.x;
        v[5] += hi.y;
        v[6] += hi.z;
        v[7] += hi.w;
    }
}

// Eight columns of a thread, held as pairs for the two-lane float32 instructions: the accesses
// [chunk 8 / VEC, (chunk + 1) 8 / VEC) of VEC columns, the accesses of a row T VEC columns apart.
// `c` is the thread's first column, d the row's end; WHOLE: every column is inside.
template <int VEC, bool WHOLE, typename L>
__device__ __forceinline__ void get8(int chunk, int c, int stride, int d, float2 (&f)[4], L load) {
#pragma unroll
    for (int i = 0; i < 8 / VEC; ++i) {
        const int col = c + (chunk * (8 / VEC) + i) * stride;
        float v[VEC];
        if (!WHOLE)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
        if (WHOLE || col < d) load(col, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) (((i * VEC + j) & 1) ? f[(i * VEC + j) / 2].y : f[(i * VEC + j) / 2].x) = v[j];
    }
}
template <int VEC, bool WHOLE, typename S>
__device__ __forceinline__ void put8(int chunk, int c, int stride, int d, const float2 (&f)[4], S store) {
#pragma unroll
    for (int i = 0; i < 8 / VEC; ++i) {
        const int col = c + (chunk * (8 / VEC) + i) * stride;
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = ((i * VEC + j) & 1) ? f[(i * VEC + j) / 2].y : f[(i * VEC + j) / 2].x;
        if (WHOLE || col < d) store(col, v);
    }
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Begins to copy the 16-byte pieces that hold src[0, count) to `dst`, which is 16-byte aligned:
// src[i] comes to lie at dst[ahead(src) + i].  Nothing before `array`, where src's array starts,
// is read, and nothing behind src[count - 1]: at least 16 bytes of zeros follow it, more than ahead()
// can put one row before another, so that an earlier row's end does not show behind it.  The block's
// threads share the pieces.
template <typename T>
__device__ __forceinline__ int ahead(const T* src) {
    return (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
}
template <typename T>
__device__ __forceinline__ void copy_span(T* dst, const T* array, const T* src, int count) {
    const uintptr_t start = reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15;
    const int bytes = (ahead(src) + count) * (int)sizeof(T);
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    for (int i = 16 * threadIdx.x; i < bytes + 16; i += 16 * blockDim.x) {
        if (start + i >= reinterpret_cast<uintptr_t>(array)) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i), "l"(start + i),
                         "r"(max(0, min(16, bytes - i)))
                         : "memory");
        } else {  // the first piece of an array that starts inside it
            const int from = ahead(src);
            for (int j = from; j < 16 / (int)sizeof(T); ++j) dst[j] = j < from + count ? src[j - from] : T(0.0f);
        }
    }
}

// What a call has.  kAllWhole: x, d_h, d_y and post_weight, and the threads' columns are the row's.
// kParts: d_y, and post_weight or no x.  kFewParts: no d_y, or x without post_weight; then e = d_h
// whatever h holds, or d_x = dq whatever x holds, so that their arithmetic is left out instead of
// multiplied by zero, which infinities, NaN and rows of zeros (eps 0) would turn into NaN.  A form of
// its own, since these branches cost the others 2 to 10% (12000 float16 rows of 2050: 148 us to 161).
enum NormForm { kAllWhole, kParts, kFewParts };
template <typename TR, typename TX, int VEC, int EL, bool OWN_GATE, NormForm FORM>
__global__ void __launch_bounds__(512) norm_grad_kernel(NormGrad k) {
    next_kernel_may_start();
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) float red[2][16 * 8];
    __shared__ __align__(16) float peer_sums[2][8];
    namespace cg = cooperative_groups;
    constexpr bool WHOLE = FORM == kAllWhole;
    const NormArgs& a = k.a;
    const int tid = threadIdx.x, T = blockDim.x, warps = T >> 5;
    const int64_t width = a.width;
    const int rank = k.cluster > 1 ? (int)(blockIdx.x % k.cluster) : 0;
    const int64_t col0 = (int64_t)rank * k.block_width, worker = blockIdx.x / k.cluster, workers = gridDim.x / k.cluster;
    const int d = (int)min((int64_t)k.block_width, width - col0);  // columns of this block, counted from col0
    constexpr bool kSpans = VEC == 1;
    const int slots = T * EL + (kSpans ? 16 : 0), c = tid * VEC, stride = T * VEC;
    const float inv_d = 1.0f / (float)width;
    const bool has_x = WHOLE || k.x != nullptr, has_dh = WHOLE || k.dh != nullptr, has_dy = WHOLE || k.dy != nullptr;
    const bool has_post = WHOLE || a.post_w != nullptr;
    // whether h and d_y, and the second mean's sums, take part
    const bool use_h = FORM != kFewParts || has_dy, use_mean = FORM != kFewParts || has_post;
    const int64_t pitch = align_up(width, 8);
    // a stage: h, dh, x, dy
    const int stage_bytes = slots * 2 * (int)(sizeof(TR) + sizeof(TX));
    auto stage_r = [&](int s, int i) { return reinterpret_cast<TR*>(smem + s * stage_bytes) + i * slots; };
    auto stage_x = [&](int s, int i) {
        return reinterpret_cast<TX*>(smem + s * stage_bytes + 2 * slots * (int)sizeof(TR)) + i * slots;
    };
    auto fetch = [&](int s, int64_t r) {
        const int64_t at = r * width + col0;
        const TR *h = static_cast<const TR*>(k.h) + at, *dh = static_cast<const TR*>(k.dh) + at;
        const TX *x = static_cast<const TX*>(k.x) + at, *dy = static_cast<const TX*>(k.dy) + at;
        TR *sh = stage_r(s, 0), *sdh = stage_r(s, 1);
        TX *sx = stage_x(s, 0), *sdy = stage_x(s, 1);
        if constexpr (kSpans) {
            if (use_h) copy_span(sh, static_cast<const TR*>(k.h), h, d);
            if (has_x) copy_span(sx, static_cast<const TX*>(k.x), x, d);
            if (has_dh) copy_span(sdh, static_cast<const TR*>(k.dh), dh, d);
            if (has_dy) copy_span(sdy, static_cast<const TX*>(k.dy), dy, d);
            return;
        }
#pragma unroll
        for (int i = 0; i < EL / VEC; ++i) {
            const int col = c + i * stride;
            if (!WHOLE && col >= d) break;
            if (use_h) copy_vec<TR, VEC>(sh + col, h + col);
            if (has_x) copy_vec<TX, VEC>(sx + col, x + col);
            if (has_dh) copy_vec<TR, VEC>(sdh + col, dh + col);
            if (has_dy) copy_vec<TX, VEC>(sdy + col, dy + col);
        }
    };
    auto block_sync = [&] {
        if (warps > 1)
            __syncthreads();
        else
            __syncwarp();
    };
    constexpr int Q = EL / 8;
    float2 pre[Q][4], post[Q][4], sum_b[Q][4], sum_pre[Q][4];
    // factors of the thread's columns: v = 1, then v *= each array
    auto factors = [&](float2 (&v)[Q][4], float start) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[q][j] = both(start);
    };
    auto multiply = [&](float2 (&v)[Q][4], const void* p, int dtype, int64_t at) {
        with_any(p, dtype, [&](auto* w) {
            using T0 = std::remove_cv_t<std::remove_pointer_t<decltype(w)>>;
            float2 f[Q][4];
#pragma unroll
            for (int q = 0; q < Q; ++q)
                get8<VEC, WHOLE>(q, c, stride, d, f[q],
                                 [&](int col, float (&x)[VEC]) { load_global<T0, VEC>(w + at + col, x); });
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[q][j] = __fmul2_rn(v[q][j], f[q][j]);
        });
    };
    if (!WHOLE) {  // absent arrays and the columns behind the row read as zero: no bounds checks then
        for (int st = 0; st < k.stages; ++st) {
            for (int i = tid + (has_dh ? d : 0); i < slots; i += T) stage_r(st, 1)[i] = TR(0.0f);
            for (int i = tid + (has_x ? d : 0); i < slots; i += T) stage_x(st, 0)[i] = TX(0.0f);
            for (int i = tid + (has_dy ? d : 0); i < slots; i += T) stage_x(st, 1)[i] = TX(0.0f);
            for (int i = tid + (use_h ? d : 0); i < slots; i += T) stage_r(st, 0)[i] = TR(0.0f);
        }
        block_sync();
    }
    factors(pre, has_dy ? 1.0f : 0.0f);
    if (has_dy) multiply(pre, a.pre_w, a.w_dtype, col0);
    factors(sum_pre, 0.0f);
    int parity = 0;
    for (int64_t u = worker; u < k.units; u += workers) {
        const int64_t g = u / k.units_per_gate, part = u % k.units_per_gate;
        const int64_t r0 = g * a.rows_per_gate + part * a.rows_per_gate / k.units_per_gate;
        const int64_t r1 = g * a.rows_per_gate + (part + 1) * a.rows_per_gate / k.units_per_gate;
        for (int i = 0; i < k.stages - 1; ++i) {
            if (r0 + i < r1) fetch(i, r0 + i);
            copy_commit();
        }
        factors(post, has_x ? a.scale : 0.0f);  // A of above; with OWN_GATE without the gate
        if (has_post) multiply(post, a.post_w, a.w_dtype, col0);
        if (a.gate != nullptr && !OWN_GATE) multiply(post, a.gate, a.gate_dtype, g * width + col0);
        factors(sum_b, 0.0f);
        int s = 0;
        for (int64_t r = r0; r < r1; ++r) {
            if (k.stages == 1) {
                if (kSpans) block_sync();
                fetch(0, r);
                copy_commit();
            }
            if (k.stages >= 4)
                copy_wait<2>();
            else if (k.stages == 3)
                copy_wait<1>();
            else
                copy_wait<0>();
            const int64_t at = r * width + col0;
            const TR *sh = stage_r(s, 0), *sdh = stage_r(s, 1);
            const TX *sx = stage_x(s, 0), *sdy = stage_x(s, 1);
            if constexpr (kSpans) {
                block_sync();  // the other threads' pieces
                sh += ahead(static_cast<const TR*>(k.h) + at);
                sdh += ahead(static_cast<const TR*>(k.dh) + at);
                sx += ahead(static_cast<const TX*>(k.x) + at);
                sdy += ahead(static_cast<const TX*>(k.dy) + at);
            }
            auto load_r = [&](int q, const TR* p, float2 (&f)[4]) {
                get8<VEC, true>(q, c, stride, d, f, [&](int col, float (&v)[VEC]) { load_vec<TR, VEC>(p + col, v); });
            };
            auto load_x = [&](int q, const TX* p, float2 (&f)[4]) {
                get8<VEC, true>(q, c, stride, d, f, [&](int col, float (&v)[VEC]) { load_vec<TX, VEC>(p + col, v); });
            };
            auto load_gate = [&](int q, float2 (&f)[4]) {
                with_any(a.gate, a.gate_dtype, [&](auto* w) {
                    using T0 = std::remove_cv_t<std::remove_pointer_t<decltype(w)>>;
                    get8<VEC, true>(q, c, stride, d, f, [&](int col, float (&v)[VEC]) {
                        load_global<T0, VEC>(w + at + (WHOLE ? col : min(col, d - VEC)), v);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) v[j] = WHOLE || col < d ? v[j] : 0.0f;
                    });
                });
            };
            float2 t2[6] = {};
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                float2 h[4], x[4], dh[4], dy[4], gate[4];
                if constexpr (FORM == kFewParts) {
                    if (use_h) {
                        load_r(q, sh, h);
                        load_x(q, sdy, dy);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            t2[0] = __ffma2_rn(h[j], h[j], t2[0]);
                            t2[2] = __ffma2_rn(__fmul2_rn(dy[j], pre[q][j]), h[j], t2[2]);
                        }
                    }
                    if (use_mean) {  // and no d_y
                        load_x(q, sx, x);
                        load_r(q, sdh, dh);
                        if (OWN_GATE) load_gate(q, gate);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float2 ax = __fmul2_rn(post[q][j], x[j]);
                            if (OWN_GATE) ax = __fmul2_rn(ax, gate[j]);
                            t2[1] = __ffma2_rn(x[j], x[j], t2[1]);
                            t2[3] = __ffma2_rn(ax, dh[j], t2[3]);
                        }
                    }
                    continue;
                }
                load_r(q, sh, h);
                load_x(q, sx, x);
                load_r(q, sdh, dh);
                load_x(q, sdy, dy);
                if (OWN_GATE) load_gate(q, gate);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 dn = __fmul2_rn(dy[j], pre[q][j]);
                    float2 ax = __fmul2_rn(post[q][j], x[j]);
                    if (OWN_GATE) ax = __fmul2_rn(ax, gate[j]);
                    t2[0] = __ffma2_rn(h[j], h[j], t2[0]);
                    t2[1] = __ffma2_rn(x[j], x[j], t2[1]);
                    t2[2] = __ffma2_rn(dn, h[j], t2[2]);
                    t2[3] = __ffma2_rn(ax, dh[j], t2[3]);
                    t2[4] = __ffma2_rn(ax, dn, t2[4]);
                    t2[5] = __ffma2_rn(ax, h[j], t2[5]);
                }
            }
            float t[8] = {};
#pragma unroll
            for (int i = 0; i < 6; ++i) t[i] = t2[i].x + t2[i].y;
            sum8(t, red[parity], warps);
            if (k.cluster > 1) {
                cg::cluster_group cluster = cg::this_cluster();
                if (tid == 0)
#pragma unroll
                    for (int i = 0; i < 8; ++i) peer_sums[parity][i] = t[i];
                cluster.sync();
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = 0.0f;
                for (int q = 0; q < k.cluster; ++q) {
                    const float* peer = cluster.map_shared_rank(peer_sums[parity], q);
#pragma unroll
                    for (int i = 0; i < 6; ++i) t[i] += peer[i];
                }
            }
            parity ^= 1;
            // every thread has left the previous row: its stage takes the row stages - 1 ahead
            if (k.stages > 1) {
                const int free_stage = s == 0 ? k.stages - 1 : s - 1;
                if (r + k.stages - 1 < r1) fetch(free_stage, r + k.stages - 1);
                copy_commit();
            }
            const float rh = use_h ? rsqrtf(t[0] * inv_d + a.eps) : 0.0f;
            const float m1 = t[2] * rh * inv_d;
            float rx = 1.0f, m2 = 0.0f;
            if (has_post) {
                rx = rsqrtf(t[1] * inv_d + a.eps);
                m2 = rx * inv_d * (t[3] + rh * (t[4] - rh * m1 * t[5]));
            }
            const float2 minus_m1 = both(-m1), minus_m2 = both(-m2), rh2 = both(rh), rx2 = both(rx);
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                float2 h[4], x[4], e[4], dy[4], gate[4];
                load_r(q, sh, h);
                load_x(q, sx, x);
                load_r(q, sdh, e);
                load_x(q, sdy, dy);
                if (OWN_GATE) load_gate(q, gate);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 n = __fmul2_rn(h[j], rh2), p = __fmul2_rn(x[j], rx2);
                    if (use_h) e[j] = __ffma2_rn(rh2, __ffma2_rn(n, minus_m1, __fmul2_rn(dy[j], pre[q][j])), e[j]);
                    float2 dq = __fmul2_rn(post[q][j], e[j]);
                    if (OWN_GATE) {
                        dy[j] = __fmul2_rn(dy[j], n);
                        sum_pre[q][j] = __fadd2_rn(sum_pre[q][j], dy[j]);
                        dy[j] = __fmul2_rn(dq, p);  // d_gate
                        dq = __fmul2_rn(dq, gate[j]);
                        sum_b[q][j] = __ffma2_rn(__fmul2_rn(e[j], gate[j]), p, sum_b[q][j]);
                    } else {
                        sum_pre[q][j] = __ffma2_rn(dy[j], n, sum_pre[q][j]);
                        sum_b[q][j] = __ffma2_rn(e[j], p, sum_b[q][j]);
                    }
                    x[j] = use_mean ? __fmul2_rn(rx2, __ffma2_rn(p, minus_m2, dq)) : dq;  // d_x
                }
                put8<VEC, WHOLE>(q, c, stride, d, e, [&](int col, const float (&v)[VEC]) {
                    store_global<TR, VEC>(static_cast<TR*>(k.dres) + at + col, v);
                });
                if (has_x)
                    put8<VEC, WHOLE>(q, c, stride, d, x, [&](int col, const float (&v)[VEC]) {
                        store_global<TX, VEC>(static_cast<TX*>(k.dx) + at + col, v);
                    });
                if (OWN_GATE)
                    put8<VEC, WHOLE>(q, c, stride, d, dy, [&](int col, const float (&v)[VEC]) {
                        store_any_vec<VEC>(k.dgate, a.gate_dtype, at + col, v);
                    });
            }
            s = s == k.stages - 1 ? 0 : s + 1;
        }
        copy_wait<0>();
        block_sync();  // the next unit fills the stages again
        if (has_x)
#pragma unroll
            for (int q = 0; q < Q; ++q)
                put8<VEC, WHOLE>(q, c, stride, d, sum_b[q], [&](int col, const float (&v)[VEC]) {
                    store_global<float, VEC>(k.part_b + u * pitch + col0 + col, v);
                });
    }
    if (has_dy)
#pragma unroll
        for (int q = 0; q < Q; ++q)
            put8<VEC, WHOLE>(q, c, stride, d, sum_pre[q], [&](int col, const float (&v)[VEC]) {
                store_global<float, VEC>(k.part_pre + worker * pitch + col0 + col, v);
            });
    if (k.cluster > 1) cg::this_cluster().sync();  // a peer may still read this block's sums
}

// Sums of `count` consecutive rows of `part` (width columns, rows align_up(width, 8)
// apart) for each group y: a block takes 32 columns, its 8 warps every eighth row.
//   sum B of the group:  d_gate[y] = scale post B,  and scale gate[y] B into `out` or,
//                        with more than one group, into row y of `post_rows`
//   plain sums:          into `out` (which = 1: pre weight, 2: post weight over groups)
struct NormColumns {
    const float* part;
    int64_t count, groups;
    int which;  // 0: sum B
    void *out, *dgate;
    float* post_rows;
};

// Two such jobs in one launch, blockIdx.z apart.
__global__ void __launch_bounds__(kThreads) norm_columns_kernel(NormArgs a, NormColumns first, NormColumns second) {
    __shared__ float sh[kWarps][32];
    const NormColumns& k = blockIdx.z == 0 ? first : second;
    next_kernel_may_start();
    previous_kernel_done();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane, d = a.width, pitch = align_up(d, 8);
    for (int64_t g = blockIdx.y; g < k.groups; g += gridDim.y) {
        float s = 0.0f;
        if (c < d)
            for (int64_t i = warp; i < k.count; i += kWarps) s += k.part[(g * k.count + i) * pitch + c];
        sh[warp][lane] = s;
        __syncthreads();
        if (warp == 0 && c < d) {
            s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) s += sh[w][lane];
            if (k.which != 0) {
                store_any(k.out, a.w_dtype, c, s);
            } else {
                s *= a.scale;
                if (k.dgate != nullptr)
                    store_any(k.dgate, a.gate_dtype, g * d + c,
                              a.post_w != nullptr ? s * load_any(a.post_w, a.w_dtype, c) : s);
                if (a.post_w != nullptr) {
                    if (k.dgate != nullptr) s *= load_any(a.gate, a.gate_dtype, g * d + c);
                    if (k.groups > 1)
                        k.post_rows[g * pitch + c] = s;
                    else
                        store_any(k.out, a.w_dtype, c, s);
                }
            }
        }
        __syncthreads();
    }
}

// Threads of a block, resident blocks to fill and the units of a backward pass, from
// the sizes alone.
struct NormGradPlan {
    NormShape shape;
    int64_t workers, units, units_per_gate;  // workers: blocks or clusters
    int64_t off_b, off_pre, off_post, bytes;
};
static NormGradPlan norm_grad_plan(int64_t n, int64_t width, int64_t gate_rows, int elems) {
    NormGradPlan p{};
    p.shape = norm_shape(width, elems);
    const int64_t want = 148 * std::max(1, 512 / p.shape.threads) / p.shape.cluster;
    const bool own = gate_rows == n && n > 1;
    const int64_t groups = own || gate_rows < 1 ? 1 : gate_rows;
    const int64_t rows = n / groups;
    p.units_per_gate = std::min(rows, std::max<int64_t>(1, want / groups));
    p.units = groups * p.units_per_gate;
    p.workers = std::min(p.units, want);
    const int64_t pitch = 4 * align_up(width, 8);
    p.off_b = 0;
    p.off_pre = align_up(p.off_b + p.units * pitch, 256);
    p.off_post = align_up(p.off_pre + p.workers * pitch, 256);
    p.bytes = align_up(p.off_post + (groups > 1 ? groups : 0) * pitch, 256);
    return p;
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
    CRESSO_REQUIRE(width <= kNormMaxWidth && n <= CRESSO_TRAIN_MAX_ROWS / 8, CRESSO_EUNSUPPORTED,
                   "block_norm: more than %d columns or 2^28 - 32 rows", kNormMaxWidth);
    CRESSO_REQUIRE(residual != nullptr && (x == nullptr || h != nullptr) && (pre_weight == nullptr) == (y == nullptr) &&
                       (x != nullptr || y != nullptr),
                   CRESSO_EINVAL, "block_norm: NULL pointer, or y without pre_weight");
    NvtxRange range("block_norm n=%lld", (long long)n);
    const NormArgs a{post_weight, pre_weight, gate, n, width, gate != nullptr ? n / gate_rows : n,
                     (int)weight_dtype, (int)gate_dtype, (float)scale, (float)eps};
    const int64_t rb = dtype_bytes(res_dtype), xb = dtype_bytes(act_dtype), wb = dtype_bytes(weight_dtype),
                  gb = dtype_bytes(gate_dtype);
    // the widest accesses that the width and the addresses allow
    auto fits = [&](int64_t vec) {
        auto ok = [&](const void* q, int64_t bytes) { return aligned_to(q, std::min<int64_t>(32, vec * bytes)); };
        return width % vec == 0 && ok(residual, rb) && ok(h, rb) && ok(x, xb) && ok(y, xb) && ok(post_weight, wb) &&
               ok(pre_weight, wb) && ok(gate, gb);
    };
    const int vec = fits(8) ? 8 : fits(2) ? 2 : 1;
    // single columns: 12000 bfloat16 rows of 1031 take 60 us with 8 a thread and 66 with 16; of 2051 they
    // take 133 and 138, float32 ones 110 and 85
    const NormShape p = norm_shape(width, n < kNormFewRows || (vec == 1 && width <= 2048) ? 8 : 16);
    return with_norm_types(res_dtype, act_dtype, [&](auto tr, auto tx) {
        using TR = decltype(tr);
        using TX = decltype(tx);
        auto launch = [&](auto kernel) {
            const int rows = p.threads == 32 ? 4 : 1;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((unsigned)(ceil_div(n, rows) * p.cluster));
            cfg.blockDim = dim3((unsigned)p.threads, (unsigned)rows);
            cfg.stream = (cudaStream_t)stream;
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = (unsigned)p.cluster;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = p.cluster > 1 ? 1 : 0;
            CRESSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, static_cast<const TR*>(residual), static_cast<const TX*>(x),
                                           static_cast<TR*>(h), static_cast<TX*>(y), p.cluster, p.block_width));
            CRESSO_LAUNCHED("norm_kernel");
            return (int)CRESSO_OK;
        };
        if (p.elems == 8)
            return vec == 8   ? launch(norm_kernel<TR, TX, 8, 8>)
                   : vec == 2 ? launch(norm_kernel<TR, TX, 2, 8>)
                              : launch(norm_kernel<TR, TX, 1, 8>);
        return vec == 8   ? launch(norm_kernel<TR, TX, 8, 16>)
               : vec == 2 ? launch(norm_kernel<TR, TX, 2, 16>)
                          : launch(norm_kernel<TR, TX, 1, 16>);
    });
}

int cresso_block_norm_grad_scratch_bytes(int64_t n, int64_t width, int64_t gate_rows, int64_t* bytes) {
    CRESSO_REQUIRE(bytes != nullptr, CRESSO_EINVAL, "block_norm_grad_scratch_bytes: NULL result");
    CRESSO_REQUIRE(n >= 0 && width >= 0 && gate_rows >= 0, CRESSO_EINVAL, "block_norm_grad: negative size");
    CRESSO_REQUIRE(width <= kNormMaxWidth, CRESSO_EUNSUPPORTED, "block_norm_grad: width above %d", kNormMaxWidth);
    *bytes = n == 0 || width == 0 ? 0
                                   : std::max(norm_grad_plan(n, width, gate_rows, 8).bytes,
                                              norm_grad_plan(n, width, gate_rows, 16).bytes);
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
    CRESSO_REQUIRE(width <= kNormMaxWidth && n <= CRESSO_TRAIN_MAX_ROWS / 8, CRESSO_EUNSUPPORTED,
                   "block_norm_grad: more than %d columns or 2^28 - 32 rows", kNormMaxWidth);
    CRESSO_REQUIRE(x != nullptr || (post_weight == nullptr && gate == nullptr), CRESSO_EINVAL,
                   "block_norm_grad: a post weight or a gate needs x");
    CRESSO_REQUIRE(h != nullptr && d_residual != nullptr && (d_h != nullptr || d_y != nullptr) &&
                       (d_y == nullptr || pre_weight != nullptr),
                   CRESSO_EINVAL, "block_norm_grad: NULL pointer, or d_y without pre_weight");
    CRESSO_REQUIRE((x != nullptr) == (d_x != nullptr) && (post_weight != nullptr) == (d_post_weight != nullptr) &&
                       (d_y != nullptr) == (d_pre_weight != nullptr) && (gate != nullptr) == (d_gate != nullptr),
                   CRESSO_EINVAL, "block_norm_grad: an input without its gradient, or a gradient without its input");
    const bool own = gate != nullptr && gate_rows == n && n > 1;
    const int64_t rb = dtype_bytes(res_dtype), xb = dtype_bytes(act_dtype), gb = dtype_bytes(gate_dtype);
    // the widest accesses that the width and the addresses allow
    auto fits = [&](int vec) {
        if (width % vec != 0) return false;
        const int64_t ar = std::min<int64_t>(32, vec * rb), ax = std::min<int64_t>(32, vec * xb);
        const int64_t ag = std::min<int64_t>(32, vec * gb), aw = std::min<int64_t>(32, vec * dtype_bytes(weight_dtype));
        return aligned_to(h, ar) && aligned_to(d_h, ar) && aligned_to(d_residual, ar) && aligned_to(x, ax) &&
               aligned_to(d_y, ax) && aligned_to(d_x, ax) && aligned_to(gate, ag) && (!own || aligned_to(d_gate, ag)) &&
               aligned_to(post_weight, aw) && aligned_to(pre_weight, aw);
    };
    const int vec = fits(8) ? 8 : fits(2) ? 2 : 1;
    // narrow accesses cost instructions: 8 columns a thread (1023 rows of 2050 float16: 24 us
    // instead of 31); wide ones leave fewer warps to the reduction with 16 (1100 rows of 4096
    // bfloat16: 24.5 us instead of 29.8; 100 rows: 10.3 instead of 11.5)
    const NormGradPlan p = norm_grad_plan(n, width, gate != nullptr ? gate_rows : 0, vec < 8 ? 8 : 16);
    CRESSO_REQUIRE(scratch != nullptr && scratch_bytes >= p.bytes, CRESSO_ESCRATCH,
                   "block_norm_grad: scratch has %lld bytes, %lld are needed", (long long)scratch_bytes,
                   (long long)p.bytes);
    CRESSO_REQUIRE(aligned_to(scratch, 32), CRESSO_EINVAL, "block_norm_grad: scratch is not 32-byte aligned");
    NvtxRange range("block_norm_grad n=%lld", (long long)n);
    const int64_t groups = gate == nullptr || own ? 1 : gate_rows;
    NormGrad k{};
    k.a = NormArgs{post_weight, pre_weight, gate, n, width, n / groups, (int)weight_dtype, (int)gate_dtype,
                   (float)scale, (float)eps};
    k.h = h;
    k.x = x;
    k.dh = d_h;
    k.dy = d_y;
    k.dres = d_residual;
    k.dx = d_x;
    k.dgate = own ? d_gate : nullptr;
    unsigned char* base = static_cast<unsigned char*>(scratch);
    k.part_b = reinterpret_cast<float*>(base + p.off_b);
    k.part_pre = reinterpret_cast<float*>(base + p.off_pre);
    k.units = p.units;
    k.units_per_gate = p.units_per_gate;
    k.cluster = p.shape.cluster;
    k.block_width = p.shape.block_width;
    const int stage = (int)((p.shape.threads * p.shape.elems + (vec == 1 ? 16 : 0)) * 2 * (rb + xb));
    // as many blocks an SM as the registers admit where each of them has two stages, else
    // as many stages as fit for one block
    const int share = kNormStageBytes / std::max(1, 512 / p.shape.threads) - 2048;
    k.stages = 2 * stage <= share ? std::min(4, share / stage) : std::min(4, kNormStageBytes / stage);
    const int smem = k.stages * stage;
    const int rc = with_norm_types(res_dtype, act_dtype, [&](auto tr, auto tx) {
        using TR = decltype(tr);
        using TX = decltype(tx);
        auto launch = [&](auto kernel) {
            // with the static part, 48 KB need no leave; one bound for all calls, since a kernel's bound
            // is shared by the host's threads and another one's smaller stages must not lower it
            if (smem > 40 * 1024)
                CRESSO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormStageBytes));
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((unsigned)(p.workers * p.shape.cluster));
            cfg.blockDim = dim3((unsigned)p.shape.threads);
            cfg.dynamicSmemBytes = (size_t)smem;
            cfg.stream = s;
            cudaLaunchAttribute attr{};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = (unsigned)p.shape.cluster;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = p.shape.cluster > 1 ? 1 : 0;
            CRESSO_CUDA(cudaLaunchKernelEx(&cfg, kernel, k));
            CRESSO_LAUNCHED("norm_grad_kernel");
            return (int)CRESSO_OK;
        };
        const bool whole = x != nullptr && d_h != nullptr && d_y != nullptr && post_weight != nullptr &&
                           p.shape.cluster == 1 && width == (int64_t)p.shape.threads * 16;
        auto with_form = [&](auto form) {
            constexpr NormForm F = decltype(form)::value;
            if (vec == 8)
                return own ? launch(norm_grad_kernel<TR, TX, 8, 16, true, F>) : launch(norm_grad_kernel<TR, TX, 8, 16, false, F>);
            if (p.shape.elems == 16)  // a row wider than 4096
                return vec == 2 ? (own ? launch(norm_grad_kernel<TR, TX, 2, 16, true, F>)
                                       : launch(norm_grad_kernel<TR, TX, 2, 16, false, F>))
                                : (own ? launch(norm_grad_kernel<TR, TX, 1, 16, true, F>)
                                       : launch(norm_grad_kernel<TR, TX, 1, 16, false, F>));
            if (vec == 2)
                return own ? launch(norm_grad_kernel<TR, TX, 2, 8, true, F>) : launch(norm_grad_kernel<TR, TX, 2, 8, false, F>);
            return own ? launch(norm_grad_kernel<TR, TX, 1, 8, true, F>) : launch(norm_grad_kernel<TR, TX, 1, 8, false, F>);
        };
        if (vec == 8 && !own && whole) return launch(norm_grad_kernel<TR, TX, 8, 16, false, kAllWhole>);
        if (d_y == nullptr || (x != nullptr && post_weight == nullptr))
            return with_form(std::integral_constant<NormForm, kFewParts>());
        return with_form(std::integral_constant<NormForm, kParts>());
    });
    if (rc != CRESSO_OK) return rc;
    float* post_rows = reinterpret_cast<float*>(base + p.off_post);
    NormArgs args = k.a;
    if (own) args.gate = nullptr;
    const bool sum_b = post_weight != nullptr || (gate != nullptr && !own), sum_pre = d_y != nullptr;
    const NormColumns job_b{k.part_b, p.units_per_gate, groups, 0, d_post_weight, own ? nullptr : d_gate, post_rows};
    const NormColumns job_pre{k.part_pre, p.workers, 1, 1, d_pre_weight, nullptr, nullptr};
    const unsigned blocks = (unsigned)ceil_div(width, 32);
    if (sum_b || sum_pre) {
        const dim3 grid(blocks, sum_b ? (unsigned)std::min<int64_t>(65535, groups) : 1, sum_b && sum_pre ? 2 : 1);
        CRESSO_CUDA(launch_overlapped(norm_columns_kernel, grid, kThreads, 0, s, args, sum_b ? job_b : job_pre, job_pre));
        CRESSO_LAUNCHED("norm_columns_kernel");
    }
    if (post_weight != nullptr && groups > 1) {  // the groups' rows to one
        const NormColumns job{post_rows, groups, 1, 2, d_post_weight, nullptr, nullptr};
        CRESSO_CUDA(launch_overlapped(norm_columns_kernel, dim3(blocks), kThreads, 0, s, args, job, job));
        CRESSO_LAUNCHED("norm_columns_kernel");
    }
    return CRESSO_OK;
}

}  // extern "C"

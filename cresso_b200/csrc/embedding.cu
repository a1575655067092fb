// Scaled embedding lookup and its gradient by sorted tokens.
//
// Lookup: out[t] = scale * W[token_t - row0].  Gradient: dW[r] = scale * sum of
// g[t] over the positions t whose token is row r.  The positions are brought into
// row order by a stable counting sort (positions ascending inside a row), so every
// row is summed in float32 in the order of its tokens: no atomics on values, the
// same bits every run, one rounding at the end.
#include "train_common.cuh"

#include <algorithm>

namespace cresso {

// ------------------------------------------------------------------ lookup ---

template <typename TW, typename TO>
__global__ void __launch_bounds__(kThreads) gather_kernel(const TW* __restrict__ w, int64_t rows, int64_t width,
                                                          int64_t stride, const void* __restrict__ tokens,
                                                          int token_bytes, int64_t row0, float scale,
                                                          TO* __restrict__ out) {
    const int64_t t = blockIdx.x;
    const uint64_t r = (uint64_t)load_id(tokens, token_bytes, t) - (uint64_t)row0;
    const bool inside = r < (uint64_t)rows;
    for (int64_t c = threadIdx.x; c < width; c += kThreads)
        out[t * width + c] = inside ? from_float<TO>(scale * to_float(w[(int64_t)r * stride + c])) : from_float<TO>(0.0f);
}

// ---------------------------------------------------------------- the sort ---
//
// One launch without any exchange between blocks: block b owns the rows
// [b * rb, (b + 1) * rb) and reads all tokens (they sit in L2).  Its 32 warps take
// equal contiguous ranges of positions.  First scan: each warp counts its tokens
// per row in shared memory, and the tokens below the block's rows, whose number is
// where the block's part of the order begins.  A scan over (row, warp) turns the
// counts into first places; the second scan puts each position at its place, lanes
// of one row ranked by a warp match, which keeps the positions ascending.
constexpr int kSortWarps = 32;
constexpr int kSortThreads = kSortWarps * 32;
constexpr int kSortMaxRows = 1536;  // rows of a block: kSortWarps counters each, 192 KB of shared memory

struct TokenWindow {
    const void* tokens;
    int token_bytes;
    int has_padding;
    int64_t n, rows, row0, padding;
};

// Row of position i in the window, -1 when the token takes no part.
__device__ __forceinline__ int window_row(const TokenWindow& w, int64_t i) {
    if (i >= w.n) return -1;
    const int64_t tok = load_id(w.tokens, w.token_bytes, i);
    const uint64_t r = (uint64_t)tok - (uint64_t)w.row0;
    return (r >= (uint64_t)w.rows || (w.has_padding && tok == w.padding)) ? -1 : (int)r;
}

__global__ void __launch_bounds__(kSortThreads) sort_kernel(TokenWindow win, int rb, int* __restrict__ row_start,
                                                            int* __restrict__ order) {
    extern __shared__ int cnt[];  // [kSortWarps][rb]
    __shared__ int warp_tot[kSortWarps], base_sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r0 = blockIdx.x * rb;
    const int nr = (int)min((int64_t)rb, win.rows - r0);
    for (int i = threadIdx.x; i < kSortWarps * rb; i += kSortThreads) cnt[i] = 0;
    if (threadIdx.x == 0) base_sh = 0;
    __syncthreads();
    const int64_t seg = ceil_div(ceil_div(win.n, kSortWarps), 32) * 32;
    const int64_t i0 = warp * seg, i1 = min(win.n, i0 + seg);
    int* mine = cnt + warp * rb;
    int below = 0;
    for (int64_t i = i0 + lane; i < i1; i += 32) {
        const int r = window_row(win, i) - r0;
        if (r >= 0 && r < nr) atomicAdd(&mine[r], 1);
        below += (r < 0 && r >= -r0) ? 1 : 0;  // r = -1 - r0: no part
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
    if (lane == 0 && below) atomicAdd(&base_sh, below);
    __syncthreads();
    // exclusive scan over the rows of the block, kSortThreads rows a turn
    int carry = base_sh;
    for (int c = 0; c < nr; c += kSortThreads) {
        const int r = c + threadIdx.x;
        int tot = 0;
        if (r < nr)
            for (int w = 0; w < kSortWarps; ++w) tot += cnt[w * rb + r];
        int incl = tot;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_tot[warp] = incl;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < kSortWarps; ++w) {
            const int v = warp_tot[w];
            before += w < warp ? v : 0;
            all += v;
        }
        int at = carry + before + incl - tot;
        if (r < nr) {
            row_start[r0 + r] = at;
            for (int w = 0; w < kSortWarps; ++w) {
                const int v = cnt[w * rb + r];
                cnt[w * rb + r] = at;
                at += v;
            }
        }
        carry += all;
        __syncthreads();
    }
    if (r0 + nr == win.rows && threadIdx.x == 0) row_start[win.rows] = carry;
    for (int64_t i = i0; i < i1; i += 32) {
        const int r = window_row(win, i + lane < i1 ? i + lane : win.n) - r0;
        const bool in = r >= 0 && r < nr;
        const unsigned any = __ballot_sync(0xffffffffu, in);
        if (any == 0) continue;
        if (in) {
            const unsigned same = __match_any_sync(any, r);
            const int rank = __popc(same & ((1u << lane) - 1u));
            const int at = mine[r];
            order[at + rank] = (int)(i + lane);
            __syncwarp(any);
            if (rank == 0) mine[r] = at + __popc(same);
        }
        __syncwarp();
    }
}

// One block sums one row.
template <typename TG, typename TO>
__global__ void __launch_bounds__(kThreads) grad_kernel(const TG* __restrict__ g, int64_t width, int64_t stride,
                                                        const int* __restrict__ row_start,
                                                        const int* __restrict__ order, float scale,
                                                        TO* __restrict__ out, int accumulate) {
    const int64_t r = blockIdx.x;
    const int s = row_start[r], e = row_start[r + 1];
    if (accumulate && s == e) return;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
        float acc = 0.0f;
        for (int j = s; j < e; ++j) acc += to_float(g[(int64_t)order[j] * stride + c]);
        acc *= scale;
        if (accumulate) acc += to_float(out[r * width + c]);
        out[r * width + c] = from_float<TO>(acc);
    }
}

}  // namespace cresso

using namespace cresso;

extern "C" {

int cresso_embedding_gather(const void* weight, int64_t weight_dtype, int64_t rows, int64_t width,
                            int64_t weight_stride, const void* tokens, int64_t token_bytes, int64_t n, int64_t row0,
                            double scale, void* out, int64_t out_dtype, cresso_stream_t stream) {
    CRESSO_REQUIRE(train_dtype_ok(weight_dtype) && train_dtype_ok(out_dtype), CRESSO_EUNSUPPORTED,
                   "embedding_gather: element types are float32, float16 and bfloat16");
    CRESSO_REQUIRE(token_bytes == 4 || token_bytes == 8, CRESSO_EINVAL, "embedding_gather: tokens are int32 or int64");
    CRESSO_REQUIRE(n >= 0 && rows >= 0 && width >= 0 && weight_stride >= width, CRESSO_EINVAL,
                   "embedding_gather: negative size, or row stride below the width");
    CRESSO_REQUIRE(n <= CRESSO_TRAIN_MAX_ROWS && rows <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED,
                   "embedding_gather: more than 2^31 - 256 tokens or rows");
    if (n == 0 || width == 0) return CRESSO_OK;
    CRESSO_REQUIRE((weight != nullptr || rows == 0) && tokens != nullptr && out != nullptr, CRESSO_EINVAL,
                   "embedding_gather: NULL pointer");
    NvtxRange range("embedding_gather n=%lld", (long long)n);
    return with_dtype(weight_dtype, [&](auto tw) {
        return with_dtype(out_dtype, [&](auto to) {
            using TW = decltype(tw);
            using TO = decltype(to);
            gather_kernel<TW, TO><<<(unsigned)n, kThreads, 0, (cudaStream_t)stream>>>(
                static_cast<const TW*>(weight), rows, width, weight_stride, tokens, (int)token_bytes, row0,
                (float)scale, static_cast<TO*>(out));
            CRESSO_LAUNCHED("gather_kernel");
            return (int)CRESSO_OK;
        });
    });
}

// scratch: row_start [rows + 1], order [n]
int cresso_embedding_grad_scratch_bytes(int64_t n, int64_t rows, int64_t width, int64_t* bytes) {
    CRESSO_REQUIRE(bytes != nullptr, CRESSO_EINVAL, "embedding_grad_scratch_bytes: NULL result");
    CRESSO_REQUIRE(n >= 0 && rows >= 0 && width >= 0, CRESSO_EINVAL, "embedding_grad: negative size");
    CRESSO_REQUIRE(n <= CRESSO_TRAIN_MAX_ROWS && rows <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED,
                   "embedding_grad: more than 2^31 - 256 tokens or rows");
    *bytes = align_up(4 * (rows + 1), 256) + align_up(4 * n, 256);
    return CRESSO_OK;
}

int cresso_embedding_grad(const void* grad, int64_t grad_dtype, int64_t n, int64_t width, int64_t grad_stride,
                          const void* tokens, int64_t token_bytes, int64_t rows, int64_t row0, int64_t has_padding,
                          int64_t padding, double scale, void* out, int64_t out_dtype, int64_t accumulate,
                          void* scratch, int64_t scratch_bytes, cresso_stream_t stream) {
    CRESSO_REQUIRE(train_dtype_ok(grad_dtype) && train_dtype_ok(out_dtype), CRESSO_EUNSUPPORTED,
                   "embedding_grad: element types are float32, float16 and bfloat16");
    CRESSO_REQUIRE(token_bytes == 4 || token_bytes == 8, CRESSO_EINVAL, "embedding_grad: tokens are int32 or int64");
    CRESSO_REQUIRE(grad_stride >= width, CRESSO_EINVAL, "embedding_grad: row stride below the width");
    int64_t need = 0;
    const int st = cresso_embedding_grad_scratch_bytes(n, rows, width, &need);
    if (st != CRESSO_OK) return st;
    if (rows == 0 || width == 0 || (n == 0 && accumulate)) return CRESSO_OK;
    CRESSO_REQUIRE(out != nullptr, CRESSO_EINVAL, "embedding_grad: NULL output");
    const cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        CRESSO_CUDA(cudaMemsetAsync(out, 0, (size_t)(rows * width * dtype_bytes(out_dtype)), s));
        return CRESSO_OK;
    }
    CRESSO_REQUIRE(grad != nullptr && tokens != nullptr, CRESSO_EINVAL, "embedding_grad: NULL pointer");
    CRESSO_REQUIRE(scratch != nullptr && scratch_bytes >= need, CRESSO_ESCRATCH,
                   "embedding_grad: scratch has %lld bytes, %lld are needed", (long long)scratch_bytes, (long long)need);
    NvtxRange range("embedding_grad n=%lld rows=%lld", (long long)n, (long long)rows);
    int* row_start = static_cast<int*>(scratch);
    int* order = reinterpret_cast<int*>(static_cast<unsigned char*>(scratch) + align_up(4 * (rows + 1), 256));
    const TokenWindow win{tokens, (int)token_bytes, has_padding != 0, n, rows, row0, padding};
    const int rb = (int)std::min<int64_t>(kSortMaxRows, std::max<int64_t>(1, ceil_div(rows, 148)));
    const int smem = kSortWarps * rb * 4;
    if (smem > 48 * 1024)
        CRESSO_CUDA(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kSortWarps * kSortMaxRows * 4));
    sort_kernel<<<(unsigned)ceil_div(rows, rb), kSortThreads, smem, s>>>(win, rb, row_start, order);
    CRESSO_LAUNCHED("sort_kernel");
    return with_dtype(grad_dtype, [&](auto tg) {
        return with_dtype(out_dtype, [&](auto to) {
            using TG = decltype(tg);
            using TO = decltype(to);
            grad_kernel<TG, TO><<<(unsigned)rows, kThreads, 0, s>>>(static_cast<const TG*>(grad), width, grad_stride,
                                                                   row_start, order, (float)scale,
                                                                   static_cast<TO*>(out), accumulate != 0);
            CRESSO_LAUNCHED("grad_kernel");
            return (int)CRESSO_OK;
        });
    });
}

}  // extern "C"

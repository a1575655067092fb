// Scaled embedding lookup and its gradient by sorted tokens.
//
// Lookup: out[t] = scale * W[token_t - row0].  Gradient: dW[r] = scale * sum of
// g[t] over the positions t whose token is row r.  The positions are brought into
// row order by a stable counting sort (positions ascending inside a row), so every
// row is summed in float32 in the order of its tokens: no atomics on values, the
// same bits every run, one rounding at the end.
#include "train_common.cuh"

#include <algorithm>
#include <type_traits>

namespace cresso {

// A row of `width` columns is taken by `tpr` threads (a power of two up to the block),
// VEC columns an access, COLS / VEC accesses of a thread in flight.
constexpr int kRowCols = 16;
template <int VEC>
constexpr int row_cols() { return VEC == 1 ? 8 : kRowCols; }
static int threads_per_row(int64_t width, int vec) {
    return (int)std::min<int64_t>(kThreads, pow2_ceil(ceil_div(width, vec)));
}

// f(std::integral_constant<int, VEC>) for the widest of 8, 4, 2 and 1 columns an access that
// the sizes and the addresses allow.
template <typename F>
int with_vec(int64_t width, int64_t stride, const void* p, int64_t p_bytes, const void* q, int64_t q_bytes, F f) {
    auto fits = [&](int vec) {
        return width % vec == 0 && stride % vec == 0 && aligned_to(p, std::min<int64_t>(16, vec * p_bytes)) &&
               aligned_to(q, std::min<int64_t>(16, vec * q_bytes));
    };
    if (fits(8)) return f(std::integral_constant<int, 8>());
    if (fits(4)) return f(std::integral_constant<int, 4>());
    if (fits(2)) return f(std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 1>());
}

// ------------------------------------------------------------------ lookup ---

template <typename TW, typename TO, int VEC>
__global__ void __launch_bounds__(kThreads) gather_kernel(const TW* __restrict__ w, int64_t rows, int64_t width,
                                                          int64_t stride, const void* __restrict__ tokens,
                                                          int token_bytes, int64_t n, int64_t row0, float scale,
                                                          TO* __restrict__ out, int tpr) {
    constexpr int U = row_cols<VEC>() / VEC;
    const int64_t t = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    if (t >= n) return;
    const uint64_t r = (uint64_t)load_id(tokens, token_bytes, t) - (uint64_t)row0;
    const bool inside = r < (uint64_t)rows;
    const TW* src = w + (inside ? (int64_t)r * stride : 0);
    TO* dst = out + t * width;
    for (int64_t c0 = (int64_t)(threadIdx.x & (tpr - 1)) * VEC; c0 < width; c0 += (int64_t)tpr * VEC * U) {
        float f[U][VEC] = {};
        if (inside)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + (int64_t)u * tpr * VEC;
                if (c < width) load_vec<TW, VEC>(src + c, f[u]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t c = c0 + (int64_t)u * tpr * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[u][j] = inside ? f[u][j] * scale : 0.0f;
            if (c < width) store_vec<TO, VEC>(dst + c, f[u]);
        }
    }
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
constexpr int kSortBatch = 8;      // tokens of a thread in flight
constexpr int kSortMaxRows = 1536;  // rows of a block: kSortWarps counters each, 192 KB of shared memory

struct TokenWindow {
    const void* tokens;
    int has_padding;
    int64_t n, rows, row0, padding;
};

// Rows in the window of the positions i, i + 32, ... below end; -1 where there is no position
// or the token takes no part.  All loads are issued before the first is used.
template <typename ID>
__device__ __forceinline__ void window_rows(const TokenWindow& w, int64_t i, int64_t end, int (&row)[kSortBatch]) {
    ID id[kSortBatch];
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) id[b] = static_cast<const ID*>(w.tokens)[min(i + 32 * b, w.n - 1)];
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
        const int64_t tok = (int64_t)id[b];
        const uint64_t r = (uint64_t)tok - (uint64_t)w.row0;
        const bool part = i + 32 * b < end && r < (uint64_t)w.rows && !(w.has_padding && tok == w.padding);
        row[b] = part ? (int)r : -1;
    }
}

template <typename ID>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(TokenWindow win, int rb, int* __restrict__ row_start,
                                                            int2* __restrict__ order) {
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
    for (int64_t i = i0 + lane; i < i1; i += 32 * kSortBatch) {
        int row[kSortBatch];
        window_rows<ID>(win, i, i1, row);
#pragma unroll
        for (int b = 0; b < kSortBatch; ++b) {
            if (row[b] >= r0 && row[b] - r0 < nr) atomicAdd(&mine[row[b] - r0], 1);
            below += row[b] >= 0 && row[b] < r0 ? 1 : 0;
        }
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
    for (int64_t i = i0; i < i1; i += 32 * kSortBatch) {
        int row[kSortBatch];
        window_rows<ID>(win, i + lane, i1, row);
#pragma unroll
        for (int b = 0; b < kSortBatch; ++b) {
            const int r = row[b] - r0;
            const bool in = r >= 0 && r < nr;
            const unsigned any = __ballot_sync(0xffffffffu, in);
            if (any == 0) continue;
            if (in) {
                const unsigned same = __match_any_sync(any, r);
                const int rank = __popc(same & ((1u << lane) - 1u));
                const int at = mine[r];
                order[at + rank] = make_int2((int)(i + 32 * b + lane), row[b]);
                __syncwarp(any);
                if (rank == 0) mine[r] = at + __popc(same);
            }
            __syncwarp();
        }
    }
}

// ----------------------------------------------------------------- the sums ---
//
// The order is cut into tiles of kTile positions, one work item each, so that the work is
// even however the tokens fall.  A tile reads its positions kFlight at a time whatever rows
// they belong to, and writes a row's sum where the row ends.  A row of up to kTile
// positions belongs to the tile it begins in.  A longer one is summed tile by tile into
// partial rows, which a second kernel adds in their order; a tile meets at most two such
// rows, one that reaches it from the left (partial 2 tile) and one that begins inside and
// leaves it to the right (partial 2 tile + 1).  Further items write the rows without a
// token, kEmptyRows rows each.
constexpr int kTile = 32;
constexpr int kEmptyRows = 8;
constexpr int kSumCols = 8;  // columns of a thread

// out row = scale * acc (+ out row)
template <typename TO, int VEC, int U>
__device__ __forceinline__ void write_row(TO* __restrict__ out, int64_t width, int64_t c0, int tpr, float scale,
                                          int accumulate, float (&acc)[U][VEC]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t c = c0 + (int64_t)u * tpr * VEC;
        if (c >= width) continue;
        float old[VEC] = {};
        if (accumulate) load_vec<TO, VEC>(out + c, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[u][i] = acc[u][i] * scale + old[i];
        store_vec<TO, VEC>(out + c, acc[u]);
    }
}

struct GradSums {
    const int* row_start;
    const int2* order;  // (position, row)
    float* partial;     // [2 tiles][pitch]
    int64_t rows, width, stride, tiles, pitch;
    float scale;
    int accumulate, tpr;
};

template <typename TG, typename TO, int VEC>
__global__ void __launch_bounds__(kThreads, VEC == 1 ? 3 : 4) grad_kernel(GradSums k, const TG* __restrict__ g,
                                                           TO* __restrict__ out) {
    constexpr int U = kSumCols / VEC;
    constexpr int kFlight = VEC <= 2 || sizeof(TG) == 4 ? 2 : 4;  // more of them would spill
    const int tpr = k.tpr;
    const int64_t item = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    const int64_t c0 = (int64_t)blockIdx.y * tpr * kSumCols + (int64_t)(threadIdx.x & (tpr - 1)) * VEC;
    float acc[U][VEC] = {};
    if (item >= k.tiles) {
        if (k.accumulate) return;  // a block's last groups
        const int64_t r0 = (item - k.tiles) * kEmptyRows;
        int start[kEmptyRows + 1];
#pragma unroll
        for (int i = 0; i <= kEmptyRows; ++i) start[i] = k.row_start[min(r0 + i, k.rows)];
#pragma unroll
        for (int i = 0; i < kEmptyRows; ++i)
            if (r0 + i < k.rows && start[i] == start[i + 1])
                write_row<TO, VEC, U>(out + (r0 + i) * k.width, k.width, c0, tpr, 1.0f, 0, acc);
        return;
    }
    const int total = k.row_start[k.rows];
    const int a = (int)item * kTile, b = min(a + kTile, total);
    if (a >= total) return;
    const int first = k.order[a].y, last = k.order[b - 1].y;
    const int first_start = k.row_start[first], first_end = k.row_start[first + 1];
    const int last_start = k.row_start[last], last_end = k.row_start[last + 1];
    // [from, to): the positions this item adds
    const int from = first_end - first_start > kTile || first_start == a ? a : min(first_end, b);
    const int to = last_end - last_start > kTile ? b : last_start >= a ? last_end : from;
    int row = -1, row_end = 0;
    for (int j = from; j < to; j += kFlight) {
        Raw<TG, VEC> f[kFlight][U];
        int rows[kFlight];
#pragma unroll
        for (int p = 0; p < kFlight; ++p) {
            const int2 o = k.order[min(j + p, to - 1)];
            rows[p] = o.y;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + (int64_t)u * tpr * VEC;
                if (c < k.width) f[p][u].load_once(g + (int64_t)o.x * k.stride + c);
            }
        }
#pragma unroll
        for (int p = 0; p < kFlight; ++p) {
            if (j + p >= to) break;
            if (rows[p] != row) {
                row = rows[p];
                row_end = k.row_start[row + 1];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[u][i] = 0.0f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c0 + (int64_t)u * tpr * VEC < k.width)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[u][i] += f[p][u].get(i);
            if (j + p + 1 != row_end && j + p + 1 != to) continue;
            // the row ends here, or the item does: a long row leaves a partial row
            const int begin = row == first ? first_start : row == last ? last_start : 0;
            const bool is_long = (row == first || row == last) && row_end - begin > kTile;
            if (is_long)
                write_row<float, VEC, U>(k.partial + (2 * item + (begin > a ? 1 : 0)) * k.pitch, k.width, c0, tpr, 1.0f,
                                         0, acc);
            else
                write_row<TO, VEC, U>(out + (int64_t)row * k.width, k.width, c0, tpr, k.scale, k.accumulate, acc);
        }
    }
}

// Adds the partial rows of the long row that begins in tile blockIdx.x; a thread has a column.
template <typename TO>
__global__ void __launch_bounds__(kThreads) grad_join_kernel(GradSums k, TO* __restrict__ out) {
    const int total = k.row_start[k.rows];
    const int64_t tile = blockIdx.x;
    const int a = (int)tile * kTile, b = min(a + kTile, total);
    if (a >= total) return;
    const int64_t r = k.order[b - 1].y;
    const int s = k.row_start[r], e = k.row_start[r + 1];
    if (e - s <= kTile || s < a) return;
    const int64_t last = (e - 1) / kTile;
    for (int64_t c = (int64_t)blockIdx.y * kThreads + threadIdx.x; c < k.width; c += (int64_t)gridDim.y * kThreads) {
        float acc = k.partial[(2 * tile + (s > a ? 1 : 0)) * k.pitch + c];
#pragma unroll 8
        for (int64_t i = tile + 1; i <= last; ++i) acc += k.partial[2 * i * k.pitch + c];
        acc *= k.scale;
        if (k.accumulate) acc += to_float(out[r * k.width + c]);
        out[r * k.width + c] = from_float<TO>(acc);
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
            return with_vec(width, weight_stride, weight, sizeof(TW), out, sizeof(TO), [&](auto vec) {
                constexpr int VEC = decltype(vec)::value;
                const int tpr = threads_per_row(width, VEC);
                gather_kernel<TW, TO, VEC><<<(unsigned)ceil_div(n, kThreads / tpr), kThreads, 0, (cudaStream_t)stream>>>(
                    static_cast<const TW*>(weight), rows, width, weight_stride, tokens, (int)token_bytes, n, row0,
                    (float)scale, static_cast<TO*>(out), tpr);
                CRESSO_LAUNCHED("gather_kernel");
                return (int)CRESSO_OK;
            });
        });
    });
}

// scratch: row_start [rows + 1], order [n], partial rows [2 ceil(n / kTile)][align_up(width, 4)]
static int64_t grad_partials(int64_t n) { return n > kTile ? 2 * ceil_div(n, kTile) : 0; }
int cresso_embedding_grad_scratch_bytes(int64_t n, int64_t rows, int64_t width, int64_t* bytes) {
    CRESSO_REQUIRE(bytes != nullptr, CRESSO_EINVAL, "embedding_grad_scratch_bytes: NULL result");
    CRESSO_REQUIRE(n >= 0 && rows >= 0 && width >= 0, CRESSO_EINVAL, "embedding_grad: negative size");
    CRESSO_REQUIRE(n <= CRESSO_TRAIN_MAX_ROWS && rows <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED,
                   "embedding_grad: more than 2^31 - 256 tokens or rows");
    *bytes = align_up(4 * (rows + 1), 256) + align_up(8 * n, 256) + grad_partials(n) * align_up(width, 4) * 4;
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
    CRESSO_REQUIRE(width <= CRESSO_TRAIN_MAX_EMBEDDING_WIDTH, CRESSO_EUNSUPPORTED, "embedding_grad: width above %d",
                   (int)CRESSO_TRAIN_MAX_EMBEDDING_WIDTH);
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
    CRESSO_REQUIRE(aligned_to(scratch, 16), CRESSO_EINVAL, "embedding_grad: scratch is not 16-byte aligned");
    NvtxRange range("embedding_grad n=%lld rows=%lld", (long long)n, (long long)rows);
    int* row_start = static_cast<int*>(scratch);
    unsigned char* after = static_cast<unsigned char*>(scratch) + align_up(4 * (rows + 1), 256);
    int2* order = reinterpret_cast<int2*>(after);
    const TokenWindow win{tokens, has_padding != 0, n, rows, row0, padding};
    const int rb = (int)std::min<int64_t>(kSortMaxRows, std::max<int64_t>(1, ceil_div(rows, 148)));
    const int smem = kSortWarps * rb * 4;
    auto sort = [&](auto kernel) {
        if (smem > 48 * 1024)
            CRESSO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kSortWarps * kSortMaxRows * 4));
        kernel<<<(unsigned)ceil_div(rows, rb), kSortThreads, smem, s>>>(win, rb, row_start, order);
        CRESSO_LAUNCHED("sort_kernel");
        return (int)CRESSO_OK;
    };
    const int rs = token_bytes == 8 ? sort(sort_kernel<int64_t>) : sort(sort_kernel<int32_t>);
    if (rs != CRESSO_OK) return rs;
    GradSums k{row_start, order, reinterpret_cast<float*>(after + align_up(8 * n, 256)), rows, width, grad_stride,
               ceil_div(n, kTile), align_up(width, 4), (float)scale, accumulate != 0, 0};
    const int64_t items = k.tiles + (accumulate ? 0 : ceil_div(rows, kEmptyRows));
    return with_dtype(grad_dtype, [&](auto tg) {
        return with_dtype(out_dtype, [&](auto to) {
            using TG = decltype(tg);
            using TO = decltype(to);
            const int rc = with_vec(width, grad_stride, grad, sizeof(TG), out, sizeof(TO), [&](auto vec) {
                constexpr int VEC = decltype(vec)::value;
                k.tpr = threads_per_row(width, kSumCols);
                const dim3 grid((unsigned)ceil_div(items, kThreads / k.tpr),
                                (unsigned)ceil_div(width, k.tpr * kSumCols));
                grad_kernel<TG, TO, VEC><<<grid, kThreads, 0, s>>>(
                    k, static_cast<const TG*>(grad), static_cast<TO*>(out));
                CRESSO_LAUNCHED("grad_kernel");
                return (int)CRESSO_OK;
            });
            if (rc != CRESSO_OK || grad_partials(n) == 0) return rc;
            const dim3 grid((unsigned)k.tiles, (unsigned)std::min<int64_t>(64, ceil_div(width, kThreads)));
            grad_join_kernel<TO><<<grid, kThreads, 0, s>>>(k, static_cast<TO*>(out));
            CRESSO_LAUNCHED("grad_join_kernel");
            return (int)CRESSO_OK;
        });
    });
}

}  // extern "C"

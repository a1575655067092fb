// Scaled embedding lookup and its gradient by sorted tokens.
//
// Lookup: out[t] = scale * W[token_t - row0].  Gradient: dW[r] = scale * sum of
// g[t] over the positions t whose token is row r.  The positions are brought into
// row order by a stable counting sort (positions ascending inside a row), so every
// row is summed in float32 in a fixed order, that of its tokens or, for long rows, of
// tiles of them: no atomics on values, the same bits every run, one rounding at the end.
#include "train_common.cuh"

#include <algorithm>
#include <type_traits>

namespace cresso {

// A row of `width` columns is taken by `tpr` threads, a power of two up to the block.
static int threads_per_row(int64_t width, int vec) {
    return (int)std::min<int64_t>(kThreads, pow2_ceil(ceil_div(width, vec)));
}

// f(std::integral_constant<int, VEC>) for the widest of 8, 4, 2 and 1 columns an access that
// the sizes and the addresses allow.
template <typename F>
int with_vec(int64_t width, int64_t stride, const void* p, int64_t p_bytes, const void* q, int64_t q_bytes, F f) {
    auto fits = [&](int vec) {
        return width % vec == 0 && stride % vec == 0 && aligned_to(p, std::min<int64_t>(32, vec * p_bytes)) &&
               aligned_to(q, std::min<int64_t>(32, vec * q_bytes));
    };
    if (fits(8)) return f(std::integral_constant<int, 8>());
    if (fits(4)) return f(std::integral_constant<int, 4>());
    if (fits(2)) return f(std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 1>());
}

// token - row0 in 64 bits is the row for every token if the window's last row has a 64-bit number; the
// difference would wrap into a longer window from the other end.
static bool window_ok(int64_t row0, int64_t rows) { return rows == 0 || row0 <= INT64_MAX - (rows - 1); }

// ------------------------------------------------------------------ lookup ---
//
// Bound by memory: the distinct rows are read, every row is written.  16384 of 32000 x 4096
// float32 rows to bfloat16 take 41.5 us, 229 MB at 5.5 TB/s; 32 columns a thread in flight by 128
// threads a row were the best of 16 to 32 columns and 64 to 256 threads (41.5 to 53 us).

template <typename TW, typename TO, int VEC>
__global__ void __launch_bounds__(kThreads, 5) gather_kernel(const TW* __restrict__ w, int64_t rows, int64_t width,
                                                          int64_t stride, const void* __restrict__ tokens,
                                                          int token_bytes, int64_t n, int64_t row0, float scale,
                                                          TO* __restrict__ out, int tpr) {
    constexpr int U = VEC == 1 ? 8 : 32 / VEC;  // accesses of a thread in flight
    const int64_t t = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    if (t >= n) return;
    const uint64_t r = (uint64_t)load_id(tokens, token_bytes, t) - (uint64_t)row0;
    const int64_t first = (int64_t)(threadIdx.x & (tpr - 1)) * VEC;
    const int step = tpr * VEC;
    TO* dst = out + t * width + first;
    if (r >= (uint64_t)rows) {
        const float zero[VEC] = {};
        for (int64_t c = first; c < width; c += step, dst += step) store_global<TO, VEC>(dst, zero);
        return;
    }
    const TW* src = w + (int64_t)r * stride + first;
    for (int64_t left = width - first; left > 0; left -= U * step, src += U * step, dst += U * step) {
        Raw<TW, VEC> f[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u * step < left) f[u].load_global(src + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u * step >= left) break;
            float v[VEC];
            f[u].to(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] *= scale;
            store_global<TO, VEC>(dst + u * step, v);
        }
    }
}

// ---------------------------------------------------------------- the sort ---
//
// One launch without any exchange between blocks: of `blocks` (a power of two) blocks,
// block b owns the rows r = b modulo blocks, so that frequent rows, which often have
// neighbouring numbers, fall to different blocks.  The order holds the rows block by
// block.  Every block reads all tokens (they sit in L2); its warps take equal contiguous
// ranges of positions.  First scan: each warp counts its tokens per owned row in shared
// memory, and the tokens of the blocks before, whose number is where the block's part of
// the order begins.  A scan over (row, warp) turns the counts into first places; the second
// scan puts each position at its place, lanes of one row ranked by a warp match, which
// keeps the positions of a row ascending.
// Bound by instructions and by the latency of a few dependent steps: 4 us for up to 2048 tokens,
// 12 us for 16384 tokens of 32000 rows; 16 warps, other batches or 256 blocks were 1 to 9 us
// slower.  Rows dealt out in ranges instead of in turn cost 7 us more where half of the tokens
// are frequent words.
constexpr int kSortMaxWarps = 32;
constexpr int kSortBatch = 8;         // tokens of a thread in flight
constexpr int kSortCounters = 49152;  // of a block, row ends among them: 192 KB of shared memory
constexpr int kSortLogBlocks = 7;     // at least 128 blocks

struct TokenWindow {
    const void* tokens;
    int64_t n, row0;
    uint32_t rows, padding_row;  // padding_row: 2^32 - 1 where no token is left out
    int log_blocks;
};

constexpr uint32_t kNoRow = 0xffffffffu;
constexpr uint32_t kLastOfRow = 0x80000000u;  // mark of a row's last position in the order

// Rows in the window of the positions i, i + 32, ... below end; kNoRow where there is no
// position or the token takes no part.  All loads are issued before the first is used.
template <typename ID>
__device__ __forceinline__ void window_rows(const TokenWindow& w, int i, int end, uint32_t (&row)[kSortBatch]) {
    ID id[kSortBatch];
    const ID* tokens = static_cast<const ID*>(w.tokens);
    const bool whole = i + 32 * (kSortBatch - 1) < end;
    if (whole) {
#pragma unroll
        for (int b = 0; b < kSortBatch; ++b) id[b] = tokens[(int64_t)i + 32 * b];
    } else {
#pragma unroll
        for (int b = 0; b < kSortBatch; ++b) id[b] = tokens[(int64_t)i + 32 * b < end ? (int64_t)i + 32 * b : end - 1];
    }
#pragma unroll
    for (int b = 0; b < kSortBatch; ++b) {
        const uint64_t d = (uint64_t)(int64_t)id[b] - (uint64_t)w.row0;
        const uint32_t r = (uint32_t)d;
        const bool part = (uint32_t)(d >> 32) == 0 && r < w.rows && r != w.padding_row;
        row[b] = part && (whole || (int64_t)i + 32 * b < end) ? r : kNoRow;
    }
}

template <typename ID>
__global__ void __launch_bounds__(kSortMaxWarps * 32) sort_kernel(TokenWindow win, int nr_max, int2* __restrict__ range,
                                                                  int2* __restrict__ order, int* __restrict__ total) {
    next_kernel_may_start();
    extern __shared__ int cnt[];  // [warps][nr_max], then the end of each row [nr_max]
    __shared__ int warp_tot[kSortMaxWarps], base_sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x, warps = threads >> 5;
    const int log_b = win.log_blocks, blocks = 1 << log_b, b0 = blockIdx.x;
    const int nr = (int)((win.rows + (uint32_t)(blocks - 1 - b0)) >> log_b);
    for (int i = threadIdx.x; i < warps * nr_max; i += threads) cnt[i] = 0;
    if (threadIdx.x == 0) base_sh = 0;
    __syncthreads();
    const int64_t seg = ceil_div(ceil_div(win.n, warps), 32) * 32;
    const int i0 = (int)min(win.n, warp * seg), i1 = (int)min(win.n, (warp + 1) * seg);
    int *mine = cnt + warp * nr_max, *row_end = cnt + warps * nr_max;
    auto owner = [&](uint32_t row) { return row == kNoRow ? blocks : (int)(row & (uint32_t)(blocks - 1)); };
    int below = 0;
    auto count = [&](const uint32_t(&row)[kSortBatch]) {
#pragma unroll
        for (int b = 0; b < kSortBatch; ++b) {
            const int o = owner(row[b]);
            if (o == b0) atomicAdd(&mine[row[b] >> log_b], 1);
            below += o < b0 ? 1 : 0;
        }
    };
    // the rows of two batches stay in registers for the second scan, which is all of a warp's
    // range up to 16384 tokens
    constexpr int kStep = 32 * kSortBatch;
    uint32_t held[2][kSortBatch];
    if (i0 < i1) window_rows<ID>(win, i0 + lane, i1, held[0]);
    if (i0 + kStep < i1) window_rows<ID>(win, i0 + kStep + lane, i1, held[1]);
    if (i0 < i1) count(held[0]);
    if (i0 + kStep < i1) count(held[1]);
    for (int64_t i = (int64_t)i0 + 2 * kStep; i < i1; i += kStep) {
        uint32_t row[kSortBatch];
        window_rows<ID>(win, (int)i + lane, i1, row);
        count(row);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
    if (lane == 0 && below) atomicAdd(&base_sh, below);
    __syncthreads();
    // exclusive scan over the rows of the block, a row a thread and `threads` rows a turn
    int carry = base_sh;
    for (int c = 0; c < nr; c += threads) {
        const int r = c + threadIdx.x;
        int tot = 0;
        if (r < nr)
#pragma unroll 8
            for (int w = 0; w < warps; ++w) tot += cnt[w * nr_max + r];
        int incl = tot;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_tot[warp] = incl;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < warps; ++w) {
            const int v = warp_tot[w];
            before += w < warp ? v : 0;
            all += v;
        }
        int at = carry + before + incl - tot;
        if (r < nr) {
            range[((int64_t)r << log_b) + b0] = make_int2(at, at + tot);
            row_end[r] = at + tot;
            if (tot > 0)
#pragma unroll 8
                for (int w = 0; w < warps; ++w) {
                    const int v = cnt[w * nr_max + r];
                    cnt[w * nr_max + r] = at;
                    at += v;
                }
        }
        carry += all;
        __syncthreads();
    }
    if (b0 == blocks - 1 && threadIdx.x == 0) *total = carry;
    auto place = [&](const uint32_t(&row)[kSortBatch], int i) {
#pragma unroll
        for (int b = 0; b < kSortBatch; ++b) {
            const bool in = owner(row[b]) == b0;
            const unsigned any = __ballot_sync(0xffffffffu, in);
            if (any == 0) continue;
            if (in) {
                const int r = (int)(row[b] >> log_b);
                const unsigned same = __match_any_sync(any, r);
                const int rank = __popc(same & ((1u << lane) - 1u));
                const int at = mine[r];
                const uint32_t last = at + rank + 1 == row_end[r] ? kLastOfRow : 0;
                order[at + rank] = make_int2(i + lane + 32 * b, (int)(row[b] | last));
                __syncwarp(any);
                if (rank == 0) mine[r] = at + __popc(same);
            }
            __syncwarp();
        }
    };
    if (i0 < i1) place(held[0], i0);
    if (i0 + kStep < i1) place(held[1], i0 + kStep);
    for (int64_t i = (int64_t)i0 + 2 * kStep; i < i1; i += kStep) {
        uint32_t row[kSortBatch];
        window_rows<ID>(win, (int)i + lane, i1, row);
        place(row, (int)i);
    }
}

// ----------------------------------------------------------------- the sums ---
//
// The order is cut into tiles of `tile` positions, one work item each, so that the work is
// even however the tokens fall.  A tile fetches its positions ahead whatever rows they
// belong to, and writes a row's sum where the row ends.  A row of up to `tile`
// positions belongs to the tile it begins in.  A longer one is summed tile by tile into
// partial rows, which a second kernel adds in a fixed order; a tile meets at most two such
// rows, one that reaches it from the left (partial 2 tile) and one that begins inside and
// leaves it to the right (partial 2 tile + 1).  Further items write the rows without a
// token, kEmptyRows rows each.
// Bound by memory: 16384 bfloat16 rows of 4096 into (32000, 4096) float32 take 116 us, of which the
// empty rows are 70 us (a plain fill of the whole gradient takes 72) and the tiles 46 us (230 MB at
// 5 TB/s); entries of the order read when they were needed cost 3 us.  Single columns cost
// instructions: 16384 bfloat16 rows of 2051 into 50000 take 160 us with the sort, of 2048 62 us.  One
// row an item took 1264 us (a frequent row is one long chain), rows in order with their own tiles 188 us.  Rows in flight in registers spilled (163 us); in shared memory, fetched
// by the thread that adds them, they need neither registers nor a barrier.
constexpr int kEmptyRows = 8;
constexpr int kSumCols = 8;    // columns of a thread
constexpr int kJoinCols = 128;

// out row = scale * acc (+ out row)
template <typename TO, int VEC, int U>
__device__ __forceinline__ void write_row(TO* __restrict__ out, int64_t c0, int left, int tpr, float scale, int accumulate,
                                          float (&acc)[U][VEC]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = u * tpr * VEC;
        if (c >= left) continue;
        float old[VEC] = {};
        if (accumulate) load_vec<TO, VEC>(out + c0 + c, old);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[u][i] = acc[u][i] * scale + old[i];
        store_global<TO, VEC>(out + c0 + c, acc[u]);
    }
}

// p[0, n) = 0 by `threads` threads, of which this is number t: 16 bytes a store but for the ends
template <typename T>
__device__ __forceinline__ void clear_span(T* p, int n, int t, int threads) {
    constexpr int kPiece = 16 / (int)sizeof(T);
    const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T)));
    const int pieces = (n - head) / kPiece;
    for (int i = t; i < head; i += threads) p[i] = T(0.0f);
    for (int i = t; i < pieces; i += threads) reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0, 0, 0, 0);
    for (int i = head + pieces * kPiece + t; i < n; i += threads) p[i] = T(0.0f);
}

// Begins to copy the first `bytes` (2 or 4) of an aligned word to shared memory.
__device__ __forceinline__ void copy_word(void* dst, const char* word, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(word),
                 "r"(bytes)
                 : "memory");
}

struct GradSums {
    const int2* range;  // (begin, end) of each row in the order
    const int2* order;  // (position, row | kLastOfRow)
    const int* total;   // length of the order
    float* partial;     // [2 tiles][pitch]
    int64_t rows, width, stride, tiles, pitch;
    float scale;
    int accumulate, tpr, tile;
};

__device__ __forceinline__ int order_row(int2 entry) { return entry.y & (int)~kLastOfRow; }

template <typename TG, typename TO, int VEC>
__global__ void __launch_bounds__(kThreads, 5) grad_kernel(GradSums k, const TG* __restrict__ g,
                                                           TO* __restrict__ out) {
    constexpr int U = kSumCols / VEC;
    // single 16-bit columns come as the aligned words that hold them, which cp.async can copy
    constexpr bool kWords = VEC * sizeof(TG) == 2;
    constexpr int kDepth = kWords ? 4 : 16 / sizeof(TG);  // positions in 32 KB of shared memory
    __shared__ __align__(16) TG ring[kDepth * kThreads * kSumCols * (kWords ? 2 : 1)];
    const int tpr = k.tpr;
    const int64_t item = (int64_t)blockIdx.x * (kThreads / tpr) + threadIdx.x / tpr;
    const int64_t c0 = (int64_t)blockIdx.y * tpr * kSumCols + (int64_t)(threadIdx.x & (tpr - 1)) * VEC;
    const int left = (int)min(k.width - c0, (int64_t)tpr * kSumCols);  // columns from the thread's first one on
    float acc[U][VEC] = {};
    next_kernel_may_start();
    previous_kernel_done();
    if (item >= k.tiles) {
        if (k.accumulate) return;  // a block's last groups
        const int64_t r0 = (item - k.tiles) * kEmptyRows;
        bool empty[kEmptyRows];
#pragma unroll
        for (int i = 0; i < kEmptyRows; ++i) {
            const int2 at = k.range[min(r0 + i, k.rows - 1)];
            empty[i] = r0 + i < k.rows && at.x == at.y;
        }
#pragma unroll
        for (int i = 0; i < kEmptyRows; ++i)
            if (empty[i]) {
                if constexpr (VEC == kSumCols) {
                    write_row<TO, VEC, U>(out + (r0 + i) * k.width, c0, left, tpr, 1.0f, 0, acc);
                } else {
                    const int64_t c = (int64_t)blockIdx.y * tpr * kSumCols;
                    clear_span(out + (r0 + i) * k.width + c, (int)min(k.width - c, (int64_t)tpr * kSumCols),
                               threadIdx.x & (tpr - 1), tpr);
                }
            }
        return;
    }
    const int total = *k.total;
    const int a = (int)item * k.tile, b = min(a + k.tile, total);
    if (a >= total) return;
    const int first = order_row(k.order[a]), last = order_row(k.order[b - 1]);
    const int2 fr = k.range[first], lr = k.range[last];
    const bool first_long = fr.y - fr.x > k.tile, last_long = lr.y - lr.x > k.tile;
    // [from, to): the positions this item adds
    const int from = first_long || fr.x == a ? a : min(fr.y, b);
    const int to = last_long ? b : lr.x >= a ? lr.y : from;
    if (from >= to) return;
    // each thread fetches its columns of the next kDepth - 1 positions ahead
    constexpr int kNext = kThreads * (kWords ? 2 : VEC);
    TG* mine = ring + threadIdx.x * (kWords ? 2 : VEC);
    auto fetch = [&](int position, int slot) {
        const TG* src = g + (int64_t)position * k.stride + c0;
        TG* dst = mine + slot * U * kNext;
        if constexpr (kWords) {  // tpr is even: the same half of each word
            const bool upper = (reinterpret_cast<uintptr_t>(src) & 2) != 0;
            const char* word = reinterpret_cast<const char*>(src) - (upper ? 2 : 0);
            if (upper && position == 0 && c0 == 0) {  // the gradient starts inside the word
                dst[1] = src[0];
            } else if (left > 0) {
                copy_word(dst, word, upper || left > 1 ? 4 : 2);
            }
#pragma unroll
            for (int u = 1; u < U; ++u)
                if (u * tpr < left) copy_word(dst + u * kNext, word + 2 * u * tpr, upper || u * tpr + 1 < left ? 4 : 2);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u * tpr * VEC < left) copy_vec<TG, VEC>(dst + u * kNext, src + u * tpr * VEC);
        }
    };
    int early[kDepth - 1];
#pragma unroll
    for (int p = 0; p < kDepth - 1; ++p) early[p] = k.order[min(from + p, to - 1)].x;
#pragma unroll
    for (int p = 0; p < kDepth - 1; ++p) {
        if (from + p < to) fetch(early[p], p);
        copy_commit();
    }
    // entries of the order are read an iteration before they are used
    int2 entry = k.order[from];
    int next = k.order[min(from + kDepth - 1, to - 1)].x;
    int slot = 0;
    for (int j = from; j < to; ++j) {
        const int mark = entry.y;
        // the half of a word that the thread's columns are in
        const int half = kWords ? (int)(reinterpret_cast<uintptr_t>(g + (int64_t)entry.x * k.stride + c0) >> 1 & 1) : 0;
        copy_wait<kDepth - 2>();
        // columns behind the row as well, whose sums are not written
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[VEC];
            load_vec<TG, VEC>(mine + (slot * U + u) * kNext + half, f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[u][i] += f[i];
        }
        if (j + kDepth - 1 < to) fetch(next, slot == 0 ? kDepth - 1 : slot - 1);
        copy_commit();
        next = k.order[min(j + kDepth, to - 1)].x;
        entry = k.order[min(j + 1, to - 1)];
        slot = slot == kDepth - 1 ? 0 : slot + 1;
        if (mark >= 0 && j + 1 < to) continue;
        // the row ends here, or the item does: a long row leaves a partial row
        const int row = mark & (int)~kLastOfRow;
        if ((row == first && first_long) || (row == last && last_long))
            write_row<float, VEC, U>(k.partial + (2 * item + ((row == first ? fr.x : lr.x) > a ? 1 : 0)) * k.pitch,
                                     c0, left, tpr, 1.0f, 0, acc);
        else
            write_row<TO, VEC, U>(out + (int64_t)row * k.width, c0, left, tpr, k.scale, k.accumulate, acc);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[u][i] = 0.0f;
    }
}

// Adds the partial rows of the long rows that begin in the tiles [256 x, 256 x + 256): a
// thread looks at a tile each, then the block takes every gridDim.z-th of the rows found, 128
// columns of it, and its eight warps add every eighth partial row.  4 to 5 us, mostly the three
// dependent loads that find the rows.
template <typename TO>
__global__ void __launch_bounds__(kThreads) grad_join_kernel(GradSums k, TO* __restrict__ out) {
    __shared__ int found[kThreads], warp_count[kWarps];
    __shared__ __align__(16) float part[kWarps][kJoinCols];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t tile = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    previous_kernel_done();
    const int total = *k.total;
    int row = -1;
    if (tile < k.tiles && tile * k.tile < total) {
        const int a = (int)tile * k.tile;
        const int r = order_row(k.order[min(a + k.tile, total) - 1]);
        const int2 at = k.range[r];
        if (at.x >= a && at.y - at.x > k.tile) row = r;
    }
    const unsigned here = __ballot_sync(0xffffffffu, row >= 0);
    if (lane == 0) warp_count[warp] = __popc(here);
    __syncthreads();
    int before = 0, count = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        before += w < warp ? warp_count[w] : 0;
        count += warp_count[w];
    }
    if (row >= 0) found[before + __popc(here & ((1u << lane) - 1u))] = row;
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.y * kJoinCols + 4 * lane, own = (int64_t)blockIdx.y * kJoinCols + threadIdx.x;
    for (int i = blockIdx.z; i < count; i += gridDim.z) {
        const int64_t r = found[i];
        const int2 at = k.range[r];
        const int64_t t0 = at.x / k.tile, t1 = (at.y - 1) / k.tile;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c < k.width) {
#pragma unroll 4
            for (int64_t t = t0 + warp; t <= t1; t += kWarps) {
                const float4 v = *reinterpret_cast<const float4*>(
                    k.partial + (2 * t + (t == t0 && at.x > t0 * k.tile ? 1 : 0)) * k.pitch + c);
                acc.x += v.x;
                acc.y += v.y;
                acc.z += v.z;
                acc.w += v.w;
            }
        }
        *reinterpret_cast<float4*>(&part[warp][4 * lane]) = acc;
        __syncthreads();
        if (threadIdx.x < kJoinCols && own < k.width) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += part[w][threadIdx.x];
            v *= k.scale;
            if (k.accumulate) v += to_float(out[r * k.width + own]);
            out[r * k.width + own] = from_float<TO>(v);
        }
        __syncthreads();
    }
}

// Positions of a tile: 8 where few elements leave SMs idle, so that more latencies overlap (2047
// tokens of 1024: 11 us with 8, 20 us with 32; 16384 of 512: 31 us and 47 us), 32 where there are
// many, since a tile costs partial rows (16384 of 4096: 126 us with 32, 133 us with 8).  Few tiles
// at last, for a frequent row's partial rows are one chain (2000000 tokens of 64: 1015 us with 128,
// 1013 us with 32, 1143 us with 8).
static int grad_tile(int64_t n, int64_t width) {
    return n <= 4096 || (n <= 131072 && n * width <= ((int64_t)1 << 24)) ? 8 : n <= 1048576 ? 32 : 128;
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
    CRESSO_REQUIRE(window_ok(row0, rows), CRESSO_EINVAL, "embedding_gather: the last row's number exceeds 64 bits");
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
                const int tpr = std::min(kThreads / 2, threads_per_row(width, VEC));
                gather_kernel<TW, TO, VEC><<<(unsigned)ceil_div(n, kThreads / tpr), kThreads, 0, (cudaStream_t)stream>>>(
                    static_cast<const TW*>(weight), rows, width, weight_stride, tokens, (int)token_bytes, n, row0,
                    (float)scale, static_cast<TO*>(out), tpr);
                CRESSO_LAUNCHED("gather_kernel");
                return (int)CRESSO_OK;
            });
        });
    });
}

// scratch: range [rows], order [n], total, partial rows [2 tiles][align_up(width, 8)]
struct GradScratch {
    int64_t tile, tiles, order, total, partial, bytes;
};
static GradScratch grad_scratch(int64_t n, int64_t rows, int64_t width) {
    GradScratch p{};
    p.tile = grad_tile(n, width);
    p.tiles = ceil_div(n, p.tile);
    p.order = align_up(8 * rows, 256);
    p.total = p.order + align_up(8 * n, 256);
    p.partial = p.total + 256;
    p.bytes = p.partial + (p.tiles > 1 ? 2 * p.tiles * align_up(width, 8) * 4 : 0);
    return p;
}

int cresso_embedding_grad_scratch_bytes(int64_t n, int64_t rows, int64_t width, int64_t* bytes) {
    CRESSO_REQUIRE(bytes != nullptr, CRESSO_EINVAL, "embedding_grad_scratch_bytes: NULL result");
    CRESSO_REQUIRE(n >= 0 && rows >= 0 && width >= 0, CRESSO_EINVAL, "embedding_grad: negative size");
    CRESSO_REQUIRE(n <= CRESSO_TRAIN_MAX_ROWS && rows <= CRESSO_TRAIN_MAX_ROWS, CRESSO_EUNSUPPORTED,
                   "embedding_grad: more than 2^31 - 256 tokens or rows");
    CRESSO_REQUIRE(width <= CRESSO_TRAIN_MAX_EMBEDDING_WIDTH, CRESSO_EUNSUPPORTED, "embedding_grad: width above %d",
                   (int)CRESSO_TRAIN_MAX_EMBEDDING_WIDTH);
    *bytes = grad_scratch(n, rows, width).bytes;
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
    CRESSO_REQUIRE(window_ok(row0, rows), CRESSO_EINVAL, "embedding_grad: the last row's number exceeds 64 bits");
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
    CRESSO_REQUIRE(aligned_to(scratch, 32), CRESSO_EINVAL, "embedding_grad: scratch is not 32-byte aligned");
    NvtxRange range("embedding_grad n=%lld rows=%lld", (long long)n, (long long)rows);
    const GradScratch at = grad_scratch(n, rows, width);
    unsigned char* base = static_cast<unsigned char*>(scratch);
    int2 *ranges = reinterpret_cast<int2*>(base), *order = reinterpret_cast<int2*>(base + at.order);
    int* total = reinterpret_cast<int*>(base + at.total);
    // warps that have a batch of tokens each (eight scan the rows quickly); blocks whose counters fit shared memory
    const int warps = std::max(8, std::min(kSortMaxWarps, pow2_ceil(ceil_div(n, 32 * kSortBatch))));
    int log_blocks = kSortLogBlocks;
    while ((warps + 1) * ceil_div(rows, (int64_t)1 << log_blocks) > kSortCounters) ++log_blocks;
    const int nr_max = (int)ceil_div(rows, (int64_t)1 << log_blocks);
    const uint64_t pad = (uint64_t)padding - (uint64_t)row0;
    const TokenWindow win{tokens, n, row0, (uint32_t)rows, has_padding != 0 && pad < (uint64_t)rows ? (uint32_t)pad : kNoRow,
                          log_blocks};
    const int smem = (warps + 1) * nr_max * 4;
    auto sort = [&](auto kernel) {
        if (smem > 40 * 1024)  // with the static part, 48 KB need no leave
            CRESSO_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortCounters * 4));
        kernel<<<1u << log_blocks, warps * 32, smem, s>>>(win, nr_max, ranges, order, total);
        CRESSO_LAUNCHED("sort_kernel");
        return (int)CRESSO_OK;
    };
    const int rs = token_bytes == 8 ? sort(sort_kernel<int64_t>) : sort(sort_kernel<int32_t>);
    if (rs != CRESSO_OK) return rs;
    GradSums k{ranges, order, total, reinterpret_cast<float*>(base + at.partial), rows, width, grad_stride, at.tiles,
               align_up(width, 8), (float)scale, accumulate != 0, 0, (int)at.tile};
    const int64_t items = k.tiles + (accumulate ? 0 : ceil_div(rows, kEmptyRows));
    return with_dtype(grad_dtype, [&](auto tg) {
        return with_dtype(out_dtype, [&](auto to) {
            using TG = decltype(tg);
            using TO = decltype(to);
            const int rc = with_vec(width, grad_stride, grad, sizeof(TG), out, sizeof(TO), [&](auto vec) {
                constexpr int VEC = decltype(vec)::value;
                k.tpr = std::max(2, threads_per_row(width, kSumCols));
                const dim3 grid((unsigned)ceil_div(items, kThreads / k.tpr),
                                (unsigned)ceil_div(width, k.tpr * kSumCols));
                CRESSO_CUDA(launch_overlapped(grad_kernel<TG, TO, VEC>, grid, kThreads, 0, s, k,
                                              static_cast<const TG*>(grad), static_cast<TO*>(out)));
                CRESSO_LAUNCHED("grad_kernel");
                return (int)CRESSO_OK;
            });
            if (rc != CRESSO_OK || k.tiles == 1) return rc;  // one tile holds no long row
            const int64_t parts = ceil_div(width, kJoinCols);
            const dim3 grid((unsigned)ceil_div(k.tiles, kThreads), (unsigned)parts,
                            (unsigned)std::max<int64_t>(1, std::min<int64_t>(32, 512 / parts)));
            CRESSO_CUDA(launch_overlapped(grad_join_kernel<TO>, grid, kThreads, 0, s, k, static_cast<TO*>(out)));
            CRESSO_LAUNCHED("grad_join_kernel");
            return (int)CRESSO_OK;
        });
    });
}

}  // extern "C"

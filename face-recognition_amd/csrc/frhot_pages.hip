// HIP kernels that move, free and squeeze the rows of a gallery (gfx950).
//
// A gallery keeps its rows in tiles of 256 (its pages), inside a tile chunk by chunk of 64 components:
//   component c of row r  ->  half index ((r / 256 * (D/64) + c / 64) * 256 + r % 256) * 64 + c % 64
// so a run of rows is, per chunk, one contiguous run of 128-byte pieces.  All of these kernels are copies: what bounds them
// is HBM (every moved byte is read once and written once), and each lane moves 16 bytes at a time, eight lanes a row's piece.
#include <hip/hip_runtime.h>
#include "frhot_kernels.h"

namespace frhot {

typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));
#define FR_DEV __device__ __forceinline__

namespace {

constexpr int32_t kDead = -1;

// byte offset of chunk j of row r
FR_DEV size_t tiled_at(int64_t r, int j, int nk) {
    return ((((size_t)(r >> 8) * (size_t)nk + (size_t)j) << 8) + (size_t)(r & 255)) * 128;
}
template <bool DENSE>
FR_DEV size_t piece_at(int64_t r, int j, int nk) {
    if constexpr (DENSE) return ((size_t)r * nk + j) * 128;
    return tiled_at(r, j, nk);
}

FR_DEV int ceil_log2(int n) { return n <= 1 ? 0 : 32 - __builtin_clz((unsigned)(n - 1)); }

// NT: past the caches.  Moves of more than kStreamBytes gain 3 % by it (1 M rows of 512: 405 -> 393 us); smaller ones lose what the next
// call would have found in the 256 MiB Infinity Cache (20,011 rows of 4096 squeezed, then read: 99 -> 105 us).
constexpr size_t kStreamBytes = (size_t)512 << 20;
template <bool NT>
FR_DEV uint4v load16(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load((const uint4v*)p);
    return *(const uint4v*)p;
}
template <bool NT>
FR_DEV void store16(void* p, uint4v v) {
    if constexpr (NT) __builtin_nontemporal_store(v, (uint4v*)p);
    else *(uint4v*)p = v;
}

// 1 M rows of 512 in 997 runs: 400 us, 2.05 GB, 5.1 TB/s; three runs of 500 x 4096: 3.3 us, the launch.
// One item (a run of up to 256 rows) and `per` chunks of it per block; the pieces are taken chunk by chunk, rows fastest, a
// power of two of row slots per chunk so that no index needs a division.
template <bool SD, bool DD, bool NT>
FR_DEV void move_item(const PageSide& src, const PageSide& dst, const PageItem& it, int nk, int per) {
    const int j0 = blockIdx.y * per, j1 = min(nk, j0 + per);
    const int lg = ceil_log2(it.n), mask = (1 << lg) - 1;
    const int total = (j1 - j0) << (lg + 3);
    const int part = (threadIdx.x & 7) * 16;
    constexpr int U = 4;
    for (int base = threadIdx.x; base < total; base += 256 * U) {
        uint4v v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int idx = base + 256 * u;
            const int i = (idx >> 3) & mask, j = j0 + (idx >> (lg + 3));
            if (idx < total && i < it.n) v[u] = load16<NT>((const char*)src.rows + piece_at<SD>(it.src + i, j, nk) + part);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int idx = base + 256 * u;
            const int i = (idx >> 3) & mask, j = j0 + (idx >> (lg + 3));
            if (idx < total && i < it.n) store16<NT>((char*)dst.rows + piece_at<DD>(it.dst + i, j, nk) + part, v[u]);
        }
    }
    if (blockIdx.y == 0 && dst.keys && (int)threadIdx.x < it.n)
        dst.keys[it.dst + threadIdx.x] = it.key == kKeepKey ? src.keys[it.src + threadIdx.x] : it.key;
}
template <bool SD, bool DD, bool NT>
__global__ __launch_bounds__(256) void page_move_kernel(PageSide src, PageSide dst, const PageItem* __restrict__ items, int nk, int per) {
    const PageItem it = items[blockIdx.x];
    move_item<SD, DD, NT>(src, dst, it, nk, per);
}
// Short lists travel in the kernel's arguments: one in host memory costs every block a trip over PCIe before its first load.
struct InlineItems { PageItem it[kPageInline]; };
template <bool SD, bool DD>
__global__ __launch_bounds__(256) void page_move_inline_kernel(PageSide src, PageSide dst, InlineItems items, int nk, int per) {
    const PageItem it = items.it[blockIdx.x];
    move_item<SD, DD, false>(src, dst, it, nk, per);
}

// A value for the host, which polls page-locked memory for it.
FR_DEV void tell_host(int32_t* p, int32_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM); }

// One run of up to kFreeTiles tiles per block; few bytes, so bound by the launch (1 M rows' keys in 245 runs: 8.4 us).
FR_DEV void free_tiles(int32_t* __restrict__ gk, const TileRun& run, const int32_t* __restrict__ keys, int nkeys, int32_t* count) {
    __shared__ int red[4];
    int mine = 0;
    for (int t = 0; t < run.n; ++t) {
        const int64_t r = (int64_t)(run.first + t) * 256 + threadIdx.x;
        const int32_t k = gk[r];
        int lo = 0, hi = nkeys;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (keys[mid] < k) lo = mid + 1; else hi = mid;
        }
        const bool hit = lo < nkeys && keys[lo] == k;
        if (hit) gk[r] = kDead;
        mine += __popcll(__ballot(hit));
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mine;
    __syncthreads();
    if (threadIdx.x == 0) tell_host(count, red[0] + red[1] + red[2] + red[3]);
}
__global__ __launch_bounds__(256) void page_free_kernel(int32_t* __restrict__ gk, const TileRun* __restrict__ runs,
                                                        const int32_t* __restrict__ keys, int nkeys, int32_t* __restrict__ counts) {
    const TileRun run = runs[blockIdx.x];
    free_tiles(gk, run, keys, nkeys, counts + blockIdx.x);
}
struct InlineRuns { TileRun run[kFreeInline]; };
__global__ __launch_bounds__(256) void page_free_inline_kernel(int32_t* __restrict__ gk, InlineRuns runs, int32_t key, int32_t* __restrict__ counts) {
    const TileRun run = runs.run[blockIdx.x];
    free_tiles(gk, run, &key, 1, counts + blockIdx.x);
}

// live rows of every tile; a wave takes one tile
__global__ __launch_bounds__(256) void page_count_kernel(const int32_t* __restrict__ gk, int64_t rows, int ntiles, int32_t* __restrict__ counts) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= ntiles) return;
    int c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = (int64_t)t * 256 + i * 64 + lane;
        c += __popcll(__ballot(r < rows && gk[r < rows ? r : 0] >= 0));
    }
    if (lane == 0) counts[t] = c;
}

// counts -> exclusive sums in place (and to host_offsets, if not null), the whole in offsets[n] and *total; one block
__global__ __launch_bounds__(1024) void page_scan_kernel(int32_t* __restrict__ offsets, int n, int32_t* host_offsets, int32_t* total) {
    __shared__ int wsum[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int carry = 0;
    for (int base = 0; base < n; base += 1024) {
        const int i = base + tid;
        const int c = i < n ? offsets[i] : 0;
        int v = c;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int u = __shfl_up(v, s);
            if (lane >= s) v += u;
        }
        if (lane == 63) wsum[wave] = v;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wsum[w] : 0;
            all += wsum[w];
        }
        if (i < n) offsets[i] = carry + before + v - c;
        if (i < n && host_offsets) tell_host(host_offsets + i, carry + before + v - c);
        carry += all;
        __syncthreads();
    }
    if (tid == 0) { offsets[n] = carry; tell_host(total, carry); }
}

// Both at once for up to kSmallTiles tiles (65,536 rows): a launch less.  (The keys of a gallery fill whole tiles.)
constexpr int kSmallTiles = 256;
__global__ __launch_bounds__(1024) void page_count_scan_kernel(const int32_t* __restrict__ gk, int64_t rows, int ntiles, int32_t* __restrict__ offsets,
                                                               int32_t* host_offsets, int32_t* total) {
    __shared__ int cnt[kSmallTiles];
    __shared__ int wsum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int t0 = wave; t0 < ntiles; t0 += 64) {        // four tiles' keys in flight a wave, four consecutive ones a lane
        int4v k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = t0 + 16 * u;
            k[u] = *(const int4v*)(gk + (size_t)(t < ntiles ? t : t0) * 256 + lane * 4);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = t0 + 16 * u;
            const int64_t r = (int64_t)t * 256 + lane * 4;
            int c = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) c += __popcll(__ballot(r + j < rows && k[u][j] >= 0));
            if (lane == 0 && t < ntiles) cnt[t] = c;
        }
    }
    __syncthreads();
    const int c = tid < ntiles ? cnt[tid] : 0;          // (ntiles <= 256: the first four waves)
    int v = c;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int u = __shfl_up(v, s);
        if (lane >= s) v += u;
    }
    if (wave < 4 && lane == 63) wsum[wave] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        before += w < wave ? wsum[w] : 0;
        all += wsum[w];
    }
    if (tid < ntiles) offsets[tid] = before + v - c;
    if (tid < ntiles && host_offsets) tell_host(host_offsets + tid, before + v - c);
    if (tid == 0) { offsets[ntiles] = all; tell_host(total, all); }
}

// 2 M rows of 512, a quarter dead in runs: 586 us, 3.1 GB, 5.3 TB/s; 20,011 of 4096, 30 % dead one by one: 45.6 us, 5.0 TB/s.
// One tile of the source and `per` chunks of it per block: its live rows, in order, go to dst rows offsets[tile] and up.
template <bool NT>
__global__ __launch_bounds__(256) void page_compact_kernel(const char* __restrict__ src, const int32_t* __restrict__ sk, int64_t src_rows, int ntiles,
                                                           char* __restrict__ dst, int32_t* __restrict__ dk, int64_t dst_rows, int nk,
                                                           int per, const int32_t* __restrict__ offsets, int64_t* __restrict__ new_rows) {
    __shared__ unsigned char list[256];
    __shared__ int wcnt[4];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = (int64_t)t * 256 + tid;
    const int live_all = offsets[ntiles];
    if (blockIdx.y == 0 && r >= live_all && r < dst_rows) dk[r] = kDead;        // what the squeezed rows left behind
    if (t >= ntiles) return;
    const int32_t key = r < src_rows ? sk[r] : kDead;
    const unsigned long long b = __ballot(key >= 0);
    if (lane == 0) wcnt[wave] = __popcll(b);
    __syncthreads();
    int rank = __popcll(b & ((1ull << lane) - 1)), live = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        rank += w < wave ? wcnt[w] : 0;
        live += wcnt[w];
    }
    const int64_t first = offsets[t];
    if (key >= 0) list[rank] = (unsigned char)tid;
    if (blockIdx.y == 0) {
        if (key >= 0) dk[first + rank] = key;
        if (new_rows && r < src_rows) new_rows[r] = key >= 0 ? first + rank : -1;
    }
    __syncthreads();
    if (live == 0) return;
    const int j0 = blockIdx.y * per, j1 = min(nk, j0 + per);
    const int lg = ceil_log2(live), mask = (1 << lg) - 1;
    const int total = (j1 - j0) << (lg + 3);
    const int part = (tid & 7) * 16;
    constexpr int U = 4;
    for (int base = tid; base < total; base += 256 * U) {
        uint4v v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int idx = base + 256 * u;
            const int i = (idx >> 3) & mask, j = j0 + (idx >> (lg + 3));
            if (idx < total && i < live) v[u] = load16<NT>(src + tiled_at((int64_t)t * 256 + list[i], j, nk) + part);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int idx = base + 256 * u;
            const int i = (idx >> 3) & mask, j = j0 + (idx >> (lg + 3));
            if (idx < total && i < live) store16<NT>(dst + tiled_at(first + i, j, nk) + part, v[u]);
        }
    }
}

__global__ __launch_bounds__(256) void page_rows_kernel(const char* __restrict__ src, char* __restrict__ out, size_t pieces, int nk) {
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;       // 16 bytes: piece t >> 3 of the output = chunk j of row r
    if (t >= pieces * 8) return;
    const int64_t r = (int64_t)((t >> 3) / (unsigned)nk);
    const int j = (int)((t >> 3) % (unsigned)nk);
    *(uint4v*)(out + t * 16) = *(const uint4v*)(src + tiled_at(r, j, nk) + (t & 7) * 16);
}

__global__ __launch_bounds__(256) void page_kill_kernel(int32_t* __restrict__ gk, int64_t lo, int64_t hi) {
    const int64_t r = lo + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r < hi) gk[r] = kDead;
}

}  // namespace

hipError_t launch_page_move(const PageSide& src, const PageSide& dst, const PageItem* items, int n, int64_t rows, int D, hipStream_t s) {
    if (!src.rows || !dst.rows || !items || n <= 0 || rows <= 0 || D <= 0 || D % 64 || (src.dense && dst.dense)) return hipErrorInvalidValue;
    // one chunk a block while that makes no more than four blocks per CU, up to about 64 KiB a block beyond (256-row items of two
    // chunks a block: 411 us for 1 M rows of 512 against 404)
    const int nk = D / 64;
    int per = 1;
    while (per < nk && rows / n * per < 400 && (int64_t)n * ((nk + per - 1) / per) > 1024) per *= 2;
    const unsigned parts = (unsigned)((nk + per - 1) / per);
    if (n <= kPageInline) {
        InlineItems list;
        for (int i = 0; i < kPageInline; ++i) list.it[i] = items[i < n ? i : 0];
        const dim3 grid((unsigned)n, parts);
        if (src.dense) hipLaunchKernelGGL((page_move_inline_kernel<true, false>), grid, dim3(256), 0, s, src, dst, list, nk, per);
        else if (dst.dense) hipLaunchKernelGGL((page_move_inline_kernel<false, true>), grid, dim3(256), 0, s, src, dst, list, nk, per);
        else hipLaunchKernelGGL((page_move_inline_kernel<false, false>), grid, dim3(256), 0, s, src, dst, list, nk, per);
        return hipGetLastError();
    }
    const bool nt = (size_t)rows * D * 2 >= kStreamBytes;
    const auto kern = src.dense   ? (nt ? page_move_kernel<true, false, true> : page_move_kernel<true, false, false>)
                      : dst.dense ? (nt ? page_move_kernel<false, true, true> : page_move_kernel<false, true, false>)
                                  : (nt ? page_move_kernel<false, false, true> : page_move_kernel<false, false, false>);
    constexpr int kLaunch = 1 << 22;            // (a launch may have fewer than 2^32 threads)
    for (int at = 0; at < n; at += kLaunch) {
        hipLaunchKernelGGL(kern, dim3((unsigned)(n - at < kLaunch ? n - at : kLaunch), parts), dim3(256), 0, s, src, dst, items + at, nk, per);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (n - at <= kLaunch) break;
    }
    return hipSuccess;
}

hipError_t launch_page_free(int32_t* gk, const TileRun* runs, int nruns, const int32_t* keys, int nkeys, int32_t* counts, hipStream_t s) {
    if (!gk || !runs || !keys || !counts || nruns <= 0 || nkeys <= 0) return hipErrorInvalidValue;
    if (nruns <= kFreeInline && nkeys == 1) {
        InlineRuns list;
        for (int i = 0; i < kFreeInline; ++i) list.run[i] = runs[i < nruns ? i : 0];
        hipLaunchKernelGGL(page_free_inline_kernel, dim3((unsigned)nruns), dim3(256), 0, s, gk, list, keys[0], counts);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(page_free_kernel, dim3((unsigned)nruns), dim3(256), 0, s, gk, runs, keys, nkeys, counts);
    return hipGetLastError();
}

hipError_t launch_page_count(const int32_t* gk, int64_t rows, int32_t* offsets, int32_t* host_offsets, int32_t* total, hipStream_t s) {
    if (!gk || !offsets || !total || rows <= 0) return hipErrorInvalidValue;
    const int ntiles = (int)((rows + 255) / 256);
    if (ntiles <= kSmallTiles) {
        hipLaunchKernelGGL(page_count_scan_kernel, dim3(1), dim3(1024), 0, s, gk, rows, ntiles, offsets, host_offsets, total);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(page_count_kernel, dim3((unsigned)((ntiles + 3) / 4)), dim3(256), 0, s, gk, rows, ntiles, offsets);
    hipLaunchKernelGGL(page_scan_kernel, dim3(1), dim3(1024), 0, s, offsets, ntiles, host_offsets, total);
    return hipGetLastError();
}

hipError_t launch_page_compact(const void* src, const int32_t* sk, int64_t src_rows, void* dst, int32_t* dk, int64_t dst_rows, int D,
                               int32_t* offsets, int64_t* new_rows, int32_t* host_offsets, int32_t* total, hipStream_t s) {
    if (!src || !sk || !dst || !dk || !offsets || !total || src_rows <= 0 || D <= 0 || D % 64) return hipErrorInvalidValue;
    const int ntiles = (int)((src_rows + 255) / 256), dtiles = (int)((dst_rows + 255) / 256), nk = D / 64;
    const hipError_t e = launch_page_count(sk, src_rows, offsets, host_offsets, total, s);
    if (e != hipSuccess) return e;
    // One chunk a block, or two or four where that brings all blocks to run at once, eight a CU (20,011 rows of 4096, 70 % of them
    // live: 47.9 us with one chunk a block, 45.6 with four; 2 M rows of 512: 587 with one, 596 with four)
    int per = 1;
    const int64_t tiles = ntiles > dtiles ? ntiles : dtiles;
    if (tiles * ((nk + 3) / 4) <= 2048)
        while (tiles * ((nk + per - 1) / per) > 2048) per *= 2;
    const dim3 grid((unsigned)tiles, (unsigned)((nk + per - 1) / per));
    const auto kern = (size_t)src_rows * D * 2 >= kStreamBytes ? page_compact_kernel<true> : page_compact_kernel<false>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, (const char*)src, sk, src_rows, ntiles, (char*)dst, dk, dst_rows, nk, per,
                       (const int32_t*)offsets, new_rows);
    return hipGetLastError();
}

hipError_t launch_page_rows(const void* tile_start, void* out, int64_t n, int D, hipStream_t s) {
    if (!tile_start || !out || n <= 0 || D <= 0 || D % 64) return hipErrorInvalidValue;
    const size_t pieces = (size_t)n * (D / 64);
    hipLaunchKernelGGL(page_rows_kernel, dim3((unsigned)((pieces * 8 + 255) / 256)), dim3(256), 0, s, (const char*)tile_start, (char*)out,
                       pieces, D / 64);
    return hipGetLastError();
}

hipError_t launch_page_kill(int32_t* gk, int64_t lo, int64_t hi, hipStream_t s) {
    if (!gk || lo < 0) return hipErrorInvalidValue;
    if (hi <= lo) return hipSuccess;
    hipLaunchKernelGGL(page_kill_kernel, dim3((unsigned)((hi - lo + 255) / 256)), dim3(256), 0, s, gk, lo, hi);
    return hipGetLastError();
}

}  // namespace frhot

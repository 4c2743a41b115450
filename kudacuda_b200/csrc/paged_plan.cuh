// paged_plan.cuh -- how the work of a ragged batch of paged attention is
// shared out.
//
// A sequence with n new tokens and G query heads per key head has n * G query
// rows per key head (row R: token R / G, head R % G); ROWS of them are a tile,
// and (sequence, key head, tile) is an item whose keys come in blocks of KT.
// Every item has a cost (its last row's keys, counted per query row, and OVER
// keys for its start and end), the items stand in one line, and worker c of N
// takes the stretch [c U / N, (c + 1) U / N) of the total cost U.  A stretch
// that ends inside an item is rounded down to a block, by the same formula for
// both neighbours, so lengths of any mix load every worker alike and an item
// is cut only where a stretch ends.  A cut item's pieces are left as partial
// results (accumulator, maximum, sum) and joined by a second kernel
// (paged_combine.cuh).
//
// The costs have a closed form per sequence, so a worker finds its place from
// the lengths alone: no host work and no plan kernel, and the lengths may
// change under a captured graph.
#pragma once

#include "kc_common.cuh"
#include "kc_launch.h"

namespace kc {

// One per worker: the item that goes on from an earlier worker's stretch into this
// one's, where it is cut (rows 0: there is none).
struct PagedCut {
    int first, last;      // the workers that may have a piece of it
    int piece;            // 1: this worker left one (in its slot 0; the first worker's is in slot 1)
    int row0;             // first row (token) of the item's sequence in the batch
    int r0, rows;         // first tile row R and the number of rows
    int kvh;
    int pad;
};

// (almost always both fit 32 bits, whose division is several times as fast)
__device__ __forceinline__ int64_t paged_div(int64_t x, int64_t y) {
    if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
    return x / y;
}
// How the line is cut: the first `rest` workers take size + 1, the others size.
struct PagedShares {
    int64_t size, rest;
    int workers;
    // No more workers than there is work for: about `least` keys a worker.
    __device__ __forceinline__ void set(int64_t total, int group, int least, int most) {
        const float w = __fdividef(static_cast<float>(total), static_cast<float>(group) * static_cast<float>(least));
        workers = w < static_cast<float>(most) ? max(static_cast<int>(w), 1) : most;
        size = paged_div(total, workers);
        rest = total - size * workers;
    }
    __device__ __forceinline__ int64_t from(int worker) const {
        return size * worker + (worker < rest ? worker : rest);
    }
    // the worker whose stretch holds x
    __device__ __forceinline__ int of(int64_t x) const {
        const int64_t high = (size + 1) * rest;
        return static_cast<int>(x < high ? paged_div(x, size + 1) : rest + paged_div(x - high, max(size, int64_t{1})));
    }
};

struct PagedSeq {
    int start, n, len;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
    PagedSeq s;
    const int a = p.query_start[b], e = p.query_start[b + 1], l = p.kv_len[b];
    s.start = min(max(a, 0), p.rows);
    s.n = min(max(e, s.start), p.rows) - s.start;
    s.len = max(l, 0);
    return s;
}

template <int ROWS, int KT, int OVER>
struct PagedWalk {
    // the line
    int64_t x0, x1;
    // the sequence at hand
    int b, start, n, len, rows, tiles_q;
    int64_t head_cost, head_at;  // cost of one key head of it; where the current one begins
    int next_kvh, next_q;
    // the piece at hand
    int piece_b, piece_start, piece_n, piece_len;
    int kvh, q, item_rows, limit, least, t0, t1, tiles;  // limit, least: keys of the last row and of the first
    int64_t item_end;

    // cost of the first k tiles of a key head
    __device__ __forceinline__ int64_t cost(int group, int k) const {
        const int64_t base = static_cast<int64_t>(max(len - n, 0) + OVER) * group;
        if (k >= tiles_q)
            return tiles_q * base + static_cast<int64_t>(ROWS / 2) * (tiles_q - 1) * tiles_q + rows;
        return k * base + static_cast<int64_t>(ROWS / 2) * k * (k + 1);
    }
    __device__ __forceinline__ void load(const PagedBatch& p, int group) {
        const PagedSeq s = paged_seq(p, b);
        start = s.start;
        n = s.n;
        len = s.len;
        rows = n * group;
        tiles_q = (rows + ROWS - 1) / ROWS;
        head_cost = tiles_q > 0 ? cost(group, tiles_q) : 0;
    }
    __device__ __forceinline__ void skip_empty(const PagedBatch& p, int group) {
        while (b < p.batch) {
            load(p, group);
            if (tiles_q > 0) return;
            ++b;
        }
    }
    // a worker's stretch, which begins in or after sequence `seq`, whose cost begins at `at`
    __device__ __forceinline__ void begin(const PagedBatch& p, int group, const PagedShares& shares, int worker, int seq,
                                          int64_t at) {
        x0 = shares.from(worker);
        x1 = shares.from(worker + 1);
        b = seq;
        head_at = at;
        next_kvh = next_q = 0;
        tiles_q = 0;
        skip_empty(p, group);
        if (b >= p.batch || x0 <= at) return;
        next_kvh = static_cast<int>(min(paged_div(x0 - at, head_cost), static_cast<int64_t>(p.kv_heads - 1)));
        head_at = at + next_kvh * head_cost;
        int lo = 0, hi = tiles_q - 1;  // the last tile that begins at or before x0
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (head_at + cost(group, mid) <= x0) lo = mid;
            else hi = mid - 1;
        }
        next_q = lo;
    }
    // the item that comes next; its cost begins at the value returned and ends at item_end
    __device__ __forceinline__ int64_t item(const PagedBatch& p, int group) {
        const int64_t lo = head_at + cost(group, next_q);
        item_end = head_at + cost(group, next_q + 1);
        kvh = next_kvh;
        q = next_q;
        item_rows = min(ROWS, rows - q * ROWS);
        const int last_token = q == tiles_q - 1 ? n - 1 : (q * ROWS + ROWS - 1) / group;
        limit = min(max(len - n + last_token + 1, 0), p.table_width * p.page_size);
        least = min(max(len - n + q * ROWS / group + 1, 0), limit);
        tiles = max((limit + KT - 1) / KT, 1);
        return lo;
    }
    // the item's block in which x lies (the same expression on both sides of a cut, so the two agree)
    __device__ __forceinline__ int block_of(int64_t x, int64_t lo) const {
        const float each = __fdividef(static_cast<float>(tiles), static_cast<float>(item_end - lo));
        return x <= lo ? 0 : x >= item_end ? tiles : min(tiles, static_cast<int>(static_cast<float>(x - lo) * each));
    }
    // the next piece with a block in it
    __device__ __forceinline__ bool next(const PagedBatch& p, int group) {
        while (b < p.batch) {
            if (head_at + cost(group, next_q) >= x1) return false;
            const int64_t lo = item(p, group);
            t0 = block_of(x0, lo);
            t1 = block_of(x1, lo);
            piece_b = b;
            piece_start = start;
            piece_n = n;
            piece_len = len;
            if (++next_q == tiles_q) {
                next_q = 0;
                head_at += head_cost;
                if (++next_kvh == p.kv_heads) {
                    next_kvh = 0;
                    ++b;
                    skip_empty(p, group);
                }
            }
            if (t0 < t1) return true;
        }
        return false;
    }
    // after begin(): the item that goes on into this worker's stretch
    __device__ __forceinline__ PagedCut record(const PagedBatch& p, int group, const PagedShares& shares, int worker) {
        PagedCut c;
        c.first = c.last = c.piece = c.row0 = c.r0 = c.rows = c.kvh = c.pad = 0;
        if (b >= p.batch) return c;
        const int64_t lo = item(p, group);
        if (x0 <= lo || x0 >= item_end) return c;
        int first = shares.of(lo);  // (its share may be less than a block)
        while (first < worker && block_of(shares.from(first + 1), lo) == 0) ++first;
        if (first == worker || block_of(shares.from(first + 1), lo) == tiles) return c;  // not cut before here
        c.first = first;
        c.last = shares.of(item_end - 1);
        c.piece = block_of(x0, lo) < block_of(x1, lo) ? 1 : 0;
        c.row0 = start;
        c.r0 = q * ROWS;
        c.rows = item_rows;
        c.kvh = kvh;
        return c;
    }
    // whether some rows of the piece do not attend all of its keys
    __device__ __forceinline__ bool uneven() const { return least < min(limit, t1 * KT); }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == tiles; }
};

// Block-wide: how the work is shared (at most `most` workers, each with LEAST keys
// or more), and for `worker` the sequence in which its stretch begins (seq) and
// that sequence's place (at).  `sums` has one word per warp.  Ends with a barrier.
template <class W, int LEAST, int THREADS>
__device__ __forceinline__ PagedShares paged_place(const PagedBatch& p, int group, int worker, int most,
                                                   int64_t* sums, int* seq, int64_t* at) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b0 = static_cast<int>(static_cast<int64_t>(p.batch) * tid / THREADS);
    const int b1 = static_cast<int>(static_cast<int64_t>(p.batch) * (tid + 1) / THREADS);
    W w;
    int64_t mine = 0;
    for (w.b = b0; w.b < b1; ++w.b) {
        w.load(p, group);
        mine += w.head_cost * p.kv_heads;
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    if (tid == 0) {
        *seq = p.batch;
        *at = 0;
    }
    __syncthreads();
    int64_t total = 0, before = 0;
    for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) before += sums[i];
        total += sums[i];
    }
    int64_t from = before + upto - mine;
    PagedShares shares;
    shares.set(total, group, LEAST, most);
    const int64_t x = shares.from(worker);
    if (worker < shares.workers && mine > 0 && x >= from && x < from + mine) {
        int64_t c = from;
        for (w.b = b0; w.b < b1; ++w.b) {
            w.load(p, group);
            const int64_t e = c + w.head_cost * p.kv_heads;
            if (x < e) break;
            c = e;
        }
        *seq = w.b;
        *at = c;
    }
    __syncthreads();
    return shares;
}

// Where a worker's partial results lie: slot 0 the end of an item begun by an
// earlier worker, slot 1 the beginning of an item that later ones end.  A slot
// is ROWS (maximum, sum) pairs and the accumulator, as its writer finds it best.
template <int ROWS, int D>
struct PagedPartial {
    static constexpr int64_t kFloats = static_cast<int64_t>(ROWS) * (D + 2);
    static __host__ __device__ int64_t bytes(int64_t workers) {
        return (workers * sizeof(PagedCut) + 255) / 256 * 256 + workers * 2 * kFloats * 4;
    }
    static __device__ __forceinline__ PagedCut* cuts(void* ws) { return static_cast<PagedCut*>(ws); }
    static __device__ __forceinline__ float* slot(void* ws, int workers, int worker, int s) {
        char* base = static_cast<char*>(ws) + (static_cast<int64_t>(workers) * sizeof(PagedCut) + 255) / 256 * 256;
        return reinterpret_cast<float*>(base) + (static_cast<int64_t>(worker) * 2 + s) * kFloats;
    }
};

}  // namespace kc

// paged_decode.cu -- paged attention with few query rows a key head (decoding):
// the cache is read once, at the speed of memory.
//
// A block of eight warps is a worker (paged_plan.cuh): it takes a stretch of the
// batch's work, items of 16 query rows (mma.m16n8k16's M; a single token of a
// group of 8 fills half of it, which costs nothing here) against blocks of 16
// keys, which go round the warps.  In the loop a warp needs no other: its own
// ring of K and V blocks in shared memory, fetched by TMA page by page (128-byte
// swizzle), its own barriers, its own running maximum, sum and 16 x head_dim
// accumulator in registers.  So the loop waits for nothing but memory, and
// two to three blocks of every warp are in flight: 128-192 KB on every SM, three
// to four times what covers the latency of 6.5 TB/s.  Only at the end of a piece
// do the warps meet, in shared memory, in a fixed order.
//
// S = Q K^T with exact products and 32-bit sums; softmax in the log2 domain; P
// is split into two 16-bit halves (P = hi + lo to about twice the type's
// precision), so P V is as good as with 32-bit probabilities.  f16 has no small
// numbers to spare for that: its P are 2^15 times as large (kShift), so that the
// largest is just below the type's end and what rounds away is below 2^-40 of it.
// Items of at most 8 rows put lo into the fragment's other 8 rows, whose sum with the first 8 is
// taken at the end: half of the products, and the tensor cores keep time to
// spare while the cache arrives.
// A value that is not finite reaches the rows that attend it alone: where a block has
// keys past some row's own, it is looked through for one first, and if there is one
// the product is taken row by row.
//
// Measured (128 dims): 2 sequences of 70 001 to 130 001 keys, 8 key heads of 4: 130 us,
// 6.0 TB/s of the card's 6.55 (the join of the pieces, 4 us, does not overlap); 64
// of 32 to 2048 keys, 2 key heads of 8: 19.4 us, 30 MB, of which the loop takes 8:
// the rest is the chain before it (lengths, shares, page numbers) and after it
// (meeting, pieces, join) and two launches.  1 of 509 keys: 12.5 us.
#include "kc_common.cuh"
#include "kc_launch.h"
#include "kc_tcgen05.cuh"
#include "kc_tma.h"
#include "paged_combine.cuh"
#include "paged_plan.cuh"

namespace kc {
namespace {

constexpr int kRows = 16;
constexpr int kKeys = 16;
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
// An item's start and end cost about as much as kOver keys, and a worker has kLeast
// or more, a block or so for every warp.  Thirteen batches together 377 us; with
// kLeast 320 or 448 381 and 383, with both 128 380, both 256 381.
constexpr int kOver = 384;
constexpr int kLeast = 192;

// m is the running maximum less this, in the log2 domain; O / l does not depend on it.
// With 0, 131071 f16 keys of weight 2^-25.1 beside one of 1 were lost: 0.4% of O.
template <int DT>
constexpr float kShift = DT == kF16 ? 15.F : 0.F;

template <int D>
struct DecodeSmem {
    static constexpr int kHalves = D / 64;
    static constexpr int kBlock = kHalves * kKeys * 128;  // [D / 64][16][128 B]
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kWarpBytes = kStages * 2 * kBlock;
    static constexpr int kMeet = kWarps / 2 * kRows * D * 4;  // accumulators of half of the warps
    static constexpr int kBytes = 1024 + kWarps * kWarpBytes + kMeet;
};

template <int DT>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (DT == kBF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if constexpr (DT == kBF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// the halves of a word that hold keys `key` and `key` + 1, where these are below `left`
__device__ __forceinline__ uint32_t keep_below(int key, int left) {
    return (key < left ? 0xffffu : 0u) | (key + 1 < left ? 0xffff0000u : 0u);
}
// Whether one of the first `keys` rows of a warp's V block holds an infinity or a NaN.
template <int DT, int D>
__device__ __forceinline__ bool not_finite(uint32_t block, int keys) {
    constexpr uint32_t kTop = DT == kBF16 ? 0x7f80u : 0x7c00u;
    bool found = false;
    for (int i = threadIdx.x & 31; i < D / 64 * kKeys * 8; i += 32) {  // 16-byte words, eight a row of 64 dims
        uint32_t x[4];
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                     : "r"(block + 16 * i));
        if ((i >> 3) % kKeys >= keys) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) found = found || (x[k] & kTop) == kTop || (x[k] >> 16 & kTop) == kTop;
    }
    return __any_sync(0xffffffffu, found);
}

// What the warps need of a piece; thread 0 lists them, kList at a time.
struct Piece {
    int b, start, n, len, kvh, r0, rows, limit, least, t0, t1;
    int whole;
};
constexpr int kList = 12;

// (one block an SM, said aloud, gives the loop 244 registers instead of 175: 64
// sequences of 500 keys, 4 key heads, take 21.8 us instead of 24.0)
template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const PagedAttentionArgs a) {
    using M = DecodeSmem<D>;
    using W = PagedWalk<kRows, kKeys, kOver>;
    using Part = PagedPartial<kRows, D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[kWarps][M::kStages];
    __shared__ float2 row_ml[kWarps][kRows];  // a warp's (maximum, sum) of a row
    __shared__ int64_t sums[kWarps], place_at;
    __shared__ int place_seq, listed;
    __shared__ Piece list[kList];
    const PagedBatch& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* const smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    uint8_t* const ring = smem + warp * M::kWarpBytes;
    float* const meet = reinterpret_cast<float*>(smem + kWarps * M::kWarpBytes);
    if (lane == 0) {
        for (int i = 0; i < M::kStages; ++i) mbar_init(&full[warp][i], 1);
        fence_mbar_init();
    }
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const int group = p.q_heads / p.kv_heads;
    const int worker = blockIdx.x;
    // (an item's rows are few: exact without an integer division)
    const float per_token = __frcp_rn(static_cast<float>(group));
    auto token_of = [&](int row) { return static_cast<int>((static_cast<float>(row) + 0.5F) * per_token); };
    const PagedShares shares =
        paged_place<W, kLeast, kThreads>(p, group, worker, gridDim.x, sums, &place_seq, &place_at);
    W w;  // (thread 0's)
    if (tid == 0) w.begin(p, group, shares, worker, place_seq, place_at);
    if (tid == 32) {
        W v;
        v.begin(p, group, shares, worker, place_seq, place_at);
        Part::cuts(a.workspace)[worker] = v.record(p, group, shares, worker);
    }
    bool ok = true;
    uint32_t fetched = 0, used = 0;
    for (;;) {
        // ---- the next pieces of the stretch
        if (tid == 0) {
            int n = 0;
            while (n < kList && w.next(p, group)) {
                Piece& e = list[n++];
                e.b = w.piece_b;
                e.start = w.piece_start;
                e.n = w.piece_n;
                e.len = w.piece_len;
                e.kvh = w.kvh;
                e.r0 = w.q * kRows;
                e.rows = w.item_rows;
                e.limit = w.limit;
                e.least = w.least;
                e.t0 = w.t0;
                e.t1 = w.t1;
                e.whole = w.whole() ? 1 : 0;
                if (w.piece_len > p.table_width * p.page_size && p.err != nullptr) atomicOr(p.err, 2);
            }
            listed = n;
        }
        __syncthreads();
        const int pieces = listed;
        if (pieces == 0) break;
        // the pieces' blocks are numbered through; this warp has those with number % kWarps == warp
        int ahead = -1, ahead_j = 0, ahead_t1 = 0, turn_ahead = 0;  // the block to be fetched next
        // the next piece with a block of this warp: its queries come into L1 while the blocks before it are worked on
        auto step = [&]() {
            while (++ahead < pieces) {
                const int t0 = list[ahead].t0;
                ahead_t1 = list[ahead].t1;
                ahead_j = t0 + ((warp - turn_ahead) & (kWarps - 1));
                turn_ahead += ahead_t1 - t0;
                if (ahead_j < ahead_t1) break;
            }
            if (ahead >= pieces) return;
            const Piece& e = list[ahead];
            const int r = lane & 15;
            if (r < e.rows) {
                const int token = token_of(e.r0 + r), head = (e.r0 + r) - token * group;
                const uint16_t* q = static_cast<const uint16_t*>(a.q) + (e.start + token) * a.q_stride +
                                    static_cast<int64_t>(e.kvh * group + head) * D + (lane >> 4) * (D / 2);
                asm volatile("prefetch.global.L1 [%0];" ::"l"(q));
            }
        };
        // fetch the next block, K and V, into its stage (which its reader has left)
        auto fetch = [&]() {
            if (ahead < 0 || ahead_j >= ahead_t1) step();
            if (ahead >= pieces) return;
            const Piece& e = list[ahead];
            const int key0 = ahead_j * kKeys;
            const bool some = key0 < e.limit;  // (an item without keys has one block without)
            const uint32_t s = fetched % M::kStages;
            uint8_t* const stage = ring + s * 2 * M::kBlock;
            if (lane == 0) mbar_arrive_expect_tx(&full[warp][s], some ? 2 * M::kBlock : 0);
            __syncwarp();
            if (some && lane < 2 * M::kHalves) {
                const int half = lane >> 1, v = lane & 1;
                const int page = p.table[e.b * p.table_stride + key0 / p.page_size];
                int row = -kKeys;  // a missing page reads as zeros: a box that begins before the tensor
                if (page >= 0 && page < p.num_pages)
                    row = (page * p.kv_heads + e.kvh) * p.page_size + (key0 & (p.page_size - 1));
                else if (p.err != nullptr) atomicOr(p.err, 2);
                tma_load_2d(stage + v * M::kBlock + half * (kKeys * 128), v ? &map_v : &map_k, half * 64, row,
                            &full[warp][s]);
            }
            ++fetched;
            ahead_j += kWarps;
        };

        const float c = a.scale * kLog2E;
        const int g = lane >> 2, t4 = lane & 3;  // an accumulator's rows g and g + 8, columns 2 t4 and 2 t4 + 1
        int turn = 0;
#pragma unroll 1
        for (int piece = 0; piece < pieces; ++piece) {
            const Piece e = list[piece];
            const bool narrow = e.rows <= 8;
            const int first = e.t0 + ((warp - turn) & (kWarps - 1));
            turn += e.t1 - e.t0;
            float o[D / 8][4];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.F;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.F, 0.F};
            // Q: the A fragments of the item's 16 rows, straight from memory
            uint32_t qf[D / 16][4];
            int row_keys[2] = {0, 0};
            if (first < e.t1) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = g + 8 * h, token = token_of(e.r0 + r), head = (e.r0 + r) - token * group;
                    const bool live = r < e.rows;
                    const uint16_t* q = static_cast<const uint16_t*>(a.q) +
                                        (live ? (e.start + token) * a.q_stride +
                                                    static_cast<int64_t>(e.kvh * group + head) * D
                                              : 0);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            qf[k][2 * x + h] = live ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8 * x + 2 * t4) : 0u;
                    row_keys[h] = live ? min(max(e.len - e.n + token + 1, 0), e.limit) : 0;
                }
            }
            // (the first blocks are on their way while the queries come)
            for (; piece == 0 && fetched - used < M::kStages - 1 && ahead < pieces;) fetch();
#pragma unroll 1
            for (int j = first; j < e.t1; j += kWarps) {
                fetch();
                const uint32_t s = used % M::kStages;
                ok = ok && mbar_wait_bounded(&full[warp][s], (used / M::kStages) & 1);
                ++used;
                if (!__all_sync(0xffffffffu, ok)) {  // the piece stays wrong, the error word says so
                    ok = false;
                    continue;
                }
                const uint32_t kb = smem_u32(ring + s * 2 * M::kBlock), vb = kb + M::kBlock;
                // S: 16 rows x 16 keys, two tiles of 8 keys
                float sc[kKeys / 8][4], sc2[kKeys / 8][4];  // even and odd steps of 16 dims: two chains
#pragma unroll
                for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[n][i] = sc2[n][i] = 0.F;
#pragma unroll
                for (int n2 = 0; n2 < kKeys / 16; ++n2) {
                    // ldmatrix: keys 16 n2 .. + 15 (two tiles), 16 dims (two 8-dim words)
                    const int key = 16 * n2 + (lane & 7) + ((lane >> 4) << 3);
                    const uint32_t row = kb + key * 128;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const int word = 2 * (k & 3) + ((lane >> 3) & 1);
                        uint32_t b[4];
                        ldsm4(b, row + (k >> 2) * (kKeys * 128) + ((word ^ (key & 7)) << 4));
                        mma16816<DT>(k & 1 ? sc2[2 * n2] : sc[2 * n2], qf[k], b[0], b[1]);
                        mma16816<DT>(k & 1 ? sc2[2 * n2 + 1] : sc[2 * n2 + 1], qf[k], b[2], b[3]);
                    }
                }
                const int key0 = j * kKeys;
                const int valid = e.limit - key0;  // keys of the block that exist
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + 8 * n + 2 * t4 + (i & 1);
                        const float x = key < row_keys[i >> 1] ? (sc[n][i] + sc2[n][i]) * c : -INFINITY;
                        sc[n][i] = x;
                        top[i >> 1] = fmaxf(top[i >> 1], x);
                    }
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                    const float mn = fmaxf(m[h], top[h] - kShift<DT>);
                    f[h] = mn == -INFINITY ? 1.F : ex2(m[h] - mn);
                    m[h] = mn;
                    l[h] *= f[h];
                }
                if (narrow) f[1] = f[0];
                if (__any_sync(0xffffffffu, f[0] != 1.F || f[1] != 1.F)) {
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        o[i][0] *= f[0];
                        o[i][1] *= f[0];
                        o[i][2] *= f[1];
                        o[i][3] *= f[1];
                    }
                }
                if (narrow) {
                    m[1] = -INFINITY;  // (rows 8 .. 15 hold the low halves of rows 0 .. 7)
                    l[1] = 0.F;
                }
                const float sub[2] = {m[0] == -INFINITY ? 0.F : m[0], m[1] == -INFINITY ? 0.F : m[1]};
                // P in A-fragment order, 16 keys a fragment, as hi + lo
                uint32_t ph[kKeys / 16][4], pl[kKeys / 16][4];  // (narrow: one fragment of both)
#pragma unroll
                for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float e0 = ex2(sc[n][2 * h] - sub[h]), e1 = ex2(sc[n][2 * h + 1] - sub[h]);
                        l[h] += e0 + e1;
                        const uint32_t hi = pack2<DT>(e0, e1);
                        const float2 back = unpack2<DT>(hi);
                        const uint32_t lo = pack2<DT>(e0 - back.x, e1 - back.y);
                        if (!narrow || h == 0) ph[n >> 1][2 * (n & 1) + h] = hi;
                        if (narrow && h == 0) ph[n >> 1][2 * (n & 1) + 1] = lo;
                        pl[n >> 1][2 * (n & 1) + h] = lo;
                    }
                if (e.least < min(key0 + kKeys, e.limit) && not_finite<DT, D>(vb, valid)) {
                    // (rare) a value that only some of the rows may see, and 0 times it is not 0: the product
                    // is taken for each row by itself, with the values past its keys left out
#pragma unroll 1
                    for (int r = 0; r < e.rows; ++r) {
                        const int left = __shfl_sync(0xffffffffu, r < 8 ? row_keys[0] : row_keys[1], 4 * (r & 7)) - key0;
                        if (left <= 0) continue;
                        const bool mine = g == (r & 7);
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
                            const int key = lane & 15, word = 2 * (d & 3) + (lane >> 4);
                            uint32_t b[4];
                            ldsm4t(b, vb + key * 128 + (d >> 2) * (kKeys * 128) + ((word ^ (key & 7)) << 4));
                            const uint32_t keep0 = keep_below(2 * t4, left), keep1 = keep_below(2 * t4 + 8, left);
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                float one[4] = {0.F, 0.F, 0.F, 0.F};
                                mma16816<DT>(one, ph[0], b[2 * x] & keep0, b[2 * x + 1] & keep1);
                                if (!narrow) mma16816<DT>(one, pl[0], b[2 * x] & keep0, b[2 * x + 1] & keep1);
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (mine && (narrow || i >> 1 == r >> 3)) o[2 * d + x][i] += one[i];
                            }
                        }
                    }
                    __syncwarp();
                    continue;
                }
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk) {
                    const int key = 16 * kk + (lane & 15);
                    const uint32_t row = vb + key * 128;
                    // slots without a key may hold anything, a NaN too: their V must not meet P = 0
                    const int left = valid - 16 * kk;
                    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                    if (left < 16) {
                        keep0 = keep_below(2 * t4, left);
                        keep1 = keep_below(2 * t4 + 8, left);
                    }
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        const int word = 2 * (d & 3) + (lane >> 4);
                        uint32_t b[4];
                        ldsm4t(b, row + (d >> 2) * (kKeys * 128) + ((word ^ (key & 7)) << 4));
                        b[0] &= keep0;
                        b[1] &= keep1;
                        b[2] &= keep0;
                        b[3] &= keep1;
                        mma16816<DT>(o[2 * d], ph[kk], b[0], b[1]);
                        mma16816<DT>(o[2 * d + 1], ph[kk], b[2], b[3]);
                        if (!narrow) {
                            mma16816<DT>(o[2 * d], pl[kk], b[0], b[1]);
                            mma16816<DT>(o[2 * d + 1], pl[kk], b[2], b[3]);
                        }
                    }
                }
                // this stage is refilled one block from now: every lane has read it (the
                // next fetch() begins with the warp's barrier) before the copy starts
                __syncwarp();
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                if (t4 == 0) row_ml[warp][g + 8 * h] = make_float2(m[h], l[h]);
            }
            if (narrow) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    o[i][0] += o[i][2];
                    o[i][1] += o[i][3];
                }
            }
            // The warps meet: every one brings its accumulator to the row's maximum, the
            // upper four leave theirs, the lower four add one each and leave the sum, and
            // all threads add those four.  (columns are swizzled by the row)
            __syncthreads();
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = row_ml[0][g + 8 * h].x;
                for (int i = 1; i < kWarps; ++i) mx = fmaxf(mx, row_ml[i][g + 8 * h].x);
                f[h] = m[h] == -INFINITY ? 0.F : ex2(m[h] - mx);
            }
            float* const spot = meet + (warp & 3) * kRows * D;
            auto place = [&](int i, int h) {
                return reinterpret_cast<float2*>(spot + (g + 8 * h) * D + (8 * (i ^ g) + 2 * t4));
            };
            if (warp >= 4) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) *place(i, h) = make_float2(o[i][2 * h] * f[h], o[i][2 * h + 1] * f[h]);
            }
            __syncthreads();
            if (warp < 4) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 x = *place(i, h);
                        *place(i, h) = make_float2(o[i][2 * h] * f[h] + x.x, o[i][2 * h + 1] * f[h] + x.y);
                    }
            }
            __syncthreads();
            float* const part = Part::slot(a.workspace, gridDim.x, worker, e.t0 > 0 ? 0 : 1);
            for (int i = tid; i < e.rows * (D / 4); i += kThreads) {
                const int r = i / (D / 4), d = 4 * (i % (D / 4));
                float mx = -INFINITY, sum = 0.F;
                for (int v = 0; v < kWarps; ++v) mx = fmaxf(mx, row_ml[v][r].x);
                for (int v = 0; v < kWarps; ++v) {
                    const float2 x = row_ml[v][r];
                    sum += x.y * (x.x == -INFINITY ? 0.F : ex2(x.x - mx));
                }
                const float* at = meet + r * D + ((((d >> 3) ^ (r & 7)) << 3) | (d & 7));
                float4 x = *reinterpret_cast<const float4*>(at);
#pragma unroll
                for (int v = 1; v < 4; ++v) {
                    const float4 y = *reinterpret_cast<const float4*>(at + v * kRows * D);
                    x.x += y.x;
                    x.y += y.y;
                    x.z += y.z;
                    x.w += y.w;
                }
                if (e.whole) {
                    const int token = token_of(e.r0 + r);
                    const int64_t row = e.start + token;
                    const int head = e.kvh * group + (e.r0 + r) - token * group;
                    const float inv = sum == 0.F ? 0.F : 1.F / sum;
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * a.out_stride +
                                              static_cast<int64_t>(head) * D + d) =
                        make_uint2(pack2<DT>(x.x * inv, x.y * inv), pack2<DT>(x.z * inv, x.w * inv));
                    if (d == 0 && a.lse != nullptr)
                        a.lse[row * p.q_heads + head] = sum == 0.F ? -INFINITY : mx * kLn2 + logf(sum);
                } else {
                    if (d == 0) __stcg(reinterpret_cast<float2*>(part) + r, make_float2(mx, sum));
                    __stcg(reinterpret_cast<float4*>(part + 2 * kRows + r * D + d), x);
                }
            }
            __syncthreads();  // `meet`, `row_ml` and in the end the list are free again
        }
        if (pieces < kList) break;
    }
    if (!ok) {
        if (lane == 0 && p.err != nullptr) atomicOr(p.err, 16);
        // no copy may still be on its way when the block ends
        for (uint32_t i = fetched > M::kStages ? fetched - M::kStages : 0; i < fetched; ++i)
            mbar_wait_bounded(&full[warp][i % M::kStages], (i / M::kStages) & 1);
    }
}

constexpr int kMaxBlocks = 148;

template <int DT, int D>
cudaError_t launch_decode(const PagedAttentionArgs& a, cudaStream_t s) {
    const PagedBatch& p = a.p;
    const uint64_t rows = static_cast<uint64_t>(p.num_pages) * p.kv_heads * p.page_size;
    const uint32_t box = kKeys;  // no page is smaller
    CUtensorMap mk, mv;
    const CUtensorMapDataType type =
        DT == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    cudaError_t st = encode_tmap_2d(&mk, type, a.k_pages, D, rows, D * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (st == cudaSuccess)
        st = encode_tmap_2d(&mv, type, a.v_pages, D, rows, D * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (st != cudaSuccess) return st;
    auto kernel = paged_decode_kernel<DT, D>;
    static std::atomic<uint64_t> opted{0};
    st = opt_in_smem(reinterpret_cast<const void*>(kernel), DecodeSmem<D>::kBytes, opted);
    if (st != cudaSuccess) return st;
    const int blocks = device_sm_count() < kMaxBlocks ? device_sm_count() : kMaxBlocks;
    st = launch_pdl(kernel, dim3(blocks), dim3(kThreads), DecodeSmem<D>::kBytes, s, mk, mv, a);
    if (st != cudaSuccess) return st;
    return launch_pdl(paged_join_kernel<DT, D, kRows, true>, dim3(blocks), dim3(kJoinThreads), 0, s, a);
}

}  // namespace

int64_t paged_decode_workspace_bytes(int head_dim) {
    return head_dim == 128 ? PagedPartial<kRows, 128>::bytes(kMaxBlocks)
                           : PagedPartial<kRows, 64>::bytes(kMaxBlocks);
}

cudaError_t paged_decode(const PagedAttentionArgs& a, int dt, cudaStream_t s) {
    if (dt == kBF16) return a.p.head_dim == 128 ? launch_decode<kBF16, 128>(a, s) : launch_decode<kBF16, 64>(a, s);
    return a.p.head_dim == 128 ? launch_decode<kF16, 128>(a, s) : launch_decode<kF16, 64>(a, s);
}

}  // namespace kc

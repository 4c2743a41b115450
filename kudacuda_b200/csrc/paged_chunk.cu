// paged_chunk.cu -- paged attention with many query rows a key head (chunks of
// a prompt, mixed steps) on the tcgen05 tensor cores.
//
// One CTA per SM takes a stretch of the batch's work (paged_plan.cuh): items
// of 256 query rows (two tiles of 128: a tile's rows are the tensor memory's
// lanes) against blocks of 128 keys.  Per block j and tile t
//   S_t = Q_t K_j^T   (Q, K from shared memory; 128 x 128 fp32 in tensor memory)
//   P_t = exp2(c S_t - m_t), rounded to the cache's type over S_t's columns
//   O_t += P_t V_j    (P from tensor memory, V from shared memory, MN-major)
// with the running maximum m in the log2 domain (c = scale log2 e).  A thread
// owns one row, so maximum and sum need no exchange.  m only follows the true
// maximum when that has grown by more than kLazy (a factor of 256, far inside fp32
// and bf16, or of 16 in f16): O is then rescaled in tensor memory, which is rare.
// The final O / l does not depend on m.
//
// Warps: 0-3 and 4-7 softmax, tile 0 and 1; 8 K/V producer (TMA, one box per
// page and 64 dims, 128-byte swizzle); 9 MMA issuer; 10 fetches Q and cleans the
// rows of V that not every row of the item attends: their P is 0 for those that do
// not, but 0 times a NaN is not.  Rows past the item's last key go to 0; the others
// are looked through for values that are not finite, which are taken out and in the
// end added to the rows that attend them; 11 only writes the record of the item that goes
// on into this stretch.
//
// P is rounded to the cache's type because that is what the matrix instruction
// takes (its error, half a step of the type, is that of the output's own rounding;
// sum and maximum are of the unrounded values).  f16 P are scaled up, or the small
// ones would not be there (kShift).  The two tiles take turns: while
// one's scores are exponentiated the other's products run, and the first half of
// P multiplies while the second is made.  Two tiles fill the tensor memory (S 2 x
// 128, O 2 x 128 columns).
//
// Measured, 4 prompts of 2048 tokens of 16 heads over 8192 keys (2 key heads of 128
// bf16 dims; 0.48 Tflop): 375 us on a cool card, 1.28 Pflop/s (the library's
// largest product: 1.63), and 431 us after a second of it, when the power limit
// brings the clocks down (1.12, the library's product: 1.36).  A step of both
// tiles takes 3550 clocks, of which the products could use 2048; the rest is the
// chain from a score to its product with V (load from tensor memory 60, maximum
// 300, exponentials and stores 1250) and six barrier waits of about 180.  Without
// exponentials it takes as long, without any arithmetic on the scores 3300.
// What did not help: blocks of 64 keys with doubled scores (652 us where this took
// 432), part of the exponentials by polynomial, exponentials before the maximum
// is known, one arrival a warp instead of one a thread, waiting by polling.
#include <cuda_bf16.h>

#include "kc_common.cuh"
#include "kc_launch.h"
#include "kc_tcgen05.cuh"
#include "kc_tma.h"
#include "paged_combine.cuh"
#include "paged_plan.cuh"

namespace kc {
namespace {

constexpr int kRows = 256;   // query rows of an item
constexpr int kKeys = 128;   // keys of a block
constexpr int kThreads = 384;
// An item's start and end cost about as much as these keys: eight ragged batches
// together 414 us, with 256 430, with 512 416.
constexpr int kOver = 384;
constexpr int kLeast = 128;  // (96, 192 and 256: within 3% on 24 batches, none better throughout)
// m is a running maximum less kShift, and the true one, less kShift too, may exceed it
// by kLazy.  f16 ends at 2^16 and 2^-25: with P up to 2^15, what rounds to nothing is a
// weight below 2^-36 of the largest (with kShift 0 below 2^-25, and 131071 keys of 2^-25.1
// beside one of 1 were lost: 0.4% of O).  f16 with kLazy 8, 6, 4, 2, 0: the large case 441, 439,
// 441, 468, 485 us, 24 mixed sequences 56.8, 56.8, 56.9, 58.9, 59.3.
template <int DT>
constexpr float kLazy = DT == kF16 ? 4.F : 8.F;
template <int DT>
constexpr float kShift = DT == kF16 ? 15.F - kLazy<DT> : 0.F;

template <int D>
struct ChunkSmem {
    static constexpr int kHalves = D / 64;
    static constexpr int kTile = kHalves * 128 * 128;  // 128 rows of Q, K or V: [D / 64][128][128 B]
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr int kBytes = 1024 + 2 * kTile + kStages * kTile;
};

// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ float max3(float x, float y, float z) {  // NaN if one is
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}
// two 32-bit numbers in a register pair
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float low(uint64_t v) {
    float x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
    return x;
}
__device__ __forceinline__ float high(uint64_t v) {
    float x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
    return y;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
// A wait that may last for whole pieces (one of 2^20 blocks takes a second, 2^17
// tries end after 0.2): it gives up when no block has been fetched for as long as
// any other wait would last (the ring holds a few).
__device__ __forceinline__ bool bar_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                              const volatile int* beat) {
    for (int round = 0, seen = 0;; ++round) {
        for (uint32_t i = 0; i < (1u << 17); ++i) {
            if (mbar_try_wait(bar, parity)) return true;
            if (*abort_flag) return false;
        }
        const int now = *beat;
        if (round > 0 && now == seen) break;
        seen = now;
    }
    *abort_flag = 1;
    return false;
}
// whether block j has rows that not every row of the item attends, as its last ones
__device__ __forceinline__ bool is_tail(int j, int least) { return (j + 1) * kKeys > least; }
// 16-bit values from this magnitude on are not finite
template <int DT>
constexpr uint32_t kNotFinite = DT == kBF16 ? 0x7f80u : 0x7c00u;
// the two 16-bit values of x, 0 where not finite
template <int DT>
__device__ __forceinline__ uint32_t finite_only(uint32_t x) {
    const uint32_t size = x & 0x7fff7fffu;
    return x & ((size & 0xffffu) >= kNotFinite<DT> ? 0xffff0000u : 0xffffffffu) &
           (size >> 16 >= kNotFinite<DT> ? 0xffffu : 0xffffffffu);
}

struct ChunkBars {
    uint64_t kv_full[8], kv_empty[8];
    uint64_t v_tail[8];  // a block of V has landed whose last rows are to be looked at first
    uint64_t q_full, q_empty;
    uint64_t s_full[2], p_half[2], p_ready[2], o_done[2];
};

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_q, const PagedAttentionArgs a, int q_by_tma) {
    using M = ChunkSmem<D>;
    using W = PagedWalk<kRows, kKeys, kOver>;
    using Part = PagedPartial<kRows, D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) ChunkBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, beat_count;
    __shared__ int odd_first, odd_last;  // the pieces from whose V something was taken out
    __shared__ int64_t sums[kThreads / 32], place_at;
    __shared__ int place_seq;
    const PagedBatch& p = a.p;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    uint8_t* const base = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    uint8_t* const qs = base;
    uint8_t* const ring = base + 2 * M::kTile;

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        for (int i = 0; i < M::kStages; ++i) {
            mbar_init(&bars.kv_full[i], 1);
            mbar_init(&bars.kv_empty[i], 1);
            mbar_init(&bars.v_tail[i], 1);
        }
        mbar_init(&bars.q_full, 1);
        mbar_init(&bars.q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_half[i], 128);
            mbar_init(&bars.p_ready[i], 128);
            mbar_init(&bars.o_done[i], 1);
        }
        abort_flag = beat_count = 0;
        odd_first = 0x7fffffff;
        odd_last = -1;
        fence_mbar_init();
    }
    tc_fence_before();
    pdl_wait_on_producer();
    const int group = p.q_heads / p.kv_heads;
    const int worker = blockIdx.x;
    const PagedShares shares =
        paged_place<W, kLeast, kThreads>(p, group, worker, gridDim.x, sums, &place_seq, &place_at);
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = __reduce_max_sync(0xffffffffu, tmem_slot);
    volatile int* const abort_p = &abort_flag;
    volatile int* const beat = &beat_count;  // blocks fetched
    W w;
    w.begin(p, group, shares, worker, place_seq, place_at);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ---- K/V producer: K_0, V_0, K_1, V_1, ... of every piece through the ring
            uint32_t seq = 0, tail_use = 0, tail_parity = 0;  // per stage: its last copy was a tail, tails so far
            bool ok = true;
            while (ok && w.next(p, group)) {
                const int32_t* table = p.table + w.piece_b * p.table_stride;
                for (int j = w.t0; j < w.t1 && ok; ++j) {
                    const int pages = min(kKeys, w.limit - j * kKeys + p.page_size - 1) / p.page_size;
                    const int part = lane / M::kHalves, half = lane % M::kHalves;
                    const bool mine = part < pages;
                    int row = 0;
                    if (mine) {
                        const int page = table[j * (kKeys / p.page_size) + part];
                        // a missing page reads as zeros: a box that begins before the tensor
                        row = -p.page_size;
                        if (page >= 0 && page < p.num_pages) row = (page * p.kv_heads + w.kvh) * p.page_size;
                        else if (half == 0 && p.err != nullptr) atomicOr(p.err, 2);
                    }
                    for (int v = 0; v < 2; ++v, ++seq) {
                        const int s = seq % M::kStages;
                        if (seq >= M::kStages) ok = bar_wait(&bars.kv_empty[s], (seq / M::kStages - 1) & 1, abort_p);
                        if (!ok) break;
                        // a tail of V goes through warp 10, which then completes kv_full
                        const bool tail = v == 1 && is_tail(j, w.least);
                        tail_use = tail ? tail_use | 1u << s : tail_use & ~(1u << s);
                        if (tail) tail_parity ^= 1u << s;
                        uint64_t* const full = tail ? &bars.v_tail[s] : &bars.kv_full[s];
                        if (lane == 0) {
                            *beat = static_cast<int>(seq);
                            mbar_arrive_expect_tx(full, pages * p.page_size * 128 * M::kHalves);
                        }
                        __syncwarp();
                        if (mine)
                            tma_load_2d(ring + s * M::kTile + half * (128 * 128) + part * p.page_size * 128,
                                        v ? &map_v : &map_k, half * 64, row, full);
                    }
                }
                if (w.piece_len > p.table_width * p.page_size && lane == 0 && p.err != nullptr) atomicOr(p.err, 2);
            }
            // every copy has landed before the CTA may exit (normally already true)
            const uint32_t first = seq > M::kStages ? seq - M::kStages : 0;
            for (uint32_t i = first; i < seq; ++i) {
                const uint32_t s = i % M::kStages;
                if (tail_use >> s & 1) bar_wait(&bars.v_tail[s], ~tail_parity >> s & 1, abort_p, false);
                else bar_wait(&bars.kv_full[s], (i / M::kStages) & 1, abort_p, false);
            }
        } else if (warp == 9) {
            // ---- MMA issuer: the warp runs converged, one lane issues
            constexpr uint32_t kIdescS = umma_idesc(DT == kBF16, 128, 128, false);
            constexpr uint32_t kIdescO = umma_idesc(DT == kBF16, 128, D, true);
            uint32_t seq = 0, items = 0, np[2] = {0, 0};
            const uint32_t q_addr = smem_u32(qs), r_addr = smem_u32(ring);
            while (__any_sync(0xffffffffu, w.next(p, group))) {
                const int active = __reduce_max_sync(0xffffffffu, w.item_rows > 128 ? 2 : 1);
                const int n = __reduce_max_sync(0xffffffffu, w.t1 - w.t0);
                bar_wait(&bars.q_full, items & 1, abort_p);
                for (int j = 0; j <= n; ++j) {
                    // O_t += P_t(j - 1) V(j - 1), then S_t = Q_t K(j)^T over P_t(j - 1)'s
                    // columns: the matrix instructions of one thread run in order
                    const uint32_t sv = seq + 2 * j - 1, sk = seq + 2 * j;
                    if (j > 0) bar_wait(&bars.kv_full[sv % M::kStages], (sv / M::kStages) & 1, abort_p);
                    if (j < n) bar_wait(&bars.kv_full[sk % M::kStages], (sk / M::kStages) & 1, abort_p);
                    tc_fence_after();
                    const uint32_t va = r_addr + (sv % M::kStages) * M::kTile;
                    const uint32_t ka = r_addr + (sk % M::kStages) * M::kTile;
                    for (int t = 0; t < active; ++t) {
                        if (j > 0) {
                            // (the first half of P multiplies while the second is still being made)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                bar_wait(h ? &bars.p_ready[t] : &bars.p_half[t], np[t] & 1, abort_p);
                                tc_fence_after();
                                if (elect_one()) {
#pragma unroll
                                    for (int k = h * (kKeys / 32); k < (h + 1) * (kKeys / 32); ++k)
                                        umma_bf16_ts(tmem + 256 + t * D, tmem + t * 128 + 8 * k,
                                                     umma_desc_sw128_mn(va + 2048 * k, 128 * 128), kIdescO,
                                                     (j > 1 || k > 0) ? 1u : 0u);
                                }
                                __syncwarp();
                            }
                            ++np[t];
                        }
                        if (elect_one()) {
                            if (j < n) {
#pragma unroll
                                for (int k = 0; k < D / 16; ++k) {
                                    const uint32_t off = (k / 4) * (128 * 128) + (k % 4) * 32;
                                    umma_bf16(tmem + t * 128, umma_desc_sw128(q_addr + t * M::kTile + off),
                                              umma_desc_sw128(ka + off), kIdescS, k > 0 ? 1u : 0u);
                                }
                                umma_commit(&bars.s_full[t]);
                            } else {
                                umma_commit(&bars.o_done[t]);
                            }
                            if (t == active - 1) {
                                if (j > 0) umma_commit(&bars.kv_empty[sv % M::kStages]);
                                if (j < n) umma_commit(&bars.kv_empty[sk % M::kStages]);
                                if (j == n - 1) umma_commit(&bars.q_empty);
                            }
                        }
                        __syncwarp();
                    }
                }
                seq += 2 * n;
                ++items;
            }
        } else if (warp == 10) {
            // ---- Q: row R of the item is token R / group, head R % group; rows past the item are zero
            uint32_t items = 0, seq = 0, tail_parity = 0;
            const uint16_t* q = static_cast<const uint16_t*>(a.q);
            while (w.next(p, group)) {
                // (the whole of the piece before)
                if (items > 0 && !bar_wait_long(&bars.q_empty, (items - 1) & 1, abort_p, beat)) break;
                const int r_all = w.item_rows > 128 ? 256 : 128;
                if (q_by_tma) {  // 128 / group whole tokens a tile (rows past the item are other tokens': not stored)
                    if (lane == 0) mbar_arrive_expect_tx(&bars.q_full, r_all * D * 2);
                    __syncwarp();
                    const int t = lane / M::kHalves, half = lane % M::kHalves;
                    if (t * 128 < r_all)
                        tma_load_3d(qs + t * M::kTile + half * (128 * 128), &map_q, half * 64, w.kvh * group,
                                    w.piece_start + (w.q * kRows + t * 128) / group, &bars.q_full);
                } else {
                    for (int r = lane; r < r_all; r += 32) {  // a lane a row
                        const bool live = r < w.item_rows;
                        const int token = (w.q * kRows + r) / group, head = (w.q * kRows + r) - token * group;
                        const uint16_t* src =
                            q + (live ? (w.piece_start + token) * a.q_stride +
                                            static_cast<int64_t>(w.kvh * group + head) * D
                                      : 0);
                        const uint32_t dst = smem_u32(qs) + (r >> 7) * M::kTile + (r & 127) * 128;
#pragma unroll
                        for (int c = 0; c < D / 8; ++c)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                             dst + (c >> 3) * (128 * 128) + (((c & 7) ^ (r & 7)) << 4)),
                                         "l"(src + 8 * c), "r"(live ? 16 : 0)
                                         : "memory");
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&bars.q_full);
                }
                ++items;
                bool ok = true;
                for (int j = max(w.t0, w.least / kKeys); j < w.t1; ++j) {
                    const uint32_t sv = (seq + 2 * (j - w.t0) + 1) % M::kStages;
                    ok = bar_wait_long(&bars.v_tail[sv], tail_parity >> sv & 1, abort_p, beat);
                    if (!ok) break;
                    tail_parity ^= 1u << sv;
                    // rows from `some` on are attended by some rows of the item, from `none` on by none
                    const int some = max(w.least - j * kKeys, 0), none = min(w.limit - j * kKeys, kKeys);
                    uint4* const v = reinterpret_cast<uint4*>(ring + sv * M::kTile);
                    uint32_t most = 0;  // the largest magnitude of either half
#pragma unroll 4
                    for (int i = some * 8 + lane; i < none * 8; i += 32)
#pragma unroll
                        for (int h = 0; h < M::kHalves; ++h) {
                            const uint4 x = v[h * (128 * 8) + i];
                            most = __vmaxu2(most, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu));
                            most = __vmaxu2(most, __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
                        }
                    if (__any_sync(0xffffffffu, max(most & 0xffffu, most >> 16) >= kNotFinite<DT>)) {
                        for (int i = some * 8 + lane; i < none * 8; i += 32)
                            for (int h = 0; h < M::kHalves; ++h) {
                                const uint4 x = v[h * (128 * 8) + i];
                                v[h * (128 * 8) + i] = make_uint4(finite_only<DT>(x.x), finite_only<DT>(x.y),
                                                                  finite_only<DT>(x.z), finite_only<DT>(x.w));
                            }
                        odd_first = min(odd_first, static_cast<int>(items) - 1);
                        odd_last = static_cast<int>(items) - 1;
                    }
                    for (int i = none * 8 + lane; i < kKeys * 8; i += 32)
#pragma unroll
                        for (int h = 0; h < M::kHalves; ++h) v[h * (128 * 8) + i] = make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&bars.kv_full[sv]);
                }
                if (!ok) break;
                seq += 2 * (w.t1 - w.t0);
            }
            if (q_by_tma && items > 0) bar_wait(&bars.q_full, (items - 1) & 1, abort_p, false);  // Q has landed
        }
    } else {
        // ---- softmax: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * D;
        const int r = t * 128 + 32 * (warp & 3) + lane;
        const float c = a.scale * kLog2E;
        uint32_t ns = 0, no = 0;
        while (w.next(p, group)) {
            if (t == 1 && w.item_rows <= 128) continue;
            const bool live = r < w.item_rows;
            const int token = (w.q * kRows + r) / group;
            // this row's keys, relative to the item: never more than the item's
            const int row_keys = live ? min(max(w.piece_len - w.piece_n + token + 1, 0), w.limit) : w.limit;
            const bool idle = !__any_sync(0xffffffffu, live);  // a warp of rows past the item: it only keeps step
            float m = -INFINITY, l = 0.F;
            for (int j = w.t0; j < w.t1; ++j) {
                // (the second tile's first block: the whole of every piece without that tile)
                bar_wait_long(&bars.s_full[t], ns++ & 1, abort_p, beat);
                tc_fence_after();
                if (idle) {  // (what its lanes of P hold reaches no row of the item)
                    tc_fence_before();
                    bar_arrive(&bars.p_half[t]);
                    bar_arrive(&bars.p_ready[t]);
                    continue;
                }
                float s[kKeys];
#pragma unroll
                for (int i = 0; i < kKeys; i += 32) tmem_ld32(ts + i, s + i);
                tmem_wait_ld();
                const int keys = row_keys - j * kKeys;
                if (__any_sync(0xffffffffu, keys < kKeys)) {
#pragma unroll
                    for (int i = 0; i < kKeys; ++i) s[i] = i < keys ? s[i] : -INFINITY;
                }
                float mx[2] = {s[0], s[1]};
#pragma unroll
                for (int i = 2; i < kKeys - 2; i += 4) {
                    mx[0] = max3(mx[0], s[i], s[i + 1]);
                    mx[1] = max3(mx[1], s[i + 2], s[i + 3]);
                }
                const float top = fmaf(max3(max3(mx[0], s[kKeys - 2], s[kKeys - 1]), mx[1], mx[1]), c, -kShift<DT>);
                if (top != top) l = top;  // a NaN score makes the row NaN
                const bool grow = top > m + kLazy<DT>;  // from -inf: any finite maximum
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = grow ? top : m;
                    const float f = grow ? ex2(m - mn) : 1.F;
                    l *= f;
                    m = mn;
                    if (j > w.t0) {
                        // S_t(j) is complete, so every earlier matrix instruction on O_t is too
#pragma unroll 1
                        for (int i = 0; i < D; i += 32) {
                            float o[32];
                            tmem_ld32(to + i, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] *= f;
                            tmem_st32(to + i, reinterpret_cast<uint32_t*>(o));
                        }
                    }
                }
                const float sub = m == -INFINITY ? 0.F : m;
                const uint64_t c2 = pair(c, c), sub2 = pair(-sub, -sub);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint64_t x = fma2(pair(s[64 * h + 2 * i], s[64 * h + 2 * i + 1]), c2, sub2);
                        const uint64_t e = pair(ex2(low(x)), ex2(high(x)));
                        sum2[i & 1] = add2(sum2[i & 1], e);
                        pk[i] = pack2<DT>(low(e), high(e));
                    }
                    tmem_st32(ts + 32 * h, pk);
                    tmem_wait_st();
                    tc_fence_before();
                    bar_arrive(h ? &bars.p_ready[t] : &bars.p_half[t]);
                }
                sum2[0] = add2(sum2[0], sum2[1]);
                l += low(sum2[0]) + high(sum2[0]);
            }
            // ---- the piece's end
            bar_wait(&bars.o_done[t], no++ & 1, abort_p);
            tc_fence_after();
            if (idle) continue;
            if (w.whole()) {
                const float inv = l == 0.F ? 0.F : 1.F / l;
                const int64_t row = w.piece_start + token;
                const int head = w.kvh * group + (w.q * kRows + r) % group;
                uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.out_stride + static_cast<int64_t>(head) * D;
#pragma unroll 1
                for (int i = 0; i < D; i += 32) {
                    float o[32];
                    tmem_ld32(to + i, o);
                    tmem_wait_ld();
                    if (live) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            uint32_t x[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) x[y] = pack2<DT>(o[k + 2 * y] * inv, o[k + 2 * y + 1] * inv);
                            *reinterpret_cast<uint4*>(out + i + k) = make_uint4(x[0], x[1], x[2], x[3]);
                        }
                    }
                }
                if (live && a.lse != nullptr) a.lse[row * p.q_heads + head] = l == 0.F ? -INFINITY : m * kLn2 + logf(l);
            } else {
                float* part = Part::slot(a.workspace, gridDim.x, worker, w.t0 > 0 ? 0 : 1);
                if (live) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(m, l);
                float4* acc = reinterpret_cast<float4*>(part + 2 * kRows);
#pragma unroll 1
                for (int i = 0; i < D; i += 32) {
                    float o[32];
                    tmem_ld32(to + i, o);
                    tmem_wait_ld();
                    if (!live) continue;
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        __stcg(acc + ((i + k) >> 2) * kRows + r, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                }
            }
            tc_fence_before();
        }
    }
    // what the join needs to know of the item that goes on into this stretch
    if (tid == 352) {
        W v;
        v.begin(p, group, shares, worker, place_seq, place_at);
        Part::cuts(a.workspace)[worker] = v.record(p, group, shares, worker);
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort_p && p.err != nullptr) atomicOr(p.err, 16);  // (every wait is over)
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
    // (rare) what was taken out of V, to the rows that attend it: thread = row, as above
    if (odd_first > odd_last || warp >= 8) return;
    W v;
    v.begin(p, group, shares, worker, place_seq, place_at);
#pragma unroll 1
    for (int piece = 0; piece <= odd_last && v.next(p, group); ++piece) {
        const int token = (v.q * kRows + tid) / group;
        if (piece < odd_first || tid >= v.item_rows) continue;
        const int end = min(min(max(v.piece_len - v.piece_n + token + 1, 0), v.limit), v.t1 * kKeys);
        uint16_t* const out = static_cast<uint16_t*>(a.out) + (v.piece_start + token) * a.out_stride +
                              static_cast<int64_t>(v.kvh * group + (v.q * kRows + tid) % group) * D;
        float* const part = Part::slot(a.workspace, gridDim.x, worker, v.t0 > 0 ? 0 : 1) + 2 * kRows + tid * 4;
#pragma unroll 1
        for (int key = max(v.t0 * kKeys, v.least); key < end; ++key) {
            const int page = p.table[v.piece_b * p.table_stride + key / p.page_size];
            if (page < 0 || page >= p.num_pages) continue;
            const uint16_t* const x = static_cast<const uint16_t*>(a.v_pages) +
                                      ((static_cast<int64_t>(page) * p.kv_heads + v.kvh) * p.page_size +
                                       (key & (p.page_size - 1))) * D;
#pragma unroll 1
            for (int i = 0; i < D; ++i) {
                if ((x[i] & 0x7fffu) < kNotFinite<DT>) continue;
                const float y = DT == kBF16 ? bf16_bits_to_f32(x[i]) : f16_bits_to_f32(x[i]);
                float* const at = part + (i >> 2) * (kRows * 4) + (i & 3);
                if (v.whole()) {
                    const float z = DT == kBF16 ? bf16_bits_to_f32(out[i]) : f16_bits_to_f32(out[i]);
                    out[i] = static_cast<uint16_t>(pack2<DT>(z + y, 0.F));
                } else {
                    *at += y;
                }
            }
        }
    }
}

}  // namespace

namespace {
constexpr int kMaxWorkers = 148;

template <int DT, int D>
cudaError_t launch_chunk(const PagedAttentionArgs& a, cudaStream_t s) {
    const PagedBatch& p = a.p;
    const uint64_t rows = static_cast<uint64_t>(p.num_pages) * p.kv_heads * p.page_size;
    CUtensorMap mk, mv, mq;
    const CUtensorMapDataType type =
        DT == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    cudaError_t st = encode_tmap_2d(&mk, type, a.k_pages, D, rows, D * 2, 64, p.page_size, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (st == cudaSuccess)
        st = encode_tmap_2d(&mv, type, a.v_pages, D, rows, D * 2, 64, p.page_size, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (st != cudaSuccess) return st;
    // a tile of 128 rows is whole tokens when the group divides it: then Q comes by TMA too
    const int group = p.q_heads / p.kv_heads;
    const int by_tma = group <= 128 && 128 % group == 0 ? 1 : 0;
    if (by_tma) {
        st = encode_tmap_3d(&mq, type, a.q, D, p.q_heads, p.rows, D * 2, a.q_stride * 2, 64, group, 128 / group,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
        if (st != cudaSuccess) return st;
    } else {
        mq = mk;
    }
    auto kernel = paged_chunk_kernel<DT, D>;
    static std::atomic<uint64_t> opted{0};
    st = opt_in_smem(reinterpret_cast<const void*>(kernel), ChunkSmem<D>::kBytes, opted);
    if (st != cudaSuccess) return st;
    const int workers = device_sm_count() < kMaxWorkers ? device_sm_count() : kMaxWorkers;
    st = launch_pdl(kernel, dim3(workers), dim3(kThreads), ChunkSmem<D>::kBytes, s, mk, mv, mq, a, by_tma);
    if (st != cudaSuccess) return st;
    // Blocks of the join: with about a full item of 256 rows for every two workers
    // four a worker (24 ragged sequences of 39 tokens each, 32 heads: 64.8 us in all,
    // with two 66.2, when the rest was slower), else two (4 tokens of 8 heads over 100:
    // 11.1 us, with four 11.8).
    const int ways = static_cast<int64_t>(p.rows) * p.q_heads >= workers * (kRows / 2) ? 4 : 2;
    return launch_pdl(paged_join_kernel<DT, D, kRows, false>, dim3(workers, ways), dim3(kJoinThreads), 0, s, a);
}
}  // namespace

int64_t paged_chunk_workspace_bytes(int head_dim) {
    return head_dim == 128 ? PagedPartial<kRows, 128>::bytes(kMaxWorkers) : PagedPartial<kRows, 64>::bytes(kMaxWorkers);
}

cudaError_t paged_chunk(const PagedAttentionArgs& a, int dt, cudaStream_t s) {
    if (dt == kBF16) return a.p.head_dim == 128 ? launch_chunk<kBF16, 128>(a, s) : launch_chunk<kBF16, 64>(a, s);
    return a.p.head_dim == 128 ? launch_chunk<kF16, 128>(a, s) : launch_chunk<kF16, 64>(a, s);
}

}  // namespace kc

// paged_decode.cu -- paged attention with few query rows a key head (decoding):
// the cache is read once, at the speed of memory.
//
// A warp is a worker (paged_plan.cuh): it takes a stretch of the batch's work,
// items of 16 query rows (mma.m16n8k16's M; a single token of a group of 8
// fills half of it, which costs nothing here) against blocks of 32 keys, and
// needs no other warp: its own ring of K and V blocks in shared memory, fetched
// by TMA page by page (128-byte swizzle), its own barriers, its own running
// maximum, sum and 16 x head_dim accumulator in registers.  So nothing in the
// loop waits for anything but memory, and kStages blocks of a warp are in
// flight: 4 warps x 3 blocks x 16 KB on every SM, seven times what covers the
// latency of 6.5 TB/s.
//
// S = Q K^T with exact products and 32-bit sums; softmax in the log2 domain; P
// is split into two 16-bit halves (P = hi + lo to about twice the type's
// precision), so P V is as good as with 32-bit probabilities: the tensor cores
// have time to spare while the cache arrives.
#include "kc_common.cuh"
#include "kc_launch.h"
#include "kc_tcgen05.cuh"
#include "kc_tma.h"
#include "paged_combine.cuh"
#include "paged_plan.cuh"

namespace kc {
namespace {

constexpr int kRows = 16;
constexpr int kKeys = 32;
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

template <int D>
struct DecodeSmem {
    static constexpr int kHalves = D / 64;
    static constexpr int kBlock = kHalves * kKeys * 128;  // [D / 64][32][128 B]
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kWarpBytes = kStages * 2 * kBlock;
    static constexpr int kBytes = 1024 + kWarps * kWarpBytes;
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

template <int DT, int D>
__global__ void __launch_bounds__(kThreads)
    paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const PagedAttentionArgs a) {
    using M = DecodeSmem<D>;
    using W = PagedWalk<kRows, kKeys>;
    using Part = PagedPartial<kRows, D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[kWarps][M::kStages];
    __shared__ int64_t sums[kWarps], place_at[kWarps];
    __shared__ int place_seq[kWarps];
    const PagedBatch& p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* const ring =
        smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw)) + warp * M::kWarpBytes;
    if (lane == 0) {
        for (int i = 0; i < M::kStages; ++i) mbar_init(&full[warp][i], 1);
        fence_mbar_init();
    }
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const int group = p.q_heads / p.kv_heads;
    // (worker = warp-major, so that few workers lie on many SMs)
    const int slots = gridDim.x * kWarps, worker = warp * gridDim.x + blockIdx.x;
    int workers = slots;
    const int64_t total = paged_places<kRows, kKeys, kThreads>(p, group, blockIdx.x, gridDim.x, kWarps, workers, sums,
                                                               place_seq, place_at);
    W w, ahead;  // the piece at hand; the piece whose blocks are being fetched
    w.begin(p, group, paged_bound(total, worker, workers), paged_bound(total, worker + 1, workers), place_seq[warp],
            place_at[warp]);
    ahead = w;
    bool more = ahead.next(p, group);
    int ahead_j = more ? ahead.t0 : 0;
    uint32_t fetched = 0, used = 0;

    // fetch the next block, K and V, into its stage (which its reader has left)
    auto fetch = [&]() {
        if (!more) return;
        const int key0 = ahead_j * kKeys;
        const int box = min(p.page_size, kKeys);  // keys of a TMA box
        const int boxes = min(kKeys, ahead.limit - key0 + box - 1) / box;
        const int part = lane / (2 * M::kHalves), half = (lane >> 1) % M::kHalves, v = lane & 1;
        const uint32_t s = fetched % M::kStages;
        uint8_t* const stage = ring + s * 2 * M::kBlock;
        int row = 0;
        if (part < boxes) {
            const int key = key0 + part * box, page = p.table[ahead.piece_b * p.table_stride + key / p.page_size];
            row = -box;  // a missing page reads as zeros: a box that begins before the tensor
            if (page >= 0 && page < p.num_pages)
                row = (page * p.kv_heads + ahead.kvh) * p.page_size + key % p.page_size;
            else if (p.err != nullptr) atomicOr(p.err, 2);
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[warp][s], boxes * box * 128 * M::kHalves * 2);
        __syncwarp();
        if (part < boxes)
            tma_load_2d(stage + v * M::kBlock + half * (kKeys * 128) + part * box * 128, v ? &map_v : &map_k, half * 64,
                        row, &full[warp][s]);
        ++fetched;
        if (++ahead_j == ahead.t1) {
            more = ahead.next(p, group);
            ahead_j = more ? ahead.t0 : 0;
        }
    };
    for (int i = 0; i < M::kStages - 1; ++i) fetch();

    const float c = a.scale * kLog2E;
    const int g = lane >> 2, t4 = lane & 3;  // an accumulator's rows g and g + 8, columns 2 t4 and 2 t4 + 1
    PagedCut cut;
    cut.valid = cut.tail = cut.row0 = cut.r0 = cut.rows = cut.kvh = cut.last = cut.pad = 0;
    bool ok = true;
    while (w.next(p, group)) {
        if (w.piece_len > p.table_width * p.page_size && lane == 0 && p.err != nullptr) atomicOr(p.err, 2);
        // Q: the A fragments of the item's 16 rows, straight from memory
        uint32_t qf[D / 16][4];
        int row_keys[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h, token = (w.q * kRows + r) / group, head = (w.q * kRows + r) % group;
            const bool live = r < w.item_rows;
            const uint16_t* q = static_cast<const uint16_t*>(a.q) +
                                (live ? (w.piece_start + token) * a.q_stride + static_cast<int64_t>(w.kvh * group + head) * D : 0);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    qf[k][2 * e + h] = live ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8 * e + 2 * t4) : 0u;
            row_keys[h] = live ? min(max(w.piece_len - w.piece_n + token + 1, 0), w.limit) : 0;
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.F;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.F, 0.F};
        for (int j = w.t0; j < w.t1; ++j) {
            fetch();
            const uint32_t s = used % M::kStages;
            if (!mbar_wait_bounded(&full[warp][s], (used / M::kStages) & 1)) ok = false;
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            ++used;
            const uint32_t kb = smem_u32(ring + s * 2 * M::kBlock), vb = kb + M::kBlock;
            // S: 16 rows x 32 keys, four tiles of 8 keys
            float sc[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.F;
#pragma unroll
            for (int n2 = 0; n2 < 2; ++n2) {
                // ldmatrix: keys 16 n2 .. + 15 (two tiles), 16 dims (two 8-dim words)
                const int key = 16 * n2 + (lane & 7) + ((lane >> 4) << 3);
                const uint32_t row = kb + key * 128;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const int word = 2 * (k & 3) + ((lane >> 3) & 1);
                    uint32_t b[4];
                    ldsm4(b, row + (k >> 2) * (kKeys * 128) + ((word ^ (key & 7)) << 4));
                    mma16816<DT>(sc[2 * n2], qf[k], b[0], b[1]);
                    mma16816<DT>(sc[2 * n2 + 1], qf[k], b[2], b[3]);
                }
            }
            const int key0 = j * kKeys;
            const int valid = w.limit - key0;  // keys of the block that exist
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + 8 * n + 2 * t4 + (e & 1);
                    const float x = key < row_keys[e >> 1] ? sc[n][e] * c : -INFINITY;
                    sc[n][e] = x;
                    top[e >> 1] = fmaxf(top[e >> 1], x);
                }
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const float mn = fmaxf(m[h], top[h]);
                f[h] = mn == -INFINITY ? 1.F : ex2(m[h] - mn);
                m[h] = mn;
                l[h] *= f[h];
            }
            if (__any_sync(0xffffffffu, f[0] != 1.F || f[1] != 1.F)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    o[i][0] *= f[0];
                    o[i][1] *= f[0];
                    o[i][2] *= f[1];
                    o[i][3] *= f[1];
                }
            }
            const float sub[2] = {m[0] == -INFINITY ? 0.F : m[0], m[1] == -INFINITY ? 0.F : m[1]};
            // P in A-fragment order, 16 keys a fragment, as hi + lo
            uint32_t ph[2][4], pl[2][4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float e0 = ex2(sc[n][2 * h] - sub[h]), e1 = ex2(sc[n][2 * h + 1] - sub[h]);
                    l[h] += e0 + e1;
                    const uint32_t hi = pack2<DT>(e0, e1);
                    const float2 back = unpack2<DT>(hi);
                    ph[n >> 1][2 * (n & 1) + h] = hi;
                    pl[n >> 1][2 * (n & 1) + h] = pack2<DT>(e0 - back.x, e1 - back.y);
                }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int key = 16 * kk + (lane & 15);
                const uint32_t row = vb + key * 128;
                // slots without a key may hold anything, a NaN too: their V must not meet P = 0
                const int left = valid - 16 * kk;
                uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                if (left < 16) {
                    const int k0 = 2 * t4, k1 = 2 * t4 + 8;
                    keep0 = (k0 < left ? 0xffffu : 0u) | (k0 + 1 < left ? 0xffff0000u : 0u);
                    keep1 = (k1 < left ? 0xffffu : 0u) | (k1 + 1 < left ? 0xffff0000u : 0u);
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
                    mma16816<DT>(o[2 * d], pl[kk], b[0], b[1]);
                    mma16816<DT>(o[2 * d + 1], ph[kk], b[2], b[3]);
                    mma16816<DT>(o[2 * d + 1], pl[kk], b[2], b[3]);
                }
            }
            // this stage is refilled one block from now: every lane has read it (the
            // next fetch() begins with the warp's barrier) before the copy starts
            __syncwarp();
        }
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
        if (w.whole()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = g + 8 * h;
                if (r >= w.item_rows) continue;
                const int64_t row = w.piece_start + (w.q * kRows + r) / group;
                const int head = w.kvh * group + (w.q * kRows + r) % group;
                const float inv = l[h] > 0.F ? 1.F / l[h] : 0.F;
                uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.out_stride + static_cast<int64_t>(head) * D;
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    *reinterpret_cast<uint32_t*>(out + 8 * i + 2 * t4) = pack2<DT>(o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
                if (t4 == 0 && a.lse != nullptr)
                    a.lse[row * p.q_heads + head] = l[h] > 0.F ? m[h] * kLn2 + logf(l[h]) : -INFINITY;
            }
        } else {
            float* part = Part::slot(a.workspace, slots, worker, w.t0 > 0 ? 0 : 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = g + 8 * h;
                if (r >= w.item_rows) continue;
                if (t4 == 0) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(m[h], l[h]);
                float* acc = part + 2 * kRows;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const int d = 8 * i + 2 * t4;
                    __stcg(reinterpret_cast<float2*>(acc + ((d >> 2) * kRows + r) * 4 + (d & 3)),
                           make_float2(o[i][2 * h], o[i][2 * h + 1]));
                }
            }
            if (w.t0 > 0) {
                cut.tail = 1;
            } else {
                cut.valid = 1;
                cut.row0 = w.piece_start;
                cut.r0 = w.q * kRows;
                cut.rows = w.item_rows;
                cut.kvh = w.kvh;
                cut.last = static_cast<int>((w.item_end * workers + total - 1) / total - 1);
            }
        }
    }
    if (!ok) {
        if (lane == 0 && p.err != nullptr) atomicOr(p.err, 16);
        // no copy may still be on its way when the block ends
        for (; used < fetched; ++used) mbar_wait_bounded(&full[warp][used % M::kStages], (used / M::kStages) & 1);
    }
    if (lane == 0) Part::cuts(a.workspace)[worker] = cut;
}

constexpr int kMaxBlocks = 148;

template <int DT, int D>
cudaError_t launch_decode(const PagedAttentionArgs& a, cudaStream_t s) {
    const PagedBatch& p = a.p;
    const uint64_t rows = static_cast<uint64_t>(p.num_pages) * p.kv_heads * p.page_size;
    const uint32_t box = p.page_size < kKeys ? p.page_size : kKeys;
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
    return launch_pdl(paged_combine_kernel<DT, D, kRows>, dim3(blocks * kWarps, 1), dim3(256), 0, s, a, blocks * kWarps);
}

}  // namespace

int64_t paged_decode_workspace_bytes(int head_dim) {
    return head_dim == 128 ? PagedPartial<kRows, 128>::bytes(kMaxBlocks * kWarps)
                           : PagedPartial<kRows, 64>::bytes(kMaxBlocks * kWarps);
}

cudaError_t paged_decode(const PagedAttentionArgs& a, int dt, cudaStream_t s) {
    if (dt == kBF16) return a.p.head_dim == 128 ? launch_decode<kBF16, 128>(a, s) : launch_decode<kBF16, 64>(a, s);
    return a.p.head_dim == 128 ? launch_decode<kF16, 128>(a, s) : launch_decode<kF16, 64>(a, s);
}

}  // namespace kc

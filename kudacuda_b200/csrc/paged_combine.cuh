// paged_combine.cuh -- the join of the items that paged attention's workers
// cut, and what its two kernels share besides.
#pragma once

#include "paged_plan.cuh"

namespace kc {

constexpr float kLn2 = 0.6931471805599453F;
constexpr float kLog2E = 1.4426950408889634F;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (DT == kBF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The join of cut items: with M the largest of the pieces' maxima,
// O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in a fixed order of the
// pieces (the same bits on every run).
//
// What it costs is reading the pieces, from L2.  A long sequence's item has pieces
// from many workers (4 key heads of 8000 keys: 37 each), more than one SM reads
// quickly: with a block for an item, two tokens of 8 heads over 8000 keys took
// 38 us, of which this kernel took 27.  So an item is dealt out, in patches of rows
// and dims, to the blocks of the workers that it went through: 15 us and 4.  A
// warp takes a patch; with fewer patches than warps several share a patch's
// pieces (share i has pieces i, i + shares, ...) and meet in shared memory.
//
// BY_ROW: accumulators lie as [row][dim] and a patch is two whole rows; else as
// [dim / 4][row][4], and a patch is eight rows (so that whole 128-byte lines are
// read) by half of the dims.  gridDim.y blocks stand for a worker.
constexpr int kJoinThreads = 256;
template <int DT, int D, int ROWS, bool BY_ROW>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedAttentionArgs a) {
    using Part = PagedPartial<ROWS, D>;
    constexpr int kWarps = kJoinThreads / 32;
    constexpr int kAhead = 2;  // pieces of a warp that are loaded together
    constexpr int kVecs = BY_ROW ? D / 64 : D / 32;                            // float4 of a lane
    constexpr int kPatchRows = BY_ROW ? 2 : 8, kAcross = BY_ROW ? 1 : D / 16 / kVecs;  // patches across the dims
    __shared__ float4 meet[kWarps][kVecs][32];
    __shared__ float2 meet_ml[kWarps][kVecs][32];
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const int me = blockIdx.x, workers = gridDim.x, ways = gridDim.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const PagedCut* cuts = Part::cuts(a.workspace);
    // the item that this worker's stretch began with, and the one that it ended with
    const PagedCut old = cuts[me], begun = cuts[min(me + 1, workers - 1)];
    const bool begins = begun.rows > 0 && begun.first == me && me + 1 < workers;
    const int old_pieces = old.rows > 0 ? old.last - old.first + 1 : 0;
    const int begun_pieces = begins ? begun.last - begun.first + 1 : 0;
    // this block is number k of n for either, and takes the patches k, k + n, ...
    const int old_n = old_pieces * ways, old_k = (me - old.first) * ways + blockIdx.y;
    const int old_all = (old.rows + kPatchRows - 1) / kPatchRows * kAcross;
    const int begun_n = begun_pieces * ways, begun_k = blockIdx.y;
    const int begun_all = (begun.rows + kPatchRows - 1) / kPatchRows * kAcross;
    const int old_here = old_pieces > 0 && old_k < old_all ? (old_all - old_k + old_n - 1) / old_n : 0;
    const int here = old_here + (begins && begun_k < begun_all ? (begun_all - begun_k + begun_n - 1) / begun_n : 0);
    const int pieces = max(old_pieces, begun_pieces);
    for (int base = 0; base < here; base += kWarps) {
        const int count = min(kWarps, here - base), share = warp / count;
        const int shares = min(kWarps / count, (pieces + kAhead - 1) / kAhead);
        const int t = base + warp % count;
        const bool is_old = t < old_here;
        const PagedCut& cut = is_old ? old : begun;
        const int patch = is_old ? old_k + t * old_n : begun_k + (t - old_here) * begun_n;
        const int patch_r = patch / kAcross * kPatchRows, patch_v = patch % kAcross * 4 * kVecs;
        float m[kVecs], l[kVecs];
        float4 acc[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.F;
            acc[i] = make_float4(0.F, 0.F, 0.F, 0.F);
        }
        auto join = [&](int i, const float2& ml, const float4& x) {
            const float mn = fmaxf(m[i], ml.x);
            const float f = m[i] == -INFINITY ? 0.F : ex2(m[i] - mn), g = ml.x == -INFINITY ? 0.F : ex2(ml.x - mn);
            l[i] = l[i] * f + ml.y * g;
            acc[i].x = acc[i].x * f + x.x * g;
            acc[i].y = acc[i].y * f + x.y * g;
            acc[i].z = acc[i].z * f + x.z * g;
            acc[i].w = acc[i].w * f + x.w * g;
            m[i] = mn;
        };
        // a lane's i-th four dims of the patch
        auto row_of = [&](int i) { return patch_r + (BY_ROW ? (lane + 32 * i) / (D / 4) : lane & 7); };
        auto vec_of = [&](int i) { return BY_ROW ? (lane + 32 * i) % (D / 4) : patch_v + (lane >> 3) + 4 * i; };
        if (share < shares) {
            for (int c0 = cut.first + share; c0 <= cut.last; c0 += kAhead * shares) {
                float2 ml[kAhead][kVecs];
                float4 x[kAhead][kVecs];
                bool there[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int c = c0 + u * shares;
                    there[u] = c <= cut.last;
                    if (!there[u]) continue;
                    // (read whether the worker left a piece or not: one round trip for everything)
                    const float* part = Part::slot(a.workspace, workers, c, c == cut.first ? 1 : 0);
                    there[u] = c == cut.first || cuts[c].piece;
#pragma unroll
                    for (int i = 0; i < kVecs; ++i) {
                        ml[u][i] = __ldcg(reinterpret_cast<const float2*>(part) + row_of(i));
                        x[u][i] = __ldcg(reinterpret_cast<const float4*>(part + 2 * ROWS) +
                                         (BY_ROW ? row_of(i) * (D / 4) + vec_of(i) : vec_of(i) * ROWS + row_of(i)));
                    }
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (!there[u]) continue;
#pragma unroll
                    for (int i = 0; i < kVecs; ++i) join(i, ml[u][i], x[u][i]);
                }
            }
        }
        if (shares > 1) {  // (in the last round only)
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                meet[warp][i][lane] = acc[i];
                meet_ml[warp][i][lane] = make_float2(m[i], l[i]);
            }
            __syncthreads();
        }
        if (share != 0) continue;
        for (int k = 1; k < shares; ++k)
#pragma unroll
            for (int i = 0; i < kVecs; ++i) join(i, meet_ml[warp + k * count][i][lane], meet[warp + k * count][i][lane]);
        const PagedBatch& p = a.p;
        const int group = p.q_heads / p.kv_heads;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int r = row_of(i), v = vec_of(i);
            if (r >= cut.rows) continue;
            const int64_t row = cut.row0 + (cut.r0 + r) / group;
            const int head = cut.kvh * group + (cut.r0 + r) % group;
            const float inv = l[i] == 0.F ? 0.F : 1.F / l[i];
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + row * a.out_stride + static_cast<int64_t>(head) * D +
                                      4 * v) =
                make_uint2(pack2<DT>(acc[i].x * inv, acc[i].y * inv), pack2<DT>(acc[i].z * inv, acc[i].w * inv));
            if (v == 0 && a.lse != nullptr)
                a.lse[row * p.q_heads + head] = l[i] == 0.F ? -INFINITY : m[i] * kLn2 + logf(l[i]);
        }
    }
}

}  // namespace kc

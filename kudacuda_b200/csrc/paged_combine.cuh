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
// O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in the order of the pieces
// (the same bits on every run).  One block per worker that began a cut item
// and 32 of the item's rows: lane = row, warp = a share of the dims.
template <int DT, int D, int ROWS>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedAttentionArgs a, int workers) {
    using Part = PagedPartial<ROWS, D>;
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const int owner = blockIdx.x;
    const PagedCut* cuts = Part::cuts(a.workspace);
    const PagedCut cut = cuts[owner];
    constexpr int kLanes = 32, kShares = 256 / kLanes;
    const int lane = threadIdx.x % kLanes, share = threadIdx.x / kLanes;
    const int r = blockIdx.y * kLanes + lane;
    if (!cut.valid || r >= cut.rows) return;
    constexpr int kVecs = (D / 4 + kShares - 1) / kShares;  // float4 of a thread
    constexpr int kAhead = 2;  // pieces whose loads are in flight together: an item is rarely cut twice
    float m = -INFINITY, l = 0.F;
    float4 acc[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) acc[i] = make_float4(0.F, 0.F, 0.F, 0.F);
    const int last = min(cut.last, workers - 1);
    for (int c0 = owner; c0 <= last; c0 += kAhead) {
        float2 ml[kAhead];
        float4 x[kAhead][kVecs];
        bool there[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int c = min(c0 + u, last);
            there[u] = c0 + u <= last && (c == owner || cuts[c].tail);
            // (read whether it is there or not: one round trip for everything)
            const float* part = Part::slot(a.workspace, workers, c, c == owner ? 1 : 0);
            ml[u] = __ldcg(reinterpret_cast<const float2*>(part) + r);
            const float4* o = reinterpret_cast<const float4*>(part + 2 * ROWS);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) x[u][i] = __ldcg(o + min(share + i * kShares, D / 4 - 1) * ROWS + r);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (!there[u]) continue;
            const float mn = fmaxf(m, ml[u].x);
            const float f = m == -INFINITY ? 0.F : exp2f(m - mn), g = ml[u].x == -INFINITY ? 0.F : exp2f(ml[u].x - mn);
            l = l * f + ml[u].y * g;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                acc[i].x = acc[i].x * f + x[u][i].x * g;
                acc[i].y = acc[i].y * f + x[u][i].y * g;
                acc[i].z = acc[i].z * f + x[u][i].z * g;
                acc[i].w = acc[i].w * f + x[u][i].w * g;
            }
            m = mn;
        }
    }
    const PagedBatch& p = a.p;
    const int group = p.q_heads / p.kv_heads;
    const int64_t row = cut.row0 + (cut.r0 + r) / group;
    const int head = cut.kvh * group + (cut.r0 + r) % group;
    const float inv = l == 0.F ? 0.F : 1.F / l;
    uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.out_stride + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int v = share + i * kShares;
        if (v >= D / 4) break;
        *reinterpret_cast<uint2*>(out + 4 * v) = make_uint2(pack2<DT>(acc[i].x * inv, acc[i].y * inv),
                                                            pack2<DT>(acc[i].z * inv, acc[i].w * inv));
    }
    if (share == 0 && a.lse != nullptr) a.lse[row * p.q_heads + head] = l == 0.F ? -INFINITY : m * kLn2 + logf(l);
}

}  // namespace kc

// paged_attention.cu -- attention of a ragged batch of new tokens over a paged
// KV cache.
//
// Row r (token i of its sequence, position pos) and query head h:
//   S_j = scale q . k_j for keys j <= pos, P = softmax(S), O = P V,
//   lse = log sum_j exp(S_j);  a row without keys has O = 0, lse = -inf.
#include "kc_common.cuh"
#include "kc_launch.h"

namespace kc {
namespace {

constexpr float kLn2 = 0.6931471805599453F;
constexpr float kLog2E = 1.4426950408889634F;

// One warp per (row, head): the keys one after the other, a running maximum
// and sum in 32 bits.
template <int DT>
__global__ void __launch_bounds__(128) paged_attention_rows_kernel(const PagedAttentionArgs a) {
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const PagedBatch& p = a.p;
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int row = static_cast<int>(w / p.q_heads), head = static_cast<int>(w - static_cast<int64_t>(row) * p.q_heads);
    if (row >= p.rows) return;
    int seq = 0;
    for (int j = 0; j < p.batch; j += 32) {
        const int k = j + lane;
        const int end = k < p.batch ? p.query_start[k + 1] : 0x7fffffff;
        seq += __popc(__ballot_sync(0xffffffffu, end <= row));
    }
    if (seq >= p.batch || row < p.query_start[seq]) return;
    const int pos = p.kv_len[seq] - (p.query_start[seq + 1] - row);
    const int kvh = head / (p.q_heads / p.kv_heads);
    const int per = p.head_dim >> 5;  // dims a lane: 2 or 4, dim = i * 32 + lane
    float q[4], acc[4] = {0.F, 0.F, 0.F, 0.F};
    const int64_t qo = static_cast<int64_t>(row) * a.q_stride + static_cast<int64_t>(head) * p.head_dim;
    for (int i = 0; i < 4; ++i) q[i] = i < per ? load_elem<DT>(a.q, qo + i * 32 + lane) * (a.scale * kLog2E) : 0.F;
    float m = -INFINITY, l = 0.F;
    for (int j = 0; j <= pos; ++j) {
        const int n = j / p.page_size;
        const int page = n < p.table_width ? p.table[seq * p.table_stride + n] : -1;
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0 && p.err != nullptr) atomicOr(p.err, 2);
            break;
        }
        const int64_t ko = ((static_cast<int64_t>(page) * p.kv_heads + kvh) * p.page_size + j % p.page_size) * p.head_dim;
        float dot = 0.F;
        for (int i = 0; i < per; ++i) dot += q[i] * load_elem<DT>(a.k_pages, ko + i * 32 + lane);
        dot = warp_sum(dot);
        const float mn = fmaxf(m, dot);
        const float scale = mn == -INFINITY ? 1.F : exp2f(m - mn), e = mn == -INFINITY ? 0.F : exp2f(dot - mn);
        l = l * scale + e;
        for (int i = 0; i < per; ++i) acc[i] = acc[i] * scale + e * load_elem<DT>(a.v_pages, ko + i * 32 + lane);
        m = mn;
    }
    const float inv = l > 0.F ? 1.F / l : 0.F;
    const int64_t oo = static_cast<int64_t>(row) * a.out_stride + static_cast<int64_t>(head) * p.head_dim;
    for (int i = 0; i < per; ++i) store_elem<DT>(a.out, oo + i * 32 + lane, acc[i] * inv);
    if (a.lse != nullptr && lane == 0)
        a.lse[static_cast<int64_t>(row) * p.q_heads + head] = l > 0.F ? m * kLn2 + logf(l) : -INFINITY;
}

}  // namespace

int64_t paged_attention_workspace_bytes(int64_t batch, int64_t rows, int64_t max_query, int64_t q_heads,
                                        int64_t kv_heads, int64_t head_dim, int64_t max_kv) {
    return paged_chunk_workspace_bytes(static_cast<int>(head_dim));
}

cudaError_t paged_attention(const PagedAttentionArgs& a, int dt, cudaStream_t s) {
    if (a.p.rows == 0 || a.p.batch == 0) return cudaSuccess;
    return paged_chunk(a, dt, s);
}

}  // namespace kc

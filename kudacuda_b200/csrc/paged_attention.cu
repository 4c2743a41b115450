// paged_attention.cu -- attention of a ragged batch of new tokens over a paged
// KV cache.
//
// Row r (token i of its sequence, position pos) and query head h:
//   S_j = scale q . k_j for keys j <= pos, P = softmax(S), O = P V,
//   lse = log sum_j exp(S_j);  a row without keys has O = 0, lse = -inf.
//
// Two kernels share the work out alike (paged_plan.cuh): paged_decode.cu for few
// query rows a key head, bound by reading the cache; paged_chunk.cu for many,
// bound by the tensor cores.
#include "kc_common.cuh"
#include "kc_launch.h"

namespace kc {

// Query rows a key head (of the longest sequence) up to which the decode kernel
// serves: its tile, for a second one it reads the cache again.  It also keeps the
// probabilities to twice the type's precision, where the chunk kernel rounds them to
// the type: against 64 bits the relative error is 0.0022 (24 mixed sequences) and
// 0.0023 (4 x 2048 tokens over 8192 keys) where the output's rounding alone makes
// 0.0017.  max_query is the caller's, who may name a smaller one to have the decode
// kernel.  Decode and chunk kernel, us, 4
// key heads of 128 bf16 dims, 1 token of 8 heads / 2 / 3:
//   64 sequences of 500 keys    25.5, 26.2 / 28.4, 26.4 / 41.6, 26.5
//   16 of 2000                  22.9, 23.3 / 24.6, 23.4 / 32.8, 23.5
//   1 of 8000                   15.0, 17.2 / 15.8, 17.5 / 19.6, 17.7
//   2 of 100000                 74.5, 77.5 / 76.3, 78.2 / 136, 78.4
// (two tokens of eight heads are 16 rows: 5 to 8% lost on short caches, 3 to 10%
// won on long ones, and the probabilities)
constexpr int64_t kDecodeRows = 16;

int64_t paged_attention_workspace_bytes(int64_t batch, int64_t rows, int64_t max_query, int64_t q_heads,
                                        int64_t kv_heads, int64_t head_dim, int64_t max_kv) {
    return max_query * (q_heads / kv_heads) <= kDecodeRows ? paged_decode_workspace_bytes(static_cast<int>(head_dim))
                                                           : paged_chunk_workspace_bytes(static_cast<int>(head_dim));
}

cudaError_t paged_attention(const PagedAttentionArgs& a, int dt, cudaStream_t s) {
    if (a.p.rows == 0 || a.p.batch == 0) return cudaSuccess;
    const int64_t rows = static_cast<int64_t>(a.max_query) * (a.p.q_heads / a.p.kv_heads);
    return rows <= kDecodeRows ? paged_decode(a, dt, s) : paged_chunk(a, dt, s);
}

}  // namespace kc

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
// probabilities to twice the type's precision.  Decode and chunk kernel, us, 4
// key heads of 128 bf16 dims, 1 token of 8 heads / 2 / 3:
//   64 sequences of 500 keys    25.8, 27.6 / 28.8, 27.9 / 42.4, 28.2
//   16 of 2000                  22.9, 23.9 / 24.8, 24.1 / 32.7, 24.5
//   1 of 8000                   15.1, 17.8 / 15.8, 18.0 / 19.7, 18.4
//   2 of 100000                 74.4, 79.8 / 75.9, 80.5 / 135, 81.1
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

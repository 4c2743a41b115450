// paged.cu -- the paged KV cache's writers: rotary positions fused with the
// append of a ragged batch's new keys and values into their pages, and the
// copies that fork and compact a cache.
//
// The reference appends through Transformers' cache classes, one contiguous
// cache per sequence (python/kudacuda_static_decode.py:147-153); it has no
// pages.
#include "kc_common.cuh"
#include "kc_launch.h"

namespace kc {
namespace {

// 16 bytes = 8 elements of a 16-bit type, in 32 bits
template <int DT>
__device__ __forceinline__ void unpack8(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kBF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kBF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------------------
// rope_append_paged: y0 = x0 c - x1 s, y1 = x1 c + x0 s over the first
// rotary_dim dims of every q and k head, in 32 bits, one rounding to the
// cache's type; v and the dims past rotary_dim pass through.
//
// A warp owns one token: its lanes split a head into units of 16 elements
// (two 16-byte words: eight pairs of a rotated unit, or 16 elements that pass
// through), 32 / (head_dim / 16) heads abreast, and walk `iters` such groups
// of heads with the unit's eight cos and sin in registers, all their loads in flight
// at once.  Bound by memory: 8192 rows of 32 + 16 heads, every element read and
// written once, 5.6 TB/s; few rows by the chain of loads from the lengths to
// the page number (64 rows of 16 + 4 heads: 3 us).
constexpr int kRopeThreads = 128;
// Warps from which four groups of heads share one: 32 + 16 heads of 128 dims, four
// against one: 16 rows 3.3 and 2.7 us, 256 rows 3.8 and 3.8, 1024 6.2 and 7.2,
// 8192 34.8 and 45.0.
constexpr int64_t kRopeWarps = 4096;

template <int DT, int ITERS>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeAppendArgs a, int groups) {
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const PagedBatch& p = a.p;
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int row = static_cast<int>(w / groups), group = static_cast<int>(w - static_cast<int64_t>(row) * groups);
    if (row >= p.rows) return;
    // the sequence of the row: how many sequences end at or before it
    int seq = 0;
    for (int j = 0; j < p.batch; j += 32) {
        const int k = j + lane;
        const int end = k < p.batch ? p.query_start[k + 1] : 0x7fffffff;
        seq += __popc(__ballot_sync(0xffffffffu, end <= row));
    }
    if (seq >= p.batch) return;  // a row of no sequence
    const int start = p.query_start[seq], end = p.query_start[seq + 1];
    const int pos = p.kv_len[seq] - (end - row);
    int page = -1;
    if (row >= start && pos >= 0 && (a.rotary_dim == 0 || pos < a.max_pos) && pos / p.page_size < p.table_width)
        page = p.table[seq * p.table_stride + pos / p.page_size];
    if (page < 0 || page >= p.num_pages) {
        if (lane == 0 && p.err != nullptr) atomicOr(p.err, 2);
        return;
    }
    const int units = p.head_dim >> 4, abreast = 32 / units;
    const int u = lane % units, hslot = lane / units;
    const int half = a.rotary_dim >> 1;
    const bool turned = u < (a.rotary_dim >> 4);
    // element offsets in the head of the unit's two words
    int o0 = 16 * u, o1 = o0 + 8;
    if (turned && !a.interleaved) {
        o0 = 8 * u;
        o1 = half + 8 * u;
    }
    float c[8], s[8];
    if (turned) {
        const float4* cp = reinterpret_cast<const float4*>(a.cos + static_cast<int64_t>(pos) * half + 8 * u);
        const float4* sp = reinterpret_cast<const float4*>(a.sin + static_cast<int64_t>(pos) * half + 8 * u);
        *reinterpret_cast<float4*>(c) = cp[0];
        *reinterpret_cast<float4*>(c + 4) = cp[1];
        *reinterpret_cast<float4*>(s) = sp[0];
        *reinterpret_cast<float4*>(s + 4) = sp[1];
    }
    const uint16_t* in = static_cast<const uint16_t*>(a.qkv) + static_cast<int64_t>(row) * a.qkv_stride;
    const int heads = p.q_heads + 2 * p.kv_heads;
    const int64_t slot = static_cast<int64_t>(pos & (p.page_size - 1)) * p.head_dim;
    const int64_t head_elems = static_cast<int64_t>(p.page_size) * p.head_dim;
    uint4 in0[ITERS], in1[ITERS];
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int h = (group * ITERS + it) * abreast + hslot;
        if (h >= heads) break;
        in0[it] = __ldcs(reinterpret_cast<const uint4*>(in + h * p.head_dim + o0));
        in1[it] = __ldcs(reinterpret_cast<const uint4*>(in + h * p.head_dim + o1));
    }
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int h = (group * ITERS + it) * abreast + hslot;
        if (h >= heads) break;
        const int64_t off = static_cast<int64_t>(h) * p.head_dim;
        uint4 v0 = in0[it], v1 = in1[it];
        const bool rotate = turned && h < p.q_heads + p.kv_heads;
        if (rotate || a.bias != nullptr) {
            float x[16];
            unpack8<DT>(v0, x);
            unpack8<DT>(v1, x + 8);
            if (a.bias != nullptr) {  // the projection's own output: rounded once after its bias
                const uint16_t* bp = static_cast<const uint16_t*>(a.bias) + off;
                float t[16];
                unpack8<DT>(*reinterpret_cast<const uint4*>(bp + o0), t);
                unpack8<DT>(*reinterpret_cast<const uint4*>(bp + o1), t + 8);
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] += t[i];
                v0 = pack8<DT>(x);
                v1 = pack8<DT>(x + 8);
                unpack8<DT>(v0, x);
                unpack8<DT>(v1, x + 8);
            }
            if (rotate) {
                if (a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x0 = x[2 * i], x1 = x[2 * i + 1];
                        x[2 * i] = x0 * c[i] - x1 * s[i];
                        x[2 * i + 1] = x1 * c[i] + x0 * s[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x0 = x[i], x1 = x[8 + i];
                        x[i] = x0 * c[i] - x1 * s[i];
                        x[8 + i] = x1 * c[i] + x0 * s[i];
                    }
                }
                v0 = pack8<DT>(x);
                v1 = pack8<DT>(x + 8);
            }
        }
        uint16_t* out;
        if (h < p.q_heads) {
            out = static_cast<uint16_t*>(a.q_out) + static_cast<int64_t>(row) * a.q_stride + off;
        } else {
            const int kv = h - p.q_heads;
            const bool isk = kv < p.kv_heads;
            out = static_cast<uint16_t*>(isk ? a.k_pages : a.v_pages) +
                  (static_cast<int64_t>(page) * p.kv_heads + (isk ? kv : kv - p.kv_heads)) * head_elems + slot;
        }
        *reinterpret_cast<uint4*>(out + o0) = v0;
        *reinterpret_cast<uint4*>(out + o1) = v1;
    }
}

// ---------------------------------------------------------------------------
// kv_pages_copy: page from -> page to for every pair, K and V, every layer;
// then every entry of the block tables through page_map.  No page is both a
// source and a target of one call, so the order of the copies is free.  Bound by
// memory: 300 pages of 32 layers, 1.26 GB read and written, 190 us, 6.6 TB/s.
// Four words in flight a thread: the blocks resident on an SM then have 128 KB
// on their way.
constexpr int kCopyThreads = 256;
constexpr int kCopyWords = 4;  // 16-byte words a thread

__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const PagesCopyArgs a, int chunks,
                                                                  int64_t copy_blocks) {
    pdl_launch_dependents();
    pdl_wait_on_producer();
    int64_t blk = blockIdx.x;
    if (blk >= copy_blocks) {  // the tables
        const int64_t i = (blk - copy_blocks) * kCopyThreads + threadIdx.x;
        if (i < static_cast<int64_t>(a.table_rows) * a.table_width) {
            const int64_t r = i / a.table_width;
            int32_t* e = a.table + r * a.table_stride + (i - r * a.table_width);
            const int32_t page = *e;
            if (page >= 0 && page < a.num_pages) *e = a.page_map[page];
        }
        return;
    }
    const int chunk = static_cast<int>(blk % chunks);
    blk /= chunks;
    const int pair = static_cast<int>(blk % a.count);
    blk /= a.count;
    const int layer = static_cast<int>(blk >> 1);
    const int from = a.pairs[2 * pair], to = a.pairs[2 * pair + 1];
    if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages) {
        if (threadIdx.x == 0 && a.err != nullptr) atomicOr(a.err, 2);
        return;
    }
    char* base = static_cast<char*>((blk & 1) ? a.v_pages : a.k_pages) + layer * a.layer_stride;
    const uint4* src = reinterpret_cast<const uint4*>(base + from * a.page_bytes);
    uint4* dst = reinterpret_cast<uint4*>(base + to * a.page_bytes);
    const int64_t words = a.page_bytes >> 4;
    const int64_t w0 = static_cast<int64_t>(chunk) * kCopyThreads * kCopyWords + threadIdx.x;
    uint4 v[kCopyWords];
#pragma unroll
    for (int i = 0; i < kCopyWords; ++i)
        if (w0 + i * kCopyThreads < words) v[i] = __ldcs(src + w0 + i * kCopyThreads);
#pragma unroll
    for (int i = 0; i < kCopyWords; ++i)
        if (w0 + i * kCopyThreads < words) __stcs(dst + w0 + i * kCopyThreads, v[i]);
}

}  // namespace

cudaError_t rope_append_paged(const RopeAppendArgs& a, int dt, cudaStream_t s) {
    if (a.p.rows == 0 || a.p.batch == 0) return cudaSuccess;
    const int abreast = 32 / (a.p.head_dim / 16);
    const int need = (a.p.q_heads + 2 * a.p.kv_heads + abreast - 1) / abreast;
    // many rows: four groups of heads a warp share the table's row and the lookup;
    // few: a warp for every group, for the shortest chain
    const int iters = static_cast<int64_t>(a.p.rows) * need >= kRopeWarps ? 4 : 1;
    const int groups = (need + iters - 1) / iters;
    const int64_t warps = static_cast<int64_t>(a.p.rows) * groups;
    const int64_t blocks = (warps + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    auto kernel = dt == kBF16 ? (iters == 4 ? rope_append_kernel<kBF16, 4> : rope_append_kernel<kBF16, 1>)
                              : (iters == 4 ? rope_append_kernel<kF16, 4> : rope_append_kernel<kF16, 1>);
    return launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kRopeThreads), 0, s, a, groups);
}

cudaError_t kv_pages_copy(const PagesCopyArgs& a, cudaStream_t s) {
    const int64_t words = a.page_bytes >> 4;
    const int64_t chunks = (words + kCopyThreads * kCopyWords - 1) / (kCopyThreads * kCopyWords);
    const int64_t copy_blocks = chunks * a.count * a.layers * 2;
    const int64_t entries = a.table != nullptr ? static_cast<int64_t>(a.table_rows) * a.table_width : 0;
    const int64_t blocks = copy_blocks + (entries + kCopyThreads - 1) / kCopyThreads;
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_pdl(pages_copy_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kCopyThreads), 0, s, a,
                      static_cast<int>(chunks), copy_blocks);
}

}  // namespace kc

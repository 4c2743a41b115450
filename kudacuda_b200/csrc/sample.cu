// sample.cu -- the next token of every row from its logits: temperature,
// top-k, top-p, min-p and one given uniform number.
//
// With x the logits in 32 bits (NaN counts as -inf) and m their maximum:
//   w_i = 1 where x_i == m, else exp((x_i - m) * (1 / T));  W_i = rint(2^38 w_i)
// (an infinite T: w_i = 1 for every finite x_i, 0 for -inf).
// The masses W are whole numbers, so every sum below is exact and does not
// depend on the order in which threads or blocks add: the same row gives the
// same token whatever shares its batch.  In the order of (x descending, index
// ascending): top-k keeps the first k (mass K), top-p the shortest prefix of
// those whose mass reaches ceil(p K), min-p the entries with w >= min_p.  The
// token is the first kept index whose inclusive kept mass exceeds
// floor(u M), M the kept mass.  T <= 0 is the lowest index of the maximum; a
// row without any entry above -inf gives token -1 and log-probability -inf.
#include <type_traits>

#include "kc_common.cuh"
#include "kc_launch.h"

namespace kc {
namespace {

constexpr float kMassOne = 274877906944.F;  // 2^38: sums of 2^24 entries stay below 2^62

__device__ __forceinline__ uint32_t ordered_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
template <int DT>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
    const float x = load_elem<DT>(p, i) + 0.F;  // -0 and +0 are one value
    return x != x ? -INFINITY : x;
}

// 1 / T, never 0: for an infinite T the smallest 32-bit number stands for it, by
// which x - m of a -inf stays -inf (weight 0), where 0 would make it NaN.
__device__ __forceinline__ float inverse_temperature(float t) { return fmaxf(1.F / t, 1.4e-45F); }

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, F f, T* buf) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    v = buf[0];
    for (int i = 1; i < static_cast<int>(blockDim.x >> 5); ++i) v = f(v, buf[i]);
    return v;
}

template <int DT>
__global__ void __launch_bounds__(1024) sample_rows_kernel(const SampleArgs a) {
    __shared__ int64_t buf[32];
    __shared__ int64_t warp_mass[32];
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const int row = blockIdx.x, tid = threadIdx.x, n = a.vocab;
    const int64_t base = row * a.row_stride;
    auto add = [](int64_t x, int64_t y) { return x + y; };
    auto least = [](int64_t x, int64_t y) { return x < y ? x : y; };
    float best = -INFINITY;
    for (int i = tid; i < n; i += 1024) best = fmaxf(best, load_logit<DT>(a.logits, base + i));
    const float m = block_reduce(best, [](float x, float y) { return fmaxf(x, y); }, reinterpret_cast<float*>(buf));
    if (m == -INFINITY) {
        if (tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
        }
        return;
    }
    const float t = a.temperature != nullptr ? a.temperature[row] : 1.F;
    if (!(t > 0.F)) {
        int64_t first = n;
        for (int i = tid; i < n; i += 1024)
            if (load_logit<DT>(a.logits, base + i) == m) first = least(first, i);
        first = block_reduce(first, least, buf);
        if (tid == 0) {
            a.tokens[row] = static_cast<int32_t>(first);
            if (a.logprobs != nullptr) a.logprobs[row] = 0.F;
        }
        return;
    }
    const float inv = inverse_temperature(t);
    const float full = t == INFINITY && m < INFINITY ? -3.402823466e38F : m;  // from here on the weight is 1
    auto weight = [&](float x) { return x >= full ? 1.F : expf((x - m) * inv); };
    auto mass = [&](float x) { return __float2ll_rn(weight(x) * kMassOne); };
    // kept: key > cut, or key == cut and index < tie_end
    uint32_t cut = 0;
    int64_t tie_end = n;
    const int k = a.top_k != nullptr ? a.top_k[row] : 0;
    const float p = a.top_p != nullptr ? a.top_p[row] : 1.F;
    // the index after the `count`-th entry with this key
    auto nth_tie = [&](uint32_t key, int64_t count) {
        int64_t lo = 0, hi = n;  // smallest e with #(key, index < e) >= count
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            int64_t c = 0;
            for (int64_t i = tid; i < mid; i += 1024) c += ordered_key(load_logit<DT>(a.logits, base + i)) == key;
            if (block_reduce(c, add, buf) >= count) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    };
    if (k > 0 && k < n) {
        uint32_t lo = 0, hi = 0xffffffffu;  // largest key with at least k entries at or above
        while (lo < hi) {
            const uint32_t mid = lo + ((hi - lo) >> 1) + 1;
            int64_t c = 0;
            for (int i = tid; i < n; i += 1024) c += ordered_key(load_logit<DT>(a.logits, base + i)) >= mid;
            if (block_reduce(c, add, buf) >= k) lo = mid;
            else hi = mid - 1;
        }
        int64_t above = 0;
        for (int i = tid; i < n; i += 1024) above += ordered_key(load_logit<DT>(a.logits, base + i)) > lo;
        above = block_reduce(above, add, buf);
        cut = lo;
        tie_end = nth_tie(lo, k - above);
    }
    auto in = [&](uint32_t key, int64_t i) { return key > cut || (key == cut && i < tie_end); };
    if (p < 1.F) {
        int64_t sum = 0;
        for (int i = tid; i < n; i += 1024) {
            const float x = load_logit<DT>(a.logits, base + i);
            if (in(ordered_key(x), i)) sum += mass(x);
        }
        const int64_t total = block_reduce(sum, add, buf);
        int64_t reach = __double2ll_ru(__dmul_rn(static_cast<double>(p), __ll2double_rn(total)));
        reach = reach < 1 ? 1 : reach;
        // largest key with kept mass at or above it >= reach
        uint32_t lo = cut, hi = 0xffffffffu;
        while (lo < hi) {
            const uint32_t mid = lo + ((hi - lo) >> 1) + 1;
            int64_t c = 0;
            for (int i = tid; i < n; i += 1024) {
                const float x = load_logit<DT>(a.logits, base + i);
                const uint32_t key = ordered_key(x);
                if (key >= mid && in(key, i)) c += mass(x);
            }
            if (block_reduce(c, add, buf) >= reach) lo = mid;
            else hi = mid - 1;
        }
        int64_t above = 0, each = 0;
        for (int i = tid; i < n; i += 1024) {
            const float x = load_logit<DT>(a.logits, base + i);
            const uint32_t key = ordered_key(x);
            if (key > lo && in(key, i)) above += mass(x);
            if (key == lo) each = mass(x);
        }
        above = block_reduce(above, add, buf);
        each = block_reduce(each, [](int64_t x, int64_t y) { return x > y ? x : y; }, buf);
        const int64_t end = each > 0 ? nth_tie(lo, (reach - above + each - 1) / each) : n;
        if (lo > cut) tie_end = end;
        else tie_end = end < tie_end ? end : tie_end;
        cut = lo;
    }
    float low = a.min_p != nullptr ? a.min_p[row] : 0.F;
    low = low > 1.F ? 1.F : low;
    // each thread's share is a run of indexes: the draw goes by the order of index
    const int per = (n + 1023) / 1024;
    const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int64_t mine = 0;
    for (int i = i0; i < i1; ++i) {
        const float x = load_logit<DT>(a.logits, base + i);
        if (in(ordered_key(x), i) && !(weight(x) < low)) mine += mass(x);
    }
    const int lane = tid & 31, warp = tid >> 5;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_mass[warp] = upto;
    __syncthreads();
    int64_t before = 0, whole = 0;
    for (int i = 0; i < 32; ++i) {
        if (i < warp) before += warp_mass[i];
        whole += warp_mass[i];
    }
    upto += before;
    int64_t aim = __double2ll_rd(__dmul_rn(static_cast<double>(a.uniform[row]), __ll2double_rn(whole)));
    aim = aim < 0 ? 0 : aim >= whole ? whole - 1 : aim;
    if (upto - mine <= aim && aim < upto) {
        int64_t c = upto - mine;
        for (int i = i0; i < i1; ++i) {
            const float x = load_logit<DT>(a.logits, base + i);
            if (!in(ordered_key(x), i) || weight(x) < low) continue;
            const int64_t w = mass(x);
            c += w;
            if (c > aim) {
                a.tokens[row] = i;
                if (a.logprobs != nullptr)
                    a.logprobs[row] = static_cast<float>(log(__ll2double_rn(w) / __ll2double_rn(whole)));
                break;
            }
        }
    }
}


// ---------------------------------------------------------------------------
// The row held in the shared memory of a thread-block cluster.
//
// The logits become ordered keys (whole numbers in the order of the values,
// 16 bits wide for the 16-bit types), read from memory once.  What remains is
// to find the key at which the kept prefix ends: kPivots keys that split the
// range still possible are tried at once - each thread counts the entries at or
// above each of them, and sums their masses, in registers - and the cluster
// exchanges the sums through distributed shared memory with one barrier.  When
// at most kList entries are left, every block gets all of their keys and
// finishes alone; when at most kBins keys are left (16-bit types), the entries of
// each are counted.  Both use atomics only where their order does not show: for
// places in a list that is only summed over, and for whole numbers.
//
// The logits are read once, so memory asks 3 us of 64 rows of 151 936 16-bit
// logits and 10 us of 333 rows of 50 257 32-bit ones.  What they do cost, rows of
// all kinds mixed, is 41 to 75 and 90 to 103 us, depending on the rows (means of 16
// draws 51 and 95): instructions
// in the first try and in the pass in index order (an exponential and two roundings
// an entry, three additions more for every key tried), and waits: a row goes
// through six or so barriers of its cluster, 1 to 2 us each with what lies between,
// and the slowest row holds up the rest (64 rows, all of one kind: greedy 10 us,
// min-p 14, temperature alone 23, top-k 29, both limits 34, top-p 64).  One row
// takes 16 us in 16 blocks.
constexpr int kPivots = 5;
constexpr float kFirst = 2.5F;
constexpr int kMaxCluster = 16;  // more than 8 need the kernel's consent (launch_cluster)
constexpr int kMaxSampleThreads = 512;
constexpr int kList = 1024;
constexpr int kBins = 512;  // (256: 64 rows 53.4 us for 52.3, mean of eight seeds)
static_assert(2 * kBins <= kList && kBins % kMaxCluster == 0);

template <int DT>
struct Keys {
    using Key = uint16_t;
    using Raw = uint16_t;
    static constexpr int kVec = 8;  // entries of a 16-byte word
    static __device__ __forceinline__ uint32_t key(Raw raw) {
        const bool nan = (raw & 0x7fffu) > (DT == kBF16 ? 0x7f80u : 0x7c00u);
        const uint32_t b = nan ? (DT == kBF16 ? 0xff80u : 0xfc00u) : (raw & 0x7fffu) == 0 ? 0u : raw;
        return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        const uint16_t b = static_cast<uint16_t>((k & 0x8000u) ? (k & 0x7fffu) : ~k);
        return DT == kBF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
    }
    // the largest of a word's eight
    static __device__ __forceinline__ uint32_t largest(const Key* k) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(k);
        const uint32_t m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
        return max(m & 0xffffu, m >> 16);
    }
    // a word's eight keys; at: the largest so far of either half
    static __device__ __forceinline__ uint4 pack(const uint4& in, uint32_t& at) {
        constexpr uint32_t kNan = DT == kBF16 ? 0x007f007fu : 0x03ff03ffu;  // carries a NaN's magnitude into bit 15
        const uint32_t w[4] = {in.x, in.y, in.z, in.w};
        uint32_t k[4], odd = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t size = w[i] & 0x7fff7fffu, sign = (w[i] >> 15) & 0x00010001u;
            odd |= (size + kNan) | (w[i] & ~(size + 0x7fff7fffu));  // bit 15: a NaN, or -0
            k[i] = w[i] ^ (sign * 0xffffu | 0x80008000u);
        }
        if (odd & 0x80008000u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) k[i] = key(w[i] & 0xffffu) | key(w[i] >> 16) << 16;
        }
        at = __vmaxu2(at, __vmaxu2(__vmaxu2(k[0], k[1]), __vmaxu2(k[2], k[3])));
        return make_uint4(k[0], k[1], k[2], k[3]);
    }
    static __device__ __forceinline__ uint32_t top(uint32_t at) { return max(at & 0xffffu, at >> 16); }
    static __device__ __forceinline__ uint32_t near(float x) {
        return key(DT == kBF16 ? f32_to_bf16_bits(x) : f32_to_f16_bits(x));
    }
};
template <>
struct Keys<kF32> {
    using Key = uint32_t;
    using Raw = uint32_t;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ uint32_t key(Raw raw) {
        const uint32_t b = (raw & 0x7fffffffu) > 0x7f800000u ? 0xff800000u : (raw & 0x7fffffffu) == 0 ? 0u : raw;
        return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    }
    static __device__ __forceinline__ float value(uint32_t k) {
        return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
    }
    static __device__ __forceinline__ uint32_t largest(const Key* k) { return max(max(k[0], k[1]), max(k[2], k[3])); }
    static __device__ __forceinline__ uint4 pack(const uint4& in, uint32_t& at) {
        const uint4 k = make_uint4(key(in.x), key(in.y), key(in.z), key(in.w));
        at = max(at, max(max(k.x, k.y), max(k.z, k.w)));
        return k;
    }
    static __device__ __forceinline__ uint32_t top(uint32_t at) { return at; }
    static __device__ __forceinline__ uint32_t near(float x) { return key(__float_as_uint(x)); }
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void store_remote(const int64_t* p, uint32_t rank, int64_t v) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

__device__ __forceinline__ void store_remote32(const uint32_t* p, uint32_t rank, uint32_t v) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

constexpr int kSums = 2 * kPivots + 1;  // masses, their total, numbers
struct SampleShared {
    int64_t warp[kSums][32];
    int64_t from[2][kSums][kMaxCluster];  // what each block of the cluster sent, alternating halves
    // the search, kept by warp 0
    uint32_t pv[kPivots], lo, hi;
    int64_t above, target;
    int at_hi;           // entries at or above hi
    int listed, start;   // entries of the list that is made next, or -1; where this block's go in it
    int everything;      // 1: it holds all entries at or above lo, 0: those below hi
    int counted;         // 1: so few keys are left that each is counted
    int own_count;
    uint32_t list[kList];
    // this block's share of the list, then the list's masses; in the end every thread's mass
    union {
        uint32_t own[kList];
        int64_t mass[kList];
    };
};
static_assert(kMaxSampleThreads <= kList);

__device__ __forceinline__ int64_t warp_sum64(int64_t x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// inclusive prefix over the lanes
__device__ __forceinline__ int64_t warp_scan64(int64_t x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (static_cast<int>(threadIdx.x & 31) >= o) x += y;
    }
    return x;
}
// the warp's sum of a value in [0, 2^48), as two sums of 24-bit halves
__device__ __forceinline__ int64_t warp_sum48(int64_t x) {
    const uint32_t lo = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x) & 0xffffffu);
    const uint32_t hi = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x >> 24));
    return (static_cast<int64_t>(hi) << 24) + lo;
}
// Lane i of warp 0 gets the block's sum of sh.warp[i], i < n.
__device__ __forceinline__ int64_t block_sums(const SampleShared& sh, int n) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    int64_t x = 0;
    if (lane < n)
        for (int w = 0; w < warps; ++w) x += sh.warp[lane][w];
    return x;
}
// Lane i of warp 0, i < n, sends its value to every block of the cluster.
__device__ __forceinline__ void cluster_send(SampleShared& sh, int turn, int n, int64_t x) {
    const int lane = threadIdx.x & 31;
    const uint32_t ranks = cluster_size(), me = cluster_rank();
    if (lane < n)
        for (uint32_t r = 0; r < ranks; ++r) store_remote(&sh.from[turn][lane][me], r, x);
}
// The largest of a value per thread, over the cluster.
__device__ __forceinline__ uint32_t cluster_max(SampleShared& sh, int& turn, uint32_t v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    v = __reduce_max_sync(0xffffffffu, v);
    if (lane == 0) sh.warp[0][warp] = v;
    __syncthreads();
    turn ^= 1;
    const uint32_t ranks = cluster_size();
    if (warp == 0) {
        v = __reduce_max_sync(0xffffffffu, lane < warps ? static_cast<uint32_t>(sh.warp[0][lane]) : 0u);
        if (lane < static_cast<int>(ranks)) store_remote(&sh.from[turn][0][cluster_rank()], lane, v);
    }
    cluster_barrier();
    v = lane < static_cast<int>(ranks) ? static_cast<uint32_t>(sh.from[turn][0][lane]) : 0u;
    return __reduce_max_sync(0xffffffffu, v);
}

// rint(2^38 w) of a w in [0, 1] as 2^19 hi + lo: adding 2^23 (1.5 2^23) leaves a
// number below 2^22 rounded to a whole one in the low mantissa bits, and both
// differences and scalings are exact, so this is the one rounding of 2^38 w.
// Two 32-bit sums cost what a 64-bit one does, and no conversion instruction.
__device__ __forceinline__ void split_mass(float w, int& hi, int& lo) {
    const float x = __fmul_rn(w, 524288.F);
    const float y = __fadd_rn(x, 8388608.F);
    hi = __float_as_int(y) - 0x4B000000;
    const float r = __fsub_rn(x, __fsub_rn(y, 8388608.F));
    lo = __float_as_int(__fmaf_rn(r, 524288.F, 12582912.F)) - 0x4B400000;
}
__device__ __forceinline__ int64_t join_mass(int hi, int lo) { return (static_cast<int64_t>(hi) << 19) + lo; }

template <int DT>
__global__ void __launch_bounds__(kMaxSampleThreads, 2) sample_cluster_kernel(const SampleArgs a) {
    using K = Keys<DT>;
    using Key = typename K::Key;
    constexpr int VE = K::kVec;
    extern __shared__ __align__(16) uint8_t sample_smem[];
    __shared__ SampleShared sh;
    Key* const keys = reinterpret_cast<Key*>(sample_smem);
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // every block runs before the first remote store
    pdl_launch_dependents();
    pdl_wait_on_producer();
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ranks = cluster_size(), rank = cluster_rank();
    const int row = blockIdx.x / ranks, n = a.vocab;
    int turn = 0;
    // the row as aligned 16-byte words; this block's words, slot s of them is entry first + s
    const auto* src = static_cast<const typename K::Raw*>(a.logits) + row * a.row_stride;
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(typename K::Raw));
    const int words = (n + shift + VE - 1) / VE;
    const int word0 = static_cast<int>(static_cast<int64_t>(words) * rank / ranks);
    const int mine = static_cast<int>(static_cast<int64_t>(words) * (rank + 1) / ranks) - word0;
    const int first = word0 * VE - shift;
    uint32_t best = 0, edge = 0;
    constexpr int kAhead = 4;  // words in flight a thread
    for (int w0 = tid; w0 < mine; w0 += kAhead * threads) {
        uint4 in[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = first + (w0 + u * threads) * VE;
            if (w0 + u * threads < mine && i >= 0 && i + VE <= n) in[u] = __ldcs(reinterpret_cast<const uint4*>(src + i));
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int w = w0 + u * threads, i = first + w * VE;
            if (w >= mine) break;
            if (i >= 0 && i + VE <= n) {
                *reinterpret_cast<uint4*>(keys + w * VE) = K::pack(in[u], best);
                continue;
            }
            for (int e = 0; e < VE; ++e) {  // the row's ends: a slot outside is below every entry's key
                const uint32_t k = i + e >= 0 && i + e < n ? K::key(src[i + e]) : 0;
                keys[w * VE + e] = static_cast<Key>(k);
                edge = max(edge, k);
            }
        }
    }
    asm volatile("barrier.cluster.wait;" ::: "memory");
    const uint32_t top = cluster_max(sh, turn, max(K::top(best), edge));  // its barriers also publish `keys` to the block
    const float m = K::value(top);
    const bool lead = rank == 0 && tid == 0;
    if (m == -INFINITY) {
        if (lead) {
            a.tokens[row] = -1;
            if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
        }
        cluster_barrier();
        return;
    }
    const float t = a.temperature != nullptr ? a.temperature[row] : 1.F;
    if (!(t > 0.F)) {
        uint32_t after = 0;  // entries from the earliest maximum on
        for (int w = tid; w < mine && after == 0; w += threads) {
            Key k[VE];
            *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(keys + w * VE);
#pragma unroll
            for (int e = VE - 1; e >= 0; --e)
                if (k[e] == top) after = static_cast<uint32_t>(n - (first + w * VE + e));
        }
        after = cluster_max(sh, turn, after);
        if (lead) {
            a.tokens[row] = n - static_cast<int32_t>(after);
            if (a.logprobs != nullptr) a.logprobs[row] = 0.F;
        }
        cluster_barrier();
        return;
    }
    const float inv = inverse_temperature(t);
    // keys from here on weigh 1: the maximum, for an infinite T every finite one
    const uint32_t full = t == INFINITY && m < INFINITY ? K::near(-INFINITY) + 1 : top;
    // (written so that nothing branches: a branch an entry, over the exponential or
    // over the sums of a pivot, made 64 rows 60 us instead of 53)
    auto weight = [&](uint32_t k) {
        const float e = expf((K::value(k) - m) * inv);
        return k >= full ? 1.F : e;
    };
    auto mass = [&](uint32_t k) {
        int hi, lo;
        split_mass(weight(k), hi, lo);
        return join_mass(hi, lo);
    };
    // f(key) for every entry with key >= from, in any order, and for some below; a
    // word whose entries all lie below is skipped as a whole, the rest goes
    // without branches (per-entry ones cost more than they save)
    auto sweep = [&](uint32_t from, auto f) {
        for (int w = tid; w < mine; w += threads) {
            Key k[VE];
            *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(keys + w * VE);
            if (K::largest(k) < from) continue;
#pragma unroll
            for (int e = 0; e < VE; ++e) f(static_cast<uint32_t>(k[e]));
        }
    };
    // f(key) for the entries with from <= key < end, few of them: one branch a word
    auto hits = [&](uint32_t from, uint32_t end, auto f) {
        for (int w = tid; w < mine; w += threads) {
            Key k[VE];
            *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(keys + w * VE);
            uint32_t in = 0;
#pragma unroll
            for (int e = 0; e < VE; ++e) in |= (k[e] - from < end - from ? 1u : 0u) << e;
            while (in != 0) {
                f(static_cast<uint32_t>(keys[w * VE + __ffs(in) - 1]));
                in &= in - 1;
            }
        }
    };
    // No mass lies below: exp(-28) 2^38 rounds to none.
    const uint32_t none = K::near(m - 28.F * t);
    // Pivot i of n, falling, for the next try in (lo, hi).  They split the range evenly:
    // by value while it is wide (by key, a range about 0 is almost all tiny
    // numbers), by key once it is narrow.
    auto next_pivot = [&](uint32_t lo, uint32_t hi, int tries, int i, uint32_t share) {  // share: 2^32 / (n + 1)
        const float x_hi = K::value(min(hi, top)), x_lo = fmaxf(K::value(lo), m - 30.F * t);
        const uint32_t part = share * static_cast<uint32_t>(i + 1);
        const float below = (x_hi - x_lo) * (static_cast<float>(part) * 2.3283064e-10F);
        const bool by_value = tries < 3 && below > 0.F && below < 1.0e30F;
        const uint32_t key = by_value ? K::near(x_hi - below) : hi - __umulhi(hi - lo, part);
        return max(min(key, hi - 1), lo + 1);
    };
    // The search: the largest key whose entries at or above it reach a target (in
    // number, or in mass).  lo reaches it (or is where the search began), hi does
    // not; above: what lies at or above hi, in the end above lo.
    int listed = -1;          // entries in sh.list, or -1
    bool everything = false;  // the list holds all entries at or above its lowest
    // The end of it, on the list, every block by itself: a warp tries two keys a
    // round and all warps read all sums (two halves of sh.warp in turn, so that a
    // round has one barrier).  base: what lies above the list; at_lo, at_hi: entries
    // of the list at or above lo, hi.
    auto finish = [&](auto by_mass, uint32_t& lo, uint32_t hi, int64_t base, int at_lo, int at_hi, int64_t& above,
                      int64_t target) {
        const int pivots = 2 * (threads >> 5);
        const uint32_t share = 0xffffffffu / static_cast<uint32_t>(pivots + 1);
        for (int tries = 0; hi - lo > 1 && at_lo - at_hi > 1; ++tries) {
            const uint32_t p0 = next_pivot(lo, hi, tries, 2 * warp, share);
            const uint32_t p1 = next_pivot(lo, hi, tries, 2 * warp + 1, share);
            int64_t m0 = 0, m1 = 0;
            int c0 = 0, c1 = 0;
            for (int i = lane; i < listed; i += 32) {
                const uint32_t k = sh.list[i];
                c0 += k >= p0;
                c1 += k >= p1;
                if constexpr (by_mass) {
                    const int64_t w = sh.mass[i];
                    m0 += k >= p0 ? w : 0;
                    m1 += k >= p1 ? w : 0;
                }
            }
            c0 = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(c0)));
            c1 = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(c1)));
            if constexpr (by_mass) {
                m0 = warp_sum48(m0);
                m1 = warp_sum48(m1);
            }
            int64_t* const sums = sh.warp[2 * (tries & 1)];
            int64_t* const counts = sh.warp[2 * (tries & 1) + 1];
            if (lane == 0) {
                counts[2 * warp] = c0;
                counts[2 * warp + 1] = c1;
                sums[2 * warp] = by_mass ? m0 : c0;
                sums[2 * warp + 1] = by_mass ? m1 : c1;
            }
            __syncthreads();
            const int64_t x = lane < pivots ? sums[lane] : 0;
            const unsigned reach = __ballot_sync(0xffffffffu, lane < pivots && base + x >= target);
            const int at = reach != 0 ? __ffs(reach) - 1 : pivots;
            const uint32_t was_lo = lo, was_hi = hi;
            if (at < pivots) {
                lo = next_pivot(was_lo, was_hi, tries, at, share);
                at_lo = static_cast<int>(counts[at]);
            }
            if (at > 0) {
                hi = next_pivot(was_lo, was_hi, tries, at - 1, share);
                at_hi = static_cast<int>(counts[at - 1]);
                above = base + sums[at - 1];
            }
        }
        if (hi - lo > 1 && at_lo - at_hi == 1) {  // one entry is left
            uint32_t k = 0;
            for (int i = lane; i < listed; i += 32)
                if (sh.list[i] < hi) k = max(k, sh.list[i]);
            k = __reduce_max_sync(0xffffffffu, k);
            if (above + (by_mass ? mass(k) : 1) >= target) lo = k;
            else above += by_mass ? mass(k) : 1;
        }
        __syncthreads();
    };
    // All of it.  The target may depend on the sum over the entries above the first
    // lo, which the first try brings along.  The sums of a try meet in warp 0
    // (lane i: sum i), which alone decides; the other warps read its decision.
    auto locate = [&](auto by_mass, auto target_of, bool want_list, uint32_t& lo, int64_t& above, int64_t& target) {
        if (by_mass && listed >= 0 && everything) {  // the search by number has left the entries that are kept
            int64_t over = 0;
            int count = 0;
            for (int i = tid; i < listed; i += threads) sh.mass[i] = mass(sh.list[i]);
            __syncthreads();
            for (int i = lane; i < listed; i += 32)
                if (sh.list[i] > lo) {
                    over += sh.mass[i];
                    ++count;
                }
            count = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(count)));
            target = target_of(warp_sum48(over));
            above = 0;
            finish(by_mass, lo, top + 1, 0, count, 0, above, target);
            return;
        }
        constexpr int N = by_mass ? kSums : kPivots, kCounts = by_mass ? kPivots + 1 : 0;
        int hi_number = 0;  // (warp 0's) entries at or above hi; lane i: of block i
        if (warp == 0) {
            // The first try: every kFirst temperatures below the maximum, which is where a
            // nucleus of ordinary logits tends to end.  Five keys that far apart, means of
            // four seeds (64 rows of 16 bits, 333 of 32), when the rest was slower: 60 and
            // 103 us; four, 3 apart: 64 and 108; at 1.5, 3.5, 6, 9, 13: 66 and 110; six, to
            // 14: 65 and 107.
            // (with lo == top no key lies between: every pivot is top + 1, where nothing is)
            if (lane < kPivots) sh.pv[lane] = max(min(K::near(m - kFirst * (lane + 1) * t), top), lo + 1);
            if (lane == 0) {
                sh.lo = lo;
                sh.hi = top + 1;  // nothing lies at or above it
                sh.above = 0;
                sh.at_hi = 0;
            }
        }
        __syncthreads();
        for (int tries = 0;; ++tries) {
            uint32_t pv[kPivots];  // falling
#pragma unroll
            for (int i = 0; i < kPivots; ++i) pv[i] = sh.pv[i];
            // sums over the entries at or above each pivot, and above the first lo
            int vh[kPivots + 1], vl[kPivots + 1], vc[kPivots];
#pragma unroll
            for (int i = 0; i <= kPivots; ++i) vh[i] = vl[i] = 0;
#pragma unroll
            for (int i = 0; i < kPivots; ++i) vc[i] = 0;
            const uint32_t from = by_mass && tries == 0 ? max(lo + 1, none) : pv[kPivots - 1];
            sweep(from, [&](uint32_t k) {
                if constexpr (by_mass) {
                    int h, l;
                    const float e = weight(k);
                    split_mass(k >= from ? e : 0.F, h, l);
                    vh[kPivots] += h;
                    vl[kPivots] += l;
#pragma unroll
                    for (int i = 0; i < kPivots; ++i) {
                        const bool in = k >= pv[i];
                        vh[i] += in ? h : 0;
                        vl[i] += in ? l : 0;
                        vc[i] += in;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kPivots; ++i) vc[i] += k >= pv[i];
                }
            });
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int64_t x;
                if (by_mass && i <= kPivots) x = warp_sum48(join_mass(vh[i], vl[i]));
                else x = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(vc[by_mass ? i - kPivots - 1 : i]));
                if (lane == 0) sh.warp[i][warp] = x;
            }
            __syncthreads();
            turn ^= 1;
            if (warp == 0) cluster_send(sh, turn, N, block_sums(sh, N));
            cluster_barrier();
            if (warp == 0) {
                int64_t x = 0;
                if (lane < N)
                    for (uint32_t r = 0; r < ranks; ++r) x += sh.from[turn][lane][r];
                if (tries == 0) {
                    const int64_t t0 = target_of(__shfl_sync(0xffffffffu, x, kPivots));
                    if (lane == 0) sh.target = t0;
                    __syncwarp();
                }
                const uint32_t my_pv = sh.pv[lane < kPivots ? lane : 0];
                const unsigned reach = __ballot_sync(0xffffffffu, lane < kPivots && x >= sh.target);
                // the first pivot that reaches the target is the new lo, the one before it the new hi
                const int at = reach != 0 ? __ffs(reach) - 1 : kPivots;
                const int i_lo = min(at, kPivots - 1), i_hi = max(at - 1, 0);
                const uint32_t nlo = __shfl_sync(0xffffffffu, my_pv, i_lo), nhi = __shfl_sync(0xffffffffu, my_pv, i_hi);
                const int64_t sum_hi = __shfl_sync(0xffffffffu, x, i_hi);
                const int number_lo = static_cast<int>(__shfl_sync(0xffffffffu, x, kCounts + i_lo));
                const int number_hi = static_cast<int>(__shfl_sync(0xffffffffu, x, kCounts + i_hi));
                const uint32_t new_lo = at < kPivots ? nlo : sh.lo, new_hi = at > 0 ? nhi : sh.hi;
                const int all_hi = at > 0 ? number_hi : sh.at_hi;
                const bool real = lane < static_cast<int>(ranks);
                if (at > 0) hi_number = real ? static_cast<int>(sh.from[turn][kCounts + i_hi][lane]) : 0;
                // A list of all that lies above lo, or of what lies between, if they are few.
                const bool narrow = new_hi - new_lo <= 1;
                const bool all = at < kPivots && number_lo <= kList && (!narrow || want_list);
                const bool some = at < kPivots && number_lo - all_hi <= kList && !narrow;
                const int own_lo = real ? static_cast<int>(sh.from[turn][kCounts + i_lo][lane]) : 0;
                const int own = all || some ? own_lo - (all ? 0 : hi_number) : 0;
                // (entries of the blocks before this one)
                const int before = static_cast<int>(
                    __reduce_add_sync(0xffffffffu, static_cast<unsigned>(lane < static_cast<int>(rank) ? own : 0)));
                const uint32_t pivot = next_pivot(new_lo, new_hi, tries, lane, 0xffffffffu / (kPivots + 1));
                __syncwarp();
                if (lane < kPivots) sh.pv[lane] = pivot;
                if (lane == 0) {
                    sh.lo = new_lo;
                    sh.hi = new_hi;
                    if (at > 0) sh.above = sum_hi;
                    sh.at_hi = all_hi;
                    sh.listed = all ? number_lo : some ? number_lo - all_hi : -1;
                    sh.everything = all ? 1 : 0;
                    sh.counted = at < kPivots && new_hi - new_lo <= kBins ? 1 : 0;
                    sh.start = before;
                    sh.own_count = 0;
                }
            }
            __syncthreads();
            if (sh.listed >= 0 || sh.hi - sh.lo <= 1 || sh.counted != 0) break;
        }
        const uint32_t hi = sh.hi;
        listed = sh.listed;
        everything = sh.everything != 0;
        lo = sh.lo;
        above = sh.above;
        target = sh.target;
        if (listed >= 0) {  // the keys of every block to every block
            const uint32_t end = everything ? top + 1 : hi;
            hits(lo, end, [&](uint32_t k) { sh.own[atomicAdd(&sh.own_count, 1)] = k; });
            __syncthreads();
            const int own = sh.own_count, start = sh.start;
            for (int i = tid; i < own * static_cast<int>(ranks); i += threads) {
                const int r = i / own, j = i - r * own;
                store_remote32(&sh.list[start + j], r, sh.own[j]);
            }
            cluster_barrier();
            if constexpr (by_mass) {
                for (int i = tid; i < listed; i += threads) sh.mass[i] = mass(sh.list[i]);
                __syncthreads();
            }
            const int at_hi = everything ? sh.at_hi : 0;
            finish(by_mass, lo, hi, everything ? 0 : above, listed, at_hi, above, target);
        } else if (hi - lo > 1) {
            // Many entries of few keys (16-bit types): counters, one a key, in the places of
            // the list and its masses.  Block i adds up the keys number i, i + ranks, ... of all blocks
            // and tells them.
            const uint32_t span = hi - lo;
            const int per = kBins / static_cast<int>(ranks);
            uint32_t* const bin = sh.list;
            uint32_t* const got = sh.list + kBins;
            uint32_t* const sum = sh.own;
            for (int i = tid; i < kBins; i += threads) bin[i] = 0;
            __syncthreads();
            hits(lo, hi, [&](uint32_t k) { atomicAdd(&bin[k - lo], 1u); });
            __syncthreads();
            for (int i = tid; i < kBins; i += threads) {
                const int owner = i & (static_cast<int>(ranks) - 1);
                store_remote32(&got[rank * per + i / ranks], owner, bin[i]);
            }
            cluster_barrier();
            for (int i = tid; i < per; i += threads) {
                uint32_t c = 0;
                for (uint32_t r = 0; r < ranks; ++r) c += got[r * per + i];
                for (uint32_t r = 0; r < ranks; ++r) store_remote32(&sum[i * ranks + rank], r, c);
            }
            cluster_barrier();
            // every warp: a lane has kBins / 32 keys in a row, the highest first
            constexpr int kEach = kBins / 32;
            auto part = [&](uint32_t back) {  // of the key that many below hi - 1
                const int64_t x = back < span ? static_cast<int64_t>(sum[span - 1 - back]) : 0;
                if constexpr (by_mass) return x * mass(hi - 1 - min(back, span - 1));
                else return x;
            };
            int64_t mine_sum = 0;
#pragma unroll 4
            for (int i = 0; i < kEach; ++i) mine_sum += part(lane * kEach + i);
            const int64_t upto = warp_scan64(mine_sum);
            const unsigned reach = __ballot_sync(0xffffffffu, above + upto >= target);
            const int at = reach != 0 ? __ffs(reach) - 1 : 31;  // (lo reaches the target, so some lane does)
            int64_t c = above + upto - mine_sum;
            uint32_t found = lo;
            if (lane == at) {
                for (int i = 0; i < kEach && found == lo; ++i) {
                    const uint32_t back = lane * kEach + i;
                    if (back + 1 >= span) break;
                    const int64_t x = part(back);
                    if (c + x >= target) found = hi - 1 - back;
                    else c += x;
                }
            }
            __syncwarp();
            lo = __shfl_sync(0xffffffffu, found, at);
            above = __shfl_sync(0xffffffffu, c, at);
            __syncthreads();
        } else {
            __syncthreads();
        }
    };
    // kept: key > cut, and the first `ties` (by index) of the entries with key == cut
    uint32_t cut = 0;  // below every entry: all are kept
    int64_t ties = 0;
    bool some_ties = false;  // not all of the entries at `cut` are kept
    const int k_ = a.top_k != nullptr ? a.top_k[row] : 0;
    const float p = a.top_p != nullptr ? a.top_p[row] : 1.F;
    constexpr std::integral_constant<bool, false> by_number{};
    constexpr std::integral_constant<bool, true> by_mass{};
    if (k_ > 0 && k_ < n) {
        int64_t above, target;
        locate(by_number, [&](int64_t) { return static_cast<int64_t>(k_); }, p < 1.F, cut, above, target);
        ties = k_ - above;
        some_ties = true;
    }
    if (p < 1.F) {
        // (with the range empty, lo == cut == top, the one try only brings the sum: nothing lies above)
        uint32_t lo = cut;
        int64_t above, reach;
        locate(by_mass, [&](int64_t over) {
            const int64_t whole = over + (some_ties ? ties * mass(cut) : 0);
            const int64_t r = __double2ll_ru(__dmul_rn(static_cast<double>(p), __ll2double_rn(whole)));
            return r < 1 ? 1 : r;
        }, false, lo, above, reach);
        const int64_t each = lo > 0 ? mass(lo) : 0;
        const int64_t need = each > 0 ? (reach - above + each - 1) / each : 0;
        if (each > 0 && (lo > cut || need < ties)) ties = need;
        some_ties = some_ties || lo > 0;
        cut = lo;
    }
    float low = a.min_p != nullptr ? a.min_p[row] : 0.F;
    low = low > 1.F ? 1.F : low;
    // Index order from here.  A thread's entries are a run of words (an odd number,
    // so that a warp's reads hit all banks); it sums what it keeps above `cut` and
    // counts its entries at `cut`.
    const int run = ((mine + threads - 1) / threads) | 1;
    const int w0 = min(mine, tid * run), w1 = min(mine, w0 + run);
    const uint32_t least = max(max(cut, none), low > 0.F ? K::near(m + t * (logf(low) * 1.001F - 0.001F)) : 0u);
    int sum_h = 0, sum_l = 0, at_cut = 0;
    for (int w = w0; w < w1; ++w) {
        Key k[VE];
        *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(keys + w * VE);
        if (K::largest(k) < least) continue;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float x = weight(k[e]);
            int h, l;
            split_mass(k[e] > cut && !(x < low) ? x : 0.F, h, l);
            sum_h += h;
            sum_l += l;
            at_cut += k[e] == cut;
        }
    }
    if (!some_ties) at_cut = 0;
    const int64_t thread_mass = join_mass(sum_h, sum_l);
    sh.mass[tid] = thread_mass;  // (the list is done with)
    sh.list[tid] = at_cut;
    const int64_t warp_mass = warp_sum48(thread_mass);
    const int64_t warp_ties = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(at_cut));
    if (lane == 0) {
        sh.warp[0][warp] = warp_mass;
        sh.warp[1][warp] = warp_ties;
    }
    __syncthreads();
    turn ^= 1;
    if (warp == 0) cluster_send(sh, turn, 2, block_sums(sh, 2));
    cluster_barrier();
    if (warp == 0) {
        // the blocks' shares (lane = block), then this block's warps' (lane = warp)
        const int64_t each = some_ties && !(weight(cut) < low) ? mass(cut) : 0;
        const bool real = lane < static_cast<int>(ranks);
        const int64_t block_ties = real ? sh.from[turn][1][lane] : 0;
        const int64_t block_ties_before = warp_scan64(block_ties) - block_ties;
        const int64_t block_quota = min(max(ties - block_ties_before, static_cast<int64_t>(0)), block_ties);
        const int64_t block_mass = (real ? sh.from[turn][0][lane] : 0) + block_quota * each;
        const int64_t block_upto = warp_scan64(block_mass);
        const int64_t whole = __shfl_sync(0xffffffffu, block_upto, 31);
        const int64_t before = __shfl_sync(0xffffffffu, block_upto - block_mass, rank);
        const int64_t ties_before = __shfl_sync(0xffffffffu, block_ties_before, rank);
        int64_t aim = __double2ll_rd(__dmul_rn(static_cast<double>(a.uniform[row]), __ll2double_rn(whole)));
        aim = (aim < 0 ? 0 : aim >= whole ? whole - 1 : aim) - before;
        if (aim >= 0 && aim < __shfl_sync(0xffffffffu, block_mass, rank)) {
            const bool real_warp = lane < (threads >> 5);
            const int64_t ties_of = real_warp ? sh.warp[1][lane] : 0;
            const int64_t ties_at_warp = ties_before + warp_scan64(ties_of) - ties_of;
            const int64_t quota_of = min(max(ties - ties_at_warp, static_cast<int64_t>(0)), ties_of);
            const int64_t all_of = (real_warp ? sh.warp[0][lane] : 0) + quota_of * each;
            const int64_t upto_of = warp_scan64(all_of);
            const int hit = __ffs(__ballot_sync(0xffffffffu, upto_of > aim)) - 1;
            // that warp's threads (lane = thread), then the words of the one that holds the
            // token, 32 at a time, a lane's entries in order
            int64_t at = __shfl_sync(0xffffffffu, upto_of - all_of, hit), left = __shfl_sync(0xffffffffu, quota_of, hit);
            const int ties_here = sh.list[32 * hit + lane];
            const int64_t ties_before_here = warp_scan64(ties_here) - ties_here;
            const int64_t quota_here =
                min(max(left - ties_before_here, static_cast<int64_t>(0)), static_cast<int64_t>(ties_here));
            const int64_t mass_here = sh.mass[32 * hit + lane] + quota_here * each;
            const int64_t upto_here = warp_scan64(mass_here);
            const int hit_lane = __ffs(__ballot_sync(0xffffffffu, at + upto_here > aim)) - 1;
            at += __shfl_sync(0xffffffffu, upto_here - mass_here, hit_lane);
            left = __shfl_sync(0xffffffffu, quota_here, hit_lane);
            const int h0 = min(mine, (32 * hit + hit_lane) * run), h1 = min(mine, h0 + run);
            for (int w = h0; w < h1; w += 32) {
                Key k[VE];
                *reinterpret_cast<uint4*>(k) =
                    w + lane < h1 ? *reinterpret_cast<const uint4*>(keys + (w + lane) * VE) : make_uint4(0, 0, 0, 0);
                int64_t x[VE], sum = 0;
                int c = 0;
#pragma unroll
                for (int e = 0; e < VE; ++e) c += some_ties && k[e] == cut;
                const int64_t ties_at = warp_scan64(c);
                int64_t mine_left = left - (ties_at - c);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const bool in = k[e] > cut || (some_ties && k[e] == cut && mine_left-- > 0);
                    x[e] = in && !(weight(k[e]) < low) ? mass(k[e]) : 0;
                    sum += x[e];
                }
                const int64_t upto = warp_scan64(sum);
                if (at + upto - sum <= aim && aim < at + upto) {
                    int64_t c2 = at + upto - sum, drawn = 0;
                    int place = -1;
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        c2 += x[e];
                        if (place < 0 && c2 > aim) {
                            place = e;
                            drawn = x[e];
                        }
                    }
                    a.tokens[row] = first + (w + lane) * VE + place;
                    if (a.logprobs != nullptr)
                        a.logprobs[row] = static_cast<float>(log(__ll2double_rn(drawn) / __ll2double_rn(whole)));
                }
                at += __shfl_sync(0xffffffffu, upto, 31);
                left -= __shfl_sync(0xffffffffu, ties_at, 31);
                if (at > aim) break;
            }
        }
    }
    cluster_barrier();  // no block leaves while another may still write into its shared memory
}

constexpr int kSampleSmem = 200 * 1024;  // the largest slice of a row

// One row to `cluster` blocks of `threads`: the kernel's 64 registers leave 1024
// threads an SM, which the blocks that are resident together share (blocks of up
// to 2048 threads in all, in two turns: 64 rows 50 us for 47, 333 rows 102 for 88).
template <int DT>
cudaError_t launch_cluster(const SampleArgs& a, int cluster, cudaStream_t s) {
    using K = Keys<DT>;
    auto kernel = sample_cluster_kernel<DT>;
    const int words = (a.vocab + 2 * K::kVec - 2) / K::kVec;
    const int slice = (words + cluster - 1) / cluster * 16;
    const int fit = 228 * 1024 / (slice + static_cast<int>(sizeof(SampleShared)) + 1024);
    const int64_t blocks = static_cast<int64_t>(a.rows) * cluster;
    const int64_t per_sm = (blocks + device_sm_count() - 1) / device_sm_count();
    int threads = 512;
    while (threads > 128 && (threads * (per_sm < fit ? per_sm : fit) > 1024 || threads > 2 * (slice / 16))) threads >>= 1;
    static std::atomic<uint64_t> opted{0};
    cudaError_t st = opt_in_smem(reinterpret_cast<const void*>(kernel), kSampleSmem, opted);
    if (st == cudaSuccess && cluster > 8)
        st = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (st != cudaSuccess) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows * cluster));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = slice;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t sample_rows(const SampleArgs& a, int dt, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    const int64_t bytes = static_cast<int64_t>(a.vocab) * (dt == kF32 ? 4 : 2) + 16;
    // 16 blocks a row while that is one an SM: 1 row of 304 KB 26 us for 28 in 8, 9 rows 28 for 35; 64 rows 89 for 87
    // (and where 8 cannot hold it)
    const bool wide = static_cast<int64_t>(a.rows) * kMaxCluster <= device_sm_count() || bytes / 8 + 16 > kSampleSmem;
    int cluster = wide ? kMaxCluster : 8;
    // fewer blocks a row once the rows fill the SMs by themselves, but no slice over 56 KB (three blocks an SM):
    // 333 rows of 201 KB 88 us in 4 blocks, 90 in 8, 110 in 2
    while (cluster > 1 && static_cast<int64_t>(a.rows) * cluster > 4 * device_sm_count() &&
           bytes / (cluster / 2) <= 56 * 1024)
        cluster >>= 1;
    // and none so small that its barrier costs more than its share of the row: 300 rows of 2 KB 23 us in 1 block,
    // 28 in 4, 49 in 8; of 64 KB 83 in 4, 87 in 8
    while (cluster > 1 && bytes / cluster < 4096) cluster >>= 1;
    if (bytes / cluster + 16 > kSampleSmem) {  // longer than a cluster holds
        // (this way 152 000 logits take 1.7 ms: a pass over memory for every bit of a key)
        auto kernel = dt == kBF16  ? sample_rows_kernel<kBF16>
                      : dt == kF16 ? sample_rows_kernel<kF16>
                                   : sample_rows_kernel<kF32>;
        return launch_pdl(kernel, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
    }
    return dt == kBF16 ? launch_cluster<kBF16>(a, cluster, s) : dt == kF16 ? launch_cluster<kF16>(a, cluster, s)
                                                                         : launch_cluster<kF32>(a, cluster, s);
}

}  // namespace kc

// sample.cu -- the next token of every row from its logits: temperature,
// top-k, top-p, min-p and one given uniform number.
//
// With x the logits in 32 bits (NaN counts as -inf) and m their maximum:
//   w_i = 1 where x_i == m, else exp((x_i - m) * (1 / T));  W_i = rint(2^38 w_i)
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
    const float inv = 1.F / t;
    auto weight = [&](float x) { return x == m ? 1.F : expf((x - m) * inv); };
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
// to find the key at which the kept prefix ends: seven keys that split the
// range still possible are tried at once - each thread counts, or sums the
// masses of, the entries at or above each of them in registers - and the
// cluster exchanges the sums through distributed shared memory with one
// barrier.  The first seven lie at fixed distances below the maximum (in units
// of the temperature), which leaves few entries; then each try takes three bits
// off the range.  No sort, no atomics.
constexpr int kPivots = 7;
constexpr int kMaxCluster = 8;
constexpr int kMaxSampleThreads = 1024;

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

struct SampleShared {
    int64_t warp[32][kPivots + 1];
    int64_t from[2][kMaxCluster][kPivots + 1];  // what each block of the cluster sent, alternating halves
    int64_t scan[32];
};

// Sum (or maximum) over the block and the cluster of n values a thread; in
// `each`, the blocks' own contributions stay readable until the call after next.
template <int N, bool MAX>
__device__ __forceinline__ void cluster_reduce(SampleShared& sh, int& turn, int64_t (&v)[N]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const int64_t x = __shfl_xor_sync(0xffffffffu, v[i], o);
            v[i] = MAX ? (x > v[i] ? x : v[i]) : v[i] + x;
        }
        if (lane == 0) sh.warp[warp][i] = v[i];
    }
    __syncthreads();
    const uint32_t ranks = cluster_size(), me = cluster_rank();
    turn ^= 1;
    if (threadIdx.x < N) {
        int64_t s = sh.warp[0][threadIdx.x];
        for (int w = 1; w < warps; ++w) {
            const int64_t x = sh.warp[w][threadIdx.x];
            s = MAX ? (x > s ? x : s) : s + x;
        }
        for (uint32_t r = 0; r < ranks; ++r) store_remote(&sh.from[turn][me][threadIdx.x], r, s);
    }
    cluster_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        int64_t s = sh.from[turn][0][i];
        for (uint32_t r = 1; r < ranks; ++r) {
            const int64_t x = sh.from[turn][r][i];
            s = MAX ? (x > s ? x : s) : s + x;
        }
        v[i] = s;
    }
}

template <int DT>
__global__ void __launch_bounds__(kMaxSampleThreads) sample_cluster_kernel(const SampleArgs a) {
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
    uint32_t best = 0;
    for (int w = tid; w < mine; w += threads) {
        const int i = first + w * VE;
        typename K::Raw raw[VE];
        Key out[VE];
        const bool all = i >= 0 && i + VE <= n;
        if (all) *reinterpret_cast<uint4*>(raw) = __ldcs(reinterpret_cast<const uint4*>(src + i));
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            uint32_t k = 0;  // below every entry's key: slots outside the row
            if (all) k = K::key(raw[e]);
            else if (i + e >= 0 && i + e < n) k = K::key(src[i + e]);
            best = max(best, k);
            out[e] = static_cast<Key>(k);
        }
        *reinterpret_cast<uint4*>(keys + w * VE) = *reinterpret_cast<const uint4*>(out);
    }
    asm volatile("barrier.cluster.wait;" ::: "memory");
    int64_t red[1] = {static_cast<int64_t>(best)};
    cluster_reduce<1, true>(sh, turn, red);  // its barriers also publish `keys` to the block
    const uint32_t top = static_cast<uint32_t>(red[0]);
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
    const int slots = mine * VE;
    if (!(t > 0.F)) {
        int at = 0x7fffffff;
        for (int s = tid; s < slots; s += threads)
            if (keys[s] == top) at = min(at, first + s);
        red[0] = -static_cast<int64_t>(at);
        cluster_reduce<1, true>(sh, turn, red);
        if (lead) {
            a.tokens[row] = static_cast<int32_t>(-red[0]);
            if (a.logprobs != nullptr) a.logprobs[row] = 0.F;
        }
        cluster_barrier();
        return;
    }
    const float inv = 1.F / t;
    auto weight = [&](uint32_t k) { return k == top ? 1.F : expf((K::value(k) - m) * inv); };
    auto mass = [&](uint32_t k) { return __float2ll_rn(weight(k) * kMassOne); };
    // f(key) for every entry at or above `floor_key`, in any order
    auto sweep = [&](uint32_t floor_key, auto f) {
        for (int w = tid; w < mine; w += threads) {
            Key k[VE];
            *reinterpret_cast<uint4*>(k) = *reinterpret_cast<const uint4*>(keys + w * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (k[e] >= floor_key) f(static_cast<uint32_t>(k[e]));
        }
    };
    // The largest key whose entries at or above it reach `target` (in number, or
    // in mass): lo reaches it, hi does not.  above: what lies above lo.
    auto locate = [&](auto by_mass, int64_t target, uint32_t& lo, int64_t& above) {
        uint32_t hi = top + 1;  // nothing lies at or above it
        above = 0;
        bool started = false;
        while (hi - lo > 1) {
            uint32_t pv[kPivots];
            if (!started) {
                const float d[kPivots] = {0.7F, 1.6F, 2.8F, 4.2F, 6.F, 8.5F, 12.F};
#pragma unroll
                for (int i = 0; i < kPivots; ++i) pv[i] = min(max(K::near(m - d[i] * t), lo + 1), hi - 1);
                started = true;
            } else {
                const uint64_t span = hi - lo;
#pragma unroll
                for (int i = 0; i < kPivots; ++i)
                    pv[i] = min(max(hi - static_cast<uint32_t>(span * (i + 1) / (kPivots + 1)), lo + 1), hi - 1);
            }
            // pv falls; entries at or above hi count for every one of them and are known
            int64_t v[kPivots];
#pragma unroll
            for (int i = 0; i < kPivots; ++i) v[i] = 0;
            sweep(pv[kPivots - 1], [&](uint32_t k) {
                if (k >= hi) return;
                const int64_t x = by_mass ? mass(k) : 1;
#pragma unroll
                for (int i = 0; i < kPivots; ++i)
                    if (k >= pv[i]) v[i] += x;
            });
            cluster_reduce<kPivots, false>(sh, turn, v);
            // the first pivot that reaches the target is the new lo, the one before it the new hi
            uint32_t nlo = lo, nhi = hi;
            int64_t at_hi = above;
            bool found = false;
#pragma unroll
            for (int i = 0; i < kPivots; ++i) {
                if (found) continue;
                if (above + v[i] >= target) {
                    nlo = pv[i];
                    found = true;
                } else {
                    nhi = pv[i];
                    at_hi = above + v[i];
                }
            }
            above = at_hi;
            lo = nlo;
            hi = nhi;
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
        int64_t above;
        locate(by_number, k_, cut, above);
        ties = k_ - above;
        some_ties = true;
    }
    if (p < 1.F) {
        int64_t sum[1] = {0};
        sweep(cut + 1, [&](uint32_t k) { sum[0] += mass(k); });
        cluster_reduce<1, false>(sh, turn, sum);
        const int64_t whole = sum[0] + (some_ties ? ties * mass(cut) : 0);
        int64_t reach = __double2ll_ru(__dmul_rn(static_cast<double>(p), __ll2double_rn(whole)));
        reach = reach < 1 ? 1 : reach;
        uint32_t lo = cut;
        int64_t above;
        locate(by_mass, reach, lo, above);
        const int64_t each = lo > 0 ? mass(lo) : 0;
        const int64_t need = each > 0 ? (reach - above + each - 1) / each : 0;
        if (each > 0 && (lo > cut || need < ties)) ties = need;
        some_ties = some_ties || lo > 0;
        cut = lo;
    }
    // Index order from here: a thread's entries are a run of slots, the block's follow one another
    const int per = ((slots + threads - 1) / threads) | 1;
    const int s0 = min(slots, tid * per), s1 = min(slots, s0 + per);
    // inclusive prefix of v over the block; total: the block's sum
    auto block_scan = [&](int64_t v, int64_t& total) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        __syncthreads();
        if (lane == 31) sh.scan[warp] = v;
        __syncthreads();
        total = 0;
        int64_t before = 0;
        for (int w = 0; w < (threads >> 5); ++w) {
            if (w < warp) before += sh.scan[w];
            total += sh.scan[w];
        }
        return v + before;
    };
    int64_t quota = 0;  // how many of this run's entries at `cut` are kept
    if (some_ties) {
        int64_t c = 0;
        for (int s = s0; s < s1; ++s) c += keys[s] == cut;
        int64_t block_total;
        const int64_t upto = block_scan(c, block_total);
        int64_t v[1] = {tid == 0 ? block_total : 0};
        cluster_reduce<1, false>(sh, turn, v);
        int64_t before = upto - c;
        for (uint32_t r = 0; r < rank; ++r) before += sh.from[turn][r][0];
        quota = min(max(ties - before, static_cast<int64_t>(0)), c);
    }
    float low = a.min_p != nullptr ? a.min_p[row] : 0.F;
    low = low > 1.F ? 1.F : low;
    int64_t sum = 0;
    {
        int64_t left = quota;
        for (int s = s0; s < s1; ++s) {
            const uint32_t k = keys[s];
            const bool in = k > cut || (k == cut && left-- > 0);
            if (in && !(weight(k) < low)) sum += mass(k);
        }
    }
    int64_t block_total;
    const int64_t upto = block_scan(sum, block_total);
    int64_t v[1] = {tid == 0 ? block_total : 0};
    cluster_reduce<1, false>(sh, turn, v);
    const int64_t whole = v[0];
    int64_t before = 0;
    for (uint32_t r = 0; r < rank; ++r) before += sh.from[turn][r][0];
    int64_t aim = __double2ll_rd(__dmul_rn(static_cast<double>(a.uniform[row]), __ll2double_rn(whole)));
    aim = (aim < 0 ? 0 : aim >= whole ? whole - 1 : aim) - before;
    if (upto - sum <= aim && aim < upto) {
        int64_t c = upto - sum, left = quota;
        for (int s = s0; s < s1; ++s) {
            const uint32_t k = keys[s];
            const bool in = k > cut || (k == cut && left-- > 0);
            if (!in || weight(k) < low) continue;
            const int64_t w = mass(k);
            c += w;
            if (c > aim) {
                a.tokens[row] = first + s;
                if (a.logprobs != nullptr)
                    a.logprobs[row] = static_cast<float>(log(__ll2double_rn(w) / __ll2double_rn(whole)));
                break;
            }
        }
    }
    cluster_barrier();  // no block leaves while another may still write into its shared memory
}

constexpr int kSampleSmem = 200 * 1024;  // the largest slice of a row

// One row to `cluster` blocks of `threads`.  The slice should leave room for
// two blocks an SM (their barriers overlap), and all rows together should fill
// the SMs' threads once.
template <int DT>
cudaError_t launch_cluster(const SampleArgs& a, int cluster, cudaStream_t s) {
    using K = Keys<DT>;
    auto kernel = sample_cluster_kernel<DT>;
    const int words = (a.vocab + 2 * K::kVec - 2) / K::kVec;
    const int slice = (words + cluster - 1) / cluster * 16;
    const int fit = static_cast<int>(220 * 1024 / (slice + 8 * 1024));
    int threads = fit >= 8 ? 256 : fit >= 4 ? 512 : 1024;
    if (static_cast<int64_t>(a.rows) * cluster <= 2 * device_sm_count()) threads = 1024;
    while (threads > 128 && threads > 2 * (slice / 16)) threads >>= 1;
    static std::atomic<uint64_t> opted{0};
    const cudaError_t st = opt_in_smem(reinterpret_cast<const void*>(kernel), kSampleSmem, opted);
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
    int cluster = kMaxCluster;
    // fewer blocks a row once the rows fill the SMs by themselves, but no slice over 100 KB
    while (cluster > 1 && static_cast<int64_t>(a.rows) * cluster > 4 * device_sm_count() &&
           bytes / (cluster / 2) <= 100 * 1024)
        cluster >>= 1;
    // and none so small that its barrier costs more than its share of the row
    while (cluster > 1 && bytes / cluster < 4096) cluster >>= 1;
    if (bytes / cluster + 16 > kSampleSmem) {  // longer than a cluster holds
        auto kernel = dt == kBF16 ? sample_rows_kernel<kBF16> : dt == kF16 ? sample_rows_kernel<kF16> : sample_rows_kernel<kF32>;
        return launch_pdl(kernel, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
    }
    return dt == kBF16 ? launch_cluster<kBF16>(a, cluster, s) : dt == kF16 ? launch_cluster<kF16>(a, cluster, s)
                                                                         : launch_cluster<kF32>(a, cluster, s);
}

}  // namespace kc

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

}  // namespace

cudaError_t sample_rows(const SampleArgs& a, int dt, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    auto kernel = dt == kBF16 ? sample_rows_kernel<kBF16> : dt == kF16 ? sample_rows_kernel<kF16> : sample_rows_kernel<kF32>;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
}

}  // namespace kc

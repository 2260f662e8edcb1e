// One token of each row of logits, drawn with a given random number under a temperature,
// top-k, top-p and min-p, gfx950.
//
//   w_j = exp((x_j - max x) / T);  kept: w_j >= min_p; of those the k largest (equal logits: the
//   lower index); of those, in that order, the shortest run whose sum reaches top_p of their
//   sum;  token: the lowest index whose running sum of kept weights exceeds u times their total
//
// Weights are whole numbers, round(2^42 w): their sums do not depend on an order, so that
// atomics and any split of a row give the same bits, and two passes that form the same
// sum agree on every border.  They are formed in float64, as a running sum of a whole vocabulary has borders
// that float32 would miss (a wrong token in a hundred rows).  Nothing is sorted.  Every filter keeps a run of the order
// (logit, lower index), so all that is looked for is its last element:
//   sample_max     each part's largest and least logit
//   sample_hist    counts (top-k) and sums (top-p) of the kept by bins that are even in log w
//   sample_gather  the bins that the borders of top-k and top-p fall into: their elements are
//                  listed, and what lies above them is summed for each part
//   sample_finish  the borders themselves, by comparing the listed elements with each other (long lists,
//                  or the row if it overflows, by the digits of their keys), the total, the part that
//                  holds u times it, and the element within it
// The logits are read once from memory and twice more from the caches behind the L2.  The passes
// are bound by issue slots, of which a weight takes about 25: where an element can be told by its
// logit alone not to count, none is formed.  256 x 151936 bf16, settings of each row: 15, 40, 30 and 31 us (fp16 16,
// 61, 30 and 30); 4 x 151936: 4, 9, 8 and 9, chains of latencies; 64 x 32000 float32, top-p: 5, 9, 8 and 16.
#include "gdn2_common.h"
#include "gdn2_internal.h"

namespace gdn2 {
namespace {

typedef unsigned long long u64;

constexpr int kFrac = 42;             // bits of a weight below 1
constexpr float kFloor = -43.0f;      // log2 of weights that round to nothing
constexpr int kThreads = 256;         // of the passes over parts
constexpr int kFinish = kSampleFinishThreads;
constexpr int kOwn = kSampleList / kFinish;
constexpr int kPairs = 256;  // listed elements that are compared each with each (4 us; by digits 6)
constexpr double kLog2e = 1.4426950408889634074;

// 2^y in units of 2^-42 (at least 1), kFloor < y <= 0: 2^f by its series, |f| <= 1/2 (the first term left out is under
// 9e-15 of it), rounded by the addition of 2^52.
__device__ __forceinline__ u64 weight_of(double y)
{
    constexpr double c[12] = {1.0, 6.931471805599453094e-1, 2.402265069591007123e-1, 5.550410866482157995e-2,
                              9.618129107628477162e-3, 1.333355814642844343e-3, 1.540353039338160995e-4,
                              1.525273380405984028e-5, 1.321548679014430949e-6, 1.017808600923969973e-7,
                              7.054911620801123329e-9, 4.445538271870811498e-10};
    const double n = __builtin_rint(y), f = y - n;
    double p = c[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) p = fma(p, f, c[i]);
    const double v = __builtin_amdgcn_ldexp(p, static_cast<int>(n) + kFrac) + 0x1p52;
    const u64 w = static_cast<u64>(__double_as_longlong(v)) & 0xfffffffffffffULL;
    return w > 0 ? w : 1;
}
__device__ __forceinline__ bool counts(double y) { return y > static_cast<double>(kFloor); }  // not for NaN

// Order of the elements: larger logit first (-0 = 0, NaN above all), of equal ones the lower
// index.  24 bits of index under 32 of the logit, of 16-bit logits 16.
template <typename T>
struct Key {
    static __device__ __forceinline__ u64 of(float v, int i)
    {
        const unsigned b = __float_as_uint(v + 0.0f);
        unsigned k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
        if (v != v) k = 0xffffffffu;
        if constexpr (sizeof(T) == 2) {
            if constexpr (std::is_same<T, f16_t>::value) {
                const uint16_t h = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v + 0.0f));
                k = v != v ? 0xffffu : (h & 0x8000u) ? static_cast<uint16_t>(~h) : (h | 0x8000u);
            } else {
                k >>= 16;
            }
        }
        return (static_cast<u64>(k) << 24) | (0xffffffu - static_cast<unsigned>(i));
    }
    static __device__ __forceinline__ float value(u64 key)
    {
        unsigned k = static_cast<unsigned>(key >> 24);
        if constexpr (std::is_same<T, f16_t>::value) {
            if (k == 0xffffu) return __uint_as_float(0x7fc00000u);
            const uint16_t h = static_cast<uint16_t>((k & 0x8000u) ? (k & 0x7fffu) : ~k);
            return static_cast<float>(__builtin_bit_cast(_Float16, h));
        }
        if constexpr (sizeof(T) == 2) k = k << 16 | (k & 0x8000u ? 0u : 0xffffu);
        if (k == 0xffffffffu || k == 0xffff0000u) return __uint_as_float(0x7fc00000u);
        return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
    }
    static __device__ __forceinline__ int index(u64 key) { return 0xffffff - static_cast<int>(key & 0xffffffu); }
};

// A row, read by 16-byte pieces of its memory; elements outside the row (the first and last
// piece's) come as -inf, or (NEAR) as the row's nearest.
template <typename T>
struct Logits {
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    const T *x, *xa;
    int n, off, pieces;
    __device__ __forceinline__ Logits(const SampleParams &p, int64_t row)
    {
        const int64_t b = row / p.inner;
        x = static_cast<const T *>(p.x) + b * p.outer_stride + (row - b * p.inner) * p.row_stride;
        n = p.n;
        off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / static_cast<int>(sizeof(T));
        xa = x - off;
        pieces = (off + n + N - 1) / N;
    }
    __device__ __forceinline__ int first(int c) const { return c * N - off; }
    template <bool NEAR = false>
    __device__ __forceinline__ void load(int c, float (&v)[N]) const
    {
        const int i0 = first(c);
        if (i0 >= 0 && i0 + N <= n) {
            const uint4 u = *reinterpret_cast<const uint4 *>(xa + static_cast<int64_t>(c) * N);
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    v[i] = __uint_as_float(w[i]);
                } else if constexpr (std::is_same<T, bf16_t>::value) {
                    v[2 * i] = __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                } else {
                    v[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] & 0xffffu)));
                    v[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = i0 + e < 0 ? 0 : i0 + e < n ? i0 + e : n - 1;
                v[e] = io<T>::ld(x, i);
                if (!NEAR && i != i0 + e) v[e] = -INFINITY;
            }
        }
    }
};

__device__ __forceinline__ u64 shfl_xor64(u64 x, int o) { return __shfl_xor(x, o, 64); }
// Over the wave's lanes, by DPP within rows of 16 (exchanges through LDS take ten times as long).
template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <typename F>
__device__ __forceinline__ float wave_all(float x, F f)
{
    x = f(x, dpp<0xb1>(x));   // quad_perm [1, 0, 3, 2]
    x = f(x, dpp<0x4e>(x));   // quad_perm [2, 3, 0, 1]
    x = f(x, dpp<0x141>(x));  // row_half_mirror
    x = f(x, dpp<0x140>(x));  // row_mirror
    const int i = __float_as_int(x);
    return f(f(__int_as_float(__builtin_amdgcn_readlane(i, 0)), __int_as_float(__builtin_amdgcn_readlane(i, 16))),
             f(__int_as_float(__builtin_amdgcn_readlane(i, 32)), __int_as_float(__builtin_amdgcn_readlane(i, 48))));
}
// The larger, NaN above all.
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }
__device__ __forceinline__ float min_of(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ u64 wave_sum64(u64 x)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += shfl_xor64(x, o);
    return x;
}
// Sum over the lanes up to and with this one.
__device__ __forceinline__ u64 wave_scan64(u64 x, int lane)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(x, o, 64);
        x += lane >= o ? y : 0;
    }
    return x;
}

// A row's settings and what the first pass found.
struct RowState {
    float top;     // largest logit
    bool greedy;   // T = 0, or a largest logit that is not finite: the token is the first of them
    double per;    // log2 of the weight of a difference of 1
    u64 least;     // smallest weight that min-p keeps (at least 1)
    float scale;   // bins per factor of 2
    double share;  // top_p; 1 and above: off
    int k;         // top_k; 0: off
};

__device__ __forceinline__ RowState row_state(const SampleParams &p, int64_t row, int lane)
{
    RowState s;
    const float2 own = lane < p.parts ? p.part_top[row * kSampleParts + lane] : make_float2(-INFINITY, INFINITY);
    s.top = wave_all(own.x, max_nan);
    const float low = wave_all(own.y, min_of);
    const float t = p.temperature ? p.temperature[row] : p.temperature_all;
    const float m = p.min_p ? p.min_p[row] : p.min_p_all, share = p.top_p ? p.top_p[row] : p.top_p_all;
    const int k = p.top_k ? p.top_k[row] : p.top_k_all;
    s.greedy = !(t > 0.0f) || !(fabsf(s.top) < INFINITY);
    s.per = kLog2e / static_cast<double>(fmaxf(t, 1e-30f));
    const double least = m > 0.0f ? ceil(static_cast<double>(fminf(m, 1.0f)) * 0x1p42) : 1.0;
    s.least = least > 1.0 ? static_cast<u64>(least) : 1;
    // Bins over the weights that there are: down to 2^-43, the least logit's, or min-p's.
    float range = fminf(-kFloor, static_cast<float>((static_cast<double>(s.top) - static_cast<double>(low)) * s.per));
    if (m > 0.0f) range = fminf(range, 1e-3f - 1.0001f * __builtin_amdgcn_logf(fminf(m, 1.0f)));
    s.scale = range > 0.0f ? kSampleBins / range : 0.0f;
    s.share = share < 1.0f ? (share > 1e-30f ? static_cast<double>(share) : 1e-30) : 1.0;
    if (share != share) s.share = 1.0;
    s.k = k > 0 && k < p.n ? k : 0;
    return s;
}
__device__ __forceinline__ bool filters(const RowState &s) { return s.k > 0 || s.share < 1.0; }
// Whether the bins hold sums: for top-p's border, and so that what top-k keeps for certain need not be summed again
// unless it is little.
__device__ __forceinline__ bool binned_sums(const RowState &s) { return s.share < 1.0 || s.k > 1024; }

__device__ __forceinline__ double log_weight(const RowState &s, float x)
{
    return (static_cast<double>(x) - static_cast<double>(s.top)) * s.per;
}
__device__ __forceinline__ int bin_of(const RowState &s, double y)
{
    const int b = static_cast<int>(static_cast<float>(-y) * s.scale);
    return b < kSampleBins ? b : kSampleBins - 1;
}

// The pieces of a part.
__device__ __forceinline__ void part_range(const SampleParams &p, int pieces, int part, int &lo, int &hi)
{
    lo = part * p.part_pieces;
    hi = lo + p.part_pieces < pieces ? lo + p.part_pieces : pieces;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleParams p)
{
    constexpr int N = Logits<T>::N, U = 4;
    __shared__ float s_top[kThreads / 64], s_low[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / p.parts;
    const int part = static_cast<int>(blockIdx.x - row * p.parts);
    if (part == 0) {  // what the next pass adds to
        u64 *h = p.hist + row * (2 * kSampleBins);
        for (int i = tid; i < 2 * kSampleBins; i += kThreads) h[i] = 0;
    }
    const Logits<T> x(p, row);
    int lo, hi;
    part_range(p, x.pieces, part, lo, hi);
    float top = -INFINITY, low = INFINITY;
    bool nan = false;
    for (int c0 = lo + tid; c0 < hi; c0 += U * kThreads) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * kThreads < hi) x.template load<true>(c0 + u * kThreads, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c0 + u * kThreads >= hi) break;
#pragma unroll
            for (int e = 0; e < N; e += 2) {  // NaN does not show in a maximum
                top = fmaxf(fmaxf(v[u][e], v[u][e + 1]), top);
                low = fminf(fminf(v[u][e], v[u][e + 1]), low);
                nan |= __builtin_isunordered(v[u][e], v[u][e + 1]);
            }
        }
    }
    top = wave_all(nan ? __uint_as_float(0x7fc00000u) : top, max_nan);
    low = wave_all(low, min_of);
    if (lane == 0) {
        s_top[wave] = top;
        s_low[wave] = low;
    }
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < kThreads / 64; ++w) {
            top = max_nan(top, s_top[w]);
            low = fminf(low, s_low[w]);
        }
        p.part_top[row * kSampleParts + part] = make_float2(top, low);
    }
}

// bf16 parts of some length: an exponential for each value that occurs instead of each element.  Values of the 16 octaves
// up to the largest that counts are counted; the few nearer zero, and those of other types, take one each.
// 256 x 151936, settings of each row: 40 us, one by one 64 (fp16, always one by one: 61).
constexpr int kCounters = 2 * 16 * 128, kCounted = 8192;

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_hist_kernel(SampleParams p)
{
    constexpr int N = Logits<T>::N, U = 4;
    constexpr bool kBf16 = std::is_same<T, bf16_t>::value;
    __shared__ u64 s_sum[kSampleBins];
    __shared__ unsigned s_count[kSampleBins];
    __shared__ unsigned s_values[kBf16 ? kCounters + 64 : 1];
    __shared__ u64 s_part[kThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / p.parts;
    const int part = static_cast<int>(blockIdx.x - row * p.parts);
    const Logits<T> x(p, row);
    int lo, hi;
    part_range(p, x.pieces, part, lo, hi);
    float v[U][N];
    auto fetch = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * kThreads < hi) x.load(c0 + u * kThreads, v[u]);
    };
    fetch(lo + tid);  // in flight while the row's settings are formed
    const RowState s = row_state(p, row, lane);
    if (s.greedy) return;
    const bool bins = filters(s), sums = !bins || binned_sums(s);
    const bool counted = kBf16 && p.part_pieces * N >= kCounted;
    if (bins) {
        for (int i = tid; i < kSampleBins; i += kThreads) {
            s_sum[i] = 0;
            s_count[i] = 0;
        }
    }
    if (counted)
        for (int i = tid; i < kCounters; i += kThreads) s_values[i] = 0;
    if (bins || counted) __syncthreads();
    u64 sum = 0;
    // `n` elements of logit a.
    auto add = [&](float a, unsigned n) __attribute__((always_inline)) {
        const double y = log_weight(s, a);
        if (!counts(y)) return;
        u64 w = 0;
        if (sums || s.least > 1) {
            w = weight_of(y);
            if (w < s.least) return;
        }
        if (bins) {
            const int b = bin_of(s, y);
            if (sums) atomicAdd(&s_sum[b], w * n);
            if (s.k > 0) atomicAdd(&s_count[b], n);
        } else {
            sum += w * n;
        }
    };
    if (counted) {
        // No logit below `floor` counts; the largest magnitude of those that do.
        const float floor = static_cast<float>(static_cast<double>(s.top) + 1.01 * static_cast<double>(kFloor) / s.per);
        const unsigned most = __float_as_uint(fmaxf(fabsf(s.top), fabsf(floor))) >> 23;
        const unsigned base = (most > 15 ? most - 15 : 0) << 7, none = kCounters + lane;
        for (int c0 = lo + tid; c0 < hi; c0 += U * kThreads) {
            unsigned mask = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c0 + u * kThreads >= hi) break;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    // Counters of no value, one a lane, take the others without a branch.
                    const unsigned bits = __float_as_uint(v[u][e]) >> 16, at = (bits & 0x7fffu) - base;
                    const bool inside = at < kCounters / 2;
                    atomicAdd(&s_values[inside ? at + (bits >> 15) * (kCounters / 2) : none], 1u);
                    if (__any(!inside))
                        mask |= !inside && v[u][e] >= floor && v[u][e] > -INFINITY ? 1u << (u * N + e) : 0u;
                }
            }
            const int at = c0;
            fetch(c0 + U * kThreads);
            for (; mask; mask &= mask - 1) {
                const int bit = __ffs(mask) - 1;
                add(io<T>::ld(x.x, x.first(at + bit / N * kThreads) + bit % N), 1);
            }
        }
        __syncthreads();
        for (int i = tid; i < kCounters; i += kThreads) {
            const unsigned n = s_values[i];
            if (n == 0) continue;
            const unsigned mag = (i & (kCounters / 2 - 1)) + base;
            add(__uint_as_float((mag | (i >= kCounters / 2 ? 0x8000u : 0u)) << 16), n);
        }
    } else {
        for (int c0 = lo + tid; c0 < hi; c0 += U * kThreads) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c0 + u * kThreads >= hi) break;
#pragma unroll
                for (int e = 0; e < N; ++e) add(v[u][e], 1);
            }
            fetch(c0 + U * kThreads);
        }
    }
    if (!bins) {
        sum = wave_sum64(sum);
        if (lane == 0) s_part[wave] = sum;
        __syncthreads();
        if (tid == 0) p.part_sum[row * kSampleParts + part] = (s_part[0] + s_part[1]) + (s_part[2] + s_part[3]);
        return;
    }
    __syncthreads();
    u64 *h = p.hist + row * (2 * kSampleBins), *own = p.part_hist + (row * p.parts + part) * kSampleBins;
    for (int i = tid; i < kSampleBins; i += kThreads) {
        if (sums) own[i] = s_sum[i];
        if (s_sum[i] != 0) atomicAdd(h + 2 * i, s_sum[i]);
        if (s_count[i] != 0) atomicAdd(h + 2 * i + 1, static_cast<u64>(s_count[i]));
    }
}

using Borders = SampleBorders;

// By one wave, from a row's bins: 8 in turn a lane.
__device__ __forceinline__ Borders borders_of(const RowState &s, const u64 *hist, int lane)
{
    constexpr int E = kSampleBins / 64;
    u64 sum[E], count[E], own_s = 0, own_c = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const ulonglong2 h = *reinterpret_cast<const ulonglong2 *>(hist + 2 * (lane * E + e));
        sum[e] = own_s += h.x;
        count[e] = own_c += h.y;
    }
    const u64 base_s = wave_scan64(own_s, lane) - own_s, base_c = wave_scan64(own_c, lane) - own_c;
    Borders r;
    r.total = __shfl(base_s + own_s, 63, 64);
    const u64 all = __shfl(base_c + own_c, 63, 64);
    // The first lane whose condition holds for some bin, and that bin: bins are in order, so
    // the least bin over the wave.
    auto least = [&](int b) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_xor(b, o, 64);
            b = b < y ? b : y;
        }
        return b;
    };
    auto before = [&](int b, u64 &ps, u64 &pc) {  // sums before bin b
        u64 a = 0, c = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane * E + e == b) {
                a = base_s + (e ? sum[e - 1] : 0);
                c = base_c + (e ? count[e - 1] : 0);
            }
        ps = wave_sum64(a);
        pc = wave_sum64(c);
    };
    r.k_bin = -1;
    r.k_sum = r.k_count = 0;
    u64 lo_sum = r.total, hi_sum = r.total;  // bounds of what top-k leaves
    int last = kSampleBins - 1;
    if (s.k > 0 && static_cast<u64>(s.k) < all) {
        int b = kSampleBins;
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if (base_c + count[e] >= static_cast<u64>(s.k)) b = lane * E + e;
        r.k_bin = last = least(b);
        before(r.k_bin, r.k_sum, r.k_count);
        lo_sum = r.k_sum;
        u64 dummy;
        hi_sum = r.total;
        if (r.k_bin + 1 < kSampleBins) before(r.k_bin + 1, hi_sum, dummy);
    }
    r.p_lo = kSampleBins;
    r.p_hi = -1;
    r.p_sum = 0;
    r.sure = r.k_bin >= 0 ? r.k_bin : kSampleBins;
    if (s.share < 1.0) {
        // An element is kept if what precedes it is less than the share: a whole bin if even
        // its end is, none of it if its beginning is not.
        const double low = s.share * static_cast<double>(lo_sum), high = s.share * static_cast<double>(hi_sum);
        int a = kSampleBins, b = kSampleBins;
#pragma unroll
        for (int e = E - 1; e >= 0; --e) {
            if (!(static_cast<double>(base_s + sum[e]) < low)) a = lane * E + e;
            if (!(static_cast<double>(base_s + (e ? sum[e - 1] : 0)) < high)) b = lane * E + e;
        }
        a = least(a);
        b = least(b) - 1;
        r.p_lo = a < last ? a : last;
        r.p_hi = b < last ? b : last;
        u64 dummy;
        before(r.p_lo, r.p_sum, dummy);
        r.sure = r.p_lo < r.sure ? r.p_lo : r.sure;
    }
    return r;
}

// The logit where bin b begins, moved by a little more than the roundings: logits above it with SIGN -1, of
// bins up to b - 1, below it with 1, of bins from b on.
template <int SIGN>
__device__ __forceinline__ float edge_of(const RowState &s, int b)
{
    if (b >= kSampleBins || !(s.scale > 0.0f)) return SIGN < 0 ? -INFINITY : INFINITY;
    const double y = -static_cast<double>(b) / static_cast<double>(s.scale) * (1.0 - SIGN * 1e-5) + SIGN * 1e-5;
    const double x = static_cast<double>(s.top) + y / s.per;
    return static_cast<float>(x + SIGN * 1e-6 * (x < 0.0 ? -x : x));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleParams p)
{
    constexpr int N = Logits<T>::N, U = 4;
    __shared__ u64 s_part[kThreads / 64];
    __shared__ unsigned s_n;
    __shared__ Borders s_borders;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / p.parts;
    const int part = static_cast<int>(blockIdx.x - row * p.parts);
    const Logits<T> x(p, row);
    int lo, hi;
    part_range(p, x.pieces, part, lo, hi);
    float v[U][N];
    auto fetch = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * kThreads < hi) x.load(c0 + u * kThreads, v[u]);
    };
    fetch(lo + tid);  // in flight while the borders are found
    const RowState s = row_state(p, row, lane);
    if (s.greedy || !filters(s)) return;
    if (wave == 0) {
        const Borders found = borders_of(s, p.hist + row * (2 * kSampleBins), lane);
        if (lane == 0) {
            s_borders = found;
            if (part == 0) p.borders[row] = found;
        }
    }
    // A list of each part's own (one for the row, and its number added to by every wave, took 40 us of 64 rows of 32000).
    u64 *list = p.list + (row * p.parts + part) * p.list_len;
    if (tid == 0) s_n = 0;
    __syncthreads();
    const Borders b = s_borders;
    // What is kept for certain is summed from the part's own bins, or (few) with the listed bins' elements.
    const bool binned = binned_sums(s);
    const int need = b.p_hi > b.k_bin ? b.p_hi : b.k_bin;  // no bin past this one is wanted
    const float cut = edge_of<-1>(s, (need > b.sure - 1 ? need : b.sure - 1) + 1);
    const float high = binned ? edge_of<1>(s, b.sure) : INFINITY;
    u64 sum = 0;
    if (binned) {
        const u64 *own = p.part_hist + (row * p.parts + part) * kSampleBins;
        for (int i = tid; i < b.sure; i += kThreads) sum += own[i];
    }
    for (int c0 = lo + tid; c0 < hi; c0 += U * kThreads) {
        // Which of the thread's elements may count, then those one after another, of all lanes together.
        unsigned mask = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c0 + u * kThreads >= hi) break;
#pragma unroll
            for (int e = 0; e < N; ++e) mask |= v[u][e] >= cut && v[u][e] <= high && v[u][e] > -INFINITY ? 1u << (u * N + e) : 0u;
        }
        fetch(c0 + U * kThreads);
        while (__ballot(mask != 0)) {
            const int bit = mask ? __ffs(mask) - 1 : 0;
            const int i = x.first(c0 + bit / N * kThreads) + bit % N;
            bool have = false;
            u64 key = 0;
            if (mask) {
                const float a = io<T>::ld(x.x, i);
                const double y = log_weight(s, a);
                const int bin = bin_of(s, y);
                if (counts(y) && ((bin < b.sure && !binned) || b.listed(bin))) {
                    const u64 w = weight_of(y);
                    if (w >= s.least) {
                        sum += bin < b.sure ? w : 0;
                        have = bin >= b.sure;  // listed bins are not below `sure`
                        key = Key<T>::of(a, i);
                    }
                }
            }
            const u64 all = __ballot(have);
            if (all) {
                unsigned at = 0;
                if (lane == 0) at = atomicAdd(&s_n, static_cast<unsigned>(__popcll(all)));
                at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((1ull << lane) - 1));
                if (have && at < static_cast<unsigned>(p.list_len)) list[at] = key;
            }
            mask &= mask - 1;
        }
    }
    sum = wave_sum64(sum);
    if (lane == 0) s_part[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        p.part_sum[row * kSampleParts + part] = (s_part[0] + s_part[1]) + (s_part[2] + s_part[3]);
        p.part_listed[row * kSampleParts + part] = s_n;
    }
}

template <typename T>
__global__ __launch_bounds__(kFinish) void sample_finish_kernel(SampleParams p)
{
    constexpr int N = Logits<T>::N, kW = kFinish / 64;
    __shared__ u64 s_sum[256], s_count[256], s_part[kSampleParts], s_wave[kW];
    __shared__ u64 s_pick[4], s_last, s_least[2], s_total;
    __shared__ ulonglong2 s_list[kPairs];
    __shared__ unsigned s_upto[64];
    __shared__ int s_found;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const RowState s = row_state(p, row, lane);
    const Logits<T> x(p, row);
    // The first of the largest: the token of a greedy row.
    auto first_top = [&]() {
        const float own = lane < p.parts ? p.part_top[row * kSampleParts + lane].x : 0.0f;
        const u64 have = __ballot(lane < p.parts && (own == s.top || (own != own && s.top != s.top)));
        int lo, hi;
        part_range(p, x.pieces, __ffsll(have) - 1, lo, hi);
        if (tid == 0) s_found = x.n;
        __syncthreads();
        for (int c = lo + tid; c < hi; c += kFinish) {
            float v[N];
            x.load(c, v);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = x.first(c) + e;
                if (i >= 0 && i < x.n && (v[e] == s.top || (v[e] != v[e] && s.top != s.top))) atomicMin(&s_found, i);
            }
        }
        __syncthreads();
        if (tid == 0) p.out[row] = s_found;
    };
    if (s.greedy) {
        first_top();
        return;
    }
    if (tid < kSampleParts) s_part[tid] = tid < p.parts ? p.part_sum[row * kSampleParts + tid] : 0;
    if (tid == 0) s_found = 0;
    u64 thr = 0;  // the last kept key
    if (filters(s)) {
        const Borders b = p.borders[row];
        // The parts' lists, one after another.
        const unsigned have = lane < p.parts ? p.part_listed[row * kSampleParts + lane] : 0;
        const unsigned upto = static_cast<unsigned>(wave_scan64(have, lane)), n = __shfl(upto, 63, 64);
        const bool from_list = n <= static_cast<unsigned>(kSampleList) &&
                               !__any(have > static_cast<unsigned>(p.list_len));
        if (wave == 0) s_upto[lane] = upto;
        __syncthreads();
        u64 own[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const unsigned at = tid + i * kFinish;
            own[i] = 0;  // no element's key is 0
            if (from_list && at < n) {
                int part = 0;
#pragma unroll
                for (int step = 32; step > 0; step >>= 1) part += s_upto[part + step - 1] <= at ? step : 0;
                const unsigned before = part > 0 ? s_upto[part - 1] : 0;
                own[i] = p.list[(row * p.parts + part) * p.list_len + (at - before)];
            }
        }
        // f(key, weight, bin) of the listed bins' elements, from the list or the row.
        auto each = [&](auto f) __attribute__((always_inline)) {
            if (from_list) {
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    if (own[i] == 0) continue;
                    const double y = log_weight(s, Key<T>::value(own[i]));
                    f(own[i], weight_of(y), bin_of(s, y));
                }
            } else {
                for (int c = tid; c < x.pieces; c += kFinish) {
                    float v[N];
                    x.load(c, v);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const double y = log_weight(s, v[e]);
                        if (!counts(y)) continue;
                        const int bin = bin_of(s, y);
                        if (!b.listed(bin)) continue;
                        const u64 w = weight_of(y);
                        if (w >= s.least) f(Key<T>::of(v[e], x.first(c) + e), w, bin);
                    }
                }
            }
        };
        // The last of the elements in bins lo .. hi with keys from `least` on before which there is
        // less than the target (`by_sum`: of sum, else of number), `sum0` and `count0` preceding them all.
        // By 8 bits of the key at a time, from the highest in which the elements differ (where they agree, all would
        // meet in one counter).  `sum0` becomes the sum up to and with it.
        auto select = [&](bool by_sum, double target, int lo, int hi, u64 least, u64 &sum0, u64 count0) {
            u64 low = ~0ull, high = 0;
            each([&](u64 key, u64, int bin) __attribute__((always_inline)) {
                if (bin < lo || bin > hi || key < least) return;
                low = key < low ? key : low;
                high = key > high ? key : high;
            });
            __syncthreads();  // s_least is read
            if (tid == 0) {
                s_least[0] = ~0ull;
                s_least[1] = 0;
            }
            __syncthreads();
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 a = shfl_xor64(low, o), b2 = shfl_xor64(high, o);
                low = a < low ? a : low;
                high = b2 > high ? b2 : high;
            }
            if (lane == 0 && high > 0) {
                atomicMin(&s_least[0], low);
                atomicMax(&s_least[1], high);
            }
            __syncthreads();
            low = s_least[0];
            high = s_least[1];
            if (high == 0) return ~0ull;  // none
            int known = low == high ? 8 : 64 - __clzll(static_cast<long long>(low ^ high));  // the bits from here on agree
            known = known < 8 ? 8 : known;
            u64 prefix = high >> known;
            for (;;) {
                const int shift = known > 8 ? known - 8 : 0;
                __syncthreads();
                if (tid < 256) s_sum[tid] = s_count[tid] = 0;
                __syncthreads();
                each([&](u64 key, u64 w, int bin) __attribute__((always_inline)) {
                    if (bin < lo || bin > hi || key < least || key >> known != prefix) return;
                    const int d = 255 - static_cast<int>((key >> shift) & 255);
                    atomicAdd(&s_sum[d], w);
                    atomicAdd(&s_count[d], 1ull);
                });
                __syncthreads();
                if (wave == 0) {
                    // Digits from the highest down, four in turn a lane.
                    u64 a[4], c[4], as = 0, cs = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = s_sum[4 * lane + e];
                        c[e] = s_count[4 * lane + e];
                        as += a[e];
                        cs += c[e];
                    }
                    u64 bs = sum0 + wave_scan64(as, lane) - as, bc = count0 + wave_scan64(cs, lane) - cs;
                    int best = -1;
                    u64 best_s = 0, best_c = 0, best_n = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (c[e] > 0 && (by_sum ? static_cast<double>(bs) : static_cast<double>(bc)) < target) {
                            best = 4 * lane + e;
                            best_s = bs;
                            best_c = bc;
                            best_n = c[e];
                        }
                        bs += a[e];
                        bc += c[e];
                    }
                    int top = best;
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) {
                        const int y = __shfl_xor(top, o, 64);
                        top = top > y ? top : y;
                    }
                    if (top >= 0 && best == top) {
                        s_pick[0] = top;
                        s_pick[1] = best_s;
                        s_pick[2] = best_c;
                        s_pick[3] = best_n;
                    }
                    if (top < 0 && lane == 0) s_pick[0] = 256;
                }
                __syncthreads();
                if (s_pick[0] == 256) return ~0ull;  // none
                // The digit's upper bits are known ones where fewer than 8 were left.
                prefix = prefix << (known - shift) | ((255 - s_pick[0]) & ((1ull << (known - shift)) - 1));
                known = shift;
                sum0 = s_pick[1];
                count0 = s_pick[2];
                if (s_pick[3] == 1 || shift == 0) {
                    // A single element is left: its own key, as others than these elements may share
                    // the digits so far.
                    sum0 += s_sum[static_cast<int>(s_pick[0])];
                    each([&](u64 key, u64, int bin) __attribute__((always_inline)) {
                        if (bin >= lo && bin <= hi && key >= least && key >> shift == prefix) s_last = key;
                    });
                    __syncthreads();
                    return s_last;
                }
            }
        };
        if (from_list && n <= static_cast<unsigned>(kPairs)) {
            // Every element against every other: how many of top-k's bin, and what sum of top-p's, lie before
            // it; thread (i, q) compares element i with each n2-th of the others.
            const u64 mine = own[0];
            u64 w = 0;
            int bin = 0;
            if (mine) {
                const double y = log_weight(s, Key<T>::value(mine));
                w = weight_of(y);
                bin = bin_of(s, y);
            }
            if (tid == 0) {
                s_total = b.k_bin >= 0 ? b.k_sum : b.total;
                s_least[0] = s_least[1] = ~0ull;
            }
            if (tid < kPairs) {
                s_list[tid] = make_ulonglong2(mine, w);
                s_sum[tid] = s_count[tid] = 0;
            }
            __syncthreads();
            unsigned n2 = 64;
            while (n2 < n) n2 *= 2;
            const unsigned i = tid & (n2 - 1);
            const u64 key = s_list[i].x;
            u64 before = 0, number = 0;
            for (unsigned j = tid / n2; j < n; j += kFinish / n2) {
                const ulonglong2 o = s_list[j];
                const bool more = o.x > key;
                before += more ? o.y : 0;
                number += more ? 1 : 0;
            }
            atomicAdd(&s_sum[i], before);
            atomicAdd(&s_count[i], number);
            __syncthreads();
            const bool in_k = mine && bin == b.k_bin, in_p = mine && bin >= b.p_lo && bin <= b.p_hi;
            before = tid < kPairs ? b.p_sum + s_sum[tid] : 0;
            number = tid < kPairs ? b.k_count + s_count[tid] : 0;
            // What was counted of the other border's bins: top-p's lie before top-k's, or are the same.
            const u64 all = static_cast<u64>(__syncthreads_count(in_p && !in_k));
            const bool kept_k = mine && (!in_k || number - all < static_cast<u64>(s.k));
            if (in_k && kept_k) {
                atomicAdd(&s_total, w);
                atomicMin(&s_least[0], mine);
            }
            __syncthreads();
            const double most = s.share * static_cast<double>(s_total);
            if (in_p && kept_k && (s.share >= 1.0 || static_cast<double>(before) < most)) atomicMin(&s_least[1], mine);
            __syncthreads();
            if (b.k_bin >= 0) thr = s_least[0];
            if (s.share < 1.0) thr = s_least[1] == ~0ull ? ~0ull : (thr > s_least[1] ? thr : s_least[1]);
        } else {
            u64 total = b.total;
            if (b.k_bin >= 0) {
                total = b.k_sum;
                thr = select(false, static_cast<double>(s.k), b.k_bin, b.k_bin, 0, total, b.k_count);
            }
            if (s.share < 1.0) {
                u64 sum = b.p_sum;
                const u64 at = select(true, s.share * static_cast<double>(total), b.p_lo, b.p_hi, thr, sum, 0);
                // No listed element is kept: the border lies at the end of the bins before.
                thr = at == ~0ull ? ~0ull : (thr > at ? thr : at);
            }
        }
        __syncthreads();
        // What the list adds to the parts.
        each([&](u64 key, u64 w, int bin) __attribute__((always_inline)) {
            if (key >= thr && bin >= b.sure)
                atomicAdd(&s_part[(Key<T>::index(key) + x.off) / N / p.part_pieces], w);
        });
        if (thr == ~0ull) {
            // Elements of whole bins are told by their bin alone.
            thr = 0;
            s_pick[0] = b.sure;
        } else {
            s_pick[0] = kSampleBins;
        }
    } else {
        s_pick[0] = kSampleBins;
    }
    __syncthreads();
    const int bins = static_cast<int>(s_pick[0]);
    // The part that holds u times the total (every wave by itself), and what is left of it there.
    const u64 own = lane < kSampleParts ? s_part[lane] : 0;
    const u64 upto = wave_scan64(own, lane), total = __shfl(upto, 63, 64);
    const float u = p.u[row];
    const double share = u > 0.0f ? static_cast<double>(u) * static_cast<double>(total) : 0.0;
    u64 target = share < static_cast<double>(total) ? static_cast<u64>(share) : total;
    if (target >= total) target = total > 0 ? total - 1 : 0;
    const u64 past = __ballot(upto > target);
    const int part = past ? __ffsll(past) - 1 : 0;
    target -= __shfl(upto - own, part, 64);
    int lo, hi;
    part_range(p, x.pieces, part, lo, hi);
    // The element: running sums of the part's pieces, one a thread.
    u64 run = 0;
    for (int c0 = lo; c0 < hi; c0 += kFinish) {
        const int c = c0 + tid;
        u64 w[N], mine = 0;
        if (c < hi) {
            float v[N];
            x.load(c, v);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const double y = log_weight(s, v[e]);
                w[e] = 0;
                if (counts(y) && Key<T>::of(v[e], x.first(c) + e) >= thr && bin_of(s, y) < bins) {
                    const u64 a = weight_of(y);
                    w[e] = a >= s.least ? a : 0;
                }
                mine += w[e];
            }
        }
        const u64 in = wave_scan64(mine, lane);
        if (lane == 63) s_wave[wave] = in;
        __syncthreads();
        u64 base = run, all = run;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            const u64 y = s_wave[i];
            base += i < wave ? y : 0;
            all += y;
        }
        u64 at = base + in - mine;
        if (mine > 0 && at <= target && target < base + in) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (w[e] > 0 && at <= target && target < at + w[e]) {
                    p.out[row] = x.first(c) + e;
                    s_found = 1;
                }
                at += w[e];
            }
        }
        run = all;
        __syncthreads();  // s_wave is read
        if (run > target) break;
    }
    __syncthreads();
    const bool found = s_found;
    __syncthreads();
    if (!found) first_top();  // not reached: the parts' sums are the sums of their elements
}

template <typename T>
hipError_t sample_t(const SampleParams &p, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>(p.rows * p.parts));
    hipLaunchKernelGGL((sample_max_kernel<T>), grid, dim3(kThreads), 0, s, p);
    hipError_t e = hipGetLastError();
    // What the settings given to all rows make needless is not launched.
    const bool greedy = !p.temperature && !(p.temperature_all > 0.0f);
    const bool filtered = p.top_k || p.top_p || p.top_k_all > 0 || p.top_p_all < 1.0f;
    if (e == hipSuccess && !greedy) {
        hipLaunchKernelGGL((sample_hist_kernel<T>), grid, dim3(kThreads), 0, s, p);
        e = hipGetLastError();
        if (e == hipSuccess && filtered) {
            hipLaunchKernelGGL((sample_gather_kernel<T>), grid, dim3(kThreads), 0, s, p);
            e = hipGetLastError();
        }
    }
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((sample_finish_kernel<T>), dim3(static_cast<unsigned>(p.rows)), dim3(kFinish), 0, s, p);
    return hipGetLastError();
}

}  // namespace

// Parts of a row: enough workgroups for the card, none under 4096 elements (4 x 151936: 30 us, of 2048 32), at most a wave's lanes.
int sample_parts(int64_t rows, int64_t n)
{
    const int64_t most = (n + 4095) / 4096;
    int64_t c = (2048 + rows - 1) / rows;
    c = c < most ? c : most;
    return static_cast<int>(c < 1 ? 1 : (c > kSampleParts ? kSampleParts : c));
}

static int sample_list(int64_t n) { return static_cast<int>(n < kSamplePartList ? n : kSamplePartList); }

// A row's workspace: bins; its parts' lists, bins, sums, largest and least logits and numbers listed; borders.
size_t sample_workspace(int64_t rows, int64_t n)
{
    const int64_t parts = sample_parts(rows, n);
    return rows * (2 * kSampleBins * sizeof(u64) + parts * (sample_list(n) + kSampleBins) * sizeof(u64) +
                   kSampleParts * (sizeof(u64) + sizeof(float2) + sizeof(unsigned)) + sizeof(SampleBorders));
}

hipError_t launch_sample(SampleParams p, void *workspace, int io_dtype, hipStream_t s)
{
    u64 *w = static_cast<u64 *>(workspace);
    p.parts = sample_parts(p.rows, p.n);
    p.list_len = sample_list(p.n);
    p.hist = w;
    w += p.rows * 2 * kSampleBins;
    p.list = w;
    w += p.rows * p.parts * p.list_len;
    p.part_sum = w;
    w += p.rows * kSampleParts;
    p.part_hist = w;
    w += p.rows * p.parts * kSampleBins;
    p.borders = reinterpret_cast<SampleBorders *>(w);
    w = reinterpret_cast<u64 *>(p.borders + p.rows);
    p.part_top = reinterpret_cast<float2 *>(w);
    p.part_listed = reinterpret_cast<unsigned *>(p.part_top + p.rows * kSampleParts);
    const int per = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    const int pieces = (p.n + per - 1) / per + 1;  // of a row at any alignment
    p.part_pieces = (pieces + p.parts - 1) / p.parts;
    switch (io_dtype) {
    case GDN2_DTYPE_F32: return sample_t<float>(p, s);
    case GDN2_DTYPE_BF16: return sample_t<bf16_t>(p, s);
    default: return sample_t<f16_t>(p, s);
    }
}

}  // namespace gdn2

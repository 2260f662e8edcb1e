// Log probabilities of given tokens from a row of logits, with the row's
// entropy and its most probable alternatives, and their gradient, gfx950.
//
//   lse = m + ln sum_j e^(x_j - m),  logp = x_t - lse,
//   H = -sum_j p_j ln p_j = ln S - U / S  with  S = sum e^(x - m), U = sum (x - m) e^(x - m)
//   d x_j = -p_j (g_logp + g_H (ln p_j + H)) + g_logp [j = t]
//
// The forward reads the logits once.  A row is cut into parts, one wave each; a
// wave walks its part in chunks of 64 lanes x kU 16-byte pieces held in
// registers: the chunk's maximum first, then one exponential per element, with
// per-lane running (maximum, S, U).  Alternatives: the k-th largest of the 64
// lane maxima (its upper bits, found by ballots) bounds the k-th largest element from
// below, so few elements of the first chunk pass it; they meet in an LDS list, whose k best are found by
// counting, and later chunks need to beat the list's last.  An element is
// ordered by (value, lower index first), NaN above everything, in one 64-bit key.
// A second launch merges the parts of a row (one wave per row); rows of one part
// finish in the first.  Bound by the read: per element about nine issue slots
// (a hardware exponential is four of them) against the ten to fourteen that
// the memory leaves per bf16 element.
#include "gdn2_common.h"
#include "gdn2_internal.h"

namespace gdn2 {
namespace {

constexpr int kU = 8;         // pieces per lane and chunk
constexpr int kCand = 256;    // entries of a wave's candidate list
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef unsigned long long u64;

// Order-preserving key: larger value first, of equal ones (-0 = 0) the lower
// index, NaN above everything.  0 is below every element.
__device__ __forceinline__ u64 key_of(float v, unsigned idx)
{
    const unsigned b = __float_as_uint(v + 0.0f);
    unsigned k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    if (v != v) k = 0xffffffffu;
    return (static_cast<u64>(k) << 32) | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_value(u64 key)
{
    const unsigned k = static_cast<unsigned>(key >> 32);
    if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned key_index(u64 key) { return 0xffffffffu - static_cast<unsigned>(key); }

template <typename T>
struct Piece {
    static constexpr int N = 16 / static_cast<int>(sizeof(T));
    static __device__ __forceinline__ void widen(uint4 u, float (&f)[N])
    {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same<T, bf16_t>::value) {
                    f[2 * i] = __uint_as_float(w[i] << 16);
                    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                } else {
                    f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] & 0xffffu)));
                    f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
                }
            }
        }
    }
};

// Running (maximum, S, U) of a lane, U in base-2 units.
struct Stat {
    float m, s, u;
};
__device__ __forceinline__ void rebase(Stat &a, float m)
{
    if (m == a.m) return;  // also both -inf
    const float d = (a.m - m) * kL2e;
    const float r = __builtin_amdgcn_exp2f(d);
    a.u = a.s == 0.0f ? 0.0f : r * fmaf(d, a.s, a.u);
    if (r == 0.0f) a.u = 0.0f;  // d may be -inf
    a.s *= r;
    a.m = m;
}
__device__ __forceinline__ void add_element(Stat &a, float x)
{
    // NaN and +inf are kept out of m; they make S NaN or infinite, and the row NaN at the end.
    const float t = (x - a.m) * kL2e;
    const float e = __builtin_amdgcn_exp2f(t);
    a.s += e;
    a.u = fmaf(fmaxf(t, -1000.0f), e, a.u);  // x = -inf: 0, not 0 * inf
}
__device__ __forceinline__ Stat merge(Stat a, Stat b)
{
    const float m = fmaxf(a.m, b.m);
    rebase(a, m);
    rebase(b, m);
    return {m, a.s + b.s, a.u + b.u};
}
__device__ __forceinline__ Stat wave_merge(Stat a)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        Stat b = {__shfl_xor(a.m, o, 64), __shfl_xor(a.s, o, 64), __shfl_xor(a.u, o, 64)};
        // Both partners add in the same order: every lane ends with the same bits.
        a = (threadIdx.x & o) ? merge(b, a) : merge(a, b);
    }
    return a;
}

// The wave's candidate list: n entries of `list` (LDS, this wave's own).
struct Top {
    u64 *list;
    int n, k;
    float last;   // with n >= k after keep_best: the k-th best value
    bool sorted;  // nothing was appended since keep_best
};

// Keeps the k best of the list, in order.
__device__ __forceinline__ void keep_best(Top &t, int lane)
{
    if (t.sorted) return;
    t.sorted = true;
    wave_fence();
    u64 own[kCand / 64];
    int rank[kCand / 64];
#pragma unroll
    for (int i = 0; i < kCand / 64; ++i) {
        own[i] = lane + 64 * i < t.n ? t.list[lane + 64 * i] : 0;
        rank[i] = 0;
    }
    if (t.n <= 64) {
        for (int j = 0; j < t.n; ++j) rank[0] += t.list[j] > own[0];
    } else {
        for (int j = 0; j < t.n; ++j) {
            const u64 x = t.list[j];
#pragma unroll
            for (int i = 0; i < kCand / 64; ++i) rank[i] += x > own[i];
        }
    }
    wave_fence();
#pragma unroll
    for (int i = 0; i < kCand / 64; ++i)
        if (lane + 64 * i < t.n && rank[i] < t.k) t.list[rank[i]] = own[i];  // keys differ: ranks are a permutation
    wave_fence();
    t.n = t.n < t.k ? t.n : t.k;
    t.last = t.n == t.k ? key_value(t.list[t.k - 1]) : -INFINITY;
}

// Appends the keys of the lanes with `have`.
__device__ __forceinline__ void push(Top &t, bool have, u64 key, int lane)
{
    const u64 mask = __ballot(have);
    if (!mask) return;
    if (t.n + 64 > kCand) keep_best(t, lane);
    if (have) t.list[t.n + __popcll(mask & ((1ull << lane) - 1))] = key;
    t.n += __popcll(mask);
    t.sorted = false;
}

// A lower bound of the k-th largest of the lanes' ordered values (key_of's high
// word), its upper 16 bits found bit by bit by counting lanes: a filter, which may let a
// few more elements through than the exact value would.
__device__ __forceinline__ unsigned kth_bound(unsigned mine, int k)
{
    unsigned t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned trial = t | (1u << bit);
        if (__popcll(__ballot(mine >= trial)) >= k) t = trial;
    }
    return t;
}

__device__ __forceinline__ int64_t row_offset(const LogprobParams &p, int64_t row)
{
    const int64_t b = row / p.inner;
    return b * p.outer_stride + (row - b * p.inner) * p.row_stride;
}

// Leading elements of a row before its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T *x, int64_t n)
{
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15);
    const int h = off == 0 ? 0 : (16 - off) / static_cast<int>(sizeof(T));
    return h < n ? h : static_cast<int>(n);
}

// The row's results from its statistics and its sorted list of k keys.
template <typename T>
__device__ __forceinline__ void finish_row(const LogprobParams &p, int64_t row, Stat a, const u64 *list, int lane)
{
    // S is at most n unless an element was +inf: the formula's inf - inf.
    if (!(a.s < INFINITY)) a.s = __uint_as_float(0x7fc00000u);
    const float ln_s = __builtin_amdgcn_logf(a.s) * kLn2;
    if (lane == 0) {
        const int64_t t = p.targets[row];
        float lp = 0.0f;
        if (t >= 0 && t < p.n && t != p.ignore)
            lp = (io<T>::ld(static_cast<const T *>(p.x) + row_offset(p, row), t) - a.m) - ln_s;
        else if (t != p.ignore)
            lp = __uint_as_float(0x7fc00000u);
        p.logp[row] = lp;
        p.entropy[row] = ln_s - a.u / a.s * kLn2;
        if (p.lse) {
            p.lse[2 * row] = a.m;
            p.lse[2 * row + 1] = ln_s;
        }
    }
    if (lane < p.top) {
        const u64 key = list[lane];
        p.top_logp[row * p.top + lane] = (key_value(key) - a.m) - ln_s;
        p.top_ids[row * p.top + lane] = key_index(key);
    }
}

// 8192 x 32000 bf16, no alternatives: 114 us, 4.6 TB/s (20 alternatives: 163); 1000 x 151936
// float32, 5 alternatives: 127 us, 4.8 TB/s, as a large copy; 4 x 151936 bf16, 20
// alternatives: 11 us, a chain of one chunk's latencies.
template <typename T, bool TOP>
__global__ __launch_bounds__(64) void logp_part_kernel(LogprobParams p)
{
    constexpr int EPP = Piece<T>::N;
    __shared__ u64 s_list[TOP ? kCand : 1];
    const int lane = threadIdx.x;
    const unsigned r = blockIdx.x / p.parts;
    const int64_t row = p.row0 + r;
    const int part = static_cast<int>(blockIdx.x - r * p.parts);
    const T *x = static_cast<const T *>(p.x) + row_offset(p, row);
    const int head = head_of(x, p.n);
    const int64_t pieces = (p.n - head) / EPP;
    const int64_t c_lo = static_cast<int64_t>(part) * p.pieces_per_part;
    const int64_t c_hi = c_lo + p.pieces_per_part < pieces ? c_lo + p.pieces_per_part : pieces;
    const T *xa = x + head;  // 16-byte aligned
    Stat a = {-INFINITY, 0.0f, 0.0f};
    Top top = {s_list, 0, p.top, -INFINITY, true};
    // The row's ragged ends, one element per lane: what precedes the first
    // piece belongs to the first part and comes first, what follows the last
    // piece to the last part and comes last (the lists below rely on it: later
    // elements have higher indices).
    const int64_t tail0 = head + pieces * EPP;
    auto ragged = [&](int64_t i) __attribute__((always_inline)) {
        const float v = i >= 0 ? io<T>::ld(x, i) : -INFINITY;
        if (v != -INFINITY) {
            Stat b = {v < INFINITY ? v : -INFINITY, 0.0f, 0.0f};
            add_element(b, v);
            a = merge(a, b);
        }
        if constexpr (TOP) push(top, i >= 0, key_of(v, static_cast<unsigned>(i)), lane);
    };
    if (part == 0 && head > 0) ragged(lane < head ? lane : -1);
    bool first = true;
    // One chunk from piece c0 on; FULL: all 64 kU pieces are there, else the
    // missing ones are skipped (a lane's pieces by its own count, whole rows of 64 by branch).
    auto chunk = [&](int64_t c0, auto full_c) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full_c)::value;
        uint4 raw[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int64_t c = c0 + 64 * u + lane;
            if (FULL || c0 + 64 * u < c_hi) raw[u] = *reinterpret_cast<const uint4 *>(xa + (FULL || c < c_hi ? c : c_hi - 1) * EPP);
        }
        // Runs f(element, its number in the chunk) over the lane's elements.
        auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (!FULL && c0 + 64 * u >= c_hi) break;
                float v[EPP];
                Piece<T>::widen(raw[u], v);
                if (FULL || c0 + 64 * u + lane < c_hi)
#pragma unroll
                    for (int e = 0; e < EPP; ++e) f(v[e], u * EPP + e);
            }
        };
        float mx = -INFINITY;  // of this lane, NaN left out
        bool nan = false;
        each([&](float v, int) __attribute__((always_inline)) {
            mx = fmaxf(mx, v);
            if constexpr (TOP) nan |= v != v;
        });
        // +inf stays out of the reference (its terms are NaN, as the formula's).
        rebase(a, fmaxf(a.m, mx < INFINITY ? mx : -INFINITY));
        if (a.m == -INFINITY) {
            // Nothing finite yet: -inf adds nothing, +inf and NaN make the row NaN.
            each([&](float v, int) __attribute__((always_inline)) {
                if (v != -INFINITY) a.s = a.u = __uint_as_float(0x7fc00000u);
            });
        } else {
            float s0 = 0.0f, u0 = 0.0f;
            each([&](float v, int) __attribute__((always_inline)) {
                const float t = (v - a.m) * kL2e;
                const float ex = __builtin_amdgcn_exp2f(t);
                s0 += ex;
                u0 = fmaf(fmaxf(t, -1000.0f), ex, u0);  // t = -inf: 0, not inf * 0; t = NaN: ex is NaN
            });
            a.s += s0;
            a.u += u0;
        }
        if constexpr (TOP) {
            // Which of the chunk's elements may be among the k best: in the
            // first chunk those that reach (a bound of) the k-th largest lane
            // maximum, later those beyond the list's last (an equal one comes after it).
            const float lane_mx = nan ? __uint_as_float(0x7fc00000u) : mx;
            float thr = top.last;
            if (first)
                thr = key_value(static_cast<u64>(kth_bound(static_cast<unsigned>(key_of(lane_mx, 0) >> 32), p.top)) << 32);
            const bool strict = !first;
            const bool any = strict ? !(lane_mx <= thr) : !(lane_mx < thr);
            if (__ballot(any)) {
                u64 mask = 0;
                each([&](float v, int i) __attribute__((always_inline)) {
                    if (strict ? !(v <= thr) : !(v < thr)) mask |= 1ull << i;
                });
                if (!any) mask = 0;
                while (__ballot(mask != 0)) {
                    const bool have = mask != 0;
                    const int bit = have ? __ffsll(mask) - 1 : 0;
                    const int64_t c = c0 + 64 * (bit / EPP) + lane;
                    const int64_t i = c * EPP + bit % EPP;  // of xa
                    float v = 0.0f;
                    if (have) v = io<T>::ld(xa, i);
                    push(top, have, key_of(v, static_cast<unsigned>(i + head)), lane);
                    mask &= mask - 1;
                }
                keep_best(top, lane);
            }
            first = top.n < p.top;
        }
    };
    int64_t c0 = c_lo;
    for (; c0 + 64 * kU <= c_hi; c0 += 64 * kU) chunk(c0, std::true_type{});
    if (c0 < c_hi) chunk(c0, std::false_type{});
    if (part == p.parts - 1 && tail0 < p.n) ragged(tail0 + lane < p.n ? tail0 + lane : -1);
    a = wave_merge(a);
    if constexpr (TOP) keep_best(top, lane);
    if (p.parts == 1) {
        finish_row<T>(p, row, a, s_list, lane);
        return;
    }
    float *st = p.part_stat + (row * p.parts + part) * 4;
    if (lane < 3) st[lane] = lane == 0 ? a.m : lane == 1 ? a.s : a.u;
    if constexpr (TOP) {
        if (lane < p.top) p.part_top[(row * p.parts + part) * p.top + lane] = lane < top.n ? s_list[lane] : 0;
    }
}

// One wave per row: the parts' statistics and lists (37 parts of 20 keys: 6.8 us).
template <typename T, bool TOP>
__global__ __launch_bounds__(64) void logp_merge_kernel(LogprobParams p)
{
    __shared__ u64 s_list[TOP ? kCand : 1];
    const int lane = threadIdx.x;
    const int64_t row = p.row0 + blockIdx.x;
    Stat a = {-INFINITY, 0.0f, 0.0f};
    for (int i = lane; i < p.parts; i += 64) {
        const float4 st = *reinterpret_cast<const float4 *>(p.part_stat + (row * p.parts + i) * 4);
        a = merge(a, Stat{st.x, st.y, st.z});
    }
    a = wave_merge(a);
    Top top = {s_list, 0, p.top, -INFINITY, true};
    if constexpr (TOP) {
        // kB keys per lane at a time, requested together; the bound from the first of
        // them (the k-th largest of some is at most that of all) filters every one.
        constexpr int kB = 16;
        const u64 *src = p.part_top + row * p.parts * p.top;
        const int n = p.parts * p.top;
        u64 thr = 1;  // 0 is no element
        for (int i0 = 0; i0 < n; i0 += 64 * kB) {
            u64 key[kB];
#pragma unroll
            for (int b = 0; b < kB; ++b) {
                const int i = i0 + 64 * b + lane;
                key[b] = src[i < n ? i : n - 1];
                if (i >= n) key[b] = 0;
            }
            if (i0 == 0) {
                u64 best = 0;  // the lane's largest
#pragma unroll
                for (int b = 0; b < kB; ++b) best = key[b] > best ? key[b] : best;
                const u64 t = static_cast<u64>(kth_bound(static_cast<unsigned>(best >> 32), p.top)) << 32;
                thr = t > thr ? t : thr;
            }
#pragma unroll
            for (int b = 0; b < kB; ++b) push(top, key[b] >= thr, key[b], lane);
        }
        keep_best(top, lane);
    }
    finish_row<T>(p, row, a, s_list, lane);
}

// Gradient: one workgroup per (row, share of it).  VEC: rows of x and dx start
// at the same offset from a 16-byte boundary.  Reads the logits again and writes as much:
// 8192 x 32000 bf16 180 us, 5.8 TB/s; 1000 x 151936 float32 206 us, 5.9 TB/s.  Without VEC,
// an element at a time: 8192 x 50257 bf16 752 us, and 301 with it.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void logp_bwd_kernel(LogprobParams p)
{
    constexpr int EPP = Piece<T>::N;
    const unsigned r = blockIdx.x / p.parts;
    const int64_t row = p.row0 + r;
    const int64_t part = blockIdx.x - r * p.parts;
    const T *x = static_cast<const T *>(p.x) + row_offset(p, row);
    T *dx = static_cast<T *>(p.dx) + row * p.n;
    const int64_t t = p.targets[row];
    const bool known = t >= 0 && t < p.n && t != p.ignore;
    float gl = t != p.ignore && p.dlogp ? p.dlogp[row] : 0.0f;
    if (!known && gl != 0.0f) gl = __uint_as_float(0x7fc00000u);  // of a NaN; where none arrives, none passes
    const float ge = p.dent ? p.dent[row] : 0.0f;
    const float m = p.lse[2 * row], ln_s = p.lse[2 * row + 1], h = ge == 0.0f ? 0.0f : p.entropy[row];
    const bool nothing = gl == 0.0f && ge == 0.0f;  // no gradient arrives: zeros, whatever the logits
    auto grad = [&](float v, int64_t j) __attribute__((always_inline)) {
        const float lp = (v - m) - ln_s;
        const float pr = __builtin_amdgcn_exp2f(lp * kL2e);
        float d = pr == 0.0f ? 0.0f : -pr * (ge == 0.0f ? gl : fmaf(ge, lp + h, gl));
        if (j == t) d += gl;
        return d;
    };
    const int head = VEC ? head_of(x, p.n) : 0;
    const int64_t pieces = VEC ? (p.n - head) / EPP : 0;
    const int64_t lo = part * p.pieces_per_part;
    const int64_t hi = lo + p.pieces_per_part < pieces ? lo + p.pieces_per_part : pieces;
    if constexpr (VEC) {
        constexpr int W = 4;  // pieces requested together
        for (int64_t c0 = lo + threadIdx.x; c0 < hi; c0 += 256 * W) {
            uint4 raw[W];
            if (!nothing) {
#pragma unroll
                for (int u = 0; u < W; ++u) {
                    const int64_t c = c0 + 256 * u;
                    raw[u] = *reinterpret_cast<const uint4 *>(x + head + (c < hi ? c : c0) * EPP);
                }
            }
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const int64_t c = c0 + 256 * u;
                if (c >= hi) break;
                const int64_t j0 = head + c * EPP;
                uint4 out = make_uint4(0, 0, 0, 0);
                if (!nothing) {
                    float f[EPP];
                    Piece<T>::widen(raw[u], f);
#pragma unroll
                    for (int e = 0; e < EPP; ++e) f[e] = grad(f[e], j0 + e);
                    if constexpr (sizeof(T) == 4) {
                        out = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                         __float_as_uint(f[3]));
                    } else if constexpr (std::is_same<T, bf16_t>::value) {
                        out = make_uint4(f32x2_to_bf16x2_bits(f[0], f[1]), f32x2_to_bf16x2_bits(f[2], f[3]),
                                         f32x2_to_bf16x2_bits(f[4], f[5]), f32x2_to_bf16x2_bits(f[6], f[7]));
                    } else {
                        unsigned w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = static_cast<unsigned>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(f[2 * i]))) |
                                   (static_cast<unsigned>(
                                        __builtin_bit_cast(uint16_t, static_cast<_Float16>(f[2 * i + 1])))
                                    << 16);
                        out = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                *reinterpret_cast<uint4 *>(dx + j0) = out;
            }
        }
        // Ragged ends (fewer than a piece each).
        if (part == 0 && threadIdx.x < head) {
            const int64_t j = threadIdx.x;
            io<T>::st(dx, j, nothing ? 0.0f : grad(io<T>::ld(x, j), j));
        }
        const int64_t tail0 = head + pieces * EPP;
        if (part == p.parts - 1 && tail0 + threadIdx.x < p.n) {
            const int64_t j = tail0 + threadIdx.x;
            io<T>::st(dx, j, nothing ? 0.0f : grad(io<T>::ld(x, j), j));
        }
    } else {
        const int64_t e_lo = lo * EPP, e_end = e_lo + p.pieces_per_part * EPP;
        for (int64_t j = e_lo + threadIdx.x; j < e_end && j < p.n; j += 256)
            io<T>::st(dx, j, nothing ? 0.0f : grad(io<T>::ld(x, j), j));
    }
}

// launch(p, rows) over all rows, as many at a time as one launch of `threads` per part takes.
template <typename Launch>
hipError_t by_rows(LogprobParams p, int threads, Launch launch)
{
    const int64_t most = max_workgroups(threads) / p.parts;
    for (p.row0 = 0; p.row0 < p.rows; p.row0 += most) {
        launch(p, p.rows - p.row0 < most ? p.rows - p.row0 : most);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename T>
hipError_t fwd_launch(const LogprobParams &all, hipStream_t s)
{
    return by_rows(all, 64, [&](const LogprobParams &p, int64_t rows) {
        const dim3 grid(static_cast<unsigned>(rows * p.parts)), merges(static_cast<unsigned>(rows));
        if (p.top > 0)
            hipLaunchKernelGGL((logp_part_kernel<T, true>), grid, dim3(64), 0, s, p);
        else
            hipLaunchKernelGGL((logp_part_kernel<T, false>), grid, dim3(64), 0, s, p);
        if (p.parts == 1) return;
        if (p.top > 0)
            hipLaunchKernelGGL((logp_merge_kernel<T, true>), merges, dim3(64), 0, s, p);
        else
            hipLaunchKernelGGL((logp_merge_kernel<T, false>), merges, dim3(64), 0, s, p);
    });
}

template <typename T>
hipError_t bwd_launch(LogprobParams p, hipStream_t s)
{
    constexpr int EPP = Piece<T>::N;
    // Whole rows of x at the same offsets from 16-byte boundaries as dx's.
    const bool vec = ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dx)) & 15) == 0 &&
                     ((p.row_stride == p.n && (p.rows <= p.inner || p.outer_stride == p.inner * p.n)) ||
                      (p.n % EPP == 0 && (p.inner == 1 || p.row_stride % EPP == 0) &&
                       (p.rows <= p.inner || p.outer_stride % EPP == 0)));
    const int64_t pieces = (p.n + EPP - 1) / EPP;
    p.pieces_per_part = 2048;
    p.parts = static_cast<int>((pieces + p.pieces_per_part - 1) / p.pieces_per_part);
    return by_rows(p, 256, [&](const LogprobParams &p, int64_t rows) {
        const dim3 grid(static_cast<unsigned>(rows * p.parts));
        if (vec)
            hipLaunchKernelGGL((logp_bwd_kernel<T, true>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((logp_bwd_kernel<T, false>), grid, dim3(256), 0, s, p);
    });
}

}  // namespace

// Parts per row: enough waves to fill the card where rows are few, whole rows
// (no second launch) where they are many.
int logprob_parts(int64_t rows, int64_t n, int io_dtype)
{
    const int64_t epp = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    const int64_t most = (n / epp + 64 * kU - 1) / (64 * kU);
    int64_t want = rows > 0 ? (16384 + rows - 1) / rows : 1;
    want = want < most ? want : most;
    return static_cast<int>(want < 1 ? 1 : (want > 4096 ? 4096 : want));
}

hipError_t launch_logprobs(LogprobParams p, int io_dtype, hipStream_t s)
{
    const int64_t epp = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    const int64_t chunks = (p.n / epp + 64 * kU - 1) / (64 * kU);
    p.pieces_per_part = (chunks + p.parts - 1) / p.parts * (64 * kU);
    if (p.pieces_per_part == 0) p.pieces_per_part = 64 * kU;
    switch (io_dtype) {
    case GDN2_DTYPE_F32: return fwd_launch<float>(p, s);
    case GDN2_DTYPE_BF16: return fwd_launch<bf16_t>(p, s);
    default: return fwd_launch<f16_t>(p, s);
    }
}

hipError_t launch_logprobs_bwd(const LogprobParams &p, int io_dtype, hipStream_t s)
{
    switch (io_dtype) {
    case GDN2_DTYPE_F32: return bwd_launch<float>(p, s);
    case GDN2_DTYPE_BF16: return bwd_launch<bf16_t>(p, s);
    default: return bwd_launch<f16_t>(p, s);
    }
}

}  // namespace gdn2

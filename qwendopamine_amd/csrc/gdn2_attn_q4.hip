// Decode attention over a key / value cache held in 4 bits, gfx950: RoPE of the
// token's q and k, the store of its k and v as codes, and softmax attention over
// the cache up to each sequence's position; and the store and the read-back of
// whole prompts.
//
// A group of 64 channels shares a minimum and a scale (bf16 each):
//   min = bf16(min x), scale = bf16((max x - min) / 15), code = rint((x - min) / scale) in 0 .. 15,
// in fp32 with 1 / scale rounded once, so a code is the same on every path.  What
// attention sees is scale * code + min.
//
// Codes enter the matrix products without being converted: a nibble n shifted into
// the top of a 16-bit float's mantissa under the exponent of 1 is 1 + n / 16,
// exact, two elements per shift and and-or.  The offsets leave through fp32 sums:
//   q . k = sum_groups 16 scale (q . (1 + n/16) - sum q) + min sum q     (accumulators start at -sum q)
//   o_d   = sum_j P'_j (1 + n_jd/16) + sum_j (p_j min_j - P'_j),  P'_j = 16 p_j scale_j
// P' is split into two bf16 numbers (16 significant bits) and both halves are
// multiplied: one alone would leave an error of half a bf16 step of 1 + n/16,
// several times that of the values themselves.
//
// v_mfma_f32_16x16x32 throughout: a wave takes 32 positions a step, the group's
// query heads are the 16 columns.  Scores come out with 4 positions of one
// head per lane and tile, which is the B operand of the value product.  Bound
// by the read of the codes: D / 2 + 4 D / 64 bytes per position, k and v each.
#include "gdn2_common.h"
#include "gdn2_internal.h"
#include "gdn2_mfma.h"

namespace gdn2 {
namespace {

constexpr int kQ4Waves = 4;
constexpr int kStep = 32;  // positions per wave and step
constexpr float kNoMax = -3.0e38f;
constexpr float kLazy = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;

struct __attribute__((aligned(4))) U4 {
    unsigned x[4];
};

// 8 codes of a word as A operand: register r holds nibbles r and r + 4, each as 1 + n / 16.
template <PrecKind PK>
__device__ __forceinline__ uint4 codes_frag(unsigned w)
{
    if constexpr (PK == PrecKind::BF16) {
        constexpr unsigned M = 0x00780078u, E = 0x3f803f80u;
        return make_uint4(((w << 3) & M) | E, ((w >> 1) & M) | E, ((w >> 5) & M) | E, ((w >> 9) & M) | E);
    } else {
        constexpr unsigned M = 0x03c003c0u, E = 0x3c003c00u;
        return make_uint4(((w << 6) & M) | E, ((w << 2) & M) | E, ((w >> 2) & M) | E, ((w >> 6) & M) | E);
    }
}

// Nibble c of both halves of a word (two positions, one channel) as two bf16 1 + n / 16.
template <int C>
__device__ __forceinline__ unsigned pair_frag(unsigned w)
{
    constexpr unsigned M = 0x00780078u, E = 0x3f803f80u;
    constexpr int s = 3 - 4 * C;
    if constexpr (s >= 0)
        return ((w << s) & M) | E;
    else
        return ((w >> -s) & M) | E;
}

template <PrecKind PK>
__device__ __forceinline__ f32x4 mma16(f32x4 acc, uint4 a, uint4 b)
{
    typename Prec<PK>::frag fa, fb;
    fa.u = a;
    fb.u = b;
    return Prec<PK>::mma(acc, fa, fb);
}

__device__ __forceinline__ float rows_max(float x)
{
    unsigned u = __float_as_uint(x);
    auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    u = __float_as_uint(x);
    s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float rows_sum(float x)
{
    unsigned u = __float_as_uint(x);
    auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    u = __float_as_uint(x);
    s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Pair rotation with every product and sum rounded by itself, as torch's
// separate operations round (a fused multiply-add would move a code at its border).
template <typename T>
__device__ __forceinline__ void rotate(float x0, float x1, float c, float s, float &y0, float &y1)
{
#pragma clang fp contract(off)
    const float a = x0 * c, b = x1 * s, d = x0 * s, e = x1 * c;
    y0 = round_to<T>(a - b);
    y1 = round_to<T>(d + e);
}

// (scale, min) of a group from its extremes, as packed bf16 bits; a group with
// anything not finite gets NaN for both.
__device__ __forceinline__ unsigned group_meta(float lo, float hi, bool finite)
{
#pragma clang fp contract(off)
    if (!finite) return 0x7fc07fc0u;
    const unsigned mn = f32_to_bf16_bits(lo);
    const float sc = fmaxf((hi - __uint_as_float(mn << 16)) / 15.0f, 0.0f);
    return f32_to_bf16_bits(sc) | (mn << 16);
}
__device__ __forceinline__ float inv_scale(unsigned meta)
{
    const float sc = __uint_as_float(meta << 16);
    return sc > 0.0f ? 1.0f / sc : 0.0f;
}
__device__ __forceinline__ unsigned code_of(float x, unsigned meta, float inv)
{
#pragma clang fp contract(off)
    const float d = x - __uint_as_float(meta & 0xffff0000u);
    const float n = __builtin_rintf(d * inv);
    return n >= 15.0f ? 15u : (n > 0.0f ? static_cast<unsigned>(n) : 0u);  // NaN: 0
}

template <typename T, PrecKind PK, int D>
__global__ __launch_bounds__(64 * kQ4Waves) void attn_q4_kernel(AttnQ4Params p)
{
    constexpr int NG = D / 64, RB = D / 2;  // groups, bytes of a row of codes
    __shared__ __align__(16) float s_o[kQ4Waves][16][D];
    __shared__ float s_m[kQ4Waves][16], s_l[kQ4Waves][16];
    __shared__ __align__(16) uint16_t s_q[16][D];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const int bg = blockIdx.x, b = bg / p.G, qpk = p.qpk;
    const int64_t pos = p.pos[p.pos_stride * b];
    const int H = p.G * qpk;
    T *out = static_cast<T *>(p.out) + (static_cast<int64_t>(b) * H + (bg - b * p.G) * qpk) * D;
    float *part = p.part + (static_cast<int64_t>(bg) * p.splits + blockIdx.y) * qpk * (D + 2);
    const bool inside = pos >= 0 && pos < p.max_len;
    const int len = inside ? static_cast<int>(pos) + 1 : 0;
    // This workgroup's positions: whole steps of its waves.
    constexpr int kRound = kStep * kQ4Waves;
    const int rounds = (len + kRound - 1) / kRound;
    const int per = (rounds + p.splits - 1) / p.splits * kRound;
    const int lo = static_cast<int>(blockIdx.y) * per;
    const int hi = lo + per < len ? lo + per : len;
    if (lo >= hi) {
        // Nothing here: an empty partial state, or (outside the caches) zeros.
        for (int e = tid; e < qpk * D; e += 64 * kQ4Waves) {
            if (p.splits == 1) {
                io<T>::st(out, e, 0.0f);
            } else {
                const int h = e / D, d = e - h * D;
                part[h * (D + 2) + d] = 0.0f;
                if (d < 2) part[h * (D + 2) + D + d] = d == 0 ? kNoMax : 0.0f;
            }
        }
        return;
    }
    const T *x = static_cast<const T *>(p.qkv) + static_cast<int64_t>(bg) * (qpk + 2) * D;
    const int64_t row0 = static_cast<int64_t>(bg) * p.max_len;
    uint8_t *kc = p.k_codes + row0 * RB, *vc = p.v_codes + row0 * RB;
    unsigned *km = p.k_meta + row0 * NG, *vm = p.v_meta + row0 * NG;
    const float *cs = p.cos + p.rope_stride * pos, *sn = p.sin + p.rope_stride * pos;

    // ---- the token: q rotated into LDS; the workgroup that holds its position
    // rotates k, turns k and v into codes and stores them ----
    for (int e = tid; e < 16 * (D / 2); e += 64 * kQ4Waves) {
        const int h = e / (D / 2), i = e - h * (D / 2);
        float y0 = 0.0f, y1 = 0.0f;
        if (h < qpk) {
            y0 = io<T>::ld(x, h * D + 2 * i);
            y1 = io<T>::ld(x, h * D + 2 * i + 1);
            if (i < p.rope_pairs) rotate<T>(y0, y1, cs[i], sn[i], y0, y1);
        }
        s_q[h][2 * i] = Prec<PK>::from_f32(y0);
        s_q[h][2 * i + 1] = Prec<PK>::from_f32(y1);
    }
    if (hi == len) {
        for (int gi = wave; gi < 2 * NG; gi += kQ4Waves) {
            const int grp = gi % NG, ch = grp * 64 + lane;
            const bool is_k = gi < NG;
            float y = io<T>::ld(x, (is_k ? qpk : qpk + 1) * D + ch);
            if (is_k) {
                // Channel 2 i and 2 i + 1 of a pair lie in neighbouring lanes.
                const float other = __shfl_xor(y, 1, 64);
                const int i = ch >> 1;
                if (i < p.rope_pairs) {
                    float y0, y1;
                    rotate<T>(ch & 1 ? other : y, ch & 1 ? y : other, cs[i], sn[i], y0, y1);
                    y = ch & 1 ? y1 : y0;
                }
            }
            float mn = y, mx = y;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                mn = fminf(mn, __shfl_xor(mn, o, 64));
                mx = fmaxf(mx, __shfl_xor(mx, o, 64));
            }
            const bool finite = __ballot(!(fabsf(y) < INFINITY)) == 0;
            const unsigned meta = group_meta(mn, mx, finite);
            unsigned w = finite ? code_of(y, meta, inv_scale(meta)) << (4 * (lane & 7)) : 0u;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) w |= __shfl_xor(w, o, 64);
            uint8_t *dst = (is_k ? kc : vc) + pos * RB + grp * 32;
            if ((lane & 7) == 0) reinterpret_cast<unsigned *>(dst)[lane >> 3] = w;
            if (lane == 0) (is_k ? km : vm)[pos * NG + grp] = meta;
        }
    }
    __syncthreads();  // q in LDS; the token's codes visible to this workgroup

    // ---- q as B operand: MFMA (g, w) takes channels 64 g + 16 kg + 8 w + {0, 4, 1, 5, 2, 6, 3, 7} ----
    uint4 qf[NG][2];
    float qs[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint16_t *s = &s_q[n][64 * g + 16 * kg + 8 * w];
            unsigned r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = s[i] | (static_cast<unsigned>(s[i + 4]) << 16);
                sum += Prec<PK>::to_f32(s[i]) + Prec<PK>::to_f32(s[i + 4]);
            }
            qf[g][w] = make_uint4(r[0], r[1], r[2], r[3]);
        }
        qs[g] = rows_sum(sum);
    }
    const float c = p.scale * kLog2e;

    float m = kNoMax, l = 0.0f, corr[NG];
    f32x4 acc[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        corr[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] = zero4();
    }
    for (int j0 = lo + wave * kStep; j0 < hi; j0 += kRound) {
        // Requests of the step.  Positions past the end read the last one.
        uint2 kw[2][NG];
        unsigned vw[8][NG], mk[2][4 * NG], mv[2][4 * NG];
        const bool full = j0 + kStep <= hi;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            int j = j0 + 16 * a + n;
            j = j < hi ? j : hi - 1;
#pragma unroll
            for (int g = 0; g < NG; ++g)
                kw[a][g] = *reinterpret_cast<const uint2 *>(kc + static_cast<int64_t>(j) * RB + 32 * g + 8 * kg);
            const int jm = j0 + 16 * a + 4 * kg;
            if (full) {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const U4 uk = *reinterpret_cast<const U4 *>(km + static_cast<int64_t>(jm) * NG + 4 * g);
                    const U4 uv = *reinterpret_cast<const U4 *>(vm + static_cast<int64_t>(jm) * NG + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mk[a][4 * g + i] = uk.x[i];
                        mv[a][4 * g + i] = uv.x[i];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4 * NG; ++i) {
                    const bool in = jm + i / NG < hi;
                    const int64_t at = static_cast<int64_t>(in ? jm + i / NG : hi - 1) * NG + i % NG;
                    mk[a][i] = km[at];
                    mv[a][i] = in ? vm[at] : 0u;  // hidden: P' and p min are 0 whatever lies there
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int jv = jm + i;
                jv = jv < hi ? jv : hi - 1;
#pragma unroll
                for (int g = 0; g < NG; ++g)
                    vw[4 * a + i][g] = *reinterpret_cast<const uint16_t *>(vc + static_cast<int64_t>(jv) * RB + 32 * g + 2 * n);
            }
        }
        // Scores: 8 per lane, position j0 + 16 a + 4 kg + i of head n.
        float s[8];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * a + i] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 t = {-qs[g], -qs[g], -qs[g], -qs[g]};
                t = mma16<PK>(t, codes_frag<PK>(kw[a][g].x), qf[g][0]);
                t = mma16<PK>(t, codes_frag<PK>(kw[a][g].y), qf[g][1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned u = mk[a][i * NG + g];
                    const float sc16 = 16.0f * __uint_as_float(u << 16), mn = __uint_as_float(u & 0xffff0000u);
                    s[4 * a + i] = fmaf(sc16, t[i], fmaf(mn, qs[g], s[4 * a + i]));
                }
            }
        }
        if (!full) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                s[i] = j0 + 16 * (i >> 2) + 4 * kg + (i & 3) < hi ? s[i] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        mx = rows_max(mx) * c;
        if (__any(mx > m + kLazy)) {
            const float mn = fmaxf(m, mx);
            const float r = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= r;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                corr[g] *= r;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[g][i] *= r;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -m));
            l += s[i];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float ph[8], pl[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const unsigned u = mv[i >> 2][(i & 3) * NG + g];
                const float t = s[i] * (16.0f * __uint_as_float(u << 16));
                corr[g] += fmaf(s[i], __uint_as_float(u & 0xffff0000u), -t);
                ph[i] = t;
            }
            uint4 bh, bl;
            unsigned *h4 = &bh.x, *l4 = &bl.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h4[i] = f32x2_to_bf16x2_bits(ph[2 * i], ph[2 * i + 1]);
                pl[2 * i] = ph[2 * i] - __uint_as_float(h4[i] << 16);
                pl[2 * i + 1] = ph[2 * i + 1] - __uint_as_float(h4[i] & 0xffff0000u);
                l4[i] = f32x2_to_bf16x2_bits(pl[2 * i], pl[2 * i + 1]);
            }
            unsigned vp[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) vp[i] = vw[2 * i][g] | (vw[2 * i + 1][g] << 16);
            const uint4 a0 = make_uint4(pair_frag<0>(vp[0]), pair_frag<0>(vp[1]), pair_frag<0>(vp[2]), pair_frag<0>(vp[3]));
            const uint4 a1 = make_uint4(pair_frag<1>(vp[0]), pair_frag<1>(vp[1]), pair_frag<1>(vp[2]), pair_frag<1>(vp[3]));
            const uint4 a2 = make_uint4(pair_frag<2>(vp[0]), pair_frag<2>(vp[1]), pair_frag<2>(vp[2]), pair_frag<2>(vp[3]));
            const uint4 a3 = make_uint4(pair_frag<3>(vp[0]), pair_frag<3>(vp[1]), pair_frag<3>(vp[2]), pair_frag<3>(vp[3]));
            acc[g][0] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][0], a0, bh), a0, bl);
            acc[g][1] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][1], a1, bh), a1, bl);
            acc[g][2] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][2], a2, bh), a2, bl);
            acc[g][3] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][3], a3, bh), a3, bl);
        }
    }
    // ---- the waves' states meet in LDS ----
    l = rows_sum(l);
#pragma unroll
    for (int g = 0; g < NG; ++g) corr[g] = rows_sum(corr[g]);
    if (n < qpk) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)  // row 4 kg + i of product cc is channel 64 g + 4 (4 kg + i) + cc
                *reinterpret_cast<float4 *>(&s_o[wave][n][64 * g + 16 * kg + 4 * i]) =
                    make_float4(acc[g][0][i] + corr[g], acc[g][1][i] + corr[g], acc[g][2][i] + corr[g],
                                acc[g][3][i] + corr[g]);
        if (kg == 0) {
            s_m[wave][n] = m;
            s_l[wave][n] = l;
        }
    }
    __syncthreads();
    for (int e = tid; e < qpk * D; e += 64 * kQ4Waves) {
        const int h = e / D, d = e - h * D;
        float mx = kNoMax;
#pragma unroll
        for (int w = 0; w < kQ4Waves; ++w) mx = fmaxf(mx, s_m[w][h]);
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < kQ4Waves; ++w) {
            const float r = __builtin_amdgcn_exp2f(s_m[w][h] - mx);
            num = fmaf(s_o[w][h][d], r, num);
            den = fmaf(s_l[w][h], r, den);
        }
        if (p.splits == 1) {
            io<T>::st(out, e, num / den);
        } else {
            part[h * (D + 2) + d] = num;
            if (d == 0) {
                part[h * (D + 2) + D] = mx;
                part[h * (D + 2) + D + 1] = den;
            }
        }
    }
}

// The splits' partial states of one (sequence, head) per workgroup of D threads.
template <typename T, int D>
__global__ __launch_bounds__(D) void attn_q4_merge_kernel(AttnQ4Params p)
{
    const int d = threadIdx.x, h = static_cast<int>(blockIdx.x % p.qpk);
    const int64_t bg = blockIdx.x / p.qpk;
    const float *part = p.part + (bg * p.splits * p.qpk + h) * (D + 2);
    const int64_t stride = static_cast<int64_t>(p.qpk) * (D + 2);
    float mx = kNoMax;
    for (int s = 0; s < p.splits; ++s) mx = fmaxf(mx, part[s * stride + D]);
    float num = 0.0f, den = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float r = __builtin_amdgcn_exp2f(part[s * stride + D] - mx);
        num = fmaf(part[s * stride + d], r, num);
        den = fmaf(part[s * stride + D + 1], r, den);
    }
    // No position at all (outside the caches): zeros.
    io<T>::st(static_cast<T *>(p.out), static_cast<int64_t>(blockIdx.x) * D + d, den == 0.0f ? 0.0f : num / den);
}

// Whole prompts into the cache: 8 lanes per group of 64 channels, one 16-byte
// piece each; the lanes of a wave take 8 consecutive tokens of one group, whose
// codes are consecutive in the cache.
template <typename T>
__global__ __launch_bounds__(256) void q4_store_kernel(Q4StoreParams p)
{
    const int NG = p.D / 64;
    const int64_t tiles = (p.T + 7) / 8;
    const int64_t wv = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, e = lane & 7;
    // (which of k, v; batch; head; group; tile of 8 tokens), tiles fastest
    const int64_t per = tiles * NG * p.G * p.B;
    if (wv >= 2 * per) return;
    const bool is_k = wv < per;
    int64_t r = is_k ? wv : wv - per;
    const int64_t tile = r % tiles;
    r /= tiles;
    const int grp = static_cast<int>(r % NG);
    r /= NG;
    const int g = static_cast<int>(r % p.G), b = static_cast<int>(r / p.G);
    const int64_t t = tile * 8 + (lane >> 3);
    const int64_t pos = (p.start ? p.start[p.start_stride * b] : 0) + t;
    const bool in = t < p.T && pos >= 0 && pos < p.max_len;  // positions outside the cache are not stored
    const int64_t *st = is_k ? p.ks : p.vs;
    const T *x = static_cast<const T *>(is_k ? p.k : p.v) + b * st[0] + (t < p.T ? t : 0) * st[1] + g * st[2] + grp * 64 + e * 8;
    float v[8];
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(x)[0], c = reinterpret_cast<const float4 *>(x)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = c.x; v[5] = c.y; v[6] = c.z; v[7] = c.w;
    } else {
        constexpr PrecKind PK = std::is_same<T, bf16_t>::value ? PrecKind::BF16 : PrecKind::F16;
        typename Prec<PK>::frag f;
        f.u = *reinterpret_cast<const uint4 *>(x);
        unpack_frag<PK>(f, v);
    }
    float mn = v[0], mx = v[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, v[i]);
        mx = fmaxf(mx, v[i]);
        finite = finite && fabsf(v[i]) < INFINITY;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        mn = fminf(mn, __shfl_xor(mn, o, 64));
        mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    }
    finite = ((__ballot(!finite) >> (lane & ~7)) & 0xff) == 0;
    const unsigned meta = group_meta(mn, mx, finite);
    const float inv = inv_scale(meta);
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= code_of(v[i], meta, inv) << (4 * i);
    if (!finite) w = 0;
    if (!in) return;
    const int64_t row = (static_cast<int64_t>(b) * p.G + g) * p.max_len + pos;
    reinterpret_cast<unsigned *>((is_k ? p.k_codes : p.v_codes) + row * (p.D / 2) + grp * 32)[e] = w;
    if (e == 0) (is_k ? p.k_meta : p.v_meta)[row * NG + grp] = meta;
}

// What positions start .. start + T - 1 stand for, [B, T, G, D] in T (zeros
// outside the cache).  scale * code has 12 significant bits, so the sum is
// rounded once with or without fusing.
template <typename T>
__global__ __launch_bounds__(256) void q4_load_kernel(Q4LoadParams p)
{
    const int W = p.D / 8, NG = p.D / 64;
    const int64_t per = static_cast<int64_t>(p.B) * p.T * p.G * W;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= 2 * per) return;
    const bool is_k = i < per;
    const int64_t o = is_k ? i : i - per;
    int64_t r = o;
    const int w = static_cast<int>(r % W);
    r /= W;
    const int g = static_cast<int>(r % p.G);
    r /= p.G;
    const int64_t t = r % p.T;
    const int b = static_cast<int>(r / p.T);
    const int64_t pos = (p.start ? p.start[p.start_stride * b] : 0) + t;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (pos >= 0 && pos < p.max_len) {
        const int64_t row = (static_cast<int64_t>(b) * p.G + g) * p.max_len + pos;
        const unsigned u = reinterpret_cast<const unsigned *>((is_k ? p.k_codes : p.v_codes) + row * (p.D / 2))[w];
        const unsigned meta = (is_k ? p.k_meta : p.v_meta)[row * NG + w / 8];
        const float sc = __uint_as_float(meta << 16), mn = __uint_as_float(meta & 0xffff0000u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(static_cast<float>((u >> (4 * e)) & 15u), sc, mn);
    }
    T *y = static_cast<T *>(is_k ? p.k : p.v) + o * 8;
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        constexpr PrecKind PK = std::is_same<T, bf16_t>::value ? PrecKind::BF16 : PrecKind::F16;
        *reinterpret_cast<uint4 *>(y) = pack_frag<PK>(v).u;
    }
}

template <typename T, PrecKind PK, int D>
hipError_t decode_d(const AttnQ4Params &p, hipStream_t s)
{
    hipLaunchKernelGGL((attn_q4_kernel<T, PK, D>), dim3(static_cast<unsigned>(p.B * p.G), p.splits),
                       dim3(64 * kQ4Waves), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((attn_q4_merge_kernel<T, D>), dim3(static_cast<unsigned>(p.B * p.G * p.qpk)), dim3(D), 0, s, p);
    return hipGetLastError();
}

}  // namespace

int attn_q4_splits(int B, int G, int64_t max_len)
{
    // Enough workgroups for every CU, of at least two rounds of their waves.
    const int64_t most = (max_len + 2 * kStep * kQ4Waves - 1) / (2 * kStep * kQ4Waves);
    int64_t s = (1024 + static_cast<int64_t>(B) * G - 1) / (static_cast<int64_t>(B) * G);
    s = s < most ? s : most;
    return static_cast<int>(s < 1 ? 1 : (s > 256 ? 256 : s));
}

size_t attn_q4_workspace_floats(int B, int G, int qpk, int D, int64_t max_len)
{
    const int s = attn_q4_splits(B, G, max_len);
    return s == 1 ? 0 : static_cast<size_t>(B) * G * s * qpk * (D + 2);
}

bool attn_q4_supported(int io_dtype, int qpk, int D)
{
    return (io_dtype == GDN2_DTYPE_BF16 || io_dtype == GDN2_DTYPE_F16) && qpk >= 1 && qpk <= 16 && (D == 64 || D == 128);
}

hipError_t launch_attn_q4(const AttnQ4Params &p, int io_dtype, hipStream_t s)
{
    if (io_dtype == GDN2_DTYPE_BF16)
        return p.D == 64 ? decode_d<bf16_t, PrecKind::BF16, 64>(p, s) : decode_d<bf16_t, PrecKind::BF16, 128>(p, s);
    return p.D == 64 ? decode_d<f16_t, PrecKind::F16, 64>(p, s) : decode_d<f16_t, PrecKind::F16, 128>(p, s);
}

hipError_t launch_q4_store(const Q4StoreParams &p, int io_dtype, hipStream_t s)
{
    const int64_t waves = 2 * ((p.T + 7) / 8) * (p.D / 64) * p.G * p.B;
    const dim3 grid(static_cast<unsigned>((waves + 3) / 4));
    switch (io_dtype) {
    case GDN2_DTYPE_F32: hipLaunchKernelGGL((q4_store_kernel<float>), grid, dim3(256), 0, s, p); break;
    case GDN2_DTYPE_BF16: hipLaunchKernelGGL((q4_store_kernel<bf16_t>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((q4_store_kernel<f16_t>), grid, dim3(256), 0, s, p); break;
    }
    return hipGetLastError();
}

hipError_t launch_q4_load(const Q4LoadParams &p, int io_dtype, hipStream_t s)
{
    const int64_t threads = 2 * static_cast<int64_t>(p.B) * p.T * p.G * (p.D / 8);
    const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
    switch (io_dtype) {
    case GDN2_DTYPE_F32: hipLaunchKernelGGL((q4_load_kernel<float>), grid, dim3(256), 0, s, p); break;
    case GDN2_DTYPE_BF16: hipLaunchKernelGGL((q4_load_kernel<bf16_t>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((q4_load_kernel<f16_t>), grid, dim3(256), 0, s, p); break;
    }
    return hipGetLastError();
}

}  // namespace gdn2

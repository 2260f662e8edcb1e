// Decode attention over a key / value cache held in 4 bits, gfx950: RoPE of the
// token's q and k, the store of its k and v as codes, and softmax attention over
// the cache up to each sequence's position; and the store and the read-back of
// whole prompts.
//
// A group of 64 channels shares a minimum and a scale (bf16 each):
//   min = bf16(min x), scale = bf16((max x - min) (1 / 15)), code = rint((x - min) (1 / scale)) in 0 .. 15,
// in fp32 with both reciprocals rounded once (as torch divides by a number on the
// GPU), so a code is the same on every path.  What
// attention sees is scale * code + min.
//
// Codes enter the matrix products without being converted: a nibble n shifted into
// the top of a 16-bit float's mantissa under the exponent of 16 is 16 + n,
// exact, two elements per shift and and-or.  The offsets leave through fp32 sums:
//   q . k = sum_groups scale (q . (16 + n) - 16 sum q) + min sum q     (accumulators start at -16 sum q)
//   o_d   = sum_j P'_j (16 + n_jd) + sum_j p_j min_j - 16 sum_j P'_j,  P'_j = p_j scale_j
// P' is split into two bf16 numbers (16 significant bits) and both halves are
// multiplied: one alone would leave an error of half a bf16 step of 16 + n,
// several times that of the values themselves.
//
// v_mfma_f32_16x16x32 throughout, positions as rows, query heads as the 16 columns:
// scores come out with 4 positions of one head per lane and 16-position tile,
// which is the B operand of the value product.  With few heads per group the
// columns repeat them kSub = 16 / heads times, and column block u keeps only the
// scores of tile u: the work per score (scales, exponential, splitting P') is then
// done once and not kSub times over, and each column carries its own softmax
// state (4 heads per group, D = 128: 427 -> 257 vector instructions per 32
// positions).  Zeros in the other blocks keep a tile's P' to its columns.
// Bound by the read of the codes: D / 2 + 4 D / 64 bytes per position, k and v each.
#include "gdn2_common.h"
#include "gdn2_internal.h"
#include "gdn2_mfma.h"

namespace gdn2 {
namespace {

constexpr int kQ4Waves = 4;
constexpr int kQ4MaxSplits = 256;
constexpr float kNoMax = -3.0e38f;
constexpr float kLazy = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;

struct __attribute__((aligned(4))) U4 {
    unsigned x[4];
};

// Mask and exponent of "nibble n -> 16 + n", kept in registers (one scalar, one
// vector) so that v_and_or_b32 can take both: as literals they need two instructions.
struct Magic {
    unsigned mask, one;
};
template <PrecKind PK>
__device__ __forceinline__ Magic magic()
{
    Magic m = PK == PrecKind::BF16 ? Magic{0x00780078u, 0x41804180u} : Magic{0x03c003c0u, 0x4c004c00u};
    asm volatile("" : "+s"(m.mask));
    asm volatile("" : "+v"(m.one));
    return m;
}

// 8 codes of a word as A operand: register r holds nibbles r and r + 4, each as 16 + n.
template <PrecKind PK>
__device__ __forceinline__ uint4 codes_frag(unsigned w, Magic m)
{
    if constexpr (PK == PrecKind::BF16)
        return make_uint4(((w << 3) & m.mask) | m.one, ((w >> 1) & m.mask) | m.one, ((w >> 5) & m.mask) | m.one,
                          ((w >> 9) & m.mask) | m.one);
    else
        return make_uint4(((w << 6) & m.mask) | m.one, ((w << 2) & m.mask) | m.one, ((w >> 2) & m.mask) | m.one,
                          ((w >> 6) & m.mask) | m.one);
}

// Nibble C of both halves of four words (two positions each, one channel) as bf16 16 + n.
template <int C>
__device__ __forceinline__ uint4 pair_frag(const unsigned (&w)[4], Magic m)
{
    constexpr int s = 3 - 4 * C;
    unsigned r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = ((s >= 0 ? w[i] << (s >= 0 ? s : 0) : w[i] >> (s >= 0 ? 0 : -s)) & m.mask) | m.one;
    return make_uint4(r[0], r[1], r[2], r[3]);
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
    const float sc = fmaxf((hi - __uint_as_float(mn << 16)) * (1.0f / 15.0f), 0.0f);
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

// Positions per workgroup: whole rounds of its waves, the longest sequence over p.splits.
__device__ __forceinline__ int q4_share(const AttnQ4Params &p, int len, int lane)
{
    int longest = len;
    if (p.splits > 1 && p.pos_stride != 0) {
        for (int b = lane; b < p.B; b += 64) {
            const int64_t x = p.pos[p.pos_stride * b];
            if (x >= 0 && x < p.max_len) longest = longest > x + 1 ? longest : static_cast<int>(x) + 1;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_xor(longest, o, 64);
            longest = longest > y ? longest : y;
        }
    }
    const int rounds = (longest + p.round - 1) / p.round;
    return (rounds + p.splits - 1) / p.splits * p.round;
}

// kSub column blocks (1, 2 or 4).  B32 of unequal positions up to 32768, H32 G8 D128: 135 us,
// 4.5 TB/s of codes, scales and minima (a large copy: 4.8); B4 at 2074 of 2304, H16 D64: 7.8 us.
template <typename T, PrecKind PK, int D, int kSub>
__global__ __launch_bounds__(64 * kQ4Waves, 2) void attn_q4_kernel(AttnQ4Params p)
{
    constexpr int NG = D / 64, RB = D / 2;           // groups, bytes of a row of codes
    constexpr int kTiles = kSub < 2 ? 2 : kSub;      // 16-position tiles per step
    constexpr int kStep = 16 * kTiles, kRound = kStep * kQ4Waves;
    constexpr int kOwn = kTiles / kSub;              // tiles whose scores a lane keeps
    constexpr int kHeads = 16 / kSub;                // heads per column block
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
    // This workgroup's positions: share blockIdx.y of those of the longest
    // sequence, so that all workgroups that have any have equally many.
    const int per = q4_share(p, len, lane);
    const int sub = n / kHeads;  // this column's block
    const int lo = static_cast<int>(blockIdx.y) * per;
    const int hi = lo + per < len ? lo + per : len;
    if (lo >= hi) {
        // Nothing here (the merge does not read this share); outside the caches: zeros.
        if (p.splits == 1)
            for (int e = tid; e < qpk * D; e += 64 * kQ4Waves) io<T>::st(out, e, 0.0f);
        return;
    }
    const T *x = static_cast<const T *>(p.qkv) + static_cast<int64_t>(bg) * (qpk + 2) * D;
    const int64_t row0 = static_cast<int64_t>(bg) * p.max_len;
    uint8_t *kc = p.k_codes + row0 * RB, *vc = p.v_codes + row0 * RB;
    unsigned *km = p.k_meta + row0 * NG, *vm = p.v_meta + row0 * NG;
    const float *cs = p.cos + p.rope_stride * pos, *sn = p.sin + p.rope_stride * pos;

    // ---- a step's requests: codes of kStep positions, (scale, minimum) of the lane's share of them ----
    struct Step {
        uint2 k[kTiles][NG];
        unsigned v[4 * kTiles][NG], mk[kOwn][4 * NG], mv[kOwn][4 * NG];
    };
    const int64_t row = lo + wave * kStep;
    const uint8_t *kp = kc + (row + n) * RB + 8 * kg;
    const uint8_t *vp = vc + (row + 4 * kg) * RB + 2 * n;
    const unsigned *kmp = km + (row + 16 * kOwn * sub + 4 * kg) * NG;
    const unsigned *vmp = vm + (row + 16 * kOwn * sub + 4 * kg) * NG;
    // The step at the pointers, which then move to the wave's next.
    auto request = [&](Step &st) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < kTiles; ++a)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                st.k[a][g] = *reinterpret_cast<const uint2 *>(kp + 16 * a * RB + 32 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    st.v[4 * a + i][g] = *reinterpret_cast<const uint16_t *>(vp + (16 * a + i) * RB + 32 * g);
            }
#pragma unroll
        for (int a = 0; a < kOwn; ++a)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const U4 uk = *reinterpret_cast<const U4 *>(kmp + 16 * a * NG + 4 * g);
                const U4 uv = *reinterpret_cast<const U4 *>(vmp + 16 * a * NG + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    st.mk[a][4 * g + i] = uk.x[i];
                    st.mv[a][4 * g + i] = uv.x[i];
                }
            }
        kp += kRound * RB;
        vp += kRound * RB;
        kmp += kRound * NG;
        vmp += kRound * NG;
    };
    // A last step of fewer positions, from j0: those past the end read the last
    // one, and their values count for nothing whatever lies there.
    auto request_part = [&](Step &st, int j0) {
#pragma unroll
        for (int a = 0; a < kTiles; ++a) {
            int j = j0 + 16 * a + n;
            j = j < hi ? j : hi - 1;
#pragma unroll
            for (int g = 0; g < NG; ++g)
                st.k[a][g] = *reinterpret_cast<const uint2 *>(kc + static_cast<int64_t>(j) * RB + 32 * g + 8 * kg);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int jv = j0 + 16 * a + 4 * kg + i;
                jv = jv < hi ? jv : hi - 1;
#pragma unroll
                for (int g = 0; g < NG; ++g)
                    st.v[4 * a + i][g] =
                        *reinterpret_cast<const uint16_t *>(vc + static_cast<int64_t>(jv) * RB + 32 * g + 2 * n);
            }
        }
#pragma unroll
        for (int a = 0; a < kOwn; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int jm = j0 + 16 * (kOwn * sub + a) + 4 * kg + i;
                const bool in = jm < hi;
                const int64_t at = in ? jm : hi - 1;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    st.mk[a][i * NG + g] = km[at * NG + g];
                    st.mv[a][i * NG + g] = in ? vm[at * NG + g] : 0u;
                }
            }
    };
    const int jw = lo + wave * kStep;                                       // the wave's first position
    const int whole = hi - jw >= kStep ? (hi - jw - kStep) / kRound + 1 : 0;  // its whole steps
    Step cur;
    // The first step is requested before the token is worked on, unless the token is in it.
    const bool early = whole > 0 && jw + kStep < len;
    if (early) request(cur);

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
    float qs[NG], q16[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint16_t *s = &s_q[n % kHeads][64 * g + 16 * kg + 8 * w];
            unsigned r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = s[i] | (static_cast<unsigned>(s[i + 4]) << 16);
                sum += Prec<PK>::to_f32(s[i]) + Prec<PK>::to_f32(s[i + 4]);
            }
            qf[g][w] = make_uint4(r[0], r[1], r[2], r[3]);
        }
        qs[g] = rows_sum(sum);
        q16[g] = -16.0f * qs[g];
    }
    const float c = p.scale * kLog2e;
    const Magic mg_k = magic<PK>(), mg_v = magic<PrecKind::BF16>();

    float m = kNoMax, l = 0.0f, cm[NG], cp[NG];  // sums of p, of p min and of P'
    f32x4 acc[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        cm[g] = cp[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] = zero4();
    }
    // ---- one step; PART: the last one, of which positions from hi on are hidden ----
    auto step = [&](const Step &st, int j0, auto part_c) __attribute__((always_inline)) {
        constexpr bool PART = decltype(part_c)::value;
        // Scores: 4 per tile that the lane keeps, positions j0 + 16 tile + 4 kg + i.
        float s[4 * kOwn];
#pragma unroll
        for (int i = 0; i < 4 * kOwn; ++i) s[i] = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x4 t[kTiles];
#pragma unroll
            for (int a = 0; a < kTiles; ++a) {
                t[a] = f32x4{q16[g], q16[g], q16[g], q16[g]};
                t[a] = mma16<PK>(t[a], codes_frag<PK>(st.k[a][g].x, mg_k), qf[g][0]);
                t[a] = mma16<PK>(t[a], codes_frag<PK>(st.k[a][g].y, mg_k), qf[g][1]);
            }
            if constexpr (kSub > 1) {
#pragma unroll
                for (int a = 1; a < kTiles; ++a)
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[0][i] = sub == a ? t[a][i] : t[0][i];
            }
#pragma unroll
            for (int a = 0; a < kOwn; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned u = st.mk[a][i * NG + g];
                    const float sc = __uint_as_float(u << 16), mn = __uint_as_float(u & 0xffff0000u);
                    s[4 * a + i] = fmaf(sc, t[a][i], fmaf(mn, qs[g], s[4 * a + i]));
                }
        }
        if constexpr (PART) {
#pragma unroll
            for (int i = 0; i < 4 * kOwn; ++i)
                s[i] = j0 + 16 * (kOwn * sub + (i >> 2)) + 4 * kg + (i & 3) < hi ? s[i] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 4 * kOwn; ++i) mx = fmaxf(mx, s[i]);
        mx = rows_max(mx) * c;
        if (__any(mx > m + kLazy)) {
            const float mn = fmaxf(m, mx);
            const float r = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= r;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                cm[g] *= r;
                cp[g] *= r;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[g][i] *= r;
            }
        }
#pragma unroll
        for (int i = 0; i < 4 * kOwn; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -m));
            l += s[i];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            unsigned ph[2 * kOwn], pl[2 * kOwn];  // both halves of P', two positions per register
#pragma unroll
            for (int i = 0; i < 2 * kOwn; ++i) {
                float t[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int x = 2 * i + e;
                    const unsigned u = st.mv[x >> 2][(x & 3) * NG + g];
                    t[e] = s[x] * __uint_as_float(u << 16);
                    cp[g] += t[e];
                    cm[g] = fmaf(s[x], __uint_as_float(u & 0xffff0000u), cm[g]);
                }
                ph[i] = f32x2_to_bf16x2_bits(t[0], t[1]);
                pl[i] = f32x2_to_bf16x2_bits(t[0] - __uint_as_float(ph[i] << 16),
                                             t[1] - __uint_as_float(ph[i] & 0xffff0000u));
            }
#pragma unroll
            for (int cc = 0; cc < kTiles / 2; ++cc) {  // 32 positions: tiles 2 cc and 2 cc + 1
                uint4 bh, bl;
                if constexpr (kSub == 1) {
                    bh = make_uint4(ph[0], ph[1], ph[2], ph[3]);
                    bl = make_uint4(pl[0], pl[1], pl[2], pl[3]);
                } else {
                    const bool e0 = sub == 2 * cc, e1 = sub == 2 * cc + 1;
                    bh = make_uint4(e0 ? ph[0] : 0u, e0 ? ph[1] : 0u, e1 ? ph[0] : 0u, e1 ? ph[1] : 0u);
                    bl = make_uint4(e0 ? pl[0] : 0u, e0 ? pl[1] : 0u, e1 ? pl[0] : 0u, e1 ? pl[1] : 0u);
                }
                unsigned vp2[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    vp2[i] = st.v[8 * cc + 2 * i][g] | (st.v[8 * cc + 2 * i + 1][g] << 16);
                const uint4 a0 = pair_frag<0>(vp2, mg_v), a1 = pair_frag<1>(vp2, mg_v);
                const uint4 a2 = pair_frag<2>(vp2, mg_v), a3 = pair_frag<3>(vp2, mg_v);
                acc[g][0] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][0], a0, bh), a0, bl);
                acc[g][1] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][1], a1, bh), a1, bl);
                acc[g][2] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][2], a2, bh), a2, bl);
                acc[g][3] = mma16<PrecKind::BF16>(mma16<PrecKind::BF16>(acc[g][3], a3, bh), a3, bl);
            }
        }
    };
    // Two register sets in turn: the next step's requests are in flight during this one.
    if (!early && whole > 0) request(cur);
    Step alt;
    int it = 0;
    for (; it + 2 <= whole; it += 2) {
        request(alt);
        step(cur, 0, std::false_type{});
        if (it + 2 < whole) request(cur);
        step(alt, 0, std::false_type{});
    }
    if (it < whole) step(cur, 0, std::false_type{});
    const int j_end = jw + whole * kRound;
    if (j_end < hi) {
        request_part(cur, j_end);
        step(cur, j_end, std::true_type{});
    }
    // ---- the waves' states meet in LDS ----
    l = rows_sum(l);
#pragma unroll
    for (int g = 0; g < NG; ++g) cm[g] = rows_sum(fmaf(-16.0f, cp[g], cm[g]));
    if (n % kHeads < qpk) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)  // row 4 kg + i of product cc is channel 64 g + 4 (4 kg + i) + cc
                *reinterpret_cast<float4 *>(&s_o[wave][n][64 * g + 16 * kg + 4 * i]) =
                    make_float4(acc[g][0][i] + cm[g], acc[g][1][i] + cm[g], acc[g][2][i] + cm[g],
                                acc[g][3][i] + cm[g]);
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
        for (int w = 0; w < kQ4Waves * kSub; ++w) mx = fmaxf(mx, s_m[w / kSub][w % kSub * kHeads + h]);
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int w = 0; w < kQ4Waves * kSub; ++w) {
            const int col = w % kSub * kHeads + h;
            const float r = __builtin_amdgcn_exp2f(s_m[w / kSub][col] - mx);
            num = fmaf(s_o[w / kSub][col][d], r, num);
            den = fmaf(s_l[w / kSub][col], r, den);
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

// The shares' partial states of one (sequence, head) per workgroup: weights first
// (a thread each), then the values, 256 / D threads per channel.  4 to 6 us, its latency.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_q4_merge_kernel(AttnQ4Params p)
{
    constexpr int N = 256 / D;
    __shared__ float s_w[kQ4MaxSplits], s_red[4], s_den[4], s_num[N][D];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = static_cast<int>(blockIdx.x % p.qpk);
    const int64_t bg = blockIdx.x / p.qpk;
    const int64_t pos = p.pos[p.pos_stride * (bg / p.G)];
    const int len = pos >= 0 && pos < p.max_len ? static_cast<int>(pos) + 1 : 0;
    const int per = q4_share(p, len, lane);
    const int used = len > 0 ? (len + per - 1) / per : 0;  // shares that hold anything
    const float *part = p.part + (bg * p.splits * p.qpk + h) * (D + 2);
    const int64_t stride = static_cast<int64_t>(p.qpk) * (D + 2);
    const float mx = tid < used ? part[tid * stride + D] : kNoMax;
    float den = tid < used ? part[tid * stride + D + 1] : 0.0f;
    float m = mx;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (lane == 0) s_red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float w = __builtin_amdgcn_exp2f(mx - m);
    s_w[tid] = w;
    den = wave_sum(den * w);
    if (lane == 0) s_den[wave] = den;
    __syncthreads();
    const int d = tid % D, g = tid / D;
    float num = 0.0f;
#pragma unroll 8
    for (int s = g; s < used; s += N) num = fmaf(part[s * stride + d], s_w[s], num);
    s_num[g][d] = num;
    __syncthreads();
    if (tid >= D) return;
    den = (s_den[0] + s_den[1]) + (s_den[2] + s_den[3]);
#pragma unroll
    for (int i = 1; i < N; ++i) num += s_num[i][d];
    // No position at all (outside the caches): zeros.
    io<T>::st(static_cast<T *>(p.out), static_cast<int64_t>(blockIdx.x) * D + d, den == 0.0f ? 0.0f : num / den);
}

// ---- whole prompts in and out of the cache.  8 lanes per group of 64 channels, 8
// channels each; a wave takes 8 consecutive tokens at a time, whose codes are consecutive
// in the cache, and kQ4Tiles such tiles with all of their reads requested first.  A
// workgroup works on one (k or v, sequence, head, group).
constexpr int kQ4Tiles = 4;
constexpr int kQ4BlockTokens = 8 * kQ4Tiles * 4;

struct Q4Place {
    bool is_k;
    int b, g, grp;
    int64_t t0;  // this lane's first token; its others 8 on each
    int e;       // its 8 channels
};

__device__ __forceinline__ Q4Place q4_place(int64_t T, int B, int G, int NG)
{
    const unsigned blocks = static_cast<unsigned>((T + kQ4BlockTokens - 1) / kQ4BlockTokens);
    unsigned r = blockIdx.x / blocks;
    const unsigned blk = blockIdx.x - r * blocks;
    Q4Place x;
    x.grp = static_cast<int>(r % NG);
    r /= NG;
    x.g = static_cast<int>(r % G);
    r /= G;
    x.b = static_cast<int>(r % B);
    x.is_k = r / B == 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x.t0 = static_cast<int64_t>(blk) * kQ4BlockTokens + wave * (8 * kQ4Tiles) + (lane >> 3);
    x.e = lane & 7;
    return x;
}

template <typename T>
__device__ __forceinline__ void load8(const T *x, float (&v)[8])
{
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
}

// Codes, scales and minima of positions start .. start + T - 1.  B4 T2048 G16 D64 bf16
// (k and v): 15.1 us, 2.8 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void q4_store_kernel(Q4StoreParams p)
{
    const int NG = p.D / 64, lane = threadIdx.x & 63;
    const Q4Place at = q4_place(p.T, p.B, p.G, NG);
    const int64_t *st = at.is_k ? p.ks : p.vs;
    const T *x = static_cast<const T *>(at.is_k ? p.k : p.v) + at.b * st[0] + at.g * st[2] + at.grp * 64 + at.e * 8;
    const int64_t first = p.start ? p.start[p.start_stride * at.b] : 0;
    const int64_t row0 = (static_cast<int64_t>(at.b) * p.G + at.g) * p.max_len;
    unsigned *codes = reinterpret_cast<unsigned *>((at.is_k ? p.k_codes : p.v_codes) + at.grp * 32);
    unsigned *meta_out = (at.is_k ? p.k_meta : p.v_meta) + at.grp;
    float v[kQ4Tiles][8];
#pragma unroll
    for (int u = 0; u < kQ4Tiles; ++u) {
        const int64_t t = at.t0 + 8 * u;
        load8(x + (t < p.T ? t : 0) * st[1], v[u]);
    }
#pragma unroll
    for (int u = 0; u < kQ4Tiles; ++u) {
        float mn = v[u][0], mx = v[u][0];
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            mn = fminf(mn, v[u][i]);
            mx = fmaxf(mx, v[u][i]);
            finite = finite && fabsf(v[u][i]) < INFINITY;
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
        for (int i = 0; i < 8; ++i) w |= code_of(v[u][i], meta, inv) << (4 * i);
        if (!finite) w = 0;
        const int64_t t = at.t0 + 8 * u, pos = first + t;
        if (t < p.T && pos >= 0 && pos < p.max_len) {  // positions outside the cache are not stored
            codes[(row0 + pos) * (p.D / 8) + at.e] = w;
            if (at.e == 0) meta_out[(row0 + pos) * NG] = meta;
        }
    }
}

// What positions start .. start + T - 1 stand for, [B, T, G, D] in T (zeros
// outside the cache).  scale * code has 12 significant bits, so the sum is
// rounded once with or without fusing.  B4 T2048 G16 D64: 9.8 us, 4.4 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void q4_load_kernel(Q4LoadParams p)
{
    const int NG = p.D / 64;
    const Q4Place at = q4_place(p.T, p.B, p.G, NG);
    const int64_t first = p.start ? p.start[p.start_stride * at.b] : 0;
    const int64_t row0 = (static_cast<int64_t>(at.b) * p.G + at.g) * p.max_len;
    const unsigned *codes = reinterpret_cast<const unsigned *>((at.is_k ? p.k_codes : p.v_codes) + at.grp * 32);
    const unsigned *metas = (at.is_k ? p.k_meta : p.v_meta) + at.grp;
    unsigned w[kQ4Tiles], m[kQ4Tiles];
#pragma unroll
    for (int u = 0; u < kQ4Tiles; ++u) {
        const int64_t t = at.t0 + 8 * u, pos = first + t;
        const bool in = t < p.T && pos >= 0 && pos < p.max_len;
        const int64_t row = row0 + (in ? pos : 0);
        const unsigned cw = codes[row * (p.D / 8) + at.e], cm = metas[row * NG];
        w[u] = in ? cw : 0u;
        m[u] = in ? cm : 0u;
    }
#pragma unroll
    for (int u = 0; u < kQ4Tiles; ++u) {
        const int64_t t = at.t0 + 8 * u;
        if (t >= p.T) break;
        const float sc = __uint_as_float(m[u] << 16), mn = __uint_as_float(m[u] & 0xffff0000u);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(static_cast<float>((w[u] >> (4 * i)) & 15u), sc, mn);
        T *y = static_cast<T *>(at.is_k ? p.k : p.v) + ((at.b * p.T + t) * p.G + at.g) * p.D + at.grp * 64 + at.e * 8;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            constexpr PrecKind PK = std::is_same<T, bf16_t>::value ? PrecKind::BF16 : PrecKind::F16;
            *reinterpret_cast<uint4 *>(y) = pack_frag<PK>(v).u;
        }
    }
}

unsigned q4_blocks(int64_t T, int B, int G, int D)
{
    return static_cast<unsigned>(2 * ((T + kQ4BlockTokens - 1) / kQ4BlockTokens) * (D / 64) * G * B);
}

template <typename T, PrecKind PK, int D>
hipError_t decode_d(AttnQ4Params p, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>(p.B * p.G), p.splits), block(64 * kQ4Waves);
    p.round = (p.qpk <= 4 ? 64 : 32) * kQ4Waves;
    if (p.qpk <= 4)
        hipLaunchKernelGGL((attn_q4_kernel<T, PK, D, 4>), grid, block, 0, s, p);
    else if (p.qpk <= 8)
        hipLaunchKernelGGL((attn_q4_kernel<T, PK, D, 2>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((attn_q4_kernel<T, PK, D, 1>), grid, block, 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((attn_q4_merge_kernel<T, D>), dim3(static_cast<unsigned>(p.B * p.G * p.qpk)), dim3(256), 0, s,
                       p);
    return hipGetLastError();
}

}  // namespace

// Workgroups per (sequence, KV group): 512 in all (two per CU), more where a share
// would exceed 4096 positions of a full cache, so that sequences of unequal lengths
// even out; but shares of 512 positions or more, of 1024 where the sequences alone
// occupy half the card (a merge costs about 4 us).  us a call with 256 / 512 / 1024 /
// 2048 / 4096 workgroups wanted: 32 sequences of up to 32768, 8 groups of 4 heads, D128
// 198 / 171 / 156 / 137 / 146; 8 x 7373 positions, 16 groups, D64 21.4 / 20.2 / 22.0 / 25.0 / 24.8;
// 64 x 922 positions, 4 groups of 4, D128 13.2 / 18.8 / 18.6 / 18.6 / 18.7.
int attn_q4_splits(int B, int G, int64_t max_len)
{
    const int64_t bg = static_cast<int64_t>(B) * G;
    const int64_t least = bg < 128 ? 512 : 1024, most = (max_len + least - 1) / least;
    int64_t s = (512 + bg - 1) / bg;
    const int64_t by_share = (max_len + 4095) / 4096;
    s = s > by_share ? s : by_share;
    s = s < most ? s : most;
    return static_cast<int>(s < 1 ? 1 : (s > kQ4MaxSplits ? kQ4MaxSplits : s));
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
    const dim3 grid(q4_blocks(p.T, p.B, p.G, p.D));
    switch (io_dtype) {
    case GDN2_DTYPE_F32: hipLaunchKernelGGL((q4_store_kernel<float>), grid, dim3(256), 0, s, p); break;
    case GDN2_DTYPE_BF16: hipLaunchKernelGGL((q4_store_kernel<bf16_t>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((q4_store_kernel<f16_t>), grid, dim3(256), 0, s, p); break;
    }
    return hipGetLastError();
}

hipError_t launch_q4_load(const Q4LoadParams &p, int io_dtype, hipStream_t s)
{
    const dim3 grid(q4_blocks(p.T, p.B, p.G, p.D));
    switch (io_dtype) {
    case GDN2_DTYPE_F32: hipLaunchKernelGGL((q4_load_kernel<float>), grid, dim3(256), 0, s, p); break;
    case GDN2_DTYPE_BF16: hipLaunchKernelGGL((q4_load_kernel<bf16_t>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((q4_load_kernel<f16_t>), grid, dim3(256), 0, s, p); break;
    }
    return hipGetLastError();
}

}  // namespace gdn2

// Softmax attention over a paged key / value cache, gfx950: from one token of each
// sequence to pieces of prompts, every sequence at its own position.
//
//   o_t = sum_j p_tj v_j / sum_j p_tj,  p_tj = exp(scale q_t . k_j),  j <= pos + t
//   k_j, v_j: row j mod S of page table[b][j / S], pages [P][G][S][D]
//
// Few rows (a group's query heads times the tokens): v_mfma_f32_16x16x32, positions as rows and
// the rows of the group as columns, 16 C of them: a lane's 16 bytes of a key row are the A
// operand as they lie in memory, so keys go from memory to the matrix units
// without passing through LDS, and the scores come out with four positions of one
// column per lane, which is the B operand of the value product.  Its A operand
// has positions along the contraction: a lane takes CH = D / 16 channels of four
// rows and pairs them by byte permutes.  Waves take 32 positions at a time in
// turn, each with a running reference and sum of its own, and meet in LDS; long
// contexts are split into shares that a second launch joins.  A wave looks the
// pages of its next 32 steps up at once (a lane each), so that no key waits for
// a page number.  One token a sequence is bound by the read of its keys and values.
#include "gdn2_common.h"
#include "gdn2_internal.h"
#include "gdn2_mfma.h"
#include "gdn2_attn_tiles.h"

namespace gdn2 {
namespace {

constexpr int kWaves = 4;
constexpr int kStep = 32;               // positions of a wave's step: two tiles of 16
constexpr int kRound = kStep * kWaves;  // positions that a workgroup's waves take at a time
constexpr int kMaxSplits = 256;
constexpr unsigned kNoPage = 0xffffffffu;
constexpr int kTileRows = 32 * kWaves;  // rows of a workgroup whose keys lie in LDS

template <PrecKind PK>
__device__ __forceinline__ f32x4 mma16(f32x4 acc, uint4 a, uint4 b)
{
    typename Prec<PK>::frag fa, fb;
    fa.u = a;
    fb.u = b;
    return Prec<PK>::mma(acc, fa, fb);
}

// Over the four lanes of a column.
__device__ __forceinline__ float col_max(float x)
{
    unsigned u = __float_as_uint(x);
    auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    u = __float_as_uint(x);
    s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float col_sum(float x)
{
    unsigned u = __float_as_uint(x);
    auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    u = __float_as_uint(x);
    s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

template <PrecKind PK>
__device__ __forceinline__ unsigned pack2(float a, float b)
{
    if constexpr (PK == PrecKind::BF16)
        return f32x2_to_bf16x2_bits(a, b);
    else
        return Prec<PK>::from_f32(a) | static_cast<unsigned>(Prec<PK>::from_f32(b)) << 16;
}

// Requests from the 16 rows at `tile` (uniform), by the lane's offset: buffer requests take the base in
// scalar registers, where flat ones hold a 64-bit address a row in vector ones.
template <int N, int STEP>
__device__ __forceinline__ void load_rows(uint4 (&x)[N], const char *tile, unsigned off)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass does not know the builtins' types
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(tile), 0, 0x10000, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i)
        x[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + i * STEP, 0, 0));
#endif
}
template <int N>
__device__ __forceinline__ void load_row(unsigned (&x)[N], const char *tile, unsigned off)
{
#ifdef __HIP_DEVICE_COMPILE__
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(tile), 0, 0x10000, 0x00020000);
    if constexpr (N == 2) {
        const uint2 u = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, 0));
        x[0] = u.x;
        x[1] = u.y;
    } else {
        const uint4 u = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
        x[0] = u.x;
        x[1] = u.y;
        x[2] = u.z;
        x[3] = u.w;
    }
#endif
}

// What a workgroup works on: rows m0 .. of group g of sequence b, tokens t0 .. t1 - 1 of
// which are there, and their positions.
struct Where {
    int b, g, m0;
    int t0, t1;  // t1 <= t0: none
    int pos;     // position of token 0
    int n;       // keys that some row sees
};

// Tokens of sequence b that are there and inside the cache.
__device__ __forceinline__ int tokens_of(const AttnPagedParams &p, int b, int &pos)
{
    const int64_t at = p.pos[p.pos_stride * b], cap = p.cap;
    int64_t t = p.T;
    if (p.lengths) {
        const int64_t l = p.lengths[b];
        t = l < 0 ? 0 : l < t ? l : t;
    }
    if (at < 0 || at >= cap) {
        pos = 0;
        return 0;
    }
    pos = static_cast<int>(at);
    return static_cast<int>(t < cap - at ? t : cap - at);
}

__device__ __forceinline__ Where where(const AttnPagedParams &p, int rows, int bg, int tile)
{
    Where w;
    w.b = bg / p.G;
    w.g = bg - w.b * p.G;
    w.m0 = tile * rows;
    const int there = tokens_of(p, w.b, w.pos);
    const int all = p.T * p.R, last = (w.m0 + rows < all ? w.m0 + rows : all) - 1;
    w.t0 = w.m0 / p.R;
    const int t1 = last / p.R + 1;
    w.t1 = t1 < there ? t1 : there;
    w.n = w.t1 > w.t0 ? w.pos + w.t1 : 0;
    return w;
}

// Positions of a share: whole rounds, the longest sequence's keys over p.splits, so that all
// shares that hold any are equally long.
__device__ __forceinline__ int share_of(const AttnPagedParams &p, int lane)
{
    int longest = 1;
    for (int b = lane; b < p.B; b += 64) {
        int pos;
        const int t = tokens_of(p, b, pos);
        longest = t > 0 && pos + t > longest ? pos + t : longest;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_xor(longest, o, 64);
        longest = longest > y ? longest : y;
    }
    const int rounds = (longest + kRound - 1) / kRound;
    return (rounds + p.splits - 1) / p.splits * kRound;
}

// Rounds of sequence b, for a group of few rows (one workgroup holds them all).
__device__ __forceinline__ int rounds_of(const AttnPagedParams &p, int b)
{
    int pos;
    const int t = tokens_of(p, b, pos);
    return t > 0 ? (pos + t + kRound - 1) / kRound : 0;
}

// The sequences' rounds in a row, dealt to p.workers workgroups in equal runs, which may begin and end
// within a sequence (no run under kLeast): sequences of unequal lengths then keep all of them
// busy to the end.  Worker w's part of sequence b is slot w + b, as both only grow along the row.
constexpr int kLeast = 2;
// By a wave: the rounds before sequence `upto`.
__device__ __forceinline__ int rounds_before(const AttnPagedParams &p, int upto, int lane)
{
    int sum = 0;
    for (int b = lane; b < upto; b += 64) sum += rounds_of(p, b);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    return sum;
}
__device__ __forceinline__ int run_of(const AttnPagedParams &p, int total)
{
    const int r = (total + p.workers - 1) / p.workers;
    return r > kLeast ? r : kLeast;
}
// The sequence in which round `at` of all lies, and the rounds before it.
__device__ __forceinline__ int sequence_at(const AttnPagedParams &p, int at, int lane, int &before)
{
    int base = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int r = b0 + lane < p.B ? rounds_of(p, b0 + lane) : 0;
        int in = r;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(in, o, 64);
            in += lane >= o ? y : 0;
        }
        const uint64_t hit = __ballot(base + in > at);
        if (hit) {
            const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            before = base + __builtin_amdgcn_readlane(in - r, l);
            return b0 + l;
        }
        base += __builtin_amdgcn_readlane(in, 63);
    }
    before = base;  // not reached: `at` is less than all
    return p.B - 1;
}

// A row's place in a [B, T, H, ...] tensor's rows.
__device__ __forceinline__ int64_t out_row(const AttnPagedParams &p, const Where &w, int x)
{
    const int t = x / p.R;
    return (static_cast<int64_t>(w.b) * p.T + t) * (p.G * p.R) + w.g * p.R + (x - t * p.R);
}

// 32 tokens over contexts spread to 32768, H32 G8 D128, pages of 16: 370 us, 5.8 TB/s of keys and values (a large copy 5.2,
// equal contexts 6.1), and the join 7; 4 over 2074 of 2304, H16 D64: 13 us, four steps' latencies.
// C column tiles hold all the T R rows of a group.  SPREAD: workgroup (worker, group) takes its run of all
// sequences' rounds, and attn_paged_join_kernel joins the parts; else workgroup (b, group) one sequence.
template <typename T, PrecKind PK, int D, int C, bool SPREAD>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_paged_kernel(AttnPagedParams p)
{
    constexpr int KS = D / 32, CH = D / 16, VW = CH / 2;  // contraction steps, channels and dwords of a lane's value row
    constexpr int kRows = 16 * C;
    __shared__ __align__(16) float s_o[kWaves][16][D];
    __shared__ float s_m[kWaves][C][16], s_l[kWaves][C][16];
    __shared__ uint4 s_q[C * KS][64];  // the query operands: registers are for keys and values
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, kg = lane >> 4;
    const int g = blockIdx.y, all = p.T * p.R;
    T *out = static_cast<T *>(p.out);
    int b = blockIdx.x, from = 0, left = 0;  // this part: from round `from` of sequence b, `left` rounds to go in all
    if constexpr (SPREAD) {
        const int total = rounds_before(p, p.B, lane), run = run_of(p, total);
        const int64_t at = static_cast<int64_t>(blockIdx.x) * run;
        if (at >= total) return;
        int before;
        b = __builtin_amdgcn_readfirstlane(sequence_at(p, static_cast<int>(at), lane, before));
        from = __builtin_amdgcn_readfirstlane(static_cast<int>(at) - before);
        left = __builtin_amdgcn_readfirstlane(total - at < run ? total - static_cast<int>(at) : run);
    }
    for (;;) {
    Where w = where(p, kRows, b * p.G + g, 0);
    // In scalar registers, although loaded after stores.
    w.pos = __builtin_amdgcn_readfirstlane(w.pos);
    w.t1 = __builtin_amdgcn_readfirstlane(w.t1);
    w.n = __builtin_amdgcn_readfirstlane(w.n);
    const int lo = from * kRound;
    int hi = w.n;
    if constexpr (SPREAD) hi = (from + left) * kRound < w.n ? (from + left) * kRound : w.n;
    if (lo >= hi) {
        if constexpr (SPREAD) {  // a sequence without keys: on to the next
            if (++b >= p.B) return;
            continue;
        }
        for (int e = tid; e < all * D; e += 64 * kWaves) io<T>::st(out, out_row(p, w, e / D) * D + e % D, 0.0f);
        return;
    }

    // ---- this lane's columns: query rows as B operands, and the keys they see ----
    int lim[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        int x = 16 * c + n;
        const int end = w.t1 * p.R;
        x = x < end ? x : end - 1;  // rows past the end repeat the last one
        const int t = x / p.R;
        lim[c] = w.pos + t + 1;
        if (c % kWaves == wave) {
            const T *q = static_cast<const T *>(p.q) + w.b * p.qs[0] + t * p.qs[1] + (g * p.R + (x - t * p.R)) * p.qs[2];
#pragma unroll
            for (int s = 0; s < KS; ++s) s_q[c * KS + s][lane] = *reinterpret_cast<const uint4 *>(q + 32 * s + 8 * kg);
        }
    }
    const int seen = w.pos + w.t0 + 1;  // every row sees these

    // ---- pages: lane 2 i + a holds the row of the cache where tile a of the wave's step i begins ----
    const int steps = hi - lo > wave * kStep ? (hi - lo - wave * kStep + kRound - 1) / kRound : 0;
    const int *table = p.table + w.b * p.table_stride;
    auto look_up = [&](int base) __attribute__((always_inline)) {
        const int j = lo + ((base + (lane >> 1)) * kWaves + wave) * kStep + (lane & 1) * 16;
        unsigned r = kNoPage;
        if (j < hi) {
            const int col = j / p.page;
            const int64_t pg = table[col];
            if (pg >= 0 && pg < p.pages) r = static_cast<unsigned>((pg * p.G + w.g) * p.page + (j - col * p.page));
        }
        return r;
    };

    struct Step {
        uint4 k[2][KS];
        unsigned v[2][4][VW];
    };
    const char *kb = static_cast<const char *>(p.k), *vb = static_cast<const char *>(p.v);
    // Positions j0 .. j0 + 31, a tile of 16 from the row of the cache r0, the other from r1; those past the
    // last key read that one again.  A tile without a page reads row 0 of the cache, and is hidden.
    auto request = [&](Step &st, int j0, unsigned r0, unsigned r1) __attribute__((always_inline)) {
        const int end = w.n - 1 - j0;  // the last key, from j0
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const bool past = a && end < 16;  // no key in this tile: the other's
            const unsigned r = a && !past ? r1 : r0;
            const int last = end - (a && !past ? 16 : 0), top = last < 15 ? last : 15;
            const int64_t at = static_cast<int64_t>(r == kNoPage ? 0 : r) * (2 * D);
            const int rk = n < top ? n : top;
            load_rows<KS, 64>(st.k[a], kb + at, rk * (2 * D) + kg * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rv = 4 * kg + i < top ? 4 * kg + i : top;
                load_row<VW>(st.v[a][i], vb + at, rv * (2 * D) + n * (2 * CH));
            }
        }
    };

    const float scale = p.scale * kLog2e;
    float m[C], l[C];
    f32x4 acc[C][CH];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        m[c] = kNoMax;
        l[c] = 0.0f;
#pragma unroll
        for (int e = 0; e < CH; ++e) acc[c][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto step = [&](Step &st, int j0, bool bad0, bool bad1) __attribute__((always_inline)) {
        const bool hide = bad0 || bad1 || j0 + kStep > seen;
        if (bad0 || bad1) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    st.v[0][i][e] = bad0 ? 0u : st.v[0][i][e];
                    st.v[1][i][e] = bad1 ? 0u : st.v[1][i][e];
                }
        }
        uint4 ph[C], pl[C];
        const int at_q = opaque(lane);  // read anew at each step
#pragma unroll
        for (int c = 0; c < C; ++c) {
            uint4 qf[KS];
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] = s_q[c * KS + s][at_q];
            f32x4 t[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                t[a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < KS; ++s) t[a] = mma16<PK>(t[a], st.k[a][s], qf[s]);
            }
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = t[i >> 2][i & 3];
            if (hide) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int j = j0 + 16 * (i >> 2) + 4 * kg + (i & 3);
                    s[i] = j < lim[c] && !(i < 4 ? bad0 : bad1) ? s[i] : -INFINITY;
                }
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
            mx = col_max(mx) * scale;
            if (__any(mx > m[c] + (Ref<PK>::down + Ref<PK>::lazy))) {
                const float mn = fmaxf(m[c], mx - Ref<PK>::down);
                const float r = __builtin_amdgcn_exp2f(m[c] - mn);
                m[c] = mn;
                l[c] *= r;
#pragma unroll
                for (int e = 0; e < CH; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[c][e][i] *= r;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], scale, -m[c]));
                l[c] += s[i];
            }
            // Probabilities in two parts: rounded once they would cost half a step of the
            // result; the products are cheap beside the read.
            unsigned h[4], lw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = pack2<PK>(s[2 * i], s[2 * i + 1]);
                lw[i] = pack2<PK>(s[2 * i] - Prec<PK>::to_f32(static_cast<uint16_t>(h[i] & 0xffffu)),
                                  s[2 * i + 1] - Prec<PK>::to_f32(static_cast<uint16_t>(h[i] >> 16)));
            }
            ph[c] = make_uint4(h[0], h[1], h[2], h[3]);
            pl[c] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
        }
#pragma unroll
        for (int e = 0; e < CH; ++e) {
            const unsigned sel = e & 1 ? 0x07060302u : 0x05040100u;
            const uint4 a = make_uint4(__builtin_amdgcn_perm(st.v[0][1][e / 2], st.v[0][0][e / 2], sel),
                                       __builtin_amdgcn_perm(st.v[0][3][e / 2], st.v[0][2][e / 2], sel),
                                       __builtin_amdgcn_perm(st.v[1][1][e / 2], st.v[1][0][e / 2], sel),
                                       __builtin_amdgcn_perm(st.v[1][3][e / 2], st.v[1][2][e / 2], sel));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                acc[c][e] = mma16<PK>(acc[c][e], a, ph[c]);
                acc[c][e] = mma16<PK>(acc[c][e], a, pl[c]);
            }
        }
    };

    // ---- the steps, the next one's keys and values in flight during each ----
    Step cur, alt;
    unsigned next = look_up(0);
    if (steps == 0) __syncthreads();  // as the others below
    for (int base = 0; base < steps; base += 32) {
        const unsigned rows = next;
        if (base + 32 < steps) next = look_up(base + 32);
        const int cnt = steps - base < 32 ? steps - base : 32;
        const int jw = lo + (base * kWaves + wave) * kStep;
        auto row = [&](int i) __attribute__((always_inline)) {
            return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(rows), i));
        };
        auto get = [&](Step &st, int i) __attribute__((always_inline)) {
            request(st, jw + i * kRound, row(2 * i), row(2 * i + 1));
        };
        auto run = [&](Step &st, int i) __attribute__((always_inline)) {
            const int j0 = jw + i * kRound;
            // A tile past the last key has no page either, and is hidden by its positions; it
            // read the one before it.
            const bool bad = row(2 * i) == kNoPage;
            step(st, j0, bad, row(2 * i + 1) == kNoPage && (bad || j0 + 16 < hi));
        };
        get(cur, 0);
        if (base == 0) __syncthreads();  // the queries are there
        for (int i = 0; i < cnt; i += 2) {
            if (i + 1 < cnt) get(alt, i + 1);
            run(cur, i);
            if (i + 1 < cnt) {
                if (i + 2 < cnt) get(cur, i + 2);
                run(alt, i + 1);
            }
        }
    }

    // ---- the waves' states meet in LDS, a column tile at a time ----
#pragma unroll
    for (int c = 0; c < C; ++c) {
        l[c] = col_sum(l[c]);
        if (kg == 0) {
            s_m[wave][c][n] = m[c];
            s_l[wave][c][n] = l[c];
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (c > 0) __syncthreads();  // the last tile's sums are read
#pragma unroll
        for (int i = 0; i < 4; ++i)  // row 4 kg + i of product e is channel CH (4 kg + i) + e
#pragma unroll
            for (int e = 0; e < CH; e += 4)
                *reinterpret_cast<float4 *>(&s_o[wave][n][CH * (4 * kg + i) + e]) =
                    make_float4(acc[c][e][i], acc[c][e + 1][i], acc[c][e + 2][i], acc[c][e + 3][i]);
        __syncthreads();
        for (int e = tid; e < 16 * D; e += 64 * kWaves) {
            const int h = e / D, d = e - h * D, x = w.m0 + 16 * c + h;
            if (x >= all) continue;
            float mx = kNoMax;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) mx = fmaxf(mx, s_m[v][c][h]);
            float num = 0.0f, den = 0.0f;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const float r = __builtin_amdgcn_exp2f(s_m[v][c][h] - mx);
                num = fmaf(s_o[v][h][d], r, num);
                den = fmaf(s_l[v][c][h], r, den);
            }
            if constexpr (SPREAD) {
                float *part = p.part + ((static_cast<int64_t>(blockIdx.x + b) * p.G + g) * all + x) * (D + 2);
                part[d] = num;
                if (d == 0) {
                    part[D] = mx;
                    part[D + 1] = den;
                }
            } else {
                // Padding, and rows whose every key is without a page: zeros.
                io<T>::st(out, out_row(p, w, x) * D + d, x < w.t1 * p.R && den != 0.0f ? num / den : 0.0f);
            }
        }
    }
    if constexpr (!SPREAD) return;
    left -= (hi - lo + kRound - 1) / kRound;
    if (left <= 0 || ++b >= p.B) return;
    from = 0;
    __syncthreads();  // the next part overwrites what was read
    }
}

// The parts of one row: weights first (a thread each), then the values, 256 / D threads per channel.
constexpr int kMaxWorkers = 512;
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(AttnPagedParams p)
{
    constexpr int N = 256 / D, kEach = kMaxWorkers / 256;
    __shared__ float s_w[kMaxWorkers], s_red[4], s_den[4], s_num[N][D];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int H = p.G * p.R;
    const int64_t row = blockIdx.x;
    const int h = static_cast<int>(row % H), bt = static_cast<int>(row / H), b = bt / p.T, t = bt - b * p.T;
    const int g = h / p.R, x = t * p.R + (h - g * p.R);
    int pos;
    const int there = tokens_of(p, b, pos);
    const int total = rounds_before(p, p.B, lane), before = rounds_before(p, b, lane), run = run_of(p, total);
    const int first = before / run, last = (before + rounds_of(p, b) - 1) / run;  // workers
    const int used = t < there ? last - first + 1 : 0;
    const int64_t step = static_cast<int64_t>(p.G) * p.T * p.R * (D + 2);  // from one slot to the next
    const float *part = p.part + (first + b) * step + (static_cast<int64_t>(g) * p.T * p.R + x) * (D + 2);
    float mx[kEach], m = kNoMax, den = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = tid + 256 * i;
        mx[i] = s < used ? part[s * step + D] : kNoMax;
        m = fmaxf(m, mx[i]);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (lane == 0) s_red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = tid + 256 * i;
        const float r = __builtin_amdgcn_exp2f(mx[i] - m);
        s_w[s] = r;
        den = fmaf(s < used ? part[s * step + D + 1] : 0.0f, r, den);
    }
    den = wave_sum(den);
    if (lane == 0) s_den[wave] = den;
    __syncthreads();
    const int d = tid % D, k = tid / D;
    float num = 0.0f;
#pragma unroll 8
    for (int s = k; s < used; s += N) num = fmaf(part[s * step + d], s_w[s], num);
    s_num[k][d] = num;
    __syncthreads();
    if (tid >= D) return;
    den = (s_den[0] + s_den[1]) + (s_den[2] + s_den[3]);
#pragma unroll
    for (int i = 1; i < N; ++i) num += s_num[i][d];
    io<T>::st(static_cast<T *>(p.out), row * D + d, den == 0.0f ? 0.0f : num / den);
}

// ---- many rows: tiles of 64 positions in LDS, which 128 rows read ----

// A lane's place among the 16 rows of a page's piece, for the request that it makes of them (rows as
// they lie, their 16-byte pieces permuted as the tile's: swz).
template <int D>
struct Place {
    int row;            // of the piece
    unsigned piece16;   // byte within the row
    int sub;            // the request's piece of the tile, it adds kPer * it
    static constexpr int kP = D / 8, kR = 64 / kP, kIt = kTile / kR / kWaves;  // pieces, rows, requests of a wave
    static constexpr int kPer = kWaves * kR / 16;
    __device__ __forceinline__ Place(int wave, int lane)
    {
        const int r = wave * kR + lane / kP;
        row = r & 15;
        sub = r >> 4;
        piece16 = ((lane % kP) ^ swz<D>(r)) * 16;
    }
};

// Positions row0 .. row0 + 63 requested into LDS: piece a of 16 from the row of the cache that lane
// i0 + a of `rows` holds.  Positions past the last, n - 1, repeat it; a piece without a page is zeros.
template <int D>
__device__ __forceinline__ void stage_pages(const char *pool, unsigned rows, int i0, int row0, int n, bool plain, char *lds,
                                            const Place<D> &at, int wave, int lane)
{
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass does not know the builtins' types
    constexpr int IT = Place<D>::kIt, PER = Place<D>::kPer;
    typedef __attribute__((address_space(3))) char *lds_ptr;
    const int wsub = __builtin_amdgcn_readfirstlane(at.sub);
    auto load = [&](unsigned row, char *to, unsigned off) __attribute__((always_inline)) {
        // Raw buffer from this row on, 32-bit elements.
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char *>(pool + static_cast<uint64_t>(row) * (2 * D)), 0, 16 * 2 * D, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)to, 16, off, 0, 0, 0);
    };
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        char *const to = lds + (it * kWaves + wave) * 1024;
        const int sub = wsub + PER * it;
        if (plain) {
            load(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(rows), i0 + sub)), to,
                 at.row * (2 * D) + at.piece16);
        } else {
            const int last = n - 1 - row0, subc = sub < (last >> 4) ? sub : last >> 4;
            const unsigned row = static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(rows), i0 + subc));
            const int r = 16 * sub + at.row < last ? 16 * sub + at.row : last;
            if (row == kNoPage)
                *reinterpret_cast<uint4 *>(to + lane * 16) = make_uint4(0, 0, 0, 0);
            else
                load(row, to, (r - 16 * subc) * (2 * D) + at.piece16);
        }
    }
#endif
}

// 2048 tokens over 16384, H32 G8 D128 causal: 504 us, 930 TFLOP/s (a large library product 1216); three pieces to 517 over
// contexts to 9000, H16 G4 D128: 78 us in four shares, whose unequal ends leave CUs idle, and their join 11.
// The products, statistics and layouts of the forward over whole sequences (gdn2_attn_train.hip), keys
// and values by pages: a wave looks the pages of 16 tiles up at once.  Probabilities are rounded once
// for their product, as there: off by 1.4 to 1.5 times the rounding of the result.
template <PrecKind PK, int D>
__global__ __launch_bounds__(64 * kWaves, D == 64 ? 3 : 2) void attn_paged_tiles_kernel(AttnPagedParams p)
{
    constexpr int KS = D / 16, DT = D / 32, BM = kTileRows;
    constexpr int kBytes = kTile * D * 2, kAhead = 16;  // tiles whose pages are looked up at once
    // Arrays of their own, so that reads of one and requests into another are known not to meet.
    __shared__ __align__(256) char sk0[kBytes], sk1[kBytes], sv0[kBytes], sv1[kBytes];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int rb = row_base<D>(lane), cb = col_base<D>(lane);
    // All groups' last tiles, the longest, then those before.  (A group's tiles dealt to one XCD: the same,
    // B4 T2048 over 16384 H32 G8 D128 1965 us either way, B1 496 and 543.)
    const int groups = p.B * p.G, turn = blockIdx.x / groups;
    const Where w = where(p, BM, static_cast<int>(blockIdx.x) - turn * groups, p.tiles - 1 - turn);
    const int all = p.T * p.R, end = w.t1 * p.R;  // rows, and those that are there
    const int per = p.splits > 1 ? share_of(p, lane) : (w.n + kRound - 1) / kRound * kRound;
    const int lo = static_cast<int>(blockIdx.y) * per, hi = lo + per < w.n ? lo + per : w.n;
    uint16_t *out = static_cast<uint16_t *>(p.out);
    if (lo >= hi) {
        if (p.splits == 1)
            for (int e = tid; e < BM * (D / 8); e += 64 * kWaves) {
                const int x = w.m0 + e / (D / 8);
                if (x < all) *reinterpret_cast<uint4 *>(out + out_row(p, w, x) * D + e % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
            }
        return;
    }
    const int x = w.m0 + 32 * wave + n, xc = x < end ? x : end - 1;  // this lane's row
    const int t_of = xc / p.R;
    const uint16_t *qr = static_cast<const uint16_t *>(p.q) + w.b * p.qs[0] + t_of * p.qs[1] +
                         (w.g * p.R + (xc - t_of * p.R)) * p.qs[2];
    uint4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const uint4 *>(qr + 16 * s + 8 * h);
    // Keys that this lane sees, all of the wave see, none of the wave sees more than, all of the workgroup see.
    const int lim = w.pos + t_of + 1;
    const int wfirst = w.m0 + 32 * wave < end ? w.m0 + 32 * wave : end - 1;
    const int wlast = wfirst + 31 < end ? wfirst + 31 : end - 1;
    const int wlim = w.pos + wfirst / p.R + 1, wend = w.pos + wlast / p.R + 1, glim = w.pos + w.t0 + 1;
    const float c = p.scale * kLog2e;

    const int first = lo / kTile, nt = (hi + kTile - 1) / kTile;
    const int *table = p.table + w.b * p.table_stride;
    auto look_up = [&](int tile) __attribute__((always_inline)) {
        const int j = tile * kTile + lane * 16;
        unsigned r = kNoPage;
        if (j < hi) {
            const int col = j / p.page;
            const int64_t pg = table[col];
            if (pg >= 0 && pg < p.pages) r = static_cast<unsigned>((pg * p.G + w.g) * p.page + (j - col * p.page));
        }
        return r;
    };
    // A bit for each piece of 16 positions that has none.
    auto missing = [&](unsigned rows, int tile) __attribute__((always_inline)) {
        return __ballot(rows == kNoPage && tile * kTile + lane * 16 < hi);
    };
    unsigned rows = look_up(first), next = look_up(first + kAhead);
    uint64_t lost = missing(rows, first);
    const Place<D> at(wave, lane);
    const char *kp = static_cast<const char *>(p.k), *vp = static_cast<const char *>(p.v);
    auto stage = [&](int t, char *tk, char *tv) __attribute__((always_inline)) {
        const int i0 = (t - first) % kAhead * 4;
        const bool plain = (t + 1) * kTile <= hi && ((lost >> i0) & 15) == 0;
        stage_pages<D>(kp, rows, i0, t * kTile, hi, plain, tk, at, wave, lane);
        stage_pages<D>(vp, rows, i0, t * kTile, hi, plain, tv, at, wave, lane);
    };

    float m = 0.0f, l = 0.0f;
    bool fresh = true;  // no visible key yet
    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = zero16();
    stage(first, sk0, sv0);
    auto step = [&](int t, int gone, auto buf, auto hidden) __attribute__((always_inline)) {
        constexpr bool kOdd = decltype(buf)::value, kHide = decltype(hidden)::value;
        const char *const tk = kOdd ? sk1 : sk0, *const tv = kOdd ? sv1 : sv0;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();  // tile t has landed, and every wave is done with tile t - 1
        if (t + 1 < nt) {
            if (kOdd && (t + 1 - first) % kAhead == 0) {
                rows = next;
                lost = missing(rows, t + 1);
                next = look_up(t + 1 + kAhead);
            }
            stage(t + 1, kOdd ? sk0 : sk1, kOdd ? sv0 : sv1);
        }
        const int j0 = t * kTile;
        if (kHide && j0 >= wend) return;
        const int kr = opaque(rb), vc = opaque(cb);
        if constexpr (D == 128) mix_reads();
        f32x16 s[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            s[a] = zero16();
#pragma unroll
            for (int st = 0; st < KS; ++st) s[a] = mma32<PK>(s[a], row_frag<D>(tk, kr, 32 * a, st), qf[st]);
        }
        if (kHide && j0 + kTile > wlim) {
            hide<true>(s[0], j0, h, lim);
            hide<true>(s[1], j0 + 32, h, lim);
        }
        if (kHide && gone) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[a][i] = (gone >> (2 * a + (i >> 3))) & 1 ? -INFINITY : s[a][i];
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[a][i] = fmaf(s[a][i], c, -m);
                mx[i & 3] = fmaxf(mx[i & 3], s[a][i]);
            }
        const float top = half_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
        constexpr float kDown = Ref<PK>::down;
        if (__any(top > (fresh ? -INFINITY : kDown + Ref<PK>::lazy))) {
            // The first visible key sets the reference, later ones raise it.
            const bool set = fresh && top > -INFINITY;
            const float d = set ? top - kDown : fmaxf(top - kDown, 0.0f);
            const float r = fresh ? 1.0f : __builtin_amdgcn_exp2f(-d);  // nothing to rescale yet
            m += d;
            fresh = fresh && !set;
            l *= r;
#pragma unroll
            for (int e = 0; e < DT; ++e)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[e][i] *= r;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[a][i] -= d;
        }
        float sum = 0.0f;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[a][i] = __builtin_amdgcn_exp2f(s[a][i]);
                sum += s[a][i];
            }
        l += sum;
#pragma unroll
        for (int a = 0; a < 2; ++a) add_columns<PK, D, false>(acc, tv, vc, 32 * a, s[a]);
    };
    for (int t = first; t < nt; t += 2) {
        // (lost belongs to this pair's tiles: both lie among the 16 that were looked up last.)
        const int gone = static_cast<int>(lost >> ((t - first) % kAhead * 4)) & 255;
        if ((t + 2) * kTile <= glim && t + 2 <= nt && gone == 0) {
            step(t, 0, std::false_type{}, std::false_type{});
            step(t + 1, 0, std::true_type{}, std::false_type{});
        } else {
            step(t, gone & 15, std::false_type{}, std::true_type{});
            if (t + 1 < nt) step(t + 1, gone >> 4, std::true_type{}, std::true_type{});
        }
    }
    l = half_add(l);
    m = fresh ? kNoMax : m;
    if (p.splits > 1) {
        if (x >= end) return;
        // This share's state; attn_paged_join_tiles_kernel puts the shares together.
        const int64_t rows_all = static_cast<int64_t>(p.B) * p.T * (p.G * p.R);
        const int64_t to = blockIdx.y * rows_all + out_row(p, w, x);
        if (h == 0) *reinterpret_cast<float2 *>(p.part + p.splits * rows_all * D + 2 * to) = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4 *>(p.part + to * D + 32 * d + 8 * i + 4 * h) =
                    make_float4(acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]);
        return;
    }
    const bool none = l == 0.0f || x >= end;  // padding, or no key with a page
    const float inv = 1.0f / l;
    __syncthreads();  // the tiles are done with
    char *const so = wave == 0 ? sk0 : wave == 1 ? sk1 : wave == 2 ? sv0 : sv1;
    put_rows<D>(so, lane, acc, [&](float a, float b, float cc, float d) __attribute__((always_inline)) {
        return none ? pack4<PK>(0.0f, 0.0f, 0.0f, 0.0f) : pack4<PK>(a * inv, b * inv, cc * inv, d * inv);
    });
    write_rows<D>(so, lane, out, [&](int r) __attribute__((always_inline)) {
        const int xr = w.m0 + 32 * wave + r;
        return xr < all ? out_row(p, w, xr) * D : int64_t{-1};
    });
}

// The shares of a row in their order; thread: 4 channels of a row.
template <PrecKind PK, int D>
__global__ __launch_bounds__(256) void attn_paged_join_tiles_kernel(AttnPagedParams p)
{
    const int H = p.G * p.R;
    const int64_t rows = static_cast<int64_t>(p.B) * p.T * H;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (1024 / D) + threadIdx.x / (D / 4);
    const int per = share_of(p, threadIdx.x & 63);
    if (row >= rows) return;
    const int ch = threadIdx.x % (D / 4) * 4;
    const unsigned bt = static_cast<unsigned>(row / H), hh = static_cast<unsigned>(row - static_cast<int64_t>(bt) * H);
    const unsigned b = bt / p.T, t = bt - b * p.T, g = hh / p.R;
    const Where w = where(p, kTileRows, static_cast<int>(b * p.G + g), static_cast<int>((t * p.R + (hh - g * p.R)) / kTileRows));
    const int used = static_cast<int>(t) < w.t1 ? (w.n + per - 1) / per : 0;
    const float2 *ml = reinterpret_cast<const float2 *>(p.part + p.splits * rows * D);
    float m = kNoMax;
    for (int s = 0; s < used; ++s) m = fmaxf(m, ml[s * rows + row].x);
    float l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = 0; s < used; ++s) {
        const float2 st = ml[s * rows + row];
        const float4 y = *reinterpret_cast<const float4 *>(p.part + (s * rows + row) * D + ch);
        const float r = __builtin_amdgcn_exp2f(st.x - m);
        l = fmaf(st.y, r, l);
        x.x = fmaf(y.x, r, x.x);
        x.y = fmaf(y.y, r, x.y);
        x.z = fmaf(y.z, r, x.z);
        x.w = fmaf(y.w, r, x.w);
    }
    const float inv = 1.0f / l;
    const Q4<PK> y = l == 0.0f ? pack4<PK>(0.0f, 0.0f, 0.0f, 0.0f) : pack4<PK>(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    st_q4<PK>(static_cast<uint16_t *>(p.out) + row * D + ch, y);
}

template <PrecKind PK, int D>
hipError_t paged_tiles(AttnPagedParams &p, hipStream_t s)
{
    const unsigned x = static_cast<unsigned>(p.B) * p.G * p.tiles;
    hipLaunchKernelGGL((attn_paged_tiles_kernel<PK, D>), dim3(x, p.splits), dim3(64 * kWaves), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t rows = static_cast<int64_t>(p.B) * p.T * p.G * p.R;
    hipLaunchKernelGGL((attn_paged_join_tiles_kernel<PK, D>), dim3(static_cast<unsigned>((rows + 1024 / D - 1) / (1024 / D))),
                       dim3(256), 0, s, p);
    return hipGetLastError();
}

template <typename T, PrecKind PK, int D, int C>
hipError_t paged_c(AttnPagedParams &p, hipStream_t s)
{
    if (p.workers == 0) {
        hipLaunchKernelGGL((attn_paged_kernel<T, PK, D, C, false>), dim3(p.B, p.G), dim3(64 * kWaves), 0, s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((attn_paged_kernel<T, PK, D, C, true>), dim3(p.workers, p.G), dim3(64 * kWaves), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_paged_join_kernel<T, D>), dim3(static_cast<unsigned>(p.B) * p.G * p.T * p.R), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <typename T, PrecKind PK, int D>
hipError_t paged_d(AttnPagedParams &p, hipStream_t s)
{
    if (p.rows == 16) return paged_c<T, PK, D, 1>(p, s);
    if constexpr (D == 64) {
        if (p.rows == 32) return paged_c<T, PK, D, 2>(p, s);
    }
    return paged_tiles<PK, D>(p, s);
}

}  // namespace

// How a call is divided.  Rows of a workgroup: the keys of up to 16 rows (D = 64: 32) go from memory to the
// matrix units, those of more by tiles in LDS (20 rows over 4 x 16384 positions, G8 D128: 54 us, and 107 with two
// column tiles in registers, which spill; D = 64 20 rows, G16: 57 and 48).
AttnPagedPlan attn_paged_plan(int B, int64_t T, int G, int R, int D, int64_t cap)
{
    AttnPagedPlan a = {};
    const int64_t rows = T * R;
    a.rows = rows <= 16 ? 16 : rows <= 32 && D == 64 ? 32 : kTileRows;
    a.tiles = static_cast<int>((rows + a.rows - 1) / a.rows);
    a.splits = 1;
    const int64_t groups = static_cast<int64_t>(B) * G;
    if (a.rows == kTileRows) {
        const int64_t wg = groups * a.tiles, most = (cap + 511) / 512;
        int64_t s = wg >= 512 ? 1 : (640 + wg - 1) / wg;
        s = s < most ? s : most;
        a.splits = static_cast<int>(s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : s));
        a.floats = a.splits == 1 ? 0 : static_cast<size_t>(a.splits) * groups * rows * (D + 2);
        return a;
    }
    // One workgroup a sequence and group for short contexts (1024 positions, B1 G8 D128: 14 us, 17 by runs),
    // and where there are many times more than the card holds; else runs, 512 workgroups in all: 32
    // contexts spread over 32768 positions, G8 D128, 377 us (one a sequence 581), 64 over 4096 125 (152); of
    // equal lengths the runs lose (32 of 4096: 105, 86), but lengths are not known here.  Fewer
    // workgroups where little is to be done.
    const int64_t per = (cap + kRound - 1) / kRound;
    const double rounds = static_cast<double>(B) * per;
    if (cap > 1024 && groups < 4096 && rounds < 2.0e9) {
        const int64_t some = (256 + G - 1) / G, many = (512 + G - 1) / G, by_work = static_cast<int64_t>(rounds / 4);
        const int64_t workers = by_work < some ? some : (by_work < many ? by_work : many);
        const int64_t used = workers < kMaxWorkers ? workers : kMaxWorkers;
        // A run's end is counted from the start of a sequence, past whose own end it may lie, in 31 bits.
        const double end = per + rounds / used + kLeast;
        if ((end < rounds ? end : rounds) * kRound < 2147483648.0) {
            a.workers = static_cast<int>(used);
            a.floats = static_cast<size_t>(a.workers + B) * G * rows * (D + 2);
        }
    }
    return a;
}

bool attn_paged_supported(int io_dtype, int D)
{
    return (io_dtype == GDN2_DTYPE_BF16 || io_dtype == GDN2_DTYPE_F16) && (D == 64 || D == 128);
}

hipError_t launch_attn_paged(AttnPagedParams p, int io_dtype, hipStream_t s)
{
    if (io_dtype == GDN2_DTYPE_BF16)
        return p.D == 64 ? paged_d<bf16_t, PrecKind::BF16, 64>(p, s) : paged_d<bf16_t, PrecKind::BF16, 128>(p, s);
    return p.D == 64 ? paged_d<f16_t, PrecKind::F16, 64>(p, s) : paged_d<f16_t, PrecKind::F16, 128>(p, s);
}

}  // namespace gdn2

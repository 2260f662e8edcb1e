// Softmax attention over whole sequences with its gradient, gfx950: the
// training and prefill side of the hybrid decoder host's attention layers.
//
//   S = scale Q K^T, hidden keys at -inf, P = softmax(S), O = P V
//   L = log sum exp(S) (kept per query), D = dO . O
//   dV = P^T dO,  dS = P (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// The probabilities are never stored: the forward makes one pass over the keys
// with a running maximum and sum, the backward recomputes P = exp(S - L) tile
// by tile, once with the queries resident (dQ) and once with the keys resident
// (dK, dV, summed over the query heads of a group in registers).  Every output
// element is summed by one wave in a fixed order: no atomics on values, the
// same bits in every run.
//
// Layout of the products (v_mfma_f32_32x32x16): lane l = n + 32 h (n < 32,
// h < 2) supplies contraction indices 8 h + j (j < 8) of row / column n, and
// the accumulator element i holds row 8 (i / 4) + 4 h + i % 4 of column n.
// The resident side (32 queries, or 32 keys, per wave) is always the column:
// softmax statistics are then per-lane scalars, and an accumulator feeds the
// next product as its B operand unmoved, since elements 8 t .. 8 t + 7 of half
// h are the contraction indices 16 t + {4 h + 0..3, 8 + 4 h + 0..3} and the
// A operand is read with the same assignment.  The streamed side lies in LDS
// row-major and serves both products: rows by 16-byte reads, columns by
// ds_read_b64_tr_b16 (a 16-lane group reads 4 rows x 16 columns and each lane
// receives one column's 4 rows).
#include "gdn2_common.h"
#include "gdn2_internal.h"
#include "gdn2_mfma.h"

namespace gdn2 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
// Reference of a share of the keys that holds none a query sees: finite, below
// every score, so that differences of references are never inf - inf.
constexpr float kNoMax = -3.0e38f;
// The reference of the exponents lies `down` below the running maximum, and moves only when
// a score exceeds the maximum it was set by by `lazy`: until then the probabilities
// are at most 2^(down + lazy), exact in the same number of bits, and the accumulators need
// no rescaling.  bf16 has the exponents of fp32 and keeps a probability's 8 bits anywhere.
// fp16 is normal from 2^-14 on only: with the largest probability held at 2^13 .. 2^15,
// 2^-27 of it still has 11 bits, and what is below is off by at most 2^-38 of it (at
// down = 0 a row lost every key under 2^-25 of its largest, while the sum counted them).
// Its smaller `lazy` costs 0.5% (fp16 forward, against down 0 and lazy 8: B2 T8192 H16 G4 D128
// causal 571 and 575 us, B4 T2048 H16 D64 54.2 and 54.4).
template <PrecKind PK>
struct Ref {
    static constexpr float down = PK == PrecKind::F16 ? 13.0f : 0.0f, lazy = PK == PrecKind::F16 ? 2.0f : 8.0f;
    static constexpr float undo = PK == PrecKind::F16 ? 0x1p-13f : 1.0f;  // 2^-down
};
constexpr int kTile = 64;  // rows of the streamed side per LDS tile

template <PrecKind PK>
__device__ __forceinline__ f32x16 mma32(f32x16 acc, uint4 a, uint4 b)
{
    if constexpr (PK == PrecKind::BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b),
                                                      acc, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16()
{
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// Elements 8 t .. 8 t + 7 of an accumulator, rounded to the operand type: the
// B operand of the next product.
template <PrecKind PK>
__device__ __forceinline__ uint4 pack8(const f32x16 &x, int t)
{
    const Q4<PK> lo = pack4<PK>(x[8 * t], x[8 * t + 1], x[8 * t + 2], x[8 * t + 3]);
    const Q4<PK> hi = pack4<PK>(x[8 * t + 4], x[8 * t + 5], x[8 * t + 6], x[8 * t + 7]);
    return make_uint4(lo.u.x, lo.u.y, hi.u.x, hi.u.y);
}

// What pack8 left out of the same elements, rounded in its turn.
template <PrecKind PK>
__device__ __forceinline__ uint4 rest8(const f32x16 &x, int t, uint4 hi)
{
    Q4<PK> a, b;
    a.u = make_uint2(hi.x, hi.y);
    b.u = make_uint2(hi.z, hi.w);
    float f[4], g[4];
    unpack4<PK>(a, f);
    unpack4<PK>(b, g);
    a = pack4<PK>(x[8 * t] - f[0], x[8 * t + 1] - f[1], x[8 * t + 2] - f[2], x[8 * t + 3] - f[3]);
    b = pack4<PK>(x[8 * t + 4] - g[0], x[8 * t + 5] - g[1], x[8 * t + 6] - g[2], x[8 * t + 7] - g[3]);
    return make_uint4(a.u.x, a.u.y, b.u.x, b.u.y);
}

// The other half's value (lane l ^ 32) combined with this lane's.
__device__ __forceinline__ float half_max(float x)
{
    const unsigned u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ float half_add(float x)
{
    const unsigned u = __float_as_uint(x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// LDS tile [rows][D]: a row's 16-byte pieces are permuted by XOR with swz(row).  64
// banks serve 256 bytes per clock: of a row read 16 lanes (the same piece of 16
// rows, which must land on 16 places; at D = 64 two rows share the banks, so 8 of each
// parity), of a column read 32 (4 pieces of 4 rows: at D = 128 the rows must
// differ in the upper two bits, at D = 64 each two of a parity in the uppermost).  A
// wave's row read then takes 4.8 clocks, a column read 2.9 (8.2 and 4.2 with a
// conflict in each pair of lanes; all waves of a CU reading).
template <int D>
__device__ __forceinline__ int swz(int row)
{
    return D == 64 ? ((row << 1) & 4) | ((row >> 2) & 3) : ((row << 2) & 12) | ((row >> 2) & 3);
}

// A streamed matrix: rows ts bytes apart, and this lane's place in a request (its
// row of the first R and its 16-byte piece; later requests of a tile are whole
// multiples of 16 rows on, where the permutation repeats, so that a tile's
// requests differ in their scalar base alone).
struct Stream {
    const char *base;
    int64_t ts;
    unsigned lane_off;
};
template <int D, int NW>
__device__ __forceinline__ Stream stream_of(const uint16_t *base, int64_t ts, int wave, int lane)
{
    constexpr int P = D / 8, R = 64 / P;  // pieces per row, rows per request
    static_assert(NW * R % 16 == 0, "the permutation repeats from one of a wave's requests to its next");
    const int r = wave * R + lane / P;
    return {reinterpret_cast<const char *>(base), 2 * ts,
            static_cast<unsigned>(r * static_cast<int>(2 * ts) + ((lane % P) ^ swz<D>(r)) * 16)};
}

// One tile, row0 .. row0 + ROWS - 1 of nrows rows, requested into LDS.  Rows past the
// end repeat the last row (never out of bounds, never another sequence's row);
// the scores of such rows are hidden.  Buffer requests: they take a tile's scalar base,
// a lane's offset and a request's scalar one as they are, and unlike flat ones leave
// the counts of outstanding LDS reads exact.
template <int D, int NW, int ROWS = kTile>
__device__ __forceinline__ void stage(const Stream &x, int row0, int nrows, char *lds, int wave, int lane)
{
    constexpr int P = D / 8, R = 64 / P, IT = ROWS / R;  // requests per tile
    static_assert(IT % NW == 0, "every wave issues as many requests");
    static_assert((ROWS - 1) * (2 * kMaxTokenStride) + 2 * D <= 0xffffffffLL, "offsets within a tile are 32 bits");
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass does not know the builtins' types
    typedef __attribute__((address_space(3))) char *lds_ptr;
    const uint64_t at = reinterpret_cast<uint64_t>(x.base + row0 * x.ts);
    const uint64_t tile = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<unsigned>(at >> 32))) << 32 |
                          static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<unsigned>(at)));
    // Raw buffer, 32-bit elements, offsets below 2^32.
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(tile), 0, 0xffffffffu, 0x00020000);
    const unsigned ts = static_cast<unsigned>(x.ts);
    if (row0 + ROWS <= nrows) {
#pragma unroll
        for (int it = 0; it < IT / NW; ++it)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(lds + (it * NW + wave) * 1024), 16, x.lane_off,
                                                     it * (NW * R) * ts, 0, 0);
    } else {
#pragma unroll
        for (int it = 0; it < IT / NW; ++it) {
            const int r = (it * NW + wave) * R + lane / P;
            const int rc = row0 + r < nrows ? r : nrows - 1 - row0;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(lds + (it * NW + wave) * 1024), 16,
                                                     rc * ts + ((lane % P) ^ swz<D>(r)) * 16, 0, 0, 0);
        }
    }
#endif
}

// A lane's byte offset within a tile for row reads (row l & 31, its half of the
// 16 channels of step 0) and for column reads (rows 4 h + 0..3 of 16, channel
// l & 31 of 32).  A row's pitch is a power of two, so that the permutation of
// any step and channel block is one XOR of the offset with a constant.
template <int D>
__device__ __forceinline__ int row_base(int lane)
{
    return (lane & 31) * (2 * D) + (((lane >> 5) ^ swz<D>(lane & 31)) * 16);
}
template <int D>
__device__ __forceinline__ int col_base(int lane)
{
    const int i = lane & 15, grp = (lane >> 4) & 1, r = 4 * (lane >> 5) + (i >> 2);
    return r * (2 * D) + (((grp * 2 + ((i & 3) >> 1)) ^ swz<D>(r)) * 16) + (i & 1) * 8;
}

// A operand, rows r0 + (l & 31) of the tile, contraction step s of the row (16
// channels); `at` is row_base.
template <int D>
__device__ __forceinline__ uint4 row_frag(const char *tile, int at, int r0, int s)
{
    return *reinterpret_cast<const uint4 *>(tile + r0 * (2 * D) + (at ^ (32 * s)));
}

// A operand of the transposed tile: channels 32 dt + (l & 31), contraction
// over rows r0 + {4 h + 0..3, 8 + 4 h + 0..3}; `at` is col_base.
template <int D>
__device__ __forceinline__ uint4 col_frag(const char *tile, int at, int r0, int dt)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 *lds_s4;
    uint2 r[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        r[u] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                             (lds_s4)(tile + (r0 + 8 * u) * (2 * D) + (at ^ (64 * dt + 32 * u)))));
    return make_uint4(r[0].x, r[0].y, r[1].x, r[1].y);
}

// acc[d] += (columns 32 d .. of the tile)^T X for rows r0 + 16 t .. of it, X the elements 8 t ..
// 8 t + 7 of x.  X is rounded to the operand type: a relative error of half a step
// each (fp16: of what Ref and ds_scale keep normal), as large as the rounding of the result, so
// that results are off by 1.4 to 1.5 times that rounding.  Of FINE calls (attn_fine) also
// what that left out is multiplied.
template <PrecKind PK, int D, bool FINE>
__device__ __forceinline__ void add_columns(f32x16 (&acc)[D / 32], const char *tile, int at, int r0, const f32x16 &x)
{
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint4 hi = pack8<PK>(x, t);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) acc[d] = mma32<PK>(acc[d], col_frag<D>(tile, at, r0 + 16 * t, d), hi);
        if constexpr (FINE) {
            const uint4 lo = rest8<PK>(x, t, hi);
#pragma unroll
            for (int d = 0; d < D / 32; ++d) acc[d] = mma32<PK>(acc[d], col_frag<D>(tile, at, r0 + 16 * t, d), lo);
        }
    }
}

// Keeps the compiler from forming every step's address before the loop, where
// they would hold registers throughout.
__device__ __forceinline__ int opaque(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

// What a workgroup works on: a tile of group g of sequence s, and the sequence's extent.
struct Where {
    int s, g, tile;
    int64_t q0, k0;  // first query / key token within the batch row
    int bq, bk;      // batch row of q and k
    int nq, nk;      // queries, visible keys
    int shift;       // causal: query i sees keys j <= i + shift
    int share;       // which share of the streamed side
};

__device__ __forceinline__ void where_rows(const AttnTrainParams &p, Where &w)
{
    if (p.cu) {
        const int64_t a = p.cu[w.s], b = p.cu[w.s + 1];
        w.q0 = w.k0 = a;
        w.bq = w.bk = 0;
        w.nq = w.nk = static_cast<int>(b - a);
        w.shift = 0;
    } else {
        w.q0 = w.k0 = 0;
        w.bq = w.bk = w.s;
        w.nq = p.Tq;
        w.nk = p.Tk;
        w.shift = p.Tk - p.Tq;
        if (p.kv_len) {
            const int64_t n = p.kv_len[w.s];
            w.nk = n < 0 ? 0 : (n < p.Tk ? static_cast<int>(n) : p.Tk);
        }
    }
}

// Asks the scheduler to alternate LDS reads and matrix products in a block (D = 128, where
// the products bound it: forward 516 -> 507 us, forward and backward 2250 -> 2196, B2
// T8192 H16 G4; at D = 64 the backward lost 3%).
__device__ __forceinline__ void mix_reads()
{
    __builtin_amdgcn_iglp_opt(0);
}

// Which of `groups` (a sequence's heads that share keys) and of a group's `tiles`, the
// longest first, workgroup b takes.  Those of equal place in successive rounds over the
// 256 CUs share a CU, so every other round runs backwards: a CU's tiles then add up to
// about the same length.
//   dealt (many rounds, set_grid): workgroups go to the 8 XCDs in turn, each with an L2 of its own; the
//     groups are dealt out to them, and an XCD does one group's tiles after the other's,
//     whose keys it then holds (200 packed documents, 62381 tokens, H16 G4 D128 forward:
//     257 us, against 296 the other way).  A last deal may be short (group >= groups).
//   else: all groups' first tiles (of `row` workgroups each), then their second, which mixes
//     long and short ones better (B4 T2048 H16 D64, one round: 48 us against 54).
struct Turn {
    int group, tile;
};
__device__ __forceinline__ int backwards(int x, int round, int all)
{
    const int r = x / round, base = r * round;
    const int last = base + round < all ? base + round - 1 : all - 1;
    return r & 1 ? base + last - x : x;
}
__device__ __forceinline__ Turn turn_of(bool dealt, int b, int groups, int tiles, int row)
{
    if (dealt) {
        const int x = backwards(b >> 3, 32, (groups + 7) / 8 * tiles), g = x / tiles;
        return {g * 8 + (b & 7), x - g * tiles};
    }
    const int x = b / groups, m = groups * row < 256 ? 256 / (groups * row) : 1;  // tiles per round
    const int t = x / row;
    return {b - x * groups, backwards(t, m, tiles / row) * row + x - t * row};
}

template <int CTRL>
__device__ __forceinline__ int dpp_add(int x)
{
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
// The sum over the wave's lanes, in a scalar register.
__device__ __forceinline__ int lanes_sum(int x)
{
    x = dpp_add<0xb1>(x);   // quad_perm [1, 0, 3, 2]
    x = dpp_add<0x4e>(x);   // quad_perm [2, 3, 0, 1]
    x = dpp_add<0x141>(x);  // row_half_mirror: the quads hold equal values
    x = dpp_add<0x140>(x);  // row_mirror
    return __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) +
           __builtin_amdgcn_readlane(x, 48);
}

// Packed sequences of very unequal lengths (packed_ranked): tile t of all their tiles,
// in an order that starts with long work: by the tile's number in its sequence
// (`level`, causal work grows with it; from the end for key tiles), the highest
// first; past kRanked sequences, where a lane would hold too many lengths, in the
// order of the sequences.  The launch then holds no more workgroups than there are tiles.
constexpr int kRanked = 256;
struct Packed {
    int s, level, tiles;  // sequence, and its number of tiles; s < 0: none
};
__device__ __forceinline__ int seq_tiles(const int64_t *cu, int nseq, int rows, int s)
{
    const int64_t n = s < nseq ? (cu[s + 1] - cu[s]) * rows : 0;
    return n > 0 ? static_cast<int>((n + 127) >> 7) : 0;
}
// rows: of a token (its query heads in the query-resident kernels, 1 in the other).
__device__ __forceinline__ Packed packed_tile(const int64_t *cu, int nseq, int rows, int longest, int t)
{
    const int lane = threadIdx.x & 63;
    if (nseq <= kRanked) {
        constexpr int U = kRanked / 64;
        int n[U];
#pragma unroll
        for (int u = 0; u < U; ++u) n[u] = 64 * u < nseq ? seq_tiles(cu, nseq, rows, 64 * u + lane) : 0;
        auto at_least = [&](int x) {  // tiles of level x and above
            int c = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) c += n[u] > x ? n[u] - x : 0;
            return lanes_sum(c);
        };
        int lo = 0, hi = longest;  // the highest level with more than t tiles at or above it
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (at_least(mid) > t) lo = mid;
            else hi = mid;
        }
        int r = t - at_least(lo + 1);  // the r-th of the sequences that have this level
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t have = __ballot(n[u] > lo);
            const int c = __popcll(have);
            if (r >= 0 && r < c) {
                const int before = __popcll(have & ((1ull << lane) - 1));
                const int l = __ffsll(static_cast<unsigned long long>(__ballot(n[u] > lo && before == r))) - 1;
                return {64 * u + l, lo, __builtin_amdgcn_readlane(n[u], l)};
            }
            r -= c;
        }
        return {-1, 0, 0};
    }
    // Each lane's range of sequences first, then 64 sequences at a time within it.
    auto before = [&](int x) {  // sum over the lanes below
        int y = x;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int z = __shfl_up(y, d);
            y += lane >= d ? z : 0;
        }
        return y - x;
    };
    const int each = (nseq + 63) / 64;
    int c = 0;
    for (int i = 0; i < each; ++i) c += seq_tiles(cu, nseq, rows, lane * each + i);
    int b = before(c);
    uint64_t hit = __ballot(t >= b && t - b < c);
    if (!hit) return {-1, 0, 0};
    int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
    t -= __builtin_amdgcn_readlane(b, l);
    for (int s0 = l * each, end = s0 + each; s0 < end; s0 += 64) {
        c = s0 + lane < end ? seq_tiles(cu, nseq, rows, s0 + lane) : 0;
        b = before(c);
        hit = __ballot(t >= b && t - b < c);
        if (hit) {
            l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            const int tiles = __builtin_amdgcn_readlane(c, l);
            return {s0 + l, tiles - 1 - (t - __builtin_amdgcn_readlane(b, l)), tiles};
        }
        t -= lanes_sum(c);
    }
    return {-1, 0, 0};
}

// Query-resident kernels: a group's rows are its queries' heads, row x the head x % qpk of
// query x / qpk, so that a tile of keys serves every head that reads it (few queries of
// many heads fill a tile, and causal tiles of 128 rows span 128 / qpk queries: B1 Tq1
// Tk16384 H32 G8 D128 29 us against 43 with a workgroup per head).  Long causal
// tiles first; w.share of `shares` of the keys; w.nq rows.
__device__ __forceinline__ Where where_q(const AttnTrainParams &p, int shares)
{
    Where w;
    const int nbg = (p.ranked ? 1 : p.nseq) * p.G;
    const int tiles = p.ranked ? static_cast<int>(p.q_tiles) : p.tiles;
    const Turn u = turn_of(p.dealt, blockIdx.x, nbg, tiles * shares, shares);
    const int t = u.tile / shares;
    w.share = u.tile - t * shares;
    w.s = u.group / p.G;
    w.g = u.group - w.s * p.G;
    w.tile = tiles - 1 - t;
    if (u.group >= nbg) {
        w.s = 0;
        w.tile = p.tiles;  // past every sequence's rows
    } else if (p.ranked) {
        const Packed x = packed_tile(p.cu, p.nseq, p.H / p.G, p.tiles, t);
        w.s = x.s < 0 ? 0 : x.s;
        w.tile = x.s < 0 ? p.tiles : x.level;
    }
    where_rows(p, w);
    return w;
}

// A lane's row of a query-resident kernel: its query and head; rows past the end repeat the last.
struct Row {
    int q, h;
};
// x / qpk, 0 <= x < 2^31: x times m = 2^(31 + s) / qpk rounded up, 2^s >= qpk; the
// rounding adds less than x 2^s / 2^(31 + s) < 1 / qpk (by division these six of a
// workgroup took 0.2 us).
__device__ __forceinline__ int query_of(const AttnTrainParams &p, int x)
{
    return static_cast<int>((static_cast<uint64_t>(static_cast<unsigned>(x)) * p.qpk_m) >> (31 + p.qpk_s));
}
__device__ __forceinline__ Row row_of(const AttnTrainParams &p, int x, int rows, int g, int qpk)
{
    const int c = x < rows ? x : rows - 1, q = query_of(p, c);
    return {q, g * qpk + (c - q * qpk)};
}

// exp2 of a tile's scaled scores relative to ref, hidden keys to 0.  keys of
// the accumulator: j0 + 8 (i / 4) + 4 h + i % 4.
template <bool MASK>
__device__ __forceinline__ void hide(f32x16 &s, int j0, int h, int limit)
{
    if constexpr (MASK) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int j = j0 + 8 * (i >> 2) + 4 * h + (i & 3);
            s[i] = j < limit ? s[i] : -INFINITY;
        }
    }
}

// A wave's 32 results of D channels, 16-bit, into rows of memory by way of 32 rows of LDS:
// written from the accumulators eight bytes a row at a time, lines were left half
// written when others took their place in the L2 (B64 T64 H16 G4 D128 forward, 512
// workgroups 128 KB apart: 33 us, and 14 as whole rows).  make(a, b, c, d): four
// channels' bits; to(r): the first element of row r, or -1.
template <int D, typename Make>
__device__ __forceinline__ void put_rows(char *so, int lane, const f32x16 (&x)[D / 32], Make make)
{
    constexpr int P = D / 8;
    const int n = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint2 *>(so + n * (2 * D) + (((4 * d + i) ^ n) & (P - 1)) * 16 + 8 * h) =
                make(x[d][4 * i], x[d][4 * i + 1], x[d][4 * i + 2], x[d][4 * i + 3]).u;
    wave_fence();  // write_rows reads what other lanes stored
}
template <int D, typename To>
__device__ __forceinline__ void write_rows(const char *so, int lane, uint16_t *out, To to)
{
    constexpr int P = D / 8;
#pragma unroll
    for (int it = 0; it < P / 2; ++it) {
        const int r = it * (64 / P) + lane / P;
        const uint4 v = *reinterpret_cast<const uint4 *>(so + r * (2 * D) + ((lane ^ r) & (P - 1)) * 16);
        const int64_t at = to(r);
        if (at >= 0) *reinterpret_cast<uint4 *>(out + at + (lane % P) * 8) = v;
    }
    wave_fence();  // the next put_rows overwrites what other lanes read
}

// ---------------------------------------------------------------- forward

// L in base 2 from the reference and the sum.  A query that sees no key: +inf, which makes its
// recomputed P zero.
template <PrecKind PK>
__device__ __forceinline__ float log_sum(float m, float l)
{
    return l == 0.0f ? INFINITY : (m + Ref<PK>::down) + __builtin_amdgcn_logf(l * Ref<PK>::undo);
}

// Four channels of O, and, for D = dO . O, what their rounding left out: without it D is
// off by half a step of O, which shows in dS where few keys carry the weight
// and dP - D cancels.  What is below the sums' own error is dropped: O of a
// single key is then exactly its V.
template <PrecKind PK>
__device__ __forceinline__ Q4<PK> left_out(float a, float b, float c, float d)
{
    const float y[4] = {a, b, c, d};
    float z[4];
    unpack4<PK>(pack4<PK>(a, b, c, d), z);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        z[e] = y[e] - z[e];
        z[e] = fabsf(z[e]) > 0x1p-18f * fabsf(y[e]) ? z[e] : 0.0f;
    }
    return pack4<PK>(z[0], z[1], z[2], z[3]);
}

// One pass over the keys with the running maximum and sum.  D = 128 is bound by the
// matrix units (B2 T8192 H16 G4 causal: 503 us, 1094 TFLOP/s; a large library product
// reaches 1121), D = 64 by vector arithmetic, as a score costs a scaling, a maximum, an
// exponential of four issue slots, a sum and half a conversion whatever D is (B4
// T2048 H16 causal: 47 us, 732 TFLOP/s, vector units busy 77% of the time, matrix
// units 40%).  Few queries over many keys: B1 Tq1 Tk16384 H32 G8 D128, keys in shares, 29 us.
template <PrecKind PK, int D, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, D == 64 ? 4 : 2) void attn_fwd_kernel(AttnTrainParams p)
{
    constexpr int KS = D / 16, DT = D / 32, BM = 32 * NW;
    constexpr int kBytes = kTile * D * 2;
    // Two tiles of k and of v, each an array of its own: reads of one and requests into
    // another are then known not to meet.  In one array the compiler waited for
    // the request of the next tile before the first read of this one.
    __shared__ __align__(256) char sk0[kBytes], sk1[kBytes], sv0[kBytes], sv1[kBytes];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int rb = row_base<D>(lane), cb = col_base<D>(lane);
    const Where w = where_q(p, p.splits_f);
    const int m0 = w.tile * BM;
    const int qpk = p.H / p.G, rows = w.nq * qpk;
    if (m0 >= rows) return;
    const int x = m0 + 32 * wave + n;  // this lane's row
    const Row row = row_of(p, x, rows, w.g, qpk);
    const uint16_t *kb = static_cast<const uint16_t *>(p.k) + w.bk * p.ks[0] + w.k0 * p.ks[1] + w.g * p.ks[2];
    const uint16_t *vb = static_cast<const uint16_t *>(p.v) + w.bk * p.vs[0] + w.k0 * p.vs[1] + w.g * p.vs[2];
    const Stream ks = stream_of<D, NW>(kb, p.ks[1], wave, lane), vs = stream_of<D, NW>(vb, p.vs[1], wave, lane);
    const uint16_t *qr = static_cast<const uint16_t *>(p.q) + w.bq * p.qs[0] + (w.q0 + row.q) * p.qs[1] + row.h * p.qs[2];
    uint4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const uint4 *>(qr + 16 * s + 8 * h);

    // Keys of the workgroup, of this wave and of this lane.
    int kend = w.nk;
    if (p.causal) {
        const int last = query_of(p, (m0 + BM < rows ? m0 + BM : rows) - 1) + 1 + w.shift;
        kend = last < kend ? last : kend;
    }
    const int lim = p.causal && row.q + w.shift + 1 < w.nk ? row.q + w.shift + 1 : w.nk;
    const int wmin = query_of(p, m0 + 32 * wave), wmax = query_of(p, m0 + 32 * wave + 31);
    const int wlim = p.causal && wmin + w.shift + 1 < w.nk ? wmin + w.shift + 1 : w.nk;  // all of the wave see these
    const int wend = p.causal && wmax + w.shift + 1 < w.nk ? wmax + w.shift + 1 : w.nk;  // none sees more
    const float c = p.scale * kLog2e;

    // Reference of the exponents (Ref) and their sum.
    float m = 0.0f, l = 0.0f;
    bool fresh = true;  // no visible key yet
    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = zero16();

    const int all = kend > 0 ? (kend + kTile - 1) / kTile : 0;
    const int first = static_cast<int>(static_cast<int64_t>(all) * w.share / p.splits_f);
    const int nt = static_cast<int>(static_cast<int64_t>(all) * (w.share + 1) / p.splits_f);
    const int gmin = query_of(p, m0);
    int glim = p.causal && gmin + w.shift + 1 < w.nk ? gmin + w.shift + 1 : w.nk;  // all of the workgroup see these
    glim = glim < nt * kTile ? glim : nt * kTile;
    if (first < nt) {
        stage<D, NW>(ks, first * kTile, w.nk, sk0, wave, lane);
        stage<D, NW>(vs, first * kTile, w.nk, sv0, wave, lane);
    }
    auto step = [&](int t, auto buf, auto hidden) __attribute__((always_inline)) {
        constexpr bool kOdd = decltype(buf)::value, kHide = decltype(hidden)::value;
        const char *const tk = kOdd ? sk1 : sk0, *const tv = kOdd ? sv1 : sv0;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();  // tile t has landed, and every wave is done with tile t - 1
        if (t + 1 < nt) {
            stage<D, NW>(ks, (t + 1) * kTile, w.nk, kOdd ? sk0 : sk1, wave, lane);
            stage<D, NW>(vs, (t + 1) * kTile, w.nk, kOdd ? sv0 : sv1, wave, lane);
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
        // Exponents relative to the reference so far, and their maximum (taken
        // from them and not from the scores: fmaxf of a product's result costs a
        // second instruction, to quiet a NaN it might hold).
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
        // The probabilities are rounded for this product, their sum l is not.
#pragma unroll
        for (int a = 0; a < 2; ++a) add_columns<PK, D, FINE>(acc, tv, vc, 32 * a, s[a]);
    };
    // Pairs of tiles that every query of the workgroup sees, then the others.
    int t = first;
    for (; (t + 2) * kTile <= glim; t += 2) {
        step(t, std::false_type{}, std::false_type{});
        step(t + 1, std::true_type{}, std::false_type{});
    }
    for (; t < nt; t += 2) {
        step(t, std::false_type{}, std::true_type{});
        if (t + 1 < nt) step(t + 1, std::true_type{}, std::true_type{});
    }
    l = half_add(l);
    m = fresh ? kNoMax : m;
    if (p.splits_f > 1) {
        if (x >= rows) return;
        // This share's state; attn_fwd_join_kernel puts the shares together.
        const int64_t orow = (w.bq * static_cast<int64_t>(p.Tq) + w.q0 + row.q) * p.H + row.h;
        const int64_t at = w.share * (static_cast<int64_t>(p.B) * p.Tq * p.H) + orow;
        if (h == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4 *>(p.part + at * D + 32 * d + 8 * i + 4 * h) =
                    make_float4(acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (h == 0 && x < rows)
        p.lse[(static_cast<int64_t>(w.bq) * p.H + row.h) * p.Tq + w.q0 + row.q] = log_sum<PK>(m, l);
    __syncthreads();  // the tiles are done with
    char *const so = wave == 0 ? sk0 : wave == 1 ? sk1 : wave == 2 ? sv0 : sv1;
    auto to = [&](int r) __attribute__((always_inline)) {
        const int xr = m0 + 32 * wave + r;
        const Row at = row_of(p, xr, rows, w.g, qpk);
        return xr < rows ? ((w.bq * static_cast<int64_t>(p.Tq) + w.q0 + at.q) * p.H + at.h) * D : int64_t{-1};
    };
    put_rows<D>(so, lane, acc, [&](float a, float b, float c, float d) __attribute__((always_inline)) {
        return pack4<PK>(a * inv, b * inv, c * inv, d * inv);
    });
    write_rows<D>(so, lane, static_cast<uint16_t *>(p.o), to);
    if (!p.o_lo) return;
    put_rows<D>(so, lane, acc, [&](float a, float b, float c, float d) __attribute__((always_inline)) {
        return left_out<PK>(a * inv, b * inv, c * inv, d * inv);
    });
    write_rows<D>(so, lane, static_cast<uint16_t *>(p.o_lo), to);
}

// The shares of a query's keys, in their order; thread: 4 channels of a row.  Bound by
// its launch: it follows at most 512 workgroups' partial results (B1 Tq64 Tk8192 H8
// D64: 19 us with the kernel above).
template <PrecKind PK>
__global__ __launch_bounds__(256) void attn_fwd_join_kernel(AttnTrainParams p)
{
    const int64_t rows = static_cast<int64_t>(p.B) * p.Tq * p.H;
    const int64_t e = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    const int64_t row = e / p.D;
    if (row >= rows) return;
    float m = kNoMax;
    for (int s = 0; s < p.splits_f; ++s) m = fmaxf(m, p.part_ml[2 * (s * rows + row)]);
    float l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = 0; s < p.splits_f; ++s) {
        const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + 2 * (s * rows + row));
        const float4 y = *reinterpret_cast<const float4 *>(p.part + s * rows * p.D + e);
        const float r = __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(ml.y, r, l);
        x.x = fmaf(y.x, r, x.x);
        x.y = fmaf(y.y, r, x.y);
        x.z = fmaf(y.z, r, x.z);
        x.w = fmaf(y.w, r, x.w);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (e == row * p.D) {
        const int64_t bt = row / p.H;
        const int hh = static_cast<int>(row - bt * p.H);
        const int64_t b = bt / p.Tq;
        p.lse[(b * p.H + hh) * p.Tq + (bt - b * p.Tq)] = log_sum<PK>(m, l);
    }
    const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    st_q4<PK>(static_cast<uint16_t *>(p.o) + e, pack4<PK>(y[0], y[1], y[2], y[3]));
    if (p.o_lo) st_q4<PK>(static_cast<uint16_t *>(p.o_lo) + e, left_out<PK>(y[0], y[1], y[2], y[3]));
}

// ---------------------------------------------------------------- backward

// fp16 only: the largest squared row norms of dO per (batch row, head) and of V per
// (batch row, group), from which the kernels below scale dS into fp16's range;
// kNormParts workgroups each, [B][heads][kNormParts].  B8 T509 H8 D64: 5 us.  Bound by the
// latency of one row at a time in few workgroups where a row is long: B1 T16384 H16 G4
// D128 157 us before a backward of 3820, 62381 packed tokens 600 before 616 (D64 294 before
// 335).  Rows that are not finite,
// or past the row's length, do not count.  `first`: of the launch's workgroups, where
// there are more than one launch takes.
constexpr int kNormParts = 4;
template <int D>
__global__ __launch_bounds__(256) void norm_max_kernel(AttnTrainParams p, unsigned first)
{
    constexpr int P = D / 8, R = 256 / P;
    __shared__ float s_best[4];
    const int ndo = p.B * p.H;
    const unsigned wg = first + blockIdx.x;
    const int part = static_cast<int>(wg % kNormParts);
    int bh = static_cast<int>(wg / kNormParts);
    const bool is_v = bh >= ndo;
    if (is_v) bh -= ndo;
    const int heads = is_v ? p.G : p.H, b = bh / heads, hh = bh - b * heads;
    const int64_t HD = static_cast<int64_t>(p.H) * D;
    const uint16_t *x = is_v ? static_cast<const uint16_t *>(p.v) + b * p.vs[0] + hh * p.vs[2]
                             : static_cast<const uint16_t *>(p.dout) + b * p.Tq * HD + hh * D;
    const int64_t st = is_v ? p.vs[1] : HD;
    int T = is_v ? p.Tk : p.Tq;
    if (is_v && p.kv_len && p.kv_len[b] < T) T = static_cast<int>(p.kv_len[b] < 0 ? 0 : p.kv_len[b]);
    const int piece = threadIdx.x % P;
    float best = 0.0f;
    for (int t = part * R + threadIdx.x / P; t < T; t += kNormParts * R) {
        typename Prec<PrecKind::F16>::frag f;
        f.u = *reinterpret_cast<const uint4 *>(x + t * st + piece * 8);
        float v[8];
        unpack_frag<PrecKind::F16>(f, v);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(v[e], v[e], s);
#pragma unroll
        for (int k = 1; k < P; k <<= 1) s += __shfl_xor(s, k, 64);
        best = s < INFINITY ? fmaxf(best, s) : best;
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) best = fmaxf(best, __shfl_xor(best, k, 64));
    if ((threadIdx.x & 63) == 0) s_best[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0)
        (is_v ? p.mx_v : p.mx_do)[bh * kNormParts + part] =
            fmaxf(fmaxf(s_best[0], s_best[1]), fmaxf(s_best[2], s_best[3]));
}

// fp16: P is held scaled by 2^kP16 (P = 1 / T of long rows stays a normal
// number), dS by a power of two that brings 2 max |dO_i| max |v_j|, its bound,
// to 2^14.  Exact scalings, undone in fp32.
constexpr float kP16 = 14.0f;

template <PrecKind PK>
__device__ __forceinline__ float ds_scale(const AttnTrainParams &p, const Where &w, int head)
{
    if constexpr (PK != PrecKind::F16) return 1.0f;
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int i = 0; i < kNormParts; ++i) {
        a = fmaxf(a, p.mx_do[(w.bq * p.H + head) * kNormParts + i]);
        b = fmaxf(b, p.mx_v[(w.bk * p.G + w.g) * kNormParts + i]);
    }
    const float bound = 2.0f * sqrtf(a) * sqrtf(b);
    if (!(bound > 0.0f)) return 1.0f;
    int e = 13 - ilogbf(bound);
    e = e < -60 ? -60 : (e > 100 ? 100 : e);
    return ldexpf(1.0f, e);
}

// dQ: queries resident, one pass over the keys.  Also forms D = dO . (O + what its
// rounding left out) per query, which the kernel below reads.  Three products a tile:
// B2 T8192 H16 G4 D128 causal 710 us, 1160 TFLOP/s, the matrix units' rate; B4 T2048
// H16 D64 63 us, 815 TFLOP/s, vector units busy 60% and matrix units 49%.
template <PrecKind PK, int D, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, D == 64 && !FINE ? 4 : 2) void attn_dq_kernel(AttnTrainParams p)
{
    constexpr int KS = D / 16, DT = D / 32, BM = 32 * NW;
    constexpr int kBytes = kTile * D * 2;
    __shared__ __align__(256) char sk0[kBytes], sk1[kBytes], sv0[kBytes], sv1[kBytes];  // as in the forward
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int rb = row_base<D>(lane), cb = col_base<D>(lane);
    const Where w = where_q(p, p.splits_q);
    const int m0 = w.tile * BM;
    const int qpk = p.H / p.G, rows = w.nq * qpk;
    if (m0 >= rows) return;
    const int x = m0 + 32 * wave + n;
    const Row row = row_of(p, x, rows, w.g, qpk);
    const uint16_t *kb = static_cast<const uint16_t *>(p.k) + w.bk * p.ks[0] + w.k0 * p.ks[1] + w.g * p.ks[2];
    const uint16_t *vb = static_cast<const uint16_t *>(p.v) + w.bk * p.vs[0] + w.k0 * p.vs[1] + w.g * p.vs[2];
    const Stream ks = stream_of<D, NW>(kb, p.ks[1], wave, lane), vs = stream_of<D, NW>(vb, p.vs[1], wave, lane);
    const uint16_t *qr = static_cast<const uint16_t *>(p.q) + w.bq * p.qs[0] + (w.q0 + row.q) * p.qs[1] + row.h * p.qs[2];
    const int64_t orow = ((w.bq * static_cast<int64_t>(p.Tq) + w.q0 + row.q) * p.H + row.h) * D;
    const uint16_t *dr = static_cast<const uint16_t *>(p.dout) + orow;
    const int64_t srow = (static_cast<int64_t>(w.bq) * p.H + row.h) * p.Tq + w.q0 + row.q;
    uint4 qf[KS], df[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        qf[s] = *reinterpret_cast<const uint4 *>(qr + 16 * s + 8 * h);
        df[s] = *reinterpret_cast<const uint4 *>(dr + 16 * s + 8 * h);
    }
    const float sc = ds_scale<PK>(p, w, row.h);
    // D = dO . O as the diagonal of a product of the same shape, operands and order as
    // dP: where a query sees a single key, O is that key's V and D is dP to the
    // bit, so that its dS is the formula's zero and not the difference of two sums.
    float dl = 0.0f;
    {
        f32x16 t = zero16(), tl = zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint4 fo = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.o) + orow + 16 * s + 8 * h);
            const uint4 fl = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.o_lo) + orow + 16 * s + 8 * h);
            t = mma32<PK>(t, fo, df[s]);
            tl = mma32<PK>(tl, fl, df[s]);
        }
        // Row n of column n: element 4 (n / 8) + n % 4 of half (n / 4) % 2.
        const int at = (n >> 3) * 4 + (n & 3);
#pragma unroll
        for (int i = 0; i < 16; ++i) dl = at == i ? t[i] + tl[i] : dl;
        dl = ((n >> 2) & 1) == h ? dl : 0.0f;
        dl = half_add(dl);
    }
    if (h == 0 && x < rows && w.share == 0) p.delta[srow] = dl;
    dl *= sc;
    const float lse = p.lse[srow];

    int kend = w.nk;
    if (p.causal) {
        const int last = query_of(p, (m0 + BM < rows ? m0 + BM : rows) - 1) + 1 + w.shift;
        kend = last < kend ? last : kend;
    }
    const int lim = p.causal && row.q + w.shift + 1 < w.nk ? row.q + w.shift + 1 : w.nk;
    const int wmin = query_of(p, m0 + 32 * wave), wmax = query_of(p, m0 + 32 * wave + 31);
    const int wlim = p.causal && wmin + w.shift + 1 < w.nk ? wmin + w.shift + 1 : w.nk;
    const int wend = p.causal && wmax + w.shift + 1 < w.nk ? wmax + w.shift + 1 : w.nk;
    const float c = p.scale * kLog2e;

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = zero16();
    const int all = kend > 0 ? (kend + kTile - 1) / kTile : 0;
    const int first = static_cast<int>(static_cast<int64_t>(all) * w.share / p.splits_q);
    const int nt = static_cast<int>(static_cast<int64_t>(all) * (w.share + 1) / p.splits_q);
    const int gmin = query_of(p, m0);
    int glim = p.causal && gmin + w.shift + 1 < w.nk ? gmin + w.shift + 1 : w.nk;  // all of the workgroup see these
    glim = glim < nt * kTile ? glim : nt * kTile;
    if (first < nt) {
        stage<D, NW>(ks, first * kTile, w.nk, sk0, wave, lane);
        stage<D, NW>(vs, first * kTile, w.nk, sv0, wave, lane);
    }
    auto step = [&](int t, auto buf, auto hidden) __attribute__((always_inline)) {
        constexpr bool kOdd = decltype(buf)::value, kHide = decltype(hidden)::value;
        const char *const tk = kOdd ? sk1 : sk0, *const tv = kOdd ? sv1 : sv0;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 1 < nt) {
            stage<D, NW>(ks, (t + 1) * kTile, w.nk, kOdd ? sk0 : sk1, wave, lane);
            stage<D, NW>(vs, (t + 1) * kTile, w.nk, kOdd ? sv0 : sv1, wave, lane);
        }
        const int j0 = t * kTile;
        if (kHide && j0 >= wend) return;
        const int rr = opaque(rb), kc = opaque(cb);
        if constexpr (D == 128) mix_reads();
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int st = 0; st < KS; ++st) s = mma32<PK>(s, row_frag<D>(tk, rr, 32 * a, st), qf[st]);
#pragma unroll
            for (int st = 0; st < KS; ++st) dp = mma32<PK>(dp, row_frag<D>(tv, rr, 32 * a, st), df[st]);
            if (kHide && j0 + kTile > wlim) hide<true>(s, j0 + 32 * a, h, lim);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float pr = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse));
                s[i] = pr * fmaf(dp[i], sc, -dl);
            }
            add_columns<PK, D, FINE>(acc, tk, kc, 32 * a, s);
        }
    };
    // Pairs of tiles that every query of the workgroup sees, then the others.  At D = 64 one loop
    // for all: within 128 registers four waves fit a SIMD, which count for more than the
    // masks' branches (B4 T2048 H16: 67 us against 72 with both loops and three waves).
    int t = first;
    if constexpr (D == 128)
        for (; (t + 2) * kTile <= glim; t += 2) {
            step(t, std::false_type{}, std::false_type{});
            step(t + 1, std::true_type{}, std::false_type{});
        }
    for (; t < nt; t += 2) {
        step(t, std::false_type{}, std::true_type{});
        if (t + 1 < nt) step(t + 1, std::true_type{}, std::true_type{});
    }
    const float f = p.scale / sc;
    if (p.splits_q > 1) {
        if (x >= rows) return;
        float *part = p.part_q + w.share * (static_cast<int64_t>(p.B) * p.Tq * p.H * D) + orow;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4 *>(part + 32 * d + 8 * i + 4 * h) =
                    make_float4(acc[d][4 * i] * f, acc[d][4 * i + 1] * f, acc[d][4 * i + 2] * f, acc[d][4 * i + 3] * f);
        return;
    }
    __syncthreads();  // the tiles are done with
    char *const so = wave == 0 ? sk0 : wave == 1 ? sk1 : wave == 2 ? sv0 : sv1;
    put_rows<D>(so, lane, acc, [&](float a, float b, float c, float d) __attribute__((always_inline)) {
        return pack4<PK>(a * f, b * f, c * f, d * f);
    });
    write_rows<D>(so, lane, static_cast<uint16_t *>(p.dq), [&](int r) __attribute__((always_inline)) {
        const int xr = m0 + 32 * wave + r;
        const Row at = row_of(p, xr, rows, w.g, qpk);
        return xr < rows ? ((w.bq * static_cast<int64_t>(p.Tq) + w.q0 + at.q) * p.H + at.h) * D : int64_t{-1};
    });
}

// dK, dV: keys resident, one pass over the queries of every head of the group,
// or, where that leaves too few or too uneven workgroups (attn_bwd_splits), over
// one of p.splits equal shares of it, whose fp32 sums attn_sum_kernel adds.  Four
// products a tile: B2 T8192 H16 G4 D128 causal 1000 us, 1100 TFLOP/s; B4 T2048 H16 D64
// 85 us, 808 TFLOP/s, vector and matrix units each busy 46%, two waves per SIMD that wait
// for each other's products in turn (three, within 168 registers, gained 4 us, but
// lost 3 over short rows, B8 T509 H8, forward and backward 60).
template <PrecKind PK, int D, int NW, int BQ, bool FINE>
__global__ __launch_bounds__(64 * NW, 2) void attn_dkv_kernel(AttnTrainParams p)
{
    constexpr int KS = D / 16, DT = D / 32, BN = 32 * NW;
    constexpr int kBytes = BQ * D * 2;
    // D = 128: V's fragments are read from LDS, K's stay in registers.  Both in
    // registers is 64 beside 128 of accumulators and 32 of S and dP, and the
    // kernel spilled 59 (B2 T8192 H16 G4, this kernel alone: 3172 us against 1777).
    constexpr bool kVLds = D == 128;
    // Two tiles of q and of dout, V's rows, and per tile L and scaled D of its queries
    // (arrays of their own, as in the forward).
    __shared__ __align__(256) char sq0[kBytes], sq1[kBytes], sd0[kBytes], sd1[kBytes], sv[kVLds ? BN * D * 2 : 16];
    __shared__ __align__(16) float sl0[2 * BQ], sl1[2 * BQ];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int rb = row_base<D>(lane), cb = col_base<D>(lane);
    Where w;
    const int nbg = (p.ranked ? 1 : p.nseq) * p.G, qpk = p.H / p.G;
    // Dealt as in turn_of, or all groups' first tiles first, both the longest (causal) ones first.
    int ts = blockIdx.x / nbg, jg = blockIdx.x - ts * nbg;
    if (p.dealt) {
        const int per = static_cast<int>(p.ranked ? p.k_tiles : p.tiles) * p.splits, x = blockIdx.x >> 3, g = x / per;
        ts = x - g * per;
        jg = g * 8 + (blockIdx.x & 7);
        if (jg >= nbg) return;
    }
    w.tile = ts / p.splits;
    const int share = ts - w.tile * p.splits;
    w.s = jg / p.G;
    w.g = jg - w.s * p.G;
    if (p.ranked) {
        const Packed x = packed_tile(p.cu, p.nseq, 1, p.tiles, w.tile);
        w.s = x.s < 0 ? 0 : x.s;
        w.tile = x.s < 0 ? p.tiles : x.tiles - 1 - x.level;
    }
    const int head0 = w.g * qpk;  // the group's first query head
    where_rows(p, w);
    const int n0 = w.tile * BN;
    const int kall = p.cu ? w.nk : p.Tk;  // rows that dk and dv have (hidden ones get zeros)
    if (n0 >= kall) return;
    const int kj = n0 + 32 * wave + n;  // this lane's key
    const int kc = kj < w.nk ? kj : (w.nk > 0 ? w.nk - 1 : 0);
    const uint16_t *kr = static_cast<const uint16_t *>(p.k) + w.bk * p.ks[0] + (w.k0 + kc) * p.ks[1] + w.g * p.ks[2];
    const uint16_t *vb = static_cast<const uint16_t *>(p.v) + w.bk * p.vs[0] + w.k0 * p.vs[1] + w.g * p.vs[2];
    const uint16_t *vr = vb + kc * p.vs[1];
    uint4 kf[KS], vf[kVLds ? 1 : KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        kf[s] = *reinterpret_cast<const uint4 *>(kr + 16 * s + 8 * h);
        if constexpr (!kVLds) vf[s] = *reinterpret_cast<const uint4 *>(vr + 16 * s + 8 * h);
    }
    // First query that sees this lane's key, any of the wave's, all of the wave's.
    const int big = 0x7fffffff;
    const int first = kj >= w.nk ? big : (p.causal ? kj - w.shift : 0);
    const int wk0 = n0 + 32 * wave;
    const int wfirst = wk0 >= w.nk ? big : (p.causal ? wk0 - w.shift : 0);
    const int wall = wk0 + 31 >= w.nk ? big : (p.causal ? wk0 + 31 - w.shift : 0);
    int gfirst = n0 >= w.nk ? big : (p.causal ? n0 - w.shift : 0);
    gfirst = gfirst < 0 ? 0 : gfirst;
    const int t0 = gfirst / BQ;
    const int nt = gfirst >= w.nq ? 0 : (w.nq + BQ - 1) / BQ - t0;
    const float c = p.scale * kLog2e;
    const float p16 = PK == PrecKind::F16 ? kP16 : 0.0f;

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        dk[d] = zero16();
        dv[d] = zero16();
    }
    // fp16: one scale for every head of the group, the smallest of theirs.
    float sc = 1.0f;
    if constexpr (PK == PrecKind::F16) {
        sc = ds_scale<PK>(p, w, head0);
        for (int r = 1; r < qpk; ++r) sc = fminf(sc, ds_scale<PK>(p, w, head0 + r));
    }
    const float ds_mul = PK == PrecKind::F16 ? sc * ldexpf(1.0f, -14) : 1.0f;

    // Steps: the first nm query tiles of each head of the group, which not every key of the
    // workgroup's sees whole, then the others of each head; this share's are x0 .. x0 + steps - 1.
    // At D = 64 all are taken as the first kind: the second loop costs more than it saves there
    // (forward and backward, with it and without: B4 T2048 H16 D64 216 and 205 us, B2 T8192 H16
    // G4 D128 2279 and 2309).
    const int gall = n0 + BN > w.nk ? big : (p.causal ? n0 + BN - 1 - w.shift : 0);
    int nm = gall >= w.nq ? nt : (gall + BQ - 1) / BQ - t0;
    nm = D == 64 ? nt : (nm < 0 ? 0 : nm);
    const int x0 = static_cast<int>(static_cast<int64_t>(nt) * qpk * share / p.splits);
    const int steps = static_cast<int>(static_cast<int64_t>(nt) * qpk * (share + 1) / p.splits) - x0;
    const uint16_t *qb = static_cast<const uint16_t *>(p.q) + w.bq * p.qs[0] + w.q0 * p.qs[1];
    const uint16_t *db = static_cast<const uint16_t *>(p.dout) + (w.bq * static_cast<int64_t>(p.Tq) + w.q0) * p.H * D;
    const Stream qs = stream_of<D, NW>(qb, p.qs[1], wave, lane);
    const Stream ds = stream_of<D, NW>(db, static_cast<int64_t>(p.H) * D, wave, lane);
    const int64_t sb = static_cast<int64_t>(w.bq) * p.H * p.Tq + w.q0;
    const int masked = nm * qpk - x0;  // steps of the first kind left to this share
    int lo = masked > 0 ? 0 : nm, hi = masked > 0 ? nm : nt;  // tiles of the kind
    const int y0 = masked > 0 ? x0 : -masked;
    int rh = hi > lo ? y0 / (hi - lo) : 0, rt = hi > lo ? lo + y0 - rh * (hi - lo) : 0;  // of the step requested next
    int ci = 0, ni = 0;  // first query of the current step, and of the one requested last
    // L and D of the queries of a step travel through a register (`next`), stored after
    // the products of the step before: stored at once, the store would wait for
    // every tile request ahead of it.
    float next = 0.0f;
    auto keep = [&](float *sl) __attribute__((always_inline)) {
        if (tid < 2 * BQ) sl[tid] = tid < BQ ? next - p16 : next * ds_mul;
    };
    auto request = [&](char *tq, char *td) __attribute__((always_inline)) {
        const int hh = head0 + rh, row0 = (t0 + rt) * BQ;
        ni = row0;
        Stream qh = qs, dh = ds;
        qh.base += 2 * hh * p.qs[2];
        dh.base += 2 * hh * D;
        stage<D, NW, BQ>(qh, row0, w.nq, tq, wave, lane);
        stage<D, NW, BQ>(dh, row0, w.nq, td, wave, lane);
        if (tid < 2 * BQ) {
            const int r = row0 + (tid & (BQ - 1));
            const float *src = (tid < BQ ? p.lse : p.delta) + sb + static_cast<int64_t>(hh) * p.Tq;
            // Queries past the end: L = +inf hides them.
            next = r < w.nq ? src[r] : (tid < BQ ? INFINITY : 0.0f);
        }
        if (++rt == hi) {
            if (++rh == qpk) {
                rh = 0;
                lo = nm;
                hi = nt;
            }
            rt = lo;
        }
    };
    if (steps > 0) {
        request(sq0, sd0);
        if constexpr (kVLds) {
            // A tile of kTile rows at a time, each from a base of its own; of one past the
            // last key (whose rows are hidden) that key.
            const Stream vt = stream_of<D, NW>(vb, p.vs[1], wave, lane);
#pragma unroll
            for (int r = 0; r < BN; r += kTile)
                stage<D, NW>(vt, n0 + r < w.nk ? n0 + r : w.nk - 1, w.nk, sv + r * D * 2, wave, lane);
        }
    }
    auto step = [&](int x, auto buf, auto hidden) __attribute__((always_inline)) {
        constexpr bool kOdd = decltype(buf)::value, kHide = decltype(hidden)::value;
        const char *const tq = kOdd ? sq1 : sq0, *const td = kOdd ? sd1 : sd0;
        keep(kOdd ? sl1 : sl0);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        ci = ni;
        if (x + 1 < steps) request(kOdd ? sq0 : sq1, kOdd ? sd0 : sd1);
        const int i0 = ci;
        if (kHide && i0 + BQ <= wfirst) return;
        const int rr = opaque(rb), cc = opaque(cb);
        if constexpr (D == 128) mix_reads();
        const float *const lt = kOdd ? sl1 : sl0, *const et = lt + BQ;
#pragma unroll
        for (int a = 0; a < BQ / 32; ++a) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int st = 0; st < KS; ++st) s = mma32<PK>(s, row_frag<D>(tq, rr, 32 * a, st), kf[st]);
            if (kHide && i0 < wall) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int qi = i0 + 32 * a + 8 * (i >> 2) + 4 * h + (i & 3);
                    s[i] = qi >= first ? s[i] : -INFINITY;
                }
            }
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                uint4 bv;
                if constexpr (kVLds)
                    bv = row_frag<D>(sv, rr, 32 * wave, st);
                else
                    bv = vf[st];
                dp = mma32<PK>(dp, row_frag<D>(td, rr, 32 * a, st), bv);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 lv = *reinterpret_cast<const float4 *>(lt + 32 * a + 8 * b + 4 * h);
                const float ls[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * b + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * b + i], c, -ls[i]));
            }
            // add_columns, written out: through it the compiler spilled 13 registers here and
            // not 3 (B2 T8192 H16 G4 D128 forward and backward 2320 us against 2269).
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint4 pf = pack8<PK>(s, u);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint4 cf = col_frag<D>(td, cc, 32 * a + 16 * u, d);
                    dv[d] = mma32<PK>(dv[d], cf, pf);
                    if constexpr (FINE) dv[d] = mma32<PK>(dv[d], cf, rest8<PK>(s, u, pf));
                }
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 ev = *reinterpret_cast<const float4 *>(et + 32 * a + 8 * b + 4 * h);
                const float es[4] = {ev.x, ev.y, ev.z, ev.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[4 * b + i] *= PK == PrecKind::F16 ? fmaf(dp[4 * b + i], ds_mul, -es[i]) : dp[4 * b + i] - es[i];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint4 pf = pack8<PK>(s, u);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint4 cf = col_frag<D>(tq, cc, 32 * a + 16 * u, d);
                    dk[d] = mma32<PK>(dk[d], cf, pf);
                    if constexpr (FINE) dk[d] = mma32<PK>(dk[d], cf, rest8<PK>(s, u, pf));
                }
            }
        }
    };
    int x = 0;
    for (; x < steps && x < masked; x += 2) {
        step(x, std::false_type{}, std::true_type{});
        if (x + 1 < steps) step(x + 1, std::true_type{}, std::true_type{});
    }
    if constexpr (D == 128)
        for (; x < steps; x += 2) {
            step(x, std::false_type{}, std::false_type{});
            if (x + 1 < steps) step(x + 1, std::true_type{}, std::false_type{});
        }
    const float fk = p.scale / sc, fv = PK == PrecKind::F16 ? ldexpf(1.0f, -14) : 1.0f;
    const int64_t krow = ((w.bk * static_cast<int64_t>(p.Tk) + w.k0 + kj) * p.G + w.g) * D;
    if (p.splits > 1) {
        if (kj >= kall) return;
        const int64_t all = static_cast<int64_t>(p.B) * p.Tk * p.G * D;
        float *pk = p.part + 2 * share * all + krow, *pv = pk + all;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *reinterpret_cast<float4 *>(pk + 32 * d + 8 * i + 4 * h) = make_float4(
                    dk[d][4 * i] * fk, dk[d][4 * i + 1] * fk, dk[d][4 * i + 2] * fk, dk[d][4 * i + 3] * fk);
                *reinterpret_cast<float4 *>(pv + 32 * d + 8 * i + 4 * h) = make_float4(
                    dv[d][4 * i] * fv, dv[d][4 * i + 1] * fv, dv[d][4 * i + 2] * fv, dv[d][4 * i + 3] * fv);
            }
        return;
    }
    __syncthreads();  // the tiles are done with
    char *const so = wave == 0 ? sq0 : wave == 1 ? sq1 : wave == 2 ? sd0 : sd1;
    auto to = [&](int r) __attribute__((always_inline)) {
        const int kr = n0 + 32 * wave + r;
        return kr < kall ? ((w.bk * static_cast<int64_t>(p.Tk) + w.k0 + kr) * p.G + w.g) * D : int64_t{-1};
    };
    put_rows<D>(so, lane, dk, [&](float a, float b, float c, float d) __attribute__((always_inline)) {
        return pack4<PK>(a * fk, b * fk, c * fk, d * fk);
    });
    write_rows<D>(so, lane, static_cast<uint16_t *>(p.dk), to);
    put_rows<D>(so, lane, dv, [&](float a, float b, float c, float d) __attribute__((always_inline)) {
        return pack4<PK>(a * fv, b * fv, c * fv, d * fv);
    });
    write_rows<D>(so, lane, static_cast<uint16_t *>(p.dv), to);
}

// Sums of n shares of `all` values each, stride apart, in their order, rounded; thread: 4
// values.  Of a second result (blockIdx.y = 1) each share follows the first's.  Bound by
// the read: B1 T7013 G4 D128, dk and dv in 4 shares (115 MB) 20 us, 5.7 TB/s.
template <PrecKind PK>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float *part, int64_t stride, int n, uint16_t *out,
                                                       uint16_t *out1, int64_t all)
{
    if (blockIdx.y) {
        part += all;
        out = out1;
    }
    const int64_t e = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (e >= all) return;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const float4 y = *reinterpret_cast<const float4 *>(part + s * stride + e);
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
    }
    st_q4<PK>(out + e, pack4<PK>(x.x, x.y, x.z, x.w));
}

template <PrecKind PK>
hipError_t sum_shares(const float *part, int64_t stride, int n, void *out, void *out1, int64_t all, hipStream_t s)
{
    hipLaunchKernelGGL((attn_sum_kernel<PK>), dim3(static_cast<unsigned>((all / 4 + 255) / 256), out1 ? 2 : 1),
                       dim3(256), 0, s, part, stride, n, static_cast<uint16_t *>(out), static_cast<uint16_t *>(out1), all);
    return hipGetLastError();
}

// Four waves per workgroup, two workgroups per CU: against eight waves and one, the
// same time on long rows and less on short ones, whose few workgroups fill the card
// more evenly (forward, with the first tiles: B1 T4096 H16 D64 72 us against 87; packed, 9
// sequences of 7013 tokens, H16 D128 78 against 97; B2 T8192 H16 D128 556 against 574).
constexpr int kWaves = 4;
static_assert(32 * kWaves == 128, "q_tiles, k_tiles and packed_tile count tiles of 128 rows");

// Tiles of one head, each sequence having as many as the longest, or looked up.  A
// workgroup without a tile ends after 0.7 ns of the card's time, a lookup costs it 2
// (hundreds of sequences) to 6 (thousands).  H16 G4 D128, forward and backward, looked
// up against not: one document of 16384 tokens among 400 of 20 .. 200 (51000 against 900
// tiles) 7030 us against 8102; 1000 of 20 .. 100 (1000, all of them there; H16 G16 D64)
// 1146 against 794; 9 of 259 .. 1348 (99 against 62) 327 against 324.
// Sets that, the tiles, and `dealt` (turn_of), for a launch over `all` tiles of a group (a
// token being `rows` of their rows) in `shares`; returns its workgroups.  Dealt from 4096
// workgroups (four to eight rounds), of enough groups that a short last deal does not count.
int64_t set_grid(AttnTrainParams &p, int64_t all, int64_t rows, int shares)
{
    p.tiles = static_cast<int>(p.cu ? (p.max_q * rows + 127) / 128 : all / p.nseq);
    const int64_t even = static_cast<int64_t>(p.nseq) * p.tiles;
    p.ranked = p.cu && even > 8 * all;
    const int64_t groups = static_cast<int64_t>(p.ranked ? 1 : p.nseq) * p.G;
    const int64_t tiles = (p.ranked ? all : p.tiles) * shares;
    p.dealt = tiles * groups >= 4096 && (groups % 8 == 0 || groups >= 64);
    return (p.dealt ? (groups + 7) / 8 * 8 : groups) * tiles;
}

// Whether P and dS are multiplied in two parts.  In short sequences few rounded terms make
// up a gradient, and one of them shows in D values of it: rounded once, the error
// of dk against 64 bits is 2.8 times that of rounding the exact result at 2 tokens, 1.6 at
// 8, 1.5 at 64 and below 1.5 past 128; in two parts it is the same as that.  The products
// they add are cheap there (when they came: forward and backward in two parts and in one, B64
// T64 H8 D64 27.2 and 26.2 us, B256 T128 H16 D64 366 and 359, B64 T128 H16 G4 D128 124
// and 121).
bool attn_fine(const AttnTrainParams &p)
{
    return p.max_q <= 128 && (p.cu || p.Tk <= 128);
}

template <PrecKind PK, int D>
hipError_t fwd_d(AttnTrainParams p, hipStream_t s)
{
    const unsigned grid = static_cast<unsigned>(set_grid(p, p.q_tiles, p.H / p.G, p.splits_f));
    hipLaunchKernelGGL((attn_fine(p) ? attn_fwd_kernel<PK, D, kWaves, true> : attn_fwd_kernel<PK, D, kWaves, false>),
                       dim3(grid), dim3(64 * kWaves), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits_f == 1) return e;
    const int64_t threads = static_cast<int64_t>(p.B) * p.Tq * p.H * (D / 4);
    hipLaunchKernelGGL((attn_fwd_join_kernel<PK>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, s,
                       p);
    return hipGetLastError();
}

template <PrecKind PK, int D>
hipError_t bwd_d(AttnTrainParams p, hipStream_t s)
{
    hipError_t e;
    if constexpr (PK == PrecKind::F16) {
        const int64_t all = static_cast<int64_t>(kNormParts) * p.B * (p.H + p.G), most = max_workgroups(256);
        for (int64_t first = 0; first < all; first += most) {
            hipLaunchKernelGGL((norm_max_kernel<D>), dim3(static_cast<unsigned>(all - first < most ? all - first : most)),
                               dim3(256), 0, s, p, static_cast<unsigned>(first));
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    if (p.Tq > 0 && p.max_q > 0) {
        const unsigned grid = static_cast<unsigned>(set_grid(p, p.q_tiles, p.H / p.G, p.splits_q));
        hipLaunchKernelGGL((attn_fine(p) ? attn_dq_kernel<PK, D, kWaves, true> : attn_dq_kernel<PK, D, kWaves, false>),
                           dim3(grid), dim3(64 * kWaves), 0, s, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        const int64_t all = static_cast<int64_t>(p.B) * p.Tq * p.H * D;
        if (p.splits_q > 1 && (e = sum_shares<PK>(p.part_q, all, p.splits_q, p.dq, nullptr, all, s)) != hipSuccess) return e;
    }
    if (p.Tk > 0) {
        // Query rows per tile: at D = 128 half of the other's, so that two
        // workgroups' tiles and V rows fit a CU's LDS.
        constexpr int BQ = D == 64 ? 64 : 32;
        const unsigned grid = static_cast<unsigned>(set_grid(p, p.k_tiles, 1, p.splits));
        hipLaunchKernelGGL((attn_fine(p) ? attn_dkv_kernel<PK, D, kWaves, BQ, true>
                                         : attn_dkv_kernel<PK, D, kWaves, BQ, false>),
                           dim3(grid), dim3(64 * kWaves), 0, s, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        const int64_t all = static_cast<int64_t>(p.B) * p.Tk * p.G * D;
        if (p.splits > 1) e = sum_shares<PK>(p.part, 2 * all, p.splits, p.dk, p.dv, all, s);
        return e;
    }
    return hipGetLastError();
}

}  // namespace

bool attn_train_supported(int io_dtype, int D)
{
    return (io_dtype == GDN2_DTYPE_BF16 || io_dtype == GDN2_DTYPE_F16) && (D == 64 || D == 128);
}

// The joins and sums of shares are small: shares are made of few workgroups.
bool attn_launchable(const AttnTrainParams &p, bool backward)
{
    AttnTrainParams q = p;
    const int64_t most = max_workgroups(64 * kWaves);
    // Before the exact count: every tile takes a workgroup, and the products below fit 64 bits.
    if (static_cast<double>(p.q_tiles) * p.G * p.splits_f > static_cast<double>(most) ||
        (backward && static_cast<double>(p.k_tiles) * p.G * p.splits > static_cast<double>(most)))
        return false;
    if (p.nseq == 0) return true;
    return (p.q_tiles == 0 || set_grid(q, p.q_tiles, p.H / p.G, p.splits_f) <= most) &&
           (!backward || p.k_tiles == 0 || set_grid(q, p.k_tiles, 1, p.splits) <= most);
}

// Shares of a key tile's queries in attn_dkv_kernel.  Two workgroups fit a CU: 512
// fill the card, and causal ones, of unequal length, even out over two rounds with
// the longest first.  Fewer are split, as long as a share keeps 16 query tiles of 64 (a
// shorter one is over before its start and its sums' traffic are paid).  Backward in
// us, with the first tiles, with 1 / 2 / 4 / 8 shares: B2 T8192 H16 G4 D128 causal (512 workgroups)
// 2314 / 1812 / 1814 / 1913; packed 7013 tokens, H16 G4 D128 (240) 310 / 217 / 184 / 223;
// B1 T4096 H16 G2 D64 (64) 795 / 456 / 288 / 213; B4 T2048 H16 D64 (1024)
// 162 / 207 / 274 / 421; B8 T509 H8 D64, not causal (256, 8 tiles each) 53 / 59 / 63 / 80.
// With the present ones, for 1024 and 512 causal workgroups, forward and backward: B2
// T8192 2211 and 2524, packed 296 and 312.
int attn_bwd_splits(const AttnTrainParams &p)
{
    const int64_t wgs = p.k_tiles * p.G, want = p.causal ? 1024 : 512;
    const int64_t steps = static_cast<int64_t>(p.H / p.G) * ((p.max_q + 63) / 64);
    int64_t s = wgs > 0 ? (want + wgs / 2) / wgs : 1;
    s = s < steps / 16 ? s : steps / 16;
    return static_cast<int>(s < 1 ? 1 : (s > 16 ? 16 : s));
}

// Shares of the keys in the query-resident kernels, where few queries face many
// keys: up to 512 workgroups, of at least 8 key tiles of the row each (of packed rows too,
// whose sequences may be shorter: shares of a short one then hold less, or nothing).
int attn_key_shares(const AttnTrainParams &p)
{
    const int64_t wgs = p.q_tiles * p.G, tiles = (p.Tk + kTile - 1) / kTile;
    if (wgs == 0 || wgs >= 256) return 1;
    int64_t s = 512 / wgs;
    s = s < tiles / 8 ? s : tiles / 8;
    return static_cast<int>(s < 1 ? 1 : (s > 64 ? 64 : s));
}

static size_t up16(size_t x) { return (x + 15) & ~static_cast<size_t>(15); }

// The shares' values, maxima and sums.
size_t attn_fwd_workspace_bytes(const AttnTrainParams &p)
{
    const size_t rows = static_cast<size_t>(p.B) * p.Tq * p.H;
    return p.splits_f > 1 ? p.splits_f * rows * (p.D + 2) * sizeof(float) : 0;
}

void attn_fwd_workspace(AttnTrainParams &p, void *workspace)
{
    p.part = static_cast<float *>(workspace);
    p.part_ml = p.part + static_cast<size_t>(p.splits_f) * p.B * p.Tq * p.H * p.D;
}

// D per query, fp16's norms, the shares' sums of dk and dv and of dq.
size_t attn_bwd_workspace_bytes(const AttnTrainParams &p)
{
    AttnTrainParams q = p;
    return attn_bwd_workspace(q, nullptr);
}

size_t attn_bwd_workspace(AttnTrainParams &p, void *workspace)
{
    char *w = static_cast<char *>(workspace);
    size_t at = 0;
    auto take = [&](size_t floats) {
        float *x = reinterpret_cast<float *>(w + at);
        at += up16(floats * sizeof(float));
        return x;
    };
    const size_t q = static_cast<size_t>(p.B) * p.Tq * p.H, k = static_cast<size_t>(p.B) * p.Tk * p.G;
    p.delta = take(q);
    p.mx_do = take(static_cast<size_t>(p.B) * p.H * kNormParts);
    p.mx_v = take(static_cast<size_t>(p.B) * p.G * kNormParts);
    p.part = take(p.splits > 1 ? p.splits * 2 * k * p.D : 0);
    p.part_q = take(p.splits_q > 1 ? p.splits_q * q * p.D : 0);
    return at;
}

hipError_t launch_attn_fwd(const AttnTrainParams &p, int io_dtype, hipStream_t s)
{
    if (io_dtype == GDN2_DTYPE_BF16)
        return p.D == 64 ? fwd_d<PrecKind::BF16, 64>(p, s) : fwd_d<PrecKind::BF16, 128>(p, s);
    return p.D == 64 ? fwd_d<PrecKind::F16, 64>(p, s) : fwd_d<PrecKind::F16, 128>(p, s);
}

hipError_t launch_attn_bwd(const AttnTrainParams &p, int io_dtype, hipStream_t s)
{
    if (io_dtype == GDN2_DTYPE_BF16)
        return p.D == 64 ? bwd_d<PrecKind::BF16, 64>(p, s) : bwd_d<PrecKind::BF16, 128>(p, s);
    return p.D == 64 ? bwd_d<PrecKind::F16, 64>(p, s) : bwd_d<PrecKind::F16, 128>(p, s);
}

}  // namespace gdn2

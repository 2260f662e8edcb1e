// Tiles of the attention kernels over whole sequences and over pieces of prompts
// (v_mfma_f32_32x32x16; layouts in gdn2_attn_train.hip): operands from rows and columns of LDS
// tiles, accumulators as the next product's operands, results as whole rows.
#pragma once

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

// Asks the scheduler to alternate LDS reads and matrix products in a block (D = 128, where
// the products bound it: forward 516 -> 507 us, forward and backward 2250 -> 2196, B2
// T8192 H16 G4; at D = 64 the backward lost 3%).
__device__ __forceinline__ void mix_reads()
{
    __builtin_amdgcn_iglp_opt(0);
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

}  // namespace
}  // namespace gdn2

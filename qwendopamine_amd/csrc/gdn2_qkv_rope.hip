// Norms of queries and keys for each head with the rotation of positions, in one
// pass over a fused projection, their gradient, and the same pass storing keys and
// values into a paged cache, gfx950.
//
//   r = (mean x^2 + eps)^-1/2,  n = x r w                       (or n = x, without weights)
//   y_2i = n_2i c_i - n_2i+1 s_i,  y_2i+1 = n_2i s_i + n_2i+1 c_i   (2 i < rot; y = n above)
// with the gradient, dn the inverse rotation of dy,
//   dw = sum dn x r,  dx = r (dn w - x r mean(dn w x r))
//
// A row of D channels is LPR lanes of 8 channels, so that a pair never leaves its
// lane and the mean is log2(LPR) exchanges; a wave takes U x 64 / LPR rows of one
// token, all requested before the first is used, and the token's angles once for
// all of them.  Nothing is kept for the backward but the projection itself: r costs
// one mean, and reading it back would cost more than forming it.  Both directions
// are bound by memory: 16384 tokens H32 G8 D128 without norms 62 us, 5.5 TB/s (float32 150); B4 T2048 H16 G16
// D64 with norms 16 us forward (4.2 TB/s) and 28 backward (4.8), its weights' sum 4; into pages 22 (3.8).
#include "gdn2_common.h"
#include "gdn2_internal.h"

namespace gdn2 {
namespace {

// U: rows in flight per lane.  The backward holds two tensors' rows and the weights' sums: with 2 it is 28 us at
// B4 T2048 H16 G16 D64 and 26 at T7013 H16 G4 D128, with 4, at fewer waves, 38 and 36.
constexpr int kRowsFwd = 4, kRowsBwd = 2;

struct Row8 {
    float x[8];
};

template <typename T>
__device__ __forceinline__ Row8 load8(const T *p)
{
    Row8 r;
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        r.x[0] = a.x; r.x[1] = a.y; r.x[2] = a.z; r.x[3] = a.w;
        r.x[4] = b.x; r.x[5] = b.y; r.x[6] = b.z; r.x[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t lo = static_cast<uint16_t>(w[i] & 0xffffu), hi = static_cast<uint16_t>(w[i] >> 16);
            if constexpr (std::is_same<T, bf16_t>::value) {
                r.x[2 * i] = bf16_bits_to_f32(lo);
                r.x[2 * i + 1] = bf16_bits_to_f32(hi);
            } else {
                r.x[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, lo));
                r.x[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, hi));
            }
        }
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const Row8 &r)
{
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(r.x[0], r.x[1], r.x[2], r.x[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(r.x[4], r.x[5], r.x[6], r.x[7]);
    } else {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, bf16_t>::value) {
                w[i] = f32x2_to_bf16x2_bits(r.x[2 * i], r.x[2 * i + 1]);
            } else {
                w[i] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(r.x[2 * i])) |
                       static_cast<unsigned>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(r.x[2 * i + 1]))) << 16;
            }
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Sum over the LPR lanes of a row.
template <int LPR>
__device__ __forceinline__ float row_sum(float x)
{
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// A lane's angles: pairs 4 c .. 4 c + 3 of the token's position; 1, 0 past the rotated channels.
struct Angles {
    float c[4], s[4];
    bool on[4];
};
__device__ __forceinline__ Angles angles_of(const QkvRopeParams &p, int64_t pos, int c)
{
    Angles a;
    const float *cr = p.cos + pos * p.pairs, *sr = p.sin + pos * p.pairs;
    if (p.pairs % 4 == 0 && p.wide_tables) {
        const bool on = 4 * c < p.pairs;
        const float4 u = on ? *reinterpret_cast<const float4 *>(cr + 4 * c) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        const float4 v = on ? *reinterpret_cast<const float4 *>(sr + 4 * c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        a.c[0] = u.x; a.c[1] = u.y; a.c[2] = u.z; a.c[3] = u.w;
        a.s[0] = v.x; a.s[1] = v.y; a.s[2] = v.z; a.s[3] = v.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) a.on[i] = on;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a.on[i] = 4 * c + i < p.pairs;
            a.c[i] = a.on[i] ? cr[4 * c + i] : 1.0f;
            a.s[i] = a.on[i] ? sr[4 * c + i] : 0.0f;
        }
    }
    return a;
}

// Rotation by the angles (BACK: by their negatives), every product and sum rounded by
// itself, as torch's separate operations round.
template <bool BACK>
__device__ __forceinline__ void rotate(Row8 &r, const Angles &a)
{
#pragma clang fp contract(off)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = r.x[2 * i], y = r.x[2 * i + 1];
        const float xc = x * a.c[i], ys = y * a.s[i], xs = x * a.s[i], yc = y * a.c[i];
        r.x[2 * i] = a.on[i] ? (BACK ? xc + ys : xc - ys) : x;
        r.x[2 * i + 1] = a.on[i] ? (BACK ? yc - xs : xs + yc) : y;
    }
}

template <typename T>
__device__ __forceinline__ Row8 weights(const QkvRopeParams &p, const void *w, int ch)
{
    return p.w_f32 ? load8(static_cast<const float *>(w) + ch) : load8(static_cast<const T *>(w) + ch);
}

// What a unit (a wave's work) is: token b, t and its rows row0 .. row0 + U 64 / LPR - 1.
struct Unit {
    int b, t, row0;
};
template <int LPR, int U>
__device__ __forceinline__ Unit unit_of(const QkvRopeParams &p, int64_t unit)
{
    const unsigned u = static_cast<unsigned>(unit);
    const unsigned token = u / p.units, b = token / p.T;
    return {static_cast<int>(b), static_cast<int>(token - b * p.T),
            static_cast<int>(u - token * p.units) * (U * (64 / LPR))};
}

// The token's position; -1 where it has none (outside the tables, or padding).
__device__ __forceinline__ int64_t position_of(const QkvRopeParams &p, const Unit &w)
{
    if (p.lengths && w.t >= p.lengths[w.b]) return -1;
    int64_t pos = w.t;
    if (p.pos) {
        pos = p.pos[w.b * p.pos_b + w.t * p.pos_t];
        if (p.pos_add_t) pos = pos >= 0 && pos < p.table_rows ? pos + w.t : -1;
    }
    return pos >= 0 && pos < p.table_rows ? pos : -1;
}

// Row i of a token's `per` rows a group (R query heads, the key, with PAGED the values).
struct Head {
    int g, slot;
};
__device__ __forceinline__ Head head_of(const QkvRopeParams &p, int i)
{
    const int g = static_cast<int>(__umulhi(static_cast<unsigned>(i), p.per_m));
    return {g, i - g * p.per};
}

// Rows are dealt to lanes i = row0 + u 64 / LPR + lane / LPR; ROPE: q and k rows into q and
// k, PAGED: k and v rows into pages.  A token without a position has zeros for q (and k).
template <typename T, int LPR, bool PAGED, bool NORM>
__global__ __launch_bounds__(256) void qkv_rope_kernel(QkvRopeParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (unit >= p.all_units) return;
    const Unit w = unit_of<LPR, kRowsFwd>(p, unit);
    const int c = lane & (LPR - 1), ch = 8 * c;
    const bool in = ch < p.D;
    const int64_t token = static_cast<int64_t>(w.b) * p.T + w.t;
    const T *x = static_cast<const T *>(p.qkv) + w.b * p.stride_b + w.t * p.stride_t + (in ? ch : 0);
    const int R = p.R, D = p.D;
    Head hd[kRowsFwd];
    Row8 v[kRowsFwd];
    bool have[kRowsFwd];
#pragma unroll
    for (int u = 0; u < kRowsFwd; ++u) {
        const int i = w.row0 + u * (64 / LPR) + lane / LPR;
        have[u] = in && i < p.G * p.per;
        hd[u] = head_of(p, have[u] ? i : 0);
        v[u] = load8(x + (hd[u].g * (R + 2) + hd[u].slot) * D);
    }
    int64_t pos = position_of(p, w);
    // The token's place in the cache.
    int64_t page = -1;
    int at = 0;
    if constexpr (PAGED) {
        const int64_t n = static_cast<int64_t>(p.table_cols) * p.page;
        if (pos >= n) pos = -1;
        if (pos >= 0) {
            const int col = static_cast<int>(pos) / p.page;
            at = static_cast<int>(pos) - col * p.page;
            page = p.table[w.b * p.table_stride + col];
            if (page >= p.pages) page = -1;
        }
    }
    T *q = static_cast<T *>(p.q) + token * p.G * R * D + ch;
    if (pos < 0) {
        const Row8 zero = {};
#pragma unroll
        for (int u = 0; u < kRowsFwd; ++u) {
            if (!have[u]) continue;
            if (hd[u].slot < R)
                store8(q + (hd[u].g * R + hd[u].slot) * D, zero);
            else if constexpr (!PAGED)
                store8(static_cast<T *>(p.k) + (token * p.G + hd[u].g) * D + ch, zero);
        }
        return;
    }
    const Angles a = angles_of(p, pos, c);
    Row8 wq, wk;
    if constexpr (NORM) {
        wq = weights<T>(p, p.wq, in ? ch : 0);
        wk = weights<T>(p, p.wk, in ? ch : 0);
    }
#pragma unroll
    for (int u = 0; u < kRowsFwd; ++u) {
        const bool is_q = hd[u].slot < R;
        Row8 y = v[u];
        if constexpr (NORM) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(y.x[e], y.x[e], ss);
            ss = row_sum<LPR>(in ? ss : 0.0f);
            const float r = rsqrtf(ss / static_cast<float>(D) + p.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) y.x[e] = y.x[e] * r * (is_q ? wq.x[e] : wk.x[e]);
        }
        rotate<false>(y, a);
        if (!have[u]) continue;
        if (is_q) {
            store8(q + (hd[u].g * R + hd[u].slot) * D, y);
        } else if constexpr (PAGED) {
            if (page >= 0) {
                const int64_t to = ((page * p.G + hd[u].g) * p.page + at) * D + ch;
                if (hd[u].slot == R)
                    store8(static_cast<T *>(p.k) + to, y);
                else
                    store8(static_cast<T *>(p.v) + to, v[u]);
            }
        } else {
            store8(static_cast<T *>(p.k) + (token * p.G + hd[u].g) * D + ch, y);
        }
    }
}

// Gradient.  Workgroups walk the units in a fixed stride; the weights' gradients are summed
// in the lanes, then over the wave's rows and the waves, and left as one row [2][D] for
// each workgroup, which qkv_rope_dw_kernel adds in a fixed order.
template <typename T, int LPR, bool NORM>
__global__ __launch_bounds__(256) void qkv_rope_bwd_kernel(QkvRopeParams p)
{
    constexpr int RPW = 64 / LPR;
    __shared__ float s_dw[4][2][8 * LPR];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & (LPR - 1), ch = 8 * c;
    const bool in = ch < p.D;
    const int R = p.R, D = p.D;
    Row8 wq, wk, gq = {}, gk = {};
    if constexpr (NORM) {
        wq = weights<T>(p, p.wq, in ? ch : 0);
        wk = weights<T>(p, p.wk, in ? ch : 0);
    }
    for (int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave; unit < p.all_units; unit += 4LL * gridDim.x) {
        const Unit w = unit_of<LPR, kRowsBwd>(p, unit);
        const int64_t token = static_cast<int64_t>(w.b) * p.T + w.t;
        const T *x = static_cast<const T *>(p.qkv) + w.b * p.stride_b + w.t * p.stride_t + (in ? ch : 0);
        Head hd[kRowsBwd];
        Row8 dy[kRowsBwd], v[kRowsBwd];
        bool have[kRowsBwd];
#pragma unroll
        for (int u = 0; u < kRowsBwd; ++u) {
            const int i = w.row0 + u * RPW + lane / LPR;
            have[u] = in && i < p.G * p.per;
            hd[u] = head_of(p, have[u] ? i : 0);
            const int cin = in ? ch : 0;
            const T *from = hd[u].slot < R
                                ? static_cast<const T *>(p.q) + (token * p.G * R + hd[u].g * R + hd[u].slot) * D + cin
                                : static_cast<const T *>(hd[u].slot == R ? p.k : p.v) + (token * p.G + hd[u].g) * D + cin;
            dy[u] = load8(from);
            if constexpr (NORM) v[u] = load8(x + (hd[u].g * (R + 2) + hd[u].slot) * D);
        }
        const int64_t pos = position_of(p, w);
        const Angles a = angles_of(p, pos < 0 ? 0 : pos, c);
        T *dx = static_cast<T *>(p.dqkv) + token * p.G * (R + 2) * D + ch;
#pragma unroll
        for (int u = 0; u < kRowsBwd; ++u) {
            const bool is_v = hd[u].slot > R, is_q = hd[u].slot < R;
            Row8 d = dy[u];
            rotate<true>(d, a);
            if constexpr (NORM) {
                float ss = 0.0f, dot = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float xe = v[u].x[e];
                    ss = fmaf(xe, xe, ss);
                    dot = fmaf(d.x[e] * (is_q ? wq.x[e] : wk.x[e]), xe, dot);
                }
                ss = row_sum<LPR>(in ? ss : 0.0f);
                dot = row_sum<LPR>(in ? dot : 0.0f);
                const float r = rsqrtf(ss / static_cast<float>(D) + p.eps);
                const float m = dot * r / static_cast<float>(D);
                const bool count = have[u] && !is_v && pos >= 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float xr = v[u].x[e] * r, g = d.x[e] * xr;
                    gq.x[e] += count && is_q ? g : 0.0f;
                    gk.x[e] += count && !is_q ? g : 0.0f;
                    d.x[e] = (d.x[e] * (is_q ? wq.x[e] : wk.x[e]) - xr * m) * r;
                }
            }
            if (pos < 0) d = Row8{};
            if (have[u]) store8(dx + (hd[u].g * (R + 2) + hd[u].slot) * D, is_v ? dy[u] : d);
        }
    }
    if constexpr (NORM) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int o = LPR; o < 64; o <<= 1) {
                gq.x[e] += __shfl_xor(gq.x[e], o, 64);
                gk.x[e] += __shfl_xor(gk.x[e], o, 64);
            }
        }
        if (lane < LPR) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s_dw[wave][0][ch + e] = gq.x[e];
                s_dw[wave][1][ch + e] = gk.x[e];
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 2 * D; e += 256) {
            const int k = e >= D, d = e - k * D;
            p.part[static_cast<int64_t>(blockIdx.x) * 2 * D + e] =
                (s_dw[0][k][d] + s_dw[1][k][d]) + (s_dw[2][k][d] + s_dw[3][k][d]);
        }
    }
}

constexpr int kSumWaves = 16, kSumDeep = 8;
template <typename T>
__global__ __launch_bounds__(64 * kSumWaves) void qkv_rope_dw_kernel(QkvRopeParams p, int parts)
{
    __shared__ float s_sum[kSumWaves][64];
    const int E = 2 * p.D;
    const int e = blockIdx.x * 64 + (threadIdx.x & 63);
    const float s = sum_parts<kSumWaves, kSumDeep>(p.part, parts, E, e < E ? e : E - 1, s_sum);
    if (threadIdx.x >= 64 || e >= E) return;
    void *to = e < p.D ? p.dwq : p.dwk;
    const int d = e < p.D ? e : e - p.D;
    if (p.w_f32)
        static_cast<float *>(to)[d] = s;
    else
        io<T>::st(static_cast<T *>(to), d, s);
}

template <typename T, int LPR>
hipError_t fwd_l(QkvRopeParams p, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>((p.all_units + 3) / 4)), block(256);
    const bool norm = p.wq != nullptr;
    if (p.table) {
        if (norm)
            hipLaunchKernelGGL((qkv_rope_kernel<T, LPR, true, true>), grid, block, 0, s, p);
        else
            hipLaunchKernelGGL((qkv_rope_kernel<T, LPR, true, false>), grid, block, 0, s, p);
    } else if (norm) {
        hipLaunchKernelGGL((qkv_rope_kernel<T, LPR, false, true>), grid, block, 0, s, p);
    } else {
        hipLaunchKernelGGL((qkv_rope_kernel<T, LPR, false, false>), grid, block, 0, s, p);
    }
    return hipGetLastError();
}

template <typename T, int LPR>
hipError_t bwd_l(QkvRopeParams p, hipStream_t s)
{
    const int blocks = qkv_rope_bwd_blocks(p.all_units);
    if (!p.wq) {
        hipLaunchKernelGGL((qkv_rope_bwd_kernel<T, LPR, false>), dim3(blocks), dim3(256), 0, s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((qkv_rope_bwd_kernel<T, LPR, true>), dim3(blocks), dim3(256), 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((qkv_rope_dw_kernel<T>), dim3((2 * p.D + 63) / 64), dim3(64 * kSumWaves), 0, s, p, blocks);
    return hipGetLastError();
}

template <typename T, bool BWD>
hipError_t rope_t(const QkvRopeParams &p, hipStream_t s)
{
    switch (qkv_rope_lanes(p.D)) {
    case 1: return BWD ? bwd_l<T, 1>(p, s) : fwd_l<T, 1>(p, s);
    case 2: return BWD ? bwd_l<T, 2>(p, s) : fwd_l<T, 2>(p, s);
    case 4: return BWD ? bwd_l<T, 4>(p, s) : fwd_l<T, 4>(p, s);
    case 8: return BWD ? bwd_l<T, 8>(p, s) : fwd_l<T, 8>(p, s);
    case 16: return BWD ? bwd_l<T, 16>(p, s) : fwd_l<T, 16>(p, s);
    default: return BWD ? bwd_l<T, 32>(p, s) : fwd_l<T, 32>(p, s);
    }
}

template <bool BWD>
hipError_t rope_d(QkvRopeParams &p, int io_dtype, hipStream_t s)
{
    // Rows of a group: the values are copied into pages, and in the gradient.
    p.per = p.R + (BWD || p.table ? 2 : 1);
    p.per_m = static_cast<unsigned>((0x100000000ULL + p.per - 1) / p.per);
    p.units = qkv_rope_units(p.G * p.per, p.D, BWD);
    p.all_units = static_cast<int64_t>(p.B) * p.T * p.units;
    p.wide_tables = ((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15) == 0;
    switch (io_dtype) {
    case GDN2_DTYPE_F32: return rope_t<float, BWD>(p, s);
    case GDN2_DTYPE_BF16: return rope_t<bf16_t, BWD>(p, s);
    default: return rope_t<f16_t, BWD>(p, s);
    }
}

}  // namespace

int qkv_rope_lanes(int D)
{
    int l = 1;
    while (8 * l < D) l *= 2;
    return l;
}

int qkv_rope_units(int rows, int D, bool backward)
{
    const int per = (backward ? kRowsBwd : kRowsFwd) * (64 / qkv_rope_lanes(D));
    return (rows + per - 1) / per;
}

// Few enough that their rows of partial sums cost little, and enough for every CU to
// hold four workgroups.
int qkv_rope_bwd_blocks(int64_t units)
{
    const int64_t b = (units + 3) / 4;
    return static_cast<int>(b < 1024 ? b : 1024);
}

hipError_t launch_qkv_rope_fwd(QkvRopeParams p, int io_dtype, hipStream_t s) { return rope_d<false>(p, io_dtype, s); }
hipError_t launch_qkv_rope_bwd(QkvRopeParams p, int io_dtype, hipStream_t s) { return rope_d<true>(p, io_dtype, s); }

}  // namespace gdn2

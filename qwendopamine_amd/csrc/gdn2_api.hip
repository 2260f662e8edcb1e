// extern "C" entry points of libgdn2_hip.so: argument validation and dispatch.
// Declarations and the reference interfaces they replace: include/gdn2_hip.h.

#include "gdn2_chunk.h"
#include "gdn2_common.h"
#include "gdn2_internal.h"

using namespace gdn2;

static bool valid_dtype(int d)
{
    return d == GDN2_DTYPE_F32 || d == GDN2_DTYPE_BF16 || d == GDN2_DTYPE_F16;
}

static int check_chunk_args(int io_dtype, int g_dtype, const int64_t *cu_seqlens,
                            const int64_t *cu_seqlens_host, int num_seqs, int B, int T, int H,
                            int K, int V, unsigned flags, const float *A_log)
{
    if (!valid_dtype(io_dtype) || !valid_dtype(g_dtype)) return GDN2_ERR_INVALID;
    if (B < 0 || T < 0 || H <= 0 || K <= 0 || V <= 0) return GDN2_ERR_INVALID;
    if (flags & ~(GDN2_FLAG_L2NORM_QK | GDN2_FLAG_GATE_IN_KERNEL | GDN2_FLAG_LOWER_BOUND |
                  GDN2_FLAG_SAVE_FOR_BWD | GDN2_FLAG_TRANSPOSE_STATE | GDN2_FLAG_SIGMOID_BW))
        return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_LOWER_BOUND) && !(flags & GDN2_FLAG_GATE_IN_KERNEL))
        return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_GATE_IN_KERNEL) && !A_log) return GDN2_ERR_INVALID;
    // Gate logits are an inference option: the backward reads b and w as given.
    if ((flags & GDN2_FLAG_SIGMOID_BW) && (flags & GDN2_FLAG_SAVE_FOR_BWD)) return GDN2_ERR_INVALID;
    if ((cu_seqlens == nullptr) != (cu_seqlens_host == nullptr)) return GDN2_ERR_INVALID;
    if (cu_seqlens && (B != 1 || num_seqs < 0)) return GDN2_ERR_INVALID;
    if (cu_seqlens_host) {
        if (cu_seqlens_host[0] != 0 || cu_seqlens_host[num_seqs] != T) return GDN2_ERR_INVALID;
        for (int i = 0; i < num_seqs; ++i)
            if (cu_seqlens_host[i + 1] < cu_seqlens_host[i]) return GDN2_ERR_INVALID;
    }
    return GDN2_OK;
}

static void fill_chunk_args(ChunkFwdArgs &a, const void *q, const void *k, const void *v,
                            const void *g, const void *b, const void *w, void *o,
                            const float *h0, float *ht, const float *A_log, const float *dt_bias,
                            float lower_bound, const int64_t *cu_seqlens, const int64_t *cu_host,
                            int num_seqs, int B, int T, int H, int K, int V, float scale,
                            unsigned flags, void *workspace, size_t workspace_bytes)
{
    a.q = q; a.k = k; a.v = v; a.g = g; a.b = b; a.w = w; a.o = o;
    a.h0 = h0;
    a.ht = ht;
    a.A_log = A_log;
    a.dt_bias = dt_bias;
    a.lower_bound = lower_bound;
    a.cu_seqlens = cu_seqlens;
    a.cu_host = cu_host;
    a.num_seqs = cu_seqlens ? num_seqs : B;
    a.B = B; a.T = T; a.H = H; a.K = K; a.V = V;
    a.scale = scale;
    a.flags = flags;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    a.stages = 3;
}

extern "C" {

int gdn2_abi_version(void) { return GDN2_ABI_VERSION; }

const char *gdn2_status_string(int status)
{
    switch (status) {
    case GDN2_OK: return "ok";
    case GDN2_ERR_INVALID: return "invalid argument";
    case GDN2_ERR_UNSUPPORTED: return "unsupported shape, dtype or option";
    case GDN2_ERR_LAUNCH: return "kernel launch failed";
    case GDN2_ERR_WORKSPACE: return "workspace missing or too small";
    case GDN2_ERR_SCRATCH:
        return "the shape needs more than the static scratch array of gdn2_chunk_fwd_static "
               "holds (GDN2_STATIC_SCRATCH_BYTES = 72 MiB); use gdn2_chunk_fwd with a workspace";
    default: return "unknown status";
    }
}

int gdn2_recurrent_fwd_ex(const void *q, const void *k, const void *v, const void *g,
                          const void *b, const void *w, int io_dtype, int g_dtype, void *o,
                          const float *initial_state, int64_t initial_state_rows,
                          int64_t initial_state_row_stride, float *final_state,
                          int64_t final_state_rows, int64_t final_state_row_stride,
                          const float *A_log, const float *dt_bias, float lower_bound,
                          const int64_t *cu_seqlens, int num_seqs,
                          const void *ssm_state_indices, int indices_dtype,
                          int64_t indices_numel, int64_t indices_seq_stride,
                          const void *num_accepted_tokens, int accepted_dtype, int B, int T,
                          int H, int HV, int K, int V, float scale, unsigned flags,
                          void *stream)
{
    if (!valid_dtype(io_dtype) || !valid_dtype(g_dtype)) return GDN2_ERR_INVALID;
    if (B < 0 || T < 0 || H <= 0 || HV <= 0 || K <= 0 || V <= 0) return GDN2_ERR_INVALID;
    if (HV % H != 0) return GDN2_ERR_INVALID;
    if (flags & ~(GDN2_FLAG_L2NORM_QK | GDN2_FLAG_GATE_IN_KERNEL | GDN2_FLAG_LOWER_BOUND |
                  GDN2_FLAG_TRANSPOSE_STATE | GDN2_FLAG_INPLACE_FINAL_STATE | GDN2_FLAG_SIGMOID_BW |
                  GDN2_FLAG_SHORT_SEQS))
        return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_LOWER_BOUND) && !(flags & GDN2_FLAG_GATE_IN_KERNEL))
        return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_GATE_IN_KERNEL) && !A_log) return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_SHORT_SEQS) && !cu_seqlens) return GDN2_ERR_INVALID;
    if (K > 256 || (V % 4) != 0) return GDN2_ERR_UNSUPPORTED;
    if ((flags & GDN2_FLAG_TRANSPOSE_STATE) && (K % 4) != 0) return GDN2_ERR_UNSUPPORTED;
    int N = B;
    if (cu_seqlens) {
        if (B != 1 || num_seqs < 0) return GDN2_ERR_INVALID;
        N = num_seqs;
    }
    const int64_t ntok = static_cast<int64_t>(B) * T;
    if (ntok > 0 && (!q || !k || !v || !g || !b || !w || !o)) return GDN2_ERR_INVALID;
    // State rows: 16-byte aligned, non-overlapping heads.
    const int64_t slab = static_cast<int64_t>(HV) * K * V;
    const bool pooled = ssm_state_indices != nullptr;
    if (initial_state) {
        if (initial_state_row_stride < slab || (initial_state_row_stride % 4) != 0 ||
            initial_state_rows < 0 || (reinterpret_cast<uintptr_t>(initial_state) & 15) != 0)
            return GDN2_ERR_INVALID;
        if (!pooled && initial_state_rows < N) return GDN2_ERR_INVALID;
    }
    if (final_state) {
        if (final_state_row_stride < slab || (final_state_row_stride % 4) != 0 ||
            final_state_rows < 0 || (reinterpret_cast<uintptr_t>(final_state) & 15) != 0)
            return GDN2_ERR_INVALID;
        if (!pooled && final_state_rows < N) return GDN2_ERR_INVALID;
    }
    if (pooled) {
        if (indices_dtype != GDN2_DTYPE_I32 && indices_dtype != GDN2_DTYPE_I64) return GDN2_ERR_INVALID;
        if (indices_numel < 0 || indices_seq_stride < 0) return GDN2_ERR_INVALID;
        if (num_accepted_tokens && accepted_dtype != GDN2_DTYPE_I32 &&
            accepted_dtype != GDN2_DTYPE_I64)
            return GDN2_ERR_INVALID;
    }
    if (N == 0) return GDN2_OK;
    if (static_cast<int64_t>(N) * HV > 2147483647LL) return GDN2_ERR_UNSUPPORTED;

    RecurrentParams p;
    p.q = q; p.k = k; p.v = v; p.g = g; p.b = b; p.w = w; p.o = o;
    p.h0 = initial_state;
    p.ht = final_state;
    p.A_log = A_log;
    p.dt_bias = dt_bias;
    p.lower_bound = lower_bound;
    p.cu_seqlens = cu_seqlens;
    p.T = T; p.H = H; p.HV = HV; p.K = K; p.V = V;
    p.scale = scale;
    p.flags = flags;
    p.h0_rows = initial_state ? initial_state_rows : 0;
    p.h0_stride = initial_state_row_stride;
    p.ht_rows = final_state ? final_state_rows : 0;
    p.ht_stride = final_state_row_stride;
    p.state_indices = ssm_state_indices;
    p.accepted = pooled ? num_accepted_tokens : nullptr;
    p.idx_numel = pooled ? indices_numel : 0;
    p.idx_seq_stride = pooled ? indices_seq_stride : 0;
    p.idx_i64 = indices_dtype == GDN2_DTYPE_I64;
    p.acc_i64 = accepted_dtype == GDN2_DTYPE_I64;
    const hipError_t err =
        launch_recurrent_fwd(p, io_dtype, g_dtype, N, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_recurrent_fwd(const void *q, const void *k, const void *v, const void *g,
                       const void *b, const void *w, int io_dtype, int g_dtype, void *o,
                       const float *initial_state, float *final_state, const float *A_log,
                       const float *dt_bias, float lower_bound, const int64_t *cu_seqlens,
                       int num_seqs, int B, int T, int H, int HV, int K, int V, float scale,
                       unsigned flags, void *stream)
{
    if (flags & (GDN2_FLAG_TRANSPOSE_STATE | GDN2_FLAG_INPLACE_FINAL_STATE)) return GDN2_ERR_INVALID;
    const int64_t rows = cu_seqlens ? num_seqs : B;
    const int64_t slab = static_cast<int64_t>(HV) * K * V;
    return gdn2_recurrent_fwd_ex(q, k, v, g, b, w, io_dtype, g_dtype, o, initial_state, rows,
                                 slab, final_state, rows, slab, A_log, dt_bias, lower_bound,
                                 cu_seqlens, num_seqs, nullptr, GDN2_DTYPE_I64, 0, 0, nullptr,
                                 GDN2_DTYPE_I64, B, T, H, HV, K, V, scale, flags, stream);
}

int gdn2_short_conv_fwd(int ntensors, const void *const *x, const void *const *weight,
                        const void *const *bias, const void *const *cache_in,
                        void *const *cache_out, void *const *y, const int *dims, int io_dtype,
                        int B, int T, int W, int silu, void *stream)
{
    return gdn2_short_conv_fwd_ex(ntensors, x, nullptr, weight, bias, cache_in, cache_out, y, dims,
                                  io_dtype, B, T, W, silu, stream);
}

int gdn2_short_conv_fwd_ex(int ntensors, const void *const *x, const int64_t *x_row_stride,
                           const void *const *weight, const void *const *bias,
                           const void *const *cache_in, void *const *cache_out, void *const *y,
                           const int *dims, int io_dtype, int B, int T, int W, int silu, void *stream)
{
    if (!valid_dtype(io_dtype)) return GDN2_ERR_INVALID;
    if (ntensors < 1 || ntensors > 3 || !x || !weight || !y || !dims) return GDN2_ERR_INVALID;
    if (B < 0 || T < 0 || W < 1) return GDN2_ERR_INVALID;
    if (W > 8) return GDN2_ERR_UNSUPPORTED;
    ConvParams p;
    p.B = B; p.T = T; p.W = W;
    p.ncache = T == 1 ? W - 1 : (T < W - 1 ? T : W - 1);
    p.silu = silu != 0;
    int maxD = 0;
    for (int i = 0; i < 3; ++i) {
        const int j = i < ntensors ? i : 0;
        ConvTensor &c = p.t[i];
        c.D = dims[j];
        if (c.D <= 0) return GDN2_ERR_INVALID;
        c.ldx = x_row_stride ? x_row_stride[j] : c.D;
        if (c.ldx < c.D) return GDN2_ERR_INVALID;
        if (B * static_cast<int64_t>(T) > 0 && (!x[j] || !weight[j] || !y[j])) return GDN2_ERR_INVALID;
        c.x = x[j]; c.w = weight[j]; c.y = y[j];
        c.bias = bias ? bias[j] : nullptr;
        c.cache_in = cache_in ? cache_in[j] : nullptr;
        c.cache_out = cache_out ? cache_out[j] : nullptr;
        if (i < ntensors && c.D > maxD) maxD = c.D;
    }
    if (B == 0 || T == 0) return GDN2_OK;
    const hipError_t err = launch_short_conv(p, io_dtype, maxD, ntensors, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_gated_rmsnorm_fwd(const void *x, const void *z, const void *weight, int weight_dtype,
                           void *out, int io_dtype, int64_t rows, int N, float eps, void *stream)
{
    if (!valid_dtype(io_dtype) || !valid_dtype(weight_dtype)) return GDN2_ERR_INVALID;
    if (weight_dtype != io_dtype && weight_dtype != GDN2_DTYPE_F32) return GDN2_ERR_INVALID;
    if (rows < 0 || N <= 0) return GDN2_ERR_INVALID;
    if (N > 2048) return GDN2_ERR_UNSUPPORTED;
    if (rows == 0) return GDN2_OK;
    if (!x || !weight || !out) return GDN2_ERR_INVALID;  // z may be NULL: no gate
    if ((rows + 3) / 4 > 2147483647LL) return GDN2_ERR_UNSUPPORTED;
    NormParams p;
    p.x = x; p.z = z; p.weight = weight; p.out = out;
    p.rows = rows; p.N = N; p.eps = eps;
    p.w_f32 = weight_dtype == GDN2_DTYPE_F32 && io_dtype != GDN2_DTYPE_F32;
    const hipError_t err = launch_gated_rmsnorm(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_add_rms_norm_fwd(const void *x, const void *residual, void *sum_out, const void *weight,
                          int weight_dtype, void *out, int io_dtype, int64_t rows, int N, float eps,
                          void *stream)
{
    if (!valid_dtype(io_dtype) || !valid_dtype(weight_dtype)) return GDN2_ERR_INVALID;
    if (weight_dtype != io_dtype && weight_dtype != GDN2_DTYPE_F32) return GDN2_ERR_INVALID;
    if (rows < 0 || N <= 0) return GDN2_ERR_INVALID;
    if (rows == 0) return GDN2_OK;
    if (!x || !residual || !sum_out || !weight || !out) return GDN2_ERR_INVALID;
    // One vectorised pass: rows of 4..256 16-byte pieces (a power of two), 16-byte aligned.
    const int epv = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    const int pieces = N / epv;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                           reinterpret_cast<uintptr_t>(sum_out) | reinterpret_cast<uintptr_t>(out);
    if (N % epv != 0 || pieces < 4 || pieces > 256 || (pieces & (pieces - 1)) != 0 || (addr & 15) != 0)
        return GDN2_ERR_UNSUPPORTED;
    if (rows > 2147483647LL) return GDN2_ERR_UNSUPPORTED;
    NormParams p;
    p.x = x; p.z = nullptr; p.weight = weight; p.out = out;
    p.rows = rows; p.N = N; p.eps = eps;
    p.w_f32 = weight_dtype == GDN2_DTYPE_F32 && io_dtype != GDN2_DTYPE_F32;
    p.res = residual; p.sum_out = sum_out;
    const hipError_t err = launch_gated_rmsnorm(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_silu_mul_fwd(const void *ab, int64_t ab_row_stride, void *out, int io_dtype, int64_t rows,
                      int H, void *stream)
{
    if (!valid_dtype(io_dtype) || rows < 0 || H <= 0) return GDN2_ERR_INVALID;
    if (rows == 0) return GDN2_OK;
    if (!ab || !out || ab_row_stride < 2LL * H) return GDN2_ERR_INVALID;
    const int epv = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    if (H % epv != 0 || ab_row_stride % epv != 0 ||
        ((reinterpret_cast<uintptr_t>(ab) | reinterpret_cast<uintptr_t>(out)) & 15) != 0)
        return GDN2_ERR_UNSUPPORTED;
    if ((rows * (H / epv) + 255) / 256 > 2147483647LL) return GDN2_ERR_UNSUPPORTED;
    SiluMulParams p;
    p.ab = ab; p.out = out; p.rows = rows; p.ld = ab_row_stride; p.H = H;
    const hipError_t err = launch_silu_mul(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_skinny_linear(const void *x, int64_t x_row_stride, const void *weight, int64_t weight_row_stride,
                       const void *bias, void *y, int64_t y_row_stride, int io_dtype, int M, int N, int K,
                       void *stream)
{
    if (!valid_dtype(io_dtype) || M < 0 || N < 0 || K < 0) return GDN2_ERR_INVALID;
    if (M == 0 || N == 0) return GDN2_OK;
    if (!x || !weight || !y || x_row_stride < K || weight_row_stride < K || y_row_stride < N) return GDN2_ERR_INVALID;
    if (!skinny_linear_supported(io_dtype, M, K)) return GDN2_ERR_UNSUPPORTED;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight)) & 15) != 0 ||
        x_row_stride % 8 != 0 || weight_row_stride % 8 != 0)
        return GDN2_ERR_UNSUPPORTED;
    if (N > 2147483647 - 8) return GDN2_ERR_UNSUPPORTED;
    SkinnyParams p;
    p.x = x; p.w = weight; p.bias = bias; p.y = y;
    p.ldx = x_row_stride; p.ldw = weight_row_stride; p.ldy = y_row_stride;
    p.M = M; p.N = N; p.K = K;
    const hipError_t err = launch_skinny_linear(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

static int skinny_addnorm_impl(const void *x, int64_t x_row_stride, const void *residual,
                               int64_t residual_row_stride, void *sum_out, int64_t sum_row_stride,
                               const void *norm_weight, float eps, const void *weight, int64_t weight_row_stride,
                               const void *bias, void *y, int64_t y_row_stride, int io_dtype, int M, int N, int K,
                               int glu, void *stream)
{
    if (!valid_dtype(io_dtype) || M < 0 || N < 0 || K < 0) return GDN2_ERR_INVALID;
    if (M == 0 || N == 0) return GDN2_OK;
    if (glu && N % 2 != 0) return GDN2_ERR_INVALID;
    if (!x || !residual || !sum_out || !norm_weight || !weight || !y || x_row_stride < K ||
        residual_row_stride < K || sum_row_stride < K || weight_row_stride < K || y_row_stride < (glu ? N / 2 : N))
        return GDN2_ERR_INVALID;
    if (!skinny_linear_supported(io_dtype, M, K) || M > 4 || K > 2048) return GDN2_ERR_UNSUPPORTED;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
          reinterpret_cast<uintptr_t>(sum_out) | reinterpret_cast<uintptr_t>(weight) |
          reinterpret_cast<uintptr_t>(norm_weight)) & 15) != 0 ||
        x_row_stride % 8 != 0 || residual_row_stride % 8 != 0 || sum_row_stride % 8 != 0 || weight_row_stride % 8 != 0)
        return GDN2_ERR_UNSUPPORTED;
    if (N > 2147483647 - 8) return GDN2_ERR_UNSUPPORTED;
    SkinnyParams p;
    p.x = x; p.w = weight; p.bias = bias; p.y = y;
    p.ldx = x_row_stride; p.ldw = weight_row_stride; p.ldy = y_row_stride;
    p.M = M; p.N = N; p.K = K;
    p.norm = 1; p.res = residual; p.nw = norm_weight; p.sum_out = sum_out;
    p.ldres = residual_row_stride; p.ldsum = sum_row_stride; p.eps = eps;
    p.glu_out = glu;
    const hipError_t err = launch_skinny_linear(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_skinny_linear_addnorm(const void *x, int64_t x_row_stride, const void *residual,
                               int64_t residual_row_stride, void *sum_out, int64_t sum_row_stride,
                               const void *norm_weight, float eps, const void *weight, int64_t weight_row_stride,
                               const void *bias, void *y, int64_t y_row_stride, int io_dtype, int M, int N, int K,
                               void *stream)
{
    return skinny_addnorm_impl(x, x_row_stride, residual, residual_row_stride, sum_out, sum_row_stride, norm_weight,
                               eps, weight, weight_row_stride, bias, y, y_row_stride, io_dtype, M, N, K, 0, stream);
}

int gdn2_skinny_linear_addnorm_swiglu(const void *x, int64_t x_row_stride, const void *residual,
                                      int64_t residual_row_stride, void *sum_out, int64_t sum_row_stride,
                                      const void *norm_weight, float eps, const void *weight,
                                      int64_t weight_row_stride, const void *bias, void *y, int64_t y_row_stride,
                                      int io_dtype, int M, int N, int K, void *stream)
{
    return skinny_addnorm_impl(x, x_row_stride, residual, residual_row_stride, sum_out, sum_row_stride, norm_weight,
                               eps, weight, weight_row_stride, bias, y, y_row_stride, io_dtype, M, N, K, 1, stream);
}

int gdn2_small_linear_pair(const void *x0, int64_t x0_row_stride, const void *weight0, const void *bias0, void *y0,
                           int64_t y0_row_stride, int N0, const void *x1, int64_t x1_row_stride,
                           const void *weight1, const void *bias1, void *y1, int64_t y1_row_stride, int N1,
                           int io_dtype, int M, int K, void *stream)
{
    if (!valid_dtype(io_dtype) || M < 0 || K < 1 || N0 < 0 || N1 < 0) return GDN2_ERR_INVALID;
    if (M == 0 || (N0 == 0 && N1 == 0)) return GDN2_OK;
    if (!small_linear_supported(io_dtype, M, K)) return GDN2_ERR_UNSUPPORTED;
    SmallLinearParams p;
    p.M = M; p.K = K;
    int n = 0;
    const void *xs[2] = {x0, x1}, *ws[2] = {weight0, weight1}, *bs[2] = {bias0, bias1};
    void *ys[2] = {y0, y1};
    const int64_t lx[2] = {x0_row_stride, x1_row_stride}, ly[2] = {y0_row_stride, y1_row_stride};
    const int Ns[2] = {N0, N1};
    for (int i = 0; i < 2; ++i) {
        if (Ns[i] == 0) continue;
        if (!xs[i] || !ws[i] || !ys[i] || lx[i] < K || ly[i] < Ns[i]) return GDN2_ERR_INVALID;
        if (((reinterpret_cast<uintptr_t>(xs[i]) | reinterpret_cast<uintptr_t>(ws[i])) & 15) != 0 || lx[i] % 8 != 0)
            return GDN2_ERR_UNSUPPORTED;
        SmallLinearProblem &q = p.prob[n++];
        q.x = xs[i]; q.w = ws[i]; q.bias = bs[i]; q.y = ys[i]; q.ldx = lx[i]; q.ldy = ly[i]; q.N = Ns[i];
    }
    const hipError_t err = launch_small_linear(p, n, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_argmax_rows_workspace_size(int64_t rows, int64_t n, int io_dtype)
{
    if (!valid_dtype(io_dtype) || rows < 1 || n < 1 || rows > 65535) return 0;
    const int s = argmax_splits(n, io_dtype);
    return s > 1 ? static_cast<size_t>(rows) * s * (sizeof(int64_t) + sizeof(float)) : 0;
}

int gdn2_argmax_rows(const void *x, int64_t x_row_stride, int io_dtype, int64_t rows, int64_t n, int64_t *out,
                     int64_t out_stride, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!valid_dtype(io_dtype) || rows < 0 || n < 1) return GDN2_ERR_INVALID;
    if (rows == 0) return GDN2_OK;
    if (!x || !out || x_row_stride < n || out_stride < 1) return GDN2_ERR_INVALID;
    const int es = io_dtype == GDN2_DTYPE_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(x) & 15) != 0 || (x_row_stride * es) % 16 != 0) return GDN2_ERR_UNSUPPORTED;
    if (rows > 2147483647LL) return GDN2_ERR_UNSUPPORTED;
    ArgmaxParams p;
    p.x = x; p.ld = x_row_stride; p.rows = rows; p.n = n; p.out = out; p.out_stride = out_stride;
    p.splits = 1; p.pps = 0; p.part_v = nullptr; p.part_i = nullptr;
    const size_t need = gdn2_argmax_rows_workspace_size(rows, n, io_dtype);
    if (workspace && need > 0) {
        if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0) return GDN2_ERR_WORKSPACE;
        p.splits = argmax_splits(n, io_dtype);
        const int64_t pieces = n / (io_dtype == GDN2_DTYPE_F32 ? 4 : 8);
        p.pps = (pieces + p.splits - 1) / p.splits;
        p.part_i = static_cast<int64_t *>(workspace);
        p.part_v = reinterpret_cast<float *>(p.part_i + rows * p.splits);
    }
    const hipError_t err = launch_argmax_rows(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_attn_decode_workspace_size(int B, int G, int qpk, int D, int64_t max_len)
{
    if (B < 0 || G < 0 || qpk < 1 || D < 1 || max_len < 1) return 0;
    return attn_decode_workspace_floats(B, G, qpk, D, max_len) * sizeof(float);
}

int gdn2_attn_decode(const void *qkv, const float *cos, const float *sin, int rope_pairs, int64_t rope_row_stride,
                     const int64_t *pos, void *k_cache, void *v_cache, void *out, int io_dtype, int B, int G,
                     int qpk, int D, int64_t max_len, float scale, void *workspace, size_t workspace_bytes,
                     void *stream)
{
    if (!valid_dtype(io_dtype) || B < 0 || G < 0 || qpk < 1 || D < 1 || max_len < 1) return GDN2_ERR_INVALID;
    if (B == 0 || G == 0) return GDN2_OK;
    if (!qkv || !pos || !k_cache || !v_cache || !out) return GDN2_ERR_INVALID;
    if (rope_pairs < 0 || 2 * rope_pairs > D) return GDN2_ERR_INVALID;
    if (rope_pairs > 0 && (!cos || !sin)) return GDN2_ERR_INVALID;
    if (rope_row_stride < 0 || (rope_row_stride > 0 && rope_row_stride < rope_pairs)) return GDN2_ERR_INVALID;
    if (!attn_decode_supported(io_dtype, qpk, D)) return GDN2_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(B) * G > 2147483647LL || max_len > 2147483647LL) return GDN2_ERR_UNSUPPORTED;
    AttnDecodeParams p;
    p.qkv = qkv; p.cos = cos; p.sin = sin;
    p.rope_pairs = rope_pairs;
    p.rope_stride = rope_row_stride;
    p.pos = pos; p.k_cache = k_cache; p.v_cache = v_cache; p.out = out;
    p.max_len = max_len; p.B = B; p.G = G; p.qpk = qpk; p.D = D; p.scale = scale;
    p.splits = attn_decode_splits(max_len);
    p.part = static_cast<float *>(workspace);
    if (p.splits > 1 && (!workspace || workspace_bytes < gdn2_attn_decode_workspace_size(B, G, qpk, D, max_len)))
        return GDN2_ERR_WORKSPACE;
    const hipError_t err = launch_attn_decode(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

static int check_q4_cache(const void *kc, const void *km, const void *vc, const void *vm, int B, int G, int D,
                          int64_t max_len)
{
    if (B < 0 || G < 1 || D < 1 || max_len < 1) return GDN2_ERR_INVALID;
    if (D % 64 != 0 || D > 1024) return GDN2_ERR_UNSUPPORTED;
    if (max_len > (1 << 30) || static_cast<int64_t>(B) * G > max_workgroups(256)) return GDN2_ERR_UNSUPPORTED;
    if (B > 0 && (!kc || !km || !vc || !vm)) return GDN2_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(kc) | reinterpret_cast<uintptr_t>(vc)) & 15) return GDN2_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(km) | reinterpret_cast<uintptr_t>(vm)) & 3) return GDN2_ERR_INVALID;
    return GDN2_OK;
}

// One launch (workgroups of 128 tokens of one head's group each).
static bool q4_launchable(int B, int64_t T, int G, int D)
{
    return T <= (1 << 30) &&
           2.0 * ((T + 127) / 128) * (D / 64) * G * B <= static_cast<double>(max_workgroups(256));
}

size_t gdn2_attn_decode_q4_workspace_size(int B, int G, int qpk, int D, int64_t max_len)
{
    if (B < 1 || G < 1 || qpk < 1 || D < 1 || max_len < 1) return 0;
    return attn_q4_workspace_floats(B, G, qpk, D, max_len) * sizeof(float);
}

int gdn2_attn_decode_q4(const void *qkv, const float *cos, const float *sin, int rope_pairs, int64_t rope_row_stride,
                        const int64_t *pos, int64_t pos_stride, void *k_codes, void *k_meta, void *v_codes,
                        void *v_meta, void *out, int io_dtype, int B, int G, int qpk, int D, int64_t max_len,
                        float scale, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!valid_dtype(io_dtype) || qpk < 1 || pos_stride < 0) return GDN2_ERR_INVALID;
    const int st = check_q4_cache(k_codes, k_meta, v_codes, v_meta, B, G, D, max_len);
    if (st != GDN2_OK) return st;
    if (rope_pairs < 0 || 2 * rope_pairs > D || (rope_pairs > 0 && (!cos || !sin))) return GDN2_ERR_INVALID;
    if (rope_row_stride < 0 || (rope_row_stride > 0 && rope_row_stride < rope_pairs)) return GDN2_ERR_INVALID;
    if (!attn_q4_supported(io_dtype, qpk, D) || !(scale > 0.0f) || scale > 1e30f) return GDN2_ERR_UNSUPPORTED;
    if (B == 0) return GDN2_OK;
    if (!qkv || !pos || !out) return GDN2_ERR_INVALID;
    const int splits = attn_q4_splits(B, G, max_len);
    if (splits > 1 && static_cast<int64_t>(B) * G * qpk > max_workgroups(256)) return GDN2_ERR_UNSUPPORTED;  // the merge
    AttnQ4Params p = {};
    p.qkv = qkv; p.cos = cos; p.sin = sin;
    p.rope_pairs = rope_pairs;
    p.rope_stride = rope_row_stride;
    p.pos = pos; p.pos_stride = pos_stride;
    p.k_codes = static_cast<uint8_t *>(k_codes); p.v_codes = static_cast<uint8_t *>(v_codes);
    p.k_meta = static_cast<unsigned *>(k_meta); p.v_meta = static_cast<unsigned *>(v_meta);
    p.out = out;
    p.max_len = max_len; p.B = B; p.G = G; p.qpk = qpk; p.D = D; p.scale = scale;
    p.splits = splits;
    p.part = static_cast<float *>(workspace);
    if (p.splits > 1 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
                         workspace_bytes < gdn2_attn_decode_q4_workspace_size(B, G, qpk, D, max_len)))
        return GDN2_ERR_WORKSPACE;
    return launch_attn_q4(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_kv_cache_q4_store(const void *k, const void *v, const int64_t *strides, int io_dtype, const int64_t *start,
                           int64_t start_stride, void *k_codes, void *k_meta, void *v_codes, void *v_meta, int B,
                           int64_t T, int G, int D, int64_t max_len, void *stream)
{
    if (!valid_dtype(io_dtype) || T < 0 || start_stride < 0 || !strides) return GDN2_ERR_INVALID;
    const int st = check_q4_cache(k_codes, k_meta, v_codes, v_meta, B, G, D, max_len);
    if (st != GDN2_OK) return st;
    if (B == 0 || T == 0) return GDN2_OK;
    if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return GDN2_ERR_INVALID;
    if (!q4_launchable(B, T, G, D)) return GDN2_ERR_UNSUPPORTED;
    Q4StoreParams p = {};
    const int64_t size[6] = {B, T, G, B, T, G};
    const int per = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    for (int i = 0; i < 6; ++i) {
        if (strides[i] < 0 || (size[i] > 1 && strides[i] % per != 0)) return GDN2_ERR_INVALID;
        (i < 3 ? p.ks : p.vs)[i % 3] = strides[i];
    }
    p.k = k; p.v = v;
    p.start = start; p.start_stride = start_stride;
    p.k_codes = static_cast<uint8_t *>(k_codes); p.v_codes = static_cast<uint8_t *>(v_codes);
    p.k_meta = static_cast<unsigned *>(k_meta); p.v_meta = static_cast<unsigned *>(v_meta);
    p.max_len = max_len; p.T = T; p.B = B; p.G = G; p.D = D;
    return launch_q4_store(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_kv_cache_q4_load(const void *k_codes, const void *k_meta, const void *v_codes, const void *v_meta,
                          const int64_t *start, int64_t start_stride, void *k, void *v, int io_dtype, int B, int64_t T,
                          int G, int D, int64_t max_len, void *stream)
{
    if (!valid_dtype(io_dtype) || T < 0 || start_stride < 0) return GDN2_ERR_INVALID;
    const int st = check_q4_cache(k_codes, k_meta, v_codes, v_meta, B, G, D, max_len);
    if (st != GDN2_OK) return st;
    if (B == 0 || T == 0) return GDN2_OK;
    if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) return GDN2_ERR_INVALID;
    if (!q4_launchable(B, T, G, D)) return GDN2_ERR_UNSUPPORTED;
    Q4LoadParams p = {};
    p.k = k; p.v = v;
    p.start = start; p.start_stride = start_stride;
    p.k_codes = static_cast<const uint8_t *>(k_codes); p.v_codes = static_cast<const uint8_t *>(v_codes);
    p.k_meta = static_cast<const unsigned *>(k_meta); p.v_meta = static_cast<const unsigned *>(v_meta);
    p.max_len = max_len; p.T = T; p.B = B; p.G = G; p.D = D;
    return launch_q4_load(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

// What the passes over a fused projection share: its rows, the norm's weights and the angles.
static int check_qkv_rope(QkvRopeParams &p, const void *qkv, int64_t stride_b, int64_t stride_t, int io_dtype,
                          const void *wq, const void *wk, int w_dtype, float eps, const float *cos, const float *sin,
                          int pairs, int64_t table_rows, int B, int64_t T, int G, int R, int D)
{
    if (!valid_dtype(io_dtype) || B < 0 || T < 0 || G < 1 || R < 1 || D < 1) return GDN2_ERR_INVALID;
    if (D % 8 != 0 || D > 256) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(G) * (R + 2) > 65535) return GDN2_ERR_UNSUPPORTED;
    if ((wq != nullptr) != (wk != nullptr)) return GDN2_ERR_INVALID;
    if (wq && w_dtype != io_dtype && w_dtype != GDN2_DTYPE_F32) return GDN2_ERR_INVALID;
    if (pairs < 0 || 2 * pairs > D || table_rows < 0 || table_rows > 2147483647LL) return GDN2_ERR_INVALID;
    if (B == 0 || T == 0) return GDN2_OK;
    const int per = io_dtype == GDN2_DTYPE_F32 ? 4 : 8;
    if (!qkv || (pairs > 0 && table_rows > 0 && (!cos || !sin))) return GDN2_ERR_INVALID;
    if (stride_b < 0 || stride_t < 0 || (B > 1 && stride_b % per != 0) || (T > 1 && stride_t % per != 0))
        return GDN2_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(wq) | reinterpret_cast<uintptr_t>(wk)) & 15)
        return GDN2_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 3) return GDN2_ERR_INVALID;
    if (T > 2147483647LL || static_cast<double>(B) * T * qkv_rope_units(G * (R + 2), D, true) / 4 + 1 >
                                static_cast<double>(max_workgroups(256)))
        return GDN2_ERR_UNSUPPORTED;
    p.qkv = qkv; p.stride_b = stride_b; p.stride_t = stride_t;
    p.wq = wq; p.wk = wk; p.w_f32 = w_dtype == GDN2_DTYPE_F32; p.eps = eps;
    // Tables of no rows hold no angles: no token has a position, and none is read (the backward reads a row for
    // tokens without one, too).
    p.cos = cos; p.sin = sin; p.pairs = table_rows > 0 ? pairs : 0; p.table_rows = table_rows;
    p.B = B; p.T = static_cast<int>(T); p.G = G; p.R = R; p.D = D;
    return GDN2_OK;
}

static bool aligned16(const void *a, const void *b, const void *c)
{
    return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & 15) == 0;
}

int gdn2_qkv_norm_rope_fwd(const void *qkv, int64_t stride_b, int64_t stride_t, int io_dtype, const void *wq,
                           const void *wk, int w_dtype, float eps, const float *cos, const float *sin, int pairs,
                           int64_t table_rows, const int64_t *pos, int64_t pos_stride_b, int64_t pos_stride_t, void *q,
                           void *k, int B, int64_t T, int G, int R, int D, void *stream)
{
    QkvRopeParams p = {};
    const int st = check_qkv_rope(p, qkv, stride_b, stride_t, io_dtype, wq, wk, w_dtype, eps, cos, sin, pairs, table_rows,
                                  B, T, G, R, D);
    if (st != GDN2_OK) return st;
    if (B == 0 || T == 0) return GDN2_OK;
    if (!q || !k || !aligned16(q, k, nullptr) || pos_stride_b < 0 || pos_stride_t < 0) return GDN2_ERR_INVALID;
    p.pos = pos; p.pos_b = pos_stride_b; p.pos_t = pos_stride_t;
    p.q = q; p.k = k;
    return launch_qkv_rope_fwd(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_qkv_norm_rope_bwd_workspace_size(int B, int64_t T, int G, int R, int D)
{
    if (B < 1 || T < 1 || G < 1 || R < 1 || D < 1 || D > 256) return 0;
    return static_cast<size_t>(qkv_rope_bwd_blocks(static_cast<int64_t>(B) * T * qkv_rope_units(G * (R + 2), D, true))) * 2 * D *
           sizeof(float);
}

int gdn2_qkv_norm_rope_bwd(const void *qkv, int64_t stride_b, int64_t stride_t, int io_dtype, const void *wq,
                           const void *wk, int w_dtype, float eps, const float *cos, const float *sin, int pairs,
                           int64_t table_rows, const int64_t *pos, int64_t pos_stride_b, int64_t pos_stride_t,
                           const void *dq, const void *dk, const void *dv, void *dqkv, void *dwq, void *dwk, int B,
                           int64_t T, int G, int R, int D, void *workspace, size_t workspace_bytes, void *stream)
{
    QkvRopeParams p = {};
    const int st = check_qkv_rope(p, qkv, stride_b, stride_t, io_dtype, wq, wk, w_dtype, eps, cos, sin, pairs, table_rows,
                                  B, T, G, R, D);
    if (st != GDN2_OK) return st;
    if (B == 0 || T == 0) return GDN2_OK;
    if (!dq || !dk || !dv || !dqkv || !aligned16(dq, dk, dv) || !aligned16(dqkv, nullptr, nullptr) || pos_stride_b < 0 ||
        pos_stride_t < 0)
        return GDN2_ERR_INVALID;
    if (wq && (!dwq || !dwk)) return GDN2_ERR_INVALID;
    if (wq && (!workspace || workspace_bytes < gdn2_qkv_norm_rope_bwd_workspace_size(B, T, G, R, D) ||
               (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return GDN2_ERR_WORKSPACE;
    p.pos = pos; p.pos_b = pos_stride_b; p.pos_t = pos_stride_t;
    p.q = const_cast<void *>(dq); p.k = const_cast<void *>(dk); p.v = const_cast<void *>(dv);
    p.dqkv = dqkv; p.dwq = dwq; p.dwk = dwk;
    p.part = static_cast<float *>(workspace);
    return launch_qkv_rope_bwd(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

// A paged cache: pages [pages][G][page_size][D] of keys and of values, and the table.
static int check_paged(const void *k_pages, const void *v_pages, int64_t pages, int page_size, const int *table,
                       int64_t table_stride, int table_cols, int B, int G, int D)
{
    if (pages < 1 || page_size < 1 || table_cols < 1 || table_stride < 0 || B < 0 || G < 1 || D < 1)
        return GDN2_ERR_INVALID;
    if (page_size % 16 != 0) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(page_size) * table_cols > (1 << 30)) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<double>(pages) * G * page_size > 4.0e9) return GDN2_ERR_UNSUPPORTED;  // rows are counted in 32 bits
    if (B > 0 && (!k_pages || !v_pages || !table)) return GDN2_ERR_INVALID;
    if (!aligned16(k_pages, v_pages, nullptr) || (reinterpret_cast<uintptr_t>(table) & 3)) return GDN2_ERR_INVALID;
    return GDN2_OK;
}

int gdn2_kv_cache_paged_append(const void *qkv, int64_t stride_b, int64_t stride_t, int io_dtype, const void *wq,
                               const void *wk, int w_dtype, float eps, const float *cos, const float *sin, int pairs,
                               int64_t table_rows, const int64_t *pos, int64_t pos_stride, const int64_t *lengths, void *q,
                               void *k_pages, void *v_pages, int64_t pages, int page_size, const int *table,
                               int64_t table_stride, int table_cols, int B, int64_t T, int G, int R, int D, void *stream)
{
    QkvRopeParams p = {};
    int st = check_qkv_rope(p, qkv, stride_b, stride_t, io_dtype, wq, wk, w_dtype, eps, cos, sin, pairs, table_rows, B, T,
                            G, R, D);
    if (st != GDN2_OK) return st;
    st = check_paged(k_pages, v_pages, pages, page_size, table, table_stride, table_cols, B, G, D);
    if (st != GDN2_OK) return st;
    if (B == 0 || T == 0) return GDN2_OK;
    if (!q || !pos || pos_stride < 0 || !aligned16(q, nullptr, nullptr)) return GDN2_ERR_INVALID;
    p.pos = pos; p.pos_b = pos_stride; p.pos_t = 0; p.pos_add_t = 1;
    p.lengths = lengths;
    p.q = q; p.k = k_pages; p.v = v_pages;
    p.table = table; p.table_stride = table_stride; p.table_cols = table_cols;
    p.pages = pages; p.page = page_size;
    return launch_qkv_rope_fwd(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_attn_paged_workspace_size(int B, int64_t T, int G, int R, int D, int64_t positions)
{
    if (B < 1 || T < 1 || G < 1 || R < 1 || D < 1 || positions < 1) return 0;
    return attn_paged_plan(B, T, G, R, D, positions).floats * sizeof(float);
}

int gdn2_attn_paged(const void *q, const int64_t *strides, int io_dtype, const void *k_pages, const void *v_pages,
                    int64_t pages, int page_size, const int *table, int64_t table_stride, int table_cols,
                    const int64_t *pos, int64_t pos_stride, const int64_t *lengths, void *out, int B, int64_t T, int G,
                    int R, int D, float scale, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!valid_dtype(io_dtype) || T < 0 || R < 1 || pos_stride < 0 || !strides) return GDN2_ERR_INVALID;
    const int st = check_paged(k_pages, v_pages, pages, page_size, table, table_stride, table_cols, B, G, D);
    if (st != GDN2_OK) return st;
    if (!attn_paged_supported(io_dtype, D) || !(scale > 0.0f) || scale > 1e30f) return GDN2_ERR_UNSUPPORTED;
    if (B == 0 || T == 0) return GDN2_OK;
    // Rows of a group in 31 bits, and every launch within HIP's limits: a workgroup for each tile and share and then 1024 /
    // D rows of the join, or (few rows) for each group, and with runs of the keys a row of the join.
    if (static_cast<double>(T) * R > 1073741824.0 || G > 65535) return GDN2_ERR_UNSUPPORTED;
    const AttnPagedPlan plan = attn_paged_plan(B, T, G, R, D, static_cast<int64_t>(page_size) * table_cols);
    const double all_rows = static_cast<double>(B) * G * R * T, groups = static_cast<double>(B) * G;
    const double join = plan.splits > 1 ? all_rows * D / 1024 + 1 : plan.workers > 0 ? all_rows : 0;
    if (groups * plan.tiles * plan.splits > max_workgroups(256) || join > max_workgroups(256)) return GDN2_ERR_UNSUPPORTED;
    if (!q || !pos || !out || !aligned16(q, out, nullptr)) return GDN2_ERR_INVALID;
    const int64_t size[3] = {B, T, static_cast<int64_t>(G) * R};
    AttnPagedParams p = {};
    for (int i = 0; i < 3; ++i) {
        if (strides[i] < 0 || (size[i] > 1 && strides[i] % 8 != 0)) return GDN2_ERR_INVALID;
        p.qs[i] = strides[i];
    }
    p.q = q; p.k = k_pages; p.v = v_pages;
    p.table = table; p.table_stride = table_stride; p.pages = pages; p.page = page_size;
    p.cap = page_size * table_cols;
    p.pos = pos; p.pos_stride = pos_stride; p.lengths = lengths;
    p.out = out; p.B = B; p.T = static_cast<int>(T); p.G = G; p.R = R; p.D = D; p.scale = scale;
    p.rows = plan.rows; p.tiles = plan.tiles; p.splits = plan.splits; p.workers = plan.workers;
    p.part = static_cast<float *>(workspace);
    if (plan.floats > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
                            workspace_bytes < plan.floats * sizeof(float)))
        return GDN2_ERR_WORKSPACE;
    return launch_attn_paged(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_sample_tokens_workspace_size(int64_t rows, int64_t n)
{
    return rows < 1 || n < 1 ? 0 : sample_workspace(rows, n);
}

int gdn2_sample_tokens(const void *x, int64_t inner, int64_t outer_stride, int64_t row_stride, int io_dtype, int64_t rows,
                       int64_t n, const float *u, const float *temperature, float temperature_all, const int *top_k,
                       int top_k_all, const float *top_p, float top_p_all, const float *min_p, float min_p_all,
                       int64_t *out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!valid_dtype(io_dtype) || rows < 0 || n < 1 || inner < 1 || outer_stride < 0 || row_stride < 0)
        return GDN2_ERR_INVALID;
    if (n > kSampleMax) return GDN2_ERR_UNSUPPORTED;
    if (!temperature && !(temperature_all >= 0.0f && temperature_all <= 3.0e38f)) return GDN2_ERR_INVALID;
    if (!top_p && !(top_p_all > 0.0f && top_p_all <= 1.0f)) return GDN2_ERR_INVALID;
    if (!min_p && !(min_p_all >= 0.0f && min_p_all <= 1.0f)) return GDN2_ERR_INVALID;
    if (!top_k && top_k_all < 0) return GDN2_ERR_INVALID;
    if (rows == 0) return GDN2_OK;
    const uintptr_t size = io_dtype == GDN2_DTYPE_F32 ? 4 : 2;
    if (!x || !u || !out || (reinterpret_cast<uintptr_t>(x) & (size - 1))) return GDN2_ERR_INVALID;
    // A workgroup for each part of a row, and one for the row.
    if (rows > max_workgroups(kSampleFinishThreads) || rows * sample_parts(rows, n) > max_workgroups(256))
        return GDN2_ERR_UNSUPPORTED;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < gdn2_sample_tokens_workspace_size(rows, n))
        return GDN2_ERR_WORKSPACE;
    SampleParams p = {};
    p.x = x; p.inner = inner; p.outer_stride = outer_stride; p.row_stride = row_stride; p.rows = rows;
    p.n = static_cast<int>(n);
    p.u = u; p.out = out;
    p.temperature = temperature; p.temperature_all = temperature_all;
    p.top_k = top_k; p.top_k_all = top_k_all;
    p.top_p = top_p; p.top_p_all = top_p_all;
    p.min_p = min_p; p.min_p_all = min_p_all;
    return launch_sample(p, workspace, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

static int fill_logprob_args(LogprobParams &p, const void *x, int64_t inner, int64_t outer_stride, int64_t row_stride,
                             int io_dtype, int64_t rows, int64_t n, const int64_t *targets, int64_t ignore)
{
    if (!valid_dtype(io_dtype) || rows < 0 || n < 1 || inner < 1 || outer_stride < 0 || row_stride < 0)
        return GDN2_ERR_INVALID;
    if (rows > 0 && (!x || !targets)) return GDN2_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(x) % (io_dtype == GDN2_DTYPE_F32 ? 4 : 2) != 0) return GDN2_ERR_INVALID;
    // Indices of a row, and of a row's parts, in 32 bits.
    if (rows > (1 << 27) || n > (1 << 30)) return GDN2_ERR_UNSUPPORTED;
    p.x = x;
    p.inner = inner; p.outer_stride = outer_stride; p.row_stride = row_stride;
    p.rows = rows; p.n = n;
    p.targets = targets;
    p.ignore = ignore;
    return GDN2_OK;
}

size_t gdn2_token_logprobs_workspace_size(int64_t rows, int64_t n, int top_k, int io_dtype)
{
    if (!valid_dtype(io_dtype) || rows < 1 || n < 1 || rows > (1 << 27) || n > (1 << 30) || top_k < 0 || top_k > 32)
        return 0;
    const int parts = logprob_parts(rows, n, io_dtype);
    return parts == 1 ? 0 : static_cast<size_t>(rows) * parts * (4 * sizeof(float) + static_cast<size_t>(top_k) * 8);
}

int gdn2_token_logprobs_fwd(const void *x, int64_t inner_rows, int64_t outer_stride, int64_t row_stride, int io_dtype,
                            int64_t rows, int64_t n, const int64_t *targets, int64_t ignore_index, float *logp,
                            float *entropy, float *lse, int top_k, float *top_logp, int64_t *top_ids, void *workspace,
                            size_t workspace_bytes, void *stream)
{
    LogprobParams p = {};
    const int st = fill_logprob_args(p, x, inner_rows, outer_stride, row_stride, io_dtype, rows, n, targets,
                                     ignore_index);
    if (st != GDN2_OK) return st;
    if (top_k < 0 || top_k > n) return GDN2_ERR_INVALID;
    if (top_k > 32) return GDN2_ERR_UNSUPPORTED;
    if (rows == 0) return GDN2_OK;
    if (!logp || !entropy || (top_k > 0 && (!top_logp || !top_ids))) return GDN2_ERR_INVALID;
    const size_t need = gdn2_token_logprobs_workspace_size(rows, n, top_k, io_dtype);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return GDN2_ERR_WORKSPACE;
    p.logp = logp; p.entropy = entropy; p.lse = lse;
    p.top = top_k; p.top_logp = top_logp; p.top_ids = top_ids;
    p.parts = logprob_parts(rows, n, io_dtype);
    p.part_stat = static_cast<float *>(workspace);
    p.part_top = reinterpret_cast<unsigned long long *>(p.part_stat + rows * p.parts * 4);
    return launch_logprobs(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_token_logprobs_bwd(const void *x, int64_t inner_rows, int64_t outer_stride, int64_t row_stride, int io_dtype,
                            int64_t rows, int64_t n, const int64_t *targets, int64_t ignore_index,
                            const float *entropy, const float *lse, const float *dlogp, const float *dentropy,
                            void *dx, void *stream)
{
    LogprobParams p = {};
    const int st = fill_logprob_args(p, x, inner_rows, outer_stride, row_stride, io_dtype, rows, n, targets,
                                     ignore_index);
    if (st != GDN2_OK) return st;
    if (rows == 0) return GDN2_OK;
    if (!entropy || !lse || !dx || reinterpret_cast<uintptr_t>(dx) % (io_dtype == GDN2_DTYPE_F32 ? 4 : 2) != 0)
        return GDN2_ERR_INVALID;
    p.entropy = const_cast<float *>(entropy);
    p.lse = const_cast<float *>(lse);
    p.dlogp = dlogp; p.dent = dentropy;
    p.dx = dx;
    return launch_logprobs_bwd(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

// The sizes gdn2_attn_fwd, gdn2_attn_bwd and its workspace depend on, checked.  `backward`: also what
// the gradient's launches take (of a forward that keeps what they read as well, so that none
// succeeds whose gradient is refused).
static int fill_attn_sizes(AttnTrainParams &p, const int64_t *cu_host, int num_seqs, int B, int Tq, int Tk, int H,
                           int G, int D, int causal, bool backward)
{
    if (B < 0 || Tq < 0 || Tk < 0 || H < 1 || G < 1 || D < 1 || H % G != 0) return GDN2_ERR_INVALID;
    if (Tq > (1 << 30) || Tk > (1 << 30) || B > (1 << 30) || H > (1 << 20) || D > (1 << 20) || num_seqs > (1 << 30))
        return GDN2_ERR_UNSUPPORTED;
    p.max_q = Tq;
    const int64_t qpk = H / G;
    if (Tq * qpk > (1 << 30)) return GDN2_ERR_UNSUPPORTED;  // a group's rows are counted in 32 bits
    while ((static_cast<int64_t>(1) << p.qpk_s) < qpk) ++p.qpk_s;
    p.qpk_m = static_cast<unsigned>(((static_cast<int64_t>(1) << (31 + p.qpk_s)) + qpk - 1) / qpk);
    p.q_tiles = B * ((Tq * qpk + 127) / 128);
    p.k_tiles = static_cast<int64_t>(B) * ((Tk + 127) / 128);
    if (cu_host) {
        if (B != 1 || Tq != Tk || num_seqs < 0) return GDN2_ERR_INVALID;
        if (cu_host[0] != 0 || cu_host[num_seqs] != Tq) return GDN2_ERR_INVALID;
        p.max_q = 0;
        p.q_tiles = p.k_tiles = 0;
        for (int i = 0; i < num_seqs; ++i) {
            const int64_t n = cu_host[i + 1] - cu_host[i];
            if (n < 0 || n > Tq) return GDN2_ERR_INVALID;
            if (n > p.max_q) p.max_q = static_cast<int>(n);
            p.q_tiles += (n * qpk + 127) / 128;
            p.k_tiles += (n + 127) / 128;
        }
    }
    p.nseq = cu_host ? num_seqs : B;
    p.B = B; p.Tq = Tq; p.Tk = Tk; p.H = H; p.G = G; p.D = D;
    p.causal = causal != 0;
    p.splits = attn_bwd_splits(p);
    p.splits_f = p.splits_q = attn_key_shares(p);
    if (!attn_launchable(p, backward) || static_cast<double>(B) * Tq * H > 17179869184.0 ||
        static_cast<double>(B) * (H + G) > 500000000.0 || static_cast<double>(B) * Tk * G * D > 500000000000.0)
        return GDN2_ERR_UNSUPPORTED;
    return GDN2_OK;
}

// Shared by gdn2_attn_fwd and gdn2_attn_bwd: checks, and the parameters both take.
static int fill_attn_args(AttnTrainParams &p, const void *q, const void *k, const void *v, const int64_t *strides,
                          int io_dtype, const int64_t *kv_lengths, const int64_t *cu, const int64_t *cu_host,
                          int num_seqs, int B, int Tq, int Tk, int H, int G, int D, float scale, int causal,
                          bool backward)
{
    if (!valid_dtype(io_dtype) || !strides || (cu == nullptr) != (cu_host == nullptr) || (cu && kv_lengths))
        return GDN2_ERR_INVALID;
    const int st = fill_attn_sizes(p, cu_host, num_seqs, B, Tq, Tk, H, G, D, causal, backward);
    if (st != GDN2_OK) return st;
    if (!attn_train_supported(io_dtype, D)) return GDN2_ERR_UNSUPPORTED;
    if (!(scale > 0.0f) || scale > 1e30f) return GDN2_ERR_UNSUPPORTED;
    if ((B > 0 && Tq > 0 && !q) || (B > 0 && Tk > 0 && (!k || !v))) return GDN2_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)
        return GDN2_ERR_INVALID;
    const int size[9] = {B, Tq, H, B, Tk, G, B, Tk, G};
    for (int i = 0; i < 9; ++i) {
        if (strides[i] < 0 || (size[i] > 1 && strides[i] % 8 != 0)) return GDN2_ERR_INVALID;
        // A token's offset within a tile of them is 32 bits in the kernels.
        if (i % 3 == 1 && size[i] > 1 && strides[i] > kMaxTokenStride) return GDN2_ERR_UNSUPPORTED;
        (i < 3 ? p.qs : i < 6 ? p.ks : p.vs)[i % 3] = size[i] > 1 ? strides[i] : 0;
    }
    if (static_cast<int64_t>(H) * D > kMaxTokenStride) return GDN2_ERR_UNSUPPORTED;  // of dout
    p.q = q; p.k = k; p.v = v;
    p.kv_len = kv_lengths;
    p.cu = cu;
    p.scale = scale;
    return GDN2_OK;
}

int gdn2_attn_fwd(const void *q, const void *k, const void *v, const int64_t *strides, void *o, void *o_lo, float *lse,
                  int io_dtype, const int64_t *kv_lengths, const int64_t *cu_seqlens,
                  const int64_t *cu_seqlens_host, int num_seqs, int B, int Tq, int Tk, int H, int G, int D,
                  float scale, int causal, void *workspace, size_t workspace_bytes, void *stream)
{
    AttnTrainParams p = {};
    const int st = fill_attn_args(p, q, k, v, strides, io_dtype, kv_lengths, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                  Tq, Tk, H, G, D, scale, causal, o_lo != nullptr);
    if (st != GDN2_OK) return st;
    if (B == 0 || Tq == 0 || p.nseq == 0) return GDN2_OK;
    if (!o || !lse || ((reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(o_lo)) & 15)) return GDN2_ERR_INVALID;
    const size_t need = attn_fwd_workspace_bytes(p);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return GDN2_ERR_WORKSPACE;
    p.o = o;
    p.o_lo = o_lo;
    p.lse = lse;
    attn_fwd_workspace(p, workspace);
    return launch_attn_fwd(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_attn_fwd_workspace_size(const int64_t *cu_seqlens_host, int num_seqs, int B, int Tq, int Tk, int H, int G,
                                    int D, int causal)
{
    AttnTrainParams p = {};
    if (fill_attn_sizes(p, cu_seqlens_host, num_seqs, B, Tq, Tk, H, G, D, causal, false) != GDN2_OK) return 0;
    return attn_fwd_workspace_bytes(p);
}

size_t gdn2_attn_bwd_workspace_size(const int64_t *cu_seqlens_host, int num_seqs, int B, int Tq, int Tk, int H, int G,
                                    int D, int causal)
{
    AttnTrainParams p = {};
    if (fill_attn_sizes(p, cu_seqlens_host, num_seqs, B, Tq, Tk, H, G, D, causal, true) != GDN2_OK) return 0;
    return attn_bwd_workspace_bytes(p);
}

int gdn2_attn_bwd(const void *q, const void *k, const void *v, const int64_t *strides, const void *o,
                  const void *o_lo, const float *lse, const void *dout, void *dq, void *dk, void *dv, int io_dtype,
                  const int64_t *kv_lengths, const int64_t *cu_seqlens, const int64_t *cu_seqlens_host,
                  int num_seqs, int B, int Tq, int Tk, int H, int G, int D, float scale, int causal,
                  void *workspace, size_t workspace_bytes, void *stream)
{
    AttnTrainParams p = {};
    const int st = fill_attn_args(p, q, k, v, strides, io_dtype, kv_lengths, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                  Tq, Tk, H, G, D, scale, causal, true);
    if (st != GDN2_OK) return st;
    if (B == 0 || p.nseq == 0 || (Tq == 0 && Tk == 0)) return GDN2_OK;
    if ((Tq > 0 && (!o || !o_lo || !lse || !dout || !dq)) || (Tk > 0 && (!dk || !dv))) return GDN2_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(o_lo) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
         reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) & 15)
        return GDN2_ERR_INVALID;
    if (!workspace || workspace_bytes < attn_bwd_workspace_bytes(p) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return GDN2_ERR_WORKSPACE;
    p.o = const_cast<void *>(o);
    p.o_lo = const_cast<void *>(o_lo);
    p.lse = const_cast<float *>(lse);
    p.dout = dout;
    p.dq = dq; p.dk = dk; p.dv = dv;
    attn_bwd_workspace(p, workspace);
    return launch_attn_bwd(p, io_dtype, static_cast<hipStream_t>(stream)) == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_gate_bwd_workspace_size(int64_t tokens, int H, int K, int has_dt_bias)
{
    if (tokens < 0 || H <= 0 || K <= 0 || K > 256) return 0;
    return gate_bwd_workspace_bytes(tokens, H, K, has_dt_bias != 0);
}

static int check_gate_args(const void *g_raw, int g_dtype, const float *A_log, unsigned flags, int64_t tokens,
                           int H, int K)
{
    if (!valid_dtype(g_dtype) || tokens < 0 || H <= 0 || K <= 0) return GDN2_ERR_INVALID;
    if (flags & ~(GDN2_FLAG_LOWER_BOUND | GDN2_FLAG_LIBRARY_MATH)) return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_LOWER_BOUND) && (flags & GDN2_FLAG_LIBRARY_MATH)) return GDN2_ERR_INVALID;
    if (K > 256) return GDN2_ERR_UNSUPPORTED;
    if (!A_log || (tokens > 0 && !g_raw)) return GDN2_ERR_INVALID;
    return GDN2_OK;
}

int gdn2_gate_fwd(const void *g_raw, int g_dtype, const float *A_log, const float *dt_bias, float lower_bound,
                  unsigned flags, float *y, int64_t tokens, int H, int K, void *stream)
{
    const int st = check_gate_args(g_raw, g_dtype, A_log, flags, tokens, H, K);
    if (st != GDN2_OK) return st;
    if (tokens > 0 && !y) return GDN2_ERR_INVALID;
    return launch_gate_fwd(g_raw, g_dtype, A_log, dt_bias, lower_bound, flags, y, tokens, H, K,
                           static_cast<hipStream_t>(stream));
}

int gdn2_gate_bwd(const void *g_raw, int g_dtype, const float *A_log, const float *dt_bias, float lower_bound,
                  unsigned flags, const float *dy, void *dg_raw, float *dA_log, float *ddt_bias, int64_t tokens,
                  int H, int K, void *workspace, size_t workspace_bytes, void *stream)
{
    const int st = check_gate_args(g_raw, g_dtype, A_log, flags, tokens, H, K);
    if (st != GDN2_OK) return st;
    if ((tokens > 0 && (!dy || !dg_raw)) || !dA_log || (dt_bias != nullptr) != (ddt_bias != nullptr))
        return GDN2_ERR_INVALID;
    if (!workspace || workspace_bytes < gate_bwd_workspace_bytes(tokens, H, K, dt_bias != nullptr))
        return GDN2_ERR_WORKSPACE;
    return launch_gate_bwd(g_raw, g_dtype, A_log, dt_bias, lower_bound, flags, dy, dg_raw, dA_log, ddt_bias,
                           tokens, H, K, workspace, static_cast<hipStream_t>(stream));
}

size_t gdn2_short_conv_bwd_workspace_size(int B, int T, int D, int conv_width)
{
    if (B < 0 || T < 0 || D < 0 || conv_width < 1 || conv_width > 8) return 0;
    return static_cast<size_t>(conv_bwd_partial_floats(B, T, D, conv_width)) * sizeof(float);
}

int gdn2_short_conv_bwd(const void *x, int64_t x_row_stride, const void *weight, const void *bias,
                        const void *dy, void *dx, void *dweight, void *dbias, int io_dtype, int B,
                        int T, int D, int conv_width, int silu, void *workspace,
                        size_t workspace_bytes, void *stream)
{
    if (!valid_dtype(io_dtype) || B < 0 || T < 0 || D < 0) return GDN2_ERR_INVALID;
    if (conv_width < 1 || conv_width > 8) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(B) * T * D == 0) return GDN2_OK;
    if (!x || !weight || !dy || !dx || !dweight || (dbias && !bias) || x_row_stride < D)
        return GDN2_ERR_INVALID;
    if (static_cast<int64_t>(B) * ((T + 31) / 32) > 65535) return GDN2_ERR_UNSUPPORTED;  // grid.y
    if (!workspace || workspace_bytes < gdn2_short_conv_bwd_workspace_size(B, T, D, conv_width))
        return GDN2_ERR_WORKSPACE;
    ConvBwdParams p;
    p.x = x; p.w = weight; p.bias = bias; p.dy = dy; p.dx = dx; p.dw = dweight; p.dbias = dbias;
    p.part = static_cast<float *>(workspace);
    p.B = B; p.T = T; p.D = D; p.W = conv_width; p.ldx = x_row_stride; p.silu = silu != 0;
    const hipError_t err = launch_short_conv_bwd(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_gated_rmsnorm_bwd_workspace_size(int64_t rows, int N)
{
    if (rows < 0 || N <= 0 || N > 256) return 0;
    return static_cast<size_t>(norm_bwd_blocks(rows) * N) * sizeof(float);
}

int gdn2_gated_rmsnorm_bwd(const void *x, const void *z, const void *weight, int weight_dtype,
                           const void *dy, void *dx, void *dz, void *dweight, int io_dtype,
                           int64_t rows, int N, float eps, void *workspace, size_t workspace_bytes,
                           void *stream)
{
    if (!valid_dtype(io_dtype) || !valid_dtype(weight_dtype)) return GDN2_ERR_INVALID;
    if (weight_dtype != io_dtype && weight_dtype != GDN2_DTYPE_F32) return GDN2_ERR_INVALID;
    if (rows < 0 || N <= 0) return GDN2_ERR_INVALID;
    if (N > 256) return GDN2_ERR_UNSUPPORTED;
    if (rows == 0) return GDN2_OK;
    if (!x || !z || !weight || !dy || !dx || !dz || !dweight) return GDN2_ERR_INVALID;
    if (!workspace || workspace_bytes < gdn2_gated_rmsnorm_bwd_workspace_size(rows, N))
        return GDN2_ERR_WORKSPACE;
    NormBwdParams p;
    p.x = x; p.z = z; p.weight = weight; p.dy = dy; p.dx = dx; p.dz = dz; p.dweight = dweight;
    p.part = static_cast<float *>(workspace);
    p.rows = rows; p.N = N; p.eps = eps;
    p.w_f32 = weight_dtype == GDN2_DTYPE_F32;
    const hipError_t err = launch_gated_rmsnorm_bwd(p, io_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

int gdn2_decode_fused(const void *const raw_qkv[3], const int64_t ld_qkv[3], const void *g,
                      int64_t ldg, int g_dtype, const void *b, int64_t ldb, const void *w,
                      int64_t ldw, const void *const conv_weight[3], const void *const conv_bias[3],
                      int conv_width, const void *const conv_cache_in[3],
                      void *const conv_cache_out[3], const float *initial_state,
                      int64_t initial_state_row_stride, float *final_state,
                      int64_t final_state_row_stride, const float *A_log, const float *dt_bias,
                      float lower_bound, const void *gate, int64_t ld_gate,
                      const void *norm_weight, int norm_weight_dtype, float eps, void *o,
                      int io_dtype, int N, int H, int K, int V, float scale, unsigned flags,
                      void *stream)
{
    if (!valid_dtype(io_dtype) || !valid_dtype(g_dtype)) return GDN2_ERR_INVALID;
    if (g_dtype != GDN2_DTYPE_F32 && g_dtype != io_dtype) return GDN2_ERR_UNSUPPORTED;
    if (N < 0 || H <= 0 || K <= 0 || V <= 0) return GDN2_ERR_INVALID;
    if (K != V || (K != 64 && K != 128) || conv_width != 4) return GDN2_ERR_UNSUPPORTED;
    if (flags & ~(GDN2_FLAG_L2NORM_QK | GDN2_FLAG_GATE_IN_KERNEL | GDN2_FLAG_LOWER_BOUND |
                  GDN2_FLAG_SIGMOID_BW))
        return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_LOWER_BOUND) && !(flags & GDN2_FLAG_GATE_IN_KERNEL)) return GDN2_ERR_INVALID;
    if ((flags & GDN2_FLAG_GATE_IN_KERNEL) && !A_log) return GDN2_ERR_INVALID;
    if (static_cast<int64_t>(N) * H > 2147483647LL) return GDN2_ERR_UNSUPPORTED;
    if (N == 0) return GDN2_OK;
    if (!raw_qkv || !ld_qkv || !conv_weight || !g || !b || !w || !o) return GDN2_ERR_INVALID;
    const int64_t HD = static_cast<int64_t>(H) * K;
    DecodeFusedParams p;
    for (int t = 0; t < 3; ++t) {
        if (!raw_qkv[t] || !conv_weight[t] || ld_qkv[t] < HD) return GDN2_ERR_INVALID;
        p.x[t] = raw_qkv[t];
        p.ldx[t] = ld_qkv[t];
        p.cw[t] = conv_weight[t];
        p.cb[t] = conv_bias ? conv_bias[t] : nullptr;
        p.cin[t] = conv_cache_in ? conv_cache_in[t] : nullptr;
        p.cout[t] = conv_cache_out ? conv_cache_out[t] : nullptr;
    }
    if (ldg < HD || ldb < HD || ldw < HD) return GDN2_ERR_INVALID;
    if (gate && (ld_gate < HD || !norm_weight)) return GDN2_ERR_INVALID;
    if (norm_weight && norm_weight_dtype != GDN2_DTYPE_F32 && norm_weight_dtype != io_dtype)
        return GDN2_ERR_INVALID;
    const int64_t slab = HD * V;
    for (const void *st : {static_cast<const void *>(initial_state), static_cast<const void *>(final_state)})
        if (st && (reinterpret_cast<uintptr_t>(st) % 16)) return GDN2_ERR_INVALID;
    if (initial_state && (initial_state_row_stride < slab || initial_state_row_stride % 4))
        return GDN2_ERR_INVALID;
    if (final_state && (final_state_row_stride < slab || final_state_row_stride % 4))
        return GDN2_ERR_INVALID;
    p.g = g; p.b = b; p.w = w;
    p.ldg = ldg; p.ldb = ldb; p.ldw = ldw;
    p.h0 = initial_state;
    p.ht = final_state;
    p.h0_stride = initial_state_row_stride;
    p.ht_stride = final_state_row_stride;
    p.A_log = A_log;
    p.dt_bias = dt_bias;
    p.lower_bound = lower_bound;
    p.z = gate;
    p.ldz = ld_gate;
    p.nw = norm_weight;
    p.nw_f32 = norm_weight && norm_weight_dtype == GDN2_DTYPE_F32 && io_dtype != GDN2_DTYPE_F32;
    p.eps = eps;
    p.o = o;
    p.N = N; p.H = H; p.D = K;
    p.scale = scale;
    p.flags = flags;
    const hipError_t err = launch_decode_fused(p, io_dtype, g_dtype, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_chunk_fwd_workspace_size(int B, int T, int H, int K, int V, int io_dtype,
                                     const int64_t *cu_seqlens_host, int num_seqs)
{
    if (B < 0 || T < 0 || H <= 0 || K <= 0 || V <= 0 || !valid_dtype(io_dtype)) return 0;
    return chunk_fwd_workspace_bytes(B, T, H, K, V, io_dtype, cu_seqlens_host, num_seqs);
}

int gdn2_chunk_fwd(const void *q, const void *k, const void *v, const void *g, const void *b,
                   const void *w, int io_dtype, int g_dtype, void *o,
                   const float *initial_state, float *final_state, const float *A_log,
                   const float *dt_bias, float lower_bound, const int64_t *cu_seqlens,
                   const int64_t *cu_seqlens_host, int num_seqs, int B, int T, int H, int K,
                   int V, float scale, unsigned flags, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    ChunkFwdArgs a;
    const int st = check_chunk_args(io_dtype, g_dtype, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                    T, H, K, V, flags, A_log);
    if (st != GDN2_OK) return st;
    if (static_cast<int64_t>(B) * T > 0 && (!q || !k || !v || !g || !b || !w || !o))
        return GDN2_ERR_INVALID;
    fill_chunk_args(a, q, k, v, g, b, w, o, initial_state, final_state, A_log, dt_bias,
                    lower_bound, cu_seqlens, cu_seqlens_host, num_seqs, B, T, H, K, V, scale,
                    flags, workspace, workspace_bytes);
    a.stages = 3;
    return launch_chunk_fwd(a, io_dtype, g_dtype, static_cast<hipStream_t>(stream));
}

int gdn2_chunk_fwd_gated_norm(const void *q, const void *k, const void *v, const void *g,
                              const void *b, const void *w, int io_dtype, int g_dtype, void *o,
                              const void *gate, int64_t ld_gate, const void *norm_weight, float eps,
                              const float *initial_state, float *final_state, const float *A_log,
                              const float *dt_bias, float lower_bound, const int64_t *cu_seqlens,
                              const int64_t *cu_seqlens_host, int num_seqs, int B, int T, int H,
                              int K, int V, float scale, unsigned flags, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    ChunkFwdArgs a;
    const int st = check_chunk_args(io_dtype, g_dtype, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                    T, H, K, V, flags, A_log);
    if (st != GDN2_OK) return st;
    if (flags & GDN2_FLAG_SAVE_FOR_BWD) return GDN2_ERR_INVALID;  // an inference epilogue
    if (io_dtype != GDN2_DTYPE_BF16 || (V != 16 && V != 32 && V != 64)) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(B) * T > 0 &&
        (!q || !k || !v || !g || !b || !w || !o || !gate || !norm_weight))
        return GDN2_ERR_INVALID;
    // 8-byte gate and output accesses: 4-value groups of every row.
    if (ld_gate < static_cast<int64_t>(H) * V || (ld_gate % 4) != 0 ||
        (reinterpret_cast<uintptr_t>(gate) % 8) != 0 || (reinterpret_cast<uintptr_t>(o) % 8) != 0)
        return GDN2_ERR_INVALID;
    fill_chunk_args(a, q, k, v, g, b, w, o, initial_state, final_state, A_log, dt_bias,
                    lower_bound, cu_seqlens, cu_seqlens_host, num_seqs, B, T, H, K, V, scale,
                    flags, workspace, workspace_bytes);
    a.stages = 3;
    a.z = gate;
    a.ldz = ld_gate;
    a.nw = norm_weight;
    a.eps = eps;
    return launch_chunk_fwd(a, io_dtype, g_dtype, static_cast<hipStream_t>(stream));
}

int gdn2_chunk_fwd_conv(const void *q, int64_t ld_q, const void *k, int64_t ld_k, const void *v, int64_t ld_v,
                        const void *conv_q, const void *conv_k, const void *conv_v, int conv_width,
                        int conv_silu, const void *g, const void *b, const void *w, int io_dtype,
                        int g_dtype, void *o, const void *gate, int64_t ld_gate,
                        const void *norm_weight, float eps, const float *initial_state,
                        float *final_state, const float *A_log, const float *dt_bias, float lower_bound,
                        const int64_t *cu_seqlens, const int64_t *cu_seqlens_host, int num_seqs, int B,
                        int T, int H, int K, int V, float scale, unsigned flags, void *workspace,
                        size_t workspace_bytes, void *stream)
{
    ChunkFwdArgs a;
    const int st = check_chunk_args(io_dtype, g_dtype, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                    T, H, K, V, flags, A_log);
    if (st != GDN2_OK) return st;
    if (flags & GDN2_FLAG_SAVE_FOR_BWD) return GDN2_ERR_INVALID;  // an inference prologue
    if (conv_width != 4 || (conv_silu != 0 && conv_silu != 1)) return GDN2_ERR_UNSUPPORTED;
    if (io_dtype != GDN2_DTYPE_BF16 || (K != 32 && K != 64 && K != 128) || V % 16 != 0)
        return GDN2_ERR_UNSUPPORTED;
    if (gate && V != 16 && V != 32 && V != 64) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(B) * T > 0 &&
        (!q || !k || !v || !g || !b || !w || !o || !conv_q || !conv_k || !conv_v || (gate && !norm_weight)))
        return GDN2_ERR_INVALID;
    // 16-byte row pieces of q, k, v, w and the taps.
    auto a16 = [](const void *x) { return (reinterpret_cast<uintptr_t>(x) % 16) == 0; };
    if (ld_q < static_cast<int64_t>(H) * K || ld_k < static_cast<int64_t>(H) * K ||
        ld_v < static_cast<int64_t>(H) * V || ld_q % 8 || ld_k % 8 || ld_v % 8 || !a16(q) || !a16(k) ||
        !a16(v) || !a16(w) || !a16(b) || !a16(g) || !a16(conv_q) || !a16(conv_k) || !a16(conv_v))
        return GDN2_ERR_INVALID;
    if (gate && (ld_gate < static_cast<int64_t>(H) * V || (ld_gate % 4) != 0 ||
                 (reinterpret_cast<uintptr_t>(gate) % 8) != 0 || (reinterpret_cast<uintptr_t>(o) % 8) != 0))
        return GDN2_ERR_INVALID;
    fill_chunk_args(a, q, k, v, g, b, w, o, initial_state, final_state, A_log, dt_bias,
                    lower_bound, cu_seqlens, cu_seqlens_host, num_seqs, B, T, H, K, V, scale,
                    flags, workspace, workspace_bytes);
    a.stages = 3;
    a.conv_w[0] = conv_q;
    a.conv_w[1] = conv_k;
    a.conv_w[2] = conv_v;
    a.ldq = ld_q;
    a.ldk = ld_k;
    a.ldv = ld_v;
    a.conv_silu = conv_silu;
    if (gate) {
        a.z = gate;
        a.ldz = ld_gate;
        a.nw = norm_weight;
        a.eps = eps;
    }
    return launch_chunk_fwd(a, io_dtype, g_dtype, static_cast<hipStream_t>(stream));
}

int gdn2_chunk_fwd_prep(const void *q, const void *k, const void *g, const void *b,
                        int io_dtype, int g_dtype, const float *A_log, const float *dt_bias,
                        float lower_bound, const int64_t *cu_seqlens,
                        const int64_t *cu_seqlens_host, int num_seqs, int B, int T, int H,
                        int K, int V, float scale, unsigned flags, void *workspace,
                        size_t workspace_bytes, void *stream)
{
    ChunkFwdArgs a;
    const int st = check_chunk_args(io_dtype, g_dtype, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                    T, H, K, V, flags, A_log);
    if (st != GDN2_OK) return st;
    // The separate scan entry point has no flags, so w could not be activated there.
    if (flags & GDN2_FLAG_SIGMOID_BW) return GDN2_ERR_INVALID;
    if (static_cast<int64_t>(B) * T > 0 && (!q || !k || !g || !b)) return GDN2_ERR_INVALID;
    fill_chunk_args(a, q, k, nullptr, g, b, nullptr, nullptr, nullptr, nullptr, A_log, dt_bias,
                    lower_bound, cu_seqlens, cu_seqlens_host, num_seqs, B, T, H, K, V, scale,
                    flags, workspace, workspace_bytes);
    a.stages = 1;
    return launch_chunk_fwd(a, io_dtype, g_dtype, static_cast<hipStream_t>(stream));
}

int gdn2_chunk_fwd_scan(const void *v, const void *w, int io_dtype, void *o,
                        const float *initial_state, float *final_state,
                        const int64_t *cu_seqlens, const int64_t *cu_seqlens_host, int num_seqs,
                        int B, int T, int H, int K, int V, void *workspace,
                        size_t workspace_bytes, void *stream)
{
    ChunkFwdArgs a;
    const int st = check_chunk_args(io_dtype, GDN2_DTYPE_F32, cu_seqlens, cu_seqlens_host,
                                    num_seqs, B, T, H, K, V, 0u, nullptr);
    if (st != GDN2_OK) return st;
    if (static_cast<int64_t>(B) * T > 0 && (!v || !w || !o)) return GDN2_ERR_INVALID;
    fill_chunk_args(a, nullptr, nullptr, v, nullptr, nullptr, w, o, initial_state, final_state,
                    nullptr, nullptr, 0.f, cu_seqlens, cu_seqlens_host, num_seqs, B, T, H, K, V,
                    1.f, 0u, workspace, workspace_bytes);
    a.stages = 2;
    return launch_chunk_fwd(a, io_dtype, GDN2_DTYPE_F32, static_cast<hipStream_t>(stream));
}

size_t gdn2_chunk_train_workspace_size(int B, int T, int H, int K, int V, int io_dtype,
                                       const int64_t *cu_seqlens_host, int num_seqs)
{
    if (B < 0 || T < 0 || H <= 0 || K <= 0 || V <= 0 || !valid_dtype(io_dtype)) return 0;
    return chunk_train_workspace_bytes(B, T, H, K, V, io_dtype, cu_seqlens_host, num_seqs);
}

int gdn2_chunk_states(const void *saved, size_t saved_bytes, int io_dtype, void *out, int transpose,
                      const int64_t *cu_seqlens_host, int num_seqs, int B, int T, int H, int K,
                      int V, void *stream)
{
    if (!valid_dtype(io_dtype) || B < 0 || T < 0 || H <= 0 || K <= 0 || V <= 0) return GDN2_ERR_INVALID;
    if (cu_seqlens_host && (B != 1 || num_seqs < 0)) return GDN2_ERR_INVALID;
    const bool wide = chunk_wide(K, io_dtype);
    if (!wide && !chunk_k_supported(K, io_dtype)) return GDN2_ERR_UNSUPPORTED;
    const int64_t nc = count_chunks(B, T, cu_seqlens_host, num_seqs);
    if (nc == 0) return GDN2_OK;
    if (!saved || !out) return GDN2_ERR_INVALID;
    if (wide) {
        if (saved_bytes < wide_train_workspace_bytes(B, T, H, K, V, cu_seqlens_host, num_seqs))
            return GDN2_ERR_WORKSPACE;
        const hipError_t err = launch_chunk_states_wide(saved, out, transpose != 0, nc, H, K, V,
                                                        static_cast<hipStream_t>(stream));
        return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
    }
    const TrainLayout tl = train_layout(nc, H, K, V, io_dtype);
    if (saved_bytes < static_cast<size_t>(tl.total)) return GDN2_ERR_WORKSPACE;
    const hipError_t err = launch_chunk_states(static_cast<const unsigned char *>(saved) + tl.hs, io_dtype, out,
                                               transpose != 0, nc, H, K, V, static_cast<hipStream_t>(stream));
    return err == hipSuccess ? GDN2_OK : GDN2_ERR_LAUNCH;
}

size_t gdn2_chunk_bwd_workspace_size(int B, int T, int H, int K, int V, int io_dtype,
                                     const int64_t *cu_seqlens_host, int num_seqs)
{
    if (B < 0 || T < 0 || H <= 0 || K <= 0 || V <= 0 || !valid_dtype(io_dtype)) return 0;
    return chunk_bwd_workspace_bytes(B, T, H, K, V, io_dtype, cu_seqlens_host, num_seqs);
}

int gdn2_chunk_bwd(const void *q, const void *k, const void *v, const void *g, const void *b,
                   const void *w, int io_dtype, int g_dtype, const void *dout,
                   const float *dht, void *dq, void *dk, void *dv, void *dg, void *db, void *dw,
                   float *dh0, const int64_t *cu_seqlens, const int64_t *cu_seqlens_host,
                   int num_seqs, int B, int T, int H, int K, int V, float scale,
                   unsigned flags, const void *saved, size_t saved_bytes, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    const int st = check_chunk_args(io_dtype, g_dtype, cu_seqlens, cu_seqlens_host, num_seqs, B,
                                    T, H, K, V, flags & ~GDN2_FLAG_SAVE_FOR_BWD, nullptr);
    if (st != GDN2_OK) return st;
    if (flags & (GDN2_FLAG_GATE_IN_KERNEL | GDN2_FLAG_LOWER_BOUND)) return GDN2_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(B) * T > 0 &&
        (!q || !k || !v || !g || !b || !w || !dout || !dq || !dk || !dv || !dg || !db || !dw))
        return GDN2_ERR_INVALID;
    ChunkBwdArgs a;
    a.q = q; a.k = k; a.v = v; a.g = g; a.b = b; a.w = w; a.dout = dout;
    a.dht = dht;
    a.dq = dq; a.dk = dk; a.dv = dv; a.dg = dg; a.db = db; a.dw = dw;
    a.dh0 = dh0;
    a.cu_seqlens = cu_seqlens;
    a.cu_host = cu_seqlens_host;
    a.num_seqs = cu_seqlens ? num_seqs : B;
    a.B = B; a.T = T; a.H = H; a.K = K; a.V = V;
    a.scale = scale;
    a.flags = flags;
    a.saved = saved;
    a.saved_bytes = saved_bytes;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    return launch_chunk_bwd(a, io_dtype, g_dtype, static_cast<hipStream_t>(stream));
}

}  // extern "C"

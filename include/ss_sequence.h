/*
 * ss_sequence.h — C-ABI of the sequence operators (libss_sequence.so): leaky attention over a [T][B] sequence or one step, the root-mean-square norm with
 * the residual's addition (16 / 32-bit output with gradients, or 8-bit codes with scales), and the 8-bit integer product with scales.
 *
 * Conventions: those of ss_neuron.h.  Plain device pointers and sizes, nothing allocated, no state kept; asynchronous on `stream` (a hipStream_t as void*);
 * 0 or a negative errno-style code, nothing thrown across the ABI; deterministic (fixed-order second passes, no float atomics); every launch may be
 * recorded into a graph (no host synchronisation, no memset).  Strides count ELEMENTS; the last axis of every operand is contiguous.
 */
#ifndef SS_SEQUENCE_H
#define SS_SEQUENCE_H

#ifdef __cplusplus
extern "C" {
#endif

#define SS_SEQ_OK        0
#define SS_SEQ_EINVAL  (-22)
#define SS_SEQ_ELAUNCH  (-5)

/* element type of activations */
#define SS_SEQ_F32   0
#define SS_SEQ_F16   1
#define SS_SEQ_BF16  2

#define SS_SEQ_ABI_VERSION 1
int ss_seq_abi_version(void);

/*
 * Leaky map.  With lambda_h = exp(log_decay[h]), for every stream b and head h, over the valid steps i = 0 .. n-1 of the stream
 * (n = lengths ? clamp(lengths[b], 0, T) : T), counted from the first step (reverse = 0) or from the last valid one backwards (reverse = 1):
 *
 *      S_i   = lambda S_{i-1} + b_scale * b_i c_i^T          [DA][DC], fp32
 *      out_i = o_scale * a_i^T S_i
 *
 * S_{-1} = s_in (NULL: zero).  reverse = 1 takes s_in UNDECAYED at its first step and hands s_out decayed once more (the adjoint of the forward map);
 * s_out (NULL: not wanted) is the state after the last valid step, s_in itself if there is none.  out rows of steps >= n are written as zeros.
 *
 *   forward: a, b, c = q, k, v, b_scale 1, o_scale scale.  Each token gradient is such a map too (ss_seq_leaky_bwd).
 *
 * a [T][B][H / a_group][DA], b [T][B][H / b_group][DA], c [T][B][H / c_group][DC], out [T][B][H][DC] with the strides given; head h reads operand head
 * h / group.  s_in / s_out: [B][H] matrices DA x DC, element (i, j) at i * s_*_row + j * s_*_col, matrices DA * DC apart.  s_in may be s_out itself
 * when T = 1 and their strides are the same.
 */
struct ss_seq_leaky_desc {
    unsigned size;                       /* sizeof(struct ss_seq_leaky_desc) */
    int dtype, out_dtype;                /* of a, b, c; of out (dtype or SS_SEQ_F32) */
    int T, B, H, DA, DC;                 /* DA, DC <= 256 */
    int reverse;
    float b_scale, o_scale;
    const void *a, *b, *c;
    void* out;
    long long a_t, a_b, a_h, b_t, b_b, b_h, c_t, c_b, c_h, o_t, o_b, o_h;
    int a_group, b_group, c_group;
    const float* log_decay;              /* [H] */
    const int* lengths;                  /* [B] or NULL */
    const float* s_in;
    float* s_out;
    int s_in_row, s_in_col, s_out_row, s_out_col;
    float* ws;                           /* ss_seq_leaky_ws_floats() floats, NULL if that is 0 */
};
long long ss_seq_leaky_ws_floats(const struct ss_seq_leaky_desc* d);
int ss_seq_leaky(const struct ss_seq_leaky_desc* d, void* stream);

/*
 * Gradients of the forward map o = leaky(q, k, v) with H query heads on Hk key / value heads, from g = dL/do and g_last = dL/d(last state) (NULL: zero):
 *
 *      g_q  a, b, c = g, v, k   forward, from s_in transposed           o_scale scale
 *      g_k  a, b, c = v, g, q   reverse, from g_last transposed         b_scale scale
 *      g_v  a, b, c = k, q, g   reverse, from g_last                    b_scale scale;   g_s, the gradient of s_in, is its last state
 *
 * g_k, g_v: summed over the query heads that share a head (in fp32, in their order), rounded once.  g_q [T][B][H][Dk], g_k [T][B][Hk][Dk],
 * g_v [T][B][Hk][Dv] contiguous in dtype, each NULL if not wanted; g_s fp32 [B][H][Dk][Dv] or NULL, wants g_v.  s_in: [B][H][Dk][Dv] contiguous or NULL, as
 * the forward pass had it.  states: the workspace of the forward pass (same sizes, type and lengths), as it left it.
 */
struct ss_seq_leaky_bwd_desc {
    unsigned size;                       /* sizeof(struct ss_seq_leaky_bwd_desc) */
    int dtype, T, B, H, Hk, Dk, Dv;
    float scale;
    const void *q, *k, *v, *g;
    long long q_t, q_b, q_h, k_t, k_b, k_h, v_t, v_b, v_h, g_t, g_b, g_h;
    void *g_q, *g_k, *g_v;
    const float* log_decay;
    const int* lengths;
    const float *s_in, *g_last;
    float* g_s;
    const float* states;                 /* NULL if ss_seq_leaky_ws_floats() was 0 */
    float* ws;                           /* ss_seq_leaky_bwd_ws_floats() floats, 16-byte aligned, NULL if that is 0 */
};
long long ss_seq_leaky_bwd_ws_floats(const struct ss_seq_leaky_bwd_desc* d);
int ss_seq_leaky_bwd(const struct ss_seq_leaky_bwd_desc* d, void* stream);

/* out[r][j] = sum over the `group` consecutive rows of x [rows * group][D] (fp32), rounded once to dtype: the gradients of heads that several heads read */
int ss_seq_group_sum(const float* x, void* out, long long rows, int group, int D, int dtype, void* stream);

/*
 * Add + root-mean-square norm:   h = round(x + residual)  (residual NULL: h = x, sum not written),
 *                                y = h * rstd * weight,   rstd = 1 / sqrt(mean(h^2) + eps)
 * x, residual: rows of C with their own row strides; y, sum: [rows][C] contiguous; weight fp32 [C]; rstd fp32 [rows] (NULL: not wanted).
 * Sums in fp32 (in fp64 where fp32 leaves its range); rstd is fp32, so sqrt(mean(h^2) + eps) has to be at least 3e-39.
 */
int ss_seq_rms_norm_fwd(const void* x, long long x_stride, const void* residual, long long r_stride, const float* weight, void* y, void* sum, float* rstd,
                        long long rows, int C, float eps, int dtype, void* stream);
/*
 * Its gradients: with n = h * rstd,   g_h = rstd * (weight g_y - n * mean(weight g_y n)) + g_sum     (g_sum NULL: none; g_y NULL: zero)
 *                                     g_w = sum over rows of g_y n        (NULL: not wanted; fixed order: ss_seq_rms_norm_ws_floats() floats in ws)
 * g_y, g_sum, h, g_h: [rows][C] contiguous.
 */
long long ss_seq_rms_norm_ws_floats(long long rows, int C, int dtype);
int ss_seq_rms_norm_bwd(const void* g_y, const void* g_sum, const void* h, const float* weight, const float* rstd, void* g_h, float* g_w, float* ws,
                        long long rows, int C, int dtype, void* stream);
/*
 * The same norm handed on in 8 bits: u = h * weight, top = max |u| of the row, codes = rint(127 u / top) (ties to even, exact: values next to a border are
 * decided in fp64), scales[row] = top * rstd / 127, so codes * scale is the norm.  A row of zeros has scale 0; a row in
 * which h or the weight holds a NaN or an infinity has codes 0 and scale NaN (finite values may have products beyond fp32).
 */
int ss_seq_rms_norm_int8(const void* x, long long x_stride, const void* residual, long long r_stride, const float* weight, signed char* codes, float* scales,
                         void* sum, long long rows, int C, float eps, int dtype, void* stream);
/* out[r][j] = codes[r][j] * scales[r] rounded once to dtype; codes, out contiguous */
int ss_seq_dequant_int8(const signed char* codes, const float* scales, void* out, long long rows, int C, int dtype, void* stream);

/*
 * 8-bit integer product:  out[m][n] = (sum_k a[m][k] * w[n][k]) * a_scale[m] * w_scale[n] + bias[n]
 * a [M][K] (row stride lda), w [N][K] (row stride ldw), sums exact in 32-bit integers (K < 131072), out [M][N] contiguous in out_dtype; bias may be NULL.
 * Any row strides and alignment; rows that are not aligned to 16 bytes are copied into the workspace first.  M, N <= 2^27, less than 2^24 tiles of 128 x 128 outputs.
 */
long long ss_seq_int8_linear_ws_ints(const signed char* a, long long lda, const signed char* w, long long ldw, long long M, int N, int K);      /* of ws */
int ss_seq_int8_linear(const signed char* a, long long lda, const float* a_scale, const signed char* w, long long ldw, const float* w_scale,
                       const float* bias, void* out, long long M, int N, int K, int out_dtype, int* ws, void* stream);

#ifdef __cplusplus
}
#endif
#endif

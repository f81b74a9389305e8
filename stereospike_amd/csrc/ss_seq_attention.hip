// ss_seq_attention.hip — leaky attention: a matrix-valued leaky integrator per head, read by a query.
//
//   S_i = lambda S_{i-1} + b_scale b_i c_i^T,   out_i = o_scale a_i^T S_i,   lambda = exp(log_decay) of the head
//
// The forward pass and the three token gradients are this one map with other operands, forwards or backwards in time (ss_sequence.h).
#include "ss_seq_common.hpp"

namespace {

struct LeakyArgs {
    int T, B, H, DA, DC, reverse;
    float b_scale, o_scale;
    const void *a, *b, *c;
    void* out;
    long long a_t, a_b, a_h, b_t, b_b, b_h, c_t, c_b, c_h, o_t, o_b, o_h;
    int a_group, b_group, c_group;
    const float* log_decay;
    const int* lengths;
    const float* s_in;
    float* s_out;
    int s_in_row, s_in_col, s_out_row, s_out_col;
};

// The recurrence itself, one step after the other with the state in registers: HBM-bound on reading and writing the state when T is small (the single-step
// call).  A workgroup owns 64 columns of one head's state: thread (g, x) holds rows g + 16 r of columns 4 x .. 4 x + 3.
template <int DT, int ODT, int R, bool V4> __global__ __launch_bounds__(256) void leaky_steps_kernel(const LeakyArgs p)
{
    __shared__ float sa[256], sb[256], red[4][64];
    const int tid = threadIdx.x, x = tid & 15, g = tid >> 4;
    const int bh = blockIdx.y, b = bh / p.H, h = bh % p.H, j0 = blockIdx.x * 64 + 4 * x;
    int n = p.T;
    if (p.lengths) { n = p.lengths[b]; n = n < 0 ? 0 : n > p.T ? p.T : n; }
    // lambda S as S + S * expm1(g) while lambda is over a half: a rounded lambda near 1 would drift over many steps (2^-25 of it each)
    const float g_h = fmaxf(p.log_decay[h], -1e30f), lam = expf(g_h), leak = g_h > -0.69f ? expm1f(g_h) : lam, kept = g_h > -0.69f ? 1.f : 0.f;
    const elem_t<DT>* pa = static_cast<const elem_t<DT>*>(p.a) + b * p.a_b + (h / p.a_group) * p.a_h;
    const elem_t<DT>* pb = static_cast<const elem_t<DT>*>(p.b) + b * p.b_b + (h / p.b_group) * p.b_h;
    const elem_t<DT>* pc = static_cast<const elem_t<DT>*>(p.c) + b * p.c_b + (h / p.c_group) * p.c_h;
    elem_t<ODT>* po = static_cast<elem_t<ODT>*>(p.out) + b * p.o_b + h * p.o_h;
    const float* s_in = p.s_in ? p.s_in + (long long)bh * p.DA * p.DC : nullptr;
    float* s_out = p.s_out ? p.s_out + (long long)bh * p.DA * p.DC : nullptr;
    f32x4 S[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        S[r] = (f32x4){0.f, 0.f, 0.f, 0.f};
        const int i = g + 16 * r;
        if (s_in && i < p.DA) {
            if constexpr (V4) { if (j0 < p.DC) S[r] = *reinterpret_cast<const f32x4*>(s_in + i * p.s_in_row + j0); }
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) if (j0 + e < p.DC) S[r][e] = s_in[i * p.s_in_row + (j0 + e) * p.s_in_col];
        }
    }
    for (int i = 0; i < n; ++i) {
        const long long t = p.reverse ? n - 1 - i : i;
        __syncthreads();
        if (tid < p.DA) { sa[tid] = widen<DT>(pa[t * p.a_t + tid]) * p.o_scale; sb[tid] = widen<DT>(pb[t * p.b_t + tid]) * p.b_scale; }
        __syncthreads();
        f32x4 c = {0.f, 0.f, 0.f, 0.f}, o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) if (j0 + e < p.DC) c[e] = widen<DT>(pc[t * p.c_t + j0 + e]);
        const bool leaks = i > 0 || !p.reverse;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = g + 16 * r;
            if (row < p.DA) {
                const float bi = sb[row], ai = sa[row];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float s = S[r][e];
                    if (leaks) s = fmaf(s, leak, s * kept);
                    s = fmaf(bi, c[e], s);
                    o[e] = fmaf(ai, s, o[e]);
                    S[r][e] = s;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e] += __shfl_xor(o[e], 16);
            o[e] += __shfl_xor(o[e], 32);
        }
        if ((tid & 48) == 0) *reinterpret_cast<f32x4*>(&red[tid >> 6][4 * x]) = o;
        __syncthreads();
        if (tid < 64 && blockIdx.x * 64 + tid < p.DC)
            po[t * p.o_t + blockIdx.x * 64 + tid] = narrow<ODT>(red[0][tid] + red[1][tid] + red[2][tid] + red[3][tid]);
    }
    if (tid < 64 && blockIdx.x * 64 + tid < p.DC)
        for (int t = n; t < p.T; ++t) po[t * p.o_t + blockIdx.x * 64 + tid] = 0;
    if (s_out) {
        const float last = p.reverse && n > 0 ? lam : 1.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = g + 16 * r;
            if (i < p.DA) {
                if constexpr (V4) { if (j0 < p.DC) *reinterpret_cast<f32x4*>(s_out + i * p.s_out_row + j0) = S[r] * last; }
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (j0 + e < p.DC) s_out[i * p.s_out_row + (j0 + e) * p.s_out_col] = S[r][e] * last;
            }
        }
    }
}

template <int DT, int ODT> int steps(const LeakyArgs& p, hipStream_t s)
{
    const bool v4 = p.DC % 4 == 0 && (!p.s_in || (p.s_in_col == 1 && p.s_in_row % 4 == 0 && aligned(p.s_in, 16))) &&
                    (!p.s_out || (p.s_out_col == 1 && p.s_out_row % 4 == 0 && aligned(p.s_out, 16)));
    const dim3 grid((unsigned)((p.DC + 63) / 64), (unsigned)(p.B * p.H));
    auto go = [&](auto R) {
        if (v4) leaky_steps_kernel<DT, ODT, R.value, true><<<grid, 256, 0, s>>>(p);
        else leaky_steps_kernel<DT, ODT, R.value, false><<<grid, 256, 0, s>>>(p);
        return launched();
    };
    if (p.DA <= 64) return go(std::integral_constant<int, 4>());
    if (p.DA <= 128) return go(std::integral_constant<int, 8>());
    return go(std::integral_constant<int, 16>());
}

template <int DT> int leaky_dt(const LeakyArgs& p, bool f32_out, hipStream_t s)
{
    if constexpr (DT != SS_SEQ_F32) { if (f32_out) return steps<DT, SS_SEQ_F32>(p, s); }
    return steps<DT, DT>(p, s);
}

template <int DT> __global__ __launch_bounds__(256) void group_sum_kernel(const float* __restrict__ x, elem_t<DT>* __restrict__ out, long long n, int group, int D)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long r = i / D;
        const float* q = x + r * group * D + (i - r * D);
        float s = q[0];
        for (int k = 1; k < group; ++k) s += q[(long long)k * D];
        out[i] = narrow<DT>(s);
    }
}

bool desc_ok(const ss_seq_leaky_desc* d)
{
    if (!d || d->size != sizeof(ss_seq_leaky_desc)) return false;
    if (d->dtype != SS_SEQ_F32 && d->dtype != SS_SEQ_F16 && d->dtype != SS_SEQ_BF16) return false;
    if (d->out_dtype != d->dtype && d->out_dtype != SS_SEQ_F32) return false;
    if (d->T < 1 || d->B < 1 || d->H < 1 || (long long)d->B * d->H > 65535 || d->DA < 1 || d->DA > 256 || d->DC < 1 || d->DC > 256) return false;
    if (d->a_group < 1 || d->b_group < 1 || d->c_group < 1 || d->H % d->a_group || d->H % d->b_group || d->H % d->c_group) return false;
    if (!d->a || !d->b || !d->c || !d->out || !d->log_decay) return false;
    return true;
}

}  // namespace

extern "C" {

long long ss_seq_leaky_ws_floats(const ss_seq_leaky_desc*) { return 0; }

int ss_seq_leaky(const ss_seq_leaky_desc* d, void* stream)
{
    if (!desc_ok(d)) return SS_SEQ_EINVAL;
    const LeakyArgs p{d->T, d->B, d->H, d->DA, d->DC, d->reverse, d->b_scale, d->o_scale, d->a, d->b, d->c, d->out,
                      d->a_t, d->a_b, d->a_h, d->b_t, d->b_b, d->b_h, d->c_t, d->c_b, d->c_h, d->o_t, d->o_b, d->o_h,
                      d->a_group, d->b_group, d->c_group, d->log_decay, d->lengths, d->s_in, d->s_out,
                      d->s_in_row, d->s_in_col, d->s_out_row, d->s_out_col};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f32_out = d->out_dtype == SS_SEQ_F32;
    return d->dtype == SS_SEQ_F32 ? leaky_dt<SS_SEQ_F32>(p, f32_out, s) : d->dtype == SS_SEQ_F16 ? leaky_dt<SS_SEQ_F16>(p, f32_out, s)
                                                                                               : leaky_dt<SS_SEQ_BF16>(p, f32_out, s);
}

int ss_seq_group_sum(const float* x, void* out, long long rows, int group, int D, int dtype, void* stream)
{
    if (!x || !out || rows < 1 || group < 1 || D < 1) return SS_SEQ_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const long long n = rows * D, want = (n + 255) / 256;
    const unsigned grid = (unsigned)(want < 8192 ? want : 8192);
    if (dtype == SS_SEQ_F32) group_sum_kernel<SS_SEQ_F32><<<grid, 256, 0, s>>>(x, static_cast<float*>(out), n, group, D);
    else if (dtype == SS_SEQ_F16) group_sum_kernel<SS_SEQ_F16><<<grid, 256, 0, s>>>(x, static_cast<unsigned short*>(out), n, group, D);
    else if (dtype == SS_SEQ_BF16) group_sum_kernel<SS_SEQ_BF16><<<grid, 256, 0, s>>>(x, static_cast<unsigned short*>(out), n, group, D);
    else return SS_SEQ_EINVAL;
    return launched();
}

}  // extern "C"

// ss_seq_attention.hip — leaky attention: checks, dispatch by element type, and the sum over heads that share an operand.
#include "ss_seq_attention.hpp"

namespace {

// the gradient of a shared head: the sum over its `group` query heads in their order, fp32; V consecutive values of a thread, the heads' loads in flight together.
// HBM-bound (4662 rows of 8 heads of 96, fp32: 14.3 MB read, 7.2 written in 5 us)
template <int DT, int V> __global__ __launch_bounds__(256) void group_sum_kernel(const float* __restrict__ x, elem_t<DT>* __restrict__ out, long long n, int group, int D)
{
    typedef Pack<SS_SEQ_F32, V> F;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < n; i += (long long)gridDim.x * 256 * V) {
        const long long r = n <= 0x7FFFFFFF ? (long long)((unsigned)i / (unsigned)D) : i / D;
        const float* q = x + r * group * D + (i - r * D);
        F s = *reinterpret_cast<const F*>(q);
        for (int k = 1; k < group; k += 4) {
            F v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const F*>(q + (long long)min(k + u, group - 1) * D);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k + u < group)
#pragma unroll
                    for (int e = 0; e < V; ++e) s.v[e] += v[u].v[e];
        }
        Pack<DT, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = narrow<DT>(s.v[e]);
        *reinterpret_cast<Pack<DT, V>*>(out + i) = o;
    }
}

bool desc_ok(const ss_seq_leaky_desc* d)
{
    if (!d || d->size != sizeof(ss_seq_leaky_desc)) return false;
    if (d->dtype != SS_SEQ_F32 && d->dtype != SS_SEQ_F16 && d->dtype != SS_SEQ_BF16) return false;
    if (d->out_dtype != d->dtype && d->out_dtype != SS_SEQ_F32) return false;
    if (d->T < 1 || d->T > (1 << 30) || d->B < 1 || d->H < 1 || (long long)d->B * d->H > 65535 || d->DA < 1 || d->DA > 256 || d->DC < 1 || d->DC > 256) return false;
    if (d->a_group < 1 || d->b_group < 1 || d->c_group < 1 || d->H % d->a_group || d->H % d->b_group || d->H % d->c_group) return false;
    if (!d->a || !d->b || !d->c || !d->out || !d->log_decay) return false;
    // in place: one step, element for element (a segment may read the first state after another wrote the last)
    if (d->s_in && d->s_in == d->s_out && (d->T > 1 || d->s_in_row != d->s_out_row || d->s_in_col != d->s_out_col)) return false;
    return true;
}

LeakyArgs args_of(const ss_seq_leaky_desc* d)
{
    return {d->T, d->B, d->H, d->DA, d->DC, d->reverse, d->b_scale, d->o_scale, d->a, d->b, d->c, d->out,
            d->a_t, d->a_b, d->a_h, d->b_t, d->b_b, d->b_h, d->c_t, d->c_b, d->c_h, d->o_t, d->o_b, d->o_h,
            d->a_group, d->b_group, d->c_group, d->log_decay, d->lengths, d->s_in, d->s_out,
            d->s_in_row, d->s_in_col, d->s_out_row, d->s_out_col, d->out_dtype == SS_SEQ_F32};
}

bool bwd_ok(const ss_seq_leaky_bwd_desc* d)
{
    if (!d || d->size != sizeof(ss_seq_leaky_bwd_desc)) return false;
    if (d->dtype != SS_SEQ_F32 && d->dtype != SS_SEQ_F16 && d->dtype != SS_SEQ_BF16) return false;
    if (d->T < 1 || d->T > (1 << 30) || d->B < 1 || d->H < 1 || d->Hk < 1 || d->H % d->Hk || (long long)d->B * d->H > 65535) return false;
    if (d->Dk < 1 || d->Dk > 256 || d->Dv < 1 || d->Dv > 256) return false;
    if (!d->q || !d->k || !d->v || !d->g || !d->log_decay || (d->g_s && !d->g_v)) return false;
    return true;
}

LeakyBwdArgs bwd_of(const ss_seq_leaky_bwd_desc* d)
{
    const int group = d->H / d->Hk;
    return {d->T, d->B, d->H, d->Hk, d->Dk, d->Dv, d->scale, {d->q, d->q_t, d->q_b, d->q_h, 1}, {d->k, d->k_t, d->k_b, d->k_h, group},
            {d->v, d->v_t, d->v_b, d->v_h, group}, {d->g, d->g_t, d->g_b, d->g_h, 1}, d->g_q, d->g_k, d->g_v, d->log_decay, d->lengths,
            d->s_in, d->g_last, d->g_s, d->states, d->ws};
}

}  // namespace

extern "C" {

long long ss_seq_leaky_ws_floats(const ss_seq_leaky_desc* d)
{
    if (!desc_ok(d)) return 0;
    const LeakyArgs p = args_of(d);
    return d->dtype == SS_SEQ_F32 ? ss_seq_leaky_ws_f32(p) : d->dtype == SS_SEQ_F16 ? ss_seq_leaky_ws_f16(p) : ss_seq_leaky_ws_bf16(p);
}

int ss_seq_leaky(const ss_seq_leaky_desc* d, void* stream)
{
    if (!desc_ok(d)) return SS_SEQ_EINVAL;
    const LeakyArgs p = args_of(d);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return d->dtype == SS_SEQ_F32 ? ss_seq_leaky_f32(p, d->ws, s) : d->dtype == SS_SEQ_F16 ? ss_seq_leaky_f16(p, d->ws, s) : ss_seq_leaky_bf16(p, d->ws, s);
}

long long ss_seq_leaky_bwd_ws_floats(const ss_seq_leaky_bwd_desc* d)
{
    if (!bwd_ok(d)) return 0;
    const LeakyBwdArgs p = bwd_of(d);
    return d->dtype == SS_SEQ_F32 ? ss_seq_leaky_bwd_ws_f32(p) : d->dtype == SS_SEQ_F16 ? ss_seq_leaky_bwd_ws_f16(p) : ss_seq_leaky_bwd_ws_bf16(p);
}

int ss_seq_leaky_bwd(const ss_seq_leaky_bwd_desc* d, void* stream)
{
    if (!bwd_ok(d)) return SS_SEQ_EINVAL;
    const LeakyBwdArgs p = bwd_of(d);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return d->dtype == SS_SEQ_F32 ? ss_seq_leaky_bwd_f32(p, s) : d->dtype == SS_SEQ_F16 ? ss_seq_leaky_bwd_f16(p, s) : ss_seq_leaky_bwd_bf16(p, s);
}

int ss_seq_group_sum(const float* x, void* out, long long rows, int group, int D, int dtype, void* stream)
{
    if (!x || !out || rows < 1 || group < 1 || D < 1) return SS_SEQ_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const long long n = rows * D;
    const bool four = D % 4 == 0 && aligned(x, 16) && aligned(out, 16);
    const long long want = (n / (four ? 4 : 1) + 255) / 256;
    const unsigned grid = (unsigned)(want < 8192 ? want : 8192);
    auto go = [&](auto DTC) {
        constexpr int DT = DTC.value;
        if (four) group_sum_kernel<DT, 4><<<grid, 256, 0, s>>>(x, static_cast<elem_t<DT>*>(out), n, group, D);
        else group_sum_kernel<DT, 1><<<grid, 256, 0, s>>>(x, static_cast<elem_t<DT>*>(out), n, group, D);
    };
    if (dtype == SS_SEQ_F32) go(std::integral_constant<int, SS_SEQ_F32>());
    else if (dtype == SS_SEQ_F16) go(std::integral_constant<int, SS_SEQ_F16>());
    else if (dtype == SS_SEQ_BF16) go(std::integral_constant<int, SS_SEQ_BF16>());
    else return SS_SEQ_EINVAL;
    return launched();
}

}  // extern "C"

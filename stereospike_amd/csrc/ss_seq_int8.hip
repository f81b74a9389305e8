// ss_seq_int8.hip — 8-bit integer product with a scale for each token (row of a) and channel (row of w).
//
//   out[m][n] = (sum_k a[m][k] w[n][k]) * a_scale[m] * w_scale[n] + bias[n]
//
// v_mfma_i32_32x32x32_i8: both operands give lane l the 16 consecutive k of row l % 32 that start at 16 * (l / 32); the sum is exact in 32 bits for
// K < 131072 (128 * 128 * 131071 < 2^31).
#include "ss_seq_common.hpp"

namespace {

struct MmArgs {
    const signed char *a, *w;
    long long lda, ldw;
    const float *as, *wsc, *bias;
    void* out;
    long long M;
    int N, K;
};

// 64 x 64 outputs per workgroup, 64 k per step.  VEC: rows of 16-byte granules (K % 16 == 0, aligned rows); otherwise bytes.
template <int DT, bool VEC> __global__ __launch_bounds__(256) void mm64_kernel(const MmArgs p)
{
    constexpr int LD = 80;                                 // 64 + 16: rows 20 banks apart
    __shared__ __attribute__((aligned(16))) signed char sa[64 * LD], sw[64 * LD];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const long long m0 = (long long)blockIdx.y * 64;
    const int n0 = blockIdx.x * 64;
    const int wm = (wv >> 1) * 32, wn = (wv & 1) * 32;
    i32x16 acc = {};
    for (int k0 = 0; k0 < p.K; k0 += 64) {
        __syncthreads();
        if constexpr (VEC) {
            const int r = tid >> 2, c = (tid & 3) * 16;
            i32x4 va = {}, vw = {};
            if (k0 + c < p.K) {
                if (m0 + r < p.M) va = *reinterpret_cast<const i32x4*>(p.a + (m0 + r) * p.lda + k0 + c);
                if (n0 + r < p.N) vw = *reinterpret_cast<const i32x4*>(p.w + (long long)(n0 + r) * p.ldw + k0 + c);
            }
            *reinterpret_cast<i32x4*>(sa + r * LD + c) = va;
            *reinterpret_cast<i32x4*>(sw + r * LD + c) = vw;
        } else {
            for (int i = tid; i < 64 * 64; i += 256) {
                const int r = i >> 6, c = i & 63;
                const bool in = k0 + c < p.K;
                sa[r * LD + c] = in && m0 + r < p.M ? p.a[(m0 + r) * p.lda + k0 + c] : (signed char)0;
                sw[r * LD + c] = in && n0 + r < p.N ? p.w[(long long)(n0 + r) * p.ldw + k0 + c] : (signed char)0;
            }
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const i32x4 fa = *reinterpret_cast<const i32x4*>(sa + (wm + (lane & 31)) * LD + ks * 32 + (lane >> 5) * 16);
            const i32x4 fw = *reinterpret_cast<const i32x4*>(sw + (wn + (lane & 31)) * LD + ks * 32 + (lane >> 5) * 16);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa, fw, acc, 0, 0, 0);
        }
    }
    const int n = n0 + wn + (lane & 31);
    if (n >= p.N) return;
    const float ws = p.wsc[n], b = p.bias ? p.bias[n] : 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long m = m0 + wm + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        if (m < p.M) static_cast<elem_t<DT>*>(p.out)[m * p.N + n] = narrow<DT>((float)acc[r] * p.as[m] * ws + b);
    }
}

}  // namespace

extern "C" {

long long ss_seq_int8_linear_ws_ints(long long, int, int) { return 0; }

int ss_seq_int8_linear(const signed char* a, long long lda, const float* a_scale, const signed char* w, long long ldw, const float* w_scale,
                       const float* bias, void* out, long long M, int N, int K, int out_dtype, int*, void* stream)
{
    if (M < 0 || N <= 0 || K <= 0 || K >= 131072 || lda < 0 || ldw < 0) return SS_SEQ_EINVAL;
    if (out_dtype != SS_SEQ_F32 && out_dtype != SS_SEQ_F16 && out_dtype != SS_SEQ_BF16) return SS_SEQ_EINVAL;
    if (M == 0) return SS_SEQ_OK;
    if (!a || !a_scale || !w || !w_scale || !out) return SS_SEQ_EINVAL;
    const MmArgs p{a, w, lda, ldw, a_scale, w_scale, bias, out, M, N, K};
    const bool vec = K % 16 == 0 && lda % 16 == 0 && ldw % 16 == 0 && aligned(a, 16) && aligned(w, 16);
    const long long gm = (M + 63) / 64;
    if (gm > 65535) return SS_SEQ_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)gm);
    auto go = [&](auto DTC) {
        constexpr int DT = DTC.value;
        if (vec) mm64_kernel<DT, true><<<grid, 256, 0, s>>>(p);
        else mm64_kernel<DT, false><<<grid, 256, 0, s>>>(p);
        return launched();
    };
    return out_dtype == SS_SEQ_F32 ? go(std::integral_constant<int, SS_SEQ_F32>())
           : out_dtype == SS_SEQ_F16 ? go(std::integral_constant<int, SS_SEQ_F16>()) : go(std::integral_constant<int, SS_SEQ_BF16>());
}

}  // extern "C"

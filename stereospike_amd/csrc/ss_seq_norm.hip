// ss_seq_norm.hip — add + root-mean-square norm: forward, gradients, and the 8-bit form.
//
//   h = round(x + residual);  n = h * rstd,  rstd = (mean h^2 + eps)^(-1/2);  y = n * weight
//
// One pass: a row's h stays in registers between the sum of squares and the output, so every element is read once and written once (HBM-bound: 4 accesses
// per element with a residual).  TPR threads share a row: a wavefront (no barrier) up to 4 accesses of 16 bytes per lane, then 256 or 1024 threads.  Blocks
// walk rows with a grid stride so that the weight is read once per block.
#include "ss_seq_common.hpp"

namespace {

constexpr int kMaxC = 16384;
constexpr int kBwdBlocks = 1024;        // partials of the weight's gradient: 4 blocks of 4 wavefronts for each of 256 CUs

struct NormArgs {
    const void *x, *r;
    long long xs, rs;
    const float* w;
    void *y, *sum;
    float* rstd;
    signed char* codes;
    float* scales;
    long long rows;
    int C;
    float eps;
};

// The row's value of v over its TPR threads, by every thread.  `red`: one slot per wavefront (unused for TPR = 64).  One barrier: the caller alternates between
// slots, so that those of the last reduction are free again only after the barrier of the next.
template <int TPR, bool MAX, typename V> __device__ __forceinline__ V row_reduce(V v, V* red)
{
    if constexpr (MAX) v = wave_max(v); else v = wave_sum(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v = MAX ? (v > red[i] ? v : red[i]) : v + red[i];
    }
    return v;
}

// fp32 sums of squares leave their range for |h| beyond 1e18 or below 1e-14: those rows are summed again in fp64.  (The same branch for all threads of a row.)
template <int TPR, int NE> __device__ __forceinline__ float rstd_of(float s, const float (&h)[NE], int C, float eps, double* redd, bool& broken)
{
    broken = false;
    if (s < 1e37f && s > 1e-25f) return rsqrtf(s / (float)C + eps);
    double d = 0.;
#pragma unroll
    for (int i = 0; i < NE; ++i) d += (double)h[i] * (double)h[i];
    if constexpr (TPR > 64) __syncthreads();               // the slots' last values have been read
    d = row_reduce<TPR, false>(d, redd);
    if constexpr (TPR > 64) __syncthreads();
    broken = !(d <= 1.7976931348623157e308);              // a NaN or an infinity in the row
    return (float)(1.0 / sqrt(d / (double)C + (double)eps));
}

// HBM-bound; the next row's loads are under way while a row is reduced and written.  (bf16, 16384 x 4096 with a residual: 537 MB in 103 us, 5.2 TB/s; in 8 bits 470 MB
// in 111 us, 4.2 TB/s: the codes' roundings and the exact decision next to a border show.)
template <int DT, int VEC, int TPR, int NV, bool INT8>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_fwd_kernel(const NormArgs p)
{
    constexpr int BLOCK = TPR == 64 ? 256 : TPR, RPB = BLOCK / TPR, NE = NV * VEC;
    __shared__ float redf[2][16], redm[16];
    __shared__ double redd[16];
    typedef Pack<DT, VEC> P;
    const int lane = threadIdx.x % TPR;
    int turn = 0;                                          // which slots: see row_reduce
    float w[NE];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int j = (v * TPR + lane) * VEC + e;
            const float t = p.w[min(j, p.C - 1)];
            w[v * VEC + e] = j < p.C ? t : 0.f;
        }
    bool wild = false;                                     // a weight that is not finite: h * w is not either, whatever h (0 * infinity is a NaN)
    if constexpr (INT8)
#pragma unroll
        for (int i = 0; i < NE; ++i) wild = wild || !(fabsf(w[i]) <= 3.402823466e38f);
    const bool add = p.r != nullptr;
    P px[NV], pr[NV];
    auto load = [&](long long row) {                       // behind the row's end: its last access, counted as zeros below
        const elem_t<DT>* x = static_cast<const elem_t<DT>*>(p.x) + row * p.xs;
        const elem_t<DT>* r = static_cast<const elem_t<DT>*>(p.r) + row * p.rs;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int j = min((v * TPR + lane) * VEC, p.C - VEC);
            px[v] = *reinterpret_cast<const P*>(x + j);
            if (add) pr[v] = *reinterpret_cast<const P*>(r + j);
        }
    };
    const long long stride = (long long)gridDim.x * RPB;
    long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
    if (row < p.rows) load(row);
    for (; row < p.rows; row += stride) {
        float h[NE];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int j = (v * TPR + lane) * VEC;
            const bool in = j < p.C;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (add) px[v].v[e] = narrow<DT>(widen<DT>(px[v].v[e]) + widen<DT>(pr[v].v[e]));         // the sum is kept, and normed, in the input's type
                const float t = widen<DT>(px[v].v[e]);
                h[v * VEC + e] = in ? t : 0.f;
            }
            if (add && in) *reinterpret_cast<P*>(static_cast<elem_t<DT>*>(p.sum) + row * p.C + j) = px[v];
        }
        if (row + stride < p.rows) load(row + stride);     // under way while this row is reduced and written
        float sum = 0.f, most = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            sum = fmaf(h[i], h[i], sum);
            if constexpr (INT8) most = fmaxf(most, fabsf(h[i] * w[i]));
        }
        float top = 0.f;
        if constexpr (INT8) {                              // both over the row with one barrier
            top = wave_max(most);
            if constexpr (TPR > 64) { if ((threadIdx.x & 63) == 0) redm[threadIdx.x >> 6] = top; }
        }
        sum = row_reduce<TPR, false>(sum, redf[turn]);
        if constexpr (INT8 && TPR > 64)
#pragma unroll
            for (int i = 0; i < TPR / 64; ++i) top = fmaxf(top, redm[i]);
        if constexpr (!INT8) turn ^= 1;
        bool broken;
        const float rstd = rstd_of<TPR, NE>(sum, h, p.C, p.eps, redd, broken);
        if constexpr (!INT8) {
            if (p.rstd && lane == 0) p.rstd[row] = rstd;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int j = (v * TPR + lane) * VEC;
                if (j < p.C) {
                    P o;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o.v[e] = narrow<DT>(h[v * VEC + e] * rstd * w[v * VEC + e]);
                    *reinterpret_cast<P*>(static_cast<elem_t<DT>*>(p.y) + row * p.C + j) = o;
                }
            }
        } else {
            // codes = rint(127 u / top), u = h w: rstd cancels.  In fp32 the quotient is off by at most 127 * 4 * 2^-24 = 3e-5; values within 1e-4 of the
            // border of two codes (2 in 10^4) are decided in fp64, where u is exact, so codes do not depend on how the sum of squares was rounded.
            double top64 = 0.;                             // rounding keeps order: the largest u in fp64 is among those whose rounded value is the largest
            if (most == top)
#pragma unroll
                for (int i = 0; i < NE; ++i) top64 = fmax(top64, fabs((double)h[i] * (double)w[i]));
            if (wild) top64 = __builtin_inf();             // (the maxima pass over NaN)
            top64 = row_reduce<TPR, true>(top64, redd);
            broken = broken || !(top64 <= 1.7976931348623157e308);
            const float c = 127.f / top;
            const bool plain = top > 1e-30f && top <= 3.402823466e38f && !broken;        // 127 / top in range
            if (lane == 0) p.scales[row] = broken ? __uint_as_float(0x7FC00000u) : top64 == 0. ? 0.f : (float)(top64 * (double)rstd / 127.0);
            int code[NE];
            bool close = !plain;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float t = h[i] * w[i] * c, q = rintf(t);
                code[i] = (int)q;
                close = close || fabsf(t - q) > 0.4999f;
            }
            if (close)                                     // one branch for the thread's values, not one each
#pragma unroll
                for (int i = 0; i < NE; ++i) code[i] = broken || top64 == 0. ? 0 : (int)rint((double)h[i] * (double)w[i] * 127.0 / top64);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int j = (v * TPR + lane) * VEC;
                if (j < p.C) {
                    struct alignas(VEC) { signed char v[VEC]; } o;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o.v[e] = (signed char)code[v * VEC + e];
                    *reinterpret_cast<decltype(o)*>(p.codes + row * p.C + j) = o;
                }
            }
        }
    }
}

struct NormBwdArgs {
    const void *gy, *gs, *h;
    const float *w, *rstd;
    void* gh;
    float* ws;                              // [gridDim.x][C] partials of the weight's gradient, or NULL
    long long rows;
    int C;
};

// g_h = rstd (w g_y - n mean(w g_y n)) + g_sum in one pass over h, g_y, g_sum; a block keeps its rows' part of the weight's gradient in registers and leaves one row
// of partials, so no atomics.  HBM-bound (29920 x 512, bf16, both gradients: 123 MB in 28 us, 4.4 TB/s).
template <int DT, int VEC, int TPR, int NV>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void rms_bwd_kernel(const NormBwdArgs p)
{
    constexpr int BLOCK = TPR == 64 ? 256 : TPR, RPB = BLOCK / TPR, NE = NV * VEC;
    __shared__ float redf[2][16];
    int turn = 0;
    __shared__ float part[TPR == 64 ? 3 * 64 * NE : 1];
    typedef Pack<DT, VEC> P;
    const int lane = threadIdx.x % TPR;
    float w[NE], gw[NE];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int j = (v * TPR + lane) * VEC + e;
            const float t = p.w[min(j, p.C - 1)];
            w[v * VEC + e] = j < p.C ? t : 0.f;
            gw[v * VEC + e] = 0.f;
        }
    for (long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR; row < p.rows; row += (long long)gridDim.x * RPB) {
        P pg[NV], ph[NV], ps[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {                     // behind the row's end: its last access, counted as zeros
            const long long j = row * p.C + min((v * TPR + lane) * VEC, p.C - VEC);
            ph[v] = *reinterpret_cast<const P*>(static_cast<const elem_t<DT>*>(p.h) + j);
            if (p.gy) pg[v] = *reinterpret_cast<const P*>(static_cast<const elem_t<DT>*>(p.gy) + j);
            if (p.gs) ps[v] = *reinterpret_cast<const P*>(static_cast<const elem_t<DT>*>(p.gs) + j);
        }
        const float rstd = p.rstd[row];
        float n[NE], g[NE], dot = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const bool in = (v * TPR + lane) * VEC < p.C;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = v * VEC + e;
                n[i] = in ? widen<DT>(ph[v].v[e]) * rstd : 0.f;
                g[i] = in && p.gy ? widen<DT>(pg[v].v[e]) : 0.f;
                gw[i] = fmaf(g[i], n[i], gw[i]);
                g[i] *= w[i];
                dot = fmaf(g[i], n[i], dot);
            }
        }
        dot = row_reduce<TPR, false>(dot, redf[turn]) / (float)p.C;
        turn ^= 1;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int j = (v * TPR + lane) * VEC;
            if (j < p.C) {
                P o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = v * VEC + e;
                    float d = rstd * (g[i] - n[i] * dot);
                    if (p.gs) d += widen<DT>(ps[v].v[e]);
                    o.v[e] = narrow<DT>(d);
                }
                *reinterpret_cast<P*>(static_cast<elem_t<DT>*>(p.gh) + row * p.C + j) = o;
            }
        }
    }
    if (!p.ws) return;
    if constexpr (TPR == 64) {                             // the block's four rows share their columns: one partial per block
        const int wv = threadIdx.x >> 6;
        if (wv)
#pragma unroll
            for (int i = 0; i < NE; ++i) part[((wv - 1) * NE + i) * 64 + lane] = gw[i];
        __syncthreads();
        if (wv) return;
#pragma unroll
        for (int i = 0; i < NE; ++i) gw[i] += part[i * 64 + lane] + part[(NE + i) * 64 + lane] + part[(2 * NE + i) * 64 + lane];
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int j = (v * TPR + lane) * VEC + e;
            if (j < p.C) p.ws[(long long)blockIdx.x * p.C + j] = gw[v * VEC + e];
        }
}

// g_w[j] = sum of the blocks' partials, in a fixed order: 16 columns x 64 slices per block, 16 partials of a slice in flight, so that it is one latency long
// (1024 partials of 512 columns: 3.9 us)
__global__ __launch_bounds__(1024) void rms_gw_kernel(const float* __restrict__ ws, float* __restrict__ gw, int P, int C)
{
    __shared__ float red[64][17];
    const int cx = threadIdx.x & 15, sl = threadIdx.x >> 4, j = blockIdx.x * 16 + cx;
    float s = 0.f;
    if (j < C) {
        int i = sl;
        for (; i + 15 * 64 < P; i += 16 * 64) {
            float v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) v[u] = ws[(long long)(i + 64 * u) * C + j];
#pragma unroll
            for (int u = 0; u < 16; ++u) s += v[u];
        }
        for (; i < P; i += 64) s += ws[(long long)i * C + j];
    }
    red[sl][cx] = s;
    __syncthreads();
    for (int k = 32; k; k >>= 1) {
        if (sl < k) red[sl][cx] += red[sl + k][cx];
        __syncthreads();
    }
    if (sl == 0 && j < C) gw[j] = red[0][cx];
}

// codes -> values, a wavefront a row, four accesses a lane.  HBM-bound (16384 x 4096 to bf16: 201 MB in 34 us, 5.9 TB/s).
template <int DT, int VEC> __global__ __launch_bounds__(256) void dequant_kernel(const signed char* __restrict__ q, const float* __restrict__ sc,
                                                                                 elem_t<DT>* __restrict__ out, long long rows, int C)
{
    const int cv = (C + VEC - 1) / VEC;                    // C % VEC == 0 where VEC > 1
    for (long long row = (long long)blockIdx.y * 4 + (threadIdx.x >> 6); row < rows; row += (long long)gridDim.y * 4) {
        const float s = sc[row];
        for (int v = blockIdx.x * 64 + (threadIdx.x & 63); v < cv; v += gridDim.x * 64) {
            struct alignas(VEC) Q { signed char v[VEC]; };
            const Q a = *reinterpret_cast<const Q*>(q + row * C + (long long)v * VEC);
            Pack<DT, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o.v[e] = narrow<DT>((float)a.v[e] * s);
            *reinterpret_cast<Pack<DT, VEC>*>(out + row * C + (long long)v * VEC) = o;
        }
    }
}

// Threads of a row and accesses per thread: 16 values a thread at most (more spill).  A wavefront up to 1024 values, where its reductions need no barrier; then
// 256 threads up to 4096, then 1024.  (bf16, with a residual, norm / norm in 8 bits: 16384 x 1024 by a wavefront 26.6 / 33 us, by 256 threads 25.1 / 47; 16384 x
// 4096 by 256 threads 103 / 115 us, by 1024 99 / 235.  More threads for few rows gain nothing: 64 x 4096, fp32: 4.8 / 5.5 us either way.)
template <int VEC, typename F> int with_shape(int C, F&& f)
{
    constexpr int N1 = 1, N2 = VEC == 1 ? 4 : 2, N3 = 16 / VEC;
    const int acc = (C + VEC - 1) / VEC;
    auto by = [&](auto TPR) {
        if (acc <= N1 * TPR.value) return f(TPR, std::integral_constant<int, N1>());
        if (N2 < N3 && acc <= N2 * TPR.value) return f(TPR, std::integral_constant<int, N2>());
        return f(TPR, std::integral_constant<int, N3>());
    };
    if (C <= 1024) return by(std::integral_constant<int, 64>());
    if (C <= 4096) return by(std::integral_constant<int, 256>());
    return by(std::integral_constant<int, 1024>());
}

template <int DT, bool INT8> int fwd_dt(const NormArgs& p, hipStream_t s)
{
    constexpr int V = DT == SS_SEQ_F32 ? 4 : 8;
    const void* out = INT8 ? (const void*)p.codes : p.y;
    const bool vec = p.C % V == 0 && p.xs % V == 0 && aligned(p.x, 16) && (!p.r || (p.rs % V == 0 && aligned(p.r, 16) && aligned(p.sum, 16))) && aligned(out, INT8 ? V : 16);
    auto go = [&](auto VC) {
        return with_shape<VC.value>(p.C, [&](auto TPR, auto NV) {
            constexpr int block = TPR.value == 64 ? 256 : TPR.value, rpb = block / TPR.value;
            const long long want = (p.rows + rpb - 1) / rpb, cap = 256 * (2048 / block);          // 32 wavefronts for each of 256 CUs
            rms_fwd_kernel<DT, VC.value, TPR.value, NV.value, INT8><<<(unsigned)(want < cap ? want : cap), block, 0, s>>>(p);
            return launched();
        });
    };
    return vec ? go(std::integral_constant<int, V>()) : go(std::integral_constant<int, 1>());
}

template <int DT> int bwd_dt(const NormBwdArgs& p, float* gw, hipStream_t s)
{
    constexpr int V = DT == SS_SEQ_F32 ? 4 : 8;
    const bool vec = p.C % V == 0 && aligned(p.gy, 16) && aligned(p.gs, 16) && aligned(p.h, 16) && aligned(p.gh, 16);
    auto go = [&](auto VC) {
        return with_shape<VC.value>(p.C, [&](auto TPR, auto NV) {
            constexpr int block = TPR.value == 64 ? 256 : TPR.value, rpb = block / TPR.value;
            const long long want = (p.rows + rpb - 1) / rpb;
            const unsigned grid = (unsigned)(want < kBwdBlocks ? want : kBwdBlocks);
            rms_bwd_kernel<DT, VC.value, TPR.value, NV.value><<<grid, block, 0, s>>>(p);
            if (int rc = launched()) return rc;
            if (gw) {
                rms_gw_kernel<<<(p.C + 15) / 16, 1024, 0, s>>>(p.ws, gw, (int)grid, p.C);
                return launched();
            }
            return SS_SEQ_OK;
        });
    };
    return vec ? go(std::integral_constant<int, V>()) : go(std::integral_constant<int, 1>());
}

bool sizes_ok(long long rows, int C, int dtype) { return rows >= 0 && C > 0 && C <= kMaxC && (dtype == SS_SEQ_F32 || dtype == SS_SEQ_F16 || dtype == SS_SEQ_BF16); }

}  // namespace

extern "C" {

int ss_seq_abi_version(void) { return SS_SEQ_ABI_VERSION; }

int ss_seq_rms_norm_fwd(const void* x, long long x_stride, const void* residual, long long r_stride, const float* weight, void* y, void* sum, float* rstd,
                        long long rows, int C, float eps, int dtype, void* stream)
{
    if (!sizes_ok(rows, C, dtype) || !(eps >= 0.f)) return SS_SEQ_EINVAL;
    if (rows == 0) return SS_SEQ_OK;
    if (!x || !weight || !y || (residual && !sum)) return SS_SEQ_EINVAL;
    const NormArgs p{x, residual, x_stride, r_stride, weight, y, sum, rstd, nullptr, nullptr, rows, C, eps};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SS_SEQ_F32 ? fwd_dt<SS_SEQ_F32, false>(p, s) : dtype == SS_SEQ_F16 ? fwd_dt<SS_SEQ_F16, false>(p, s) : fwd_dt<SS_SEQ_BF16, false>(p, s);
}

int ss_seq_rms_norm_int8(const void* x, long long x_stride, const void* residual, long long r_stride, const float* weight, signed char* codes, float* scales,
                         void* sum, long long rows, int C, float eps, int dtype, void* stream)
{
    if (!sizes_ok(rows, C, dtype) || !(eps >= 0.f)) return SS_SEQ_EINVAL;
    if (rows == 0) return SS_SEQ_OK;
    if (!x || !weight || !codes || !scales || (residual && !sum)) return SS_SEQ_EINVAL;
    const NormArgs p{x, residual, x_stride, r_stride, weight, nullptr, sum, nullptr, codes, scales, rows, C, eps};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SS_SEQ_F32 ? fwd_dt<SS_SEQ_F32, true>(p, s) : dtype == SS_SEQ_F16 ? fwd_dt<SS_SEQ_F16, true>(p, s) : fwd_dt<SS_SEQ_BF16, true>(p, s);
}

long long ss_seq_rms_norm_ws_floats(long long rows, int C, int dtype)
{
    if (!sizes_ok(rows, C, dtype)) return 0;
    return (rows < kBwdBlocks ? rows : kBwdBlocks) * (long long)C;
}

int ss_seq_rms_norm_bwd(const void* g_y, const void* g_sum, const void* h, const float* weight, const float* rstd, void* g_h, float* g_w, float* ws,
                        long long rows, int C, int dtype, void* stream)
{
    if (!sizes_ok(rows, C, dtype) || rows == 0 || !h || !weight || !rstd || !g_h || (g_w && !ws)) return SS_SEQ_EINVAL;
    const NormBwdArgs p{g_y, g_sum, h, weight, rstd, g_h, g_w ? ws : nullptr, rows, C};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == SS_SEQ_F32 ? bwd_dt<SS_SEQ_F32>(p, g_w, s) : dtype == SS_SEQ_F16 ? bwd_dt<SS_SEQ_F16>(p, g_w, s) : bwd_dt<SS_SEQ_BF16>(p, g_w, s);
}

int ss_seq_dequant_int8(const signed char* codes, const float* scales, void* out, long long rows, int C, int dtype, void* stream)
{
    if (rows < 0 || C <= 0 || (dtype != SS_SEQ_F32 && dtype != SS_SEQ_F16 && dtype != SS_SEQ_BF16)) return SS_SEQ_EINVAL;
    if (rows == 0) return SS_SEQ_OK;
    if (!codes || !scales || !out) return SS_SEQ_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool vec = C % 8 == 0 && aligned(codes, 8) && aligned(out, 32);
    const int cv = vec ? C / 8 : C;
    const int gx = (cv + 255) / 256;                       // four accesses per lane
    const dim3 grid((unsigned)gx, (unsigned)(rows < 65536ll * 4 ? (rows + 3) / 4 : 65535));
    auto go = [&](auto DTC) {
        constexpr int DT = DTC.value;
        elem_t<DT>* o = static_cast<elem_t<DT>*>(out);
        if (vec) dequant_kernel<DT, 8><<<grid, 256, 0, s>>>(codes, scales, o, rows, C);
        else dequant_kernel<DT, 1><<<grid, 256, 0, s>>>(codes, scales, o, rows, C);
        return launched();
    };
    return dtype == SS_SEQ_F32 ? go(std::integral_constant<int, SS_SEQ_F32>()) : dtype == SS_SEQ_F16 ? go(std::integral_constant<int, SS_SEQ_F16>())
                                                                                                     : go(std::integral_constant<int, SS_SEQ_BF16>());
}

}  // extern "C"

// ss_seq_attention.hpp — leaky attention: a matrix-valued leaky integrator per head, read by a query.
//
//   S_i = lambda S_{i-1} + b_scale b_i c_i^T,   out_i = o_scale a_i^T S_i,   lambda = exp(log_decay) of the head
//
// The forward pass and the three token gradients are this one map with other operands, forwards or backwards in time (ss_sequence.h).  One unit per element
// type instantiates it (ss_seq_attention_{f32,f16,bf16}.hip).
#pragma once
#include "ss_seq_common.hpp"

// (in ss_seq_attention.hip: checks and dispatch by element type)
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
    int out_f32;
};

struct LeakyView {
    const void* p;
    long long t, b, h;                       // strides
    int group;                               // query heads that read a head of it
};
struct LeakyBwdArgs {
    int T, B, H, Hk, Dk, Dv;
    float scale;
    LeakyView q, k, v, g;
    void *g_q, *g_k, *g_v;
    const float* log_decay;
    const int* lengths;
    const float *s_in, *g_last;
    float* g_s;
    const float* states;
    float* ws;
};

long long ss_seq_leaky_bwd_ws_f32(const LeakyBwdArgs&);
long long ss_seq_leaky_bwd_ws_f16(const LeakyBwdArgs&);
long long ss_seq_leaky_bwd_ws_bf16(const LeakyBwdArgs&);
int ss_seq_leaky_bwd_f32(const LeakyBwdArgs&, hipStream_t);
int ss_seq_leaky_bwd_f16(const LeakyBwdArgs&, hipStream_t);
int ss_seq_leaky_bwd_bf16(const LeakyBwdArgs&, hipStream_t);
long long ss_seq_leaky_ws_f32(const LeakyArgs&);
long long ss_seq_leaky_ws_f16(const LeakyArgs&);
long long ss_seq_leaky_ws_bf16(const LeakyArgs&);
int ss_seq_leaky_f32(const LeakyArgs&, float* ws, hipStream_t);
int ss_seq_leaky_f16(const LeakyArgs&, float* ws, hipStream_t);
int ss_seq_leaky_bf16(const LeakyArgs&, float* ws, hipStream_t);

namespace {


// One step, S = lambda S + b c^T and out = a^T S (in reverse the leak comes after: s_out = lambda S).  HBM-bound: the state is read, updated and written once,
// 8 bytes for each of its values.  A workgroup has 64 columns of one head's state, thread (g, x) rows g + 16 r of columns 4 x .. 4 x + 3, all R of them in
// flight at once.  (512 streams of 16 heads of 128 x 128, bf16: 1.08 GB in 213 us, a large copy's rate; one stream of 8 heads of 64 x 64: 4.2 us,
// little over an empty launch.)  V4: the state's rows take 16-byte accesses.
template <int DT, int ODT, int R, bool V4> __global__ __launch_bounds__(256) void leaky_step_kernel(const LeakyArgs p)
{
    __shared__ float sa[256], sb[256], red[4][64];
    const int tid = threadIdx.x, x = tid & 15, g = tid >> 4;
    const int bh = blockIdx.y, b = bh / p.H, h = bh - b * p.H, j0 = blockIdx.x * 64 + 4 * x;
    const bool valid = !p.lengths || p.lengths[b] > 0;     // no step: the state as it is, an output of zeros
    f32x4 S[R];
    // (rows and columns outside are read at the nearest inside: a branch per load would end the loads' flight together)
    if (p.s_in) {
        const float* s_in = p.s_in + (long long)bh * p.DA * p.DC;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float* row = s_in + min(g + 16 * r, p.DA - 1) * p.s_in_row;
            if constexpr (V4) S[r] = *reinterpret_cast<const f32x4*>(row + min(j0, p.DC - 4));
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) S[r][e] = row[min(j0 + e, p.DC - 1) * p.s_in_col];
        }
    } else
#pragma unroll
        for (int r = 0; r < R; ++r) S[r] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const float lam = expf(p.log_decay[h]), before = p.reverse || !valid ? 1.f : lam, after = p.reverse && valid ? lam : 1.f;
    if (tid < p.DA) {
        sa[tid] = valid ? widen<DT>(static_cast<const elem_t<DT>*>(p.a)[b * p.a_b + (h / p.a_group) * p.a_h + tid]) * p.o_scale : 0.f;
        sb[tid] = valid ? widen<DT>(static_cast<const elem_t<DT>*>(p.b)[b * p.b_b + (h / p.b_group) * p.b_h + tid]) * p.b_scale : 0.f;
    }
    f32x4 c = {0.f, 0.f, 0.f, 0.f}, o = {0.f, 0.f, 0.f, 0.f};
    if (valid)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j0 + e < p.DC) c[e] = widen<DT>(static_cast<const elem_t<DT>*>(p.c)[b * p.c_b + (h / p.c_group) * p.c_h + j0 + e]);
    __syncthreads();
    float* s_out = p.s_out ? p.s_out + (long long)bh * p.DA * p.DC : nullptr;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = g + 16 * r;
        if (j0 < p.DC && row < p.DA) {
            const f32x4 s = S[r] * before + sb[row] * c;
            o += sa[row] * s;
            if constexpr (V4) { if (s_out) *reinterpret_cast<f32x4*>(s_out + row * p.s_out_row + j0) = s * after; }
            else if (s_out)
#pragma unroll
                for (int e = 0; e < 4; ++e) if (j0 + e < p.DC) s_out[row * p.s_out_row + (j0 + e) * p.s_out_col] = s[e] * after;
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
        static_cast<elem_t<ODT>*>(p.out)[b * p.o_b + h * p.o_h + blockIdx.x * 64 + tid] =
            valid ? narrow<ODT>(red[0][tid] + red[1][tid] + red[2][tid] + red[3][tid]) : elem_t<ODT>(0);
}

template <int DT, int ODT> int step(const LeakyArgs& p, hipStream_t s)
{
    const bool v4 = p.DC % 4 == 0 && (!p.s_in || (p.s_in_col == 1 && p.s_in_row % 4 == 0 && aligned(p.s_in, 16))) &&
                    (!p.s_out || (p.s_out_col == 1 && p.s_out_row % 4 == 0 && aligned(p.s_out, 16)));
    const dim3 grid((unsigned)((p.DC + 63) / 64), (unsigned)(p.B * p.H));
    auto go = [&](auto R) {
        if (v4) leaky_step_kernel<DT, ODT, R.value, true><<<grid, 256, 0, s>>>(p);
        else leaky_step_kernel<DT, ODT, R.value, false><<<grid, 256, 0, s>>>(p);
        return launched();
    };
    if (p.DA <= 64) return go(std::integral_constant<int, 4>());
    if (p.DA <= 128) return go(std::integral_constant<int, 8>());
    return go(std::integral_constant<int, 16>());
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// The tile form.  A chunk of CH steps is four products, with W the state as the NEXT step would see it (already leaked once):
//
//   P_ij  = a_i . b_j * lambda^(i-j)  (j <= i)             (1)
//   out_i = sum_j P_ij c_j                                 (2)
//         + lambda^i a_i W                                 (3)
//   W    <- lambda^CH W + sum_j lambda^(CH-j) b_j c_j^T    (4)
//
// A workgroup owns a block of columns of one head's state for one SEGMENT of the steps, a wavefront 16 or 32 of them with all DA rows of W in its registers.
// Several segments: a first pass computes what each adds to the state (STATE: (4) alone, of b and c), a scan or the second pass joins them, the second pass
// computes the outputs.  That reads b and c twice, which costs less than the steps one after the other: a head's time axis is cut until the card is filled.
// Products are taken so that accumulators ARE the next product's operand: a 16 x 16 accumulator gives lane l rows 4 (l / 16) .. + 3 of column l % 16; two
// of them, one above the other, are the 8 contraction values of a 16x16x32 operand in the order {4g .. 4g+3, 16+4g .. 16+4g+3} (four 16x16x4 operands in
// fp32).  a and b are staged in LDS in that order, so W never leaves the registers; P is shared between the wavefronts through LDS in operand order.
// Out comes out transposed: a lane stores four consecutive columns of one step.
//
// Rounding (16-bit operands): W has two terms of the operands' type in (3) and P two in (2), the rounded value and what that leaves, so the output's own rounding is
// the only one that shows (with one term of W the error against 64 bits was 1.35 - 1.4 times that of outputs rounded once; the second costs 2 - 9 %: T = 4096,
// 64 heads of 128 x 128, bf16: 122 -> 132 us).  (4) splits lambda^(CH-j) c_j into three bf16 or two fp16 terms (24 and 23 bits), so the state keeps fp32 accuracy.
// fp16's range is too short for P, W and c's terms: they are scaled by powers of two, taken from the largest value of a tile of P, of a wavefront's columns of W,
// of a column of c.  fp32 operands run on the fp32 matrix instructions.
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;

// log2 of lambda; minus infinity becomes a number, so that lambda^0 is 1
__device__ __forceinline__ float log2_decay(float log_decay) { return (log_decay < -1e30f ? -1e30f : log_decay) * 1.44269504088896341f; }

struct LeakyPlan {
    int nseg, seg;                           // segments and their steps (a multiple of the chunk)
    int ncb;                                 // column blocks
    int fold;                                // the output pass joins the segments' states itself (no scan launch)
    // the states between segments, as the state pass of this map or of the map with b and c exchanged (trans) left them: per head and column block of `dcb`
    // columns, nseg - 1 matrices in accumulator order (wavefronts of 16 nt columns, `ka` row tiles)
    int trans, ka, nt, dcb, sncb;
};
struct LeakyMap {
    LeakyArgs p;
    LeakyPlan plan;
    float* ws;                               // the states between segments
    int vec, vec_out;                        // 16-byte accesses to the operands, to the output
};
// the maps of one launch: `per` workgroups each
struct LeakyMaps {
    LeakyMap m[3];
    unsigned per;
};

// the 16 x 16 tile of rows 16 rt, columns 16 ct of a state left in accumulator order: its first element
__device__ __forceinline__ long long state_tile(const LeakyPlan& p, long long bh, int s, int rt, int ct)
{
    const int cb = 16 * ct / p.dcb, t = ct - cb * (p.dcb / 16), w = t / p.nt, n = t - w * p.nt;
    return ((bh * p.sncb + cb) * (p.nseg - 1) + s) * (16ll * p.ka * p.dcb) + ((w * p.ka + rt) * p.nt + n) * 256;
}
// this lane's four values of the tile (rows 4 g .. + 3 of column l16) of the state that entered segment s + 1, or of its transpose
__device__ __forceinline__ f32x4 state_read(const LeakyPlan& p, const float* __restrict__ ws, long long bh, int s, int rt, int ct, int lane)
{
    if (!p.trans) return *reinterpret_cast<const f32x4*>(ws + state_tile(p, bh, s, rt, ct) + lane * 4);
    const float* at = ws + state_tile(p, bh, s, ct, rt) + ((lane & 15) >> 2) * 64 + (lane >> 4) * 16 + (lane & 3);
    return (f32x4){at[0], at[4], at[8], at[12]};
}

__device__ __forceinline__ unsigned pack_hi16(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }
__device__ __forceinline__ float top16(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
__device__ __forceinline__ bf16x8 mk8(unsigned a, unsigned b, unsigned c, unsigned d)
{
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(bf16x8, (u32x4){a, b, c, d});
}
__device__ __forceinline__ unsigned round_pk(float lo, float hi)
{
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, (bf16x2){(__bf16)lo, (__bf16)hi});
}

// The tile form on fp32 operands: the 16x16x4 fp32 matrix instructions, a workgroup of WV (4 or 8) wavefronts with 16 columns each, two workgroups on a CU.
// Bound by those instructions (157 TFLOP/s) and, where streams are ragged, by the longest one's chunks in a row (5 us each with 128 columns, 3.5 of them the
// instructions' own); the 16-row tiles behind DA and the wavefronts behind DC are left out (training, 48 heads of 80 and 96, 777 steps: 218 -> 196 us).  Blocks of
// 64 columns with twice the workgroups took 203.
template <int DA, int WV, bool STATE>
__global__ __launch_bounds__(64 * WV, DA == 64 || (DA == 128 && WV == 8) ? 4 : 2) void leaky_chunk_kernel(const LeakyMaps maps)
{
    constexpr int CH = 32, NTH = 64 * WV, DCB = 16 * WV, KA = DA / 16;
    constexpr int SA = DA + 4, SC = DCB + 4;                             // LDS rows 16 bytes longer than a power of two
    constexpr int GA = CH * DA / 4 / NTH, GC = CH * DCB / 4 / NTH;       // 16-byte granules of a thread
    __shared__ __attribute__((aligned(16))) float sa[STATE ? 8 : CH * SA];
    __shared__ __attribute__((aligned(16))) float sb[CH * SA];
    __shared__ __attribute__((aligned(16))) float sc[CH * SC];
    __shared__ __attribute__((aligned(16))) float sp[STATE ? 8 : 3 * 64 * 4];                // P: the tiles (0, 0), (1, 0), (1, 1)
    __shared__ __attribute__((aligned(16))) float rw[CH];                // lambda^(e - j) b_scale of the chunk's steps

    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const unsigned which = blockIdx.x / maps.per, block = blockIdx.x - which * maps.per;
    const LeakyMap& map = maps.m[which];
    const LeakyArgs& p = map.p;
    const LeakyPlan& plan = map.plan;
    float* __restrict__ ws = map.ws;
    const int cb = block % plan.ncb, rest = block / plan.ncb;
    const int nst = STATE ? plan.nseg - 1 : plan.nseg, seg = rest % nst, bh = rest / nst, b = bh / p.H, h = bh - b * p.H;
    int n = p.T;
    if (p.lengths) { n = p.lengths[b]; n = n < 0 ? 0 : n > p.T ? p.T : n; }
    const int start = seg * plan.seg, stop = n < start + plan.seg ? n : start + plan.seg;      // this segment's valid steps
    if (STATE && n <= start + plan.seg) return;                          // no later segment reads this one's state
    const float gl = log2_decay(p.log_decay[h]);
    const int c0 = cb * DCB, col0 = c0 + wv * 16, ka = (p.DA + 15) / 16;
    const bool on = col0 < p.DC;                                         // this wavefront has columns
    const float* pa = static_cast<const float*>(p.a) + b * p.a_b + (h / p.a_group) * p.a_h;
    const float* pb = static_cast<const float*>(p.b) + b * p.b_b + (h / p.b_group) * p.b_h;
    const float* pc = static_cast<const float*>(p.c) + b * p.c_b + (h / p.c_group) * p.c_h + c0;
    const int dc = p.DC - c0 < DCB ? p.DC - c0 : DCB;

    // ---- the state that enters the segment
    f32x4 W[KA];
#pragma unroll
    for (int kt = 0; kt < KA; ++kt) W[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (seg == 0) {
        if (p.s_in) {
            const float* s_in = p.s_in + (long long)bh * p.DA * p.DC;
            const float first = exp2f(gl * (float)((p.reverse || n == 0 ? 0 : 1) + (STATE ? plan.seg : 0)));
#pragma unroll
            for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * kt + 4 * g + r, j = col0 + l16;
                    const bool in = i < p.DA && j < p.DC;
                    const float v = s_in[in ? i * p.s_in_row + j * p.s_in_col : 0];
                    W[kt][r] = in ? v * first : 0.f;
                }
        }
    } else if (!STATE && start < n && on) {
        const float leak = exp2f(gl * (float)plan.seg);
        for (int s = plan.fold ? 0 : seg - 1; s < seg; ++s)
#pragma unroll
            for (int kt = 0; kt < KA; ++kt)
                if (kt < ka) W[kt] = W[kt] * leak + state_read(plan, ws, bh, s, kt, col0 / 16, lane);
    }

    // ---- staging: global -> registers (one chunk ahead) -> LDS
    f32x4 ra[STATE ? 1 : GA], rb[GA], rc[GC];
    auto fetch = [&](f32x4* dst, const float* base, long long st, int i0, int d, auto SPRC) {
        constexpr int SPR = SPRC.value;                                  // granules of a row
#pragma unroll
        for (int u = 0; u < CH * SPR / NTH; ++u) {
            const int x = tid + NTH * u, q = x % SPR, i = i0 + x / SPR;
            const float* src = base + (long long)(p.reverse ? n - 1 - i : i) * st + 4 * q;
            dst[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (i < stop && 4 * q < d) {
                if (map.vec) dst[u] = *reinterpret_cast<const f32x4*>(src);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (4 * q + e < d) dst[u][e] = src[e];
            }
        }
    };
    auto put = [&](float* dst, const f32x4* v, int stride, auto SPRC) {
        constexpr int SPR = SPRC.value;
#pragma unroll
        for (int u = 0; u < CH * SPR / NTH; ++u) {
            const int x = tid + NTH * u;
            *reinterpret_cast<f32x4*>(dst + x / SPR * stride + 4 * (x % SPR)) = v[u];
        }
    };
    typedef std::integral_constant<int, DA / 4> QA;
    typedef std::integral_constant<int, DCB / 4> QC;
    auto load = [&](int i0) {
        if constexpr (!STATE) fetch(ra, pa, p.a_t, i0, p.DA, QA());
        fetch(rb, pb, p.b_t, i0, p.DA, QA());
        fetch(rc, pc, p.c_t, i0, dc, QC());
    };
    auto store = [&](int i, int col, const f32x4& v) {                   // four columns of step i
        if (i >= p.T || col >= p.DC) return;
        const bool live = i < n;
        float* q = static_cast<float*>(p.out) + b * p.o_b + h * p.o_h + (live && p.reverse ? n - 1 - i : i) * p.o_t + col;
        const f32x4 o = live ? v : (f32x4){0.f, 0.f, 0.f, 0.f};
        if (map.vec_out) *reinterpret_cast<f32x4*>(q) = o;
        else
#pragma unroll
            for (int e = 0; e < 4; ++e) if (col + e < p.DC) q[e] = o[e];
    };

    float row_scale[2];                                                  // lambda^i o_scale of this lane's steps
#pragma unroll
    for (int it = 0; it < 2; ++it) row_scale[it] = exp2f(gl * (float)(16 * it + l16)) * p.o_scale;
    if (tid < CH) rw[tid] = exp2f(gl * (float)(CH - tid)) * p.b_scale;

    load(start);
    int i0 = start;
    for (; i0 < stop; i0 += CH) {
        const int cnt = stop - i0 < CH ? stop - i0 : CH;
        // the last chunk of the stream leaves the state as it is after its last step (forward) or leaked once more (reverse)
        const int e = i0 + cnt == n && !p.reverse ? cnt - 1 : cnt;
        __syncthreads();                                                 // the last chunk has been read
        if constexpr (!STATE) put(sa, ra, SA, QA());
        put(sb, rb, SA, QA());
        put(sc, rc, SC, QC());
        if (e != CH && tid < CH) rw[tid] = exp2f(gl * (float)(e > tid ? e - tid : 0)) * p.b_scale;
        __syncthreads();
        if (i0 + CH < stop) load(i0 + CH);

        f32x4 acc[2];
        if constexpr (!STATE) {
            // (1) wavefronts 0 .. 2: a tile of P each
            if (wv < 3) {
                const int it = (wv + 1) >> 1, jt = wv >> 1;
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
                const float *qa = sa + (16 * it + l16) * SA + 4 * g, *qb = sb + (16 * jt + l16) * SA + 4 * g;
#pragma unroll
                for (int k = 0; k < KA; ++k)
                    if (k < ka) {
                        const f32x4 fb = *reinterpret_cast<const f32x4*>(qb + 16 * k), fa = *reinterpret_cast<const f32x4*>(qa + 16 * k);
#pragma unroll
                        for (int r = 0; r < 4; ++r) s = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[r], fa[r], s, 0, 0, 0);
                    }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * (it - jt) + l16 - 4 * g - r;      // i - j
                    s[r] = d < 0 ? 0.f : s[r] * (exp2f(gl * (float)d) * p.b_scale * p.o_scale);
                }
                *reinterpret_cast<f32x4*>(sp + (wv * 64 + lane) * 4) = s;
            }
            // (3)
            acc[0] = acc[1] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (on) {
#pragma unroll
                for (int k = 0; k < KA; ++k)
                    if (k < ka) {
                        const float* q = sa + l16 * SA + 16 * k + 4 * g;
                        const f32x4 f0 = *reinterpret_cast<const f32x4*>(q), f1 = *reinterpret_cast<const f32x4*>(q + 16 * SA);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(W[k][r], f0[r], acc[0], 0, 0, 0);
                            acc[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(W[k][r], f1[r], acc[1], 0, 0, 0);
                        }
                    }
#pragma unroll
                for (int it = 0; it < 2; ++it) acc[it] *= row_scale[it];
            }
            __syncthreads();                                             // P is there
        }
        if (!on) continue;
        // (2) and (4) share the wavefront's columns of c
        // (the state pass weighs by the distance to the segment's end, so W only accumulates)
        const float tail = STATE ? exp2f(gl * (float)(stop - CH - i0)) : 1.f;
        if constexpr (!STATE) {
            const float keep = exp2f(gl * (float)e);
#pragma unroll
            for (int kt = 0; kt < KA; ++kt) W[kt] *= keep;
        }
        bool wild = false;
        float fc[2][4];
#pragma unroll
        for (int jt = 0; jt < 2; ++jt) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(rw + 16 * jt + 4 * g) * tail;
            float fin[4];                                                // without what is not finite: 0 * NaN would reach steps before it
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                fc[jt][r] = sc[(16 * jt + 4 * g + r) * SC + wv * 16 + l16];
                const bool odd = !(fabsf(fc[jt][r]) < __builtin_inff());
                fin[r] = odd ? 0.f : fc[jt][r];
                wild = wild || odd;
                fc[jt][r] *= w[r];
            }
            if constexpr (!STATE) {
#pragma unroll
                for (int it = jt; it < 2; ++it) {
                    const f32x4 fp = *reinterpret_cast<const f32x4*>(sp + ((it + jt) * 64 + lane) * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[it] = __builtin_amdgcn_mfma_f32_16x16x4f32(fin[r], fp[r], acc[it], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int kt = 0; kt < KA; ++kt)
            if (kt < ka) {
#pragma unroll
                for (int jt = 0; jt < 2; ++jt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) W[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(sb[(16 * jt + 4 * g + r) * SA + 16 * kt + l16], fc[jt][r], W[kt], 0, 0, 0);
            }
        if constexpr (!STATE) {
            if (__any(wild))                                             // rare: those terms one by one, where j <= i
#pragma unroll 1
                for (int j = 0; j < CH; ++j)
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        if (j > 16 * it + l16) continue;
                        const float pij = sp[((it + (j >> 4)) * 64 + 16 * (j >> 2 & 3) + l16) * 4 + (j & 3)];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float c = sc[j * SC + wv * 16 + 4 * g + r];
                            if (!(fabsf(c) < __builtin_inff())) acc[it][r] += pij * c;
                        }
                    }
#pragma unroll
            for (int it = 0; it < 2; ++it) store(i0 + 16 * it + l16, col0 + 4 * g, acc[it]);
        }
    }

    if constexpr (STATE) {
        float* mine = ws + (((long long)bh * plan.ncb + cb) * (plan.nseg - 1) + seg) * ((long long)DA * DCB) + wv * KA * 256 + lane * 4;
#pragma unroll
        for (int kt = 0; kt < KA; ++kt) *reinterpret_cast<f32x4*>(mine + kt * 256) = W[kt];
    } else {
        // steps of the segment behind the stream's last: zeros (the loop above has written its own chunks to their end)
        const int end = start + plan.seg < p.T ? start + plan.seg : p.T;
        for (; i0 < end; i0 += CH)
#pragma unroll
            for (int it = 0; it < 2; ++it) store(i0 + 16 * it + l16, col0 + 4 * g, (f32x4){0.f, 0.f, 0.f, 0.f});
        if (p.s_out && ((start < n && n <= start + plan.seg) || (n == 0 && seg == 0))) {
            float* s_out = p.s_out + (long long)bh * p.DA * p.DC;
#pragma unroll
            for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * kt + 4 * g + r, j = col0 + l16;
                    if (i < p.DA && j < p.DC) s_out[i * p.s_out_row + j * p.s_out_col] = W[kt][r];
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// The tile form on 16-bit operands: chunks of 32 steps, a workgroup of four wavefronts owns 64 NT columns, a wavefront 16 NT of them (W: KA tiles of 16 rows
// in its registers; DA is the power of two that rows have in LDS).  a, b, c of the next chunk are on their way to registers while this one is computed, then go to
// the other of two LDS buffers: one barrier for the buffers and one for P per chunk, two workgroups on a CU.
// Bound by the vector instructions beside the products (of 784 in a wavefront's chunk 91 are products; the split of lambda^(CH-j) c and the terms of W lead): they issue
// 59 % of the output pass's time, the matrix cores are busy 28 % of it.  64 heads of 128 x 128, 4096 steps, bf16: 38 us for the states (134 MB), 10 for the scan, 87 for the
// outputs (300 MB).  Chunks of 64 steps in eight wavefronts took 209 us for the whole where this form took 118 (both with one term of W).
// Rows are unpadded; the 16-byte granule q of row r lies in slot q ^ f(r), f chosen so that the three ways they are read (a granule of 16 rows, half granules
// of 16 rows, and the transposing 4 x 16 read) meet no bank twice.
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
template <int SPR> __device__ __forceinline__ int swz(int row) { return SPR >= 16 ? ((row & 7) << 1) | ((row >> 3) & 1) : (((row >> 1) & 3) << 1) | ((row >> 3) & 1); }
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
template <int DT> __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c)
{
    if constexpr (DT == SS_SEQ_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// |x|, 0 for what is not finite
__device__ __forceinline__ float finite(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.f; }
// what is left of x behind its rounded value; 0 where that is not finite
__device__ __forceinline__ float behind(float x, float rounded) { return fabsf(rounded) < __builtin_inff() ? x - rounded : 0.f; }
// a power of two that takes `most` into [2^14, 2^15), fp16's upper end, and its inverse; 1 for zero and for what is not finite
__device__ __forceinline__ void fp16_scale(float most, float& up, float& down)
{
    int e = (int)(__float_as_uint(most) >> 23 & 255);      // biased exponent
    e = e == 0 || e == 255 ? 141 : e < 30 ? 30 : e;
    up = __uint_as_float((unsigned)(268 - e) << 23);       // 2^(14 - (e - 127))
    down = __uint_as_float((unsigned)(e - 14) << 23);
}
// eight fp32 values, times `up` for fp16, as two terms of the operands' type: the rounded value and what that leaves.  CAREFUL: for any value; else for finite ones
template <int DT, bool CAREFUL> __device__ __forceinline__ void two_terms(const f32x4& x, const f32x4& y, float up, s16x8& first, s16x8& second)
{
    if constexpr (DT == SS_SEQ_F16) {
        f16x8 p, q;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = (i < 4 ? x[i & 3] : y[i & 3]) * up;
            p[i] = (_Float16)v;
            q[i] = (_Float16)(CAREFUL ? behind(v, (float)p[i]) : v - (float)p[i]);
        }
        first = __builtin_bit_cast(s16x8, p);
        second = __builtin_bit_cast(s16x8, q);
    } else {
        unsigned p[4];
        float z[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = i < 2 ? x[2 * i] : y[2 * i - 4], b = i < 2 ? x[2 * i + 1] : y[2 * i - 3];
            p[i] = round_pk(a, b);
            const float pa = __uint_as_float(p[i] << 16), pb = __uint_as_float(p[i] & 0xFFFF0000u);
            z[2 * i] = CAREFUL ? behind(a, pa) : a - pa;
            z[2 * i + 1] = CAREFUL ? behind(b, pb) : b - pb;
        }
        first = __builtin_bit_cast(s16x8, mk8(p[0], p[1], p[2], p[3]));
        second = __builtin_bit_cast(s16x8, mk8(round_pk(z[0], z[1]), round_pk(z[2], z[3]), round_pk(z[4], z[5]), round_pk(z[6], z[7])));
    }
}
// this wavefront's LDS operations are done, then the barrier: unlike __syncthreads() it does not wait for loads on their way to LDS or for stores
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int DT, int DA, int KA, int NT, bool STATE, bool VEC>
__global__ __launch_bounds__(256, DA * NT <= 256 ? 2 : 1) void leaky_tile_kernel(const LeakyMaps maps)
{
    constexpr int CH = 32, DCB = 64 * NT, SA = DA / 8, SC = DCB / 8;                          // SA, SC: granules of a row
    constexpr int PL = 2 * 64 * 8;
    constexpr int BA = CH * DA, BC = CH * DCB, BUF = (STATE ? 1 : 2) * BA + BC;              // elements of a buffer: [a] b c
    __shared__ __attribute__((aligned(1024))) unsigned short lds[2 * BUF];
    __shared__ __attribute__((aligned(16))) unsigned short sp[STATE ? 8 : 2 * PL];           // P's two terms in operand order, by tile of 16 steps
    __shared__ __attribute__((aligned(16))) float rw[CH];                                    // lambda^(e - j) b_scale of the chunk's steps
    __shared__ float p_down[4];                                                              // fp16: what undoes the scale of P's three tiles
    constexpr bool H = DT == SS_SEQ_F16;

    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const unsigned which = blockIdx.x / maps.per, block = blockIdx.x - which * maps.per;
    const LeakyMap& map = maps.m[which];
    const LeakyArgs& p = map.p;
    const LeakyPlan& plan = map.plan;
    float* __restrict__ ws = map.ws;
    const int cb = block % plan.ncb, rest = block / plan.ncb;
    const int nst = STATE ? plan.nseg - 1 : plan.nseg, seg = rest % nst, bh = rest / nst, b = bh / p.H, h = bh - b * p.H;
    int n = p.T;
    if (p.lengths) { n = p.lengths[b]; n = n < 0 ? 0 : n > p.T ? p.T : n; }
    const int start = seg * plan.seg, stop = n < start + plan.seg ? n : start + plan.seg;    // this segment's valid steps
    if (STATE && n <= start + plan.seg) return;                          // no later segment reads this one's state
    const float gl = log2_decay(p.log_decay[h]);
    const int c0 = cb * DCB, col0 = c0 + wv * 16 * NT;
    const unsigned short* pa = static_cast<const unsigned short*>(p.a) + b * p.a_b + (h / p.a_group) * p.a_h;
    const unsigned short* pb = static_cast<const unsigned short*>(p.b) + b * p.b_b + (h / p.b_group) * p.b_h;
    const unsigned short* pc = static_cast<const unsigned short*>(p.c) + b * p.c_b + (h / p.c_group) * p.c_h + c0;
    const int dc = p.DC - c0 < DCB ? p.DC - c0 : DCB;

    // ---- the state that enters the segment
    f32x4 W[KA][NT];
    {
#pragma unroll
        for (int kt = 0; kt < KA; ++kt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) W[kt][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (seg == 0) {
            if (p.s_in) {
                const float* s_in = p.s_in + (long long)bh * p.DA * p.DC;
                const float first = exp2f(gl * (float)((p.reverse || n == 0 ? 0 : 1) + (STATE ? plan.seg : 0)));
#pragma unroll
                for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int i = 16 * kt + 4 * g + r, j = col0 + 16 * nt + l16;
                            const bool in = i < p.DA && j < p.DC;
                            const float v = s_in[in ? i * p.s_in_row + j * p.s_in_col : 0];
                            W[kt][nt][r] = in ? v * first : 0.f;
                        }
            }
        } else if (!STATE && start < n) {
            const float leak = exp2f(gl * (float)plan.seg);
            for (int s = plan.fold ? 0 : seg - 1; s < seg; ++s)
#pragma unroll
                for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) W[kt][nt] = W[kt][nt] * leak + state_read(plan, ws, bh, s, kt, col0 / 16 + nt, lane);
        }
    }

    // ---- staging: 16-byte granules of [CH][D] rows, global -> registers -> LDS
    constexpr int GA = CH * SA / 256, GC = CH * SC / 256;
    u16x8 ra[STATE ? 1 : GA], rb[GA], rc[GC];
    auto fetch = [&](u16x8* dst, const unsigned short* base, long long st, int i0, int d, auto SPRC) {
        constexpr int SPR = SPRC.value;
#pragma unroll
        for (int u = 0; u < CH * SPR / 256; ++u) {
            const int x = tid + 256 * u, row = x / SPR, q = x % SPR, i = i0 + row;
            const unsigned short* src = base + (long long)(p.reverse ? n - 1 - i : i) * st + 8 * q;
            if (VEC && i0 + CH <= stop && d == 8 * SPR) dst[u] = *reinterpret_cast<const u16x8*>(src);       // nothing to leave out: no branch per granule
            else {
                dst[u] = (u16x8){0, 0, 0, 0, 0, 0, 0, 0};
                if (i < stop && 8 * q < d) {
                    if constexpr (VEC) dst[u] = *reinterpret_cast<const u16x8*>(src);
                    else                                                 // rows that are not whole aligned granules
#pragma unroll
                        for (int e = 0; e < 8; ++e) if (8 * q + e < d) dst[u][e] = src[e];
                }
            }
        }
    };
    auto put = [&](unsigned short* dst, const u16x8* v, auto SPRC) {
        constexpr int SPR = SPRC.value;
#pragma unroll
        for (int u = 0; u < CH * SPR / 256; ++u) {
            const int x = tid + 256 * u, row = x / SPR, q = x % SPR;
            *reinterpret_cast<u16x8*>(dst + (row * SPR + (q ^ swz<SPR>(row))) * 8) = v[u];
        }
    };
    auto load = [&](int i0) {
        if constexpr (!STATE) fetch(ra, pa, p.a_t, i0, p.DA, std::integral_constant<int, SA>());
        fetch(rb, pb, p.b_t, i0, p.DA, std::integral_constant<int, SA>());
        fetch(rc, pc, p.c_t, i0, dc, std::integral_constant<int, SC>());
    };
    auto stage = [&](int buf) {
        unsigned short* at = lds + buf * BUF;
        if constexpr (!STATE) { put(at, ra, std::integral_constant<int, SA>()); at += BA; }
        put(at, rb, std::integral_constant<int, SA>());
        put(at + BA, rc, std::integral_constant<int, SC>());
    };
    auto put_out = [&](void* q, const f32x4& o) {
        if (p.out_f32) *static_cast<f32x4*>(q) = o;
        else *static_cast<u16x4*>(q) = (u16x4){narrow<DT>(o[0]), narrow<DT>(o[1]), narrow<DT>(o[2]), narrow<DT>(o[3])};
    };
    // the chunk's outputs: a lane has four columns of steps 16 it + l16
    auto store = [&](int i0, const f32x4 (&v)[2][NT]) {
        const int es = p.out_f32 ? 4 : 2;
        char* out = static_cast<char*>(p.out) + (b * p.o_b + h * p.o_h + col0) * es;
        if (VEC && i0 + CH <= stop && col0 + 16 * NT <= p.DC) {
            char* to = out + (long long)(p.reverse ? n - CH - i0 : i0) * p.o_t * es;
            const unsigned step = (unsigned)p.o_t * es;
#pragma unroll
            for (int it = 0; it < 2; ++it)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    put_out(to + ((unsigned)(p.reverse ? CH - 1 - 16 * it - l16 : 16 * it + l16) * step + (unsigned)((16 * nt + 4 * g) * es)), v[it][nt]);
            return;
        }
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int i = i0 + 16 * it + l16, col = 16 * nt + 4 * g, left = p.DC - col0 - col;
                if (i >= p.T || left <= 0) continue;
                const bool live = i < n;                                 // steps behind the last: zeros
                char* q = out + ((long long)(live && p.reverse ? n - 1 - i : i) * p.o_t + col) * es;
                const f32x4 o = live ? v[it][nt] : (f32x4){0.f, 0.f, 0.f, 0.f};
                if constexpr (VEC) put_out(q, o);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < left) {
                            if (p.out_f32) reinterpret_cast<float*>(q)[e] = o[e];
                            else reinterpret_cast<unsigned short*>(q)[e] = narrow<DT>(o[e]);
                        }
            }
    };

    if constexpr (!STATE) *reinterpret_cast<f32x4*>(sp + tid * 8) = (f32x4){0.f, 0.f, 0.f, 0.f};         // the half of P above the diagonal stays zero
    if (tid < CH) rw[tid] = exp2f(gl * (float)(CH - tid)) * p.b_scale;
    // lambda^i o_scale of this lane's steps; lambda^(i - j) and both scales for this lane's entries of the wavefront's tile of P (0: above the diagonal)
    const int it1 = (wv + 1) >> 1, jt1 = wv >> 1;
    float row_scale[2], p_scale[4];
#pragma unroll
    for (int it = 0; it < 2; ++it) row_scale[it] = exp2f(gl * (float)(16 * it + l16)) * p.o_scale;
#pragma unroll
    for (int r = 0; r < 4; ++r) p_scale[r] = exp2f(gl * (float)max(16 * (it1 - jt1) + l16 - 4 * g - r, 0)) * p.b_scale * p.o_scale;
    const float keep_all = exp2f(gl * (float)CH);
    // byte offsets of this lane's operands in a buffer; 32 (64) bytes of the row further on is an XOR of the slot
    const int fa = swz<SA>(l16), o1 = l16 * DA * 2 + ((g ^ fa) << 4), o3 = l16 * DA * 2 + (((g >> 1) ^ fa) << 4) + ((g & 1) << 3);
    const int tr = 4 * g + (l16 >> 2), y = (l16 & 3) >> 1;
    const int o4 = tr * DA * 2 + ((y ^ swz<SA>(tr)) << 4) + ((l16 & 1) << 3), oc = tr * DCB * 2 + (((2 * NT * wv + y) ^ swz<SC>(tr)) << 4) + ((l16 & 1) << 3);

    int i0 = start, buf = 0;
    if (start < stop) {
        load(start);
        stage(0);
    }
    for (; i0 < stop; i0 += CH, buf ^= 1) {
        const int cnt = stop - i0 < CH ? stop - i0 : CH;
        // the last chunk of the stream leaves the state as it is after its last step (forward) or leaked once more (reverse)
        const int e = i0 + cnt == n && !p.reverse ? cnt - 1 : cnt;
        lds_barrier();                                                   // this chunk is there, and the other buffer has been read
        if (i0 + CH < stop) load(i0 + CH);
        const char* la = reinterpret_cast<const char*>(lds + buf * BUF);
        const char* lb = la + (STATE ? 0 : BA * 2);
        const char* lc = lb + BA * 2;
        if (e != CH && tid < CH) rw[tid] = exp2f(gl * (float)(e > tid ? e - tid : 0)) * p.b_scale;
        f32x4 acc[2][NT];
        if constexpr (!STATE) {
            // (1) wavefronts 0 .. 2: the tiles (0, 0), (1, 0), (1, 1)
            if (wv < 3) {
                const int it = it1, jt = jt1;
                f32x4 s = {0.f, 0.f, 0.f, 0.f}, s2 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KA / 2; ++k) {
                    const s16x8 xa = *reinterpret_cast<const s16x8*>(la + it * 16 * DA * 2 + (o1 ^ (64 * k)));
                    const s16x8 xb = *reinterpret_cast<const s16x8*>(lb + jt * 16 * DA * 2 + (o1 ^ (64 * k)));
                    if (k & 1) s2 = mfma16<DT>(xb, xa, s2);
                    else s = mfma16<DT>(xb, xa, s);
                }
                s += s2;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[r] = 16 * (it - jt) + l16 - 4 * g - r < 0 ? 0.f : s[r] * p_scale[r];
                }
                if constexpr (H) {
                    float up, down;
                    fp16_scale(wave_max(fmaxf(fmaxf(finite(s[0]), finite(s[1])), fmaxf(finite(s[2]), finite(s[3])))), up, down);
                    f16x4 x, z;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = (_Float16)(s[r] * up);
                        z[r] = (_Float16)behind(s[r] * up, (float)x[r]);
                    }
                    *reinterpret_cast<f16x4*>(sp + (wv * 64 + lane) * 4) = x;
                    *reinterpret_cast<f16x4*>(sp + PL + (wv * 64 + lane) * 4) = z;
                    if (lane == 0) p_down[wv] = down;
                } else {
                    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                    f32x4 z;
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[r] = behind(s[r], (float)(__bf16)s[r]);
                    *reinterpret_cast<u32x2*>(sp + (it * 64 + lane) * 8 + jt * 4) = (u32x2){round_pk(s[0], s[1]), round_pk(s[2], s[3])};
                    *reinterpret_cast<u32x2*>(sp + PL + (it * 64 + lane) * 8 + jt * 4) = (u32x2){round_pk(z[0], z[1]), round_pk(z[2], z[3])};
                }
            }
            // (3)
            float up = 1.f, down = 1.f;
            bool odd = false;                                            // this wavefront's W holds an infinity
            if constexpr (H) {
                float most = 0.f;
#pragma unroll
                for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(W[kt][nt][r]));
                most = wave_max(most);
                if (most == __builtin_inff()) {                          // rare: the others' scale without what is infinite
                    odd = true;
                    most = 0.f;
#pragma unroll
                    for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) most = fmaxf(most, finite(W[kt][nt][r]));
                    most = wave_max(most);
                }
                fp16_scale(most, up, down);
            }
            // CAREFUL: the second term is 0 behind what is not finite (infinity - infinity would make a NaN of it)
            auto read = [&](auto CAREFUL) {
#pragma unroll
                for (int it = 0; it < 2; ++it)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) acc[it][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KA / 2; ++k) {
                    s16x8 xa[2];
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        const char* q = la + it * 16 * DA * 2 + (o3 ^ (64 * k));
                        const char* q2 = la + it * 16 * DA * 2 + (o3 ^ (64 * k + 32));
                        xa[it] = __builtin_shufflevector(*reinterpret_cast<const s16x4*>(q), *reinterpret_cast<const s16x4*>(q2), 0, 1, 2, 3, 4, 5, 6, 7);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const f32x4 x = W[2 * k][nt], z = W[2 * k + 1][nt];
                        s16x8 f0, f1;
                        two_terms<DT, CAREFUL.value>(x, z, up, f0, f1);
#pragma unroll
                        for (int it = 0; it < 2; ++it) acc[it][nt] = mfma16<DT>(f0, xa[it], mfma16<DT>(f1, xa[it], acc[it][nt]));
                    }
                    // the conversions of all of W at once do not fit the registers (32 heads of 256 x 256, bf16: 180 us with the spills, 127 without)
                    if constexpr (KA * NT >= 12) if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            };
            if constexpr (H) {
                if (odd) read(std::true_type());
                else read(std::false_type());
            } else {
                read(std::false_type());
                f32x4 sum = acc[0][0] + acc[1][0];
#pragma unroll
                for (int nt = 1; nt < NT; ++nt) sum += acc[0][nt] + acc[1][nt];
                sum[0] += sum[1] + sum[2] + sum[3];
                if (__any(!(sum[0] == sum[0]))) {                        // rare: again, with care
#pragma unroll
                    for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) asm("" : "+v"(W[kt][nt]));       // (or the first terms of all of W are kept for this branch, and spill)
                    read(std::true_type());
                }
            }
#pragma unroll
            for (int it = 0; it < 2; ++it)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[it][nt] *= row_scale[it] * down;
            lds_barrier();                                               // P is there
        }
        // (2) and (4) share the wavefront's columns of c
        s16x8 t0[NT], t1[NT], t2[NT];
        float c_down[NT];
        bool wild = false;
        {
            // (the state pass weighs by the distance to the segment's end, so W only accumulates)
            const float tail = STATE ? exp2f(gl * (float)(stop - CH - i0)) : 1.f;
            const f32x4 w0 = *reinterpret_cast<const f32x4*>(rw + 4 * g) * tail, w1 = *reinterpret_cast<const f32x4*>(rw + 16 + 4 * g) * tail;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const char* q = lc + (oc ^ (32 * nt));
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)q), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(q + 16 * DCB * 2));
                const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                // what is not finite (exponent all ones: one more carries into the sign's place) is left out of the product (2): 0 * NaN would reach steps before it
                s16x8 fin = both;
                if constexpr (!STATE) {
                    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
                    constexpr unsigned EXP = H ? 0x7C007C00u : 0x7F807F80u, ONE = H ? 0x04000400u : 0x00800080u;
                    const u32x4 c2 = __builtin_bit_cast(u32x4, both), t = (c2 & EXP) + ONE;
                    if (__any(((t[0] | t[1] | t[2] | t[3]) & 0x80008000u) != 0)) {
                        wild = true;
                        const s16x8 odd = (both & (short)EXP) == (short)EXP;
                        fin = both & ~odd;
                    }
                }
                if constexpr (!STATE && H) {               // a product of 16 steps for each tile of P, its scale undone as it is added
                    const f16x4 *fp = reinterpret_cast<const f16x4*>(sp) + lane, cl = __builtin_bit_cast(f16x4, (s16x4)__builtin_shufflevector(fin, fin, 0, 1, 2, 3)), ch = __builtin_bit_cast(f16x4, (s16x4)__builtin_shufflevector(fin, fin, 4, 5, 6, 7));
                    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
                    auto both_terms = [&](const f16x4& c, int t) {
                        return __builtin_amdgcn_mfma_f32_16x16x16f16(c, fp[64 * t], __builtin_amdgcn_mfma_f32_16x16x16f16(c, fp[PL / 4 + 64 * t], z, 0, 0, 0), 0, 0, 0);
                    };
                    acc[0][nt] += both_terms(cl, 0) * p_down[0];
                    acc[1][nt] += both_terms(cl, 1) * p_down[1] + both_terms(ch, 2) * p_down[2];
                } else if constexpr (!STATE) {
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        acc[it][nt] = mfma16<DT>(fin, *reinterpret_cast<const s16x8*>(sp + PL + (it * 64 + lane) * 8), acc[it][nt]);
                        acc[it][nt] = mfma16<DT>(fin, *reinterpret_cast<const s16x8*>(sp + (it * 64 + lane) * 8), acc[it][nt]);
                    }
                }
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = widen<DT>((unsigned short)both[i]) * (i < 4 ? w0[i & 3] : w1[i & 3]);
                if constexpr (H) {
                    float most = 0.f, up;
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    fp16_scale(most, up, c_down[nt]);
                    f16x8 x, z;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = (_Float16)(v[i] * up);
                        z[i] = (_Float16)(v[i] * up - (float)x[i]);
                    }
                    t0[nt] = __builtin_bit_cast(s16x8, x);
                    t1[nt] = __builtin_bit_cast(s16x8, z);
                } else {
                    float x[8], z[8], u[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        x[i] = top16(v[i]);
                        z[i] = v[i] - x[i];
                        u[i] = z[i] - top16(z[i]);
                    }
                    t0[nt] = __builtin_bit_cast(s16x8, mk8(pack_hi16(x[0], x[1]), pack_hi16(x[2], x[3]), pack_hi16(x[4], x[5]), pack_hi16(x[6], x[7])));
                    t1[nt] = __builtin_bit_cast(s16x8, mk8(pack_hi16(z[0], z[1]), pack_hi16(z[2], z[3]), pack_hi16(z[4], z[5]), pack_hi16(z[6], z[7])));
                    t2[nt] = __builtin_bit_cast(s16x8, mk8(pack_hi16(u[0], u[1]), pack_hi16(u[2], u[3]), pack_hi16(u[4], u[5]), pack_hi16(u[6], u[7])));
                }
            }
        }
        if (!STATE && wild)                                       // rare: those terms one by one, where j <= i
#pragma unroll 1
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int it = 0; it < 2; ++it) {
                    if (j > 16 * it + l16) continue;
                    const int jl = 16 * (j >> 2 & 3) + l16;              // the lane that holds P_ij
                    const unsigned short* at = sp + (H ? ((it + (j >> 4)) * 64 + jl) * 4 : (it * 64 + jl) * 8 + (j >> 4) * 4) + (j & 3);
                    const float pij = (widen<DT>(at[0]) + widen<DT>(at[PL])) * (H ? p_down[it + (j >> 4)] : 1.f);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int col = wv * 16 * NT + 16 * nt + 4 * g + r;
                            const float c = widen<DT>(*reinterpret_cast<const unsigned short*>(lc + j * DCB * 2 + (((col >> 3) ^ swz<SC>(j)) << 4) + ((col & 7) << 1)));
                            if (!(fabsf(c) < __builtin_inff())) acc[it][nt][r] += pij * c;
                        }
                }
        if constexpr (!STATE) store(i0, acc);
        const float keep = STATE ? 1.f : e == CH ? keep_all : exp2f(gl * (float)e);
#pragma unroll
        for (int kt = 0; kt < KA; ++kt) {
            const char* q = lb + (o4 ^ (32 * kt));
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)q), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(q + 16 * DA * 2));
            const s16x8 fb = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            if constexpr (H) {
                f32x4 d[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) d[nt] = mfma16<DT>(fb, t1[nt], (f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) d[nt] = mfma16<DT>(fb, t0[nt], d[nt]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) W[kt][nt] = (STATE ? W[kt][nt] : W[kt][nt] * keep) + d[nt] * c_down[nt];
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) W[kt][nt] = mfma16<DT>(fb, t2[nt], STATE ? W[kt][nt] : W[kt][nt] * keep);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) W[kt][nt] = mfma16<DT>(fb, t1[nt], W[kt][nt]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) W[kt][nt] = mfma16<DT>(fb, t0[nt], W[kt][nt]);
            }
        }
        if (i0 + CH < stop) stage(buf ^ 1);
    }

    if constexpr (STATE) {
        const long long per = (long long)DA * DCB;
        float* mine = ws + (((long long)bh * plan.ncb + cb) * (plan.nseg - 1) + seg) * per + wv * (DA / 16) * NT * 256 + lane * 4;
#pragma unroll
        for (int kt = 0; kt < KA; ++kt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<f32x4*>(mine + (kt * NT + nt) * 256) = W[kt][nt];
    } else {
        // steps of the segment behind the stream's last: zeros (the loop above has written its own chunks to their end)
        const int end = start + plan.seg < p.T ? start + plan.seg : p.T;
        f32x4 none[2][NT];
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) none[it][nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (; i0 < end; i0 += CH) store(i0, none);
        if (p.s_out && ((start < n && n <= start + plan.seg) || (n == 0 && seg == 0))) {
            float* s_out = p.s_out + (long long)bh * p.DA * p.DC;
#pragma unroll
            for (int kt = 0; kt < KA; ++kt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 16 * kt + 4 * g + r, j = col0 + 16 * nt + l16;
                        if (i < p.DA && j < p.DC) s_out[i * p.s_out_row + j * p.s_out_col] = W[kt][nt][r];
                    }
        }
    }
}

// ws[s] (what segment s adds to the state) -> the state that enters segment s + 1, in fp32.  HBM-bound (64 heads of 128 x 128, 7 states: 59 MB in 10 us).
__global__ __launch_bounds__(256) void leaky_scan_kernel(float* __restrict__ ws, const float* __restrict__ log_decay, int H, int ncb, int per, int nstate, int seg)
{
    const unsigned parts = per / 1024, head = blockIdx.x / parts, bh = head / ncb;
    const float leak = exp2f(log2_decay(log_decay[bh % H]) * (float)seg);
    float* at = ws + (long long)head * nstate * per + ((blockIdx.x - head * parts) * 256 + threadIdx.x) * 4;
    f32x4 s = *reinterpret_cast<const f32x4*>(at);
    constexpr int U = 16;                    // states in flight: with one at a time the scan is their latencies (63 of them: 23 us)
    for (int k = 1; k < nstate; k += U) {
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const f32x4*>(at + (long long)min(u + 1, nstate - k) * per);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s = s * leak + v[u];
            if (k + u < nstate) *reinterpret_cast<f32x4*>(at + (long long)(u + 1) * per) = s;
        }
        at += (long long)U * per;
    }
}

template <int DT> struct LeakyShape {
    static constexpr int CH = 32;
    static int pad(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
    // row tiles of a state in a kernel's registers: three quarters of the padded width where they suffice (2048 steps, bf16: 64 heads of 96 x 96 76 -> 68 us, 32 of
    // 192 x 192 101 -> 88; the fp32 kernel leaves tiles out as it runs)
    static int row_tiles(int d) { return DT != SS_SEQ_F32 && d > 64 && d <= pad(d) / 4 * 3 ? pad(d) / 64 * 3 : pad(d) / 16; }
    // columns of a workgroup's block: 64 where the state of 128 would not leave two workgroups on a CU (16-bit heads over 128 wide; 2048 steps, 32 heads, bf16:
    // 256 x 256 in blocks of 128 174 us, of 64 119; 192 x 192 167 and 95, with one term of W), else up to 128
    static int cols(int DA, int DC) { return DC <= 64 || (DT != SS_SEQ_F32 && DA > 128) ? 64 : 128; }
    static int blocks(int DA, int DC) { return (DC + cols(DA, DC) - 1) / cols(DA, DC); }
    static LeakyPlan plan(int T, int B, int H, int DA, int DC)
    {
        LeakyPlan r;
        r.ncb = r.sncb = blocks(DA, DC);
        // Segments: the count with the least estimated time, in chunks.  A round of workgroups (two on a CU; one for fp32, whose matrix instructions one workgroup
        // fills) takes a segment's chunks and two for its state; the state pass half of that; joining costs half a chunk per state in the output pass up to 5
        // segments, else a scan; each further launch two.  (64 heads, 4096 steps, bf16: 4 segments 152 us, 8 132, 16 169; 48 heads, 777 steps, fp32 training:
        // 4 segments 179 us, 5 147, 7 165.)
        const int chunks = (T + CH - 1) / CH;
        const double base = (double)B * H * r.ncb, slots = DT == SS_SEQ_F32 ? 256. : 512.;
        int best = 1;
        double least = 0.;
        for (int n = 1; n <= 128 && n <= chunks; ++n) {
            const double per = (chunks + n - 1) / n;
            double t = ceil(base * n / slots) * (per + 2. + (n <= 5 ? 0.5 * (n - 1) : 0.));
            if (n > 1) t += ceil(base * (n - 1) / slots) * (0.5 * per + 1.) + 2.;
            if (n > 5) t += 4. + n / 16.;
            if (n == 1 || t < least) { best = n; least = t; }
        }
        const int per = (chunks + best - 1) / best;
        r.seg = per * CH;
        r.nseg = (chunks + per - 1) / per;
        r.fold = r.nseg <= 5;
        r.trans = 0;
        r.ka = pad(DA) / 16;
        r.dcb = cols(DA, DC);
        r.nt = DT == SS_SEQ_F32 || r.dcb == 64 ? 1 : 2;
        return r;
    }
    static long long state_floats(int T, int B, int H, int DA, int DC)
    {
        if (T == 1) return 0;
        const LeakyPlan r = plan(T, B, H, DA, DC);
        return (long long)B * H * (r.nseg - 1) * (r.ncb * r.dcb) * pad(DA);
    }
    static LeakyMap map_of(const LeakyArgs& p, const LeakyPlan& r, float* ws, bool state)
    {
        // rows of whole 16-byte granules; a chunk of the output within 32-bit offsets
        constexpr int E = DT == SS_SEQ_F32 ? 4 : 8;
        auto ok = [&](const void* q, long long t, long long b, long long h) { return aligned(q, 16) && t % E == 0 && b % E == 0 && h % E == 0; };
        const int vec = p.DA % E == 0 && p.DC % E == 0 && (state || ok(p.a, p.a_t, p.a_b, p.a_h)) && ok(p.b, p.b_t, p.b_b, p.b_h) && ok(p.c, p.c_t, p.c_b, p.c_h);
        const int vec_out = state || (p.DC % 4 == 0 && p.o_t % 4 == 0 && p.o_b % 4 == 0 && p.o_h % 4 == 0 && aligned(p.out, 16) && p.o_t >= 0 && p.o_t < (1 << 24));
        return {p, r, ws, vec, vec_out};
    }
    template <int DA, int KA, int WV, bool STATE> static int launch(LeakyMaps& maps, int count, hipStream_t s)
    {
        const LeakyPlan& r = maps.m[0].plan;               // maps of one launch have the same segments and column blocks
        maps.per = (unsigned)(maps.m[0].p.B * maps.m[0].p.H * r.ncb) * (STATE ? r.nseg - 1 : r.nseg);
        const unsigned grid = maps.per * count;
        if constexpr (DT == SS_SEQ_F32) leaky_chunk_kernel<DA, WV, STATE><<<grid, 64 * WV, 0, s>>>(maps);
        else {
            bool all = true;
            for (int i = 0; i < count; ++i) all = all && maps.m[i].vec && maps.m[i].vec_out;
            if (all) leaky_tile_kernel<DT, DA, KA, WV / 4, STATE, true><<<grid, 256, 0, s>>>(maps);
            else leaky_tile_kernel<DT, DA, KA, WV / 4, STATE, false><<<grid, 256, 0, s>>>(maps);
        }
        return launched();
    }
    // `count` maps of the same padded sizes, row tiles and column blocks in one launch
    template <bool STATE> static int pass(LeakyMaps& maps, int count, hipStream_t s)
    {
        const int DA = maps.m[0].p.DA, DC = maps.m[0].p.DC;
        auto by_dc = [&](auto DAC, auto KAC) {
            if constexpr (DT == SS_SEQ_F32 || DAC.value <= 128)
                if (cols(DA, DC) == 128) return launch<DAC.value, KAC.value, 8, STATE>(maps, count, s);
            return launch<DAC.value, KAC.value, 4, STATE>(maps, count, s);
        };
        auto by_ka = [&](auto DAC) {
            if constexpr (DT != SS_SEQ_F32 && DAC.value > 64)
                if (row_tiles(DA) * 16 < DAC.value) return by_dc(DAC, std::integral_constant<int, DAC.value / 16 * 3 / 4>());
            return by_dc(DAC, std::integral_constant<int, DAC.value / 16>());
        };
        return DA <= 64 ? by_ka(std::integral_constant<int, 64>()) : DA <= 128 ? by_ka(std::integral_constant<int, 128>()) : by_ka(std::integral_constant<int, 256>());
    }
    // the states that enter the segments, into ws (nothing where there is one segment)
    static int states(const LeakyArgs& p, const LeakyPlan& r, float* ws, hipStream_t s)
    {
        if (r.nseg == 1) return SS_SEQ_OK;
        if (!ws || !aligned(ws, 16)) return SS_SEQ_EINVAL;
        LeakyMaps one{{map_of(p, r, ws, true)}, 0};
        if (int rc = pass<true>(one, 1, s)) return rc;
        if (r.fold) return SS_SEQ_OK;
        const int per = pad(p.DA) * r.dcb;
        leaky_scan_kernel<<<(unsigned)(p.B * p.H * r.ncb) * (per / 1024), 256, 0, s>>>(ws, p.log_decay, p.H, r.ncb, per, r.nseg - 1, r.seg);
        return launched();
    }
    static int run(const LeakyArgs& p, float* ws, hipStream_t s)
    {
        // one step has its own kernel; from two on a tile (8 heads of 64 x 64, bf16: a kernel that walks the steps 4.8 us for 2, 6.4 for 4, 9.3 for 7, the tile form
        // 7 for any; 128 heads of 128 x 128: 54, 70 and 95 against 15)
        if (p.T == 1) return p.out_f32 ? step<DT, SS_SEQ_F32>(p, s) : step<DT, DT>(p, s);
        const LeakyPlan r = plan(p.T, p.B, p.H, p.DA, p.DC);
        if (int rc = states(p, r, ws, s)) return rc;
        LeakyMaps one{{map_of(p, r, ws, false)}, 0};
        return pass<false>(one, 1, s);
    }

    // ---- the gradients: three maps.  dq reads the forward pass's states transposed; dk and dv run backwards in time and share the states of (q, g).  dq and
    // dk are of one shape and run in one launch, with dv where its row tiles and column blocks are theirs: the ends of one map's streams fill with the next map's workgroups
    // (48 heads of 80 and 96, 777 ragged steps, fp32: three launches 196 us a training step, one 158).
    static long long round4(long long n) { return (n + 3) / 4 * 4; }
    static long long heads_floats(const LeakyBwdArgs& d, int D) { return d.H == d.Hk ? 0 : round4((long long)d.T * d.B * d.H * D); }
    static long long bwd_floats(const LeakyBwdArgs& d) { return heads_floats(d, d.Dk) + heads_floats(d, d.Dv) + state_floats(d.T, d.B, d.H, d.Dk, d.Dv); }
    static int bwd(const LeakyBwdArgs& d, hipStream_t s)
    {
        const int group = d.H / d.Hk;
        float *each_k = d.ws, *each_v = each_k + heads_floats(d, d.Dk), *rstate = each_v + heads_floats(d, d.Dv);      // gradients by query head
        const bool tiles = d.T > 1;
        const LeakyPlan fwd = plan(d.T, d.B, d.H, d.Dk, d.Dv);
        if (bwd_floats(d) && (!d.ws || !aligned(d.ws, 16))) return SS_SEQ_EINVAL;
        if (tiles && fwd.nseg > 1 && d.g_q && (!d.states || !aligned(d.states, 16))) return SS_SEQ_EINVAL;
        // contiguous results: [T][B][heads][D]
        auto map = [&](int DA, int DC, int reverse, float bs, float os, const LeakyView& a, const LeakyView& b, const LeakyView& c, void* out, bool f32) {
            LeakyArgs p{};
            p.T = d.T; p.B = d.B; p.H = d.H; p.DA = DA; p.DC = DC; p.reverse = reverse; p.b_scale = bs; p.o_scale = os;
            p.a = a.p; p.a_t = a.t; p.a_b = a.b; p.a_h = a.h; p.a_group = a.group;
            p.b = b.p; p.b_t = b.t; p.b_b = b.b; p.b_h = b.h; p.b_group = b.group;
            p.c = c.p; p.c_t = c.t; p.c_b = c.b; p.c_h = c.h; p.c_group = c.group;
            p.out = out; p.o_h = DC; p.o_b = (long long)d.H * DC; p.o_t = p.o_b * d.B;
            p.log_decay = d.log_decay; p.lengths = d.lengths; p.out_f32 = f32;
            return p;
        };
        LeakyArgs pv = map(d.Dk, d.Dv, 1, d.scale, 1.f, d.k, d.q, d.g, group == 1 ? d.g_v : each_v, group > 1 || DT == SS_SEQ_F32);
        pv.s_in = d.g_last; pv.s_in_row = d.Dv; pv.s_in_col = 1;
        pv.s_out = d.g_s; pv.s_out_row = d.Dv; pv.s_out_col = 1;
        LeakyArgs pq = map(d.Dv, d.Dk, 0, 1.f, d.scale, d.g, d.v, d.k, d.g_q, DT == SS_SEQ_F32);
        pq.s_in = d.s_in; pq.s_in_row = 1; pq.s_in_col = d.Dv;
        LeakyArgs pk = map(d.Dv, d.Dk, 1, d.scale, 1.f, d.v, d.g, d.q, group == 1 ? d.g_k : each_k, group > 1 || DT == SS_SEQ_F32);
        pk.s_in = d.g_last; pk.s_in_row = 1; pk.s_in_col = d.Dv;
        if (!tiles) {
            auto go = [&](const LeakyArgs& p) { return p.out_f32 ? step<DT, SS_SEQ_F32>(p, s) : step<DT, DT>(p, s); };
            if (d.g_q) if (int rc = go(pq)) return rc;
            if (d.g_v) if (int rc = go(pv)) return rc;
            if (d.g_k) if (int rc = go(pk)) return rc;
        } else {
            if (d.g_k || d.g_v) if (int rc = states(pv, fwd, rstate, s)) return rc;
            LeakyMaps maps{};
            int count = 0;
            auto add = [&](const LeakyArgs& p, float* ws, int trans) {
                LeakyPlan r = fwd;                         // the forward pass's segments, whatever this map's own sizes
                r.ncb = blocks(p.DA, p.DC);
                r.trans = trans;
                maps.m[count++] = map_of(p, r, ws, false);
            };
            if (d.g_q) add(pq, const_cast<float*>(d.states), 1);
            if (d.g_k) add(pk, rstate, 1);
            if (d.g_v && count && !(pad(d.Dk) == pad(d.Dv) && row_tiles(d.Dk) == row_tiles(d.Dv) && blocks(d.Dk, d.Dv) == blocks(d.Dv, d.Dk))) {
                if (int rc = pass<false>(maps, count, s)) return rc;
                count = 0;
            }
            if (d.g_v) add(pv, rstate, 0);
            if (int rc = count ? pass<false>(maps, count, s) : SS_SEQ_OK) return rc;
        }
        auto sum = [&](const float* each, void* out, int D) { return ss_seq_group_sum(each, out, (long long)d.T * d.B * d.Hk, group, D, DT, s); };
        if (group > 1 && d.g_k) if (int rc = sum(each_k, d.g_k, d.Dk)) return rc;
        if (group > 1 && d.g_v) if (int rc = sum(each_v, d.g_v, d.Dv)) return rc;
        return SS_SEQ_OK;
    }
};

}  // namespace

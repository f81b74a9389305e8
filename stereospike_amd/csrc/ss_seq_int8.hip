// ss_seq_int8.hip — 8-bit integer product with a scale for each token (row of a) and channel (row of w).
//
//   out[m][n] = (sum_k a[m][k] w[n][k]) * a_scale[m] * w_scale[n] + bias[n]
//
// The sum is exact in 32 bits for K < 131072 (128 * 128 * 131071 < 2^31), so no order of summation and no split over k changes a result.
//
// Three forms, by a rule on the sizes alone (choose()):
//   rows   at most 32 tokens, or at most 64 channels: the other operand is streamed once from memory, straight into matrix operands (bound by reading it).
//   tile   256 x 256 or 128 x 128 outputs per workgroup, both operands through LDS (bound by the matrix cores and LDS reads).
//   split  the tile form over parts of k into 32-bit partials, joined by a second pass, where there are too few tiles to fill the card.
// Rows that are not aligned to 16 bytes are copied into aligned, zero-padded rows first (tile form) or read unaligned (rows form).
#include "ss_seq_common.hpp"

namespace {

typedef i32x4 __attribute__((aligned(1))) i32x4_u;         // 16 bytes at any address

struct MmArgs {
    const signed char *a, *w;
    long long lda, ldw;
    const float *as, *wsc, *bias;
    void* out;
    long long M;
    int N, K;
};

__device__ __forceinline__ float scaled(int acc, float as, float ws, float bias) { return (float)acc * as * ws + bias; }

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// rows: X has R rows and is read once; Y has S <= 16 MT rows.  v_mfma_i32_16x16x64_i8: lane l holds the 16 consecutive k of row l % 16 that start at
// 16 (l / 16), so one load of a wavefront is 64 consecutive bytes of 16 rows, and the product gives lane l rows 4 (l / 16) .. + 3 of X against row l % 16 of Y.
// The four wavefronts of a workgroup take every fourth 64 k of the same 16 rows of X (256 consecutive bytes of a row at a time) and add up in LDS.
// SWAP: X is a (few channels), else X is w (few tokens).
// (1 x 8192 x 4096, 33.6 MB: 12 us with another weight every call, 2.8 TB/s, 9 with the same one, which the L2 caches hold in part: 64 KB of a workgroup's rows are two
// bursts and their latency.)
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
template <int DT, int MT, bool SWAP> __global__ __launch_bounds__(256) void mm_rows_kernel(const MmArgs p)
{
    __shared__ __attribute__((aligned(16))) int red[3][MT][64][4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const signed char *X = SWAP ? p.a : p.w, *Y = SWAP ? p.w : p.a;
    const long long ldx = SWAP ? p.lda : p.ldw, ldy = SWAP ? p.ldw : p.lda, R = SWAP ? p.M : p.N, S = SWAP ? p.N : p.M;
    const long long x0 = (long long)blockIdx.x * 16, xr = x0 + l16 < R ? x0 + l16 : R - 1;             // rows behind the last: any row, not stored
    const signed char* px = X + xr * ldx + 16 * g;
    const signed char* py[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const long long yr = 16 * t + l16 < S ? 16 * t + l16 : S - 1;
        py[t] = Y + yr * ldy + 16 * g;
    }
    i32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = (i32x4){0, 0, 0, 0};
    const int whole = p.K / 64;                            // steps without an end in them
    constexpr int U = MT == 1 ? 8 : 4;
    int k = wv;
    for (; k + 4 * (U - 1) < whole; k += 4 * U) {
        i32x4 fx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) fx[u] = *reinterpret_cast<const i32x4_u*>(px + 64 * (k + 4 * u));
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx[u], *reinterpret_cast<const i32x4_u*>(py[t] + 64 * (k + 4 * u)), acc[t], 0, 0, 0);
    }
    for (; k < whole; k += 4) {
        const i32x4 fx = *reinterpret_cast<const i32x4_u*>(px + 64 * k);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx, *reinterpret_cast<const i32x4_u*>(py[t] + 64 * k), acc[t], 0, 0, 0);
    }
    if (k == whole && 64 * whole < p.K) {                  // the last, partial step: byte by byte, zeros behind the end
        const int left = p.K - 64 * whole - 16 * g;
        auto tail = [&](const signed char* q) {
            i32x4 v = {0, 0, 0, 0};
            for (int i = 0; i < 16 && i < left; ++i) v[i >> 2] |= (int)(unsigned char)q[64 * whole + i] << (8 * (i & 3));
            return v;
        };
        const i32x4 fx = tail(px);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx, tail(py[t]), acc[t], 0, 0, 0);
    }
    if (wv)
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<i32x4*>(&red[wv - 1][t][lane][0]) = acc[t];
    __syncthreads();
    if (wv) return;
    elem_t<DT>* out = static_cast<elem_t<DT>*>(p.out);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const long long y = 16 * t + l16;
#pragma unroll
        for (int i = 0; i < 3; ++i) acc[t] += *reinterpret_cast<const i32x4*>(&red[i][t][lane][0]);
        if (y >= S) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long long x = x0 + 4 * g + r;
            if (x >= R) continue;
            const long long m = SWAP ? x : y, n = SWAP ? y : x;
            out[m * p.N + n] = narrow<DT>(scaled(acc[t][r], p.as[m], p.wsc[n], p.bias ? p.bias[n] : 0.f));
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------------------
// tile: WM x WN wavefronts, each 32 TI channels x 32 TJ tokens in v_mfma_i32_32x32x32_i8 (lane l: row l % 32, 16 k from 16 (l / 32); taken as w a^T, so a
// lane ends with four consecutive channels of one token).  128 k per step: rows of 128 bytes travel global -> LDS without registers into the other of two
// buffers while this step is computed; granule q of row r lies in slot q ^ (r / 2 % 8), which 16 rows of one granule read without a bank conflict.  The result
// goes through LDS once more, so that stores are whole 128-byte lines.  (8192 x 8192 x 4096, spread codes: 550 GOP in 277 us, 1985 TOP/s; the library's product of
// 8192 cubed reaches 2110.  29920 x 512 x 4608: 141 GOP in 72 us.)  Bound by the matrix cores with LDS reads beside them: 8 fragments feed 8 products.
// ---------------------------------------------------------------------------------------------------------------------------------------------------------
struct TileGrid {
    int tm, tn;                             // tiles
    int steps;                              // k steps of one part
    int* part;                              // [parts][M][N] partial sums, or NULL: finished outputs
    int vec;                                // rows of out take 16-byte stores
};

template <int WM, int WN, int TI, int TJ> struct TileShape {
    static constexpr int BN = WN * TI * 32, BM = WM * TJ * 32, THREADS = WM * WN * 64;
    static constexpr int STAGE = (BM + BN) * 128;
    static constexpr int ROW = TI * 32 * 4 + 16;           // bytes of a token's channels on their way out (32-bit)
};

// one step's rows to LDS, 8 rows per wavefront and instruction
template <int ROWS, int WAVES> __device__ __forceinline__ void tile_load(signed char* __restrict dst, const signed char* __restrict src, const unsigned (&off)[ROWS / 8 / WAVES], int wv)
{
#pragma unroll
    for (int u = 0; u < ROWS / 8 / WAVES; ++u)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + off[u]),
                                         (__attribute__((address_space(3))) void*)(dst + (u * WAVES + wv) * 1024), 16, 0, 0);
}

template <int DT, int WM, int WN, int TI, int TJ>
__global__ __launch_bounds__(WM * WN * 64, 2) void mm_tile_kernel(const MmArgs p, const TileGrid tg)
{
    typedef TileShape<WM, WN, TI, TJ> Sh;
    constexpr int BM = Sh::BM, BN = Sh::BN, WAVES = WM * WN;
    static_assert(WAVES * 32 * Sh::ROW <= 2 * Sh::STAGE, "the result's rows fit the buffers");
    __shared__ __attribute__((aligned(1024))) signed char lds[2 * Sh::STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hi = lane >> 5;
    const int wn = wv % WN, wm = wv / WN;
    // tiles: each of the 8 L2 caches (workgroup i runs on XCD i % 8) gets consecutive tiles, and those run 8 tiles of tokens by 4 of channels at a time
    int tile = blockIdx.x;
    {
        const int total = tg.tm * tg.tn, per = (total + 7) / 8, x = tile & 7, i = tile >> 3;
        const int full = total - 8 * (per - 1);            // XCDs with `per` tiles; the others have one fewer
        tile = x < full ? x * per + i : full * per + (x - full) * (per - 1) + i;
    }
    constexpr int GM = 8;
    const int band = tile / (GM * tg.tn), first = band * GM, high = tg.tm - first < GM ? tg.tm - first : GM;
    const int in = tile - band * GM * tg.tn, mt = first + in % high, nt = in / high;
    const long long m0 = (long long)mt * BM;
    const int n0 = nt * BN;
    const int k_first = blockIdx.y * tg.steps, all = (p.K + 127) / 128, k_last = k_first + tg.steps < all ? k_first + tg.steps : all;

    // this lane's granules: row and place in the row do not change from step to step
    const int r8 = lane >> 3, slot = lane & 7;
    unsigned offa[BM / 8 / WAVES], offw[BN / 8 / WAVES];
#pragma unroll
    for (int u = 0; u < BM / 8 / WAVES; ++u) {
        const int row = (u * WAVES + wv) * 8 + r8;
        const long long left = p.M - m0 - 1;
        offa[u] = (unsigned)((row < left ? row : (int)left) * p.lda) + 16 * (slot ^ (row >> 1 & 7));      // rows behind the last: any row, not stored
    }
#pragma unroll
    for (int u = 0; u < BN / 8 / WAVES; ++u) {
        const int row = (u * WAVES + wv) * 8 + r8, left = p.N - n0 - 1;
        offw[u] = (unsigned)((row < left ? row : left) * p.ldw) + 16 * (slot ^ (row >> 1 & 7));
    }
    const signed char* ga = p.a + m0 * p.lda;
    const signed char* gw = p.w + (long long)n0 * p.ldw;

    i32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    auto fetch = [&](signed char* __restrict dst, const signed char* __restrict a, const signed char* __restrict w, int kt) {
        if ((kt + 1) * 128 <= p.K) {
            tile_load<BM, WAVES>(dst, a + (long long)kt * 128, offa, wv);
            tile_load<BN, WAVES>(dst + BM * 128, w + (long long)kt * 128, offw, wv);
        } else {                                           // granules behind the end of the rows: any granule (a's become zeros below)
            const int most = p.K - 16 - kt * 128;
            unsigned oa[BM / 8 / WAVES], ow[BN / 8 / WAVES];
#pragma unroll
            for (int u = 0; u < BM / 8 / WAVES; ++u) {
                const int row = (u * WAVES + wv) * 8 + r8, q = 16 * (slot ^ (row >> 1 & 7));
                oa[u] = offa[u] - (q > most ? q - most : 0);
            }
#pragma unroll
            for (int u = 0; u < BN / 8 / WAVES; ++u) {
                const int row = (u * WAVES + wv) * 8 + r8, q = 16 * (slot ^ (row >> 1 & 7));
                ow[u] = offw[u] - (q > most ? q - most : 0);
            }
            tile_load<BM, WAVES>(dst, a + (long long)kt * 128, oa, wv);
            tile_load<BN, WAVES>(dst + BM * 128, w + (long long)kt * 128, ow, wv);
        }
    };
    // rows of 32 l32 + ..: (row / 2) % 8 = (l32 / 2) % 8 for every fragment
    const int sw = l32 >> 1 & 7;
    auto step = [&](signed char* __restrict next, const signed char* __restrict cur, const signed char* __restrict a, const signed char* __restrict w, int kt) {
        if (kt + 1 < k_last) fetch(next, a, w, kt + 1);
        const signed char* fa = cur + (wm * TJ * 32 + l32) * 128;
        const signed char* fw = cur + BM * 128 + (wn * TI * 32 + l32) * 128;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int at = ((2 * ks + hi) ^ sw) * 16;
            i32x4 xa[TJ], xw[TI];
#pragma unroll
            for (int i = 0; i < TI; ++i) xw[i] = *reinterpret_cast<const i32x4*>(fw + i * 4096 + at);
#pragma unroll
            for (int j = 0; j < TJ; ++j) xa[j] = *reinterpret_cast<const i32x4*>(fa + j * 4096 + at);
#pragma unroll
            for (int j = 0; j < TJ; ++j)
#pragma unroll
                for (int i = 0; i < TI; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xw[i], xa[j], acc[i][j], 0, 0, 0);
        }
    };
    if (k_first < k_last) fetch(lds, ga, gw, k_first);
    for (int kt = k_first, buf = 0; kt < k_last; ++kt, buf ^= 1) {
        // this step's rows are there, and nobody reads the other buffer any more
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if ((kt + 1) * 128 > p.K) {                        // the rows end within this step: a's granules behind the end become zeros
            for (int i = tid; i < BM * 8; i += Sh::THREADS)
                if (kt * 128 + 16 * ((i & 7) ^ (i >> 4 & 7)) >= p.K) *reinterpret_cast<i32x4*>(lds + buf * Sh::STAGE + i * 16) = (i32x4){0, 0, 0, 0};
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        step(lds + (buf ^ 1) * Sh::STAGE, lds + buf * Sh::STAGE, ga, gw, kt);
    }
    __syncthreads();

    // 32 tokens at a time through this wavefront's part of LDS: lane -> 4 channels of a token; then whole rows
    signed char* mine = lds + wv * 32 * Sh::ROW;
    const int nw = n0 + wn * TI * 32;
    constexpr int ES = sizeof(elem_t<DT>);
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
        const long long mb = m0 + (wm * TJ + j) * 32;
        if (tg.part) {
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<i32x4*>(mine + l32 * Sh::ROW + (i * 32 + q * 8 + 4 * hi) * 4) = (i32x4){acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        } else {
            const float as = mb + l32 < p.M ? p.as[mb + l32] : 0.f;
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    Pack<DT, 4> o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int n = nw + i * 32 + q * 8 + 4 * hi + r, nc = n < p.N ? n : p.N - 1;
                        o.v[r] = narrow<DT>(scaled(acc[i][j][4 * q + r], as, p.wsc[nc], p.bias ? p.bias[nc] : 0.f));
                    }
                    *reinterpret_cast<Pack<DT, 4>*>(mine + l32 * Sh::ROW + (i * 32 + q * 8 + 4 * hi) * ES) = o;
                }
        }
        __builtin_amdgcn_wave_barrier();
        const int es = tg.part ? 4 : ES, lanes = TI * 32 * es / 16;          // lanes of 16 bytes in a row
        for (int r0 = 0; r0 < 32; r0 += 64 / lanes) {
            const int row = r0 + lane / lanes, c = (lane % lanes) * (16 / es);
            const long long m = mb + row;
            const i32x4 v = *reinterpret_cast<const i32x4*>(mine + row * Sh::ROW + c * es);
            if (m >= p.M || nw + c >= p.N) continue;
            signed char* dst = (tg.part ? reinterpret_cast<signed char*>(tg.part + (long long)blockIdx.y * p.M * p.N) : static_cast<signed char*>(p.out)) + (m * p.N + nw + c) * es;
            if (tg.vec) *reinterpret_cast<i32x4*>(dst) = v;
            else if (es == 4) {
#pragma unroll
                for (int e = 0; e < 4; ++e) if (nw + c + e < p.N) reinterpret_cast<int*>(dst)[e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) if (nw + c + e < p.N) reinterpret_cast<unsigned short*>(dst)[e] = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// the parts' sums, scaled; V consecutive outputs of a thread, 8 parts in flight
template <int DT, int V> __global__ __launch_bounds__(256) void mm_join_kernel(const MmArgs p, const int* __restrict__ part, int parts)
{
    struct alignas(4 * V) Sums { int v[V]; };
    const long long mn = p.M * p.N;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < mn; i += (long long)gridDim.x * 256 * V) {
        Sums s = *reinterpret_cast<const Sums*>(part + i);
        for (int k = 1; k < parts; k += 8) {
            Sums x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const Sums*>(part + min(k + u, parts - 1) * mn + i);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k + u < parts)
#pragma unroll
                    for (int e = 0; e < V; ++e) s.v[e] += x[u].v[e];
        }
        const long long m = i / p.N;
        const int n = (int)(i - m * p.N);
        Pack<DT, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = narrow<DT>(scaled(s.v[e], p.as[m], p.wsc[n + e], p.bias ? p.bias[n + e] : 0.f));
        *reinterpret_cast<Pack<DT, V>*>(static_cast<elem_t<DT>*>(p.out) + i) = o;
    }
}

// rows of any alignment -> rows of kp bytes (a multiple of 16), zeros behind the end
__global__ __launch_bounds__(256) void mm_align_kernel(const signed char* __restrict__ src, long long ld, signed char* __restrict__ dst, long long rows, int K, int kp)
{
    const int gr = kp / 16;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * gr; i += (long long)gridDim.x * 256) {
        const long long r = i / gr;
        const int k = (int)(i - r * gr) * 16;
        i32x4 v = {0, 0, 0, 0};
        if (k + 16 <= K) v = *reinterpret_cast<const i32x4_u*>(src + r * ld + k);
        else
            for (int e = 0; e < 16 && k + e < K; ++e) v[e >> 2] |= (int)(unsigned char)src[r * ld + k + e] << (8 * (e & 3));
        *reinterpret_cast<i32x4*>(dst + r * kp + k) = v;
    }
}

struct MmPlan {
    int form;                               // 0 rows (X = w), 1 rows (X = a), 2 tile of 128, 3 tile of 256
    int parts, steps;
    bool align_a, align_w;
    long long ws;                           // ints: [parts][M][N], then the aligned copies
    int kp;
};

MmPlan choose(long long M, int N, int K, bool a_ok, bool w_ok)
{
    MmPlan r{};
    // few rows on one side: the other side's bytes are all that matters.  (N = K = 4096: 33 rows streamed 11.3 us, tiles 11.8; 48 rows 12.7 and 12.6; 64 rows 14.5
    // and 13.5; N = 512, K = 4608: 64 rows 14.6 and 10.5.  Few channels are streamed up to 64: 4096 rows, 64 channels 13.7 us, tiles 14.3.)
    if (M <= 32 && M <= N) { r.form = 0; return r; }
    if (N <= 64) { r.form = 1; return r; }
    const long long t256 = ((M + 255) / 256) * ((N + 255) / 256), t128 = ((M + 127) / 128) * ((N + 127) / 128);
    const int all = (K + 127) / 128;
    // 256 x 256 reads each operand half as often as 128 x 128, but needs a tile for most CUs.  (K = 4096: 48 tiles 58 us, those of 128 27; 80 tiles 59 and 35; 176
    // tiles 60 to 62 and 62; 208 tiles 61 and 73; 256 tiles 73 and 83.)
    r.form = t256 >= 176 ? 3 : 2;
    r.parts = 1;
    if (r.form == 2 && t128 < 256) {
        // Parts of k: the count with the least estimated time in us, 0.75 for a step of 128 k and 2 around them, 4 for the joining launch and the partials' way out
        // and in at 4 TB/s; two workgroups fit a CU.  (512 x 512 x 4608: whole 24.6 us, 6 parts 13.0; 256 x 256 x 16384: 74 and 14.8 in 32 parts; 1536 x 1536 x 1024:
        // whole 10.6, two parts 20.7.)
        double least = 0.;
        for (int n = 1; n <= 512 / t128 && n <= all; ++n) {
            const double t = ((all + n - 1) / n) * 0.75 + 2. + (n > 1 ? 4. + (double)n * M * N * 8e-6 / 4. : 0.);
            if (n == 1 || t < least) { r.parts = n; least = t; }
        }
    }
    r.steps = (all + r.parts - 1) / r.parts;
    r.parts = (all + r.steps - 1) / r.steps;
    r.kp = (K + 15) / 16 * 16;
    r.align_a = !a_ok;
    r.align_w = !w_ok;
    const long long part = r.parts > 1 ? (long long)r.parts * M * N : 0;
    r.ws = (part + 3) / 4 * 4 + (r.align_a ? M * (long long)(r.kp / 4) : 0) + (r.align_w ? N * (long long)(r.kp / 4) : 0);
    return r;
}

bool row_ok(const signed char* p, long long ld, int K) { return K % 16 == 0 && ld % 16 == 0 && aligned(p, 16) && ld < (1 << 23); }

template <int DT, int WM, int WN, int TI, int TJ> int tiles(const MmArgs& p, const MmPlan& r, int* part, hipStream_t s)
{
    typedef TileShape<WM, WN, TI, TJ> Sh;
    TileGrid tg{(int)((p.M + Sh::BM - 1) / Sh::BM), (p.N + Sh::BN - 1) / Sh::BN, r.steps, r.parts > 1 ? part : nullptr, 0};
    const int es = tg.part ? 4 : (int)sizeof(elem_t<DT>);
    tg.vec = p.N * (long long)es % 16 == 0 && aligned(tg.part ? (const void*)tg.part : p.out, 16);
    mm_tile_kernel<DT, WM, WN, TI, TJ><<<dim3((unsigned)(tg.tm * tg.tn), (unsigned)r.parts), Sh::THREADS, 0, s>>>(p, tg);
    if (int rc = launched()) return rc;
    if (tg.part) {
        const bool four = p.N % 4 == 0 && aligned(p.out, 16);
        const long long want = (p.M * p.N / (four ? 4 : 1) + 255) / 256;
        const unsigned grid = (unsigned)(want < 4096 ? want : 4096);
        if (four) mm_join_kernel<DT, 4><<<grid, 256, 0, s>>>(p, tg.part, r.parts);
        else mm_join_kernel<DT, 1><<<grid, 256, 0, s>>>(p, tg.part, r.parts);
        return launched();
    }
    return SS_SEQ_OK;
}

template <int DT> int run(MmArgs p, const MmPlan& r, int* ws, hipStream_t s)
{
    if (r.form < 2) {
        const long long X = r.form ? p.M : p.N, S = r.form ? p.N : p.M;
        const unsigned grid = (unsigned)((X + 15) / 16);
        auto go = [&](auto MT) {
            if (r.form) mm_rows_kernel<DT, MT.value, true><<<grid, 256, 0, s>>>(p);
            else mm_rows_kernel<DT, MT.value, false><<<grid, 256, 0, s>>>(p);
            return launched();
        };
        return S <= 16 ? go(std::integral_constant<int, 1>()) : S <= 32 ? go(std::integral_constant<int, 2>()) : go(std::integral_constant<int, 4>());
    }
    int* part = ws;
    signed char* copy = reinterpret_cast<signed char*>(ws + (r.parts > 1 ? ((long long)r.parts * p.M * p.N + 3) / 4 * 4 : 0));
    auto align = [&](const signed char*& src, long long& ld, long long rows) {
        const long long want = (rows * (r.kp / 16) + 255) / 256;
        mm_align_kernel<<<(unsigned)(want < 8192 ? want : 8192), 256, 0, s>>>(src, ld, copy, rows, p.K, r.kp);
        src = copy;
        ld = r.kp;
        copy += rows * r.kp;
        return launched();
    };
    if (r.align_a) if (int rc = align(p.a, p.lda, p.M)) return rc;
    if (r.align_w) if (int rc = align(p.w, p.ldw, p.N)) return rc;
    p.K = r.kp;
    return r.form == 3 ? tiles<DT, 2, 4, 2, 4>(p, r, part, s) : tiles<DT, 2, 2, 2, 2>(p, r, part, s);
}

}  // namespace

extern "C" {

long long ss_seq_int8_linear_ws_ints(const signed char* a, long long lda, const signed char* w, long long ldw, long long M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return choose(M, N, K, row_ok(a, lda, K), row_ok(w, ldw, K)).ws;
}

int ss_seq_int8_linear(const signed char* a, long long lda, const float* a_scale, const signed char* w, long long ldw, const float* w_scale,
                       const float* bias, void* out, long long M, int N, int K, int out_dtype, int* ws, void* stream)
{
    if (M < 0 || M > (1 << 27) || N <= 0 || N > (1 << 27) || ((M + 127) / 128) * ((N + 127ll) / 128) >= (1 << 24) || K <= 0 || K >= 131072 || lda < 0 || ldw < 0) return SS_SEQ_EINVAL;
    if (out_dtype != SS_SEQ_F32 && out_dtype != SS_SEQ_F16 && out_dtype != SS_SEQ_BF16) return SS_SEQ_EINVAL;
    if (M == 0) return SS_SEQ_OK;
    if (!a || !a_scale || !w || !w_scale || !out) return SS_SEQ_EINVAL;
    const MmArgs p{a, w, lda, ldw, a_scale, w_scale, bias, out, M, N, K};
    const MmPlan r = choose(M, N, K, row_ok(a, lda, K), row_ok(w, ldw, K));
    if (r.ws && (!ws || !aligned(ws, 16))) return SS_SEQ_EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return out_dtype == SS_SEQ_F32 ? run<SS_SEQ_F32>(p, r, ws, s) : out_dtype == SS_SEQ_F16 ? run<SS_SEQ_F16>(p, r, ws, s) : run<SS_SEQ_BF16>(p, r, ws, s);
}

}  // extern "C"

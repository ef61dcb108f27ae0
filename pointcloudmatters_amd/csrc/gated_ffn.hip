// gated_ffn.hip -- the gated feed-forward block and its backward pass.
//
//   a = x Wg^T + bg,  u = x Wu^T + bu,  h = act(a) * u,  y = h Wd^T + bd            (act: SiLU, GELU (erf) or ReLU)
//   dh = dy Wd,  da = dh * u * act'(a),  du = dh * act(a),
//   dx = da Wg + du Wu,  dWg = da^T x,  dWu = du^T x,  dWd = dy^T h,  bias gradients = column sums.
//
// Every product is one tile engine (v_mfma_f32_32x32x16_bf16, fp32 accumulators) with two operand forms: contracted index contiguous in
// memory (read from LDS as 16-byte pieces), or the other index contiguous (read through ds_read_b64_tr_b16, which transposes on the
// way).  The element-wise parts are epilogues: both projections share one launch -- a wave's 64 output columns are 32 of the gate and
// the same 32 of the up projection, so act(a) * u needs no exchange -- and so do dh, da and du.  a, u, h, da, du are rounded to bf16
// where they are stored as operands of the next product (one half step, 2^-8 relative at most); outputs are rounded once.
//
// a, u, h have rows of Fp = F rounded up to 64 values; the columns from F on are zero, so contractions over F need no edge.  Matrices
// whose rows do not start at 16-byte boundaries (an odd width) are copied into padded rows first, one launch for all of a call's.
#include "pcm_attn.hpp"

namespace {

constexpr int GF_BK = 32;

// A matrix of 2-byte values, rows at `ld`; rows from `split` on come from the second part (gate | up weights).
struct GfMat {
    const u16 *p0, *p1;
    long ld;
    int split, rows0, rows1, cols;  // rows of each part, columns (a multiple of 8)
};

struct GfParams {
    GfMat a, b;
    long M, N, K;
    int act, nsplit;
    long F, Fp, osplit;          // weight gradients: output rows from osplit on go to out1; F rows each
    const u16 *bias0, *bias1;
    u16 *out, *out1, *h;         // see the epilogues
    const u16 *ea, *eu;
    long ldo;
    float *part;
};

enum { EP_GLU, EP_OUT, EP_DGLU, EP_WGRAD };

// Phi(a) = (1 + erf(a / sqrt 2)) / 2 and exp(-a^2 / 2): erfc(x) = (t (a1 + t (a2 + .. a5 t^4))) exp(-x^2), t = 1 / (1 + p x), x >= 0
// (Abramowitz and Stegun 7.1.26, |error| <= 1.5e-7): one exponential, which the derivative needs as well, and one reciprocal, where the
// library's erff takes three times as many operations -- with one evaluation per hidden value that was a fifth of the launch.
__device__ __forceinline__ float2 gf_phi(float a)
{
    const float x = fabsf(a) * 0.70710678118654752f, e = __expf(-x * x), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
    float q = 1.061405429f;
    q = __builtin_fmaf(q, t, -1.453152027f), q = __builtin_fmaf(q, t, 1.421413741f);
    q = __builtin_fmaf(q, t, -0.284496736f), q = __builtin_fmaf(q, t, 0.254829592f);
    const float half_erfc = 0.5f * q * t * e;
    return make_float2(a < 0.f ? half_erfc : 1.f - half_erfc, e);
}
__device__ __forceinline__ float gf_act(float a, int act)
{
    if (act == 0) return a * __builtin_amdgcn_rcpf(1.f + __expf(-a));
    if (act == 1) return a * gf_phi(a).x;
    return a > 0.f ? a : (a == a ? 0.f : a);
}
// act(a) and act'(a)
__device__ __forceinline__ float2 gf_act_grad(float a, int act)
{
    if (act == 0) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-a));
        return make_float2(a * s, s * __builtin_fmaf(a, 1.f - s, 1.f));
    }
    if (act == 1) {
        const float2 g = gf_phi(a);
        return make_float2(a * g.x, __builtin_fmaf(a * 0.39894228040143267f, g.y, g.x));
    }
    return make_float2(a > 0.f ? a : (a == a ? 0.f : a), a > 0.f ? 1.f : 0.f);
}
__device__ __forceinline__ u16 gf_bf(float v) { return (u16)cvt_pk_bf16(v, 0.f); }
__device__ __forceinline__ uint4 gf_bf8(const float (&v)[8])
{
    return make_uint4(cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]), cvt_pk_bf16(v[4], v[5]), cvt_pk_bf16(v[6], v[7]));
}
__device__ __forceinline__ void gf_f8(const uint4 &w, float (&v)[8])
{
    v[0] = __uint_as_float(w.x << 16), v[1] = __uint_as_float(w.x & 0xFFFF0000u), v[2] = __uint_as_float(w.y << 16), v[3] = __uint_as_float(w.y & 0xFFFF0000u);
    v[4] = __uint_as_float(w.z << 16), v[5] = __uint_as_float(w.z & 0xFFFF0000u), v[6] = __uint_as_float(w.w << 16), v[7] = __uint_as_float(w.w & 0xFFFF0000u);
}

typedef s4 __attribute__((address_space(3))) * gf_lds_s4;
typedef __attribute__((address_space(3))) void *gf_lds_p;
typedef const __attribute__((address_space(1))) void *gf_glb_p;
__device__ uint4 gf_zeros;  // what pieces outside a matrix are read from

// One operand's tile of GF_BK contracted values, ROWS values of the operand's own index.
// COL false: [ROWS][32], contracted index contiguous, four 16-byte pieces a row.  COL true: [32][ROWS], ROWS / 8 pieces a row.
// global_load_lds writes a wave's 64 pieces to consecutive addresses, so the layout cannot be padded; instead the piece a slot holds is
// permuted (the lane picks its source).  64 banks of 4 bytes: ds_read_b128 serves the lanes 0-3, 12-15, 20-23, 24-27 of 32 together, then the
// other 16, and rows of 64 bytes share banks every 4, so the row's bits 2 and 3 pick the slot; ds_read_b64_tr_b16 serves 32 lanes together,
// 64 bytes of each of 4 neighbouring contracted rows, which have to lie in different 64-byte groups.
template <bool COL, int ROWS>
struct GfTile {
    static constexpr int PIECES = COL ? ROWS / 8 : 4, SIZE = ROWS * GF_BK, LOADS = SIZE / 8 / 256;
    static __device__ __forceinline__ int swz(int r)
    {
        if constexpr (!COL) return (r >> 2) & 3;
        else if constexpr (ROWS >= 128) return (r & 3) << 2;
        else return ((r >> 1) & 1) << 2;
    }
    // The thread's n-th piece stands n * NROWS tile rows below its first (the permutation is the same: NROWS is a multiple of 8).
    static constexpr int NROWS = 256 / PIECES;
    const u16 *base;  // the first piece at contracted index 0
    long step;        // values from one piece to the next
    int left, koff;   // COL false: matrix rows left from the first piece's on; true: 1 or 0, columns in or outside.  koff: contracted index inside the tile
    int each;         // matrix rows from one piece to the next (GLU: 64 virtual rows are 32)

    __device__ __forceinline__ void init(const GfMat &m, long i0, bool glu)
    {
        const int r = (int)threadIdx.x / PIECES, c = ((int)threadIdx.x - r * PIECES) ^ swz(r);
        if constexpr (COL) {
            const long col = i0 + 8 * c;
            left = col < m.cols, koff = r, each = 0, step = NROWS * m.ld;
            base = m.p0 + (left ? col : 0) + r * m.ld;
        } else {
            long row = i0 + r;
            if (glu) row = (row >> 6) * 32 + (row & 31) + ((row & 32) ? m.split : 0);  // virtual row -> gate | up weight row
            const bool second = row >= m.split;
            const long rr = second ? row - m.split : row;
            left = (int)((second ? m.rows1 : m.rows0) - rr), koff = 8 * c, each = glu ? NROWS / 2 : NROWS, step = each * m.ld;
            base = (second ? m.p1 : m.p0) + rr * m.ld + 8 * c;
        }
    }
    // the tile of contracted indices k .. k + 31 on its way into LDS
    __device__ __forceinline__ void load(const GfMat &m, u16 *tile, long k, long kend) const
    {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        // a tile never straddles the parts: `split` is a multiple of 64
        const bool second = COL && k >= m.split;
        const int rest = (int)((COL ? min(kend, second ? m.split + (long)m.rows1 : (long)m.rows0) : kend) - k);
        const long at = COL ? k * m.ld + (second ? (long)(m.p1 - m.p0) - (long)m.split * m.ld : 0) : k;
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const bool in = COL ? left && koff + n * NROWS < rest : n * each < left && koff < rest;
            const u16 *src = in ? base + (at + n * step) : (const u16 *)&gf_zeros;
            __builtin_amdgcn_global_load_lds((gf_glb_p)src, (gf_lds_p)(tile + (n * 256 + wave * 64) * 8), 16, 0, 0);
        }
    }
    // operand of rows i .. i + 31, contracted values 16 kk .. + 15
    static __device__ __forceinline__ bf8 operand(const u16 *t, int i, int kk, int lane)
    {
        const int h = lane >> 5;
        if constexpr (COL) {
            const int p = lane & 15, r = 16 * kk + 8 * h + (p >> 2), c = (i >> 3) + 2 * ((lane >> 4) & 1) + ((p >> 1) & 1);
            const u16 *q = t + (r * PIECES + (c ^ swz(r))) * 8 + 4 * (p & 1);
            const u16 *q4 = t + ((r + 4) * PIECES + (c ^ swz(r + 4))) * 8 + 4 * (p & 1);
            return cat8(__builtin_amdgcn_ds_read_tr16_b64_v4i16((gf_lds_s4)q), __builtin_amdgcn_ds_read_tr16_b64_v4i16((gf_lds_s4)q4));
        } else {
            const int r = i + (lane & 31), c = 2 * kk + h;
            return lds_bf8(t + (r * PIECES + (c ^ swz(r))) * 8);
        }
    }
};

// vmcnt(N) lgkmcnt(0): all but the wave's last N requests have arrived, its LDS reads are done
template <int N>
__device__ __forceinline__ void gf_wait()
{
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
}

// The tile engine.  4 waves, 2 x 2; a wave owns MI x NI tiles of 32 x 32.  Three LDS buffers of 32 contracted values each: in step t all
// operands of tile t come out of LDS, tile t + 2's pieces are requested straight into the buffer that step t - 1 read
// (global_load_lds: no registers, no LDS write instructions), then the step's matrix instructions run.  One barrier a step, which waits
// for tile t alone: tile t + 1 stays in flight.  (With one tile in flight a step took 2800 clocks for two workgroups on a compute unit, 1024 of
// matrix work: every tile row's first reader waits for memory, and the others with it.)  The buffers are three variables, so that the
// compiler can tell the reads of one from the requests into another and inserts no wait of its own between them.
template <int EP, bool ACOL, bool BCOL, int MI, int NI>
__global__ void __launch_bounds__(256, 2) pcm_gated_gemm_kernel(GfParams P)
{
    constexpr int BM = 64 * MI, BN = 64 * NI, COLS = 32 * NI, SLAB = COLS + 4;
    typedef GfTile<ACOL, BM> TA;
    typedef GfTile<BCOL, BN> TB;
    constexpr int STAGE = (TA::SIZE + TB::SIZE) * 2, BYTES = STAGE > 2 * 32 * SLAB * 4 ? STAGE : 2 * 32 * SLAB * 4, LOADS = TA::LOADS + TB::LOADS;
    __shared__ __attribute__((aligned(1024))) unsigned char sm0[BYTES], sm1[BYTES], sm2[BYTES];
    const int M = (int)P.M, N = (int)P.N;
    const long mt = (P.M + BM - 1) / BM, nt = (P.N + BN - 1) / BN, items = mt * nt * P.nsplit, per = (items + 7) / 8;
    const long item = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);  // one XCD's L2 sees consecutive tiles
    if (item >= items) return;
    const long m0 = item / nt % mt * BM, n0 = item % nt * BN, split = item / (nt * mt);
    const long kt = (P.K + GF_BK - 1) / GF_BK, kper = (kt + P.nsplit - 1) / P.nsplit * GF_BK;
    const long k0 = split * kper, kend = k0 + kper < P.K ? k0 + kper : P.K;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = (wave >> 1) * 32 * MI, wn = (wave & 1) * COLS;
    f16v acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    TA ga;
    TB gb;
    ga.init(P.a, m0, false), gb.init(P.b, n0, EP == EP_GLU);
    // every step requests a tile, behind the end one of zeros: the count of requests in flight stays the same
    const auto request = [&](unsigned char *sm, long k) {
        ga.load(P.a, (u16 *)sm, k, kend), gb.load(P.b, (u16 *)sm + TA::SIZE, k, kend);
    };
    const auto step = [&](const unsigned char *cur, unsigned char *free, long k) {
        gf_wait<LOADS>();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const u16 *ta = (const u16 *)cur, *tb = ta + TA::SIZE;
        bf8 a[2][MI], b[2][NI];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
            for (int i = 0; i < MI; ++i) a[kk][i] = TA::operand(ta, wm + 32 * i, kk, lane);
#pragma unroll
            for (int j = 0; j < NI; ++j) b[kk][j] = TB::operand(tb, wn + 32 * j, kk, lane);
        }
        request(free, k + 2 * GF_BK);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = PCM_MFMA16(a[kk][i], b[kk][j], acc[i][j]);
    };
    if (k0 < kend) {
        request(sm0, k0);
        request(sm1, k0 + GF_BK);
        long k = k0;
        for (; k + 2 * GF_BK < kend; k += 3 * GF_BK) {
            step(sm0, sm2, k);
            step(sm1, sm0, k + GF_BK);
            step(sm2, sm1, k + 2 * GF_BK);
        }
        if (k < kend) step(sm0, sm2, k);
        if (k + GF_BK < kend) step(sm1, sm0, k + GF_BK);
    }
    gf_wait<0>();  // the last requests (of zeros) must not land in the slabs
    __syncthreads();
    // Epilogue: 32 rows at a time through a slab of the wave's own (an accumulator holds a column a lane), out of it 8 neighbouring
    // columns a lane, the same ones in every pass: 16-byte accesses to everything that is read and written beside the products.
    float *const slab = (float *)(wave < 2 ? sm0 : sm1) + (wave & 1) * 32 * SLAB;
    constexpr int GROUPS = EP == EP_GLU ? 4 : COLS / 8;  // groups of 8 columns a row
    static_assert(64 % GROUPS == 0, "a lane's columns are the same in every pass");
    const int c = 8 * (lane % GROUPS), r0 = lane / GROUPS, col = (int)(EP == EP_GLU ? (n0 + wn) / 2 : n0 + wn) + c;
    const int width = EP == EP_GLU || EP == EP_DGLU ? (int)P.F : N;  // columns that carry values; Fp of them are written in the hidden forms
    const bool vec = P.ldo % 8 == 0 && (((uintptr_t)P.out | (uintptr_t)P.out1) & 15) == 0 && col + 8 <= width;
    float bias0[8], bias1[8];  // EP_DGLU: the column sums of da, du
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        bias0[e] = (EP == EP_GLU || EP == EP_OUT) && P.bias0 && P.nsplit == 1 && col + e < width ? bf2f(P.bias0[col + e]) : 0.f;
        bias1[e] = EP == EP_GLU && P.bias1 && col + e < width ? bf2f(P.bias1[col + e]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) slab[crow(r, lane) * SLAB + 32 * j + (lane & 31)] = acc[i][j][r];
        __builtin_amdgcn_wave_barrier();  // the wave's LDS operations complete in order
#pragma unroll
        for (int g = 0; g < 32 * GROUPS / 64; ++g) {
            const int r = r0 + g * (64 / GROUPS);
            const long row = m0 + wm + 32 * i + r;
            if ((int)row >= M) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = slab[r * SLAB + c + e];
            if constexpr (EP == EP_GLU) {
                float u[8], hv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = slab[r * SLAB + 32 + c + e];
#pragma unroll
                for (int e = 0; e < 8; ++e) {  // columns from F on: weights and biases are zeros, and so are a, u and h
                    v[e] += bias0[e], u[e] += bias1[e];
                    hv[e] = gf_act(v[e], P.act) * u[e];
                }
                const long at = row * P.Fp + col;
                if (P.out) *(uint4 *)(P.out + at) = gf_bf8(v), *(uint4 *)(P.out1 + at) = gf_bf8(u);
                *(uint4 *)(P.h + at) = gf_bf8(hv);
            } else if constexpr (EP == EP_DGLU) {
                if (col >= P.Fp) continue;
                float a[8], u[8];
                gf_f8(*(const uint4 *)(P.ea + row * P.Fp + col), a), gf_f8(*(const uint4 *)(P.eu + row * P.Fp + col), u);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 g2 = gf_act_grad(a[e], P.act);
                    const float dh = col + e < width ? v[e] : 0.f;
                    v[e] = dh * u[e] * g2.y, u[e] = dh * g2.x;
                    bias0[e] += v[e], bias1[e] += u[e];
                }
                u16 *o = P.out + row * 2 * P.Fp + col;
                *(uint4 *)o = gf_bf8(v), *(uint4 *)(o + P.Fp) = gf_bf8(u);
            } else {
                if (col >= N) continue;
                if (P.nsplit > 1) {
                    float *o = P.part + (split * P.M + row) * P.N + col;
                    if (col + 8 <= N && N % 4 == 0) {
                        *(float4 *)o = make_float4(v[0], v[1], v[2], v[3]), *(float4 *)(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + e < N) o[e] = v[e];
                    }
                    continue;
                }
                const bool second = row >= P.osplit;
                const long rr = second ? row - P.osplit : row;
                if (rr >= P.F) continue;
                u16 *o = (second ? P.out1 : P.out) + rr * P.ldo + col;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += bias0[e];
                if (vec) *(uint4 *)o = gf_bf8(v);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e < N) o[e] = gf_bf(v[e]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if constexpr (EP == EP_DGLU) {
        if (P.part == nullptr) return;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            for (int d = GROUPS; d < 64; d <<= 1) bias0[e] += __shfl_xor(bias0[e], d), bias1[e] += __shfl_xor(bias1[e], d);
        if (lane >= GROUPS || col >= P.Fp) return;
        float *o = P.part + (m0 / (32 * MI) + (wave >> 1)) * 2 * P.Fp + col;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = bias0[e], o[P.Fp + e] = bias1[e];
    }
}

// out = sum of the splits in split order (+ bias)
__global__ void __launch_bounds__(256) pcm_gated_join_kernel(GfParams P)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= P.M * P.N) return;
    const long row = i / P.N, n = i - row * P.N;
    const bool second = row >= P.osplit;
    const long rr = second ? row - P.osplit : row;
    if (rr >= P.F) return;
    float s = P.bias0 ? bf2f(P.bias0[n]) : 0.f;
    for (int k = 0; k < P.nsplit; ++k) s += P.part[(long)k * P.M * P.N + i];
    (second ? P.out1 : P.out)[rr * P.ldo + n] = gf_bf(s);
}

// Bias gradients.  The sums of da | du over a wave's rows leave the epilogue that forms them (one partial row per wave row: reading
// da | du again would cost as much as writing it); dy is summed here, `slots` partial rows of fixed row ranges.  Then one wave per 16
// columns, 4 lanes per column over interleaved partial rows, joined by two exchanges: the order never changes.
struct GfSums {
    const u16 *g;
    long ld, rows;
    int C[2], slots[2];
    const float *part[2];
    float *part1;
    u16 *out[3];
    int E, F, Fp;
};
__global__ void __launch_bounds__(256) pcm_gated_colsum_kernel(GfSums P)
{
    const int c = (int)blockIdx.x * 512 + 2 * (int)threadIdx.x;
    if (c >= P.C[1]) return;
    const long per = (P.rows + P.slots[1] - 1) / P.slots[1], r0 = blockIdx.y * per, r1 = r0 + per < P.rows ? r0 + per : P.rows;
    float a = 0.f, b = 0.f;
#pragma unroll 8
    for (long r = r0; r < r1; ++r) {
        const uint32_t w = *(const uint32_t *)(P.g + r * P.ld + c);
        a += __uint_as_float(w << 16), b += __uint_as_float(w & 0xFFFF0000u);
    }
    *(float2 *)(P.part1 + (long)blockIdx.y * P.C[1] + c) = make_float2(a, b);
}
__global__ void __launch_bounds__(256) pcm_gated_colsum_join_kernel(GfSums P)
{
    const int j = blockIdx.y, lane = threadIdx.x & 63, c = ((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6)) * 16 + (lane & 15);
    float s = 0.f;
    if (c < P.C[j]) {
#pragma unroll 8
        for (int k = lane >> 4; k < P.slots[j]; k += 4) s += P.part[j][(long)k * P.C[j] + c];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane >= 16 || c >= P.C[j]) return;
    if (j == 1) {
        if (c < P.E) P.out[2][c] = gf_bf(s);
    } else if (c < P.F) {
        P.out[0][c] = gf_bf(s);
    } else if (c >= P.Fp && c - P.Fp < P.F) {
        P.out[1][c - P.Fp] = gf_bf(s);
    }
}

// rows copied into padded rows (zero behind the last column): up to five matrices in one launch
struct GfPack {
    const u16 *src[5];
    u16 *dst[5];
    long rows[5], ld[5], end[5];  // end: running sum of destination values / 8
    int cols[5], ldp[5], n;
};
__global__ void __launch_bounds__(256) pcm_gated_pack_kernel(GfPack P)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    int j = 0;
    while (j < P.n && i >= P.end[j]) ++j;
    if (j == P.n) return;
    const long e = (i - (j ? P.end[j - 1] : 0)) * 8, r = e / P.ldp[j];
    const int c = (int)(e - r * P.ldp[j]);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const u16 *s = P.src[j] + r * P.ld[j] + c + 2 * k;
        const uint32_t lo = c + 2 * k < P.cols[j] ? s[0] : 0, hi = c + 2 * k + 1 < P.cols[j] ? s[1] : 0;
        w[k] = lo | (hi << 16);
    }
    *(uint4 *)(P.dst[j] + e) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- few rows: one token of a rollout ----------------------------------------------------------------------------------------------
// With up to 8 rows the weights are all there is to read and a 64-row tile would leave most of the chip idle: one wave per output column
// reads that column's weight row once, 16 bytes a lane, and keeps all rows' sums.  Rows of any alignment (no padded copies).
struct __attribute__((packed, aligned(2))) GfAny16 {
    uint32_t w[4];
};
__device__ __forceinline__ void gf_any8(const u16 *p, float (&v)[8])
{
    const GfAny16 a = *(const GfAny16 *)p;
    gf_f8(make_uint4(a.w[0], a.w[1], a.w[2], a.w[3]), v);
}
constexpr int GF_FEW = 8;

// a, u, h of one hidden column
template <int NR>
__global__ void __launch_bounds__(256) pcm_gated_few_in_kernel(GfParams P)
{
    const int lane = threadIdx.x & 63, f = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), E = (int)P.K, R = (int)P.M;
    if (f >= P.Fp) return;
    float sg[NR], su[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) sg[r] = su[r] = 0.f;
    if (f < P.F) {
        const u16 *wg = P.b.p0 + f * P.b.ld, *wu = P.b.p1 + f * P.b.ld;
#pragma unroll 2
        for (int c = 8 * lane; c + 8 <= E; c += 512) {
            float g[8], u[8];
            gf_any8(wg + c, g), gf_any8(wu + c, u);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float x[8];
                if (r < R) {
                    gf_any8(P.a.p0 + r * P.a.ld + c, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sg[r] = __builtin_fmaf(x[e], g[e], sg[r]), su[r] = __builtin_fmaf(x[e], u[e], su[r]);
                }
            }
        }
        const int tail = (E & ~7) + lane;
        if (tail < E)
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (r < R) {
                    const float x = bf2f(P.a.p0[r * P.a.ld + tail]);
                    sg[r] = __builtin_fmaf(x, bf2f(wg[tail]), sg[r]), su[r] = __builtin_fmaf(x, bf2f(wu[tail]), su[r]);
                }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float g = wave_sum(sg[r]), u = wave_sum(su[r]);
        if (lane == r) sg[0] = g, su[0] = u;  // lane r finishes row r
    }
    if (lane >= R) return;
    const bool in = f < P.F;
    const float a = in ? sg[0] + (P.bias0 ? bf2f(P.bias0[f]) : 0.f) : 0.f, u = in ? su[0] + (P.bias1 ? bf2f(P.bias1[f]) : 0.f) : 0.f;
    const long at = lane * P.Fp + f;
    if (P.out) P.out[at] = gf_bf(a), P.out1[at] = gf_bf(u);
    P.h[at] = gf_bf(gf_act(a, P.act) * u);
}

// y of one output column
template <int NR>
__global__ void __launch_bounds__(256) pcm_gated_few_out_kernel(GfParams P)
{
    const int lane = threadIdx.x & 63, n = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), K = (int)P.K, R = (int)P.M;
    if (n >= P.N) return;
    float s[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) s[r] = 0.f;
    const u16 *w = P.b.p0 + n * P.b.ld;
#pragma unroll 4
    for (int c = 8 * lane; c + 8 <= K; c += 512) {
        float v[8];
        gf_any8(w + c, v);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float x[8];
            if (r < R) {
                gf_f8(*(const uint4 *)(P.a.p0 + r * P.a.ld + c), x);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[r] = __builtin_fmaf(x[e], v[e], s[r]);
            }
        }
    }
    const int tail = (K & ~7) + lane;
    if (tail < K)
#pragma unroll
        for (int r = 0; r < NR; ++r)
            if (r < R) s[r] = __builtin_fmaf(bf2f(P.a.p0[r * P.a.ld + tail]), bf2f(w[tail]), s[r]);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const float t = wave_sum(s[r]);
        if (lane == r) s[0] = t;
    }
    if (lane < R) P.out[lane * P.ldo + n] = gf_bf(s[0] + (P.bias0 ? bf2f(P.bias0[n]) : 0.f));
}

#define GF_BY_ROWS(kernel, R, grid, s, P)                                                       \
    do {                                                                                        \
        if ((R) == 1) hipLaunchKernelGGL((kernel<1>), dim3(grid), dim3(256), 0, s, P);          \
        else if ((R) <= 2) hipLaunchKernelGGL((kernel<2>), dim3(grid), dim3(256), 0, s, P);     \
        else if ((R) <= 4) hipLaunchKernelGGL((kernel<4>), dim3(grid), dim3(256), 0, s, P);     \
        else hipLaunchKernelGGL((kernel<GF_FEW>), dim3(grid), dim3(256), 0, s, P);              \
    } while (0)

long gf_up(long v, long m) { return (v + m - 1) / m * m; }
bool gf_fits(const void *p, long ld, int cols) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && cols % 8 == 0; }

// Lays out the copies a call needs: `get` returns the matrix to use in place of p.
struct GfPacker {
    GfPack P;
    char *at, *end;
    GfPacker(void *ws, long bytes) : at((char *)ws), end((char *)ws + bytes) { P.n = 0; }
    const u16 *get(const void *p, long rows, int cols, long &ld)
    {
        if (gf_fits(p, ld, cols)) return (const u16 *)p;
        const int ldp = (int)gf_up(cols, 8), j = P.n++;
        const long bytes = gf_up(rows * ldp * 2, 256);
        P.src[j] = (const u16 *)p, P.dst[j] = (u16 *)at, P.rows[j] = rows, P.ld[j] = ld, P.cols[j] = cols, P.ldp[j] = ldp;
        P.end[j] = (j ? P.end[j - 1] : 0) + rows * ldp / 8;
        at += bytes;
        ld = ldp;
        return P.dst[j];
    }
    bool room() const { return at <= end; }
    void run(hipStream_t s)
    {
        if (P.n) hipLaunchKernelGGL(pcm_gated_pack_kernel, dim3((unsigned)((P.end[P.n - 1] + 255) / 256)), dim3(256), 0, s, P);
    }
};

GfMat gf_mat(const u16 *p, long ld, long rows, long cols) { return GfMat{p, p, ld, 0x7FFFFFFF, (int)rows, 0, (int)cols}; }
GfMat gf_mat2(const u16 *p0, const u16 *p1, long ld, long split, long rows, long cols) { return GfMat{p0, p1, ld, (int)split, (int)rows, (int)rows, (int)cols}; }

long gf_tiles(long M, long N, int mi, int ni) { return (M + 64 * mi - 1) / (64 * mi) * ((N + 64 * ni - 1) / (64 * ni)); }

template <int EP, bool ACOL, bool BCOL, int MI, int NI>
void gf_launch_tile(const GfParams &P, hipStream_t s)
{
    hipLaunchKernelGGL((pcm_gated_gemm_kernel<EP, ACOL, BCOL, MI, NI>), dim3((unsigned)gf_up(gf_tiles(P.M, P.N, MI, NI) * P.nsplit, 8)), dim3(256), 0, s, P);
}

// Tile of a product: the largest that gives every compute unit a workgroup or two.  A wave of 128 x 64 reads 12 operand pieces for 16
// matrix instructions, one of 32 x 64 six for four: large tiles are bound by the matrix cores, small ones by LDS, but 52 workgroups of
// the large kind leave four fifths of the chip idle.
int gf_tile_mi(long M, long N, int nsplit) { return gf_tiles(M, N, 4, 2) * nsplit >= 400 ? 4 : (gf_tiles(M, N, 2, 2) * nsplit >= 256 ? 2 : 1); }

template <int EP, bool ACOL, bool BCOL>
void gf_launch(const GfParams &P, hipStream_t s)
{
    const int mi = gf_tile_mi(P.M, P.N, P.nsplit);
    if (mi == 4) gf_launch_tile<EP, ACOL, BCOL, 4, 2>(P, s);
    else if (mi == 2) gf_launch_tile<EP, ACOL, BCOL, 2, 2>(P, s);
    else gf_launch_tile<EP, ACOL, BCOL, 1, 2>(P, s);
    if (P.nsplit > 1) hipLaunchKernelGGL(pcm_gated_join_kernel, dim3((unsigned)((P.M * P.N + 255) / 256)), dim3(256), 0, s, P);
}

// Splits of a product's contraction where its output has too few tiles: weight gradients contract over all rows, the outer products of
// few rows over all hidden values.  Shared out until about 512 workgroups run, at least 256 contracted values each (a split writes and
// re-reads the fp32 output).
int gf_splits(long M, long N, long K)
{
    const long tiles = gf_tiles(M, N, 4, 2) >= 64 ? gf_tiles(M, N, 4, 2) : (gf_tiles(M, N, 2, 2) >= 64 ? gf_tiles(M, N, 2, 2) : gf_tiles(M, N, 1, 2));
    if (tiles >= 256) return 1;
    long n = (512 + tiles - 1) / tiles;
    n = n < K / 256 ? n : K / 256;
    return (int)(n < 1 ? 1 : (n > 32 ? 32 : n));
}
long gf_part_bytes(long M, long N, long K) { const int n = gf_splits(M, N, K); return n > 1 ? gf_up(n * M * N * 4, 256) : 0; }

// the backward products run one after another and share one buffer of partial sums
long gf_back_part_bytes(long R, int E, int F)
{
    const long Fp = gf_up(F, 64), a = gf_part_bytes(2 * Fp, E, R), b = gf_part_bytes(E, F, R), c = gf_part_bytes(R, E, 2 * Fp);
    return a > b ? (a > c ? a : c) : (b > c ? b : c);
}
int gf_slots(long R) { return (int)(R < 64 ? 1 : (R / 32 > 128 ? 128 : R / 32)); }
// partial rows of da | du: two wave rows per tile row
long gf_wave_rows(long R, long Fp) { const int mi = gf_tile_mi(R, Fp, 1); return (R + 64 * mi - 1) / (64 * mi) * 2; }
long gf_sum_bytes(long R, int E, long Fp) { return gf_up((gf_wave_rows(R, Fp) * 2 * Fp + gf_slots(R) * gf_up(E, 8)) * 4, 256); }
bool gf_sizes_ok(long R, int E, int F) { return R <= 0x3FFFFFFFL && E <= (1 << 20) && F <= (1 << 20); }
long gf_pack_bytes(long rows, int cols) { return gf_up(rows * gf_up(cols, 8) * 2, 256); }

}  // namespace

extern "C" long pcm_gated_ffn_hidden_ld(int F) { return F > 0 ? gf_up(F, 64) : 0; }

extern "C" long pcm_gated_ffn_ws_bytes(long R, int E, int F, int backward)
{
    if (R <= 0 || E <= 0 || F <= 0) return 0;
    const long Fp = gf_up(F, 64);
    if (!backward && R <= GF_FEW) return 0;
    // copies: x and dy (any strides), the three weights
    long n = gf_pack_bytes(R, E) * (backward ? 2 : 1) + 2 * gf_pack_bytes(F, E) + gf_pack_bytes(E, F);
    if (!backward) n += gf_part_bytes(R, E, gf_up(F, 8));
    if (backward) {
        n += gf_up(R * 2 * Fp * 2, 256);  // da | du
        n += gf_back_part_bytes(R, E, F);
        n += gf_sum_bytes(R, E, Fp);
    }
    return n;
}

extern "C" int pcm_gated_ffn_forward_hip(long R, int E, int F, int act, const void *x, long x_ls, const void *wg, const void *wu, const void *wd,
                                         const void *bg, const void *bu, const void *bd, void *y, void *a, void *u, void *h, void *ws,
                                         long ws_bytes, void *stream)
{
    if (R < 0 || E < 0 || F < 0) return PCM_ERR_BAD_ARG;
    if (R == 0) return PCM_OK;
    if (E == 0 || F == 0 || act < 0 || act > 2 || !x || !wg || !wu || !wd || !y || !h || (!a != !u)) return PCM_ERR_BAD_ARG;
    if (!gf_sizes_ok(R, E, F)) return PCM_ERR_UNSUPPORTED;
    if ((((uintptr_t)a | (uintptr_t)u | (uintptr_t)h | (uintptr_t)ws) & 15) != 0) return PCM_ERR_BAD_ARG;
    const hipStream_t s = (hipStream_t)stream;
    const long Fp = gf_up(F, 64);
    if (R <= GF_FEW) {
        GfParams P{};
        P.a.p0 = (const u16 *)x, P.a.ld = x_ls, P.b.p0 = (const u16 *)wg, P.b.p1 = (const u16 *)wu, P.b.ld = E;
        P.M = R, P.K = E, P.act = act, P.F = F, P.Fp = Fp, P.bias0 = (const u16 *)bg, P.bias1 = (const u16 *)bu;
        P.out = (u16 *)a, P.out1 = (u16 *)u, P.h = (u16 *)h;
        GF_BY_ROWS(pcm_gated_few_in_kernel, R, (unsigned)(Fp / 4), s, P);
        GfParams Q{};
        Q.a.p0 = (const u16 *)h, Q.a.ld = Fp, Q.b.p0 = (const u16 *)wd, Q.b.ld = F, Q.M = R, Q.N = E, Q.K = F;
        Q.bias0 = (const u16 *)bd, Q.out = (u16 *)y, Q.ldo = E;
        GF_BY_ROWS(pcm_gated_few_out_kernel, R, (unsigned)((E + 3) / 4), s, Q);
        return PCM_LAUNCH_STATUS();
    }
    if (ws_bytes < pcm_gated_ffn_ws_bytes(R, E, F, 0) || !ws) return PCM_ERR_BAD_ARG;
    float *const part = (float *)ws;
    const long part_bytes = gf_part_bytes(R, E, gf_up(F, 8));
    GfPacker pk((char *)ws + part_bytes, ws_bytes - part_bytes);
    long ldx = x_ls, ldg = E, ldu = E, ldd = F;
    const u16 *px = pk.get(x, R, E, ldx);
    const u16 *pg = pk.get(wg, F, E, ldg), *pu = pk.get(wu, F, E, ldu);  // one row length either way
    const u16 *pd = pk.get(wd, E, F, ldd);
    if (!pk.room()) return PCM_ERR_BAD_ARG;
    pk.run(s);
    const long Ep = gf_up(E, 8);
    GfParams P{};
    P.a = gf_mat(px, ldx, R, Ep), P.b = gf_mat2(pg, pu, ldg, Fp, F, Ep);
    P.M = R, P.N = 2 * Fp, P.K = Ep, P.act = act, P.nsplit = 1, P.F = F, P.Fp = Fp;
    P.bias0 = (const u16 *)bg, P.bias1 = (const u16 *)bu, P.out = (u16 *)a, P.out1 = (u16 *)u, P.h = (u16 *)h;
    gf_launch<EP_GLU, false, false>(P, s);
    GfParams Q{};
    Q.a = gf_mat((const u16 *)h, Fp, R, Fp), Q.b = gf_mat(pd, ldd, E, gf_up(F, 8));
    Q.M = R, Q.N = E, Q.K = gf_up(F, 8), Q.nsplit = gf_splits(R, E, Q.K), Q.part = part, Q.bias0 = (const u16 *)bd, Q.F = Q.osplit = R, Q.out = (u16 *)y, Q.ldo = E;
    gf_launch<EP_OUT, false, false>(Q, s);
    return PCM_LAUNCH_STATUS();
}

extern "C" int pcm_gated_ffn_backward_hip(long R, int E, int F, int act, const void *x, long x_ls, const void *wg, const void *wu, const void *wd,
                                          const void *a, const void *u, const void *h, const void *dy, long dy_ls, void *dx, void *dwg,
                                          void *dwu, void *dwd, void *dbg, void *dbu, void *dbd, void *ws, long ws_bytes, void *stream)
{
    if (R < 0 || E < 0 || F < 0) return PCM_ERR_BAD_ARG;
    if (R == 0) return PCM_OK;
    if (E == 0 || F == 0 || act < 0 || act > 2 || !x || !wg || !wu || !wd || !a || !u || !h || !dy || !ws || (!dwg != !dwu) || (!dbg != !dbu)) return PCM_ERR_BAD_ARG;
    if (!gf_sizes_ok(R, E, F)) return PCM_ERR_UNSUPPORTED;
    if ((((uintptr_t)a | (uintptr_t)u | (uintptr_t)h | (uintptr_t)ws) & 15) != 0 || ws_bytes < pcm_gated_ffn_ws_bytes(R, E, F, 1)) return PCM_ERR_BAD_ARG;
    const hipStream_t s = (hipStream_t)stream;
    const long Fp = gf_up(F, 64), Ep = gf_up(E, 8);
    const bool hidden = dx || dwg || dbg;
    u16 *dau = (u16 *)ws;
    char *at = (char *)ws + gf_up(R * 2 * Fp * 2, 256);
    float *sums = (float *)at;
    at += gf_sum_bytes(R, E, Fp);
    float *part = (float *)at;
    at += gf_back_part_bytes(R, E, F);
    GfPacker pk(at, (char *)ws + ws_bytes - at);
    long ldx = x_ls, ldy = dy_ls, ldg = E, ldu = E, ldd = F;
    const u16 *py = pk.get(dy, R, E, ldy), *px = dwg ? pk.get(x, R, E, ldx) : nullptr;
    const u16 *pg = dx ? pk.get(wg, F, E, ldg) : nullptr, *pu = dx ? pk.get(wu, F, E, ldu) : nullptr;
    const u16 *pd = hidden ? pk.get(wd, E, F, ldd) : nullptr;
    if (!pk.room()) return PCM_ERR_BAD_ARG;
    pk.run(s);
    if (hidden) {
        GfParams P{};
        P.a = gf_mat(py, ldy, R, Ep), P.b = gf_mat(pd, ldd, E, gf_up(F, 8));
        P.M = R, P.N = Fp, P.K = Ep, P.act = act, P.nsplit = 1, P.F = F, P.Fp = Fp;
        P.out = dau, P.ea = (const u16 *)a, P.eu = (const u16 *)u, P.part = dbg ? sums : nullptr;
        gf_launch<EP_DGLU, false, true>(P, s);
    }
    if (dx) {
        GfParams P{};
        P.a = gf_mat(dau, 2 * Fp, R, 2 * Fp), P.b = gf_mat2(pg, pu, ldg, Fp, F, Ep);
        P.M = R, P.N = E, P.K = 2 * Fp, P.nsplit = gf_splits(P.M, P.N, P.K), P.part = part, P.F = P.osplit = R, P.out = (u16 *)dx, P.ldo = E;
        gf_launch<EP_OUT, false, true>(P, s);
    }
    if (dwg) {
        GfParams P{};
        P.a = gf_mat(dau, 2 * Fp, R, 2 * Fp), P.b = gf_mat(px, ldx, R, Ep);
        P.M = 2 * Fp, P.N = E, P.K = R, P.nsplit = gf_splits(P.M, P.N, P.K), P.F = F, P.out = (u16 *)dwg, P.out1 = (u16 *)dwu, P.ldo = E, P.part = part;
        P.osplit = Fp;
        gf_launch<EP_WGRAD, true, true>(P, s);
    }
    if (dwd) {
        GfParams P{};
        P.a = gf_mat(py, ldy, R, Ep), P.b = gf_mat((const u16 *)h, Fp, R, Fp);
        P.M = E, P.N = F, P.K = R, P.nsplit = gf_splits(P.M, P.N, P.K), P.F = E, P.osplit = E, P.out = (u16 *)dwd, P.ldo = F, P.part = part;
        gf_launch<EP_WGRAD, true, true>(P, s);
    }
    if (dbg || dbd) {
        GfSums P{};
        P.rows = R, P.E = E, P.F = F, P.Fp = (int)Fp, P.g = py, P.ld = ldy;
        P.slots[0] = (int)gf_wave_rows(R, Fp), P.C[0] = dbg ? (int)(2 * Fp) : 0, P.part[0] = sums;
        P.slots[1] = gf_slots(R), P.C[1] = dbd ? (int)Ep : 0, P.part1 = sums + P.slots[0] * 2 * Fp, P.part[1] = P.part1;
        P.out[0] = (u16 *)dbg, P.out[1] = (u16 *)dbu, P.out[2] = (u16 *)dbd;
        if (dbd) hipLaunchKernelGGL(pcm_gated_colsum_kernel, dim3((unsigned)((Ep + 511) / 512), P.slots[1]), dim3(256), 0, s, P);
        const long widest = P.C[0] > P.C[1] ? P.C[0] : P.C[1];
        hipLaunchKernelGGL(pcm_gated_colsum_join_kernel, dim3((unsigned)((widest + 63) / 64), 2), dim3(256), 0, s, P);
    }
    return PCM_LAUNCH_STATUS();
}

// gated_ffn.hip -- the gated feed-forward block and its backward pass.
//
//   a = x Wg^T + bg,  u = x Wu^T + bu,  h = act(a) * u,  y = h Wd^T + bd            (act: SiLU, GELU (erf) or ReLU)
//   dh = dy Wd,  da = dh * u * act'(a),  du = dh * act(a),
//   dx = da Wg + du Wu,  dWg = da^T x,  dWu = du^T x,  dWd = dy^T h,  bias gradients = column sums.
//
// Every product is one tile engine (v_mfma_f32_32x32x16_bf16, fp32 accumulators) with two operand forms: contracted index contiguous in
// memory (read from LDS as 16-byte pieces), or the other index contiguous (read through ds_read_b64_tr_b16, which transposes on the
// way).  The element-wise parts are epilogues: both projections share one launch -- a wave's 64 output columns are 32 of the gate and
// the same 32 of the up projection, so act(a) * u needs no exchange -- and so do dh, da and du.  h, da and du are rounded to bf16
// where they are stored as operands of the next product (one half step, 2^-8 relative at most); outputs are rounded once.  a and u, of which
// the backward pass forms da and du, are kept in fp32: as bf16 they brought dx, the weight and the bias gradients from 2.3e-3 of their norm
// (the roundings of da, du and the output) to 3.0e-3, for 5 % less time (16408 rows, 512 -> 2048, forward and backward).
//
// a, u, h have rows of Fp = F rounded up to 64 values; the columns from F on are zero, so contractions over F need no edge.  Matrices
// whose rows do not start at 16-byte boundaries (an odd width) are copied into padded rows first, one launch for all of a call's.
#include "pcm_attn.hpp"

namespace {

constexpr int GF_BK = 64;  // contracted values of a step: 128 bytes of a row

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
    float *ka, *ku;              // a and u: what the forward pass keeps for the backward one
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
__device__ __forceinline__ void gf_store8(float *p, const float (&v)[8])
{
    *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]), *(float4 *)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
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

// One operand's tile of GF_BK contracted values, ROWS values of the operand's own index, requested by THREADS threads.
// COL false: [ROWS][64], contracted index contiguous, eight 16-byte pieces a row.  COL true: [64][ROWS], ROWS / 8 pieces a row.
// global_load_lds writes a wave's 64 pieces to consecutive addresses, so the layout cannot be padded; instead the piece a slot holds is
// permuted (the lane picks its source).  64 banks of 4 bytes: ds_read_b128 serves the lanes 0-3, 12-15, 20-23, 24-27 of 32 together, then the
// other 16, and rows of 128 bytes share banks every other row, so three bits of the row pick the slot; ds_read_b64_tr_b16 serves 32 lanes
// together, 64 bytes of each of 4 neighbouring contracted rows, which have to lie in different 64-byte groups.
template <bool COL, int ROWS, int THREADS>
struct GfTile {
    static constexpr int PIECES = COL ? ROWS / 8 : 8, SIZE = ROWS * GF_BK, LOADS = SIZE / 8 / THREADS;
    static __device__ __forceinline__ int swz(int r)
    {
        if constexpr (!COL) return (r >> 1) & 7;
        else if constexpr (ROWS >= 128) return (r & 3) << 2;
        else return ((r >> 1) & 1) << 2;
    }
    // The thread's n-th piece stands n * NROWS tile rows below its first (the permutation is the same: NROWS is a multiple of 16).
    static constexpr int NROWS = THREADS / PIECES;
    static_assert(COL || NROWS % 16 == 0, "the permutation repeats every 16 rows");
    static_assert(!COL || NROWS % 4 == 0, "the permutation repeats every 4 rows");
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
            left = 0, each = NROWS;
            if (glu) {  // virtual row -> gate | up weight row: 32 and 32 of every 64
                row = (row >> 6) * 32 + (row & 31) + ((row & 32) ? m.split : 0);
                if constexpr (NROWS % 64 == 0) each = NROWS / 2;
            }
            const bool second = row >= m.split;
            const long rr = second ? row - m.split : row;
            left = (int)((second ? m.rows1 : m.rows0) - rr), koff = 8 * c, step = each * m.ld;
            base = (second ? m.p1 : m.p0) + rr * m.ld + 8 * c;
        }
    }
    // the tile of contracted indices k .. k + 63 on its way into LDS
    // (its pieces n0 .. n1 - 1)
    template <bool GLU>
    __device__ __forceinline__ void load(const GfMat &m, u16 *tile, long k, long kend, int n0 = 0, int n1 = LOADS) const
    {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        // a tile never straddles the parts: `split` is a multiple of 64
        const bool second = COL && k >= m.split;
        const int rest = (int)((COL ? min(kend, second ? m.split + (long)m.rows1 : (long)m.rows0) : kend) - k);
        const long at = COL ? k * m.ld + (second ? (long)(m.p1 - m.p0) - (long)m.split * m.ld : 0) : k;
#pragma unroll
        for (int n = n0; n < n1; ++n) {
            bool in = COL ? left && koff + n * NROWS < rest : n * each < left && koff < rest;
            const u16 *src = base + (at + n * step);
            if constexpr (GLU && !COL && NROWS % 64 != 0) {  // 32 rows a pass: gate and up rows alternate
                static_assert(!(GLU && !COL) || NROWS % 64 == 0 || NROWS == 32, "a pass covers whole runs of 32");
                const int f = (n >> 1) * 32;
                in = f < left && koff < rest;
                src = base + (at + f * m.ld + ((n & 1) ? (long)(m.p1 - m.p0) : 0));
            }
            __builtin_amdgcn_global_load_lds((gf_glb_p)(in ? (const void *)src : (const void *)&gf_zeros),
                                             (gf_lds_p)(tile + (n * THREADS + wave * 64) * 8), 16, 0, 0);
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

// The tile engine.  2 x WN waves; a wave owns MI x NI tiles of 32 x 32.  Two LDS buffers of 64 contracted values each: once tile t has arrived,
// tile t + 1 is requested into the other buffer (global_load_lds: no registers, no LDS write instructions) and the step's matrix
// instructions run meanwhile; one barrier a step.  A step takes 128 bytes of a row because that is a cache line: with steps of 64 bytes
// the other half of every line had left the 32 KB cache before its turn, the lines went through it twice, and 256 x 128 tiles kept the
// matrix cores at half of what they do here.  The buffers are two variables, so that the compiler can tell the reads of one from the requests into
// the other and inserts no wait of its own between them.
template <int EP, bool ACOL, bool BCOL, int MI, int NI, int WN>
__global__ void __launch_bounds__(128 * WN, 2) pcm_gated_gemm_kernel(GfParams P)
{
    constexpr int THREADS = 128 * WN, BM = 64 * MI, BN = 32 * NI * WN, COLS = 32 * NI, SLAB = COLS + 4;
    typedef GfTile<ACOL, BM, THREADS> TA;
    typedef GfTile<BCOL, BN, THREADS> TB;
    constexpr int STAGE = (TA::SIZE + TB::SIZE) * 2, BYTES = STAGE > WN * 32 * SLAB * 4 ? STAGE : WN * 32 * SLAB * 4;
    __shared__ __attribute__((aligned(1024))) unsigned char sm0[BYTES], sm1[BYTES];
    const int M = (int)P.M, N = (int)P.N;
    const long mt = (P.M + BM - 1) / BM, nt = (P.N + BN - 1) / BN, items = mt * nt * P.nsplit, per = (items + 7) / 8;
    const long item = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);  // one XCD's L2 sees consecutive tiles
    if ((long)(blockIdx.x >> 3) >= per || item >= items) return;
    const long m0 = item / nt % mt * BM, n0 = item % nt * BN, split = item / (nt * mt);
    const long kt = (P.K + GF_BK - 1) / GF_BK, kper = (kt + P.nsplit - 1) / P.nsplit * GF_BK;
    const long k0 = split * kper, kend = k0 + kper < P.K ? k0 + kper : P.K;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = (wave / WN) * 32 * MI, wn = (wave % WN) * COLS;
    f16v acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    TA ga;
    TB gb;
    ga.init(P.a, m0, false), gb.init(P.b, n0, EP == EP_GLU);
    const auto request = [&](unsigned char *sm, long k) {
        ga.template load<false>(P.a, (u16 *)sm, k, kend), gb.template load<EP == EP_GLU>(P.b, (u16 *)sm + TA::SIZE, k, kend);
    };
    const auto step = [&](const unsigned char *cur, unsigned char *other, long k) {
        __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0) lgkmcnt(0): this wave's pieces have arrived, its reads of the other buffer are done
        __syncthreads();                   // ... and everybody's
        const u16 *ta = (const u16 *)cur, *tb = ta + TA::SIZE;
        // One workgroup a compute unit (8 waves): all requests at once would hold up every wave's first products until the last is
        // accepted (0.6 us for 64 KB), so they are spread over the step's first half.  With two or three workgroups the others multiply
        // meanwhile, and the earliest request is best: 128 x 128 tiles took 8 % longer with spread requests, 256 x 256 ones 12 % less.
        constexpr bool SPREAD = WN == 4;
        constexpr int KK = GF_BK / 16, ALL = TA::LOADS + TB::LOADS, SLOTS = 2 * MI;
        if (!SPREAD) {
            if (k + GF_BK < kend) request(other, k + GF_BK);
            __builtin_amdgcn_sched_barrier(0);
        }
        bf8 a[2][MI], b[2][NI];
        const auto read = [&](int kk) {
#pragma unroll
            for (int i = 0; i < MI; ++i) a[kk & 1][i] = TA::operand(ta, wm + 32 * i, kk, lane);
#pragma unroll
            for (int j = 0; j < NI; ++j) b[kk & 1][j] = TB::operand(tb, wn + 32 * j, kk, lane);
        };
        read(0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            if (kk + 1 < KK) read(kk + 1);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                if constexpr (SPREAD) {
                    if (kk < 2 && k + GF_BK < kend) {
                        const int p0 = (kk * MI + i) * ALL / SLOTS, p1 = (kk * MI + i + 1) * ALL / SLOTS;
                        ga.template load<false>(P.a, (u16 *)other, k + GF_BK, kend, min(p0, TA::LOADS), min(p1, TA::LOADS));
                        gb.template load<EP == EP_GLU>(P.b, (u16 *)other + TA::SIZE, k + GF_BK, kend, max(p0 - TA::LOADS, 0), max(p1 - TA::LOADS, 0));
                    }
                }
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = PCM_MFMA16(a[kk & 1][i], b[kk & 1][j], acc[i][j]);
                if (SPREAD && kk < 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    if (k0 < kend) {
        request(sm0, k0);
        long k = k0;
        for (; k + GF_BK < kend; k += 2 * GF_BK) {
            step(sm0, sm1, k);
            step(sm1, sm0, k + GF_BK);
        }
        if (k < kend) step(sm0, sm1, k);
    }
    __syncthreads();
    // Epilogue: 32 rows at a time through a slab of the wave's own (an accumulator holds a column a lane), out of it 8 neighbouring
    // columns a lane, the same ones in every pass: 16-byte accesses to everything that is read and written beside the products.
    float *const slab = (float *)(wave < WN ? sm0 : sm1) + (wave % WN) * 32 * SLAB;
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
    constexpr int PASSES = 32 * GROUPS / 64, AHEAD = EP == EP_DGLU ? PASSES / 2 : 1;
    float4 ea[2][AHEAD][2], eu[2][AHEAD][2];
    const auto fetch = [&](int half) {  // a and u of half a slab, requested half a slab ahead
#pragma unroll
        for (int g = 0; g < AHEAD; ++g) {
            // rows and columns outside are read from the last ones inside: no branch that the loads could sink into
            const long row = min(m0 + wm + 16 * half + r0 + g * (64 / GROUPS), P.M - 1), at = row * P.Fp + min((long)col, P.Fp - 8);
#pragma unroll
            for (int e = 0; e < 2; ++e) ea[half & 1][g][e] = *(const float4 *)(P.ka + at + 4 * e), eu[half & 1][g][e] = *(const float4 *)(P.ku + at + 4 * e);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (EP == EP_DGLU) fetch(0);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) slab[crow(r, lane) * SLAB + 32 * j + (lane & 31)] = acc[i][j][r];
        __builtin_amdgcn_wave_barrier();  // the wave's LDS operations complete in order
#pragma unroll
        for (int g = 0; g < PASSES; ++g) {
            if constexpr (EP == EP_DGLU)
                if (g % AHEAD == 0 && 2 * i + g / AHEAD + 1 < 2 * MI) fetch(2 * i + g / AHEAD + 1);
            const int r = r0 + g * (64 / GROUPS);
            const long row = m0 + wm + 32 * i + r;
            if ((int)row >= M) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = slab[r * SLAB + c + e];
            if constexpr (EP == EP_GLU) {
                if (col >= P.Fp) continue;  // a tile of 256 columns, 128 of each projection, may end behind the last of 64 k
                float u[8], hv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = slab[r * SLAB + 32 + c + e];
#pragma unroll
                for (int e = 0; e < 8; ++e) {  // columns from F on: weights and biases are zeros, and so are a, u and h
                    v[e] += bias0[e], u[e] += bias1[e];
                    hv[e] = gf_act(v[e], P.act) * u[e];
                }
                const long at = row * P.Fp + col;
                if (P.ka) gf_store8(P.ka + at, v), gf_store8(P.ku + at, u);
                *(uint4 *)(P.h + at) = gf_bf8(hv);
            } else if constexpr (EP == EP_DGLU) {
                if (col >= P.Fp) continue;
                const float4(&fa)[2] = ea[g / AHEAD][g % AHEAD], (&fu)[2] = eu[g / AHEAD][g % AHEAD];
                const float a[8] = {fa[0].x, fa[0].y, fa[0].z, fa[0].w, fa[1].x, fa[1].y, fa[1].z, fa[1].w};
                float u[8] = {fu[0].x, fu[0].y, fu[0].z, fu[0].w, fu[1].x, fu[1].y, fu[1].z, fu[1].w};
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
                        gf_store8(o, v);
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
        float *o = P.part + (m0 / (32 * MI) + wave / WN) * 2 * P.Fp + col;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = bias0[e], o[P.Fp + e] = bias1[e];
    }
}

// Bias gradients.  The sums of da | du over a wave's rows leave the epilogue that forms them (one partial row per wave row: reading
// da | du again would cost as much as writing it); dy is summed here, `slots` partial rows of fixed row ranges.  pcm_gated_close_kernel
// sums the partial rows; the order never changes.
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
// What closes a pass, in one launch: split contractions summed in split order (+ bias), four values a thread, and the bias gradients'
// partial rows, 16 columns and 16 interleaved row lanes a workgroup.
struct GfJoin {
    const float *part;
    u16 *out, *out1;
    const u16 *bias;
    long M, N, osplit, F, ldo, end;  // end: running count of workgroups
    int nsplit;
};
struct GfClose {
    GfJoin j[3];
    int n;
    GfSums s;
    int sums;  // workgroups of the first part's columns (da | du), then of the second's (dy)
};
__global__ void __launch_bounds__(256) pcm_gated_close_kernel(GfClose P)
{
    __shared__ float lds[4][16];
    long blk = blockIdx.x;
    int j = 0;
    while (j < P.n && blk >= P.j[j].end) ++j;
    if (j < P.n) {
        const GfJoin &J = P.j[j];
        const long first = (blk - (j ? P.j[j - 1].end : 0)) * 1024, size = J.M * J.N;
        if (J.N % 4 == 0) {
            const long i = first + 4 * (int)threadIdx.x;
            if (i >= size) return;
            const long row = i / J.N, n = i - row * J.N;
            const bool second = row >= J.osplit;
            const long rr = second ? row - J.osplit : row;
            if (rr >= J.F) return;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int k = 0; k < J.nsplit; ++k) {
                const float4 v = *(const float4 *)(J.part + k * size + i);
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            if (J.bias) s.x += bf2f(J.bias[n]), s.y += bf2f(J.bias[n + 1]), s.z += bf2f(J.bias[n + 2]), s.w += bf2f(J.bias[n + 3]);
            u16 *o = (second ? J.out1 : J.out) + rr * J.ldo + n;
            if (((uintptr_t)o & 7) == 0) *(uint2 *)o = make_uint2(cvt_pk_bf16(s.x, s.y), cvt_pk_bf16(s.z, s.w));
            else o[0] = gf_bf(s.x), o[1] = gf_bf(s.y), o[2] = gf_bf(s.z), o[3] = gf_bf(s.w);
            return;
        }
        for (long e = first + (int)threadIdx.x; e < first + 1024 && e < size; e += 256) {
            const long row = e / J.N, n = e - row * J.N;
            const bool second = row >= J.osplit;
            const long rr = second ? row - J.osplit : row;
            if (rr >= J.F) continue;
            float s = 0.f;
#pragma unroll 4
            for (int k = 0; k < J.nsplit; ++k) s += J.part[k * size + e];
            (second ? J.out1 : J.out)[rr * J.ldo + n] = gf_bf(s + (J.bias ? bf2f(J.bias[n]) : 0.f));
        }
        return;
    }
    blk -= P.n ? P.j[P.n - 1].end : 0;
    const int part = blk >= P.sums, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)(blk - (part ? P.sums : 0)) * 16 + (lane & 15);
    const GfSums &S = P.s;
    float s = 0.f;
    if (c < S.C[part]) {
#pragma unroll 8
        for (int k = wave * 4 + (lane >> 4); k < S.slots[part]; k += 16) s += S.part[part][(long)k * S.C[part] + c];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16) lds[wave][lane] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || c >= S.C[part]) return;
    s = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
    if (part) {
        if (c < S.E) S.out[2][c] = gf_bf(s);
    } else if (c < S.F) {
        S.out[0][c] = gf_bf(s);
    } else if (c >= S.Fp && c - S.Fp < S.F) {
        S.out[1][c - S.Fp] = gf_bf(s);
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
    if (P.ka) P.ka[at] = a, P.ku[at] = u;
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

// Tiles: 256 x 256 (8 waves of 128 x 64, one workgroup a compute unit), 128 x 128 and 64 x 128 (4 waves, two or three a compute unit).
struct GfShape {
    int bm, bn;
};
constexpr GfShape GF_LARGE{256, 256}, GF_MIDDLE{128, 128}, GF_SMALL{64, 128};
long gf_tiles(long M, long N, GfShape s) { return (M + s.bm - 1) / s.bm * ((N + s.bn - 1) / s.bn); }

// The shape of a product's tiles: large ones pass the least data per product through LDS and cache, but a launch of 257 of them takes as long as one
// of 512.  Taken: the largest shape whose last round of workgroups is not mostly empty (256 compute units, 1 / 2 / 3 workgroups each); over a short
// contraction the smaller ones, of which one multiplies while its neighbour is in the epilogue (both projections of 16384 rows, 512 -> 2048, the shortest
// one for large tiles: 145 us with them, 188 with 128 x 128).  Weight gradients, both of whose operands are read
// transposed, have no registers left for large ones.
GfShape gf_shape(long M, long N, long K, int nsplit, bool wgrad)
{
    const long large = gf_tiles(M, N, GF_LARGE) * nsplit, middle = gf_tiles(M, N, GF_MIDDLE) * nsplit;
    if (!wgrad && K / nsplit >= 512 && large >= 200 && large * 10 >= (large + 255) / 256 * 256 * 7) return GF_LARGE;
    return middle >= 256 ? GF_MIDDLE : GF_SMALL;
}

// Rows of a product's first launch.  Tiles a little over whole rounds of workgroups (one / two / three a compute unit) leave the last round nearly
// empty: 16408 rows are 64 row tiles of 256 and 24 rows, 4 rounds and 16 tiles of a fifth.  Where the last round has under a third of a round's
// tiles and a round is worth the launch (2^24 products a compute unit, some 20 us), its rows are multiplied by a second launch, in smaller tiles
// and shared-out contractions of its own choice (16408 rows of 512 -> 2048, forward and backward: 602 us, 633 with one launch a
// product).
long gf_first_rows(long M, long N, long K)
{
    const GfShape t = gf_shape(M, N, K, 1, false);
    const long per = t.bm == 256 ? 1 : (t.bm == 128 ? 2 : 3), slots = 256 * per, nt = (N + t.bn - 1) / t.bn;
    const long whole = gf_tiles(M, N, t) / slots, rest = gf_tiles(M, N, t) - whole * slots;
    if (whole == 0 || rest == 0 || rest * 3 > slots || t.bm * t.bn * per * K < 1L << 24) return M;
    const long rows = whole * slots / nt * t.bm;  // none where one row of tiles is more than the whole rounds hold: the rows stay together
    return rows > 0 && rows < M ? rows : M;
}

template <int EP, bool ACOL, bool BCOL>
void gf_launch(const GfParams &P, hipStream_t s)
{
    const GfShape t = gf_shape(P.M, P.N, P.K, P.nsplit, EP == EP_WGRAD);
    const dim3 grid((unsigned)((gf_tiles(P.M, P.N, t) * P.nsplit + 7) / 8 * 8));
    if (t.bm == 256) {
        if constexpr (EP != EP_WGRAD) hipLaunchKernelGGL((pcm_gated_gemm_kernel<EP, ACOL, BCOL, 4, 2, 4>), grid, dim3(512), 0, s, P);
    } else if (t.bm == 128) hipLaunchKernelGGL((pcm_gated_gemm_kernel<EP, ACOL, BCOL, 2, 2, 2>), grid, dim3(256), 0, s, P);
    else hipLaunchKernelGGL((pcm_gated_gemm_kernel<EP, ACOL, BCOL, 1, 2, 2>), grid, dim3(256), 0, s, P);
}

long gf_tile_rows(long M, long N, long K) { const int bm = gf_shape(M, N, K, 1, false).bm; return (M + bm - 1) / bm; }

// adds a product's joining to what closes the pass
void gf_join(GfClose &c, const GfParams &P)
{
    if (P.nsplit <= 1) return;
    GfJoin &j = c.j[c.n++];
    j = GfJoin{P.part, P.out, P.out1, P.bias0, P.M, P.N, P.osplit, P.F, P.ldo, 0, P.nsplit};
    j.end = (c.n > 1 ? c.j[c.n - 2].end : 0) + (P.M * P.N + 1023) / 1024;
}
void gf_close(GfClose &c, hipStream_t s)
{
    c.sums = (c.s.C[0] + 15) / 16;
    const long blocks = (c.n ? c.j[c.n - 1].end : 0) + c.sums + (c.s.C[1] + 15) / 16;
    if (blocks) hipLaunchKernelGGL(pcm_gated_close_kernel, dim3((unsigned)blocks), dim3(256), 0, s, c);
}

// Splits of a product's contraction where its output has too few tiles: weight gradients contract over all rows, the outer products of
// few rows over all hidden values.  Shared out until about 512 workgroups run, at least 256 contracted values each (a split writes and
// re-reads the fp32 output).
int gf_splits(long M, long N, long K)
{
    const long middle = gf_tiles(M, N, GF_MIDDLE), tiles = middle >= 64 ? middle : gf_tiles(M, N, GF_SMALL);
    if (tiles >= 256) return 1;
    long n = 512 / tiles;
    n = n < K / 256 ? n : K / 256;
    return (int)(n < 1 ? 1 : (n > 32 ? 32 : n));
}
// the row products' second launch
template <int EP, bool BCOL>
bool gf_launch_rows(GfParams &P, hipStream_t s)  // false: one launch; true: P is the second one
{
    const long M = P.M, first = P.nsplit > 1 ? M : gf_first_rows(M, P.N, P.K);
    P.M = first;
    if (EP == EP_OUT) P.F = P.osplit = first;
    gf_launch<EP, false, BCOL>(P, s);
    if (first == M) return false;
    P.M = M - first, P.a.p0 += first * P.a.ld, P.a.rows0 -= (int)first;
    if (EP == EP_OUT) {
        P.F = P.osplit = P.M, P.out += first * P.ldo, P.nsplit = gf_splits(P.M, P.N, P.K);
    } else {
        P.ka = P.ka ? P.ka + first * P.Fp : nullptr, P.ku = P.ku ? P.ku + first * P.Fp : nullptr;
        if (EP == EP_GLU) P.h += first * P.Fp;
        if (EP == EP_DGLU) P.out += first * 2 * P.Fp, P.part = P.part ? P.part + gf_tile_rows(first, P.N, P.K) * 4 * P.Fp : nullptr;
    }
    gf_launch<EP, false, BCOL>(P, s);
    return true;
}
long gf_part_bytes(long M, long N, long K) { const int n = gf_splits(M, N, K); return n > 1 ? gf_up(n * M * N * 4, 256) : 0; }

// partial sums of a row product: of all of it, or of its second launch
long gf_row_part_bytes(long M, long N, long K)
{
    if (gf_splits(M, N, K) > 1) return gf_part_bytes(M, N, K);
    const long first = gf_first_rows(M, N, K);
    return first < M ? gf_part_bytes(M - first, N, K) : 0;
}

// partial sums of the three backward products, joined together at the end
long gf_back_part_bytes(long R, int E, int F)
{
    const long Fp = gf_up(F, 64);
    return gf_row_part_bytes(R, E, 2 * Fp) + gf_part_bytes(2 * Fp, E, R) + gf_part_bytes(E, F, R);
}
int gf_slots(long R) { return (int)(R < 64 ? 1 : (R / 32 > 512 ? 512 : R / 32)); }
// partial rows of da | du: two wave rows per tile row
long gf_wave_rows(long R, int E, long Fp)
{
    const long Ep = gf_up(E, 8), first = gf_first_rows(R, Fp, Ep);
    return 2 * (gf_tile_rows(first, Fp, Ep) + (first < R ? gf_tile_rows(R - first, Fp, Ep) : 0));
}
long gf_sum_bytes(long R, int E, long Fp) { return gf_up((gf_wave_rows(R, E, Fp) * 2 * Fp + gf_slots(R) * gf_up(E, 8)) * 4, 256); }
// 32-bit rows and columns inside a tile; no launch has 2^32 threads (a copy of x, dy and three weights takes one for eight values)
bool gf_sizes_ok(long R, int E, int F)
{
    return R <= 0x3FFFFFFFL && E <= (1 << 20) && F <= (1 << 20) && R * gf_up(E, 8) <= 1L << 33 && R * gf_up(F, 64) <= 1L << 36 && (long)F * E <= 1L << 32;
}
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
    if (!backward) n += gf_row_part_bytes(R, E, gf_up(F, 8));
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
        P.ka = (float *)a, P.ku = (float *)u, P.h = (u16 *)h;
        GF_BY_ROWS(pcm_gated_few_in_kernel, R, (unsigned)(Fp / 4), s, P);
        GfParams Q{};
        Q.a.p0 = (const u16 *)h, Q.a.ld = Fp, Q.b.p0 = (const u16 *)wd, Q.b.ld = F, Q.M = R, Q.N = E, Q.K = F;
        Q.bias0 = (const u16 *)bd, Q.out = (u16 *)y, Q.ldo = E;
        GF_BY_ROWS(pcm_gated_few_out_kernel, R, (unsigned)((E + 3) / 4), s, Q);
        return PCM_LAUNCH_STATUS();
    }
    if (ws_bytes < pcm_gated_ffn_ws_bytes(R, E, F, 0) || !ws) return PCM_ERR_BAD_ARG;
    float *const part = (float *)ws;
    const long part_bytes = gf_row_part_bytes(R, E, gf_up(F, 8));
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
    P.bias0 = (const u16 *)bg, P.bias1 = (const u16 *)bu, P.ka = (float *)a, P.ku = (float *)u, P.h = (u16 *)h;
    gf_launch_rows<EP_GLU, false>(P, s);
    GfParams Q{};
    Q.a = gf_mat((const u16 *)h, Fp, R, Fp), Q.b = gf_mat(pd, ldd, E, gf_up(F, 8));
    Q.M = R, Q.N = E, Q.K = gf_up(F, 8), Q.nsplit = gf_splits(R, E, Q.K), Q.part = part, Q.bias0 = (const u16 *)bd, Q.out = (u16 *)y, Q.ldo = E;
    gf_launch_rows<EP_OUT, false>(Q, s);
    GfClose c{};
    gf_join(c, Q);
    gf_close(c, s);
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
    float *const part_dx = (float *)at, *const part_w1 = part_dx + gf_row_part_bytes(R, E, 2 * Fp) / 4, *const part_w2 = part_w1 + gf_part_bytes(2 * Fp, E, R) / 4;
    at += gf_back_part_bytes(R, E, F);
    GfClose c{};
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
        P.out = dau, P.ka = (float *)a, P.ku = (float *)u, P.part = dbg ? sums : nullptr;
        gf_launch_rows<EP_DGLU, true>(P, s);
    }
    if (dx) {
        GfParams P{};
        P.a = gf_mat(dau, 2 * Fp, R, 2 * Fp), P.b = gf_mat2(pg, pu, ldg, Fp, F, Ep);
        P.M = R, P.N = E, P.K = 2 * Fp, P.nsplit = gf_splits(P.M, P.N, P.K), P.part = part_dx, P.out = (u16 *)dx, P.ldo = E;
        gf_launch_rows<EP_OUT, true>(P, s);
        gf_join(c, P);
    }
    if (dwg) {
        GfParams P{};
        P.a = gf_mat(dau, 2 * Fp, R, 2 * Fp), P.b = gf_mat(px, ldx, R, Ep);
        P.M = 2 * Fp, P.N = E, P.K = R, P.nsplit = gf_splits(P.M, P.N, P.K), P.F = F, P.out = (u16 *)dwg, P.out1 = (u16 *)dwu, P.ldo = E, P.part = part_w1;
        P.osplit = Fp;
        gf_launch<EP_WGRAD, true, true>(P, s);
        gf_join(c, P);
    }
    if (dwd) {
        GfParams P{};
        P.a = gf_mat(py, ldy, R, Ep), P.b = gf_mat((const u16 *)h, Fp, R, Fp);
        P.M = E, P.N = F, P.K = R, P.nsplit = gf_splits(P.M, P.N, P.K), P.F = E, P.osplit = E, P.out = (u16 *)dwd, P.ldo = F, P.part = part_w2;
        gf_launch<EP_WGRAD, true, true>(P, s);
        gf_join(c, P);
    }
    if (dbg || dbd) {
        GfSums &P = c.s;
        P.rows = R, P.E = E, P.F = F, P.Fp = (int)Fp, P.g = py, P.ld = ldy;
        P.slots[0] = (int)gf_wave_rows(R, E, Fp), P.C[0] = dbg ? (int)(2 * Fp) : 0, P.part[0] = sums;
        P.slots[1] = gf_slots(R), P.C[1] = dbd ? (int)Ep : 0, P.part1 = sums + P.slots[0] * 2 * Fp, P.part[1] = P.part1;
        P.out[0] = (u16 *)dbg, P.out[1] = (u16 *)dbu, P.out[2] = (u16 *)dbd;
        if (dbd) hipLaunchKernelGGL(pcm_gated_colsum_kernel, dim3((unsigned)((Ep + 511) / 512), P.slots[1]), dim3(256), 0, s, P);
    }
    gf_close(c, s);
    return PCM_LAUNCH_STATUS();
}

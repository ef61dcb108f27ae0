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

constexpr int GF_BM = 128, GF_BN = 128, GF_BK = 64;

// A matrix of 2-byte values, rows at `ld`; rows from `split` on come from the second part (gate | up weights).
struct GfMat {
    const u16 *p0, *p1;
    long ld;
    int split, rows0, rows1, cols;  // rows of each part, columns (a multiple of 8)
};

struct GfParams {
    GfMat a, b;
    long M, N, K;
    int glu_rows;   // B's virtual rows: 32 of the gate, 32 of the up projection, alternating
    int act, nsplit;
    long F, Fp, osplit;          // weight gradients: output rows from osplit on go to out1; F rows each
    const u16 *bias0, *bias1;
    u16 *out, *out1, *h;         // see the epilogues
    const u16 *ea, *eu;
    long ldo;
    float *part;
};

enum { EP_GLU, EP_OUT, EP_DGLU, EP_DX, EP_WGRAD };

__device__ __forceinline__ float gf_act(float a, int act)
{
    if (act == 0) return a / (1.f + __expf(-a));
    if (act == 1) return 0.5f * a * (1.f + erff(a * 0.70710678118654752f));
    return a > 0.f ? a : (a == a ? 0.f : a);
}
// act(a) and act'(a)
__device__ __forceinline__ float2 gf_act_grad(float a, int act)
{
    if (act == 0) {
        const float s = 1.f / (1.f + __expf(-a));
        return make_float2(a * s, s * __builtin_fmaf(a, 1.f - s, 1.f));
    }
    if (act == 1) {
        const float c = 0.5f * (1.f + erff(a * 0.70710678118654752f));
        return make_float2(a * c, __builtin_fmaf(a * 0.39894228040143267f, __expf(-0.5f * a * a), c));
    }
    return make_float2(a > 0.f ? a : (a == a ? 0.f : a), a > 0.f ? 1.f : 0.f);
}
__device__ __forceinline__ u16 gf_bf(float v) { return (u16)cvt_pk_bf16(v, 0.f); }

// 16 bytes of matrix row r, columns c .. c + 7 (zero outside)
__device__ __forceinline__ uint4 gf_piece(const GfMat &m, long r, long c, bool ok)
{
    const bool second = r >= m.split;
    const long rr = second ? r - m.split : r;
    ok = ok && c < m.cols && rr < (second ? m.rows1 : m.rows0);
    return ok ? *(const uint4 *)((second ? m.p1 : m.p0) + rr * m.ld + c) : make_uint4(0, 0, 0, 0);
}

typedef s4 __attribute__((address_space(3))) * gf_lds_s4;

// One operand's tile: `COL` false: 128 rows of the operand x 64 contracted values; true: 64 contracted rows x 128 columns.
template <bool COL>
struct GfTile {
    static constexpr int PIECES = COL ? 16 : 8, LD = COL ? 136 : 72, SIZE = COL ? 64 * 136 : 128 * 72;
    uint4 d[4];
    __device__ __forceinline__ void load(const GfMat &m, long i0, long k0, long kend, bool glu)
    {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int c = threadIdx.x + 256 * n, r = c / PIECES, p = c - r * PIECES;
            if constexpr (COL) {
                d[n] = gf_piece(m, k0 + r, i0 + 8 * p, k0 + r < kend);
            } else {
                long row = i0 + r;
                if (glu) row = (row >> 6) * 32 + (row & 31) + ((row & 32) ? m.split : 0);  // virtual row -> gate | up weight row
                d[n] = gf_piece(m, row, k0 + 8 * p, k0 + 8 * p < kend);
            }
        }
    }
    __device__ __forceinline__ void store(u16 *t) const
    {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int c = threadIdx.x + 256 * n, r = c / PIECES, p = c - r * PIECES;
            *(uint4 *)(t + r * LD + 8 * p) = d[n];
        }
    }
    // operand of 32 rows i .. i + 31, contracted values 16 kk .. + 15
    static __device__ __forceinline__ bf8 operand(const u16 *t, int i, int kk, int lane)
    {
        const int h = lane >> 5;
        if constexpr (COL) {
            const int p = lane & 15, g = (lane >> 4) & 1;
            const u16 *q = t + (16 * kk + 8 * h + (p >> 2)) * LD + i + 16 * g + 4 * (p & 3);
            return cat8(__builtin_amdgcn_ds_read_tr16_b64_v4i16((gf_lds_s4)q), __builtin_amdgcn_ds_read_tr16_b64_v4i16((gf_lds_s4)(q + 4 * LD)));
        } else {
            return lds_bf8(t + (i + (lane & 31)) * LD + 16 * kk + 8 * h);
        }
    }
};

template <int EP, bool ACOL, bool BCOL>
__global__ void __launch_bounds__(256, 2) pcm_gated_gemm_kernel(GfParams P)
{
    __shared__ __attribute__((aligned(16))) u16 ta[GfTile<ACOL>::SIZE], tb[GfTile<BCOL>::SIZE];
    const long mt = (P.M + GF_BM - 1) / GF_BM, nt = (P.N + GF_BN - 1) / GF_BN, items = mt * nt * P.nsplit, per = (items + 7) / 8;
    const long item = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);  // one XCD's L2 sees consecutive tiles
    if (item >= items) return;
    const long m0 = item / nt % mt * GF_BM, n0 = item % nt * GF_BN, split = item / (nt * mt);
    const long kt = (P.K + GF_BK - 1) / GF_BK, kper = (kt + P.nsplit - 1) / P.nsplit * GF_BK;
    const long k0 = split * kper, kend = k0 + kper < P.K ? k0 + kper : P.K;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    f16v acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    GfTile<ACOL> ga;
    GfTile<BCOL> gb;
    if (k0 < kend) ga.load(P.a, m0, k0, kend, false), gb.load(P.b, n0, k0, kend, P.glu_rows);
    for (long k = k0; k < kend; k += GF_BK) {
        __syncthreads();
        ga.store(ta), gb.store(tb);
        __syncthreads();
        if (k + GF_BK < kend) ga.load(P.a, m0, k + GF_BK, kend, false), gb.load(P.b, n0, k + GF_BK, kend, P.glu_rows);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const bf8 a0 = GfTile<ACOL>::operand(ta, wm, kk, lane), a1 = GfTile<ACOL>::operand(ta, wm + 32, kk, lane);
            const bf8 b0 = GfTile<BCOL>::operand(tb, wn, kk, lane), b1 = GfTile<BCOL>::operand(tb, wn + 32, kk, lane);
            acc[0][0] = PCM_MFMA16(a0, b0, acc[0][0]), acc[0][1] = PCM_MFMA16(a0, b1, acc[0][1]);
            acc[1][0] = PCM_MFMA16(a1, b0, acc[1][0]), acc[1][1] = PCM_MFMA16(a1, b1, acc[1][1]);
        }
    }
    const int col = lane & 31;
    if constexpr (EP == EP_GLU) {
        const long f = (n0 + wn) / 2 + col;
        const bool in = f < P.F;
        const float ba = in && P.bias0 ? bf2f(P.bias0[f]) : 0.f, bu = in && P.bias1 ? bf2f(P.bias1[f]) : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const long row = m0 + wm + 32 * i + crow(r, lane);
                if (row >= P.M) continue;
                const float a = acc[i][0][r] + ba, u = acc[i][1][r] + bu;
                if (P.out) P.out[row * P.Fp + f] = gf_bf(in ? a : 0.f), P.out1[row * P.Fp + f] = gf_bf(in ? u : 0.f);
                P.h[row * P.Fp + f] = gf_bf(in ? gf_act(a, P.act) * u : 0.f);
            }
    } else if constexpr (EP == EP_DGLU) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long f = n0 + wn + 32 * j + col;
            if (f >= P.Fp) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const long row = m0 + wm + 32 * i + crow(r, lane);
                    if (row >= P.M) continue;
                    const float a = bf2f(P.ea[row * P.Fp + f]), u = bf2f(P.eu[row * P.Fp + f]), dh = acc[i][j][r];
                    const float2 g = gf_act_grad(a, P.act);
                    P.out[row * 2 * P.Fp + f] = gf_bf(f < P.F ? dh * u * g.y : 0.f);
                    P.out[row * 2 * P.Fp + P.Fp + f] = gf_bf(f < P.F ? dh * g.x : 0.f);
                }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long n = n0 + wn + 32 * j + col;
            if (n >= P.N) continue;
            const float bias = EP == EP_OUT && P.bias0 ? bf2f(P.bias0[n]) : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const long row = m0 + wm + 32 * i + crow(r, lane);
                    if (row >= P.M) continue;
                    if (P.nsplit > 1) {
                        P.part[(split * P.M + row) * P.N + n] = acc[i][j][r];
                    } else if constexpr (EP == EP_WGRAD) {  // rows of the second part go to the second gradient
                        const bool second = row >= P.osplit;
                        const long rr = second ? row - P.osplit : row;
                        if (rr < P.F) (second ? P.out1 : P.out)[rr * P.ldo + n] = gf_bf(acc[i][j][r]);
                    } else {
                        P.out[row * P.ldo + n] = gf_bf(acc[i][j][r] + bias);
                    }
                }
        }
    }
}

// out = sum of the splits in split order
__global__ void __launch_bounds__(256) pcm_gated_join_kernel(GfParams P)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= P.M * P.N) return;
    const long row = i / P.N, n = i - row * P.N;
    const bool second = row >= P.osplit;
    const long rr = second ? row - P.osplit : row;
    if (rr >= P.F) return;
    float s = 0.f;
    for (int k = 0; k < P.nsplit; ++k) s += P.part[(long)k * P.M * P.N + i];
    (second ? P.out1 : P.out)[rr * P.ldo + n] = gf_bf(s);
}

// Column sums of da | du and of dy for the bias gradients: `slots` partial rows each (fixed row ranges: the order never changes),
// then one thread per column.
struct GfSums {
    const u16 *g[2];
    long ld[2], rows;
    int C[2], slots;
    float *part[2];
    u16 *out[3];
    int F, Fp;
};
__global__ void __launch_bounds__(256) pcm_gated_colsum_kernel(GfSums P)
{
    const int j = blockIdx.z, c = (int)blockIdx.x * 512 + 2 * (int)threadIdx.x;
    if (c >= P.C[j]) return;
    const long per = (P.rows + P.slots - 1) / P.slots, r0 = blockIdx.y * per, r1 = r0 + per < P.rows ? r0 + per : P.rows;
    float a = 0.f, b = 0.f;
#pragma unroll 8
    for (long r = r0; r < r1; ++r) {
        const uint32_t w = *(const uint32_t *)(P.g[j] + r * P.ld[j] + c);
        a += __uint_as_float(w << 16), b += __uint_as_float(w & 0xFFFF0000u);
    }
    *(float2 *)(P.part[j] + (long)blockIdx.y * P.C[j] + c) = make_float2(a, b);
}
__global__ void __launch_bounds__(256) pcm_gated_colsum_join_kernel(GfSums P, int E)
{
    const int j = blockIdx.z, c = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (c >= P.C[j]) return;
    float s = 0.f;
    for (int k = 0; k < P.slots; ++k) s += P.part[j][(long)k * P.C[j] + c];
    if (j == 1) {
        if (c < E) P.out[2][c] = gf_bf(s);
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

long gf_up(long v, long m) { return (v + m - 1) / m * m; }
bool gf_fits(const void *p, long ld, int cols) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && cols % 8 == 0; }

// Lays out the copies a call needs: `get` returns the matrix to use in place of p.
struct GfPacker {
    GfPack P;
    char *at, *end;
    long used;
    GfPacker(void *ws, long bytes) : at((char *)ws), end((char *)ws + bytes), used(0) { P.n = 0; }
    const u16 *get(const void *p, long rows, int cols, long &ld)
    {
        if (gf_fits(p, ld, cols)) return (const u16 *)p;
        const int ldp = (int)gf_up(cols, 8), j = P.n++;
        const long bytes = gf_up(rows * ldp * 2, 256);
        P.src[j] = (const u16 *)p, P.dst[j] = (u16 *)at, P.rows[j] = rows, P.ld[j] = ld, P.cols[j] = cols, P.ldp[j] = ldp;
        P.end[j] = (j ? P.end[j - 1] : 0) + rows * ldp / 8;
        at += bytes, used += bytes;
        ld = ldp;
        return P.dst[j];
    }
    bool room() const { return used == 0 || at <= end; }
    void run(hipStream_t s)
    {
        if (P.n) hipLaunchKernelGGL(pcm_gated_pack_kernel, dim3((unsigned)((P.end[P.n - 1] + 255) / 256)), dim3(256), 0, s, P);
    }
};

GfMat gf_mat(const u16 *p, long ld, long rows, long cols) { return GfMat{p, p, ld, 0x7FFFFFFF, (int)rows, 0, (int)cols}; }
GfMat gf_mat2(const u16 *p0, const u16 *p1, long ld, long split, long rows, long cols) { return GfMat{p0, p1, ld, (int)split, (int)rows, (int)rows, (int)cols}; }

template <int EP, bool ACOL, bool BCOL>
void gf_launch(const GfParams &P, hipStream_t s)
{
    const long items = gf_up(P.M, GF_BM) / GF_BM * (gf_up(P.N, GF_BN) / GF_BN) * P.nsplit;
    hipLaunchKernelGGL((pcm_gated_gemm_kernel<EP, ACOL, BCOL>), dim3((unsigned)gf_up(items, 8)), dim3(256), 0, s, P);
}

// Splits of a weight gradient's contraction (over the rows): its output has few tiles and the contraction is long, so the rows are
// shared out until about 512 workgroups run, at least 512 rows each (a split writes and re-reads the fp32 output).
int gf_splits(long M, long N, long K)
{
    const long tiles = gf_up(M, GF_BM) / GF_BM * (gf_up(N, GF_BN) / GF_BN);
    long n = (512 + tiles - 1) / tiles;
    n = n < K / 512 ? n : K / 512;
    return (int)(n < 1 ? 1 : (n > 32 ? 32 : n));
}

int gf_slots(long R) { return (int)(R < 64 ? 1 : (R / 32 > 128 ? 128 : R / 32)); }
long gf_sum_bytes(long R, int E, long Fp) { return gf_up(gf_slots(R) * (2 * Fp + gf_up(E, 8)) * 4, 256); }
bool gf_sizes_ok(long R, int E, int F) { return R <= 0x3FFFFFFFL && E <= (1 << 20) && F <= (1 << 20); }
long gf_pack_bytes(long rows, int cols) { return gf_up(rows * gf_up(cols, 8) * 2, 256); }

}  // namespace

extern "C" long pcm_gated_ffn_hidden_ld(int F) { return F > 0 ? gf_up(F, 64) : 0; }

extern "C" long pcm_gated_ffn_ws_bytes(long R, int E, int F, int backward)
{
    if (R <= 0 || E <= 0 || F <= 0) return 0;
    const long Fp = gf_up(F, 64);
    // copies: x and dy (any strides), the three weights
    long n = gf_pack_bytes(R, E) * (backward ? 2 : 1) + 2 * gf_pack_bytes(F, E) + gf_pack_bytes(E, F);
    if (backward) {
        n += gf_up(R * 2 * Fp * 2, 256);  // da | du
        const long w1 = gf_splits(2 * Fp, E, R) > 1 ? gf_splits(2 * Fp, E, R) * 2 * Fp * E * 4 : 0;
        const long w2 = gf_splits(E, F, R) > 1 ? gf_splits(E, F, R) * (long)E * F * 4 : 0;
        n += gf_up(w1 > w2 ? w1 : w2, 256);
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
    GfPacker pk(ws, ws ? ws_bytes : 0);
    long ldx = x_ls, ldg = E, ldu = E, ldd = F;
    const u16 *px = pk.get(x, R, E, ldx);
    const u16 *pg = pk.get(wg, F, E, ldg), *pu = pk.get(wu, F, E, ldu);  // one row length either way
    const u16 *pd = pk.get(wd, E, F, ldd);
    if (!pk.room()) return PCM_ERR_BAD_ARG;
    pk.run(s);
    const long Ep = gf_up(E, 8);
    GfParams P{};
    P.a = gf_mat(px, ldx, R, Ep), P.b = gf_mat2(pg, pu, ldg, Fp, F, Ep);
    P.M = R, P.N = 2 * Fp, P.K = Ep, P.glu_rows = 1, P.act = act, P.nsplit = 1, P.F = F, P.Fp = Fp;
    P.bias0 = (const u16 *)bg, P.bias1 = (const u16 *)bu, P.out = (u16 *)a, P.out1 = (u16 *)u, P.h = (u16 *)h;
    gf_launch<EP_GLU, false, false>(P, s);
    GfParams Q{};
    Q.a = gf_mat((const u16 *)h, Fp, R, Fp), Q.b = gf_mat(pd, ldd, E, gf_up(F, 8));
    Q.M = R, Q.N = E, Q.K = gf_up(F, 8), Q.nsplit = 1, Q.bias0 = (const u16 *)bd, Q.out = (u16 *)y, Q.ldo = E;
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
    const int s1 = gf_splits(2 * Fp, E, R), s2 = gf_splits(E, F, R);
    const long w1 = s1 > 1 ? s1 * 2 * Fp * E * 4 : 0, w2 = s2 > 1 ? s2 * (long)E * F * 4 : 0;
    at += gf_up(w1 > w2 ? w1 : w2, 256);
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
        P.out = dau, P.ea = (const u16 *)a, P.eu = (const u16 *)u;
        gf_launch<EP_DGLU, false, true>(P, s);
    }
    if (dx) {
        GfParams P{};
        P.a = gf_mat(dau, 2 * Fp, R, 2 * Fp), P.b = gf_mat2(pg, pu, ldg, Fp, F, Ep);
        P.M = R, P.N = E, P.K = 2 * Fp, P.nsplit = 1, P.out = (u16 *)dx, P.ldo = E;
        gf_launch<EP_DX, false, true>(P, s);
    }
    if (dwg) {
        GfParams P{};
        P.a = gf_mat(dau, 2 * Fp, R, 2 * Fp), P.b = gf_mat(px, ldx, R, Ep);
        P.M = 2 * Fp, P.N = E, P.K = R, P.nsplit = s1, P.F = F, P.out = (u16 *)dwg, P.out1 = (u16 *)dwu, P.ldo = E, P.part = part;
        P.osplit = Fp;
        gf_launch<EP_WGRAD, true, true>(P, s);
        if (s1 > 1) hipLaunchKernelGGL(pcm_gated_join_kernel, dim3((unsigned)((P.M * P.N + 255) / 256)), dim3(256), 0, s, P);
    }
    if (dwd) {
        GfParams P{};
        P.a = gf_mat(py, ldy, R, Ep), P.b = gf_mat((const u16 *)h, Fp, R, Fp);
        P.M = E, P.N = F, P.K = R, P.nsplit = s2, P.F = E, P.osplit = E, P.out = (u16 *)dwd, P.ldo = F, P.part = part;
        gf_launch<EP_WGRAD, true, true>(P, s);
        if (s2 > 1) hipLaunchKernelGGL(pcm_gated_join_kernel, dim3((unsigned)((P.M * P.N + 255) / 256)), dim3(256), 0, s, P);
    }
    if (dbg || dbd) {
        GfSums P{};
        P.rows = R, P.slots = gf_slots(R), P.F = F, P.Fp = (int)Fp;
        P.g[0] = dau, P.ld[0] = 2 * Fp, P.C[0] = dbg ? (int)(2 * Fp) : 0, P.part[0] = sums, P.out[0] = (u16 *)dbg, P.out[1] = (u16 *)dbu;
        P.g[1] = py, P.ld[1] = ldy, P.C[1] = dbd ? (int)Ep : 0, P.part[1] = sums + P.slots * 2 * Fp, P.out[2] = (u16 *)dbd;
        const long widest = P.C[0] > P.C[1] ? P.C[0] : P.C[1];
        hipLaunchKernelGGL(pcm_gated_colsum_kernel, dim3((unsigned)((widest + 511) / 512), P.slots, 2), dim3(256), 0, s, P);
        hipLaunchKernelGGL(pcm_gated_colsum_join_kernel, dim3((unsigned)((widest + 255) / 256), 1, 2), dim3(256), 0, s, P, E);
    }
    return PCM_LAUNCH_STATUS();
}

// cross_attn.hip -- attention of a set of queries over an encoder's states of another length.
//
//   O = softmax(scale * Q K^T) V per head; the keys of a row are those of its sequence that the padding mask leaves; a row without a
//   key is zero (its lse is -inf and its gradients are zero).  Query head h reads key head h / G, G = H / Hkv.
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO * O),  dQ = scale dS K,  dK = scale dS^T Q.
//
// Sides.  Each side is padded (sequence b at base + b * batch stride, all of one length) or packed (all rows side by side, sequence b
// = rows [offset[b - 1], offset[b]), the layout of this library's point clouds).  Rows of a packed side behind the last sequence form
// one more sequence without partners: their outputs and gradients are zero.  Offsets are clamped to the row count on the device.
// The rows of one (sequence, key head) are its tokens times its G heads, r = token * G + g: the heads that share a key head fill a tile
// together, whatever L is, and their dK / dV sums need no second pass.
//
// Matrix operands (v_mfma_f32_32x32x16_bf16).  Scores are computed TRANSPOSED in the row kernels (S^T = K Q^T: a lane owns one row, 16
// keys of each 32 in its registers), so the softmax statistics are lane-local up to one exchange between the two 32-lane halves, and
// the exponentials, packed in register order, ARE the B operand of O^T = V^T P^T: the order of the contracted keys is free as long as
// V^T's operand uses the same, and ds_read_b64_tr_b16 delivers V^T from the row-major tile in that order.  The key kernel is the mirror
// image (S = Q K^T: a lane owns one key).  Nothing is ever transposed through registers or a second LDS copy.
//
// Masked or absent keys are zeroed in K and V where a tile is staged (a NaN or infinity in padding must not meet a zero weight) and
// their scores are replaced by -inf.  Sums, maxima, lse, delta and accumulators are fp32; P and dS are rounded to bf16 (one half step,
// 2^-8 relative at most) because the matrix operands are bf16; outputs are rounded once.
#include "pcm_attn.hpp"

namespace {

constexpr int XA_ROWS = 128;  // rows of a row kernel's workgroup, keys of the key kernel's (4 waves of 32)
constexpr int XA_TILE = 64;   // rows of the other side staged at a time
constexpr float XA_LOG2E = 1.44269504088896340736f;

struct XaParams {
    const u16 *q, *k, *v, *dout;
    long q_bs, q_ls, q_hs, k_bs, k_ls, k_hs, v_bs, v_ls, v_hs, g_bs, g_ls, g_hs;
    const unsigned char *mask;
    long mask_bs;
    const int *q_off, *kv_off;
    int B, H, Hkv, G, D, L, S;
    long q_rows, kv_rows;
    float scale;
    int tiles, nsplit;
    u16 *out, *dq, *dk, *dv;
    float *lse, *delta, *part_o, *part_ml;
};

// One side of one sequence: row0 = index of its first row among all rows of the side, n = its rows.
struct XaSpan {
    long row0;
    int n;
};
__device__ __forceinline__ XaSpan xa_span(const int *off, int b, int B, int len, long rows)
{
    if (off == nullptr) return {(long)b * len, len};
    long lo = b > 0 ? (long)off[b - 1] : 0l, hi = b < B ? (long)off[b] : rows;
    lo = lo < 0 ? 0 : (lo > rows ? rows : lo), hi = hi < lo ? lo : (hi > rows ? rows : hi);
    return {lo, (int)(hi - lo)};
}

// Which (sequence, tile of it) is the t-th tile of a side, `per` tile rows, `mult` rows per token.  False: no such tile.  A packed side's
// tile counts are summed 64 sequences at a time, one per lane (an inclusive scan and one ballot).
__device__ __forceinline__ bool xa_locate(const int *off, int B, int len, long rows, int mult, int per, int t, int lane, int &b, int &tile)
{
    if (off == nullptr) {
        const int each = (int)(((long)len * mult + per - 1) / per);
        b = t / each, tile = t - b * each;
        return b < B;
    }
    long run = 0;
    for (int base = 0; base <= B; base += 64) {
        const int i = base + lane;
        const int mine = i <= B ? (int)(((long)xa_span(off, i, B, 0, rows).n * mult + per - 1) / per) : 0;
        int incl = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(incl, d);
            if (lane >= d) incl += up;
        }
        const unsigned long long past = __ballot(run + incl > t);
        if (past != 0) {
            const int f = __ffsll(past) - 1;
            b = base + f, tile = (int)(t - run) - (__shfl(incl, f) - __shfl(mine, f));
            return true;
        }
        run += __shfl(incl, 63);
    }
    return false;
}

// consecutive work items (the tiles of one key head, which read the same K and V) go to one XCD's contiguous share
__device__ __forceinline__ long xa_item(long items)
{
    const long per = (items + 7) / 8;
    return (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
}

typedef s4 __attribute__((address_space(3))) * xa_lds_s4;
__device__ __forceinline__ s4 xa_tr(const u16 *p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((xa_lds_s4)p); }

// Transposed operand: lane <-> channel 32 * blk + lane % 32, contracted index i of half h <-> tile row row16 + 4 h + i % 4 + 8 (i / 4):
// the order in which a 32 x 32 accumulator holds 16 of its rows.
template <int LD>
__device__ __forceinline__ bf8 xa_transposed(const u16 *tile, int row16, int blk, int lane)
{
    const int p = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
    const u16 *a = tile + (row16 + 4 * h + (p >> 2)) * LD + 32 * blk + 16 * g + 4 * (p & 3);
    return cat8(xa_tr(a), xa_tr(a + 8 * LD));
}
__device__ __forceinline__ f16v xa_zero16()
{
    f16v z = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    return z;
}
__device__ __forceinline__ bf8 xa_pack(const f16v &s, int u)  // rows 16 u .. + 15 of a 32-row accumulator, in operand order
{
    return as_bf8(make_uint4(cvt_pk_bf16(s[8 * u], s[8 * u + 1]), cvt_pk_bf16(s[8 * u + 2], s[8 * u + 3]), cvt_pk_bf16(s[8 * u + 4], s[8 * u + 5]),
                             cvt_pk_bf16(s[8 * u + 6], s[8 * u + 7])));
}
// the 16-byte pieces of one row (lane % 32 owns the row, the halves alternate 8 channels): a register-resident B operand
template <int DP>
__device__ __forceinline__ void xa_row_operand(const u16 *row, bool ok, int D, int h, bf8 (&f)[DP / 16])
{
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
        f[t] = as_bf8(ok && 16 * t + 8 * h < D ? *(const uint4 *)(row + 16 * t + 8 * h) : make_uint4(0, 0, 0, 0));
}

// 64 rows of a strided matrix on their way into LDS: 16-byte pieces, DP / 32 per thread, requested together.
template <int DP>
struct XaStage {
    static constexpr int N = DP / 32, PIECES = DP / 8, LD = DP + 8;
    uint4 d[N];
    __device__ __forceinline__ void load(const u16 *base, long ls, int row0, int n, int D)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + 256 * i, r = c / PIECES, p = c - r * PIECES;
            d[i] = row0 + r < n && 8 * p < D ? *(const uint4 *)(base + (long)(row0 + r) * ls + 8 * p) : make_uint4(0, 0, 0, 0);
        }
    }
    // visible: bit r <-> row r of the tile
    __device__ __forceinline__ void store(u16 *tile, unsigned long long visible) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + 256 * i, r = c / PIECES, p = c - r * PIECES;
            const bool keep = (visible >> r) & 1;
            *(uint4 *)(tile + r * LD + 8 * p) = keep ? d[i] : make_uint4(0, 0, 0, 0);
        }
    }
};

// rows r = token * G + g of a strided (token, head, channel) matrix
template <int DP>
struct XaRowStage {
    static constexpr int N = DP / 32, PIECES = DP / 8, LD = DP + 8;
    uint4 d[N];
    __device__ __forceinline__ void load(const u16 *base, long ls, long hs, int row0, int n, int G, int D)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + 256 * i, r = c / PIECES, p = c - r * PIECES, row = row0 + r, tok = row / G;
            d[i] = row < n && 8 * p < D ? *(const uint4 *)(base + (long)tok * ls + (long)(row - tok * G) * hs + 8 * p) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(u16 *tile) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = threadIdx.x + 256 * i, r = c / PIECES, p = c - r * PIECES;
            *(uint4 *)(tile + r * LD + 8 * p) = d[i];
        }
    }
};

__device__ __forceinline__ unsigned xa_mask_byte(const unsigned char *m, int key, int n) { return m != nullptr && key < n ? (unsigned)m[key] : 0u; }

__device__ __forceinline__ void xa_store_row(u16 *row, int D, int h, int blk, const f16v &o, float f)
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = 32 * blk + 8 * g + 4 * h;
        if (d < D) *(uint2 *)(row + d) = make_uint2(cvt_pk_bf16(o[4 * g] * f, o[4 * g + 1] * f), cvt_pk_bf16(o[4 * g + 2] * f, o[4 * g + 3] * f));
    }
}
__device__ __forceinline__ void xa_store_part(float *row, int D, int h, int blk, const f16v &o)
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = 32 * blk + 8 * g + 4 * h;
        if (d < D) *(float4 *)(row + d) = make_float4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
    }
}

// What a row kernel's workgroup works on.
struct XaRows {
    int b, kvh, split, row, tok, head, nrows, key_lo, key_hi;  // key range: multiples of XA_TILE
    bool ok;
    XaSpan qs, ks;
    const u16 *k, *v;
    const unsigned char *mask;
    long out_row;  // (q row) * H + head
};
__device__ __forceinline__ bool xa_rows(const XaParams &P, int lane, int wave, XaRows &R)
{
    const long items = (long)P.tiles * P.Hkv * P.nsplit, item = xa_item(items);
    if (item >= items) return false;
    int tile;
    const long rest = item / P.tiles;
    R.kvh = (int)(rest % P.Hkv), R.split = (int)(rest / P.Hkv);
    if (!xa_locate(P.q_off, P.B, P.L, P.q_rows, P.G, XA_ROWS, (int)(item % P.tiles), lane, R.b, tile)) return false;
    R.qs = xa_span(P.q_off, R.b, P.B, P.L, P.q_rows);
    R.ks = R.b < P.B ? xa_span(P.kv_off, R.b, P.B, P.S, P.kv_rows) : XaSpan{0, 0};
    R.nrows = R.qs.n * P.G;
    R.row = tile * XA_ROWS + wave * 32 + (lane & 31), R.ok = R.row < R.nrows;
    R.tok = R.ok ? R.row / P.G : 0, R.head = R.kvh * P.G + (R.ok ? R.row - R.tok * P.G : 0);
    R.out_row = (R.qs.row0 + R.tok) * P.H + R.head;
    const int kt = (R.ks.n + XA_TILE - 1) / XA_TILE, per = (kt + P.nsplit - 1) / P.nsplit;
    R.key_lo = R.split * per * XA_TILE, R.key_hi = min(R.ks.n, R.key_lo + per * XA_TILE);
    const long kb = P.kv_off ? 0 : (long)R.b, kr = P.kv_off ? R.ks.row0 : 0;
    if (R.ks.n == 0) return true;
    R.k = P.k + kb * P.k_bs + kr * P.k_ls + (long)R.kvh * P.k_hs;
    R.v = P.v + kb * P.v_bs + kr * P.v_ls + (long)R.kvh * P.v_hs;
    R.mask = P.mask ? P.mask + (P.kv_off ? R.ks.row0 : kb * P.mask_bs) : nullptr;
    return true;
}
__device__ __forceinline__ const u16 *xa_q_row(const XaParams &P, const u16 *base, long bs, long ls, long hs, const XaRows &R)
{
    return base + (P.q_off ? (R.qs.row0 + R.tok) * ls : R.b * bs + R.tok * ls) + (long)R.head * hs;
}

template <int DP>
__global__ void __launch_bounds__(256, 2) pcm_xattn_fwd_kernel(XaParams P)
{
    constexpr int LD = DP + 8;
    __shared__ __attribute__((aligned(16))) u16 sk[XA_TILE * LD], sv[XA_TILE * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
    XaRows R;
    if (!xa_rows(P, lane, wave, R)) return;
    bf8 qf[DP / 16];
    xa_row_operand<DP>(xa_q_row(P, P.q, P.q_bs, P.q_ls, P.q_hs, R), R.ok, P.D, h, qf);
    f16v o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = xa_zero16();
    float m = -INFINITY, l = 0.f;
    const float c = P.scale * XA_LOG2E;
    XaStage<DP> gk, gv;
    unsigned mb = 0;
    if (R.key_lo < R.key_hi) {
        mb = xa_mask_byte(R.mask, R.key_lo + lane, R.ks.n);
        gk.load(R.k, P.k_ls, R.key_lo, R.ks.n, P.D), gv.load(R.v, P.v_ls, R.key_lo, R.ks.n, P.D);
    }
    for (int key0 = R.key_lo; key0 < R.key_hi; key0 += XA_TILE) {
        const unsigned long long vis = __ballot(key0 + lane < R.ks.n && mb == 0u);
        __syncthreads();
        gk.store(sk, vis), gv.store(sv, vis);
        __syncthreads();
        if (key0 + XA_TILE < R.key_hi) {
            mb = xa_mask_byte(R.mask, key0 + XA_TILE + lane, R.ks.n);
            gk.load(R.k, P.k_ls, key0 + XA_TILE, R.ks.n, P.D), gv.load(R.v, P.v_ls, key0 + XA_TILE, R.ks.n, P.D);
        }
        if (vis == 0) continue;
        f16v s[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            s[j] = xa_zero16();
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) s[j] = PCM_MFMA16(lds_bf8(sk + (32 * j + col) * LD + 16 * t + 8 * h), qf[t], s[j]);
        }
        if (vis != ~0ull) {
            const unsigned long long mine = vis >> (4 * h);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (32 * j + (r & 3) + 8 * (r >> 2))) & 1)) s[j][r] = -INFINITY;
        }
        float mx = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = max3f(mx, s[0][r], s[1][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mc = mx == -INFINITY ? 0.f : mx * c;
        const float alpha = __builtin_amdgcn_exp2f(__builtin_fmaf(m, c, -mc));
        m = mx;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], c, -mc));
                sum += s[j][r];
            }
        l = __builtin_fmaf(l, alpha, sum);
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) o[i] *= alpha;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const bf8 p = xa_pack(s[t >> 1], t & 1);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] = PCM_MFMA16(xa_transposed<LD>(sv, 16 * t, i, lane), p, o[i]);
        }
    }
    l += __shfl_xor(l, 32);
    if (!R.ok) return;
    if (P.nsplit > 1) {
        const long at = (long)R.split * P.q_rows * P.H + R.out_row;
        if (h == 0) *(float2 *)(P.part_ml + 2 * at) = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) xa_store_part(P.part_o + at * P.D, P.D, h, i, o[i]);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // l >= 1 with a key (its largest weight is 1), NaN with a NaN among the scores
    if (P.lse && h == 0) P.lse[R.out_row] = l == 0.f ? -INFINITY : m * P.scale + __logf(l);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) xa_store_row(P.out + R.out_row * P.D, P.D, h, i, o[i], inv);
}

// joins the splits of a row: one wave per (row, head), lanes over channels
__global__ void __launch_bounds__(256) pcm_xattn_join_kernel(XaParams P)
{
    const long rows = P.q_rows * P.H, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    float m = -INFINITY;
    for (int s = 0; s < P.nsplit; ++s) m = fmaxf(m, P.part_ml[2 * (s * rows + row)]);
    const float c = P.scale * XA_LOG2E;
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int s = 0; s < P.nsplit; ++s) {
        const float2 ml = *(const float2 *)(P.part_ml + 2 * (s * rows + row));
        if (ml.y == 0.f) continue;  // no key in this split
        const float w = __builtin_amdgcn_exp2f((ml.x - m) * c);
        l = __builtin_fmaf(ml.y, w, l);
        const float *po = P.part_o + (s * rows + row) * P.D;
        if (2 * lane < P.D) o0 = __builtin_fmaf(po[2 * lane], w, o0), o1 = __builtin_fmaf(po[2 * lane + 1], w, o1);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (P.lse && lane == 0) P.lse[row] = l == 0.f ? -INFINITY : m * P.scale + __logf(l);
    if (2 * lane < P.D) *(uint32_t *)(P.out + row * P.D + 2 * lane) = cvt_pk_bf16(o0 * inv, o1 * inv);
}

// delta = rowsum(dO * O): 16 lanes per (row, head), 8 channels each
__global__ void __launch_bounds__(256) pcm_xattn_delta_kernel(XaParams P)
{
    const long row = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int d = 8 * (threadIdx.x & 15);
    float s = 0.f;
    if (row < P.q_rows * P.H && d < P.D) {
        const long tok = row / P.H, head = row - tok * P.H;
        const long b = P.q_off ? 0 : tok / P.L, l = P.q_off ? tok : tok - b * P.L;
        const uint4 a = *(const uint4 *)(P.out + row * P.D + d), g = *(const uint4 *)(P.dout + b * P.g_bs + l * P.g_ls + head * P.g_hs + d);
        const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s = __builtin_fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
            s = __builtin_fmaf(__uint_as_float(x[i] & 0xFFFF0000u), __uint_as_float(y[i] & 0xFFFF0000u), s);
        }
    }
    for (int k = 8; k > 0; k >>= 1) s += __shfl_xor(s, k);
    if ((threadIdx.x & 15) == 0 && row < P.q_rows * P.H) P.delta[row] = s;
}

template <int DP>
__global__ void __launch_bounds__(256, 2) pcm_xattn_dq_kernel(XaParams P)
{
    constexpr int LD = DP + 8;
    __shared__ __attribute__((aligned(16))) u16 sk[XA_TILE * LD], sv[XA_TILE * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
    XaRows R;
    if (!xa_rows(P, lane, wave, R)) return;
    bf8 qf[DP / 16], gf[DP / 16];
    xa_row_operand<DP>(xa_q_row(P, P.q, P.q_bs, P.q_ls, P.q_hs, R), R.ok, P.D, h, qf);
    xa_row_operand<DP>(xa_q_row(P, P.dout, P.g_bs, P.g_ls, P.g_hs, R), R.ok, P.D, h, gf);
    const float lse = R.ok ? P.lse[R.out_row] : -INFINITY, delta = R.ok ? P.delta[R.out_row] : 0.f;
    const float l2 = lse == -INFINITY ? INFINITY : lse * XA_LOG2E;  // a row without a key: every weight 2^-inf = 0
    const float c = P.scale * XA_LOG2E;
    f16v o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = xa_zero16();
    XaStage<DP> gk, gv;
    unsigned mb = 0;
    if (R.key_lo < R.key_hi) {
        mb = xa_mask_byte(R.mask, R.key_lo + lane, R.ks.n);
        gk.load(R.k, P.k_ls, R.key_lo, R.ks.n, P.D), gv.load(R.v, P.v_ls, R.key_lo, R.ks.n, P.D);
    }
    for (int key0 = R.key_lo; key0 < R.key_hi; key0 += XA_TILE) {
        const unsigned long long vis = __ballot(key0 + lane < R.ks.n && mb == 0u);
        __syncthreads();
        gk.store(sk, vis), gv.store(sv, vis);
        __syncthreads();
        if (key0 + XA_TILE < R.key_hi) {
            mb = xa_mask_byte(R.mask, key0 + XA_TILE + lane, R.ks.n);
            gk.load(R.k, P.k_ls, key0 + XA_TILE, R.ks.n, P.D), gv.load(R.v, P.v_ls, key0 + XA_TILE, R.ks.n, P.D);
        }
        if (vis == 0) continue;
        const unsigned long long mine = vis >> (4 * h);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f16v s = xa_zero16(), dp = xa_zero16();
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                s = PCM_MFMA16(lds_bf8(sk + (32 * j + col) * LD + 16 * t + 8 * h), qf[t], s);
                dp = PCM_MFMA16(lds_bf8(sv + (32 * j + col) * LD + 16 * t + 8 * h), gf[t], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -l2));
                s[r] = p * (dp[r] - delta);
            }
            if (vis != ~0ull) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (32 * j + (r & 3) + 8 * (r >> 2))) & 1)) s[r] = 0.f;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bf8 ds = xa_pack(s, u);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) o[i] = PCM_MFMA16(xa_transposed<LD>(sk, 32 * j + 16 * u, i, lane), ds, o[i]);
            }
        }
    }
    if (!R.ok) return;
    const long at = (long)R.split * P.q_rows * P.H + R.out_row;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        if (P.nsplit > 1) xa_store_part(P.part_o + at * P.D, P.D, h, i, o[i]);
        else xa_store_row(P.dq + R.out_row * P.D, P.D, h, i, o[i], P.scale);
    }
}

// dQ of a row out of its splits, in split order
__global__ void __launch_bounds__(256) pcm_xattn_dq_join_kernel(XaParams P)
{
    const long pairs = P.q_rows * P.H * (P.D / 2), i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= pairs) return;
    float a = 0.f, b = 0.f;
    for (int s = 0; s < P.nsplit; ++s) {
        const float2 v = *(const float2 *)(P.part_o + 2 * (s * pairs + i));
        a += v.x, b += v.y;
    }
    *(uint32_t *)(P.dq + 2 * i) = cvt_pk_bf16(a * P.scale, b * P.scale);
}

template <int DP>
__global__ void __launch_bounds__(256, DP > 64 ? 1 : 2) pcm_xattn_dkv_kernel(XaParams P)
{
    constexpr int LD = DP + 8;
    __shared__ __attribute__((aligned(16))) u16 sq[XA_TILE * LD], sg[XA_TILE * LD];
    __shared__ __attribute__((aligned(16))) float sl[XA_TILE], sd[XA_TILE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
    const long items = (long)P.tiles * P.Hkv, item = xa_item(items);
    if (item >= items) return;
    int b, tile;
    const int kvh = (int)(item / P.tiles);
    if (!xa_locate(P.kv_off, P.B, P.S, P.kv_rows, 1, XA_ROWS, (int)(item % P.tiles), lane, b, tile)) return;
    const XaSpan ks = xa_span(P.kv_off, b, P.B, P.S, P.kv_rows);
    const XaSpan qs = b < P.B ? xa_span(P.q_off, b, P.B, P.L, P.q_rows) : XaSpan{0, 0};
    const int key = tile * XA_ROWS + wave * 32 + col, nrows = qs.n * P.G;
    const bool held = key < ks.n;
    const long key_row = ks.row0 + key, kb = P.kv_off ? 0 : (long)b, kr = P.kv_off ? key_row : (long)key;
    const bool seen = held && (P.mask == nullptr || P.mask[P.kv_off ? key_row : kb * P.mask_bs + key] == 0);
    bf8 kf[DP / 16], vf[DP / 16];
    xa_row_operand<DP>(P.k + kb * P.k_bs + kr * P.k_ls + (long)kvh * P.k_hs, seen, P.D, h, kf);
    xa_row_operand<DP>(P.v + kb * P.v_bs + kr * P.v_ls + (long)kvh * P.v_hs, seen, P.D, h, vf);
    const u16 *qb = nrows == 0 ? nullptr : P.q + (P.q_off ? qs.row0 * P.q_ls : b * P.q_bs) + (long)kvh * P.G * P.q_hs;
    const u16 *gb = nrows == 0 ? nullptr : P.dout + (P.q_off ? qs.row0 * P.g_ls : b * P.g_bs) + (long)kvh * P.G * P.g_hs;
    const float c = P.scale * XA_LOG2E;
    f16v dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = xa_zero16(), dv[i] = xa_zero16();
    XaRowStage<DP> rq, rg;
    float rl = INFINITY, rd = 0.f;
    const auto stats = [&](int row0) {  // thread t < 64: row row0 + t
        const int row = row0 + (int)threadIdx.x, tok = row / P.G;
        rl = INFINITY, rd = 0.f;
        if (threadIdx.x < XA_TILE && row < nrows) {
            const long at = (qs.row0 + tok) * P.H + kvh * P.G + (row - tok * P.G);
            const float lse = P.lse[at];
            rl = lse == -INFINITY ? INFINITY : lse * XA_LOG2E, rd = P.delta[at];
        }
    };
    if (nrows > 0) rq.load(qb, P.q_ls, P.q_hs, 0, nrows, P.G, P.D), rg.load(gb, P.g_ls, P.g_hs, 0, nrows, P.G, P.D), stats(0);
    for (int row0 = 0; row0 < nrows; row0 += XA_TILE) {
        __syncthreads();
        rq.store(sq), rg.store(sg);
        if (threadIdx.x < XA_TILE) sl[threadIdx.x] = rl, sd[threadIdx.x] = rd;
        __syncthreads();
        if (row0 + XA_TILE < nrows)
            rq.load(qb, P.q_ls, P.q_hs, row0 + XA_TILE, nrows, P.G, P.D), rg.load(gb, P.g_ls, P.g_hs, row0 + XA_TILE, nrows, P.G, P.D), stats(row0 + XA_TILE);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f16v s = xa_zero16(), dp = xa_zero16();
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
                s = PCM_MFMA16(lds_bf8(sq + (32 * j + col) * LD + 16 * t + 8 * h), kf[t], s);
                dp = PCM_MFMA16(lds_bf8(sg + (32 * j + col) * LD + 16 * t + 8 * h), vf[t], dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 l2 = *(const float4 *)(sl + 32 * j + 8 * g + 4 * h), de = *(const float4 *)(sd + 32 * j + 8 * g + 4 * h);
                const float a[4] = {l2.x, l2.y, l2.z, l2.w}, e[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 4 * g + i;
                    const float p = seen ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -a[i])) : 0.f;
                    dp[r] = p * (dp[r] - e[i]), s[r] = p;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bf8 p = xa_pack(s, u), ds = xa_pack(dp, u);
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    dv[i] = PCM_MFMA16(xa_transposed<LD>(sg, 32 * j + 16 * u, i, lane), p, dv[i]);
                    dk[i] = PCM_MFMA16(xa_transposed<LD>(sq, 32 * j + 16 * u, i, lane), ds, dk[i]);
                }
            }
        }
    }
    if (!held) return;
    const long at = (key_row * P.Hkv + kvh) * P.D;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        xa_store_row(P.dk + at, P.D, h, i, dk[i], P.scale);
        xa_store_row(P.dv + at, P.D, h, i, dv[i], 1.f);
    }
}

#define XA_BY_DIM(kernel, grid, s, P)                                                                       \
    do {                                                                                                    \
        if ((P).D <= 32) hipLaunchKernelGGL((kernel<32>), dim3(grid), dim3(256), 0, s, P);                  \
        else if ((P).D <= 64) hipLaunchKernelGGL((kernel<64>), dim3(grid), dim3(256), 0, s, P);             \
        else if ((P).D <= 96) hipLaunchKernelGGL((kernel<96>), dim3(grid), dim3(256), 0, s, P);             \
        else hipLaunchKernelGGL((kernel<128>), dim3(grid), dim3(256), 0, s, P);                             \
    } while (0)

bool xa_shape_ok(int H, int Hkv, int D) { return H > 0 && Hkv > 0 && H % Hkv == 0 && D >= 8 && D <= 128 && D % 8 == 0; }

// an upper bound on the tiles of a side: a packed side's sequences end inside a tile each
long xa_tiles(int packed, int B, int len, long rows, int mult, int per)
{
    return packed ? (rows * mult + per - 1) / per + B + 1 : (long)B * (((long)len * mult + per - 1) / per);
}

// Splits of the keys.  A workgroup per (tile, key head) is too few for 256 compute units when the rows are few (one token of a rollout,
// a decoder's 100 queries): the keys are then shared out until about 512 workgroups run, with at least 256 keys (4 tiles) each, since a
// split writes and re-reads its row's fp32 sums.
int xa_splits(int B, int H, int Hkv, int L, long q_rows, int q_packed, int S, long kv_rows, int kv_packed)
{
    const int G = H / Hkv;
    const long work = (q_packed ? (q_rows * G + XA_ROWS - 1) / XA_ROWS + B - 1 : xa_tiles(0, B, L, q_rows, G, XA_ROWS)) * Hkv;
    const long keys = kv_packed ? (kv_rows + B - 1) / B : S;
    long n = (512 + work - 1) / (work > 0 ? work : 1);
    n = n < keys / 256 ? n : keys / 256;
    return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
}

bool xa_strides_ok(const void *p, long bs, long ls, long hs) { return (((uintptr_t)p) & 15) == 0 && ((bs | ls | hs) & 7) == 0; }

int xa_fill(XaParams &P, int B, int H, int Hkv, int D, int L, long q_rows, const int *q_offset, int S, long kv_rows, const int *kv_offset,
            const void *q, long q_bs, long q_ls, long q_hs, const void *k, long k_bs, long k_ls, long k_hs, const void *v, long v_bs, long v_ls,
            long v_hs, const unsigned char *mask, long mask_bs, float scale)
{
    P = XaParams{};
    if (!xa_shape_ok(H, Hkv, D)) return PCM_ERR_UNSUPPORTED;
    if (!(scale > 0.f) || scale > 3.0e38f) return PCM_ERR_BAD_ARG;
    if (!q_offset) q_rows = (long)B * L;
    if (!kv_offset) kv_rows = (long)B * S;
    if (q_rows * H > 0x7FFFFFFFL || kv_rows > 0x7FFFFFFFL || (kv_rows + 127) / 128 * Hkv + (long)B * Hkv > 0x3FFFFFFFL) return PCM_ERR_UNSUPPORTED;
    if ((q_rows > 0 && !q) || (kv_rows > 0 && (!k || !v))) return PCM_ERR_BAD_ARG;
    if (!xa_strides_ok(q, q_bs, q_ls, q_hs) || !xa_strides_ok(k, k_bs, k_ls, k_hs) || !xa_strides_ok(v, v_bs, v_ls, v_hs)) return PCM_ERR_UNSUPPORTED;
    P.q = (const u16 *)q, P.k = (const u16 *)k, P.v = (const u16 *)v;
    P.q_bs = q_bs, P.q_ls = q_ls, P.q_hs = q_hs, P.k_bs = k_bs, P.k_ls = k_ls, P.k_hs = k_hs, P.v_bs = v_bs, P.v_ls = v_ls, P.v_hs = v_hs;
    P.mask = mask, P.mask_bs = mask_bs, P.q_off = q_offset, P.kv_off = kv_offset;
    P.B = B, P.H = H, P.Hkv = Hkv, P.G = H / Hkv, P.D = D, P.L = L, P.S = S, P.q_rows = q_rows, P.kv_rows = kv_rows, P.scale = scale;
    return PCM_OK;
}

unsigned xa_grid(long items) { return (unsigned)((items + 7) / 8 * 8); }

}  // namespace

extern "C" int pcm_cross_attn_supported(int H, int Hkv, int D) { return xa_shape_ok(H, Hkv, D) ? 1 : 0; }

extern "C" long pcm_cross_attn_ws_bytes(int B, int H, int Hkv, int D, int L, long q_rows, int q_packed, int S, long kv_rows, int kv_packed)
{
    if (B <= 0 || L < 0 || S < 0 || q_rows < 0 || kv_rows < 0 || !xa_shape_ok(H, Hkv, D)) return 0;
    if (!q_packed) q_rows = (long)B * L;
    const int n = xa_splits(B, H, Hkv, L, q_rows, q_packed, S, kv_rows, kv_packed);
    return n > 1 ? (long)n * q_rows * H * (D + 2) * 4 : 0;
}

extern "C" int pcm_cross_attn_forward_hip(int B, int H, int Hkv, int D, int L, long q_rows, const int *q_offset, int S, long kv_rows,
                                          const int *kv_offset, const void *q, long q_bs, long q_ls, long q_hs, const void *k, long k_bs,
                                          long k_ls, long k_hs, const void *v, long v_bs, long v_ls, long v_hs, const unsigned char *mask,
                                          long mask_bs, float scale, void *out, float *lse, void *ws, long ws_bytes, void *stream)
{
    if (B < 0 || H < 0 || Hkv < 0 || D < 0 || L < 0 || S < 0 || q_rows < 0 || kv_rows < 0) return PCM_ERR_BAD_ARG;
    if (B == 0 || (q_offset ? q_rows == 0 : L == 0)) return PCM_OK;
    XaParams P;
    const int bad = xa_fill(P, B, H, Hkv, D, L, q_rows, q_offset, S, kv_rows, kv_offset, q, q_bs, q_ls, q_hs, k, k_bs, k_ls, k_hs, v, v_bs, v_ls, v_hs,
                            mask, mask_bs, scale);
    if (bad) return bad;
    if (!out || (((uintptr_t)out | (uintptr_t)ws) & 15) != 0) return PCM_ERR_BAD_ARG;
    P.out = (u16 *)out, P.lse = lse;
    P.nsplit = xa_splits(B, H, Hkv, L, P.q_rows, q_offset != nullptr, S, P.kv_rows, kv_offset != nullptr);
    if (P.nsplit > 1) {
        if (!ws || ws_bytes < (long)P.nsplit * P.q_rows * H * (D + 2) * 4) return PCM_ERR_BAD_ARG;
        P.part_o = (float *)ws, P.part_ml = (float *)ws + (long)P.nsplit * P.q_rows * H * D;
    }
    P.tiles = (int)xa_tiles(q_offset != nullptr, B, L, P.q_rows, P.G, XA_ROWS);
    const hipStream_t s = (hipStream_t)stream;
    XA_BY_DIM(pcm_xattn_fwd_kernel, xa_grid((long)P.tiles * Hkv * P.nsplit), s, P);
    if (P.nsplit > 1) hipLaunchKernelGGL(pcm_xattn_join_kernel, dim3((unsigned)((P.q_rows * H + 3) / 4)), dim3(256), 0, s, P);
    return PCM_LAUNCH_STATUS();
}

extern "C" int pcm_cross_attn_backward_hip(int B, int H, int Hkv, int D, int L, long q_rows, const int *q_offset, int S, long kv_rows,
                                           const int *kv_offset, const void *q, long q_bs, long q_ls, long q_hs, const void *k, long k_bs,
                                           long k_ls, long k_hs, const void *v, long v_bs, long v_ls, long v_hs, const unsigned char *mask,
                                           long mask_bs, float scale, const void *out, const float *lse, const void *dout, long g_bs, long g_ls,
                                           long g_hs, float *delta, void *dq, void *dk, void *dv, void *ws, long ws_bytes, void *stream)
{
    if (B < 0 || H < 0 || Hkv < 0 || D < 0 || L < 0 || S < 0 || q_rows < 0 || kv_rows < 0) return PCM_ERR_BAD_ARG;
    if (B == 0) return PCM_OK;
    XaParams P;
    const int bad = xa_fill(P, B, H, Hkv, D, L, q_rows, q_offset, S, kv_rows, kv_offset, q, q_bs, q_ls, q_hs, k, k_bs, k_ls, k_hs, v, v_bs, v_ls, v_hs,
                            mask, mask_bs, scale);
    if (bad) return bad;
    if (P.q_rows > 0 && (!out || !lse || !dout || !delta || !dq)) return PCM_ERR_BAD_ARG;
    if (P.kv_rows > 0 && (!dk || !dv)) return PCM_ERR_BAD_ARG;
    if (!xa_strides_ok(dout, g_bs, g_ls, g_hs)) return PCM_ERR_UNSUPPORTED;
    if ((((uintptr_t)out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15) != 0) return PCM_ERR_BAD_ARG;
    P.out = (u16 *)out, P.lse = (float *)lse, P.dout = (const u16 *)dout, P.g_bs = g_bs, P.g_ls = g_ls, P.g_hs = g_hs;
    P.delta = delta, P.dq = (u16 *)dq, P.dk = (u16 *)dk, P.dv = (u16 *)dv;
    const hipStream_t s = (hipStream_t)stream;
    if (P.q_rows > 0) {
        P.nsplit = xa_splits(B, H, Hkv, L, P.q_rows, q_offset != nullptr, S, P.kv_rows, kv_offset != nullptr);
        if (P.nsplit > 1) {
            if (!ws || ws_bytes < (long)P.nsplit * P.q_rows * H * D * 4) return PCM_ERR_BAD_ARG;
            P.part_o = (float *)ws;
        }
        hipLaunchKernelGGL(pcm_xattn_delta_kernel, dim3((unsigned)((P.q_rows * H + 15) / 16)), dim3(256), 0, s, P);
        P.tiles = (int)xa_tiles(q_offset != nullptr, B, L, P.q_rows, P.G, XA_ROWS);
        XA_BY_DIM(pcm_xattn_dq_kernel, xa_grid((long)P.tiles * Hkv * P.nsplit), s, P);
        if (P.nsplit > 1) hipLaunchKernelGGL(pcm_xattn_dq_join_kernel, dim3((unsigned)((P.q_rows * H * (D / 2) + 255) / 256)), dim3(256), 0, s, P);
    }
    if (P.kv_rows > 0) {
        P.tiles = (int)xa_tiles(kv_offset != nullptr, B, S, P.kv_rows, 1, XA_ROWS);
        XA_BY_DIM(pcm_xattn_dkv_kernel, xa_grid((long)P.tiles * Hkv), s, P);
    }
    return PCM_LAUNCH_STATUS();
}

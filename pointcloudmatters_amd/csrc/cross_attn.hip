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
// their scores start from -inf.  Sums, maxima, lse, delta and accumulators are fp32; P and dS are rounded to bf16 (one half step,
// 2^-8 relative at most) because the matrix operands are bf16; outputs are rounded once.  For delta O is
// kept in fp32 beside lse: over few keys a rounded O took dQ and dK from 2.4e-3 of their norm to 2.9e-3.
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
    int tiles, each, nsplit;  // each: tiles of a padded sequence
    u16 *out, *dq, *dk, *dv;
    float *o32, *lse, *delta, *part_o, *part_ml;
    // row / G by one multiplication: g_inv = 2^g_shift / G rounded up, 2^(g_shift - 31) >= G.  g_inv * G exceeds 2^g_shift by less than G,
    // so the product is off by less than row * G <= 2^31 * 2^(g_shift - 31) of 2^g_shift: exact for every row below 2^31
    uint32_t g_inv;
    int g_shift;
    __device__ __forceinline__ int token(int row) const { return (int)(((uint64_t)(uint32_t)row * g_inv) >> g_shift); }
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
            b = base + f, tile = __builtin_amdgcn_readfirstlane((int)(t - run) - (__shfl(incl, f) - __shfl(mine, f)));
            return true;
        }
        run += __shfl(incl, 63);
    }
    return false;
}

// Consecutive work items (the tiles of one key head, which read the same K and V) go to one XCD's contiguous share.  Padded sides: where a
// share is whole runs of `each` tiles, the runs' first tiles are started first and their last ones, which are ragged, at the end.
__device__ __forceinline__ long xa_item(long items, int each)
{
    const int per = (int)((items + 7) / 8), x = blockIdx.x & 7, i = blockIdx.x >> 3;
    if (each <= 1 || per % each != 0) return (long)x * per + i;
    const int runs = per / each, tile = i / runs;
    return (long)x * per + (long)(i - tile * runs) * each + tile;
}

typedef s4 __attribute__((address_space(3))) * xa_lds_s4;
__device__ __forceinline__ s4 xa_tr(const u16 *p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((xa_lds_s4)p); }

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

// Tiles of 64 rows x DP channels in LDS, filled by buffer_load ... lds: a wave's 64 16-byte pieces go to consecutive addresses, no registers
// and no LDS write instructions.  That layout cannot be padded, so the piece a slot holds is permuted by its row (the lane picks its
// source), see xa_swz.  The descriptor starts at the tile's first row and covers 2 GB; a lane has one 32-bit offset a piece.  Pieces outside
// (absent or masked rows, channels from D on) get an offset behind it, which reads zeros: one selection where 64-bit addresses took six
// operations, with holes in the mask a sixth of the row kernels' vector instructions.
typedef __attribute__((address_space(3))) void *xa_lds_p;
constexpr unsigned XA_SPAN = 0x7FFFFFFFu, XA_OUT = 0x80000000u;
constexpr long XA_NEAR = 1 << 22;  // strides below it: 128 rows, 64 tokens and their heads are less than 2 GB apart
__device__ __forceinline__ __amdgpu_buffer_rsrc_t xa_from(const u16 *p)  // p: the same in all lanes
{
    const uint64_t a = (uint64_t)p;
    const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
    return __builtin_amdgcn_make_buffer_rsrc((void *)u, 0, XA_SPAN, 0x00027000);  // raw, 32-bit data
}

// 64 banks of 4 bytes.  ds_read_b128 serves the lanes 0-3, 12-15, 20-23, 24-27 of 32 together, then the other 16: the rows of either set
// that share a place modulo 256 bytes must hold a piece in different slots.  ds_read_b64_tr_b16 serves 32 lanes together, 64 bytes of
// each of 4 neighbouring rows: those must lie in different 64-byte groups.  Both hold for these bit permutations of the row (counted:
// SQ_LDS_BANK_CONFLICT was half of the LDS cycles with a permutation made for 8 neighbouring lanes).
template <int DP>
__device__ __forceinline__ constexpr int xa_swz(int r)
{
    return DP == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (DP == 64 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : (r >> 2) & 3);
}
template <int DP>
__device__ __forceinline__ int xa_at(int row, int piece)  // value offset of a piece inside a tile
{
    return row * DP + ((piece ^ xa_swz<DP>(row)) << 3);
}

// THREADS threads (a workgroup or one wave) request ROWS rows; a thread's n-th piece stands n * NR rows below its first.
template <int DP, int ROWS, int THREADS>
struct XaStage {
    static constexpr int PIECES = DP / 8, NR = THREADS / PIECES, N = ROWS / NR;
    int r;        // tile row of the first piece
    int p;        // its channel
    int dim;
    static_assert((NR & (NR - 1)) == 0 && ROWS % NR == 0, "r < NR and NR is a power of two: the permutation's bits separate");
    __device__ __forceinline__ void init(int t, int D)
    {
        r = t / PIECES, p = 8 * ((t - r * PIECES) ^ xa_swz<DP>(r)), dim = D;
    }
    __device__ __forceinline__ int channel(int n) const { return p ^ (8 * xa_swz<DP>(n * NR)); }
    static __device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t from, unsigned at, u16 *tile, int n, int wave)
    {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (xa_lds_p)(tile + (n * THREADS + wave * 64) * 8), 16, at, 0, 0, 0);
    }
    // rows row0 .. of a matrix at row stride ls; visible: bit i <-> tile row i
    __device__ __forceinline__ void load(const u16 *base, long ls, long row0, unsigned long long visible, u16 *tile, int wave) const
    {
        const __amdgpu_buffer_rsrc_t from = xa_from(base + row0 * ls);
        const bool all = visible == (ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1);
        const unsigned long long mine = visible >> r;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = channel(n);
            unsigned at = 2u * (unsigned)((r + n * NR) * (int)ls + c);
            if (c >= dim) at = XA_OUT;
            if (!all) at = (mine >> (n * NR)) & 1 ? at : XA_OUT;
            put(from, at, tile, n, wave);
        }
    }
    // rows = token * G + g of two (token, head, channel) matrices
    __device__ __forceinline__ void load_rows(const u16 *a, long a_ls, long a_hs, u16 *ta, const u16 *b, long b_ls, long b_hs, u16 *tb, int row0, int n,
                                              const XaParams &P, int wave) const
    {
        const int tok0 = P.token(row0);
        const __amdgpu_buffer_rsrc_t af = xa_from(a + tok0 * a_ls), bf = xa_from(b + tok0 * b_ls);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = row0 + r + i * NR, tok = P.token(row), g = row - tok * P.G, c = channel(i);
            const bool ok = c < dim && row < n;
            put(af, ok ? 2u * (unsigned)((tok - tok0) * (int)a_ls + g * (int)a_hs + c) : XA_OUT, ta, i, wave);
            put(bf, ok ? 2u * (unsigned)((tok - tok0) * (int)b_ls + g * (int)b_hs + c) : XA_OUT, tb, i, wave);
        }
    }
};
// all of this wave's requests have arrived and its LDS reads are done; then the same of every wave
__device__ __forceinline__ void xa_arrived()
{
    __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0) lgkmcnt(0)
    __syncthreads();
}
// which of the 64 (or fewer) keys from key0 on are there and seen: bit i <-> key0 + i
__device__ __forceinline__ unsigned long long xa_visible(const unsigned char *mask, unsigned byte, int key0, int n, int lane)
{
    if (mask != nullptr) return __ballot(key0 + lane < n && byte == 0u);
    const int left = n - key0;
    return left >= 64 ? ~0ull : (left <= 0 ? 0ull : (1ull << left) - 1);
}
// What the scores of 32 keys start from: 0, or -inf for keys that are not to be seen (their K and V are zeros).  A matrix instruction adds to it,
// so a hole in the mask costs four LDS reads of the keys' biases instead of a test and a selection a score.
__device__ __forceinline__ float xa_bias(unsigned long long visible, int i) { return (visible >> i) & 1 ? 0.f : -INFINITY; }
__device__ __forceinline__ f16v xa_start(const float *bias, int h)
{
    f16v s;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const float4 b = *(const float4 *)(bias + 8 * g + 4 * h);
        s[4 * g] = b.x, s[4 * g + 1] = b.y, s[4 * g + 2] = b.z, s[4 * g + 3] = b.w;
    }
    return s;
}

// Transposed operand: lane <-> channel 32 * blk + lane % 32, contracted index i of half h <-> tile row row16 + 4 h + i % 4 + 8 (i / 4):
// the order in which a 32 x 32 accumulator holds 16 of its rows.
// A lane's two offsets serve every operand of every tile: the permutation is a XOR of the piece with bits of the row, so another piece is
// a XOR of the offset, and rows a multiple of 16 further are a constant.
template <int DP>
struct XaLane {
    int row, tr;
    __device__ __forceinline__ XaLane(int lane)
    {
        const int p = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
        row = xa_at<DP>(lane & 31, h), tr = xa_at<DP>(4 * h + (p >> 2), 2 * g + ((p >> 1) & 1)) + 4 * (p & 1);
    }
    // A copy whose offsets the compiler cannot trace back: it would form all 16 of them in front of a loop and, where registers are short,
    // read each back from scratch memory; formed at their use they cost one operation.
    __device__ __forceinline__ XaLane here() const
    {
        XaLane c = *this;
        asm volatile("" : "+v"(c.row), "+v"(c.tr));
        return c;
    }
    __device__ __forceinline__ bf8 rows(const u16 *tile, int row0, int t) const  // lane <-> row, channels 16 t + 8 h ..; row0: a multiple of 32
    {
        return lds_bf8(tile + row0 * DP + (row ^ (16 * t)));
    }
    __device__ __forceinline__ bf8 transposed(const u16 *tile, int row16, int blk) const  // 8 rows further the permutation's piece bit 1 flips
    {
        return cat8(xa_tr(tile + row16 * DP + (tr ^ (32 * blk))), xa_tr(tile + (row16 + 8) * DP + (tr ^ (32 * blk + 16))));
    }
};

// LDS reads and matrix instructions keep their order here (vector operations may pass).  The compiler reads an operand right in front of its
// use and waits out the whole LDS latency each time; with one or two waves a SIMD that was most of the time of a tile.
__device__ __forceinline__ void xa_keep() { __builtin_amdgcn_sched_barrier(0x406); }

// A wave among matrix instructions goes before one among exponentials: the matrix cores are fed while others calculate weights (forward pass:
// 171 and 166 us over a scene's 12000 keys, heads of 128 39 and 36 us).
#define xa_matrix(on) __builtin_amdgcn_s_setprio(on)

// acc[j] += A_j B_j over the DP channels, for N products: the operands of the next 16 channels are read before the present ones are multiplied
template <int DP, int N, class FA, class FB>
__device__ __forceinline__ void xa_products(f16v (&acc)[N], FA a, FB b)
{
    bf8 x[2][N], y[2][N];
    xa_matrix(1);
#pragma unroll
    for (int j = 0; j < N; ++j) x[0][j] = a(j, 0), y[0][j] = b(j, 0);
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        if (t + 1 < DP / 16) {
#pragma unroll
            for (int j = 0; j < N; ++j) x[(t + 1) & 1][j] = a(j, t + 1), y[(t + 1) & 1][j] = b(j, t + 1);
        }
        xa_keep();
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = PCM_MFMA16(x[t & 1][j], y[t & 1][j], acc[j]);
        xa_keep();
    }
    xa_matrix(0);
}

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
    bool ok, work;  // the lane's row is there; a row of the wave is
    XaSpan qs, ks;
    const u16 *k, *v;
    const unsigned char *mask;
    long out_row;  // (q row) * H + head
};
__device__ __forceinline__ bool xa_rows(const XaParams &P, int lane, int wave, XaRows &R)
{
    const long items = (long)P.tiles * P.Hkv * P.nsplit, item = xa_item(items, P.each);
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
    R.work = __ballot(R.ok) != 0;
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

// One 32-row column of the forward pass: reference m, sum l (of this lane's half of the keys) and O^T.
// m is a score that the row has met, at least its maximum less XA_SLACK / c: moving it with every new maximum would multiply O^T nearly each
// tile (32 rows, of which one has a new maximum more often than not) and exchange the halves' maxima; weights up to 2^8 are as good, the sums
// are fp32 and the bf16 of a weight has the same relative step everywhere.
constexpr float XA_SLACK = 8.f;
template <int DP>
struct XaSoftmax {
    f16v o[DP / 32];
    float m, l;
    __device__ __forceinline__ void init()
    {
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) o[i] = xa_zero16();
        m = -INFINITY, l = 0.f;
    }
    // NJ * 32 keys of a tile, c = scale * log2 e
    template <int NJ>
    __device__ __forceinline__ void tile(const u16 *sk, const u16 *sv, const bf8 (&qf)[DP / 16], bool all, const float *bias, float c, const XaLane<DP> &ln0, int h)
    {
        const XaLane<DP> ln = ln0.here();
        f16v s[NJ];
        const auto keys = [&](int j, int t) { return ln.rows(sk, 32 * j, t); };
        const auto rows = [&](int, int t) { return qf[t]; };
        if (all) {  // twice, so that zeros need no registers: a matrix instruction takes the constant
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[j] = xa_zero16();
            xa_products<DP>(s, keys, rows);
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) s[j] = xa_start(bias + 32 * j, h);
            xa_products<DP>(s, keys, rows);
        }
        bf8 vt[2][DP / 32];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) vt[0][i] = ln.transposed(sv, 0, i);
        xa_keep();
        float mx = m;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 2) mx = max3f(mx, s[j][r], s[j][r + 1]);
        if (__ballot((mx - m) * c > XA_SLACK) != 0) {  // the first tile; then a rare case
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float alpha = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mx) * c);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] *= alpha;
            m = mx;
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], c, -mc));
                sum += s[j][r];
            }
        l += sum;
        xa_matrix(1);
#pragma unroll
        for (int t = 0; t < 2 * NJ; ++t) {
            if (t + 1 < 2 * NJ) {
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) vt[(t + 1) & 1][i] = ln.transposed(sv, 16 * (t + 1), i);
            }
            const bf8 p = xa_pack(s[t >> 1], t & 1);
            xa_keep();
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) o[i] = PCM_MFMA16(vt[t & 1][i], p, o[i]);
            xa_keep();
        }
        xa_matrix(0);
    }
};

// the end of a row: its result, or its part of a split
template <int DP>
__device__ __forceinline__ void xa_finish(const XaParams &P, const XaRows &R, const f16v (&o)[DP / 32], float m, float l, int h)
{
    if (!R.ok) return;
    if (P.nsplit > 1) {
        const long at = (long)R.split * P.q_rows * P.H + R.out_row;
        if (h == 0) *(float2 *)(P.part_ml + 2 * at) = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) xa_store_part(P.part_o + at * P.D, P.D, h, i, o[i]);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // l >= 1 with a key (the reference score's own weight is 1, the largest at most 2^8), NaN with a NaN among the scores
    if (P.lse && h == 0) P.lse[R.out_row] = l == 0.f ? -INFINITY : m * P.scale + __logf(l);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        xa_store_row(P.out + R.out_row * P.D, P.D, h, i, o[i], inv);
        if (P.o32) xa_store_part(P.o32 + R.out_row * P.D, P.D, h, i, o[i] * inv);
    }
}

// The keys of a row kernel, 64 at a time through two LDS buffers of K and V: while tile t is worked on, tile t + 1 is on its way.  The
// buffers are variables of their own, so that the compiler can tell reads of one from requests into the other.
template <int DP, class F>
__device__ __forceinline__ void xa_key_loop(const XaRows &R, const XaParams &P, u16 *sk0, u16 *sv0, u16 *sk1, u16 *sv1, float (*bias)[XA_TILE], int lane, int wave,
                                            F body)
{
    if (R.key_lo >= R.key_hi) return;
    XaStage<DP, XA_TILE, 256> st;
    st.init((int)threadIdx.x, P.D);
    unsigned mb = xa_mask_byte(R.mask, R.key_lo + lane, R.ks.n);
    unsigned long long next = 0;
    const auto request = [&](int key0, u16 *tk, u16 *tv, float *tb) {
        next = xa_visible(R.mask, mb, key0, R.ks.n, lane);
        if (next != ~0ull && wave == 0) tb[lane] = xa_bias(next, lane);
        st.load(R.k, P.k_ls, key0, next, tk, wave), st.load(R.v, P.v_ls, key0, next, tv, wave);
        mb = xa_mask_byte(R.mask, key0 + XA_TILE + lane, R.ks.n);
    };
    const auto step = [&](int key0, int buf, const u16 *tk, const u16 *tv, u16 *nk, u16 *nv) {
        xa_arrived();
        const unsigned long long vis = next;
        if (key0 + XA_TILE < R.key_hi) request(key0 + XA_TILE, nk, nv, bias[1 - buf]);
        if (vis != 0 && R.work) body(tk, tv, vis == ~0ull, bias[buf]);
    };
    request(R.key_lo, sk0, sv0, bias[0]);
    int key0 = R.key_lo;
    for (; key0 + XA_TILE < R.key_hi; key0 += 2 * XA_TILE) {
        step(key0, 0, sk0, sv0, sk1, sv1);
        step(key0 + XA_TILE, 1, sk1, sv1, sk0, sv0);
    }
    if (key0 < R.key_hi) step(key0, 0, sk0, sv0, sk1, sv1);
}

template <int DP>
__global__ void __launch_bounds__(256, 2) pcm_xattn_fwd_kernel(XaParams P)
{
    __shared__ __attribute__((aligned(1024))) u16 sk0[XA_TILE * DP], sv0[XA_TILE * DP], sk1[XA_TILE * DP], sv1[XA_TILE * DP];
    __shared__ __attribute__((aligned(16))) float bias[2][XA_TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5;
    const XaLane<DP> ln(lane);
    XaRows R;
    if (!xa_rows(P, lane, wave, R)) return;
    bf8 qf[DP / 16];
    xa_row_operand<DP>(xa_q_row(P, P.q, P.q_bs, P.q_ls, P.q_hs, R), R.ok, P.D, h, qf);
    XaSoftmax<DP> w;
    w.init();
    const float c = P.scale * XA_LOG2E;
    xa_key_loop<DP>(R, P, sk0, sv0, sk1, sv1, bias, lane, wave,
                    [&](const u16 *tk, const u16 *tv, bool all, const float *tb) { w.template tile<2>(tk, tv, qf, all, tb, c, ln, h); });
    w.l += __shfl_xor(w.l, 32);
    xa_finish<DP>(P, R, w.o, w.m, w.l, h);
}

// Few rows (up to 32 of a key head: one token of a rollout, a group of heads that share one): all waves hold the same rows and share
// the keys, wave w every WAVES-th run of 32, each with LDS tiles and waits of its own (no barrier until the end).  K and V are read once and
// nothing else is long, so what counts is requests in flight: two tiles of K and V a wave (128 KB for 8 waves and heads of 64, for
// 4 and 128).  The waves' sums are joined through LDS.
template <int DP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) pcm_xattn_few_kernel(XaParams P)
{
    constexpr int TILE = 32 * DP, STEP = 32 * WAVES;
    __shared__ __attribute__((aligned(1024))) u16 t0[WAVES * 2 * TILE], t1[WAVES * 2 * TILE];
    __shared__ float sm[WAVES][32], sl[WAVES][32];
    __shared__ __attribute__((aligned(16))) float bias[WAVES][2][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    const XaLane<DP> ln(lane);
    XaRows R;
    if (!xa_rows(P, lane, 0, R)) return;
    bf8 qf[DP / 16];
    xa_row_operand<DP>(xa_q_row(P, P.q, P.q_bs, P.q_ls, P.q_hs, R), R.ok, P.D, h, qf);
    XaSoftmax<DP> w;
    w.init();
    const float c = P.scale * XA_LOG2E;
    XaStage<DP, 32, 64> st;
    st.init(lane, P.D);
    u16 *const k0 = t0 + wave * 2 * TILE, *const k1 = t1 + wave * 2 * TILE;
    unsigned mb = 0;
    unsigned long long vis = 0, next = 0;
    const auto request = [&](int key0, u16 *tk, float *tb) {
        next = xa_visible(R.mask, mb, key0, R.ks.n, lane) & 0xFFFFFFFFull;
        if (next != 0xFFFFFFFFull && lane < 32) tb[lane] = xa_bias(next, lane);
        st.load(R.k, P.k_ls, key0, next, tk, 0), st.load(R.v, P.v_ls, key0, next, tk + TILE, 0);
        mb = xa_mask_byte(R.mask, key0 + STEP + lane, R.ks.n);
    };
    const auto step = [&](int key0, int buf, const u16 *tk, u16 *nk) {
        __builtin_amdgcn_s_waitcnt(0x70);  // this wave's tile has arrived, its reads of the other are done
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        vis = next;
        if (key0 + STEP < R.key_hi) request(key0 + STEP, nk, bias[wave][1 - buf]);
        if (vis != 0) w.template tile<1>(tk, tk + TILE, qf, vis == 0xFFFFFFFFull, bias[wave][buf], c, ln, h);
    };
    int key0 = R.key_lo + 32 * wave;
    if (key0 < R.key_hi) {
        mb = xa_mask_byte(R.mask, key0 + lane, R.ks.n);
        request(key0, k0, bias[wave][0]);
        for (; key0 + STEP < R.key_hi; key0 += 2 * STEP) {
            step(key0, 0, k0, k1);
            step(key0 + STEP, 1, k1, k0);
        }
        if (key0 < R.key_hi) step(key0, 0, k0, k1);
    }
    w.l += __shfl_xor(w.l, 32);
    if (h == 0) sm[wave][col] = w.m, sl[wave][col] = w.l;
    __syncthreads();
    float m = sm[0][col];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) m = fmaxf(m, sm[i][col]);
    float l = 0.f, mine = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const float f = sl[i][col] == 0.f ? 0.f : __builtin_amdgcn_exp2f((sm[i][col] - m) * c);
        if (sl[i][col] != 0.f) l = __builtin_fmaf(sl[i][col], f, l);
        if (i == wave) mine = f;
    }
    // O^T of the waves, one after the other in wave order: [register][lane] in the first tiles' memory
    float *const sum = (float *)t0;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float v = mine == 0.f && w.l == 0.f ? 0.f : w.o[i][r] * mine;
            if (wave != 0) sum[((wave - 1) * (DP / 2) + 16 * i + r) * 64 + lane] = v;
            else w.o[i][r] = v;
        }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int k = 0; k < WAVES - 1; ++k) w.o[i][r] += sum[(k * (DP / 2) + 16 * i + r) * 64 + lane];
    xa_finish<DP>(P, R, w.o, m, l, h);
}

// joins the splits of a row in split order: LPR lanes per (row, head), four channels each
template <int LPR>
__global__ void __launch_bounds__(256) pcm_xattn_join_kernel(XaParams P)
{
    const long rows = P.q_rows * P.H, row = (long)blockIdx.x * (256 / LPR) + (int)threadIdx.x / LPR;
    const int d = 4 * ((int)threadIdx.x % LPR);
    if (row >= rows) return;
    const float2 *ml = (const float2 *)P.part_ml + row;
    float m = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < P.nsplit; ++s) m = fmaxf(m, ml[s * rows].x);
    const float c = P.scale * XA_LOG2E;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < P.D) {
#pragma unroll 4
        for (int s = 0; s < P.nsplit; ++s) {
            const float2 w = ml[s * rows];
            const float4 v = *(const float4 *)(P.part_o + (s * rows + row) * P.D + d);
            if (w.y != 0.f) {  // a split without a key holds no sum
                const float f = __builtin_amdgcn_exp2f((w.x - m) * c);
                l = __builtin_fmaf(w.y, f, l);
                o.x = __builtin_fmaf(v.x, f, o.x), o.y = __builtin_fmaf(v.y, f, o.y), o.z = __builtin_fmaf(v.z, f, o.z), o.w = __builtin_fmaf(v.w, f, o.w);
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (P.lse && d == 0) P.lse[row] = l == 0.f ? -INFINITY : m * P.scale + __logf(l);
        o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        *(uint2 *)(P.out + row * P.D + d) = make_uint2(cvt_pk_bf16(o.x, o.y), cvt_pk_bf16(o.z, o.w));
        if (P.o32) *(float4 *)(P.o32 + row * P.D + d) = o;
    }
}

// dQ, and delta = rowsum(dO * O) on the way (the key kernel, launched behind, reads it)
template <int DP>
__global__ void __launch_bounds__(256, 2) pcm_xattn_dq_kernel(XaParams P)
{
    __shared__ __attribute__((aligned(1024))) u16 sk0[XA_TILE * DP], sv0[XA_TILE * DP], sk1[XA_TILE * DP], sv1[XA_TILE * DP];
    __shared__ __attribute__((aligned(16))) float bias[2][XA_TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5;
    const XaLane<DP> ln0(lane);
    XaRows R;
    if (!xa_rows(P, lane, wave, R)) return;
    bf8 qf[DP / 16], gf[DP / 16];
    float delta = 0.f;
    {
        xa_row_operand<DP>(xa_q_row(P, P.dout, P.g_bs, P.g_ls, P.g_hs, R), R.ok, P.D, h, gf);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            if (!R.ok || 16 * t + 8 * h >= P.D) continue;
            const float *const row = P.o32 + R.out_row * P.D + 16 * t + 8 * h;
            const float4 a = *(const float4 *)row, b = *(const float4 *)(row + 4);
            const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(f[e], (float)gf[t][e], delta);
        }
        delta += __shfl_xor(delta, 32);
    }
    xa_row_operand<DP>(xa_q_row(P, P.q, P.q_bs, P.q_ls, P.q_hs, R), R.ok, P.D, h, qf);
    if (R.ok && h == 0 && R.split == 0) P.delta[R.out_row] = delta;
    const float lse = R.ok ? P.lse[R.out_row] : -INFINITY;
    const float l2 = lse == -INFINITY ? INFINITY : lse * XA_LOG2E;  // a row without a key: every weight 2^-inf = 0
    const float c = P.scale * XA_LOG2E;
    f16v o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = xa_zero16();
    xa_key_loop<DP>(R, P, sk0, sv0, sk1, sv1, bias, lane, wave, [&](const u16 *tk, const u16 *tv, bool all, const float *tb) {
        const XaLane<DP> ln = ln0.here();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f16v s[2] = {xa_zero16(), xa_zero16()};  // scores, dP
            const auto keys = [&](int n, int t) { return ln.rows(n ? tv : tk, 32 * j, t); };
            const auto rows = [&](int n, int t) { return n ? gf[t] : qf[t]; };
            if (all) {
                xa_products<DP>(s, keys, rows);
            } else {
                s[0] = xa_start(tb + 32 * j, h);
                xa_products<DP>(s, keys, rows);
            }
            bf8 kt[2][DP / 32];
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) kt[0][i] = ln.transposed(tk, 32 * j, i);
            xa_keep();
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], c, -l2));
                s[0][r] = p * (s[1][r] - delta);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (u == 0) {
#pragma unroll
                    for (int i = 0; i < DP / 32; ++i) kt[1][i] = ln.transposed(tk, 32 * j + 16, i);
                }
                const bf8 ds = xa_pack(s[0], u);
                xa_keep();
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) o[i] = PCM_MFMA16(kt[u][i], ds, o[i]);
                xa_keep();
            }
        }
    });
    if (!R.ok) return;
    const long at = (long)R.split * P.q_rows * P.H + R.out_row;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        if (P.nsplit > 1) xa_store_part(P.part_o + at * P.D, P.D, h, i, o[i]);
        else xa_store_row(P.dq + R.out_row * P.D, P.D, h, i, o[i], P.scale);
    }
}

// dQ of a row out of its splits, in split order: four channels a thread (D is a multiple of 8)
__global__ void __launch_bounds__(256) pcm_xattn_dq_join_kernel(XaParams P)
{
    const long quads = P.q_rows * P.H * (P.D / 4), i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < P.nsplit; ++s) {
        const float4 v = *(const float4 *)(P.part_o + 4 * (s * quads + i));
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
    *(uint2 *)(P.dq + 4 * i) = make_uint2(cvt_pk_bf16(a.x * P.scale, a.y * P.scale), cvt_pk_bf16(a.z * P.scale, a.w * P.scale));
}

// What a key kernel's workgroup works on: 128 keys of a (sequence, key head), and a share of its rows.
struct XaKeys {
    int b, kvh, split, key0, lo, nrows;  // rows lo .. nrows - 1
    XaSpan qs, ks;
    long kb, kr;  // batch and first row of the sequence in K and V
    const unsigned char *mask;
};
__device__ __forceinline__ bool xa_keys(const XaParams &P, int lane, XaKeys &K)
{
    const long items = (long)P.tiles * P.Hkv * P.nsplit, item = xa_item(items, P.each);
    if (item >= items) return false;
    int tile;
    const long rest = item / P.tiles;
    K.kvh = (int)(rest % P.Hkv), K.split = (int)(rest / P.Hkv);
    if (!xa_locate(P.kv_off, P.B, P.S, P.kv_rows, 1, XA_ROWS, (int)(item % P.tiles), lane, K.b, tile)) return false;
    K.ks = xa_span(P.kv_off, K.b, P.B, P.S, P.kv_rows);
    K.qs = K.b < P.B ? xa_span(P.q_off, K.b, P.B, P.L, P.q_rows) : XaSpan{0, 0};
    K.key0 = tile * XA_ROWS;
    const int all = K.qs.n * P.G, rt = (all + XA_TILE - 1) / XA_TILE, per = (rt + P.nsplit - 1) / P.nsplit * XA_TILE;
    K.lo = K.split * per, K.nrows = min(all, K.lo + per);
    K.kb = P.kv_off ? 0 : (long)K.b, K.kr = P.kv_off ? K.ks.row0 : 0;
    K.mask = P.mask ? P.mask + (P.kv_off ? K.ks.row0 : K.kb * P.mask_bs) : nullptr;
    if (K.mask != nullptr) {  // keys that are all masked (padding): no rows to go through
        const int k0 = K.key0 + lane, k1 = k0 + 64;
        if (__ballot((k0 < K.ks.n && K.mask[k0] == 0) || (k1 < K.ks.n && K.mask[k1] == 0)) == 0) K.nrows = K.lo;
    }
    return true;
}

// The rows of a key kernel, 64 at a time through two LDS buffers of Q and dO and of the rows' statistics.
template <int DP, int THREADS>
struct XaRowLoop {
    static constexpr int PIECES = DP / 8, ROWT = XA_TILE * PIECES < THREADS ? XA_TILE * PIECES : THREADS;  // threads that request a tile
    const XaParams &P;
    const XaKeys &K;
    const int wave;
    XaStage<DP, XA_TILE, ROWT> st;
    const u16 *qb, *gb;
    float rl, rd;
    __device__ __forceinline__ XaRowLoop(const XaParams &P_, const XaKeys &K_, int wave_) : P(P_), K(K_), wave(wave_), qb(nullptr), gb(nullptr)
    {
        st.init((int)threadIdx.x, P.D);
        if (K.lo >= K.nrows) return;
        qb = P.q + (P.q_off ? K.qs.row0 * P.q_ls : K.b * P.q_bs) + (long)K.kvh * P.G * P.q_hs;
        gb = P.dout + (P.q_off ? K.qs.row0 * P.g_ls : K.b * P.g_bs) + (long)K.kvh * P.G * P.g_hs;
    }
    __device__ __forceinline__ void request(int row0, u16 *tq, u16 *tg)
    {
        // the statistics first, untouched until they are stored: waiting for them then leaves the tiles behind them in flight
        const int row = row0 + (int)threadIdx.x, tok = P.token(row);
        rl = -INFINITY, rd = 0.f;
        if (threadIdx.x < XA_TILE && row < K.nrows) {
            const long at = (K.qs.row0 + tok) * P.H + K.kvh * P.G + (row - tok * P.G);
            rl = P.lse[at], rd = P.delta[at];
        }
        if (ROWT == THREADS || wave < ROWT / 64) st.load_rows(qb, P.q_ls, P.q_hs, tq, gb, P.g_ls, P.g_hs, tg, row0, K.nrows, P, wave);
    }
    template <class F>
    __device__ __forceinline__ void step(int row0, int buf, const u16 *tq, const u16 *tg, u16 *nq, u16 *ng, float (*sl)[XA_TILE], float (*sd)[XA_TILE], F &body)
    {
        if (threadIdx.x < XA_TILE) sl[buf][threadIdx.x] = rl == -INFINITY ? INFINITY : rl * XA_LOG2E, sd[buf][threadIdx.x] = rd;
        xa_arrived();
        if (row0 + XA_TILE < K.nrows) request(row0 + XA_TILE, nq, ng);
        body(buf, tq, tg);
    }
    template <class F>
    __device__ __forceinline__ void run(u16 *sq0, u16 *sg0, u16 *sq1, u16 *sg1, float (*sl)[XA_TILE], float (*sd)[XA_TILE], F &body)
    {
        if (K.lo >= K.nrows) return;
        request(K.lo, sq0, sg0);
        int row0 = K.lo;
        for (; row0 + XA_TILE < K.nrows; row0 += 2 * XA_TILE) {
            step(row0, 0, sq0, sg0, sq1, sg1, sl, sd, body);
            step(row0 + XA_TILE, 1, sq1, sg1, sq0, sg0, sl, sd, body);
        }
        if (row0 < K.nrows) step(row0, 0, sq0, sg0, sq1, sg1, sl, sd, body);
    }
};
// s := P, dp := dS of a 32 x 32 tile (a lane's key, 16 rows in its registers)
__device__ __forceinline__ void xa_weights(f16v &s, f16v &dp, const float *sl, const float *sd, float c, bool seen, int h)
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const float4 l2 = *(const float4 *)(sl + 8 * g + 4 * h), de = *(const float4 *)(sd + 8 * g + 4 * h);
        const float a[4] = {l2.x, l2.y, l2.z, l2.w}, e[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * g + i;
            const float p = seen ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -a[i])) : 0.f;
            dp[r] = p * (dp[r] - e[i]), s[r] = p;
        }
    }
}
// dV += dO^T P, dK += Q^T dS over 32 rows of a tile
template <int DP>
__device__ __forceinline__ void xa_key_products(f16v (&dk)[DP / 32], f16v (&dv)[DP / 32], const f16v &p, const f16v &ds, const XaLane<DP> &ln, const u16 *tq,
                                                const u16 *tg, int row0)
{
    constexpr int N = DP / 16;  // (16 rows, 32 channels) steps
    bf8 g[2], q[2];
    g[0] = ln.transposed(tg, row0, 0), q[0] = ln.transposed(tq, row0, 0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int u = n / (DP / 32), i = n % (DP / 32);
        if (n + 1 < N) {
            const int u1 = (n + 1) / (DP / 32), i1 = (n + 1) % (DP / 32);
            g[(n + 1) & 1] = ln.transposed(tg, row0 + 16 * u1, i1), q[(n + 1) & 1] = ln.transposed(tq, row0 + 16 * u1, i1);
        }
        xa_keep();
        dv[i] = PCM_MFMA16(g[n & 1], xa_pack(p, u), dv[i]);
        dk[i] = PCM_MFMA16(q[n & 1], xa_pack(ds, u), dk[i]);
        xa_keep();
    }
}
template <int DP>
__device__ __forceinline__ void xa_store_keys(const XaParams &P, const XaKeys &K, int key, int h, const f16v (&dk)[DP / 32], const f16v (&dv)[DP / 32])
{
    const long at = ((K.ks.row0 + key) * P.Hkv + K.kvh) * P.D, whole = P.kv_rows * P.Hkv * P.D;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        if (P.nsplit > 1) {
            xa_store_part(P.part_o + 2 * K.split * whole + at, P.D, h, i, dk[i]);
            xa_store_part(P.part_o + (2 * K.split + 1) * whole + at, P.D, h, i, dv[i]);
        } else {
            xa_store_row(P.dk + at, P.D, h, i, dk[i], P.scale);
            xa_store_row(P.dv + at, P.D, h, i, dv[i], 1.f);
        }
    }
}

// dK and dV of 128 keys, heads wider than 64.  8 waves: four groups of 32 keys times the two halves of every 64-row tile of Q and dO, whose sums
// are added at the end.  K and V stand in LDS beside the two buffers of Q and dO (128 KB): held in registers, as operands of 4 waves,
// they left one wave a SIMD, which waited for its own LDS reads and exponentials (515 x 4 rows over 1027 keys: 119 us, now 74).
// nsplit > 1: the rows are shared out and each share writes fp32 sums.
template <int DP>
__global__ void __launch_bounds__(512, 2) pcm_xattn_dkv_wide_kernel(XaParams P)
{
    __shared__ __attribute__((aligned(1024))) u16 sq0[XA_TILE * DP], sg0[XA_TILE * DP], sq1[XA_TILE * DP], sg1[XA_TILE * DP], sk[XA_ROWS * DP],
        sv[XA_ROWS * DP];
    __shared__ __attribute__((aligned(16))) float sl[2][XA_TILE], sd[2][XA_TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    const XaLane<DP> ln0(lane);
    const int kg = wave & 3, half = wave >> 2;
    XaKeys K;
    if (!xa_keys(P, lane, K)) return;
    const int key = K.key0 + kg * 32 + col;
    const bool held = key < K.ks.n, seen = held && (K.mask == nullptr || K.mask[key] == 0);
    const float c = P.scale * XA_LOG2E;
    f16v dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = xa_zero16(), dv[i] = xa_zero16();
    if (K.lo < K.nrows) {  // K and V, zeros for keys that are not there or not seen
        XaStage<DP, XA_ROWS, 512> kt;
        kt.init((int)threadIdx.x, P.D);
        const __amdgpu_buffer_rsrc_t kf = xa_from(P.k + K.kb * P.k_bs + (K.kr + K.key0) * P.k_ls + (long)K.kvh * P.k_hs),
                                     vf = xa_from(P.v + K.kb * P.v_bs + (K.kr + K.key0) * P.v_ls + (long)K.kvh * P.v_hs);
#pragma unroll
        for (int n = 0; n < kt.N; ++n) {
            const int i = kt.r + n * kt.NR, j = K.key0 + i, c = kt.channel(n);
            const bool ok = c < P.D && j < K.ks.n && (K.mask == nullptr || K.mask[j] == 0);
            kt.put(kf, ok ? 2u * (unsigned)(i * (int)P.k_ls + c) : XA_OUT, sk, n, wave), kt.put(vf, ok ? 2u * (unsigned)(i * (int)P.v_ls + c) : XA_OUT, sv, n, wave);
        }
    }
    XaRowLoop<DP, 512> rows(P, K, wave);
    const bool work = __ballot(seen) != 0;  // a wave whose keys are absent or masked only takes part in the loading
    const auto body = [&](int buf, const u16 *tq, const u16 *tg) {
        if (!work) return;
        const XaLane<DP> ln = ln0.here();
        f16v s[2] = {xa_zero16(), xa_zero16()};  // scores, dP
        xa_products<DP>(s, [&](int n, int t) { return ln.rows(n ? tg : tq, 32 * half, t); }, [&](int n, int t) { return ln.rows(n ? sv : sk, 32 * kg, t); });
        xa_weights(s[0], s[1], sl[buf] + 32 * half, sd[buf] + 32 * half, c, seen, h);
        xa_key_products<DP>(dk, dv, s[0], s[1], ln, tq, tg, 32 * half);
    };
    rows.run(sq0, sg0, sq1, sg1, sl, sd, body);
    // the two halves: [register][lane], dK and then dV, 128 * DP values in the place of K and V
    float *const sum = (float *)(kg < 2 ? sk : sv) + (kg & 1) * 32 * DP;
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        if (half == 1) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[(16 * i + r) * 64 + lane] = part ? dv[i][r] : dk[i][r];
        }
        __syncthreads();
        if (half == 0) {
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float v = sum[(16 * i + r) * 64 + lane];
                    if (part) dv[i][r] += v;
                    else dk[i][r] += v;
                }
        }
        __syncthreads();
    }
    if (half == 0 && held) xa_store_keys<DP>(P, K, key, h, dk, dv);
}

// The same for heads of up to 64: 4 waves, K and V of a wave's 32 keys in registers, both halves of a row tile one after the other.
template <int DP>
__global__ void __launch_bounds__(256, 2) pcm_xattn_dkv_narrow_kernel(XaParams P)
{
    __shared__ __attribute__((aligned(1024))) u16 sq0[XA_TILE * DP], sg0[XA_TILE * DP], sq1[XA_TILE * DP], sg1[XA_TILE * DP];
    __shared__ __attribute__((aligned(16))) float sl[2][XA_TILE], sd[2][XA_TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    const XaLane<DP> ln0(lane);
    XaKeys K;
    if (!xa_keys(P, lane, K)) return;
    const int key = K.key0 + wave * 32 + col;
    const bool held = key < K.ks.n, seen = held && (K.mask == nullptr || K.mask[key] == 0);
    const long at_k = K.kb * P.k_bs + (K.kr + key) * P.k_ls + (long)K.kvh * P.k_hs, at_v = K.kb * P.v_bs + (K.kr + key) * P.v_ls + (long)K.kvh * P.v_hs;
    bf8 kf[DP / 16], vf[DP / 16];
    xa_row_operand<DP>(P.k + (seen ? at_k : 0), seen, P.D, h, kf);
    xa_row_operand<DP>(P.v + (seen ? at_v : 0), seen, P.D, h, vf);
    const float c = P.scale * XA_LOG2E;
    f16v dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = xa_zero16(), dv[i] = xa_zero16();
    XaRowLoop<DP, 256> rows(P, K, wave);
    const bool work = __ballot(seen) != 0;
    const auto body = [&](int buf, const u16 *tq, const u16 *tg) {
        if (!work) return;
        const XaLane<DP> ln = ln0.here();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f16v s[2] = {xa_zero16(), xa_zero16()};
            xa_products<DP>(s, [&](int n, int t) { return ln.rows(n ? tg : tq, 32 * j, t); }, [&](int n, int t) { return n ? vf[t] : kf[t]; });
            xa_weights(s[0], s[1], sl[buf] + 32 * j, sd[buf] + 32 * j, c, seen, h);
            xa_key_products<DP>(dk, dv, s[0], s[1], ln, tq, tg, 32 * j);
        }
    };
    rows.run(sq0, sg0, sq1, sg1, sl, sd, body);
    if (held) xa_store_keys<DP>(P, K, key, h, dk, dv);
}

// dK and dV out of the shares of their rows, in order: four channels a thread, dK then dV
__global__ void __launch_bounds__(256) pcm_xattn_dkv_join_kernel(XaParams P)
{
    const long quads = P.kv_rows * P.Hkv * (P.D / 4);
    long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * quads) return;
    const int part = i >= quads;
    i -= part * quads;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < P.nsplit; ++s) {
        const float4 v = *(const float4 *)(P.part_o + 4 * ((2 * s + part) * quads + i));
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
    const float f = part ? 1.f : P.scale;
    *(uint2 *)((part ? P.dv : P.dk) + 4 * i) = make_uint2(cvt_pk_bf16(a.x * f, a.y * f), cvt_pk_bf16(a.z * f, a.w * f));
}

#define XA_BY_DIM(kernel, threads, grid, s, P)                                                              \
    do {                                                                                                    \
        if ((P).D <= 32) hipLaunchKernelGGL((kernel<32>), dim3(grid), dim3(threads), 0, s, P);              \
        else if ((P).D <= 64) hipLaunchKernelGGL((kernel<64>), dim3(grid), dim3(threads), 0, s, P);         \
        else hipLaunchKernelGGL((kernel<128>), dim3(grid), dim3(threads), 0, s, P);                         \
    } while (0)

bool xa_shape_ok(int H, int Hkv, int D) { return H > 0 && Hkv > 0 && H % Hkv == 0 && D >= 8 && D <= 128 && D % 8 == 0; }

// an upper bound on the tiles of a side: a packed side's sequences end inside a tile each
long xa_tiles(int packed, int B, int len, long rows, int mult, int per)
{
    return packed ? (rows * mult + per - 1) / per + B + 1 : (long)B * (((long)len * mult + per - 1) / per);
}

// The forward pass of few rows (see pcm_xattn_few_kernel): every (sequence, key head) has 32 rows at most.  A packed side's longest
// sequence is not known here: only its total counts.
bool xa_few(int L, long q_rows, int q_packed, int G) { return (q_packed ? q_rows : (long)L) * G <= 32; }

// Splits of the keys.  A workgroup per (tile, key head) is too few for 256 compute units when the rows are few (a decoder's 100 queries): the
// keys are then shared out until about 512 workgroups run, two a compute unit.  A split writes and re-reads its row's fp32 sums and costs a
// second launch (4 - 7 us), so it has 256 keys at least.  The kernel of few rows shares the keys among its own waves (8, or 4 for heads wider
// than 64), so a split of its has 2048 keys (1024) at least, 256 a wave: one split up to 4095 keys, two up to 6143 and so on.  Measured at one
// row over 2051 keys, 8 heads of 64: 13.4 us without a split, 10.4 + 4.8 with 7.  What counts is a wave's chain of tiles, so a call takes 16.2 us
// over 2051 keys, 19.6 over 4095 and, with two splits, 16.2 over 4096 and 20.6 over 6143.  Long states are shared out further, to three
// workgroups a compute unit and two rounds of them: a third wave hides the others' waits, and ragged sequences even out (4500 rows over 12000
// keys on average, 8 heads of 64: 230 us with one split, 173 + 7 for the joining with two, 167 + 10 with four).
int xa_splits(int B, int H, int Hkv, int D, int L, long q_rows, int q_packed, int S, long kv_rows, int kv_packed, bool backward)
{
    const int G = H / Hkv;
    const bool few = !backward && xa_few(L, q_rows, q_packed, G);
    const long work = (q_packed ? (q_rows * G + XA_ROWS - 1) / XA_ROWS + B - 1 : xa_tiles(0, B, L, q_rows, G, XA_ROWS)) * Hkv;
    const long keys = kv_packed ? (kv_rows + B - 1) / B : S, w = work > 0 ? work : 1;
    const long least = few ? (D <= 64 ? 2048 : 1024) : 256;
    long n = 512 / w < keys / least ? 512 / w : keys / least;
    const long more = 1536 / w < keys / 2048 ? 1536 / w : keys / 2048;
    n = n > more ? n : more;
    return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
}
int xa_splits(const XaParams &P, bool backward)
{
    return xa_splits(P.B, P.H, P.Hkv, P.D, P.L, P.q_rows, P.q_off != nullptr, P.S, P.kv_rows, P.kv_off != nullptr, backward);
}

// Splits of the rows for dK and dV, where few keys leave compute units idle: at least 512 rows (8 tiles) each.
int xa_row_splits(int B, int Hkv, int G, long q_rows, int S, long kv_rows, int kv_packed)
{
    const long work = (kv_packed ? (kv_rows + XA_ROWS - 1) / XA_ROWS + B - 1 : xa_tiles(0, B, S, kv_rows, 1, XA_ROWS)) * Hkv;
    const long rows = q_rows * G / B, w = work > 0 ? work : 1;
    const long n = 256 / w < rows / 512 ? 256 / w : rows / 512;
    return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
}
int xa_row_splits(const XaParams &P) { return xa_row_splits(P.B, P.Hkv, P.G, P.q_rows, P.S, P.kv_rows, P.kv_off != nullptr); }

// heads: those of a key head where a tile holds several (queries)
bool xa_strides_ok(const void *p, long bs, long ls, long hs, long heads)
{
    return (((uintptr_t)p) & 15) == 0 && ((bs | ls | hs) & 7) == 0 && ls >= 0 && hs >= 0 && ls < XA_NEAR && hs * (heads - 1) < 1L << 29;
}

int xa_fill(XaParams &P, int B, int H, int Hkv, int D, int L, long q_rows, const int *q_offset, int S, long kv_rows, const int *kv_offset,
            const void *q, long q_bs, long q_ls, long q_hs, const void *k, long k_bs, long k_ls, long k_hs, const void *v, long v_bs, long v_ls,
            long v_hs, const unsigned char *mask, long mask_bs, float scale)
{
    P = XaParams{};
    if (!xa_shape_ok(H, Hkv, D)) return PCM_ERR_UNSUPPORTED;
    if (!(scale > 0.f) || scale > 3.0e38f) return PCM_ERR_BAD_ARG;
    if (!q_offset) q_rows = (long)B * L;
    if (!kv_offset) kv_rows = (long)B * S;
    // rows and keys are 32-bit numbers inside a sequence, with room for the steps that pass its end; a launch has fewer than 2^32 threads
    // (splits only multiply launches of a few hundred workgroups)
    if (q_rows > 0x7FFFFC00L / H || kv_rows > 0x7FFFFC00L) return PCM_ERR_UNSUPPORTED;
    if (xa_tiles(q_offset != nullptr, B, L, q_rows, H / Hkv, XA_ROWS) > 0xFFFFF000L / 256 / Hkv ||
        xa_tiles(kv_offset != nullptr, B, S, kv_rows, 1, XA_ROWS) > 0xFFFFF000L / 512 / Hkv)
        return PCM_ERR_UNSUPPORTED;
    if ((q_rows > 0 && !q) || (kv_rows > 0 && (!k || !v))) return PCM_ERR_BAD_ARG;
    if (!xa_strides_ok(q, q_bs, q_ls, q_hs, H / Hkv) || !xa_strides_ok(k, k_bs, k_ls, k_hs, 1) || !xa_strides_ok(v, v_bs, v_ls, v_hs, 1)) return PCM_ERR_UNSUPPORTED;
    P.q = (const u16 *)q, P.k = (const u16 *)k, P.v = (const u16 *)v;
    P.q_bs = q_bs, P.q_ls = q_ls, P.q_hs = q_hs, P.k_bs = k_bs, P.k_ls = k_ls, P.k_hs = k_hs, P.v_bs = v_bs, P.v_ls = v_ls, P.v_hs = v_hs;
    P.mask = mask, P.mask_bs = mask_bs, P.q_off = q_offset, P.kv_off = kv_offset;
    P.B = B, P.H = H, P.Hkv = Hkv, P.G = H / Hkv, P.D = D, P.L = L, P.S = S, P.q_rows = q_rows, P.kv_rows = kv_rows, P.scale = scale;
    P.g_shift = 31;
    while ((1L << (P.g_shift - 31)) < P.G) ++P.g_shift;
    P.g_inv = (uint32_t)(((1ull << P.g_shift) + P.G - 1) / P.G);
    return PCM_OK;
}

unsigned xa_grid(long items) { return (unsigned)((items + 7) / 8 * 8); }

}  // namespace

extern "C" int pcm_cross_attn_supported(int H, int Hkv, int D) { return xa_shape_ok(H, Hkv, D) ? 1 : 0; }

extern "C" long pcm_cross_attn_ws_bytes(int B, int H, int Hkv, int D, int L, long q_rows, int q_packed, int S, long kv_rows, int kv_packed,
                                        int backward)
{
    if (B <= 0 || L < 0 || S < 0 || q_rows < 0 || kv_rows < 0 || !xa_shape_ok(H, Hkv, D)) return 0;
    if (!q_packed) q_rows = (long)B * L;
    if (!kv_packed) kv_rows = (long)B * S;
    const int n = xa_splits(B, H, Hkv, D, L, q_rows, q_packed, S, kv_rows, kv_packed, backward != 0);
    const int m = backward ? xa_row_splits(B, Hkv, H / Hkv, q_rows, S, kv_rows, kv_packed) : 1;
    const long rows = n > 1 ? (long)n * q_rows * H * (D + 2) * 4 : 0, keys = m > 1 ? (long)m * 2 * kv_rows * Hkv * D * 4 : 0;
    return rows > keys ? rows : keys;
}

extern "C" int pcm_cross_attn_forward_hip(int B, int H, int Hkv, int D, int L, long q_rows, const int *q_offset, int S, long kv_rows,
                                          const int *kv_offset, const void *q, long q_bs, long q_ls, long q_hs, const void *k, long k_bs,
                                          long k_ls, long k_hs, const void *v, long v_bs, long v_ls, long v_hs, const unsigned char *mask,
                                          long mask_bs, float scale, void *out, float *out32, float *lse, void *ws, long ws_bytes, void *stream)
{
    if (B < 0 || H < 0 || Hkv < 0 || D < 0 || L < 0 || S < 0 || q_rows < 0 || kv_rows < 0) return PCM_ERR_BAD_ARG;
    if (B == 0 || (q_offset ? q_rows == 0 : L == 0)) return PCM_OK;
    XaParams P;
    const int bad = xa_fill(P, B, H, Hkv, D, L, q_rows, q_offset, S, kv_rows, kv_offset, q, q_bs, q_ls, q_hs, k, k_bs, k_ls, k_hs, v, v_bs, v_ls, v_hs,
                            mask, mask_bs, scale);
    if (bad) return bad;
    if (!out || (((uintptr_t)out | (uintptr_t)out32 | (uintptr_t)ws) & 15) != 0) return PCM_ERR_BAD_ARG;
    P.out = (u16 *)out, P.o32 = out32, P.lse = lse;
    P.nsplit = xa_splits(P, false);
    if (P.nsplit > 1) {
        if (!ws || ws_bytes < (long)P.nsplit * P.q_rows * H * (D + 2) * 4) return PCM_ERR_BAD_ARG;
        P.part_o = (float *)ws, P.part_ml = (float *)ws + (long)P.nsplit * P.q_rows * H * D;
    }
    P.tiles = (int)xa_tiles(q_offset != nullptr, B, L, P.q_rows, P.G, XA_ROWS), P.each = q_offset ? 1 : P.tiles / B;
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid(xa_grid((long)P.tiles * Hkv * P.nsplit));
    // xa_fill's limit on the tiles is that of workgroups of 256 threads: more than half as many stay with those
    const bool few = xa_few(L, P.q_rows, q_offset != nullptr, P.G) && (D > 64 || grid.x < 0xFFFFF000u / 512);
    if (few && D <= 32) hipLaunchKernelGGL((pcm_xattn_few_kernel<32, 8>), grid, dim3(512), 0, s, P);
    else if (few && D <= 64) hipLaunchKernelGGL((pcm_xattn_few_kernel<64, 8>), grid, dim3(512), 0, s, P);
    else if (few) hipLaunchKernelGGL((pcm_xattn_few_kernel<128, 4>), grid, dim3(256), 0, s, P);
    else XA_BY_DIM(pcm_xattn_fwd_kernel, 256, xa_grid((long)P.tiles * Hkv * P.nsplit), s, P);
    if (P.nsplit > 1) {
        const long rows = P.q_rows * H;
        if (D <= 32) hipLaunchKernelGGL((pcm_xattn_join_kernel<8>), dim3((unsigned)((rows + 31) / 32)), dim3(256), 0, s, P);
        else if (D <= 64) hipLaunchKernelGGL((pcm_xattn_join_kernel<16>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, s, P);
        else hipLaunchKernelGGL((pcm_xattn_join_kernel<32>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, P);
    }
    return PCM_LAUNCH_STATUS();
}

extern "C" int pcm_cross_attn_backward_hip(int B, int H, int Hkv, int D, int L, long q_rows, const int *q_offset, int S, long kv_rows,
                                           const int *kv_offset, const void *q, long q_bs, long q_ls, long q_hs, const void *k, long k_bs,
                                           long k_ls, long k_hs, const void *v, long v_bs, long v_ls, long v_hs, const unsigned char *mask,
                                           long mask_bs, float scale, const float *out32, const float *lse, const void *dout, long g_bs, long g_ls,
                                           long g_hs, float *delta, void *dq, void *dk, void *dv, void *ws, long ws_bytes, void *stream)
{
    if (B < 0 || H < 0 || Hkv < 0 || D < 0 || L < 0 || S < 0 || q_rows < 0 || kv_rows < 0) return PCM_ERR_BAD_ARG;
    if (B == 0) return PCM_OK;
    XaParams P;
    const int bad = xa_fill(P, B, H, Hkv, D, L, q_rows, q_offset, S, kv_rows, kv_offset, q, q_bs, q_ls, q_hs, k, k_bs, k_ls, k_hs, v, v_bs, v_ls, v_hs,
                            mask, mask_bs, scale);
    if (bad) return bad;
    if (P.q_rows > 0 && (!out32 || !lse || !dout || !delta || !dq)) return PCM_ERR_BAD_ARG;
    if (!dk != !dv) return PCM_ERR_BAD_ARG;  // neither: states that need no gradient
    if (!xa_strides_ok(dout, g_bs, g_ls, g_hs, H / Hkv)) return PCM_ERR_UNSUPPORTED;
    if ((((uintptr_t)out32 | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15) != 0) return PCM_ERR_BAD_ARG;
    P.o32 = (float *)out32, P.lse = (float *)lse, P.dout = (const u16 *)dout, P.g_bs = g_bs, P.g_ls = g_ls, P.g_hs = g_hs;
    P.delta = delta, P.dq = (u16 *)dq, P.dk = (u16 *)dk, P.dv = (u16 *)dv;
    const hipStream_t s = (hipStream_t)stream;
    if (P.q_rows > 0) {
        P.nsplit = xa_splits(P, true);
        if (P.nsplit > 1) {
            if (!ws || ws_bytes < (long)P.nsplit * P.q_rows * H * D * 4) return PCM_ERR_BAD_ARG;
            P.part_o = (float *)ws;
        }
        P.tiles = (int)xa_tiles(q_offset != nullptr, B, L, P.q_rows, P.G, XA_ROWS), P.each = q_offset ? 1 : P.tiles / B;
        XA_BY_DIM(pcm_xattn_dq_kernel, 256, xa_grid((long)P.tiles * Hkv * P.nsplit), s, P);
        if (P.nsplit > 1) hipLaunchKernelGGL(pcm_xattn_dq_join_kernel, dim3((unsigned)((P.q_rows * H * (D / 4) + 255) / 256)), dim3(256), 0, s, P);
    }
    if (P.kv_rows > 0 && dk) {
        P.tiles = (int)xa_tiles(kv_offset != nullptr, B, S, P.kv_rows, 1, XA_ROWS), P.each = kv_offset ? 1 : P.tiles / B;
        P.nsplit = xa_row_splits(P);
        if (P.nsplit > 1) {
            if (!ws || ws_bytes < (long)P.nsplit * 2 * P.kv_rows * Hkv * D * 4) return PCM_ERR_BAD_ARG;
            P.part_o = (float *)ws;
        }
        const dim3 grid(xa_grid((long)P.tiles * Hkv * P.nsplit));
        if (D <= 32) hipLaunchKernelGGL((pcm_xattn_dkv_narrow_kernel<32>), grid, dim3(256), 0, s, P);
        else if (D <= 64) hipLaunchKernelGGL((pcm_xattn_dkv_narrow_kernel<64>), grid, dim3(256), 0, s, P);
        else hipLaunchKernelGGL((pcm_xattn_dkv_wide_kernel<128>), grid, dim3(512), 0, s, P);
        if (P.nsplit > 1) hipLaunchKernelGGL(pcm_xattn_dkv_join_kernel, dim3((unsigned)((P.kv_rows * Hkv * (D / 2) + 255) / 256)), dim3(256), 0, s, P);
    }
    return PCM_LAUNCH_STATUS();
}

// rotary.hip -- rotary positions over several axes (x, y, z of a point token; time, height, width of a frame).
//
// Pair j (of n_a) of axis a turns by  theta = coord_a * base^(-j / n_a):
//     (u, v) -> (u cos theta - v sin theta, u sin theta + v cos theta),
// with the pairs of all axes side by side: pair i holds the channels (i, i + half), or (2 i, 2 i + 1) when interleaved; channels from
// 2 * half on pass through.  The transpose of a turn is the turn by -theta: the backward pass is the same kernel with `inverse`.
//
// Angles.  In fp32, coord * frequency at a coordinate of 2^20 is off by 2^-4 radians.  The product is therefore formed in fp64 and in
// REVOLUTIONS (the host divides the frequencies by 2 pi): the quarter turn k and the remainder |r| <= 1/8 revolution come out of one
// fp64 subtraction, and only the remainder (times 2 pi, |x| <= pi / 4) is rounded to fp32, for two short Taylor sums (truncation
// 2e-9 relative: x^11 / 11! and x^12 / 12! at pi / 4).
//
// Bound by memory: 3 operations a value.  The angle does not depend on the head, so a workgroup first puts (cos, sin) of its tokens
// into LDS (one fp64 product and ~25 operations per token and pair, once) and then streams its tokens' heads in memory order.
#include "pcm_elem.hpp"

namespace {

constexpr int ROT_MAX_HALF = 128, ROT_MAX_AXES = 8, ROT_THREADS = 256, ROT_TABLE = 2048, ROT_TOKENS = 256;

struct RotArgs {
    const void *x;
    void *out;
    const void *coords;
    long L, rows;
    long x_bs, x_ls, x_hs, o_bs, o_ls, o_hs, c_bs, c_ls;
    int H, D, half, coords_type, tokens;
    float sign;
    double rev[ROT_MAX_HALF];          // revolutions per unit of the pair's coordinate
    unsigned char axis[ROT_MAX_HALF];  // the pair's axis
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

template <int N>
__device__ __forceinline__ Pack<float, N> from_f(const float (&v)[N], float)
{
    Pack<float, N> p;
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = v[i];
    return p;
}
template <int N>
__device__ __forceinline__ Pack<uint16_t, N> from_f(const float (&v)[N], uint16_t)
{
    Pack<uint16_t, N> p;  // round to nearest even, once
    if constexpr (N == 1) {
        p.v[0] = (uint16_t)pcm_cvt_pk_bf16(v[0], 0.f);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint32_t w = pcm_cvt_pk_bf16(v[i], v[i + 1]);
            p.v[i] = (uint16_t)w, p.v[i + 1] = (uint16_t)(w >> 16);
        }
    }
    return p;
}

__device__ __forceinline__ float2 rot_cos_sin(double coord, double rev, float sign)
{
    const double t = coord * rev;  // revolutions
    const double q = rint(4.0 * t);
    const float x = (float)((t - 0.25 * q) * 6.283185307179586476925);
    const float k = (float)(q - 4.0 * floor(0.25 * q));  // quarter turns 0 .. 3 (a NaN coordinate stays one in x)
    const float y = x * x;
    float s = 2.7557319e-6f, c = -2.7557319e-7f;
    s = __builtin_fmaf(s, y, -1.9841270e-4f), c = __builtin_fmaf(c, y, 2.4801587e-5f);
    s = __builtin_fmaf(s, y, 8.3333333e-3f), c = __builtin_fmaf(c, y, -1.3888889e-3f);
    s = __builtin_fmaf(s, y, -1.6666667e-1f), c = __builtin_fmaf(c, y, 4.1666667e-2f);
    s = __builtin_fmaf(s * y, x, x), c = __builtin_fmaf(c, y, -0.5f);
    c = __builtin_fmaf(c, y, 1.f);
    const bool odd = k == 1.f || k == 3.f;
    const float cc = odd ? s : c, ss = odd ? c : s;
    return make_float2((k == 1.f || k == 2.f) ? -cc : cc, sign * (k >= 2.f ? -ss : ss));
}

// One item of the stream: V channels of each half of V pairs; V neighbouring channels, V / 2 pairs, when interleaved (one pair of single
// channels for V = 1); or V channels behind the pairs.
template <typename T, int V, bool INTER>
struct RotItem {
    typedef Pack<T, V> Vec;
    static constexpr bool TWO = !INTER || V == 1;   // two accesses
    static constexpr int PAIRS = TWO ? V : V / 2;
    Vec a, e;
    T *o0, *o1;
    const float2 *cs;  // nullptr: channels that pass through
    __device__ __forceinline__ void load(const RotArgs &P, const long *xo, const long *oo, const float2 *table, int t, int h, int c, int turned)
    {
        const T *x = (const T *)P.x + xo[t] + h * P.x_hs;
        T *o = (T *)P.out + oo[t] + h * P.o_hs;
        if (c >= turned) {
            const int d = 2 * P.half + (c - turned) * V;
            a = *(const Vec *)(x + d), o0 = o + d, cs = nullptr;
            return;
        }
        const int d0 = INTER ? 2 * c * PAIRS : c * V, d1 = INTER ? d0 + 1 : P.half + c * V;
        a = *(const Vec *)(x + d0), o0 = o + d0, cs = table + t * P.half + c * PAIRS;
        if constexpr (TWO) e = *(const Vec *)(x + d1), o1 = o + d1;
    }
    __device__ __forceinline__ void finish() const
    {
        if (cs == nullptr) {
            *(Vec *)o0 = a;
            return;
        }
        float u[V], v[V];
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const float2 w = cs[j];
            if constexpr (TWO) {
                const float p = to_f(a.v[j]), q = to_f(e.v[j]);
                u[j] = __builtin_fmaf(p, w.x, -(q * w.y)), v[j] = __builtin_fmaf(p, w.y, q * w.x);
            } else {
                const float p = to_f(a.v[2 * j]), q = to_f(a.v[2 * j + 1]);
                u[2 * j] = __builtin_fmaf(p, w.x, -(q * w.y)), u[2 * j + 1] = __builtin_fmaf(p, w.y, q * w.x);
            }
        }
        *(Vec *)o0 = from_f<V>(u, T());
        if constexpr (TWO) *(Vec *)o1 = from_f<V>(v, T());
    }
};

// T: uint16_t (bf16 bits) or float.  V: channels a thread takes from each half of the pairs, one aligned access of V values.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(ROT_THREADS) pcm_rotary_kernel(RotArgs P)
{
    __shared__ float2 table[ROT_TABLE];  // [token][half]
    __shared__ long xo[ROT_TOKENS], oo[ROT_TOKENS];
    const long t0 = (long)blockIdx.x * P.tokens;
    const int nt = (int)(P.rows - t0 < P.tokens ? P.rows - t0 : P.tokens);
    for (int t = threadIdx.x; t < nt; t += ROT_THREADS) {
        const long b = (t0 + t) / P.L, l = t0 + t - b * P.L;
        xo[t] = b * P.x_bs + l * P.x_ls, oo[t] = b * P.o_bs + l * P.o_ls;
    }
    for (int i = threadIdx.x; i < nt * P.half; i += ROT_THREADS) {
        const int t = i / P.half, j = i - t * P.half;
        const long tok = t0 + t, b = tok / P.L;
        const long at = b * P.c_bs + (tok - b * P.L) * P.c_ls + P.axis[j];
        const double c = P.coords_type == 0 ? (double)((const float *)P.coords)[at]
                         : P.coords_type == 1 ? (double)((const int *)P.coords)[at]
                                              : (double)((const long *)P.coords)[at];
        table[i] = rot_cos_sin(c, P.rev[j], P.sign);
    }
    __syncthreads();
    // items in memory order, (token, head, chunk) carried along instead of divided out; the loads of U items in flight
    const int turned = P.half / RotItem<T, V, INTER>::PAIRS, chunks = turned + (P.D - 2 * P.half) / V, per_token = P.H * chunks, all = nt * per_token;
    const int dt = ROT_THREADS / per_token, rest = ROT_THREADS - dt * per_token, dh = rest / chunks, dc = rest - dh * chunks;
    int t = (int)threadIdx.x / per_token, h = ((int)threadIdx.x - t * per_token) / chunks, c = (int)threadIdx.x - t * per_token - h * chunks;
    const auto next = [&]() {
        c += dc;
        if (c >= chunks) c -= chunks, ++h;
        h += dh;
        if (h >= P.H) h -= P.H, ++t;
        t += dt;
    };
    constexpr int U = RotItem<T, V, INTER>::TWO ? 1 : 4;
    RotItem<T, V, INTER> x[U];
    int i = threadIdx.x;
    for (; i + (U - 1) * ROT_THREADS < all; i += U * ROT_THREADS) {
#pragma unroll
        for (int n = 0; n < U; ++n) {
            x[n].load(P, xo, oo, table, t, h, c, turned);
            next();
        }
#pragma unroll
        for (int n = 0; n < U; ++n) x[n].finish();
    }
    for (; i < all; i += ROT_THREADS) {
        x[0].load(P, xo, oo, table, t, h, c, turned);
        next();
        x[0].finish();
    }
}

template <typename T, int V>
void rot_launch(const RotArgs &P, int interleaved, hipStream_t s)
{
    const dim3 grid((unsigned)((P.rows + P.tokens - 1) / P.tokens));
    if (interleaved) hipLaunchKernelGGL((pcm_rotary_kernel<T, V, true>), grid, dim3(ROT_THREADS), 0, s, P);
    else hipLaunchKernelGGL((pcm_rotary_kernel<T, V, false>), grid, dim3(ROT_THREADS), 0, s, P);
}

}  // namespace

extern "C" int pcm_rotary_axes_hip(long B, long L, int H, int D, int x_is_bf16, const void *x, long x_bs, long x_ls, long x_hs, void *out,
                                   long o_bs, long o_ls, long o_hs, int coords_type, const void *coords, long c_bs, long c_ls, int axes,
                                   const int *sections, double base, int interleaved, int inverse, void *stream)
{
    if (B < 0 || L < 0 || H < 0 || D < 0 || axes < 0) return PCM_ERR_BAD_ARG;
    if (B == 0 || L == 0 || H == 0 || D == 0) return PCM_OK;
    if (!x || !out || !coords || !sections || axes < 1 || axes > ROT_MAX_AXES || coords_type < 0 || coords_type > 2) return PCM_ERR_BAD_ARG;
    if (!(base > 0.0)) return PCM_ERR_BAD_ARG;
    if (L > (1L << 40) / B || (long)H * D > (1L << 22)) return PCM_ERR_UNSUPPORTED;  // a workgroup's items are a 32-bit number
    RotArgs P;
    P.half = 0;
    for (int a = 0; a < axes; ++a) {
        if (sections[a] < 0 || sections[a] > ROT_MAX_HALF - P.half) return PCM_ERR_UNSUPPORTED;
        for (int j = 0; j < sections[a]; ++j) {
            P.rev[P.half + j] = pow(base, -(double)j / (double)sections[a]) / 6.283185307179586476925;
            P.axis[P.half + j] = (unsigned char)a;
        }
        P.half += sections[a];
    }
    if (P.half < 1 || 2 * P.half > D) return PCM_ERR_BAD_ARG;
    P.x = x, P.out = out, P.coords = coords, P.L = L, P.rows = B * L;
    P.x_bs = x_bs, P.x_ls = x_ls, P.x_hs = x_hs, P.o_bs = o_bs, P.o_ls = o_ls, P.o_hs = o_hs, P.c_bs = c_bs, P.c_ls = c_ls;
    P.H = H, P.D = D, P.coords_type = coords_type, P.sign = inverse ? -1.f : 1.f;
    // tokens of a workgroup: as many as the table holds (a long stream per workgroup), fewer while that leaves compute units idle
    P.tokens = ROT_TABLE / P.half < ROT_TOKENS ? ROT_TABLE / P.half : ROT_TOKENS;
    while (P.tokens > 1 && P.rows / P.tokens < 1024) P.tokens = (P.tokens + 1) / 2;
    if ((P.rows + P.tokens - 1) / P.tokens > 0xFFFFFFL) return PCM_ERR_UNSUPPORTED;  // fewer than 2^32 threads
    // the widest access that every channel offset and address is aligned to (16 bytes when strides and sections allow)
    const int size = x_is_bf16 ? 2 : 4;
    int V = 16 / size;
    const long all = x_bs | x_ls | x_hs | o_bs | o_ls | o_hs | P.half | D;
    while (V > 1 && (all % V != 0 || ((uintptr_t)x | (uintptr_t)out) % (uintptr_t)(V * size) != 0)) V /= 2;
    const hipStream_t s = (hipStream_t)stream;
    if (x_is_bf16) {
        if (V == 8) rot_launch<uint16_t, 8>(P, interleaved, s);
        else if (V == 4) rot_launch<uint16_t, 4>(P, interleaved, s);
        else if (V == 2) rot_launch<uint16_t, 2>(P, interleaved, s);
        else rot_launch<uint16_t, 1>(P, interleaved, s);
    } else {
        if (V == 4) rot_launch<float, 4>(P, interleaved, s);
        else if (V == 2) rot_launch<float, 2>(P, interleaved, s);
        else rot_launch<float, 1>(P, interleaved, s);
    }
    return PCM_LAUNCH_STATUS();
}

// ops_attention.hpp -- device code of the windowed attention (see artemis_ops.h for what it computes).
//
// Everything is built from 16 x 16 blocks on the matrix cores.  One block product mma() contracts over 16:
// lane (i = lane % 16, g = lane / 16) holds A[row i][4g .. 4g+3] and B[4g .. 4g+3][column i] and gets
// D[4g .. 4g+3][column i]: four fp32 instructions of depth 4 or one 16-bit instruction of depth 16.  The result of a
// block product therefore has the layout of a B operand, so that the scores are computed transposed,
//     S^T = K Q^T  (rows: keys, lane: query),
// the softmax over keys is a sum within a lane and over the four lane groups, and P^T goes straight from
// registers into  O^T = V^T P^T  (rows: channels, lane: query): no shuffle, no trip through LDS for P.
#pragma once
#include "ops_common.hpp"

namespace aops {

constexpr int kAttnThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;

struct WindowArgs {
    int B, D, H, W;
    int heads, hd;           // head_dim
    int wd, wh, ww, n;       // window, its tokens
    int sd, sh, sw;          // shift
    int nd, nh, nw;          // windows along the axes
    int label_maps;
    int rd, rh;              // radices of the bias index: (2wh-1)(2ww-1), 2ww-1
    int entries;             // of the bias table
    long long windows;       // B * nd * nh * nw
    float scale, outside2;   // outside * log2(e); -inf: never
};

template <class T>
struct Mma;

template <>
struct Mma<float> {
    using Frag = f32x4;
    static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c)
    {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[0], b[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[1], b[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[2], b[2], c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(a[3], b[3], c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag frag(f32x4 v) { return v; }
};
template <>
struct Mma<__bf16> {
    using Frag = bf16x4;
    static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag frag(f32x4 v)
    {
        return Frag{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
};
template <>
struct Mma<_Float16> {
    using Frag = f16x4;
    static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag frag(f32x4 v)
    {
        return Frag{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    }
};

// a column of four rows of a row-major LDS tile: the A operand (row = channel, contraction over tokens)
template <class T, int STRIDE>
__device__ __forceinline__ typename Mma<T>::Frag column(const T *tile, int token, int channel)
{
    typename Mma<T>::Frag f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = tile[(token + r) * STRIDE + channel];
    return f;
}
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag row4(const T *p)
{
    return *(const typename Mma<T>::Frag *)p;
}

// Where a token of a window lies, and its region.  `live`: it exists and is not padding.
struct Place {
    int token;   // on the (B, D, H, W) map, -1: none
    int label;
    int wrap;    // which axes the shift wrapped around, one bit each
};

__device__ __forceinline__ Place place_of(const WindowArgs &a, const int *__restrict__ labels, long long window, int t)
{
    Place r{-1, -1, 0};
    if (window >= a.windows) return r;
    const unsigned w = (unsigned)window;
    const unsigned kw = w % (unsigned)a.nw, w1 = w / (unsigned)a.nw;
    const unsigned kh = w1 % (unsigned)a.nh, w2 = w1 / (unsigned)a.nh;
    const unsigned kd = w2 % (unsigned)a.nd, b = w2 / (unsigned)a.nd;
    const unsigned tw = (unsigned)t % (unsigned)a.ww, t1 = (unsigned)t / (unsigned)a.ww;
    const unsigned th = t1 % (unsigned)a.wh, td = t1 / (unsigned)a.wh;
    int d = (int)(kd * a.wd + td) + a.sd, h = (int)(kh * a.wh + th) + a.sh, x = (int)(kw * a.ww + tw) + a.sw;
    if (d >= a.D) d -= a.D, r.wrap |= 1;
    if (h >= a.H) h -= a.H, r.wrap |= 2;
    if (x >= a.W) x -= a.W, r.wrap |= 4;
    const int at = (d * a.H + h) * a.W + x;
    r.token = (int)b * a.D * a.H * a.W + at;
    r.label = labels ? labels[(size_t)(a.label_maps > 1 ? b : 0) * a.D * a.H * a.W + at] : 0;
    return r;
}

// the bias index of a pair is corner(a) - corner(b) + middle
__device__ __forceinline__ int corner(const WindowArgs &a, int t)
{
    const int tw = t % a.ww, t1 = t / a.ww;
    return (t1 / a.wh) * a.rd + (t1 % a.wh) * a.rh + tw;
}
__device__ __forceinline__ int middle(const WindowArgs &a) { return (a.wd - 1) * a.rd + (a.wh - 1) * a.rh + a.ww - 1; }

__device__ __forceinline__ float fold_max(float x)
{
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float fold_sum(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Loads four channels of a token's row, zeros where there is no token or no channel
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag load4(const T *__restrict__ base, long long stride, int token, int c, int hd)
{
    typename Mma<T>::Frag f{};
    if (token >= 0 && c < hd) f = *(const typename Mma<T>::Frag *)(base + (long long)token * stride + c);
    return f;
}

// ================================================================================================
// Windows of at most 64 tokens.  A tile is 64 slots: units of 16 * NB slots, each holding one window (NB > 1) or
// as many as fit 16 slots (NB = 1).  Wave w has the queries of slots 16w .. 16w+15; their keys are the NB
// blocks of the unit.  A workgroup keeps one head and goes through tiles, so that the bias of its pairs stays in registers
// (-inf where a pair is of two windows or of empty slots).
// Bound by memory for the model's sizes (64 tokens, 32 channels: 16 products for each value read).
// ================================================================================================

// the head and first tile of a workgroup, and its step.  Workgroups 8 apart run on one XCD; the heads of a tile,
// which share cache lines of the tokens' rows, are kept there.
struct Walk {
    int head;
    long long tile, step;
};
__device__ __forceinline__ Walk walk_of(int heads)
{
    const unsigned x = blockIdx.x % 8, i = blockIdx.x / 8;
    return {(int)(i % (unsigned)heads), (long long)(i / (unsigned)heads) * 8 + x, (long long)(gridDim.x / (unsigned)heads)};
}

template <int NB>
struct Slots {
    // slot -> window (of the tile's) and token; token -1: empty slot
    static __device__ __forceinline__ void of(const WindowArgs &a, int slot, int &window, int &t)
    {
        const int unit = slot / (16 * NB), r = slot % (16 * NB);
        const int fit = NB == 1 ? 16 / a.n : 1;
        const int i = r / a.n;
        window = unit * fit + i;
        t = i < fit ? r % a.n : -1;
    }
    static __host__ __device__ int per_tile(int n) { return 4 / NB * (NB == 1 ? 16 / n : 1); }
};

// bias of (query slot of this lane, four keys of block kb), times log2 e
template <int NB>
__device__ __forceinline__ f32x4 pair_bias(const WindowArgs &a, const float *__restrict__ table, int head, int q, int key)
{
    f32x4 b;
    int qw, qt;
    Slots<NB>::of(a, q, qw, qt);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        int kw, kt;
        Slots<NB>::of(a, key + r, kw, kt);
        b[r] = -INFINITY;
        if (qt >= 0 && kt >= 0 && qw == kw)
            b[r] = table ? table[(size_t)(corner(a, qt) - corner(a, kt) + middle(a)) * a.heads + head] * kLog2e : 0.f;
    }
    return b;
}

// x = scores in the exponent of 2, masked: -inf for what may not be seen
__device__ __forceinline__ float masked(float x, int ql, int qr, int kl, int kr, float outside2)
{
    const bool out = ql != kl || qr != kr;
    if (ql < 0 || kl < 0) return -INFINITY;
    if (!out) return x;
    return outside2 == -INFINITY ? -INFINITY : x + outside2;
}

template <class T, int HD, int NB>
__global__ __launch_bounds__(kAttnThreads) void window_fwd(const WindowArgs a, const T *__restrict__ qkv,
                                                           const float *__restrict__ table,
                                                           const int *__restrict__ labels, T *__restrict__ out)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int STRIDE = HD + 4;  // rows 4 elements apart from a power of two: 16 rows on different banks
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * STRIDE];
    __shared__ __align__(16) T Vs[64 * STRIDE];
    __shared__ int token_s[64], label_s[64], wrap_s[64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16;
    const Walk walk = walk_of(a.heads);
    const int C = a.heads * a.hd;
    const long long stride = 3LL * C;
    const T *base = qkv + (size_t)walk.head * a.hd;
    const int per = Slots<NB>::per_tile(a.n);
    const long long tiles = (a.windows + per - 1) / per;
    const bool mask = labels || a.sd || a.sh || a.sw;
    const int kb0 = wave / NB * NB;  // the first key block of this wave's unit
    const int q = wave * 16 + i;
    f32x4 bias[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) bias[j] = pair_bias<NB>(a, table, walk.head, q, (kb0 + j) * 16 + 4 * g);
    const float scale2 = a.scale * kLog2e;

    for (long long tile = walk.tile; tile < tiles; tile += walk.step) {
        __syncthreads();  // the tile before has been used
        if (threadIdx.x < 64) {
            int w, t;
            Slots<NB>::of(a, threadIdx.x, w, t);
            Place p{-1, -1, 0};
            if (t >= 0) p = place_of(a, labels, tile * per + w, t);
            token_s[threadIdx.x] = p.token;
            label_s[threadIdx.x] = p.label;
            wrap_s[threadIdx.x] = p.wrap;
        }
        __syncthreads();
        for (int k = threadIdx.x; k < 64 * (HD / 4); k += kAttnThreads) {
            const int s = k / (HD / 4), c = k % (HD / 4) * 4;
            const int t = label_s[s] < 0 ? -1 : token_s[s];
            *(Frag *)&Ks[s * STRIDE + c] = load4<T>(base + C, stride, t, c, a.hd);
            *(Frag *)&Vs[s * STRIDE + c] = load4<T>(base + 2 * C, stride, t, c, a.hd);
        }
        const int mine = token_s[q], ql = label_s[q], qr = wrap_s[q];
        Frag qf[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) qf[c] = load4<T>(base, stride, ql < 0 ? -1 : mine, c * 16 + 4 * g, a.hd);
        __syncthreads();
        f32x4 s[NB];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            f32x4 acc{};
#pragma unroll
            for (int c = 0; c < CB; ++c) acc = M::run(row4<T>(&Ks[((kb0 + j) * 16 + i) * STRIDE + c * 16 + 4 * g]), qf[c], acc);
            const int key = (kb0 + j) * 16 + 4 * g;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = bias[j][r] == -INFINITY ? -INFINITY : acc[r] * scale2 + bias[j][r];
                if (mask) x = masked(x, ql, qr, label_s[key + r], wrap_s[key + r], a.outside2);
                s[j][r] = x;
                top = fmaxf(top, x);
            }
        }
        top = fold_max(top);
        if (top == -INFINITY) top = 0.f;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = exp2f(s[j][r] - top);
                sum += s[j][r];
            }
        sum = fold_sum(sum);
        const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        Frag p[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) p[j] = M::frag(s[j] * inv);  // 16 bit: rounded once, as the product takes it
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            f32x4 o{};
#pragma unroll
            for (int j = 0; j < NB; ++j)
                o = M::run(column<T, STRIDE>(Vs, (kb0 + j) * 16 + 4 * g, c * 16 + i), p[j], o);
            if (mine >= 0 && c * 16 + 4 * g < a.hd)
                *(Frag *)(out + (size_t)mine * C + walk.head * a.hd + c * 16 + 4 * g) = M::frag(o);
        }
    }
}

// Backward pass of a tile.  Wave w first has the queries of block w: P^T and dP^T as in the forward pass, the row sums
// delta = sum P dP, dS^T = P^T (dP^T - delta), dQ^T = K^T dS^T.  P and dS go through LDS once; then wave w
// has the keys of block w: dV^T = dO^T P and dK^T = Q^T dS, contracted over the queries of its unit.  The sum
// of dS over the workgroup's windows, from which the table's gradient follows, stays in registers.
template <class T, int HD, int NB>
__global__ __launch_bounds__(kAttnThreads) void window_bwd(const WindowArgs a, const T *__restrict__ qkv,
                                                           const float *__restrict__ table,
                                                           const int *__restrict__ labels,
                                                           const T *__restrict__ dout, T *__restrict__ dqkv,
                                                           float *__restrict__ pairs)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int STRIDE = HD + 4;
    constexpr int PS = 16 * NB + 4;
    constexpr int CB = HD / 16;
    constexpr int TILE = 64 * STRIDE, PAIRS = 2 * 64 * PS;
    __shared__ __align__(16) T Qs[TILE];
    __shared__ __align__(16) T Ks[TILE];
    __shared__ __align__(16) T Gs[TILE];
    __shared__ __align__(16) T Vs[TILE > PAIRS ? TILE : PAIRS];  // V, then P and dS
    T *const Ps = Vs, *const Ss = Vs + 64 * PS;
    __shared__ int token_s[64], label_s[64], wrap_s[64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16;
    const Walk walk = walk_of(a.heads);
    const int C = a.heads * a.hd;
    const long long stride = 3LL * C;
    const T *base = qkv + (size_t)walk.head * a.hd;
    T *dbase = dqkv + (size_t)walk.head * a.hd;
    const int per = Slots<NB>::per_tile(a.n);
    const long long tiles = (a.windows + per - 1) / per;
    const bool mask = labels || a.sd || a.sh || a.sw;
    const int kb0 = wave / NB * NB;
    const int q = wave * 16 + i;
    f32x4 bias[NB], dbias[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        bias[j] = pair_bias<NB>(a, table, walk.head, q, (kb0 + j) * 16 + 4 * g);
        dbias[j] = f32x4{};
    }
    const float scale2 = a.scale * kLog2e;

    for (long long tile = walk.tile; tile < tiles; tile += walk.step) {
        __syncthreads();
        if (threadIdx.x < 64) {
            int w, t;
            Slots<NB>::of(a, threadIdx.x, w, t);
            Place p{-1, -1, 0};
            if (t >= 0) p = place_of(a, labels, tile * per + w, t);
            token_s[threadIdx.x] = p.token;
            label_s[threadIdx.x] = p.label;
            wrap_s[threadIdx.x] = p.wrap;
        }
        __syncthreads();
        for (int k = threadIdx.x; k < 64 * (HD / 4); k += kAttnThreads) {
            const int s = k / (HD / 4), c = k % (HD / 4) * 4;
            const int t = label_s[s] < 0 ? -1 : token_s[s];
            *(Frag *)&Qs[s * STRIDE + c] = load4<T>(base, stride, t, c, a.hd);
            *(Frag *)&Ks[s * STRIDE + c] = load4<T>(base + C, stride, t, c, a.hd);
            *(Frag *)&Vs[s * STRIDE + c] = load4<T>(base + 2 * C, stride, t, c, a.hd);
            *(Frag *)&Gs[s * STRIDE + c] = load4<T>(dout + (size_t)walk.head * a.hd, C, t, c, a.hd);
        }
        const int mine = token_s[q], ql = label_s[q], qr = wrap_s[q];
        __syncthreads();
        Frag qf[CB], gf[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            qf[c] = row4<T>(&Qs[q * STRIDE + c * 16 + 4 * g]);
            gf[c] = row4<T>(&Gs[q * STRIDE + c * 16 + 4 * g]);
        }
        f32x4 s[NB], dp[NB];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            f32x4 acc{}, acc2{};
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const int at = ((kb0 + j) * 16 + i) * STRIDE + c * 16 + 4 * g;
                acc = M::run(row4<T>(&Ks[at]), qf[c], acc);
                acc2 = M::run(row4<T>(&Vs[at]), gf[c], acc2);
            }
            dp[j] = acc2;
            const int key = (kb0 + j) * 16 + 4 * g;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = bias[j][r] == -INFINITY ? -INFINITY : acc[r] * scale2 + bias[j][r];
                if (mask) x = masked(x, ql, qr, label_s[key + r], wrap_s[key + r], a.outside2);
                s[j][r] = x;
                top = fmaxf(top, x);
            }
        }
        top = fold_max(top);
        if (top == -INFINITY) top = 0.f;
        float sum = 0.f, delta = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = exp2f(s[j][r] - top);
                sum += s[j][r];
                delta += s[j][r] * dp[j][r];
            }
        sum = fold_sum(sum);
        const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        delta = fold_sum(delta) * inv;
        Frag ds[NB], p[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const f32x4 pv = s[j] * inv;
            const f32x4 d = pv * (dp[j] - delta);
            dbias[j] += d;
            p[j] = M::frag(pv);
            ds[j] = M::frag(d);  // 16 bit: rounded once, as the products take it; the table's gradient sums it unrounded
        }
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            f32x4 dq{};
#pragma unroll
            for (int j = 0; j < NB; ++j)
                dq = M::run(column<T, STRIDE>(Ks, (kb0 + j) * 16 + 4 * g, c * 16 + i), ds[j], dq);
            if (mine >= 0 && c * 16 + 4 * g < a.hd)
                *(Frag *)(dbase + (size_t)mine * stride + c * 16 + 4 * g) = M::frag(dq * a.scale);
        }
        __syncthreads();  // V has been used
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            *(Frag *)&Ps[q * PS + j * 16 + 4 * g] = p[j];
            *(Frag *)&Ss[q * PS + j * 16 + 4 * g] = ds[j];
        }
        __syncthreads();
        const int kc = wave % NB * 16 + i;  // this lane's key within the unit
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            f32x4 dv{}, dk{};
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int qb = (kb0 + j) * 16 + 4 * g;
                dv = M::run(column<T, STRIDE>(Gs, qb, c * 16 + i), column<T, PS>(Ps, qb, kc), dv);
                dk = M::run(column<T, STRIDE>(Qs, qb, c * 16 + i), column<T, PS>(Ss, qb, kc), dk);
            }
            if (mine >= 0 && c * 16 + 4 * g < a.hd) {  // (slot q is also this lane's key)
                T *to = dbase + (size_t)mine * stride + c * 16 + 4 * g;
                *(Frag *)(to + C) = M::frag(dk * a.scale);
                *(Frag *)(to + 2 * C) = M::frag(dv);
            }
        }
    }
    if (!pairs) return;
    float *to = pairs + (size_t)blockIdx.x * 64 * 16 * NB;
#pragma unroll
    for (int j = 0; j < NB; ++j) *(f32x4 *)&to[q * 16 * NB + j * 16 + 4 * g] = dbias[j];
}


// ================================================================================================
// Longer windows (65 .. 4096 tokens): tiles of 64 queries against tiles of 64 keys, with the running maximum and sum
// of a softmax over the key tiles.  The bias comes from a copy of the table with one head's entries in a row.
// ================================================================================================

struct LongTile {
    long long window;
    int head, first;  // the tile's first token
};
__device__ __forceinline__ LongTile long_tile(const WindowArgs &a)
{
    const unsigned tiles = (unsigned)(a.n + 63) / 64;
    const unsigned t = blockIdx.x % tiles, r = blockIdx.x / tiles;
    return {(long long)(r / (unsigned)a.heads), (int)(r % (unsigned)a.heads), (int)t * 64};
}

struct TokenRow {
    int token[64], label[64], wrap[64], corner[64];
    __device__ __forceinline__ void fill(const WindowArgs &a, const int *labels, long long window, int first, int s)
    {
        Place p{-1, -1, 0};
        int c = 0;
        if (first + s < a.n) {
            p = place_of(a, labels, window, first + s);
            c = ::aops::corner(a, first + s);
        }
        token[s] = p.token;
        label[s] = p.token < 0 ? -1 : p.label;
        wrap[s] = p.wrap;
        corner[s] = c;
    }
};

template <class T, int HD>
__device__ __forceinline__ void stage(T *tile, const T *__restrict__ base, long long stride, const TokenRow &row, int hd)
{
    constexpr int STRIDE = HD + 4;
    for (int k = threadIdx.x; k < 64 * (HD / 4); k += kAttnThreads) {
        const int s = k / (HD / 4), c = k % (HD / 4) * 4;
        *(typename Mma<T>::Frag *)&tile[s * STRIDE + c] = load4<T>(base, stride, row.label[s] < 0 ? -1 : row.token[s], c, hd);
    }
}

template <class T, int HD>
__global__ __launch_bounds__(kAttnThreads) void long_fwd(const WindowArgs a, const T *__restrict__ qkv,
                                                         const float *__restrict__ bias_by_head,
                                                         const int *__restrict__ labels, T *__restrict__ out,
                                                         float *__restrict__ lse)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int STRIDE = HD + 4;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * STRIDE];
    __shared__ __align__(16) T Vs[64 * STRIDE];
    __shared__ TokenRow qrow, krow;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, q = wave * 16 + i;
    const LongTile lt = long_tile(a);
    const int C = a.heads * a.hd;
    const long long stride = 3LL * C;
    const T *base = qkv + (size_t)lt.head * a.hd;
    const float *bias = bias_by_head ? bias_by_head + (size_t)lt.head * a.entries : nullptr;
    if (threadIdx.x < 64) qrow.fill(a, labels, lt.window, lt.first, threadIdx.x);
    __syncthreads();
    const int mine = qrow.token[q], ql = qrow.label[q], qr = qrow.wrap[q], qc = qrow.corner[q] + middle(a);
    Frag qf[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) qf[c] = load4<T>(base, stride, ql < 0 ? -1 : mine, c * 16 + 4 * g, a.hd);
    const float scale2 = a.scale * kLog2e;
    float top = -INFINITY, sum = 0.f;
    f32x4 o[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) o[c] = f32x4{};
    for (int k0 = 0; k0 < a.n; k0 += 64) {
        __syncthreads();
        if (threadIdx.x < 64) krow.fill(a, labels, lt.window, k0, threadIdx.x);
        __syncthreads();
        stage<T, HD>(Ks, base + C, stride, krow, a.hd);
        stage<T, HD>(Vs, base + 2 * C, stride, krow, a.hd);
        __syncthreads();
        f32x4 s[4];
        float high = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 acc{};
#pragma unroll
            for (int c = 0; c < CB; ++c) acc = M::run(row4<T>(&Ks[(j * 16 + i) * STRIDE + c * 16 + 4 * g]), qf[c], acc);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = j * 16 + 4 * g + r;
                float x = acc[r] * scale2;
                if (bias) x += bias[qc - krow.corner[key]];
                x = masked(x, ql, qr, krow.label[key], krow.wrap[key], a.outside2);
                s[j][r] = x;
                high = fmaxf(high, x);
            }
        }
        high = fmaxf(fold_max(high), top);
        const float at = high == -INFINITY ? 0.f : high;
        const float fade = exp2f(top - at);
        top = high;
        float part = 0.f;
        Frag p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = exp2f(s[j][r] - at);
                part += s[j][r];
            }
            p[j] = M::frag(s[j]);
        }
        sum = sum * fade + part;
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            o[c] *= fade;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[c] = M::run(column<T, STRIDE>(Vs, j * 16 + 4 * g, c * 16 + i), p[j], o[c]);
        }
    }
    sum = fold_sum(sum);
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    if (mine < 0) return;
#pragma unroll
    for (int c = 0; c < CB; ++c)
        if (c * 16 + 4 * g < a.hd)
            *(Frag *)(out + (size_t)mine * C + lt.head * a.hd + c * 16 + 4 * g) = M::frag(o[c] * inv);
    // log2 of the row's sum of 2^x; +inf for an empty row, so that its P is 0 in the backward pass
    if (lse && g == 0)
        lse[((size_t)lt.window * a.heads + lt.head) * a.n + lt.first + q] = top == -INFINITY ? INFINITY : top + log2f(sum);
}

// dQ, and delta = sum over keys of P dP for each query.  delta is also the product of out and dout; in 16 bits `out` is
// rounded, so that product c is only near: dS = P (dP - c) serves dQ, which is rounded as coarsely itself, and
// c + sum P (dP - c), summed here in fp32, is the delta that the table's gradient and dK are computed with.
template <class T, int HD>
__global__ __launch_bounds__(kAttnThreads) void long_bwd_q(const WindowArgs a, const T *__restrict__ qkv,
                                                           const float *__restrict__ bias_by_head,
                                                           const int *__restrict__ labels, const T *__restrict__ out,
                                                           const float *__restrict__ lse, const T *__restrict__ dout,
                                                           T *__restrict__ dqkv, float *__restrict__ delta)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int STRIDE = HD + 4;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * STRIDE];
    __shared__ __align__(16) T Vs[64 * STRIDE];
    __shared__ TokenRow qrow, krow;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, q = wave * 16 + i;
    const LongTile lt = long_tile(a);
    const int C = a.heads * a.hd;
    const long long stride = 3LL * C;
    const T *base = qkv + (size_t)lt.head * a.hd;
    const float *bias = bias_by_head ? bias_by_head + (size_t)lt.head * a.entries : nullptr;
    if (threadIdx.x < 64) qrow.fill(a, labels, lt.window, lt.first, threadIdx.x);
    __syncthreads();
    const int mine = qrow.token[q], ql = qrow.label[q], qr = qrow.wrap[q], qc = qrow.corner[q] + middle(a);
    const int live = ql < 0 ? -1 : mine;
    Frag qf[CB], gf[CB];
    float near = 0.f;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        qf[c] = load4<T>(base, stride, live, c * 16 + 4 * g, a.hd);
        gf[c] = load4<T>(dout + (size_t)lt.head * a.hd, C, live, c * 16 + 4 * g, a.hd);
        const Frag of = load4<T>(out + (size_t)lt.head * a.hd, C, live, c * 16 + 4 * g, a.hd);
#pragma unroll
        for (int r = 0; r < 4; ++r) near += (float)of[r] * (float)gf[c][r];
    }
    near = fold_sum(near);
    const size_t line = ((size_t)lt.window * a.heads + lt.head) * a.n + lt.first + q;
    const float shift = mine >= 0 ? lse[line] : INFINITY;
    const float scale2 = a.scale * kLog2e;
    float rest = 0.f;
    f32x4 dq[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) dq[c] = f32x4{};
    for (int k0 = 0; k0 < a.n; k0 += 64) {
        __syncthreads();
        if (threadIdx.x < 64) krow.fill(a, labels, lt.window, k0, threadIdx.x);
        __syncthreads();
        stage<T, HD>(Ks, base + C, stride, krow, a.hd);
        stage<T, HD>(Vs, base + 2 * C, stride, krow, a.hd);
        __syncthreads();
        Frag ds[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 acc{}, acc2{};
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const int at = (j * 16 + i) * STRIDE + c * 16 + 4 * g;
                acc = M::run(row4<T>(&Ks[at]), qf[c], acc);
                acc2 = M::run(row4<T>(&Vs[at]), gf[c], acc2);
            }
            f32x4 d;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = j * 16 + 4 * g + r;
                float x = acc[r] * scale2;
                if (bias) x += bias[qc - krow.corner[key]];
                x = masked(x, ql, qr, krow.label[key], krow.wrap[key], a.outside2);
                d[r] = x == -INFINITY ? 0.f : exp2f(x - shift) * (acc2[r] - near);
                rest += d[r];
            }
            ds[j] = M::frag(d);
        }
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) dq[c] = M::run(column<T, STRIDE>(Ks, j * 16 + 4 * g, c * 16 + i), ds[j], dq[c]);
    }
    rest = fold_sum(rest);
    if (mine < 0) return;
    if (g == 0) delta[line] = near + rest;
#pragma unroll
    for (int c = 0; c < CB; ++c)
        if (c * 16 + 4 * g < a.hd)
            *(Frag *)(dqkv + (size_t)mine * stride + lt.head * a.hd + c * 16 + 4 * g) = M::frag(dq[c] * a.scale);
}

// dK and dV: wave w has 16 keys and goes through the queries, S = Q K^T (rows: queries, lane: key), so that P and dS have the
// layout of the B operands of dV^T = dO^T P and dK^T = Q^T dS.
template <class T, int HD>
__global__ __launch_bounds__(kAttnThreads) void long_bwd_kv(const WindowArgs a, const T *__restrict__ qkv,
                                                            const float *__restrict__ bias_by_head,
                                                            const int *__restrict__ labels,
                                                            const float *__restrict__ lse, const T *__restrict__ dout,
                                                            T *__restrict__ dqkv, const float *__restrict__ delta)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int STRIDE = HD + 4;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Qs[64 * STRIDE];
    __shared__ __align__(16) T Gs[64 * STRIDE];
    __shared__ TokenRow qrow, krow;
    __shared__ float lse_s[64], delta_s[64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, k = wave * 16 + i;
    const LongTile lt = long_tile(a);
    const int C = a.heads * a.hd;
    const long long stride = 3LL * C;
    const T *base = qkv + (size_t)lt.head * a.hd;
    const float *bias = bias_by_head ? bias_by_head + (size_t)lt.head * a.entries : nullptr;
    if (threadIdx.x < 64) krow.fill(a, labels, lt.window, lt.first, threadIdx.x);
    __syncthreads();
    const int mine = krow.token[k], kl = krow.label[k], kr = krow.wrap[k], kc = middle(a) - krow.corner[k];
    const int live = kl < 0 ? -1 : mine;
    Frag kf[CB], vf[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        kf[c] = load4<T>(base + C, stride, live, c * 16 + 4 * g, a.hd);
        vf[c] = load4<T>(base + 2 * C, stride, live, c * 16 + 4 * g, a.hd);
    }
    const float scale2 = a.scale * kLog2e;
    const size_t lines = ((size_t)lt.window * a.heads + lt.head) * a.n;
    f32x4 dk[CB], dv[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) dk[c] = dv[c] = f32x4{};
    for (int q0 = 0; q0 < a.n; q0 += 64) {
        __syncthreads();
        if (threadIdx.x < 64) {
            qrow.fill(a, labels, lt.window, q0, threadIdx.x);
            const bool in = q0 + (int)threadIdx.x < a.n;
            lse_s[threadIdx.x] = in ? lse[lines + q0 + threadIdx.x] : INFINITY;
            delta_s[threadIdx.x] = in ? delta[lines + q0 + threadIdx.x] : 0.f;
        }
        __syncthreads();
        stage<T, HD>(Qs, base, stride, qrow, a.hd);
        stage<T, HD>(Gs, dout + (size_t)lt.head * a.hd, C, qrow, a.hd);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 acc{}, acc2{};
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const int at = (j * 16 + i) * STRIDE + c * 16 + 4 * g;
                acc = M::run(row4<T>(&Qs[at]), kf[c], acc);
                acc2 = M::run(row4<T>(&Gs[at]), vf[c], acc2);
            }
            f32x4 p, d;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int q = j * 16 + 4 * g + r;
                float x = acc[r] * scale2;
                if (bias) x += bias[qrow.corner[q] + kc];
                x = masked(x, qrow.label[q], qrow.wrap[q], kl, kr, a.outside2);
                p[r] = x == -INFINITY ? 0.f : exp2f(x - lse_s[q]);
                d[r] = p[r] * (acc2[r] - delta_s[q]);
            }
            const Frag pf = M::frag(p), df = M::frag(d);
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                dv[c] = M::run(column<T, STRIDE>(Gs, j * 16 + 4 * g, c * 16 + i), pf, dv[c]);
                dk[c] = M::run(column<T, STRIDE>(Qs, j * 16 + 4 * g, c * 16 + i), df, dk[c]);
            }
        }
    }
    if (mine < 0) return;
#pragma unroll
    for (int c = 0; c < CB; ++c)
        if (c * 16 + 4 * g < a.hd) {
            T *to = dqkv + (size_t)mine * stride + lt.head * a.hd + c * 16 + 4 * g;
            *(Frag *)(to + C) = M::frag(dk[c] * a.scale);
            *(Frag *)(to + 2 * C) = M::frag(dv[c]);
        }
}

// dense[head][query][key] = the sum of dS over the windows, for one tile of 64 x 64 pairs of one head
template <class T, int HD>
__global__ __launch_bounds__(kAttnThreads) void long_bwd_pairs(const WindowArgs a, const T *__restrict__ qkv,
                                                               const float *__restrict__ bias_by_head,
                                                               const int *__restrict__ labels,
                                                               const float *__restrict__ lse, const T *__restrict__ dout,
                                                               const float *__restrict__ delta, float *__restrict__ dense)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int STRIDE = HD + 4;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * STRIDE];
    __shared__ __align__(16) T Vs[64 * STRIDE];
    __shared__ TokenRow qrow, krow;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, q = wave * 16 + i;
    const unsigned tiles = (unsigned)(a.n + 63) / 64;
    const int k0 = (int)(blockIdx.x % tiles) * 64, q0 = (int)(blockIdx.x / tiles % tiles) * 64;
    const int head = (int)(blockIdx.x / tiles / tiles);
    const int C = a.heads * a.hd;
    const long long stride = 3LL * C;
    const T *base = qkv + (size_t)head * a.hd;
    const float *bias = bias_by_head ? bias_by_head + (size_t)head * a.entries : nullptr;
    const float scale2 = a.scale * kLog2e;
    f32x4 sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = f32x4{};
    for (long long window = 0; window < a.windows; ++window) {
        __syncthreads();
        if (threadIdx.x < 64)
            qrow.fill(a, labels, window, q0, threadIdx.x);
        else if (threadIdx.x < 128)
            krow.fill(a, labels, window, k0, threadIdx.x - 64);
        __syncthreads();
        stage<T, HD>(Ks, base + C, stride, krow, a.hd);
        stage<T, HD>(Vs, base + 2 * C, stride, krow, a.hd);
        const int mine = qrow.token[q], ql = qrow.label[q], qr = qrow.wrap[q], qc = qrow.corner[q] + middle(a);
        const int live = ql < 0 ? -1 : mine;
        Frag qf[CB], gf[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            qf[c] = load4<T>(base, stride, live, c * 16 + 4 * g, a.hd);
            gf[c] = load4<T>(dout + (size_t)head * a.hd, C, live, c * 16 + 4 * g, a.hd);
        }
        const size_t line = ((size_t)window * a.heads + head) * a.n + q0 + q;
        const float shift = mine >= 0 ? lse[line] : INFINITY, del = mine >= 0 ? delta[line] : 0.f;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 acc{}, acc2{};
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                const int at = (j * 16 + i) * STRIDE + c * 16 + 4 * g;
                acc = M::run(row4<T>(&Ks[at]), qf[c], acc);
                acc2 = M::run(row4<T>(&Vs[at]), gf[c], acc2);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = j * 16 + 4 * g + r;
                float x = acc[r] * scale2;
                if (bias) x += bias[qc - krow.corner[key]];
                x = masked(x, ql, qr, krow.label[key], krow.wrap[key], a.outside2);
                if (x != -INFINITY) sum[j][r] += exp2f(x - shift) * (acc2[r] - del);
            }
        }
    }
    if (q0 + q >= a.n) return;
    float *to = dense + ((size_t)head * a.n + q0 + q) * a.n + k0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (k0 + j * 16 + 4 * g + r < a.n) to[j * 16 + 4 * g + r] = sum[j][r];
}

// launchers, one translation unit for each element type
struct AttnBuffers {
    const void *qkv;
    const float *table;         // as given
    const float *bias_by_head;  // long windows: the copy
    const int *labels;
    const void *out_in;
    void *out;
    float *lse;
    const void *dout;
    void *dqkv;
    float *pairs, *dense, *delta;
    int groups;                 // workgroups of window_fwd / window_bwd
};
template <class T>
void launch_attention_fwd(const WindowArgs &a, const AttnBuffers &b, hipStream_t st);
template <class T>
void launch_attention_bwd(const WindowArgs &a, const AttnBuffers &b, hipStream_t st);

}  // namespace aops

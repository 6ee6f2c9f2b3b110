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
// Waves of a SIMD that the register budget is for: at two (256 registers) the compiler keeps products in vector registers; at
// one it puts them into accumulation registers, and every value costs a move.  128 fp32 channels need more than 256.
template <class T, int HD>
constexpr int kWaves = HD * sizeof(T) <= 256 ? 2 : 1;
constexpr float kLog2e = 1.44269504088896340736f;

// Division of numbers below 2^31 by a constant d: q = (mulhi(x, m) + x) >> s with m = floor(2^32 (2^s - d) / d) + 1,
// s = ceil(log2 d) -- the reciprocal rounded up to 33 bits, whose top one is the added x.
struct Divider {
    unsigned m = 1, s = 0;
    Divider() = default;
    explicit Divider(unsigned d)
    {
        while ((1ull << s) < d) ++s;
        m = (unsigned)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    }
    __device__ __forceinline__ unsigned of(unsigned x) const { return (__umulhi(x, m) + x) >> s; }
};

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
    Divider by_nd, by_nh, by_nw;
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
    static __device__ __forceinline__ f32x4 run2(Frag a0, Frag a1, Frag b0, Frag b1, f32x4 c)
    {
        return run(a1, b1, run(a0, b0, c));
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
    // two block products at once, depth 32: any order of the contraction will do, as long as a and b share it
    static __device__ __forceinline__ f32x4 run2(Frag a0, Frag a1, Frag b0, Frag b1, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7),
                                                       __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7), c, 0, 0, 0);
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
    static __device__ __forceinline__ f32x4 run2(Frag a0, Frag a1, Frag b0, Frag b1, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7),
                                                      __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag frag(f32x4 v)
    {
        return Frag{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    }
};

// fp16 operands.  Below 2^-14 the type's steps stay 2^-24 wide, and beyond 65504 there is nothing.  P of thousands of keys, and
// dS = P (dP - delta) the more so where dout is small, lie below, though their sums do not (dS unscaled: at 4096 tokens and dout of
// 1e-3, dQ and dK off by 7e-3 of their size); dS with a scaled loss may lie above.  So P enters the products times 2^15 (nothing is
// above 1), and dS times a power of two of its column: a query in dQ, a key in dK, both of which a lane's column of the result
// belongs to, and so does the way back.  bf16 has fp32's exponents and takes both as they are.
template <class T>
constexpr int kLift = 0;
template <>
inline constexpr int kLift<_Float16> = 15;
template <class T>
constexpr float kDown = kLift<T> ? 0x1p-15f : 1.f;

// the exponent of a magnitude, -98 at least: its power of two and that one's reciprocal, times up to 2^29, are normal numbers
__device__ __forceinline__ int exponent_of(float m)
{
    const int e = (int)(__builtin_bit_cast(unsigned, m) >> 23) - 127;
    return e < -98 ? -98 : e;
}
__device__ __forceinline__ float two_to(int e) { return __builtin_bit_cast(float, (unsigned)(127 + e) << 23); }

// four neighbours of an LDS tile as an operand
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag row4(const T *p)
{
    return *(const typename Mma<T>::Frag *)p;
}

// Where a token of a window lies, and its region.
struct Place {
    int token;   // on the (B, D, H, W) map, -1: none
    int label;   // < 0: padding
    int wrap;    // which axes the shift wrapped around, one bit each
};

// `td`, `th`, `tw`: the token's coordinates in the window
__device__ __forceinline__ Place place_of(const WindowArgs &a, const int *__restrict__ labels, long long window, int td, int th,
                                          int tw)
{
    Place r{-1, -1, 0};
    if (window >= a.windows) return r;
    const unsigned w = (unsigned)window;
    const unsigned w1 = a.by_nw.of(w), kw = w - w1 * a.nw;
    const unsigned w2 = a.by_nh.of(w1), kh = w1 - w2 * a.nh;
    const unsigned b = a.by_nd.of(w2), kd = w2 - b * a.nd;
    // (unsigned: in front of the wrap a coordinate may pass 2^31)
    const unsigned D = (unsigned)a.D, H = (unsigned)a.H, W = (unsigned)a.W;
    unsigned d = kd * a.wd + td + a.sd, h = kh * a.wh + th + a.sh, x = kw * a.ww + tw + a.sw;
    if (d >= D) d -= D, r.wrap |= 1;
    if (h >= H) h -= H, r.wrap |= 2;
    if (x >= W) x -= W, r.wrap |= 4;
    const int at = (int)((d * H + h) * W + x);
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

// the largest finite magnitude of a lane's values (NaN: left out; an infinity: none is to be had)
template <int N>
__device__ __forceinline__ float largest(const f32x4 (&x)[N])
{
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int r = 0; r < 4; r += 2) m = fmaxf(m, fmaxf(fabsf(x[j][r]), fabsf(x[j][r + 1])));
    return m;
}

// The power of two that brings a column's largest magnitude to 2^14 ..: all of the column is here.  1 where it is not finite.
__device__ __forceinline__ float column_scale(float m)
{
    m = fold_max(m);
    return m < INFINITY ? two_to(14 - exponent_of(m)) : 1.f;
}

// The same where a column comes tile by tile: the scale follows the largest magnitude met so far, and what has been summed
// follows the scale.  A new one leaves room for 16 times as much, so that changes are few.
struct RunningScale {
    float s = 1.f, limit = 0.f;
    template <int N, int C>
    __device__ __forceinline__ void apply(f32x4 (&x)[N], f32x4 (&sum)[C])
    {
        float m = largest(x);
        if (__any(m > limit)) {
            m = fold_max(m);
            if (m > limit && m < INFINITY) {  // (the same in the column's four lanes)
                const int e = exponent_of(m);
                const float to = two_to(10 - e), by = to / s;
                s = to;
                limit = two_to(e) * 32.f;  // 2^15 when scaled
#pragma unroll
                for (int c = 0; c < C; ++c) sum[c] *= by;
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= s;
    }
};

// Four channels of a token's row.  Loaded whether or not there is such a token and channel (from the tensor's first token
// or the head's first channels then), and cleared where it is used: a load under a condition shares its registers with the
// zeros, and the compiler waits for all loads in flight before it writes those.  (So guarded, a tile's eight
// loads went one after the other: 118 us for what took 89 without in the kernel of the table's gradient, at 4096 tokens and 8 heads.)
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag raw4(const T *__restrict__ base, unsigned stride, int token, int c, int hd)
{
    return *(const typename Mma<T>::Frag *)(base + (unsigned long long)(unsigned)(token < 0 ? 0 : token) * stride +
                                               (c < hd ? c : 0));
}
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag cleared(typename Mma<T>::Frag f, bool keep)
{
    return keep ? f : typename Mma<T>::Frag{};
}
template <class T>
__device__ __forceinline__ typename Mma<T>::Frag load4(const T *__restrict__ base, unsigned stride, int token, int c, int hd)
{
    return cleared<T>(raw4<T>(base, stride, token, c, hd), token >= 0 && c < hd);
}

// Nothing below is loaded before x is there.  Where a register's next value is loaded while this one is still wanted, the
// compiler loads into another and copies that, which waits for the load: so what becomes of this one is had first.
template <class X>
__device__ __forceinline__ void settle(X &x)
{
    asm volatile("" : "+v"(x)::"memory");
}

// 64 rows on their way to LDS: HD / 16 pieces of four channels in each thread
template <class T, int HD>
struct Rows {
    using Frag = typename Mma<T>::Frag;
    static constexpr int kPieces = HD / 16, kRowStep = kAttnThreads / (HD / 4);
    Frag f[kPieces];
    static __device__ __forceinline__ int row(int m) { return threadIdx.x / (HD / 4) + m * kRowStep; }
    static __device__ __forceinline__ int channel() { return threadIdx.x % (HD / 4) * 4; }
    __device__ __forceinline__ void load(const T *__restrict__ base, unsigned stride, const int (&token)[kPieces], int hd)
    {
#pragma unroll
        for (int m = 0; m < kPieces; ++m) f[m] = raw4<T>(base, stride, token[m], channel(), hd);
    }
    __device__ __forceinline__ void arrive()
    {
#pragma unroll
        for (int m = 0; m < kPieces; ++m) settle(f[m]);
    }
    // `none`: bit m: there is no such piece.  For whole tiles it is 0 in every thread: one branch.
    __device__ __forceinline__ void clear(unsigned none)
    {
        if (!__any(none != 0)) return;
#pragma unroll
        for (int m = 0; m < kPieces; ++m) f[m] = cleared<T>(f[m], !(none >> m & 1));
    }
    static __device__ __forceinline__ unsigned none_of(const int (&token)[kPieces], int hd)
    {
        unsigned none = channel() < hd ? 0u : ~0u;
#pragma unroll
        for (int m = 0; m < kPieces; ++m) none |= (unsigned)(token[m] < 0) << m;
        return none;
    }
    __device__ __forceinline__ void store_rows(T *tile) const  // [64][HD + 4]
    {
#pragma unroll
        for (int m = 0; m < kPieces; ++m) *(Frag *)&tile[row(m) * (HD + 4) + channel()] = f[m];
    }
    __device__ __forceinline__ void store_columns(T *tile) const  // [HD][64 + 4]
    {
#pragma unroll
        for (int m = 0; m < kPieces; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) tile[(channel() + e) * 68 + row(m)] = f[m][e];
    }
};

// D[token 4g ..][column i] for a block of 16 rows of a row-major tile against a lane's operand: contraction over channels
template <class T, int HD>
__device__ __forceinline__ f32x4 over_channels(const T *rows, int first, const typename Mma<T>::Frag *own)
{
    using M = Mma<T>;
    const int i = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
    const T *p = rows + (first + i) * (HD + 4) + 4 * g;
    f32x4 acc{};
    if constexpr (HD >= 32) {
#pragma unroll
        for (int c = 0; c < HD / 16; c += 2) acc = M::run2(row4<T>(p + c * 16), row4<T>(p + c * 16 + 16), own[c], own[c + 1], acc);
    } else {
        acc = M::run(row4<T>(p), own[0], acc);
    }
    return acc;
}

// The A operand of a contraction over tokens (row: channel c * 16 + i; tokens at + 4g ..): one read of a tile stored by
// columns, four of one stored by rows
template <class T, int HD, bool BY_ROWS>
__device__ __forceinline__ typename Mma<T>::Frag column(const T *tile, int c, int at)
{
    const int i = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
    if constexpr (BY_ROWS) {
        typename Mma<T>::Frag f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = tile[(at + 4 * g + r) * (HD + 4) + c * 16 + i];
        return f;
    }
    return row4<T>(tile + (c * 16 + i) * 68 + at + 4 * g);
}

// acc[c] += tile^T (channels c * 16 .., tokens first ..) times N blocks of B operands: contraction over 16 N tokens
template <class T, int HD, int N, bool BY_ROWS = false>
__device__ __forceinline__ void over_tokens(f32x4 (&acc)[HD / 16], const T *tile, int first,
                                            const typename Mma<T>::Frag (&b)[N])
{
    using M = Mma<T>;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) {
        if constexpr (N == 1)
            acc[c] = M::run(column<T, HD, BY_ROWS>(tile, c, first), b[0], acc[c]);
        else
#pragma unroll
            for (int j = 0; j < N; j += 2)
                acc[c] = M::run2(column<T, HD, BY_ROWS>(tile, c, first + j * 16),
                                 column<T, HD, BY_ROWS>(tile, c, first + j * 16 + 16), b[j], b[j + 1], acc[c]);
    }
}

// the same of a whole tile with two operands, each piece of the tile read once
template <class T, int HD>
__device__ __forceinline__ void over_tokens_both(f32x4 (&x)[HD / 16], f32x4 (&y)[HD / 16], const T *tile,
                                                 const typename Mma<T>::Frag (&bx)[4], const typename Mma<T>::Frag (&by)[4])
{
    using M = Mma<T>;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const typename M::Frag f0 = column<T, HD, false>(tile, c, j * 16), f1 = column<T, HD, false>(tile, c, j * 16 + 16);
            x[c] = M::run2(f0, f1, bx[j], bx[j + 1], x[c]);
            y[c] = M::run2(f0, f1, by[j], by[j + 1], y[c]);
        }
}

// ================================================================================================
// Windows of at most 64 tokens.  A tile is 64 slots: units of 16 * NB slots, each holding one window (NB > 1) or
// as many as fit 16 slots (NB = 1).  Wave w has the queries of slots 16w .. 16w+15; their keys are the NB
// blocks of the unit.  A workgroup keeps one head and goes through tiles, so that the bias of its pairs stays in registers
// (-inf where a pair is of two windows or of empty slots).
// Bound by memory where windows are small or 16 bit, by memory and products together in fp32 at 64 tokens: 8192 windows with 2
// heads of 32 channels take 124 us forward (537 MB at 4.3 TB/s) and 288 backward (940 MB at 3.3 TB/s; matrix units busy for half
// of it, a quarter of the waves' time spent waiting), in bf16 71 (3.8 TB/s) and 151 (3.1); 131072 tokens in windows of 4, 4
// heads: 70 us (3.8 TB/s) and 95 (4.9); bf16, 8160 shifted windows of 64, 4 heads, forward: 140 us (3.8 TB/s).  (Kernels alone, by
// a trace of 200 passes.)  Registers for 3 and 4 waves on a SIMD were slower (spills), as was reading the operands of the
// next products ahead of those at hand (by 8 %).
// P (16 bit, and dS) is rounded to the type as the operand of a product that matrix instructions take, its sum is of the
// unrounded ones.  Outputs then lie 0.0023 of their size (bf16) from the definition instead of the 0.0017 that their own rounding
// makes; two operands, the rounded one and what is left of it, would double those products and their conversions.
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

// x = scores in the exponent of 2, masked: -inf for what may not be seen
__device__ __forceinline__ float masked(float x, int ql, int qr, int kl, int kr, float outside2)
{
    const bool out = ql != kl || qr != kr;
    if (ql < 0 || kl < 0) return -INFINITY;
    if (!out) return x;
    return outside2 == -INFINITY ? -INFINITY : x + outside2;
}

// What the 64 slots of a tile hold.  `mixed`: some are of different regions, or padding.
struct Spots {
    int token[64], label[64], wrap[64];
    int source[64];  // the token, or -1 for padding too
    int mixed;
};

// The slot of this thread (the first wave's), and the spots of one tile after the other
template <int NB>
struct Spotter {
    int window, t, td, th, tw;
    __device__ __forceinline__ explicit Spotter(const WindowArgs &a)
    {
        Slots<NB>::of(a, threadIdx.x % 64, window, t);
        const int u = t < 0 ? 0 : t, u1 = u / a.ww;
        tw = u % a.ww, th = u1 % a.wh, td = u1 / a.wh;
    }
    __device__ __forceinline__ Place look(const WindowArgs &a, const int *labels, long long first) const
    {
        return t < 0 ? Place{-1, -1, 0} : place_of(a, labels, first + window, td, th, tw);
    }
    // where the bias table is entered: the slot's corner, and its window or -1
    __device__ __forceinline__ void write_corners(const WindowArgs &a, Spots &to) const
    {
        to.token[threadIdx.x] = td * a.rd + th * a.rh + tw;
        to.label[threadIdx.x] = t < 0 ? -1 : window;
    }
    // (only pairs within a window meet, but one comparison serves all windows of the tile)
    __device__ __forceinline__ void write(Spots &to, const Place &p) const
    {
        const int s = threadIdx.x;
        to.token[s] = p.token;
        to.source[s] = p.label < 0 ? -1 : p.token;
        to.label[s] = p.label;
        to.wrap[s] = p.wrap;
        const int label = __shfl(p.label, 0), wrap = __shfl(p.wrap, 0);
        const bool mixed = !__all(t < 0 || p.token < 0 || (p.label >= 0 && p.label == label && p.wrap == wrap));
        if (s == 0) to.mixed = mixed;
    }
};

// biases of (query slot q, key slots of NB blocks), times log2 e; -inf where the two are not of one window
template <int NB>
__device__ __forceinline__ void pair_biases(f32x4 (&b)[NB], const WindowArgs &a, const Spots &corners,
                                            const float *__restrict__ table, int head, int q, int key)
{
    const int from = corners.token[q] + middle(a), window = corners.label[q];
    unsigned meet = 0;
    int entry[NB][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool m = window == corners.label[key + j * 16 + r];
            entry[j][r] = m ? (from - corners.token[key + j * 16 + r]) * a.heads + head : 0;
            meet |= (unsigned)m << (j * 4 + r);
        }
    if (window < 0) meet = 0;
#pragma unroll
    for (int j = 0; j < NB; ++j) b[j] = f32x4{};
    if (table) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) b[j][r] = table[entry[j][r]];
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) b[j][r] = meet >> (j * 4 + r) & 1 ? b[j][r] * kLog2e : -INFINITY;
}

// the mask of (query slot q, key slots of NB blocks)
template <int NB>
__device__ __forceinline__ void mask_slots(f32x4 (&s)[NB], const Spots &at, int q, int key, float outside2)
{
    const int ql = at.label[q], qr = at.wrap[q];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        __builtin_amdgcn_sched_barrier(0);  // (few labels at a time: their registers cost all tiles a wave)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            s[j][r] = masked(s[j][r], ql, qr, at.label[key + j * 16 + r], at.wrap[key + j * 16 + r], outside2);
    }
}

template <class T, int HD>
__device__ __forceinline__ void tokens_at(const Spots &at, int (&token)[Rows<T, HD>::kPieces])
{
#pragma unroll
    for (int m = 0; m < Rows<T, HD>::kPieces; ++m) token[m] = at.source[Rows<T, HD>::row(m)];
}

// Windows that share a block of 16 slots meet in its products, where an operand 0 does not undo an infinity or a NaN of
// another window's tokens.  Where a tile holds any (kept in a flag beside it), the products over tokens are made
// window by window instead, with the other windows' tokens taken for 0, and each lane keeps its own window's.
template <class T, int HD, int NB, bool BY_ROWS = false>
__device__ __forceinline__ void over_unit(f32x4 (&acc)[HD / 16], const T *tile, int first,
                                          const typename Mma<T>::Frag (&b)[NB], bool odd, int n)
{
    if constexpr (NB == 1) {
        if (odd) {
            using M = Mma<T>;
            const int i = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
            for (int w = 0; w < 16 / n; ++w)
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    typename M::Frag f = column<T, HD, BY_ROWS>(tile, c, first), e = b[0];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((4 * g + r) / n != w) f[r] = (T)0.f, e[r] = (T)0.f;
                    const f32x4 o = M::run(f, e, f32x4{});
                    if (i / n == w) acc[c] += o;
                }
            return;
        }
    }
    over_tokens<T, HD, NB, BY_ROWS>(acc, tile, first, b);
}

// whether a thread's pieces hold an infinity or a NaN
template <class T, int HD>
__device__ __forceinline__ bool not_finite(const Rows<T, HD> &r)
{
    float x = 0.f;
#pragma unroll
    for (int m = 0; m < Rows<T, HD>::kPieces; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) x += (float)r.f[m][e] * 0.f;
    return x != 0.f;  // 0, or NaN
}

// Stores are not made under a condition either: a wait for the next tile's loads counts the stores behind them, and where
// their number is not known it waits for all of them.  What belongs to no token goes to `spare`.
template <class T>
__device__ __forceinline__ T *store_at(T *real, T *spare, bool wanted)
{
    return wanted ? real : spare + threadIdx.x % 64 * 4;
}
constexpr size_t kSpareBytes = 64 * 4 * sizeof(float);

template <class T, int HD, int NB, bool LABELS>
__global__ __launch_bounds__(kAttnThreads, (kWaves<T, HD>)) void window_fwd(const WindowArgs a, const T *__restrict__ qkv,
                                                           const float *__restrict__ table, const int *__restrict__ label_map,
                                                           T *__restrict__ out, T *__restrict__ spare)
{
    const int *const labels = LABELS ? label_map : nullptr;
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using R = Rows<T, HD>;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * (HD + 4)];
    __shared__ __align__(16) T Vt[HD * 68];
    __shared__ Spots spots[3];
    __shared__ int odd_s[3];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16;
    const Walk walk = walk_of(a.heads);
    const int C = a.heads * a.hd;
    const unsigned stride = 3u * C;
    const T *base = qkv + (size_t)walk.head * a.hd;
    const int per = Slots<NB>::per_tile(a.n);
    const long long tiles = (a.windows + per - 1) / per;
    if (walk.tile >= tiles) return;
    const int kb0 = wave / NB * NB;  // the first key block of this wave's unit
    const int q = wave * 16 + i;
    const bool gaps = NB > 1 && a.n < 16 * NB;  // slots without a token beside a window's
    f32x4 bias[NB];
    const float scale2 = a.scale * kLog2e;
    const Spotter<NB> spotter(a);
    const bool first_wave = threadIdx.x < 64;
    if (first_wave) {
        spotter.write(spots[0], spotter.look(a, labels, walk.tile * per));
        spotter.write(spots[1], spotter.look(a, labels, (walk.tile + walk.step) * per));
        spotter.write_corners(a, spots[2]);  // (tokens are written there in the first tile, behind its barriers)
    }
    if (threadIdx.x < 3) odd_s[threadIdx.x] = 0;
    __syncthreads();
    pair_biases<NB>(bias, a, spots[2], table, walk.head, q, kb0 * 16 + 4 * g);
    R kr, vr;
    Frag qn[CB];
    unsigned none = 0;
    auto fetch = [&](const Spots &at) {
        int token[R::kPieces];
        tokens_at<T, HD>(at, token);
        kr.load(base + C, stride, token, a.hd);
        vr.load(base + 2 * C, stride, token, a.hd);
        none = R::none_of(token, a.hd);
#pragma unroll
        for (int c = 0; c < CB; ++c) qn[c] = raw4<T>(base, stride, at.source[q], c * 16 + 4 * g, a.hd);
    };
    fetch(spots[0]);
    kr.arrive();  // (so that within the loop the number of loads and stores behind a load is known)
    vr.arrive();
#pragma unroll
    for (int c = 0; c < CB; ++c) settle(qn[c]);
    int now = 0;  // of three spots: this tile's, the next one's, and the one being looked up
    for (long long tile = walk.tile; tile < tiles; tile += walk.step) {
        const int next = now == 2 ? 0 : now + 1, after = next == 2 ? 0 : next + 1;
        __syncthreads();  // the tile before has been used
        kr.clear(none);
        vr.clear(none);
        kr.store_rows(Ks);
        vr.store_columns(Vt);
        if constexpr (NB == 1) {
            if (not_finite(vr)) odd_s[now] = 1;
        }
        const Spots &at = spots[now];
        Frag qf[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) qf[c] = cleared<T>(qn[c], at.source[q] >= 0 && c * 16 + 4 * g < a.hd);
        __syncthreads();
        const bool mixed = at.mixed;
        if (NB == 1 && threadIdx.x == 0) odd_s[next] = 0;  // (its last readers were two tiles ago)
        Place coming;
        if (first_wave) coming = spotter.look(a, labels, (tile + 2 * walk.step) * per);
        fetch(spots[next]);  // (behind the last tile: the first token's)
        f32x4 s[NB];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const f32x4 acc = over_channels<T, HD>(Ks, (kb0 + j) * 16, qf);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = acc[r] * scale2 + bias[j][r];
                if (NB == 1 && bias[j][r] == -INFINITY) s[j][r] = -INFINITY;  // (of another window: whatever it is)
            }
        }
        if (gaps || mixed) {
            if (gaps) {  // empty slots: 0 times an infinity is NaN
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[j][r] = bias[j][r] == -INFINITY ? -INFINITY : s[j][r];
            }
            if (mixed) mask_slots<NB>(s, at, q, kb0 * 16 + 4 * g, a.outside2);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[j][r]);
        top = fold_max(top);
        if (top == -INFINITY) top = 0.f;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(s[j][r] - top);
                sum += s[j][r];
            }
        sum = fold_sum(sum);
        const float inv = sum > 0.f || sum != sum ? 1.0f / kDown<T> / sum : 0.f;
        Frag p[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) p[j] = M::frag(s[j] * inv);  // 16 bit: rounded once, as the product takes it
        f32x4 o[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) o[c] = f32x4{};
        over_unit<T, HD, NB>(o, Vt, kb0 * 16, p, NB == 1 && odd_s[now], a.n);
        const int mine = at.token[q];
        const bool padding = LABELS && at.source[q] < 0;  // (0 whatever its window holds: 0 times an infinity is NaN)
#pragma unroll
        for (int c = 0; c < CB; ++c)
            *(Frag *)store_at(out + (unsigned long long)(unsigned)mine * (unsigned)C + walk.head * a.hd + c * 16 + 4 * g, spare,
                              mine >= 0 && c * 16 + 4 * g < a.hd) = cleared<T>(M::frag(o[c] * kDown<T>), !padding);
        if (first_wave) spotter.write(spots[after], coming);
        now = next;
    }
}

// Where (key, query of its unit) lies in an LDS tile of 64 keys: rows of 4 NB quads of queries, without gaps, the quads
// permuted within a row so that neither the writes (one query of four groups of keys) nor the reads (a quad of 16 keys) meet in
// a bank.
template <int NB>
__device__ __forceinline__ int pair_at(int key, int query)
{
    return key * 16 * NB + ((query / 4) ^ (key / (4 / NB) % (4 * NB))) * 4 + query % 4;
}

// Backward pass of a tile.  Wave w first has the queries of block w: P^T and dP^T as in the forward pass, the row sums
// delta = sum P dP, dS^T = P^T (dP^T - delta), dQ^T = K^T dS^T.  P and dS go through LDS once; then wave w
// has the keys of block w: dV^T = dO^T P and dK^T = Q^T dS, contracted over the queries of its unit.  The sum
// of dS over the workgroup's windows, from which the table's gradient follows, stays in registers.
template <class T, int HD, int NB, bool LABELS>
__global__ __launch_bounds__(kAttnThreads, (kWaves<T, HD>)) void window_bwd(const WindowArgs a, const T *__restrict__ qkv,
                                                           const float *__restrict__ table, const int *__restrict__ label_map,
                                                           const T *__restrict__ dout, T *__restrict__ dqkv,
                                                           float *__restrict__ pairs, T *__restrict__ spare)
{
    const int *const labels = LABELS ? label_map : nullptr;
    using M = Mma<T>;
    using Frag = typename M::Frag;
    using R = Rows<T, HD>;
    constexpr int CB = HD / 16;
    constexpr int ROWS = 64 * (HD + 4), COLUMNS = HD * 68, PAIRS = 64 * 16 * NB;
    // K by rows and (128 fp32 channels: no room) by columns, V by rows; then, in their place, P and dS by keys.  Q and dO by
    // columns.  (32 fp32 channels: 52 KB, three workgroups on a CU.)
    constexpr bool K_BY_ROWS = HD * sizeof(T) > 256;
    constexpr int KV = 2 * ROWS + (K_BY_ROWS ? 0 : COLUMNS);
    __shared__ __align__(16) T Ks[KV > 2 * PAIRS ? KV : 2 * PAIRS];
    __shared__ __align__(16) T Qt[COLUMNS];
    __shared__ __align__(16) T Gt[COLUMNS];
    T *const Vs = Ks + ROWS, *const Kt = Vs + ROWS, *const Ps = Ks, *const Ss = Ks + PAIRS;
    __shared__ Spots spots[3];
    __shared__ int odd_s[3];
    constexpr bool SCALED = kLift<T> != 0;
    __shared__ __align__(16) float back_s[SCALED ? 64 : 4];  // by query: what undoes the scale of its dS
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16;
    const Walk walk = walk_of(a.heads);
    const int C = a.heads * a.hd;
    const unsigned stride = 3u * C;
    const T *base = qkv + (size_t)walk.head * a.hd, *gbase = dout + (size_t)walk.head * a.hd;
    T *dbase = dqkv + (size_t)walk.head * a.hd;
    const int per = Slots<NB>::per_tile(a.n);
    const long long tiles = (a.windows + per - 1) / per;
    const int kb0 = wave / NB * NB;
    const int q = wave * 16 + i;
    const bool gaps = NB > 1 && a.n < 16 * NB;  // slots without a token beside a window's
    f32x4 bias[NB], dbias[NB];
    const float scale2 = a.scale * kLog2e;
    const Spotter<NB> spotter(a);
    const bool first_wave = threadIdx.x < 64;
    if (first_wave) {
        spotter.write(spots[0], spotter.look(a, labels, walk.tile * per));
        spotter.write(spots[1], spotter.look(a, labels, (walk.tile + walk.step) * per));
        spotter.write_corners(a, spots[2]);
    }
    if (threadIdx.x < 3) odd_s[threadIdx.x] = 0;
    __syncthreads();
    pair_biases<NB>(bias, a, spots[2], table, walk.head, q, kb0 * 16 + 4 * g);
#pragma unroll
    for (int j = 0; j < NB; ++j) dbias[j] = f32x4{};
    R qr_, kr, vr, gr;
    unsigned none = 0;
    auto fetch = [&](const Spots &at) {
        int token[R::kPieces];
        tokens_at<T, HD>(at, token);
        qr_.load(base, stride, token, a.hd);
        kr.load(base + C, stride, token, a.hd);
        vr.load(base + 2 * C, stride, token, a.hd);
        gr.load(gbase, C, token, a.hd);
        none = R::none_of(token, a.hd);
    };
    fetch(spots[0]);
    qr_.arrive();
    kr.arrive();
    vr.arrive();
    gr.arrive();
    int now = 0;
    for (long long tile = walk.tile; tile < tiles; tile += walk.step) {
        const int next = now == 2 ? 0 : now + 1, after = next == 2 ? 0 : next + 1;
        __syncthreads();
        qr_.clear(none);
        kr.clear(none);
        vr.clear(none);
        gr.clear(none);
        qr_.store_columns(Qt);
        kr.store_rows(Ks);
        if constexpr (!K_BY_ROWS) kr.store_columns(Kt);
        vr.store_rows(Vs);
        gr.store_columns(Gt);
        if constexpr (NB == 1) {
            if (not_finite(qr_) || not_finite(kr) || not_finite(vr) || not_finite(gr)) odd_s[now] = 1;
        }
        __syncthreads();
        const Spots &at = spots[now];
        const bool mixed = at.mixed, odd = NB == 1 && odd_s[now];
        if (NB == 1 && threadIdx.x == 0) odd_s[next] = 0;  // (its last readers were two tiles ago)
        Place coming;
        if (first_wave) coming = spotter.look(a, labels, (tile + 2 * walk.step) * per);
        fetch(spots[next]);  // (behind the last tile: the first token's)
        Frag qf[CB], gf[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                qf[c][r] = Qt[(c * 16 + 4 * g + r) * 68 + q];
                gf[c][r] = Gt[(c * 16 + 4 * g + r) * 68 + q];
            }
        f32x4 s[NB], dp[NB];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const f32x4 acc = over_channels<T, HD>(Ks, (kb0 + j) * 16, qf);
            dp[j] = over_channels<T, HD>(Vs, (kb0 + j) * 16, gf);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = acc[r] * scale2 + bias[j][r];
                if (NB == 1 && bias[j][r] == -INFINITY) s[j][r] = -INFINITY, dp[j][r] = 0.f;
            }
        }
        if (gaps || mixed) {
            if (gaps) {  // empty slots: 0 times an infinity is NaN
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[j][r] = bias[j][r] == -INFINITY ? -INFINITY : s[j][r];
            }
            if (mixed) {
                mask_slots<NB>(s, at, q, kb0 * 16 + 4 * g, a.outside2);
                if (LABELS && at.source[q] < 0) {  // (as a query: its P is 0, and 0 times an infinity is NaN)
#pragma unroll
                    for (int j = 0; j < NB; ++j) dp[j] = f32x4{};
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[j][r]);
        top = fold_max(top);
        if (top == -INFINITY) top = 0.f;
        float sum = 0.f, delta = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(s[j][r] - top);
                sum += s[j][r];
                delta += s[j][r] * dp[j][r];
            }
        sum = fold_sum(sum);
        const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        delta = fold_sum(delta) * inv;
        Frag ds[NB], p[NB];
        f32x4 d[NB];  // (times 2^kLift)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            f32x4 pv = s[j] * (inv * (1.0f / kDown<T>));
            d[j] = pv * (dp[j] - delta);
            if constexpr (NB == 1) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (bias[j][r] == -INFINITY) pv[r] = d[j][r] = 0.f;
            }
            dbias[j] += d[j];
            p[j] = M::frag(pv);
        }
        float to_dq = a.scale * kDown<T>;
        if constexpr (SCALED) {
            const float up = column_scale(largest(d));
#pragma unroll
            for (int j = 0; j < NB; ++j) d[j] *= up;
            if (g == 0) back_s[q] = 1.0f / up;
            to_dq /= up;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) ds[j] = M::frag(d[j]);  // 16 bit: rounded once, as the products take it; the table's
                                                             // gradient sums it unrounded
        f32x4 acc[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[c] = f32x4{};
        over_unit<T, HD, NB, K_BY_ROWS>(acc, K_BY_ROWS ? Ks : Kt, kb0 * 16, ds, odd, a.n);
        const int mine = at.token[q];
        const bool padding = LABELS && at.source[q] < 0;
#pragma unroll
        for (int c = 0; c < CB; ++c)
            *(Frag *)store_at(dbase + (unsigned long long)(unsigned)mine * stride + c * 16 + 4 * g, spare, mine >= 0 && c * 16 + 4 * g < a.hd) =
                cleared<T>(M::frag(acc[c] * to_dq), !padding);
        __syncthreads();  // K and V have been used
        const int ql_ = wave % NB * 16 + i;  // this lane's query within its unit
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            settle(p[j]);  // (the rounded values, not their rounding once more)
            settle(ds[j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = pair_at<NB>((kb0 + j) * 16 + 4 * g + r, ql_);
                Ps[at] = p[j][r];
                Ss[at] = ds[j][r];
            }
        }
        __syncthreads();
        // now slot q is this lane's key
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int at = pair_at<NB>(q, j * 16 + 4 * g);
            p[j] = row4<T>(&Ps[at]);
            ds[j] = row4<T>(&Ss[at]);
        }
        float to_dk = a.scale * kDown<T>;
        if constexpr (SCALED) {  // from the queries' scales to this key's: exact but for what is 2^-29 of its largest
            f32x4 v[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const f32x4 back = *(const f32x4 *)&back_s[kb0 * 16 + j * 16 + 4 * g];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[j][r] = (float)ds[j][r] * back[r];
            }
            const float up = column_scale(largest(v));
            to_dk /= up;
#pragma unroll
            for (int j = 0; j < NB; ++j) ds[j] = M::frag(v[j] * up);
        }
        f32x4 dv[CB];
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[c] = dv[c] = f32x4{};
        over_unit<T, HD, NB>(dv, Gt, kb0 * 16, p, odd, a.n);
        over_unit<T, HD, NB>(acc, Qt, kb0 * 16, ds, odd, a.n);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            T *to = dbase + (unsigned long long)(unsigned)mine * stride + c * 16 + 4 * g;
            const bool wanted = mine >= 0 && c * 16 + 4 * g < a.hd;
            *(Frag *)store_at(to + C, spare, wanted) = cleared<T>(M::frag(acc[c] * to_dk), !padding);
            *(Frag *)store_at(to + 2 * C, spare, wanted) = cleared<T>(M::frag(dv[c] * kDown<T>), !padding);
        }
        if (first_wave) spotter.write(spots[after], coming);
        now = next;
    }
    if (!pairs) return;
    float *to = pairs + (size_t)blockIdx.x * 64 * 16 * NB;
#pragma unroll
    for (int j = 0; j < NB; ++j) *(f32x4 *)&to[q * 16 * NB + j * 16 + 4 * g] = dbias[j] * kDown<T>;
}

// ================================================================================================
// Longer windows (65 .. 4096 tokens): tiles of 64 queries against tiles of 64 keys, with the running maximum and sum
// of a softmax over the key tiles.  A head's scores take about eleven vector instructions for each pair beside its
// products (scale and bias, maximum, exponential, sum, rounding), against 4 hd / 1024 matrix instructions: with the
// model's 32 channels the vector units are busy for half of the forward pass (a third to two fifths of dQ, dK and dV, a quarter of
// the table's gradient), the matrix units for a tenth, and waves wait a third of their time, at the two barriers of a
// tile above all.  So the pair loop holds nothing else --
//  * where tokens lie and what region they are of is written once for each call (`places`, `tiles`): a pair of
//    tiles of one region needs no mask, one of two regions that never meet is skipped with its loads;
//  * the bias comes from a copy of the table with one head's entries in a row, forwards and backwards, so that four
//    neighbouring keys (or queries) have neighbouring entries: a pair of tiles needs one run of it, which goes through LDS,
//    where rows of the window are multiples of 4;
//  * the next tile's rows are in flight while this one is used, and what is contracted over tokens lies in LDS
//    transposed, so that an operand is one read.
// ================================================================================================

struct PlaceAt {
    int token, corner, label, wrap;  // token -1: none (behind the window's end); label < 0: padding
};
struct TileAt {
    int state, label, wrap;  // kEven: live tokens of one region; kPadded: of one region beside padding; kDead: no live
    int corner;              // token; kMixed: of several regions.  corner: of the tile's first token
};
constexpr int kMixed = 0, kEven = 1, kPadded = 2, kDead = 3;

struct LongMap {
    const PlaceAt *places;   // (windows, tiles * 64)
    const int *live;         // the same: the token, -1 for none and for padding
    const TileAt *tiles_at;  // (windows, tiles)
    const float *bias;       // (heads, entries) * log2 e, or NULL
    const float *rev;        // the same, every head's entries in reverse
    int tiles;               // of 64 tokens in a window, at most 64
};

// Few workgroups: `splits` of them share a tile's partners, and their sums are joined by a second kernel.
struct Split {
    int splits;
    float *a, *b;  // [split][window, head, tile, 64][head_dim]: sums of the products over tokens
    float *rows;   // [split][window, head, tile, 64][2]: forward: maximum and sum of the softmax; dQ: near and rest
};

struct LongTile {
    long long window;
    int head, tile;
};
// Workgroups 8 apart run on one XCD: each XCD takes a run of neighbouring tiles, head by head, so that its cache holds few
// heads' rows and biases, and so that tiles with more to do than others (the last row of every plane padding, say) do not
// all fall to one XCD, as they do where tile t goes to XCD t % 8.
__device__ __forceinline__ LongTile long_tile(const WindowArgs &a, int tiles)
{
    const unsigned x = blockIdx.x % 8, each = gridDim.x / 8, more = gridDim.x % 8;
    const unsigned id = x * each + (x < more ? x : more) + blockIdx.x / 8;
    const unsigned t = id % (unsigned)tiles, r = id / (unsigned)tiles;
    return {(long long)(r / (unsigned)a.heads), (int)(r % (unsigned)a.heads), (int)t};
}

// Whether tokens `x` meet tile `y` at all, and whether they need a mask.  Padding among x needs none: its row is cleared
// at the end; PADDING_OK: padding among y neither (queries: their lse is infinite, their P 0).
template <bool PADDING_OK>
__device__ __forceinline__ void relation(const TileAt &x, const TileAt &y, float outside2, bool &any, bool &mixed)
{
    const bool single = x.state != kMixed && y.state != kMixed;
    const bool same = x.label == y.label && x.wrap == y.wrap;
    any = x.state != kDead && y.state != kDead && !(single && !same && outside2 == -INFINITY);
    mixed = any && !(single && same && (PADDING_OK || y.state == kEven));
}

// what the lanes of a wave hold: a token each
__device__ __forceinline__ TileAt tile_of(const PlaceAt &p, int corner)
{
    const unsigned long long live = __ballot(p.label >= 0);
    const int first = live ? __builtin_ctzll(live) : 0;
    const int label = __shfl(p.label, first), wrap = __shfl(p.wrap, first);
    const bool one = __all(p.label < 0 || (p.label == label && p.wrap == wrap));
    return {live == 0 ? kDead : !one ? kMixed : live == ~0ull ? kEven : kPadded, label, wrap, corner};
}

// Which tiles a wave's 16 tokens meet, one bit each (every lane looks at one tile); the workgroup goes through those that any
// of its waves meets, or every splits-th of them.
struct Meets {
    unsigned long long todo, any, mixed, masks;  // masks: `mixed` of any wave
    unsigned long long gaps;                     // tiles that may hold padding, or a window's end
    int corner;  // this lane's tile's first token's
};
template <bool PADDING_OK>
__device__ __forceinline__ Meets meets(const LongMap &m, long long window, const PlaceAt &own, float outside2, int splits)
{
    constexpr int W = kAttnThreads / 64;
    __shared__ unsigned long long bits[2 * W];
    const int lane = threadIdx.x % 64;
    TileAt other{kDead, 0, 0, 0};
    if (lane < m.tiles) other = m.tiles_at[window * m.tiles + lane];
    bool any, mixed;
    relation<PADDING_OK>(tile_of(own, 0), other, outside2, any, mixed);
    const unsigned long long mine = __ballot(any), masked = __ballot(mixed);
    if (lane == 0) bits[threadIdx.x / 64] = mine, bits[W + threadIdx.x / 64] = masked;
    __syncthreads();
    unsigned long long all = 0, masks = 0;
#pragma unroll
    for (int k = 0; k < W; ++k) all |= bits[k], masks |= bits[W + k];
    if (splits > 1) all = __ballot((all >> lane & 1) && __popcll(all & ((1ull << lane) - 1)) % splits == (int)blockIdx.y);
    return {all, mine, masked, masks, __ballot(other.state != kEven), other.corner};
}

// The bias of a tile's pairs.
// EVEN (64 tokens tile the window, its rows are multiples of 4, and two tiles' distances span at most kSpan entries): the
// entries of a pair of tiles are one run of the row, which the workgroup copies to LDS, a tile ahead; a lane's four lie
// behind each other there.  (Loading them from the row itself is 16 bytes a lane at any alignment, and was a third of all
// the work of the address units.)
// Else: each by itself, from a copy of the head's whole row in LDS where it has at most TABLE entries.  (From the row itself
// a tile's sixteen loads wait for the next tile's rows, which were asked for before: 7872 tiles of windows of 72 tokens, 64 channels
// in fp16, take 99 us forward, 89 with the copy.  With 128 channels the registers for both forms leave one wave less on a SIMD:
// 189 us instead of 160.)
constexpr int kSpan = 512;
template <int HD>
constexpr int kTable = HD <= 64 ? 2048 : 0;
template <bool EVEN, int TABLE>
struct Biases {
    f32x4 now[4];
    float ahead[2];
    int at[4], start;
    const float *row;  // this head's entries
    bool copied;       // into LDS, all of them
    // `sign`: an entry's place grows with +-corner(own); `own`, `partner`: corners of this lane's token and of the first tile's
    __device__ __forceinline__ Biases(const float *head_row, const WindowArgs &a, int own, int own_tile, const PlaceAt *first_tile)
        : row(head_row), copied(!EVEN && TABLE > 0 && a.entries <= TABLE)
    {
        const int g = threadIdx.x % 64 / 16;
        const int reach = EVEN ? first_tile[63].corner : 0;  // between the first and the last token of a tile
        start = middle(a) - own_tile - reach;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            now[j] = f32x4{};
            at[j] = EVEN ? reach - (own - own_tile) + first_tile[j * 16 + 4 * g].corner : middle(a) - own;
        }
    }
    // (there is a barrier between this and take())
    __device__ __forceinline__ void copy(const WindowArgs &a, float *to) const
    {
        if (TABLE == 0 || !row || !copied) return;
#pragma unroll 2
        for (int e = threadIdx.x; e < a.entries; e += kAttnThreads) to[e] = row[e];
    }
    __device__ __forceinline__ void fetch(const WindowArgs &a, int tile_corner)
    {
        if (!EVEN || !row) return;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            // (what lies outside the row is never used)
            ahead[k] = row[min(max(start + tile_corner + k * kAttnThreads + (int)threadIdx.x, 0), a.entries - 1)];
        }
    }
    __device__ __forceinline__ void store(float *run)
    {
        if (!EVEN || !row) return;
        run[threadIdx.x] = ahead[0];
        run[threadIdx.x + kAttnThreads] = ahead[1];
    }
    __device__ __forceinline__ void take(const float *run, const PlaceAt *tile)
    {
        if (!row) return;
        const int g = threadIdx.x % 64 / 16;
        if (EVEN || (TABLE > 0 && copied)) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) now[j][r] = run[at[j] + (EVEN ? r : tile[j * 16 + 4 * g + r].corner)];
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) now[j][r] = row[at[j] + tile[j * 16 + 4 * g + r].corner];
    }
};

// The scores of a tile in the exponent of 2: all products first (one after the other they would each be waited for), then
// one branch for the mask.
template <class T, int HD>
__device__ __forceinline__ void scores(f32x4 (&x)[4], const T *rows, const typename Mma<T>::Frag *own_row, float scale2,
                                       const f32x4 (&bias)[4], bool mixed, const PlaceAt &own, const PlaceAt *at, float outside2)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[j] = over_channels<T, HD>(rows, j * 16, own_row);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[j][r] = x[j][r] * scale2 + bias[j][r];
    }
    if (mixed) {
        const int g = threadIdx.x % 64 / 16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const PlaceAt &p = at[j * 16 + 4 * g + r];
                x[j][r] = masked(x[j][r], own.label, own.wrap, p.label, p.wrap, outside2);
            }
    }
}

// What a thread has in flight of the tiles to come: the rows of the next one, the tokens of the one after it.  Nothing here is
// loaded under a condition (see raw4).
template <class T, int HD>
struct Ahead {
    using R = Rows<T, HD>;
    R x, y;         // rows of two tensors
    unsigned none;  // of their pieces
    int token[R::kPieces];
    __device__ __forceinline__ void tokens(const int *live, int t)
    {
        settle(none);  // (the tokens before have become addresses and `none`)
#pragma unroll
        for (int m = 0; m < R::kPieces; ++m) token[m] = live[t * 64 + R::row(m)];
    }
    __device__ __forceinline__ void rows(const T *xb, long long xs, const T *yb, long long ys, int hd)
    {
        x.load(xb, xs, token, hd);
        y.load(yb, ys, token, hd);
        none = R::none_of(token, hd);
    }
    __device__ __forceinline__ void clear()
    {
        x.clear(none);
        y.clear(none);
    }
};

// Where the tokens of a tile lie and what they are, into LDS.  EVEN: wanted where there is a mask only, and loaded then.
template <bool EVEN>
struct TilePlaces {
    i32x4 ahead;
    __device__ __forceinline__ void fetch(const PlaceAt *tile)
    {
        if constexpr (!EVEN) ahead = *(const i32x4 *)(tile + threadIdx.x % 64);
    }
    __device__ __forceinline__ void store(PlaceAt *to, const PlaceAt *tile, bool wanted)
    {
        if constexpr (EVEN) {
            if (wanted && threadIdx.x < 64) to[threadIdx.x] = tile[threadIdx.x];
        } else if (threadIdx.x < 64) {
            *(i32x4 *)(to + threadIdx.x) = ahead;
        }
    }
};

// log2 of a row's sum of 2^x; +inf for an empty row, so that its P is 0 in the backward pass (a sum of NaN alone stays NaN)
template <class T>
__device__ __forceinline__ float lse_of(float top, float sum)
{
    return top == -INFINITY && sum == 0.f ? INFINITY : top + (log2f(sum) - kLift<T>);
}

template <class T, int HD, bool EVEN>
__global__ __launch_bounds__(kAttnThreads, (kWaves<T, HD>)) void long_fwd(const WindowArgs a, const LongMap map, const Split split,
                                                         const T *__restrict__ qkv, T *__restrict__ out,
                                                         float *__restrict__ lse)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * (HD + 4)];
    __shared__ __align__(16) T Vt[HD * 68];
    __shared__ __align__(16) PlaceAt at_s[64];
    __shared__ float bias_s[EVEN ? kSpan : kTable<HD> + 1];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, q = wave * 16 + i;
    const LongTile lt = long_tile(a, map.tiles);
    const int C = a.heads * a.hd;
    const unsigned stride = 3u * C;
    const T *base = qkv + (size_t)lt.head * a.hd;
    const PlaceAt *window = map.places + lt.window * map.tiles * 64;
    const PlaceAt own = window[lt.tile * 64 + q];
    const Meets meet = meets<false>(map, lt.window, own, a.outside2, split.splits);
    const int *live = map.live + lt.window * map.tiles * 64;
    unsigned long long todo = meet.todo, later = todo & (todo - 1);
    Ahead<T, HD> ahead;
    TilePlaces<EVEN> at;
    auto rows = [&](int t) {
        ahead.rows(base + C, stride, base + 2 * C, stride, a.hd);
        at.fetch(window + t * 64);
    };
    ahead.none = 0;
    ahead.tokens(live, todo ? __builtin_ctzll(todo) : 0);
    // entry of the reversed row: middle - corner(q) + corner(k)
    Biases<EVEN, kTable<HD>> bias(map.rev ? map.rev + (size_t)lt.head * a.entries : nullptr, a, own.corner,
                      window[lt.tile * 64].corner, window);
    bias.copy(a, bias_s);
    if (todo) {
        rows(__builtin_ctzll(todo));
        bias.fetch(a, __builtin_amdgcn_readlane(meet.corner, __builtin_ctzll(todo)));
        ahead.tokens(live, later ? __builtin_ctzll(later) : 0);
    }
    Frag qf[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) qf[c] = load4<T>(base, stride, own.label < 0 ? -1 : own.token, c * 16 + 4 * g, a.hd);
    const float scale2 = a.scale * kLog2e;
    float top = -INFINITY, sum = 0.f;
    f32x4 o[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) o[c] = f32x4{};
    while (todo) {
        const int now = __builtin_ctzll(todo);
        const bool mixed = meet.mixed >> now & 1, any = meet.any >> now & 1;
        todo = later;
        later &= later - 1;
        __syncthreads();  // the tile before has been used
        ahead.clear();
        ahead.x.store_rows(Ks);
        ahead.y.store_columns(Vt);
        at.store(at_s, window + now * 64, meet.masks >> now & 1);
        bias.store(bias_s);
        __syncthreads();
        if (todo) {
            rows(__builtin_ctzll(todo));
            bias.fetch(a, __builtin_amdgcn_readlane(meet.corner, __builtin_ctzll(todo)));
            ahead.tokens(live, later ? __builtin_ctzll(later) : 0);
        }
        if (!any) continue;  // (the barriers are at the loop's head)
        bias.take(bias_s, at_s);
        f32x4 s[4];
        float high = top;
        scores<T, HD>(s, Ks, qf, scale2, bias.now, mixed, own, at_s, a.outside2);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) high = fmaxf(high, s[j][r]);
        high = fold_max(high);
        const float base2 = high == -INFINITY ? 0.f : high;
        const float fade = __builtin_amdgcn_exp2f(top - base2);
        top = high;
        float part = 0.f;
        Frag p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(s[j][r] - (base2 - kLift<T>));
                part += s[j][r];
            }
            p[j] = M::frag(s[j]);  // 16 bit: rounded as the product takes it, the sum is of the unrounded ones
        }
        sum = sum * fade + part;
#pragma unroll
        for (int c = 0; c < CB; ++c) o[c] *= fade;
        over_tokens<T, HD>(o, Vt, 0, p);
    }
    sum = fold_sum(sum);
    if (own.label < 0) {  // padding: an empty row
        top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int c = 0; c < CB; ++c) o[c] = f32x4{};
    }
    const size_t padded = (((size_t)lt.window * a.heads + lt.head) * map.tiles + lt.tile) * 64 + q;
    if (split.splits > 1) {
        const size_t line = (size_t)blockIdx.y * gridDim.x * 64 + padded;
#pragma unroll
        for (int c = 0; c < CB; ++c)
            if (c * 16 + 4 * g < a.hd) *(f32x4 *)(split.a + line * a.hd + c * 16 + 4 * g) = o[c];
        if (g == 0) split.rows[line * 2] = top, split.rows[line * 2 + 1] = sum;
        return;
    }
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    if (own.token < 0) return;
#pragma unroll
    for (int c = 0; c < CB; ++c)
        if (c * 16 + 4 * g < a.hd)
            *(Frag *)(out + (size_t)own.token * C + lt.head * a.hd + c * 16 + 4 * g) = M::frag(o[c] * inv);
    if (lse && g == 0) lse[padded] = lse_of<T>(top, sum);
}

// Joins the shares of a forward pass: hd / 4 threads for a query, each with four channels
template <class T>
__global__ __launch_bounds__(kAttnThreads) void long_fwd_join(const WindowArgs a, const LongMap map, const Split split,
                                                              T *__restrict__ out, float *__restrict__ lse)
{
    const size_t lines = (size_t)a.windows * a.heads * map.tiles * 64;
    const unsigned per = (unsigned)a.hd / 4;
    const size_t id = (size_t)blockIdx.x * kAttnThreads + threadIdx.x, line = id / per;
    const int c = (int)(id % per) * 4;
    if (line >= lines) return;
    const size_t r = line / ((size_t)map.tiles * 64);
    const int head = (int)(r % (size_t)a.heads);
    const PlaceAt own = map.places[r / (size_t)a.heads * (size_t)map.tiles * 64 + line % ((size_t)map.tiles * 64)];
    if (own.token < 0) return;
    float top = -INFINITY;
    for (int k = 0; k < split.splits; ++k) top = fmaxf(top, split.rows[(k * lines + line) * 2]);
    const float base2 = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o{};
    for (int k = 0; k < split.splits; ++k) {
        const float fade = __builtin_amdgcn_exp2f(split.rows[(k * lines + line) * 2] - base2);
        sum += split.rows[(k * lines + line) * 2 + 1] * fade;
        o += *(const f32x4 *)(split.a + (k * lines + line) * a.hd + c) * fade;
    }
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    *(typename Mma<T>::Frag *)(out + (size_t)own.token * a.heads * a.hd + head * a.hd + c) = Mma<T>::frag(o * inv);
    if (lse && c == 0) lse[line] = lse_of<T>(top, sum);
}

// dQ, and delta = sum over keys of P dP for each query.  delta is also the product of out and dout; in 16 bits `out` is
// rounded, so that product c is only near: off by about half a step of |out| |dout|.  Where keys and values have a mean, as
// behind a projection with a bias, that times sum P K is as large as dQ itself (4 deviations, 4096 tokens, bf16: dQ off by as much
// as its size).  So dS = P (dP - c) is what the product with K takes, rest = sum P (dP - c), summed in fp32, gives
// delta = c + rest, which the table's gradient and dK are computed with, and
//     dQ = sum dS K - rest sum P K,
// in which the rounding of P counts only for what c was off by.  In fp32 c is as near as any sum here: no second product.
template <class T, int HD, bool EVEN>
__global__ __launch_bounds__(kAttnThreads, (kWaves<T, HD>)) void long_bwd_q(const WindowArgs a, const LongMap map, const Split split,
                                                           const T *__restrict__ qkv, const T *__restrict__ out,
                                                           const float *__restrict__ lse, const T *__restrict__ dout,
                                                           T *__restrict__ dqkv, float *__restrict__ delta)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * (HD + 4)];
    __shared__ __align__(16) T Kt[HD * 68];
    __shared__ __align__(16) T Vs[64 * (HD + 4)];
    __shared__ __align__(16) PlaceAt at_s[64];
    __shared__ float bias_s[EVEN ? kSpan : kTable<HD> + 1];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, q = wave * 16 + i;
    const LongTile lt = long_tile(a, map.tiles);
    const int C = a.heads * a.hd;
    const unsigned stride = 3u * C;
    const T *base = qkv + (size_t)lt.head * a.hd;
    const PlaceAt *window = map.places + lt.window * map.tiles * 64;
    const PlaceAt own = window[lt.tile * 64 + q];
    const Meets meet = meets<false>(map, lt.window, own, a.outside2, split.splits);
    const int *live = map.live + lt.window * map.tiles * 64;
    unsigned long long todo = meet.todo, later = todo & (todo - 1);
    Ahead<T, HD> ahead;
    TilePlaces<EVEN> at;
    auto rows = [&](int t) {
        ahead.rows(base + C, stride, base + 2 * C, stride, a.hd);
        at.fetch(window + t * 64);
    };
    ahead.none = 0;
    ahead.tokens(live, todo ? __builtin_ctzll(todo) : 0);
    const int mine = own.label < 0 ? -1 : own.token;
    Biases<EVEN, kTable<HD>> bias(map.rev ? map.rev + (size_t)lt.head * a.entries : nullptr, a, own.corner,
                      window[lt.tile * 64].corner, window);
    bias.copy(a, bias_s);
    if (todo) {
        rows(__builtin_ctzll(todo));
        bias.fetch(a, __builtin_amdgcn_readlane(meet.corner, __builtin_ctzll(todo)));
        ahead.tokens(live, later ? __builtin_ctzll(later) : 0);
    }
    Frag qf[CB], gf[CB];
    float near = 0.f;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        qf[c] = load4<T>(base, stride, mine, c * 16 + 4 * g, a.hd);
        gf[c] = load4<T>(dout + (size_t)lt.head * a.hd, C, mine, c * 16 + 4 * g, a.hd);
        const Frag of = load4<T>(out + (size_t)lt.head * a.hd, C, mine, c * 16 + 4 * g, a.hd);
#pragma unroll
        for (int r = 0; r < 4; ++r) near += (float)of[r] * (float)gf[c][r];
    }
    near = fold_sum(near);
    const size_t padded = (((size_t)lt.window * a.heads + lt.head) * map.tiles + lt.tile) * 64 + q;
    const float shift = own.token >= 0 ? lse[padded] : INFINITY;
    const float scale2 = a.scale * kLog2e;
    float rest = 0.f;
    RunningScale fit;
    f32x4 dq[CB], pk[CB];  // pk: sum P K
#pragma unroll
    for (int c = 0; c < CB; ++c) dq[c] = pk[c] = f32x4{};
    while (todo) {
        const int now = __builtin_ctzll(todo);
        const bool mixed = meet.mixed >> now & 1, any = meet.any >> now & 1;
        todo = later;
        later &= later - 1;
        __syncthreads();
        ahead.clear();
        ahead.x.store_rows(Ks);
        ahead.x.store_columns(Kt);
        ahead.y.store_rows(Vs);
        at.store(at_s, window + now * 64, meet.masks >> now & 1);
        bias.store(bias_s);
        __syncthreads();
        if (todo) {
            rows(__builtin_ctzll(todo));
            bias.fetch(a, __builtin_amdgcn_readlane(meet.corner, __builtin_ctzll(todo)));
            ahead.tokens(live, later ? __builtin_ctzll(later) : 0);
        }
        if (!any) continue;  // (the barriers are at the loop's head)
        bias.take(bias_s, at_s);
        Frag ds[4], pf[4];
        f32x4 x[4], dp[4], d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[j] = over_channels<T, HD>(Vs, j * 16, gf);
        scores<T, HD>(x, Ks, qf, scale2, bias.now, mixed, own, at_s, a.outside2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 p;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // (an empty row: -inf against +inf)
                p[r] = __builtin_amdgcn_exp2f(x[j][r] - shift);
                d[j][r] = p[r] * (dp[j][r] - near);
                rest += d[j][r];
            }
            if constexpr (sizeof(T) == 2) pf[j] = M::frag(p);
        }
        if constexpr (kLift<T> != 0) fit.apply(d, dq);
#pragma unroll
        for (int j = 0; j < 4; ++j) ds[j] = M::frag(d[j]);
        if constexpr (sizeof(T) == 2)
            over_tokens_both<T, HD>(dq, pk, Kt, ds, pf);
        else
            over_tokens<T, HD>(dq, Kt, 0, ds);
    }
    rest = fold_sum(rest);
    if constexpr (kLift<T> != 0) {
#pragma unroll
        for (int c = 0; c < CB; ++c) dq[c] *= 1.0f / fit.s;
    }
    if (own.label < 0) {
        near = rest = 0.f;
#pragma unroll
        for (int c = 0; c < CB; ++c) dq[c] = pk[c] = f32x4{};
    }
    if (split.splits > 1) {
        const size_t line = (size_t)blockIdx.y * gridDim.x * 64 + padded;
#pragma unroll
        for (int c = 0; c < CB; ++c)
            if (c * 16 + 4 * g < a.hd) {
                *(f32x4 *)(split.a + line * a.hd + c * 16 + 4 * g) = dq[c];
                if constexpr (sizeof(T) == 2) *(f32x4 *)(split.b + line * a.hd + c * 16 + 4 * g) = pk[c];
            }
        if (g == 0) split.rows[line * 2] = near, split.rows[line * 2 + 1] = rest;
        return;
    }
    if (own.token < 0) return;
    if (g == 0) delta[padded] = near + rest;
#pragma unroll
    for (int c = 0; c < CB; ++c)
        if (c * 16 + 4 * g < a.hd) {
            if constexpr (sizeof(T) == 2) dq[c] -= pk[c] * rest;
            *(Frag *)(dqkv + (size_t)own.token * stride + lt.head * a.hd + c * 16 + 4 * g) = M::frag(dq[c] * a.scale);
        }
}

// dK and dV: wave w has 16 keys and goes through the queries, S = Q K^T (rows: queries, lane: key), so that P and dS have the
// layout of the B operands of dV^T = dO^T P and dK^T = Q^T dS.
template <class T, int HD, bool EVEN>
__global__ __launch_bounds__(kAttnThreads, (kWaves<T, HD>)) void long_bwd_kv(const WindowArgs a, const LongMap map, const Split split,
                                                            const T *__restrict__ qkv, const float *__restrict__ lse,
                                                            const T *__restrict__ dout, T *__restrict__ dqkv,
                                                            const float *__restrict__ delta)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Qs[64 * (HD + 4)];
    __shared__ __align__(16) T Qt[HD * 68];
    __shared__ __align__(16) T Gs[64 * (HD + 4)];
    __shared__ __align__(16) T Gt[HD * 68];
    __shared__ __align__(16) PlaceAt at_s[64];
    __shared__ float bias_s[EVEN ? kSpan : kTable<HD> + 1];
    __shared__ __align__(16) float lse_s[64], delta_s[64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, k = wave * 16 + i;
    const LongTile lt = long_tile(a, map.tiles);
    const int C = a.heads * a.hd;
    const unsigned stride = 3u * C;
    const T *base = qkv + (size_t)lt.head * a.hd, *gbase = dout + (size_t)lt.head * a.hd;
    const PlaceAt *window = map.places + lt.window * map.tiles * 64;
    const size_t lines = ((size_t)lt.window * a.heads + lt.head) * map.tiles * 64;
    const PlaceAt own = window[lt.tile * 64 + k];
    const Meets meet = meets<true>(map, lt.window, own, a.outside2, split.splits);
    const int *live = map.live + lt.window * map.tiles * 64;
    unsigned long long todo = meet.todo, later = todo & (todo - 1);
    Ahead<T, HD> ahead;
    TilePlaces<EVEN> at;
    float shift = 0.f, del = 0.f;
    int some = -1;  // (lse and delta of no token were never written)
    auto rows = [&](int t) {
        ahead.rows(base, stride, gbase, C, a.hd);
        at.fetch(window + t * 64);
        some = live[t * 64 + threadIdx.x % 64];
        shift = lse[lines + t * 64 + threadIdx.x % 64];
        del = delta[lines + t * 64 + threadIdx.x % 64];
    };
    ahead.none = 0;
    ahead.tokens(live, todo ? __builtin_ctzll(todo) : 0);
    const int mine = own.label < 0 ? -1 : own.token;
    // entry: corner(q) + middle - corner(k)
    Biases<EVEN, kTable<HD>> bias(map.bias ? map.bias + (size_t)lt.head * a.entries : nullptr, a, own.corner,
                      window[lt.tile * 64].corner, window);
    bias.copy(a, bias_s);
    if (todo) {
        rows(__builtin_ctzll(todo));
        bias.fetch(a, __builtin_amdgcn_readlane(meet.corner, __builtin_ctzll(todo)));
        ahead.tokens(live, later ? __builtin_ctzll(later) : 0);
    }
    Frag kf[CB], vf[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) {
        kf[c] = load4<T>(base + C, stride, mine, c * 16 + 4 * g, a.hd);
        vf[c] = load4<T>(base + 2 * C, stride, mine, c * 16 + 4 * g, a.hd);
    }
    // Where there is no query its row is zeros, and 0 times an infinity of a key is NaN: where there are such keys, tiles with such
    // rows are masked too.  (An infinity of V needs nothing: all that it meets in dK is NaN by itself.)
    float zero = 0.f;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) zero += (float)kf[c][r] * 0.f;
    const unsigned long long gaps = __syncthreads_or(zero != 0.f) ? meet.gaps : 0;
    const float scale2 = a.scale * kLog2e;
    RunningScale fit;
    f32x4 dk[CB], dv[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) dk[c] = dv[c] = f32x4{};
    while (todo) {
        const int now = __builtin_ctzll(todo);
        const bool mixed = (meet.mixed | gaps) >> now & 1, any = meet.any >> now & 1;
        todo = later;
        later &= later - 1;
        __syncthreads();
        ahead.clear();
        ahead.x.store_rows(Qs);
        ahead.x.store_columns(Qt);
        ahead.y.store_rows(Gs);
        ahead.y.store_columns(Gt);
        at.store(at_s, window + now * 64, (meet.masks | gaps) >> now & 1);
        if (threadIdx.x < 64) {
            lse_s[threadIdx.x] = some >= 0 ? shift - kLift<T> : INFINITY;
            delta_s[threadIdx.x] = some >= 0 ? del : 0.f;
        }
        bias.store(bias_s);
        __syncthreads();
        if (todo) {
            rows(__builtin_ctzll(todo));
            bias.fetch(a, __builtin_amdgcn_readlane(meet.corner, __builtin_ctzll(todo)));
            ahead.tokens(live, later ? __builtin_ctzll(later) : 0);
        }
        if (!any) continue;  // (the barriers are at the loop's head)
        bias.take(bias_s, at_s);
        Frag p[4], ds[4];
        f32x4 x[4], dp[4], d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[j] = over_channels<T, HD>(Gs, j * 16, vf);
        scores<T, HD>(x, Qs, kf, scale2, bias.now, mixed, own, at_s, a.outside2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 l = *(const f32x4 *)&lse_s[j * 16 + 4 * g], del4 = *(const f32x4 *)&delta_s[j * 16 + 4 * g];
            f32x4 pv;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pv[r] = __builtin_amdgcn_exp2f(x[j][r] - l[r]);
                d[j][r] = pv[r] * (dp[j][r] - del4[r]);
            }
            p[j] = M::frag(pv);
        }
        if constexpr (kLift<T> != 0) fit.apply(d, dk);
#pragma unroll
        for (int j = 0; j < 4; ++j) ds[j] = M::frag(d[j]);
        over_tokens<T, HD>(dv, Gt, 0, p);
        over_tokens<T, HD>(dk, Qt, 0, ds);
    }
    if constexpr (kLift<T> != 0) {
#pragma unroll
        for (int c = 0; c < CB; ++c) dk[c] *= kDown<T> / fit.s, dv[c] *= kDown<T>;
    }
    if (own.label < 0) {
#pragma unroll
        for (int c = 0; c < CB; ++c) dk[c] = dv[c] = f32x4{};
    }
    if (split.splits > 1) {
        const size_t line = (size_t)blockIdx.y * gridDim.x * 64 + lines + lt.tile * 64 + k;
#pragma unroll
        for (int c = 0; c < CB; ++c)
            if (c * 16 + 4 * g < a.hd) {
                *(f32x4 *)(split.a + line * a.hd + c * 16 + 4 * g) = dk[c];
                *(f32x4 *)(split.b + line * a.hd + c * 16 + 4 * g) = dv[c];
            }
        return;
    }
    if (own.token < 0) return;
#pragma unroll
    for (int c = 0; c < CB; ++c)
        if (c * 16 + 4 * g < a.hd) {
            T *to = dqkv + (size_t)own.token * stride + lt.head * a.hd + c * 16 + 4 * g;
            *(Frag *)(to + C) = M::frag(dk[c] * a.scale);
            *(Frag *)(to + 2 * C) = M::frag(dv[c]);
        }
}

// Joins the shares of a backward pass: hd / 4 threads for a token, each with four channels.  KV: dK and dV; else dQ and delta.
template <class T, bool KV>
__global__ __launch_bounds__(kAttnThreads) void long_bwd_join(const WindowArgs a, const LongMap map, const Split split,
                                                              T *__restrict__ dqkv, float *__restrict__ delta)
{
    const size_t lines = (size_t)a.windows * a.heads * map.tiles * 64;
    const unsigned per = (unsigned)a.hd / 4;
    const size_t id = (size_t)blockIdx.x * kAttnThreads + threadIdx.x, line = id / per;
    const int c = (int)(id % per) * 4;
    if (line >= lines) return;
    const size_t r = line / ((size_t)map.tiles * 64);
    const int head = (int)(r % (size_t)a.heads), C = a.heads * a.hd;
    const PlaceAt own = map.places[r / (size_t)a.heads * (size_t)map.tiles * 64 + line % ((size_t)map.tiles * 64)];
    if (own.token < 0) return;
    constexpr bool TAKE_BACK = !KV && sizeof(T) == 2;  // what delta was off by, times sum P K: see long_bwd_q
    f32x4 x{}, y{};
    float rest = 0.f;
    for (int k = 0; k < split.splits; ++k) {
        x += *(const f32x4 *)(split.a + (k * lines + line) * a.hd + c);
        if constexpr (KV || TAKE_BACK) y += *(const f32x4 *)(split.b + (k * lines + line) * a.hd + c);
        if constexpr (!KV) rest += split.rows[(k * lines + line) * 2 + 1];
    }
    if constexpr (TAKE_BACK) x -= y * rest;
    T *to = dqkv + (size_t)own.token * 3 * C + head * a.hd + c;
    *(typename Mma<T>::Frag *)(to + (KV ? C : 0)) = Mma<T>::frag(x * a.scale);
    if constexpr (KV)
        *(typename Mma<T>::Frag *)(to + 2 * C) = Mma<T>::frag(y);
    else if (c == 0)
        delta[line] = split.rows[line * 2] + rest;  // (`near` is the same in every share)
}

// The table's gradient sums dS over all pairs of one distance.  Where 64 tokens tile the window evenly (ed x eh x ew tokens,
// all three dividing the window's), the distances of a pair of tiles depend on the tiles' own distance alone: a
// workgroup takes one distance of tiles and one head, goes through all such pairs of tiles of its share of the windows, and
// adds their dS up in registers, where the bias is kept too.  64 x 64 sums for each distance of tiles are left.
// Windows that 64 tokens do not tile: a workgroup takes one pair of tiles in its share of the windows, and the sums are of n x n
// pairs.
struct PairWork {
    int gd, gh, gw;    // tiles along the axes; 0: not tiled evenly
    int chunks;        // shares of the windows
};
template <class T, int HD>
__global__ __launch_bounds__(kAttnThreads, (kWaves<T, HD>)) void long_bwd_pairs(const WindowArgs a, const LongMap map, const PairWork w,
                                                               const T *__restrict__ qkv, const float *__restrict__ lse,
                                                               const T *__restrict__ dout, const float *__restrict__ delta,
                                                               float *__restrict__ dense)
{
    using M = Mma<T>;
    using Frag = typename M::Frag;
    constexpr int CB = HD / 16;
    __shared__ __align__(16) T Ks[64 * (HD + 4)];
    __shared__ __align__(16) T Vs[64 * (HD + 4)];
    __shared__ __align__(16) PlaceAt at_s[64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16, q = wave * 16 + i;
    const bool even = w.gd > 0;
    // which tiles: query tile qt0 + step against key tile kt0 + step, for nz * ny * nx <= 64 steps
    unsigned id = blockIdx.x;
    const int chunk = (int)(id % (unsigned)w.chunks);
    id /= (unsigned)w.chunks;
    const int head = (int)(id % (unsigned)a.heads);
    id /= (unsigned)a.heads;
    int qt0, kt0, nz = 1, ny = 1, nx = 1, distance = 0;
    if (even) {
        // Distances in the order 0, 1, -1, 2, -2, ... along each axis, the one with most tiles outermost: those with most pairs
        // start first, and many and few are mixed in every CU (a window of 4 x 16 tiles, 8 heads: 84 us, 88 in raster order).
        auto take = [&](int n) {
            const int u = (int)(id % (unsigned)(2 * n - 1));
            id /= (unsigned)(2 * n - 1);
            return u;
        };
        auto signed_of = [](int u) { return u & 1 ? (u + 1) / 2 : -(u / 2); };
        int ux, uy, uz;
        if (w.gd >= w.gh && w.gd >= w.gw)
            ux = take(w.gw), uy = take(w.gh), uz = take(w.gd);
        else if (w.gh >= w.gw)
            uz = take(w.gd), ux = take(w.gw), uy = take(w.gh);
        else
            uz = take(w.gd), uy = take(w.gh), ux = take(w.gw);
        distance = (uz * (2 * w.gh - 1) + uy) * (2 * w.gw - 1) + ux;
        const int dx = signed_of(ux), dy = signed_of(uy), dz = signed_of(uz);
        nz = w.gd - abs(dz), ny = w.gh - abs(dy), nx = w.gw - abs(dx);
        qt0 = (max(dz, 0) * w.gh + max(dy, 0)) * w.gw + max(dx, 0);
        kt0 = (max(-dz, 0) * w.gh + max(-dy, 0)) * w.gw + max(-dx, 0);
    } else {
        kt0 = (int)(id % (unsigned)map.tiles);
        qt0 = (int)(id / (unsigned)map.tiles);
    }
    const int C = a.heads * a.hd;
    const unsigned stride = 3u * C;
    const T *base = qkv + (size_t)head * a.hd, *gbase = dout + (size_t)head * a.hd;
    const float scale2 = a.scale * kLog2e;
    f32x4 sum[4], bias[4];
    {
        const float *row = map.bias ? map.bias + (size_t)head * a.entries : nullptr;
        const PlaceAt *first = map.places;  // any window's: corners are the same in all
        const int cq = first[qt0 * 64 + q].corner + middle(a);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sum[j] = f32x4{};
#pragma unroll
            for (int r = 0; r < 4; ++r)
                bias[j][r] = row ? row[cq - first[kt0 * 64 + j * 16 + 4 * g + r].corner] : 0.f;
        }
    }
    // lane u's step, and of the window in hand which steps meet, one bit each; the next window's tiles are loaded ahead
    const int sx = lane % nx, sy = lane / nx % ny, sz = lane / nx / ny;
    const bool in = lane < nz * ny * nx;
    const int step = in ? (sz * w.gh + sy) * w.gw + sx : 0;
    const long long w1 = a.windows * (chunk + 1) / w.chunks;
    long long window = a.windows * chunk / w.chunks - 1;
    unsigned long long todo = 0, mask = 0;
    TileAt tq{kDead, 0, 0, 0}, tk{kDead, 0, 0, 0};
    auto look = [&](long long at) {
        if (at >= w1) return;
        tq = map.tiles_at[at * map.tiles + qt0 + step];
        tk = map.tiles_at[at * map.tiles + kt0 + step];
    };
    look(window + 1);
    struct Pair {
        long long window;
        int qt, kt;
        bool mixed, some;
    };
    auto advance = [&]() {
        while (!todo) {
            if (++window >= w1) return Pair{0, 0, 0, false, false};
            bool any, mixed;
            relation<false>(tq, tk, a.outside2, any, mixed);
            todo = __ballot(any && in);
            mask = __ballot(mixed);
            look(window + 1);
        }
        const int u = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int by = __builtin_amdgcn_readlane(step, u);
        return Pair{window, qt0 + by, kt0 + by, (bool)(mask >> u & 1), true};
    };
    Ahead<T, HD> ahead;
    ahead.none = 0;
    Frag qn[CB], gn[CB];
    int mine = -1;
    unsigned no_row = 0;
    float shift_next = 0.f, del_next = 0.f;
    auto tokens = [&](const Pair &p) {
        const int *live = map.live + p.window * map.tiles * 64;
        ahead.tokens(live, p.kt);
        mine = live[p.qt * 64 + q];
    };
    auto rows = [&](const Pair &p) {
        ahead.rows(base + C, stride, base + 2 * C, stride, a.hd);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            qn[c] = raw4<T>(base, stride, mine, c * 16 + 4 * g, a.hd);
            gn[c] = raw4<T>(gbase, C, mine, c * 16 + 4 * g, a.hd);
        }
        const size_t line = (((size_t)p.window * a.heads + head) * map.tiles + p.qt) * 64 + q;
        shift_next = lse[line];
        del_next = delta[line];
        no_row = mine < 0 ? 1u : 0u;
        settle(no_row);
    };
    // (where there are no more pairs, the first window's first tiles are loaded for nothing: see raw4)
    Pair now = advance(), next{};
    tokens(now);
    rows(now);
    next = advance();
    tokens(next);
    while (now.some) {
        const Pair hand = now;
        Frag qf[CB], gf[CB];
        __syncthreads();
        ahead.clear();
        ahead.x.store_rows(Ks);
        ahead.y.store_rows(Vs);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
            const bool in = !no_row && c * 16 + 4 * g < a.hd;
            qf[c] = cleared<T>(qn[c], in);
            gf[c] = cleared<T>(gn[c], in);
            settle(qf[c]);
            settle(gf[c]);
        }
        float shift = no_row ? INFINITY : shift_next, del = no_row ? 0.f : del_next;
        unsigned empty = no_row;
        settle(shift);
        settle(del);
        settle(empty);
        PlaceAt own{};
        if (hand.mixed) {  // (loaded when wanted)
            const PlaceAt *window = map.places + hand.window * map.tiles * 64;
            own = window[hand.qt * 64 + q];
            if (threadIdx.x < 64) at_s[threadIdx.x] = window[hand.kt * 64 + threadIdx.x];
            settle(own.label);
            settle(own.wrap);
        }
        __syncthreads();
        now = next;
        rows(now);
        next = advance();
        tokens(next);
        f32x4 x[4], dp[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[j] = over_channels<T, HD>(Vs, j * 16, gf);
        scores<T, HD>(x, Ks, qf, scale2, bias, hand.mixed, own, at_s, a.outside2);
        if (__any(empty != 0)) {  // the rows of no query are zeros, and 0 times an infinity of K or V is NaN
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[j][r] = empty ? 0.f : x[j][r], dp[j][r] = empty ? 0.f : dp[j][r];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[j][r] += __builtin_amdgcn_exp2f(x[j][r] - shift) * (dp[j][r] - del);
    }
    if (even) {  // [chunk][distance of tiles][head][64][64]
        const unsigned each = (unsigned)(w.chunks * a.heads);
        float *to = dense + (((size_t)chunk * (gridDim.x / each) + distance) * a.heads + head) * 4096 + q * 64;
#pragma unroll
        for (int j = 0; j < 4; ++j) *(f32x4 *)&to[j * 16 + 4 * g] = sum[j];
        return;
    }
    if (qt0 * 64 + q >= a.n) return;
    float *to = dense + (((size_t)chunk * a.heads + head) * a.n + qt0 * 64 + q) * a.n + kt0 * 64;  // [chunk][head][n][n]
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (kt0 * 64 + j * 16 + 4 * g + r < a.n) to[j * 16 + 4 * g + r] = sum[j][r];
}

// launchers, one translation unit for each element type
struct AttnBuffers {
    const void *qkv;
    const float *table;         // as given
    LongMap map;                // long windows
    bool even;                  // see Biases
    Split split;
    PairWork work;
    const int *labels;
    const void *out_in;
    void *out;
    float *lse;
    const void *dout;
    void *dqkv;
    float *pairs, *dense, *delta;
    void *spare;                // kSpareBytes that are written and never read
    int groups;                 // workgroups of window_fwd / window_bwd
};
template <class T>
void launch_attention_fwd(const WindowArgs &a, const AttnBuffers &b, hipStream_t st);
template <class T>
void launch_attention_bwd(const WindowArgs &a, const AttnBuffers &b, hipStream_t st);

}  // namespace aops

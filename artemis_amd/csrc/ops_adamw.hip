// ops_adamw.hip -- one AdamW step over many tensors, with 32-bit or 8-bit moments.
//
//   p *= 1 - lr wd;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Elementwise, so bound by memory: 28 bytes for an fp32 parameter with 32-bit moments, 16 with 8-bit ones.  A
// launch takes the addresses of up to 90 tensors (8 bit: 59) as its arguments (no copy of a table, nothing kept
// between calls); a workgroup finds its tensor and its share of 1024 elements by a search in the shares' prefix sums.
//
// 8-bit moments.  A positive fp32 number's bit pattern orders as the number does; its top 11 bits are 8 of
// exponent and 3 of mantissa.  256 elements share a base, and a code counts those 11 bits up from it: v, which
// has no sign, gets 255 codes (32 binades), m a sign and 127 (16 binades).  What is cut off is rounded up or down
// at random with the right mean: to the nearest of 8 steps in a binade, v would never move, since one step of
// b2 = 0.999 changes it by far less than half a step of its code.  16 random bits decide, from a counter-based
// generator, so that a step gives the same bits wherever it runs.  A positive v never becomes 0 (its code stops
// at 1: the quotient m / sqrt(v) stays bounded); an m below the smallest code becomes that or 0, with the right
// mean.
#include "ops_common.hpp"

namespace aops {
namespace {

constexpr int kThreads = 256;
// Elements a workgroup takes: four a thread.  Short-lived workgroups keep loads and stores of different ones in flight
// together: 29.1 M fp32 parameters with 32-bit moments take 163 us (5.0 TB/s) at 1024, 174 at 2048, 190 at 4096; with
// 8-bit ones 120, 140 and 174 us.
constexpr int kShare = 1024;
constexpr int kGroup = 256;   // elements that share a base

// A launch's tensors, as many as its 4 KB of arguments hold
struct Tensor32 {
    static constexpr int kMost = 90;
    void *p;
    const void *g;
    void *m, *v;
    long long count;
    Tensor32() = default;
    Tensor32(const artemis_ops_tensor &t, unsigned) : p(t.param), g(t.grad), m(t.m), v(t.v), count(t.count) {}
};
struct Tensor8 {
    static constexpr int kMost = 59;
    void *p;
    const void *g;
    void *m, *v;
    int *mb, *vb;
    long long count;
    unsigned place;  // among all tensors, in groups of kGroup
    Tensor8() = default;
    Tensor8(const artemis_ops_tensor &t, unsigned at)
        : p(t.param), g(t.grad), m(t.m), v(t.v), mb(t.m_base), vb(t.v_base), count(t.count), place(at) {}
};
template <class Tensor>
struct Batch {
    Tensor t[Tensor::kMost];
    int first[Tensor::kMost];  // the first workgroup of each tensor
    int n;
};

struct Coef {
    float keep;      // 1 - lr wd
    float b1, c1;    // b1, 1 - b1
    float b2, c2;    // b2, 1 - b2
    float step;      // lr / (1 - b1^t)
    float unbias;    // 1 / sqrt(1 - b2^t)
    float eps;
    unsigned key;    // of the generator: seed and step
};

// One element.  Every operation rounds by itself (no fused multiply-add): the new moments decide codes, and a
// last bit that depends on the compiler's choice would make them differ from build to build.
__device__ __forceinline__ void update(float &p, float g, float &m, float &v, const Coef &c)
{
#pragma clang fp contract(off)
    m = m * c.b1 + g * c.c1;
    v = v * c.b2 + (g * g) * c.c2;
    p = p * c.keep;
    p = p - (m * c.step) / (sqrtf(v) * c.unbias + c.eps);
}

template <class Tensor>
__device__ __forceinline__ int find(const Batch<Tensor> &b)
{
    int lo = 0, hi = b.n - 1;  // the last tensor whose first workgroup is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (b.first[mid] <= (int)blockIdx.x)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <class T>
__global__ __launch_bounds__(kThreads) void adamw32(const Batch<Tensor32> b, const Coef c)
{
    const int which = find(b);
    const Tensor32 t = b.t[which];
    const long long at = (long long)(blockIdx.x - b.first[which]) * kShare;
    T *p = (T *)t.p + at;
    const T *g = (const T *)t.g + at;
    float *m = (float *)t.m + at, *v = (float *)t.v + at;
    const int n = (int)(t.count - at < kShare ? t.count - at : kShare);
    const bool aligned = (((size_t)m | (size_t)v) & 15) == 0 && (((size_t)p | (size_t)g) & (4 * sizeof(T) - 1)) == 0;
    if (aligned && n == kShare) {
        constexpr int K = kShare / (4 * kThreads);
        Vec<T, 4> pv[K], gv[K];  // all loads in front of the first store
        f32x4 mv[K], vv[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = k * kThreads + threadIdx.x;
            pv[k] = ((Vec<T, 4> *)p)[i];
            gv[k] = ((const Vec<T, 4> *)g)[i];
            mv[k] = ((f32x4 *)m)[i];
            vv[k] = ((f32x4 *)v)[i];
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = k * kThreads + threadIdx.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = to_f32(pv[k].v[e]), a = mv[k][e], q = vv[k][e];
                update(x, to_f32(gv[k].v[e]), a, q, c);
                pv[k].v[e] = from_f32<T>(x);
                mv[k][e] = a;
                vv[k][e] = q;
            }
            ((Vec<T, 4> *)p)[i] = pv[k];
            ((f32x4 *)m)[i] = mv[k];
            ((f32x4 *)v)[i] = vv[k];
        }
        return;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        float x = to_f32(p[i]), a = m[i], q = v[i];
        update(x, to_f32(g[i]), a, q, c);
        p[i] = from_f32<T>(x);
        m[i] = a;
        v[i] = q;
    }
}

// 32 random bits from a counter: two rounds of multiplication by odd constants (the first 32 bits of the fraction of
// sqrt 2; those of sqrt 3 but for the first) between shifts, so that every bit of the counter reaches every bit of the result.
__device__ __forceinline__ unsigned noise(unsigned counter)
{
    unsigned z = counter;
    z = (z ^ (z >> 16)) * 0x6A09E667u;
    z = (z ^ (z >> 15)) * 0x3B67AE85u;
    return z ^ (z >> 16);
}

__device__ __forceinline__ float decode(unsigned code, int base)
{
    return code ? __uint_as_float((code + (unsigned)base) << 20) : 0.f;
}

__device__ __forceinline__ float decode_signed(unsigned code, int base)
{
    const float v = decode(code & 127u, base);
    return code & 128u ? -v : v;
}

// the base of a group whose largest magnitude has the bit pattern `top`: one code is left for rounding up
__device__ __forceinline__ int base_for(unsigned top, int codes)
{
    const int b = (int)(top >> 20) + 1 - codes;
    return b > 0 ? b : 0;
}

__device__ __forceinline__ unsigned encode(float v, int base, unsigned random16)
{
    if (!(v > 0.f) && !(v != v)) return 0;
    const int q = (int)((__float_as_uint(v) + (random16 << 4)) >> 20) - base;
    return (unsigned)(q < 1 ? 1 : q > 255 ? 255 : q);
}

__device__ __forceinline__ unsigned encode_signed(float m, int base, unsigned random16)
{
#pragma clang fp contract(off)
    const float a = fabsf(m);
    const float least = __uint_as_float((unsigned)(base + 1) << 20);
    int q;
    if (a < least) {
        q = a * 65536.0f > (float)random16 * least;
    } else {
        q = (int)((__float_as_uint(a) + (random16 << 4)) >> 20) - base;
        if (q > 127) q = 127;
    }
    return (unsigned)q | (m < 0.f && q ? 128u : 0u);
}

// The largest of 64 lanes' values: within rows of 16 by shifted copies, then across the rows.
__device__ __forceinline__ unsigned wave_max(unsigned x)
{
    auto step = [&](int y) { x = (unsigned)y > x ? (unsigned)y : x; };
    step(__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));
    step(__shfl_xor((int)x, 16));
    step(__shfl_xor((int)x, 32));
    return x;
}

// What a lane holds of a group: four neighbouring elements, the first n of them.
template <class T>
struct Held {
    Vec<T, 4> p, g;
    Vec<unsigned char, 4> m, v;
    int mb, vb;
};

// A wave takes groups of 256 elements, four neighbours in each lane; all groups' loads are in front of the first store.
template <class T>
__global__ __launch_bounds__(kThreads) void adamw8(const Batch<Tensor8> b, const Coef c)
{
    constexpr int K = kShare / kGroup / (kThreads / 64);
    const int which = find(b);
    const Tensor8 t = b.t[which];
    const long long at = (long long)(blockIdx.x - b.first[which]) * kShare;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const unsigned place = t.place;
    const bool aligned = ((size_t)t.p % (4 * sizeof(T)) | (size_t)t.g % (4 * sizeof(T)) |
                          ((size_t)t.m & 3) | ((size_t)t.v & 3)) == 0;
    Held<T> held[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i0 = at + (wave * K + k) * kGroup, i = i0 + lane * 4;
        Held<T> &h = held[k];
        h = Held<T>{};
        if (i0 >= t.count) continue;
        const T *p = (const T *)t.p + i, *g = (const T *)t.g + i;
        const unsigned char *mc = (const unsigned char *)t.m + i, *vc = (const unsigned char *)t.v + i;
        h.mb = t.mb[i0 / kGroup];
        h.vb = t.vb[i0 / kGroup];
        if (aligned && i + 4 <= t.count) {
            h.p = *(const Vec<T, 4> *)p;
            h.g = *(const Vec<T, 4> *)g;
            h.m = *(const Vec<unsigned char, 4> *)mc;
            h.v = *(const Vec<unsigned char, 4> *)vc;
        } else {
            for (int e = 0; e < 4 && i + e < t.count; ++e) {
                h.p.v[e] = p[e];
                h.g.v[e] = g[e];
                h.m.v[e] = mc[e];
                h.v.v[e] = vc[e];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i0 = at + (wave * K + k) * kGroup, i = i0 + lane * 4, group = i0 / kGroup;
        if (i0 >= t.count) break;
        Held<T> &h = held[k];
        float m[4], v[4];
        unsigned top_m = 0, top_v = 0;
        // (elements behind the tensor's end are zeros all through: they do not raise the largest)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = to_f32(h.p.v[e]);
            m[e] = decode_signed(h.m.v[e], h.mb);
            v[e] = decode(h.v.v[e], h.vb);
            update(x, to_f32(h.g.v[e]), m[e], v[e], c);
            h.p.v[e] = from_f32<T>(x);
            const unsigned a = __float_as_uint(fabsf(m[e])), q = __float_as_uint(v[e]) & 0x7FFFFFFFu;
            top_m = a > top_m ? a : top_m;
            top_v = q > top_v ? q : top_v;
        }
        const int nmb = base_for(wave_max(top_m), 127), nvb = base_for(wave_max(top_v), 255);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned z = noise((place + (unsigned)group) * (unsigned)kGroup + lane * 4 + e + c.key);
            h.m.v[e] = (unsigned char)encode_signed(m[e], nmb, z & 0xFFFFu);
            h.v.v[e] = (unsigned char)encode(v[e], nvb, z >> 16);
        }
        T *p = (T *)t.p + i;
        unsigned char *mc = (unsigned char *)t.m + i, *vc = (unsigned char *)t.v + i;
        if (aligned && i + 4 <= t.count) {
            *(Vec<T, 4> *)p = h.p;
            *(Vec<unsigned char, 4> *)mc = h.m;
            *(Vec<unsigned char, 4> *)vc = h.v;
        } else {
            for (int e = 0; e < 4 && i + e < t.count; ++e) {
                p[e] = h.p.v[e];
                mc[e] = h.m.v[e];
                vc[e] = h.v.v[e];
            }
        }
        if (lane == 0) {
            t.mb[group] = nmb;
            t.vb[group] = nvb;
        }
    }
}

template <bool SIGNED>
__global__ __launch_bounds__(kThreads) void moments_from_8bit(const Batch<Tensor8> b)
{
    const int which = find(b);
    const Tensor8 t = b.t[which];
    const long long at = (long long)(blockIdx.x - b.first[which]) * kShare;
    float *out = (float *)t.p;
    const unsigned char *codes = (const unsigned char *)t.m;
    const bool aligned = (((size_t)out & 15) | ((size_t)codes & 3)) == 0;
#pragma unroll
    for (int k = 0; k < kShare / (4 * kThreads); ++k) {
        const long long i = at + (k * kThreads + threadIdx.x) * 4LL;
        if (i >= t.count) break;
        const int base = t.mb[i / kGroup];
        if (aligned && i + 4 <= t.count) {
            const Vec<unsigned char, 4> q = *(const Vec<unsigned char, 4> *)(codes + i);
            f32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = SIGNED ? decode_signed(q.v[e], base) : decode(q.v[e], base);
            *(f32x4 *)(out + i) = o;
        } else {
            for (long long j = i; j < t.count && j < i + 4; ++j)
                out[j] = SIGNED ? decode_signed(codes[j], base) : decode(codes[j], base);
        }
    }
}

// Calls launch(batch, workgroups) for every batch of tensors: as many as fit the arguments and 2^23 workgroups
// (check_tensors holds each of them to that; a launch has at most 2^32 threads).
template <class Tensor, class F>
int in_batches(const artemis_ops_tensor *tensors, int n, const char *what, F launch)
{
    static_assert(sizeof(Batch<Tensor>) + sizeof(Coef) <= 4096, "a launch's arguments");
    Batch<Tensor> b;
    b.n = 0;
    long long blocks = 0;
    unsigned place = 0;
    constexpr long long kMost = 1 << 23;
    auto flush = [&]() -> int {
        if (b.n == 0) return 0;
        launch(b, (unsigned)blocks);
        b.n = 0;
        blocks = 0;
        return check_launch(what);
    };
    for (int i = 0; i < n; ++i) {
        const long long count = tensors[i].count;
        if (count == 0) continue;
        const long long need = (count + kShare - 1) / kShare;
        if (b.n == Tensor::kMost || blocks + need > kMost)
            if (int rc = flush()) return rc;
        b.t[b.n] = Tensor(tensors[i], place);
        b.first[b.n] = (int)blocks;
        ++b.n;
        blocks += need;
        place += (unsigned)((count + kGroup - 1) / kGroup);
    }
    return flush();
}

int check_tensors(const artemis_ops_tensor *tensors, int n, bool grads, bool bases, const char *what)
{
    if (n < 0) return fail(hipErrorInvalidValue, "%s: negative number of tensors", what);
    if (n > 0 && !tensors) return fail(hipErrorInvalidValue, "%s: NULL array of tensors", what);
    long long groups = 0;
    for (int i = 0; i < n; ++i) {
        const artemis_ops_tensor &t = tensors[i];
        if (t.count < 0 || t.count > ((1LL << 23) * kShare))
            return fail(hipErrorInvalidValue, "%s: tensor %d has %lld elements (0 .. 2^33)", what, i, t.count);
        groups += (t.count + kGroup - 1) / kGroup;
        if (t.count == 0) continue;
        if (!t.param || !t.m || (grads && (!t.grad || !t.v)) || (bases && (!t.m_base || (grads && !t.v_base))))
            return fail(hipErrorInvalidValue, "%s: tensor %d has a NULL pointer", what, i);
    }
    if (bases && grads && groups > (1LL << 24))
        return fail(hipErrorInvalidValue, "%s: more than 2^32 elements with 8-bit moments", what);
    return 0;
}

}  // namespace
}  // namespace aops

using namespace aops;

extern "C" {

int artemis_ops_adamw(const artemis_ops_tensor *tensors, int n_tensors, int dtype, int bits, double lr,
                      double beta1, double beta2, double eps, double weight_decay, long long step, unsigned seed,
                      void *stream)
{
    const char *what = "artemis_ops_adamw";
    if (dtype != ARTEMIS_OPS_F32 && dtype != ARTEMIS_OPS_BF16 && dtype != ARTEMIS_OPS_F16)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d", what, dtype);
    if (bits != 32 && bits != 8) return fail(hipErrorInvalidValue, "%s: moments of %d bits (32 or 8)", what, bits);
    if (!(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) ||
        !(weight_decay >= 0) || step < 1)
        return fail(hipErrorInvalidValue,
                    "%s: lr=%g betas=(%g, %g) eps=%g weight_decay=%g step=%lld: lr, eps, weight_decay >= 0, betas "
                    "in [0, 1) and step >= 1 are wanted", what, lr, beta1, beta2, eps, weight_decay, step);
    if (int rc = check_tensors(tensors, n_tensors, true, bits == 8, what)) return rc;
    // in 64 bits: 1 - beta^t loses most of its digits in 32 for small t
    Coef c;
    c.keep = (float)(1.0 - lr * weight_decay);
    c.b1 = (float)beta1;
    c.c1 = (float)(1.0 - beta1);
    c.b2 = (float)beta2;
    c.c2 = (float)(1.0 - beta2);
    c.step = (float)(lr / (1.0 - pow(beta1, (double)step)));
    c.unbias = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    c.eps = (float)eps;
    c.key = seed * 0x9E3779B1u + (unsigned)step * 0x6A09E667u;
    hipStream_t st = (hipStream_t)stream;
    if (bits == 32)
        return in_batches<Tensor32>(tensors, n_tensors, what, [&](const Batch<Tensor32> &b, unsigned blocks) {
            const dim3 grid(blocks), block(kThreads);
            if (dtype == ARTEMIS_OPS_F32)
                hipLaunchKernelGGL((adamw32<float>), grid, block, 0, st, b, c);
            else if (dtype == ARTEMIS_OPS_BF16)
                hipLaunchKernelGGL((adamw32<__bf16>), grid, block, 0, st, b, c);
            else
                hipLaunchKernelGGL((adamw32<_Float16>), grid, block, 0, st, b, c);
        });
    return in_batches<Tensor8>(tensors, n_tensors, what, [&](const Batch<Tensor8> &b, unsigned blocks) {
        const dim3 grid(blocks), block(kThreads);
        if (dtype == ARTEMIS_OPS_F32)
            hipLaunchKernelGGL((adamw8<float>), grid, block, 0, st, b, c);
        else if (dtype == ARTEMIS_OPS_BF16)
            hipLaunchKernelGGL((adamw8<__bf16>), grid, block, 0, st, b, c);
        else
            hipLaunchKernelGGL((adamw8<_Float16>), grid, block, 0, st, b, c);
    });
}

int artemis_ops_moments_from_8bit(const artemis_ops_tensor *tensors, int n_tensors, int is_signed, void *stream)
{
    const char *what = "artemis_ops_moments_from_8bit";
    if (int rc = check_tensors(tensors, n_tensors, false, true, what)) return rc;
    hipStream_t st = (hipStream_t)stream;
    return in_batches<Tensor8>(tensors, n_tensors, what, [&](const Batch<Tensor8> &b, unsigned blocks) {
        if (is_signed)
            hipLaunchKernelGGL((moments_from_8bit<true>), dim3(blocks), dim3(kThreads), 0, st, b);
        else
            hipLaunchKernelGGL((moments_from_8bit<false>), dim3(blocks), dim3(kThreads), 0, st, b);
    });
}

}  // extern "C"

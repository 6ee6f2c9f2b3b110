// ops_norm.hip -- layer norm over the last dimension, forward and backward.
//
//   y  = (x - mean) rstd w + b                        rstd = (var + eps)^-1/2
//   dx = rstd (a - mean(a) - xh mean(a xh))           a = dy w, xh = (x - mean) rstd
//   dw = sum over rows of dy xh,  db = sum of dy
//
// Both passes are bound by memory: 2 (forward) and 4 (whole training pass: x, dy in, y, dx out) values moved
// for each element, a few operations on each.  A row is therefore read once and stays in registers: L lanes of
// a wave hold it, NV vectors of 16 bytes each.  The variance is the mean of squared deviations from the mean
// in the registers, not E[x^2] - mean^2, which cancels for features far from zero.  Measured at 33 M elements (rows of 64 to 8192,
// divisible or not): forward 39 to 45 us in fp32 (5.8 to 6.9 TB/s), 20 to 34 in 16 bits, backward 77 to 120 in fp32 (5.1 to
// 3.3 TB/s) with 1024 shares of dw and db.
// The weight's gradient is summed over the rows that a workgroup meets in registers, then over its row
// groups through LDS in a fixed order, then over the workgroups by a second kernel: no atomics, so every run
// gives the same bits.
#include "ops_common.hpp"

namespace aops {
namespace {

constexpr int kThreads = 256;

// Where a lane's vectors lie in a row.  Vector j has the columns from j * VEC on; the last one of a row that VEC does not
// divide ends with the row and starts earlier, and so do vectors behind the row's end: their first `skip` elements belong
// to others (or there is nothing for them to do: skip >= VEC), are left out of the sums, and get the value from
// both.  So every load is one of 16 bytes, made without a condition; rows and pointers need no alignment beyond the element's.
// WHOLE: the lanes' vectors are exactly the row.
template <int VEC, int L, int NV, bool WHOLE>
struct Columns {
    int start[NV], skip[NV];
    __device__ __forceinline__ Columns(int lane, int cols)
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (lane + i * L) * VEC;
            start[i] = WHOLE ? at : min(at, cols - VEC);
            skip[i] = at - start[i];
        }
    }
    __device__ __forceinline__ bool has(int i, int e) const { return WHOLE || e >= skip[i]; }
    __device__ __forceinline__ bool any(int i) const { return WHOLE || skip[i] < VEC; }
};

template <int VEC, class T>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T *p)
{
    Vec<T, VEC> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <int VEC, class T>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, VEC> &v)
{
    __builtin_memcpy(p, &v, sizeof(v));
}

// VEC parameters from column `start` on; `none` where there are no parameters
template <int VEC>
__device__ __forceinline__ void load_params(float (&to)[VEC], const float *__restrict__ p, int start, float none)
{
#pragma unroll
    for (int e = 0; e < VEC; ++e) to[e] = none;
    if (!p) return;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const Vec<float, 4> v = load_vec<4>(p + start + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) to[e + k] = v.v[k];
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) to[e] = p[start + e];
    }
}

// The sum over a row's L lanes, in all of them.  Over a whole workgroup it goes through LDS: `part` may be used again once all
// have passed another such sum.
template <int L>
__device__ __forceinline__ float row_sum(float x, float *part)
{
    if constexpr (L <= 64) return group_sum<L>(x);
    x = group_sum<64>(x);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// Rows of `cols` elements as NV vectors of VEC elements in each of L lanes; lane i holds the vectors i, i + L, ...
// R rows are in flight at once: one row's 16 bytes for a lane, read, summed and written in turn, leave the memory
// waiting for the sums (524288 rows of 64 in fp32: 96 us one by one, 46 with four).  Loads under a condition are as bad:
// 130560 rows of 256 in bf16 34 us, without 28; 8191 rows of 1001 in fp16 by single elements 20, by vectors 8.6.
template <class T, int VEC, int L, int NV, int R, bool WHOLE>
__global__ __launch_bounds__(kThreads) void norm_fwd(const T *__restrict__ x, const float *__restrict__ w,
                                                     const float *__restrict__ b, T *__restrict__ y,
                                                     float *__restrict__ mean_out, float *__restrict__ rstd_out,
                                                     long long rows, int cols, float eps)
{
    constexpr int G = kThreads / L;
    __shared__ float part[2][kThreads / 64];
    const int lane = threadIdx.x % L;
    const Columns<VEC, L, NV, WHOLE> at(lane, cols);
    const float inv = 1.0f / (float)cols;
    // (whole groups of L lanes leave the loop together: the sums below stay within a group)
    for (long long row0 = (long long)blockIdx.x * (G * R) + threadIdx.x / L; row0 < rows;
         row0 += (long long)gridDim.x * (G * R)) {
        Vec<T, VEC> t[R][NV];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long row = min(row0 + k * G, rows - 1);
#pragma unroll
            for (int i = 0; i < NV; ++i) t[k][i] = load_vec<VEC>(x + row * cols + at.start[i]);
        }
        float wv[NV][VEC], bv[NV][VEC];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            load_params<VEC>(wv[i], w, at.start[i], 1.f);
            load_params<VEC>(bv[i], b, at.start[i], 0.f);
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long row = row0 + k * G;
            if (row >= rows) break;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) s += at.has(i, e) ? to_f32(t[k][i].v[e]) : 0.f;
            const float mean = row_sum<L>(s, part[0]) * inv;
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float d = at.has(i, e) ? to_f32(t[k][i].v[e]) - mean : 0.f;
                    q += d * d;
                }
            const float rstd = 1.0f / sqrtf(row_sum<L>(q, part[1]) * inv + eps);
            if (lane == 0 && mean_out) {
                mean_out[row] = mean;
                rstd_out[row] = rstd;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!at.any(i)) continue;
                Vec<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    o.v[e] = from_f32<T>((to_f32(t[k][i].v[e]) - mean) * rstd * wv[i][e] + bv[i][e]);
                store_vec<VEC>(y + row * cols + at.start[i], o);
            }
        }
    }
}

// One workgroup for a row of any width: three passes over it, the later two from the caches.
template <class T>
__global__ __launch_bounds__(kThreads) void norm_fwd_wide(const T *__restrict__ x, const float *__restrict__ w,
                                                          const float *__restrict__ b, T *__restrict__ y,
                                                          float *__restrict__ mean_out,
                                                          float *__restrict__ rstd_out, long long rows, int cols,
                                                          float eps)
{
    __shared__ float part[2][kThreads / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * cols;
    T *yr = y + row * cols;
    float s = 0.f;
    for (int c = threadIdx.x; c < cols; c += kThreads) s += to_f32(xr[c]);
    s = group_sum<64>(s);
    if (threadIdx.x % 64 == 0) part[0][threadIdx.x / 64] = s;  // (the row before read it in front of its 2nd barrier)
    __syncthreads();
    const float mean = (part[0][0] + part[0][1] + part[0][2] + part[0][3]) / (float)cols;
    float q = 0.f;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
        const float d = to_f32(xr[c]) - mean;
        q += d * d;
    }
    q = group_sum<64>(q);
    if (threadIdx.x % 64 == 0) part[1][threadIdx.x / 64] = q;
    __syncthreads();
    const float rstd = 1.0f / sqrtf((part[1][0] + part[1][1] + part[1][2] + part[1][3]) / (float)cols + eps);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    for (int c = threadIdx.x; c < cols; c += kThreads) {
        float v = (to_f32(xr[c]) - mean) * rstd;
        if (w) v *= w[c];
        if (b) v += b[c];
        yr[c] = from_f32<T>(v);
    }
    __syncthreads();  // part[1] has been read
    }
}

// partial (gridDim.x, 2, cols): this workgroup's share of dw and db; NULL: not asked for
template <class T, int VEC, int L, int NV, bool WHOLE>
__global__ __launch_bounds__(kThreads) void norm_bwd(const T *__restrict__ x, const T *__restrict__ dy,
                                                     const float *__restrict__ w,
                                                     const float *__restrict__ mean_in,
                                                     const float *__restrict__ rstd_in, T *__restrict__ dx,
                                                     float *__restrict__ partial, long long rows, int cols)
{
    constexpr int G = kThreads / L;  // row groups of a workgroup
    __shared__ float fold[G > 1 ? G * L * NV * VEC : 1], part[2][2][kThreads / 64];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const Columns<VEC, L, NV, WHOLE> at(lane, cols);
    const float inv = 1.0f / (float)cols;
    float wv[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
        load_params<VEC>(wv[i], w, at.start[i], 1.f);
    }
    int odd = 0;  // rows alternate between two places for the sums over a workgroup
    for (long long row = (long long)blockIdx.x * G + group; row < rows; row += (long long)gridDim.x * G) {
        const float mean = mean_in[row], rstd = rstd_in[row];
        Vec<T, VEC> tx[NV], tg[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            tx[i] = load_vec<VEC>(x + row * cols + at.start[i]);
            tg[i] = load_vec<VEC>(dy + row * cols + at.start[i]);
        }
        float xh[NV][VEC], a[NV][VEC];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = to_f32(tg[i].v[e]), h = (to_f32(tx[i].v[e]) - mean) * rstd;
                xh[i][e] = h;
                a[i][e] = g * wv[i][e];
                s1 += at.has(i, e) ? a[i][e] : 0.f;
                s2 += at.has(i, e) ? a[i][e] * h : 0.f;
                dw[i][e] += g * h;
                db[i][e] += g;
            }
        if (!dx) continue;
        const float m1 = row_sum<L>(s1, part[odd][0]) * inv, m2 = row_sum<L>(s2, part[odd][1]) * inv;
        odd ^= 1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!at.any(i)) continue;
            Vec<T, VEC> t;
#pragma unroll
            for (int e = 0; e < VEC; ++e) t.v[e] = from_f32<T>(rstd * (a[i][e] - m1 - xh[i][e] * m2));
            store_vec<VEC>(dx + row * cols + at.start[i], t);
        }
    }
    if (!partial) return;
    float *out = partial + (size_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (G == 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (at.has(i, e) && at.any(i)) out[which * cols + at.start[i] + e] = which ? db[i][e] : dw[i][e];
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (at.has(i, e) && at.any(i))
                        fold[group * (L * NV * VEC) + at.start[i] + e] = which ? db[i][e] : dw[i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += kThreads) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < G; ++k) s += fold[k * (L * NV * VEC) + c];
                out[which * cols + c] = s;
            }
        }
    }
}

// Wide rows: a workgroup takes rows blockIdx.x, blockIdx.x + gridDim.x, ...; its columns' sums for dw and db
// stay in the partial buffer, where every thread adds to its own columns only.
template <class T>
__global__ __launch_bounds__(kThreads) void norm_bwd_wide(const T *__restrict__ x, const T *__restrict__ dy,
                                                          const float *__restrict__ w,
                                                          const float *__restrict__ mean_in,
                                                          const float *__restrict__ rstd_in, T *__restrict__ dx,
                                                          float *__restrict__ partial, long long rows, int cols)
{
    __shared__ float part[2][kThreads / 64];
    float *out = partial ? partial + (size_t)blockIdx.x * 2 * cols : nullptr;
    bool first = true;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols, *gr = dy + row * cols;
        const float mean = mean_in[row], rstd = rstd_in[row];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < cols; c += kThreads) {
            const float g = to_f32(gr[c]), xh = (to_f32(xr[c]) - mean) * rstd;
            const float a = w ? g * w[c] : g;
            s1 += a;
            s2 += a * xh;
            if (out) {
                out[c] = first ? g * xh : out[c] + g * xh;
                out[cols + c] = first ? g : out[cols + c] + g;
            }
        }
        first = false;
        if (!dx) continue;
        s1 = group_sum<64>(s1);
        s2 = group_sum<64>(s2);
        __syncthreads();  // the row before has been read
        if (threadIdx.x % 64 == 0) {
            part[0][threadIdx.x / 64] = s1;
            part[1][threadIdx.x / 64] = s2;
        }
        __syncthreads();
        const float m1 = (part[0][0] + part[0][1] + part[0][2] + part[0][3]) / (float)cols;
        const float m2 = (part[1][0] + part[1][1] + part[1][2] + part[1][3]) / (float)cols;
        T *dr = dx + row * cols;
        for (int c = threadIdx.x; c < cols; c += kThreads) {
            const float xh = (to_f32(xr[c]) - mean) * rstd;
            const float a = w ? to_f32(gr[c]) * w[c] : to_f32(gr[c]);
            dr[c] = from_f32<T>(rstd * (a - m1 - xh * m2));
        }
    }
}

// dw and db from the workgroups' shares: 16 columns at a time for a workgroup, 64 threads on each, joined in order.  (16 threads
// on each: 17 us for 1024 shares of 2 x 64 columns, all of it waiting for 64 loads in a row.)
constexpr int kFold = 1024;
__global__ __launch_bounds__(kFold) void norm_fold(const float *__restrict__ partial, float *__restrict__ dw,
                                                   float *__restrict__ db, int parts, int cols)
{
    __shared__ float fold[kFold / 16][17];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (long long first = blockIdx.x * 16LL; first < 2LL * cols; first += gridDim.x * 16LL) {
        const long long c = first + tx;  // of 2 * cols
        float s = 0.f;
        if (c < 2LL * cols) {
#pragma unroll 8
            for (int p = ty; p < parts; p += kFold / 16) s += partial[(size_t)p * 2 * cols + c];
        }
        fold[ty][tx] = s;
        __syncthreads();
        if (threadIdx.x < 16 && c < 2LL * cols) {
            float t = 0.f;
            for (int k = 0; k < kFold / 16; ++k) t += fold[k][tx];
            if (c < cols) {
                if (dw) dw[c] = t;
            } else if (db) {
                db[c - cols] = t;
            }
        }
        __syncthreads();  // the sums have been read
    }
}

// How a row is held: `vec` elements for a vector, `lanes` lanes, `nv` vectors in each; lanes = 0: a workgroup
// for a row, which it reads three times.  Vectors of 16 bytes where a row has as many; as few lanes as hold a row, so
// that a wave takes several narrow rows, and a whole workgroup where a wave's lanes would need more than 16 elements.
struct Shape {
    int vec, lanes, nv;
};

int element_size(int dtype) { return dtype == ARTEMIS_OPS_F32 ? 4 : 2; }

Shape shape_for(long long cols, int dtype)
{
    const int wide = 16 / element_size(dtype);
    if (cols < wide) return {1, 8, 1};
    const long long nvec = (cols + wide - 1) / wide;
    if (nvec <= 64) {
        int lanes = 8;
        while (lanes < nvec) lanes *= 2;
        return {wide, lanes, 1};
    }
    for (int nv = 2; nv * wide <= 16; nv *= 2)
        if (nvec <= 64LL * nv) return {wide, 64, nv};
    for (int nv = 2; nv * wide <= 32; nv *= 2)
        if (nvec <= 256LL * nv) return {wide, 256, nv};
    return {1, 0, 0};
}

// Workgroups of the backward pass: enough to fill 256 CUs several times over, no more than there are rows
// for, since each writes a share of dw and db.
long long bwd_blocks(long long rows, int rows_at_once)
{
    const long long need = (rows + rows_at_once - 1) / rows_at_once;
    return need < 1024 ? need : 1024;
}

// a workgroup for each group of rows, up to a launch's 2^32 threads
unsigned fwd_blocks(long long rows, int rows_at_once)
{
    const long long need = (rows + rows_at_once - 1) / rows_at_once;
    return (unsigned)(need < (1 << 22) ? need : (1 << 22));
}

// 16 columns for each workgroup of norm_fold, up to 2^20 of them (a launch has at most 2^32 threads)
unsigned fold_blocks(long long cols)
{
    const long long need = (2 * cols + 15) / 16;
    return (unsigned)(need < (1 << 20) ? need : (1 << 20));
}

template <class T, class F>
bool with_shape(const Shape &s, int cols, F f)
{
    constexpr int W = 16 / (int)sizeof(T);
    using std::integral_constant;
#define ARTEMIS_CASE(V, L, N)                                                                                   \
    if (s.vec == V && s.lanes == L && s.nv == N) {                                                              \
        if (cols == V * L * N)                                                                                  \
            f(integral_constant<int, V>{}, integral_constant<int, L>{}, integral_constant<int, N>{}, std::true_type{});  \
        else                                                                                                    \
            f(integral_constant<int, V>{}, integral_constant<int, L>{}, integral_constant<int, N>{}, std::false_type{}); \
        return true;                                                                                            \
    }
    ARTEMIS_CASE(1, 8, 1)
    ARTEMIS_CASE(W, 8, 1) ARTEMIS_CASE(W, 16, 1) ARTEMIS_CASE(W, 32, 1) ARTEMIS_CASE(W, 64, 1) ARTEMIS_CASE(W, 64, 2)
    ARTEMIS_CASE(W, 256, 2) ARTEMIS_CASE(W, 256, 4)
    if constexpr (W == 4) {
        ARTEMIS_CASE(W, 64, 4) ARTEMIS_CASE(W, 256, 8)
    }
#undef ARTEMIS_CASE
    return false;
}

template <class T>
int run_fwd(const void *x, const float *w, const float *b, void *y, float *mean, float *rstd, long long rows,
            int cols, float eps, int dtype, hipStream_t st)
{
    const Shape s = shape_for(cols, dtype);
    if (!with_shape<T>(s, cols, [&](auto V, auto L, auto N, auto WHOLE) {
            // rows in flight: as many as 64 bytes for a lane make
            constexpr int R = N == 1 ? 4 : N == 2 ? 2 : 1;
            hipLaunchKernelGGL((norm_fwd<T, V, L, N, R, WHOLE>), dim3(fwd_blocks(rows, kThreads / L * R)), dim3(kThreads), 0, st,
                               (const T *)x, w, b, (T *)y, mean, rstd, rows, cols, eps);
        }))
        hipLaunchKernelGGL((norm_fwd_wide<T>), dim3(fwd_blocks(rows, 1)), dim3(kThreads), 0, st, (const T *)x, w, b,
                           (T *)y, mean, rstd, rows, cols, eps);
    return check_launch("artemis_ops_layer_norm_forward");
}

template <class T>
int run_bwd(const void *x, const void *dy, const float *w, const float *mean, const float *rstd, void *dx,
            float *dw, float *db, long long rows, int cols, int dtype, float *partial, hipStream_t st)
{
    const Shape s = shape_for(cols, dtype);
    const int parts = (int)bwd_blocks(rows, s.lanes ? kThreads / s.lanes : 1);
    if (!with_shape<T>(s, cols, [&](auto V, auto L, auto N, auto WHOLE) {
            hipLaunchKernelGGL((norm_bwd<T, V, L, N, WHOLE>), dim3(parts), dim3(kThreads), 0, st, (const T *)x,
                               (const T *)dy, w, mean, rstd, (T *)dx, partial, rows, cols);
        }))
        hipLaunchKernelGGL((norm_bwd_wide<T>), dim3(parts), dim3(kThreads), 0, st, (const T *)x, (const T *)dy, w,
                           mean, rstd, (T *)dx, partial, rows, cols);
    if (partial)
        hipLaunchKernelGGL(norm_fold, dim3(fold_blocks(cols)), dim3(kFold), 0, st, partial, dw, db, parts, cols);
    return check_launch("artemis_ops_layer_norm_backward");
}

int check_sizes(const char *what, long long rows, long long cols, int dtype)
{
    if (rows < 0 || cols < 0 || rows >= (1LL << 31) || cols >= (1LL << 30))
        return fail(hipErrorInvalidValue, "%s: %lld rows of %lld columns (0 <= rows < 2^31, 0 <= cols < 2^30)",
                    what, rows, cols);
    if (rows > 0 && cols == 0) return fail(hipErrorInvalidValue, "%s: rows without columns", what);
    if (dtype != ARTEMIS_OPS_F32 && dtype != ARTEMIS_OPS_BF16 && dtype != ARTEMIS_OPS_F16)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d", what, dtype);
    return 0;
}

}  // namespace
}  // namespace aops

using namespace aops;

extern "C" {

int artemis_ops_layer_norm_forward(const void *x, const float *weight, const float *bias, void *y, float *mean,
                                   float *rstd, long long rows, long long cols, float eps, int dtype,
                                   void *stream)
{
    const char *what = "artemis_ops_layer_norm_forward";
    if (int rc = check_sizes(what, rows, cols, dtype)) return rc;
    if (rows == 0) return 0;
    if (!x || !y) return fail(hipErrorInvalidValue, "%s: NULL tensor pointer", what);
    if (!mean != !rstd) return fail(hipErrorInvalidValue, "%s: mean and rstd are written together", what);
    if (!(eps >= 0.f)) return fail(hipErrorInvalidValue, "%s: eps must be >= 0", what);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ARTEMIS_OPS_F32) return run_fwd<float>(x, weight, bias, y, mean, rstd, rows, (int)cols, eps, dtype, st);
    if (dtype == ARTEMIS_OPS_BF16)
        return run_fwd<__bf16>(x, weight, bias, y, mean, rstd, rows, (int)cols, eps, dtype, st);
    return run_fwd<_Float16>(x, weight, bias, y, mean, rstd, rows, (int)cols, eps, dtype, st);
}

size_t artemis_ops_layer_norm_workspace_bytes(long long rows, long long cols, int dtype)
{
    if (rows < 0 || cols <= 0 || dtype < 0 || dtype > ARTEMIS_OPS_F16) return 0;
    const Shape s = shape_for(cols, dtype);
    const long long parts = bwd_blocks(rows, s.lanes ? kThreads / s.lanes : 1);
    return (size_t)parts * 2 * (size_t)cols * sizeof(float);
}

int artemis_ops_layer_norm_backward(const void *x, const void *dy, const float *weight, const float *mean,
                                    const float *rstd, void *dx, float *dweight, float *dbias, long long rows,
                                    long long cols, int dtype, void *workspace, size_t workspace_bytes,
                                    void *stream)
{
    const char *what = "artemis_ops_layer_norm_backward";
    if (int rc = check_sizes(what, rows, cols, dtype)) return rc;
    if (cols == 0 || (!dx && !dweight && !dbias)) return 0;
    hipStream_t st = (hipStream_t)stream;
    const bool sums = dweight || dbias;
    if (rows == 0) {  // sums over nothing
        if (sums)
            hipLaunchKernelGGL(norm_fold, dim3(fold_blocks(cols)), dim3(kFold), 0, st, (const float *)nullptr, dweight, dbias, 0,
                               (int)cols);
        return check_launch(what);
    }
    if (!x || !dy || !mean || !rstd) return fail(hipErrorInvalidValue, "%s: NULL tensor pointer", what);
    if (sums && (!workspace || workspace_bytes < artemis_ops_layer_norm_workspace_bytes(rows, cols, dtype)))
        return fail(hipErrorInvalidValue, "%s: workspace of %zu bytes, %zu needed", what,
                    workspace ? workspace_bytes : (size_t)0,
                    artemis_ops_layer_norm_workspace_bytes(rows, cols, dtype));
    float *partial = sums ? (float *)workspace : nullptr;
    if (dtype == ARTEMIS_OPS_F32)
        return run_bwd<float>(x, dy, weight, mean, rstd, dx, dweight, dbias, rows, (int)cols, dtype, partial, st);
    if (dtype == ARTEMIS_OPS_BF16)
        return run_bwd<__bf16>(x, dy, weight, mean, rstd, dx, dweight, dbias, rows, (int)cols, dtype, partial, st);
    return run_bwd<_Float16>(x, dy, weight, mean, rstd, dx, dweight, dbias, rows, (int)cols, dtype, partial, st);
}

}  // extern "C"

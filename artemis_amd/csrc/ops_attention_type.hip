// ops_attention_type.hip -- the attention kernels of one element type (OPS_TYPE), and which of them a call takes:
// the head's channels rounded up to 16, 32, 64 or 128, and the size of the window.
#include "ops_attention.hpp"

namespace aops {
namespace {

template <class F>
void with_hd(int hd, F f)
{
    using std::integral_constant;
    if (hd <= 16)
        f(integral_constant<int, 16>{});
    else if (hd <= 32)
        f(integral_constant<int, 32>{});
    else if (hd <= 64)
        f(integral_constant<int, 64>{});
    else
        f(integral_constant<int, 128>{});
}

template <class F>
void with_nb(int n, F f)
{
    using std::integral_constant;
    if (n <= 16)
        f(integral_constant<int, 1>{});
    else if (n <= 32)
        f(integral_constant<int, 2>{});
    else
        f(integral_constant<int, 4>{});
}

unsigned long_grid(const WindowArgs &a) { return (unsigned)(a.windows * a.heads * ((a.n + 63) / 64)); }

// rows of the window that are multiples of 4: four neighbours' bias entries lie behind each other
template <class F>
void with_vec(int ww, F f)
{
    if (ww % 4 == 0)
        f(std::true_type{});
    else
        f(std::false_type{});
}

}  // namespace

template <>
void launch_attention_fwd<OPS_TYPE>(const WindowArgs &a, const AttnBuffers &b, hipStream_t st)
{
    using T = OPS_TYPE;
    with_hd(a.hd, [&](auto HD) {
        if (a.n <= 64)
            with_nb(a.n, [&](auto NB) {
                hipLaunchKernelGGL((window_fwd<T, HD, NB>), dim3(b.groups), dim3(kAttnThreads), 0, st, a, (const T *)b.qkv,
                                   b.table, b.labels, (T *)b.out);
            });
        else
            with_vec(a.ww, [&](auto VEC) {
                hipLaunchKernelGGL((long_fwd<T, HD, VEC>), dim3(long_grid(a)), dim3(kAttnThreads), 0, st, a, b.map,
                                   (const T *)b.qkv, (T *)b.out, b.lse);
            });
    });
}

template <>
void launch_attention_bwd<OPS_TYPE>(const WindowArgs &a, const AttnBuffers &b, hipStream_t st)
{
    using T = OPS_TYPE;
    with_hd(a.hd, [&](auto HD) {
        if (a.n <= 64) {
            with_nb(a.n, [&](auto NB) {
                hipLaunchKernelGGL((window_bwd<T, HD, NB>), dim3(b.groups), dim3(kAttnThreads), 0, st, a, (const T *)b.qkv,
                                   b.table, b.labels, (const T *)b.dout, (T *)b.dqkv, b.pairs);
            });
            return;
        }
        with_vec(a.ww, [&](auto VEC) {
            hipLaunchKernelGGL((long_bwd_q<T, HD, VEC>), dim3(long_grid(a)), dim3(kAttnThreads), 0, st, a, b.map,
                               (const T *)b.qkv, (const T *)b.out_in, b.lse, (const T *)b.dout, (T *)b.dqkv, b.delta);
            hipLaunchKernelGGL((long_bwd_kv<T, HD, VEC>), dim3(long_grid(a)), dim3(kAttnThreads), 0, st, a, b.map,
                               (const T *)b.qkv, b.lse, (const T *)b.dout, (T *)b.dqkv, b.delta);
        });
        if (b.dense) {
            const PairWork &w = b.work;
            const unsigned distances = w.gd ? (2 * w.gd - 1) * (2 * w.gh - 1) * (2 * w.gw - 1) : b.map.tiles * b.map.tiles;
            hipLaunchKernelGGL((long_bwd_pairs<T, HD>), dim3(distances * a.heads * w.chunks), dim3(kAttnThreads), 0, st, a, b.map, w,
                               (const T *)b.qkv, b.lse, (const T *)b.dout, b.delta, b.dense);
        }
    });
}

}  // namespace aops

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

dim3 long_grid(const WindowArgs &a, const AttnBuffers &b)
{
    return dim3((unsigned)(a.windows * a.heads * b.map.tiles), b.split.splits);
}
unsigned join_grid(const WindowArgs &a, const AttnBuffers &b)
{
    return (unsigned)((a.windows * a.heads * b.map.tiles * 64 * (a.hd / 4) + kAttnThreads - 1) / kAttnThreads);
}

template <class F>
void with_bool(bool is, F f)
{
    if (is)
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
                with_bool(b.labels != nullptr, [&](auto LABELS) {
                    hipLaunchKernelGGL((window_fwd<T, HD, NB, LABELS>), dim3(b.groups), dim3(kAttnThreads), 0, st, a,
                                       (const T *)b.qkv, b.table, b.labels, (T *)b.out, (T *)b.spare);
                });
            });
        else
            with_bool(b.even, [&](auto EVEN) {
                hipLaunchKernelGGL((long_fwd<T, HD, EVEN>), long_grid(a, b), dim3(kAttnThreads), 0, st, a, b.map, b.split,
                                   (const T *)b.qkv, (T *)b.out, b.lse);
            });
    });
    if (a.n > 64 && b.split.splits > 1)
        hipLaunchKernelGGL((long_fwd_join<T>), dim3(join_grid(a, b)), dim3(kAttnThreads), 0, st, a, b.map, b.split, (T *)b.out,
                           b.lse);
}

template <>
void launch_attention_bwd<OPS_TYPE>(const WindowArgs &a, const AttnBuffers &b, hipStream_t st)
{
    using T = OPS_TYPE;
    with_hd(a.hd, [&](auto HD) {
        if (a.n <= 64) {
            with_nb(a.n, [&](auto NB) {
                with_bool(b.labels != nullptr, [&](auto LABELS) {
                    hipLaunchKernelGGL((window_bwd<T, HD, NB, LABELS>), dim3(b.groups), dim3(kAttnThreads), 0, st, a,
                                       (const T *)b.qkv, b.table, b.labels, (const T *)b.dout, (T *)b.dqkv, b.pairs,
                                       (T *)b.spare);
                });
            });
            return;
        }
        const dim3 grid = long_grid(a, b), join(join_grid(a, b)), block(kAttnThreads);
        with_bool(b.even, [&](auto EVEN) {
            hipLaunchKernelGGL((long_bwd_q<T, HD, EVEN>), grid, block, 0, st, a, b.map, b.split, (const T *)b.qkv,
                               (const T *)b.out_in, b.lse, (const T *)b.dout, (T *)b.dqkv, b.delta);
            if (b.split.splits > 1)
                hipLaunchKernelGGL((long_bwd_join<T, false>), join, block, 0, st, a, b.map, b.split, (T *)b.dqkv, b.delta);
            hipLaunchKernelGGL((long_bwd_kv<T, HD, EVEN>), grid, block, 0, st, a, b.map, b.split, (const T *)b.qkv, b.lse,
                               (const T *)b.dout, (T *)b.dqkv, b.delta);
            if (b.split.splits > 1)
                hipLaunchKernelGGL((long_bwd_join<T, true>), join, block, 0, st, a, b.map, b.split, (T *)b.dqkv, b.delta);
        });
        if (b.dense) {
            const PairWork &w = b.work;
            const unsigned distances = w.gd ? (2 * w.gd - 1) * (2 * w.gh - 1) * (2 * w.gw - 1) : b.map.tiles * b.map.tiles;
            hipLaunchKernelGGL((long_bwd_pairs<T, HD>), dim3(distances * a.heads * w.chunks), dim3(kAttnThreads),
                               0, st, a, b.map, w,
                               (const T *)b.qkv, b.lse, (const T *)b.dout, b.delta, b.dense);
        }
    });
}

}  // namespace aops

// ops_attention.hip -- C ABI of the windowed attention: checks, workspace, and the kernels that do not depend on the
// element type.
#include "ops_attention.hpp"

namespace aops {
namespace {

// bias[head][entry] = table[entry][head] * log2(e), and every head's entries in reverse
__global__ __launch_bounds__(256) void bias_rows(const float *__restrict__ table, float *__restrict__ bias,
                                                 float *__restrict__ rev, int entries, int heads)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= entries * heads) return;
    const int e = i / heads, head = i % heads;
    const float v = table[i] * kLog2e;
    bias[(size_t)head * entries + e] = v;
    rev[(size_t)head * entries + entries - 1 - e] = v;
}

// Long windows: where the tokens of a window lie, and what the tiles of 64 tokens hold.  A wave for a tile.
__global__ __launch_bounds__(256) void places_of(const WindowArgs a, const int *__restrict__ labels, int tiles,
                                                 PlaceAt *__restrict__ places, int *__restrict__ live,
                                                 TileAt *__restrict__ tiles_at)
{
    const long long tile = blockIdx.x * 4LL + threadIdx.x / 64;
    if (tile >= a.windows * tiles) return;  // (a whole wave)
    const int lane = threadIdx.x % 64, t = (int)(tile % tiles) * 64 + lane;
    PlaceAt p{-1, 0, -1, 0};
    if (t < a.n) {
        const Place at = place_of(a, labels, tile / tiles, t / a.ww / a.wh, t / a.ww % a.wh, t % a.ww);
        p = PlaceAt{at.token, corner(a, t), at.label, at.wrap};
    }
    places[tile * 64 + lane] = p;
    live[tile * 64 + lane] = p.label < 0 ? -1 : p.token;
    const TileAt what = tile_of(p, __shfl(p.corner, 0));
    if (lane == 0) tiles_at[tile] = what;
}

// dense[head][e] = the sum of the shares of the workgroups that have that head, in a fixed order: 64 elements for a
// workgroup, 16 threads on each four of them
__global__ __launch_bounds__(256) void pairs_fold(const float *__restrict__ pairs, float *__restrict__ dense, int heads,
                                                  int groups, int elements)
{
    __shared__ f32x4 fold[16][16];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int head = blockIdx.y, e = blockIdx.x * 64 + tx * 4;
    // workgroup b has head b / 8 % heads (walk_of): the k-th of a head's is ((k / 8) * heads + head) * 8 + k % 8
    const int mine = groups / heads;
    f32x4 s{};
#pragma unroll 8
    for (int k = ty; k < mine; k += 16)
        s += *(const f32x4 *)(pairs + (size_t)(((k / 8) * heads + head) * 8 + k % 8) * elements + e);
    fold[ty][tx] = s;
    __syncthreads();
    if (ty == 0) {
        f32x4 t{};
        for (int k = 0; k < 16; ++k) t += fold[k][tx];
        *(f32x4 *)(dense + (size_t)head * elements + e) = t;
    }
}

// dtable[e][head]: a wave sums the pairs of entry e, queries in its lanes.  `dense` is [head][slots][width]; a window's tokens start
// at `pitch * i` for i < copies (small windows share 16 slots), and block-diagonal units start every 16 * nb slots.
__global__ __launch_bounds__(256) void table_small(const WindowArgs a, const float *__restrict__ dense,
                                                   float *__restrict__ dtable, int nb)
{
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int e = blockIdx.x * 4 + wave, head = blockIdx.y;
    if (e >= a.entries) return;
    const int dw = e % a.rh - (a.ww - 1), dh = e / a.rh % (2 * a.wh - 1) - (a.wh - 1), dd = e / a.rd - (a.wd - 1);
    const int fit = nb == 1 ? 16 / a.n : 1;
    const int r = lane % (16 * nb);
    float s = 0.f;
    if (r < fit * a.n) {
        const int t = r % a.n;
        const int tw = t % a.ww - dw, th = t / a.ww % a.wh - dh, td = t / a.ww / a.wh - dd;
        if (tw >= 0 && tw < a.ww && th >= 0 && th < a.wh && td >= 0 && td < a.wd) {
            const int key = r / a.n * a.n + (td * a.wh + th) * a.ww + tw;
            s = dense[((size_t)head * 64 + lane) * 16 * nb + key];
        }
    }
    s = group_sum<64>(s);
    if (lane == 0) dtable[(size_t)e * a.heads + head] = s;
}

// The shares of `dense`, into the first, in order.  (Summed where they are read, by few workgroups, 113 shares of 3 distances and 3
// heads took 790 us; here 11, and 8 there.)
__global__ __launch_bounds__(256) void shares_fold(float *dense, int shares, long long count)
{
    const long long i = blockIdx.x * 256LL + threadIdx.x;
    if (i >= count) return;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < shares; ++k) s += dense[k * count + i];
    dense[i] = s;
}

// dtable[e][head] for long windows that tiles of ed x eh x ew = 64 tokens divide: dense is [distance of tiles][head][64][64]
// (long_bwd_pairs).  For each query of a tile the key at this distance is one token of one tile: 64 terms, a quarter for
// each wave.  Neighbouring lanes have neighbouring distances: they read neighbouring keys.
__global__ __launch_bounds__(256) void table_tiled(const WindowArgs a, const PairWork w, const float *__restrict__ dense,
                                                   float *__restrict__ dtable)
{
    __shared__ float fold[4][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, head = blockIdx.y;
    const int e = min(blockIdx.x * 64 + lane, a.entries - 1);
    const int dw = e % a.rh - (a.ww - 1), dh = e / a.rh % (2 * a.wh - 1) - (a.wh - 1), dd = e / a.rd - (a.wd - 1);
    // One axis: tokens i of a query's tile, `size` long, at distance d.  With m = d mod size the key is i - m in the tile
    // (d - m) / size away for i >= m, and i - m + size in the tile one further for i < m: two cases, each with what it adds
    // to the distance's number (distances are counted as 0, 1, -1, 2, -2, ...) and to the key's place.
    // The sizes are powers of two.
    struct Axis {
        int m, far[2], key[2];
        __device__ Axis(int d, int log, int tiles, int distances, int pitch) : m(d & ((1 << log) - 1))
        {
            for (int k = 0; k < 2; ++k) {
                const int D = ((d - m) >> log) + k;
                far[k] = abs(D) >= tiles ? -(1 << 24) : (D > 0 ? 2 * D - 1 : -2 * D) * distances;  // beyond the window
                key[k] = ((k << log) - m) * pitch;
            }
        }
    };
    const int lw = __builtin_ctz(a.ww / w.gw), lh = __builtin_ctz(a.wh / w.gh), ld = __builtin_ctz(a.wd / w.gd);
    const Axis x(dw, lw, w.gw, 1, 1), y(dh, lh, w.gh, 2 * w.gw - 1, 1 << lw);
    const Axis z(dd, ld, w.gd, (2 * w.gh - 1) * (2 * w.gw - 1), 1 << (lw + lh));
    const unsigned stride = (unsigned)a.heads * 4096;
    float s = 0.f;
    const float *from = dense + (size_t)head * 4096;
#pragma unroll 8
    for (int q = wave * 16; q < wave * 16 + 16; ++q) {  // (the same q in every lane: its coordinates are scalars)
        const int ix = q & ((1 << lw) - 1), iy = q >> lw & ((1 << lh) - 1), iz = q >> (lw + lh);
        const int bx = ix < x.m, by = iy < y.m, bz = iz < z.m;
        const int far = (bx ? x.far[1] : x.far[0]) + (by ? y.far[1] : y.far[0]) + (bz ? z.far[1] : z.far[0]);
        const int key = (bx ? x.key[1] : x.key[0]) + (by ? y.key[1] : y.key[0]) + (bz ? z.key[1] : z.key[0]);
        // (the key's coordinates are the query's plus these: the query's place in the tile is q itself)
        if (far >= 0) s += from[(unsigned long long)(unsigned)far * stride + (unsigned)(q * 65 + key)];
    }
    fold[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && (int)blockIdx.x * 64 + lane < a.entries)
        dtable[(size_t)e * a.heads + head] = (fold[0][lane] + fold[1][lane]) + (fold[2][lane] + fold[3][lane]);
}

// dtable[e][head] for other long windows, from dense [head][n][n]: the workgroup has the entries of one (dd, dh) and goes
// through the queries' rows; a lane has one dw, so that neighbouring lanes read neighbouring keys.  Sixteen waves take every sixteenth
// row.  Eight queries' loads are in flight, also of queries that have no such key (not added): 1386 tokens, 8 heads, 50 us; one
// after the other, by four waves, 97.
__global__ __launch_bounds__(1024) void table_long(const WindowArgs a, const float *__restrict__ dense,
                                                  float *__restrict__ dtable)
{
    __shared__ float fold[16][64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int head = blockIdx.z;
    const int dh = (int)blockIdx.y % (2 * a.wh - 1) - (a.wh - 1), dd = (int)blockIdx.y / (2 * a.wh - 1) - (a.wd - 1);
    const int e = blockIdx.x * 64 + lane, dw = min(e, a.rh - 1) - (a.ww - 1);
    const int lo = max(dw, 0), hi = min(a.ww, a.ww + dw);  // queries whose key is in the row: one at least
    float s = 0.f;
    const int rows = a.wd * a.wh;
    for (int row = wave; row < rows; row += 16) {
        const int qd = row / a.wh, qh = row % a.wh, kd = qd - dd, kh = qh - dh;
        if (kd < 0 || kd >= a.wd || kh < 0 || kh >= a.wh) continue;
        const float *line = dense + ((size_t)head * a.n + (size_t)row * a.ww) * a.n + (kd * a.wh + kh) * a.ww - dw;
        for (int first = 0; first < a.ww; first += 8) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int qw = min(max(first + k, lo), hi - 1);
                x[k] = line[(size_t)qw * a.n + qw];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) s += first + k >= lo && first + k < hi ? x[k] : 0.f;
        }
    }
    fold[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || e >= a.rh) return;
    float t = 0.f;
    for (int w = 0; w < 16; ++w) t += fold[w][lane];
    dtable[((size_t)blockIdx.y * a.rh + e) * a.heads + head] = t;
}

__global__ void fill_zero(float *p, long long n)
{
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) p[i] = 0.f;
}

int small_nb(int n) { return n <= 16 ? 1 : n <= 32 ? 2 : 4; }

// Workgroups for windows of at most 64 tokens: a multiple of 8 * heads (walk_of), about `target`, at most one for
// each (tile, head).
int small_groups(const WindowArgs &a, int target)
{
    const int nb = small_nb(a.n);
    const int per = 4 / nb * (nb == 1 ? 16 / a.n : 1);
    const long long tiles = (a.windows + per - 1) / per;
    const long long most = (tiles + 7) / 8;           // times 8 * heads
    long long want = target / (8LL * a.heads);
    if (want < 1) want = 1;
    return (int)((want < most ? want : most) * 8 * a.heads);
}
// Measured with 8192 windows of 64 tokens in fp32 (2 heads of 32 channels), and 16384 of 4 (4 heads): forward 138 and 71 us for
// 2048 workgroups, 143 and 68 for 1024, 147 and 66 for 4096; backward with the sum of the table's shares 333 and 103 us for
// 768, 331 and 106 for 512, 335 and 104 for 1024.
int fwd_groups(const WindowArgs &a) { return small_groups(a, 2048); }
int bwd_groups(const WindowArgs &a) { return small_groups(a, 768); }

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

// 0 ok, > 0 invalid, -1 nothing to do
int make_args(const char *what, const artemis_ops_window *w, WindowArgs &a)
{
    if (!w) return fail(hipErrorInvalidValue, "%s: NULL description", what);
    if (w->B < 0 || w->D < 0 || w->H < 0 || w->W < 0)
        return fail(hipErrorInvalidValue, "%s: negative dimension B=%d D=%d H=%d W=%d", what, w->B, w->D, w->H, w->W);
    if (w->dtype != ARTEMIS_OPS_F32 && w->dtype != ARTEMIS_OPS_BF16 && w->dtype != ARTEMIS_OPS_F16)
        return fail(hipErrorInvalidValue, "%s: unknown dtype %d", what, w->dtype);
    if (w->heads < 1 || w->heads > 1024 || w->head_dim < 4 || w->head_dim > 128 || w->head_dim % 4)
        return fail(hipErrorInvalidValue, "%s: heads=%d head_dim=%d (heads 1..1024, head_dim a multiple of 4 up to 128)",
                    what, w->heads, w->head_dim);
    if (w->wd < 1 || w->wh < 1 || w->ww < 1 || w->wd > 4096 || w->wh > 4096 || w->ww > 4096 ||
        (long long)w->wd * w->wh * w->ww > 4096)
        return fail(hipErrorInvalidValue, "%s: window (%d, %d, %d) must hold 1..4096 tokens", what, w->wd, w->wh, w->ww);
    if (w->D % w->wd || w->H % w->wh || w->W % w->ww)
        return fail(hipErrorInvalidValue, "%s: map (%d, %d, %d) is not a multiple of the window (%d, %d, %d)", what, w->D,
                    w->H, w->W, w->wd, w->wh, w->ww);
    if (w->shift_d < 0 || w->shift_d >= w->wd || w->shift_h < 0 || w->shift_h >= w->wh || w->shift_w < 0 ||
        w->shift_w >= w->ww)
        return fail(hipErrorInvalidValue, "%s: shift (%d, %d, %d) must lie in [0, window)", what, w->shift_d, w->shift_h,
                    w->shift_w);
    if (w->label_maps < 0 || (w->label_maps > 1 && w->label_maps != w->B))
        return fail(hipErrorInvalidValue, "%s: label_maps=%d must be 0, 1 or B", what, w->label_maps);
    if (!(w->outside <= 0.f)) return fail(hipErrorInvalidValue, "%s: outside=%g must be <= 0", what, w->outside);
    if (!(fabsf(w->scale) <= 3.4e38f)) return fail(hipErrorInvalidValue, "%s: scale must be finite", what);
    const double tokens = (double)w->B * w->D * w->H * w->W;
    const int n = w->wd * w->wh * w->ww;
    if (tokens >= 2147483648.0 || tokens / n * w->heads * ((n + 63) / 64) >= 16777216.0 * 64 ||
        (n > 64 && tokens / n * w->heads * ((n + 63) / 64) >= 16777216.0))
        return fail(hipErrorInvalidValue, "%s: too many tokens or windows * heads", what);
    a = WindowArgs{w->B, w->D, w->H, w->W, w->heads, w->head_dim, w->wd, w->wh, w->ww, n, w->shift_d, w->shift_h,
                   w->shift_w, w->D / w->wd, w->H / w->wh, w->W / w->ww, w->label_maps, (2 * w->wh - 1) * (2 * w->ww - 1),
                   2 * w->ww - 1, (2 * w->wd - 1) * (2 * w->wh - 1) * (2 * w->ww - 1), 0, Divider(), Divider(), Divider(), w->scale, 0.f};
    a.windows = (long long)w->B * a.nd * a.nh * a.nw;
    if (a.windows) a.by_nd = Divider(a.nd), a.by_nh = Divider(a.nh), a.by_nw = Divider(a.nw);
    // a finite `outside` stays finite in the exponent of 2; beyond -1e30 nothing else counts beside it anyway
    a.outside2 = w->outside == -INFINITY ? -INFINITY : (w->outside < -1e30f ? -1e30f : w->outside) * kLog2e;
    return a.windows == 0 ? -1 : 0;
}

// How the table's gradient goes through a long window's pairs (long_bwd_pairs): 64 tokens in a row of the raster that fill
// whole rows, or whole planes, evenly; and shares of the windows until there is work for about 1024 workgroups.
PairWork pair_work(const WindowArgs &a)
{
    PairWork w{0, 0, 0, 1};
    const int plane = a.wh * a.ww;
    if (a.ww % 64 == 0)
        w = {a.wd, a.wh, a.ww / 64, 1};
    else if (64 % a.ww == 0 && a.wh % (64 / a.ww) == 0)
        w = {a.wd, a.wh / (64 / a.ww), 1, 1};
    else if (64 % plane == 0 && a.wd % (64 / plane) == 0)
        w = {a.wd / (64 / plane), 1, 1, 1};
    const long long tiles = (a.n + 63) / 64;
    const long long groups = (w.gd ? (2LL * w.gd - 1) * (2 * w.gh - 1) * (2 * w.gw - 1) : tiles * tiles) * a.heads;
    const long long want = 1024 / groups;
    w.chunks = (int)(want < 1 ? 1 : want < a.windows ? want : a.windows);
    return w;
}

// Workgroups that share a tile's partners where there are few tiles: about 1024 in all (as many as the card holds of them), each
// with four partners at least.  One window of 4096 tokens, 8 heads of 32 bf16 channels, 512 tiles: forward, dQ, dK and dV with
// the joins take 155 us, 156 without splitting, 161 at 2048 workgroups, 185 at 4096.
constexpr long long kSplitTarget = 1024;
int split_count(const WindowArgs &a)
{
    const long long tiles = (a.n + 63) / 64, groups = a.windows * a.heads * tiles;
    const long long want = kSplitTarget / groups, most = tiles / 4;
    return (int)(want < 1 || most < 1 ? 1 : want < most ? want : most);
}

struct Layout {
    size_t bias, rev, places, live, tiles, pairs, dense, delta, split_a, split_b, split_rows, spare, total;
    PairWork work;
    int splits;
};
Layout layout_of(const WindowArgs &a, bool backward, bool need_dtable, bool table)
{
    Layout l{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round16(bytes);
        return here;
    };
    if (a.n > 64) {
        const size_t tiles = (size_t)(a.n + 63) / 64;
        l.places = take(a.windows * tiles * 64 * sizeof(PlaceAt));
        l.live = take(a.windows * tiles * 64 * sizeof(int));
        l.tiles = take(a.windows * tiles * sizeof(TileAt));
        if (table) {
            l.bias = take((size_t)a.entries * a.heads * 4);
            l.rev = take((size_t)a.entries * a.heads * 4);
        }
        const size_t lines = (size_t)a.windows * a.heads * tiles * 64;
        if (backward) l.delta = take(lines * 4);
        l.splits = split_count(a);
        if (l.splits > 1) {
            l.split_a = take(l.splits * lines * a.hd * 4);
            if (backward) l.split_b = take(l.splits * lines * a.hd * 4);
            l.split_rows = take(l.splits * lines * 2 * 4);
        }
        if (backward && need_dtable) {
            l.work = pair_work(a);
            const PairWork &w = l.work;
            l.dense = take(w.gd ? (size_t)w.chunks * (2 * w.gd - 1) * (2 * w.gh - 1) * (2 * w.gw - 1) * a.heads * 4096 * 4
                                : (size_t)w.chunks * a.heads * a.n * a.n * 4);
        }
    } else {
        l.spare = take(kSpareBytes);
        if (backward && need_dtable) {
            const int nb = small_nb(a.n);
            l.pairs = take((size_t)bwd_groups(a) * 64 * 16 * nb * 4);
            l.dense = take((size_t)a.heads * 64 * 16 * nb * 4);
        }
    }
    l.total = at;
    return l;
}

bool aligned4(const void *p, int dtype) { return ((size_t)p & (dtype == ARTEMIS_OPS_F32 ? 15 : 7)) == 0; }

// Long windows: what the kernels find in the workspace; fills the maps
void long_buffers(AttnBuffers &b, const WindowArgs &a, const Layout &l, const float *table, const int *labels, char *ws,
                  hipStream_t st)
{
    const int last = 63;  // of a tile: how far its corners reach
    const int reach = last / a.ww / a.wh * a.rd + last / a.ww % a.wh * a.rh + last % a.ww;
    b.even = pair_work(a).gd > 0 && a.ww % 4 == 0 && 2 * reach + 4 <= kSpan;
    b.split = Split{l.splits, (float *)(ws + l.split_a), (float *)(ws + l.split_b), (float *)(ws + l.split_rows)};
    LongMap m{};
    m.tiles = (a.n + 63) / 64;
    PlaceAt *places = (PlaceAt *)(ws + l.places);
    TileAt *tiles = (TileAt *)(ws + l.tiles);
    m.places = places;
    m.tiles_at = tiles;
    int *live = (int *)(ws + l.live);
    m.live = live;
    hipLaunchKernelGGL(places_of, dim3((unsigned)((a.windows * m.tiles + 3) / 4)), dim3(256), 0, st, a, labels, m.tiles, places,
                       live, tiles);
    if (table) {
        float *bias = (float *)(ws + l.bias), *rev = (float *)(ws + l.rev);
        const int n = a.entries * a.heads;
        hipLaunchKernelGGL(bias_rows, dim3((n + 255) / 256), dim3(256), 0, st, table, bias, rev, a.entries, a.heads);
        m.bias = bias;
        m.rev = rev;
    }
    b.map = m;
}

}  // namespace
}  // namespace aops

using namespace aops;

extern "C" {

size_t artemis_ops_window_attention_lse_count(const artemis_ops_window *w)
{
    WindowArgs a;
    if (make_args("artemis_ops_window_attention", w, a)) return 0;
    return a.n > 64 ? (size_t)a.windows * a.heads * ((a.n + 63) / 64) * 64 : 0;
}

size_t artemis_ops_window_attention_workspace_bytes(const artemis_ops_window *w, int backward, int need_dtable)
{
    WindowArgs a;
    if (make_args("artemis_ops_window_attention", w, a)) return 0;
    return layout_of(a, backward != 0, need_dtable != 0, true).total;
}

int artemis_ops_window_attention_forward(const artemis_ops_window *w, const void *qkv, const float *table,
                                         const int *labels, void *out, float *lse, void *workspace,
                                         size_t workspace_bytes, void *stream)
{
    const char *what = "artemis_ops_window_attention_forward";
    WindowArgs a;
    if (const int rc = make_args(what, w, a)) return rc > 0 ? rc : 0;
    if (!qkv || !out) return fail(hipErrorInvalidValue, "%s: NULL tensor pointer", what);
    if (!labels != !w->label_maps) return fail(hipErrorInvalidValue, "%s: labels and label_maps do not match", what);
    if (!aligned4(qkv, w->dtype) || !aligned4(out, w->dtype))
        return fail(hipErrorInvalidValue, "%s: tensors must be aligned to 4 elements", what);
    const Layout l = layout_of(a, false, false, table != nullptr);
    if (l.total && (!workspace || workspace_bytes < l.total || ((size_t)workspace & 15)))
        return fail(hipErrorInvalidValue, "%s: workspace of %zu bytes aligned to 16 needed", what, l.total);
    hipStream_t st = (hipStream_t)stream;
    AttnBuffers b{};
    b.qkv = qkv;
    b.table = table;
    b.labels = labels;
    b.out = out;
    b.lse = lse;
    b.groups = a.n <= 64 ? fwd_groups(a) : 0;
    b.spare = (char *)workspace + l.spare;
    if (a.n > 64) long_buffers(b, a, l, table, labels, (char *)workspace, st);
    if (w->dtype == ARTEMIS_OPS_F32)
        launch_attention_fwd<float>(a, b, st);
    else if (w->dtype == ARTEMIS_OPS_BF16)
        launch_attention_fwd<__bf16>(a, b, st);
    else
        launch_attention_fwd<_Float16>(a, b, st);
    return check_launch(what);
}

int artemis_ops_window_attention_backward(const artemis_ops_window *w, const void *qkv, const float *table,
                                          const int *labels, const void *out, const float *lse, const void *dout,
                                          void *dqkv, float *dtable, void *workspace, size_t workspace_bytes,
                                          void *stream)
{
    const char *what = "artemis_ops_window_attention_backward";
    WindowArgs a;
    const int made = make_args(what, w, a);
    if (made > 0) return made;
    hipStream_t st = (hipStream_t)stream;
    if (made < 0) {  // no tokens: the table's gradient is a sum over nothing
        if (dtable) hipLaunchKernelGGL(fill_zero, dim3(64), dim3(256), 0, st, dtable, (long long)a.entries * a.heads);
        return check_launch(what);
    }
    const bool is_long = a.n > 64;
    if (!qkv || !dout || !dqkv || (is_long && (!out || !lse)))
        return fail(hipErrorInvalidValue, "%s: NULL tensor pointer", what);
    if (!labels != !w->label_maps) return fail(hipErrorInvalidValue, "%s: labels and label_maps do not match", what);
    if (!aligned4(qkv, w->dtype) || !aligned4(out, w->dtype) || !aligned4(dout, w->dtype) || !aligned4(dqkv, w->dtype))
        return fail(hipErrorInvalidValue, "%s: tensors must be aligned to 4 elements", what);
    const Layout l = layout_of(a, true, dtable != nullptr, table != nullptr);
    if (l.total && (!workspace || workspace_bytes < l.total || ((size_t)workspace & 15)))
        return fail(hipErrorInvalidValue, "%s: workspace of %zu bytes aligned to 16 needed", what, l.total);
    char *ws = (char *)workspace;
    AttnBuffers b{};
    b.qkv = qkv;
    b.table = table;
    b.labels = labels;
    b.out_in = out;
    b.lse = (float *)lse;
    b.dout = dout;
    b.dqkv = dqkv;
    b.groups = is_long ? 0 : bwd_groups(a);
    b.spare = ws + l.spare;
    if (is_long) b.delta = (float *)(ws + l.delta);
    if (dtable) {
        b.dense = (float *)(ws + l.dense);
        if (!is_long) b.pairs = (float *)(ws + l.pairs);
    }
    if (is_long) long_buffers(b, a, l, table, labels, ws, st);
    b.work = l.work;
    if (w->dtype == ARTEMIS_OPS_F32)
        launch_attention_bwd<float>(a, b, st);
    else if (w->dtype == ARTEMIS_OPS_BF16)
        launch_attention_bwd<__bf16>(a, b, st);
    else
        launch_attention_bwd<_Float16>(a, b, st);
    if (dtable && is_long) {
        const PairWork &p = b.work;
        const long long count = p.gd ? (2LL * p.gd - 1) * (2 * p.gh - 1) * (2 * p.gw - 1) * a.heads * 4096
                                     : (long long)a.heads * a.n * a.n;
        if (p.chunks > 1)
            hipLaunchKernelGGL(shares_fold, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, st, b.dense, p.chunks, count);
        if (p.gd)
            hipLaunchKernelGGL(table_tiled, dim3((a.entries + 63) / 64, a.heads), dim3(256), 0, st, a, p, b.dense, dtable);
        else
            hipLaunchKernelGGL(table_long, dim3((a.rh + 63) / 64, (2 * a.wd - 1) * (2 * a.wh - 1), a.heads), dim3(1024), 0, st, a,
                               b.dense, dtable);
    } else if (dtable) {
        const int nb = small_nb(a.n), elements = 64 * 16 * nb;
        hipLaunchKernelGGL(pairs_fold, dim3(elements / 64, a.heads), dim3(256), 0, st, b.pairs, b.dense, a.heads, b.groups,
                           elements);
        hipLaunchKernelGGL(table_small, dim3((a.entries + 3) / 4, a.heads), dim3(256), 0, st, a, b.dense, dtable, nb);
    }
    return check_launch(what);
}

}  // extern "C"

/*
 * artemis_ops.h -- C ABI of libartemis_ops.so: the operators of the Sep-STS encoder and of the
 * optimizer step as hand-written CDNA4 (gfx950) HIP kernels: layer norm, windowed attention with a
 * relative-position bias and region masks, and AdamW over many tensors.
 *
 * Conventions (those of artemis_synth.h)
 *  - plain C: pointers are DEVICE pointers on the current HIP device unless a comment says HOST.
 *  - the library never allocates, frees or retains caller memory; it only enqueues kernels on
 *    `stream` (a hipStream_t; NULL = the null stream) and returns.  It enqueues no memset and no
 *    copy, so every call can be captured into a HIP graph.
 *  - every function returns 0 on success or a hipError_t value (> 0); arguments that fail
 *    validation give hipErrorInvalidValue (1) before any GPU work.  artemis_ops_last_error()
 *    returns a thread-local description of the last failure on the calling thread.  No exception
 *    crosses the boundary.
 *  - entry points are reentrant and the library has no mutable state.
 *  - results are bit-reproducible from run to run: no atomics.
 *  - empty problems are a successful no-op (gradients of parameters are still written: zeros).
 */
#ifndef ARTEMIS_OPS_H
#define ARTEMIS_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ARTEMIS_OPS_ABI_VERSION 1

/* element types */
#define ARTEMIS_OPS_F32 0
#define ARTEMIS_OPS_BF16 1
#define ARTEMIS_OPS_F16 2

/* ---- layer norm over the last dimension -------------------------------------------------------
 *   y[r, c] = (x[r, c] - mean_r) * rstd_r * weight[c] + bias[c],  rstd = (var + eps)^-1/2,
 * var the mean of the squared deviations.  x and y are (rows, cols) contiguous of `dtype`, weight and
 * bias (either may be NULL: 1 and 0) fp32.  mean and rstd (rows each, fp32) are written for the backward
 * pass; both may be NULL.  Reference: nn.LayerNorm in model/sep_sts_layer.py:251,257.
 * cols >= 1 where rows > 0; rows below 2^31, cols below 2^30. */
int artemis_ops_layer_norm_forward(const void *x, const float *weight, const float *bias, void *y,
                                   float *mean, float *rstd, long long rows, long long cols, float eps,
                                   int dtype, void *stream);

/* dx (rows, cols) of `dtype`; dweight and dbias (cols) fp32; each may be NULL.  `workspace`: at least
 * artemis_ops_layer_norm_workspace_bytes bytes when dweight or dbias is asked for. */
int artemis_ops_layer_norm_backward(const void *x, const void *dy, const float *weight,
                                    const float *mean, const float *rstd, void *dx, float *dweight,
                                    float *dbias, long long rows, long long cols, int dtype,
                                    void *workspace, size_t workspace_bytes, void *stream);
size_t artemis_ops_layer_norm_workspace_bytes(long long rows, long long cols, int dtype);

/* ---- windowed attention ----------------------------------------------------------------------
 * Tokens lie on a (B, D, H, W) map, cut into windows of (wd, wh, ww) tokens after a cyclic shift: the
 * window at (i, j, k) holds the map positions ((i*wd + t + shift_d) mod D, ...).  Within a window, for
 * each head,
 *     S = scale * q k^T + T[rel(a, b)] + M(a, b),   P = softmax(S) over b,   out_a = sum_b P(a, b) v_b
 *  rel(a, b)  the difference of the tokens' coordinates in the window in mixed radix: ((ad - bd + wd - 1)
 *             * (2wh - 1) + ah - bh + wh - 1) * (2ww - 1) + aw - bw + ww - 1.
 *  M(a, b)    0 for tokens of one region, `outside` (-inf, or a finite number <= 0) for tokens of two
 *             regions; a region is what the shift wrapped around the same axes and what carries the same
 *             label.
 *  labels     (label_maps, D, H, W) int32 with label_maps = 1 (shared) or B, or NULL.  A token of a
 *             negative label is padding: its q, k, v and dout are not used, its output and gradients
 *             are 0.
 * Where M leaves a row nothing (only padding does) the output is 0.
 *   qkv    (B, D, H, W, 3, heads, head_dim) contiguous of `dtype`, aligned to 4 elements
 *   table  ((2wd-1)(2wh-1)(2ww-1), heads) fp32, or NULL: no bias
 *   out    (B, D, H, W, heads, head_dim) of `dtype`
 *   lse    fp32, artemis_ops_window_attention_lse_count elements: what the backward pass needs of the
 *          rows' softmax; may be NULL for a forward pass alone, and where the count is 0.
 * Limits: heads at most 1024; head_dim a multiple of 4, at most 128; n = wd*wh*ww at most 4096; D, H, W multiples of the
 * window; 0 <= shift < window; B*D*H*W below 2^31; windows * heads below 2^30 for n <= 64, windows * heads * ceil(n / 64)
 * below 2^24 for longer windows.  The size functions return 0 for what is refused.
 * Workspace: 1 KB for n <= 64, with dtable some 12 MB, or 144 KB for each head where that is more.  Longer windows: 20 bytes a
 * token, two copies of the table, in a backward pass 4 bytes a token and head; where there are fewer than 1024 tiles of 64
 * tokens and a head, up to 1024 * 64 * (head_dim + 2) * 4 bytes (backward: twice that) for their shares.  With dtable the
 * sums of dS: heads * n * n * 4 bytes where runs of 64 tokens do not tile the window evenly (16 heads of 3844 tokens: 946 MB),
 * 16 KB for each head and distance of two tiles where they do, both for as many shares of the windows as make about 1024
 * workgroups.
 * Reference: model/sep_sts_layer.py:108-219 (attention), :262-337 (shift and mask). */
typedef struct artemis_ops_window {
    int B, D, H, W;
    int heads, head_dim;
    int wd, wh, ww;
    int shift_d, shift_h, shift_w;
    int label_maps;
    int dtype;
    float scale, outside;
} artemis_ops_window;

size_t artemis_ops_window_attention_lse_count(const artemis_ops_window *w /* HOST */);
size_t artemis_ops_window_attention_workspace_bytes(const artemis_ops_window *w /* HOST */, int backward,
                                                    int need_dtable);
int artemis_ops_window_attention_forward(const artemis_ops_window *w /* HOST */, const void *qkv,
                                         const float *table, const int *labels, void *out, float *lse,
                                         void *workspace, size_t workspace_bytes, void *stream);
/* dqkv (like qkv) and dtable (like table), fully overwritten; dtable may be NULL. */
int artemis_ops_window_attention_backward(const artemis_ops_window *w /* HOST */, const void *qkv,
                                          const float *table, const int *labels, const void *out,
                                          const float *lse, const void *dout, void *dqkv, float *dtable,
                                          void *workspace, size_t workspace_bytes, void *stream);

/* ---- AdamW over many tensors -----------------------------------------------------------------
 *   p *= 1 - lr*weight_decay;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;
 *   p -= lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * in fp32, rounded once to the parameter's type.  `tensors` is a HOST array, read during the call.
 * Parameters and gradients are of `dtype`, `count` elements each.
 *  bits = 32: m, v fp32.
 *  bits = 8:  m, v uint8 (count each) with one int32 base for each 256 elements (m_base, v_base).  A code
 *             stands for the fp32 number whose top bits (sign excluded) are code + base above 20 zero bits:
 *             3 bits of mantissa; 0 stands for 0.  v uses codes 0..255, m a sign (bit 7) and 0..127.
 *             The new moments are rounded up or down at random with the right mean, by a counter-based
 *             generator: (seed, step, the element's place), where the tensors follow each other at
 *             multiples of 256 elements.  A gradient that is not finite spoils the 256 elements of its
 *             group.
 * step >= 1; a tensor has at most 2^33 elements.  bits = 8 holds at most 2^32 places, counted in groups of 256. */
typedef struct artemis_ops_tensor {
    void *param;
    const void *grad;
    void *m;
    void *v;
    int *m_base;
    int *v_base;
    long long count;
} artemis_ops_tensor;

int artemis_ops_adamw(const artemis_ops_tensor *tensors /* HOST */, int n_tensors, int dtype, int bits,
                      double lr, double beta1, double beta2, double eps, double weight_decay,
                      long long step, unsigned seed, void *stream);

/* 8-bit moments as fp32: out[i] (count elements) from codes and bases.  tensors[i].param = out,
 * .m = codes, .m_base = bases; the other pointers are not used. */
int artemis_ops_moments_from_8bit(const artemis_ops_tensor *tensors /* HOST */, int n_tensors,
                                  int is_signed, void *stream);

const char *artemis_ops_version(void);
const char *artemis_ops_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* ARTEMIS_OPS_H */

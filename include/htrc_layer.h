/* C ABI of the operators around the flat attention in a video transformer's layer (libhtrc_flat.so, sm_100a):
 *   rotary positions over several axes (time, height, width), with the per-head RMS norm before them and the
 *   token-major -> head-major reorder in the same pass, forward and backward;
 *   cross attention of the tokens to an encoder's states of another length, forward and backward;
 *   layer norm with a learned affine and a modulation per batch entry, forward and backward;
 *   the matrix product in 8-bit integers with a scale per token and channel, and the rows it reads.
 *
 * Pointers are device pointers on the current CUDA device unless stated otherwise; the caller owns all memory;
 * no entry point allocates or synchronises, so every call can be captured in a CUDA graph after the first one
 * on a device.  Return values are the HTRC_OK / HTRC_ERR_* codes of htrc_flat.h.  Strides count elements. */
#ifndef HTRC_LAYER_H_
#define HTRC_LAYER_H_

#include "htrc_flat.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { HTRC_LAYER_F32 = 0, HTRC_LAYER_BF16 = 1, HTRC_LAYER_F16 = 2, HTRC_LAYER_I32 = 3, HTRC_LAYER_U8 = 4,
       HTRC_LAYER_I8 = 5 }; /* types */

enum { HTRC_ROTARY_MAX_AXES = 4, HTRC_ROTARY_MAX_DIM = 256, HTRC_ROTARY_MAX_HEADS = 1024 };
/* pairs of a head's rotated width R: (2 i, 2 i + 1), or (i, i + R / 2) */
enum { HTRC_ROTARY_INTERLEAVED = 0, HTRC_ROTARY_HALF = 1 };

/* One rotated tensor: `in` (forward: x; backward: dy) -> `out` (forward: y; backward: dx), each
 * [batch][token][head][dim] through its strides (batch, token, head; the dim stride is 1). */
typedef struct {
  const void* in;
  int64_t in_stride[3];
  void* out;
  int64_t out_stride[3];
  const void* x;          /* backward with a weight: the forward's input, else NULL */
  int64_t x_stride[3];
  const void* weight;     /* [dim] RMS-norm weight, or NULL for no norm */
  void* dweight;          /* backward with a weight: [dim] gradient in weight_dtype */
  int32_t weight_dtype;   /* HTRC_LAYER_F32 / BF16 / F16 */
  int32_t heads;          /* 1 .. HTRC_ROTARY_MAX_HEADS */
} HtrcRotaryTensor;

typedef struct {
  HtrcRotaryTensor tensor[2];   /* q and k (or one tensor) */
  int32_t n_tensors;            /* 1 or 2 */
  int32_t dtype;                /* HTRC_LAYER_F32 / BF16 / F16, of in, x and out */
  int64_t batch, tokens;        /* >= 0 */
  int32_t dim;                  /* 2 .. HTRC_ROTARY_MAX_DIM */
  int32_t n_axes;               /* 1 .. HTRC_ROTARY_MAX_AXES */
  int32_t axis_width[4];        /* rotated elements per axis, even; the sum R <= dim, the rest is not rotated */
  int32_t pairs;                /* HTRC_ROTARY_INTERLEAVED / HALF */
  const void* positions;        /* [batch][token][axis], int32 or float32 */
  int32_t position_dtype;       /* HTRC_LAYER_I32 / F32 */
  int64_t position_stride[3];
  double theta;                 /* pair i of an axis of width w turns by position * theta^(-2 i / w) radians */
  const double* freqs;          /* HOST: R / 2 frequencies (radians per position) instead of theta's, or NULL */
  float eps;                    /* of the norm: x * rsqrt(mean(x^2) + eps) * weight */
  void* workspace;              /* backward with a weight: htrc_rotary_workspace_size() bytes */
  size_t workspace_bytes;
} HtrcRotaryArgs;

int htrc_rotary_forward(const HtrcRotaryArgs* args, htrc_stream_t stream);
/* dx = the transposed rotation of dy, through the norm where there is a weight; dweight summed in a fixed order */
int htrc_rotary_workspace_size(const HtrcRotaryArgs* args, size_t* bytes);
int htrc_rotary_backward(const HtrcRotaryArgs* args, htrc_stream_t stream);

/* Cross attention: out = softmax(scale * q k^T + mask) v over the keys that the mask and the key lengths leave, and
 * lse = the natural log of the softmax's sum.  A row with no key left gives 0 and -infinity.  Query head h reads
 * key head h / (heads / kv_heads).  q, k, v, out and their gradients are [batch][token][head][dim] through their
 * strides (batch, token, head; the dim stride is 1), rows 16-byte aligned, dim a multiple of 8. */
enum { HTRC_CROSS_MAX_DIM = 128 };

typedef struct {
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  void* out;              /* forward: written; backward: the forward's output */
  int64_t out_stride[3];
  float* lse;             /* [batch][heads][queries]; forward: written unless NULL; backward: the forward's */
  int64_t batch, queries, keys;   /* >= 0 */
  int32_t heads, kv_heads;        /* heads a multiple of kv_heads */
  int32_t dim;                    /* 8 .. HTRC_CROSS_MAX_DIM, a multiple of 8 */
  int32_t dtype;                  /* HTRC_LAYER_BF16 / F16 */
  float scale;                    /* > 0 */
  const int32_t* key_lengths;     /* [batch] keys per entry (clamped to 0 .. keys), or NULL */
  const void* mask;               /* [batch][head][query][key] through mask_stride (0: broadcast), or NULL */
  int32_t mask_dtype;             /* HTRC_LAYER_U8: nonzero keeps; F32 / BF16 / F16: added, -infinity excludes */
  int64_t mask_stride[4];
  int32_t* status;                /* device word the guards OR their bits into (zeroed once; htrc_flat_status
                                   * reads and clears it), or NULL */
  /* backward only */
  const void* dout;
  int64_t dout_stride[3];
  const float* dlse;              /* gradient of lse, laid out as lse, or NULL */
  void *dq, *dk, *dv;
  int64_t dq_stride[3], dk_stride[3], dv_stride[3];
  /* both: the direction's _workspace_size() bytes (the forward's may be 0), 256-byte aligned */
  void* workspace;
  size_t workspace_bytes;
} HtrcCrossArgs;

/* Keys and values that no query may see (past a length, or excluded by a mask that is the same for every query) are
 * never computed with, whatever they hold. */
int htrc_cross_forward_workspace_size(const HtrcCrossArgs* args, size_t* bytes);
int htrc_cross_forward(const HtrcCrossArgs* args, htrc_stream_t stream);
int htrc_cross_backward_workspace_size(const HtrcCrossArgs* args, size_t* bytes);
int htrc_cross_backward(const HtrcCrossArgs* args, htrc_stream_t stream);

/* Layer norm: u = (x - mean) rstd over the width, y = (u weight + bias) (1 + scale) + shift, rstd = 1 / sqrt(variance +
 * eps).  Rows are [batch][token][width] through their strides (batch, token; the width's is 1); rows that are not 16-byte
 * aligned may be read in the whole 16-byte pieces that cover them. */
enum { HTRC_NORM_MAX_WIDTH = 16384 };

typedef struct {
  const void* x;
  int64_t x_stride[2];
  int64_t batch, tokens;        /* >= 0, fewer than 2^31 rows */
  int32_t width;                /* 1 .. HTRC_NORM_MAX_WIDTH */
  int32_t dtype;                /* HTRC_LAYER_F32 / BF16 / F16, of x, out, dy and dx */
  const void *weight, *bias;    /* [width], or NULL for 1 and 0 */
  const void *scale, *shift;    /* [batch][width], batch entries scale_stride / shift_stride apart, or NULL for 0 */
  int64_t scale_stride, shift_stride;
  int32_t weight_dtype, bias_dtype, scale_dtype, shift_dtype;   /* HTRC_LAYER_F32 / BF16 / F16 */
  float eps;                    /* >= 0 */
  /* forward: rows of dtype in out, or with codes 8-bit rows (see htrc_quantize_rows) */
  void* out;
  int64_t out_stride[2];
  int8_t* codes;                /* [batch * tokens][codes_pitch] */
  int64_t codes_pitch;
  float* scales;                /* [batch * tokens] */
  float *mean, *rstd;           /* [batch * tokens]; forward: written unless NULL; backward: the forward's */
  /* backward only */
  const void* dy;
  int64_t dy_stride[2];
  void* dx;
  int64_t dx_stride[2];
  void *dweight, *dbias;        /* [width], each in its parameter's type, or NULL */
  void *dscale, *dshift;        /* [batch][width] */
  int32_t* status;              /* as in HtrcCrossArgs */
  void* workspace;              /* htrc_norm_workspace_size() bytes */
  size_t workspace_bytes;
} HtrcNormArgs;

int htrc_norm_forward(const HtrcNormArgs* args, htrc_stream_t stream);
/* of the backward; every sum in a fixed order */
int htrc_norm_workspace_size(const HtrcNormArgs* args, size_t* bytes);
int htrc_norm_backward(const HtrcNormArgs* args, htrc_stream_t stream);

/* 8-bit rows of x [batch][token][width] (strides: batch, token): codes[row][i] = the integer nearest x 127 / top, ties to
 * even, scales[row] = top / 127, top = the row's largest magnitude, 10^-30 at least.  A row with a NaN or an infinity
 * gets a scale of NaN.  pitch: bytes between rows of codes, a multiple of 16 (codes 16-byte aligned). */
int htrc_quantize_rows(const void* x, int32_t dtype, int64_t batch, int64_t tokens, int32_t width, const int64_t* stride,
                       int8_t* codes, int64_t pitch, float* scales, htrc_stream_t stream);

/* Product in 8-bit integers: out[row][n] = (sum over k of x[row][k] w[n][k]) x_scales[row] w_scales[n] + bias[n], the sum
 * an exact 32-bit integer, the rest float32, rounded once.  Rows that are not 8-bit yet are quantised into the workspace, or
 * (few of them) by the product. */
enum { HTRC_LINEAR8_MAX_WIDTH = 65536 };

typedef struct {
  const void* x;                /* [batch][token][width]; HTRC_LAYER_I8: 16-byte aligned, batch stride = tokens * token stride */
  int64_t x_stride[2];          /* HTRC_LAYER_I8: multiples of 16 */
  const float* x_scales;        /* HTRC_LAYER_I8: [batch * tokens] */
  int64_t batch, tokens;        /* >= 0, fewer than 2^31 - 1024 rows */
  int32_t width, channels;      /* >= 1; HTRC_LINEAR8_MAX_WIDTH at most (HTRC_NORM_MAX_WIDTH where x is quantised here) */
  int32_t dtype;                /* of x: HTRC_LAYER_F32 / BF16 / F16 / I8 */
  const int8_t* w;              /* [channels][width], 16-byte aligned, rows w_pitch apart, a multiple of 16 */
  int64_t w_pitch;
  const float* w_scales;        /* [channels] */
  const void* bias;             /* [channels] or NULL */
  int32_t bias_dtype, out_dtype;   /* HTRC_LAYER_F32 / BF16 / F16 */
  void* out;                    /* [batch * tokens][channels], dense */
  int32_t* status;              /* as in HtrcCrossArgs */
  void* workspace;              /* htrc_linear8_workspace_size() bytes (it may be 0), 256-byte aligned */
  size_t workspace_bytes;
} HtrcLinear8Args;

int htrc_linear8_workspace_size(const HtrcLinear8Args* args, size_t* bytes);
int htrc_linear8_forward(const HtrcLinear8Args* args, htrc_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* HTRC_LAYER_H_ */

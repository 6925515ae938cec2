/* C ABI of the operators around the flat attention in a video transformer's layer (libhtrc_flat.so, sm_100a):
 *   rotary positions over several axes (time, height, width), with the per-head RMS norm before them and the
 *   token-major -> head-major reorder in the same pass, forward and backward;
 *   cross attention of the tokens to an encoder's states of another length, forward and backward.
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

enum { HTRC_LAYER_F32 = 0, HTRC_LAYER_BF16 = 1, HTRC_LAYER_F16 = 2, HTRC_LAYER_I32 = 3, HTRC_LAYER_U8 = 4 }; /* types */

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

#ifdef __cplusplus
}
#endif

#endif /* HTRC_LAYER_H_ */

/*
 * ps_ops.h -- C ABI of the operators that a half-precision training iteration runs around the optimizer step (gfx950):
 * rotation of queries and keys by their positions, alone or behind the norm of every head; a teacher's top logits; the
 * loss of a student against them.
 *
 * Conventions are those of ps_adam.h: plain C types, device addresses in every descriptor, everything is only ENQUEUED on
 * the given stream, 0 or a negative value is returned (text: ps_last_error()), nothing throws, and the library never
 * allocates, frees or keeps tensor memory.  The descriptors are read before a call returns.
 */
#ifndef PS_OPS_H
#define PS_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "ps_adam.h"

#ifdef __cplusplus
extern "C" {
#endif

/* types of elements */
#define PS_F16 0
#define PS_BF16 1
#define PS_F32 2

#define PS_MAX_HEAD_DIM 512   /* elements of a head */
#define PS_MAX_TOP 1024       /* entries of a list of top logits */

/*
 * Queries and keys of `batch` x `tokens` tokens, and how they are rotated.  Index 0 is the queries, 1 the keys; heads[1] may be 0
 * (no keys).  Element (b, t, h, d) of an input lies `stride[0] * b + stride[1] * t + stride[2] * h + d` elements behind its
 * address; outputs are contiguous.
 *
 * Pair i of the first `rotary` elements of a head is (i, i + rotary / 2), or (2 i, 2 i + 1) if `interleaved`.  It is turned by
 *     positions[axis_i] * step_i / 2^64 turns,
 * where plan[2 i] = step_i (modulo 2^64, so the product may wrap) and plan[2 i + 1] = axis_i: any 64-bit position is exact.
 */
typedef struct ps_heads_call {
    const void* x[2];         /* inputs */
    const void* grad[2];      /* gradients of the outputs (ps_norm_rotate_heads_backward) */
    void* out[2];             /* outputs, or gradients of the inputs */
    const void* weight[2];    /* the norms' weights, `dim` elements each; NULL: ones */
    void* weight_grad[2];     /* their gradients, of the weights' type; NULL: not wanted */
    const void* positions;
    const int64_t* plan;
    int64_t x_stride[2][3];
    int64_t grad_stride[2][3];
    int64_t position_stride[3]; /* of axis, batch, token; in elements */
    int64_t batch, tokens;
    int32_t heads[2];
    int32_t dim, rotary, axes;
    int32_t dtype;            /* of x, grad, out */
    int32_t weight_dtype;     /* dtype, or PS_F32 */
    int32_t position_bytes;   /* 4 or 8 */
    int32_t interleaved;
    int32_t inverse;          /* turn the other way (ps_rotate_heads: the gradient of a rotation) */
    int32_t norm;             /* divide every head by its root mean square, and multiply by the weight, first */
    float eps;                /* added to the mean square */
    int32_t reserved[2];
} ps_heads_call;

/* out = rotation(norm(x)), for queries and keys in one launch. */
int ps_rotate_heads(const ps_heads_call* call, ps_stream_t stream);

/* Gradients of the inputs and of the norms' weights from those of the outputs.  The workspace (device memory, 16-byte aligned) is
 * the caller's; 0 bytes where no weight's gradient is wanted. */
size_t ps_norm_rotate_heads_workspace_bytes(const ps_heads_call* call);
int ps_norm_rotate_heads_backward(const ps_heads_call* call, void* d_workspace, size_t workspace_bytes, ps_stream_t stream);

/*
 * The `k` largest of every row of logits, largest first, equal ones by their place (NaN counts as larger than everything, zeros of
 * both signs as equal), and log(sum(exp(logits / temperature))) of the row.
 */
typedef struct ps_top_call {
    const void* logits;
    void* values;      /* rows x k, of the logits' type */
    int32_t* ids;      /* rows x k */
    float* lse;        /* rows */
    int64_t rows, vocab, row_stride;
    double temperature;
    int32_t k, dtype;
} ps_top_call;

int ps_top_logits(const ps_top_call* call, ps_stream_t stream);

/*
 * The loss of a student against a teacher's top logits, row by row:
 *     (1 - label_weight) * temperature^2 * KL(teacher || student) + label_weight * (cross entropy of the label),
 * both distributions at the temperature, the cross entropy at 1.  The teacher's probabilities are the softmax of its list, or, with
 * teacher_lse, exp(value / temperature - teacher_lse), and what they leave to 1 is compared with what the student gives to the
 * tokens off the list.  List entries with a negative id are not there.  Rows whose label is ignore_index count for nothing.
 * A list that names a token twice or one beyond the vocabulary, or such a label, makes its row's loss and gradient NaN.
 */
typedef struct ps_distill_call {
    const void* logits;
    const void* ids;             /* rows x k, int32 or int64 */
    const void* values;          /* rows x k */
    const float* teacher_lse;    /* rows, or NULL */
    const void* labels;          /* rows, int64 or int32, or NULL */
    float* row_loss;             /* rows */
    float* stats;                /* rows x 4: what the backward pass needs (NULL: not wanted) */
    float* loss;                 /* 1: the rows' sum, over `denominator`; NULL: not wanted */
    float* denominator;          /* 1, with `mean`: the number of rows that count (at least 1) is left here for the backward pass */
    void* grad;                  /* gradient of the logits, contiguous; NULL: not wanted */
    const float* upstream;       /* what the gradient is multiplied by; NULL: upstream_value */
    float* upstream_used;        /* 1: the factor that `grad` was made with (NULL: not wanted) */
    int64_t rows, vocab, row_stride, ids_stride, values_stride, upstream_stride;
    int64_t ignore_index;
    double temperature;
    int32_t k, dtype, values_dtype, ids_bytes, labels_bytes, mean;
    float label_weight, upstream_value;
} ps_distill_call;

/* Loss, and the gradient at `upstream` too where `grad` is given: the logits are read once for both. */
int ps_distill_loss(const ps_distill_call* call, ps_stream_t stream);

/* The gradient at upstream[row * upstream_stride] from the forward pass's stats and denominator.  With upstream_used it is made only
 * if upstream[0] is another number than that (decided on the device): `grad` then holds it already. */
int ps_distill_loss_backward(const ps_distill_call* call, ps_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* PS_OPS_H */

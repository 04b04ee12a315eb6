/* gsx_optim.h — C ABI of the optimizer operators over many tensors at once (libgsx.so): AdamW with moments in 32 or in 8 bits, the norm of all
 * gradients with the clip factor, and the row selection of 8-bit moments.  Same conventions as gsx.h: device pointers unless stated, sizes, scalars and a
 * HIP stream; no allocation, no host synchronisation, nothing kept between calls; every entry point returns a gsx_status and leaves a thread-local
 * message (gsx_last_error).  All of them may be captured into a HIP graph (they record kernels only).
 *
 * Lists of tensors are host arrays, read before the call returns; any number of tensors, empty ones included.
 *
 * The control block: GSX_CONTROL_WORDS doubles on the device, through which the norm steers the update that follows it on the stream without the host:
 *   [0] norm of all gradients   [1] factor the gradients are multiplied by   [2] not 0: the update leaves everything as it is   [3] step
 *   [4..7] the library's own, zero before the first call.
 * One block belongs to one sequence of calls: two streams (or two graphs in flight at once) take a block each. */
#ifndef GSX_OPTIM_H
#define GSX_OPTIM_H

#include "gsx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The version of this header's entry points, counted apart from GSX_ABI_VERSION (gsx.h). */
#define GSX_OPTIM_ABI_VERSION 1
int gsx_optim_abi_version(void);

typedef enum gsx_dtype { GSX_DTYPE_F32 = 0, GSX_DTYPE_BF16 = 1, GSX_DTYPE_F16 = 2 } gsx_dtype;

#define GSX_CONTROL_WORDS 8
#define GSX_MOMENT_RUN 128 /* consecutive values of a tensor that share a scale of the 8-bit moments */

/* A gradient, or one parameter tensor with all that belongs to it: [rows, cols] with rows ld values apart (ld is ignored where rows == 1), the values
 * of a row next to each other.  Any alignment that the type itself has. */
typedef struct gsx_grad_tensor {
    const void* grad;
    uint64_t rows, cols, ld;
    uint32_t dtype; /* gsx_dtype */
} gsx_grad_tensor;

typedef struct gsx_adamw_tensor {
    void* param;
    const void* grad;
    void* exp_avg;    /* m: float [rows * cols], or e4m3 codes (1 byte each) */
    void* exp_avg_sq; /* v: float [rows * cols]; 8 bits: codes of sqrt(v) */
    float* avg_scale; /* 8 bits only: [ceil(rows * cols / GSX_MOMENT_RUN)] */
    float* rms_scale;
    uint64_t rows, cols, ld_param, ld_grad;
    uint64_t step;     /* number of this step, from 1; 0: the control block's */
    uint32_t split;    /* columns [split, cols) are a second group with lr_b, weight_decay_b, hold_b; 0: one group */
    uint32_t param_dtype, grad_dtype;
    int32_t hold, hold_b; /* not 0: the group's parameters and moments stay as they are (8 bits: as values, in the run's new scale) */
    float lr, lr_b, weight_decay, weight_decay_b;
} gsx_adamw_tensor;

/* Euclidean norm of all gradients, accumulated in 64 bits (the same bits every time), into the control block:
 *   [0] = norm;  [1] = min(1, max_norm / (norm + 1e-6));  [2] = 1 if any gradient is infinite or NaN, else 0;  [3] += 1 - [2].
 * Where [2] is 1, [0] is infinite or NaN and [1] is 0.  max_norm: infinite for no clipping. */
size_t gsx_grad_norm_multi_workspace_bytes(uint32_t count, const gsx_grad_tensor* tensors);
int gsx_grad_norm_multi(uint32_t count, const gsx_grad_tensor* tensors, double max_norm, double* control, void* workspace, size_t workspace_bytes,
                        void* stream);

/* AdamW with decoupled decay, t the step, g the gradient (times the control block's factor where there is one):
 *   m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2;  p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * in 32 bits, p rounded once to its type; an eps below 2^-126 (0 too) counts as 2^-126.  control: NULL, or a control block; needed where a step is 0.
 * 1 / (1 - beta1^t) and 1 / sqrt(1 - beta2^t) of a step of the list are formed in 64 bits and rounded; those of the control block's step on the device, in 32 bits, to within
 * 2^-21 of themselves.  The quotient by the root is a product with a reciprocal of 1 unit in the last place. */
int gsx_adamw_step_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, const double* control, void* stream);

/* The same with m and r = sqrt(v) stored as OCP e4m3 numbers, one scale for each GSX_MOMENT_RUN consecutive values (the last run of a tensor may be
 * shorter): scale = max(largest finite |x| of the run * (1 / 448 in 32 bits), 2^-120), code = x / scale rounded; infinities and NaN become NaN; an r above zero is
 * never stored as zero.  Zero codes (with any finite scale) are zero moments.  The moments are formed product by product and sum by sum, each rounded to 32
 * bits ((1 - beta2) g times g), the root and the quotient x / scale too, so that the codes are a function of the inputs to the last bit (but for scales between 2^-120 and 2^-93,
 * where the quotient may be off by one place of its 24 bits).
 * stochastic 0: to the nearest code, ties to even.  Else to one of the two neighbours: away from zero if (the part of the step between them) + u >= 1,
 * u the high (m) or low (r) 16 bits of mix(i + key) / 2^16 for value i of the tensor, i taken modulo 2^32,
 *   key = mix(mix(seed + 0x9E3779B9 t) + 0xC2A6F0B5 k) + 0x61C8864F floor(i / 2^32) for tensor k of the list, all in 32 bits,
 *   mix(x): x ^= x >> 16; x *= 0x9E46A9E5; x ^= x >> 15; x *= 0xF4B0A2DB; x ^= x >> 16. */
int gsx_adamw8_step_multi(uint32_t count, const gsx_adamw_tensor* tensors, double beta1, double beta2, double eps, int stochastic, uint32_t seed,
                          const double* control, void* stream);

/* Rows of 8-bit moments into a model of other rows: row j of the new moments is row index[j] of the old ones, or zero where index[j] is outside
 * [0, rows_in).  The runs are formed anew and rounded to nearest.  New and old may not overlap. */
typedef struct gsx_moments8 {
    const void *avg_in, *rms_in;
    const float *avg_scale_in, *rms_scale_in;
    void *avg_out, *rms_out;
    float *avg_scale_out, *rms_scale_out;
    uint64_t cols;
} gsx_moments8;
int gsx_adamw8_select_rows(uint32_t count, const gsx_moments8* tensors, uint64_t rows_in, uint64_t rows_out, const int64_t* index, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GSX_OPTIM_H */

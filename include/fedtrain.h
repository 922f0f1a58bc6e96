/* libfedtrain: the dense training operators for MI355X (gfx950) behind a C ABI.
 *
 *   fedtrain_product       matrix products with bias, activation and residual in
 *                          the epilogue, of one weight matrix or grouped by
 *                          client with ragged row counts, and the products of
 *                          their gradients
 *   fedtrain_act_backward  the activation's gradient; with _sums, a bias's too
 *   fedtrain_adamw         an AdamW step over many tensors, states in 32 or 8 bits
 *
 * Every entry checks its arguments on the host, launches on `stream` (a
 * hipStream_t) of the current device, allocates nothing, synchronises nothing
 * and returns 0, FEDTRAIN_EINVAL or a positive hipError_t.  No entry throws or
 * aborts.
 */
#ifndef FEDTRAIN_H
#define FEDTRAIN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FEDTRAIN_ABI_VERSION 3
#define FEDTRAIN_EINVAL (-22)

#define FEDTRAIN_F32 0
#define FEDTRAIN_BF16 1
#define FEDTRAIN_F16 2

#define FEDTRAIN_ACT_NONE 0
#define FEDTRAIN_ACT_RELU 1
#define FEDTRAIN_ACT_GELU 2 /* z Phi(z), by erf */
#define FEDTRAIN_ACT_SILU 3

/* C[i,j] = act(sum_k A[i,k] B[j,k] + bias[j]) + res[i,j]; z takes the value before act */
#define FEDTRAIN_FORWARD 0
/* C[i,j] = sum_k A[i,k] B[k,j] */
#define FEDTRAIN_GRAD_INPUT 1
/* C[i,j] = sum_k A[k,i] B[k,j]; colsum[i] = sum_k A[k,i] */
#define FEDTRAIN_GRAD_WEIGHT 2

/* Sizes: FORWARD and GRAD_INPUT have m rows, n columns and length k;
 * GRAD_WEIGHT has m x n outputs and k rows.  Strides are in elements, the last
 * dimension has stride 1.
 * groups = 0: one weight matrix.  groups > 0: `offsets` holds groups + 1
 * ascending row numbers on the device; rows offsets[g] .. offsets[g+1] use B
 * (FORWARD, GRAD_INPUT) or make C and colsum (GRAD_WEIGHT) at g * *_group.  A
 * row in no group gets C = res, or 0.  Offsets outside the rows are cut to
 * them: no value there makes an access leave the operands.
 * More tiles than a launch can hold (2^24) are refused. */
typedef struct fedtrain_product_args {
  int32_t dtype, form, act, groups;
  int64_t m, n, k;
  const void* a;
  int64_t lda;
  const void* b;
  int64_t ldb, b_group;
  void* c; /* NULL with GRAD_WEIGHT: only colsum is wanted */
  int64_t ldc, c_group;
  const void* bias; /* [n] a group, or NULL */
  int64_t bias_group;
  const void* res; /* [m, n] or NULL */
  int64_t ldr;
  void* z; /* [m, n] or NULL */
  int64_t ldz;
  void* colsum; /* [m] a group, or NULL */
  int64_t colsum_group;
  const void* offsets;
  int32_t offsets64; /* 1: int64 offsets, 0: int32 */
  int32_t reserved;
  void* workspace; /* fedtrain_product_workspace bytes, 16-byte aligned */
  int64_t workspace_bytes;
} fedtrain_product_args;

int fedtrain_abi_version(void);
const char* fedtrain_strerror(int status);

/* Bytes of device workspace a call with these arguments needs (0: none), or
 * FEDTRAIN_EINVAL.  The workspace belongs to the call until it has run. */
int64_t fedtrain_product_workspace(const fedtrain_product_args* args);
int fedtrain_product(const fedtrain_product_args* args, void* stream);

/* The tile of C a workgroup of that call takes (1 column: the kernel for a few
 * rows), and the parts k is taken in. */
int fedtrain_product_plan(const fedtrain_product_args* args, int* rows, int* cols, int* parts);

/* dz = dy act'(z), [rows, cols] with row strides; relu takes z or act(z). */
int fedtrain_act_backward(int dtype, int act, int64_t rows, int64_t cols, const void* dy,
                          int64_t lddy, const void* z, int64_t ldz, void* dz, int64_t lddz,
                          void* stream);

/* The same for 16-bit types, and each group's bias gradient from the terms before
 * they are rounded: colsum[j] = sum_rows dy act'(z).  groups, offsets and rows of no
 * group as in fedtrain_product; groups = 0 sums all rows.  (float32's dz is not
 * rounded, and FEDTRAIN_GRAD_WEIGHT sums it.) */
typedef struct fedtrain_act_args {
  int32_t dtype, act, groups, offsets64;
  int64_t rows, cols;
  const void* dy;
  int64_t lddy;
  const void* z;
  int64_t ldz;
  void* dz;
  int64_t lddz;
  void* colsum; /* [cols] a group */
  int64_t colsum_group;
  const void* offsets;
  void* workspace; /* fedtrain_act_backward_sums_workspace bytes, 16-byte aligned */
  int64_t workspace_bytes;
} fedtrain_act_args;

int64_t fedtrain_act_backward_sums_workspace(const fedtrain_act_args* args);
int fedtrain_act_backward_sums(const fedtrain_act_args* args, void* stream);

/* One tensor of an AdamW step: n elements; g has p's type; m and v are f32
 * (state_bits 32), or e4m3 and e5m2 codes with one f32 scale for each 256
 * elements in m_scale and v_scale (state_bits 8).  block0 numbers the tensor's
 * first block of 256 in the whole step, for the rounding's random numbers.  What a
 * step writes (p, m, v, the scales) shares memory with nothing else it is given. */
typedef struct fedtrain_adamw_tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  int64_t n;
  int64_t block0;
} fedtrain_adamw_tensor;

typedef struct fedtrain_adamw_scalars {
  double lr, beta1, beta2, eps, weight_decay;
  int64_t step; /* 1 for the first; not read when a step on the device is given */
  uint32_t seed;
  int32_t maximize;
  const int64_t* device_step; /* the step's number on the device, or NULL */
  void* workspace;            /* 16 bytes on the device with device_step, 16 for each
                                 tensor with device_steps */
  const int64_t* const* device_steps; /* on the host: where on the device each tensor's
                                         own step is, or NULL (then device_step is not read) */
} fedtrain_adamw_scalars;

int fedtrain_adamw(int dtype, int state_bits, int64_t count, const fedtrain_adamw_tensor* tensors,
                   const fedtrain_adamw_scalars* scalars, void* stream);

#ifdef __cplusplus
}
#endif
#endif

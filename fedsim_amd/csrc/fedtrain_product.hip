// Matrix products with bias, activation and residual in the epilogue, of one
// weight matrix or grouped by client with ragged row counts, and the products
// of their gradients (fedtrain_product, fedtrain_act_backward).
//
//   forward       z = A B^T + bias,  C = act(z) + res      A rows, B weights
//   grad input    C = A B                                  A = dz, B weights
//   grad weight   C = A^T B, colsum = A^T 1                A = dz, B = x
#include "fedtrain_common.h"

#include <climits>

namespace {

using namespace fedtrain;

using Args = fedtrain_product_args;

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------
__device__ inline float act_value(float z, int act) {
  if (act == FEDTRAIN_ACT_RELU) return z > 0 || z != z ? z : 0.0f;
  if (act == FEDTRAIN_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  if (act == FEDTRAIN_ACT_SILU) return z / (1.0f + expf(-z));
  return z;
}

__device__ inline float act_slope(float z, int act) {
  if (act == FEDTRAIN_ACT_RELU) return z > 0 ? 1.0f : 0.0f;
  if (act == FEDTRAIN_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * expf(-0.5f * z * z) * 0.39894228040143268f;
  if (act == FEDTRAIN_ACT_SILU) {
    const float t = 1.0f / (1.0f + expf(-z));
    return t * (1.0f + z * (1.0f - t));
  }
  return 1.0f;
}

// ---------------------------------------------------------------------------
// which rows a workgroup takes
// ---------------------------------------------------------------------------
struct Rows {
  int64_t lo, hi;
  int group;  // -1: rows of no group
};

// Row numbers that bound the groups, with the rows before the first and behind
// the last group as groups of their own: 0, offsets[0 .. G], rows.
__device__ inline int64_t bound(const Args& a, int64_t rows, int i) {
  if (i <= 0) return 0;
  if (i > a.groups + 1) return rows;
  const int64_t v = a.offsets64 ? static_cast<const int64_t*>(a.offsets)[i - 1]
                                : static_cast<const int32_t*>(a.offsets)[i - 1];
  return v < 0 ? 0 : v > rows ? rows : v;
}

// Range i's tiles take the slots from bound(i) / BM + i on: enough for all of
// them, and found without a sum over the ranges before.
__device__ inline Rows rows_of(const Args& a, int64_t slot, int BM) {
  if (!a.groups) {
    const int64_t lo = slot * BM;
    return {lo, lo + BM < a.m ? lo + BM : a.m, 0};
  }
  int at = 0, n = a.groups + 2;
  while (n > 1) {
    const int half = n / 2;
    if (bound(a, a.m, at + half) / BM + at + half <= slot) {
      at += half;
      n -= half;
    } else {
      n = half;
    }
  }
  const int64_t first = bound(a, a.m, at), end = bound(a, a.m, at + 1);
  const int64_t lo = first + (slot - first / BM - at) * BM;
  return {lo, lo + BM < end ? lo + BM : end, at - 1 < a.groups ? at - 1 : -1};
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

template <int D> struct Mfma;
template <> struct Mfma<FEDTRAIN_BF16> {
  static __device__ f32x4 run(const __bf16* a, const __bf16* b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(a),
                                                   *reinterpret_cast<const bf16x8*>(b), c, 0, 0, 0);
  }
};
template <> struct Mfma<FEDTRAIN_F16> {
  static __device__ f32x4 run(const _Float16* a, const _Float16* b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const f16x8*>(a),
                                                  *reinterpret_cast<const f16x8*>(b), c, 0, 0, 0);
  }
};
template <> struct Mfma<FEDTRAIN_F32> {
  static __device__ f32x4 run(const float* a, const float* b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

constexpr int kBM = 64, kBN = 64, kBK = 32;

template <int D, int FORM> __global__ __launch_bounds__(256) void k_product(Args a, int tiles_n) {
  using T = typename Elem<D>::type;
  __shared__ __attribute__((aligned(16))) T As[kBM][kBK + 8], Bs[kBN][kBK + 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const int64_t col0 = static_cast<int64_t>(blockIdx.x % tiles_n) * kBN;
  int64_t slot = blockIdx.x / tiles_n;
  int64_t row0, rows, k0 = 0, k1 = a.k;
  int group = 0;
  if (FORM == FEDTRAIN_GRAD_WEIGHT) {
    const int64_t tiles_m = (a.m + kBM - 1) / kBM;
    if (a.groups) {
      group = static_cast<int>(slot / tiles_m);
      slot %= tiles_m;
      k0 = bound(a, a.k, group + 1);
      k1 = bound(a, a.k, group + 2);
    }
    row0 = slot * kBM;
    rows = a.m - row0 < kBM ? a.m - row0 : kBM;
  } else {
    const Rows r = rows_of(a, slot, kBM);
    if (r.lo >= r.hi) return;
    row0 = r.lo;
    rows = r.hi - r.lo;
    group = r.group;
    if (group < 0) k1 = 0;
  }
  const T* A = static_cast<const T*>(a.a);
  const T* B = static_cast<const T*>(a.b);
  if (FORM != FEDTRAIN_GRAD_WEIGHT && group > 0) B += group * a.b_group;
  const int64_t cols = a.n - col0 < kBN ? a.n - col0 : kBN;

  f32x4 acc[2][2] = {};
  f32x4 sum[2] = {};
  const bool want_sum = FORM == FEDTRAIN_GRAD_WEIGHT && a.colsum && col0 == 0;
  for (int64_t k = k0; k < k1; k += kBK) {
    for (int i = tid; i < kBM * kBK; i += 256) {
      const int r = FORM == FEDTRAIN_GRAD_WEIGHT ? i % kBM : i / kBK;
      const int c = FORM == FEDTRAIN_GRAD_WEIGHT ? i / kBM : i % kBK;
      T v = Elem<D>::down(0);
      if (r < rows && k + c < k1)
        v = FORM == FEDTRAIN_GRAD_WEIGHT ? A[(k + c) * a.lda + row0 + r]
                                         : A[(row0 + r) * a.lda + k + c];
      As[r][c] = v;
    }
    for (int i = tid; i < kBN * kBK; i += 256) {
      const int r = FORM == FEDTRAIN_FORWARD ? i / kBK : i % kBN;
      const int c = FORM == FEDTRAIN_FORWARD ? i % kBK : i / kBN;
      T v = Elem<D>::down(0);
      if (r < cols && k + c < k1)
        v = FORM == FEDTRAIN_FORWARD ? B[(col0 + r) * a.ldb + k + c]
                                     : B[(k + c) * a.ldb + col0 + r];
      Bs[r][c] = v;
    }
    __syncthreads();
    const int r = lane & 15, q = (lane >> 4) * 8;
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2; ++j)
        acc[i][j] = Mfma<D>::run(&As[wm + i * 16 + r][q], &Bs[wn + j * 16 + r][q], acc[i][j]);
    if (want_sum && wn == 0) {
      T one[8];
      for (int e = 0; e < 8; ++e) one[e] = Elem<D>::down(1.0f);
      for (int i = 0; i < 2; ++i) sum[i] = Mfma<D>::run(&As[wm + i * 16 + r][q], one, sum[i]);
    }
    __syncthreads();
  }

  T* C = static_cast<T*>(a.c);
  for (int i = 0; i < 2; ++i)
    for (int e = 0; e < 4; ++e) {
      const int r = wm + i * 16 + (lane >> 4) * 4 + e;
      if (r >= rows) continue;
      if (want_sum && wn == 0 && (lane & 15) == 0)
        static_cast<T*>(a.colsum)[group * a.colsum_group + row0 + r] = Elem<D>::down(sum[i][e]);
      for (int j = 0; j < 2; ++j) {
        const int c = wn + j * 16 + (lane & 15);
        if (c >= cols) continue;
        float v = acc[i][j][e];
        const int64_t row = row0 + r, col = col0 + c;
        if (FORM == FEDTRAIN_FORWARD) {
          if (group >= 0) {
            if (a.bias) v += Elem<D>::up(static_cast<const T*>(a.bias)[group * a.bias_group + col]);
            if (a.z) static_cast<T*>(a.z)[row * a.ldz + col] = Elem<D>::down(v);
            v = act_value(v, a.act);
          } else if (a.z) {
            static_cast<T*>(a.z)[row * a.ldz + col] = Elem<D>::down(0);
          }
          if (a.res) v += Elem<D>::up(static_cast<const T*>(a.res)[row * a.ldr + col]);
        }
        if (FORM == FEDTRAIN_GRAD_WEIGHT) {
          if (C) C[group * a.c_group + row * a.ldc + col] = Elem<D>::down(v);
        } else {
          C[row * a.ldc + col] = Elem<D>::down(v);
        }
      }
    }
}

template <int D>
__global__ __launch_bounds__(256) void k_act_backward(int act, int64_t rows, int64_t cols,
                                                      const void* dy, int64_t lddy, const void* z,
                                                      int64_t ldz, void* dz, int64_t lddz) {
  using T = typename Elem<D>::type;
  const int64_t n = rows * cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / cols, c = i % cols;
    const float g = Elem<D>::up(static_cast<const T*>(dy)[r * lddy + c]);
    const float v = Elem<D>::up(static_cast<const T*>(z)[r * ldz + c]);
    static_cast<T*>(dz)[r * lddz + c] = Elem<D>::down(g * act_slope(v, act));
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int64_t kMaxSize = INT32_MAX;  // of one dimension

bool valid(const Args* a) {
  if (!a || a->dtype < FEDTRAIN_F32 || a->dtype > FEDTRAIN_F16 || a->form < FEDTRAIN_FORWARD ||
      a->form > FEDTRAIN_GRAD_WEIGHT || a->act < FEDTRAIN_ACT_NONE || a->act > FEDTRAIN_ACT_SILU ||
      a->groups < 0 || a->m < 0 || a->n < 0 || a->k < 0 || a->m > kMaxSize || a->n > kMaxSize ||
      a->k > kMaxSize)
    return false;
  const int form = a->form;
  if (form != FEDTRAIN_FORWARD && (a->act || a->bias || a->res || a->z)) return false;
  if (form != FEDTRAIN_GRAD_WEIGHT && a->colsum) return false;
  if (a->groups && !a->offsets) return false;
  if (a->groups == INT32_MAX || a->groups > INT32_MAX - 2) return false;
  const size_t size = a->dtype == FEDTRAIN_F32 ? 4 : 2;
  const void* each[] = {a->a, a->b, a->c, a->bias, a->res, a->z, a->colsum};
  for (const void* p : each)
    if (!aligned(p, size)) return false;
  if (a->offsets && !aligned(a->offsets, a->offsets64 ? 8 : 4)) return false;
  if (a->lda < 0 || a->ldb < 0 || a->ldr < 0 || a->b_group < 0 || a->bias_group < 0) return false;
  // outputs must not overlap themselves
  const int64_t out_rows = a->m;
  if (out_rows > 1 && a->c && a->ldc < a->n) return false;
  if (out_rows > 1 && a->z && a->ldz < a->n) return false;
  if (form == FEDTRAIN_GRAD_WEIGHT && a->groups > 1) {
    if (a->c && a->c_group < (a->m > 0 ? (a->m - 1) * a->ldc + a->n : 0)) return false;
    if (a->colsum && a->colsum_group < a->m) return false;
  }
  const bool any = a->m && a->n;
  if (form == FEDTRAIN_GRAD_WEIGHT) {
    if (any && !a->c && !a->colsum) return false;
    if (a->m && a->k && (!a->a || (a->n && !a->b))) return false;
  } else if (any && (!a->c || (a->k && (!a->a || !a->b)))) {
    return false;
  }
  return true;
}

template <int D> int run(const Args& a, hipStream_t s) {
  const int64_t tiles_n = a.n ? (a.n + kBN - 1) / kBN : 1;
  int64_t slots;
  if (a.form == FEDTRAIN_GRAD_WEIGHT)
    slots = (a.m + kBM - 1) / kBM * (a.groups ? a.groups : 1);
  else
    slots = a.groups ? a.m / kBM + a.groups + 2 : (a.m + kBM - 1) / kBM;
  if (slots > INT32_MAX / tiles_n) return FEDTRAIN_EINVAL;
  const dim3 grid(static_cast<unsigned>(slots * tiles_n));
  const int tn = static_cast<int>(tiles_n);
  if (a.form == FEDTRAIN_FORWARD)
    hipLaunchKernelGGL((k_product<D, FEDTRAIN_FORWARD>), grid, dim3(256), 0, s, a, tn);
  else if (a.form == FEDTRAIN_GRAD_INPUT)
    hipLaunchKernelGGL((k_product<D, FEDTRAIN_GRAD_INPUT>), grid, dim3(256), 0, s, a, tn);
  else
    hipLaunchKernelGGL((k_product<D, FEDTRAIN_GRAD_WEIGHT>), grid, dim3(256), 0, s, a, tn);
  return launched();
}

}  // namespace

extern "C" {

int fedtrain_abi_version(void) { return FEDTRAIN_ABI_VERSION; }

const char* fedtrain_strerror(int status) {
  if (status == 0) return "success";
  if (status == FEDTRAIN_EINVAL) return "fedtrain: invalid argument";
  if (status > 0) return hipGetErrorString(static_cast<hipError_t>(status));
  return "fedtrain: unknown error";
}

int64_t fedtrain_product_workspace(const Args* args) {
  return valid(args) ? 0 : FEDTRAIN_EINVAL;
}

int fedtrain_product(const Args* args, void* stream) {
  if (!valid(args)) return FEDTRAIN_EINVAL;
  const Args& a = *args;
  if (!a.m || (!a.n && !a.colsum)) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.dtype == FEDTRAIN_F32) return run<FEDTRAIN_F32>(a, s);
  if (a.dtype == FEDTRAIN_BF16) return run<FEDTRAIN_BF16>(a, s);
  return run<FEDTRAIN_F16>(a, s);
}

int fedtrain_act_backward(int dtype, int act, int64_t rows, int64_t cols, const void* dy,
                          int64_t lddy, const void* z, int64_t ldz, void* dz, int64_t lddz,
                          void* stream) {
  if (dtype < FEDTRAIN_F32 || dtype > FEDTRAIN_F16 || act < FEDTRAIN_ACT_NONE ||
      act > FEDTRAIN_ACT_SILU || rows < 0 || cols < 0 || rows > kMaxSize || cols > kMaxSize)
    return FEDTRAIN_EINVAL;
  if (!rows || !cols) return 0;
  const size_t size = dtype == FEDTRAIN_F32 ? 4 : 2;
  if (!dy || !z || !dz || !aligned(dy, size) || !aligned(z, size) || !aligned(dz, size) ||
      lddy < 0 || ldz < 0 || (rows > 1 && lddz < cols))
    return FEDTRAIN_EINVAL;
  const int64_t want = (rows * cols + 1023) / 1024;
  const dim3 grid(static_cast<unsigned>(want < 65536 ? want : 65536));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FEDTRAIN_F32)
    hipLaunchKernelGGL(k_act_backward<FEDTRAIN_F32>, grid, dim3(256), 0, s, act, rows, cols, dy,
                       lddy, z, ldz, dz, lddz);
  else if (dtype == FEDTRAIN_BF16)
    hipLaunchKernelGGL(k_act_backward<FEDTRAIN_BF16>, grid, dim3(256), 0, s, act, rows, cols, dy,
                       lddy, z, ldz, dz, lddz);
  else
    hipLaunchKernelGGL(k_act_backward<FEDTRAIN_F16>, grid, dim3(256), 0, s, act, rows, cols, dy,
                       lddy, z, ldz, dz, lddz);
  return launched();
}

}  // extern "C"

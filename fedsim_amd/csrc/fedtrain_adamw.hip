// AdamW over many tensors in one launch (fedtrain_adamw).
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The sums are f32, each product and sum rounded on its own (no fma), so that
// a state's value does not depend on how the compiler pairs them.
//
// States in 8 bits: m is held in e4m3 and v in e5m2, in blocks of 256 elements
// that share a power of two.  Powers of two keep the grid of the codes in place
// when a block's scale changes, so an element that barely moves is barely
// rounded: with stochastic rounding the error of a step has the variance
// (change x spacing), not spacing^2 / 6, and it is 0 in the mean.  v moves by
// about (1 - b2) v a step; over its memory of 1 / (1 - b2) steps the noise adds
// up to about 0.3 v, 0.15 in sqrt(v), whatever b2 is.  Rounding to nearest would
// leave v where it is for good: (1 - b2) is far below half a spacing.
// The parameters are updated from m and v as they are before this rounding.
#include "fedtrain_common.h"

#include <cmath>

namespace {

using namespace fedtrain;

constexpr int kBlock = 256;   // elements that share a scale: 64 lanes x 4
constexpr int kChunk = 4096;  // elements a workgroup takes: 4 waves x 4 blocks
constexpr int kMost = 40;     // tensors a launch takes: 40 x 72 B of kernel arguments

struct Tensor {
  fedtrain_adamw_tensor t;
  int first;  // the tensor's first workgroup
  int wide;   // every pointer allows loads of 4 elements
};

struct Batch {
  Tensor at[kMost];
  int count;
  float b1, c1, b2, c2, decay, eps, size, root;
  unsigned key;
  float sign;
  const float* device;  // {size, root, key} computed on the device, or null
};

// two rounds of xor-shift and multiply by odd fractions of sqrt(2) and sqrt(3)
__host__ __device__ inline unsigned mix(unsigned h) {
  h ^= h >> 16;
  h *= 0x6A09E667u;
  h ^= h >> 15;
  h *= 0xBB67AE85u;
  return h ^ (h >> 16);
}

__device__ inline float from_bits(unsigned b) { return __builtin_bit_cast(float, b); }
__device__ inline unsigned to_bits(float f) { return __builtin_bit_cast(unsigned, f); }

// The largest of a wave's values.
__device__ inline float wave_max(float x) {
  for (int s = 32; s; s >>= 1) x = fmaxf(x, __shfl_xor(x, s));
  return x;
}

// The biased exponent of a block's scale: the largest magnitude over it lies
// between sqrt(3) 2^TOP and sqrt(3) 2^(TOP + 1), below the codes' largest.  A
// border at 1.0 or at the largest code would be met by sums of codes.
template <int TOP> __device__ inline int scale_exponent(float most) {
  int e = static_cast<int>(to_bits(most * 0.57735026918962576f) >> 23) - TOP;
  return e < 1 ? 1 : e;
}

// |x| in units of the scale, rounded to a float of MANT bits and smallest
// normal 2^LEAST: up with the probability of the part that is cut off
template <int MANT, int LEAST> __device__ inline float stochastic(float a, unsigned u16) {
  unsigned e = to_bits(a) >> 23;
  e = e < 127 + LEAST ? 127 + LEAST : e;
  float up = from_bits((254 - e + MANT) << 23), step = from_bits((e - MANT) << 23);
  return floorf(a * up + static_cast<float>(u16) * 0x1p-16f) * step;
}

struct Moments {
  float m, v;
};

__device__ inline Moments moments(const Batch& b, float m, float v, float g) {
  g *= b.sign;
  return {m * b.b1 + g * b.c1, v * b.b2 + (g * b.c2) * g};
}

__device__ inline float step_of(const Batch& b, float size, float root, float p, Moments s) {
  // the square root and the quotient of the hardware, each within one unit of
  // its last place: far below the rounding of p
  float d = __builtin_amdgcn_sqrtf(s.v) * root + b.eps;
  return p * b.decay - size * (s.m * __builtin_amdgcn_rcpf(d));
}

template <int D, int BITS> __global__ __launch_bounds__(256) void k_adamw(Batch b) {
  using T = typename Elem<D>::type;
  int i = 0;
  while (i + 1 < b.count && static_cast<int>(blockIdx.x) >= b.at[i + 1].first) ++i;
  const Tensor& t = b.at[i];
  float size = b.size, root = b.root;
  unsigned key = b.key;
  if (b.device) {
    size = b.device[0];
    root = b.device[1];
    key = to_bits(b.device[2]);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T* P = static_cast<T*>(t.t.p);
  const T* G = static_cast<const T*>(t.t.g);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x - t.first) * kChunk;
  for (int j = 0; j < kChunk / kBlock / 4; ++j) {
    const int64_t at = chunk + (j * 4 + wave) * kBlock + lane * 4;
    if (at - lane * 4 >= t.t.n) return;
    const int64_t blk = at / kBlock;
    float p[4], g[4], m[4], v[4];
    int live = t.t.n - at >= 4 ? 4 : t.t.n - at > 0 ? static_cast<int>(t.t.n - at) : 0;
    float ms = 1, vs = 1;
    if (BITS == 8) {
      ms = t.t.m_scale[blk];
      vs = t.t.v_scale[blk];
    }
    for (int e = 0; e < 4; ++e) {
      p[e] = g[e] = m[e] = v[e] = 0;
      if (e < live) {
        p[e] = Elem<D>::up(P[at + e]);
        g[e] = Elem<D>::up(G[at + e]);
        if (BITS == 32) {
          m[e] = static_cast<const float*>(t.t.m)[at + e];
          v[e] = static_cast<const float*>(t.t.v)[at + e];
        } else {
          m[e] = __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(t.t.m)[at + e], 0) * ms;
          v[e] = __builtin_amdgcn_cvt_f32_bf8(static_cast<const uint8_t*>(t.t.v)[at + e], 0) * vs;
        }
      }
    }
    float mm = 0, vm = 0;
    for (int e = 0; e < 4; ++e) {
      Moments s = moments(b, m[e], v[e], g[e]);
      m[e] = s.m;
      v[e] = s.v;
      p[e] = step_of(b, size, root, p[e], s);
      // an infinity or NaN is that element's alone: it does not set the scale
      if (fabsf(s.m) < INFINITY) mm = fmaxf(mm, fabsf(s.m));
      if (s.v < INFINITY) vm = fmaxf(vm, s.v);
    }
    uint8_t qm[4], qv[4];
    if (BITS == 8) {
      const int me = scale_exponent<7>(wave_max(mm)), ve = scale_exponent<14>(wave_max(vm));
      const float mi = from_bits(static_cast<unsigned>(254 - me) << 23);
      const float vi = from_bits(static_cast<unsigned>(254 - ve) << 23);
      const unsigned bk = mix(key + static_cast<unsigned>(t.t.block0 + blk) * 0x9E3779B9u);
      for (int e = 0; e < 4; ++e) {
        const unsigned h = mix(bk + static_cast<unsigned>(lane * 4 + e) * 0x9E3779B9u);
        float x = stochastic<3, -6>(fabsf(m[e]) * mi, h & 0xFFFF);
        x = copysignf(x, m[e]);
        float y = v[e] * vi;
        y = y > 0 ? fmaxf(stochastic<2, -14>(y, h >> 16), 0x1p-16f) : y;
        qm[e] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false));
        qv[e] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_bf8_f32(y, y, 0, false));
        if (!(fabsf(m[e]) < INFINITY)) qm[e] = 0x7F;
        if (!(v[e] < INFINITY)) qv[e] = v[e] == INFINITY ? 0x7C : 0x7F;
      }
      if (lane == 0) {
        t.t.m_scale[blk] = from_bits(static_cast<unsigned>(me) << 23);
        t.t.v_scale[blk] = from_bits(static_cast<unsigned>(ve) << 23);
      }
    }
    for (int e = 0; e < live; ++e) {
      P[at + e] = Elem<D>::down(p[e]);
      if (BITS == 32) {
        static_cast<float*>(t.t.m)[at + e] = m[e];
        static_cast<float*>(t.t.v)[at + e] = v[e];
      } else {
        static_cast<uint8_t*>(t.t.m)[at + e] = qm[e];
        static_cast<uint8_t*>(t.t.v)[at + e] = qv[e];
      }
    }
  }
}

struct Corrections {
  float size, root;
};

__host__ __device__ inline Corrections corrections(double lr, double b1, double b2, double t) {
  return {static_cast<float>(lr / (1 - pow(b1, t))),
          static_cast<float>(1 / sqrt(1 - pow(b2, t)))};
}

__global__ void k_adamw_scalars(double lr, double b1, double b2, unsigned seed,
                                const int64_t* step, float* out) {
  const int64_t t = *step;
  const Corrections c = corrections(lr, b1, b2, static_cast<double>(t));
  out[0] = c.size;
  out[1] = c.root;
  out[2] = from_bits(mix(seed ^ mix(static_cast<unsigned>(t))));
}

template <int D> void launch(int bits, unsigned grid, hipStream_t s, const Batch& b) {
  if (bits == 32)
    hipLaunchKernelGGL((k_adamw<D, 32>), dim3(grid), dim3(256), 0, s, b);
  else
    hipLaunchKernelGGL((k_adamw<D, 8>), dim3(grid), dim3(256), 0, s, b);
}

}  // namespace

extern "C" int fedtrain_adamw(int dtype, int state_bits, int64_t count,
                              const fedtrain_adamw_tensor* tensors,
                              const fedtrain_adamw_scalars* s, void* stream) {
  if (dtype < FEDTRAIN_F32 || dtype > FEDTRAIN_F16 || (state_bits != 8 && state_bits != 32) ||
      count < 0 || (count && !tensors) || !s)
    return FEDTRAIN_EINVAL;
  if (s->device_step ? !s->workspace || !aligned(s->workspace, 4) : s->step < 1)
    return FEDTRAIN_EINVAL;
  if (!(s->beta1 >= 0 && s->beta1 < 1 && s->beta2 >= 0 && s->beta2 < 1 && s->lr >= 0 &&
        s->eps >= 0 && s->weight_decay >= 0))
    return FEDTRAIN_EINVAL;
  const size_t esize = dtype == FEDTRAIN_F32 ? 4 : 2, ssize = state_bits == 32 ? 4 : 1;
  for (int64_t i = 0; i < count; ++i) {
    const fedtrain_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.block0 < 0) return FEDTRAIN_EINVAL;
    if (!t.n) continue;
    if (!t.p || !t.g || !t.m || !t.v || !aligned(t.p, esize) || !aligned(t.g, esize) ||
        !aligned(t.m, ssize) || !aligned(t.v, ssize))
      return FEDTRAIN_EINVAL;
    if (state_bits == 8 &&
        (!t.m_scale || !t.v_scale || !aligned(t.m_scale, 4) || !aligned(t.v_scale, 4)))
      return FEDTRAIN_EINVAL;
    if (t.n > static_cast<int64_t>(kChunk) << 30) return FEDTRAIN_EINVAL;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  Batch b;
  b.b1 = static_cast<float>(s->beta1);
  b.c1 = static_cast<float>(1 - s->beta1);
  b.b2 = static_cast<float>(s->beta2);
  b.c2 = static_cast<float>(1 - s->beta2);
  b.decay = static_cast<float>(1 - s->lr * s->weight_decay);
  b.eps = static_cast<float>(s->eps);
  b.sign = s->maximize ? -1.0f : 1.0f;
  b.device = nullptr;
  b.size = b.root = 0;
  b.key = 0;
  if (s->device_step) {
    b.device = static_cast<const float*>(s->workspace);
    hipLaunchKernelGGL(k_adamw_scalars, dim3(1), dim3(1), 0, st, s->lr, s->beta1, s->beta2,
                       s->seed, s->device_step, static_cast<float*>(s->workspace));
  } else {
    const Corrections c = corrections(s->lr, s->beta1, s->beta2, static_cast<double>(s->step));
    b.size = c.size;
    b.root = c.root;
    b.key = mix(s->seed ^ mix(static_cast<unsigned>(s->step)));
  }
  for (int64_t i = 0; i < count;) {
    int64_t grid = 0;
    b.count = 0;
    for (; i < count && b.count < kMost; ++i) {
      const fedtrain_adamw_tensor& t = tensors[i];
      if (!t.n) continue;
      const int64_t groups = (t.n + kChunk - 1) / kChunk;
      if (grid + groups > INT32_MAX) break;
      Tensor& at = b.at[b.count++];
      at.t = t;
      at.first = static_cast<int>(grid);
      at.wide = aligned(t.p, 4 * esize) && aligned(t.g, 4 * esize) && aligned(t.m, 4 * ssize) &&
                aligned(t.v, 4 * ssize);
      grid += groups;
    }
    if (!b.count) break;
    const unsigned n = static_cast<unsigned>(grid);
    if (dtype == FEDTRAIN_F32) launch<FEDTRAIN_F32>(state_bits, n, st, b);
    else if (dtype == FEDTRAIN_BF16) launch<FEDTRAIN_BF16>(state_bits, n, st, b);
    else launch<FEDTRAIN_F16>(state_bits, n, st, b);
    if (const int rc = launched()) return rc;
  }
  return 0;
}

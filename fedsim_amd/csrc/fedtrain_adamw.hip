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
//
// Memory bounds it: 125 M f32 with 32-bit states, 28 B an element, in 650 us (5.4
// TB/s; a copy reaches 4.64), 25 M bf16 in 60 tensors with 8-bit states, 10 B an
// element, in 54 us (4.6 TB/s), six tensors of 200 k in 6.2 us, a launch.
#include "fedtrain_common.h"

#include <cmath>

namespace {

using namespace fedtrain;

constexpr int kBlock = 256;   // elements that share a scale: 64 lanes x 4
constexpr int kMost = 62;     // tensors a launch takes: 62 x 64 B of the 4 KiB of arguments

struct Tensor {
  void* p;
  const void* g;
  void *m, *v;
  float *m_scale, *v_scale;
  int64_t n_wide;  // 2 n, + 1 where every pointer is 16-byte aligned
  int first;       // the tensor's first workgroup
  unsigned block0;

  __device__ int64_t n() const { return n_wide >> 1; }
  __device__ bool wide() const { return n_wide & 1; }
};

struct Batch {
  Tensor at[kMost];
  int count;
  float b1, c1, b2, c2, decay, eps, size, root;
  unsigned key;
  const float* device;  // {size, root, key} computed on the device, or null:
  int each;             // floats from one tensor's to the next one's, 0 if they share them
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

// The biased exponent of a block's scale: the largest magnitude over it lies
// between sqrt(3) 2^TOP and sqrt(3) 2^(TOP + 1), below the codes' largest.  A
// border at 1.0 or at the largest code would be met by sums of codes.
template <int TOP> __device__ inline int scale_exponent(float most) {
  int e = static_cast<int>(to_bits(most * 0.57735026918962576f) >> 23) - TOP;
  return e < 1 ? 1 : e;
}

struct Moments {
  float m, v;
};

// From states that already carry b1 and b2.  c1 has the sign of the direction.
__device__ inline Moments moments(const Batch& b, float b1m, float b2v, float g) {
  return {b1m + g * b.c1, b2v + (g * b.c2) * g};
}

struct Scalars {
  float size, root;
  unsigned key;
};

__device__ inline float step_of(const Batch& b, const Scalars& c, float p, Moments s) {
  // the square root and the quotient of the hardware, each within one unit of
  // its last place: far below the rounding of p
  // (the root takes a subnormal number for 0, which only eps = 0 would show)
  const bool tiny = s.v < 0x1p-100f;
  const float root = __builtin_amdgcn_sqrtf(tiny ? s.v * 0x1p48f : s.v);
  const float d = (tiny ? root * 0x1p-24f : root) * c.root + b.eps;
  return __builtin_fmaf(p, b.decay, -(c.size * (s.m * __builtin_amdgcn_rcpf(d))));
}

template <class T, int V> struct __attribute__((aligned(V * sizeof(T)))) Vec {
  T v[V];
};

template <class T, int V> __device__ inline Vec<T, V> get(const void* p, int64_t at) {
  return *reinterpret_cast<const Vec<T, V>*>(static_cast<const T*>(p) + at);
}
template <class T, int V> __device__ inline void set(void* p, int64_t at, const Vec<T, V>& x) {
  *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p) + at) = x;
}

// The largest of each SPAN neighbouring lanes' values.
template <int SPAN> __device__ inline float span_max(float x) {
#pragma unroll
  for (int s = SPAN / 2; s; s >>= 1) x = fmaxf(x, __shfl_xor(x, s));
  return x;
}

// The codes of V neighbouring elements of block `blk`, from its element `first`
// on; SPAN lanes share the block, and one of them stores its scales.
//
// A code is its value rounded down on the grid of codes, or up with the
// probability of the part that is cut off, floor(x / spacing + u) spacing with u
// 16 random bits over 2^16: the conversion's own rounding with u in the high half
// of its random operand, subnormal codes included (compared on 33 million values).
// An infinity or NaN gets a code of its own: NaN (m), infinity or NaN (v).
template <int V, int SPAN>
__device__ inline void requantize(const float* m, const float* v, unsigned key, int64_t blk,
                                  unsigned first, float* m_scale, float* v_scale, unsigned* qm,
                                  unsigned* qv) {
  float mm = 0, vm = 0;  // the maximum of a number and NaN is the number
#pragma unroll
  for (int e = 0; e < V; ++e) {
    mm = fmaxf(mm, fabsf(m[e]));
    vm = fmaxf(vm, v[e]);
  }
  mm = span_max<SPAN>(mm);
  vm = span_max<SPAN>(vm);
  if (__builtin_amdgcn_ballot_w64(!(mm < INFINITY && vm < INFINITY))) {
    // an infinity does not set its block's scale
    mm = vm = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      mm = fmaxf(mm, fabsf(m[e]) < INFINITY ? fabsf(m[e]) : 0.0f);
      vm = fmaxf(vm, v[e] < INFINITY ? v[e] : 0.0f);
    }
    mm = span_max<SPAN>(mm);
    vm = span_max<SPAN>(vm);
  }
  const int me = scale_exponent<7>(mm), ve = scale_exponent<14>(vm);
  const float mi = from_bits(static_cast<unsigned>(254 - me) << 23);
  const float vi = from_bits(static_cast<unsigned>(254 - ve) << 23);
  const unsigned bk = mix(key + static_cast<unsigned>(blk) * 0x9E3779B9u);
#pragma unroll
  for (int e = 0; e < V; e += 4) {
    int a = 0, c = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const unsigned h = mix(bk + (first + e + s) * 0x9E3779B9u);
      const float x = m[e + s] * mi;
      float y = v[e + s] * vi;
      // v is never rounded to zero, since it divides m: at least the least code
      if (__builtin_amdgcn_ballot_w64(y < 0x1p-16f)) y = v[e + s] > 0 ? fmaxf(y, 0x1p-16f) : y;
      switch (s) {  // the byte is a constant of the instruction
        case 0:
          a = __builtin_amdgcn_cvt_sr_fp8_f32(x, h << 16, a, 0);
          c = __builtin_amdgcn_cvt_sr_bf8_f32(y, h & 0xFFFF0000u, c, 0);
          break;
        case 1:
          a = __builtin_amdgcn_cvt_sr_fp8_f32(x, h << 16, a, 1);
          c = __builtin_amdgcn_cvt_sr_bf8_f32(y, h & 0xFFFF0000u, c, 1);
          break;
        case 2:
          a = __builtin_amdgcn_cvt_sr_fp8_f32(x, h << 16, a, 2);
          c = __builtin_amdgcn_cvt_sr_bf8_f32(y, h & 0xFFFF0000u, c, 2);
          break;
        default:
          a = __builtin_amdgcn_cvt_sr_fp8_f32(x, h << 16, a, 3);
          c = __builtin_amdgcn_cvt_sr_bf8_f32(y, h & 0xFFFF0000u, c, 3);
      }
    }
    qm[e / 4] = a;
    qv[e / 4] = c;
  }
  if ((threadIdx.x & (SPAN - 1)) == 0) {
    *m_scale = from_bits(static_cast<unsigned>(me) << 23);
    *v_scale = from_bits(static_cast<unsigned>(ve) << 23);
  }
}

// V elements of a tensor from `at` on that all exist, all pointers aligned.
template <int D, int BITS, int V>
__device__ inline void step_wide(const Batch& b, const Scalars& c, const Tensor& t, int64_t at) {
  using T = typename Elem<D>::type;
  const Vec<T, V> p = get<T, V>(t.p, at), g = get<T, V>(t.g, at);
  float m[V], v[V];
  const int64_t blk = at / kBlock;
  if constexpr (BITS == 32) {
    const Vec<float, V> mo = get<float, V>(t.m, at), vo = get<float, V>(t.v, at);
#pragma unroll
    for (int e = 0; e < V; ++e) m[e] = mo.v[e] * b.b1, v[e] = vo.v[e] * b.b2;
  } else {
    const Vec<unsigned, V / 4> mo = get<unsigned, V / 4>(t.m, at / 4);
    const Vec<unsigned, V / 4> vo = get<unsigned, V / 4>(t.v, at / 4);
    // a power of two times b1 is exact, and so is code * scale: one rounding
    const float ms = t.m_scale[blk] * b.b1, vs = t.v_scale[blk] * b.b2;
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      m[e] = __builtin_amdgcn_cvt_f32_fp8(mo.v[e / 4], 0) * ms;
      m[e + 1] = __builtin_amdgcn_cvt_f32_fp8(mo.v[e / 4], 1) * ms;
      m[e + 2] = __builtin_amdgcn_cvt_f32_fp8(mo.v[e / 4], 2) * ms;
      m[e + 3] = __builtin_amdgcn_cvt_f32_fp8(mo.v[e / 4], 3) * ms;
      v[e] = __builtin_amdgcn_cvt_f32_bf8(vo.v[e / 4], 0) * vs;
      v[e + 1] = __builtin_amdgcn_cvt_f32_bf8(vo.v[e / 4], 1) * vs;
      v[e + 2] = __builtin_amdgcn_cvt_f32_bf8(vo.v[e / 4], 2) * vs;
      v[e + 3] = __builtin_amdgcn_cvt_f32_bf8(vo.v[e / 4], 3) * vs;
    }
  }
  Vec<T, V> out;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const Moments s = moments(b, m[e], v[e], Elem<D>::up(g.v[e]));
    m[e] = s.m;
    v[e] = s.v;
    out.v[e] = Elem<D>::down(step_of(b, c, Elem<D>::up(p.v[e]), s));
  }
  set<T, V>(t.p, at, out);
  if constexpr (BITS == 32) {
    Vec<float, V> mo, vo;
#pragma unroll
    for (int e = 0; e < V; ++e) mo.v[e] = m[e], vo.v[e] = v[e];
    set<float, V>(t.m, at, mo);
    set<float, V>(t.v, at, vo);
  } else {
    Vec<unsigned, V / 4> qm, qv;
    requantize<V, kBlock / V>(m, v, c.key, t.block0 + blk, at % kBlock, t.m_scale + blk,
                              t.v_scale + blk, qm.v, qv.v);
    set<unsigned, V / 4>(t.m, at / 4, qm);
    set<unsigned, V / 4>(t.v, at / 4, qv);
  }
}

// A wave's block at any alignment, or the short last one; 4 elements a lane.
template <int D, int BITS>
__device__ void step_any(const Batch& b, const Scalars& c, const Tensor& t, int64_t at) {
  using T = typename Elem<D>::type;
  T* P = static_cast<T*>(t.p);
  const T* G = static_cast<const T*>(t.g);
  const int64_t left = t.n() - at, blk = at / kBlock;
  const int live = left >= 4 ? 4 : left > 0 ? static_cast<int>(left) : 0;
  float p[4], m[4], v[4];
  const float ms = BITS == 8 ? t.m_scale[blk] * b.b1 : b.b1;
  const float vs = BITS == 8 ? t.v_scale[blk] * b.b2 : b.b2;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float g = 0;
    p[e] = m[e] = v[e] = 0;
    if (e < live) {
      p[e] = Elem<D>::up(P[at + e]);
      g = Elem<D>::up(G[at + e]);
      if (BITS == 32) {
        m[e] = static_cast<const float*>(t.m)[at + e] * ms;
        v[e] = static_cast<const float*>(t.v)[at + e] * vs;
      } else {
        m[e] = __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(t.m)[at + e], 0) * ms;
        v[e] = __builtin_amdgcn_cvt_f32_bf8(static_cast<const uint8_t*>(t.v)[at + e], 0) * vs;
      }
    }
    const Moments s = moments(b, m[e], v[e], g);
    m[e] = s.m;
    v[e] = s.v;
    p[e] = step_of(b, c, p[e], s);
  }
  unsigned qm[1], qv[1];
  if (BITS == 8)
    requantize<4, 64>(m, v, c.key, t.block0 + blk, at % kBlock, t.m_scale + blk,
                      t.v_scale + blk, qm, qv);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (e >= live) continue;
    P[at + e] = Elem<D>::down(p[e]);
    if (BITS == 32) {
      static_cast<float*>(t.m)[at + e] = m[e];
      static_cast<float*>(t.v)[at + e] = v[e];
    } else {
      static_cast<uint8_t*>(t.m)[at + e] = static_cast<uint8_t>(qm[0] >> (8 * e));
      static_cast<uint8_t*>(t.v)[at + e] = static_cast<uint8_t>(qv[0] >> (8 * e));
    }
  }
}

// A workgroup takes `per` x 1024 elements: 1 where there is little to do, so that
// every wave has one block and one trip to memory; 4 otherwise, with states in
// 8 bits 16 elements a lane (whole 16-byte loads of the codes, and a block's
// largest value among 16 lanes).
template <int D, int BITS, int PER> __global__ __launch_bounds__(256) void k_adamw(Batch b) {
  int i = 0;
  while (i + 1 < b.count && static_cast<int>(blockIdx.x) >= b.at[i + 1].first) ++i;
  const Tensor& t = b.at[i];
  const int64_t chunk = static_cast<int64_t>(blockIdx.x - t.first) * (PER * 1024);
  Scalars c = {b.size, b.root, b.key};
  if (b.device) {
    const float* d = b.device + i * b.each;
    c = {d[0], d[1], to_bits(d[2])};
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (PER == 4 && t.wide() && chunk + PER * 1024 <= t.n()) {
    if constexpr (BITS == 8) {
      step_wide<D, BITS, 16>(b, c, t, chunk + tid * 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) step_wide<D, BITS, 4>(b, c, t, chunk + (j * 256 + tid) * 4);
    }
    return;
  }
  for (int j = 0; j < PER; ++j) {
    const int64_t first = chunk + (j * 4 + wave) * kBlock;
    if (first >= t.n()) return;
    if (t.wide() && first + kBlock <= t.n()) step_wide<D, BITS, 4>(b, c, t, first + lane * 4);
    else step_any<D, BITS>(b, c, t, first + lane * 4);
  }
}

static_assert(sizeof(Batch) <= 4096, "the arguments of a launch");

struct Corrections {
  float size, root;
};

__host__ __device__ inline Corrections corrections(double lr, double b1, double b2, double t) {
  return {static_cast<float>(lr / (1 - pow(b1, t))),
          static_cast<float>(1 / sqrt(1 - pow(b2, t)))};
}

struct Steps {
  const int64_t* at[kMost];
};

// A thread for each count on the device.
__global__ void k_adamw_scalars(double lr, double b1, double b2, unsigned seed, Steps steps,
                                float* out) {
  const int64_t t = *steps.at[threadIdx.x];
  out += threadIdx.x * 4;
  const Corrections c = corrections(lr, b1, b2, static_cast<double>(t));
  out[0] = c.size;
  out[1] = c.root;
  out[2] = from_bits(mix(seed ^ mix(static_cast<unsigned>(t))));
}

template <int D, int BITS> void launch(int per, unsigned grid, hipStream_t s, const Batch& b) {
  if (per == 1)
    hipLaunchKernelGGL((k_adamw<D, BITS, 1>), dim3(grid), dim3(256), 0, s, b);
  else
    hipLaunchKernelGGL((k_adamw<D, BITS, 4>), dim3(grid), dim3(256), 0, s, b);
}

template <int D> void launch(int bits, int per, unsigned grid, hipStream_t s, const Batch& b) {
  if (bits == 32) launch<D, 32>(per, grid, s, b);
  else launch<D, 8>(per, grid, s, b);
}

}  // namespace

extern "C" int fedtrain_adamw(int dtype, int state_bits, int64_t count,
                              const fedtrain_adamw_tensor* tensors,
                              const fedtrain_adamw_scalars* s, void* stream) {
  if (dtype < FEDTRAIN_F32 || dtype > FEDTRAIN_F16 || (state_bits != 8 && state_bits != 32) ||
      count < 0 || (count && !tensors) || !s)
    return FEDTRAIN_EINVAL;
  if (s->device_step || s->device_steps ? !s->workspace || !aligned(s->workspace, 4) : s->step < 1)
    return FEDTRAIN_EINVAL;
  if (!(s->beta1 >= 0 && s->beta1 < 1 && s->beta2 >= 0 && s->beta2 < 1 && s->lr >= 0 &&
        s->eps >= 0 && s->weight_decay >= 0))
    return FEDTRAIN_EINVAL;
  const size_t esize = dtype == FEDTRAIN_F32 ? 4 : 2, ssize = state_bits == 32 ? 4 : 1;
  int64_t total = 0;
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
    if (t.n > kMostGroups * 1024) return FEDTRAIN_EINVAL;
    if (s->device_steps && !(s->device_steps[i] && aligned(s->device_steps[i], 8)))
      return FEDTRAIN_EINVAL;
    total += t.n;
  }
  // below 4 workgroups of 1024 elements a compute unit the smaller ones win
  const int per = total < 4 * 256 * 1024 ? 1 : 4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  Batch b;
  b.b1 = static_cast<float>(s->beta1);
  b.c1 = static_cast<float>(1 - s->beta1) * (s->maximize ? -1.0f : 1.0f);
  b.b2 = static_cast<float>(s->beta2);
  b.c2 = static_cast<float>(1 - s->beta2);
  b.decay = static_cast<float>(1 - s->lr * s->weight_decay);
  // below the smallest normal number its reciprocal would be an infinity, and m = 0
  // times it NaN; the root of any v above 0 is far larger
  b.eps = s->eps > 0 ? fmaxf(static_cast<float>(s->eps), 0x1p-126f) : 0.0f;
  b.device = nullptr;
  b.each = 0;
  b.size = b.root = 0;
  b.key = 0;
  Steps steps;
  float* scalars = static_cast<float*>(s->workspace);  // of the launch's first tensor
  auto count_on_device = [&](int n) {
    b.device = scalars;
    hipLaunchKernelGGL(k_adamw_scalars, dim3(1), dim3(n), 0, st, s->lr, s->beta1, s->beta2,
                       s->seed, steps, scalars);
    return launched();
  };
  if (s->device_steps) {
    b.each = 4;
  } else if (s->device_step) {
    steps.at[0] = s->device_step;
    if (const int rc = count_on_device(1)) return rc;
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
      const int64_t groups = (t.n + per * 1024 - 1) / (per * 1024);
      if (grid + groups > kMostGroups) break;
      if (s->device_steps) steps.at[b.count] = s->device_steps[i];
      Tensor& at = b.at[b.count++];
      at.p = t.p;
      at.g = t.g;
      at.m = t.m;
      at.v = t.v;
      at.m_scale = t.m_scale;
      at.v_scale = t.v_scale;
      at.first = static_cast<int>(grid);
      at.block0 = static_cast<unsigned>(t.block0);
      at.n_wide = t.n * 2 + (aligned(t.p, 16) && aligned(t.g, 16) && aligned(t.m, 16) &&
                             aligned(t.v, 16));
      grid += groups;
    }
    if (!b.count) break;
    if (s->device_steps) {
      if (const int rc = count_on_device(b.count)) return rc;
      scalars += 4 * b.count;
    }
    const unsigned n = static_cast<unsigned>(grid);
    if (dtype == FEDTRAIN_F32) launch<FEDTRAIN_F32>(state_bits, per, n, st, b);
    else if (dtype == FEDTRAIN_BF16) launch<FEDTRAIN_BF16>(state_bits, per, n, st, b);
    else launch<FEDTRAIN_F16>(state_bits, per, n, st, b);
    if (const int rc = launched()) return rc;
  }
  return 0;
}

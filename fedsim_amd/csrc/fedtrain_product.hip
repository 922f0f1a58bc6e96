// Matrix products with bias, activation and residual in the epilogue, of one
// weight matrix or grouped by client with ragged row counts, and the products
// of their gradients (fedtrain_product, fedtrain_act_backward).
//
//   forward       z = A B^T + bias,  C = act(z) + res      A rows, B weights
//   grad input    C = A B                                  A = dz, B weights
//   grad weight   C = A^T B, colsum = A^T 1                A = dz, B = x
#include "fedtrain_common.h"

#include <climits>
#include <type_traits>

namespace {

using namespace fedtrain;

using Args = fedtrain_product_args;

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------
// erf to 1.5e-7 (Abramowitz and Stegun 7.1.26) with e = exp(-x^2) at hand: a
// fifth of erff's instructions, and far inside a 16-bit result's rounding.
__device__ inline float erf_of(float x, float e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(x), 0.3275911f, 1.0f));
  float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  p = __builtin_fmaf(t, p, 1.421413741f);
  p = __builtin_fmaf(t, p, -0.284496736f);
  p = __builtin_fmaf(t, p, 0.254829592f);
  return copysignf(__builtin_fmaf(-p * t, e, 1.0f), x);
}

constexpr float kLog2e = 1.4426950408889634f;

template <int D, int ACT> __device__ inline float act_value(float z) {
  if constexpr (ACT == FEDTRAIN_ACT_RELU) return z > 0 || z != z ? z : 0.0f;
  if constexpr (ACT == FEDTRAIN_ACT_GELU) {
    const float x = z * 0.70710678118654752f;
    const float f = D == FEDTRAIN_F32 ? erff(x)
                                      : erf_of(x, __builtin_amdgcn_exp2f(x * x * -kLog2e));
    return 0.5f * z * (1.0f + f);
  }
  if constexpr (ACT == FEDTRAIN_ACT_SILU)
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -kLog2e));
  return z;
}

template <int D, int ACT> __device__ inline float act_slope(float z) {
  if constexpr (ACT == FEDTRAIN_ACT_RELU) return z > 0 ? 1.0f : 0.0f;
  if constexpr (ACT == FEDTRAIN_ACT_GELU) {
    const float x = z * 0.70710678118654752f;
    const float e = __builtin_amdgcn_exp2f(x * x * -kLog2e);
    const float f = D == FEDTRAIN_F32 ? erff(x) : erf_of(x, e);
    // z e is 0 where e is, whatever z
    return 0.5f * (1.0f + f) + (e > 0 ? z * e : 0.0f) * 0.39894228040143268f;
  }
  if constexpr (ACT == FEDTRAIN_ACT_SILU) {
    const float t = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -kLog2e));
    return t * (1.0f + z * (1.0f - t));
  }
  return 1.0f;
}

// f(a constant of each activation)
template <class F> __device__ inline void by_act(int act, F f) {
  if (act == FEDTRAIN_ACT_NONE) f(std::integral_constant<int, FEDTRAIN_ACT_NONE>());
  else if (act == FEDTRAIN_ACT_RELU) f(std::integral_constant<int, FEDTRAIN_ACT_RELU>());
  else if (act == FEDTRAIN_ACT_GELU) f(std::integral_constant<int, FEDTRAIN_ACT_GELU>());
  else f(std::integral_constant<int, FEDTRAIN_ACT_SILU>());
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

// The group of one row, -1 if it is in none: the last range that begins at or
// before it.
__device__ inline int group_of(const Args& a, int64_t row) {
  int at = 0, n = a.groups + 2;
  while (n > 1) {
    const int half = n / 2;
    if (bound(a, a.m, at + half) <= row) {
      at += half;
      n -= half;
    } else {
      n = half;
    }
  }
  return at - 1 < a.groups ? at - 1 : -1;
}

// ---------------------------------------------------------------------------
// the product: tiles in LDS
// ---------------------------------------------------------------------------
// An operand's tile is kept as it lies in memory, in chunks of 8 elements.  Where
// k is the closest dimension (KC) a line is a row with BK of its k; else (KS) a
// line is one k with W rows' values, and the matrix unit's fragments are read
// with the transposing load.  In both a line's chunks are exchanged by xor, so
// that the lanes that LDS serves together meet different banks.
//
// f32 operands are split into three bf16 parts by cutting off bits, x = h + m + l
// exactly, one plane each; the six products hh, hm, mh, hl, mm, lh keep all but
// 2^-21 of |a b| (after Henry, Tang and Heinecke, 2019: the bf16 unit is 16
// times the f32 unit's rate, so six products are 2.7 times faster than one).

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((address_space(3))) char lds_char;

template <int D> __device__ inline f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (D == FEDTRAIN_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// How a tile of an operand lies in LDS.  NJ: the column operand's rows are read
// in the order that gives a lane 4 NJ neighbouring columns of C (0: in order).
template <bool KS_, int W_, int BK_, int NJ_> struct Tile {
  static constexpr bool KS = KS_;
  static constexpr int W = W_, BK = BK_, NJ = NJ_;
  static constexpr int per_line = (KS ? W : BK) / 8;
  static constexpr int chunks = W * BK / 8;
  static constexpr int bytes = chunks * 16;  // of one plane

  static __device__ int swizzle(int line) {
    if constexpr (KS) {
      return (((line & 3) | ((line >> 3) & 3) << 2) & (W / 16 - 1)) << 1;
    } else {
      const int high = NJ == 0 ? 2 : NJ == 1 ? 2 : NJ == 2 ? 3 : 4;  // of the next 4 lanes' rows
      if constexpr (BK == 64) return (line & 3) | ((line >> high) & 1) << 2;
      return ((line >> 1) & 1) | ((line >> high) & 1) << 1;
    }
  }
  static __device__ int at(int line, int chunk) {
    return (line * per_line + (chunk ^ swizzle(line))) * 16;
  }
  // tile t (16 rows from row0) of k step kk, for the lane
  static __device__ s16x8 fragment(const char* base, int row0, int t, int kk, int lane) {
    const int r = lane & 15, q = lane >> 4;
    if constexpr (KS) {
      const int k = kk * 32 + q * 8 + (r >> 2), row = row0 + t * 16 + (r & 3) * 4;
      s16x4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char* p = base + at(k + h * 4, row >> 3) + (row & 4) * 2;
        v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(p));
      }
      return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const int row = row0 + (NJ ? (r >> 2) * (4 * NJ) + t * 4 + (r & 3) : t * 16 + r);
      return *reinterpret_cast<const s16x8*>(base + at(row, kk * 4 + q));
    }
  }
};

// x's three bf16 parts, in the high halves.  An infinity or NaN is its first
// part alone; true for those.  (Parts below 2^-126 may be lost.)
__device__ inline bool split3(float x, unsigned& h, unsigned& m, unsigned& l) {
  const unsigned b = __builtin_bit_cast(unsigned, x);
  h = b & 0xFFFF0000u;
  const bool odd = (b & 0x7F800000u) == 0x7F800000u;
  if (odd && (b & 0xFFFFu)) h |= 0x10000u;  // a NaN stays one
  const float r = odd ? 0.0f : x - __builtin_bit_cast(float, h);
  m = __builtin_bit_cast(unsigned, r) & 0xFFFF0000u;
  l = __builtin_bit_cast(unsigned, r - __builtin_bit_cast(float, m)) & 0xFFFF0000u;
  return odd;
}

// The value that three parts stand for.
__device__ inline float joined(short h, short m, short l) {
  auto up = [](short x) {
    return __builtin_bit_cast(float, static_cast<unsigned>(static_cast<unsigned short>(x)) << 16);
  };
  return up(h) + up(m) + up(l);
}

// An operand's tile on its way to LDS: `rows` of its rows (KC) or columns (KS)
// exist, k runs to k1.
template <int D, class L, int THREADS, bool DIRECT> struct Loader {
  using T = typename Elem<D>::type;
  static constexpr int N = L::chunks / THREADS;
  static_assert(L::chunks % THREADS == 0, "chunks a thread");
  static constexpr int R = D == FEDTRAIN_F32 ? 2 : 1;
  const T* base;  // the tile at k = 0
  int64_t ld;
  int rows;
  u32x4 held[DIRECT ? 1 : N][R];
  unsigned offset[DIRECT ? N : 1];

  __device__ void init(const void* p, int64_t ld_, int64_t row0, int64_t rows_, int tid) {
    ld = ld_;
    rows = static_cast<int>(rows_ < L::W ? rows_ : L::W);
    base = static_cast<const T*>(p) + (L::KS ? row0 : row0 * ld);
    if constexpr (DIRECT) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int q = tid + i * THREADS, line = q / L::per_line;
        const int c = (q % L::per_line) ^ L::swizzle(line);
        const bool in = L::KS ? c * 8 < rows : line < rows;
        offset[i] = in ? static_cast<unsigned>(line * ld + c * 8) * 2u : ~0u;
      }
    }
  }

  // DIRECT: memory to LDS without registers.  A lane outside the operand asks
  // for an offset past the descriptor's range, which stores zeros.
  __device__ void issue(int64_t k, int64_t k1, char* to, int tid) const {
    const int64_t first = L::KS ? k * ld : k;
    auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + first), 0, 0x7FFFFFFF,
                                               0x00027000);
    const int left = k1 - k < L::BK ? static_cast<int>(k1 - k) : L::BK;
    to += __builtin_amdgcn_readfirstlane(tid & ~63) * 16;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned o = offset[i];
      if (left < L::BK) {
        const int q = tid + i * THREADS, line = q / L::per_line;
        const int c = (q % L::per_line) ^ L::swizzle(line);
        if (L::KS ? line >= left : c * 8 >= left) o = ~0u;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          d, (__attribute__((address_space(3))) void*)(to + i * THREADS * 16), 16, o, 0, 0, 0);
    }
  }

  // through registers: any alignment, any length
  __device__ void load(int64_t k, int64_t k1, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = tid + i * THREADS, line = q / L::per_line;
      const int c = (q % L::per_line) ^ L::swizzle(line);
      const int row = L::KS ? c * 8 : line;
      const int64_t kk = k + (L::KS ? line : c * 8);
      const T* p = base + (L::KS ? kk * ld + row : row * ld + kk);
      int n = L::KS ? (kk < k1 ? rows - row : 0)
                    : (row < rows ? static_cast<int>(k1 - kk < 8 ? k1 - kk : 8) : 0);
      if (n >= 8) {
        __builtin_memcpy(&held[i][0], p, 16 * R);
      } else {
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : Elem<D>::down(0);
        __builtin_memcpy(&held[i][0], v, 16 * R);
      }
    }
  }

  // f32: *odd becomes 1 where an infinity or NaN was met
  __device__ void store(char* to, int tid, int* odd) const {
    bool met = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      char* p = to + (tid + i * THREADS) * 16;
      if constexpr (D != FEDTRAIN_F32) {
        *reinterpret_cast<u32x4*>(p) = held[i][0];
      } else {
        u32x4 out[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unsigned h[2], m[2], l[2];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int n = e * 2 + s;
            const unsigned bits = held[i][n / 4][n % 4];
            met |= split3(__builtin_bit_cast(float, bits), h[s], m[s], l[s]);
          }
          out[0][e] = __builtin_amdgcn_perm(h[1], h[0], 0x07060302);
          out[1][e] = __builtin_amdgcn_perm(m[1], m[0], 0x07060302);
          out[2][e] = __builtin_amdgcn_perm(l[1], l[0], 0x07060302);
        }
#pragma unroll
        for (int e = 0; e < 3; ++e) *reinterpret_cast<u32x4*>(p + e * L::bytes) = out[e];
      }
    }
    if (D == FEDTRAIN_F32 && met) *odd = 1;
  }
};

// The shape of a workgroup: MW x NW waves, each with MI x NI tiles of 16 x 16.
template <int MW_, int NW_, int MI_, int NI_, int BK_> struct Shape {
  static constexpr int MW = MW_, NW = NW_, MI = MI_, NI = NI_, BK = BK_;
  static constexpr int BM = MW * MI * 16, BN = NW * NI * 16, THREADS = MW * NW * 64;
};

// Workgroups go to the 8 dies in turn.  Each die gets a contiguous part of the
// tiles, in bands of 8 rows of tiles, so that what its workgroups read at a time
// is shared in its own L2.
__device__ inline void place(int64_t tiles_m, int64_t tiles_n, int64_t& tm, int64_t& tn) {
  const int64_t total = tiles_m * tiles_n, id = blockIdx.x;
  const int64_t share = total / 8, more = total % 8, die = id % 8;
  const int64_t t = die * share + (die < more ? die : more) + id / 8;
  const int64_t band = t / (8 * tiles_n), in = t - band * 8 * tiles_n;
  const int64_t height = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
  tn = in / height;
  tm = band * 8 + in % height;
}

__device__ inline void arrive() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
template <int N> __device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

struct Plan {
  int64_t tiles_m, tiles_n;  // tiles_m: of one group (grad weight), or slots
  int splits;                // parts of k; over 1, C is f32 partial sums in the workspace
  int wide;                  // 1: four neighbouring values of every operand of C at a time
};

// ---------------------------------------------------------------------------
// what becomes of the sums
// ---------------------------------------------------------------------------
template <class T> struct __attribute__((aligned(4 * sizeof(T)))) Four {
  T v[4];
};

template <int D> __device__ inline void read4(const void* p, int64_t at, int n, bool wide,
                                              float* to) {
  using T = typename Elem<D>::type;
  const T* x = static_cast<const T*>(p) + at;
  if (wide) {
    const Four<T> f = *reinterpret_cast<const Four<T>*>(x);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = Elem<D>::up(f.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = e < n ? Elem<D>::up(x[e]) : 0.0f;
  }
}

template <int D> __device__ inline void write4(void* p, int64_t at, int n, bool wide,
                                               const float* v) {
  using T = typename Elem<D>::type;
  T* x = static_cast<T*>(p) + at;
  if (wide) {
    Four<T> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f.v[e] = Elem<D>::down(v[e]);
    *reinterpret_cast<Four<T>*>(x) = f;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) x[e] = Elem<D>::down(v[e]);
  }
}

// n <= 4 neighbouring sums of a row of C, to their end
template <int D, int FORM, int ACT>
__device__ inline void put(const Args& a, int group, int64_t row, int64_t col, int n, bool wide,
                           float* v) {
  if constexpr (FORM == FEDTRAIN_FORWARD) {
    if (group >= 0) {
      if (a.bias) {
        float b[4];
        read4<D>(a.bias, group * a.bias_group + col, n, wide, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += b[e];
      }
      if (a.z) write4<D>(a.z, row * a.ldz + col, n, wide, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = act_value<D, ACT>(v[e]);
    } else if (a.z) {
      write4<D>(a.z, row * a.ldz + col, n, wide, v);
    }
    if (a.res) {
      float r[4];
      read4<D>(a.res, row * a.ldr + col, n, wide, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += r[e];
    }
  }
  const int64_t first = FORM == FEDTRAIN_GRAD_WEIGHT ? group * a.c_group : 0;
  write4<D>(a.c, first + row * a.ldc + col, n, wide, v);
}

template <int D, int FORM, class S, bool DIRECT>
__global__ __launch_bounds__(S::THREADS) void k_product(Args a, Plan plan) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass needs the name alone
  using T = typename Elem<D>::type;
  constexpr bool WEIGHT = FORM == FEDTRAIN_GRAD_WEIGHT;
  constexpr int PLANES = D == FEDTRAIN_F32 ? 3 : 1;
  using LA = Tile<WEIGHT, S::BM, S::BK, 0>;
  using LB = Tile<FORM != FEDTRAIN_FORWARD, S::BN, S::BK, FORM == FEDTRAIN_FORWARD ? S::NI : 0>;
  constexpr int STAGE = PLANES * (LA::bytes + LB::bytes);
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / S::NW * (S::MI * 16), wn = wave % S::NW * (S::NI * 16);
  int64_t slot, tn;
  place(plan.tiles_m * (WEIGHT && a.groups ? a.groups : 1), plan.tiles_n, slot, tn);
  const int64_t col0 = tn * S::BN;
  int64_t row0, rows, k0 = 0, k1 = a.k;
  int group = 0;
  if (WEIGHT) {
    if (a.groups) {
      group = static_cast<int>(slot / plan.tiles_m);
      slot %= plan.tiles_m;
      k0 = bound(a, a.k, group + 1);
      k1 = bound(a, a.k, group + 2);
    }
    row0 = slot * S::BM;
    rows = a.m - row0 < S::BM ? a.m - row0 : S::BM;
  } else {
    const Rows r = rows_of(a, slot, S::BM);
    if (r.lo >= r.hi) return;
    row0 = r.lo;
    rows = r.hi - r.lo;
    group = r.group;
    if (group < 0) k1 = 0;
  }
  if (plan.splits > 1) {  // an even part, in whole tiles
    const int64_t part = ((k1 - k0 + S::BK - 1) / S::BK + plan.splits - 1) / plan.splits * S::BK;
    k0 += part * blockIdx.y;
    if (k0 + part < k1) k1 = k0 + part;
  }
  const int64_t cols = a.n - col0 < S::BN ? a.n - col0 : S::BN;
  const T* B = static_cast<const T*>(a.b);
  if (!WEIGHT && group > 0) B += group * a.b_group;

  Loader<D, LA, S::THREADS, DIRECT> la;
  Loader<D, LB, S::THREADS, DIRECT> lb;
  la.init(a.a, a.lda, row0, rows, tid);
  lb.init(B, a.ldb, col0, cols, tid);

  f32x4 acc[S::MI][S::NI] = {};
  f32x4 sum[S::MI] = {};
  const bool want_sum = WEIGHT && a.colsum && col0 == 0 && wn == 0;

  int* odd = reinterpret_cast<int*>(lds + (DIRECT ? 2 : 1) * STAGE);
  auto compute = [&](const char* at) {
    const char* pa = at;
    const char* pb = at + PLANES * LA::bytes;
#pragma unroll
    for (int kk = 0; kk < S::BK / 32; ++kk) {
      s16x8 fb[S::NI][PLANES];
#pragma unroll
      for (int j = 0; j < S::NI; ++j)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          fb[j][p] = LB::fragment(pb + p * LB::bytes, wn, j, kk, lane);
#pragma unroll
      for (int i = 0; i < S::MI; ++i) {
        s16x8 fa[PLANES];
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          fa[p] = LA::fragment(pa + p * LA::bytes, wm, i, kk, lane);
        if constexpr (D == FEDTRAIN_F32) {
          // an infinity times a part that is 0 would be NaN: with one about, the
          // f32 unit takes the values as they were
          if (*odd) {
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
              const float x = joined(fa[0][e], fa[1][e], fa[2][e]);
#pragma unroll
              for (int j = 0; j < S::NI; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    joined(fb[j][0][e], fb[j][1][e], fb[j][2][e]), x, acc[i][j], 0, 0, 0);
              if (want_sum) sum[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(1.0f, x, sum[i], 0, 0, 0);
            }
            continue;
          }
        }
        // the columns go to the rows of the unit's result: a lane gets 4
        // neighbouring columns
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p)
#pragma unroll
          for (int s = 0; s <= p; ++s)
#pragma unroll
            for (int j = 0; j < S::NI; ++j)
              acc[i][j] = mfma<D>(fb[j][s], fa[p - s], acc[i][j]);
        if (want_sum) {
          s16x8 one;
#pragma unroll
          for (int e = 0; e < 8; ++e) one[e] = D == FEDTRAIN_F16 ? 0x3C00 : 0x3F80;
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) sum[i] = mfma<D>(one, fa[p], sum[i]);
        }
      }
    }
  };

  if constexpr (DIRECT) {
    constexpr int LOADS = LA::chunks / S::THREADS + LB::chunks / S::THREADS;
    if (k0 < k1) {
      la.issue(k0, k1, lds, tid);
      lb.issue(k0, k1, lds + LA::bytes, tid);
    }
    int turn = 0;
    for (int64_t k = k0; k < k1; k += S::BK, turn ^= 1) {
      if (k + S::BK < k1) {
        char* next = lds + (turn ^ 1) * STAGE;
        la.issue(k + S::BK, k1, next, tid);
        lb.issue(k + S::BK, k1, next + LA::bytes, tid);
        wait_loads<LOADS>();
      } else {
        wait_loads<0>();
      }
      arrive();
      compute(lds + turn * STAGE);
      arrive();
    }
  } else {
    if (D == FEDTRAIN_F32) {
      if (tid == 0) *odd = 0;
      __syncthreads();
    }
    if (k0 < k1) {
      la.load(k0, k1, tid);
      lb.load(k0, k1, tid);
    }
    for (int64_t k = k0; k < k1; k += S::BK) {
      la.store(lds, tid, odd);
      lb.store(lds + PLANES * LA::bytes, tid, odd);
      __syncthreads();
      if (k + S::BK < k1) {
        la.load(k + S::BK, k1, tid);
        lb.load(k + S::BK, k1, tid);
      }
      compute(lds);
      __syncthreads();
    }
  }

  // a lane holds the columns of one row: 4 NI neighbours (forward), or 4 in each
  // tile
  const int r16 = lane & 15, q = lane >> 4;
  auto column = [&](int j) { return wn + (LB::NJ ? q * 4 * S::NI + j * 4 : j * 16 + q * 4); };
  if (plan.splits > 1) {
    const int64_t width = (a.n + 3) / 4 * 4 + (a.colsum ? 4 : 0);
#pragma unroll
    for (int i = 0; i < S::MI; ++i) {
      const int r = wm + i * 16 + r16;
      if (r >= rows) continue;
      float* P = static_cast<float*>(a.workspace) +
                 (static_cast<int64_t>(blockIdx.y) * a.m + row0 + r) * width;
#pragma unroll
      for (int j = 0; j < S::NI; ++j)
        if (column(j) < cols) *reinterpret_cast<f32x4*>(P + col0 + column(j)) = acc[i][j];
      if (want_sum && q == 0) P[width - 4] = sum[i][0];
    }
    return;
  }
  if (want_sum && q == 0) {
#pragma unroll
    for (int i = 0; i < S::MI; ++i) {
      const int r = wm + i * 16 + r16;
      if (r < rows)
        static_cast<T*>(a.colsum)[group * a.colsum_group + row0 + r] = Elem<D>::down(sum[i][0]);
    }
  }
  if (WEIGHT && !a.c) return;
  by_act(FORM == FEDTRAIN_FORWARD ? a.act : 0, [&](auto act) {
#pragma unroll
    for (int i = 0; i < S::MI; ++i) {
      const int r = wm + i * 16 + r16;
      if (r >= rows) continue;
#pragma unroll
      for (int j = 0; j < S::NI; ++j) {
        const int c = column(j), n = static_cast<int>(cols) - c;
        if (n <= 0) continue;
        float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        put<D, FORM, decltype(act)::value>(a, group, row0 + r, col0 + c, n, plan.wide && n >= 4,
                                           v);
      }
    }
  });
#endif
}

// The parts of k added up in their order, for four columns a thread.
template <int D, int FORM> __global__ __launch_bounds__(256) void k_join(Args a, Plan plan) {
  using T = typename Elem<D>::type;
  const int64_t width = (a.n + 3) / 4 * 4 + (a.colsum ? 4 : 0), per = width / 4;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= a.m * per) return;
  const int64_t row = id / per, col = id % per * 4;
  const float* P = static_cast<const float*>(a.workspace) + row * width + col;
  f32x4 x = {0, 0, 0, 0};
  for (int s = 0; s < plan.splits; ++s) x += *reinterpret_cast<const f32x4*>(P + s * a.m * width);
  if (col >= a.n) {
    if (a.colsum) static_cast<T*>(a.colsum)[row] = Elem<D>::down(x[0]);
    return;
  }
  if (FORM == FEDTRAIN_GRAD_WEIGHT && !a.c) return;
  int group = 0;
  if (FORM != FEDTRAIN_GRAD_WEIGHT && a.groups) {
    group = group_of(a, row);
    if (group < 0) x = f32x4{0, 0, 0, 0};
  }
  const int n = static_cast<int>(a.n - col < 4 ? a.n - col : 4);
  float v[4] = {x[0], x[1], x[2], x[3]};
  by_act(FORM == FEDTRAIN_FORWARD ? a.act : 0, [&](auto act) {
    put<D, FORM, decltype(act)::value>(a, group, row, col, n, plan.wide && n >= 4, v);
  });
}

// dz = dy act'(z): one pass, eight values a thread where rows allow it
template <int D, int ACT, int V>
__global__ __launch_bounds__(256) void k_act_backward(int64_t rows, int64_t cols, const void* dy,
                                                      int64_t lddy, const void* z, int64_t ldz,
                                                      void* dz, int64_t lddz) {
  using T = typename Elem<D>::type;
  struct __attribute__((aligned(V * sizeof(T)))) Vec {
    T v[V];
  };
  const int64_t per = cols / V;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t r = i / per, c = i % per * V;
  const Vec g = *reinterpret_cast<const Vec*>(static_cast<const T*>(dy) + r * lddy + c);
  const Vec x = *reinterpret_cast<const Vec*>(static_cast<const T*>(z) + r * ldz + c);
  Vec out;
#pragma unroll
  for (int e = 0; e < V; ++e)
    out.v[e] = Elem<D>::down(Elem<D>::up(g.v[e]) * act_slope<D, ACT>(Elem<D>::up(x.v[e])));
  *reinterpret_cast<Vec*>(static_cast<T*>(dz) + r * lddz + c) = out;
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

bool in_eights(const Args& a) {
  // Whether the operands' chunks of 8 can go to LDS directly: they are whole and
  // 16-byte aligned, and a tile's offsets fit the 31 bits of a descriptor.
  const int64_t m = a.form == FEDTRAIN_GRAD_WEIGHT ? a.m : a.k;
  const int64_t n = a.form == FEDTRAIN_FORWARD ? a.k : a.n;
  return a.dtype != FEDTRAIN_F32 && aligned(a.a, 16) && aligned(a.b, 16) && m % 8 == 0 &&
         n % 8 == 0 && a.lda % 8 == 0 && a.ldb % 8 == 0 && a.b_group % 8 == 0 &&
         a.lda < (1 << 21) && a.ldb < (1 << 21);
}

bool in_fours(const Args& a) {
  const size_t size = a.dtype == FEDTRAIN_F32 ? 16 : 8;
  return aligned(a.c, size) && aligned(a.z, size) && aligned(a.res, size) &&
         aligned(a.bias, size) && a.ldc % 4 == 0 && a.c_group % 4 == 0 &&
         (!a.z || a.ldz % 4 == 0) && (!a.res || a.ldr % 4 == 0) && a.bias_group % 4 == 0;
}

enum class Size { Large, Middle, Small };

struct Choice {
  Size size;
  int splits;
};

// Tiles of (256, 256), (128, 128) or (64, 64), the largest that leaves a
// workgroup for most of the 256 compute units; and where the smallest tiles do
// not, k in parts.
Choice choose(const Args& a) {
  const bool weight = a.form == FEDTRAIN_GRAD_WEIGHT;
  const int64_t groups = a.groups ? a.groups : 1;
  auto tiles = [&](int64_t b) {
    const int64_t n = a.n ? (a.n + b - 1) / b : 1;
    const int64_t m = weight ? (a.m + b - 1) / b * groups
                             : (a.m + b - 1) / b + (a.groups ? a.groups / 2 : 0);
    return m * n;
  };
  const int64_t rows = weight ? a.m : a.m / groups;  // of one weight matrix
  if (a.dtype != FEDTRAIN_F32 && in_eights(a) && rows >= 192 && a.n >= 192 && tiles(256) >= 192)
    return {Size::Large, 1};
  if (rows >= 96 && a.n >= 96 && tiles(128) >= 192) return {Size::Middle, 1};
  int64_t splits = 1;
  const int64_t have = tiles(64), steps = (a.k + 63) / 64;
  if (!(weight && a.groups) && have > 0 && have < 256) {
    splits = (512 + have - 1) / have;
    if (splits > steps / 4) splits = steps / 4;
    if (splits > 64) splits = 64;
    if (splits < 1) splits = 1;
  }
  return {Size::Small, static_cast<int>(splits)};
}

int64_t workspace(const Args& a) {
  const int s = choose(a).splits;
  if (s < 2) return 0;
  return static_cast<int64_t>(s) * a.m * ((a.n + 3) / 4 * 4 + (a.colsum ? 4 : 0)) * 4;
}

template <int D, int FORM, class S, bool DIRECT> int go(const Args& a, int splits, hipStream_t s) {
  Plan p;
  p.splits = splits;
  p.wide = in_fours(a);
  p.tiles_n = a.n ? (a.n + S::BN - 1) / S::BN : 1;
  int64_t all;
  if (FORM == FEDTRAIN_GRAD_WEIGHT) {
    p.tiles_m = (a.m + S::BM - 1) / S::BM;
    all = p.tiles_m * (a.groups ? a.groups : 1);
  } else {
    all = p.tiles_m = a.groups ? a.m / S::BM + a.groups + 2 : (a.m + S::BM - 1) / S::BM;
  }
  if (all > INT32_MAX / p.tiles_n) return FEDTRAIN_EINVAL;
  constexpr int PLANES = D == FEDTRAIN_F32 ? 3 : 1;
  constexpr int BYTES = (DIRECT ? 2 : 1) * PLANES * (S::BM + S::BN) * S::BK * 2 +
                        (D == FEDTRAIN_F32 ? 16 : 0);  // and the mark of an infinity
  auto* kernel = &k_product<D, FORM, S, DIRECT>;
  if (BYTES > 64 * 1024) {
    // for the current device; it costs about a microsecond
    const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (set != hipSuccess) return static_cast<int>(set);
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(all * p.tiles_n), splits),
                     dim3(S::THREADS), BYTES, s, a, p);
  if (splits > 1) {
    if (const int rc = launched()) return rc;
    const int64_t fours = a.m * ((a.n + 3) / 4 + (a.colsum ? 1 : 0));
    if (fours > static_cast<int64_t>(INT32_MAX) * 256) return FEDTRAIN_EINVAL;
    hipLaunchKernelGGL((k_join<D, FORM>), dim3(static_cast<unsigned>((fours + 255) / 256)),
                       dim3(256), 0, s, a, p);
  }
  return launched();
}

template <int D, int FORM> int run(const Args& a, hipStream_t s) {
  const Choice c = choose(a);
  if (c.splits > 1 && (!a.workspace || !aligned(a.workspace, 16) ||
                       a.workspace_bytes < workspace(a)))
    return FEDTRAIN_EINVAL;
  if constexpr (D == FEDTRAIN_F32) {
    if (c.size == Size::Small) return go<D, FORM, Shape<2, 2, 2, 2, 32>, false>(a, c.splits, s);
    return go<D, FORM, Shape<2, 2, 4, 4, 32>, false>(a, 1, s);
  } else {
    if (c.size == Size::Large) return go<D, FORM, Shape<2, 4, 8, 4, 64>, true>(a, 1, s);
    const bool d = in_eights(a);
    if (c.size == Size::Middle)
      return d ? go<D, FORM, Shape<2, 2, 4, 4, 64>, true>(a, 1, s)
               : go<D, FORM, Shape<2, 2, 4, 4, 64>, false>(a, 1, s);
    return d ? go<D, FORM, Shape<2, 2, 2, 2, 64>, true>(a, c.splits, s)
             : go<D, FORM, Shape<2, 2, 2, 2, 64>, false>(a, c.splits, s);
  }
}

template <int D> int run(const Args& a, hipStream_t s) {
  if (a.form == FEDTRAIN_FORWARD) return run<D, FEDTRAIN_FORWARD>(a, s);
  if (a.form == FEDTRAIN_GRAD_INPUT) return run<D, FEDTRAIN_GRAD_INPUT>(a, s);
  return run<D, FEDTRAIN_GRAD_WEIGHT>(a, s);
}

struct Slope {
  int64_t rows, cols;
  const void* dy;
  int64_t lddy;
  const void* z;
  int64_t ldz;
  void* dz;
  int64_t lddz;
};

template <int D, int ACT, int V> int slope(const Slope& x, hipStream_t s) {
  const int64_t n = x.rows * (x.cols / V);
  if (n > static_cast<int64_t>(INT32_MAX) * 256) return FEDTRAIN_EINVAL;
  hipLaunchKernelGGL((k_act_backward<D, ACT, V>), dim3(static_cast<unsigned>((n + 255) / 256)),
                     dim3(256), 0, s, x.rows, x.cols, x.dy, x.lddy, x.z, x.ldz, x.dz, x.lddz);
  return launched();
}

template <int D, int ACT> int slope(const Slope& x, hipStream_t s) {
  constexpr int V = D == FEDTRAIN_F32 ? 4 : 8;
  const bool wide = aligned(x.dy, 16) && aligned(x.z, 16) && aligned(x.dz, 16) &&
                    x.cols % V == 0 && x.lddy % V == 0 && x.ldz % V == 0 && x.lddz % V == 0;
  return wide ? slope<D, ACT, V>(x, s) : slope<D, ACT, 1>(x, s);
}

template <int D> int slope(int act, const Slope& x, hipStream_t s) {
  if (act == FEDTRAIN_ACT_RELU) return slope<D, FEDTRAIN_ACT_RELU>(x, s);
  if (act == FEDTRAIN_ACT_GELU) return slope<D, FEDTRAIN_ACT_GELU>(x, s);
  if (act == FEDTRAIN_ACT_SILU) return slope<D, FEDTRAIN_ACT_SILU>(x, s);
  return slope<D, FEDTRAIN_ACT_NONE>(x, s);
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
  return valid(args) ? workspace(*args) : FEDTRAIN_EINVAL;
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
  const Slope x = {rows, cols, dy, lddy, z, ldz, dz, lddz};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FEDTRAIN_F32) return slope<FEDTRAIN_F32>(act, x, s);
  if (dtype == FEDTRAIN_BF16) return slope<FEDTRAIN_BF16>(act, x, s);
  return slope<FEDTRAIN_F16>(act, x, s);
}

}  // extern "C"

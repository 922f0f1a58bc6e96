// Matrix products with bias, activation and residual in the epilogue, of one
// weight matrix or grouped by client with ragged row counts, and the products
// of their gradients (fedtrain_product, fedtrain_act_backward).
//
//   forward       z = A B^T + bias,  C = act(z) + res      A rows, B weights
//   grad input    C = A B                                  A = dz, B weights
//   grad weight   C = A^T B, colsum = A^T 1                A = dz, B = x
//
// Sums, bias, activation and residual are f32; C and z are rounded to their type
// once, at the store.  The activation's gradient is taken at the rounded z, and
// dz = dy act'(z) is rounded to the type before dx and dW, whose matrix instructions
// take operands of that type: in 16 bits they are 0.0024 (bf16) and 0.0003 (f16) from
// the exact result in the mean, where their own rounding alone makes 0.0017 and
// 0.0002.  f32 z and dz would be twice the bytes, and dz in two parts twice the
// products.  db is summed from dz as it is before that.
//
// One kernel (k_product) in tiles of 256 x 256, 128 x 128 and 64 x 64 (f32: 64 x
// 128), picked by choose().  What bounds it, as measured on one MI355X (a copy
// reaches 4.64 TB/s, the library's product of 8192^3 bf16 1.31 and f32 0.15
// PFLOP/s):
//   large 16-bit products   the matrix unit at the clock that power leaves:
//                           8192 x 4096 x 16384 bf16 in 830 to 960 us, 1.14 to
//                           1.32 PFLOP/s, in tiles of 256 x 256
//   large f32 products      six bf16 products each: 194 TFLOP/s at 8192^3; 2048 x 512
//                           x 3136 in 54 to 59 us, 111 to 122 TFLOP/s, and 7 to 8 for
//                           parts of k: with few workgroups on a compute unit a
//                           step's loads, split and two barriers are its time
//   1000 clients' weights   memory: 3.5 GB of weights read once, 0.82 to 0.96 ms
//   64 experts              tiles that ragged groups fill by two thirds: forward 610
//                           us, grad input 510, of 400 by memory and 290 by the matrix
//                           unit; grad weight 720 to 850, four steps of k a tile
//   a client's small batch  launches and the trip to memory: 5 to 9 us each
#include "fedtrain_common.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

namespace {

using namespace fedtrain;

using Args = fedtrain_product_args;

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------
// Phi(z), the normal distribution's sum, for a 16-bit result, with e =
// exp(-z^2 / 2) at hand.  With x = |z| / sqrt(2), erfc(x) / exp(-x^2) is a polynomial
// in t = 1 / (1 + 0.37 x) to 7.6e-7 of itself for x up to 9.6 (fitted here, least
// largest relative error; beyond, e underflows).  1 + erf would cancel for negative
// z: at z = -4.5 it is off by ten roundings of a float16, and all of it at -6.
__device__ inline float phi_of(float z, float e) {
  const float t =
      __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.37f * 0.70710678118654752f, 1.0f));
  float p = __builtin_fmaf(t, -0.142360942f, 0.434967045f);
  p = __builtin_fmaf(t, p, -0.185421152f);
  p = __builtin_fmaf(t, p, 0.316651476f);
  p = __builtin_fmaf(t, p, 0.152958472f);
  p = __builtin_fmaf(t, p, 0.214821000f);
  p = __builtin_fmaf(t, p, 0.208384861f);
  const float half = 0.5f * p * t * e;
  return z < 0 ? half : 1.0f - half;
}

// The same for f32, by the library's erfc: 8192 x 8192 outputs of 256 inputs 276 us and
// their gradient's pass 146, where erff, which cancels, made 253 and 137.
__device__ inline float phi(float z) { return 0.5f * erfcf(z * -0.70710678118654752f); }

constexpr float kLog2e = 1.4426950408889634f;

template <int D, int ACT> __device__ inline float act_value(float z) {
  if constexpr (ACT == FEDTRAIN_ACT_RELU) return z > 0 || z != z ? z : 0.0f;
  if constexpr (ACT == FEDTRAIN_ACT_GELU) {
    if (D == FEDTRAIN_F32) return z * phi(z);
    return z * phi_of(z, __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e)));
  }
  if constexpr (ACT == FEDTRAIN_ACT_SILU)
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -kLog2e));
  return z;
}

template <int D, int ACT> __device__ inline float act_slope(float z) {
  if constexpr (ACT == FEDTRAIN_ACT_RELU) return z > 0 ? 1.0f : 0.0f;
  if constexpr (ACT == FEDTRAIN_ACT_GELU) {
    const float e = __builtin_amdgcn_exp2f(z * z * (-0.5f * kLog2e));
    // z e is 0 where e is, whatever z
    return (D == FEDTRAIN_F32 ? phi(z) : phi_of(z, e)) +
           (e > 0 ? z * e : 0.0f) * 0.39894228040143268f;
  }
  if constexpr (ACT == FEDTRAIN_ACT_SILU) {
    const float t = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -kLog2e));
    // a finite sum may be an infinity in z's type: 0 and 1 there, not 0 times it
    const float finite = fminf(fmaxf(z, -FLT_MAX), FLT_MAX);
    return t * (1.0f + finite * (1.0f - t));
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
// f32 operands are split into three bf16 parts, x = h + m + l exactly, each the
// nearest to what is left, one plane each.  With 2^e <= |x| < 2^(e+1), |m| <=
// 2^(e-8) and |l| <= 2^(e-17), so the six products hh, hm, mh, hl, mm, lh keep all
// but 2^-24 of |a b|, one rounding of an f32 product (cutting bits off instead
// would leave out up to 2^-21, always towards zero).  After Henry, Tang and
// Heinecke, 2019: the bf16 unit is 16 times the f32 unit's rate, so six products
// are 2.7 times faster than one.

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

template <int D> __device__ inline f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (D == FEDTRAIN_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool KS_, int W_, int BK_> struct Tile {
  static constexpr bool KS = KS_;
  static constexpr int W = W_, BK = BK_;
  static constexpr int per_line = (KS ? W : BK) / 8;
  static constexpr int chunks = W * BK / 8;
  static constexpr int bytes = chunks * 16;  // of one plane

  static __device__ int swizzle(int line) {
    if constexpr (KS) return (((line & 3) | ((line >> 3) & 3) << 2) & (W / 16 - 1)) << 1;
    return BK == 64 ? line & 7 : (line >> 1) & 3;
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
      return *reinterpret_cast<const s16x8*>(base + at(row0 + t * 16 + r, kk * 4 + q));
    }
  }
};

// The parts of two neighbouring values, packed as they lie in LDS.  True for an
// infinity or NaN, or a number that rounds to an infinity, whose parts are wrong.
// (Parts below 2^-126 may be lost.)
__device__ inline bool split3(f32x2 x, unsigned* to) {
  auto up = [](unsigned two) {
    return f32x2{__builtin_bit_cast(float, two << 16),
                 __builtin_bit_cast(float, two & 0xFFFF0000u)};
  };
  f32x2 r = x;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    to[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(r, bf16x2));
    if (i < 2) {
      const f32x2 part = up(to[i]);
      r[0] -= part[0];
      r[1] -= part[1];
    }
  }
  return r[0] != r[0] || r[1] != r[1];
}

// The same for any value, by cutting off bits: an infinity or NaN is its first
// part alone.
__device__ inline void split3_any(float x, unsigned& h, unsigned& m, unsigned& l) {
  h = __builtin_bit_cast(unsigned, x);
  const float r = x - __builtin_bit_cast(float, h & 0xFFFF0000u);
  m = __builtin_bit_cast(unsigned, r);
  l = __builtin_bit_cast(unsigned, r - __builtin_bit_cast(float, m & 0xFFFF0000u));
  if (r == r) return;
  m = l = 0;
  if (x != x) h |= 0x10000u;  // a NaN stays one
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
  const T* from[DIRECT ? 1 : N];  // the chunk's place in the tile under way
  int some[DIRECT ? 1 : N];       // its values that exist (KS), or whether its row does (KC)
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
  //
  // The loads are written out because the compiler, which cannot tell the stages
  // apart, would wait for all of them before the next LDS read: arrive() and
  // wait_loads() are what orders them.  They have no result in a register.  A
  // descriptor's registers may come from the vector unit, 5 cycles before a load
  // may read them.  m0 cannot be named as changed, it is the compiler's own: a test
  // reads the listing for any other use of it.
  __device__ u32x4 descriptor(int64_t k) const {
    const uint64_t p = reinterpret_cast<uint64_t>(base + (L::KS ? k * ld : k));
    u32x4 d;
    d[0] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(p));
    d[1] = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(p >> 32) & 0xFFFFu);
    d[2] = 0x7FFFFFFFu;
    d[3] = 0x00027000u;
    asm volatile("s_nop 4" : "+s"(d));
    return d;
  }
  // load i of a stage, of which `left` k exist (FULL: all)
  template <bool FULL>
  __device__ void issue(int i, u32x4 d, int left, const char* to, int tid) const {
    unsigned o = offset[i];
    if (!FULL) {
      const int q = tid + i * THREADS, line = q / L::per_line;
      const int c = (q % L::per_line) ^ L::swizzle(line);
      if (L::KS ? line >= left : c * 8 >= left) o = ~0u;
    }
    const unsigned at = __builtin_amdgcn_readfirstlane(
        static_cast<unsigned>(reinterpret_cast<uintptr_t>(
            (const __attribute__((address_space(3))) char*)to)) +
        ((tid & ~63) + i * THREADS) * 16);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(at), "v"(o), "s"(d)
                 : "memory");
  }
  // the stage at k, of which some, all or no k exist
  __device__ void issue_all(int64_t k, int64_t k1, char* to, int tid) const {
    if (k > k1) k = k1;
    const u32x4 d = descriptor(k);
    const int left = k1 - k < L::BK ? static_cast<int>(k1 - k) : L::BK;
#pragma unroll
    for (int i = 0; i < N; ++i) issue<false>(i, d, left, to, tid);
  }

  // through registers: any alignment, any length.  For steps of BK from k on.
  __device__ void begin(int64_t k, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int q = tid + i * THREADS, line = q / L::per_line;
      const int c = (q % L::per_line) ^ L::swizzle(line);
      from[i] = base + (L::KS ? (k + line) * ld + c * 8 : line * ld + k + c * 8);
      some[i] = L::KS ? rows - c * 8 : line < rows ? 8 : 0;
    }
  }

  // the next tile, of which `left` k exist
  __device__ void load(int64_t left, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int n = some[i];
      if (left < L::BK) {
        const int q = tid + i * THREADS, line = q / L::per_line;
        const int c = (q % L::per_line) ^ L::swizzle(line);
        const int more = static_cast<int>(left) - (L::KS ? line : c * 8);
        n = L::KS ? (more > 0 ? n : 0) : (more < n ? more : n);
      }
      if (n >= 8) {
        __builtin_memcpy(&held[i][0], from[i], 16 * R);
      } else {
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? from[i][e] : Elem<D>::down(0);
        __builtin_memcpy(&held[i][0], v, 16 * R);
      }
      from[i] += L::KS ? L::BK * ld : L::BK;
    }
  }

  // chunk i to its place; f32: true where a value was met whose parts are right with
  // ANY alone
  template <bool ANY> __device__ bool put(int i, char* to, int tid) const {
    char* p = to + (tid + i * THREADS) * 16;
    bool met = false;
    if constexpr (D != FEDTRAIN_F32) {
      *reinterpret_cast<u32x4*>(p) = held[i][0];
    } else {
      u32x4 out[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 four = __builtin_bit_cast(f32x4, held[i][e / 2]);
        const f32x2 x = {four[e % 2 * 2], four[e % 2 * 2 + 1]};
        unsigned part[3];
        if constexpr (ANY) {
          unsigned b[2][3];
#pragma unroll
          for (int s = 0; s < 2; ++s) split3_any(x[s], b[s][0], b[s][1], b[s][2]);
#pragma unroll
          for (int j = 0; j < 3; ++j) part[j] = __builtin_amdgcn_perm(b[1][j], b[0][j], 0x07060302);
        } else {
          met |= split3(x, part);
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) out[j][e] = part[j];
      }
#pragma unroll
      for (int e = 0; e < 3; ++e) *reinterpret_cast<u32x4*>(p + e * L::bytes) = out[e];
    }
    return met;
  }
  template <bool ANY> __device__ bool put_all(char* to, int tid) const {
    bool met = false;
#pragma unroll
    for (int i = 0; i < N; ++i) met |= put<ANY>(i, to, tid);
    return met;
  }
};

// The shape of a workgroup: MW x NW waves, each with MI x NI tiles of 16 x 16.
// PASS of the MI at a time are written to C.  STAGES of tiles in LDS: 1 where they
// come through registers, more where they come without.
template <int MW_, int NW_, int MI_, int NI_, int BK_, int PASS_, int STAGES_ = 1> struct Shape {
  static constexpr int WAVES = MI_ * NI_ > 32 ? 1 : 2;  // of a SIMD: what registers allow
  static constexpr bool DIRECT = STAGES_ > 1;
  static constexpr int STAGES = STAGES_;
  static constexpr int MW = MW_, NW = NW_, MI = MI_, NI = NI_, BK = BK_, PASS = PASS_;
  static constexpr int BM = MW * MI * 16, BN = NW * NI * 16, THREADS = MW * NW * 64;
};

// Workgroups go to the 8 dies in turn.  Each die gets a contiguous part of the
// tiles, in bands of `high` rows of tiles, so that what its workgroups read at a
// time is shared in its own L2.
__device__ inline void place(int64_t tiles_m, int64_t tiles_n, int high, int64_t& tm,
                             int64_t& tn) {
  const int64_t total = tiles_m * tiles_n, id = blockIdx.x;
  const int64_t share = total / 8, more = total % 8, die = id % 8;
  const int64_t t = die * share + (die < more ? die : more) + id / 8;
  const int64_t band = t / (high * tiles_n), in = t - band * high * tiles_n;
  const int64_t height = tiles_m - band * high < high ? tiles_m - band * high : high;
  tn = in / height;
  tm = band * high + in % height;
}

__device__ inline void arrive() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
template <int N> __device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

struct Plan {
  int64_t tiles_m, tiles_n;  // tiles_m: of one group (grad weight), or slots
  int high;                  // rows of tiles in a band, see place()
  bool counted;              // see counted()
  bool once;                 // C is larger than what the caches could keep for a reader
  int splits;                // parts of k; over 1, C is f32 partial sums in the workspace
};

__device__ inline int tiles_of(const Args& a, int i, int BM) {
  const int64_t n = bound(a, a.m, i + 1) - bound(a, a.m, i);
  return n > 0 ? static_cast<int>((n + BM - 1) / BM) : 0;
}

// The rows and the column of tiles of a workgroup when every wave counts the
// ranges' tiles, 64 ranges at a time, so that the dies share the tiles that exist
// instead of the slots, of which ragged groups leave some empty.
__device__ inline Rows counted(const Args& a, const Plan& plan, int BM, int64_t& tn) {
  const int n = a.groups + 2, lane = threadIdx.x & 63;
  const Rows none = {0, 0, -1};
  int all = 0;
  for (int i = lane; i < n; i += 64) all += tiles_of(a, i, BM);
#pragma unroll
  for (int s = 32; s; s >>= 1) all += __shfl_xor(all, s);
  const int total = __builtin_amdgcn_readfirstlane(all);
  if (static_cast<int64_t>(blockIdx.x) >= total * plan.tiles_n) return none;
  int64_t slot;
  place(total, plan.tiles_n, plan.high, slot, tn);
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int mine = i0 + lane < n ? tiles_of(a, i0 + lane, BM) : 0;
    int upto = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const int x = __shfl_up(upto, s);
      if (lane >= s) upto += x;
    }
    const uint64_t over = __builtin_amdgcn_ballot_w64(before + upto > slot);
    if (over) {
      const int l = __builtin_ctzll(over), at = i0 + l;
      const int64_t skipped = before + __builtin_amdgcn_readlane(upto - mine, l);
      const int64_t first = bound(a, a.m, at), end = bound(a, a.m, at + 1);
      const int64_t lo = first + (slot - skipped) * BM;
      if (lo < first || lo >= end) return none;  // offsets that do not ascend
      return {lo, lo + BM < end ? lo + BM : end, at - 1 < a.groups ? at - 1 : -1};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return none;
}

// ---------------------------------------------------------------------------
// what becomes of the sums
// ---------------------------------------------------------------------------
// n <= 8 neighbouring values in memory; all eight are one or two accesses of 16
// bytes, which need no alignment beyond the values' own.
template <int D> __device__ inline void read8(const void* p, int64_t at, int n, float* to) {
  using T = typename Elem<D>::type;
  const T* x = static_cast<const T*>(p) + at;
  if (n >= 8) {
    T f[8];
    __builtin_memcpy(f, x, sizeof(f));
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = Elem<D>::up(f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = e < n ? Elem<D>::up(x[e]) : 0.0f;
  }
}

// ONCE: past the caches
template <int D, bool ONCE> __device__ inline void write8(void* p, int n, const float* v) {
  using T = typename Elem<D>::type;
  typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned any4;
  T* x = static_cast<T*>(p);
  if (n >= 8) {
    T f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = Elem<D>::down(v[e]);
    u32x4 t[sizeof(f) / 16];
    __builtin_memcpy(t, f, sizeof(f));
#pragma unroll
    for (unsigned i = 0; i < sizeof(f) / 16; ++i) {
      if constexpr (ONCE) __builtin_nontemporal_store(t[i], reinterpret_cast<any4*>(x) + i);
      else reinterpret_cast<any4*>(x)[i] = t[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) x[e] = Elem<D>::down(v[e]);
  }
}

struct __attribute__((aligned(16))) Eight {
  float v[8];
};

// Where eight neighbouring columns of C are written, row by row.
template <int D, int FORM> struct Out {
  using T = typename Elem<D>::type;
  T *c, *z;
  const T* res;
  float bias[8];
  int n;
  bool held;  // by a group; other rows get their residual

  __device__ Out(const Args& a, int group, int64_t row, int64_t col, int64_t n_)
      : n(static_cast<int>(n_ < 8 ? n_ : 8)), held(group >= 0) {
    const int64_t first = FORM == FEDTRAIN_GRAD_WEIGHT ? group * a.c_group : 0;
    c = static_cast<T*>(a.c) + first + row * a.ldc + col;
    if constexpr (FORM == FEDTRAIN_FORWARD) {
      z = a.z ? static_cast<T*>(a.z) + row * a.ldz + col : nullptr;
      res = a.res ? static_cast<const T*>(a.res) + row * a.ldr + col : nullptr;
      if (a.bias && held && n > 0) {
        read8<D>(a.bias, group * a.bias_group + col, n, bias);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = 0;
      }
    }
  }
  // to the row `rows` further down
  __device__ void advance(const Args& a, int rows) {
    c += rows * a.ldc;
    if constexpr (FORM == FEDTRAIN_FORWARD) {
      if (z) z += rows * a.ldz;
      if (res) res += rows * a.ldr;
    }
  }
  // a row's sums, to their end
  template <int ACT, bool ONCE = false> __device__ void put(float* v) const {
    if constexpr (FORM == FEDTRAIN_FORWARD) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += bias[e];
      if (z) write8<D, ONCE>(z, n, v);
      if (held) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = act_value<D, ACT>(v[e]);
      }
      if (res) {
        float r[8];
        read8<D>(res, 0, n, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
      }
    }
    write8<D, ONCE>(c, n, v);
  }
};

// A workgroup's tile of C.  16-bit operands whose chunks are whole and aligned go to
// LDS directly (DIRECT): no registers and no instructions of the waves, which leaves
// room for 256 sums a lane of the largest tile; the matrix unit is busy for 54 to 62 %
// of its products' cycles, counted one at a time on a rested card.  A tile of 256 x
// 256 by four waves reads 64 bytes of LDS for each product, half of what eight waves
// would (30 % slower) and a quarter of what 128 x 128 by four does.  Operands at
// any other alignment, and f32 on its way into three parts, come through
// registers: 1003 x 517 f16 at odd strides 33 to 41 us a product where memory
// needs about 9.
template <int D, int FORM, class S> __global__ __launch_bounds__(S::THREADS, S::WAVES)
void k_product(Args a, Plan plan) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass needs the name alone
  using T = typename Elem<D>::type;
  constexpr bool WEIGHT = FORM == FEDTRAIN_GRAD_WEIGHT;
  constexpr int PLANES = D == FEDTRAIN_F32 ? 3 : 1;
  using LA = Tile<WEIGHT, S::BM, S::BK>;
  using LB = Tile<FORM != FEDTRAIN_FORWARD, S::BN, S::BK>;
  constexpr int STAGE = PLANES * (LA::bytes + LB::bytes);
  extern __shared__ __attribute__((aligned(1024))) char lds[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / S::NW * (S::MI * 16), wn = wave % S::NW * (S::NI * 16);
  int64_t slot = 0, tn = 0;
  Rows taken = {};
  if (!WEIGHT && plan.counted) {
    taken = counted(a, plan, S::BM, tn);
  } else {
    place(plan.tiles_m * (WEIGHT && a.groups ? a.groups : 1), plan.tiles_n, plan.high, slot, tn);
    if (!WEIGHT) taken = rows_of(a, slot, S::BM);
  }
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
    if (taken.lo >= taken.hi) return;
    row0 = taken.lo;
    rows = taken.hi - taken.lo;
    group = taken.group;
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

  Loader<D, LA, S::THREADS, S::DIRECT> la;
  Loader<D, LB, S::THREADS, S::DIRECT> lb;
  la.init(a.a, a.lda, row0, rows, tid);
  lb.init(B, a.ldb, col0, cols, tid);

  f32x4 acc[S::MI][S::NI] = {};
  // sums of A's columns: the waves of C's first columns multiply by ones
  f32x4 sum[WEIGHT ? S::MI : 1] = {};
  const bool want_sum = WEIGHT && a.colsum && col0 == 0 && wn == 0;
  s16x8 one;
#pragma unroll
  for (int e = 0; e < 8; ++e) one[e] = D == FEDTRAIN_F16 ? 0x3C00 : 0x3F80;
  // what of the wave's rows exists; a wave without any has nothing to multiply
  const int mine_rows = static_cast<int>(rows) - wm;
  const bool live = mine_rows > 0 && (wn < cols || want_sum);

  // the columns of C go to the rows of the unit's result: a lane gets 4
  // neighbouring columns of a row of C
  if constexpr (S::DIRECT) {
    // Two stages in LDS, and a k step's fragments in registers ahead of their
    // use: a stage is read while the one before is multiplied, so there is one
    // barrier for each stage, and it is met with products still to do.
    static_assert(S::BK == 64 && S::STAGES == 2, "two k steps, two stages");
    struct Fragments {
      s16x8 a[S::MI], b[S::NI];
    };
    auto read = [&](Fragments& f, const char* at, int kk) {
#pragma unroll
      for (int j = 0; j < S::NI; ++j) f.b[j] = LB::fragment(at + LA::bytes, wn, j, kk, lane);
#pragma unroll
      for (int i = 0; i < S::MI; ++i) f.a[i] = LA::fragment(at, wm, i, kk, lane);
    };
    constexpr int LOADS = LA::chunks / S::THREADS + LB::chunks / S::THREADS;
    auto issue = [&](int64_t k, char* to) {
      la.issue_all(k, k1, to, tid);
      lb.issue_all(k, k1, to + LA::bytes, tid);
    };
    // A step's products; between them the next step's reads, and the loads of the
    // stage at k where `loads`, in the order written (the unit takes a product
    // every 16 cycles; a read or a load in between costs it nothing, a row of them
    // does).
    auto multiply = [&](const Fragments& f, Fragments& other, const char* at, int kk,
                        auto with_sum, auto loads, int64_t k, char* to) {
      constexpr bool LOAD = decltype(loads)::value;
      constexpr int NA = decltype(la)::N, NB = decltype(lb)::N;
      u32x4 da, db;
      if (!live) {
        if (LOAD) issue(k, to);
        return;
      }
      if constexpr (LOAD) {
        da = la.descriptor(k);
        db = lb.descriptor(k);
      }
      constexpr int READS = S::NI + S::MI;
      constexpr int ALL = S::MI * S::NI, EACH = (ALL + READS - 1) / READS;
      constexpr int LOADS_EACH = (NA + NB + READS - 1) / READS;
#pragma unroll
      for (int r = 0; r < READS; ++r) {
        if (r < S::NI) other.b[r < S::NI ? r : 0] = LB::fragment(at + LA::bytes, wn, r, kk, lane);
        else other.a[r < S::NI ? 0 : r - S::NI] = LA::fragment(at, wm, r - S::NI, kk, lane);
        if (LOAD) {
#pragma unroll
          for (int l = r * LOADS_EACH; l < (r + 1) * LOADS_EACH && l < NA + NB; ++l) {
            if (l < NA) la.template issue<true>(l < NA ? l : 0, da, 0, to, tid);
            else lb.template issue<true>(l < NA ? 0 : l - NA, db, 0, to + LA::bytes, tid);
          }
        }
#pragma unroll
        for (int t = r * EACH; t < (r + 1) * EACH && t < ALL; ++t) {
          const int i = t / S::NI, j = t % S::NI;
          acc[i][j] = mfma<D>(f.b[j], f.a[i], acc[i][j]);
          if constexpr (decltype(with_sum)::value)
            if (j == 0) sum[i] = mfma<D>(one, f.a[i], sum[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto loop = [&](auto with_sum) {
      Fragments f[2];
      issue(k0, lds);
      issue(k0 + S::BK, lds + STAGE);
      wait_loads<LOADS>();
      arrive();
      if (live) read(f[0], lds, 0);
      int turn = 0;
      auto stage = [&](int64_t k, auto loads) {
        char* now = lds + turn * STAGE;
        turn ^= 1;
        multiply(f[0], f[1], now, 1, with_sum, std::false_type(), 0, nullptr);
        wait_loads<0>();
        arrive();
        if (!decltype(loads)::value && k + 2 * S::BK < k1) issue(k + 2 * S::BK, now);
        multiply(f[1], f[0], lds + turn * STAGE, 0, with_sum, loads, k + 2 * S::BK, now);
      };
      int64_t k = k0;
      for (; k + 3 * S::BK <= k1; k += S::BK) stage(k, std::true_type());
      for (; k < k1; k += S::BK) stage(k, std::false_type());
    };
    if (k0 < k1) {
      if constexpr (WEIGHT) {
        // one of the two for the whole workgroup: both have its barriers
        if (a.colsum && col0 == 0) loop(std::true_type());
        else loop(std::false_type());
      } else {
        loop(std::false_type());
      }
    }
  } else {
    int* odd = reinterpret_cast<int*>(lds + STAGE);
    if (D == FEDTRAIN_F32) {
      if (tid == 0) *odd = 0;
      __syncthreads();
    }
    // the loaded tile to LDS; a value that ANY is for leaves its mark
    auto fill = [&](char* to) {
      bool met = la.template put_all<false>(to, tid);
      met |= lb.template put_all<false>(to + PLANES * LA::bytes, tid);
      return met;
    };
    auto fill_any = [&](char* to) {
      la.template put_all<true>(to, tid);
      lb.template put_all<true>(to + PLANES * LA::bytes, tid);
      *odd = 1;
    };
    auto multiply = [&](const char* pa, auto with_sum) {
      const char* pb = pa + PLANES * LA::bytes;
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
          if (S::MW == 1 && i * 16 >= mine_rows) continue;
          s16x8 fa[PLANES];
#pragma unroll
          for (int p = 0; p < PLANES; ++p)
            fa[p] = LA::fragment(pa + p * LA::bytes, wm, i, kk, lane);
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
#pragma unroll
            for (int s = 0; s <= p; ++s)
#pragma unroll
              for (int j = 0; j < S::NI; ++j)
                acc[i][j] = mfma<D>(fb[j][s], fa[p - s], acc[i][j]);
            if constexpr (decltype(with_sum)::value) sum[i] = mfma<D>(one, fa[p], sum[i]);
          }
        }
      }
    };
    // an infinity times a part that is 0 would be NaN: with one about, the f32
    // unit takes the values as they were
    auto multiply_any = [&](const char* pa, auto with_sum) {
      const char* pb = pa + PLANES * LA::bytes;
      if constexpr (D == FEDTRAIN_F32) {
#pragma unroll
        for (int i = 0; i < S::MI; ++i) {
          s16x8 x[3];
          for (int p = 0; p < 3; ++p) x[p] = LA::fragment(pa + p * LA::bytes, wm, i, 0, lane);
#pragma unroll
          for (int j = 0; j < S::NI; ++j) {
            s16x8 w[3];
            for (int p = 0; p < 3; ++p) w[p] = LB::fragment(pb + p * LB::bytes, wn, j, 0, lane);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  joined(w[0][e], w[1][e], w[2][e]), joined(x[0][e], x[1][e], x[2][e]),
                  acc[i][j], 0, 0, 0);
          }
          if constexpr (decltype(with_sum)::value) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sum[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  1.0f, joined(x[0][e], x[1][e], x[2][e]), sum[i], 0, 0, 0);
          }
        }
      }
    };
    auto load = [&](int64_t left) {
      la.load(left, tid);
      lb.load(left, tid);
    };
    auto loop = [&](auto with_sum) {
      la.begin(k0, tid);
      lb.begin(k0, tid);
      load(k1 - k0);
      for (int64_t k = k0; k < k1; k += S::BK) {
        if (fill(lds)) fill_any(lds);
        __syncthreads();
        if (k + S::BK < k1) load(k1 - k - S::BK);
        const bool plain = D != FEDTRAIN_F32 || !__builtin_amdgcn_readfirstlane(*odd);
        if (live && plain) multiply(lds, with_sum);
        if (live && !plain) multiply_any(lds, with_sum);
        __syncthreads();
      }
    };
    if (k0 < k1) {
      if constexpr (WEIGHT) {
        if (a.colsum && col0 == 0) loop(std::true_type());
        else loop(std::false_type());
      } else {
        loop(std::false_type());
      }
    }
  }

  const int64_t width = (a.n + 7) / 8 * 8 + (a.colsum ? 8 : 0);  // of a row of partial sums
  float* partial = static_cast<float*>(a.workspace) +
                   (static_cast<int64_t>(blockIdx.y) * a.m + row0) * width;
  arrive();  // LDS is free
  if constexpr (WEIGHT) {
    if (want_sum && lane < 16) {
#pragma unroll
      for (int i = 0; i < S::MI; ++i) {
        const int r = wm + i * 16 + lane;
        if (r >= rows) continue;
        if (plan.splits > 1) partial[r * width + width - 8] = sum[i][0];
        else
          static_cast<T*>(a.colsum)[group * a.colsum_group + row0 + r] =
              Elem<D>::down(sum[i][0]);
      }
    }
    if (!a.c) return;
  }

  // The sums go through the wave's own part of LDS, some rows at a time, and come
  // back as eight neighbours of a row, rows one after another: whole lines of
  // memory, and one copy of the code that follows.
  constexpr int LINE = S::NI * 16, EIGHTS = S::NI * 2, FIT = S::PASS, DOWN = 64 / EIGHTS;
  f32x4* mine = reinterpret_cast<f32x4*>(lds) + wave * (FIT * 16 * LINE / 4);
  auto spot = [](int row, int four) { return row * (LINE / 4) + (four ^ (row & (LINE / 4 - 1))); };
  const int c8 = lane % EIGHTS, c = wn + c8 * 8, n = static_cast<int>(cols) - c;
  int r = wm + lane / EIGHTS;
  Out<D, FORM> out(a, group, row0 + r, col0 + c, n);
#pragma unroll
  for (int i0 = 0; i0 < S::MI; i0 += FIT) {
#pragma unroll
    for (int i = 0; i < FIT; ++i)
#pragma unroll
      for (int j = 0; j < S::NI; ++j)
        mine[spot(i * 16 + (lane & 15), j * 4 + (lane >> 4))] = acc[i0 + i][j];
    auto leave = [&](auto act, auto once) {
#pragma unroll 4
      for (int row = lane / EIGHTS; row < FIT * 16; row += DOWN, r += DOWN) {
        const f32x4 lo = mine[spot(row, c8 * 2)], hi = mine[spot(row, c8 * 2 + 1)];
        float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (r < rows && n > 0) {
          if (plan.splits > 1) {
            Eight f;
#pragma unroll
            for (int e = 0; e < 8; ++e) f.v[e] = v[e];
            *reinterpret_cast<Eight*>(partial + r * width + col0 + c) = f;
          } else {
            out.template put<decltype(act)::value, decltype(once)::value>(v);
          }
        }
        out.advance(a, DOWN);
      }
    };
    by_act(FORM == FEDTRAIN_FORWARD ? a.act : 0, [&](auto act) {
      if (plan.once) leave(act, std::true_type());
      else leave(act, std::false_type());
    });
  }
#endif
}

// The parts of k added up in their order, for eight columns a thread: 3 us for a
// client's layer, 7 to 8 for 2048 x 512.  The order is the same in every run.
template <int D, int FORM> __global__ __launch_bounds__(256) void k_join(Args a, Plan plan) {
  using T = typename Elem<D>::type;
  const int64_t width = (a.n + 7) / 8 * 8 + (a.colsum ? 8 : 0), per = width / 8;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= a.m * per) return;
  const int64_t row = id / per, col = id % per * 8;
  const float* P = static_cast<const float*>(a.workspace) + row * width + col;
  float v[8] = {};
#pragma unroll 4
  for (int s = 0; s < plan.splits; ++s) {
    const Eight f = *reinterpret_cast<const Eight*>(P + s * a.m * width);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += f.v[e];
  }
  if (col >= a.n) {
    if (a.colsum) static_cast<T*>(a.colsum)[row] = Elem<D>::down(v[0]);
    return;
  }
  if (FORM == FEDTRAIN_GRAD_WEIGHT && !a.c) return;
  int group = 0;
  if (FORM != FEDTRAIN_GRAD_WEIGHT && a.groups) {
    group = group_of(a, row);
    if (group < 0)
      for (int e = 0; e < 8; ++e) v[e] = 0;
  }
  const Out<D, FORM> out(a, group, row, col, a.n - col);
  by_act(FORM == FEDTRAIN_FORWARD ? a.act : 0,
         [&](auto act) { out.template put<decltype(act)::value>(v); });
}

// The forward product of a few rows: the weights are read once, at the rate of
// memory, and each lane adds up its part of k by itself.  A wave takes COLS columns
// and one of PARTS parts of k, which its workgroup's other waves complete.
template <int D, int ROWS, int COLS, int PARTS>
__global__ __launch_bounds__(256) void k_few_rows(Args a) {
  using T = typename Elem<D>::type;
  constexpr int TEAMS = 4 / PARTS;
  __shared__ float part[4][ROWS * COLS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int team = wave / PARTS, mine = wave % PARTS;
  const int64_t col0 = (static_cast<int64_t>(blockIdx.x) * TEAMS + team) * COLS;
  const T* X = static_cast<const T*>(a.a);
  const T* W[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c)  // columns past the last read the last
    W[c] = static_cast<const T*>(a.b) + (col0 + c < a.n ? col0 + c : a.n - 1) * a.ldb;
  float acc[ROWS][COLS] = {};
  auto step = [&](int64_t k, int n) {
    float w[COLS][8];
#pragma unroll
    for (int c = 0; c < COLS; ++c) read8<D>(W[c], k, n, w[c]);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float x[8];
      read8<D>(X, (r < a.m ? r : 0) * a.lda + k, n, x);
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r][c] = __builtin_fmaf(x[e], w[c][e], acc[r][c]);
    }
  };
  int64_t k = (mine * 64 + lane) * 8;
#pragma unroll 2
  for (; k + 8 <= a.k; k += PARTS * 64 * 8) step(k, 8);
  if (k < a.k) step(k, static_cast<int>(a.k - k));
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
#pragma unroll
      for (int s = 32; s; s >>= 1) acc[r][c] += __shfl_xor(acc[r][c], s);
      if (lane == 0) part[wave][r * COLS + c] = acc[r][c];
    }
  __syncthreads();
  if (threadIdx.x >= TEAMS * ROWS * COLS) return;
  const int t = threadIdx.x / (ROWS * COLS), i = threadIdx.x % (ROWS * COLS);
  const int r = i / COLS;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * TEAMS + t) * COLS + i % COLS;
  if (r >= a.m || col >= a.n) return;
  float v[8] = {};
  for (int s = 0; s < PARTS; ++s) v[0] += part[t * PARTS + s][i];
  const Out<D, FEDTRAIN_FORWARD> out(a, 0, r, col, 1);
  by_act(a.act, [&](auto act) { out.template put<decltype(act)::value>(v); });
}

// dz = dy act'(z): one pass, eight values of a row a thread, at any alignment.
// Memory bounds it: 16384 x 5632 bf16 in 90 us and 8192 x 16384 in 131 (6.1 TB/s).
template <int D, int ACT, bool ONCE>
__global__ __launch_bounds__(256) void k_act_backward(int64_t rows, int64_t cols, const void* dy,
                                                      int64_t lddy, const void* z, int64_t ldz,
                                                      void* dz, int64_t lddz) {
  using T = typename Elem<D>::type;
  const int64_t per = (cols + 7) / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t r = rows == 1 ? 0 : i / per, c = (i - r * per) * 8;
  const int n = static_cast<int>(cols - c < 8 ? cols - c : 8);
  float g[8], x[8];
  read8<D>(dy, r * lddy + c, n, g);
  read8<D>(z, r * ldz + c, n, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] *= act_slope<D, ACT>(x[e]);
  write8<D, ONCE>(static_cast<T*>(dz) + r * lddz + c, n, g);
}

// The same where a bias wants its gradient too, in 16-bit types: its terms are added
// up before they are rounded (rounded ones put db off 1.5 times as far as its own
// rounding does, by several of its units where the terms cancel).  A workgroup takes
// 64 columns of up to 2^log rows of a group, 8 values a thread and 32 rows at a
// time; sums go through the wave, LDS and, where there is more than one such part,
// the workspace, in the same order in every run.  Memory and the slope's instructions
// bound it: 8192 x 16384 bf16 gelu in 149 us and 10 to join, where k_act_backward takes
// 130; 777 x 333 f16 in 8.5 and 4.
constexpr int kSumCols = 64;

// rows_of() in parts of 2^log rows, the ranges looked at 64 at a time: the last one
// whose slots begin at or before this.
__device__ inline Rows part_of(const Args& a, int64_t slot, int log) {
  int64_t first = 0, end = a.m;
  int at = 0;
  if (a.groups) {
    const int n = a.groups + 2, lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const uint64_t m =
          __builtin_amdgcn_ballot_w64(i < n && (bound(a, a.m, i) >> log) + i <= slot);
      if (m) at = i0 + 63 - __builtin_clzll(m);
    }
    first = bound(a, a.m, at);
    end = bound(a, a.m, at + 1);
  }
  const int64_t lo = first + ((slot - (first >> log) - at) << log), hi = lo + (1ll << log);
  return {lo, hi < end ? hi : end, at};
}

template <int D, int ACT, bool ONCE>
__global__ __launch_bounds__(256) void k_act_backward_sums(Args a, unsigned strips, int log,
                                                           bool joined) {
  using T = typename Elem<D>::type;
  __shared__ float part[4][kSumCols];
  const int64_t slot = blockIdx.x / strips;
  const int64_t col0 = static_cast<int64_t>(blockIdx.x % strips) * kSumCols;
  const Rows taken = part_of(a, slot, log);
  if (joined && taken.lo >= taken.hi) return;
  const int lane = threadIdx.x & 63, c = (threadIdx.x & 7) * 8;
  const int64_t col = col0 + c;
  const int n = static_cast<int>(a.n - col < 8 ? a.n - col : 8);
  float sum[8] = {};
  // two rows' loads before their sums
  auto pass = [&](int n) {
    for (int64_t r = taken.lo + (threadIdx.x >> 3); r < taken.hi; r += 64) {
      const bool both = r + 32 < taken.hi;
      float g[2][8], x[2][8];
      read8<D>(a.a, r * a.lda + col, n, g[0]);
      read8<D>(a.b, r * a.ldb + col, n, x[0]);
      if (both) {
        read8<D>(a.a, (r + 32) * a.lda + col, n, g[1]);
        read8<D>(a.b, (r + 32) * a.ldb + col, n, x[1]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j && !both) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          g[j][e] *= act_slope<D, ACT>(x[j][e]);
          sum[e] += g[j][e];
        }
        write8<D, ONCE>(static_cast<T*>(a.c) + (r + j * 32) * a.ldc + col, n, g[j]);
      }
    }
  };
  if (n >= 8) pass(8);
  else if (n > 0) pass(n);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int s = 8; s < 64; s *= 2) sum[e] += __shfl_xor(sum[e], s);
    if (lane < 8) part[threadIdx.x >> 6][c + e] = sum[e];
  }
  __syncthreads();
  if (threadIdx.x >= kSumCols || col0 + threadIdx.x >= a.n) return;
  float all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) all += part[w][threadIdx.x];
  if (joined) static_cast<float*>(a.workspace)[slot * a.n + col0 + threadIdx.x] = all;
  else static_cast<T*>(a.colsum)[col0 + threadIdx.x] = Elem<D>::down(all);
}

// A group's parts, a thread for each of its columns.
template <int D> __global__ __launch_bounds__(256) void k_sums_join(Args a, int log) {
  using T = typename Elem<D>::type;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= (a.groups ? a.groups : 1) * a.n) return;
  const int64_t group = id / a.n, col = id % a.n;
  int64_t lo = 0, hi = a.m, slot = 0;
  if (a.groups) {  // as part_of() deals them out
    const int i = static_cast<int>(group) + 1;
    lo = bound(a, a.m, i);
    hi = bound(a, a.m, i + 1);
    slot = (lo >> log) + i;
  }
  float all = 0;
#pragma unroll 8
  for (; lo < hi; lo += 1ll << log, ++slot)
    all += static_cast<const float*>(a.workspace)[slot * a.n + col];
  static_cast<T*>(a.colsum)[group * a.colsum_group + col] = Elem<D>::down(all);
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

enum class Size { Large, Middle, Small };

struct Choice {
  Size size;
  int splits;
};

// What a workgroup of a kind costs, in microseconds as measured: `first` for its
// launch, first loads and stores; a step of 64 (16 bit) or 32 (f32) k alone on a
// compute unit and with the `fit` of them that one holds.
struct Kind {
  Size size;
  int bm, bn, fit;
  double first, alone, full;
};

const Kind kDirect[] = {{Size::Large, 256, 256, 1, 13.0, 1.7, 1.7},
                        {Size::Middle, 128, 128, 2, 4.0, 0.75, 1.2},
                        {Size::Small, 64, 64, 5, 4.0, 0.45, 1.1}};
const Kind kThrough[] = {{Size::Middle, 128, 128, 2, 6.0, 1.2, 1.6},
                         {Size::Small, 64, 64, 4, 4.0, 1.1, 1.4}};
const Kind kF32[] = {{Size::Middle, 128, 128, 2, 9.0, 1.95, 2.7},
                     {Size::Small, 64, 128, 3, 6.0, 1.45, 2.3}};

// The tile and the parts of k whose estimate is the least: large tiles read each
// operand less often, small ones and parts of k fill the 256 compute units.
Choice choose(const Args& a) {
  const bool weight = a.form == FEDTRAIN_GRAD_WEIGHT, f32 = a.dtype == FEDTRAIN_F32;
  const bool d = in_eights(a);
  const Kind* kinds = f32 ? kF32 : d ? kDirect : kThrough;
  const int count = !f32 && d ? 3 : 2;
  const double groups = a.groups ? a.groups : 1;
  const double k = weight ? a.k / groups : a.k, bk = f32 ? 32 : 64;
  const double steps = std::ceil(k / bk) + (weight && a.groups ? 0.5 : 0.0);
  Choice best = {Size::Small, 1};
  double least = 1e30;
  for (int i = 0; i < count; ++i) {
    const Kind& t = kinds[i];
    double tiles = std::ceil(a.n / static_cast<double>(t.bn));
    if (tiles < 1) tiles = 1;
    if (weight) tiles *= std::ceil(a.m / static_cast<double>(t.bm)) * groups;
    else if (!a.groups) tiles *= std::ceil(a.m / static_cast<double>(t.bm));
    else tiles *= groups * std::max(1.0, a.m / groups / t.bm + 0.5);  // ragged
    for (int s = 1; s <= 32; s += s < 4 ? 1 : s < 8 ? 2 : s / 2) {
      if (s > 1 && (steps < 2 * s || (weight && a.groups) || t.size == Size::Large)) break;
      const double each = tiles * s / 256;  // workgroups a compute unit
      const double held = each < t.fit ? std::max(1.0, std::ceil(each)) : t.fit;
      const double step =
          t.fit > 1 ? t.alone + (t.full - t.alone) * (held - 1) / (t.fit - 1) : t.full;
      const double rounds = each < t.fit ? 1.0 : each < 4 * t.fit ? std::ceil(each / t.fit)
                                                                  : each / t.fit + 0.5;
      double cost = rounds * (t.first + std::ceil(steps / s) * step);
      if (s > 1) cost += 4.0 + s * static_cast<double>(a.m) * a.n * 8 / 3e6;  // k_join
      if (cost < least) {
        least = cost;
        best = {t.size, s};
      }
    }
  }
  return best;
}

// Up to 4 rows of one weight matrix, while reading the weights costs more than the
// vector unit's products.  4096 x 4096, the weights in the caches: one bf16 row 5.1 us
// (9 from memory), on the matrix unit 11.5; two 12.1 and 11.9, four 15.4 and 11.9; one,
// two and four f32 rows 12.3, 13.3 and 16.3, on the matrix unit 21.  784 x 200: 4 to 5
// us, in place of 7 (bf16) and 10 (f32) by parts of k and their sum.
bool few_rows(const Args& a) {
  return a.form == FEDTRAIN_FORWARD && !a.groups && a.m <= 4 && a.n < 1 << 28 &&
         (a.dtype == FEDTRAIN_F32 || a.m == 1 ||
          static_cast<double>(a.m) * a.n * a.k <= 1 << 24);
}

int64_t workspace(const Args& a) {
  if (few_rows(a)) return 0;
  const int s = choose(a).splits;
  if (s < 2) return 0;
  return static_cast<int64_t>(s) * a.m * ((a.n + 7) / 8 * 8 + (a.colsum ? 8 : 0)) * 4;
}

// Results this large are not in the caches (256 MB) when they are read next, and
// push out what is: storing past them takes 64 experts' grad weight from 820 to 720
// us, dz of 8192 x 16384 and 16384 x 5632 from 133 to 131 and from 93 to 90.
template <int D> bool written_once(int64_t values) {
  return values * static_cast<int64_t>(sizeof(typename Elem<D>::type)) >= 128 << 20;
}

template <int D, int FORM, class S> int go(const Args& a, int splits, hipStream_t s) {
  Plan p;
  p.splits = splits;
  p.tiles_n = a.n ? (a.n + S::BN - 1) / S::BN : 1;
  int64_t all;
  if (FORM == FEDTRAIN_GRAD_WEIGHT) {
    p.tiles_m = (a.m + S::BM - 1) / S::BM;
    all = p.tiles_m * (a.groups ? a.groups : 1);
  } else {
    all = p.tiles_m = a.groups ? a.m / S::BM + a.groups + 2 : (a.m + S::BM - 1) / S::BM;
  }
  if (all > kMostGroups / p.tiles_n) return FEDTRAIN_EINVAL;
  p.once = written_once<D>(a.m * a.n * (FORM == FEDTRAIN_GRAD_WEIGHT && a.groups ? a.groups : 1));
  // Bands of 4 (forward), 2 (grad input) and 8 rows (grad weight) took 1026, 1060
  // and 1122 us where 8, 8 and 4 took 1035, 1159 and 1151 (8192 x 4096 x 16384
  // bf16).  Ragged groups have weights of their own: the columns of one row of
  // tiles at a time read them in whole rows (64 experts 600 and 714 us, against
  // 695 and 1013 in bands of 8).
  p.high = FORM == FEDTRAIN_FORWARD ? 4 : FORM == FEDTRAIN_GRAD_INPUT ? 2 : 8;
  if (a.groups) p.high = FORM == FEDTRAIN_GRAD_WEIGHT ? 16 : 1;
  // Counting pays up to two steps of 64 ranges and over four tiles a compute unit:
  // grad input of 64 experts (2048 x 5632) 587 -> 521 us, 120 of f32 1024 x 1024 332
  // -> 285, 126 of 1024 x 2048 159 -> 151; but 250 238 -> 247, 500 of 1024 x 1024 231
  // -> 287, and ten small clients 17.6 -> 17.9.
  p.counted = a.groups && a.groups <= 126 && all * p.tiles_n > 1024;
  constexpr int PLANES = D == FEDTRAIN_F32 ? 3 : 1;
  constexpr int STAGES = S::STAGES * PLANES * (S::BM + S::BN) * S::BK * 2 +
                         (D == FEDTRAIN_F32 ? 16 : 0);  // and the mark of an infinity
  constexpr int BYTES = std::max(STAGES, S::PASS * 16 * S::BN * S::MW * 4);  // C leaves through it
  auto* kernel = &k_product<D, FORM, S>;
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
    const int64_t eights = a.m * ((a.n + 7) / 8 + (a.colsum ? 1 : 0));
    if (eights > kMostGroups * 256) return FEDTRAIN_EINVAL;
    hipLaunchKernelGGL((k_join<D, FORM>), dim3(static_cast<unsigned>((eights + 255) / 256)),
                       dim3(256), 0, s, a, p);
  }
  return launched();
}

template <int D, int ROWS, int COLS, int PARTS> int go_few_rows(const Args& a, hipStream_t s) {
  constexpr int64_t each = 4 / PARTS * COLS;
  hipLaunchKernelGGL((k_few_rows<D, ROWS, COLS, PARTS>),
                     dim3(static_cast<unsigned>((a.n + each - 1) / each)), dim3(256), 0, s, a);
  return launched();
}

template <int D, int ROWS> int go_few_rows(const Args& a, hipStream_t s) {
  // 2048 waves or more, two to a SIMD
  if (a.n >= 8192) return go_few_rows<D, ROWS, 4, 1>(a, s);
  if (a.n >= 4096) return go_few_rows<D, ROWS, 4, 2>(a, s);
  return go_few_rows<D, ROWS, 2, 4>(a, s);
}

template <int D> int run_few_rows(const Args& a, hipStream_t s) {
  if (a.m <= 1) return go_few_rows<D, 1>(a, s);
  if (a.m <= 2) return go_few_rows<D, 2>(a, s);
  return go_few_rows<D, 4>(a, s);
}

template <int D, int FORM> int run(const Args& a, hipStream_t s) {
  const Choice c = choose(a);
  if (c.splits > 1 && (!a.workspace || !aligned(a.workspace, 16) ||
                       a.workspace_bytes < workspace(a)))
    return FEDTRAIN_EINVAL;
  if constexpr (D == FEDTRAIN_F32) {
    if (c.size == Size::Small) return go<D, FORM, Shape<1, 4, 4, 2, 32, 4>>(a, c.splits, s);
    return go<D, FORM, Shape<2, 2, 4, 4, 32, 4>>(a, c.splits, s);
  } else {
    if (c.size == Size::Large) return go<D, FORM, Shape<2, 2, 8, 8, 64, 4, 2>>(a, 1, s);
    const bool d = in_eights(a);
    if (c.size != Size::Small)
      return d ? go<D, FORM, Shape<2, 2, 4, 4, 64, 4, 2>>(a, c.splits, s)
               : go<D, FORM, Shape<2, 2, 4, 4, 64, 4>>(a, c.splits, s);
    return d ? go<D, FORM, Shape<2, 2, 2, 2, 64, 2, 2>>(a, c.splits, s)
             : go<D, FORM, Shape<2, 2, 2, 2, 64, 2>>(a, c.splits, s);
  }
}

template <int D> int run(const Args& a, hipStream_t s) {
  if (few_rows(a)) return run_few_rows<D>(a, s);
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

template <int D, int ACT> int slope(const Slope& given, hipStream_t s) {
  Slope x = given;
  if (x.lddy == x.cols && x.ldz == x.cols && x.lddz == x.cols) {  // one long row
    x.cols *= x.rows;
    x.rows = 1;
  }
  const int64_t n = x.rows * ((x.cols + 7) / 8);
  if (n > kMostGroups * 256) return FEDTRAIN_EINVAL;
  auto* kernel = written_once<D>(x.rows * x.cols) ? &k_act_backward<D, ACT, true>
                                                  : &k_act_backward<D, ACT, false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s,
                     x.rows, x.cols, x.dy, x.lddy, x.z, x.ldz, x.dz, x.lddz);
  return launched();
}

template <int D> int slope(int act, const Slope& x, hipStream_t s) {
  if (act == FEDTRAIN_ACT_RELU) return slope<D, FEDTRAIN_ACT_RELU>(x, s);
  if (act == FEDTRAIN_ACT_GELU) return slope<D, FEDTRAIN_ACT_GELU>(x, s);
  if (act == FEDTRAIN_ACT_SILU) return slope<D, FEDTRAIN_ACT_SILU>(x, s);
  return slope<D, FEDTRAIN_ACT_NONE>(x, s);
}

bool valid(const fedtrain_act_args* x) {
  if (!x || (x->dtype != FEDTRAIN_BF16 && x->dtype != FEDTRAIN_F16) || x->act < FEDTRAIN_ACT_NONE ||
      x->act > FEDTRAIN_ACT_SILU || x->groups < 0 || x->groups > INT32_MAX - 2 || x->rows < 0 ||
      x->cols < 0 || x->rows > kMaxSize || x->cols > kMaxSize)
    return false;
  if (x->groups && (!x->offsets || !aligned(x->offsets, x->offsets64 ? 8 : 4))) return false;
  const void* each[] = {x->dy, x->z, x->dz, x->colsum};
  for (const void* p : each)
    if (!aligned(p, 2)) return false;
  if (x->lddy < 0 || x->ldz < 0 || (x->rows > 1 && x->lddz < x->cols) ||
      (x->groups > 1 && x->colsum_group < x->cols))
    return false;
  return !x->cols || (x->colsum && (!x->rows || (x->dy && x->z && x->dz)));
}

// Rows of a part, as a power of two: 32, so that small cases fill the card; more where
// there would be over 256 parts, which k_sums_join adds up one by one, or over 128
// workgroups a compute unit (8192 x 16384 bf16 with 128, 64 and 32 rows: 166, 148 and
// 182 us, and 6, 10 and 17 to join).
int sum_log(const fedtrain_act_args& x) {
  const int64_t strips = (x.cols + kSumCols - 1) / kSumCols;
  int log = 5;
  while (x.rows >> log > 256 || (x.rows >> log) * strips > 128 * 256) ++log;
  return log;
}
// Parts of rows, and whether their sums have to be joined: not where one workgroup
// sees all rows of its columns.
int64_t sum_slots(const fedtrain_act_args& x) {
  const int log = sum_log(x);
  if (x.groups) return (x.rows >> log) + x.groups + 2;
  return std::max<int64_t>(1, (x.rows + (1ll << log) - 1) >> log);
}
bool sums_joined(const fedtrain_act_args& x) { return x.groups || sum_slots(x) > 1; }

int64_t workspace(const fedtrain_act_args& x) {
  return sums_joined(x) ? sum_slots(x) * x.cols * 4 : 0;
}

template <int D, int ACT> int slope_sums(const fedtrain_act_args& x, hipStream_t s) {
  const int64_t strips = (x.cols + kSumCols - 1) / kSumCols, slots = sum_slots(x);
  const int64_t sums = (x.groups ? x.groups : 1) * x.cols;
  const bool joined = sums_joined(x);
  const int log = sum_log(x);
  // a launch's threads are counted in 32 bits
  if (slots > kMostGroups / strips || sums > kMostGroups * 256) return FEDTRAIN_EINVAL;
  if (joined && (!x.workspace || !aligned(x.workspace, 16) || x.workspace_bytes < workspace(x)))
    return FEDTRAIN_EINVAL;
  Args a = {};
  a.groups = x.groups;
  a.offsets = x.offsets;
  a.offsets64 = x.offsets64;
  a.m = x.rows;
  a.n = x.cols;
  a.a = x.dy;
  a.lda = x.lddy;
  a.b = x.z;
  a.ldb = x.ldz;
  a.c = x.dz;
  a.ldc = x.lddz;
  a.colsum = x.colsum;
  a.colsum_group = x.colsum_group;
  a.workspace = x.workspace;
  auto* kernel = written_once<D>(x.rows * x.cols) ? &k_act_backward_sums<D, ACT, true>
                                                  : &k_act_backward_sums<D, ACT, false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(slots * strips)), dim3(256), 0, s, a,
                     static_cast<unsigned>(strips), log, joined);
  if (joined) {
    if (const int rc = launched()) return rc;
    hipLaunchKernelGGL((k_sums_join<D>), dim3(static_cast<unsigned>((sums + 255) / 256)),
                       dim3(256), 0, s, a, log);
  }
  return launched();
}

template <int D> int slope_sums(const fedtrain_act_args& x, hipStream_t s) {
  if (x.act == FEDTRAIN_ACT_RELU) return slope_sums<D, FEDTRAIN_ACT_RELU>(x, s);
  if (x.act == FEDTRAIN_ACT_GELU) return slope_sums<D, FEDTRAIN_ACT_GELU>(x, s);
  if (x.act == FEDTRAIN_ACT_SILU) return slope_sums<D, FEDTRAIN_ACT_SILU>(x, s);
  return slope_sums<D, FEDTRAIN_ACT_NONE>(x, s);
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

int fedtrain_product_plan(const Args* args, int* rows, int* cols, int* parts) {
  if (!valid(args) || !rows || !cols || !parts) return FEDTRAIN_EINVAL;
  if (few_rows(*args)) {
    *rows = static_cast<int>(args->m);
    *cols = *parts = 1;
    return 0;
  }
  const Choice c = choose(*args);
  *rows = c.size == Size::Large ? 256 : c.size == Size::Middle ? 128 : 64;
  *cols = c.size == Size::Small && args->dtype == FEDTRAIN_F32 ? 128 : *rows;
  *parts = c.splits;
  return 0;
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

int64_t fedtrain_act_backward_sums_workspace(const fedtrain_act_args* args) {
  return valid(args) ? workspace(*args) : FEDTRAIN_EINVAL;
}

int fedtrain_act_backward_sums(const fedtrain_act_args* args, void* stream) {
  if (!valid(args)) return FEDTRAIN_EINVAL;
  if (!args->cols) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (args->dtype == FEDTRAIN_BF16) return slope_sums<FEDTRAIN_BF16>(*args, s);
  return slope_sums<FEDTRAIN_F16>(*args, s);
}

}  // extern "C"

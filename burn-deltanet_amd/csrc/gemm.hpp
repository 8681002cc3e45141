// The tile kernel of the products around the mixer: C = A·B with an epilogue,
// for bf16, fp32 and 8-bit (e4m3) operands, fp32 sums.
//
// Layouts. Each operand is either "row" (the contraction index k is fastest:
// x of x·W, W of dz·Wᵀ, 8-bit weights) or "col" (k is the slow index: W of
// x·W, both operands of xᵀ·dz). A tile of an operand is BM (BN) rows of 128
// bytes along k, or the same bytes with k slow; it lies in LDS as it lies in
// memory, in 16-byte words that an XOR spreads over the banks, so an HBM → LDS
// copy needs no registers. "row" fragments are 16-byte LDS reads; "col"
// fragments are transposing reads (bf16) or four-byte reads (fp32).
//
// A wave owns (BM/WM) × (BN/WN) of the output in 16×16 accumulators. The
// product is formed transposed (the B fragment as the matrix unit's first
// operand), so a lane holds four adjacent columns of one row; the epilogue
// passes 32 rows at a time through LDS and works on 8 adjacent columns, which
// it stores as 16-byte words.
#pragma once

#include <type_traits>
#include <utility>

#include "activations.hpp"
#include "dn_common.hpp"
#include "mfma_util.hpp"

namespace dn {

struct f8 {
  uint8_t bits;
};

typedef short i16x4 __attribute__((ext_vector_type(4)));

// What a product does with its sums.
enum GemmEpi {
  kEpiLinear = 0,  // act(scale · sum + bias) + residual
  kEpiGated = 1,   // columns in pairs: act(gate) · up, both kept on request
  kEpiDGated = 2,  // the sum is d_h: d_gate, d_up and h from the kept gate and up
};

struct GemmArgs {
  const char* a[2];     // A, and the second contraction segment's A
  const char* b[2];     // B; second segment's, second product's, or W_up's
  int64_t lda, ldb;     // bytes between rows (row) or between k (col)
  int M, N, K;          // N: output columns (gated: of h); K: of one segment
  int nseg;             // contraction segments: 1 or 2
  int npair;            // products that share A: 1 or 2 (b[z] → out[z])
  int ktiles;           // k tiles of a segment
  int split;            // workgroups along the contraction (wide: workgroups)
  int per_split;        // k tiles of each (wide: of the rest's share)
  int rounds;           // wide: whole tiles of every workgroup
  int tiles_m, tiles_n;
  // epilogue
  int act;
  void* out[2];
  int64_t ldo;          // elements, as below
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* preact;         // linear: act's argument, kept; gated: the gate's
  void* up;             // gated: kept (written); d_gated: with preact, read
  int64_t ldp;          // preact and up
  void* h;              // d_gated: h; out[0], out[1]: d_gate, d_up
  const float* row_scale;  // 8-bit: of A's rows, of B's rows
  const float* col_scale;
  float* partial;       // [split][npair][M][ldpart] fp32, or null
  int64_t ldpart;       // gated: 2·hidden columns, gate then up
};

namespace gemm {

template <class T>
struct Elem;
template <>
struct Elem<bf16> {
  static constexpr int kCh = 8, kKT = 64, kSteps = 2;
};
template <>
struct Elem<float> {
  static constexpr int kCh = 4, kKT = 32, kSteps = 2;
};
template <>
struct Elem<f8> {
  static constexpr int kCh = 16, kKT = 128, kSteps = 2;
};

// Sixteen e4m3 codes as bf16, which holds every one of them exactly. The
// products then run on the bf16 matrix instructions, whose sums are fp32: those
// on 8-bit operands add their products in fewer bits (both the 32- and the
// 128-deep one were off by up to 2^-16 of the terms' magnitude at K = 64).
struct Codes16 {
  uint4 lo, hi;
};
__device__ inline Codes16 widen(const uint4& c) {
  auto two = [](uint32_t u, auto high) {
    return __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, decltype(high)::value));
  };
  using L = std::false_type;
  using H = std::true_type;
  return {make_uint4(two(c.x, L{}), two(c.x, H{}), two(c.y, L{}), two(c.y, H{})),
          make_uint4(two(c.z, L{}), two(c.z, H{}), two(c.w, L{}), two(c.w, H{}))};
}

// The first n of a word's sixteen codes, zeros behind them: a row's last word may
// hold another matrix's columns, or NaN.
__device__ inline uint4 first_codes(uint4 v, int n) {
  auto part = [&](uint32_t u, int from) {
    const int k = n - from;
    return k >= 4 ? u : k > 0 ? u & ((1u << (8 * k)) - 1u) : 0u;
  };
  return make_uint4(part(v.x, 0), part(v.y, 4), part(v.z, 8), part(v.w, 12));
}

// f(0), …, f(N − 1) with compile-time arguments.
template <int... I, class F>
__device__ inline void each_of(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ inline void each(F f) {
  each_of(std::make_integer_sequence<int, N>{}, f);
}

// act(z) and its derivative. GELU is the exact form, z·Φ(z), with Φ by erfc:
// 1 + erf(z/√2) loses its bits below zero (4 % at z = −5, all of them at −5.6).
__device__ inline float gelu_cdf(float z) { return 0.5f * erfcf(z * -0.70710678118654752f); }
// a[i] = act(z[i]), and with SLOPE d[i] = act'(z[i]): one branch for eight (a
// may be z).
template <bool SLOPE>
__device__ inline void act8(const float (&z)[8], int kind, float (&a)[8], float (&d)[8]) {
  if (kind == DN_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = z[i], s = sigmoidf_(x);
      a[i] = x * s;
      if constexpr (SLOPE) d[i] = s * (1.0f + x * (1.0f - s));
    }
  } else if (kind == DN_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = z[i], c = gelu_cdf(x);
      a[i] = x * c;
      if constexpr (SLOPE) d[i] = c + x * 0.39894228040143268f * __expf(-0.5f * x * x);
    }
  } else if (kind == DN_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = z[i];
      a[i] = x < 0.f ? 0.f : x;  // NaN stays
      if constexpr (SLOPE) d[i] = x <= 0.f ? 0.f : 1.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = z[i];
      if constexpr (SLOPE) d[i] = 1.0f;
    }
  }
}

// Eight adjacent values of a row, `valid` of them inside it. The 16-byte
// accesses need no alignment beyond the element's own.
template <class T>
__device__ inline void load8(const T* p, float (&v)[8], int valid) {
  if (valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      uint4 u;
      __builtin_memcpy(&u, p, 16);
      unpack8(u, v);
    } else {
      __builtin_memcpy(v, p, 32);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? ld(p, i) : 0.f;
  }
}
template <class T>
__device__ inline void store8(T* p, const float (&v)[8], int valid) {
  if (valid >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = make_uint4(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]),
                                 pk_bf16(v[6], v[7]));
      __builtin_memcpy(p, &u, 16);
    } else {
      __builtin_memcpy(p, v, 32);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) st(p, i, v[i]);
  }
}

// Eight adjacent values as they lie in memory, until they are used.
template <class T>
struct Raw8 {
  static constexpr int kWords = 2 * int(sizeof(T));
  uint32_t w[kWords];
  __device__ inline void load(const T* p, int valid) {
    if (valid >= 8) {
      __builtin_memcpy(w, p, sizeof(w));
    } else {
      float v[8];
      load8(p, v, valid);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pk_bf16(v[2 * i], v[2 * i + 1]);
      }
    }
  }
  __device__ inline void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else {
      unpack8(make_uint4(w[0], w[1], w[2], w[3]), v);
    }
  }
};

// The epilogues on eight columns of a row, each in two parts, so that a caller
// can have several rows' loads in flight: what it reads (Tail), then the rest.
// Shared by the tile kernels, the few-rows kernel and the join of split
// contractions.
template <class TO, int EPI>
struct Tail {
  Raw8<TO> x, y;  // linear: the residual; d_gated: the kept gate and up
};
template <class TO, int EPI>
__device__ inline void tail_load(const GemmArgs& p, int64_t row, int col, Tail<TO, EPI>& t) {
  const int valid = p.N - col;
  if constexpr (EPI == kEpiLinear) {
    if (p.residual) t.x.load(static_cast<const TO*>(p.residual) + row * p.ldr + col, valid);
  } else if constexpr (EPI == kEpiDGated) {
    t.x.load(static_cast<const TO*>(p.preact) + row * p.ldp + col, valid);
    t.y.load(static_cast<const TO*>(p.up) + row * p.ldp + col, valid);
  }
}
// v: the product (gated: gate's, and u up's). z: which of a pair of products.
template <class TO, int EPI>
__device__ inline void tail_store(const GemmArgs& p, int z, int64_t row, int col, float (&v)[8],
                                  const float (&u)[8], Tail<TO, EPI>& t) {
  const int valid = p.N - col;
  float none[8];
  if constexpr (EPI == kEpiLinear) {
    if (p.row_scale) {
      const float rs = p.row_scale[row];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < valid) v[i] *= rs * p.col_scale[col + i];
    }
    if (p.bias) {
      float b[8];
      load8(static_cast<const TO*>(p.bias) + col, b, valid);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    if (p.preact) store8(static_cast<TO*>(p.preact) + row * p.ldp + col, v, valid);
    if (p.act != DN_ACT_IDENTITY) act8<false>(v, p.act, v, none);
    if (p.residual) {
      float r[8];
      t.x.get(r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    store8(static_cast<TO*>(z ? p.out[1] : p.out[0]) + row * p.ldo + col, v, valid);
  } else if constexpr (EPI == kEpiGated) {
    // h = act(g)·u, and the kept g and u.
    if (p.preact) {
      store8(static_cast<TO*>(p.preact) + row * p.ldp + col, v, valid);
      store8(static_cast<TO*>(p.up) + row * p.ldp + col, u, valid);
    }
    act8<false>(v, p.act, v, none);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= u[i];
    store8(static_cast<TO*>(p.out[0]) + row * p.ldo + col, v, valid);
  } else {
    // From d_h (v) and the kept g and u: d_g = d_h·u·act'(g), d_u = d_h·act(g),
    // and h again for the down projection's weight gradient.
    float dg[8], h[8], kept[8];
    t.x.get(kept);
    act8<true>(kept, p.act, h, dg);
    t.y.get(kept);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dg[i] *= v[i] * kept[i];
      v[i] *= h[i];
      h[i] *= kept[i];
    }
    store8(static_cast<TO*>(p.out[0]) + row * p.ldo + col, dg, valid);
    store8(static_cast<TO*>(p.out[1]) + row * p.ldo + col, v, valid);
    store8(static_cast<TO*>(p.h) + row * p.ldo + col, h, valid);
  }
}
// Whether the sums are stored as they are, or with a residual. The whole epilogue
// is 5 KB of code for each of the rows that a kernel unrolls, more than the
// instruction cache holds: such products go by a path of their own that is short
// (bf16 8192 x 2048 x 12304 468 -> 408 us).
template <int EPI>
__device__ inline bool stored_as_they_are(const GemmArgs& p) {
  return EPI == kEpiLinear && p.act == DN_ACT_IDENTITY && !p.bias && !p.preact && !p.row_scale;
}
// Both parts, or the sums of a split product to the workspace.
template <class TO, int EPI>
__device__ inline void finish8(const GemmArgs& p, int z, int sp, int64_t row, int col,
                               float (&v)[8], const float (&u)[8], Tail<TO, EPI>& t) {
  if (p.partial) {
    float* to = p.partial + (int64_t(sp * p.npair + z) * p.M + row) * p.ldpart + col;
    store8(to, v, p.N - col);
    if constexpr (EPI == kEpiGated) store8(to + p.N, u, p.N - col);
  } else {
    tail_store<TO, EPI>(p, z, row, col, v, u, t);
  }
}

// One HBM → LDS copy of 16 bytes a lane: lane i's word goes to `lds` + 16·i.
// No register receives it; it is complete when vmcnt says so. The compiler does
// not look inside the text, so it holds the wait that the copy owes m0. Nothing
// else in these kernels uses m0 (LDS accesses do not need it on this architecture).
__device__ inline void copy_to_lds(const char* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(src)
               : "memory");
}
// The same from a scalar base. A vector instruction may have written it just
// before, which a copy may read five wait states later, the scalar unit at once:
// that unit's copy of it also is m0's wait (with five states in its place the
// wide kernel takes 2 to 4 % longer).
__device__ inline void copy_to_lds(const char* base, uint32_t offset, uint32_t lds) {
  const char* from;
  asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
               : "=&s"(from)
               : "s"(lds), "v"(offset), "s"(base)
               : "memory");
}
// c += b·a with c held in accumulation registers. The wide kernel's 256 sums
// fill that half of the register file; left to itself the compiler moves them
// between the halves at every branch (276 moves a k tile of 128 products, and
// spills among them). What scratch memory the kernel uses now lies outside the
// products. The compiler does not see a matrix instruction here: settle_acc() is
// owed before anything else reads the sums, and settle_words() before a product
// reads operands that a vector instruction wrote.
__device__ inline void mfma16_acc(const uint4& b, const uint4& a, f32x4& c) {
  asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0"
      : "+a"(c)
      : "v"(__builtin_bit_cast(bf16x8, b)), "v"(__builtin_bit_cast(bf16x8, a)));
}
// The wait that a matrix instruction's result needs before another kind of
// instruction reads it, by itself and tied to eight of the sums.
__device__ inline void settle_products() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
__device__ inline void settle_acc(f32x4 (&c)[8]) {
  asm volatile("s_nop 15\n\ts_nop 15"
               : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]),
                 "+a"(c[6]), "+a"(c[7]));
}

// The wait that a vector instruction's result needs before a matrix instruction
// reads it, tied to widened codes. (In the products' own text the two states
// would cost the wide kernel 6 %.)
__device__ inline void settle_words(Codes16& c) {
  bf16x8 lo = __builtin_bit_cast(bf16x8, c.lo), hi = __builtin_bit_cast(bf16x8, c.hi);
  asm("s_nop 1" : "+v"(lo), "+v"(hi));
  c = {__builtin_bit_cast(uint4, lo), __builtin_bit_cast(uint4, hi)};
}

template <int N>
__device__ inline void wait_copies() {  // at most N of this wave's copies outstanding
  static_assert(N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ inline uint32_t lds_address(const void* p) {
  return uint32_t(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) const void*)p));
}

// The XOR on a word's place. "row" tiles have rows of 8 words, two rows to
// the banks' 256 bytes: the 16 rows of a fragment read meet 16 places.
__device__ inline int swizzle_row(int row) { return (row >> 1) & 7; }
// "col" tiles of R columns. bf16: a transposing read takes 32 bytes of rows
// 8q + 4h + 0…3 for the lanes' four groups q, and the eight rows of a half wave
// get eight places; k's rows are whole multiples of 256 bytes, or (R = 64) two
// make one. fp32: rows 4q + i, 64 bytes each.
template <class T, int R>
__device__ inline int swizzle_col(int k) {
  if constexpr (sizeof(T) == 4) return 4 * ((k >> 2) & 3);
  else if constexpr (R == 64) return 2 * (((k >> 1) & 1) | ((k >> 2) & 2));
  else return 2 * ((k & 3) | ((k >> 1) & 4));
}

// Which 16-byte word of an operand goes to word `L` of its tile.
// "row": row r = L / 8 and word c of its 128 bytes; "col": k = L / (R/kCh),
// word c of its R columns.
template <class T, bool COL, int R>
__device__ inline void tile_word(int L, int& r, int& c) {
  if constexpr (COL) {
    constexpr int W = R / Elem<T>::kCh;
    r = L / W;
    c = (L % W) ^ swizzle_col<T, R>(r);
  } else {
    r = L >> 3;
    c = (L & 7) ^ swizzle_row(r);
  }
}

}  // namespace gemm

// BM × BN tiles, WM × WN parts of them, each of WK waves that share the k steps
// of a tile; a ring of RING k tiles in LDS, RING − 1 in flight while one is
// worked on. ACOL, BCOL: layouts. STAGED: operands whose rows do not lie at
// 16-byte steps go through registers, with masks.
//
// Bound by LDS and the copies, 50 to 60 GB/s a CU, at two workgroups a CU 0.58 us
// a k tile of 128 x 128. Measured, bf16 x·W: 4096 x 4096 x 2048 70 us (980
// TFLOP/s), 1500 x 2048 x 12304 95 (800), 1024 x 2048 x 5632 36 (650); 8-bit
// 4096 x 4096 x 2048 62 (1100). fp32 is bound by the matrix unit: 2048 x 2048 x
// 1024 77 us (111 TFLOP/s); 500 x 256 x 1039 with unaligned rows 16, all latency.
template <class T, class TO, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, int WK,
          int RING, int EPI, bool STAGED>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void gemm_kernel(GemmArgs p) {
  using namespace gemm;
  using E = Elem<T>;
  constexpr int kWaves = WM * WN * WK, kThreads = 64 * kWaves, CH = E::kCh, KT = E::kKT;
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;  // 16×16 blocks of a wave
  constexpr int kABytes = BM * 128, kBBytes = BN * 128, kStage = kABytes + kBBytes;
  constexpr int NA = kABytes / 16 / kThreads, NB = kBBytes / 16 / kThreads;
  static_assert(NA * kThreads * 16 == kABytes && NB * kThreads * 16 == kBBytes, "whole copies");
  static_assert(NJ == 4, "the epilogue's rows of 64 columns");
  static_assert(!STAGED || RING == 2, "one tile in the registers");
  __shared__ __attribute__((aligned(16))) char smem[RING * kStage];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
  const int s = lane & 15, q = lane >> 4;

  // Workgroups go round the eight XCDs: each XCD gets a contiguous range of
  // tiles, ordered in bands of 8 tile rows, so its 32 CUs share operand tiles
  // in its L2.
  const int total = p.tiles_m * p.tiles_n * p.npair * p.split;
  int id;
  {
    const int xcd = blockIdx.x & 7, n = blockIdx.x >> 3, per = total >> 3, rem = total & 7;
    id = xcd * per + min(xcd, rem) + n;
  }
  const int tiles = p.tiles_m * p.tiles_n;
  const int zs = id / tiles, z = zs % p.npair, sp = zs / p.npair;
  int tm, tn;
  {
    const int t = id % tiles, band = 8 * p.tiles_n, g = t / band, first = g * 8;
    const int rows = min(8, p.tiles_m - first), r = t - g * band;
    tm = first + r % rows;
    tn = r / rows;
  }
  const int m0 = tm * BM;
  constexpr int kOutCols = EPI == kEpiGated ? BN / 2 : BN;
  const int n0 = tn * kOutCols;

  const char* gb0 = p.npair == 2 && z ? p.b[1] : p.b[0];

  // The source column (in elements of b[which]) of word c of a "col" B tile.
  // Gated: a wave's 64 columns are 32 of W_gate and 32 of W_up.
  auto b_col = [&](int c, int& which) {
    const int j = c * CH;
    which = 0;
    if constexpr (EPI == kEpiGated) {
      which = (j >> 5) & 1;
      return n0 + (j >> 6) * 32 + (j & 31);
    }
    return n0 + j;
  };

  // k tiles of this workgroup, counted over the segments.
  const int t0 = sp * p.per_split, t1 = min(t0 + p.per_split, p.ktiles * p.nseg);
  const bool ragged = p.K % KT != 0;

  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Word w of thread's copies: its place in the tile and its source.
  const char *pa[NA], *pb[NB];
  auto sources = [&](int seg, int kt) {  // of a segment's k tile
    const char* ga = seg ? p.a[1] : p.a[0];
#pragma unroll
    for (int w = 0; w < NA; ++w) {
      int r, c;
      tile_word<T, ACOL, BM>((w * kWaves + wave) * 64 + lane, r, c);
      if constexpr (ACOL)
        pa[w] = ga + int64_t(kt * KT + r) * p.lda +
                int64_t(min(m0 + c * CH, p.M - CH)) * int(sizeof(T));
      else
        pa[w] = ga + int64_t(min(m0 + r, p.M - 1)) * p.lda + int64_t(kt) * 128 + c * 16;
    }
#pragma unroll
    for (int w = 0; w < NB; ++w) {
      int r, c;
      tile_word<T, BCOL, BN>((w * kWaves + wave) * 64 + lane, r, c);
      if constexpr (BCOL) {
        int which;
        const int col = min(b_col(c, which), p.N - CH);
        const char* gb = EPI == kEpiGated ? (which ? p.b[1] : p.b[0]) : (seg ? p.b[1] : gb0);
        pb[w] = gb + int64_t(kt * KT + r) * p.ldb + int64_t(col) * int(sizeof(T));
      } else {
        const char* gb = seg ? p.b[1] : gb0;
        pb[w] = gb + int64_t(min(n0 + r, p.N - 1)) * p.ldb + int64_t(kt) * 128 + c * 16;
      }
    }
  };
  const int64_t step_a = ACOL ? p.lda * KT : 128, step_b = BCOL ? p.ldb * KT : 128;

  // A word with masks: columns and rows past the operand's end read as zero.
  // `k`: its first (row) or only (col) contraction index; `i`: its row (row) or
  // first column (col).
  auto masked = [&](const char* base, int64_t ldx, bool col, int k, int i, int extent) {
    uint4 v = make_uint4(0, 0, 0, 0);
    const int major = col ? k : i, minor = col ? i : k;
    const int major_end = col ? p.K : extent, minor_end = col ? extent : p.K;
    if (major < major_end && minor < minor_end) {
      const char* src = base + int64_t(major) * ldx + int64_t(minor) * int(sizeof(T));
      if (minor + CH <= minor_end) {
        __builtin_memcpy(&v, src, 16);
      } else if constexpr (sizeof(T) == 4) {
        const uint32_t* e = reinterpret_cast<const uint32_t*>(src);
        v.x = e[0];
        if (minor + 1 < minor_end) v.y = e[1];
        if (minor + 2 < minor_end) v.z = e[2];
      } else if constexpr (sizeof(T) == 2) {
        const uint16_t* e = reinterpret_cast<const uint16_t*>(src);
        uint32_t h[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) h[n] = minor + n < minor_end ? e[n] : 0u;
        v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16,
                       h[6] | h[7] << 16);
      } else {  // 8-bit rows hold whole words
        __builtin_memcpy(&v, src, 16);
        v = first_codes(v, minor_end - minor);
      }
    }
    return v;
  };
  // The next fetch's segment, and its place in it.
  int seg = p.ktiles > 0 ? t0 / p.ktiles : 0, kt = t0 - seg * p.ktiles;
  auto masked_a = [&](int w) {
    int r, c;
    tile_word<T, ACOL, BM>((w * kWaves + wave) * 64 + lane, r, c);
    const char* ga = seg ? p.a[1] : p.a[0];
    return ACOL ? masked(ga, p.lda, true, kt * KT + r, m0 + c * CH, p.M)
                : masked(ga, p.lda, false, kt * KT + c * CH, m0 + r, p.M);
  };
  auto masked_b = [&](int w) {
    int r, c, which = 0;
    tile_word<T, BCOL, BN>((w * kWaves + wave) * 64 + lane, r, c);
    if constexpr (BCOL) {
      const int col = b_col(c, which);
      const char* gb = EPI == kEpiGated ? (which ? p.b[1] : p.b[0]) : (seg ? p.b[1] : gb0);
      return masked(gb, p.ldb, true, kt * KT + r, col, p.N);
    } else {
      return masked(seg ? p.b[1] : gb0, p.ldb, false, kt * KT + c * CH, n0 + r, p.N);
    }
  };
  auto place = [&](int buf, int w, bool b) {
    return smem + buf * kStage + (b ? kABytes : 0) + ((w * kWaves + wave) * 64) * 16;
  };

  // Tile t into buffer `buf`: copies in flight, or (STAGED, or a segment's
  // ragged last tile) through registers.
  uint4 ra[STAGED ? NA : 1], rb[STAGED ? NB : 1];
  int plain = 0;  // fetches by copies since the last other one
  auto fetch = [&](int t, int buf) {
    const bool last = kt + 1 == p.ktiles;
    if constexpr (STAGED) {
#pragma unroll
      for (int w = 0; w < NA; ++w) ra[w] = masked_a(w);
#pragma unroll
      for (int w = 0; w < NB; ++w) rb[w] = masked_b(w);
    } else if (last && ragged) {
      plain = 0;
#pragma unroll
      for (int w = 0; w < NA; ++w)
        *reinterpret_cast<uint4*>(place(buf, w, false) + lane * 16) = masked_a(w);
#pragma unroll
      for (int w = 0; w < NB; ++w)
        *reinterpret_cast<uint4*>(place(buf, w, true) + lane * 16) = masked_b(w);
    } else {
      ++plain;
#pragma unroll
      for (int w = 0; w < NA; ++w) copy_to_lds(pa[w], lds_address(place(buf, w, false)));
#pragma unroll
      for (int w = 0; w < NB; ++w) copy_to_lds(pb[w], lds_address(place(buf, w, true)));
    }
    ++kt;
    if (last) {
      kt = 0;
      ++seg;
    }
    if constexpr (!STAGED) {
      if (last) {
        if (t + 1 < t1) sources(seg, 0);
      } else {
#pragma unroll
        for (int w = 0; w < NA; ++w) pa[w] += step_a;
#pragma unroll
        for (int w = 0; w < NB; ++w) pb[w] += step_b;
      }
    }
  };
  auto settle = [&](int buf) {  // STAGED: the fetched words to LDS
    if constexpr (STAGED) {
#pragma unroll
      for (int w = 0; w < NA; ++w)
        *reinterpret_cast<uint4*>(place(buf, w, false) + lane * 16) = ra[w];
#pragma unroll
      for (int w = 0; w < NB; ++w)
        *reinterpret_cast<uint4*>(place(buf, w, true) + lane * 16) = rb[w];
    }
  };

  // Fragment of 16-row block `blk` of a tile, k step kk.
  using Frag = std::conditional_t<sizeof(T) == 1, Codes16, uint4>;
  auto frag = [&](const char* tile, auto col, int width, int blk, int kk) -> Frag {
    if constexpr (decltype(col)::value) {
      if constexpr (sizeof(T) == 2) {
        // Transposing reads: lane s of group q names row 8q + 4h + s/4, columns
        // 4(s%4)…+3 of the block, and receives column s of those four rows.
        const int g = width == 64 ? (s >> 3) | ((q & 1) << 1) : (s >> 2) | ((q & 1) << 2);
        const char* at = tile + (32 * kk + 8 * q + (s >> 2)) * (width * 2) + ((blk ^ g) * 32) +
                         (s & 3) * 8;
        typedef __attribute__((address_space(3))) i16x4* P;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)at);
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 4 * width * 2));
        const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
        return make_uint4(l.x, l.y, h.x, h.y);
      } else if constexpr (sizeof(T) == 4) {
        const char* at = tile + (16 * kk + 4 * q) * (width * 4) + ((blk ^ q) * 64) + s * 4;
        uint4 v;
        v.x = *reinterpret_cast<const uint32_t*>(at);
        v.y = *reinterpret_cast<const uint32_t*>(at + width * 4);
        v.z = *reinterpret_cast<const uint32_t*>(at + 2 * width * 4);
        v.w = *reinterpret_cast<const uint32_t*>(at + 3 * width * 4);
        return v;
      } else {
        static_assert(sizeof(T) != 1, "8-bit operands have k fastest");
      }
    } else {
      const int row = blk * 16 + s;
      const char* at = tile + row * 128;
      const int x = swizzle_row(s);
      if constexpr (sizeof(T) == 1) {
        return widen(*reinterpret_cast<const uint4*>(at + (((4 * kk + q) ^ x) << 4)));
      } else {
        return *reinterpret_cast<const uint4*>(at + (((4 * kk + q) ^ x) << 4));
      }
    }
  };
  auto mul = [&](const Frag& b, const Frag& a, f32x4& c) {
    if constexpr (sizeof(T) == 1) {
      c = mfma16(b.lo, a.lo, c);
      c = mfma16(b.hi, a.hi, c);
    } else if constexpr (sizeof(T) == 2) {
      c = mfma16(b, a, c);
    } else {
      c = mfma_f32(__uint_as_float(b.x), __uint_as_float(a.x), c);
      c = mfma_f32(__uint_as_float(b.y), __uint_as_float(a.y), c);
      c = mfma_f32(__uint_as_float(b.z), __uint_as_float(a.z), c);
      c = mfma_f32(__uint_as_float(b.w), __uint_as_float(a.w), c);
    }
  };

  if (t0 < t1) {
    if constexpr (!STAGED) sources(seg, kt);
    int ready = t0;  // tiles fetched
    for (; ready < min(t1, t0 + RING - 1); ++ready) fetch(ready, ready - t0);
    settle(0);
    int buf = 0, fill = RING - 1;
    for (int t = t0; t < t1; ++t) {
      // Tile t is there when no more copies are out than the RING − 2 tiles' after
      // it, if those were all copied.
      if (RING > 2 && ready - t == RING - 1 && plain >= RING - 2)
        wait_copies<(RING - 2) * (NA + NB)>();
      else
        wait_copies<0>();
      lds_barrier();
      if (ready < t1) fetch(ready, fill);
      const char* ta = smem + buf * kStage;
      const char* tb = ta + kABytes;
#pragma unroll
      for (int kn = 0; kn < E::kSteps / WK; ++kn) {
        const int kk = kn * WK + wk;
        Frag fb[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          fb[j] = frag(tb, std::integral_constant<bool, BCOL>{}, BN, wn * NJ + j, kk);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const Frag fa = frag(ta, std::integral_constant<bool, ACOL>{}, BM, wm * MI + i, kk);
#pragma unroll
          for (int j = 0; j < NJ; ++j) mul(fb[j], fa, acc[i][j]);
        }
      }
      if (ready < t1) {
        settle(fill);
        ++ready;
      }
      fill = buf;
      buf = buf + 1 == RING ? 0 : buf + 1;
    }
  }
  __syncthreads();

  // The two waves of a part of the tile exchange sums: each keeps half of the
  // row blocks, and adds in the order of the k steps.
  constexpr int ME = MI / WK;
  if constexpr (WK == 2) {
    f32x4* mine = reinterpret_cast<f32x4*>(smem) + wave * ME * NJ * 64 + lane;
    const f32x4* other =
        reinterpret_cast<f32x4*>(smem) + (wave ^ (WM * WN)) * ME * NJ * 64 + lane;
    static_assert(kWaves * ME * NJ * 1024 <= RING * kStage, "in LDS");
#pragma unroll
    for (int i = 0; i < ME; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) mine[(i * NJ + j) * 64] = wk ? acc[i][j] : acc[ME + i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ME; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const f32x4 v = other[(i * NJ + j) * 64];
        acc[i][j] = wk ? v + acc[ME + i][j] : acc[i][j] + v;
      }
    __syncthreads();
  }

  // Epilogue: up to 32 rows of a wave at a time through its own LDS.
  constexpr int kLd = 68;  // floats a row: 64 and a pad
  constexpr int kBlocks = ME < 2 || kWaves > 4 ? 1 : 2, kRows = 16 * kBlocks;
  static_assert(kWaves * kRows * kLd * 4 <= RING * kStage, "in LDS");
  float* stage = reinterpret_cast<float*>(smem) + wave * kRows * kLd;
  const int row0 = m0 + wm * (BM / WM) + wk * (ME * 16);
  const int col0 = n0 + wn * (EPI == kEpiGated ? 32 : 64);
#pragma unroll
  for (int half = 0; half < ME / kBlocks; ++half) {
#pragma unroll
    for (int ii = 0; ii < kBlocks; ++ii)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const f32x4 a = acc[kBlocks * half + ii][j];
        *reinterpret_cast<float4*>(stage + (ii * 16 + s) * kLd + j * 16 + 4 * q) =
            make_float4(a[0], a[1], a[2], a[3]);
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int kPer = EPI == kEpiGated ? 4 : 8;  // lanes to a row
    constexpr int kIts = kRows * kPer / 64;
    Tail<TO, EPI> tails[kIts];
    const int col = col0 + (lane % kPer) * 8, c = (lane % kPer) * 8;
    auto row_of = [&](int it) {
      return int64_t(row0) + half * kRows + it * (64 / kPer) + lane / kPer;
    };
#pragma unroll
    for (int it = 0; it < kIts; ++it)
      if (!p.partial && row_of(it) < p.M && col < p.N)
        tail_load<TO, EPI>(p, row_of(it), col, tails[it]);
#pragma unroll
    for (int it = 0; it < kIts; ++it) {
      const float* at = stage + (it * (64 / kPer) + lane / kPer) * kLd + c;
      float v[8], u[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(at);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(at + 4);
      if constexpr (EPI == kEpiGated) {
        *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(at + 32);
        *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(at + 36);
      }
      if (row_of(it) < p.M && col < p.N)
        finish8<TO, EPI>(p, z, sp, row_of(it), col, v, u, tails[it]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// The same product for large sizes: 256 × 256 tiles, four waves of 128 × 128,
// one to a SIMD, so that a fragment read from LDS feeds eight products (eight
// waves of 128 × 64 read 1.5 times as many bytes).
//
// LDS holds two k tiles (128 bytes of every row) of B and three of A: all of a
// CU's 160 KB. A tile is 16 slots: for each half of its k, each of the wave's
// eight row blocks against all eight column blocks. The order is fixed in the
// source (sched_barrier): a wave issues in order, so a memory instruction
// stands between any two or three products and issues while they run. In slots
// 0…5 the fragments of the tile's second half are read; at slot 8, where the
// wave holds all it needs of the tile, is the tile's one barrier; in slots
// 8…13 the fragments of the next tile's first half are read. Copies go out one
// a slot, A's of tile t + 2 in slots 0…7, B's in 8…15: the four waves' then
// take half of the vector memory path's time; two a slot take all of it, and
// the waves wait for it in place of the matrix unit.
//
// Copies take their address as a scalar base and a 32-bit offset: with 64-bit
// addresses in registers 16 loads beside 128 products take 1200 ns, like this
// 1116, without any loads 1096.
//
// "col" operands lie in LDS as subtiles of 128 columns, so that every copy
// instruction reads one matrix; gated: gate's and up's.
//
// One workgroup to a CU. Where the tiles are no whole number of rounds, the
// rest's k tiles are dealt out evenly (per_split to a workgroup): parts of a
// tile leave their sums in the workspace, and wide_join_kernel adds them in
// the order of k.
//
// Bound by the matrix unit's clock and by what of the loop does not hide behind
// it: a k tile takes 1.65 us on all CUs (1.3 PFLOP/s), a round of tiles 5 to 9 us
// of ends. Measured, bf16: 16384 x 4096 x 2048 x·W 217 us (1270 TFLOP/s), with a
// residual 239, its gradients 485 together; 8192 x 2048 x 12304 400 (1030); the
// feed-forward of 16384 x 2048 x 5632 942, its backward 2170. 8-bit: 3.2 us a k
// tile of 128, the bf16 rate; 8192 x 4096 x 4096 282 us (975).
template <class T, class TO, bool ACOL, bool BCOL, int EPI>
__global__ __launch_bounds__(256, 1) void gemm_wide_kernel(GemmArgs p) {
  using namespace gemm;
  using E = Elem<T>;
  constexpr int CH = E::kCh, KT = E::kKT, ES = int(sizeof(T));
  constexpr int kHalf = 256 * 128;  // bytes of an operand's tile
  constexpr int NW = 8;             // copies of an operand's tile a thread
  __shared__ __attribute__((aligned(16))) char smem[5 * kHalf];  // A, A, A, B, B

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int s = lane & 15, q = lane >> 4;

  // The workgroup's work: whole tiles while there are rounds of them for all
  // workgroups, then its share of the rest's k tiles. Workgroups go round the
  // eight XCDs: by `place` each XCD has a contiguous range of tiles, ordered in
  // bands of 8 tile rows, so its 32 CUs share operand tiles in its L2.
  const int groups = gridDim.x, tiles = p.tiles_m * p.tiles_n, nk = p.ktiles * p.nseg;
  const int xcd = blockIdx.x & 7, per_xcd = groups >> 3, more_xcd = groups & 7;
  const int place = xcd * per_xcd + min(xcd, more_xcd) + (blockIdx.x >> 3);
  int round = 0;
  int64_t unit = int64_t(place) * p.per_split;  // of the rest: tile · nk + k tile
  const int64_t unit_end =
      min(unit + p.per_split, int64_t(tiles * p.npair - p.rounds * groups) * nk);
  while (true) {
  int id, t0, t1, slot_no = -1;  // slot_no: where a part of a tile leaves its sums
  if (round < p.rounds) {
    id = round * groups + place;
    t0 = 0;
    t1 = nk;
    ++round;
  } else {
    if (unit >= unit_end) break;
    const int rest = int(unit / nk);
    t0 = int(unit - int64_t(rest) * nk);
    t1 = int(min(int64_t(nk), t0 + (unit_end - unit)));
    unit += t1 - t0;
    id = p.rounds * groups + rest;
    if (t1 - t0 < nk) slot_no = place + rest;
  }
  const int z = id / tiles;
  int tm, tn;
  {
    const int t = id - z * tiles, band = 8 * p.tiles_n, g = t / band, first = g * 8;
    const int rows = min(8, p.tiles_m - first), r = t - g * band;
    tm = first + r % rows;
    tn = r / rows;
  }
  constexpr int kCols = EPI == kEpiGated ? 128 : 256;
  const int m0 = tm * 256, n0 = tn * kCols;

  // Word w of a thread's copies of an operand's tile: (r, c) is its row and
  // 16-byte word ("row"), or its k and word of the subtile `sub` ("col").
  auto word = [&](auto col, int w, int& r, int& c, int& sub) {
    const int L = (w * 4 + wave) * 64 + lane;
    if constexpr (decltype(col)::value) {
      sub = (w * 4) >> 4;  // 16 KB subtiles: 1024 words, four of each thread
      const int l = L & 1023;
      r = l >> (CH == 8 ? 4 : 5);
      c = (l & (128 / CH - 1)) ^ swizzle_col<T, 128>(r);
    } else {
      sub = 0;
      r = L >> 3;
      c = (L & 7) ^ swizzle_row(r);
    }
  };
  static_assert(!(ACOL || BCOL) || sizeof(T) == 2, "subtiles of 1024 words");
  using AC = std::integral_constant<bool, ACOL>;
  using BC = std::integral_constant<bool, BCOL>;

  // Byte offsets of the copies' sources from the tile's base: rows past the end
  // moved back to the last one, words to the last whole one (what they give is
  // not stored).
  uint32_t oa[NW], ob[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    int r, c, sub;
    word(AC{}, w, r, c, sub);
    if constexpr (ACOL)
      oa[w] = uint32_t(r * p.lda) + uint32_t(min(sub * 128 + c * CH, p.M - CH - m0) * ES);
    else
      oa[w] = uint32_t(min(r, p.M - 1 - m0) * p.lda) + uint32_t(c * 16);
    word(BC{}, w, r, c, sub);
    if constexpr (BCOL)
      ob[w] = uint32_t(r * p.ldb) +
              uint32_t(min((EPI == kEpiGated ? 0 : sub * 128) + c * CH, p.N - CH - n0) * ES);
    else
      ob[w] = uint32_t(min(r, p.N - 1 - n0) * p.ldb) + uint32_t(c * 16);
  }
  // The tile being copied: its bases, and its place in its segment, followed
  // step by step (a division and a load of the segment's pointers a tile would
  // hold up the wave). `plain`: it is inside this workgroup's range, and not a
  // segment's ragged last one.
  const int segment0 = t0 / p.ktiles;
  int kt = t0 - segment0 * p.ktiles, left = t1 - t0;
  const char* pa = segment0 ? p.a[1] : p.a[0];
  const char* pb = segment0 || (p.npair == 2 && z) ? p.b[1] : p.b[0];
  const int64_t skip_a = ACOL ? int64_t(m0) * ES : int64_t(m0) * p.lda;
  const int64_t skip_b = BCOL ? int64_t(n0) * ES : int64_t(n0) * p.ldb;
  const int64_t step_a = ACOL ? p.lda * KT : 128, step_b = BCOL ? p.ldb * KT : 128;
  const char* ba = pa + skip_a + kt * step_a;
  const char* bb = pb + skip_b + kt * step_b;
  const char* bu = p.b[1] + skip_b + kt * step_b;  // gated: up
  const char *second_a = p.a[1] + skip_a, *second_b = p.b[1] + skip_b;
  const int whole_tiles = p.K / KT, ktiles = p.ktiles;
  auto plain = [&] { return left > 0 && kt < whole_tiles; };
  auto advance = [&] {
    --left;
    ++kt;
    ba += step_a;
    bb += step_b;
    bu += step_b;
    if (kt == ktiles) {
      kt = 0;
      ba = second_a;
      bb = second_b;
      pa = p.a[1];
      pb = p.b[1];
    }
  };
  const uint32_t lds0 = lds_address(smem) + uint32_t(wave) * 1024;
  auto copy = [&](uint32_t at, uint32_t offset, const char* base) {
    copy_to_lds(base, offset, lds0 + at);
  };
  // Buffers: A's of tile t is (t − t0) % 3, B's (t − t0) % 2.
  auto copy_a = [&](int buf, int w) { copy(uint32_t(buf * kHalf + w * 4096), oa[w], ba); };
  auto copy_b = [&](int buf, int w) {
    copy(uint32_t((3 + buf) * kHalf + w * 4096), ob[w],
         EPI == kEpiGated && w >= NW / 2 ? bu : bb);
  };
  auto masked = [&](const char* base, int64_t ldx, bool col, int k, int i, int extent) {
    const int major = col ? k : i, minor = col ? i : k;
    const int major_end = col ? p.K : extent, minor_end = col ? extent : p.K;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (major < major_end && minor < minor_end) {  // whole words, as the operands hold them
      v = *reinterpret_cast<const uint4*>(base + int64_t(major) * ldx + int64_t(minor) * ES);
      if constexpr (ES == 1) v = first_codes(v, minor_end - minor);
    }
    return v;
  };
  // A segment's ragged last tile, through registers with masks.
  auto ragged_a = [&](int buf) {
    const int k0 = kt * KT;
#pragma unroll 1
    for (int w = 0; w < NW; ++w) {
      int r, c, sub;
      word(AC{}, w, r, c, sub);
      *reinterpret_cast<uint4*>(smem + buf * kHalf + (w * 4 + wave) * 1024 + lane * 16) =
          ACOL ? masked(pa, p.lda, true, k0 + r, m0 + sub * 128 + c * CH, p.M)
               : masked(pa, p.lda, false, k0 + c * CH, m0 + r, p.M);
    }
  };
  auto ragged_b = [&](int buf) {
    const int k0 = kt * KT;
#pragma unroll 1
    for (int w = 0; w < NW; ++w) {
      int r, c, sub;
      word(BC{}, w, r, c, sub);
      *reinterpret_cast<uint4*>(smem + (3 + buf) * kHalf + (w * 4 + wave) * 1024 + lane * 16) =
          BCOL ? masked(EPI == kEpiGated && sub ? p.b[1] : pb, p.ldb, true, k0 + r,
                        n0 + (EPI == kEpiGated ? 0 : sub * 128) + c * CH, p.N)
               : masked(pb, p.ldb, false, k0 + c * CH, n0 + r, p.N);
    }
  };

  // Fragment of 16-row block `blk` of 128-row subtile `sub`, half kk.
  auto frag = [&](const char* tile, auto col, int sub, int blk, int kk) -> uint4 {
    if constexpr (decltype(col)::value) {
      const int g = (s >> 2) | ((q & 1) << 2);
      const char* at = tile + sub * 16384 + (32 * kk + 8 * q + (s >> 2)) * 256 + ((blk ^ g) * 32) +
                       (s & 3) * 8;
      typedef __attribute__((address_space(3))) i16x4* P;
      const uint2 l = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)at));
      const uint2 h =
          __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 1024)));
      return make_uint4(l.x, l.y, h.x, h.y);
    } else {
      return *reinterpret_cast<const uint4*>(tile + (sub * 128 + blk * 16 + s) * 128 +
                                             (((4 * kk + q) ^ swizzle_row(s)) << 4));
    }
  };

  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint4 fa[2][8], fb[2][8];  // [half][block]
  constexpr bool kF8 = sizeof(T) == 1;
  Codes16 wb[kF8 ? 8 : 1];
  // Fragment n of half kk's sixteen, in the order of their first use.
  auto read = [&](const char* a, const char* b, auto kk_no, auto n_no) {
    constexpr int kk = decltype(kk_no)::value, n = decltype(n_no)::value;
    if constexpr (n < 8)
      fb[kk][n] = EPI == kEpiGated ? frag(b, BC{}, n >> 2, wn * 4 + (n & 3), kk)
                                   : frag(b, BC{}, wn, n, kk);
    else
      fa[kk][n - 8] = frag(a, AC{}, wm, n - 8, kk);
  };

  {
    // Tiles t0 and t0 + 1.
    for (int d = 0; d < 2; ++d) {
      if (plain()) {
        each<NW>([&](auto w) {
          copy_a(d, w);
          copy_b(d, w);
        });
      } else if (left > 0) {
        ragged_a(d);
        ragged_b(d);
      }
      advance();
    }
    wait_copies<0>();
    __syncthreads();
    const char *sa = smem, *sb = smem + 3 * kHalf;
    using Half0 = std::integral_constant<int, 0>;
    using Half1 = std::integral_constant<int, 1>;
    each<16>([&](auto n) { read(sa, sb, Half0{}, n); });
    int abuf = 0;
    for (int t = t0; t < t1; ++t) {
      const int bbuf = (t - t0) & 1, anext = abuf == 2 ? 0 : abuf + 1;
      const int afill = anext == 2 ? 0 : anext + 1;  // of t − 1 and t + 2
      const char *ca = smem + abuf * kHalf, *cb = smem + (3 + bbuf) * kHalf;
      const char *na = smem + anext * kHalf, *nb = smem + (3 + (bbuf ^ 1)) * kHalf;
      const bool more = plain();  // tile t + 2
      if (!more && left > 0) ragged_a(afill);
      auto work = [&](auto slot_no) {
        constexpr int slot = decltype(slot_no)::value, kk = slot >> 3, i = slot & 7;
        Codes16 a;
        if constexpr (kF8) {
          if constexpr (i == 0)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              wb[j] = widen(fb[kk][j]);
              settle_words(wb[j]);
            }
          a = widen(fa[kk][i]);
          settle_words(a);
        }
        each<8>([&](auto jn) {
          constexpr int j = decltype(jn)::value;
          if constexpr (kF8) {
            mfma16_acc(wb[j].lo, a.lo, acc[i][j]);
            mfma16_acc(wb[j].hi, a.hi, acc[i][j]);
          } else {
            mfma16_acc(fb[kk][j], fa[kk][i], acc[i][j]);
          }
          __builtin_amdgcn_sched_barrier(0);
          // Sixteen fragments, three a slot: of this tile's second half from slot
          // 0 on, of the next tile's first half from slot 8 on (after the last
          // tile they are of no use).
          constexpr int n = 3 * i + (j >> 1);
          if constexpr ((j == 1 || j == 3 || j == 5) && n < 16) {
            if constexpr (slot < 8) read(ca, cb, Half1{}, std::integral_constant<int, n>{});
            else read(na, nb, Half0{}, std::integral_constant<int, n>{});
          }
          if constexpr (j == 6) {
            if constexpr (slot < 8) {
              if (more) copy_a(afill, i);
            } else {
              if (more) copy_b(bbuf, i);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        });
      };
      each<8>(work);
      // A's and B's tile t + 1 have landed once no more copies are out than
      // those of A's t + 2.
      if (more) wait_copies<NW>();
      else wait_copies<0>();
      lds_barrier();
      if (!more && left > 0) ragged_b(bbuf);
      each<8>([&](auto n) { work(std::integral_constant<int, 8 + n.value>{}); });
      advance();
      abuf = anext;
      // Where the loop ends the compiler may move sums already (it did so 14 states
      // after the last product).
      if (t + 1 == t1) settle_products();
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) settle_acc(acc[i]);

  // Epilogue: half of the wave's rows (64 by 128 columns) at a time through its
  // own LDS, 16-byte words XORed by row over the banks.
  float4* stage = reinterpret_cast<float4*>(smem) + wave * 64 * 32;
  auto at = [&](int r, int c) -> float4& { return stage[r * 32 + (c ^ (r & 15))]; };
  auto flush = [&](auto half) {
    constexpr int kHalfRows = decltype(half)::value;
    constexpr int kPer = EPI == kEpiGated ? 8 : 16;  // lanes to a row
    constexpr int kAtOnce = EPI == kEpiDGated ? 4 : 2;
    const int64_t row0 = m0 + wm * 128 + kHalfRows * 64;
    const int col = n0 + wn * (EPI == kEpiGated ? 64 : 128) + (lane % kPer) * 8;
    Tail<TO, EPI> tails[kAtOnce];
    auto fetch = [&](int it) {
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        const int64_t row = row0 + (it + n) * (64 / kPer) + lane / kPer;
        if (slot_no < 0 && row < p.M && col < p.N) tail_load<TO, EPI>(p, row, col, tails[n]);
      }
    };
    const bool bare = stored_as_they_are<EPI>(p);
    if (!bare) fetch(0);
#pragma unroll
    for (int ii = 0; ii < 4; ++ii)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const f32x4 v = acc[kHalfRows * 4 + ii][j];
        at(ii * 16 + s, 4 * j + q) = make_float4(v[0], v[1], v[2], v[3]);
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    auto local = [&](int it) { return it * (64 / kPer) + lane / kPer; };
    auto take = [&](int it, float (&v)[8], float (&u)[8]) {
      const int r = local(it), c = 2 * (lane % kPer);
      *reinterpret_cast<float4*>(v) = at(r, c);
      *reinterpret_cast<float4*>(v + 4) = at(r, c + 1);
      if constexpr (EPI == kEpiGated) {
        *reinterpret_cast<float4*>(u) = at(r, 16 + c);
        *reinterpret_cast<float4*>(u + 4) = at(r, 16 + c + 1);
      }
    };
    if (slot_no >= 0) {  // a part: its sums to the workspace, gate's then up's
#pragma unroll 4
      for (int it = 0; it < kPer; ++it) {
        float v[8], u[8];
        take(it, v, u);
        float* to =
            p.partial + ((int64_t(slot_no) * 256 + int(row0 - m0) + local(it)) << 8) + (col - n0);
        store8(to, v, 8);
        if constexpr (EPI == kEpiGated) store8(to + 128, u, 8);
      }
    } else if (bare) {
#pragma unroll 1
      for (int it = 0; it < kPer; it += 4) {
        Raw8<TO> r[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int64_t row = row0 + local(it + n);
          if (p.residual && row < p.M && col < p.N)
            r[n].load(static_cast<const TO*>(p.residual) + row * p.ldr + col, p.N - col);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float v[8], u[8];
          take(it + n, v, u);
          const int64_t row = row0 + local(it + n);
          if (p.residual) {
            r[n].get(u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += u[i];
          }
          if (row < p.M && col < p.N)
            store8(static_cast<TO*>(z ? p.out[1] : p.out[0]) + row * p.ldo + col, v, p.N - col);
        }
      }
    } else {
      // What the epilogue reads for eight rows is in flight at a time, the first
      // eight's since before the sums went to LDS.
#pragma unroll 1
      for (int it = 0; it < kPer; it += kAtOnce) {
        if (it > 0) fetch(it);
        float v[kAtOnce][8], u[EPI == kEpiGated ? kAtOnce : 1][8];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) take(it + n, v[n], u[EPI == kEpiGated ? n : 0]);
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n)
          if (row0 + local(it + n) < p.M && col < p.N)
            tail_store<TO, EPI>(p, z, row0 + local(it + n), col, v[n],
                                u[EPI == kEpiGated ? n : 0], tails[n]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  flush(std::integral_constant<int, 0>{});
  flush(std::integral_constant<int, 1>{});
  __syncthreads();
  }
}

}  // namespace dn

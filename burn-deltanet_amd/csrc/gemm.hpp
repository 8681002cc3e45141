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
  int split;            // workgroups along the contraction
  int per_split;        // k tiles of each
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

// act(z) and its derivative. GELU is the exact form, z·Φ(z).
__device__ inline float gelu_cdf(float z) { return 0.5f * (1.0f + erff(z * 0.70710678118654752f)); }
__device__ inline float act_value(float z, int kind) {
  if (kind == DN_ACT_GELU) return z * gelu_cdf(z);
  return activate(z, kind);
}
__device__ inline float act_slope(float z, int kind) {
  switch (kind) {
    case DN_ACT_SILU: {
      const float s = sigmoidf_(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case DN_ACT_RELU: return z > 0.f ? 1.0f : 0.f;
    case DN_ACT_GELU:
      return gelu_cdf(z) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
    default: return 1.0f;
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

// The linear epilogue on eight columns of a row (z: the product, and on
// return act's value with the residual). Shared by the tile kernel, the
// few-rows kernel and the join of split contractions.
template <class TO>
__device__ inline void linear_tail(const GemmArgs& p, int z, int64_t row, int col, float (&v)[8]) {
  const int valid = p.N - col;
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
  if (p.act != DN_ACT_IDENTITY) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value(v[i], p.act);
  }
  if (p.residual) {
    float r[8];
    load8(static_cast<const TO*>(p.residual) + row * p.ldr + col, r, valid);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  store8(static_cast<TO*>(z ? p.out[1] : p.out[0]) + row * p.ldo + col, v, valid);
}
// h = act(g)·u, and the kept g and u.
template <class TO>
__device__ inline void gated_tail(const GemmArgs& p, int64_t row, int col, const float (&g)[8],
                                  const float (&u)[8]) {
  const int valid = p.N - col;
  if (p.preact) {
    store8(static_cast<TO*>(p.preact) + row * p.ldp + col, g, valid);
    store8(static_cast<TO*>(p.up) + row * p.ldp + col, u, valid);
  }
  float h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = act_value(g[i], p.act) * u[i];
  store8(static_cast<TO*>(p.out[0]) + row * p.ldo + col, h, valid);
}
// From d_h and the kept g and u: d_g = d_h·u·act'(g), d_u = d_h·act(g), and h
// again for the down projection's weight gradient.
template <class TO>
__device__ inline void dgated_tail(const GemmArgs& p, int64_t row, int col, const float (&dh)[8]) {
  const int valid = p.N - col;
  float g[8], u[8], dg[8], du[8], h[8];
  load8(static_cast<const TO*>(p.preact) + row * p.ldp + col, g, valid);
  load8(static_cast<const TO*>(p.up) + row * p.ldp + col, u, valid);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = act_value(g[i], p.act);
    dg[i] = dh[i] * u[i] * act_slope(g[i], p.act);
    du[i] = dh[i] * a;
    h[i] = a * u[i];
  }
  store8(static_cast<TO*>(p.out[0]) + row * p.ldo + col, dg, valid);
  store8(static_cast<TO*>(p.out[1]) + row * p.ldo + col, du, valid);
  store8(static_cast<TO*>(p.h) + row * p.ldo + col, h, valid);
}

// One HBM → LDS copy of 16 bytes a lane: lane i's word goes to `lds` + 16·i.
// No register receives it; it is complete when vmcnt says so. Nothing else in
// these kernels uses m0 (LDS accesses do not need it on this architecture).
__device__ inline void copy_to_lds(const char* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(src)
               : "memory");
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
// "col" tiles: k's rows are whole multiples of 256 bytes. bf16: a transposing
// read takes 32 bytes of rows 8q + 4h + 0…3 for the lanes' four groups q; the
// eight rows of a half wave get eight places. fp32: rows 4q + i, 64 bytes each.
template <class T>
__device__ inline int swizzle_col(int k) {
  if constexpr (sizeof(T) == 2) return 2 * ((k & 3) | ((k >> 1) & 4));
  else return 4 * ((k >> 2) & 3);
}

// Which 16-byte word of an operand goes to word `L` of its tile.
// "row": row r = L / 8 and word c of its 128 bytes; "col": k = L / (R/kCh),
// word c of its R columns.
template <class T, bool COL, int R>
__device__ inline void tile_word(int L, int& r, int& c) {
  if constexpr (COL) {
    constexpr int W = R / Elem<T>::kCh;
    r = L / W;
    c = (L % W) ^ swizzle_col<T>(r);
  } else {
    r = L >> 3;
    c = (L & 7) ^ swizzle_row(r);
  }
}

}  // namespace gemm

// BM × BN tiles, WM × WN waves. ACOL, BCOL: layouts. STAGED: operands whose
// rows do not lie at 16-byte steps go through registers, with masks.
template <class T, class TO, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, int EPI,
          bool STAGED>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs p) {
  using namespace gemm;
  using E = Elem<T>;
  constexpr int kThreads = 64 * WM * WN, CH = E::kCh, KT = E::kKT;
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;  // 16×16 blocks of a wave
  constexpr int kABytes = BM * 128, kBBytes = BN * 128, kStage = kABytes + kBBytes;
  constexpr int NA = kABytes / 16 / kThreads, NB = kBBytes / 16 / kThreads;
  static_assert(NA * kThreads * 16 == kABytes && NB * kThreads * 16 == kBBytes, "whole copies");
  static_assert(NJ == 4, "the epilogue's rows of 64 columns");
  __shared__ __attribute__((aligned(16))) char smem[2 * kStage];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
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
  auto sources = [&](int t) {  // of k tile t
    const int seg = t / p.ktiles, kt = t - seg * p.ktiles;
    const char* ga = seg ? p.a[1] : p.a[0];
#pragma unroll
    for (int w = 0; w < NA; ++w) {
      int r, c;
      tile_word<T, ACOL, BM>((w * WM * WN + wave) * 64 + lane, r, c);
      if constexpr (ACOL)
        pa[w] = ga + int64_t(kt * KT + r) * p.lda +
                int64_t(min(m0 + c * CH, p.M - CH)) * int(sizeof(T));
      else
        pa[w] = ga + int64_t(min(m0 + r, p.M - 1)) * p.lda + int64_t(kt) * 128 + c * 16;
    }
#pragma unroll
    for (int w = 0; w < NB; ++w) {
      int r, c;
      tile_word<T, BCOL, BN>((w * WM * WN + wave) * 64 + lane, r, c);
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
      }
    }
    return v;
  };
  auto masked_a = [&](int t, int w) {
    const int seg = t / p.ktiles, kt = t - seg * p.ktiles;
    int r, c;
    tile_word<T, ACOL, BM>((w * WM * WN + wave) * 64 + lane, r, c);
    const char* ga = seg ? p.a[1] : p.a[0];
    return ACOL ? masked(ga, p.lda, true, kt * KT + r, m0 + c * CH, p.M)
                : masked(ga, p.lda, false, kt * KT + c * CH, m0 + r, p.M);
  };
  auto masked_b = [&](int t, int w) {
    const int seg = t / p.ktiles, kt = t - seg * p.ktiles;
    int r, c, which = 0;
    tile_word<T, BCOL, BN>((w * WM * WN + wave) * 64 + lane, r, c);
    if constexpr (BCOL) {
      const int col = b_col(c, which);
      const char* gb = EPI == kEpiGated ? (which ? p.b[1] : p.b[0]) : (seg ? p.b[1] : gb0);
      return masked(gb, p.ldb, true, kt * KT + r, col, p.N);
    } else {
      return masked(seg ? p.b[1] : gb0, p.ldb, false, kt * KT + c * CH, n0 + r, p.N);
    }
  };
  auto place = [&](int buf, int w, bool b) {
    return smem + buf * kStage + (b ? kABytes : 0) + ((w * WM * WN + wave) * 64) * 16;
  };

  // Tile t into buffer `buf`: copies in flight, or (STAGED, or a segment's
  // ragged last tile) through registers.
  uint4 ra[STAGED ? NA : 1], rb[STAGED ? NB : 1];
  auto fetch = [&](int t, int buf) {
    if constexpr (STAGED) {
#pragma unroll
      for (int w = 0; w < NA; ++w) ra[w] = masked_a(t, w);
#pragma unroll
      for (int w = 0; w < NB; ++w) rb[w] = masked_b(t, w);
    } else {
      const bool last = (t + 1) % p.ktiles == 0;
      if (last && ragged) {
#pragma unroll
        for (int w = 0; w < NA; ++w)
          *reinterpret_cast<uint4*>(place(buf, w, false) + lane * 16) = masked_a(t, w);
#pragma unroll
        for (int w = 0; w < NB; ++w)
          *reinterpret_cast<uint4*>(place(buf, w, true) + lane * 16) = masked_b(t, w);
      } else {
#pragma unroll
        for (int w = 0; w < NA; ++w) copy_to_lds(pa[w], lds_address(place(buf, w, false)));
#pragma unroll
        for (int w = 0; w < NB; ++w) copy_to_lds(pb[w], lds_address(place(buf, w, true)));
      }
      if (last) {
        if (t + 1 < t1) sources(t + 1);
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
        const int g = (s >> 2) | ((q & 1) << 2);
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
    if constexpr (!STAGED) sources(t0);
    fetch(t0, 0);
    settle(0);
    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
      wait_copies<0>();
      __syncthreads();
      if (t + 1 < t1) fetch(t + 1, buf ^ 1);
      const char* ta = smem + buf * kStage;
      const char* tb = ta + kABytes;
#pragma unroll
      for (int kk = 0; kk < E::kSteps; ++kk) {
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
      if (t + 1 < t1) settle(buf ^ 1);
    }
  }
  __syncthreads();

  // Epilogue: 32 rows of the wave at a time through its own LDS.
  constexpr int kLd = 68;  // floats a row: 64 and a pad
  float* stage = reinterpret_cast<float*>(smem) + wave * 32 * kLd;
  const int row0 = m0 + wm * (BM / WM);
  const int col0 = n0 + wn * (EPI == kEpiGated ? 32 : 64);
#pragma unroll
  for (int half = 0; half < MI / 2; ++half) {
#pragma unroll
    for (int ii = 0; ii < 2; ++ii)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const f32x4 a = acc[2 * half + ii][j];
        *reinterpret_cast<float4*>(stage + (ii * 16 + s) * kLd + j * 16 + 4 * q) =
            make_float4(a[0], a[1], a[2], a[3]);
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int kPer = EPI == kEpiGated ? 4 : 8;  // lanes to a row
#pragma unroll
    for (int it = 0; it < 32 * kPer / 64; ++it) {
      const int r = it * (64 / kPer) + lane / kPer, c = (lane % kPer) * 8;
      const int64_t row = row0 + half * 32 + r;
      const int col = col0 + c;
      float v[8], u[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(stage + r * kLd + c);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(stage + r * kLd + c + 4);
      if constexpr (EPI == kEpiGated) {
        *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(stage + r * kLd + 32 + c);
        *reinterpret_cast<float4*>(u + 4) =
            *reinterpret_cast<const float4*>(stage + r * kLd + 36 + c);
      }
      if (row < p.M && col < p.N) {
        if (p.partial) {
          float* at = p.partial + (int64_t(sp * p.npair + z) * p.M + row) * p.ldpart + col;
          store8(at, v, p.N - col);
          if constexpr (EPI == kEpiGated)
            store8(at + p.N, u, p.N - col);
        } else if constexpr (EPI == kEpiLinear) {
          linear_tail<TO>(p, z, row, col, v);
        } else if constexpr (EPI == kEpiGated) {
          gated_tail<TO>(p, row, col, v, u);
        } else {
          dgated_tail<TO>(p, row, col, v);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace dn

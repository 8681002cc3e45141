// Products of few rows (single tokens, small batches): x·W with W [K][N] in
// bf16 or fp32, or 8-bit x·Wᵀ with W [N][K], and the gated pair of products.
//
// Bound by reading W once. A workgroup owns 64 or 32 columns and all of the
// contraction, which its 16 waves share in steps of 32 rows of W (16 in fp32;
// 64 k of 8-bit rows), with the loads of 2 to 4 steps of a wave in flight, up
// to 128 KB a CU. The waves' sums meet in LDS, halving their number at each
// turn, so one launch does it all and the order of the sums is fixed.
//
// W needs no transposition through LDS: a lane loads NC adjacent columns of the
// 8 (bf16) rows that the matrix instruction wants of it, and a permute of two
// halves a word makes them k-adjacent. Its 16 columns of instruction j are
// those NC apart, j, j + NC, …, so a lane ends with NC adjacent columns of 4
// rows.
#include <algorithm>

#include "layer.hpp"

namespace dn {
namespace {

constexpr int kFewWaves = 16;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// MT: blocks of 16 rows of x. NC: adjacent columns a lane (a workgroup has
// 16·NC). DEPTH: steps in flight. NP: products side by side (gated: 2).
template <class T, class TO, int MT, int NC, int DEPTH, int EPI>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(GemmArgs p) {
  using namespace gemm;
  constexpr bool kBf = sizeof(T) == 2, kF8 = sizeof(T) == 1;
  constexpr int NP = EPI == kEpiGated ? 2 : 1;
  constexpr int KS = kF8 ? 64 : kBf ? 32 : 16;  // contraction of a step
  constexpr int KL = KS / 4;                    // of a lane: bf16 8, fp32 4, 8-bit 16
  constexpr int ES = int(sizeof(T));
  // What a lane holds of a step: x's words, and of W 8 rows of NC columns
  // (bf16), 4 rows of NC (fp32) or 16 codes of NC columns (8-bit).
  constexpr int NW = kF8 ? NC : KL;
  constexpr int kDw = kF8 ? 4 : NC * ES / 4;  // 32-bit words of a load
  struct Step {
    u32x4 x[MT];
    uint32_t w[NP][NW][kDw];
  };
  constexpr int kFewCols = 16 * NC;
  __shared__ __attribute__((aligned(16))) float sums[kFewWaves / 2][NP][MT][4][64][NC];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.x * kFewCols, col = c0 + NC * s;
  const int K = p.K, whole = K / KS;  // whole steps

  // Rows past x's end repeat its last one: what they give is not stored.
  const char* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = p.a[0] + int64_t(min(16 * m + s, p.M - 1)) * p.lda;
  // Columns past N − NC: the last NC ones are loaded, and moved down by `over`
  // (what comes in behind them is not stored; 8-bit columns repeat the last).
  const int from = kF8 ? col : min(col, p.N - NC), over = col - from;
  const bool edge = c0 + kFewCols > p.N;
  auto fetch_w = [&](Step& st, int k, int k_end) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int r = 0; r < NW; ++r) {
        const char* at = kF8 ? p.b[n] + int64_t(min(col + r, p.N - 1)) * p.ldb + min(k, k_end - KL)
                             : p.b[n] + int64_t(min(k + r, k_end - 1)) * p.ldb + int64_t(from) * ES;
        __builtin_memcpy(st.w[n][r], at, 4 * kDw);
      }
    if (!kF8 && edge) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int r = 0; r < NW; ++r) {
          uint32_t* w = st.w[n][r];
          if constexpr (kBf && NC == 4) {
            const uint64_t v = (uint64_t(w[1]) << 32 | w[0]) >> (16 * min(over, 3));
            w[0] = uint32_t(v);
            w[1] = uint32_t(v >> 32);
          } else if constexpr (kBf) {
            w[0] >>= 16 * min(over, 1);
          } else {
#pragma unroll
            for (int o = 1; o < NC; ++o)
              if (over >= o)
#pragma unroll
                for (int e = 0; e + 1 < NC; ++e) w[e] = w[e + 1];
          }
        }
    }
  };
  auto fetch = [&](Step& st, int step) {  // of the whole ones
    if (step >= whole) return;
    const int k = step * KS + q * KL;
    fetch_w(st, k, 0x7fffffff);
#pragma unroll
    for (int m = 0; m < MT; ++m) __builtin_memcpy(&st.x[m], xr[m] + int64_t(k) * ES, 16);
  };
  // The ragged last step: what lies past K is zero in both. 8-bit rows hold whole
  // words, whose codes past K may be any.
  auto fetch_ragged = [&](Step& st) {
    const int k = whole * KS + q * KL;
    fetch_w(st, k, kF8 ? (K + KL - 1) / KL * KL : K);
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int r = 0; r < NW; ++r) {
        if constexpr (kF8) {
          uint4 v;
          __builtin_memcpy(&v, st.w[n][r], 16);
          v = first_codes(v, K - k);
          __builtin_memcpy(st.w[n][r], &v, 16);
        } else {
#pragma unroll
          for (int d = 0; d < kDw; ++d)
            if (k + r >= K) st.w[n][r][d] = 0;
        }
      }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      u32x4 v = {0, 0, 0, 0};
      if constexpr (kF8) {
        if (k < K) {
          __builtin_memcpy(&v, xr[m] + k, 16);
          v = __builtin_bit_cast(u32x4, first_codes(__builtin_bit_cast(uint4, v), K - k));
        }
      } else {
#pragma unroll
        for (int e = 0; e < KL; ++e) {
          if (k + e >= K) continue;
          if constexpr (kBf)
            v[e >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(xr[m])[k + e]) << (16 * (e & 1));
          else
            v[e] = reinterpret_cast<const uint32_t*>(xr[m])[k + e];
        }
      }
      st.x[m] = v;
    }
  };

  f32x4 acc[NP][MT][NC];
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[n][m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Step& st) {
    if constexpr (kF8) {
      Codes16 x[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m] = widen(__builtin_bit_cast(uint4, st.x[m]));
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const Codes16 w = widen(make_uint4(st.w[0][j][0], st.w[0][j][1], st.w[0][j][2],
                                           st.w[0][j][3]));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          acc[0][m][j] = mfma16(x[m].lo, w.lo, acc[0][m][j]);
          acc[0][m][j] = mfma16(x[m].hi, w.hi, acc[0][m][j]);
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          if constexpr (kBf) {
            // Column j of rows k and k + 1: two halves to a word.
            uint32_t f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              f[e] = __builtin_amdgcn_perm(st.w[n][2 * e + 1][j >> 1], st.w[n][2 * e][j >> 1],
                                           j & 1 ? 0x07060302u : 0x05040100u);
            const uint4 w = make_uint4(f[0], f[1], f[2], f[3]);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[n][m][j] = mfma16(__builtin_bit_cast(uint4, st.x[m]), w, acc[n][m][j]);
          } else {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[n][m][j] = mfma_f32(__uint_as_float(st.x[m][e]),
                                        __uint_as_float(st.w[n][e][j]), acc[n][m][j]);
          }
        }
    }
  };

  Step st[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) fetch(st[d], wave + d * kFewWaves);
  for (int step = wave; step < whole; step += DEPTH * kFewWaves) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (step + d * kFewWaves < whole) multiply(st[d]);
      fetch(st[d], step + (d + DEPTH) * kFewWaves);
    }
  }
  if (K % KS && whole % kFewWaves == wave) {
    fetch_ragged(st[0]);
    multiply(st[0]);
  }

  // The waves' sums, the upper half's added to the lower half's.
  auto put = [&](int place) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < NC; ++j) sums[place][n][m][r][lane][j] = acc[n][m][j][r];
  };
#pragma unroll 1
  for (int half = kFewWaves / 2; half; half >>= 1) {
    if (wave >= half && wave < 2 * half) put(wave - half);
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NC; ++j) acc[n][m][j][r] += sums[wave][n][m][r][lane][j];
    }
    __syncthreads();
  }
  // Sums of row 16m + 4q + r, columns col …, back through LDS: a thread
  // finishes 8 adjacent columns of a row.
  if (wave == 0) put(0);
  __syncthreads();
  constexpr int kGroups = kFewCols / 8;  // of 8 columns
  for (int i = threadIdx.x; i < 16 * MT * kGroups; i += 64 * kFewWaves) {
    const int row = i / kGroups, c8 = (i % kGroups) * 8;
    if (row >= p.M || c0 + c8 >= p.N) continue;
    const int m = row >> 4, first = ((row >> 2) & 3) * 16 + c8 / NC, r = row & 3;
    Tail<TO, EPI> tail;
    tail_load<TO, EPI>(p, row, c0 + c8, tail);
    float v[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = sums[0][0][m][r][first + e / NC][e % NC];
      if constexpr (NP == 2) u[e] = sums[0][1][m][r][first + e / NC][e % NC];
    }
    tail_store<TO, EPI>(p, 0, row, c0 + c8, v, u, tail);
  }
}

// Up to 16 rows of bf16 whose rows and W's lie at 16-byte steps. The kernel
// above loads NC·2 bytes a lane, and the vector memory path takes 16 cycles an
// instruction of 64 lanes whatever their width: 29 GB/s a CU at NC = 2. Here a
// wave copies W to its own part of LDS, 16 bytes a lane, in chunks of 32 rows by
// 16·CB columns (gated: of both matrices), with x's 32 columns beside them, and
// reads both back as fragments, W's transposed. kRing chunks are in flight, 6 to 8 KB
// of W a wave; no wave waits for another before the sums meet.
//
// Measured, one row of bf16: 2048 x 12304 10.8 us (4.7 TB/s), the gated pair of
// 2048 x 5632 13.2 (3.5), 5632 x 2048 in four parts 6.8 and the join's 3.3.
template <int CB, int EPI>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_copy_kernel(GemmArgs p) {
  using namespace gemm;
  constexpr int NP = EPI == kEpiGated ? 2 : 1;
  constexpr int kCols = 16 * CB, kRow = 32 * CB;  // columns, bytes of a row
  constexpr int kPart = 32 * kRow;                // bytes of a chunk of one matrix
  constexpr int kChunk = NP * kPart + 1024;       // and x's
  constexpr int kRing = 10240 / kChunk;
  constexpr int kCopies = kChunk / 1024;
  static_assert(kRing >= 2 && kRing * kChunk * kFewWaves <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[kRing * kChunk * kFewWaves];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = lane & 15, q = lane >> 4;
  // An XCD's workgroups have adjacent columns: rows whose parts share a line
  // are read into its L2 once.
  const int groups = gridDim.x, per = groups >> 3, rem = groups & 7, xcd = blockIdx.x & 7;
  const int c0 = (xcd * per + min(xcd, rem) + (blockIdx.x >> 3)) * kCols;
  // Whole chunks of this workgroup's share of the contraction.
  const int K = p.K, all = K / 32, lo = int(blockIdx.y) * p.per_split;
  const int chunks = min(p.per_split, all - lo);

  // Sources of a lane's copies from chunk 0 (words past N: the last whole one's).
  constexpr int kLanesRow = kRow / 16, kRows = 64 / kLanesRow;  // rows of a copy
  const int wrow = lane / kLanesRow, wcol = min(c0 + (lane % kLanesRow) * 8, p.N - 8);
  const int64_t step = int64_t(32) * p.ldb;
  const char* w0 = p.b[0] + int64_t(wrow) * p.ldb + int64_t(wcol) * 2;
  const char* w1 = NP == 2 ? p.b[1] + int64_t(wrow) * p.ldb + int64_t(wcol) * 2 : w0;
  const char* x0 = p.a[0] + int64_t(min(lane >> 2, p.M - 1)) * p.lda + (lane & 3) * 16;
  const uint32_t lds0 = lds_address(smem) + uint32_t(wave) * kRing * kChunk;
  auto fetch = [&](int slot, int c) {
    const uint32_t at = lds0 + uint32_t(slot) * kChunk;
#pragma unroll
    for (int i = 0; i < 32 / kRows; ++i)
      copy_to_lds(w0 + c * step + int64_t(i * kRows) * p.ldb, at + i * 1024);
    if constexpr (NP == 2) {
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i)
        copy_to_lds(w1 + c * step + int64_t(i * kRows) * p.ldb, at + kPart + i * 1024);
    }
    copy_to_lds(x0 + int64_t(c) * 64, at + NP * kPart);
  };

  f32x4 acc[NP][CB];
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int slot) {
    const char* at = smem + (wave * kRing + slot) * kChunk;
    const uint4 x = *reinterpret_cast<const uint4*>(at + NP * kPart + s * 64 + q * 16);
    typedef __attribute__((address_space(3))) i16x4* P;
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        const char* w = at + n * kPart + (8 * q + (s >> 2)) * kRow + j * 32 + (s & 3) * 8;
        const uint2 l = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)w));
        const uint2 h = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(w + 4 * kRow)));
        acc[n][j] = mfma16(x, make_uint4(l.x, l.y, h.x, h.y), acc[n][j]);
      }
  };

  // This wave's chunks: wave, wave + 16, …; `mine` of them.
  const int mine = chunks > wave ? (chunks - wave + kFewWaves - 1) / kFewWaves : 0;
#pragma unroll
  for (int d = 0; d < kRing; ++d)
    if (d < mine) fetch(d, lo + wave + d * kFewWaves);
  for (int n = 0; n < mine; n += kRing) {
#pragma unroll
    for (int d = 0; d < kRing; ++d) {
      if (n + d >= mine) break;
      // All but the copies of the chunks behind this one have landed.
      if (n + d + kRing <= mine) wait_copies<(kRing - 1) * kCopies>();
      else wait_copies<0>();
      multiply(d);
      if (n + d + kRing < mine) {
        // The fragments are in registers before their place is refilled.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        fetch(d, lo + wave + (n + d + kRing) * kFewWaves);
      }
    }
  }
  if (K % 32 && lo + chunks == all && chunks % kFewWaves == wave) {
    // The ragged last rows, element by element: what lies past K is zero.
    const int k = all * 32 + 8 * q;
    auto eight = [&](auto at) {
      uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < K) v[e >> 1] |= uint32_t(*at(e)) << (16 * (e & 1));
      return make_uint4(v[0], v[1], v[2], v[3]);
    };
    const char* xr = p.a[0] + int64_t(min(s, p.M - 1)) * p.lda;
    const uint4 x = eight([&](int e) { return reinterpret_cast<const uint16_t*>(xr) + k + e; });
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int j = 0; j < CB; ++j) {
        const int col = min(c0 + 16 * j + s, p.N - 1);
        const uint4 w = eight([&](int e) {
          return reinterpret_cast<const uint16_t*>(p.b[n] + int64_t(k + e) * p.ldb) + col;
        });
        acc[n][j] = mfma16(x, w, acc[n][j]);
      }
  }

  // Row 4q + r, column 16j + s of the waves' sums, added by halves. The ring's
  // place is free once every wave has read its last chunk.
  float(*sums)[NP][CB][4][64] = reinterpret_cast<float(*)[NP][CB][4][64]>(smem);
  static_assert(sizeof(float) * NP * CB * 4 * 64 * (kFewWaves / 2) <= sizeof(smem), "the sums");
  __syncthreads();
  auto put = [&](int place) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int j = 0; j < CB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[place][n][j][r][lane] = acc[n][j][r];
  };
#pragma unroll 1
  for (int half = kFewWaves / 2; half; half >>= 1) {
    if (wave >= half && wave < 2 * half) put(wave - half);
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[n][j][r] += sums[wave][n][j][r][lane];
    }
    __syncthreads();
  }
  if (wave == 0) put(0);
  __syncthreads();
  const int i = threadIdx.x, row = i / (kCols / 8), c8 = (i % (kCols / 8)) * 8;
  if (row >= p.M || row >= 16 || c0 + c8 >= p.N) return;
  Tail<bf16, EPI> tail;
  if (!p.partial) tail_load<bf16, EPI>(p, row, c0 + c8, tail);
  float v[8], u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = (row >> 2) * 16 + (c8 & 8) + e;
    v[e] = sums[0][0][c8 >> 4][row & 3][at];
    if constexpr (NP == 2) u[e] = sums[0][1][c8 >> 4][row & 3][at];
  }
  finish8<bf16, EPI>(p, 0, blockIdx.y, row, c0 + c8, v, u, tail);
}

template <int CB, int EPI>
hipError_t few_copy_launch(const GemmArgs& g, hipStream_t stream) {
  hipLaunchKernelGGL((few_rows_copy_kernel<CB, EPI>),
                     dim3(unsigned((g.N + 16 * CB - 1) / (16 * CB)), unsigned(g.split)),
                     dim3(64 * kFewWaves), 0, stream, g);
  return hipGetLastError();
}

template <class T, class TO, int MT, int NC, int DEPTH, int EPI>
hipError_t few_launch(const GemmArgs& g, hipStream_t stream) {
  hipLaunchKernelGGL((few_rows_kernel<T, TO, MT, NC, DEPTH, EPI>),
                     dim3(unsigned((g.N + 16 * NC - 1) / (16 * NC))), dim3(64 * kFewWaves), 0,
                     stream, g);
  return hipGetLastError();
}

// 32 columns a workgroup where 64 would leave half of the CUs without one.
template <class T, class TO>
hipError_t few_go(const GemmArgs& g, GemmEpi epi, hipStream_t stream) {
  const bool narrow = (g.N + 63) / 64 < device_cu_count() / 2;
  constexpr bool kWide = sizeof(T) == 4;  // fp32 steps hold twice the registers
  if constexpr (sizeof(T) > 1) {
    if (epi == kEpiGated) {
      if (g.M > 16) return few_launch<T, TO, 2, 2, kWide ? 1 : 2, kEpiGated>(g, stream);
      if (narrow) return few_launch<T, TO, 1, 2, kWide ? 2 : 3, kEpiGated>(g, stream);
      return few_launch<T, TO, 1, 4, kWide ? 1 : 2, kEpiGated>(g, stream);
    }
  }
  if (g.M > 32) return few_launch<T, TO, 4, 4, 1, kEpiLinear>(g, stream);
  if (g.M > 16) return few_launch<T, TO, 2, 4, kWide ? 1 : 2, kEpiLinear>(g, stream);
  if (narrow) return few_launch<T, TO, 1, 2, 4, kEpiLinear>(g, stream);
  return few_launch<T, TO, 1, 4, kWide ? 2 : 3, kEpiLinear>(g, stream);
}

}  // namespace

// Parts of the contraction, each a workgroup's for its columns. Few columns
// leave CUs without work, and a CU takes W's rows at 28 GB/s whatever its waves
// do: more parts where that makes up for the join's 4.5 us. One row of
// 5632 x 2048: 13.8 us whole, four parts 6.8 and their join 3.3.
int few_rows_split(const GemmArgs& g, GemmEpi epi, int dtype, bool copyable) {
  if (dtype != DN_BF16 || !copyable || g.M > 16 || epi != kEpiLinear) return 1;
  const int cus = device_cu_count(), groups = (g.N + 31) / 32, chunks = g.K / 32;
  const double alone = double(g.K) * 64 / 28e3;
  int best = 1;
  double least = alone;
  for (int s = 2; s * groups <= cus && s * 2 * kFewWaves <= chunks; ++s) {
    const double cost = alone / s + 4.5;
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

int few_rows_most(GemmEpi epi) { return epi == kEpiGated ? 32 : epi == kEpiLinear ? 64 : 0; }

hipError_t few_rows(const GemmArgs& g, GemmEpi epi, int dtype, int out_dtype, bool copyable,
                    hipStream_t stream) {
  if (dtype == DN_BF16 && copyable && g.M <= 16) {
    if (epi == kEpiGated) return few_copy_launch<2, kEpiGated>(g, stream);
    if ((g.N + 63) / 64 < device_cu_count() / 2) return few_copy_launch<2, kEpiLinear>(g, stream);
    return few_copy_launch<4, kEpiLinear>(g, stream);
  }
  if (dtype == DN_BF16) return few_go<bf16, bf16>(g, epi, stream);
  if (dtype == DN_F32) return few_go<float, float>(g, epi, stream);
  return out_dtype == DN_BF16 ? few_go<f8, bf16>(g, epi, stream)
                              : few_go<f8, float>(g, epi, stream);
}

}  // namespace dn

// What the attention kernels share: blocks of the matrix unit for bf16 and fp32,
// tiles in LDS, and where a workgroup's rows lie.
//
// All products are formed so that the accumulators of one are the operand of the
// next. A block is E × E (E = 32 for bf16, 16 for fp32): its column is the lane's
// own (c = lane % E), its rows are spread over the lane's registers and the 64 / E
// lanes of that column (h = lane / E). With scores formed as K·Qᵀ a lane holds
// scores of one query, so a softmax needs one exchange a tile, and the weights
// enter Vᵀ·P as its second operand where they are: the contraction runs over keys
// in the order in which the registers hold them, and the other operand is read
// from LDS in that order (by transposing reads in bf16).
//
// A word is 16 bytes: 8 bf16 values or 4 fp32 ones. Operand fragments cover 16
// values of the contraction, one word a lane.
#pragma once

#include "dn_common.hpp"
#include "gemm.hpp"
#include "mfma_util.hpp"

namespace dn {
namespace attn {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

template <class T>
struct Mma;

template <>
struct Mma<bf16> {
  static constexpr int kE = 32, kAcc = 16, kCh = 8;
  using Acc = f32x16;
  // The row of register i within a block.
  static __device__ inline int row(int i, int h) { return (i & 3) + 8 * (i >> 2) + 4 * h; }
  static __device__ inline void mul(const uint4& a, const uint4& b, Acc& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  // Rows 16·s … of a column of blocks as an operand.
  template <int S, int N>
  static __device__ inline uint4 operand(const Acc (&x)[N]) {
    const Acc& a = x[S / 2];
    constexpr int o = 8 * (S & 1);
    return make_uint4(pk_bf16(a[o], a[o + 1]), pk_bf16(a[o + 2], a[o + 3]),
                      pk_bf16(a[o + 4], a[o + 5]), pk_bf16(a[o + 6], a[o + 7]));
  }
  // Places words of a row: 4 adjacent rows at one column (a transposing read) and 16
  // rows at one word (an operand's read) are spread over the banks.
  template <int HD>
  static __device__ inline int spread(int row) {
    return HD == 64 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3)
                    : ((row & 3) << 2) | ((row >> 2) & 3);
  }
  static __device__ inline bool finite(const uint4& w) {
    auto ok = [](uint32_t u) {
      return (u & 0x7f80u) != 0x7f80u && (u & 0x7f800000u) != 0x7f800000u;
    };
    return ok(w.x) && ok(w.y) && ok(w.z) && ok(w.w);
  }
};

template <>
struct Mma<float> {
  static constexpr int kE = 16, kAcc = 4, kCh = 4;
  using Acc = f32x4;
  static __device__ inline int row(int i, int h) { return 4 * h + i; }
  static __device__ inline void mul(const uint4& a, const uint4& b, Acc& c) {
    c = mfma_f32(__uint_as_float(a.x), __uint_as_float(b.x), c);
    c = mfma_f32(__uint_as_float(a.y), __uint_as_float(b.y), c);
    c = mfma_f32(__uint_as_float(a.z), __uint_as_float(b.z), c);
    c = mfma_f32(__uint_as_float(a.w), __uint_as_float(b.w), c);
  }
  template <int S, int N>
  static __device__ inline uint4 operand(const Acc (&x)[N]) {
    return __builtin_bit_cast(uint4, x[S]);
  }
  template <int HD>
  static __device__ inline int spread(int row) {
    return row & 15;
  }
  static __device__ inline bool finite(const uint4& w) {
    auto ok = [](uint32_t u) { return (u & 0x7f800000u) != 0x7f800000u; };
    return ok(w.x) && ok(w.y) && ok(w.z) && ok(w.w);
  }
};

// A tile of rows of HD values in LDS.
template <class T, int HD>
struct Tile {
  using M = Mma<T>;
  static constexpr int kWords = HD / M::kCh;  // of a row
  static __device__ inline int at(int row, int word) {
    return row * kWords + (word ^ M::template spread<HD>(row));
  }
  // Rows E·blk …, values 16·step … of them.
  static __device__ inline uint4 rows(const uint4* t, int blk, int step, int c, int h) {
    return t[at(blk * M::kE + c, step * (16 / M::kCh) + h)];
  }
  // Columns E·blk … as rows, contraction over rows 16·step … in the order of an
  // accumulator's registers.
  static __device__ inline uint4 cols(const uint4* t, int blk, int step, int lane) {
    if constexpr (sizeof(T) == 2) {
      // Lane i of a 16-lane group names four columns of row i / 4, and receives
      // column i of those four rows.
      const int i = lane & 15, g = lane >> 4;
      const int row = 16 * step + 4 * (g >> 1) + (i >> 2);
      const int col = 32 * blk + 16 * (g & 1) + 4 * (i & 3);
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) v4s* P;
      const char* p = reinterpret_cast<const char*>(t) + (col & 7) * 2;
      const uint2 lo = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 16 * at(row, col >> 3))));
      const uint2 hi = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 16 * at(row + 8, col >> 3))));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      const int c = lane & 15, h = lane >> 4, col = 16 * blk + c;
      auto one = [&](int r) {
        return reinterpret_cast<const uint32_t*>(t)[4 * at(16 * step + 4 * h + r, col >> 2) +
                                                    (col & 3)];
      };
      return make_uint4(one(0), one(1), one(2), one(3));
    }
  }
  static __device__ inline float value(const uint4* t, int row, int col) {
    return ld(reinterpret_cast<const T*>(t + at(row, col / M::kCh)), size_t(col % M::kCh));
  }
};

// Division of rows by the heads of a group: row r of a group's queries is head
// r % G of token r / G.
struct Group {
  int size;
  uint32_t mul, shift;
  __device__ inline int token(int r) const {
    return size == 1 ? r : int(__umulhi(uint32_t(r), mul) >> shift);
  }
};
// ceil(2^(31 + l) / G) with 2^l >= G: exact below 2^31.
inline Group group_of(int64_t size) {
  uint32_t l = 1;
  while ((int64_t(1) << l) < size) ++l;
  const uint64_t m = ((uint64_t(1) << (31 + l)) + uint64_t(size) - 1) / uint64_t(size);
  return {int(size), size == 1 ? 0 : uint32_t(m), l - 1};
}

// Rows of a tensor [token][head][dim] as a group's queries (G > 1) or as one key
// head's tokens (G = 1). `base` is the head's first value of the sequence's first
// token.
template <class T>
struct Rows {
  const T* base;
  int64_t ld;
  int dim;
  Group group;
  __device__ inline const T* at(int r) const {
    if (group.size == 1) return base + int64_t(r) * ld;
    const int t = group.token(r);
    return base + int64_t(t) * ld + int64_t(r - t * group.size) * dim;
  }
};

// A word of a row from value `col` on; values at dim and past it are zeros.
template <class T>
__device__ inline uint4 row_word(const T* row, int col, int dim) {
  constexpr int kCh = Mma<T>::kCh;
  uint4 w = make_uint4(0, 0, 0, 0);
  if (col + kCh <= dim) {
    __builtin_memcpy(&w, row + col, 16);
  } else if (col < dim) {
    T v[kCh] = {};
#pragma unroll
    for (int i = 0; i < kCh; ++i)
      if (col + i < dim) v[i] = row[col + i];
    __builtin_memcpy(&w, v, 16);
  }
  return w;
}

// ROWS rows on their way from memory to LDS through registers.
template <class T, int HD, int ROWS, int NT>
struct Stage {
  static constexpr int kWords = Tile<T, HD>::kWords, kN = ROWS * kWords / NT;
  static_assert(ROWS * kWords % NT == 0, "whole words a thread");
  uint4 w[kN];
  // Rows from `first` on, `there` (at least 1) of them; the others become zeros.
  __device__ inline void load(const Rows<T>& src, int first, int there) {
    if (src.dim == HD) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = i * NT + int(threadIdx.x), r = e / kWords;
        __builtin_memcpy(&w[i], src.at(first + min(r, there - 1)) + (e % kWords) * Mma<T>::kCh, 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = i * NT + int(threadIdx.x), r = e / kWords;
        w[i] = row_word(src.at(first + min(r, there - 1)), (e % kWords) * Mma<T>::kCh, src.dim);
      }
    }
  }
  __device__ inline void store(uint4* tile, int there) const {
    if (there >= ROWS) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = i * NT + int(threadIdx.x);
        tile[Tile<T, HD>::at(e / kWords, e % kWords)] = w[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = i * NT + int(threadIdx.x);
        tile[Tile<T, HD>::at(e / kWords, e % kWords)] =
            e / kWords < there ? w[i] : make_uint4(0, 0, 0, 0);
      }
    }
  }
  // Whether the rows that are there hold an infinity or a NaN.
  __device__ inline int wild(int there) const {
    int bad = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      bad |= (i * NT + int(threadIdx.x)) / kWords < there && !Mma<T>::finite(w[i]);
    return bad;
  }
};

// A tile whose rows do not all count for every column of a product, and that holds
// infinities or NaN: the matrix unit would carry them into columns that do not see
// them, as 0 · inf. Their rows' part of the columns that do see them (which are then
// not finite in any case) is added here, value by value, and the tile loses them.
// For whole workgroups; the tile may be used when it returns. `sees(row)`: whether
// the lane's column does.
template <class T, int HD, int ROWS, int NT, int NB, class Sees>
__device__ void set_apart(uint4* tile, typename Mma<T>::Acc (&acc)[NB], int h, Sees sees) {
  using M = Mma<T>;
  for (int r = 0; r < ROWS; ++r) {
    const bool on = sees(r);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < M::kAcc; ++i) {
        const float v = Tile<T, HD>::value(tile, r, b * M::kE + M::row(i, h));
        if (on && !(fabsf(v) < INFINITY)) acc[b][i] += v;
      }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ROWS * HD; e += NT) {
    const int at = Tile<T, HD>::at(e / HD, e % HD / M::kCh) * M::kCh + e % M::kCh;
    T* v = reinterpret_cast<T*>(tile);
    if (!(fabsf(ld(v, size_t(at))) < INFINITY)) st(v, size_t(at), 0.f);
  }
  __syncthreads();
}

// Where the sequences of a packed batch lie.
struct Spans {
  const int* offsets;      // [sequences + 1], or null: `each` rows a sequence
  const int *key_starts, *key_lengths;  // or null: a sequence's keys are its own rows
  int sequences, tokens, key_rows, each;
  // First row of sequence s; of `sequences`, the first behind the last. Never out
  // of [0, tokens], whatever the offsets are.
  __device__ inline int first(int s) const {
    if (s <= 0) return 0;
    if (s > sequences) return tokens;
    return offsets ? min(max(offsets[s], 0), tokens) : s * each;
  }
};
// A sequence's queries and keys.
struct Seq {
  int q0, len, k0, keys;
  int tile;  // of the sequence's own
};
// Tile t of rows (`per` a token, `edge` a tile) over all sequences, one after the
// other: sequence s starts at tile floor(first·per / edge) + s, which leaves room
// for a last tile that is not full. The rows behind the last sequence count as one
// without keys. False: no rows there.
__device__ inline bool find_tile(const Spans& sp, int t, int per, int edge, Seq* out) {
  const int lane = threadIdx.x & 63;
  // The last sequence that starts at t or before: 64 places at a time.
  int lo = 0, n = sp.sequences + 1;
  while (n > 1) {
    const int step = (n + 63) / 64, s = lo + lane * step;
    const bool before =
        s < lo + n && int64_t(sp.first(s)) * per / edge + s <= t;
    const int k = max(1, int(__popcll(__ballot(before))));
    const int end = min(lo + n, lo + k * step);
    lo += (k - 1) * step;
    n = step == 1 ? 1 : end - lo;
  }
  const int s = __builtin_amdgcn_readfirstlane(lo);
  const int q0 = sp.first(s), end = max(q0, sp.first(s + 1));
  out->q0 = q0;
  out->len = end - q0;
  out->tile = t - int(int64_t(q0) * per / edge) - s;
  if (s == sp.sequences) {
    out->k0 = out->keys = 0;
  } else if (sp.key_starts) {
    out->k0 = min(max(sp.key_starts[s], 0), sp.key_rows);
    out->keys = min(max(sp.key_lengths[s], 0), sp.key_rows - out->k0);
  } else {
    out->k0 = q0;
    out->keys = end - q0;
  }
  return out->tile >= 0 && int64_t(out->tile) * edge < int64_t(out->len) * per;
}
inline int64_t tile_count(int64_t tokens, int64_t per, int64_t edge, int64_t sequences) {
  return tokens * per / edge + sequences + 1;
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kNT = 256;  // threads of a workgroup: four waves

}  // namespace attn
}  // namespace dn

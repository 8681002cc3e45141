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

#include <initializer_list>

#include "dn_common.hpp"
#include "gemm.hpp"
#include "mfma_util.hpp"

namespace dn {
namespace attn {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kNT = 256;  // threads of a workgroup: four waves

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
  // Rows 16·half … of a block as an operand.
  static constexpr int kHalves = 2;
  static __device__ inline uint4 operand(const Acc& a, int half) {
    const int o = 8 * half;
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
  static constexpr int kHalves = 1;
  static __device__ inline uint4 operand(const Acc& a, int) { return __builtin_bit_cast(uint4, a); }
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

// Where a lane's operand words lie in a tile, in bytes: for a block's first words, the
// others being a constant further.
template <class T, int HD>
struct Reader {
  using M = Mma<T>;
  using TL = Tile<T, HD>;
  static constexpr int kSpan = TL::kWords < 16 ? TL::kWords : 16;  // words that `spread` mixes
  static constexpr int kStepWords = 16 / M::kCh, kSteps = kSpan / kStepWords;
  static constexpr int kBlkWords = M::kE / M::kCh, kBlks = kSpan / kBlkWords;
  static constexpr int kParts = sizeof(T) == 2 ? 2 : 4;
  static constexpr int kRow = TL::kWords * 16;
  uint32_t row[kSteps], col[kBlks][kParts];
  __device__ inline explicit Reader(int lane) {
    const int c = lane % M::kE, h = lane / M::kE;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) row[s] = TL::at(c, s * kStepWords + h) * 16;
#pragma unroll
    for (int b = 0; b < kBlks; ++b)
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        if constexpr (sizeof(T) == 2) {
          // Lane i of a 16-lane group names four columns of row i / 4, and receives
          // column i of those four rows.
          const int i = lane & 15, g = lane >> 4;
          const int r = 4 * (g >> 1) + 8 * j + (i >> 2), x = 32 * b + 16 * (g & 1) + 4 * (i & 3);
          col[b][j] = TL::at(r, x >> 3) * 16 + (x & 7) * 2;
        } else {
          const int x = 16 * b + c;
          col[b][j] = TL::at(4 * h + j, x >> 2) * 16 + (x & 3) * 4;
        }
      }
  }
  // Rows E·blk …, values 16·step … of them.
  __device__ inline uint4 rows(const char* t, int blk, int step) const {
    return *reinterpret_cast<const uint4*>(t + row[step % kSteps] + (step / kSteps) * kSpan * 16 +
                                           blk * M::kE * kRow);
  }
  // Columns E·blk … as rows, contraction over rows 16·step … in the order of an
  // accumulator's registers.
  __device__ inline uint4 cols(const char* t, int blk, int step) const {
    const int far = (blk / kBlks) * kSpan * 16 + step * 16 * kRow;
    if constexpr (sizeof(T) == 2) {
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) v4s* P;
      const uint2 lo = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(t + col[blk % kBlks][0] + far)));
      const uint2 hi = __builtin_bit_cast(
          uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(t + col[blk % kBlks][1] + far)));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      auto one = [&](int j) {
        return *reinterpret_cast<const uint32_t*>(t + col[blk % kBlks][j] + far);
      };
      return make_uint4(one(0), one(1), one(2), one(3));
    }
  }
};

__device__ inline uint32_t wave_index() {
  return uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
}
// A pointer that is the same in all lanes, in scalar registers.
__device__ inline const char* scalar(const char* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const char*>(
      uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(u >> 32)))) << 32 |
      uint32_t(__builtin_amdgcn_readfirstlane(int(u))));
}

// Tiles of ROWS rows on their way from memory to LDS. Copies need no registers: they
// are issued a tile ahead and waited for behind the products. They take whole words at
// 16-byte steps (`words`); rows that lie otherwise go through registers at once. Where
// a step of 16 rows is the same distance everywhere (`even`), a whole tile's addresses
// are a scalar base and an offset of the lane's own that stays.
template <class T, int HD, int ROWS>
struct Feed {
  using M = Mma<T>;
  using TL = Tile<T, HD>;
  static constexpr int kN = ROWS * TL::kWords / kNT;  // words of a thread
  static constexpr int kStep = kNT / TL::kWords;      // rows from one to the next
  static constexpr int kLong = kStep < 16 ? 16 : kStep, kD = kLong / kStep;
  static_assert(ROWS * TL::kWords % kNT == 0 && ROWS % kLong == 0, "whole words a thread");
  Rows<T> src;
  bool words, even;
  bool repeat;  // what stands for rows that are not there: the last one, or zeros
  int64_t far;  // bytes of kLong rows
  uint32_t off[kD];
  bool on[kD];
  __device__ inline Feed(const Rows<T>& rows, bool can_copy, bool repeat_last = false)
      : src(rows), words(can_copy), repeat(repeat_last) {
    const int g = src.group.size;
    even = 16 % g == 0;
    far = src.ld * int64_t(sizeof(T)) * (kLong / (even ? g : 1));
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      const int e = d * kNT + int(threadIdx.x), r = e / TL::kWords;
      const int word = (e % TL::kWords) ^ M::template spread<HD>(r);
      const int t = even ? src.group.token(r) : 0;
      off[d] = uint32_t(t) * uint32_t(src.ld * int64_t(sizeof(T))) +
               uint32_t((r - t * g) * src.dim * int(sizeof(T)) + word * 16);
      on[d] = word * M::kCh < src.dim;
    }
  }
  // Words past the rows' ends, which copies do not write.
  __device__ inline void clear_rest(uint4* tile) const {
    if (src.dim == HD) return;
    for (int e = threadIdx.x; e < ROWS * TL::kWords; e += kNT)
      if (((e % TL::kWords) ^ M::template spread<HD>(e / TL::kWords)) * M::kCh >= src.dim)
        tile[e] = make_uint4(0, 0, 0, 0);
  }
  // Rows from `first` (a multiple of ROWS) on, `there` (at least 1) of them.
  __device__ inline void load(uint4* tile, int first, int there) const {
    if (words && even && there >= ROWS) {
      const char* base = scalar(reinterpret_cast<const char*>(src.base) +
                                int64_t(first / kLong) * far);
      const uint32_t to = gemm::lds_address(tile) + wave_index() * 1024;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        if (src.dim == HD)
          gemm::copy_to_lds(base + (i / kD) * far, off[i % kD], to + i * kNT * 16);
        else if (on[i % kD])
          gemm::copy_to_lds(base + (i / kD) * far, off[i % kD], to + i * kNT * 16);
      }
    } else {
      load_any(tile, first, there);
    }
  }
  __device__ inline void load_any(uint4* tile, int first, int there) const {
    const uint32_t to = gemm::lds_address(tile) + wave_index() * 1024;
#pragma unroll 1
    for (int i = 0; i < kN; ++i) {
      const int e = i * kNT + int(threadIdx.x), r = e / TL::kWords;
      const int col = ((e % TL::kWords) ^ M::template spread<HD>(r)) * M::kCh;
      const T* row = src.at(first + min(r, there - 1));
      if ((r >= there && !repeat) || col >= src.dim) tile[e] = make_uint4(0, 0, 0, 0);
      else if (words) gemm::copy_to_lds(reinterpret_cast<const char*>(row + col), to + i * kNT * 16);
      else tile[e] = row_word(row, col, src.dim);
    }
  }
  // Whether a tile in LDS holds an infinity or a NaN.
  static __device__ inline int wild(const uint4* tile) {
    int bad = 0;
    for (int i = 0; i < kN; ++i) bad |= !M::finite(tile[i * kNT + int(threadIdx.x)]);
    return bad;
  }
};
// This wave's copies have landed and its LDS accesses are done; then all waves'.
__device__ inline void feed_barrier() {
  gemm::wait_copies<0>();
  lds_barrier();
}

// step(buffer, partly, n) for the tiles 0 … count − 1 of a walk, which take the two
// buffers in turn: the first `whole` are seen whole and the others in part.
template <class Step>
__device__ inline void walk(int whole, int count, Step step) {
  using A = std::integral_constant<int, 0>;
  using B = std::integral_constant<int, 1>;
  for (int n = 0; n < count; n += 2) {
    if (n < whole) step(A{}, std::false_type{}, n);
    else step(A{}, std::true_type{}, n);
    if (n + 1 >= count) break;
    if (n + 1 < whole) step(B{}, std::false_type{}, n + 1);
    else step(B{}, std::true_type{}, n + 1);
  }
}

// N products in order, with(i, word), the words read from LDS kAhead products ahead, and
// what `with` does beside its product kept there: a SIMD's vector unit works while its
// matrix unit does, but each wave hands out its instructions in order. Left to itself
// the compiler reads every word where it is used and gathers the rest behind.
template <int N, int kAhead, class Read, class With>
__device__ inline void in_turn(Read read, With with) {
  constexpr int kRing = kAhead + 1;
  uint4 ring[kRing];
  gemm::each<(kAhead < N ? kAhead : N)>([&](auto i) { ring[decltype(i)::value] = read(i); });
  gemm::each<N>([&](auto i) {
    constexpr int at = decltype(i)::value;
    if constexpr (at + kAhead < N)
      ring[(at + kAhead) % kRing] = read(std::integral_constant<int, at + kAhead>{});
    with(i, ring[at % kRing]);
    __builtin_amdgcn_sched_barrier(0);
  });
}
// f(e) for the part of [0, TOTAL) that falls to piece I of N.
template <int TOTAL, int N, int I, class F>
__device__ inline void share(F f) {
  constexpr int lo = TOTAL * I / N, hi = TOTAL * (I + 1) / N;
#pragma unroll
  for (int e = lo; e < hi; ++e) f(e);
}

// A value of the E lanes (h) of each column, over them.
template <int E, class F>
__device__ inline float over_column(float v, F f) {
  if constexpr (E == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// A tile whose rows do not all count for every column of a product, and that holds
// infinities or NaN: the matrix unit would carry them into columns that do not see
// them, as 0 · inf. Their rows' part of the columns that do see them (which are then
// not finite in any case) is added here, value by value, and the tile loses them.
// For whole workgroups; the tile may be used when it returns. `sees(row)`: whether
// the lane's column does. `weight` stands for theirs: 1 for a softmax's, which are above
// zero; 0 for dS of a key or query that is not finite, which is 0 or NaN.
template <class T, int HD, int ROWS, int NT, int NB, class Sees>
__device__ void set_apart(uint4* tile, typename Mma<T>::Acc (&acc)[NB], int h, float weight,
                          Sees sees) {
  using M = Mma<T>;
  for (int r = 0; r < ROWS; ++r) {
    const bool on = sees(r);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < M::kAcc; ++i) {
        const float v = Tile<T, HD>::value(tile, r, b * M::kE + M::row(i, h));
        if (on && !(fabsf(v) < INFINITY)) acc[b][i] += v * weight;
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
// Whether tensors' rows can be copied to LDS: heads of whole words, at 16-byte steps,
// with 32-bit offsets between rows of a tile.
struct Lying {
  const void* p;
  int64_t ld;
};
inline bool in_words(int dtype, int dim, std::initializer_list<Lying> tensors) {
  const int64_t size = dtype == DN_BF16 ? 2 : 4;
  if (dim * size % 16) return false;
  for (const Lying& t : tensors)
    if (reinterpret_cast<uintptr_t>(t.p) % 16 || t.ld * size % 16 || t.ld >= (1 << 23)) return false;
  return true;
}
inline int64_t tile_count(int64_t tokens, int64_t per, int64_t edge, int64_t sequences) {
  return tokens * per / edge + sequences + 1;
}


}  // namespace attn
}  // namespace dn

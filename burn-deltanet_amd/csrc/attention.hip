// dn_attention: out = softmax(scale · q kᵀ) v with grouped heads over packed
// sequences, causal or not, in one pass over the keys.
//
// A workgroup takes a tile of rows, a row being one head of one token, the heads
// of a group side by side: the group's keys are read once for all of them, and one
// token's heads fill a part of a tile. Its four waves have E rows each and walk the
// keys in tiles that are copied to LDS, the next tile in flight during the products of
// this one. Scores are K·Qᵀ, a lane holds scores of one row:
// the running maximum is its own, and the sums of its two (four) lanes meet at the
// end. The maximum is followed in steps: the sums are rescaled where it has grown by
// more than 2^8, which few tiles do after the first, and the weights are below 2^8
// then.
//
// Where there are few tiles of rows the keys are split too; parts meet in the
// workspace with their maxima and sums, and a second kernel adds them in order.
//
// Sums, statistics and scores are fp32; in bf16 the weights are rounded for the
// matrix unit (their sum is not), the output once.
//
// Bound by the matrix and the vector unit in turn, which two waves a SIMD overlap only in
// part. Measured, bf16, 16 heads on 4 of 128: one causal sequence of 16384 1.13 ms a call
// (0.97 PFLOP/s; 1.24 under the tracer); one token over 65536 keys 50 us and 13 for the
// join (2.7 TB/s), 64 over 2048 to 8192 each 182 us (3.8 TB/s: a CU has 64 KB of keys in
// flight). Through registers in place of copies the first took 1.45 ms. Heads of other
// widths are padded in LDS to 64, 128 or 256; widths that are no multiple of 16 bytes are
// read without copies, and the tile's loads are not hidden (2048 tokens of 33 values: 119
// us).
#include <algorithm>

#include "attention.hpp"
#include "layer.hpp"

namespace dn {
namespace {

using namespace attn;

struct FwdArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  float* part;      // [splits][rows][dim], null: not split
  float2* part_ml;  // [splits][rows] maximum (in powers of two) and sum
  Spans spans;
  Group group;
  int64_t ldq, ldk, ldv, ldo;
  int kv_heads, dim, causal, tiles, splits;
  bool words;  // keys and values lie in whole words
  float c;  // scale · log2(e)
};

constexpr float kGrowth = 8.f;

template <class T, int HD>
struct FwdShape {
  static constexpr int kBN = sizeof(T) == 2 ? 64 : 32;  // keys of a tile
  static constexpr int kBM = 4 * Mma<T>::kE;            // rows of a workgroup
  static constexpr int kTileWords = kBN * Tile<T, HD>::kWords;
};

template <class T, int HD>
__global__ __launch_bounds__(kNT, HD <= 128 ? 2 : 1) void attention_kernel(FwdArgs p) {
  using M = Mma<T>;
  using S = FwdShape<T, HD>;
  using Acc = typename M::Acc;
  constexpr int E = M::kE, BN = S::kBN, KB = BN / E, DB = HD / E, KS = HD / 16;
  __shared__ uint4 smem[4 * S::kTileWords];  // keys, values; of two tiles
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % E, h = lane / E;
  const int G = p.group.size, heads = G * p.kv_heads;
  // Heads are the fastest: a head's tiles go to few XCDs, which then share its keys
  // in their L2. The last tiles, which see the most keys, come first.
  const int head = int(blockIdx.x) % p.kv_heads;
  Seq seq;
  if (!find_tile(p.spans, p.tiles - 1 - int(blockIdx.x) / p.kv_heads, G, S::kBM, &seq)) return;
  const int rows = seq.len * G, r0 = seq.tile * S::kBM, shift = seq.keys - seq.len;
  // Keys that any row of the tile sees, and that all do.
  int some = seq.keys, all = seq.keys;
  if (p.causal) {
    some = min(seq.keys, max(0, p.group.token(min(rows, r0 + S::kBM) - 1) + shift + 1));
    all = min(seq.keys, max(0, p.group.token(r0) + shift + 1));
  }
  const int count = (some + BN - 1) / BN, per = (count + p.splits - 1) / p.splits;
  const int n0 = min(count, int(blockIdx.y) * per), n1 = min(count, n0 + per);

  const int r = r0 + wave * E + c;
  const bool active = r0 + wave * E < rows, mine = r < rows;  // active: the whole wave
  const int token = p.group.token(min(r, rows - 1));
  const int last = p.causal ? min(seq.keys - 1, token + shift) : seq.keys - 1;
  const int64_t at = int64_t(seq.q0 + token) * heads + head * G + (min(r, rows - 1) - token * G);
  const Feed<T, HD, BN> keys(
      Rows<T>{static_cast<const T*>(p.k) + int64_t(seq.k0) * p.ldk + int64_t(head) * p.dim, p.ldk,
              p.dim, Group{1, 0, 0}},
      p.words);
  const Feed<T, HD, BN> values(
      Rows<T>{static_cast<const T*>(p.v) + int64_t(seq.k0) * p.ldv + int64_t(head) * p.dim, p.ldv,
              p.dim, Group{1, 0, 0}},
      p.words);
  const Reader<T, HD> read(lane);
  auto load = [&](int n, int buf) {
    const int there = min(BN, seq.keys - n * BN);
    keys.load(smem + buf * 2 * S::kTileWords, n * BN, there);
    values.load(smem + (buf * 2 + 1) * S::kTileWords, n * BN, there);
  };
  if (n0 < n1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) keys.clear_rest(smem + i * S::kTileWords);
    load(n0, 0);
  }
  uint4 q[KS];
  {
    const T* row = static_cast<const T*>(p.q) + int64_t(seq.q0 + token) * p.ldq +
                   int64_t(head * G + (min(r, rows - 1) - token * G)) * p.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = row_word(row, s * 16 + h * M::kCh, p.dim);
  }
  Acc o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < M::kAcc; ++i) o[b][i] = 0.f;
  float top = -INFINITY, sum = 0.f;  // the maximum in powers of two
  feed_barrier();

  // Tile n in buffer `parity`; one that a row sees in part (`partly`), or whole.
  auto step = [&](auto parity, auto partly, int n) {
    constexpr int buf = decltype(parity)::value;
    constexpr bool kPartly = decltype(partly)::value;
    uint4* const value_tile = smem + (buf * 2 + 1) * S::kTileWords;
    const char* const tk = reinterpret_cast<const char*>(smem + buf * 2 * S::kTileWords);
    const char* const tv = reinterpret_cast<const char*>(value_tile);
    if constexpr (kPartly) {
      if (__syncthreads_or(Feed<T, HD, BN>::wild(value_tile)))
        set_apart<T, HD, BN, kNT, DB>(value_tile, o, h, 1.f,
                                      [&](int j) { return n * BN + j <= last; });
    }
    // At 256 values a head some operands come back from scratch memory, which waits for
    // every copy issued before: the copies go behind the scores.
    constexpr bool kLate = HD == 256;
    if (!kLate && n + 1 < n1) load(n + 1, buf ^ 1);
    if (active) {
      Acc s[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i) s[b][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int b = 0; b < KB; ++b) M::mul(read.rows(tk, b, k), q[k], s[b]);
      if (kLate && n + 1 < n1) load(n + 1, buf ^ 1);
      if constexpr (kPartly) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int i = 0; i < M::kAcc; ++i)
            s[b][i] = n * BN + b * E + M::row(i, h) <= last ? s[b][i] : -INFINITY;
      }
      float m = s[0][0];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i) m = fmaxf(m, s[b][i]);
      m = over_column<E>(m, [](float x, float y) { return fmaxf(x, y); }) * p.c;
      if (__any(m > top + kGrowth)) {
        const float now = fmaxf(top, m);
        // Not zero, which would make NaN of infinities that were set apart: 2^-126 of the
        // sums so far is nothing beside a weight of one.
        const float f = now == top ? 1.f : fmaxf(__builtin_amdgcn_exp2f(top - now), 0x1p-126f);
        top = now;
        sum *= f;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int i = 0; i < M::kAcc; ++i) o[b][i] *= f;
      }
      // No key seen yet: the scores are −inf, and so are these exponents.
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i) {
          s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], p.c, -base));
          sum += s[b][i];
        }
#pragma unroll
      for (int st = 0; st < BN / 16; ++st) {
        const uint4 w = M::operand(s[st / M::kHalves], st % M::kHalves);
#pragma unroll
        for (int b = 0; b < DB; ++b) M::mul(read.cols(tv, b, st), w, o[b]);
      }
    } else if (kLate && n + 1 < n1) {
      load(n + 1, buf ^ 1);
    }
    feed_barrier();
  };
  walk(all / BN - n0, n1 - n0,
       [&](auto parity, auto partly, int n) { step(parity, partly, n0 + n); });
  if (!active) return;
  sum = over_column<E>(sum, [](float x, float y) { return x + y; });
  if (!mine) return;
  if (p.part) {
    const int64_t all_rows = int64_t(p.spans.tokens) * heads, to = blockIdx.y * all_rows + at;
    if (h == 0) p.part_ml[to] = make_float2(top, sum);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < M::kAcc; ++i) {
        const int col = b * E + M::row(i, h);
        if (col < p.dim) p.part[to * p.dim + col] = o[b][i];
      }
    return;
  }
  // A row that sees no key: zeros, and a log-sum of −inf. NaN stays.
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  T* out = static_cast<T*>(p.out) + int64_t(seq.q0 + token) * p.ldo +
           int64_t(at - int64_t(seq.q0 + token) * heads) * p.dim;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < M::kAcc; i += 4) {
      const int col = b * E + M::row(i, h);
      if (col + 4 <= p.dim) {
        if constexpr (sizeof(T) == 2) {
          const uint2 w = make_uint2(pk_bf16(o[b][i] * inv, o[b][i + 1] * inv),
                                     pk_bf16(o[b][i + 2] * inv, o[b][i + 3] * inv));
          __builtin_memcpy(out + col, &w, 8);
        } else {
          const float4 w = make_float4(o[b][i] * inv, o[b][i + 1] * inv, o[b][i + 2] * inv,
                                       o[b][i + 3] * inv);
          __builtin_memcpy(out + col, &w, 16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < p.dim) st(out, size_t(col + j), o[b][i + j] * inv);
      }
    }
  if (p.lse && h == 0) p.lse[at] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) / kLog2E;
}

// The parts of a row: a workgroup a row, its waves taking every fourth part, two columns a
// lane; their sums meet in LDS.
constexpr int kMostSplits = 256;
template <class T>
__global__ __launch_bounds__(kNT) void attention_join_kernel(FwdArgs p) {
  __shared__ float weight[kMostSplits], part[4][128];
  const int heads = p.group.size * p.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rows = int64_t(p.spans.tokens) * heads, row = blockIdx.x;
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) top = fmaxf(top, p.part_ml[s * rows + row].x);
#pragma unroll
  for (int w = 32; w; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int s = lane; s < p.splits; s += 64) {
    const float2 ml = p.part_ml[s * rows + row];
    const float f = __builtin_amdgcn_exp2f(ml.x - base);
    sum += ml.y * f;
    if (wave == 0) weight[s] = f;
  }
#pragma unroll
  for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w);
  __syncthreads();
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int64_t token = row / heads;
  T* out = static_cast<T*>(p.out) + token * p.ldo + (row - token * heads) * p.dim;
  for (int c0 = 0; c0 < p.dim; c0 += 128) {
    const int col = c0 + 2 * lane;
    float2 v = make_float2(0.f, 0.f);
    if (col + 1 < p.dim) {
#pragma unroll 8
      for (int s = wave; s < p.splits; s += 4) {
        float2 x;
        __builtin_memcpy(&x, p.part + (s * rows + row) * p.dim + col, 8);
        v.x = fmaf(x.x, weight[s], v.x);
        v.y = fmaf(x.y, weight[s], v.y);
      }
    } else if (col < p.dim) {
      for (int s = wave; s < p.splits; s += 4)
        v.x = fmaf(p.part[(s * rows + row) * p.dim + col], weight[s], v.x);
    }
    part[wave][2 * lane] = v.x;
    part[wave][2 * lane + 1] = v.y;
    __syncthreads();
    const int c = threadIdx.x;
    if (c < 128 && c0 + c < p.dim)
      st(out, size_t(c0 + c), (part[0][c] + part[1][c] + part[2][c] + part[3][c]) * inv);
    __syncthreads();
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[row] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) / kLog2E;
}

int padded_dim(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
int64_t tile_rows(int dtype) {
  return 4 * (dtype == DN_BF16 ? Mma<bf16>::kE : Mma<float>::kE);
}

// Parts of the keys, of at least 256 keys each on average: as many as fill the CUs twice
// where the tiles of rows do not. (More, to even out sequences of different lengths, gain
// nothing: 64 requests of a token over 2048 to 8192 keys, 16 heads on 4 of 128, 183 us
// with twice the CUs' workgroups and 186 with eight times.)
int splits_of(const dn_attention_args& a) {
  const int64_t group = a.nheads / a.kv_heads;
  const int64_t tiles =
      std::max<int64_t>(a.sequences, a.tokens * group / tile_rows(a.dtype)) * a.kv_heads;
  const int64_t want = 2 * device_cu_count() / std::max<int64_t>(1, tiles);
  const int64_t keys = a.key_starts ? a.key_rows : a.tokens;
  const int64_t most = keys / std::max<int64_t>(1, a.sequences) / 256;
  return int(std::max<int64_t>(1, std::min<int64_t>({want, most, kMostSplits})));
}

template <class T, int HD>
hipError_t fwd_go(const FwdArgs& p, hipStream_t stream) {
  const auto fn = attention_kernel<T, HD>;
  {
    ProfScope ps("dn_attention", stream);
    hipLaunchKernelGGL(fn, dim3(unsigned(p.tiles) * unsigned(p.kv_heads), unsigned(p.splits)),
                       dim3(kNT), 0, stream, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.part) return e;
  ProfScope ps("dn_attention_join", stream);
  const int64_t rows = int64_t(p.spans.tokens) * p.group.size * p.kv_heads;
  hipLaunchKernelGGL((attention_join_kernel<T>), dim3(unsigned(rows)), dim3(kNT), 0, stream, p);
  return hipGetLastError();
}
template <class T>
hipError_t fwd_typed(const FwdArgs& p, hipStream_t stream) {
  const int hd = padded_dim(p.dim);
  return hd == 64    ? fwd_go<T, 64>(p, stream)
         : hd == 128 ? fwd_go<T, 128>(p, stream)
                     : fwd_go<T, 256>(p, stream);
}

}  // namespace

size_t attention_workspace(const dn_attention_args& a) {
  const size_t splits = size_t(splits_of(a)), rows = size_t(a.tokens) * size_t(a.nheads);
  if (splits == 1) return 0;
  return align_up(splits * rows * size_t(a.head_dim) * 4, 256) + splits * rows * sizeof(float2);
}

hipError_t launch_attention(const dn_attention_args& a, float scale, void* ws, hipStream_t stream) {
  FwdArgs p{};
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.out = a.out;
  p.lse = a.lse;
  p.group = group_of(a.nheads / a.kv_heads);
  p.spans = {a.offsets, a.key_starts, a.key_lengths, int(a.sequences), int(a.tokens),
             int(a.key_starts ? a.key_rows : a.tokens),
             int(a.sequences ? a.tokens / a.sequences : 0)};
  p.ldq = a.q_stride;
  p.ldk = a.k_stride;
  p.ldv = a.v_stride;
  p.ldo = a.out_stride;
  p.kv_heads = int(a.kv_heads);
  p.dim = int(a.head_dim);
  p.causal = a.causal;
  p.tiles = int(tile_count(a.tokens, p.group.size, tile_rows(a.dtype), a.sequences));
  p.splits = splits_of(a);
  p.c = scale * kLog2E;
  p.words = in_words(a.dtype, p.dim, {{a.k, p.ldk}, {a.v, p.ldv}});
  if (p.splits > 1) {
    const size_t rows = size_t(a.tokens) * size_t(a.nheads);
    p.part = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(
        static_cast<char*>(ws) + align_up(size_t(p.splits) * rows * size_t(a.head_dim) * 4, 256));
  }
  return a.dtype == DN_BF16 ? fwd_typed<bf16>(p, stream) : fwd_typed<float>(p, stream);
}

}  // namespace dn

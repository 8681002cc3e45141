// dn_attention_bwd: the gradients of dn_attention where a sequence's keys are its
// own rows. With P = exp(scale·q kᵀ − lse), dP = d_out vᵀ, δ = d_out · out of a row
// and dS = P ⊙ (dP − δ):
//   d_q = scale·dS k,  d_k = scale·dSᵀ q,  d_v = Pᵀ d_out.
//
// Three launches: δ (with lse beside it, the rows of a group side by side); d_q, a
// workgroup a tile of rows that walks the keys; d_k and d_v, a workgroup a tile of keys
// that walks the rows of all of its group's heads. So every gradient is summed by one
// workgroup in a fixed order, without atomics, and a group's shared heads need no sum of
// their own; the price is that S and dP are formed twice (seven products in place of
// five), and S a third time (eight) where d_k and d_v are apart. Every product leaves its
// sums where the next one takes them as an operand (attention.hpp).
//
// Sums are fp32; in bf16 the matrix unit takes P and dS rounded, δ is that of the rounded
// out, and the gradients are rounded once (they are 0.0025 from a 64-bit result in the
// norm, up to 0.0035 where sequences are short, and rounding the result alone gives 0.0017).
//
// Bound by the order in which a wave hands out its instructions: at 128 values a head two
// waves a SIMD keep the matrix unit at half of its rate. Measured, one causal sequence of
// 16384, 16 heads on 4 of 128, bf16, under the tracer: d_q 1.46 ms (1.1 PFLOP/s), d_k and
// d_v 2.73 ms (1.0 PFLOP/s with S formed twice), δ 27 us; a call of them 4.09 ms.
#include <algorithm>

#include "attention.hpp"
#include "layer.hpp"

namespace dn {
namespace {

using namespace attn;

struct BwdArgs {
  const void *q, *k, *v, *out, *d_out;
  const float* lse;
  void *d_q, *d_k, *d_v;
  float2* stats;  // [kv_heads][tokens · G]: −lse / scale, −δ: where S and dP start
  Spans spans;
  Group group;
  int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  int kv_heads, dim, causal, tiles;
  bool words;  // all operands lie in whole words
  float c, scale;
};

// δ and lse of every row: 16 lanes a row.
template <class T>
__global__ __launch_bounds__(kNT) void attention_stats_kernel(BwdArgs p) {
  const int heads = p.group.size * p.kv_heads, lane = threadIdx.x & 15;
  const int64_t row = int64_t(blockIdx.x) * (kNT / 16) + (threadIdx.x >> 4);
  if (row >= int64_t(p.spans.tokens) * heads) return;
  const int64_t token = row / heads;
  const int hd = int(row - token * heads), kv = hd / p.group.size;
  const T* o = static_cast<const T*>(p.out) + token * p.ldo + int64_t(hd) * p.dim;
  const T* d = static_cast<const T*>(p.d_out) + token * p.lddo + int64_t(hd) * p.dim;
  float t = 0.f;
  for (int col = lane * 8; col < p.dim; col += 128) {
    float a[8], b[8];
    gemm::load8(o + col, a, p.dim - col);
    gemm::load8(d + col, b, p.dim - col);
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fmaf(a[i], b[i], t);
  }
#pragma unroll
  for (int w = 8; w; w >>= 1) t += __shfl_xor(t, w);
  // A row without a score above −inf was given zeros: its weights are zeros here too.
  const float lse = p.lse[row];
  if (lane == 0)
    p.stats[(int64_t(kv) * p.spans.tokens + token) * p.group.size + (hd - kv * p.group.size)] =
        make_float2(lse == -INFINITY ? lse : -lse * kLog2E / p.c, -t);
}

template <class T, int HD>
struct BwdShape {
  static constexpr int kBN = sizeof(T) == 2 ? 64 : 32;  // rows of a tile that is walked
  static constexpr int kBM = 4 * Mma<T>::kE;            // rows, or keys, of a workgroup
  static constexpr int kTileWords = kBN * Tile<T, HD>::kWords;
  static constexpr bool kApart = (sizeof(T) == 2 && HD == 128) || HD == 256;  // d_k and d_v
  // For want of registers: one block of scores at a time; and the next tile's copies go
  // behind them, as operands that come back from scratch memory wait for every copy
  // issued before.
  static constexpr bool kLarge = HD == 256;
};

// A lane's row of a gradient: blocks of sums, a column of them the lane's own.
template <class T, int NB>
__device__ inline void store_row(T* to, const typename Mma<T>::Acc (&x)[NB], float f, int dim,
                                 int h) {
  using M = Mma<T>;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < M::kAcc; i += 4) {
      const int col = b * M::kE + M::row(i, h);
      if (col + 4 <= dim) {
        if constexpr (sizeof(T) == 2) {
          const uint2 w = make_uint2(pk_bf16(x[b][i] * f, x[b][i + 1] * f),
                                     pk_bf16(x[b][i + 2] * f, x[b][i + 3] * f));
          __builtin_memcpy(to + col, &w, 8);
        } else {
          const float4 w =
              make_float4(x[b][i] * f, x[b][i + 1] * f, x[b][i + 2] * f, x[b][i + 3] * f);
          __builtin_memcpy(to + col, &w, 16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < dim) st(to, size_t(col + j), x[b][i + j] * f);
      }
    }
}

template <class T, int HD>
__global__ __launch_bounds__(kNT, HD <= 128 ? 2 : 1) void attention_dq_kernel(BwdArgs p) {
  using M = Mma<T>;
  using S = BwdShape<T, HD>;
  using Acc = typename M::Acc;
  constexpr int E = M::kE, BN = S::kBN, KB = BN / E, DB = HD / E, KS = HD / 16;
  __shared__ uint4 smem[4 * S::kTileWords];  // keys, values; of two tiles
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % E, h = lane / E;
  const int G = p.group.size;
  const int head = int(blockIdx.x) % p.kv_heads;
  Seq seq;
  if (!find_tile(p.spans, p.tiles - 1 - int(blockIdx.x) / p.kv_heads, G, S::kBM, &seq)) return;
  const int rows = seq.len * G, r0 = seq.tile * S::kBM;
  int some = seq.keys, all = seq.keys;
  if (p.causal) {
    some = min(seq.keys, p.group.token(min(rows, r0 + S::kBM) - 1) + 1);
    all = min(seq.keys, p.group.token(r0) + 1);
  }
  const int count = (some + BN - 1) / BN;
  const int r = r0 + wave * E + c, rc = min(r, rows - 1);
  const bool active = r0 + wave * E < rows;
  const int token = p.group.token(rc), hd = head * G + (rc - token * G);
  const int last = p.causal ? min(seq.keys - 1, token) : seq.keys - 1;
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
  if (count > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) keys.clear_rest(smem + i * S::kTileWords);
    load(0, 0);
  }
  uint4 q[KS], d[KS];
  {
    const T* qr = static_cast<const T*>(p.q) + int64_t(seq.q0 + token) * p.ldq + int64_t(hd) * p.dim;
    const T* dr =
        static_cast<const T*>(p.d_out) + int64_t(seq.q0 + token) * p.lddo + int64_t(hd) * p.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[s] = row_word(qr, s * 16 + h * M::kCh, p.dim);
      d[s] = row_word(dr, s * 16 + h * M::kCh, p.dim);
    }
  }
  const float2 stat = p.stats[(int64_t(head) * p.spans.tokens + seq.q0) * G + rc];
  const float lse = stat.x * p.c, delta = stat.y;  // negative
  Acc dq[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < M::kAcc; ++i) dq[b][i] = 0.f;
  feed_barrier();

  auto step = [&](auto parity, auto partly, int n) {
    constexpr int buf = decltype(parity)::value;
    constexpr bool kPartly = decltype(partly)::value;
    uint4* const key_tile = smem + buf * 2 * S::kTileWords;
    const char* const tk = reinterpret_cast<const char*>(key_tile);
    const char* const tv = reinterpret_cast<const char*>(key_tile + S::kTileWords);
    if (!S::kLarge && n + 1 < count) load(n + 1, buf ^ 1);
    static_assert(KB == 2, "a block's exponentials stand beside the other's products");
    uint4 x[BN / 16];  // dS
    Acc s[KB], g[KB];
    auto scores = [&](auto block, auto beside) {
      constexpr int b = decltype(block)::value;
#pragma unroll
      for (int i = 0; i < M::kAcc; ++i) s[b][i] = g[b][i] = 0.f;
      in_turn<2 * KS, 3>(
          [&](auto i) { return read.rows(i % 2 ? tv : tk, b, i / 2); },
          [&](auto i, const uint4& w) {
            constexpr int at = decltype(i)::value;
            if constexpr (at % 2) M::mul(w, d[at / 2], g[b]);
            else M::mul(w, q[at / 2], s[b]);
            beside(i);
          });
    };
    auto weigh = [&](int b, int i) {
      float v = __builtin_amdgcn_exp2f(fmaf(s[b][i], p.c, lse)) * (g[b][i] + delta);
      if constexpr (kPartly) v = n * BN + b * E + M::row(i, h) <= last ? v : 0.f;
      s[b][i] = v;
    };
    auto weigh_all = [&](int b) {
#pragma unroll
      for (int i = 0; i < M::kAcc; ++i) weigh(b, i);
    };
    auto pack = [&](int b) {
#pragma unroll
      for (int u = 0; u < M::kHalves; ++u) x[b * M::kHalves + u] = M::operand(s[b], u);
    };
    constexpr int kProducts = M::kHalves * DB;
    auto gradient = [&](auto block, auto beside) {
      constexpr int b = decltype(block)::value;
      in_turn<kProducts, 3>(
          [&](auto i) { return read.cols(tk, i % DB, b * M::kHalves + i / DB); },
          [&](auto i, const uint4& w) {
            constexpr int at = decltype(i)::value;
            M::mul(w, x[b * M::kHalves + at / DB], dq[at % DB]);
            beside(i);
          });
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    const auto nothing = [](auto) {};
    if (active) {
      scores(B0{}, nothing);
      if constexpr (S::kLarge) weigh_all(0);
      scores(B1{}, [&](auto i) {
        if constexpr (!S::kLarge)
          share<M::kAcc, 2 * KS, decltype(i)::value>([&](int e) { weigh(0, e); });
      });
      pack(0);
      if constexpr (kPartly || S::kLarge) weigh_all(1);
    }
    if (S::kLarge && n + 1 < count) load(n + 1, buf ^ 1);
    if constexpr (kPartly) {
      if (__syncthreads_or(Feed<T, HD, BN>::wild(key_tile)))
        set_apart<T, HD, BN, kNT, DB>(key_tile, dq, h, 0.f,
                                      [&](int j) { return n * BN + j <= last; });
    }
    if (active) {
      gradient(B0{}, [&](auto i) {
        if constexpr (!kPartly && !S::kLarge)
          share<M::kAcc, kProducts, decltype(i)::value>([&](int e) { weigh(1, e); });
      });
      pack(1);
      gradient(B1{}, nothing);
    }
    feed_barrier();
  };
  walk(all / BN, count, step);
  if (r < rows)
    store_row<T, DB>(static_cast<T*>(p.d_q) + int64_t(seq.q0 + token) * p.lddq +
                         int64_t(hd) * p.dim, dq, p.scale, p.dim, h);
}

// d_k (DK) and d_v (DV) of a tile of keys. In bf16 from 65 values a head on their sums and
// operands together are more than the 256 registers of a lane with which a SIMD has two
// waves, so they are apart, with S formed for each: one wave hands out an instruction
// every five to eight cycles, too few to keep its matrix unit busy (8192 tokens in four
// sequences, 16 heads on 4 of 128: 607 us apart, 745 together by one wave).
template <class T, int HD, bool DK, bool DV>
__device__ inline void key_gradients(const BwdArgs& p, uint4* smem, float* stats, int block) {
  using M = Mma<T>;
  using S = BwdShape<T, HD>;
  using Acc = typename M::Acc;
  constexpr int E = M::kE, BN = S::kBN, KB = BN / E, DB = HD / E, KS = HD / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % E, h = lane / E;
  const int G = p.group.size;
  const int head = block % p.kv_heads;
  Seq seq;
  if (!find_tile(p.spans, block / p.kv_heads, 1, S::kBM, &seq)) return;
  const int rows = seq.keys ? seq.len * G : 0, j0 = seq.tile * S::kBM;
  const int j = j0 + wave * E + c, jc = min(j, seq.len - 1);
  const bool active = j0 + wave * E < seq.len;
  // Rows from `first` on see the lane's key; from `whole` on all of the tile's.
  const int first = p.causal ? jc * G : 0;
  const int whole = p.causal ? min(seq.len, j0 + S::kBM) * G - G : 0;
  const int b0 = p.causal ? j0 * G / BN : 0, count = (rows + BN - 1) / BN;
  // Rows that are not there start their scores at −inf. Zeros as their queries would make
  // that NaN for a key that is not finite; the last row's do so where that row, which sees
  // every key, has NaN of its own.
  const Feed<T, HD, BN> queries(
      Rows<T>{static_cast<const T*>(p.q) + int64_t(seq.q0) * p.ldq + int64_t(head) * G * p.dim,
              p.ldq, p.dim, p.group},
      p.words, true);
  const Feed<T, HD, BN> cotangents(
      Rows<T>{static_cast<const T*>(p.d_out) + int64_t(seq.q0) * p.lddo +
                  int64_t(head) * G * p.dim,
              p.lddo, p.dim, p.group},
      p.words);
  const float2* st = p.stats + (int64_t(head) * p.spans.tokens + seq.q0) * G;
  uint4 k[KS], v[DK ? KS : 1];
  {
    const T* kr = static_cast<const T*>(p.k) + int64_t(seq.q0 + jc) * p.ldk + int64_t(head) * p.dim;
    const T* vr = static_cast<const T*>(p.v) + int64_t(seq.q0 + jc) * p.ldv + int64_t(head) * p.dim;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      k[s] = row_word(kr, s * 16 + h * M::kCh, p.dim);
      if constexpr (DK) v[s] = row_word(vr, s * 16 + h * M::kCh, p.dim);
    }
  }
  Acc dk[DK ? DB : 1], dv[DV ? DB : 1];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < M::kAcc; ++i) {
      if constexpr (DK) dk[b][i] = 0.f;
      if constexpr (DV) dv[b][i] = 0.f;
    }
  const Reader<T, HD> read(lane);
  float2 ss;
  auto load = [&](int n, int buf) {
    const int there = min(BN, rows - n * BN);
    // Before the copies: what is written to a register in flight waits for all of them.
    // Rows that are not there have weights of zero.
    ss = make_float2(-INFINITY, 0.f);
    if (int(threadIdx.x) < there) ss = st[n * BN + threadIdx.x];
    queries.load(smem + buf * 2 * S::kTileWords, n * BN, there);
    cotangents.load(smem + (buf * 2 + 1) * S::kTileWords, n * BN, there);
  };
  auto keep_stats = [&](int buf) {
    if (threadIdx.x < BN) {
      stats[buf * 2 * BN + threadIdx.x] = ss.x;
      stats[(buf * 2 + 1) * BN + threadIdx.x] = ss.y;
    }
  };
  if (b0 < count) {
#pragma unroll
    for (int i = 0; i < 4; ++i) queries.clear_rest(smem + i * S::kTileWords);
    load(count - 1, 0);
    keep_stats(0);
  }
  feed_barrier();
  // From the last rows on: all workgroups of a head then read the same rows at the same
  // time, which meet in L2.
  auto step = [&](auto parity, auto partly, int n) {
    constexpr int buf = decltype(parity)::value;
    constexpr bool kPartly = decltype(partly)::value;
    uint4* const query_tile = smem + buf * 2 * S::kTileWords;
    const char* const tq = reinterpret_cast<const char*>(query_tile);
    const char* const td = reinterpret_cast<const char*>(query_tile + S::kTileWords);
    const float *start_s = stats + buf * 2 * BN, *start_g = start_s + BN;
    if (!S::kLarge && n > b0) load(n - 1, buf ^ 1);
    static_assert(KB == 2, "a block's exponentials stand beside the other's products");
    constexpr int kTerms = (DK ? 2 : 1) * KS, kAhead = DK && sizeof(T) == 2 && HD == 128 ? 1 : 3;
    uint4 x[DK ? BN / 16 : 1], w[DV ? BN / 16 : 1];  // dS, P
    Acc s[KB], g[KB];
    auto scores = [&](auto block, auto beside) {
      constexpr int b = decltype(block)::value;
#pragma unroll
      for (int i = 0; i < M::kAcc; i += 4) {
        const float4 ls = *reinterpret_cast<const float4*>(start_s + b * E + M::row(i, h));
        s[b][i] = ls.x;
        s[b][i + 1] = ls.y;
        s[b][i + 2] = ls.z;
        s[b][i + 3] = ls.w;
        if constexpr (DK) {
          const float4 de = *reinterpret_cast<const float4*>(start_g + b * E + M::row(i, h));
          g[b][i] = de.x;
          g[b][i + 1] = de.y;
          g[b][i + 2] = de.z;
          g[b][i + 3] = de.w;
        }
      }
      in_turn<kTerms, kAhead>(
          [&](auto i) {
            return DK ? read.rows(i % 2 ? td : tq, b, i / 2) : read.rows(tq, b, i);
          },
          [&](auto i, const uint4& w) {
            constexpr int at = decltype(i)::value;
            if constexpr (!DK) M::mul(w, k[at], s[b]);
            else if constexpr (at % 2) M::mul(w, v[at / 2], g[b]);
            else M::mul(w, k[at / 2], s[b]);
            beside(i);
          });
    };
    auto weigh = [&](int b, int i) {
      const bool on = !kPartly || n * BN + b * E + M::row(i, h) >= first;
      float t = __builtin_amdgcn_exp2f(s[b][i] * p.c);
      if constexpr (DK) {
        float u = on ? t * g[b][i] : 0.f;
        g[b][i] = u;
      }
      t = on ? t : 0.f;
      s[b][i] = t;
    };
    auto weigh_all = [&](int b) {
#pragma unroll
      for (int i = 0; i < M::kAcc; ++i) weigh(b, i);
    };
    auto pack = [&](int b) {
#pragma unroll
      for (int u = 0; u < M::kHalves; ++u) {
        if constexpr (DK) x[b * M::kHalves + u] = M::operand(g[b], u);
        if constexpr (DV) w[b * M::kHalves + u] = M::operand(s[b], u);
      }
    };
    constexpr int kBoth = DK + DV, kProducts = M::kHalves * DB * kBoth;
    auto gradient = [&](auto block, auto beside) {
      constexpr int b = decltype(block)::value;
      in_turn<kProducts, kAhead>(
          [&](auto i) {
            constexpr int at = decltype(i)::value, u = at / kBoth;
            return read.cols(DK && at % kBoth == 0 ? tq : td, u % DB, b * M::kHalves + u / DB);
          },
          [&](auto i, const uint4& a) {
            constexpr int at = decltype(i)::value, u = at / kBoth;
            if constexpr (DK && at % kBoth == 0) M::mul(a, x[b * M::kHalves + u / DB], dk[u % DB]);
            else M::mul(a, w[b * M::kHalves + u / DB], dv[u % DB]);
            beside(i);
          });
    };
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    const auto nothing = [](auto) {};
    if (active) {
      scores(B0{}, nothing);
      if constexpr (S::kLarge) weigh_all(0);
      scores(B1{}, [&](auto i) {
        if constexpr (!S::kLarge)
          share<M::kAcc, kTerms, decltype(i)::value>([&](int e) { weigh(0, e); });
      });
      pack(0);
      if constexpr (kPartly || S::kLarge) weigh_all(1);
    }
    if (S::kLarge && n > b0) load(n - 1, buf ^ 1);
    if constexpr (kPartly) {
      const int bad = (DK ? Feed<T, HD, BN>::wild(query_tile) : 0) |
                      (DV ? Feed<T, HD, BN>::wild(query_tile + S::kTileWords) : 0);
      if (__syncthreads_or(bad)) {
        const auto sees = [&](int i) { return n * BN + i >= first; };
        if constexpr (DK) set_apart<T, HD, BN, kNT, DB>(query_tile, dk, h, 0.f, sees);
        if constexpr (DV)
          set_apart<T, HD, BN, kNT, DB>(query_tile + S::kTileWords, dv, h, 1.f, sees);
      }
    }
    if (active) {
      gradient(B0{}, [&](auto i) {
        if constexpr (!kPartly && !S::kLarge)
          share<M::kAcc, kProducts, decltype(i)::value>([&](int e) { weigh(1, e); });
      });
      pack(1);
      gradient(B1{}, nothing);
    }
    if (n > b0) keep_stats(buf ^ 1);
    feed_barrier();
  };
  // Tiles from `whole` on are seen whole.
  walk(count - (p.causal ? (whole + BN - 1) / BN : 0), count - b0,
       [&](auto parity, auto partly, int i) { step(parity, partly, count - 1 - i); });
  if (j >= seq.len) return;
  if constexpr (DK)
    store_row<T, DB>(static_cast<T*>(p.d_k) + int64_t(seq.q0 + j) * p.lddk +
                         int64_t(head) * p.dim, dk, p.scale, p.dim, h);
  if constexpr (DV)
    store_row<T, DB>(static_cast<T*>(p.d_v) + int64_t(seq.q0 + j) * p.lddv +
                         int64_t(head) * p.dim, dv, 1.f, p.dim, h);
}
// Apart: d_k's workgroups (`first_v` of them) come before d_v's, and either may be left
// out. Together: first_v is negative.
template <class T, int HD>
__global__ __launch_bounds__(kNT, HD <= 128 ? 2 : 1) void attention_dkv_kernel(
    BwdArgs p, int first_v) {
  using S = BwdShape<T, HD>;
  __shared__ uint4 smem[4 * S::kTileWords];  // queries, d_out; of two tiles
  __shared__ __attribute__((aligned(16))) float stats[4 * S::kBN];
  const int block = int(blockIdx.x);
  if constexpr (!S::kApart) {
    if (first_v < 0) {
      key_gradients<T, HD, true, true>(p, smem, stats, block);
      return;
    }
  }
  if (block < first_v) key_gradients<T, HD, true, false>(p, smem, stats, block);
  else key_gradients<T, HD, false, true>(p, smem, stats, block - first_v);
}

template <class T, int HD>
hipError_t bwd_go(const BwdArgs& a, hipStream_t stream) {
  using S = BwdShape<T, HD>;
  BwdArgs p = a;
  const int64_t rows = int64_t(p.spans.tokens) * p.group.size * p.kv_heads;
  {
    ProfScope ps("dn_attention_stats", stream);
    hipLaunchKernelGGL((attention_stats_kernel<T>), dim3(unsigned((rows + 15) / 16)), dim3(kNT), 0,
                       stream, p);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.d_q) {
    const auto fn = attention_dq_kernel<T, HD>;
    p.tiles = int(tile_count(p.spans.tokens, p.group.size, S::kBM, p.spans.sequences));
    ProfScope ps("dn_attention_dq", stream);
    hipLaunchKernelGGL(fn, dim3(unsigned(p.tiles) * unsigned(p.kv_heads)), dim3(kNT), 0,
                       stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (!p.d_k && !p.d_v) return hipSuccess;
  p.tiles = int(tile_count(p.spans.tokens, 1, S::kBM, p.spans.sequences));
  const int blocks = p.tiles * p.kv_heads;
  ProfScope ps("dn_attention_dkv", stream);
  // Apart too where the tiles of keys are too few to fill the CUs twice (fp32, 1000 tokens,
  // 6 heads on 2 of 40, 38 tiles: forward and gradients 211 us apart, 235 together).
  const bool both = p.d_k && p.d_v, apart = S::kApart || blocks < 2 * device_cu_count();
  hipLaunchKernelGGL((attention_dkv_kernel<T, HD>), dim3(unsigned(both && apart ? 2 * blocks : blocks)),
                     dim3(kNT), 0, stream, p, both && !apart ? -1 : p.d_k ? blocks : 0);
  return hipGetLastError();
}
template <class T>
hipError_t bwd_typed(const BwdArgs& p, hipStream_t stream) {
  return p.dim <= 64    ? bwd_go<T, 64>(p, stream)
         : p.dim <= 128 ? bwd_go<T, 128>(p, stream)
                        : bwd_go<T, 256>(p, stream);
}

}  // namespace

size_t attention_bwd_workspace(const dn_attention_bwd_args& a) {
  return size_t(a.tokens) * size_t(a.nheads) * sizeof(float2);
}

hipError_t launch_attention_bwd(const dn_attention_bwd_args& a, float scale, void* ws,
                                hipStream_t stream) {
  BwdArgs p{};
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.out = a.out;
  p.d_out = a.d_out;
  p.lse = a.lse;
  p.d_q = a.d_q;
  p.d_k = a.d_k;
  p.d_v = a.d_v;
  p.stats = static_cast<float2*>(ws);
  p.spans = {a.offsets, nullptr, nullptr, int(a.sequences), int(a.tokens), int(a.tokens),
             int(a.sequences ? a.tokens / a.sequences : 0)};
  p.group = group_of(a.nheads / a.kv_heads);
  p.ldq = a.q_stride;
  p.ldk = a.k_stride;
  p.ldv = a.v_stride;
  p.ldo = a.out_stride;
  p.lddo = a.d_out_stride;
  p.lddq = a.d_q_stride;
  p.lddk = a.d_k_stride;
  p.lddv = a.d_v_stride;
  p.kv_heads = int(a.kv_heads);
  p.dim = int(a.head_dim);
  p.causal = a.causal;
  p.c = scale * kLog2E;
  p.scale = scale;
  p.words = in_words(a.dtype, p.dim, {{a.q, p.ldq}, {a.k, p.ldk}, {a.v, p.ldv}, {a.d_out, p.lddo}});
  return a.dtype == DN_BF16 ? bwd_typed<bf16>(p, stream) : bwd_typed<float>(p, stream);
}

}  // namespace dn

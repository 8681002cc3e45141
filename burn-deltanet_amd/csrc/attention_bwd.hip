// dn_attention_bwd: the gradients of dn_attention where a sequence's keys are its
// own rows. With P = exp(scale·q kᵀ − lse), dP = d_out vᵀ, δ = d_out · out of a row
// and dS = P ⊙ (dP − δ):
//   d_q = scale·dS k,  d_k = scale·dSᵀ q,  d_v = Pᵀ d_out.
//
// Three launches: δ (with lse in powers of two beside it, the rows of a group side by
// side); d_q, a workgroup a tile of rows that walks the keys; d_k and d_v, a workgroup
// a tile of keys that walks the rows of all of its group's heads. So every gradient
// is summed by one workgroup in a fixed order, without atomics, and a group's shared
// heads need no sum of their own; the price is that S and dP are formed twice (seven
// products in place of five). Every product leaves its sums where the next one takes
// them as an operand (attention.hpp).
//
// Sums are fp32; in bf16 the matrix unit takes P and dS rounded, the gradients are
// rounded once.
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
  float2* stats;  // [kv_heads][tokens · G]: lse · log2(e), δ
  Spans spans;
  Group group;
  int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  int kv_heads, dim, causal, tiles;
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
  if (lane == 0)
    p.stats[(int64_t(kv) * p.spans.tokens + token) * p.group.size + (hd - kv * p.group.size)] =
        make_float2(p.lse[row] * kLog2E, t);
}

template <class T, int HD>
struct BwdShape {
  static constexpr int kBN = sizeof(T) == 2 ? 64 : 32;  // rows of a tile that is walked
  static constexpr int kBM = 4 * Mma<T>::kE;            // rows, or keys, of a workgroup
  static constexpr int kTileWords = kBN * Tile<T, HD>::kWords;
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
  __shared__ uint4 smem[4 * S::kTileWords];
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
  const Rows<T> ks{static_cast<const T*>(p.k) + int64_t(seq.k0) * p.ldk + int64_t(head) * p.dim,
                   p.ldk, p.dim, Group{1, 0, 0}};
  const Rows<T> vs{static_cast<const T*>(p.v) + int64_t(seq.k0) * p.ldv + int64_t(head) * p.dim,
                   p.ldv, p.dim, Group{1, 0, 0}};
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
  Acc dq[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < M::kAcc; ++i) dq[b][i] = 0.f;

  Stage<T, HD, BN, kNT> sk, sv;
  auto tile_k = [&](int n) { return smem + (n & 1) * 2 * S::kTileWords; };
  auto tile_v = [&](int n) { return tile_k(n) + S::kTileWords; };
  auto partly = [&](int n) { return p.causal && (n + 1) * BN > all; };
  int wild = 0;
  if (count > 0) {
    const int there = min(BN, seq.keys);
    sk.load(ks, 0, there);
    sv.load(vs, 0, there);
    sk.store(tile_k(0), there);
    sv.store(tile_v(0), there);
    if (partly(0)) wild = __syncthreads_or(sk.wild(there));
    else __syncthreads();
  }
  for (int n = 0; n < count; ++n) {
    const int there = min(BN, seq.keys - (n + 1) * BN);
    if (n + 1 < count) {
      sk.load(ks, (n + 1) * BN, there);
      sv.load(vs, (n + 1) * BN, there);
    }
    const uint4 *tk = tile_k(n), *tv = tile_v(n);
    Acc x[KB];
    if (active) {
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        Acc s, g;
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i) s[i] = g[i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          M::mul(Tile<T, HD>::rows(tk, b, k, c, h), q[k], s);
          M::mul(Tile<T, HD>::rows(tv, b, k, c, h), d[k], g);
        }
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i)
          x[b][i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -stat.x)) * (g[i] - stat.y);
        if ((n + 1) * BN > all) {
#pragma unroll
          for (int i = 0; i < M::kAcc; ++i)
            x[b][i] = n * BN + b * E + M::row(i, h) <= last ? x[b][i] : 0.f;
        }
      }
    }
    if (wild)  // whole workgroups, after the keys' own products
      set_apart<T, HD, BN, kNT, DB>(tile_k(n), dq, h, [&](int j) { return n * BN + j <= last; });
    if (active)
      gemm::each<BN / 16>([&](auto step) {
        constexpr int st = decltype(step)::value;
        const uint4 w = M::template operand<st>(x);
#pragma unroll
        for (int b = 0; b < DB; ++b) M::mul(Tile<T, HD>::cols(tk, b, st, lane), w, dq[b]);
      });
    if (n + 1 < count) {
      sk.store(tile_k(n + 1), there);
      sv.store(tile_v(n + 1), there);
      if (partly(n + 1)) wild = __syncthreads_or(sk.wild(there));
      else __syncthreads();
    }
  }
  if (r < rows)
    store_row<T, DB>(static_cast<T*>(p.d_q) + int64_t(seq.q0 + token) * p.lddq +
                         int64_t(hd) * p.dim, dq, p.scale, p.dim, h);
}

// d_k (DK) and d_v (DV) of a tile of keys. At 256 values a head the sums and operands
// of both do not fit in registers, and they are launches of their own.
template <class T, int HD, bool DK, bool DV>
__global__ __launch_bounds__(kNT, 1) void attention_dkv_kernel(BwdArgs p) {
  using M = Mma<T>;
  using S = BwdShape<T, HD>;
  using Acc = typename M::Acc;
  constexpr int E = M::kE, BN = S::kBN, KB = BN / E, DB = HD / E, KS = HD / 16;
  __shared__ uint4 smem[4 * S::kTileWords];
  __shared__ float2 stats[2 * BN];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % E, h = lane / E;
  const int G = p.group.size;
  const int head = int(blockIdx.x) % p.kv_heads;
  Seq seq;
  if (!find_tile(p.spans, int(blockIdx.x) / p.kv_heads, 1, S::kBM, &seq)) return;
  const int rows = seq.keys ? seq.len * G : 0, j0 = seq.tile * S::kBM;
  const int j = j0 + wave * E + c, jc = min(j, seq.len - 1);
  const bool active = j0 + wave * E < seq.len;
  // Rows from `first` on see the lane's key; from `whole` on all of the tile's.
  const int first = p.causal ? jc * G : 0;
  const int whole = p.causal ? min(seq.len, j0 + S::kBM) * G - G : 0;
  const int b0 = p.causal ? j0 * G / BN : 0, count = (rows + BN - 1) / BN;
  const Rows<T> qs{static_cast<const T*>(p.q) + int64_t(seq.q0) * p.ldq +
                       int64_t(head) * G * p.dim, p.ldq, p.dim, p.group};
  const Rows<T> ds{static_cast<const T*>(p.d_out) + int64_t(seq.q0) * p.lddo +
                       int64_t(head) * G * p.dim, p.lddo, p.dim, p.group};
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
  for (int i = 0; i < M::kAcc; ++i) {
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      if constexpr (DK) dk[b][i] = 0.f;
      if constexpr (DV) dv[b][i] = 0.f;
    }
  }
  Stage<T, HD, BN, kNT> sq, sd;
  float2 ss;
  auto tile_q = [&](int n) { return smem + (n & 1) * 2 * S::kTileWords; };
  auto tile_d = [&](int n) { return tile_q(n) + S::kTileWords; };
  auto partly = [&](int n) { return p.causal && n * BN < whole; };
  int wild = 0;
  auto load = [&](int n) {
    const int there = min(BN, rows - n * BN);
    sq.load(qs, n * BN, there);
    sd.load(ds, n * BN, there);
    // Rows that are not there: weights of zero.
    ss = make_float2(INFINITY, 0.f);
    if (int(threadIdx.x) < there) ss = st[n * BN + threadIdx.x];
  };
  auto store = [&](int n) {
    const int there = min(BN, rows - n * BN);
    sq.store(tile_q(n), there);
    sd.store(tile_d(n), there);
    if (threadIdx.x < BN) stats[(n & 1) * BN + threadIdx.x] = ss;
    wild = 0;
    if (partly(n)) wild = __syncthreads_or((DK ? sq.wild(there) : 0) | (DV ? sd.wild(there) : 0));
    else __syncthreads();
  };
  if (b0 < count) {
    load(b0);
    store(b0);
  }
  for (int n = b0; n < count; ++n) {
    if (n + 1 < count) load(n + 1);
    const uint4 *tq = tile_q(n), *td = tile_d(n);
    const float2* sn = stats + (n & 1) * BN;
    Acc pr[KB], x[KB];
    if (active) {
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        Acc s, g;
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i) s[i] = g[i] = 0.f;
#pragma unroll
        for (int u = 0; u < KS; ++u) {
          M::mul(Tile<T, HD>::rows(tq, b, u, c, h), k[u], s);
          if constexpr (DK) M::mul(Tile<T, HD>::rows(td, b, u, c, h), v[u], g);
        }
#pragma unroll
        for (int i = 0; i < M::kAcc; ++i) {
          const float2 rs = sn[b * E + M::row(i, h)];
          const float w = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -rs.x));
          const bool on = !partly(n) || n * BN + b * E + M::row(i, h) >= first;
          pr[b][i] = on ? w : 0.f;
          if constexpr (DK) x[b][i] = on ? w * (g[i] - rs.y) : 0.f;
        }
      }
    }
    if (wild) {  // whole workgroups
      const auto sees = [&](int i) { return n * BN + i >= first; };
      if constexpr (DV) set_apart<T, HD, BN, kNT, DB>(tile_d(n), dv, h, sees);
      if constexpr (DK) set_apart<T, HD, BN, kNT, DB>(tile_q(n), dk, h, sees);
    }
    if (active)
      gemm::each<BN / 16>([&](auto step) {
        constexpr int u = decltype(step)::value;
        if constexpr (DV) {
          const uint4 w = M::template operand<u>(pr);
#pragma unroll
          for (int b = 0; b < DB; ++b) M::mul(Tile<T, HD>::cols(td, b, u, lane), w, dv[b]);
        }
        if constexpr (DK) {
          const uint4 w = M::template operand<u>(x);
#pragma unroll
          for (int b = 0; b < DB; ++b) M::mul(Tile<T, HD>::cols(tq, b, u, lane), w, dk[b]);
        }
      });
    if (n + 1 < count) store(n + 1);
  }
  if (j >= seq.len) return;
  if constexpr (DK)
    store_row<T, DB>(static_cast<T*>(p.d_k) + int64_t(seq.q0 + j) * p.lddk +
                         int64_t(head) * p.dim, dk, p.scale, p.dim, h);
  if constexpr (DV)
    store_row<T, DB>(static_cast<T*>(p.d_v) + int64_t(seq.q0 + j) * p.lddv +
                         int64_t(head) * p.dim, dv, 1.f, p.dim, h);
}

template <class T, int HD, bool DK, bool DV>
hipError_t dkv_go(BwdArgs p, hipStream_t stream) {
  using S = BwdShape<T, HD>;
  const auto fn = attention_dkv_kernel<T, HD, DK, DV>;
  p.tiles = int(tile_count(p.spans.tokens, 1, S::kBM, p.spans.sequences));
  ProfScope ps("dn_attention_dkv", stream);
  hipLaunchKernelGGL(fn, dim3(unsigned(p.tiles) * unsigned(p.kv_heads)), dim3(kNT), 0,
                     stream, p);
  return hipGetLastError();
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
  if constexpr (HD <= 128) {
    if (p.d_k && p.d_v) return dkv_go<T, HD, true, true>(p, stream);
  }
  if (p.d_k && (e = dkv_go<T, HD, true, false>(p, stream)) != hipSuccess) return e;
  return p.d_v ? dkv_go<T, HD, false, true>(p, stream) : hipSuccess;
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
  return a.dtype == DN_BF16 ? bwd_typed<bf16>(p, stream) : bwd_typed<float>(p, stream);
}

}  // namespace dn

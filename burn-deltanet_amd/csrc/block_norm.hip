// dn_block_norm: what stands between two blocks of a decoder in one pass. With
// x a block's output and r the residual stream,
//   u = x / sqrt(mean(x²) + ε) · γ_post    (without γ_post: u = x)
//   s = a·r + g ⊙ u                        (g a channel, a token, an element, or 1)
//   out = s / sqrt(mean(s²) + ε) · γ_pre
// dn_block_norm_bwd: its gradient at the s that was handed out, in one pass and a
// short sum. With n = x·inv_x, w = s·inv_s and d = d_out ⊙ γ_pre:
//   d_s = inv_s·(d − w·mean(d ⊙ w)) + d_sum,   d_r = a·d_s,   d_g = d_s ⊙ u
//   e = d_s ⊙ g ⊙ γ_post,   d_x = inv_x·(e − n·mean(e ⊙ n))
// and d_γ_pre = Σ d_out ⊙ w, d_γ_post = Σ d_s ⊙ g ⊙ n, d_g of a channel, over the rows.
//
// Bound by memory: x and r in, s and out out; x, s, d_out, d_sum in, d_x and d_r
// out. A row is held in registers between its reads and its writes, eight adjacent
// values to a lane and chunk, so that every byte moves once. Rows of up to 512
// values take one wave each, the others four that meet in LDS (once for each of the
// two chained means). The backward's workgroups walk rows with the next row's reads
// in flight, and keep the column sums of their rows in registers: a second kernel
// adds the workgroups' in order. Rows too long for registers are read again. In the
// backward a part of what rows of 4097 to 8192 values need goes to scratch memory: 20
// bytes a lane in bf16, 68 with fp32 weights, some 420 in fp32.
//
// Statistics, s before its rounding and all sums are fp32. As in add_rms_norm, the
// forward normalises the unrounded s and the backward starts from the stored one (whose
// rounding makes bf16 gradients 0.0024 off in the norm, where 0.0017 is their own).
//
// Measured, bf16: 32768 x 2048 with a gate a channel 101 us (5.3 TB/s, a copy's rate), its
// gradient 168 us (4.8 TB/s) and 8 for the column sums; one row 3.5 us. As many values in
// wider rows, calls of the forward and the gradient in TB/s: 4096 columns 5.5 and 3.3, 8192
// 5.0 and 3.6, 10000 3.4 and 1.5; in fp32 4.3 and 4.8, 4.1 and 2.0, 2.5 and 1.9.
#include <algorithm>

#include "gemm.hpp"
#include "layer.hpp"

namespace dn {
namespace {

using gemm::load8;
using gemm::Raw8;
using gemm::store8;

constexpr int kThreads = 256;
// Workgroups along x: a launch of 2^32 threads or more along an axis wraps.
constexpr int kMostGroups = 1 << 20;

struct FwdArgs {
  const void *x, *residual, *pre, *post, *gate;
  void *sum, *out;
  int64_t ldx, ldr, ldg, lds, ldo;
  int rows, dim, gate_kind;
  float eps, scale;
};

// Sums over a row's WPR waves; every lane receives them. `lds`: a place of its own
// for each use between two barriers.
template <int WPR, int N>
__device__ inline void row_sums(float (&v)[N], float (*lds)[4]) {
#pragma unroll
  for (int o = 32; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) lds[i][wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lds[i][0] + lds[i][1] + lds[i][2] + lds[i][3];
  }
}

// The gate's values at eight columns; a token's gate is read once a row (`token`).
template <class T, class TW>
__device__ inline void gate8(const void* gate, int kind, int64_t row_at, float token, int col,
                             int dim, float (&g)[8]) {
  if (kind == DN_GATE_CHANNEL) {
    load8(static_cast<const TW*>(gate) + min(col, dim), g, dim - col);
  } else if (kind == DN_GATE_FULL) {
    load8(static_cast<const T*>(gate) + row_at + min(col, dim), g, dim - col);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = token;
  }
}

template <class T, class TW, int WPR, int NCH>
__global__ __launch_bounds__(kThreads) void block_norm_kernel(FwdArgs p) {
  constexpr int kLanes = 64 * WPR;
  __shared__ float red[2][1][4];
  const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t group = int64_t(blockIdx.y) * kMostGroups + blockIdx.x;
  const int64_t row = WPR == 1 ? group * 4 + (threadIdx.x >> 6) : group;
  if (row >= p.rows) return;  // whole waves; with WPR = 4 whole workgroups
  const int dim = p.dim;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* res = static_cast<const T*>(p.residual) + row * p.ldr;
  const TW *pre = static_cast<const TW*>(p.pre), *post = static_cast<const TW*>(p.post);
  T* sum = static_cast<T*>(p.sum) + row * p.lds;
  T* out = static_cast<T*>(p.out) + row * p.ldo;
  const float token =
      p.gate_kind == DN_GATE_TOKEN ? ld(static_cast<const T*>(p.gate), size_t(row * p.ldg)) : 1.f;
  const int64_t gate_at = row * p.ldg;
  // s at eight columns from x's values there.
  auto joined = [&](int col, float (&v)[8], float inv_x, const float (&r)[8]) {
    if (post) {
      float w[8];
      load8(post + min(col, dim), w, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * inv_x * w[i];
    }
    if (p.gate_kind != DN_GATE_NONE) {
      float g[8];
      gate8<T, TW>(p.gate, p.gate_kind, gate_at, token, col, dim, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(p.scale, r[i], v[i]);
  };
  float ss[1] = {0.f}, inv_x = 1.f;
  if constexpr (NCH > 0) {
    Raw8<T> rx[NCH], rr[NCH];
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      rx[n].load(x + min(col, dim), dim - col);
      rr[n].load(res + min(col, dim), dim - col);
    }
    float v[NCH][8];
#pragma unroll
    for (int n = 0; n < NCH; ++n) rx[n].get(v[n]);
    if (post) {
#pragma unroll
      for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss[0] = fmaf(v[n][i], v[n][i], ss[0]);
      row_sums<WPR, 1>(ss, red[0]);
      inv_x = 1.0f / sqrtf(ss[0] / float(dim) + p.eps);
    }
    ss[0] = 0.f;
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      float r[8];
      rr[n].get(r);
      // Past dim x and r are zeros, and a token's gate or none leaves them so.
      joined(col, v[n], inv_x, r);
      if (col >= dim) continue;
      store8(sum + col, v[n], dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss[0] = fmaf(v[n][i], v[n][i], ss[0]);
    }
    row_sums<WPR, 1>(ss, red[1]);
    const float inv = 1.0f / sqrtf(ss[0] / float(dim) + p.eps);
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      if (col >= dim) continue;
      float w[8];
      load8(pre + col, w, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[n][i] = v[n][i] * inv * w[i];
      store8(out + col, v[n], dim - col);
    }
  } else {
    // s is formed again from x and r, so that the norm is the unrounded one's: `sum`
    // may alias either, and is written last.
    if (post) {
      for (int col = lane * 8; col < dim; col += kLanes * 8) {
        float v[8];
        load8(x + col, v, dim - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss[0] = fmaf(v[i], v[i], ss[0]);
      }
      row_sums<WPR, 1>(ss, red[0]);
      inv_x = 1.0f / sqrtf(ss[0] / float(dim) + p.eps);
    }
    auto again = [&](int col, float (&v)[8]) {
      float r[8];
      load8(x + col, v, dim - col);
      load8(res + col, r, dim - col);
      joined(col, v, inv_x, r);
    };
    ss[0] = 0.f;
    for (int col = lane * 8; col < dim; col += kLanes * 8) {
      float v[8];
      again(col, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss[0] = fmaf(v[i], v[i], ss[0]);
    }
    row_sums<WPR, 1>(ss, red[1]);
    const float inv = 1.0f / sqrtf(ss[0] / float(dim) + p.eps);
    for (int col = lane * 8; col < dim; col += kLanes * 8) {
      float v[8], w[8];
      again(col, v);
      store8(sum + col, v, dim - col);
      load8(pre + col, w, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
      store8(out + col, v, dim - col);
    }
  }
}

struct BwdArgs {
  const void *x, *sum, *pre, *post, *gate, *d_out, *d_sum;
  void *d_x, *d_residual, *d_gate;
  // Column sums [workgroups][kind][dim] of the kinds that are wanted: d_γ_pre,
  // d_γ_post, d_g a channel, each at its place or −1.
  float* cols;
  int at_pre, at_post, at_gate, kinds;
  float4* row;  // long rows: inv_s, c_s, inv_x of each, for the column kernel
  int64_t ldx, lds, ldg, ldo, ldd, ldx_out, ldr_out, ldg_out;
  int rows, dim, gate_kind;
  float eps, scale;
};

// What a row's gradient needs at eight columns.
template <class T>
struct RowWords {
  Raw8<T> x, s, d, e, g;  // x, s, d_out, d_sum, a full gate
};

template <class T, class TW, int WPR, int NCH>
__global__ __launch_bounds__(kThreads) void block_norm_bwd_kernel(BwdArgs p) {
  constexpr int kLanes = 64 * WPR, R = 4 / WPR, N = NCH > 0 ? NCH : 1;
  __shared__ float red[2][2][3][4];
  const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int wave = threadIdx.x >> 6, dim = p.dim;
  const float mean = 1.0f / float(dim);
  const TW *pre = static_cast<const TW*>(p.pre), *post = static_cast<const TW*>(p.post);
  const bool full = p.gate_kind == DN_GATE_FULL, token = p.gate_kind == DN_GATE_TOKEN;
  const int64_t step = int64_t(gridDim.x) * R;
  int64_t row = int64_t(blockIdx.x) * R + (WPR == 1 ? wave : 0);
  auto at = [&](const void* t, int64_t ld) { return static_cast<const T*>(t) + row * ld; };
  int turn = 0;
  if constexpr (NCH > 0) {
    float wpre[N][8], wpost[N][8], wgate[N][8], spre[N][8] = {}, spost[N][8] = {}, sgate[N][8] = {};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int col = (n * kLanes + lane) * 8;
      load8(pre + min(col, dim), wpre[n], dim - col);
      if (post) {
        load8(post + min(col, dim), wpost[n], dim - col);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) wpost[n][i] = 1.f;
      }
      if (p.gate_kind == DN_GATE_CHANNEL) {
        load8(static_cast<const TW*>(p.gate) + min(col, dim), wgate[n], dim - col);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) wgate[n][i] = 1.f;
      }
    }
    RowWords<T> next[N];
    float next_token = 1.f;
    auto fetch = [&](int64_t r) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int col = (n * kLanes + lane) * 8, c = min(col, dim), valid = dim - col;
        next[n].x.load(static_cast<const T*>(p.x) + r * p.ldx + c, valid);
        next[n].s.load(static_cast<const T*>(p.sum) + r * p.lds + c, valid);
        // A tensor that is absent is read as zeros.
        next[n].d.load(static_cast<const T*>(p.d_out) + (p.d_out ? r * p.ldo + c : 0),
                       p.d_out ? valid : 0);
        next[n].e.load(static_cast<const T*>(p.d_sum) + (p.d_sum ? r * p.ldd + c : 0),
                       p.d_sum ? valid : 0);
        if (full) next[n].g.load(static_cast<const T*>(p.gate) + r * p.ldg + c, valid);
      }
      if (token) next_token = ld(static_cast<const T*>(p.gate), size_t(r * p.ldg));
    };
    if (row < p.rows) fetch(row);
    for (; row < p.rows; row += step, turn ^= 1) {
      RowWords<T> now[N];
#pragma unroll
      for (int n = 0; n < N; ++n) now[n] = next[n];
      const float gt = next_token;
      if (row + step < p.rows) fetch(row + step);
      float x[N][8], s[N][8], ds[N][8];
      float t[3] = {};  // Σ x², Σ s², Σ d_out γ_pre s
#pragma unroll
      for (int n = 0; n < N; ++n) {
        now[n].x.get(x[n]);
        now[n].s.get(s[n]);
        float d[8];
        now[n].d.get(d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[0] = fmaf(x[n][i], x[n][i], t[0]);
          t[1] = fmaf(s[n][i], s[n][i], t[1]);
          t[2] = fmaf(d[i] * wpre[n][i], s[n][i], t[2]);
        }
      }
      row_sums<WPR, 3>(t, red[turn][0]);
      const float inv_x = post ? 1.0f / sqrtf(t[0] * mean + p.eps) : 1.f;
      const float inv_s = 1.0f / sqrtf(t[1] * mean + p.eps);
      const float c_s = t[2] * inv_s * inv_s * mean;
      float b[2] = {};  // Σ e ⊙ n, Σ d_s ⊙ u
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int col = (n * kLanes + lane) * 8;
        float d[8], e[8], g[8];
        now[n].d.get(d);
        now[n].e.get(e);
        if (full) {
          now[n].g.get(g);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = token ? gt : wgate[n][i];
        }
        float dg[8], dr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = inv_s * (d[i] * wpre[n][i] - s[n][i] * c_s) + e[i];
          spre[n][i] = fmaf(d[i], s[n][i] * inv_s, spre[n][i]);
          x[n][i] *= inv_x;  // n
          dg[i] = v * x[n][i] * wpost[n][i];
          sgate[n][i] += dg[i];
          dr[i] = v * p.scale;
          ds[n][i] = v * g[i];
          spost[n][i] = fmaf(ds[n][i], x[n][i], spost[n][i]);
          ds[n][i] *= wpost[n][i];
          b[0] = fmaf(ds[n][i], x[n][i], b[0]);
          b[1] += dg[i];
        }
        if (col < dim) {
          if (p.d_residual)
            store8(static_cast<T*>(p.d_residual) + row * p.ldr_out + col, dr, dim - col);
          if (full && p.d_gate)
            store8(static_cast<T*>(p.d_gate) + row * p.ldg_out + col, dg, dim - col);
        }
      }
      if (post || token) row_sums<WPR, 2>(b, red[turn][1]);
      if (token && p.d_gate && lane == 0)
        st(static_cast<T*>(p.d_gate), size_t(row * p.ldg_out), b[1]);
      if (!p.d_x) continue;
      const float c_x = post ? b[0] * mean : 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int col = (n * kLanes + lane) * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = inv_x * (ds[n][i] - x[n][i] * c_x);
        if (col < dim) store8(static_cast<T*>(p.d_x) + row * p.ldx_out + col, v, dim - col);
      }
    }
    if (!p.kinds) return;
    float* out = p.cols + int64_t(blockIdx.x) * p.kinds * dim;
    auto put = [&](int kind, const float (&v)[N][8]) {
      if (kind < 0) return;
      if constexpr (WPR == 1) {
        // The four waves' sums of each column meet in LDS, a chunk at a time.
        __shared__ float part[4][64 * 8];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 8; ++i) part[wave][i * 64 + lane] = v[n][i];
          __syncthreads();
          for (int e = threadIdx.x; e < 512; e += kThreads) {
            const int col = n * 512 + (e & 63) * 8 + (e >> 6);
            if (col < dim)
              out[int64_t(kind) * dim + col] = part[0][e] + part[1][e] + part[2][e] + part[3][e];
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int col = (n * kLanes + lane) * 8;
          if (col < dim) store8(out + int64_t(kind) * dim + col, v[n], dim - col);
        }
      }
    };
    put(p.at_pre, spre);
    put(p.at_post, spost);
    put(p.at_gate, sgate);
  } else {
    for (; row < p.rows; row += step, turn ^= 1) {
      const T *x = at(p.x, p.ldx), *s = at(p.sum, p.lds);
      const T* dy = p.d_out ? at(p.d_out, p.ldo) : nullptr;
      const T* de = p.d_sum ? at(p.d_sum, p.ldd) : nullptr;
      const float gt = token ? ld(static_cast<const T*>(p.gate), size_t(row * p.ldg)) : 1.f;
      float t[3] = {};
      for (int col = lane * 8; col < dim; col += kLanes * 8) {
        float vx[8], vs[8], vd[8] = {}, w[8];
        load8(x + col, vx, dim - col);
        load8(s + col, vs, dim - col);
        if (dy) load8(dy + col, vd, dim - col);
        load8(pre + col, w, dim - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[0] = fmaf(vx[i], vx[i], t[0]);
          t[1] = fmaf(vs[i], vs[i], t[1]);
          t[2] = fmaf(vd[i] * w[i], vs[i], t[2]);
        }
      }
      row_sums<WPR, 3>(t, red[turn][0]);
      const float inv_x = post ? 1.0f / sqrtf(t[0] * mean + p.eps) : 1.f;
      const float inv_s = 1.0f / sqrtf(t[1] * mean + p.eps);
      const float c_s = t[2] * inv_s * inv_s * mean;
      if (lane == 0 && p.row) p.row[row] = make_float4(inv_s, c_s, inv_x, 0.f);
      float b[2] = {};
      // n, e and the gate's gradient at eight columns; d_s in `ds`.
      auto terms = [&](int col, float (&n)[8], float (&e)[8], float (&dg)[8], float (&ds)[8]) {
        float vs[8], vd[8] = {}, ve[8] = {}, w[8], g[8];
        load8(x + col, n, dim - col);
        load8(s + col, vs, dim - col);
        if (dy) load8(dy + col, vd, dim - col);
        if (de) load8(de + col, ve, dim - col);
        load8(pre + col, w, dim - col);
        gate8<T, TW>(p.gate, p.gate_kind, row * p.ldg, gt, col, dim, g);
        float wp[8];
        if (post) {
          load8(post + col, wp, dim - col);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) wp[i] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ds[i] = inv_s * (vd[i] * w[i] - vs[i] * c_s) + ve[i];
          n[i] *= inv_x;
          dg[i] = ds[i] * n[i] * wp[i];
          e[i] = ds[i] * g[i] * wp[i];
        }
      };
      if (post || token) {
        for (int col = lane * 8; col < dim; col += kLanes * 8) {
          float n[8], e[8], dg[8], ds[8];
          terms(col, n, e, dg, ds);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            b[0] = fmaf(e[i], n[i], b[0]);
            b[1] += dg[i];
          }
        }
        row_sums<WPR, 2>(b, red[turn][1]);
      }
      if (token && p.d_gate && lane == 0)
        st(static_cast<T*>(p.d_gate), size_t(row * p.ldg_out), b[1]);
      const float c_x = post ? b[0] * mean : 0.f;
      for (int col = lane * 8; col < dim; col += kLanes * 8) {
        float n[8], e[8], dg[8], ds[8];
        terms(col, n, e, dg, ds);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n[i] = inv_x * (e[i] - n[i] * c_x);
          ds[i] *= p.scale;
        }
        if (p.d_x) store8(static_cast<T*>(p.d_x) + row * p.ldx_out + col, n, dim - col);
        if (p.d_residual)
          store8(static_cast<T*>(p.d_residual) + row * p.ldr_out + col, ds, dim - col);
        if (full && p.d_gate)
          store8(static_cast<T*>(p.d_gate) + row * p.ldg_out + col, dg, dim - col);
      }
    }
  }
}

// Long rows: the column sums over a strip of rows, a thread to a column.
template <class T, class TW>
__global__ __launch_bounds__(256) void block_norm_cols_kernel(BwdArgs p, int per) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.dim) return;
  const int64_t r0 = int64_t(blockIdx.y) * per, r1 = min(r0 + per, int64_t(p.rows));
  const float wpre = ld(static_cast<const TW*>(p.pre), size_t(c));
  const float wpost = p.post ? ld(static_cast<const TW*>(p.post), size_t(c)) : 1.f;
  float g = 1.f, spre = 0.f, spost = 0.f, sgate = 0.f;
  if (p.gate_kind == DN_GATE_CHANNEL) g = ld(static_cast<const TW*>(p.gate), size_t(c));
  for (int64_t r = r0; r < r1; ++r) {
    const float4 st = p.row[r];
    const float s = ld(static_cast<const T*>(p.sum), size_t(r * p.lds + c));
    const float n = ld(static_cast<const T*>(p.x), size_t(r * p.ldx + c)) * st.z;
    const float d = p.d_out ? ld(static_cast<const T*>(p.d_out), size_t(r * p.ldo + c)) : 0.f;
    const float e = p.d_sum ? ld(static_cast<const T*>(p.d_sum), size_t(r * p.ldd + c)) : 0.f;
    if (p.gate_kind >= DN_GATE_TOKEN)
      g = ld(static_cast<const T*>(p.gate),
             size_t(r * p.ldg + (p.gate_kind == DN_GATE_FULL ? c : 0)));
    const float ds = st.x * (d * wpre - s * st.y) + e;
    spre = fmaf(d, s * st.x, spre);
    sgate = fmaf(ds * n, wpost, sgate);
    spost = fmaf(ds * g, n, spost);
  }
  float* out = p.cols + int64_t(blockIdx.y) * p.kinds * p.dim + c;
  if (p.at_pre >= 0) out[int64_t(p.at_pre) * p.dim] = spre;
  if (p.at_post >= 0) out[int64_t(p.at_post) * p.dim] = spost;
  if (p.at_gate >= 0) out[int64_t(p.at_gate) * p.dim] = sgate;
}

// The workgroups' column sums added in order, 64 lanes of a column taking every
// 64th workgroup, their sums by halves.
constexpr int kSumCols = 16, kSumLanes = 64;
struct ColOuts {
  void* out[3];
};
template <class TW>
__global__ __launch_bounds__(kSumCols * kSumLanes) void block_norm_sum_kernel(
    const float* cols, ColOuts outs, int parts, int kinds, int dim) {
  __shared__ float lds[kSumLanes][kSumCols];
  const int x = threadIdx.x % kSumCols, l = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + x, kind = blockIdx.y;
  float t = 0.f;
  if (c < dim) {
#pragma unroll 4
    for (int i = l; i < parts; i += kSumLanes) t += cols[(int64_t(i) * kinds + kind) * dim + c];
  }
  lds[l][x] = t;
  __syncthreads();
#pragma unroll
  for (int half = kSumLanes / 2; half; half >>= 1) {
    if (l < half) lds[l][x] += lds[l + half][x];
    __syncthreads();
  }
  if (l == 0 && c < dim) st(static_cast<TW*>(outs.out[kind]), size_t(c), lds[0][x]);
}

// Waves to a row and chunks of eight values a lane (0: a long row).
struct Shape {
  int wpr, nch;
};
Shape shape_of(int64_t dim) {
  if (dim <= 512) return {1, 1};
  return {4, dim <= 2048 ? 1 : dim <= 4096 ? 2 : dim <= 8192 ? 4 : 0};
}

// Workgroups of the backward: each walks rows and leaves one set of column sums. As many
// as a CU has registers for at once (bf16 of up to 2048 values 152 to 166 a lane, fp32 up
// to 191, longer rows more than 256): others would walk their rows alone, behind the rest
// (32768 x 2048 in bf16: 218 us with four to a CU, 170 with three). bf16 of up to 512
// values with fp32 weights takes 174, of which two fit, not three: 48 us at 32768 x 512,
// 41 with weights in bf16.
int bwd_groups(int64_t rows, const Shape& s, int dtype) {
  const int64_t all = s.wpr == 1 ? (rows + 3) / 4 : rows;
  const int cu = s.nch == 0 ? 4 : s.nch > 1 ? 1 : dtype == DN_BF16 ? 3 : 2;
  return int(std::max<int64_t>(1, std::min<int64_t>(all, cu * device_cu_count())));
}
// Long rows: rows of a strip of the column kernel (a grid has at most 65535).
int strip_rows(int64_t rows) { return int(std::max<int64_t>(64, (rows + 32767) / 32768)); }
int strip_count(int64_t rows) {
  return int(std::max<int64_t>(1, (rows + strip_rows(rows) - 1) / strip_rows(rows)));
}
int kinds_of(const dn_block_norm_bwd_args& a) {
  return (a.d_pre_weight != nullptr) + (a.d_post_weight != nullptr) +
         (a.d_gate && a.gate_kind == DN_GATE_CHANNEL);
}

template <class T, class TW>
hipError_t fwd_go(const FwdArgs& p, hipStream_t stream) {
  const Shape s = shape_of(p.dim);
  const int64_t groups = s.wpr == 1 ? (int64_t(p.rows) + 3) / 4 : p.rows;
  const dim3 grid(unsigned(std::min<int64_t>(groups, kMostGroups)),
                  unsigned((groups + kMostGroups - 1) / kMostGroups));
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p);
  };
  if (s.wpr == 1) go(block_norm_kernel<T, TW, 1, 1>);
  else if (s.nch == 1) go(block_norm_kernel<T, TW, 4, 1>);
  else if (s.nch == 2) go(block_norm_kernel<T, TW, 4, 2>);
  else if (s.nch == 4) go(block_norm_kernel<T, TW, 4, 4>);
  else go(block_norm_kernel<T, TW, 4, 0>);
  return hipGetLastError();
}

template <class T, class TW>
hipError_t bwd_go(BwdArgs p, const ColOuts& outs, void* ws, hipStream_t stream) {
  const Shape s = shape_of(p.dim);
  int parts = bwd_groups(p.rows, s, sizeof(T) == 2 ? DN_BF16 : DN_F32);
  const dim3 grid{unsigned(parts)};
  const int strips = strip_count(p.rows);
  p.cols = static_cast<float*>(ws);
  if (p.kinds && s.nch == 0)
    p.row = reinterpret_cast<float4*>(
        static_cast<char*>(ws) + align_up(size_t(strips) * size_t(p.kinds) * size_t(p.dim) * 4, 256));
  {
    ProfScope ps("dn_block_norm_bwd", stream);
    const auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p);
    };
    if (s.wpr == 1) go(block_norm_bwd_kernel<T, TW, 1, 1>);
    else if (s.nch == 1) go(block_norm_bwd_kernel<T, TW, 4, 1>);
    else if (s.nch == 2) go(block_norm_bwd_kernel<T, TW, 4, 2>);
    else if (s.nch == 4) go(block_norm_bwd_kernel<T, TW, 4, 4>);
    else go(block_norm_bwd_kernel<T, TW, 4, 0>);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.kinds) return e;
  if (s.nch == 0) {
    ProfScope ps("dn_block_norm_cols", stream);
    hipLaunchKernelGGL((block_norm_cols_kernel<T, TW>),
                       dim3(unsigned((p.dim + 255) / 256), unsigned(strips)), dim3(256), 0, stream,
                       p, strip_rows(p.rows));
    if ((e = hipGetLastError()) != hipSuccess) return e;
    parts = strips;
  }
  ProfScope ps("dn_block_norm_sum", stream);
  hipLaunchKernelGGL((block_norm_sum_kernel<TW>),
                     dim3(unsigned((p.dim + kSumCols - 1) / kSumCols), unsigned(p.kinds)),
                     dim3(kSumCols * kSumLanes), 0, stream, static_cast<const float*>(p.cols), outs,
                     parts, p.kinds, p.dim);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_norm(const dn_block_norm_args& a, hipStream_t stream) {
  FwdArgs p{};
  p.x = a.x;
  p.residual = a.residual;
  p.pre = a.pre_weight;
  p.post = a.post_weight;
  p.gate = a.gate;
  p.sum = a.sum;
  p.out = a.out;
  p.ldx = a.x_stride;
  p.ldr = a.residual_stride;
  p.ldg = a.gate_stride;
  p.lds = a.sum_stride;
  p.ldo = a.out_stride;
  p.rows = int(a.rows);
  p.dim = int(a.dim);
  p.gate_kind = a.gate_kind;
  p.eps = float(a.eps);
  p.scale = float(a.residual_scale);
  ProfScope ps("dn_block_norm", stream);
  const bool wb = a.weight_dtype == DN_BF16;
  if (a.dtype == DN_BF16) return wb ? fwd_go<bf16, bf16>(p, stream) : fwd_go<bf16, float>(p, stream);
  return wb ? fwd_go<float, bf16>(p, stream) : fwd_go<float, float>(p, stream);
}

size_t block_norm_bwd_workspace(const dn_block_norm_bwd_args& a) {
  const size_t kinds = size_t(kinds_of(a));
  if (!kinds) return 0;
  const Shape s = shape_of(a.dim);
  if (s.nch > 0) return size_t(bwd_groups(a.rows, s, a.dtype)) * kinds * size_t(a.dim) * 4;
  const size_t strips = size_t(strip_count(a.rows));
  return align_up(strips * kinds * size_t(a.dim) * 4, 256) + size_t(a.rows) * sizeof(float4);
}

hipError_t launch_block_norm_bwd(const dn_block_norm_bwd_args& a, void* ws, hipStream_t stream) {
  BwdArgs p{};
  p.x = a.x;
  p.sum = a.sum;
  p.pre = a.pre_weight;
  p.post = a.post_weight;
  p.gate = a.gate;
  p.d_out = a.d_out;
  p.d_sum = a.d_sum;
  p.d_x = a.d_x;
  p.d_residual = a.d_residual;
  p.d_gate = a.d_gate;
  p.ldx = a.x_stride;
  p.lds = a.sum_stride;
  p.ldg = a.gate_stride;
  p.ldo = a.d_out_stride;
  p.ldd = a.d_sum_stride;
  p.ldx_out = a.d_x_stride;
  p.ldr_out = a.d_residual_stride;
  p.ldg_out = a.d_gate_stride;
  p.rows = int(a.rows);
  p.dim = int(a.dim);
  p.gate_kind = a.gate_kind;
  p.eps = float(a.eps);
  p.scale = float(a.residual_scale);
  ColOuts outs{};
  const auto want = [&](void* to) {
    if (!to) return -1;
    outs.out[p.kinds] = to;
    return p.kinds++;
  };
  p.at_pre = want(a.d_pre_weight);
  p.at_post = want(a.d_post_weight);
  p.at_gate = want(a.gate_kind == DN_GATE_CHANNEL ? a.d_gate : nullptr);
  const bool wb = a.weight_dtype == DN_BF16;
  if (a.dtype == DN_BF16)
    return wb ? bwd_go<bf16, bf16>(p, outs, ws, stream) : bwd_go<bf16, float>(p, outs, ws, stream);
  return wb ? bwd_go<float, bf16>(p, outs, ws, stream) : bwd_go<float, float>(p, outs, ws, stream);
}

}  // namespace dn

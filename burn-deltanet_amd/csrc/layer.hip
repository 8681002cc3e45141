// Plans and launches of dn_linear, dn_linear_bwd, dn_gated_ffn and
// dn_gated_ffn_bwd over the tile kernel (gemm.hpp).
//
// Forward: one product with its epilogue (linear); both input projections, the
// activation and their product in one kernel, then the down projection with
// the residual (feed-forward). Backward of the feed-forward: d_out·W_downᵀ,
// whose epilogue turns d_h into d_gate, d_up and h where it forms it; then d_x
// as one product whose contraction runs over W_gate's columns and W_up's; then
// the weights' gradients, xᵀ·d_gate and xᵀ·d_up in one launch.
//
// Where the tiles of a product are too few to fill the CUs, workgroups also
// split the contraction; their fp32 sums meet in the workspace and a second
// kernel adds them in order and runs the epilogue (no atomics: the results do
// not depend on the order of arrival).
#include <algorithm>

#include "layer.hpp"

namespace dn {
namespace {

constexpr int kJoinThreads = 256;

// Adds the partial sums of a split product, in order, and runs its epilogue.
// A thread owns eight adjacent columns of a row.
template <class TO, int EPI>
__global__ __launch_bounds__(kJoinThreads) void gemm_join_kernel(GemmArgs p) {
  const int groups = (p.N + 7) / 8;
  const int64_t n = int64_t(p.M) * groups * p.npair;
  const int64_t i = int64_t(blockIdx.x) * kJoinThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t zr = i / groups;
  const int col = int(i - zr * groups) * 8, z = int(zr / p.M);
  const int64_t row = zr - int64_t(z) * p.M;
  const int valid = p.N - col;
  const int64_t hop = int64_t(p.npair) * p.M * p.ldpart;
  const float* at = p.partial + (int64_t(z) * p.M + row) * p.ldpart + col;
  float v[8] = {}, u[8] = {};
  for (int sp = 0; sp < p.split; ++sp, at += hop) {
    float w[8];
    gemm::load8(at, w, valid);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
    if constexpr (EPI == kEpiGated) {
      gemm::load8(at + p.N, w, valid);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] += w[e];
    }
  }
  if constexpr (EPI == kEpiLinear) gemm::linear_tail<TO>(p, z, row, col, v);
  else if constexpr (EPI == kEpiGated) gemm::gated_tail<TO>(p, row, col, v, u);
  else gemm::dgated_tail<TO>(p, row, col, v);
}

// d_z = d_out·act'(z) and the column sums of d_z, over a strip of rows: a
// thread owns eight columns and every eighth row, the eight row lanes meet in
// LDS, and the strip's sums go to sums[strip][N].
struct ActBwdArgs {
  const void* d_out;
  const void* z;      // null: the identity, d_z is d_out
  void* dz;           // null: not written
  float* sums;        // null: not formed
  int64_t ldd, ldz, lddz;
  int M, N, rows_per, act;
};
template <class T>
__global__ __launch_bounds__(256) void act_bwd_kernel(ActBwdArgs p) {
  const int c8 = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + c8) * 8, valid = p.N - col;
  const int64_t r0 = int64_t(blockIdx.y) * p.rows_per;
  const int64_t r1 = min(r0 + p.rows_per, int64_t(p.M));
  float sum[8] = {};
  if (valid > 0) {
    for (int64_t r = r0 + lane; r < r1; r += 8) {
      float d[8];
      gemm::load8(static_cast<const T*>(p.d_out) + r * p.ldd + col, d, valid);
      if (p.z) {
        float z[8];
        gemm::load8(static_cast<const T*>(p.z) + r * p.ldz + col, z, valid);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= gemm::act_slope(z[i], p.act);
      }
      if (p.dz) gemm::store8(static_cast<T*>(p.dz) + r * p.lddz + col, d, valid);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += d[i];
    }
  }
  if (!p.sums) return;
  __shared__ float lds[8][32 * 8 + 8];
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[lane][c8 * 8 + i] = sum[i];
  __syncthreads();
  const int c = int(blockIdx.x) * 256 + threadIdx.x;
  if (c >= p.N) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) t += lds[i][threadIdx.x];
  p.sums[int64_t(blockIdx.y) * p.N + c] = t;
}

template <class T>
__global__ __launch_bounds__(256) void strip_sum_kernel(const float* sums, T* out, int strips,
                                                        int n) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float t = 0.f;
  for (int i = 0; i < strips; ++i) t += sums[int64_t(i) * n + c];
  st(out, size_t(c), t);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t elem_size(int dtype) { return dtype == DN_F32 ? 4 : dtype == DN_BF16 ? 2 : 1; }
bool at16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How one product is cut into workgroups.
struct Plan {
  GemmTile tile;
  int tiles_m, tiles_n, ktiles, split, per_split;
  size_t partial_bytes;
};

Plan plan_product(int64_t M, int64_t N, int64_t K, int nseg, int npair, int dtype, bool gated) {
  const int kt = int(128 / elem_size(dtype));
  Plan best{};
  double best_cost = 0;
  for (int big = 0; big < 2; ++big) {
    Plan p{};
    const int b = big ? 256 : 128;
    p.tile = big ? kTile256 : kTile128;
    p.tiles_m = int(ceil_div(M, b));
    p.tiles_n = int(ceil_div(N, gated ? b / 2 : b));
    p.ktiles = int(ceil_div(K, kt));
    const int64_t ksteps = std::max<int64_t>(1, int64_t(p.ktiles) * nseg);
    const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n * npair;
    const int slots = device_cu_count() * (big ? 1 : 2);
    const double unit = big ? 1.0 : 0.56;  // a k tile's time on a full machine
    const int most = int(std::min<int64_t>(std::max<int64_t>(1, ksteps / 4), 64));
    for (int s = 1; s <= most; s = s < 4 ? s + 1 : s + s / 4) {
      const int64_t per = ceil_div(ksteps, s);
      const int split = int(ceil_div(ksteps, per));
      if (tiles * split > (int64_t(1) << 30)) break;
      const double rounds = double(ceil_div(tiles * split, slots));
      double cost = rounds * (double(per) + 6.0) * unit;
      if (split > 1)  // partial sums out and in, at a CU's share of the memory's rate
        cost += 8.0 + double(M) * N * (gated ? 2 : 1) * npair * split * 8.0 / 4.0e6;
      if (best.split == 0 || cost < best_cost) {
        best_cost = cost;
        p.split = split;
        p.per_split = int(per);
        best = p;
      }
      if (s > 1 && tiles * s >= 4 * int64_t(slots)) break;
    }
  }
  if (best.split > 1)
    best.partial_bytes = align_up(size_t(best.split) * npair * size_t(M) *
                                      size_t(gated ? 2 * N : align_up(size_t(N), 4)) * 4, 256);
  return best;
}

void apply(GemmArgs& g, const Plan& p, bool gated, float* partial) {
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.ktiles = p.ktiles;
  g.split = p.split;
  g.per_split = p.per_split;
  g.partial = p.split > 1 ? partial : nullptr;
  g.ldpart = gated ? 2 * int64_t(g.N) : int64_t(align_up(size_t(g.N), 4));
}

// Whether every operand row lies at 16-byte steps and holds whole words.
bool copyable(const GemmArgs& g, GemmForm form, int dtype, bool second) {
  const int64_t ch = int64_t(16 / elem_size(dtype));
  const bool acol = form == kFormTN, bcol = form != kFormNT;
  bool ok = at16(g.a[0]) && at16(g.b[0]) && g.lda % 16 == 0 && g.ldb % 16 == 0;
  if (second) ok = ok && at16(g.b[1]) && (g.nseg == 1 || at16(g.a[1]));
  if (acol) ok = ok && g.M % ch == 0;
  if (bcol) ok = ok && g.N % ch == 0;
  if (!acol || !bcol) ok = ok && g.K % ch == 0;
  return ok;
}

template <class TO>
hipError_t join_typed(const GemmArgs& g, GemmEpi epi, hipStream_t stream) {
  const int64_t n = int64_t(g.M) * ((g.N + 7) / 8) * g.npair;
  const dim3 grid(unsigned(ceil_div(n, kJoinThreads)));
  if (epi == kEpiLinear)
    hipLaunchKernelGGL((gemm_join_kernel<TO, kEpiLinear>), grid, dim3(kJoinThreads), 0, stream, g);
  else if (epi == kEpiGated)
    hipLaunchKernelGGL((gemm_join_kernel<TO, kEpiGated>), grid, dim3(kJoinThreads), 0, stream, g);
  else
    hipLaunchKernelGGL((gemm_join_kernel<TO, kEpiDGated>), grid, dim3(kJoinThreads), 0, stream, g);
  return hipGetLastError();
}

hipError_t run_product(GemmArgs& g, GemmForm form, GemmEpi epi, int dtype, int out_dtype,
                       const Plan& plan, float* partial, const char* name, hipStream_t stream) {
  const bool gated = epi == kEpiGated;
  apply(g, plan, gated, partial);
  const bool staged = !copyable(g, form, dtype, g.nseg == 2 || g.npair == 2 || gated);
  hipError_t e;
  {
    ProfScope ps(name, stream);
    if (dtype == DN_F8) e = gemm_f8(g, out_dtype, plan.tile, stream);
    else if (dtype == DN_BF16) e = gemm_bf16(g, form, epi, plan.tile, staged, stream);
    else e = gemm_f32(g, form, epi, plan.tile, staged, stream);
  }
  if (e != hipSuccess || plan.split == 1) return e;
  ProfScope ps("dn_product_join", stream);
  return out_dtype == DN_BF16 ? join_typed<bf16>(g, epi, stream)
                              : join_typed<float>(g, epi, stream);
}

// --- act' and the bias' gradient -------------------------------------------------

struct Strips {
  int rows_per, count;
};
// Strips of rows: enough workgroups to fill the CUs, at least 32 rows each.
Strips strips_of(int64_t M, int64_t N) {
  const int64_t across = ceil_div(N, 256);
  const int64_t want = std::max<int64_t>(1, 1024 / across);
  const int64_t per = std::max<int64_t>(32, ceil_div(M, want));
  return {int(per), int(std::max<int64_t>(1, ceil_div(M, per)))};
}

template <class T>
hipError_t act_bwd(const ActBwdArgs& a, const Strips& st, void* d_bias, hipStream_t stream) {
  {
    ProfScope ps("dn_linear_act_bwd", stream);
    hipLaunchKernelGGL((act_bwd_kernel<T>), dim3(unsigned(ceil_div(a.N, 256)), unsigned(st.count)),
                       dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.sums) return e;
  }
  ProfScope ps("dn_linear_bias_sum", stream);
  hipLaunchKernelGGL((strip_sum_kernel<T>), dim3(unsigned(ceil_div(a.N, 256))), dim3(256), 0, stream,
                     static_cast<const float*>(a.sums), static_cast<T*>(d_bias), st.count, a.N);
  return hipGetLastError();
}

struct Carve {
  char* at;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = at ? at + used : nullptr;
    used += align_up(bytes, 256);
    return p;
  }
};

// --- dn_linear --------------------------------------------------------------------

Plan linear_plan(const dn_linear_args& a) {
  return plan_product(a.rows, a.out_dim, a.in_dim, 1, 1, a.dtype, false);
}

struct LinearBwd {
  Plan dx, dw;
  Strips strips;
  int64_t lddz;
  void* dz;
  float *sums, *partial;
  size_t bytes;
};
LinearBwd linear_bwd_plan(const dn_linear_bwd_args& a, void* ws) {
  LinearBwd p{};
  size_t partial = 0;
  if (a.d_x && a.rows > 0) {
    p.dx = plan_product(a.rows, a.in_dim, a.out_dim, 1, 1, a.dtype, false);
    partial = p.dx.partial_bytes;
  }
  if (a.d_weight) {
    p.dw = plan_product(a.in_dim, a.out_dim, a.rows, 1, 1, a.dtype, false);
    partial = std::max(partial, p.dw.partial_bytes);
  }
  Carve c{static_cast<char*>(ws)};
  p.lddz = int64_t(align_up(size_t(a.out_dim), 16));
  if (a.activation != DN_ACT_IDENTITY)
    p.dz = c.take(size_t(a.rows) * size_t(p.lddz) * elem_size(a.dtype));
  p.strips = strips_of(a.rows, a.out_dim);
  if (a.d_bias) p.sums = static_cast<float*>(c.take(size_t(p.strips.count) * a.out_dim * 4));
  if (partial) p.partial = static_cast<float*>(c.take(partial));
  p.bytes = c.used;
  return p;
}

// --- dn_gated_ffn -----------------------------------------------------------------

int64_t padded(int64_t n) { return int64_t(align_up(size_t(n), 16)); }

struct FfnFwd {
  Plan in, down;
  void* h;
  float* partial;
  size_t bytes;
};
FfnFwd ffn_plan(const dn_gated_ffn_args& a, void* ws) {
  FfnFwd p{};
  p.in = plan_product(a.rows, a.hidden, a.dim, 1, 1, a.dtype, true);
  p.down = plan_product(a.rows, a.dim, a.hidden, 1, 1, a.dtype, false);
  Carve c{static_cast<char*>(ws)};
  p.h = c.take(size_t(a.rows) * size_t(padded(a.hidden)) * elem_size(a.dtype));
  const size_t partial = std::max(p.in.partial_bytes, p.down.partial_bytes);
  if (partial) p.partial = static_cast<float*>(c.take(partial));
  p.bytes = c.used;
  return p;
}

struct FfnBwd {
  Plan dh, dx, dw_in, dw_down;
  void *dg, *du, *h;
  float* partial;
  size_t bytes;
};
FfnBwd ffn_bwd_plan(const dn_gated_ffn_bwd_args& a, void* ws) {
  FfnBwd p{};
  if (a.rows > 0) p.dh = plan_product(a.rows, a.hidden, a.dim, 1, 1, a.dtype, false);
  size_t partial = p.dh.partial_bytes;
  if (a.d_x && a.rows > 0) {
    p.dx = plan_product(a.rows, a.dim, a.hidden, 2, 1, a.dtype, false);
    partial = std::max(partial, p.dx.partial_bytes);
  }
  if (a.d_w_gate) {
    p.dw_in = plan_product(a.dim, a.hidden, a.rows, 1, 2, a.dtype, false);
    partial = std::max(partial, p.dw_in.partial_bytes);
  }
  if (a.d_w_down) {
    p.dw_down = plan_product(a.hidden, a.dim, a.rows, 1, 1, a.dtype, false);
    partial = std::max(partial, p.dw_down.partial_bytes);
  }
  Carve c{static_cast<char*>(ws)};
  const size_t one = size_t(a.rows) * size_t(padded(a.hidden)) * elem_size(a.dtype);
  p.dg = c.take(one);
  p.du = c.take(one);
  p.h = c.take(one);
  if (partial) p.partial = static_cast<float*>(c.take(partial));
  p.bytes = c.used;
  return p;
}

const char* bytes_of(const void* p) { return static_cast<const char*>(p); }

GemmArgs product(int64_t M, int64_t N, int64_t K, const void* a, int64_t lda, const void* b,
                 int64_t ldb, int dtype) {
  GemmArgs g{};
  const int64_t es = int64_t(elem_size(dtype));
  g.a[0] = bytes_of(a);
  g.b[0] = bytes_of(b);
  g.lda = lda * es;
  g.ldb = ldb * es;
  g.M = int(M);
  g.N = int(N);
  g.K = int(K);
  g.nseg = g.npair = 1;
  return g;
}

}  // namespace

size_t linear_workspace(const dn_linear_args& a) { return linear_plan(a).partial_bytes; }

hipError_t launch_linear(const dn_linear_args& a, void* ws, hipStream_t stream) {
  const Plan plan = linear_plan(a);
  GemmArgs g = product(a.rows, a.out_dim, a.in_dim, a.x, a.x_stride, a.weight, a.weight_stride,
                       a.dtype);
  // 8-bit rows are padded with zeros to whole words.
  if (a.dtype == DN_F8) g.K = int(align_up(size_t(a.in_dim), 16));
  g.act = a.activation;
  g.out[0] = a.out;
  g.ldo = a.out_stride;
  g.bias = a.bias;
  g.residual = a.residual;
  g.ldr = a.residual_stride;
  g.preact = a.preact;
  g.ldp = a.preact_stride;
  g.row_scale = a.x_scale;
  g.col_scale = a.weight_scale;
  return run_product(g, a.dtype == DN_F8 ? kFormNT : kFormNN, kEpiLinear, a.dtype, a.out_dtype, plan,
                     static_cast<float*>(ws), "dn_linear", stream);
}

size_t linear_bwd_workspace(const dn_linear_bwd_args& a) {
  return linear_bwd_plan(a, nullptr).bytes;
}

hipError_t launch_linear_bwd(const dn_linear_bwd_args& a, void* ws, hipStream_t stream) {
  const LinearBwd p = linear_bwd_plan(a, ws);
  const void* dz = a.d_out;
  int64_t lddz = a.d_out_stride;
  hipError_t e;
  if (p.dz || a.d_bias) {
    ActBwdArgs b{};
    b.d_out = a.d_out;
    b.ldd = a.d_out_stride;
    b.z = p.dz ? a.preact : nullptr;
    b.ldz = a.preact_stride;
    b.dz = p.dz;
    b.lddz = p.lddz;
    b.sums = p.sums;
    b.M = int(a.rows);
    b.N = int(a.out_dim);
    b.rows_per = p.strips.rows_per;
    b.act = a.activation;
      e = a.dtype == DN_BF16 ? act_bwd<bf16>(b, p.strips, a.d_bias, stream)
                           : act_bwd<float>(b, p.strips, a.d_bias, stream);
    if (e != hipSuccess) return e;
    if (p.dz) {
      dz = p.dz;
      lddz = p.lddz;
    }
  }
  if (a.d_x && a.rows > 0) {
    GemmArgs g = product(a.rows, a.in_dim, a.out_dim, dz, lddz, a.weight, a.weight_stride, a.dtype);
    g.out[0] = a.d_x;
    g.ldo = a.d_x_stride;
      if ((e = run_product(g, kFormNT, kEpiLinear, a.dtype, a.dtype, p.dx, p.partial, "dn_linear_dx",
                         stream)) != hipSuccess)
      return e;
  }
  if (a.d_weight) {
    GemmArgs g = product(a.in_dim, a.out_dim, a.rows, a.x, a.x_stride, dz, lddz, a.dtype);
    g.out[0] = a.d_weight;
    g.ldo = a.out_dim;
      if ((e = run_product(g, kFormTN, kEpiLinear, a.dtype, a.dtype, p.dw, p.partial, "dn_linear_dw",
                         stream)) != hipSuccess)
      return e;
  }
  return hipSuccess;
}

size_t gated_ffn_workspace(const dn_gated_ffn_args& a) { return ffn_plan(a, nullptr).bytes; }

hipError_t launch_gated_ffn(const dn_gated_ffn_args& a, void* ws, hipStream_t stream) {
  const FfnFwd p = ffn_plan(a, ws);
  const int64_t ldh = padded(a.hidden);
  GemmArgs g = product(a.rows, a.hidden, a.dim, a.x, a.x_stride, a.w_gate, a.w_in_stride, a.dtype);
  g.b[1] = bytes_of(a.w_up);
  g.act = a.activation;
  g.out[0] = p.h;
  g.ldo = ldh;
  g.preact = a.gate;
  g.up = a.up;
  g.ldp = a.kept_stride;
  hipError_t e = run_product(g, kFormNN, kEpiGated, a.dtype, a.dtype, p.in, p.partial,
                             "dn_gated_ffn_in", stream);
  if (e != hipSuccess) return e;
  g = product(a.rows, a.dim, a.hidden, p.h, ldh, a.w_down, a.w_down_stride, a.dtype);
  g.out[0] = a.out;
  g.ldo = a.out_stride;
  g.residual = a.residual;
  g.ldr = a.residual_stride;
  return run_product(g, kFormNN, kEpiLinear, a.dtype, a.dtype, p.down, p.partial,
                     "dn_gated_ffn_down", stream);
}

size_t gated_ffn_bwd_workspace(const dn_gated_ffn_bwd_args& a) {
  return ffn_bwd_plan(a, nullptr).bytes;
}

hipError_t launch_gated_ffn_bwd(const dn_gated_ffn_bwd_args& a, void* ws, hipStream_t stream) {
  const FfnBwd p = ffn_bwd_plan(a, ws);
  const int64_t ldh = padded(a.hidden);
  GemmArgs g = product(a.rows, a.hidden, a.dim, a.d_out, a.d_out_stride, a.w_down, a.w_down_stride,
                       a.dtype);
  g.act = a.activation;
  g.out[0] = p.dg;
  g.out[1] = p.du;
  g.h = p.h;
  g.ldo = ldh;
  g.preact = const_cast<void*>(a.gate);
  g.up = const_cast<void*>(a.up);
  g.ldp = a.kept_stride;
  hipError_t e = hipSuccess;
  if (a.rows > 0)
    e = run_product(g, kFormNT, kEpiDGated, a.dtype, a.dtype, p.dh, p.partial, "dn_gated_ffn_dh",
                    stream);
  if (e != hipSuccess) return e;
  if (a.d_x && a.rows > 0) {
    g = product(a.rows, a.dim, a.hidden, p.dg, ldh, a.w_gate, a.w_in_stride, a.dtype);
    g.a[1] = bytes_of(p.du);
    g.b[1] = bytes_of(a.w_up);
    g.nseg = 2;
    g.out[0] = a.d_x;
    g.ldo = a.d_x_stride;
      if ((e = run_product(g, kFormNT, kEpiLinear, a.dtype, a.dtype, p.dx, p.partial,
                         "dn_gated_ffn_dx", stream)) != hipSuccess)
      return e;
  }
  if (a.d_w_gate) {
    g = product(a.dim, a.hidden, a.rows, a.x, a.x_stride, p.dg, ldh, a.dtype);
    g.b[1] = bytes_of(p.du);
    g.npair = 2;
    g.out[0] = a.d_w_gate;
    g.out[1] = a.d_w_up;
    g.ldo = a.hidden;
      if ((e = run_product(g, kFormTN, kEpiLinear, a.dtype, a.dtype, p.dw_in, p.partial,
                         "dn_gated_ffn_dw_in", stream)) != hipSuccess)
      return e;
  }
  if (a.d_w_down) {
    g = product(a.hidden, a.dim, a.rows, p.h, ldh, a.d_out, a.d_out_stride, a.dtype);
    g.out[0] = a.d_w_down;
    g.ldo = a.dim;
      if ((e = run_product(g, kFormTN, kEpiLinear, a.dtype, a.dtype, p.dw_down, p.partial,
                         "dn_gated_ffn_dw_down", stream)) != hipSuccess)
      return e;
  }
  return hipSuccess;
}

}  // namespace dn

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
//
// Roundings of a bf16 feed-forward's backward: gate and up are kept in bf16 (in
// fp32 they would be 738 MB at 16384 x 5632, and not kept they would cost the
// largest product again), and the matrix unit takes h, d_gate and d_up in bf16.
// The gradients are 0.0035 from a 64-bit result in the norm, where rounding the
// result alone gives 0.0017. The forward rounds h the same way: 0.0019.
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
  gemm::Tail<TO, EPI> tail;
  gemm::tail_load<TO, EPI>(p, row, col, tail);
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
  gemm::tail_store<TO, EPI>(p, z, row, col, v, u, tail);
}

// The same for the wide kernel's split tiles: workgroup w has the rest's k
// tiles w·per … (w + 1)·per − 1, and its part of the rest's tile t is slot
// w + t of the workspace. A workgroup of this kernel takes 8 rows of a tile.
template <class TO, int EPI>
__global__ __launch_bounds__(kJoinThreads) void wide_join_kernel(GemmArgs p) {
  constexpr int kPer = EPI == kEpiGated ? 16 : 32;  // threads to a row
  constexpr int kRows = kJoinThreads / kPer;
  const int t = blockIdx.x, nk = p.ktiles * p.nseg, tiles = p.tiles_m * p.tiles_n;
  const int64_t u0 = int64_t(t) * nk;
  const int w0 = int(u0 / p.per_split), w1 = int((u0 + nk - 1) / p.per_split);
  if (w0 == w1) return;  // in one piece
  const int id = p.rounds * p.split + t, z = id / tiles;
  int tm, tn;
  {
    const int i = id - z * tiles, band = 8 * p.tiles_n, g = i / band, first = g * 8;
    const int rows = min(8, p.tiles_m - first), r = i - g * band;
    tm = first + r % rows;
    tn = r / rows;
  }
  const int r = blockIdx.y * kRows + threadIdx.x / kPer, c = (threadIdx.x % kPer) * 8;
  const int64_t row = int64_t(tm) * 256 + r;
  const int col = tn * (EPI == kEpiGated ? 128 : 256) + c;
  if (row >= p.M || col >= p.N) return;
  gemm::Tail<TO, EPI> tail;
  gemm::tail_load<TO, EPI>(p, row, col, tail);
  float v[8] = {}, u[8] = {};
  for (int w = w0; w <= w1; ++w) {
    const float* at = p.partial + ((int64_t(w + t) * 256 + r) << 8) + c;
    float x[8];
    gemm::load8(at, x, 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
    if constexpr (EPI == kEpiGated) {
      gemm::load8(at + 128, x, 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] += x[e];
    }
  }
  gemm::tail_store<TO, EPI>(p, z, row, col, v, u, tail);
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
        float slope[8];
        gemm::act8<true>(z, p.act, z, slope);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= slope[i];
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

// The strips' sums: 64 columns a workgroup, four lanes to each, which meet in LDS.
template <class T>
__global__ __launch_bounds__(256) void strip_sum_kernel(const float* sums, T* out, int strips,
                                                        int n) {
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), lane = threadIdx.x >> 6;
  float t = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int i = lane; i < strips; i += 4) t += sums[int64_t(i) * n + c];
  }
  __shared__ float lds[4][64];
  lds[lane][threadIdx.x & 63] = t;
  __syncthreads();
  if (lane == 0 && c < n) st(out, size_t(c), lds[0][threadIdx.x] + lds[1][threadIdx.x] +
                                                 lds[2][threadIdx.x] + lds[3][threadIdx.x]);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t elem_size(int dtype) { return dtype == DN_F32 ? 4 : dtype == DN_BF16 ? 2 : 1; }
bool at16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How one product is cut into workgroups.
struct Plan {
  GemmTile tile;
  bool copyable;
  int tiles_m, tiles_n, ktiles, split, per_split, rounds;
  size_t partial_bytes;
};

// Whether every operand row lies at 16-byte steps and holds whole words.
bool is_copyable(const GemmArgs& g, GemmForm form, int dtype, bool second) {
  const int64_t ch = int64_t(16 / elem_size(dtype));
  const bool acol = form == kFormTN, bcol = form != kFormNT;
  bool ok = at16(g.a[0]) && at16(g.b[0]) && g.lda % 16 == 0 && g.ldb % 16 == 0;
  if (second) ok = ok && at16(g.b[1]) && (g.nseg == 1 || at16(g.a[1]));
  if (acol) ok = ok && g.M % ch == 0;
  if (bcol) ok = ok && g.N % ch == 0;
  if ((!acol || !bcol) && dtype != DN_F8) ok = ok && g.K % ch == 0;  // 8-bit rows do
  return ok;
}

// What the kernels take, in us, from their measured times: `lone` for a k tile
// where a CU has one workgroup, or `each` for every workgroup of the CU,
// whichever is more; `ends` for a tile's start and end.
//
// kTile128: four waves of 64 x 64; two workgroups hide each other's waits.
// kTileLone: the same tile by eight waves, two of them sharing each part's k
// steps, for one workgroup a CU (bf16 1024 x 2048 x 4096 31 -> 25 us, 8-bit
// 256 x 2048 x 12304 28 -> 22). kTile64: where 128 x 128 tiles are too few
// (bf16 512 x 2048 x 4096: 18 us, kTileLone 24). Gated, its 32 columns of each
// matrix are half lines of memory: 256 x 2048 x 5632 40 us, kTileLone 29.
struct Cost {
  double lone, each, ends;
  int most;  // workgroups of a CU at once
};
Cost cost_of(GemmTile tile, int dtype, bool gated) {
  switch (tile) {
    case kTileWide: return dtype == DN_F8 ? Cost{3.2, 3.2, 9, 1} : Cost{1.65, 1.65, 9, 1};
    case kTile128:
      return dtype == DN_F32  ? Cost{2.4, 2.1, 3, 2}
             : dtype == DN_F8 ? Cost{1.55, 1.0, 3, 2}
                              : Cost{0.85, 0.58, 3, 2};
    case kTileLone: return dtype == DN_F8 ? Cost{1.15, 1.15, 4, 1} : Cost{0.65, 0.65, 4, 1};
    default:
      return dtype == DN_F32  ? Cost{0.8, 0.56, 3, 4}
             : dtype == DN_F8 ? Cost{0.58, 0.27, 3, 4}
             : gated          ? Cost{0.5, 0.36, 3, 3}
                              : Cost{0.38, 0.22, 3, 3};
  }
}

// The wide kernel: one workgroup a CU, whole tiles in rounds, the rest's k
// tiles dealt out.
Plan plan_wide(int64_t M, int64_t N, int64_t K, int nseg, int npair, int dtype, bool gated,
               double* cost) {
  Plan p{};
  p.tile = kTileWide;
  p.tiles_m = int(ceil_div(M, 256));
  p.tiles_n = int(ceil_div(N, gated ? 128 : 256));
  p.ktiles = int(ceil_div(K, int64_t(128 / elem_size(dtype))));
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n * npair, nk = int64_t(p.ktiles) * nseg;
  const int64_t cus = device_cu_count();
  const Cost t = cost_of(kTileWide, dtype, gated);
  p.rounds = int(tiles / cus);
  const int64_t rest = tiles - p.rounds * cus;
  double c = p.rounds * (double(nk) * t.each + t.ends);
  p.split = int(p.rounds ? cus : std::max<int64_t>(1, std::min(cus, tiles)));
  p.per_split = int(nk);
  if (rest) {
    // Whole, one a workgroup; or dealt out, at least 8 k tiles each, with up to
    // two parts a workgroup (their ends, with fp32 sums to store, take longer than
    // a tile's), the join and the sums' round trip (256 KB a part at 4 TB/s).
    const double whole = double(nk) * t.each + t.ends;
    const int64_t per = std::max<int64_t>(8, ceil_div(rest * nk, cus));
    const int64_t parts = ceil_div(rest * nk, per) + rest;
    const double dealt = double(per) * t.each + 28 + 4 + double(parts) * 0.13;
    if (per < nk && dealt < whole) {
      p.per_split = int(per);
      if (!p.rounds) p.split = int(ceil_div(rest * nk, per));
      p.partial_bytes = size_t(p.split + rest) * 256 * 256 * 4;
      c += dealt;
    } else {
      c += whole;
    }
  }
  *cost = c;
  return p;
}

// A pointer into a workspace that is not there yet is null: its place is aligned.
Plan plan_product(const GemmArgs& g, GemmForm form, GemmEpi epi, int dtype) {
  const int64_t M = g.M, N = g.N, K = g.K;
  const int nseg = g.nseg, npair = g.npair;
  const bool gated = epi == kEpiGated;
  const bool copyable = is_copyable(g, form, dtype, nseg == 2 || npair == 2 || gated);
  Plan best{};
  // Few rows: up to 64 (gated 32) W's traffic binds, not the products.
  if (M <= few_rows_most(epi) && N >= 4 && form == (dtype == DN_F8 ? kFormNT : kFormNN)) {
    best.tile = kTileFew;
    best.copyable = copyable;
    const int64_t chunks = K / 32;  // of 32 rows of W
    best.per_split = int(ceil_div(std::max<int64_t>(1, chunks),
                                  few_rows_split(g, epi, dtype, copyable)));
    best.split = int(std::max<int64_t>(1, ceil_div(chunks, best.per_split)));
    if (best.split > 1)
      best.partial_bytes = align_up(size_t(best.split) * M * align_up(size_t(N), 4) * 4, 256);
    return best;
  }
  double best_cost = 0;
  // The wide kernel has no fp32 form (fp32 products are bound by the matrix
  // unit in any), takes whole words, and 32-bit offsets within 256 rows.
  if (copyable && dtype != DN_F32 && K > 0 && g.lda < (1 << 23) && g.ldb < (1 << 23))
    best = plan_wide(M, N, K, nseg, npair, dtype, gated, &best_cost);
  const int64_t cus = device_cu_count();
  for (const GemmTile tile : {kTile128, kTileLone, kTile64}) {
    if (tile == kTileLone && (!copyable || dtype == DN_F32)) continue;
    const int b = tile == kTile64 ? 64 : 128;
    const Cost t = cost_of(tile, dtype, gated);
    Plan p{};
    p.tile = tile;
    p.tiles_m = int(ceil_div(M, b));
    p.tiles_n = int(ceil_div(N, gated ? b / 2 : b));
    p.ktiles = int(ceil_div(K, int64_t(128 / elem_size(dtype))));
    const int64_t ksteps = std::max<int64_t>(1, int64_t(p.ktiles) * nseg);
    const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n * npair;
    const int most = int(std::min<int64_t>(std::max<int64_t>(1, ksteps / 2), 64));
    for (int s = 1; s <= most; s = s < 4 ? s + 1 : s + s / 4) {
      const int64_t per = ceil_div(ksteps, s);
      const int split = int(ceil_div(ksteps, per));
      // A launch of 2^32 threads or more wraps.
      if (tiles * split >= (int64_t(1) << 32) / (tile == kTileLone ? 512 : 256)) break;
      const int64_t w = ceil_div(tiles * split, cus), left = w % t.most;
      const auto turn = [&](int64_t n) {
        return double(per) * std::max(t.lone, t.each * double(n)) + t.ends;
      };
      double cost = double(w / t.most) * turn(t.most) + (left ? turn(left) : 0.0);
      if (split > 1)  // the join, and the partial sums out and in at 4 TB/s
        cost += 4 + double(M) * N * (gated ? 2 : 1) * npair * split * 8.0 / 4.0e6;
      if (best.split == 0 || cost < best_cost) {
        best_cost = cost;
        p.split = split;
        p.per_split = int(per);
        p.partial_bytes =
            split > 1 ? align_up(size_t(split) * npair * size_t(M) *
                                     size_t(gated ? 2 * N : align_up(size_t(N), 4)) * 4, 256)
                      : 0;
        best = p;
      }
      if (s > 1 && tiles * s >= 4 * t.most * cus) break;
    }
  }
  best.copyable = copyable;
  return best;
}

void apply(GemmArgs& g, const Plan& p, bool gated, float* partial) {
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.ktiles = p.ktiles;
  g.split = p.split;
  g.per_split = p.per_split;
  g.rounds = p.rounds;
  g.partial = p.partial_bytes ? partial : nullptr;
  g.ldpart = gated ? 2 * int64_t(g.N) : int64_t(align_up(size_t(g.N), 4));
}

template <class TO, int EPI>
hipError_t join_go(const GemmArgs& g, GemmTile tile, hipStream_t stream) {
  if (tile == kTileWide) {
    const int rest = g.tiles_m * g.tiles_n * g.npair - g.rounds * g.split;
    const int rows = kJoinThreads / (EPI == kEpiGated ? 16 : 32);
    hipLaunchKernelGGL((wide_join_kernel<TO, EPI>), dim3(unsigned(rest), unsigned(256 / rows)),
                       dim3(kJoinThreads), 0, stream, g);
  } else {
    const int64_t n = int64_t(g.M) * ((g.N + 7) / 8) * g.npair;
    hipLaunchKernelGGL((gemm_join_kernel<TO, EPI>), dim3(unsigned(ceil_div(n, kJoinThreads))),
                       dim3(kJoinThreads), 0, stream, g);
  }
  return hipGetLastError();
}
template <class TO>
hipError_t join_typed(const GemmArgs& g, GemmEpi epi, GemmTile tile, hipStream_t stream) {
  if (epi == kEpiLinear) return join_go<TO, kEpiLinear>(g, tile, stream);
  if (epi == kEpiGated) return join_go<TO, kEpiGated>(g, tile, stream);
  return join_go<TO, kEpiDGated>(g, tile, stream);
}

hipError_t run_product(GemmArgs& g, GemmForm form, GemmEpi epi, int dtype, int out_dtype,
                       const Plan& plan, float* partial, const char* name, hipStream_t stream) {
  if (!plan.split) return hipErrorInvalidConfiguration;  // no tile is large enough
  apply(g, plan, epi == kEpiGated, partial);
  hipError_t e;
  {
    ProfScope ps(name, stream);
    if (plan.tile == kTileFew) e = few_rows(g, epi, dtype, out_dtype, plan.copyable, stream);
    else if (dtype == DN_F8) e = gemm_f8(g, out_dtype, plan.tile, stream);
    else if (dtype == DN_BF16) e = gemm_bf16(g, form, epi, plan.tile, !plan.copyable, stream);
    else e = gemm_f32(g, form, epi, plan.tile, !plan.copyable, stream);
  }
  if (e != hipSuccess || !plan.partial_bytes) return e;
  ProfScope ps("dn_product_join", stream);
  return out_dtype == DN_BF16 ? join_typed<bf16>(g, epi, plan.tile, stream)
                              : join_typed<float>(g, epi, plan.tile, stream);
}

// --- act' and the bias' gradient -------------------------------------------------

struct Strips {
  int rows_per, count;
};
// Strips of rows: enough workgroups to fill the CUs, at least 8 rows each, one for
// a lane (of 32: 7.9 us in place of 5.2 at 500 x 1039 in fp32).
Strips strips_of(int64_t M, int64_t N) {
  const int64_t across = ceil_div(N, 256);
  const int64_t want = std::max<int64_t>(1, 1024 / across);
  const int64_t per = std::max<int64_t>(8, ceil_div(M, want));
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
  hipLaunchKernelGGL((strip_sum_kernel<T>), dim3(unsigned(ceil_div(a.N, 64))), dim3(256), 0, stream,
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

// One product of an operation.
struct Product {
  GemmArgs g;
  GemmForm form;
  GemmEpi epi;
  const char* name;
  Plan plan;
};

// An operation's products, in order, and its workspace: what they share, then
// room for the largest one's partial sums. Laid out the same with no workspace
// given (`ws` null), to size it.
struct Steps {
  int dtype, out_dtype;
  Carve carve;
  Product product[4];
  int count = 0;

  // M × N over K: a (lda elements a row) times b.
  GemmArgs& add(const char* name, GemmForm form, GemmEpi epi, int64_t M, int64_t N, int64_t K,
                const void* a, int64_t lda, const void* b, int64_t ldb) {
    const int64_t es = int64_t(elem_size(dtype));
    Product& p = product[count++];
    p = Product{};
    p.form = form;
    p.epi = epi;
    p.name = name;
    p.g.a[0] = static_cast<const char*>(a);
    p.g.b[0] = static_cast<const char*>(b);
    p.g.lda = lda * es;
    p.g.ldb = ldb * es;
    p.g.M = int(M);
    p.g.N = int(N);
    p.g.K = int(K);
    p.g.nseg = p.g.npair = 1;
    return p.g;
  }
  size_t finish() {
    size_t partial = 0;
    for (int i = 0; i < count; ++i) {
      product[i].plan = plan_product(product[i].g, product[i].form, product[i].epi, dtype);
      partial = std::max(partial, product[i].plan.partial_bytes);
    }
    partials = partial ? static_cast<float*>(carve.take(partial)) : nullptr;
    return carve.used;
  }
  hipError_t run(hipStream_t stream) {
    for (int i = 0; i < count; ++i) {
      Product& p = product[i];
      const hipError_t e = run_product(p.g, p.form, p.epi, dtype, out_dtype, p.plan, partials,
                                       p.name, stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  float* partials = nullptr;
};

int64_t padded(int64_t n) { return int64_t(align_up(size_t(n), 16)); }

size_t linear_steps(const dn_linear_args& a, void* ws, Steps& s) {
  s.dtype = a.dtype;
  s.out_dtype = a.out_dtype;
  s.carve.at = static_cast<char*>(ws);
  GemmArgs& g = s.add("dn_linear", a.dtype == DN_F8 ? kFormNT : kFormNN, kEpiLinear, a.rows,
                      a.out_dim, a.in_dim, a.x, a.x_stride, a.weight, a.weight_stride);
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
  return s.finish();
}

struct LinearBwd {
  Strips strips;
  int64_t lddz;
  void* dz;
  float* sums;
};
size_t linear_bwd_steps(const dn_linear_bwd_args& a, void* ws, Steps& s, LinearBwd& l) {
  s.dtype = s.out_dtype = a.dtype;
  s.carve.at = static_cast<char*>(ws);
  const bool act = a.activation != DN_ACT_IDENTITY;
  l.strips = strips_of(a.rows, a.out_dim);
  l.lddz = padded(a.out_dim);
  l.dz = act ? s.carve.take(size_t(a.rows) * size_t(l.lddz) * elem_size(a.dtype)) : nullptr;
  l.sums = a.d_bias
               ? static_cast<float*>(s.carve.take(size_t(l.strips.count) * size_t(a.out_dim) * 4))
               : nullptr;
  const void* dz = act ? l.dz : a.d_out;
  const int64_t lddz = act ? l.lddz : a.d_out_stride;
  if (a.d_x && a.rows > 0) {
    GemmArgs& g = s.add("dn_linear_dx", kFormNT, kEpiLinear, a.rows, a.in_dim, a.out_dim, dz, lddz,
                        a.weight, a.weight_stride);
    g.out[0] = a.d_x;
    g.ldo = a.d_x_stride;
  }
  if (a.d_weight) {
    GemmArgs& g = s.add("dn_linear_dw", kFormTN, kEpiLinear, a.in_dim, a.out_dim, a.rows, a.x,
                        a.x_stride, dz, lddz);
    g.out[0] = a.d_weight;
    g.ldo = a.out_dim;
  }
  return s.finish();
}

size_t ffn_steps(const dn_gated_ffn_args& a, void* ws, Steps& s) {
  s.dtype = s.out_dtype = a.dtype;
  s.carve.at = static_cast<char*>(ws);
  const int64_t ldh = padded(a.hidden);
  void* h = s.carve.take(size_t(a.rows) * size_t(ldh) * elem_size(a.dtype));
  GemmArgs& in = s.add("dn_gated_ffn_in", kFormNN, kEpiGated, a.rows, a.hidden, a.dim, a.x,
                       a.x_stride, a.w_gate, a.w_in_stride);
  in.b[1] = static_cast<const char*>(a.w_up);
  in.act = a.activation;
  in.out[0] = h;
  in.ldo = ldh;
  in.preact = a.gate;
  in.up = a.up;
  in.ldp = a.kept_stride;
  GemmArgs& down = s.add("dn_gated_ffn_down", kFormNN, kEpiLinear, a.rows, a.dim, a.hidden, h, ldh,
                         a.w_down, a.w_down_stride);
  down.out[0] = a.out;
  down.ldo = a.out_stride;
  down.residual = a.residual;
  down.ldr = a.residual_stride;
  return s.finish();
}

size_t ffn_bwd_steps(const dn_gated_ffn_bwd_args& a, void* ws, Steps& s) {
  s.dtype = s.out_dtype = a.dtype;
  s.carve.at = static_cast<char*>(ws);
  const int64_t ldh = padded(a.hidden);
  const size_t one = size_t(a.rows) * size_t(ldh) * elem_size(a.dtype);
  void* dg = s.carve.take(one);
  void* du = s.carve.take(one);
  void* h = s.carve.take(one);
  if (a.rows > 0) {
    GemmArgs& g = s.add("dn_gated_ffn_dh", kFormNT, kEpiDGated, a.rows, a.hidden, a.dim, a.d_out,
                        a.d_out_stride, a.w_down, a.w_down_stride);
    g.act = a.activation;
    g.out[0] = dg;
    g.out[1] = du;
    g.h = h;
    g.ldo = ldh;
    g.preact = const_cast<void*>(a.gate);
    g.up = const_cast<void*>(a.up);
    g.ldp = a.kept_stride;
  }
  if (a.d_x && a.rows > 0) {
    GemmArgs& g = s.add("dn_gated_ffn_dx", kFormNT, kEpiLinear, a.rows, a.dim, a.hidden, dg, ldh,
                        a.w_gate, a.w_in_stride);
    g.a[1] = static_cast<const char*>(du);
    g.b[1] = static_cast<const char*>(a.w_up);
    g.nseg = 2;
    g.out[0] = a.d_x;
    g.ldo = a.d_x_stride;
  }
  if (a.d_w_gate) {
    GemmArgs& g = s.add("dn_gated_ffn_dw_in", kFormTN, kEpiLinear, a.dim, a.hidden, a.rows, a.x,
                        a.x_stride, dg, ldh);
    g.b[1] = static_cast<const char*>(du);
    g.npair = 2;
    g.out[0] = a.d_w_gate;
    g.out[1] = a.d_w_up;
    g.ldo = a.hidden;
  }
  if (a.d_w_down) {
    GemmArgs& g = s.add("dn_gated_ffn_dw_down", kFormTN, kEpiLinear, a.hidden, a.dim, a.rows, h,
                        ldh, a.d_out, a.d_out_stride);
    g.out[0] = a.d_w_down;
    g.ldo = a.dim;
  }
  return s.finish();
}

}  // namespace

size_t linear_workspace(const dn_linear_args& a) {
  Steps s;
  return linear_steps(a, nullptr, s);
}

hipError_t launch_linear(const dn_linear_args& a, void* ws, hipStream_t stream) {
  Steps s;
  linear_steps(a, ws, s);
  return s.run(stream);
}

size_t linear_bwd_workspace(const dn_linear_bwd_args& a) {
  Steps s;
  LinearBwd l;
  return linear_bwd_steps(a, nullptr, s, l);
}

hipError_t launch_linear_bwd(const dn_linear_bwd_args& a, void* ws, hipStream_t stream) {
  Steps s;
  LinearBwd l;
  linear_bwd_steps(a, ws, s, l);
  if ((l.dz && a.rows > 0) || l.sums) {
    ActBwdArgs b{};
    b.d_out = a.d_out;
    b.ldd = a.d_out_stride;
    b.z = l.dz ? a.preact : nullptr;
    b.ldz = a.preact_stride;
    b.dz = l.dz;
    b.lddz = l.lddz;
    b.sums = l.sums;
    b.M = int(a.rows);
    b.N = int(a.out_dim);
    b.rows_per = l.strips.rows_per;
    b.act = a.activation;
    const hipError_t e = a.dtype == DN_BF16 ? act_bwd<bf16>(b, l.strips, a.d_bias, stream)
                                            : act_bwd<float>(b, l.strips, a.d_bias, stream);
    if (e != hipSuccess) return e;
  }
  return s.run(stream);
}

size_t gated_ffn_workspace(const dn_gated_ffn_args& a) {
  Steps s;
  return ffn_steps(a, nullptr, s);
}

hipError_t launch_gated_ffn(const dn_gated_ffn_args& a, void* ws, hipStream_t stream) {
  Steps s;
  ffn_steps(a, ws, s);
  return s.run(stream);
}

size_t gated_ffn_bwd_workspace(const dn_gated_ffn_bwd_args& a) {
  Steps s;
  return ffn_bwd_steps(a, nullptr, s);
}

hipError_t launch_gated_ffn_bwd(const dn_gated_ffn_bwd_args& a, void* ws, hipStream_t stream) {
  Steps s;
  ffn_bwd_steps(a, ws, s);
  return s.run(stream);
}

}  // namespace dn

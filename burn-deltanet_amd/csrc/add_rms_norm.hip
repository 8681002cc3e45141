// dn_add_rms_norm: s = x + residual, out = s / sqrt(mean(s²) + ε) · γ, in one
// pass; dn_add_rms_norm_bwd: its gradient in one pass and a short sum.
//
// Bound by memory: x, residual in, s, out out (the backward: s, d_out, d_s in,
// d_x out). A row is held in registers between its reads and its writes, eight
// adjacent values to a lane and chunk, so that every byte moves once. WPR
// waves share a row: one where there are rows enough to fill the CUs (no
// barrier, and a wave's loads of a row are all in flight at once), four where
// rows are few or long. Rows too long for registers are read a second time.
//
// The 8-bit output's scale is the largest |out| of the row over 448 (e4m3's
// largest finite value), found in registers before the codes are rounded.
//
// d_γ sums over the rows: a workgroup keeps its rows' sums in registers and
// writes them once; a second kernel adds the workgroups' in order.
//
// The sum and all statistics are fp32. A bf16 sum that is handed out is rounded
// once (it is the residual stream, and is read again as such); the forward
// normalises the unrounded one, the backward starts from what was handed out.
//
// Measured, bf16: 32768 x 2048 with a residual 97 us (5.5 TB/s, a copy's rate),
// its gradient 164 us (3.3 TB/s) and 6 for d_γ's sum; 256 x 2048 into 8 bits
// 4.4 us.
#include <algorithm>

#include "gemm.hpp"
#include "layer.hpp"

namespace dn {
namespace {

using gemm::load8;
using gemm::store8;

struct NormArgs {
  const void *x, *residual, *weight;
  void *sum, *out;
  float* scale;
  int64_t ldx, ldr, lds, ldo;
  int rows, dim;
  int end;  // of a row of codes
  float eps;
};

// Sums (or maxima) over a row's WPR waves; every lane receives them.
__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ inline float wave_max(float v) {  // NaN wins
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const float w = __shfl_xor(v, o);
    v = w > v || w != w ? w : v;
  }
  return v;
}
// `slot`: a place of `lds` for each use between two barriers.
template <int WPR, bool MAX>
__device__ inline float row_reduce(float v, float* lds) {
  v = MAX ? wave_max(v) : wave_sum(v);
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      const float u = lds[w];
      v = MAX ? (u > v || u != u ? u : v) : v + u;
    }
  }
  return v;
}

// Eight e4m3 codes of v / scale (v is 0 or NaN where the scale is).
__device__ inline uint2 codes8(const float (&v)[8], float scale) {
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = scale == 0.f ? v[i] : v[i] / scale;
  // A denormal scale has few bits, and the row's largest value may be up to 1.5 times
  // what 448 stands for, which the conversion makes NaN.
  if (scale < 0x1p-126f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = c[i] > 448.f ? 448.f : c[i] < -448.f ? -448.f : c[i];
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
  return make_uint2(uint32_t(lo), uint32_t(hi));
}
// Codes of columns [col, col + 8) of those before dim, and zeros up to `end`.
__device__ inline void store_codes(uint8_t* row, int end, int col, int dim, uint2 u) {
  if (col + 8 > dim) {
    // Past dim 0 / scale is NaN in a row with a value that is not finite.
    const int n = max(dim - col, 0);
    const uint64_t c = (uint64_t(u.y) << 32 | u.x) & ((uint64_t(1) << (8 * n)) - 1);
    u = make_uint2(uint32_t(c), uint32_t(c >> 32));
  }
  if (col + 8 <= end) {
    __builtin_memcpy(row + col, &u, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < end) row[col + i] = uint8_t((i < 4 ? u.x : u.y) >> (8 * (i & 3)));
  }
}

constexpr int kNormThreads = 256;
// Workgroups along x: a launch of 2^32 threads or more along an axis wraps.
constexpr int kMostGroups = 1 << 20;

// NCH chunks of 8 values a lane; NCH = 0: any length, in two passes.
template <class T, class TW, bool F8, int WPR, int NCH>
__global__ __launch_bounds__(kNormThreads) void add_rms_norm_kernel(NormArgs p) {
  constexpr int kLanes = 64 * WPR;  // lanes to a row
  __shared__ float red[2][4];
  const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t group = int64_t(blockIdx.y) * kMostGroups + blockIdx.x;
  const int64_t row = WPR == 1 ? group * 4 + (threadIdx.x >> 6) : group;
  if (row >= p.rows) return;  // whole waves; with WPR = 4 whole workgroups
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
  const TW* weight = static_cast<const TW*>(p.weight);
  T* sum = p.sum ? static_cast<T*>(p.sum) + row * p.lds : nullptr;
  const int dim = p.dim;
  auto read = [&](int col, float (&v)[8]) {
    load8(x + col, v, dim - col);
    if (res) {
      float r[8];
      load8(res + col, r, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
  };
  auto write = [&](int col, const float (&v)[8], float scale) {
    if constexpr (F8)
      store_codes(static_cast<uint8_t*>(p.out) + row * p.ldo, p.end, col, dim, codes8(v, scale));
    else
      store8(static_cast<T*>(p.out) + row * p.ldo + col, v, dim - col);
  };
  auto top = [](const float (&v)[8], float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(v[i]);
      m = a > m || a != a ? a : m;
    }
    return m;
  };
  float ss = 0.f, most = 0.f, scale = 0.f;
  if constexpr (NCH > 0) {
    float v[NCH][8];
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      if (col < dim) {
        read(col, v[n]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[n][i] = 0.f;
      }
    }
#pragma unroll
    for (int n = 0; n < NCH; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[n][i], v[n][i], ss);
    ss = row_reduce<WPR, false>(ss, red[0]);
    const float inv = 1.0f / sqrtf(ss / float(dim) + p.eps);
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      if (col >= dim) continue;
      if (sum) store8(sum + col, v[n], dim - col);
      float w[8];
      load8(weight + col, w, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[n][i] = v[n][i] * inv * w[i];
      if constexpr (F8) most = top(v[n], most);
    }
    if constexpr (F8) {
      scale = row_reduce<WPR, true>(most, red[1]) * (1.0f / 448.0f);
      if (lane == 0) p.scale[row] = scale;
    }
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      if (col < (F8 ? (dim + 15) & ~15 : dim)) write(col, v[n], scale);
    }
  } else {
    // The sum is re-read from x and the residual, so that the norm is the
    // unrounded sum's: `sum` may alias either, and is written last.
    for (int col = lane * 8; col < dim; col += kLanes * 8) {
      float v[8];
      read(col, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
    }
    ss = row_reduce<WPR, false>(ss, red[0]);
    const float inv = 1.0f / sqrtf(ss / float(dim) + p.eps);
    auto normed = [&](int col, float (&v)[8], float (&s)[8]) {
      read(col, s);
      float w[8];
      load8(weight + col, w, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s[i] * inv * w[i];
    };
    if constexpr (F8) {
      for (int col = lane * 8; col < dim; col += kLanes * 8) {
        float v[8], s[8];
        normed(col, v, s);
        most = top(v, most);
      }
      scale = row_reduce<WPR, true>(most, red[1]) * (1.0f / 448.0f);
      if (lane == 0) p.scale[row] = scale;
    }
    const int end = F8 ? (dim + 15) & ~15 : dim;
    for (int col = lane * 8; col < end; col += kLanes * 8) {
      float v[8] = {}, s[8];
      if (col < dim) {
        normed(col, v, s);
        if (sum) store8(sum + col, s, dim - col);
      }
      write(col, v, scale);
    }
  }
}

struct NormBwdArgs {
  const void *sum, *weight, *d_out, *d_sum;
  void* d_x;
  float* dw;    // [workgroups][dim]; null: not formed
  float2* row;  // NCH = 0: each row's inv and c, for the column kernel
  int64_t lds, ldo, ldd, ldx;
  int rows, dim;
  float eps;
};

// With a = Σ d_out·γ·s and inv = (mean(s²) + ε)^−½, u = s·inv:
// d_x = inv·(d_out·γ − u·inv·a/dim) + d_s. A workgroup walks rows blockIdx.x·R,
// + gridDim.x·R, … (R rows at once) and its lanes keep their columns' Σ d_out·u.
// Rows too long for registers: where d_x lies on d_out, which d_γ's sum still has
// to read, the statistics and d_x are launches of their own, before and after it
// (4096 x 16384 in bf16 210 us, else 195).
enum { kStats = 1, kGradient = 2, kBoth = 3 };
template <class T, class TW, int WPR, int NCH, int DO = kBoth>
__global__ __launch_bounds__(kNormThreads) void add_rms_norm_bwd_kernel(NormBwdArgs p) {
  constexpr int kLanes = 64 * WPR, R = 4 / WPR;
  __shared__ float red[2][2][4];
  const int lane = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int wave = threadIdx.x >> 6;
  const int dim = p.dim;
  const TW* weight = static_cast<const TW*>(p.weight);
  constexpr int N = NCH > 0 ? NCH : 1;
  float w[N][8], dw[N][8] = {};
  if constexpr (NCH > 0) {
#pragma unroll
    for (int n = 0; n < NCH; ++n) {
      const int col = (n * kLanes + lane) * 8;
      load8(weight + min(col, dim), w[n], dim - col);
    }
  }
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * R + (WPR == 1 ? wave : 0); row < p.rows;
       row += int64_t(gridDim.x) * R, turn ^= 1) {
    const T* s = static_cast<const T*>(p.sum) + row * p.lds;
    const T* dy = static_cast<const T*>(p.d_out) + row * p.ldo;
    const T* ds = p.d_sum ? static_cast<const T*>(p.d_sum) + row * p.ldd : nullptr;
    T* dx = static_cast<T*>(p.d_x) + row * p.ldx;
    float ss = 0.f, a = 0.f;
    if constexpr (NCH > 0) {
      float vs[NCH][8], vd[NCH][8], ve[NCH][8];
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int col = (n * kLanes + lane) * 8;
        load8(s + min(col, dim), vs[n], dim - col);
        load8(dy + min(col, dim), vd[n], dim - col);
        if (ds) {
          load8(ds + min(col, dim), ve[n], dim - col);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) ve[n][i] = 0.f;
        }
      }
#pragma unroll
      for (int n = 0; n < NCH; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fmaf(vs[n][i], vs[n][i], ss);
          a = fmaf(vd[n][i] * w[n][i], vs[n][i], a);
        }
      ss = row_reduce<WPR, false>(ss, red[turn][0]);
      a = row_reduce<WPR, false>(a, red[turn][1]);
      const float inv = 1.0f / sqrtf(ss / float(dim) + p.eps);
      const float c = a * inv * inv / float(dim);
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int col = (n * kLanes + lane) * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = inv * (vd[n][i] * w[n][i] - vs[n][i] * c) + ve[n][i];
          dw[n][i] = fmaf(vd[n][i], vs[n][i] * inv, dw[n][i]);
        }
        if (col < dim) store8(dx + col, v, dim - col);
      }
    } else {
      float inv, c;
      if constexpr (DO & kStats) {
        for (int col = lane * 8; col < dim; col += kLanes * 8) {
          float vs[8], vd[8], vw[8];
          load8(s + col, vs, dim - col);
          load8(dy + col, vd, dim - col);
          load8(weight + col, vw, dim - col);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss = fmaf(vs[i], vs[i], ss);
            a = fmaf(vd[i] * vw[i], vs[i], a);
          }
        }
        ss = row_reduce<WPR, false>(ss, red[turn][0]);
        a = row_reduce<WPR, false>(a, red[turn][1]);
        inv = 1.0f / sqrtf(ss / float(dim) + p.eps);
        c = a * inv * inv / float(dim);
        if (lane == 0 && p.row) p.row[row] = make_float2(inv, c);
      } else {
        inv = p.row[row].x;
        c = p.row[row].y;
      }
      if constexpr (DO & kGradient)
        for (int col = lane * 8; col < dim; col += kLanes * 8) {
          float vs[8], vd[8], vw[8], ve[8] = {};
          load8(s + col, vs, dim - col);
          load8(dy + col, vd, dim - col);
          load8(weight + col, vw, dim - col);
          if (ds) load8(ds + col, ve, dim - col);
#pragma unroll
          for (int i = 0; i < 8; ++i) ve[i] += inv * (vd[i] * vw[i] - vs[i] * c);
          store8(dx + col, ve, dim - col);
        }
    }
  }
  if constexpr (NCH > 0) {
    if (!p.dw) return;
    float* out = p.dw + int64_t(blockIdx.x) * dim;
    if constexpr (WPR == 1) {
      // The four waves' sums of each column meet in LDS, a chunk at a time.
      __shared__ float part[4][64 * 8];
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) part[wave][i * 64 + lane] = dw[n][i];
        __syncthreads();
        for (int e = threadIdx.x; e < 512; e += kNormThreads) {
          const int col = n * 512 + (e & 63) * 8 + (e >> 6);
          if (col < dim) out[col] = part[0][e] + part[1][e] + part[2][e] + part[3][e];
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NCH; ++n) {
        const int col = (n * kLanes + lane) * 8;
        if (col < dim) store8(out + col, dw[n], dim - col);
      }
    }
  }
}

// Long rows: Σ d_out·s·inv over a strip of rows, a thread to a column.
template <class T>
__global__ __launch_bounds__(256) void norm_dw_kernel(const T* d_out, const T* sum,
                                                      const float2* row, float* dw, int64_t ldo,
                                                      int64_t lds, int rows, int dim, int per) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= dim) return;
  const int64_t r0 = int64_t(blockIdx.y) * per, r1 = min(r0 + per, int64_t(rows));
  float t = 0.f;
  for (int64_t r = r0; r < r1; ++r)
    t = fmaf(ld(d_out, size_t(r * ldo + c)), ld(sum, size_t(r * lds + c)) * row[r].x, t);
  dw[int64_t(blockIdx.y) * dim + c] = t;
}

// d_γ: the workgroups' sums added in order, 64 lanes of a column taking every
// 64th workgroup, their sums by halves.
constexpr int kSumCols = 16, kSumLanes = 64;
template <class TW>
__global__ __launch_bounds__(kSumCols * kSumLanes) void norm_dw_sum_kernel(const float* dw, TW* out,
                                                                           int parts, int dim) {
  __shared__ float lds[kSumLanes][kSumCols];
  const int x = threadIdx.x % kSumCols, l = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + x;
  float t = 0.f;
  if (c < dim) {
#pragma unroll 4
    for (int i = l; i < parts; i += kSumLanes) t += dw[int64_t(i) * dim + c];
  }
  lds[l][x] = t;
  __syncthreads();
#pragma unroll
  for (int half = kSumLanes / 2; half; half >>= 1) {
    if (l < half) lds[l][x] += lds[l + half][x];
    __syncthreads();
  }
  if (l == 0 && c < dim) st(out, size_t(c), lds[0][x]);
}

// Waves to a row and chunks a lane: one wave where that leaves every CU
// eight waves and the row fits (up to 2048 values), else four (up to 8192).
struct Shape {
  int wpr, nch;
};
Shape shape_of(int64_t rows, int64_t dim) {
  if (dim <= 2048 && (rows >= 8 * device_cu_count() || dim <= 512)) {
    return {1, dim <= 512 ? 1 : dim <= 1024 ? 2 : 4};
  }
  return {4, dim <= 2048 ? 1 : dim <= 4096 ? 2 : dim <= 8192 ? 4 : 0};
}

template <class T, class TW, bool F8>
hipError_t fwd_go(const NormArgs& p, hipStream_t stream) {
  const Shape s = shape_of(p.rows, p.dim);
  const int64_t groups = s.wpr == 1 ? (int64_t(p.rows) + 3) / 4 : p.rows;
  const dim3 grid(unsigned(std::min<int64_t>(groups, kMostGroups)),
                  unsigned((groups + kMostGroups - 1) / kMostGroups)),
      block(kNormThreads);
  if (s.wpr == 1 && s.nch == 1)
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 1, 1>), grid, block, 0, stream, p);
  else if (s.wpr == 1 && s.nch == 2)
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 1, 2>), grid, block, 0, stream, p);
  else if (s.wpr == 1)
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 1, 4>), grid, block, 0, stream, p);
  else if (s.nch == 1)
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 4, 1>), grid, block, 0, stream, p);
  else if (s.nch == 2)
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 4, 2>), grid, block, 0, stream, p);
  else if (s.nch == 4)
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 4, 4>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((add_rms_norm_kernel<T, TW, F8, 4, 0>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// Workgroups of the backward, whose sums of d_γ the second kernel reads: four
// to a CU keep the memory busy.
int bwd_groups(int64_t rows, const Shape& s) {
  const int64_t all = s.wpr == 1 ? (rows + 3) / 4 : rows;
  return int(std::max<int64_t>(1, std::min<int64_t>(all, 4 * device_cu_count())));
}
// Long rows: rows of a strip of the column kernel (a grid has at most 65535).
int strip_rows(int64_t rows) { return int(std::max<int64_t>(64, (rows + 32767) / 32768)); }
int strip_count(int64_t rows) {
  return int(std::max<int64_t>(1, (rows + strip_rows(rows) - 1) / strip_rows(rows)));
}

// Whether two matrices' extents in memory have a byte in common.
template <class T>
bool meet(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int64_t dim) {
  if (rows == 0) return false;
  const auto p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  const auto bytes = [&](int64_t ld) { return uintptr_t((rows - 1) * ld + dim) * sizeof(T); };
  return p < q + bytes(ldb) && q < p + bytes(lda);
}

template <class T, class TW>
hipError_t bwd_go(NormBwdArgs p, void* d_weight, void* ws, hipStream_t stream) {
  const Shape s = shape_of(p.rows, p.dim);
  int parts = bwd_groups(p.rows, s);
  const dim3 grid{unsigned(parts)}, block(kNormThreads);
  float* dw = static_cast<float*>(ws);
  if (d_weight && s.nch > 0) p.dw = dw;
  const int strips = strip_count(p.rows);
  if (d_weight && s.nch == 0)
    p.row = reinterpret_cast<float2*>(static_cast<char*>(ws) +
                                      align_up(size_t(strips) * p.dim * 4, 256));
  const bool late = p.row && meet<T>(p.d_x, p.ldx, p.d_out, p.ldo, p.rows, p.dim);
  {
    ProfScope ps("dn_add_rms_norm_bwd", stream);
    if (s.wpr == 1 && s.nch == 1)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 1, 1>), grid, block, 0, stream, p);
    else if (s.wpr == 1 && s.nch == 2)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 1, 2>), grid, block, 0, stream, p);
    else if (s.wpr == 1)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 1, 4>), grid, block, 0, stream, p);
    else if (s.nch == 1)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 4, 1>), grid, block, 0, stream, p);
    else if (s.nch == 2)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 4, 2>), grid, block, 0, stream, p);
    else if (s.nch == 4)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 4, 4>), grid, block, 0, stream, p);
    else if (late)
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 4, 0, kStats>), grid, block, 0, stream,
                         p);
    else
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 4, 0>), grid, block, 0, stream, p);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !d_weight) return e;
  if (s.nch == 0) {
    {
      ProfScope ps("dn_add_rms_norm_dw", stream);
      hipLaunchKernelGGL((norm_dw_kernel<T>), dim3(unsigned((p.dim + 255) / 256), unsigned(strips)),
                         dim3(256), 0, stream, static_cast<const T*>(p.d_out),
                         static_cast<const T*>(p.sum), static_cast<const float2*>(p.row), dw, p.ldo,
                         p.lds, p.rows, p.dim, strip_rows(p.rows));
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (late) {
      ProfScope ps("dn_add_rms_norm_bwd", stream);
      hipLaunchKernelGGL((add_rms_norm_bwd_kernel<T, TW, 4, 0, kGradient>), grid, block, 0, stream,
                         p);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    parts = strips;
  }
  ProfScope ps("dn_add_rms_norm_dw_sum", stream);
  hipLaunchKernelGGL((norm_dw_sum_kernel<TW>), dim3(unsigned((p.dim + kSumCols - 1) / kSumCols)),
                     dim3(kSumCols * kSumLanes), 0, stream, static_cast<const float*>(dw), static_cast<TW*>(d_weight), parts, p.dim);
  return hipGetLastError();
}

template <class T>
hipError_t fwd_typed(const NormArgs& p, bool wb, bool f8out, hipStream_t stream) {
  if (wb) return f8out ? fwd_go<T, bf16, true>(p, stream) : fwd_go<T, bf16, false>(p, stream);
  return f8out ? fwd_go<T, float, true>(p, stream) : fwd_go<T, float, false>(p, stream);
}

}  // namespace

hipError_t launch_add_rms_norm(const dn_add_rms_norm_args& a, hipStream_t stream) {
  NormArgs p{};
  p.x = a.x;
  p.residual = a.residual;
  p.weight = a.weight;
  p.sum = a.sum;
  p.out = a.out;
  p.scale = a.scale;
  p.ldx = a.x_stride;
  p.ldr = a.residual_stride;
  p.lds = a.sum_stride;
  p.ldo = a.out_stride;
  p.rows = int(a.rows);
  p.dim = int(a.dim);
  // Zeros up to the next multiple of 16 where the row's storage holds them (a lone
  // row's stride may be any).
  p.end = int(std::max(a.dim, std::min(int64_t(align_up(size_t(a.dim), 16)), a.out_stride)));
  p.eps = float(a.eps);
  ProfScope ps("dn_add_rms_norm", stream);
  const bool wb = a.weight_dtype == DN_BF16, f8out = a.out_dtype == DN_F8;
  return a.dtype == DN_BF16 ? fwd_typed<bf16>(p, wb, f8out, stream)
                            : fwd_typed<float>(p, wb, f8out, stream);
}

size_t add_rms_norm_bwd_workspace(const dn_add_rms_norm_bwd_args& a) {
  if (!a.d_weight) return 0;
  const Shape s = shape_of(a.rows, a.dim);
  if (s.nch > 0) return size_t(bwd_groups(a.rows, s)) * size_t(a.dim) * 4;
  const size_t strips = size_t(strip_count(a.rows));
  return align_up(strips * size_t(a.dim) * 4, 256) + size_t(a.rows) * sizeof(float2);
}

hipError_t launch_add_rms_norm_bwd(const dn_add_rms_norm_bwd_args& a, void* ws,
                                   hipStream_t stream) {
  NormBwdArgs p{};
  p.sum = a.sum;
  p.weight = a.weight;
  p.d_out = a.d_out;
  p.d_sum = a.d_sum;
  p.d_x = a.d_x;
  p.lds = a.sum_stride;
  p.ldo = a.d_out_stride;
  p.ldd = a.d_sum_stride;
  p.ldx = a.d_x_stride;
  p.rows = int(a.rows);
  p.dim = int(a.dim);
  p.eps = float(a.eps);
  const bool wb = a.weight_dtype == DN_BF16;
  if (a.dtype == DN_BF16)
    return wb ? bwd_go<bf16, bf16>(p, a.d_weight, ws, stream)
              : bwd_go<bf16, float>(p, a.d_weight, ws, stream);
  return wb ? bwd_go<float, bf16>(p, a.d_weight, ws, stream)
            : bwd_go<float, float>(p, a.d_weight, ws, stream);
}

}  // namespace dn

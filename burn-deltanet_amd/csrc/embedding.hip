// dn_embedding: out_i = scale · table[id_i]; dn_embedding_bwd: the table's gradient,
// d_table[v] = scale · Σ d_out_i over the tokens i with id_i = v, added up in a fixed
// order. An id that is not in [0, vocab), as padding has, stands for a row of zeros
// and takes no part in the gradient.
//
// Bound by memory: the rows that the ids name in, out out; d_out in, the whole
// table's gradient out (most of its rows are zeros).
//
// The gradient takes three launches and no atomics on values:
//  1. Sorting, one workgroup a range of ids. It goes over all ids twice (they are
//     few bytes beside the rows, and come from L2): first every wave counts in its
//     share of the tokens, an id at a time, what belongs to the range and what lies
//     below it, which is where the range's tokens start in the sorted order; then
//     each wave puts down its tokens where its counts say, so that an id's tokens
//     stand in their order.
//  2. Sums of 32 (8) consecutive sorted tokens each, however few or many share an id: a run
//     that lies inside is written, one that crosses an end leaves its part in the
//     workspace (fp32). Further workgroups write the rows that no token names.
//  3. The parts of the runs that cross: four waves take every fourth, and meet in order.
//
// Measured, bf16, 16384 tokens as text has them, 50000 ids of 2048 values: lookup 26 us
// (5.1 TB/s), sort 18, sums and zeros 66 (4.1 TB/s), join 7.
#include <algorithm>

#include "gemm.hpp"
#include "layer.hpp"

namespace dn {
namespace {

using gemm::load8;
using gemm::Raw8;
using gemm::store8;

constexpr int kThreads = 256;
// Workgroups of a launch: 2^32 threads or more along an axis wrap.
constexpr int64_t kMostGroups = 1 << 20;

// Threads that share a row, eight columns each: a power of two up to a workgroup.
int lanes_of(int64_t dim) {
  int n = 1;
  while (n < kThreads && n * 8 < dim) n *= 2;
  return n;
}

template <class T, class ID>
__global__ __launch_bounds__(kThreads) void embedding_kernel(const ID* ids, const T* table, T* out,
                                                             int64_t ldt, int64_t ldo, int tokens,
                                                             int vocab, int dim, int lanes,
                                                             float scale) {
  const int rows = kThreads / lanes;
  for (int64_t row = int64_t(blockIdx.x) * rows + threadIdx.x / lanes; row < tokens;
       row += int64_t(gridDim.x) * rows) {
    const int64_t id = int64_t(ids[row]);
    const bool there = id >= 0 && id < vocab;
    const T* from = table + (there ? id : 0) * ldt;
    T* to = out + row * ldo;
    for (int col = (threadIdx.x % lanes) * 8; col < dim; col += lanes * 8) {
      float v[8] = {};
      if (there) load8(from + col, v, dim - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= scale;
      store8(to + col, v, dim - col);
    }
  }
}

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kIdsAhead = 8;  // steps of 64 tokens whose ids a wave has in flight

struct SortArgs {
  const void* ids;
  int *pos, *key, *total;  // sorted: the token and its id; how many there are
  int* count;              // [vocab] tokens of each id
  int tokens, vocab, width;  // width: ids of a workgroup
};

// Between accesses of a wave's lanes to each other's values in LDS.
__device__ inline void lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

template <class ID>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(SortArgs p) {
  extern __shared__ int counts[];  // [waves][width]
  __shared__ int scan[kSortThreads], below[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, width = p.width;
  const int lo = int(blockIdx.x) * width, n = min(width, p.vocab - lo);
  const ID* ids = static_cast<const ID*>(p.ids);
  for (int i = threadIdx.x; i < kSortWaves * width; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  // A wave's share of the tokens: whole steps of 64.
  const int share = int(((int64_t(p.tokens) + kSortThreads - 1) / kSortThreads) * 64);
  const int64_t first = int64_t(wave) * share, end = min(first + share, int64_t(p.tokens));
  int* mine = counts + wave * width;
  int less = 0;
  for (int64_t i0 = first; i0 < end; i0 += 64 * kIdsAhead) {
    ID next[kIdsAhead];
#pragma unroll
    for (int j = 0; j < kIdsAhead; ++j) {
      const int64_t i = i0 + 64 * j + lane;
      next[j] = i < end ? ids[i] : ID(-1);
    }
#pragma unroll
    for (int j = 0; j < kIdsAhead; ++j) {
      const int64_t id = int64_t(next[j]);
      if (id >= 0 && id < lo) ++less;
      if (id >= lo && id < lo + n) atomicAdd(&mine[int(id - lo)], 1);
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) less += __shfl_xor(less, o);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += below[w];
  // Where each wave's tokens of each id start: ids in order, an id's waves in order.
  for (int i0 = 0; i0 < n; i0 += kSortThreads) {
    const int i = i0 + threadIdx.x;
    int t = 0;
    if (i < n)
      for (int w = 0; w < kSortWaves; ++w) {
        const int k = counts[w * width + i];
        counts[w * width + i] = t;
        t += k;
      }
    scan[threadIdx.x] = t;
    __syncthreads();
    for (int o = 1; o < kSortThreads; o *= 2) {
      const int v = int(threadIdx.x) >= o ? scan[threadIdx.x - o] : 0;
      __syncthreads();
      scan[threadIdx.x] += v;
      __syncthreads();
    }
    if (i < n) {
      const int start = base + scan[threadIdx.x] - t;
      for (int w = 0; w < kSortWaves; ++w) counts[w * width + i] += start;
      p.count[lo + i] = t;
    }
    base += scan[kSortThreads - 1];
    __syncthreads();
  }
  if (blockIdx.x + 1 == gridDim.x && threadIdx.x == 0) *p.total = base;
  // Tokens of one id within a step stand in the order of their lanes. Lanes of one id find
  // each other by the bits of their ids (one ballot a bit: a loop over the ids of a step
  // took 81 us in place of 18 for 16384 tokens as text has them, half of whom one range
  // holds).
  int bits = 0;
  while ((1 << bits) < n) ++bits;
  for (int64_t i0 = first; i0 < end; i0 += 64 * kIdsAhead) {
    ID next[kIdsAhead];
#pragma unroll
    for (int j = 0; j < kIdsAhead; ++j) {
      const int64_t i = i0 + 64 * j + lane;
      next[j] = i < end ? ids[i] : ID(-1);
    }
#pragma unroll
    for (int j = 0; j < kIdsAhead; ++j) {
      const int64_t id = int64_t(next[j]);
      const bool in = id >= lo && id < lo + n;
      uint64_t same = __ballot(in);
      if (!same) continue;
      const int key = in ? int(id - lo) : 0;
      for (int b = 0; b < bits; ++b) {
        const bool set = key >> b & 1;
        const uint64_t all = __ballot(set);
        same &= set ? all : ~all;
      }
      const int rank = int(__popcll(same & ((uint64_t(1) << lane) - 1)));
      int at = 0;
      if (in) {
        at = mine[key] + rank;
        p.pos[at] = int(i0 + 64 * j + lane);
        p.key[at] = lo + key;
      }
      // The first lane of an id moves its place on: behind the others' reads, and before
      // those of the next step.
      lds_fence();
      if (in && rank == 0) mine[key] = at + int(__popcll(same));
      lds_fence();
    }
  }
}

struct SumArgs {
  const void* d_out;
  void* d_table;
  const int *pos, *key, *total, *count;
  int64_t groups;  // of workgroups that sum; the others write zeros
  int vocab;
  float* part;  // [runs][2][dim]: what a run of tokens leaves at its start, at its end
  int64_t ldd, ldt;
  int dim, lanes, run;  // run: sorted tokens of a sum
  float scale;
};

constexpr int kZeroRows = 32;  // of a workgroup that writes zeros

template <class T>
__global__ __launch_bounds__(kThreads) void embedding_sum_kernel(SumArgs p) {
  if (blockIdx.x >= p.groups) {  // rows of ids that no token has
    const int64_t first = (blockIdx.x - p.groups) * kZeroRows;
    const int rows = kThreads / p.lanes;
    const int col = (threadIdx.x % p.lanes + int(blockIdx.y) * p.lanes) * 8, valid = p.dim - col;
    const float zero[8] = {};
    if (valid <= 0) return;
    for (int64_t r = first + threadIdx.x / p.lanes; r < min(first + kZeroRows, int64_t(p.vocab));
         r += rows)
      if (!p.count[r]) store8(static_cast<T*>(p.d_table) + r * p.ldt + col, zero, valid);
    return;
  }
  const int64_t run = int64_t(blockIdx.x) * (kThreads / p.lanes) + threadIdx.x / p.lanes;
  const int total = *p.total;
  const int64_t p0 = run * p.run;
  if (p0 >= total) return;
  const int end = int(min(p0 + p.run, int64_t(total))), begin = int(p0);
  const int col = (threadIdx.x % p.lanes + int(blockIdx.y) * p.lanes) * 8, valid = p.dim - col;
  if (valid <= 0) return;
  const T* d = static_cast<const T*>(p.d_out) + col;
  // Whether the first id's tokens began before, and the last one's go on.
  bool open = begin > 0 && p.key[begin - 1] == p.key[begin];
  const bool on = end < total && p.key[end] == p.key[end - 1];
  float acc[8] = {};
  int key = p.key[begin];
  auto flush = [&](bool head, bool tail) {
    if (head || tail) {
      store8(p.part + (run * 2 + (head ? 0 : 1)) * p.dim + col, acc, valid);
    } else {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = acc[i] * p.scale;
      store8(static_cast<T*>(p.d_table) + int64_t(key) * p.ldt + col, v, valid);
    }
  };
  constexpr int kAhead = 8;
  for (int i = begin; i < end; i += kAhead) {
    Raw8<T> w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      w[j].load(d + int64_t(p.pos[min(i + j, end - 1)]) * p.ldd, valid);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i + j >= end) break;
      const int k = p.key[i + j];
      if (k != key) {
        flush(open, false);
        open = false;
        key = k;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      }
      float v[8];
      w[j].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[e];
    }
  }
  flush(open, on);
}

// An id whose tokens cross runs: the part at the end of the first run, then those at
// the starts of the following ones. Four lanes of rows a column, which meet in LDS.
constexpr int kJoinCols = 256;
template <class T>
__global__ __launch_bounds__(kThreads) void embedding_join_kernel(SumArgs p) {
  const int total = *p.total;
  const int64_t run = blockIdx.x, begin = run * p.run, end = begin + p.run;
  if (end >= total) return;
  const int key = p.key[end - 1];
  if (p.key[end] != key) return;                                             // ends here
  if (p.key[begin] == key && begin > 0 && p.key[begin - 1] == key) return;  // began before
  const int c = threadIdx.x & 63, lane = threadIdx.x >> 6;
  const int col = (int(blockIdx.y) * 64 + c) * 4, valid = p.dim - col;
  // Behind the last run that starts with the id: between `past` and `top`, by 64 places at
  // a time, as keys stand in order. Found first, so that the parts are read ahead: a walk
  // that asks each run took 333 us in place of 191 for 65536 tokens of 64 values, 60 % of
  // them of one id.
  int64_t past = run + 1, top = (int64_t(total) + p.run - 1) / p.run;
  for (int64_t step = 1; past < top; step = (top - past + 63) / 64) {
    const int64_t r = past + c * step;
    const int same = int(__popcll(__ballot(r < top && p.key[r * p.run] == key)));
    if (same == 0) break;
    if (same < 64) top = min(top, past + same * step);
    past += (same - 1) * step + 1;
  }
  float acc[4] = {};
  const auto add = [&](int64_t r, int side) {
    const float* at = p.part + (r * 2 + side) * p.dim + col;
    if (valid >= 4) {
      float x[4];
      __builtin_memcpy(x, at, 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += x[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < valid) acc[i] += at[i];
    }
  };
  if (lane == 0) add(run, 1);
#pragma unroll 8
  for (int64_t r = run + 1 + lane; r < past; r += 4) add(r, 0);
  __shared__ float lds[4][kJoinCols];
#pragma unroll
  for (int i = 0; i < 4; ++i) lds[lane][c * 4 + i] = acc[i];
  __syncthreads();
  const int out = int(blockIdx.y) * kJoinCols + threadIdx.x;
  if (out < p.dim)
    st(static_cast<T*>(p.d_table), size_t(int64_t(key) * p.ldt + out),
       (lds[0][threadIdx.x] + lds[1][threadIdx.x] + lds[2][threadIdx.x] + lds[3][threadIdx.x]) *
           p.scale);
}

// Ids of a sorting workgroup: one for every CU, but no more than 512 ids each (their
// counts by wave are 32 KB of LDS).
int sort_width(int64_t vocab) {
  const int64_t all = (vocab + device_cu_count() - 1) / device_cu_count();
  return int(std::max<int64_t>(1, std::min<int64_t>(all, 512)));
}

// Sorted tokens of a sum: 32, or 8 up to 4096 tokens where that leaves CUs without two
// workgroups. Short sums end sooner, but leave more parts, which one workgroup an id and
// 256 columns joins. With 8 and with 32, whole calls in bf16 and us: 3000 tokens of 256
// values 19 and 25, 4096 21 and 26, 8192 28 and 27, 65536 of 64 112 and 68; where 60 % of
// the tokens have one id 38 and 36, 45 and 39, 76 and 53, 438 and 191.
int run_of(const dn_embedding_bwd_args& a) {
  const int64_t lanes = lanes_of(a.dim), at_once = kThreads / lanes;
  const int64_t groups = a.tokens / (32 * at_once) * ((a.dim + lanes * 8 - 1) / (lanes * 8));
  return a.tokens > 4096 || groups >= 2 * device_cu_count() ? 32 : 8;
}

struct Layout {
  size_t pos, key, total, count, part, bytes;
};
Layout layout_of(const dn_embedding_bwd_args& a) {
  Layout l{};
  const size_t n = size_t(a.tokens), run = size_t(run_of(a)), runs = (n + run - 1) / run;
  l.pos = 0;
  l.key = align_up(n * 4, 256);
  l.total = l.key + align_up(n * 4, 256);
  l.count = l.total + 256;
  l.part = l.count + align_up(size_t(a.vocab) * 4, 256);
  l.bytes = l.part + (runs > 1 ? runs * 2 * size_t(a.dim) * 4 : 0);
  return l;
}

template <class T, class ID>
hipError_t bwd_go(const dn_embedding_bwd_args& a, void* ws, hipStream_t stream) {
  const Layout l = layout_of(a);
  char* base = static_cast<char*>(ws);
  SortArgs s{};
  s.ids = a.ids;
  s.pos = reinterpret_cast<int*>(base + l.pos);
  s.key = reinterpret_cast<int*>(base + l.key);
  s.total = reinterpret_cast<int*>(base + l.total);
  s.count = reinterpret_cast<int*>(base + l.count);
  s.tokens = int(a.tokens);
  s.vocab = int(a.vocab);
  s.width = sort_width(a.vocab);
  {
    ProfScope ps("dn_embedding_sort", stream);
    hipLaunchKernelGGL((embedding_sort_kernel<ID>),
                       dim3(unsigned((a.vocab + s.width - 1) / s.width)), dim3(kSortThreads),
                       size_t(kSortWaves) * size_t(s.width) * 4, stream, s);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  SumArgs p{};
  p.d_out = a.d_out;
  p.d_table = a.d_table;
  p.pos = s.pos;
  p.key = s.key;
  p.total = s.total;
  p.count = s.count;
  p.vocab = s.vocab;
  p.part = reinterpret_cast<float*>(base + l.part);
  p.ldd = a.d_out_stride;
  p.ldt = a.d_table_stride;
  p.dim = int(a.dim);
  p.lanes = lanes_of(a.dim);
  p.scale = float(a.scale);
  p.run = run_of(a);
  const int64_t runs = (a.tokens + p.run - 1) / p.run, at_once = kThreads / p.lanes;
  p.groups = (runs + at_once - 1) / at_once;
  {
    ProfScope ps("dn_embedding_sum", stream);
    hipLaunchKernelGGL((embedding_sum_kernel<T>),
                       dim3(unsigned(p.groups + (a.vocab + kZeroRows - 1) / kZeroRows),
                            unsigned((a.dim + p.lanes * 8 - 1) / (p.lanes * 8))),
                       dim3(kThreads), 0, stream, p);
  }
  e = hipGetLastError();
  if (e != hipSuccess || runs <= 1) return e;
  ProfScope ps("dn_embedding_join", stream);
  hipLaunchKernelGGL((embedding_join_kernel<T>),
                     dim3(unsigned(runs - 1), unsigned((a.dim + kJoinCols - 1) / kJoinCols)),
                     dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

template <class T, class ID>
hipError_t fwd_go(const dn_embedding_args& a, hipStream_t stream) {
  const int lanes = lanes_of(a.dim), rows = kThreads / lanes;
  hipLaunchKernelGGL((embedding_kernel<T, ID>), dim3(unsigned(std::min<int64_t>((a.tokens + rows - 1) / rows, kMostGroups))),
                     dim3(kThreads), 0, stream, static_cast<const ID*>(a.ids),
                     static_cast<const T*>(a.table), static_cast<T*>(a.out), a.table_stride,
                     a.out_stride, int(a.tokens), int(a.vocab), int(a.dim), lanes, float(a.scale));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_embedding(const dn_embedding_args& a, hipStream_t stream) {
  ProfScope ps("dn_embedding", stream);
  if (a.dtype == DN_BF16)
    return a.wide_ids ? fwd_go<bf16, int64_t>(a, stream) : fwd_go<bf16, int32_t>(a, stream);
  return a.wide_ids ? fwd_go<float, int64_t>(a, stream) : fwd_go<float, int32_t>(a, stream);
}

size_t embedding_bwd_workspace(const dn_embedding_bwd_args& a) { return layout_of(a).bytes; }

hipError_t launch_embedding_bwd(const dn_embedding_bwd_args& a, void* ws, hipStream_t stream) {
  if (a.dtype == DN_BF16)
    return a.wide_ids ? bwd_go<bf16, int64_t>(a, ws, stream) : bwd_go<bf16, int32_t>(a, ws, stream);
  return a.wide_ids ? bwd_go<float, int64_t>(a, ws, stream) : bwd_go<float, int32_t>(a, ws, stream);
}

}  // namespace dn

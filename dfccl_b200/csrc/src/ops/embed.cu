// Embedding of tokens: y = scale w[id] + p[position] per token, and the gradients of both tables by sorted tokens.
// The reference has no counterpart (it is a collective library); the GPT-2 workload's first stage uses these.
//
// Forward: a gather, bound by memory (or by its launch, for few tokens): 16 bytes per thread and access where rows allow it.
// Backward: dw[v] = scale sum over tokens with id v of g, in fp32, in the order of the tokens, rounded once.  Three launches:
//   1. one cluster of eight blocks per table sorts (id, token) by id - a stable radix sort, eight bits a pass, whose counts meet in
//      distributed shared memory - while the other blocks clear the gradients, which is what the time goes into: most rows of a
//      large table have no token;
//   2. the sorted tokens in stretches: rows whose tokens lie inside one are summed and stored, others leave one or two sums;
//   3. those are added up, stretch by stretch.
// No result is added to by atomics, so a call repeats itself bit by bit.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <algorithm>
#include "dfccl_ops.h"
#include "../common/log.h"
#include "../gemm/tc_common.h"

namespace dfccl {
namespace {

constexpr int SORT_CTAS = 8, SORT_THREADS = 1024, SORT_WARPS = SORT_CTAS * SORT_THREADS / 32;
constexpr int CLEAR_CLUSTERS = 16;             // beside the sorting ones: 128 blocks of 1024 threads
constexpr int SUM_GROUPS = 8;                  // of threads that share a row's stretches in the last step
constexpr int MAX_TABLES = 2;

template <typename... P, typename... A>
cudaError_t launchBehind(void (*kernel)(P...), dim3 grid, int block, int cluster, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension; at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, (P)args...);
}

__device__ __forceinline__ long long intAt(const void* p, int wide, size_t i) { return wide ? ((const long long*)p)[i] : ((const int*)p)[i]; }

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }

// E elements of a row: one access of E sizeof(T) bytes (16, or one element where rows are not on that grid).
template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
  T v[E];
};

struct Forward {
  const void* ids; const void* positions;        // positions may be null
  const void* w; const void* p;
  void* out;
  int wideIds, widePositions;
  int n, packs;                                  // packs of E elements per row
  long long rows, prows, ldw, ldp;               // in elements
  float scale;
};

// A thread takes U packs, a block apart, so that its loads overlap.
template <typename T, int E, int U>
__global__ void __launch_bounds__(256) embedForwardKernel(const Forward a) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  using P = Pack<T, E>;
  const long long total = (long long)a.n * a.packs, base = (long long)blockIdx.x * 256 * U + threadIdx.x;
  P w[U], p[U];
  bool bad[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = base + u * 256;
    if (i >= total) break;
    const int row = (int)(i / a.packs), c = (int)(i - (long long)row * a.packs);
    const long long id = intAt(a.ids, a.wideIds, row), at = a.positions ? intAt(a.positions, a.widePositions, row) : 0;
    bad[u] = id < 0 || id >= a.rows || (a.positions && (at < 0 || at >= a.prows));
    if (bad[u]) continue;
    w[u] = *(const P*)((const T*)a.w + id * a.ldw + (long long)c * E);
    if (a.positions) p[u] = *(const P*)((const T*)a.p + at * a.ldp + (long long)c * E);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = base + u * 256;
    if (i >= total) break;
    P o;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float y = __int_as_float(0x7fffffff);            // a token outside the table: not a number
      if (!bad[u]) y = a.positions ? fmaf(toFloat(w[u].v[e]), a.scale, toFloat(p[u].v[e])) : toFloat(w[u].v[e]) * a.scale;
      o.v[e] = fromFloat<T>(y);
    }
    ((P*)a.out)[i] = o;
  }
}

struct Table {
  const void* ids;
  int wide;
  int rows;                       // of the table; also the key of tokens without a gradient, behind all others
  long long padding;              // the id without a gradient, or -1
  int passes;                     // of eight bits
  uint2* buf[2];                  // (key, token) [n]; sorted into buf[passes & 1]
  void* grad;
  size_t gradBytes;
  float scale;
  float* sums;                    // [stretches][2][d]: of the row that goes on from the stretch in front, of the one that goes on behind
};
struct Backward {
  Table t[MAX_TABLES];
  int tables, n, d, stretch, stretches;
  const void* g;
};

__device__ __forceinline__ uint2 itemAt(const Table& t, int pass, int i) {
  if (pass) return __ldcg(&t.buf[pass & 1][i]);
  const long long id = intAt(t.ids, t.wide, i);
  return make_uint2(id >= 0 && id < t.rows && id != t.padding ? (uint32_t)id : (uint32_t)t.rows, (uint32_t)i);
}

// Every warp has a range of the items of its own; its counts of the digits, summed over the ranges in front, are where its items go.
__device__ void sortCluster(const Table& t, int n) {
  namespace cg = cooperative_groups;
  __shared__ int hist[32][256];
  __shared__ int total[256], scan[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int range = ((n + SORT_WARPS - 1) / SORT_WARPS + 31) / 32 * 32;
  const long long begin = (long long)(cta * 32 + warp) * range;
  const int first = (int)min((long long)n, begin), last = (int)min((long long)n, begin + range);
  for (int pass = 0; pass < t.passes; ++pass) {
    const int shift = pass * 8;
    uint2* dst = t.buf[(pass + 1) & 1];
    for (int i = lane; i < 256; i += 32) hist[warp][i] = 0;
    __syncwarp();
    for (int i = first; i < last; i += 32) {
      const bool in = i + lane < last;
      const int digit = in ? (int)(itemAt(t, pass, i + lane).x >> shift & 255) : 256;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      if (in && (same & ((1u << lane) - 1)) == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < 256) {                             // this block's ranges, in order
      int run = 0;
      for (int w = 0; w < 32; ++w) { const int c = hist[w][threadIdx.x]; hist[w][threadIdx.x] = run; run += c; }
      total[threadIdx.x] = run;
    }
    cluster.sync();
    int offset = 0;
    if (threadIdx.x < 256) {                             // the blocks in front, and all smaller digits
      int before = 0, all = 0;
      for (int c = 0; c < SORT_CTAS; ++c) {
        const int x = *cluster.map_shared_rank(&total[threadIdx.x], c);
        if (c < cta) before += x;
        all += x;
      }
      int inc = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += x; }
      if (lane == 31) scan[warp] = inc;
      offset = before + inc - all;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
      for (int w = 0; w < warp; ++w) offset += scan[w];
      for (int w = 0; w < 32; ++w) hist[w][threadIdx.x] += offset;
    }
    __syncthreads();
    for (int i = first; i < last; i += 32) {
      const bool in = i + lane < last;
      const uint2 item = in ? itemAt(t, pass, i + lane) : make_uint2(0u, 0u);
      const int digit = in ? (int)(item.x >> shift & 255) : 256;
      const uint32_t same = __match_any_sync(0xffffffffu, digit), before = same & ((1u << lane) - 1);
      if (in) dst[hist[warp][digit] + __popc(before)] = item;
      __syncwarp();
      if (in && before == 0) hist[warp][digit] += __popc(same);
      __syncwarp();
    }
    __threadfence();
    cluster.sync();                                      // all items in place; all counts read
  }
}

__global__ void __launch_bounds__(SORT_THREADS) sortAndClearKernel(const Backward a) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const int cluster = blockIdx.x / SORT_CTAS;
  if (cluster < a.tables) { sortCluster(a.t[cluster], a.n); return; }
  const size_t thread = (size_t)(blockIdx.x - a.tables * SORT_CTAS) * SORT_THREADS + threadIdx.x;
  const size_t threads = (size_t)(gridDim.x - a.tables * SORT_CTAS) * SORT_THREADS;
  for (int k = 0; k < a.tables; ++k) {
    uint4* dst = (uint4*)a.t[k].grad;
    const size_t packs = a.t[k].gradBytes / 16;
    for (size_t i = thread; i < packs; i += threads) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    for (size_t i = packs * 16 + thread; i < a.t[k].gradBytes; i += threads) ((uint8_t*)a.t[k].grad)[i] = 0;
  }
}

// A block sums the tokens of a stretch for its columns (E per thread), row after row.
template <typename T, int E>
__global__ void __launch_bounds__(128) sumStretchKernel(const Backward a) {
  constexpr int MAX = 128, AHEAD = 8;
  __shared__ uint32_t keys[MAX + 2], tokens[MAX];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const Table& t = a.t[blockIdx.z];
  const uint2* items = t.buf[t.passes & 1];
  const int start = blockIdx.x * a.stretch, count = min(a.stretch, a.n - start);
  for (int i = (int)threadIdx.x - 1; i <= count; i += 128) {             // and the keys on either side
    const int at = start + i;
    const uint2 item = at >= 0 && at < a.n ? __ldcg(&items[at]) : make_uint2(0xffffffffu, 0u);
    keys[i + 1] = item.x;
    if (i >= 0 && i < count) tokens[i] = item.y;
  }
  __syncthreads();
  const int col = (blockIdx.y * 128 + threadIdx.x) * E;
  if (col >= a.d) return;
  using P = Pack<T, E>;
  const T* g = (const T*)a.g + col;
  const uint32_t none = (uint32_t)t.rows;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  bool head = keys[0] == keys[1];
  for (int i = 0; i < count; i += AHEAD) {
    P p[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) if (i + u < count && keys[i + u + 1] != none) p[u] = *(const P*)(g + (size_t)tokens[i + u] * a.d);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = i + u;
      if (j >= count || keys[j + 1] == none) return;                     // (tokens without a gradient are the last)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += toFloat(p[u].v[e]);
      const bool goesOn = keys[j + 2] == keys[j + 1];
      if (goesOn && j + 1 < count) continue;
      if (head || goesOn) {                                              // not all of the row
        float* s = t.sums + ((size_t)blockIdx.x * 2 + (head ? 0 : 1)) * a.d + col;
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] = acc[e];
      } else {
        P o;
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = fromFloat<T>(acc[e] * t.scale);
        *(P*)((T*)t.grad + (size_t)keys[j + 1] * a.d + col) = o;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      head = false;
    }
  }
}

// Rows that go on behind the stretch in which they begin: a block per such stretch and 32 packs of columns; SUM_GROUPS groups of threads
// add up a part of the row's stretches each.
template <typename T, int E>
__global__ void __launch_bounds__(32 * SUM_GROUPS) joinStretchKernel(const Backward a) {
  __shared__ float part[SUM_GROUPS][32 * E];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const Table& t = a.t[blockIdx.z];
  const uint2* items = t.buf[t.passes & 1];
  const int start = blockIdx.x * a.stretch, end = start + a.stretch;     // the last stretch has nothing behind it
  const uint32_t key = __ldcg(&items[end - 1]).x;
  if (key == (uint32_t)t.rows || __ldcg(&items[end]).x != key) return;
  if (start > 0 && __ldcg(&items[start]).x == key && __ldcg(&items[start - 1]).x == key) return;      // it began further in front
  int lo = end, hi = a.n;                                                // the first item behind the row
  while (lo < hi) { const int mid = (lo + hi) >> 1; if (__ldcg(&items[mid]).x <= key) lo = mid + 1; else hi = mid; }
  const int first = blockIdx.x + 1, count = (lo - 1) / a.stretch - first + 1;      // stretches that begin with it
  const int group = threadIdx.x >> 5, lane = threadIdx.x & 31, col = (blockIdx.y * 32 + lane) * E;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (col < a.d) {
    if (group == 0) {
      const float* s = t.sums + ((size_t)blockIdx.x * 2 + 1) * a.d + col;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = s[e];
    }
    const int per = (count + SUM_GROUPS - 1) / SUM_GROUPS, from = group * per, to = min(count, from + per);
    const float* s = t.sums + (size_t)first * 2 * a.d + col;
#pragma unroll 4
    for (int i = from; i < to; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += s[(size_t)i * 2 * a.d + e];
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) part[group][lane * E + e] = acc[e];
  __syncthreads();
  if (group || col >= a.d) return;
  Pack<T, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < SUM_GROUPS; ++k) s += part[k][lane * E + e];
    o.v[e] = fromFloat<T>(s * t.scale);
  }
  *(Pack<T, E>*)((T*)t.grad + (size_t)key * a.d + col) = o;
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }
// Tokens of a stretch: 16, more (up to 128) once there are more than 4096 stretches.
int stretchOf(int n) { return std::min(128, std::max(16, (n + 4095) / 4096)); }
struct Layout { size_t items, sums; };
Layout layoutOf(int n, int d) {
  const int s = stretchOf(n);
  return Layout{up256((size_t)n * sizeof(uint2)), up256((size_t)((n + s - 1) / s) * 2 * d * sizeof(float))};
}

template <typename T, int E>
ncclResult_t forward(const Forward& a, cudaStream_t stream) {
  const long long total = (long long)a.n * a.packs;
  // Four packs a thread where that still leaves every SM two blocks.
  if (total >= 4ll * 256 * 296) {
    CUDACHECK(launchBehind(embedForwardKernel<T, E, 4>, dim3((unsigned)((total + 1023) / 1024)), 256, 1, stream, a));
  } else {
    CUDACHECK(launchBehind(embedForwardKernel<T, E, 1>, dim3((unsigned)((total + 255) / 256)), 256, 1, stream, a));
  }
  return ncclSuccess;
}

template <typename T, int E>
ncclResult_t backward(const Backward& a, cudaStream_t stream) {
  CUDACHECK(launchBehind(sortAndClearKernel, dim3(SORT_CTAS * (a.tables + CLEAR_CLUSTERS)), SORT_THREADS, SORT_CTAS, stream, a));
  const int packs = a.d / E;
  CUDACHECK(launchBehind(sumStretchKernel<T, E>, dim3(a.stretches, (packs + 127) / 128, a.tables), 128, 1, stream, a));
  if (a.stretches > 1)
    CUDACHECK(launchBehind(joinStretchKernel<T, E>, dim3(a.stretches - 1, (packs + 31) / 32, a.tables), 32 * SUM_GROUPS, 1, stream, a));
  return ncclSuccess;
}

int typeBytes(int t) { return t == ncclFloat32 ? 4 : t == ncclBfloat16 || t == ncclFloat16 ? 2 : 0; }

}  // namespace
}  // namespace dfccl

using namespace dfccl;
#define DF_API extern "C" __attribute__((visibility("default")))

DF_API ncclResult_t dfcclEmbeddingForward(const void* ids, int wideIds, int n, const void* w, int64_t rows, int64_t ldw, const void* positions, int widePositions,
                                          const void* p, int64_t prows, int64_t ldp, void* out, int d, int type, float scale, cudaStream_t stream) {
  const int bytes = typeBytes(type);
  if (n <= 0 || d <= 0 || rows <= 0 || !bytes || !ids || !w || !out || ldw < d || (positions && (!p || prows <= 0 || ldp < d))) return ncclInvalidArgument;
  Forward a{ids, positions, w, p, out, wideIds, widePositions, n, 0, rows, prows, ldw, ldp, scale};
  const uintptr_t grid = (uintptr_t)w | (uintptr_t)out | (uintptr_t)(ldw * bytes) | (uintptr_t)((size_t)d * bytes) |
                         (positions ? (uintptr_t)p | (uintptr_t)(ldp * bytes) : 0);
  const bool whole = (grid & 15) == 0;
  a.packs = whole ? d / (16 / bytes) : d;
  if ((long long)n * a.packs > 0x7fffffffll * 256) return ncclInvalidArgument;
  if (type == ncclFloat32) return whole ? forward<float, 4>(a, stream) : forward<float, 1>(a, stream);
  if (type == ncclBfloat16) return whole ? forward<__nv_bfloat16, 8>(a, stream) : forward<__nv_bfloat16, 1>(a, stream);
  return whole ? forward<__half, 8>(a, stream) : forward<__half, 1>(a, stream);
}

DF_API size_t dfcclEmbeddingBackwardWork(int n, int d, int tables) {
  if (n <= 0 || d <= 0 || tables < 1 || tables > MAX_TABLES) return 0;
  const Layout l = layoutOf(n, d);
  return tables * (2 * l.items + l.sums);
}

DF_API ncclResult_t dfcclEmbeddingBackward(const void* g, int n, int d, int type, const void* ids, int wideIds, int64_t padding, float scale, void* gw, int64_t rows,
                                           const void* positions, int widePositions, void* gp, int64_t prows, void* work, cudaStream_t stream) {
  const int bytes = typeBytes(type);
  if (n <= 0 || d <= 0 || !bytes || !g || !work || !(gw || gp) || (gw && (!ids || rows <= 0 || rows > 0x7ffffff0ll)) ||
      (gp && (!positions || prows <= 0 || prows > 0x7ffffff0ll)) || (((uintptr_t)gw | (uintptr_t)gp | (uintptr_t)work) & 15))
    return ncclInvalidArgument;
  const Layout l = layoutOf(n, d);
  Backward a;
  a.tables = 0; a.n = n; a.d = d; a.stretch = stretchOf(n); a.stretches = (n + a.stretch - 1) / a.stretch; a.g = g;
  uint8_t* at = (uint8_t*)work;
  auto add = [&](const void* idx, int wide, int64_t count, int64_t pad, void* grad, float s) {
    Table& t = a.t[a.tables++];
    t.ids = idx; t.wide = wide; t.rows = (int)count; t.padding = pad; t.grad = grad; t.gradBytes = (size_t)count * d * bytes; t.scale = s;
    t.passes = 1;
    while (t.passes < 4 && (uint64_t)count >> (8 * t.passes)) ++t.passes;
    t.buf[0] = (uint2*)at; t.buf[1] = (uint2*)(at + l.items); t.sums = (float*)(at + 2 * l.items);
    at += 2 * l.items + l.sums;
  };
  if (gw) add(ids, wideIds, rows, padding, gw, scale);
  if (gp) add(positions, widePositions, prows, -1, gp, 1.f);
  const bool whole = (((uintptr_t)g | (uintptr_t)((size_t)d * bytes)) & 15) == 0;
  if (type == ncclFloat32) return whole ? backward<float, 4>(a, stream) : backward<float, 1>(a, stream);
  if (type == ncclBfloat16) return whole ? backward<__nv_bfloat16, 8>(a, stream) : backward<__nv_bfloat16, 1>(a, stream);
  return whole ? backward<__half, 8>(a, stream) : backward<__half, 1>(a, stream);
}

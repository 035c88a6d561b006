// Embedding of tokens: y = scale w[id] + p[position] per token, and the gradients of both tables by sorted tokens.
// The reference has no counterpart (it is a collective library); the GPT-2 workload's first stage uses these.
//
// Forward: a gather, bound by memory (or by its launch, for few tokens): 16 bytes per thread and access where rows allow it.  131072 tokens of
// 1024 bf16 with positions: 60 us, 537 MB to and from L2 and 300 of DRAM; 8192: 6.7; one: 2.
// Backward: dw[v] = scale sum over tokens with id v of g, in fp32, in the order of the tokens within a stretch of them, then of the stretches (by eight
// warps where there are more than eight of them, each a share in its order), rounded once.  Four launches:
//   1. and 2. one cluster of eight blocks per table sorts (id, token) by id - a stable radix sort, eight bits a pass, whose counts meet in
//      distributed shared memory - while another launch clears the gradients, which is what the time goes into: most rows of a
//      large table have no token (50257 x 1024 bf16: 17 us; the sort of 8192 tokens 15, of 131072 49);
//   3. the sorted tokens in stretches: rows whose tokens lie inside one are summed and stored, others leave one or two sums (8192 x 1024 and
//      positions: 9 us; 131072: 90, 600 MB at 6.7 TB/s: g is read once per table);
//   4. those are added up, stretch by stretch (8 us; 16).
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
#include "embed.h"

namespace dfccl {
namespace {

constexpr int SORT_CTAS = 8, SORT_THREADS = 1024, SORT_WARPS = SORT_CTAS * SORT_THREADS / 32;
constexpr int CLEAR_BLOCKS = 128;
constexpr int JOIN_WARPS = 8;
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
  int lanes, turns;                              // of a warp that share a row (a power of two); rows one after the other
  long long rows, prows, ldw, ldp;               // in elements
  float scale;
};

// Two elements of 16 bits at a time, rounded by one instruction.
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using Type = __nv_bfloat162;
  static __device__ __forceinline__ float2 wide(Type v) { return __bfloat1622float2(v); }
  static __device__ __forceinline__ Type narrow(float a, float b) { return __floats2bfloat162_rn(a, b); }
};
template <> struct Pair<__half> {
  using Type = __half2;
  static __device__ __forceinline__ float2 wide(Type v) { return __half22float2(v); }
  static __device__ __forceinline__ Type narrow(float a, float b) { return __floats2half2_rn(a, b); }
};

// What becomes of a row: copied (scale 1), the position's row added (scale 1), or scaled in general.
enum EmbedForm { EMBED_COPY, EMBED_ADD, EMBED_SCALE, EMBED_SCALE_ADD };
template <typename T, int E, int FORM>
__device__ __forceinline__ void combine(const Pack<T, E>& x, const Pack<T, E>& y, float scale, Pack<T, E>& o) {
  if (FORM == EMBED_COPY) { o = x; return; }
  if constexpr (sizeof(T) == 2 && E > 1) {
    using P2 = typename Pair<T>::Type;
    const P2* a = (const P2*)x.v; const P2* b = (const P2*)y.v;
    P2* r = (P2*)o.v;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      // (a sum of two elements in 32 bits, rounded to 16, is the sum rounded once: 24 bits are twice those of the type and two)
      if (FORM == EMBED_ADD) { r[e] = __hadd2(a[e], b[e]); continue; }
      const float2 f = Pair<T>::wide(a[e]);
      if (FORM == EMBED_SCALE) { r[e] = Pair<T>::narrow(f.x * scale, f.y * scale); continue; }
      const float2 h = Pair<T>::wide(b[e]);
      r[e] = Pair<T>::narrow(fmaf(f.x, scale, h.x), fmaf(f.y, scale, h.y));
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = fromFloat<T>(FORM == EMBED_SCALE ? toFloat(x.v[e]) * scale : fmaf(toFloat(x.v[e]), scale, toFloat(y.v[e])));
  }
}

// A warp takes `turns` rows one after the other (`turns` times as many side by side where rows are short), 32 at most: their tokens are one
// load in front, and four packs of a lane are on their way at a time (a row of 1024 bf16 is four).
template <typename T, int E, int FORM>
__global__ void __launch_bounds__(256) embedForwardKernel(const Forward a) {
  constexpr int U = 4;
  constexpr bool POS = FORM == EMBED_ADD || FORM == EMBED_SCALE_ADD;
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  using P = Pack<T, E>;
  const int lane = threadIdx.x & 31, perWarp = 32 / a.lanes, sub = lane / a.lanes, own = lane & (a.lanes - 1);
  const long long row0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * perWarp * a.turns;
  const int rows = (int)max(0ll, min((long long)perWarp * a.turns, a.n - row0));
  long long mine = 0, minePos = 0;
  if (lane < rows) {
    mine = intAt(a.ids, a.wideIds, row0 + lane);
    if (POS) minePos = intAt(a.positions, a.widePositions, row0 + lane);
    if (mine < 0 || mine >= a.rows || (POS && (minePos < 0 || minePos >= a.prows))) mine = -1;
  }
  for (int k = 0; k < rows; k += perWarp) {
    const long long id = __shfl_sync(0xffffffffu, mine, k + sub), at = POS ? __shfl_sync(0xffffffffu, minePos, k + sub) : 0;
    if (k + sub >= rows) continue;
    P* out = (P*)a.out + (row0 + k + sub) * a.packs;
    if (id < 0) {                                            // a token outside the table: not a number
      P o;
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] = fromFloat<T>(__int_as_float(0x7fffffff));
      for (int c = own; c < a.packs; c += a.lanes) out[c] = o;
      continue;
    }
    const P* w = (const P*)((const T*)a.w + id * a.ldw);
    const P* p = (const P*)((const T*)a.p + at * a.ldp);
    for (int c = own; c < a.packs; c += U * a.lanes) {
      P x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(c + u * a.lanes, a.packs - 1);     // (no branch between the loads)
        x[u] = w[i];
        if (POS) y[u] = p[i];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = c + u * a.lanes;
        if (i >= a.packs) break;
        P o;
        combine<T, E, FORM>(x[u], y[u], a.scale, o);
        out[i] = o;
      }
    }
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
  // sums by themselves instead of a gradient: fp32 rows [n][d], used where `where` [rows] says
  float* compact;
  int* where;
  const float* weights;           // [n] of the tokens there, times gout of their row of g where given
  const float* gout;
  int goutStride, perRow;         // tokens that share a row of g
  bool dense;                     // sums at the number of their token
};
struct Backward {
  Table t[MAX_TABLES];
  int tables, n, d, stretch, stretches;
  const void* g;
};

// The lanes with an item of the same digit, bit by bit.
__device__ __forceinline__ uint32_t sameDigit(int digit, bool in) {
  uint32_t same = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint32_t set = __ballot_sync(0xffffffffu, digit >> b & 1);
    same &= digit >> b & 1 ? set : ~set;
  }
  return same;
}

// Every warp has a range of the items of its own; the counts of its digits, behind those of smaller digits and of the ranges in front,
// are where its items go.  Eight items of a lane are on their way at a time.
__device__ void sortCluster(const Table& t, int n) {
  namespace cg = cooperative_groups;
  constexpr int AHEAD = 8;
  __shared__ int hist[32][256];
  __shared__ int quarter[4][256], total[256], scan[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, digit = threadIdx.x & 255, part = threadIdx.x >> 8;
  const int range = ((n + SORT_WARPS - 1) / SORT_WARPS + 31) / 32 * 32;
  const long long begin = (long long)(cta * 32 + warp) * range;
  const int first = (int)min((long long)n, begin), last = (int)min((long long)n, begin + range);
  for (int pass = 0; pass < t.passes; ++pass) {
    const int shift = pass * 8;
    const uint2* src = t.buf[pass & 1];
    uint2* dst = t.buf[(pass + 1) & 1];
    auto load = [&](int base, uint2 (&item)[AHEAD]) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = base + u * 32 + lane;
        if (i >= last) break;
        if (pass) { item[u] = __ldcg(&src[i]); continue; }
        const long long id = intAt(t.ids, t.wide, i);
        item[u] = make_uint2(id >= 0 && id < t.rows && id != t.padding ? (uint32_t)id : (uint32_t)t.rows, (uint32_t)i);
      }
    };
    for (int i = lane; i < 256; i += 32) hist[warp][i] = 0;
    __syncwarp();
    for (int i = first; i < last; i += 32 * AHEAD) {
      uint2 item[AHEAD];
      load(i, item);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (i + u * 32 + lane < last) atomicAdd(&hist[warp][item[u].x >> shift & 255], 1);
    }
    __syncthreads();
    // the warps in front (a quarter of them per thread), the blocks in front, all smaller digits
    int own[8], run = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) own[w] = hist[part * 8 + w][digit];
#pragma unroll
    for (int w = 0; w < 8; ++w) { const int c = own[w]; own[w] = run; run += c; }
    quarter[part][digit] = run;
    __syncthreads();
    int inFront = 0, sum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) { const int c = quarter[q][digit]; inFront += q < part ? c : 0; sum += c; }
    if (part == 0) total[digit] = sum;
    cluster.sync();
    int all = 0;
    {
      int c[SORT_CTAS];
#pragma unroll
      for (int k = 0; k < SORT_CTAS; ++k) c[k] = *cluster.map_shared_rank(&total[digit], k);
#pragma unroll
      for (int k = 0; k < SORT_CTAS; ++k) { inFront += k < cta ? c[k] : 0; all += c[k]; }
    }
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += x; }
    if (part == 0 && lane == 31) scan[warp] = inc;
    __syncthreads();
    inFront += inc - all;
#pragma unroll
    for (int w = 0; w < 7; ++w) inFront += w < (warp & 7) ? scan[w] : 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) hist[part * 8 + w][digit] = inFront + own[w];
    __syncthreads();
    for (int i = first; i < last; i += 32 * AHEAD) {
      uint2 item[AHEAD];
      load(i, item);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (i + u * 32 >= last) break;
        const bool in = i + u * 32 + lane < last;
        const int d = (int)(item[u].x >> shift & 255);
        const uint32_t same = sameDigit(d, in), before = same & ((1u << lane) - 1);
        int at = 0;
        if (in) at = hist[warp][d];
        __syncwarp();
        if (in && before == 0) hist[warp][d] = at + __popc(same);
        __syncwarp();
        if (in) dst[at + __popc(before)] = item[u];
      }
    }
    __threadfence();
    cluster.sync();                                      // all items in place; all counts read
  }
}

__global__ void __launch_bounds__(SORT_THREADS) sortTokensKernel(const Backward a) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();                          // the clearing starts now
  sortCluster(a.t[blockIdx.x / SORT_CTAS], a.n);
}

// Runs beside the sort, which has seen the kernels in front of both end before it let this one start; ends behind it.  128 blocks: a
// power of two of them clears 103 MB in 16.6 us, 148 in 18.6.
__global__ void __launch_bounds__(256) clearKernel(const Backward a) {
  tc::grid_launch_dependents();
  const size_t thread = (size_t)blockIdx.x * 256 + threadIdx.x, threads = (size_t)gridDim.x * 256;
  for (int k = 0; k < a.tables; ++k) {
    uint4* dst = (uint4*)a.t[k].grad;
    const size_t packs = a.t[k].gradBytes / 16;
    for (size_t i = thread; i < packs; i += threads) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    for (size_t i = packs * 16 + thread; i < a.t[k].gradBytes; i += threads) ((uint8_t*)a.t[k].grad)[i] = 0;
  }
  tc::grid_dependency_wait();
}

// Stores the sum of a row whose last token (of the stretch in which the row begins) is the `at`-th of the sorted ones.
template <typename T, int E, bool COMPACT>
__device__ __forceinline__ void storeRow(const Table& t, uint32_t row, int at, int d, int col, const float (&acc)[E]) {
  if (COMPACT) {
    Pack<float, E> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = acc[e];
    *(Pack<float, E>*)(t.compact + (size_t)(t.dense ? (int)row : at) * d + col) = o;
    if (col == 0) t.where[row] = at;
  } else {
    Pack<T, E> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = fromFloat<T>(acc[e] * t.scale);
    *(Pack<T, E>*)((T*)t.grad + (size_t)row * d + col) = o;
  }
}

// A block sums the tokens of a stretch for its columns (E per thread), row after row; eight rows are on their way at a time.
template <typename T, int E, bool COMPACT>
__global__ void __launch_bounds__(128) sumStretchKernel(const Backward a) {
  constexpr int MAX = 128, AHEAD = 8;
  __shared__ uint32_t keys[MAX + 2], tokens[MAX];
  __shared__ float weights[MAX];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const Table& t = a.t[blockIdx.z];
  const uint2* items = t.buf[t.passes & 1];
  const int start = blockIdx.x * a.stretch, count = min(a.stretch, a.n - start);
  for (int i = (int)threadIdx.x - 1; i <= count; i += 128) {             // and the keys on either side
    const int at = start + i;
    const uint2 item = at >= 0 && at < a.n ? __ldcg(&items[at]) : make_uint2(0xffffffffu, 0u);
    keys[i + 1] = item.x;
    if (i >= 0 && i < count) {
      tokens[i] = COMPACT ? item.y / t.perRow : item.y;
      if (COMPACT) weights[i] = item.x < (uint32_t)t.rows ? t.weights[item.y] * (t.gout ? t.gout[(size_t)tokens[i] * t.goutStride] : 1.f) : 0.f;
    }
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
    for (int u = 0; u < AHEAD; ++u) p[u] = *(const P*)(g + (size_t)tokens[min(i + u, count - 1)] * a.d);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = i + u;
      if (j >= count || keys[j + 1] == none) return;                     // (tokens without a gradient are the last)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = COMPACT ? fmaf(weights[j], toFloat(p[u].v[e]), acc[e]) : acc[e] + toFloat(p[u].v[e]);
      const bool goesOn = keys[j + 2] == keys[j + 1];
      if (goesOn && j + 1 < count) continue;
      if (head || goesOn) {                                              // not all of the row
        Pack<float, E> s;
#pragma unroll
        for (int e = 0; e < E; ++e) s.v[e] = acc[e];
        *(Pack<float, E>*)(t.sums + ((size_t)blockIdx.x * 2 + (head ? 0 : 1)) * a.d + col) = s;
      } else {
        storeRow<T, E, COMPACT>(t, keys[j + 1], start + j, a.d, col, acc);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      head = false;
    }
  }
}

// acc += the sums of stretches [from, to) of a row that goes through them.
template <int E>
__device__ __forceinline__ void addStretches(const float* s, size_t step, int from, int to, float (&acc)[E]) {
#pragma unroll 4
  for (int i = from; i < to; ++i) {
    const Pack<float, E> x = *(const Pack<float, E>*)(s + i * step);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += x.v[e];
  }
}

// Rows that go on behind the stretch in which they begin, 32 packs of columns per block.  A warp looks whether its stretch has such a row
// and adds up what few stretches it goes through; one that goes through more than eight, the block's warps add up together.  (With all rows
// added up by one warp each, a row of 12000 tokens of 131072 took 35 us.)
template <typename T, int E, bool COMPACT>
__global__ void __launch_bounds__(32 * JOIN_WARPS) joinStretchKernel(const Backward a) {
  constexpr int FEW = 8;
  __shared__ float part[JOIN_WARPS][32 * E];
  __shared__ int rowKey[JOIN_WARPS], rowCount[JOIN_WARPS];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const Table& t = a.t[blockIdx.z];
  const uint2* items = t.buf[t.passes & 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = (blockIdx.y * 32 + lane) * E;
  const int own = blockIdx.x * JOIN_WARPS + warp, start = own * a.stretch, end = start + a.stretch;
  uint32_t key = 0;
  int count = 0;                                                         // stretches that begin with the row
  if (own + 1 < a.stretches) {                                           // (the last one has nothing behind it)
    key = __ldcg(&items[end - 1]).x;
    const uint32_t behind = __ldcg(&items[end]).x, front = __ldcg(&items[start]).x, before = start > 0 ? __ldcg(&items[start - 1]).x : 0xffffffffu;
    if (key != (uint32_t)t.rows && behind == key && !(front == key && before == key)) {      // goes on, and did not begin further in front
      int next = own + 1;                                                // the first that does not end with it
      for (;;) {
        const int at = next + lane;
        const bool through = at < a.stretches && __ldcg(&items[min((at + 1) * a.stretch, a.n) - 1]).x == key;
        const uint32_t stops = ~__ballot_sync(0xffffffffu, through);
        if (stops) { next += __ffs(stops) - 1; break; }
        next += 32;
      }
      count = next - own - 1 + (next < a.stretches && __ldcg(&items[next * a.stretch]).x == key ? 1 : 0);
    }
  }
  if (lane == 0) { rowKey[warp] = (int)key; rowCount[warp] = count; }
  const size_t step = (size_t)2 * a.d;
  float acc[E];
  auto begin = [&](int stretch) {                                        // what the row has in the stretch in which it begins
    const Pack<float, E> x = *(const Pack<float, E>*)(t.sums + stretch * step + a.d + col);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = x.v[e];
  };
  if (count && count <= FEW && col < a.d) {
    begin(own);
    addStretches<E>(t.sums + (own + 1) * step + col, step, 0, count, acc);
    storeRow<T, E, COMPACT>(t, key, end - 1, a.d, col, acc);
  }
  __syncthreads();
  for (int w = 0; w < JOIN_WARPS; ++w) {
    const int many = rowCount[w], first = blockIdx.x * JOIN_WARPS + w;
    if (many <= FEW) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    const int per = (many + JOIN_WARPS - 1) / JOIN_WARPS;
    if (col < a.d) {
      if (warp == 0) begin(first);
      addStretches<E>(t.sums + (first + 1) * step + col, step, min(many, warp * per), min(many, warp * per + per), acc);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][lane * E + e] = acc[e];
    __syncthreads();
    if (warp || col >= a.d) continue;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int k = 1; k < JOIN_WARPS; ++k) acc[e] += part[k][lane * E + e];
    storeRow<T, E, COMPACT>(t, (uint32_t)rowKey[w], (first + 1) * a.stretch - 1, a.d, col, acc);
  }
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }
// Tokens of a stretch: 16, more (up to 128) once there are more than 2048 stretches.
int stretchOf(int n) { return std::min(128, std::max(16, (n + 2047) / 2048)); }
int lanesOf(int packs, int most) { int l = 1; while (l < packs && l < most) l *= 2; return l; }
struct Layout { size_t items, sums; };
Layout layoutOf(int n, int d) {
  const int s = stretchOf(n);
  return Layout{up256((size_t)n * sizeof(uint2)), up256((size_t)((n + s - 1) / s) * 2 * d * sizeof(float))};
}

template <typename T, int E>
ncclResult_t forward(const Forward& a, cudaStream_t stream) {
  const long long perBlock = 8ll * (32 / a.lanes) * a.turns;
  const bool plain = a.scale == 1.f;
  auto* kernel = a.positions ? plain ? embedForwardKernel<T, E, EMBED_ADD> : embedForwardKernel<T, E, EMBED_SCALE_ADD>
                             : plain ? embedForwardKernel<T, E, EMBED_COPY> : embedForwardKernel<T, E, EMBED_SCALE>;
  CUDACHECK(launchBehind(kernel, dim3((unsigned)((a.n + perBlock - 1) / perBlock)), 256, 1, stream, a));
  return ncclSuccess;
}

template <typename T, int E, bool COMPACT>
ncclResult_t backward(const Backward& a, cudaStream_t stream) {
  if (!COMPACT) CUDACHECK(launchBehind(sortTokensKernel, dim3(SORT_CTAS * a.tables), SORT_THREADS, SORT_CTAS, stream, a));
  if (!COMPACT) CUDACHECK(launchBehind(clearKernel, dim3(CLEAR_BLOCKS), 256, 1, stream, a));
  const int packs = a.d / E;
  CUDACHECK(launchBehind(sumStretchKernel<T, E, COMPACT>, dim3(a.stretches, (packs + 127) / 128, a.tables), 128, 1, stream, a));
  if (a.stretches > 1)
    CUDACHECK(launchBehind(joinStretchKernel<T, E, COMPACT>, dim3((a.stretches + JOIN_WARPS - 2) / JOIN_WARPS, (packs + 31) / 32, a.tables), 32 * JOIN_WARPS, 1,
                           stream, a));
  return ncclSuccess;
}

void setKeys(Table* t, const void* idx, int wide, int64_t rows, int64_t padding, uint8_t* at, const Layout& l) {
  t->ids = idx; t->wide = wide; t->rows = (int)rows; t->padding = padding;
  t->passes = 1;
  while (t->passes < 4 && (uint64_t)rows >> (8 * t->passes)) ++t->passes;
  t->buf[0] = (uint2*)at; t->buf[1] = (uint2*)(at + l.items); t->sums = (float*)(at + 2 * l.items);
}

constexpr int MOST_TOKENS = 0x7fffffff - 4095;      // loops over them step up to 2048 past their end
int typeBytes(int t) { return t == ncclFloat32 ? 4 : t == ncclBfloat16 || t == ncclFloat16 ? 2 : 0; }

}  // namespace

size_t tokenSumsWork(int n, int d) {
  const Layout l = layoutOf(n, d);
  return 2 * l.items + l.sums;
}
static Backward sumsOf(int n, int d, const void* ids, int wide, int64_t ignore, int v, void* work) {
  Backward a = {};
  a.tables = 1; a.n = n; a.d = d; a.stretch = stretchOf(n); a.stretches = (n + a.stretch - 1) / a.stretch;
  setKeys(&a.t[0], ids, wide, v, ignore, (uint8_t*)work, layoutOf(n, d));
  return a;
}
const uint2* tokenSortItems(int n, int d, int v, void* work) {
  const Backward a = sumsOf(n, d, nullptr, 0, 0, v, work);
  return a.t[0].buf[a.t[0].passes & 1];
}
ncclResult_t tokenSort(int n, int d, const void* ids, int wide, int64_t ignore, int v, void* work, cudaStream_t stream) {
  CUDACHECK(launchBehind(sortTokensKernel, dim3(SORT_CTAS), SORT_THREADS, SORT_CTAS, stream, sumsOf(n, d, ids, wide, ignore, v, work)));
  return ncclSuccess;
}
ncclResult_t tokenSums(const void* x, int n, int d, int perRow, int v, const float* weights, const float* gout, int goutStride, float* sums, bool dense, int* where,
                       void* work, cudaStream_t stream) {
  if (d % 8) return ncclInvalidArgument;
  Backward a = sumsOf(n, d, nullptr, 0, 0, v, work);
  a.g = x;
  a.t[0].compact = sums; a.t[0].where = where; a.t[0].weights = weights; a.t[0].gout = gout; a.t[0].goutStride = goutStride;
  a.t[0].perRow = perRow; a.t[0].dense = dense;
  return backward<__nv_bfloat16, 8, true>(a, stream);
}

}  // namespace dfccl

using namespace dfccl;
#define DF_API extern "C" __attribute__((visibility("default")))

DF_API ncclResult_t dfcclEmbeddingForward(const void* ids, int wideIds, int n, const void* w, int64_t rows, int64_t ldw, const void* positions, int widePositions,
                                          const void* p, int64_t prows, int64_t ldp, void* out, int d, int type, float scale, cudaStream_t stream) {
  const int bytes = typeBytes(type);
  if (n <= 0 || n > MOST_TOKENS || d <= 0 || rows <= 0 || !bytes || !ids || !w || !out || ldw < d || (positions && (!p || prows <= 0 || ldp < d))) return ncclInvalidArgument;
  Forward a{ids, positions, w, p, out, wideIds, widePositions, n, 0, 0, 0, rows, prows, ldw, ldp, scale};
  const uintptr_t grid = (uintptr_t)w | (uintptr_t)out | (uintptr_t)(ldw * bytes) | (uintptr_t)((size_t)d * bytes) |
                         (positions ? (uintptr_t)p | (uintptr_t)(ldp * bytes) : 0);
  const bool whole = (grid & 15) == 0;
  a.packs = whole ? d / (16 / bytes) : d;
  a.lanes = lanesOf(a.packs, 32);
  // rows one after the other, 8 at most, once there are more than 64 warps of them per SM
  { const int64_t warps = 148 * 64, side = 32 / a.lanes; a.turns = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(8, a.lanes), n / (warps * side))); }
  if (type == ncclFloat32) return whole ? forward<float, 4>(a, stream) : forward<float, 1>(a, stream);
  if (type == ncclBfloat16) return whole ? forward<__nv_bfloat16, 8>(a, stream) : forward<__nv_bfloat16, 1>(a, stream);
  return whole ? forward<__half, 8>(a, stream) : forward<__half, 1>(a, stream);
}

DF_API size_t dfcclEmbeddingBackwardWork(int n, int d, int tables) {
  if (n <= 0 || n > MOST_TOKENS || d <= 0 || tables < 1 || tables > MAX_TABLES) return 0;
  const Layout l = layoutOf(n, d);
  return tables * (2 * l.items + l.sums);
}

DF_API ncclResult_t dfcclEmbeddingBackward(const void* g, int n, int d, int type, const void* ids, int wideIds, int64_t padding, float scale, void* gw, int64_t rows,
                                           const void* positions, int widePositions, void* gp, int64_t prows, void* work, cudaStream_t stream) {
  const int bytes = typeBytes(type);
  if (n <= 0 || n > MOST_TOKENS || d <= 0 || !bytes || !g || !work || !(gw || gp) || (gw && (!ids || rows <= 0 || rows > 0x7ffffff0ll)) ||
      (gp && (!positions || prows <= 0 || prows > 0x7ffffff0ll)) || (((uintptr_t)gw | (uintptr_t)gp) & 15) || ((uintptr_t)work & 31))
    return ncclInvalidArgument;
  const Layout l = layoutOf(n, d);
  Backward a = {};
  a.n = n; a.d = d; a.stretch = stretchOf(n); a.stretches = (n + a.stretch - 1) / a.stretch; a.g = g;
  uint8_t* at = (uint8_t*)work;
  auto add = [&](const void* idx, int wide, int64_t count, int64_t pad, void* grad, float s) {
    Table& t = a.t[a.tables++];
    setKeys(&t, idx, wide, count, pad, at, l);
    t.grad = grad; t.gradBytes = (size_t)count * d * bytes; t.scale = s;
    at += 2 * l.items + l.sums;
  };
  if (gw) add(ids, wideIds, rows, padding, gw, scale);
  if (gp) add(positions, widePositions, prows, -1, gp, 1.f);
  const bool whole = (((uintptr_t)g | (uintptr_t)((size_t)d * bytes)) & 15) == 0;
  if (type == ncclFloat32) return whole ? backward<float, 4, false>(a, stream) : backward<float, 1, false>(a, stream);
  if (type == ncclBfloat16) return whole ? backward<__nv_bfloat16, 8, false>(a, stream) : backward<__nv_bfloat16, 1, false>(a, stream);
  return whole ? backward<__half, 8, false>(a, stream) : backward<__half, 1, false>(a, stream);
}

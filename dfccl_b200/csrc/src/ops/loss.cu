// Losses of a language model's head over its vocabulary, from the head's inputs x [n, d] and its weights w [v, d] without keeping
// the logits z = x w^T: softmax cross entropy with a target per row, and distillation from a teacher's list of logits per row.
// Both are a divergence from a distribution q over a row's list of entries (one entry of weight 1: a target),
//     loss = T^2 sum_k q_k (ln q_k - ln p_k),   p = softmax(z / T),   dz = T g (p - q),
// so both run on the same products (gemm/tcgen05_vocab.cu); here are the passes around them.  They move n (k + 1) words and, behind the
// forward product, 8 bytes per row and stretch of 128 columns: microseconds beside the products'.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <algorithm>
#include "dfccl_ops.h"
#include "../common/log.h"
#include "../common/param.h"
#include "../gemm/epilogue.h"
#include "../gemm/gemm.h"
#include "../gemm/tc_common.h"
#include "../gemm/vocab.h"

namespace dfccl {
namespace {

constexpr int MAX_LIST = 256;          // entries of a teacher's list
constexpr int ROWS = 16384;            // rows of a forward product at a time: bounds its partial sums (52 MB at 50257 columns)
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;

template <typename... P, typename... A>
cudaError_t launchBehind(void (*kernel)(P...), dim3 grid, int block, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization; at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, (P)args...);
}

__device__ __forceinline__ long long intAt(const void* p, int wide, size_t i) { return wide ? ((const long long*)p)[i] : ((const int*)p)[i]; }

__device__ __forceinline__ float warpMax(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warpSum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A teacher's entries as lists in ascending order with q = softmax(logits / T); entries of token -1 or of logit -inf are left out.  A warp
// per row; an entry's place is the number of entries in front of it (256 entries: 8 x 256 comparisons a lane).
__global__ void __launch_bounds__(128) teacherRowsKernel(const void* logits, int type, const void* tokens, int wide, int n, int k, int v, float invT,
                                                         int* outTokens, float* outWeights, int* state) {
  __shared__ int tok[4][MAX_LIST];
  __shared__ float val[4][MAX_LIST];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * 4 + warp;
  if (row >= n) return;
  bool bad = false;
  float top = -INFINITY;
  for (int i = lane; i < k; i += 32) {
    const size_t at = (size_t)row * k + i;
    const long long t = intAt(tokens, wide, at);
    const float l = (type == 0 ? ((const float*)logits)[at] : type == 1 ? __bfloat162float(((const __nv_bfloat16*)logits)[at]) : __half2float(((const __half*)logits)[at])) * invT;
    const bool keep = t != -1 && l != -INFINITY;
    if (keep && (t < 0 || t >= v)) bad = true;
    tok[warp][i] = keep ? (int)t : VOCAB_NO_TOKEN;
    val[warp][i] = l;
    if (keep) top = fmaxf(top, l);
  }
  bad = __any_sync(0xffffffffu, bad);
  top = warpMax(top);
  __syncwarp();
  float sum = 0.f;
  bool some = false;
  for (int i = lane; i < k; i += 32) {
    if (tok[warp][i] == VOCAB_NO_TOKEN) continue;
    const float e = expf(val[warp][i] - top);
    val[warp][i] = e;
    sum += e;
    some = true;
  }
  some = __any_sync(0xffffffffu, some);
  sum = warpSum(sum);
  const float inv = 1.f / sum;
  __syncwarp();
  const bool usable = some && !bad;
  for (int i = lane; i < k; i += 32) {
    const int t = tok[warp][i];
    int place = 0;
    for (int j = 0; j < k; ++j) { const int u = tok[warp][j]; place += u < t || (u == t && j < i) ? 1 : 0; }
    const bool in = usable && t != VOCAB_NO_TOKEN;
    outTokens[(size_t)row * k + place] = in ? t : VOCAB_NO_TOKEN;
    outWeights[(size_t)row * k + place] = in ? val[warp][i] * inv : 0.f;
  }
  if (lane == 0) state[row] = bad ? ROW_BAD : some ? ROW_LIST : ROW_NONE;
}

// {m, s} stands for s 2^m.
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), base = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * exp2f(a.x - base) + b.y * exp2f(b.x - base));
}

// Sum or mean of the rows' losses, in 64 bits and a fixed order, and the number of rows that count; by the 1024 threads of one block.
__device__ void reduceLoss(const float* loss, const VocabRows& rows, int n, int mean, float* out, int* count) {
  __shared__ double sums[32];
  __shared__ int counts[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double s = 0.0;
  int c = 0;
  for (int i = threadIdx.x; i < n; i += 1024) { s += __ldcg(loss + i); c += rowState(rows, i) != ROW_NONE; }
#pragma unroll
  for (int o = 16; o; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); c += __shfl_xor_sync(0xffffffffu, c, o); }
  if (lane == 0) { sums[warp] = s; counts[warp] = c; }
  __syncthreads();
  if (warp) return;
  s = sums[lane]; c = counts[lane];
#pragma unroll
  for (int o = 16; o; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); c += __shfl_xor_sync(0xffffffffu, c, o); }
  if (lane == 0) { *out = (float)(mean ? s / max(c, 1) : s); *count = c; }
}

struct JoinArgs {
  VocabRows rows;               // from this launch's first row on, as `lse` and `loss`
  const float2* parts;
  const float* picked;
  int stretches, n;
  float t2;
  float* lse;
  float* loss;
  // the sum over all rows, by the block of the last launch that comes last; null: none
  VocabRows allRows;
  const float* allLoss;
  int all, mean, blocks;        // blocks of all launches
  int* ticket;
  float* out;
  int* count;
};

// 32 rows per block: warp g takes every 32nd stretch of all of them (a line of 256 bytes each), then warp r finishes row r.
__global__ void __launch_bounds__(1024) joinRowsKernel(const JoinArgs a) {
  __shared__ float2 part[32][33];
  __shared__ int last;
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = blockIdx.x * 32;
  float2 acc = make_float2(-INFINITY, 0.f);
  if (row0 + lane < a.n) {
    int i = warp;
    for (; i + 96 < a.stretches; i += 128) {
      float2 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = a.parts[(size_t)(i + 32 * u) * a.n + row0 + lane];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc = joined(acc, p[u]);
    }
    for (; i < a.stretches; i += 32) acc = joined(acc, a.parts[(size_t)i * a.n + row0 + lane]);
  }
  part[warp][lane] = acc;
  __syncthreads();
  const int row = row0 + warp;
  if (row < a.n) {
    acc = part[lane][warp];
#pragma unroll
    for (int o = 16; o; o >>= 1) acc = joined(acc, make_float2(__shfl_xor_sync(0xffffffffu, acc.x, o), __shfl_xor_sync(0xffffffffu, acc.y, o)));
    const float l = acc.x + log2f(acc.y);
    float sum = 0.f;
    const int st = rowState(a.rows, row);
    if (st == ROW_LIST)
      for (int i = lane; i < a.rows.k; i += 32) {
        const size_t at = (size_t)row * a.rows.k + i;
        if (!a.rows.targets && a.rows.tokens[at] == VOCAB_NO_TOKEN) continue;
        const float q = a.rows.targets ? 1.f : a.rows.weights[at];
        if (q == 0.f) continue;                         // 0 ln 0
        sum += q * (logf(q) - (a.picked[at] * a.rows.scale - l) * LN2);
      }
    sum = warpSum(sum);
    if (lane == 0) {
      a.lse[row] = l;
      a.loss[row] = st == ROW_LIST ? sum * a.t2 : st == ROW_NONE ? 0.f : __int_as_float(0x7fffffff);
    }
  }
  if (!a.ticket) return;
  __threadfence();                                       // this block's losses, in front of its ticket
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1) == a.blocks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  reduceLoss(a.allLoss, a.allRows, a.all, a.mean, a.out, a.count);
}

// x with zeros in the rows without a list: in the product of the weights' gradient they meet the zeros of the logits' gradient, and nothing
// that x holds there (infinities, NaN) may come through.  n d 4 bytes: 8192 x 1024 takes 6 us beside 2300.
__global__ void __launch_bounds__(256) keepRowsKernel(const uint4* x, const VocabRows rows, int n, int packs, uint4* out) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  for (int row = blockIdx.x; row < n; row += gridDim.x) {
    const bool keep = rowState(rows, row) != ROW_NONE;
    for (int i = threadIdx.x; i < packs; i += 256) out[(size_t)row * packs + i] = keep ? x[(size_t)row * packs + i] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// out = factor times the sum of the slices, rounded once; `packs` of 8 elements.
__global__ void __launch_bounds__(256) joinSlicesKernel(const float* part, int slices, size_t packs, const VocabFactor factor, __nv_bfloat16* out) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const float f = vocabFactor(factor);
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < packs; i += (size_t)gridDim.x * 256) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int s = 0; s < slices; ++s) {
      const float4* src = (const float4*)part + ((size_t)s * packs + i) * 2;
      const float4 x = src[0], y = src[1];
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
    }
    ((uint4*)out)[i] = make_uint4(tc::pack_bf16x2(a.x * f, a.y * f), tc::pack_bf16x2(a.z * f, a.w * f), tc::pack_bf16x2(b.x * f, b.y * f), tc::pack_bf16x2(b.z * f, b.w * f));
  }
}

ncclResult_t joinSlices(const float* part, int slices, size_t elements, const VocabFactor& factor, void* out, cudaStream_t stream) {
  const size_t packs = elements / 8;
  CUDACHECK(launchBehind(joinSlicesKernel, dim3((unsigned)std::min<size_t>((packs + 255) / 256, 148 * 8)), 256, stream, part, slices, packs, factor, (__nv_bfloat16*)out));
  return ncclSuccess;
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// How a backward pass goes over the vocabulary: columns of the logits' gradient that exist at a time, and what the products need.
struct BackwardPlan {
  int cols;                       // columns of a piece (all of them, or a multiple of the tile)
  VocabPlan cut;
  int slicesX, slicesW;           // of dx those of a whole piece: a shorter last one has fewer and adds to the first of them
  bool sumX, sumW;                // fp32 sums in memory: of dx because there are pieces or slices, of dw because there are slices
  size_t dz, partX, partW, kept;  // bytes
  size_t all() const { return dz + partX + partW + kept; }
};
BackwardPlan backwardPlan(int n, int v, int d, bool wantX, bool wantW) {
  BackwardPlan p;
  const int64_t limit = std::max<int64_t>(1 << 20, paramI64("LOSS_WORKSPACE_BYTES", 1ll << 30));
  const int64_t most = std::max<int64_t>(1, limit / (2ll * n) / VOCAB_TILE) * VOCAB_TILE;
  const int64_t pieces = (v + most - 1) / most;
  p.cols = pieces == 1 ? v : (int)(((v + pieces - 1) / pieces + VOCAB_TILE - 1) / VOCAB_TILE * VOCAB_TILE);
  p.cut = vocabProductPlan(n, p.cols, d, wantX, wantW, gemmPairResident());
  p.slicesX = vocabSlices(p.cols, p.cut.perX);
  p.slicesW = vocabSlices(n, p.cut.perW);
  p.sumX = wantX && (pieces > 1 || p.slicesX > 1);
  p.sumW = wantW && p.slicesW > 1;
  p.dz = up256((size_t)n * ((p.cols + 63) / 64 * 64) * 2);
  p.partX = p.sumX ? up256((size_t)p.slicesX * n * d * 4) : 0;
  p.partW = p.sumW ? up256((size_t)p.slicesW * p.cols * d * 4) : 0;
  p.kept = wantW ? up256((size_t)n * d * 2) : 0;
  return p;
}

bool sizesOk(int n, int v, int d, int k) { return n > 0 && v > 0 && v <= VOCAB_NO_TOKEN - 512 && d > 0 && d % 8 == 0 && k > 0 && k <= MAX_LIST; }

}  // namespace
}  // namespace dfccl

using namespace dfccl;
#define DF_API extern "C" __attribute__((visibility("default")))

DF_API int dfcclLinearLossMaxList(void) { return MAX_LIST; }

DF_API ncclResult_t dfcclTeacherRows(const void* logits, int logitType, const void* tokens, int wide, int n, int k, int v, float temperature, void* outTokens,
                                     void* outWeights, void* state, cudaStream_t stream) {
  const int type = logitType == ncclFloat32 ? 0 : logitType == ncclBfloat16 ? 1 : logitType == ncclFloat16 ? 2 : -1;
  if (!logits || !tokens || !outTokens || !outWeights || !state || type < 0 || !sizesOk(n, v, 8, k) || !(temperature > 0.f)) return ncclInvalidArgument;
  CUDACHECK(launchBehind(teacherRowsKernel, (n + 3) / 4, 128, stream, logits, type, tokens, wide, n, k, v, 1.f / temperature, (int*)outTokens, (float*)outWeights,
                         (int*)state));
  return ncclSuccess;
}

namespace {
struct ForwardLayout { size_t parts, picked, loss; };
ForwardLayout forwardLayout(int n, int v, int k) {
  const size_t rows = std::min(n, ROWS);
  return ForwardLayout{up256(rows * vocabParts(v) * sizeof(float2)), up256(rows * k * 4), up256((size_t)n * 4)};
}
// A target per row, or lists; from row `r` on.
VocabRows rowsOf(const void* targets, int wide, int v, int64_t ignore, const void* tokens, const void* weights, const void* state, int k, float temperature, int r) {
  const size_t at = (size_t)r * k;
  return VocabRows{targets ? (const uint8_t*)targets + (size_t)r * (wide ? 8 : 4) : nullptr, wide, v, (long long)ignore, tokens ? (const int*)tokens + at : nullptr,
                   weights ? (const float*)weights + at : nullptr, state ? (const int*)state + r : nullptr, k, LOG2E / temperature};
}
bool rowsOk(const void* targets, const void* tokens, const void* weights, const void* state, int k, float temperature) {
  return (targets ? k == 1 : tokens && weights && state) && temperature > 0.f;
}
}  // namespace

DF_API size_t dfcclLinearLossForwardWork(int n, int v, int k) {
  if (!sizesOk(n, v, 8, k)) return 0;
  const ForwardLayout l = forwardLayout(n, v, k);
  return l.parts + l.picked + l.loss + 256;
}

DF_API ncclResult_t dfcclLinearLossForward(const void* x, const void* w, int n, int v, int d, const void* targets, int wide, int64_t ignore, const void* tokens,
                                           const void* weights, const void* state, int k, float temperature, int reduction, void* work, void* lse, void* rowLoss,
                                           void* loss, void* count, cudaStream_t stream) {
  if (!sizesOk(n, v, d, k) || !x || !w || !rowsOk(targets, tokens, weights, state, k, temperature) || !work || !lse || reduction < 0 || reduction > 2) return ncclInvalidArgument;
  if ((((uintptr_t)x | (uintptr_t)w) & 15) || (reduction ? !loss || !count : !rowLoss)) return ncclInvalidArgument;
  const ForwardLayout l = forwardLayout(n, v, k);
  JoinArgs j = {};
  j.parts = (const float2*)work; j.picked = (const float*)((uint8_t*)work + l.parts);
  j.stretches = vocabParts(v); j.t2 = temperature * temperature;
  float* losses = rowLoss ? (float*)rowLoss : (float*)((uint8_t*)work + l.parts + l.picked);
  j.allRows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, 0);
  j.allLoss = losses; j.all = n; j.mean = reduction == 1;
  j.ticket = reduction ? (int*)((uint8_t*)work + l.parts + l.picked + l.loss) : nullptr;
  j.out = (float*)loss; j.count = (int*)count;
  for (int r = 0; r < n; r += ROWS) j.blocks += (std::min(ROWS, n - r) + 31) / 32;
  for (int r = 0; r < n; r += ROWS) {
    j.n = std::min(ROWS, n - r);
    j.rows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, r);
    j.lse = (float*)lse + r; j.loss = losses + r;
    DFCHECK(vocabStats((const __nv_bfloat16*)x + (size_t)r * d, w, j.n, v, d, j.rows, (float2*)j.parts, (float*)j.picked, r ? nullptr : j.ticket, stream));
    CUDACHECK(launchBehind(joinRowsKernel, (j.n + 31) / 32, 1024, stream, j));
  }
  return ncclSuccess;
}

DF_API size_t dfcclLinearLossBackwardWork(int n, int v, int d, int wantX, int wantW) {
  if (!sizesOk(n, v, d, 1) || !(wantX || wantW)) return 0;
  const BackwardPlan p = backwardPlan(n, v, d, wantX != 0, wantW != 0);
  return p.all();
}

DF_API ncclResult_t dfcclLinearLossBackward(const void* x, const void* w, int n, int v, int d, const void* targets, int wide, int64_t ignore, const void* tokens,
                                            const void* weights, const void* state, int k, float temperature, const void* lse, const void* gout, int goutStride,
                                            const void* count, void* dx, void* dw, void* work, size_t workBytes, cudaStream_t stream) {
  if (!sizesOk(n, v, d, k) || !x || !w || !rowsOk(targets, tokens, weights, state, k, temperature) || !lse || !gout || !work || !(dx || dw) || goutStride < 0) return ncclInvalidArgument;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw) & 15) return ncclInvalidArgument;
  const BackwardPlan p = backwardPlan(n, v, d, dx != nullptr, dw != nullptr);
  if (p.all() > workBytes) return ncclInvalidArgument;          // (the setting has changed since the size was asked for)
  void* dz = work;
  float* partX = p.sumX ? (float*)((uint8_t*)work + p.dz) : nullptr;
  float* partW = p.sumW ? (float*)((uint8_t*)work + p.dz + p.partX) : nullptr;
  void* kept = (uint8_t*)work + p.dz + p.partX + p.partW;
  const VocabRows rows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, 0);
  if (dw) CUDACHECK(launchBehind(keepRowsKernel, std::min(n, 148 * 8), 256, stream, (const uint4*)x, rows, n, d / 8, (uint4*)kept));
  const VocabGrad grad{(const float*)lse, goutStride ? (const float*)gout : nullptr, goutStride};
  const VocabFactor factor{goutStride ? nullptr : (const float*)gout, (const int*)count, temperature};
  for (int c = 0; c < v; c += p.cols) {
    const int cols = std::min(p.cols, v - c);
    const __nv_bfloat16* wc = (const __nv_bfloat16*)w + (size_t)c * d;
    __nv_bfloat16* dwc = dw ? (__nv_bfloat16*)dw + (size_t)c * d : nullptr;
    DFCHECK(vocabGrad(x, wc, n, cols, c, d, rows, grad, dz, stream));
    DFCHECK(vocabProducts(dz, kept, wc, n, cols, d, p.cut, factor, p.sumX ? nullptr : dx, partX, c != 0, p.sumW ? nullptr : dwc, partW, stream));
    if (p.sumW) DFCHECK(joinSlices(partW, p.slicesW, (size_t)cols * d, factor, dwc, stream));
  }
  if (p.sumX) DFCHECK(joinSlices(partX, p.slicesX, (size_t)n * d, factor, dx, stream));
  return ncclSuccess;
}

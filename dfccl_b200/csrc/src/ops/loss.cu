// Losses of a language model's head over its vocabulary, from the head's inputs x [n, d] and its weights w [v, d] without keeping
// the logits z = x w^T: softmax cross entropy with a target per row, and distillation from a teacher's list of logits per row.
// Both are a divergence from a distribution q over a row's list of entries (one entry of weight 1: a target),
//     loss = T^2 sum_k q_k (ln q_k - ln p_k),   p = softmax(z / T),   dz = T g (p - q),
// so both run on the same products (gemm/tcgen05_vocab.cu); here are the passes around them.  Behind the forward product they move 8 bytes per
// row and stretch of 256 columns; for the lists a row of w per entry twice (their logits, what they add to dx) and one of x twice (what they add
// to dw, its sums).  Beside targets that is microseconds; 8192 lists of 32 over 50257 x 1024 take 270 us of 1997.
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
#include "embed.h"

namespace dfccl {
namespace {

constexpr int MAX_LIST = 256;          // entries of a teacher's list
constexpr int MOST_SORTED = 0x7fffffff - 4096;      // entries of all lists together that are sorted, as 31 bits count them
constexpr int ROWS = 16384;            // rows of a forward product at a time: bounds its partial sums (26 MB at 50257 columns)
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
#pragma unroll 4
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
  float* rest;                  // [n][k] what is left of an entry's weight without its probability; of entries of one token all of it in the first
  // behind vocabPowers: the powers' bases and, to be written, the powers' share of a probability, 2^base / sum; rows whose sums say that
  // their base was no good raise `again`
  float* base;
  float* share;
  const uint4* x;               // and x times that, where `shared` is given; `packs` of 8 elements in a row
  uint4* shared;
  int packs;
  int* again;
  const int* only;              // nothing but the sum over all rows unless this holds something (null: always)
  // the sum over all rows, by the block of the last launch that comes last; null: none
  VocabRows allRows;
  const float* allLoss;
  int all, mean, blocks;        // blocks of all launches
  int* ticket;
  float* out;
  int* count;
};

// A base is good if it is a number and no power is above 2^60: the sums of powers times x or w stay far from the end of fp32.
constexpr float MOST_POWER = 60.f;

// 32 rows per block: warp g takes every 32nd stretch of all of them (a line of 256 bytes each), then warp r finishes row r.
// POWERS: the stretches' sums are relative to the rows' bases.  Otherwise, with `base`, the logarithms of the sums become the bases.
template <bool POWERS>
__global__ void __launch_bounds__(1024) joinRowsKernel(const JoinArgs a) {
  __shared__ float2 part[32][33];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = blockIdx.x * 32, row = row0 + warp;
  const size_t list = (size_t)row * a.rows.k;
  // The rows' lists are older than the launches that run beside this one (those have waited for them): their way is over when the parts come.
  int st = ROW_NONE, token = VOCAB_NO_TOKEN, tokenFront = VOCAB_NO_TOKEN;
  float weight = 0.f;
  if (row < a.n) {
    st = rowState(a.rows, row, token);
    if (!a.rows.targets && lane < a.rows.k) {
      token = a.rows.tokens[list + lane];
      tokenFront = lane ? a.rows.tokens[list + lane - 1] : VOCAB_NO_TOKEN;
      weight = a.rows.weights[list + lane];
    }
  }
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  auto tokenAt = [&](int i) { return i == lane ? token : a.rows.tokens[list + i]; };
  auto frontOf = [&](int i) { return i == lane ? tokenFront : a.rows.tokens[list + i - 1]; };
  auto weightAt = [&](int i) { return i == lane ? weight : a.rows.weights[list + i]; };
  auto join = [](float2 x, float2 y) { return POWERS ? make_float2(fmaxf(x.x, y.x), x.y + y.y) : joined(x, y); };
  if (!a.only || *a.only) {
    float2 acc = make_float2(-INFINITY, 0.f);
    const float mine = row < a.n && lane < a.rows.k ? a.picked[list + lane] : 0.f, base = POWERS && row < a.n ? a.base[row] : 0.f;
    auto pickedAt = [&](int i) { return i == lane ? mine : a.picked[list + i]; };
    if (row0 + lane < a.n) {
      for (int i = warp; i < a.stretches; i += 32 * 8) {
        float2 p[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) p[u] = i + 32 * u < a.stretches ? a.parts[(size_t)(i + 32 * u) * a.n + row0 + lane] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int u = 0; u < 8; ++u) acc = join(acc, p[u]);
      }
    }
    part[warp][lane] = acc;
    __syncthreads();
    if (row < a.n) {
      acc = part[lane][warp];
#pragma unroll
      for (int o = 16; o; o >>= 1) acc = join(acc, make_float2(__shfl_xor_sync(0xffffffffu, acc.x, o), __shfl_xor_sync(0xffffffffu, acc.y, o)));
      float sum = 0.f, share = st == ROW_BAD ? __int_as_float(0x7fffffff) : 1.f;
      const float2 others = POWERS ? make_float2(base, acc.y) : acc;             // of entries that the list has not
      float2 every = others;
      int distinct = 0;
      if (st == ROW_LIST) {                             // the list's own powers, each token once
        float2 own = make_float2(-INFINITY, 0.f);
        for (int i = lane; i < a.rows.k; i += 32) {
          if (!a.rows.targets && (tokenAt(i) == VOCAB_NO_TOKEN || (i && tokenAt(i) == frontOf(i)))) continue;
          own = joined(own, make_float2(pickedAt(i) * a.rows.scale, 1.f));
          ++distinct;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          own = joined(own, make_float2(__shfl_xor_sync(0xffffffffu, own.x, o), __shfl_xor_sync(0xffffffffu, own.y, o)));
          distinct += __shfl_xor_sync(0xffffffffu, distinct, o);
        }
        every = joined(others, own);
      }
      const float l = every.x + log2f(every.y);
      if (distinct == 1) {                              // all on one token: from the others' powers, however small they are beside its own
        const float u = __shfl_sync(0xffffffffu, mine, 0) * a.rows.scale, ratio = others.y * exp2f(others.x - u);
        for (int i = lane; i < a.rows.k; i += 32) {
          const float q = a.rows.targets || tokenAt(i) == VOCAB_NO_TOKEN ? 1.f : weightAt(i);
          if (q != 0.f) sum += q * logf(q);             // (of entries that share the token)
          a.rest[list + i] = 0.f;
        }
        sum = warpSum(sum);
        if (lane == 0) a.rest[list] = sum != sum ? sum : others.y * exp2f(others.x - l);      // (the teacher's weights are not numbers)
        sum += (ratio < 1e30f ? log1pf(ratio) : (l - u) * LN2);
      } else {
        for (int i = lane; i < a.rows.k; i += 32) {
          float rest = 0.f;
          if (st == ROW_LIST && tokenAt(i) != VOCAB_NO_TOKEN) {
            const int t = tokenAt(i);
            float q = weightAt(i);
            const float u = pickedAt(i) * a.rows.scale - l;
            if (q != 0.f) sum += q * (logf(q) - u * LN2);         // (0 ln 0)
            if (i == 0 || frontOf(i) != t) {
              for (int j = i + 1; j < a.rows.k && a.rows.tokens[list + j] == t; ++j) q += a.rows.weights[list + j];
              rest = q - exp2f(u);
            }
          }
          a.rest[list + i] = rest;
        }
        sum = warpSum(sum);
      }
      if (POWERS) {
        if (st == ROW_LIST) share = exp2f(others.x - l);
        if (lane == 0) {
          a.share[row] = st == ROW_NONE ? 0.f : share;
          if (st == ROW_LIST && !(acc.x <= MOST_POWER && acc.y < INFINITY && fabsf(others.x) < INFINITY)) *a.again = 1;
        }
      } else if (a.base && lane == 0) {
        a.base[row] = l;
        if (st == ROW_LIST) a.share[row] = 1.f;
      }
      // x times the row's share, rounded to bf16: the right operand of the powers' product.  A row without a target is zeros whatever it holds.
      if (a.shared)
        for (int i = lane; i < a.packs; i += 32) {
          uint4 o = make_uint4(0u, 0u, 0u, 0u);
          if (st != ROW_NONE) {
            const uint4 p = a.x[(size_t)row * a.packs + i];
            o = make_uint4(tc::pack_bf16x2(bf16Lo(p.x) * share, bf16Hi(p.x) * share), tc::pack_bf16x2(bf16Lo(p.y) * share, bf16Hi(p.y) * share),
                           tc::pack_bf16x2(bf16Lo(p.z) * share, bf16Hi(p.z) * share), tc::pack_bf16x2(bf16Lo(p.w) * share, bf16Hi(p.w) * share));
          }
          a.shared[(size_t)row * a.packs + i] = o;
        }
      if (lane == 0) {
        a.lse[row] = l;
        a.loss[row] = st == ROW_LIST ? sum * a.t2 : st == ROW_NONE ? 0.f : __int_as_float(0x7fffffff);
      }
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

// In front of the products: the logits of the rows' lists by fp32 sums, a warp for four entries of a row, -> picked [n][k].  Where `base` is
// given, a warp for a row, and the largest of its entries times `scale` is the base of its powers.  On the way, words set to their start and
// the number of rows that count.
struct PickArgs {
  const uint4* x; const uint4* w;
  VocabRows rows;
  int n, packs;                  // of 8 columns
  float* picked;
  float* base;
  int* count;                    // or null
  int* words; int nWords;        // to be 0
  int beside;                    // the sort in front runs beside this kernel, which ends behind it
};
__global__ void __launch_bounds__(256) pickLogitsKernel(const PickArgs a) {
  __shared__ int counts[8];
  if (!a.beside) tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0) {
    if (a.count) {
      int c = 0;
      for (int i = threadIdx.x; i < a.n; i += 256) c += rowState(a.rows, i) != ROW_NONE;
#pragma unroll
      for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
      if (lane == 0) counts[warp] = c;
      __syncthreads();
      if (threadIdx.x == 0) { for (int k = 1; k < 8; ++k) c += counts[k]; *a.count = c; }
    }
    for (int i = threadIdx.x; i < a.nWords; i += 256) a.words[i] = 0;
  }
  const int k = a.rows.k, fours = a.base ? 1 : (k + 3) / 4;
  for (long long item = (long long)blockIdx.x * 8 + warp; item < (long long)a.n * fours; item += (long long)gridDim.x * 8) {
    const int row = (int)(item / fours);
    int first = (int)(item - (long long)row * fours) * 4, token;
    const int end = a.base ? k : min(k, first + 4);
    const bool list = rowState(a.rows, row, token) == ROW_LIST;
    float most = -INFINITY;
    bool odd = false;                                   // (a maximum passes over what is not a number)
    for (; first < end; first += 4) {
      const uint4* w[4];
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      bool some = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int t = VOCAB_NO_TOKEN;
        if (list) t = a.rows.targets ? e ? VOCAB_NO_TOKEN : token : first + e < k ? a.rows.tokens[(size_t)row * k + first + e] : VOCAB_NO_TOKEN;
        w[e] = t == VOCAB_NO_TOKEN ? nullptr : a.w + (size_t)t * a.packs;
        some = some || w[e];
      }
      if (some)
        for (int i = lane; i < a.packs; i += 32) {
          const uint4 x = a.x[(size_t)row * a.packs + i];
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
          uint4 y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = w[e] ? w[e][i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t yw[4] = {y[e].x, y[e].y, y[e].z, y[e].w};
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[e] = fmaf(bf16Lo(xw[q]), bf16Lo(yw[q]), fmaf(bf16Hi(xw[q]), bf16Hi(yw[q]), sum[e]));
          }
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (first + e >= k) break;
        const float z = warpSum(sum[e]);
        if (lane == 0) a.picked[(size_t)row * k + first + e] = z;
        if (w[e]) { most = fmaxf(most, z); odd = odd || z != z; }
      }
    }
    if (a.base && lane == 0) a.base[row] = !list ? 0.f : odd ? __int_as_float(0x7fffffff) : most * a.rows.scale;
  }
  // (one block waits for the sort, and with it the kernel: blocks that waited would keep those behind them from starting)
  if (a.beside && blockIdx.x == gridDim.x - 1) tc::grid_dependency_wait();
}
ncclResult_t pickLogits(const PickArgs& a, cudaStream_t stream) {
  const long long items = (long long)a.n * (a.base ? 1 : (a.rows.k + 3) / 4);
  CUDACHECK(launchBehind(pickLogitsKernel, dim3((unsigned)std::min<long long>((items + 7) / 8, 148 * 8)), 256, stream, a));
  return ncclSuccess;
}

// The sum over each row's list of rest w: a block per row, a thread per pack of columns.  As many bytes of w from L2 as the list has rows, as in
// pickLogitsKernel; 8192 lists of 32 and 1024 columns take 55 us; on the way, in the product's epilogue, 128.
__global__ void __launch_bounds__(128) listSumsKernel(const uint4* w, const VocabRows rows, const float* rest, int n, int packs, float4* out) {
  __shared__ int tokens[MAX_LIST];
  __shared__ float weights[MAX_LIST];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  for (int row = blockIdx.x; row < n; row += gridDim.x) {
    __syncthreads();
    for (int i = threadIdx.x; i < rows.k; i += 128) {
      const int t = rows.tokens[(size_t)row * rows.k + i];
      const float q = rest[(size_t)row * rows.k + i];
      tokens[i] = t == VOCAB_NO_TOKEN ? 0 : t;
      weights[i] = t == VOCAB_NO_TOKEN ? 0.f : q;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < packs; i += 128) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
      for (int k = 0; k < rows.k; ++k) {
        const float q = weights[k];
        const uint4 p = q != 0.f ? w[(size_t)tokens[k] * packs + i] : make_uint4(0u, 0u, 0u, 0u);
        vocabMinus(f, -q, p);
      }
      float4* dst = out + ((size_t)row * packs + i) * 2;
      dst[0] = make_float4(f[0], f[1], f[2], f[3]); dst[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
}

// Two results times one number on the device, in place; nothing is read or written where it is 1.  (What is not a power of two rounds them to
// bf16 a second time: the number is not known when they are made, and as fp32 they would take twice the memory until then.)
__global__ void __launch_bounds__(256) scaleResultsKernel(uint4* a, size_t na, uint4* b, size_t nb, const float* scale) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const float f = *scale;
  if (f == 1.f) return;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < na + nb; i += (size_t)gridDim.x * 256) {
    uint4* p = i < na ? a + i : b + (i - na);
    const uint4 v = *p;
    *p = make_uint4(tc::pack_bf16x2(bf16Lo(v.x) * f, bf16Hi(v.x) * f), tc::pack_bf16x2(bf16Lo(v.y) * f, bf16Hi(v.y) * f),
                    tc::pack_bf16x2(bf16Lo(v.z) * f, bf16Hi(v.z) * f), tc::pack_bf16x2(bf16Lo(v.w) * f, bf16Hi(v.w) * f));
  }
}

// What the entries of few rows' lists add to the weights' gradient (VocabExact), a block per entry: the first entry of a token adds up
// g rest x over all entries of its token.  Groups of threads that share a row's packs take a part of the entries each, in their order.  On the
// way, what keepRowsKernel does.  (Every entry is compared with every other: the limit keeps that, and a token that all of them share,
// beside the gradient of the logits, which runs at the same time.)
constexpr int FEW_ENTRIES = 2048, OWN_THREADS = 256, OWN_WARPS = OWN_THREADS / 32, AT_ONCE = 4;
__global__ void __launch_bounds__(OWN_THREADS) ownSumsKernel(const uint4* x, const VocabRows rows, int n, int packs, int lanes, const float* rest, const float* gout,
                                                             int goutStride, float* sums, int* where, uint4* kept) {
  __shared__ int list[FEW_ENTRIES];
  __shared__ int counts[AT_ONCE][OWN_WARPS];
  __shared__ float part[OWN_THREADS][9];
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const int k = rows.k, entries = n * k, own = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (own % k == 0) {
    const int row = own / k;
    const bool keep = rowState(rows, row) != ROW_NONE;
    for (int i = threadIdx.x; i < packs; i += OWN_THREADS) kept[(size_t)row * packs + i] = keep ? x[(size_t)row * packs + i] : make_uint4(0u, 0u, 0u, 0u);
  }
  auto tokenOf = [&](int e) { int t; if (rows.targets) rowState(rows, e, t); else t = rows.tokens[e]; return t; };
  const int token = tokenOf(own);
  if (token == VOCAB_NO_TOKEN) return;
  int count = 0;
  for (int base = 0; base < entries; base += OWN_THREADS * AT_ONCE) {
    bool same[AT_ONCE], front = false;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int e = base + u * OWN_THREADS + threadIdx.x;
      same[u] = e < entries && tokenOf(e) == token;
      front = front || (same[u] && e < own);
    }
    if (__syncthreads_or(front)) return;                 // not the first
    uint32_t votes[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      votes[u] = __ballot_sync(0xffffffffu, same[u]);
      if (lane == 0) counts[u][warp] = __popc(votes[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      int at = count + __popc(votes[u] & ((1u << lane) - 1));
#pragma unroll
      for (int w = 0; w < OWN_WARPS; ++w) { at += w < warp ? counts[u][w] : 0; count += counts[u][w]; }
      if (same[u]) list[at] = base + u * OWN_THREADS + threadIdx.x;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) where[token] = own;
  const int groups = OWN_THREADS / lanes, group = threadIdx.x / lanes, per = (count + groups - 1) / groups;
  const int from = min(count, group * per), to = min(count, from + per);
  for (int base = 0; base < packs; base += lanes) {
    const int i = base + (threadIdx.x & (lanes - 1));
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (i < packs) {
#pragma unroll 8
      for (int m = from; m < to; ++m) {
        const int e = list[m], row = e / k;
        vocabMinus(f, -(rest[e] * (gout ? gout[(size_t)row * goutStride] : 1.f)), x[(size_t)row * packs + i]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) part[threadIdx.x][e] = f[e];
    __syncthreads();
    if (group == 0 && i < packs) {
      for (int g = 1; g < groups; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += part[g * lanes + threadIdx.x][e];
      float4* out = (float4*)sums + ((size_t)own * packs + i) * 2;
      out[0] = make_float4(f[0], f[1], f[2], f[3]); out[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  }
}

// x with zeros in the rows without a list: in the product of the weights' gradient they meet the zeros of the logits' gradient, and nothing
// that x holds there (infinities, NaN) may come through.  n d 4 bytes: 8192 x 1024 takes 15 us (cold) beside the 1700 of the losses and gradients.
__global__ void __launch_bounds__(256) keepRowsKernel(const uint4* x, const VocabRows rows, int n, int packs, uint4* out) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  for (int row = blockIdx.x; row < n; row += gridDim.x) {
    const bool keep = rowState(rows, row) != ROW_NONE;
    for (int i = threadIdx.x; i < packs; i += 256) out[(size_t)row * packs + i] = keep ? x[(size_t)row * packs + i] : make_uint4(0u, 0u, 0u, 0u);
  }
}

// out = factor times the sum of the slices, rounded once; `packs` of 8 elements, `rowPacks` to a row.  which: what `exact` adds, as in the products'
// own epilogue: 1 of dx, 2 of dw, 0 nothing.
__global__ void __launch_bounds__(256) joinSlicesKernel(const float* part, int slices, size_t packs, int rowPacks, const VocabFactor factor, const VocabExact exact,
                                                        int which, __nv_bfloat16* out) {
  tc::grid_dependency_wait();
  tc::grid_launch_dependents();
  const float scale = vocabFactor(factor);
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < packs; i += (size_t)gridDim.x * 256) {
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < slices; ++s) {                  // (eight on their way at a time: few rows leave few threads and many slices, 49 at 50257 columns)
      const float4* src = (const float4*)part + ((size_t)s * packs + i) * 2;
      const float4 x = src[0], y = src[1];
      f[0] += x.x; f[1] += x.y; f[2] += x.z; f[3] += x.w; f[4] += y.x; f[5] += y.y; f[6] += y.z; f[7] += y.w;
    }
    if (which) {
      const int row = (int)(i / rowPacks), c = (int)(i - (size_t)row * rowPacks);
      if (which == 1) {
        vocabExactX<1>(f, exact, row, rowPacks * 8, c * 8, 1);
      } else if (const float* sums = vocabSumsOf(exact, exact.first + row, rowPacks * 8)) {
        const float4 p = ((const float4*)sums)[2 * c], q = ((const float4*)sums)[2 * c + 1];
        f[0] -= p.x; f[1] -= p.y; f[2] -= p.z; f[3] -= p.w; f[4] -= q.x; f[5] -= q.y; f[6] -= q.z; f[7] -= q.w;
      }
    }
    ((uint4*)out)[i] = make_uint4(tc::pack_bf16x2(f[0] * scale, f[1] * scale), tc::pack_bf16x2(f[2] * scale, f[3] * scale), tc::pack_bf16x2(f[4] * scale, f[5] * scale),
                                  tc::pack_bf16x2(f[6] * scale, f[7] * scale));
  }
}

ncclResult_t joinSlices(const float* part, int slices, int rows, int d, const VocabFactor& factor, const VocabExact* exact, int which, void* out, cudaStream_t stream) {
  const size_t packs = (size_t)rows * d / 8;
  CUDACHECK(launchBehind(joinSlicesKernel, dim3((unsigned)std::min<size_t>((packs + 255) / 256, 148 * 8)), 256, stream, part, slices, packs, d / 8, factor,
                         exact ? *exact : VocabExact{}, exact ? which : 0, (__nv_bfloat16*)out));
  return ncclSuccess;
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// How a backward pass goes over the vocabulary: columns of the logits' gradient that exist at a time, and what the products need.
struct BackwardPlan {
  int cols;                       // columns of a piece (all of them, or a multiple of the tile)
  VocabPlan cut;
  int slicesX, slicesW;           // of dx those of a whole piece: a shorter last one has fewer and adds to the first of them
  bool sumX, sumW;                // fp32 sums in memory: of dx because there are pieces or slices, of dw because there are slices
  int exact;                      // what the entries add to the results: 0 through dz, 1 by ownSumsKernel, 2 by sorted tokens
  bool dense;                     // of the sorted entries' sums there is a row for every token of the vocabulary
  size_t dz, partX, partW, kept, sums, where, tokens, listed;     // bytes
  size_t all() const { return dz + partX + partW + kept + sums + where + tokens + listed; }
};
// k = 0: targets.  More entries go by sorted tokens (us, GPU, both gradients by themselves / sorted: targets 2048 x 2000 x 64 44 / 51, 4096 68 / 61).
// That costs lists up to as much as one product (1777 x 30011 x 640, lists of 17: 287 us; with the lists' shares rounded to bf16 in dz 238, and both
// gradients 2.3e-3 off instead of 1.7e-3, which is what rounding the results costs).  Only entries that 31 bits do not count go through dz.
BackwardPlan backwardPlan(int n, int v, int d, int k, bool wantX, bool wantW) {
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
  const int64_t entries = (int64_t)n * std::max(1, k);
  p.exact = entries <= FEW_ENTRIES ? 1 : entries <= MOST_SORTED ? 2 : 0;
  p.dense = p.exact == 2 && entries > v;
  p.sums = p.exact && wantW ? up256((p.dense ? (size_t)v : (size_t)entries) * d * 4) : 0;
  p.where = p.exact && wantW ? up256((size_t)v * 4) : 0;
  p.tokens = p.exact == 2 && wantW ? tokenSumsWork((int)entries, d) : 0;
  p.listed = p.exact && wantX && k > 4 ? up256((size_t)n * d * 4) : 0;
  return p;
}

// Loops over pieces end at the first number of rows or columns that is not below the size: at most a piece behind it, and at most 256 for each of
// the pieces, of which the smaller is 742 000 at 2^31.
constexpr int MOST_ROWS = 0x7fffffff - (1 << 20);
// A workspace's parts lie at multiples of 256 bytes behind its beginning, and are accessed 32 bytes at a time.
bool workOk(const void* work) { return work && ((uintptr_t)work & 31) == 0; }
// Below, ordinary logits (hundreds) would leave the exponents that fp32 tells apart by less than a power's range, 2^31; above, T^2 is more than
// what a rounding of fp32 leaves of the loss.
bool temperatureOk(float t) { return t >= 0x1p-20f && t <= 0x1p20f; }
bool sizesOk(int n, int v, int d, int k) {
  return n > 0 && n <= MOST_ROWS && v > 0 && v <= MOST_ROWS && d > 0 && d <= MOST_ROWS && d % 8 == 0 && k > 0 && k <= MAX_LIST;
}

}  // namespace
}  // namespace dfccl

using namespace dfccl;
#define DF_API extern "C" __attribute__((visibility("default")))

DF_API int dfcclLinearLossMaxList(void) { return MAX_LIST; }

DF_API ncclResult_t dfcclTeacherRows(const void* logits, int logitType, const void* tokens, int wide, int n, int k, int v, float temperature, void* outTokens,
                                     void* outWeights, void* state, cudaStream_t stream) {
  const int type = logitType == ncclFloat32 ? 0 : logitType == ncclBfloat16 ? 1 : logitType == ncclFloat16 ? 2 : -1;
  if (!logits || !tokens || !outTokens || !outWeights || !state || type < 0 || !sizesOk(n, v, 8, k) || !temperatureOk(temperature)) return ncclInvalidArgument;
  CUDACHECK(launchBehind(teacherRowsKernel, (n + 3) / 4, 128, stream, logits, type, tokens, wide, n, k, v, 1.f / temperature, (int*)outTokens, (float*)outWeights,
                         (int*)state));
  return ncclSuccess;
}

namespace {
struct ForwardLayout { size_t parts, picked, loss; };
ForwardLayout forwardLayout(int n, int v, int k) {
  return ForwardLayout{up256((size_t)std::min(n, ROWS) * vocabParts(v) * sizeof(float2)), up256((size_t)n * k * 4), up256((size_t)n * 4)};
}
// A target per row, or lists; from row `r` on.
VocabRows rowsOf(const void* targets, int wide, int v, int64_t ignore, const void* tokens, const void* weights, const void* state, int k, float temperature, int r) {
  const size_t at = (size_t)r * k;
  return VocabRows{targets ? (const uint8_t*)targets + (size_t)r * (wide ? 8 : 4) : nullptr, wide, v, (long long)ignore, tokens ? (const int*)tokens + at : nullptr,
                   weights ? (const float*)weights + at : nullptr, state ? (const int*)state + r : nullptr, k, LOG2E / temperature};
}
bool rowsOk(const void* targets, const void* tokens, const void* weights, const void* state, int k, float temperature) {
  return (targets ? k == 1 : tokens && weights && state) && temperatureOk(temperature);
}
}  // namespace

DF_API size_t dfcclLinearLossForwardWork(int n, int v, int k) {
  if (!sizesOk(n, v, 8, k)) return 0;
  const ForwardLayout l = forwardLayout(n, v, k);
  return l.parts + l.picked + l.loss + 256;
}

DF_API ncclResult_t dfcclLinearLossForward(const void* x, const void* w, int n, int v, int d, const void* targets, int wide, int64_t ignore, const void* tokens,
                                           const void* weights, const void* state, int k, float temperature, int reduction, void* work, void* lse, void* rest,
                                           void* rowLoss, void* loss, void* count, cudaStream_t stream) {
  if (!sizesOk(n, v, d, k) || !x || !w || !rowsOk(targets, tokens, weights, state, k, temperature) || !workOk(work) || !lse || !rest || reduction < 0 || reduction > 2) return ncclInvalidArgument;
  if ((((uintptr_t)x | (uintptr_t)w) & 15) || (reduction ? !loss || !count : !rowLoss)) return ncclInvalidArgument;
  const ForwardLayout l = forwardLayout(n, v, k);
  JoinArgs j = {};
  j.parts = (const float2*)work;
  float* picked = (float*)((uint8_t*)work + l.parts);
  j.stretches = vocabParts(v); j.t2 = temperature * temperature;
  float* losses = rowLoss ? (float*)rowLoss : (float*)((uint8_t*)work + l.parts + l.picked);
  j.allRows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, 0);
  j.allLoss = losses; j.all = n; j.mean = reduction == 1;
  j.ticket = reduction ? (int*)((uint8_t*)work + l.parts + l.picked + l.loss) : nullptr;
  j.out = (float*)loss; j.count = (int*)count;
  DFCHECK(pickLogits(PickArgs{(const uint4*)x, (const uint4*)w, j.allRows, n, d / 8, picked, nullptr, nullptr, j.ticket, j.ticket ? 1 : 0, 0}, stream));
  for (int r = 0; r < n; r += ROWS) j.blocks += (std::min(ROWS, n - r) + 31) / 32;
  for (int r = 0; r < n; r += ROWS) {
    j.n = std::min(ROWS, n - r);
    j.picked = picked + (size_t)r * k;
    j.rows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, r);
    j.lse = (float*)lse + r; j.loss = losses + r; j.rest = (float*)rest + (size_t)r * k;
    // (the first beside pickLogitsKernel)
    DFCHECK(vocabStats((const __nv_bfloat16*)x + (size_t)r * d, w, j.n, v, d, j.rows, (float2*)j.parts, nullptr, r == 0, stream));
    CUDACHECK(launchBehind(joinRowsKernel<false>, (j.n + 31) / 32, 1024, stream, j));
  }
  return ncclSuccess;
}

DF_API size_t dfcclLinearLossBackwardWork(int n, int v, int d, int k, int wantX, int wantW) {
  if (!sizesOk(n, v, d, std::max(1, k)) || k < 0 || !(wantX || wantW)) return 0;
  const BackwardPlan p = backwardPlan(n, v, d, k, wantX != 0, wantW != 0);
  return p.all();
}

DF_API ncclResult_t dfcclLinearLossBackward(const void* x, const void* w, int n, int v, int d, const void* targets, int wide, int64_t ignore, const void* tokens,
                                            const void* weights, const void* state, int k, float temperature, const void* lse, const void* rest,
                                            const void* gout, int goutStride, const void* count, void* dx, void* dw, void* work, size_t workBytes, cudaStream_t stream) {
  if (!sizesOk(n, v, d, k) || !x || !w || !rowsOk(targets, tokens, weights, state, k, temperature) || !lse || !rest || !gout || !workOk(work) || !(dx || dw) || goutStride < 0) return ncclInvalidArgument;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw) & 15) return ncclInvalidArgument;
  const BackwardPlan p = backwardPlan(n, v, d, targets ? 0 : k, dx != nullptr, dw != nullptr);
  if (p.all() > workBytes) return ncclInvalidArgument;          // (the setting has changed since the size was asked for)
  void* dz = work;
  float* partX = p.sumX ? (float*)((uint8_t*)work + p.dz) : nullptr;
  float* partW = p.sumW ? (float*)((uint8_t*)work + p.dz + p.partX) : nullptr;
  uint8_t* at = (uint8_t*)work + p.dz + p.partX + p.partW;
  void* kept = at;
  float* sums = (float*)(at + p.kept);
  int* where = (int*)(at + p.kept + p.sums);
  void* sorted = at + p.kept + p.sums + p.where;
  float* listed = p.listed ? (float*)(at + p.kept + p.sums + p.where + p.tokens) : nullptr;
  const VocabRows rows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, 0);
  const float* rowGout = goutStride ? (const float*)gout : nullptr;
  if (listed) CUDACHECK(launchBehind(listSumsKernel, std::min(n, 148 * 16), 128, stream, (const uint4*)w, rows, (const float*)rest, n, d / 8, (float4*)listed));
  if (dw && p.exact == 1) {
    int lanes = 8;
    while (lanes < OWN_THREADS && lanes < d / 8) lanes *= 2;
    CUDACHECK(launchBehind(ownSumsKernel, n * k, OWN_THREADS, stream, (const uint4*)x, rows, n, d / 8, lanes, (const float*)rest, rowGout, goutStride, sums, where,
                           (uint4*)kept));
  } else if (dw) {
    if (p.exact) {
      DFCHECK(targets ? tokenSort(n, d, targets, wide, ignore, v, sorted, stream) : tokenSort(n * k, d, tokens, 0, -1, v, sorted, stream));
      DFCHECK(tokenSums(x, n * k, d, k, v, (const float*)rest, rowGout, goutStride, sums, p.dense, where, sorted, stream));
    }
    CUDACHECK(launchBehind(keepRowsKernel, std::min(n, 148 * 8), 256, stream, (const uint4*)x, rows, n, d / 8, (uint4*)kept));
  }
  const VocabGrad grad{(const float*)lse, rowGout, goutStride, p.exact ? nullptr : (const float*)rest};
  VocabExact exact{rows, nullptr, (const float*)rest, rowGout, goutStride, (const __nv_bfloat16*)w, sums, where,
                   p.exact == 2 && dw ? tokenSortItems(n * k, d, v, sorted) : nullptr, p.exact ? n * k : 0, 0, p.dense, listed};
  const VocabExact* add = p.exact ? &exact : nullptr;
  const VocabFactor factor{goutStride ? nullptr : (const float*)gout, (const int*)count, temperature};
  for (int c = 0; c < v; c += p.cols) {
    const int cols = std::min(p.cols, v - c);
    const __nv_bfloat16* wc = (const __nv_bfloat16*)w + (size_t)c * d;
    __nv_bfloat16* dwc = dw ? (__nv_bfloat16*)dw + (size_t)c * d : nullptr;
    DFCHECK(vocabGrad(x, wc, n, cols, c, d, rows, grad, dz, dw && c == 0, stream));      // (beside the launch in front)
    exact.first = c;
    DFCHECK(vocabProducts(dz, kept, wc, n, cols, d, p.cut, factor, add, VocabResult{p.sumX ? nullptr : dx, partX, c != 0}, VocabResult{p.sumW ? nullptr : dwc, partW, false}, stream));
    if (p.sumW) DFCHECK(joinSlices(partW, p.slicesW, cols, d, factor, add, 2, dwc, stream));
  }
  if (p.sumX) DFCHECK(joinSlices(partX, p.slicesX, n, d, factor, add, 1, dx, stream));
  return ncclSuccess;
}

namespace {
// How a pass with gradients goes over the rows, and where its parts of the workspace begin.
struct OneGoPlan {
  int rows;                       // of a piece (all of them, or a multiple of the tile)
  VocabPlan cut;
  int slicesX, slicesW;
  bool sumX, sumW, dense;         // dense: of the entries' sums there is a row for every token of the vocabulary
  size_t listedBytes, listed, powers, parts, partX, partW, shared, base, share, losses, words, where, sums, tokens, picked, bytes;
};
OneGoPlan oneGoPlan(int n, int v, int d, int k, bool wantX, bool wantW) {
  OneGoPlan p = {};
  const size_t ld = (size_t)(v + 63) / 64 * 64;
  const int64_t limit = std::max<int64_t>(1 << 20, paramI64("LOSS_WORKSPACE_BYTES", 1ll << 30));
  const int64_t most = std::max<int64_t>(1, limit / (int64_t)(2 * ld) / VOCAB_TILE) * VOCAB_TILE;
  const int64_t pieces = (n + most - 1) / most;
  p.rows = pieces == 1 ? n : (int)(((n + pieces - 1) / pieces + VOCAB_TILE - 1) / VOCAB_TILE * VOCAB_TILE);
  p.cut = vocabProductPlan(p.rows, v, d, wantX, wantW, gemmPairResident());
  p.slicesX = vocabSlices(v, p.cut.perX);
  p.slicesW = vocabSlices(p.rows, p.cut.perW);
  p.sumX = wantX && p.slicesX > 1;
  p.sumW = wantW && (pieces > 1 || p.slicesW > 1);
  auto take = [&](size_t bytes) { const size_t at = p.bytes; p.bytes += up256(bytes); return at; };
  p.powers = take(p.rows * ld * 2);
  p.parts = take((size_t)p.rows * vocabParts(v) * sizeof(float2));
  p.partX = take(p.sumX ? (size_t)p.slicesX * p.rows * d * 4 : 0);
  p.partW = take(p.sumW ? (size_t)p.slicesW * v * d * 4 : 0);
  p.shared = take(wantW ? (size_t)p.rows * d * 2 : 0);
  p.base = take((size_t)n * 4); p.share = take((size_t)n * 4); p.losses = take((size_t)n * 4); p.picked = take((size_t)n * k * 4);
  p.words = take((size_t)(pieces + 1) * 4);
  p.where = take(wantW ? (size_t)v * 4 : 0);
  p.dense = (int64_t)n * k > v;
  p.sums = take(wantW ? (p.dense ? (size_t)v : (size_t)n * k) * d * 4 : 0);
  p.tokens = take(wantW ? tokenSumsWork(n * k, d) : 0);
  p.listedBytes = wantX && k > 4 ? (size_t)p.rows * d * 4 : 0;
  p.listed = take(p.listedBytes);
  return p;
}
}  // namespace

DF_API size_t dfcclLinearLossWithGradientsWork(int n, int v, int d, int k, int wantX, int wantW) {
  return sizesOk(n, v, d, k) && (int64_t)n * k <= MOST_SORTED && (wantX || wantW) ? oneGoPlan(n, v, d, k, wantX != 0, wantW != 0).bytes : 0;
}

// Per piece of rows: powers of the logits relative to the largest of the row's list (vocabPowers), their sums, x times the rows' shares, the two
// products.  What the lists themselves add to the gradients does not go through bf16 (VocabExact).  Rows with a power that is too
// large send their piece through statistics and powers once more, with the logarithms of the sums as bases: launches that find nothing
// to do otherwise (2 us each).  That is 10 n v d of such a piece, more than the 8 of gradients apart from the loss: 8192 x 50257 x 1024 1806 us without
// such a row, 2919 with one, 2630 apart.  It takes a loss above 41.6 (60 ln 2), four times that of a uniform guess among 50257.
DF_API ncclResult_t dfcclLinearLossWithGradients(const void* x, const void* w, int n, int v, int d, const void* targets, int wide, int64_t ignore, const void* tokens,
                                                 const void* weights, const void* state, int k, float temperature, int reduction, void* work, size_t workBytes,
                                                 void* lse, void* rest, void* loss, void* count, void* dx, void* dw, cudaStream_t stream) {
  if (!sizesOk(n, v, d, k) || (int64_t)n * k > MOST_SORTED || !x || !w || !rowsOk(targets, tokens, weights, state, k, temperature) || !workOk(work) || !lse ||
      !rest || !loss || !count || !(dx || dw) || reduction < 1 || reduction > 2)
    return ncclInvalidArgument;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw) & 15) return ncclInvalidArgument;
  const OneGoPlan p = oneGoPlan(n, v, d, k, dx != nullptr, dw != nullptr);
  if (p.bytes > workBytes) return ncclInvalidArgument;           // (the setting has changed since the size was asked for)
  uint8_t* at = (uint8_t*)work;
  void* powers = at + p.powers;
  float2* parts = (float2*)(at + p.parts);
  float* partX = p.sumX ? (float*)(at + p.partX) : nullptr;
  float* partW = p.sumW ? (float*)(at + p.partW) : nullptr;
  float *base = (float*)(at + p.base), *share = (float*)(at + p.share), *losses = (float*)(at + p.losses);
  int *words = (int*)(at + p.words), *where = (int*)(at + p.where);
  const VocabRows all = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, 0);
  const int pieces = (n + p.rows - 1) / p.rows, packs = d / 8;
  float* picked = (float*)(at + p.picked);
  float* listed = p.listedBytes ? (float*)(at + p.listed) : nullptr;
  if (dw) DFCHECK(targets ? tokenSort(n, d, targets, wide, ignore, v, at + p.tokens, stream) : tokenSort(n * k, d, tokens, 0, -1, v, at + p.tokens, stream));
  DFCHECK(pickLogits(PickArgs{(const uint4*)x, (const uint4*)w, all, n, packs, picked, base, (int*)count, words, pieces + 1, dw ? 1 : 0}, stream));
  const VocabFactor factor{nullptr, reduction == 1 ? (const int*)count : nullptr, temperature};
  JoinArgs j = {};
  j.parts = parts; j.stretches = vocabParts(v); j.t2 = temperature * temperature;
  j.allRows = all; j.allLoss = losses; j.all = n; j.mean = reduction == 1;
  j.out = (float*)loss; j.count = (int*)count;
  for (int r = 0; r < n; r += p.rows) j.blocks += (std::min(p.rows, n - r) + 31) / 32;
  for (int i = 0; i < pieces; ++i) {
    const int r = i * p.rows, m = std::min(p.rows, n - r);
    const __nv_bfloat16* xr = (const __nv_bfloat16*)x + (size_t)r * d;
    j.rows = rowsOf(targets, wide, v, ignore, tokens, weights, state, k, temperature, r);
    j.n = m; j.lse = (float*)lse + r; j.loss = losses + r; j.base = base + r; j.share = share + r;
    j.picked = picked + (size_t)r * k; j.rest = (float*)rest + (size_t)r * k;
    j.x = (const uint4*)xr; j.shared = dw ? (uint4*)(at + p.shared) : nullptr; j.packs = packs;
    DFCHECK(vocabPowers(xr, w, m, v, d, j.rows, base + r, parts, powers, nullptr, stream));
    j.again = words + 1 + i; j.only = nullptr; j.ticket = nullptr;
    CUDACHECK(launchBehind(joinRowsKernel<true>, (m + 31) / 32, 1024, stream, j));
    DFCHECK(vocabStats(xr, w, m, v, d, j.rows, parts, j.again, false, stream));
    j.only = j.again; j.ticket = words;
    CUDACHECK(launchBehind(joinRowsKernel<false>, (m + 31) / 32, 1024, stream, j));
    DFCHECK(vocabPowers(xr, w, m, v, d, j.rows, base + r, parts, powers, j.again, stream));
    if (dw && i == pieces - 1) DFCHECK(tokenSums(x, n * k, d, k, v, (const float*)rest, nullptr, 0, (float*)(at + p.sums), p.dense, where, at + p.tokens, stream));
    if (listed)
      CUDACHECK(launchBehind(listSumsKernel, std::min(m, 148 * 16), 128, stream, (const uint4*)w, j.rows, (const float*)rest + (size_t)r * k, m, packs, (float4*)listed));
    const VocabExact exact{j.rows, share + r, (const float*)rest + (size_t)r * k, nullptr, 0, (const __nv_bfloat16*)w, (const float*)(at + p.sums), where,
                           dw ? tokenSortItems(n * k, d, v, at + p.tokens) : nullptr, n * k, 0, p.dense, listed};
    __nv_bfloat16* dxr = dx ? (__nv_bfloat16*)dx + (size_t)r * d : nullptr;
    // (a shorter last piece has fewer slices of dw: it adds to the first of them)
    DFCHECK(vocabProducts(powers, at + p.shared, w, m, v, d, p.cut, factor, &exact, VocabResult{p.sumX ? nullptr : dxr, partX, false},
                          VocabResult{p.sumW ? nullptr : dw, partW, i != 0}, stream));
    if (p.sumX) DFCHECK(joinSlices(partX, p.slicesX, m, d, factor, &exact, 1, dxr, stream));
    if (p.sumW && i == pieces - 1) DFCHECK(joinSlices(partW, p.slicesW, v, d, factor, &exact, 2, dw, stream));
  }
  return ncclSuccess;
}

DF_API uint64_t dfcclCaptureId(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) { (void)cudaGetLastError(); return 0; }
  return status == cudaStreamCaptureStatusNone ? 0 : id;
}

DF_API ncclResult_t dfcclScaleResults(void* a, size_t na, void* b, size_t nb, const void* scale, cudaStream_t stream) {
  if (!scale || na % 8 || nb % 8 || (na && !a) || (nb && !b) || !(na || nb) || (((uintptr_t)a | (uintptr_t)b) & 15)) return ncclInvalidArgument;
  const size_t packs = (na + nb) / 8;
  CUDACHECK(launchBehind(scaleResultsKernel, dim3((unsigned)std::min<size_t>((packs + 255) / 256, 148 * 8)), 256, stream, (uint4*)a, na / 8, (uint4*)b, nb / 8,
                         (const float*)scale));
  return ncclSuccess;
}

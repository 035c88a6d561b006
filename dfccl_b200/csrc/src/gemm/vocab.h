// Internal interface of the products over a vocabulary (tcgen05_vocab.cu), for the losses of a language model's head (ops/loss.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "dfccl.h"

namespace dfccl {

constexpr int VOCAB_TILE = 256;              // rows and columns of a tile
constexpr int VOCAB_NO_TOKEN = 0x7fffffff;   // behind the last entry of a row's list

// What the rows of logits are compared with: a target each (`targets`), or a list of vocabulary entries in ascending order (VOCAB_NO_TOKEN
// behind the last one) with the weight of each.  A target is a list of one entry of weight 1.
struct VocabRows {
  const void* targets;          // [n] 64-bit integers (wide) or 32-bit, or null: lists
  int wide, v;                  // v: of the whole vocabulary
  long long ignore;
  const int* tokens;            // [n][k]
  const float* weights;         // [n][k]
  const int* state;             // [n]
  int k;                        // 1 beside targets
  float scale;                  // logits -> exponents of two: log2(e) / temperature
};
enum RowState { ROW_NONE = 0, ROW_LIST = 1, ROW_BAD = 2 };      // nothing to compare with; something; a token outside the vocabulary

#if defined(__CUDACC__)
__device__ __forceinline__ int rowState(const VocabRows& r, int row, int& token) {
  if (!r.targets) { token = VOCAB_NO_TOKEN; return r.state[row]; }
  const long long t = r.wide ? ((const long long*)r.targets)[row] : ((const int*)r.targets)[row];
  const bool in = t >= 0 && t < r.v && t != r.ignore;
  token = in ? (int)t : VOCAB_NO_TOKEN;
  return in ? ROW_LIST : t == r.ignore ? ROW_NONE : ROW_BAD;
}
__device__ __forceinline__ int rowState(const VocabRows& r, int row) { int token; return rowState(r, row, token); }
#endif

inline int vocabParts(int v) { return (v + VOCAB_TILE - 1) / VOCAB_TILE; }

// z = x [n, d] w[v, d]^T, tile by tile and never stored.  Of every row, for each of the vocabParts(v) stretches of its columns and without the
// entries of its list: {largest z scale, sum of 2^(z scale - that)} -> parts [stretch][n].  (The tensor cores cut off what does not fit an
// accumulator, step by step: a logit of 20 from 1024 products of one sign is 2.5e-5 too small, one of 4096 products 9e-5.  The logits that stand
// out, and that a loss is the difference to, are computed apart.)  `only`, where given: nothing happens unless it holds something other than 0.
// `early`: the launch in front of this one writes nothing that this one reads or writes, and lets it start when everything further in front
// has ended; the two run side by side.
ncclResult_t vocabStats(const void* x, const void* w, int n, int v, int d, const VocabRows& rows, float2* parts, const int* only, bool early, cudaStream_t stream);

// powers = 2^(z scale - base) of every row with a target, 0 elsewhere: bf16, [n][ld], ld = v rounded up to 64 (zeros behind v).  Of each stretch
// of a row's columns, without its target: {largest exponent, sum of the powers in fp32} -> parts [stretch][n].
ncclResult_t vocabPowers(const void* x, const void* w, int n, int v, int d, const VocabRows& rows, const float* base, float2* parts, void* powers, const int* only,
                         cudaStream_t stream);

// What all rows' gradients share: the gradient of the reduced loss, a mean's count, the temperature.  It does not go into dz, where its
// rounding to bf16 would be the same for all of them (a mean over 32113 rows: dx 3.1e-3 off, 1.7e-3 without), but into the results.
struct VocabFactor {
  const float* gout;            // one value, or null: the rows have their own
  const int* count;             // rows that share a mean, or null
  float temperature;
};
// dz = g (2^(z scale - lse) - weight where an entry is in the list), 0 in rows without a list and NaN in those with a token outside the
// vocabulary, for the columns [0, v) of w, which start at column `first` of the vocabulary: bf16, [n][ld], ld = v rounded up to 64 (zeros behind v).
struct VocabGrad {
  const float* lse;             // [n] log2 of the sum of 2^(z scale)
  const float* gout;            // g [n], or null: 1
  int goutStride;
};
ncclResult_t vocabGrad(const void* x, const void* w, int n, int v, int first, int d, const VocabRows& rows, const VocabGrad& grad, void* dz, bool early,
                       cudaStream_t stream);

#if defined(__CUDACC__)
__device__ __forceinline__ float vocabFactor(const VocabFactor& f) {
  float s = f.gout ? *f.gout * f.temperature : f.temperature;
  if (f.count) s /= (float)max(1, *f.count);
  return s;
}
#endif

// How the contractions of the two products are cut: blocks of 64 in a slice.
struct VocabPlan { int perX, perW; };
VocabPlan vocabProductPlan(int n, int v, int d, bool wantX, bool wantW, int pairs);
inline int vocabSlices(int k, int per) { return ((k + 63) / 64 + per - 1) / per; }

// Where dz is not the gradient of the logits but their powers (vocabPowers, targets only): what is missing of both results, in fp32.
//   dx_n = factor (scale_n (powers w)_n - w_target(n)),   dw_t = factor ((powers^T x')_t - sums_where(t))
// with x' = scale_n x_n as the right operand, sums_where(t) the sum of the x_n whose target is t.
struct VocabExact {
  VocabRows rows;               // of the n rows
  const float* scale;           // [n]
  const __nv_bfloat16* w;       // [v, d]
  const float* sums;            // rows of d
  const int* where;             // [v] a row of sums, or -1
};

// dx [n, d] = factor dz w and dw [v, d] = factor dz^T x in one launch.  A result is bf16 where `out` is given; otherwise `part` gets an fp32
// sum [slice][rows][d] of each slice of the contraction, without the factor and without what `exact` (may be null) adds, on top of what is
// there with `add`.  A result with neither is left out.
struct VocabResult {
  void* out;
  float* part;
  bool add;
};
ncclResult_t vocabProducts(const void* dz, const void* x, const void* w, int n, int v, int d, const VocabPlan& plan, const VocabFactor& factor, const VocabExact* exact,
                           const VocabResult& dx, const VocabResult& dw, cudaStream_t stream);

#if defined(__CUDACC__)
// Eight elements of a row of dx or dw from their sums.
__device__ __forceinline__ void vocabMinus(float (&f)[8], const float4* p) {
  const float4 a = p[0], b = p[1];
  f[0] -= a.x; f[1] -= a.y; f[2] -= a.z; f[3] -= a.w; f[4] -= b.x; f[5] -= b.y; f[6] -= b.z; f[7] -= b.w;
}
__device__ __forceinline__ void vocabExactX(float (&f)[8], int state, float scale, const uint4* target) {
  if (state != ROW_LIST) {
    const float none = state == ROW_BAD ? __int_as_float(0x7fffffff) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = none;
    return;
  }
  const uint4 t = *target;
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = fmaf(f[2 * e], scale, -__uint_as_float(w[e] << 16));
    f[2 * e + 1] = fmaf(f[2 * e + 1], scale, -__uint_as_float(w[e] & 0xffff0000u));
  }
}
#endif

}  // namespace dfccl

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

// powers = 2^(z scale - base) of every row with a list, 0 in the places of its entries and elsewhere: bf16, [n][ld], ld = v rounded up to 64 (zeros
// behind v).  Of each stretch of a row's columns, without the list's: {largest exponent, sum of the powers in fp32} -> parts [stretch][n].
ncclResult_t vocabPowers(const void* x, const void* w, int n, int v, int d, const VocabRows& rows, const float* base, float2* parts, void* powers, const int* only,
                         cudaStream_t stream);

// What all rows' gradients share: the gradient of the reduced loss, a mean's count, the temperature.  It does not go into dz, where its
// rounding to bf16 would be the same for all of them (a mean over 32113 rows: dx 3.1e-3 off, 1.7e-3 without), but into the results.
struct VocabFactor {
  const float* gout;            // one value, or null: the rows have their own
  const int* count;             // rows that share a mean, or null
  float temperature;
};
// dz = g 2^(z scale - lse), for the entries of a row's list -g rest instead (0 where `rest` is null), 0 in rows without a list and NaN in those with a token
// outside the vocabulary, for the columns [0, v) of w, which start at column `first` of the vocabulary: bf16, [n][ld], ld = v rounded up to 64
// (zeros behind v).
struct VocabGrad {
  const float* lse;             // [n] log2 of the sum of 2^(z scale)
  const float* gout;            // g [n], or null: 1
  int goutStride;
  const float* rest;            // [n][k] an entry's weight less its probability; of entries of one token all of it in the first
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

// What the entries of the rows' lists add to both results, in fp32, where dz has zeros in their places.  It is most of both: of few rows
// its rounding in dz would be as large as that of the results.
//   dx_n = factor (scale_n (dz w)_n - g_n sum_k rest_nk w_token(n,k)),   dw_t = factor ((dz^T x)_t - sums_where(t))
// sums_where(t): the sum of g_n rest_nk x_n over the entries of token t.
struct VocabExact {
  VocabRows rows;               // of the n rows
  const float* scale;           // [n], or null: 1
  const float* rest;            // [n][k]
  const float* gout;            // g [n], or null: 1
  int goutStride;
  const __nv_bfloat16* w;       // [v, d], the whole vocabulary
  const float* sums;            // rows of d
  const int* where;             // [v] a row of sums; of a token that no list has it may be anything:
  const uint2* items;           // it counts where items[that].x is the token, or where, with items null, the rows' entry of that number is
  int entries;                  // of items or of the rows
  int first;                    // token of dw's first row
  bool dense;                   // sums has a row for every token, at its number
  const float* listed;          // [n][d] sum_k rest_nk w_token(n,k), or null: from w on the way
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
// The row of sums of a token, or null.
__device__ __forceinline__ const float* vocabSumsOf(const VocabExact& x, int token, int d) {
  const int at = x.where[token];
  if (at < 0 || at >= x.entries) return nullptr;
  int own;
  if (x.items) own = (int)x.items[at].x;
  else if (x.rows.targets) rowState(x.rows, at, own);
  else own = x.rows.tokens[at];
  return own == token ? x.sums + (size_t)(x.dense ? token : at) * d : nullptr;
}
__device__ __forceinline__ void vocabMinus(float* f, float weight, const uint4& w) {
  const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = fmaf(-weight, __uint_as_float(p[e] << 16), f[2 * e]);
    f[2 * e + 1] = fmaf(-weight, __uint_as_float(p[e] & 0xffff0000u), f[2 * e + 1]);
  }
}
// P packs of eight columns of a row of dx from their sums, from column c of d on (the first `packs` of them).
template <int P>
__device__ __forceinline__ void vocabExactX(float (&f)[8 * P], const VocabExact& x, int row, int d, int c, int packs) {
  int token;
  const int state = rowState(x.rows, row, token);
  if (state != ROW_LIST) {
    const float none = state == ROW_BAD ? __int_as_float(0x7fffffff) : 0.f;
#pragma unroll
    for (int e = 0; e < 8 * P; ++e) f[e] = none;
    return;
  }
  if (x.scale) {
    const float s = x.scale[row];
#pragma unroll
    for (int e = 0; e < 8 * P; ++e) f[e] *= s;
  }
  const float g = x.gout ? x.gout[(size_t)row * x.goutStride] : 1.f;
  if (x.listed) {
    const float4* src = (const float4*)(x.listed + (size_t)row * d + c);
#pragma unroll
    for (int v = 0; v < 2 * P; ++v) {
      if (v / 2 >= packs) break;
      const float4 q = src[v];
      f[4 * v] = fmaf(-g, q.x, f[4 * v]); f[4 * v + 1] = fmaf(-g, q.y, f[4 * v + 1]);
      f[4 * v + 2] = fmaf(-g, q.z, f[4 * v + 2]); f[4 * v + 3] = fmaf(-g, q.w, f[4 * v + 3]);
    }
    return;
  }
  const size_t at = (size_t)row * x.rows.k;
  for (int i = 0; i < x.rows.k; i += 2) {
    const uint4* src[2];
    float weight[2];
    uint4 w[2][P];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = x.rows.targets ? u ? VOCAB_NO_TOKEN : token : i + u < x.rows.k ? x.rows.tokens[at + i + u] : VOCAB_NO_TOKEN;
      weight[u] = t == VOCAB_NO_TOKEN ? 0.f : g * x.rest[at + i + u];
      src[u] = (const uint4*)(x.w + (size_t)(t == VOCAB_NO_TOKEN ? 0 : t) * d + c);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int v = 0; v < P; ++v) w[u][v] = weight[u] != 0.f && v < packs ? src[u][v] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (weight[u] == 0.f) continue;
#pragma unroll
      for (int v = 0; v < P; ++v) vocabMinus(f + 8 * v, weight[u], w[u][v]);
    }
  }
}
#endif

}  // namespace dfccl

// Internal interface of the products over a vocabulary (tcgen05_vocab.cu), for the losses of a language model's head (ops/loss.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "dfccl.h"

namespace dfccl {

constexpr int VOCAB_TILE = 256;              // rows and columns of a tile
constexpr int VOCAB_PARTS = 2;               // epilogue warps that share 32 rows of a tile: each leaves a maximum and a sum of its own
constexpr int VOCAB_NO_TOKEN = 0x7fffffff;   // behind the last entry of a row's list

// What a row of logits is compared with: a list of vocabulary entries in ascending order (VOCAB_NO_TOKEN behind the last one) with the
// weight of each.  One entry of weight 1 is a target of the cross entropy.
struct VocabRows {
  const int* tokens;            // [n][k]
  const float* weights;         // [n][k], or null: 1
  int k;
  float scale;                  // logits -> exponents of two: log2(e) / temperature
};

inline int vocabParts(int v) { return (v + VOCAB_TILE - 1) / VOCAB_TILE * VOCAB_PARTS; }

// z = x [n, d] w[v, d]^T, tile by tile and never stored.  Of every row: for each of the vocabParts(v) stretches of its columns
// {largest z scale, sum of 2^(z scale - that)} -> parts [stretch][n], and the z of its list's entries -> picked [n][k].
ncclResult_t vocabStats(const void* x, const void* w, int n, int v, int d, const VocabRows& rows, float2* parts, float* picked, cudaStream_t stream);

// dz = coef (2^(z scale - lse) - weight where an entry is in the list) for the columns [0, v) of w, which start at column `first` of the
// vocabulary: bf16, [n][ld], ld = v rounded up to 64 (zeros behind v).
struct VocabGrad {
  const float* lse;             // [n] log2 of the sum of 2^(z scale)
  const float* gout;            // gradient of the loss: [n] or, with goutStride 0, one
  int goutStride;
  const int* count;             // rows that share a mean, or null
  const int* state;             // [n] 0: no gradient, 1: a row with a list, 2: a row with a token outside the vocabulary (NaN)
  float temperature;
};
ncclResult_t vocabGrad(const void* x, const void* w, int n, int v, int first, int d, const VocabRows& rows, const VocabGrad& grad, void* dz, cudaStream_t stream);

// How the contractions of the two products are cut: blocks of 64 in a slice.
struct VocabPlan { int perX, perW; };
VocabPlan vocabProductPlan(int n, int v, int d, bool wantX, bool wantW, int pairs);
inline int vocabSlices(int k, int per) { return ((k + 63) / 64 + per - 1) / per; }

// dx [n, d] = dz w and dw [v, d] = dz^T x in one launch; either may be left out (null).  dx is bf16 where `partX` is null, otherwise
// an fp32 sum [slice][n][d] of each slice of the vocabulary, added to what is there with `addX`; dw likewise with partW.
ncclResult_t vocabProducts(const void* dz, const void* x, const void* w, int n, int v, int d, const VocabPlan& plan, void* dx, float* partX, bool addX,
                           void* dw, float* partW, cudaStream_t stream);

}  // namespace dfccl

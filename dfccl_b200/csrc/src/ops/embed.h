// Sums of rows by token, for the losses of a language model's head (embed.cu, loss.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "dfccl.h"

namespace dfccl {

// Sorts n tokens that are inside [0, v) and not `ignore`, by token and number; the others are behind them as v.  work: tokenSumsWork bytes.
size_t tokenSumsWork(int n, int d);
ncclResult_t tokenSort(int n, int d, const void* ids, int wide, int64_t ignore, int v, void* work, cudaStream_t stream);
// The sorted (token, number) [n], once it has run.
const uint2* tokenSortItems(int n, int d, int v, void* work);
// Behind it, with the same work: for every token the fp32 sum of weights_i gout_r x_r over its numbers i, r = i / perRow (x [n / perRow, d] bf16, d % 8
// == 0; gout may be null), in their order, -> row where[token] of sums [n][d], the place of one of the token's items, or with `dense` row `token`
// of sums [v][d].  Entries of `where` [v] of other tokens are left as they are.
ncclResult_t tokenSums(const void* x, int n, int d, int perRow, int v, const float* weights, const float* gout, int goutStride, float* sums, bool dense, int* where,
                       void* work, cudaStream_t stream);

}  // namespace dfccl

// Sums of rows by token, for the losses of a language model's head (embed.cu, loss.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "dfccl.h"

namespace dfccl {

// The fp32 sum of the rows of x [n, d] (bf16, d % 8 == 0) for every token of ids that is inside [0, v) and not `ignore`, in the order of the
// rows: row where[token] of sums [n][d].  Entries of `where` [v] of other tokens are left as they are.  work: tokenSumsWork bytes.
size_t tokenSumsWork(int n, int d);
ncclResult_t tokenSums(const void* x, int n, int d, const void* ids, int wide, int64_t ignore, int v, float* sums, int* where, void* work, cudaStream_t stream);

}  // namespace dfccl

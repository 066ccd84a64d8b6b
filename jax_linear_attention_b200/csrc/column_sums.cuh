// Column sums in two steps that give the same bits every time: kernels that walk rows leave one row of partial sums per
// block in a workspace, and column_sums() adds those rows up in a fixed order. (Atomics would add them as they come.)
#pragma once

#include "common.cuh"

namespace jla {

// out[c] = sum over p of partial[p * cols + c]; `parts` rows, enqueued on `stream`; returns a jla_status.
int column_sums(const float* partial, int parts, int cols, float* out, cudaStream_t stream);

// At most this many blocks walk the rows of one column range.
constexpr int kMaxParts = 592;  // 4 blocks on each of 148 SMs

}  // namespace jla

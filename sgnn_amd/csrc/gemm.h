// The matrix product behind sgnn_linear and its backward pass (gemm.hip).
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace sgnn {

// C[m][n] = act(sum_k A(m, k) B(n, k) + bias[n]) + res[m][n].
// An operand is stored with k contiguous ("rows": A[m * lda + k]) or, where a_cols / b_cols is set, with m / n
// contiguous (A[k * lda + m]).  All operands are of type dtype.
struct Gemm {
  int32_t dtype = 0;
  int64_t M = 0, N = 0, K = 0;
  const void* A = nullptr;
  int64_t lda = 0;
  bool a_cols = false;
  // 16-bit types with b_cols: half of A in two planes (ops_types.h, split2), the second lo bytes behind the first (0: one
  // plane, A as it is).
  int64_t lo = 0;
  const void* B = nullptr;
  int64_t ldb = 0;
  bool b_cols = false;
  const void* bias = nullptr;
  int32_t act = 0;
  const void* res = nullptr;
  int64_t ldr = 0;
  float* slope = nullptr;  // act'(sum + bias), dense [M][N] as sgnn_linear describes it
  void* C = nullptr;
  int64_t ldc = 0;
};

size_t gemm_workspace_bytes(const Gemm& g);
int gemm_run(const Gemm& g, void* workspace, size_t workspace_bytes, void* stream);

}  // namespace sgnn

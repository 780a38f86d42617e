// Projections with 4-bit weights and group scales (w4.cu).
#pragma once
#include "common.cuh"

namespace b200mm {

// y[m, n] = epilogue(sum_k x[m, k] (u[n, k] - 8) s[n, k / G]); u: 4 bits, two to
// a byte, the even column low.
struct W4Args {
  const void* x; int64_t ldx;                          // [M, K] dtype
  const uint8_t* w0; const uint8_t* w1; int64_t ldw;   // [N, K / 2], row stride in bytes (w1: up weights, gate only)
  const void* s0; const void* s1; int64_t lds;         // [N, K / G] dtype
  void* y; int64_t ldy;                                // [M, N] dtype
  int M, N, K, G;
  int dtype;                                           // B200MM_F16 / BF16
  bool gate;                                           // silu(gate) * up
  void* ws;
  cudaStream_t stream;
};

size_t w4_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gate);
int w4_run(const W4Args& a);

}  // namespace b200mm

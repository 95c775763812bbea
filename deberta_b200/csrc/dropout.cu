// Dropout from a counter-based generator: out[r, c] = (residual[r, c] +) kept(r, c) ? x[r, c] / (1 - p) : 0.
// The mask is a function of (seed, r, c) (philox.cuh), so the backward pass is the same kernel on the output's gradient
// and nothing is kept in between. One vector of eight columns is one evaluation of the generator and one 16-byte access
// per operand (two for fp32); the sum with the residual is formed in fp32 and rounded once.
#include "kernels.h"
#include "philox.cuh"
#include "rows.cuh"
#include "tc05.cuh"

#include <cuda_runtime.h>

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // vectors in flight per thread

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ residual, long long ldr,
               T* __restrict__ out, long long rows, int cols, philox::Seed seed, uint32_t threshold, float scale) {
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const uint2 key = philox::load_key(seed);
  const unsigned groups = (cols + 7) >> 3;
  const long long total = rows * groups;
  const long long base = static_cast<long long>(blockIdx.x) * (kThreads * kUnroll) + threadIdx.x;
  rows::Raw<T> xr[kUnroll], rr[kUnroll];
  long long row[kUnroll];
  int group[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long long i = base + u * kThreads;
    if (i < total) {
      if (total <= 0xffffffffll) {  // (uniform) 32-bit division
        const unsigned q = static_cast<unsigned>(i) / groups;
        row[u] = q;
        group[u] = static_cast<unsigned>(i) - q * groups;
      } else {
        row[u] = i / groups;
        group[u] = static_cast<int>(i - row[u] * groups);
      }
      rows::load<VEC>(xr[u], x + row[u] * ldx, group[u] * 8, cols);
      if (residual) rows::load<VEC>(rr[u], residual + row[u] * ldr, group[u] * 8, cols);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (base + u * kThreads < total) {
      float f[8];
      rows::unpack(xr[u], f);
      philox::apply8(f, group[u], row[u], key, threshold, scale);
      if (residual) {
        float r[8];
        rows::unpack(rr[u], r);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] += r[j];
      }
      rows::store<VEC>(f, out + row[u] * cols, group[u] * 8, cols);
    }
  }
}

template <typename T>
int launch(const void* x, long long ldx, const void* residual, long long ldr, void* out, long long rows, int cols,
           philox::Seed seed, uint32_t threshold, float scale, cudaStream_t st) {
  const long long vecs = rows * ((cols + 7) / 8);
  const long long blocks = (vecs + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  if (blocks > 0x7fffffffLL) return -12;
  const bool vec = rows::vector_rows(x, ldx, cols) && rows::vector_rows(residual, ldr, cols) &&
                   rows::vector_rows(out, cols, cols);
  auto X = static_cast<const T*>(x);
  auto R = static_cast<const T*>(residual);
  auto O = static_cast<T*>(out);
  const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
  const cudaError_t rc =
      vec ? tc05::launch_pdl(dropout_kernel<T, true>, grid, block, 0, st, X, ldx, R, ldr, O, rows, cols, seed, threshold, scale)
          : tc05::launch_pdl(dropout_kernel<T, false>, grid, block, 0, st, X, ldx, R, ldr, O, rows, cols, seed, threshold, scale);
  return rc == cudaSuccess ? 0 : -4;
}

}  // namespace

extern "C" int db200_dropout(const void* x, long long ldx, const void* residual, long long ldr, void* out,
                             long long rows, int cols, int dtype, const void* seed_ptr, unsigned long long seed,
                             unsigned threshold, float scale, void* stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if (!x || !out || threshold > 65535u || ldx < cols || (residual && ldr < cols)) return -10;
  const philox::Seed s{static_cast<const unsigned long long*>(seed_ptr), seed};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case 0: return launch<__nv_bfloat16>(x, ldx, residual, ldr, out, rows, cols, s, threshold, scale, st);
    case 1: return launch<__half>(x, ldx, residual, ldr, out, rows, cols, s, threshold, scale, st);
    case 2: return launch<float>(x, ldx, residual, ldr, out, rows, cols, s, threshold, scale, st);
  }
  return -11;
}

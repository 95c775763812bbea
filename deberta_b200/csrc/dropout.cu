// Dropout from a counter-based generator: out[r, c] = (residual[r, c] +) kept(r, c) ? x[r, c] / (1 - p) : 0.
// The mask is a function of (seed, r, c) (philox.cuh), so the backward pass is the same kernel on the output's gradient
// and nothing is kept in between. One vector of eight columns is one evaluation of the generator and one 16-byte access
// per operand (two for fp32); the sum with the residual is formed in fp32 and rounded once. 16384 x 768 bf16, both directions:
// 23.1 us for 101 MB (4.4 TB/s; the ALU pipe, which the generator and the selects run on, is 58 % busy).
#include "kernels.h"
#include "philox.cuh"
#include "rows.cuh"
#include "tc05.cuh"

#include <cuda_runtime.h>

namespace {

constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 4;  // 16384 x 768 bf16, both directions: 23.1 us (a copy of as many bytes: 17.9), one vector per thread: 25.6

// i / d for 0 <= i < 2^31 by a multiplication: m = ceil(2^(31 + b) / d) with 2^(b-1) < d <= 2^b, which is exact in that range
struct Divider {
  unsigned d, m, shift;
};
Divider make_divider(unsigned d) {
  unsigned b = 0;
  while ((1ull << b) < d) ++b;
  return {d, static_cast<unsigned>(((1ull << (31 + b)) + d - 1) / d), b};
}

// WIDE: more than 2^31 vectors (64-bit division). A thread takes every gridDim-th vector; the next one's operands are
// asked for before the current one's bits are drawn.
template <typename T, bool VEC, bool WIDE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
dropout_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ residual, long long ldr,
               T* __restrict__ out, long long total, Divider groups, int cols, philox::Seed seed, uint32_t threshold,
               float scale) {
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= total) return;
  const uint2 key = philox::load_key(seed);
  rows::Raw<T> xr, rr;
  long long row;
  unsigned group;
  auto fetch = [&](long long at, rows::Raw<T>& xo, rows::Raw<T>& ro, long long& r, unsigned& g) {
    if constexpr (WIDE) {
      r = at / groups.d;
      g = static_cast<unsigned>(at - r * groups.d);
    } else {
      const unsigned q = static_cast<unsigned>((static_cast<unsigned long long>(static_cast<unsigned>(at)) * groups.m) >> 31) >>
                         groups.shift;
      r = q;
      g = static_cast<unsigned>(at) - q * groups.d;
    }
    rows::load<VEC>(xo, x + r * ldx, static_cast<int>(g * 8), cols);
    if (residual) rows::load<VEC>(ro, residual + r * ldr, static_cast<int>(g * 8), cols);
  };
  fetch(i, xr, rr, row, group);
  for (; i < total; i += step) {
    const long long next = i + step;
    rows::Raw<T> xn, rn;
    long long row_n = 0;
    unsigned group_n = 0;
    if (next < total) fetch(next, xn, rn, row_n, group_n);
    float f[8];
    const uint4 bits = philox::words(group, row, key);
    rows::unpack(xr, f);
    const uint32_t high = threshold << 16;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = philox::keeps(bits, j, high) ? f[j] * scale : 0.f;
    if (residual) {
      float r[8];
      rows::unpack(rr, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += r[j];
    }
    rows::store<VEC>(f, out + row * cols, static_cast<int>(group * 8), cols);
    xr = xn;
    rr = rn;
    row = row_n;
    group = group_n;
  }
}

template <typename T>
int launch(const void* x, long long ldx, const void* residual, long long ldr, void* out, long long rows, int cols,
           philox::Seed seed, uint32_t threshold, float scale, cudaStream_t st) {
  const Divider groups = make_divider((cols + 7) / 8);
  const long long total = rows * groups.d;
  const long long blocks = (total + kThreads - 1) / kThreads;
  const bool vec = rows::vector_rows(x, ldx, cols) && rows::vector_rows(residual, ldr, cols) &&
                   rows::vector_rows(out, cols, cols);
  using Kernel = void (*)(const T*, long long, const T*, long long, T*, long long, Divider, int, philox::Seed, uint32_t, float);
  const bool wide = total + 148ll * kBlocksPerSm * kThreads > 0x7fffffffll;
  const Kernel kern = vec ? (wide ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                          : (wide ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
  const dim3 grid(static_cast<unsigned>(blocks < 148 * kBlocksPerSm ? blocks : 148 * kBlocksPerSm));
  return tc05::launch_pdl(kern, grid, dim3(kThreads), 0, st, static_cast<const T*>(x), ldx,
                          static_cast<const T*>(residual), ldr, static_cast<T*>(out), total, groups, cols, seed, threshold,
                          scale) == cudaSuccess ? 0 : -4;
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

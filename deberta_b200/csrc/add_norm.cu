// LayerNorm / RMSNorm of a residual sum with dropout on the branch:
//   t = residual + dropout(x),   y = norm(t) * gamma (+ beta)
// forward in one pass over x and residual (t and y leave it), backward in one pass over dy, t and the gradient that
// reaches t directly:
//   dt = rstd * (dy*gamma - mean(dy*gamma) - xhat * mean(dy*gamma*xhat)) + dtotal      (RMS: without the first mean)
//   dresidual = dt,   dx = dropout'(dt)   (the mask is drawn again, philox.cuh)
// Both are bound by memory: each operand crosses the bus once. Up to 1024 columns a warp owns a row (no block barrier) and
// walks its rows over a ring of shared-memory stages that bulk copies fill two to four rows ahead, so that the row's
// reductions do not stop the loads; rows that bulk copies cannot reach (odd widths, unaligned views) are loaded straight
// into registers, and above 1024 columns a block of 256 threads owns a row. Statistics are fp32 and are
// taken of the unrounded sum; the backward pass reads the rounded one. The parameter gradients are summed in registers
// over a block's rows, written as one fp32 row per block and added up by a second kernel in a fixed order, so that they
// are the same bits in every run. Measured, both directions: RMSNorm 16384 x 1024 bf16 without dropout 48.5 us (268 MB:
// 5.5 TB/s), LayerNorm 16384 x 768 with dropout 54.3 us (226 MB: 4.2 TB/s; the generator's integer work shows).
#include "kernels.h"
#include "philox.cuh"
#include "rows.cuh"
#include "tc05.cuh"

#include <cuda_runtime.h>

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// sum over the TPR threads of a row
template <int TPR>
__device__ __forceinline__ float row_total(float v, float* red) {
  v = warp_total(v);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) v += red[w];
    __syncthreads();
  }
  return v;
}

struct FwdArgs {
  const void *x, *residual, *gamma, *beta;
  long long ldx, ldr;
  void *total, *y;
  float *mean, *rstd;  // mean: null for RMSNorm
  long long rows;
  int cols;
  float eps;
  philox::Seed seed;
  uint32_t threshold;  // 0: no dropout
  float scale;
};

// V = vectors of eight columns per thread: covers cols <= 8 * TPR * V
template <typename T, int TPR, int V, bool VEC>
__global__ void __launch_bounds__(kThreads)
add_norm_fwd_kernel(const FwdArgs p) {
  __shared__ float red[kThreads / 32];
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  constexpr int kRows = kThreads / TPR;
  const int t = threadIdx.x % TPR;
  const bool rms = p.mean == nullptr;
  const int cols = p.cols;
  uint2 key = make_uint2(0, 0);
  if (p.threshold) key = philox::load_key(p.seed);
  for (long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / TPR; row < p.rows;
       row += static_cast<long long>(gridDim.x) * kRows) {
    const T* xr = static_cast<const T*>(p.x) + row * p.ldx;
    const T* rr = static_cast<const T*>(p.residual) + row * p.ldr;
    rows::Raw<T> xv[V], rv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
        rows::load<VEC>(xv[i], xr, c, cols);
        rows::load<VEC>(rv[i], rr, c, cols);
      }
    }
    float v[V][8];
    float s = 0.f;
    T* tr = static_cast<T*>(p.total) + row * cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
        float r[8];
        rows::unpack(xv[i], v[i]);
        rows::unpack(rv[i], r);
        if (p.threshold) philox::apply8(v[i], c >> 3, row, key, p.threshold, p.scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] += r[j];  // (columns past the end: zeros)
          s += v[i][j];
        }
        rows::store<VEC>(v[i], tr, c, cols);
      }
    }
    const float mean = rms ? 0.f : row_total<TPR>(s, red) / cols;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = v[i][j] - mean;
          ss += (VEC || c + j < cols) ? d * d : 0.f;
        }
      }
    }
    const float rstd = rsqrtf(row_total<TPR>(ss, red) / cols + p.eps);
    T* yr = static_cast<T*>(p.y) + row * cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
        rows::Raw<T> w;
        float g[8], b[8] = {};
        rows::load<VEC>(w, static_cast<const T*>(p.gamma), c, cols);
        rows::unpack(w, g);
        if (p.beta) {
          rows::load<VEC>(w, static_cast<const T*>(p.beta), c, cols);
          rows::unpack(w, b);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf((v[i][j] - mean) * rstd, g[j], b[j]);
        rows::store<VEC>(v[i], yr, c, cols);
      }
    }
    if (t == 0) {
      if (!rms) p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

// ---- rows ahead of a warp: a ring of `stages` slots, each one row of NT operands, filled by bulk copies --------------------
constexpr int kMaxStages = 4;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   tc05::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc05::smem_u32(bar))
               : "memory");
}

template <int NT>
struct Ring {
  uint8_t* slots;     // this warp's
  uint64_t* bars;     // this warp's, one per slot
  volatile int* abort_flag;
  int* status;
  int stages;
  uint32_t row_bytes;  // a multiple of 16
  int slot = 0;
  uint32_t parity = 0;

  __device__ __forceinline__ uint8_t* at(int s, int operand) const {
    return slots + (static_cast<uint32_t>(s) * NT + operand) * row_bytes;
  }
  // one lane: asks for a row's operands (null: none)
  __device__ __forceinline__ void ask(int s, const void* const (&src)[NT]) {
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < NT; ++k) n += src[k] != nullptr ? 1 : 0;
    tc05::mbar_expect_tx(&bars[s], n * row_bytes);
#pragma unroll
    for (int k = 0; k < NT; ++k)
      if (src[k] != nullptr) bulk_copy(at(s, k), src[k], row_bytes, &bars[s]);
  }
  __device__ __forceinline__ bool wait() {  // whole warp: the current slot has arrived
    return __all_sync(0xffffffffu, tc05::mbar_wait(&bars[slot], parity, abort_flag, status, tc05::kErrFullWait)) != 0;
  }
  __device__ __forceinline__ void advance() {
    if (++slot == stages) {
      slot = 0;
      parity ^= 1;
    }
  }
  // after a wait that ran out: `left` slots are still in flight and must land before the block leaves
  __device__ __forceinline__ void drain(int left) {
    for (; left > 0; --left) {
      for (uint32_t i = 0; i < tc05::kSpinLimit; ++i)
        if (tc05::mbar_try_wait(&bars[slot], parity)) break;
      advance();
    }
  }
};

// Every warp initialises its own barriers; returns its ring.
template <int NT>
__device__ __forceinline__ Ring<NT> make_ring(uint8_t* smem, uint64_t (*bars)[kMaxStages], int* abort_flag, int* status,
                                              int stages, uint32_t row_bytes) {
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    for (int s = 0; s < stages; ++s) tc05::mbar_init(&bars[warp][s], 1);
    tc05::fence_barrier_init();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  __syncthreads();
  return Ring<NT>{smem + static_cast<uint32_t>(warp) * stages * NT * row_bytes, bars[warp], abort_flag, status, stages,
                  row_bytes};
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1)
add_norm_fwd_ring_kernel(const FwdArgs p, int stages, int* status) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ uint64_t bars[kWarps][kMaxStages];
  __shared__ int abort_flag;
  tc05::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int cols = p.cols;
  const bool rms = p.mean == nullptr;
  Ring<2> ring = make_ring<2>(ring_smem, bars, &abort_flag, status, stages, cols * sizeof(T));
  tc05::pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  long long row = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  auto ask = [&](int s, long long r) {
    const void* const src[2] = {static_cast<const T*>(p.x) + r * p.ldx, static_cast<const T*>(p.residual) + r * p.ldr};
    ring.ask(s, src);
  };
  if (lane == 0)
    for (int s = 0; s < stages && row + s * step < p.rows; ++s) ask(s, row + s * step);
  uint2 key = make_uint2(0, 0);
  if (p.threshold) key = philox::load_key(p.seed);
  rows::Raw<T> gv[V], bv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (lane + i * 32) * 8;
    if (c < cols) {
      gv[i] = *reinterpret_cast<const rows::Raw<T>*>(static_cast<const T*>(p.gamma) + c);
      if (p.beta) bv[i] = *reinterpret_cast<const rows::Raw<T>*>(static_cast<const T*>(p.beta) + c);
    }
  }
  const uint32_t high = p.threshold << 16;
  for (; row < p.rows; row += step) {
    if (!ring.wait()) {
      int left = 0;
      while (left < stages && row + left * step < p.rows) ++left;
      ring.drain(left);
      return;
    }
    const T* xs = reinterpret_cast<const T*>(ring.at(ring.slot, 0));
    const T* rs = reinterpret_cast<const T*>(ring.at(ring.slot, 1));
    float v[V][8];
    float s = 0.f;
    T* tr = static_cast<T*>(p.total) + row * cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (lane + i * 32) * 8;
      if (c < cols) {
        float r[8];
        rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(xs + c), v[i]);
        rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(rs + c), r);
        if (p.threshold) {
          const uint4 w = philox::words(c >> 3, row, key);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = philox::keeps(w, j, high) ? v[i][j] * p.scale : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] += r[j];
          s += v[i][j];
        }
      }
    }
    __syncwarp();  // the slot has been read
    if (lane == 0 && row + stages * step < p.rows) ask(ring.slot, row + stages * step);
    ring.advance();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (lane + i * 32) * 8;
      if (c < cols) rows::store<true>(v[i], tr, c, cols);
    }
    const float mean = rms ? 0.f : warp_total(s) / cols;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if ((lane + i * 32) * 8 < cols) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = v[i][j] - mean;
          ss += d * d;
        }
      }
    }
    const float rstd = rsqrtf(warp_total(ss) / cols + p.eps);
    T* yr = static_cast<T*>(p.y) + row * cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (lane + i * 32) * 8;
      if (c < cols) {
        float g[8], b[8] = {};
        rows::unpack(gv[i], g);
        if (p.beta) rows::unpack(bv[i], b);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf((v[i][j] - mean) * rstd, g[j], b[j]);
        rows::store<true>(v[i], yr, c, cols);
      }
    }
    if (lane == 0) {
      if (!rms) p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

struct BwdArgs {
  const void *dy, *total, *dtotal, *gamma;  // dtotal: null where nothing reaches the sum directly
  const float *mean, *rstd;
  void *dx, *dresidual;  // dresidual: null where it equals dx (no dropout)
  float *dgamma_part, *dbeta_part;  // [blocks, cols]; dbeta_part may be null
  long long rows;
  int cols;
  philox::Seed seed;
  uint32_t threshold;
  float scale;
};

// The block's warps share the columns: their sums, one row of partial sums per block.
template <int V>
__device__ __forceinline__ void write_parts(const BwdArgs& p, float (&dg)[V][8], float (&db)[V][8], float (*cross)[257]) {
  const int warp = threadIdx.x >> 5, t = threadIdx.x & 31;
  const long long out = static_cast<long long>(blockIdx.x) * p.cols;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    for (int pass = 0; pass < 2; ++pass) {
      float* part = pass == 0 ? p.dgamma_part : p.dbeta_part;
      if (part == nullptr) continue;  // uniform
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) cross[warp][t * 8 + j] = pass == 0 ? dg[i][j] : db[i][j];
      __syncthreads();
      const int col = i * 256 + threadIdx.x;
      float acc = 0.f;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) acc += cross[w][threadIdx.x];
      if (col < p.cols) part[out + col] = acc;
    }
  }
}

template <typename T, int V, bool RMS>
__global__ void __launch_bounds__(kThreads, (sizeof(T) == 2 && (V <= 3 || RMS)) ? 2 : 1)
add_norm_bwd_ring_kernel(const BwdArgs p, int stages, int* status) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ uint64_t bars[kWarps][kMaxStages];
  __shared__ int abort_flag;
  __shared__ float cross[kWarps][257];
  tc05::pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int cols = p.cols;
  const float inv_cols = 1.f / cols;
  Ring<3> ring = make_ring<3>(ring_smem, bars, &abort_flag, status, stages, cols * sizeof(T));
  tc05::pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  long long row = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  auto ask = [&](int s, long long r) {
    const long long at = r * cols;
    const void* const src[3] = {static_cast<const T*>(p.dy) + at, static_cast<const T*>(p.total) + at,
                                p.dtotal ? static_cast<const T*>(p.dtotal) + at : nullptr};
    ring.ask(s, src);
  };
  if (lane == 0)
    for (int s = 0; s < stages && row + s * step < p.rows; ++s) ask(s, row + s * step);
  uint2 key = make_uint2(0, 0);
  if (p.threshold) key = philox::load_key(p.seed);
  const uint32_t high = p.threshold << 16;
  rows::Raw<T> gv[V];  // gamma stays packed
  float dg[V][8], db[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (lane + i * 32) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[i][j] = db[i][j] = 0.f;
    if (c < cols) gv[i] = *reinterpret_cast<const rows::Raw<T>*>(static_cast<const T*>(p.gamma) + c);
  }
  float mean = 0.f, rstd = 0.f;  // (a row ahead, too: their loads would wait otherwise)
  if (row < p.rows) {
    mean = RMS ? 0.f : p.mean[row];
    rstd = p.rstd[row];
  }
  bool ok = true;
  for (; row < p.rows; row += step) {
    float mean_n = 0.f, rstd_n = 0.f;
    if (row + step < p.rows) {
      mean_n = RMS ? 0.f : p.mean[row + step];
      rstd_n = p.rstd[row + step];
    }
    ok = ring.wait();
    if (!ok) break;
    const T* ys = reinterpret_cast<const T*>(ring.at(ring.slot, 0));
    const T* ts = reinterpret_cast<const T*>(ring.at(ring.slot, 1));
    const T* es = reinterpret_cast<const T*>(ring.at(ring.slot, 2));
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (lane + i * 32) * 8;
      if (c < cols) {
        float d[8], x[8], g[8];
        rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(ys + c), d);
        rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(ts + c), x);
        rows::unpack(gv[i], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = (x[j] - mean) * rstd;
          const float dxh = d[j] * g[j];
          s1 += dxh;
          s2 += dxh * xh;
          dg[i][j] += d[j] * xh;
          if (!RMS) db[i][j] += d[j];
        }
      }
    }
    s1 = RMS ? 0.f : warp_total(s1) * inv_cols;
    s2 = warp_total(s2) * inv_cols;
    const long long at = row * cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (lane + i * 32) * 8;
      if (c < cols) {
        float d[8], x[8], g[8], e[8] = {};
        rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(ys + c), d);
        rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(ts + c), x);
        rows::unpack(gv[i], g);
        if (p.dtotal) rows::unpack(*reinterpret_cast<const rows::Raw<T>*>(es + c), e);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] += rstd * (d[j] * g[j] - s1 - (x[j] - mean) * rstd * s2);
        if (p.dresidual) rows::store<true>(e, static_cast<T*>(p.dresidual) + at, c, cols);
        if (p.threshold) {
          const uint4 w = philox::words(c >> 3, row, key);
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = philox::keeps(w, j, high) ? e[j] * p.scale : 0.f;
        }
        rows::store<true>(e, static_cast<T*>(p.dx) + at, c, cols);
      }
    }
    __syncwarp();  // the slot has been read
    if (lane == 0 && row + stages * step < p.rows) ask(ring.slot, row + stages * step);
    ring.advance();
    mean = mean_n;
    rstd = rstd_n;
  }
  if (!ok) {
    int left = 0;
    while (left < stages && row + left * step < p.rows) ++left;
    ring.drain(left);
  }
  write_parts<V>(p, dg, db, cross);
}

template <typename T, int TPR, int V, bool VEC, bool RMS>
__global__ void __launch_bounds__(kThreads)
add_norm_bwd_kernel(const BwdArgs p) {
  __shared__ float red[kThreads / 32];
  __shared__ float cross[TPR == 32 ? kThreads / 32 : 1][257];
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  constexpr int kRows = kThreads / TPR;
  const int t = threadIdx.x % TPR;
  const int cols = p.cols;
  const float inv_cols = 1.f / cols;
  uint2 key = make_uint2(0, 0);
  if (p.threshold) key = philox::load_key(p.seed);
  rows::Raw<T> gv[V];  // gamma stays packed
  float dg[V][8], db[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (t + i * TPR) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) dg[i][j] = db[i][j] = 0.f;
    if (c < cols) rows::load<VEC>(gv[i], static_cast<const T*>(p.gamma), c, cols);
  }
  for (long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / TPR; row < p.rows;
       row += static_cast<long long>(gridDim.x) * kRows) {
    const long long at = row * cols;
    rows::Raw<T> yv[V], tv[V], ev[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
        rows::load<VEC>(yv[i], static_cast<const T*>(p.dy) + at, c, cols);
        rows::load<VEC>(tv[i], static_cast<const T*>(p.total) + at, c, cols);
        if (p.dtotal) rows::load<VEC>(ev[i], static_cast<const T*>(p.dtotal) + at, c, cols);
      }
    }
    const float mean = RMS ? 0.f : p.mean[row], rstd = p.rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
        float d[8], x[8], g[8];
        rows::unpack(yv[i], d);  // (zeros past the end)
        rows::unpack(tv[i], x);
        rows::unpack(gv[i], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = (x[j] - mean) * rstd;
          const float dxh = d[j] * g[j];
          s1 += dxh;
          s2 += dxh * xh;
          dg[i][j] += d[j] * xh;
          if (!RMS) db[i][j] += d[j];
        }
      }
    }
    s1 = RMS ? 0.f : row_total<TPR>(s1, red) * inv_cols;
    s2 = row_total<TPR>(s2, red) * inv_cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
      if (c < cols) {
        float d[8], x[8], g[8], e[8] = {};
        rows::unpack(yv[i], d);
        rows::unpack(tv[i], x);
        rows::unpack(gv[i], g);
        if (p.dtotal) rows::unpack(ev[i], e);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] += rstd * (d[j] * g[j] - s1 - (x[j] - mean) * rstd * s2);
        if (p.dresidual) rows::store<VEC>(e, static_cast<T*>(p.dresidual) + at, c, cols);
        if (p.threshold) philox::apply8(e, c >> 3, row, key, p.threshold, p.scale);
        rows::store<VEC>(e, static_cast<T*>(p.dx) + at, c, cols);
      }
    }
  }
  if constexpr (TPR == 32) {
    write_parts<V>(p, dg, db, cross);
  } else {
    const long long out = static_cast<long long>(blockIdx.x) * cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (t + i * TPR) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c + j < cols) {
          p.dgamma_part[out + c + j] = dg[i][j];
          if (p.dbeta_part) p.dbeta_part[out + c + j] = db[i][j];
        }
      }
    }
  }
}

// Column sums of `parts` rows, in an order that depends on `parts` alone. blockIdx.y: 0 = gamma, 1 = beta.
struct SumArgs {
  const float* part[2];
  void* out[2];       // in the parameter's type, or null
  float* acc[2];      // fp32 buffer that the sum is added to, or null
  int parts, cols;
};

constexpr int kSumRows = 32;   // row groups of a block
constexpr int kSumAhead = 10;  // loads in flight per thread: all of 296 rows at once

template <typename T>
__global__ void __launch_bounds__(32 * kSumRows)
param_grad_kernel(const SumArgs p) {
  __shared__ float red[kSumRows][33];
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const float* part = blockIdx.y == 0 ? p.part[0] : p.part[1];
  float* buffer = blockIdx.y == 0 ? p.acc[0] : p.acc[1];
  T* out = static_cast<T*>(blockIdx.y == 0 ? p.out[0] : p.out[1]);
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + x;
  float s = 0.f;
  if (col < p.cols) {
    for (int r0 = y; r0 < p.parts; r0 += kSumRows * kSumAhead) {
      float v[kSumAhead];
#pragma unroll
      for (int u = 0; u < kSumAhead; ++u) {
        const int r = r0 + u * kSumRows;
        v[u] = r < p.parts ? part[static_cast<long long>(r) * p.cols + col] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kSumAhead; ++u) s += v[u];
    }
  }
  red[y][x] = s;
  __syncthreads();
  if (y == 0 && col < p.cols) {
#pragma unroll
    for (int r = 1; r < kSumRows; ++r) s += red[r][x];
    if (buffer) buffer[col] += s;
    else out[col] = rows::from_f<T>(s);
  }
}

// Stages of a ring of `operands` rows per warp: as many as fit beside a second block on the SM (two at least, then alone).
int ring_stages(int operands, long long row_bytes) {
  const long long slot = kWarps * operands * row_bytes;
  const long long n = (100 * 1024) / slot;
  return n >= kMaxStages ? kMaxStages : (n >= 2 ? static_cast<int>(n) : 2);
}

// The opt-in to large shared memory, once per kernel and device.
template <typename Kernel>
bool allow_smem(Kernel kern, bool (&done)[16]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) return false;
  if (!done[dev]) done[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024) == cudaSuccess;
  return done[dev];
}

template <typename T, int V>
cudaError_t run_fwd_ring(const FwdArgs& a, cudaStream_t st) {
  static bool done[16] = {};
  if (!allow_smem(add_norm_fwd_ring_kernel<T, V>, done)) return cudaErrorInvalidValue;
  const long long row_bytes = static_cast<long long>(a.cols) * sizeof(T);
  const int stages = ring_stages(2, row_bytes);
  const long long want = (a.rows + kWarps - 1) / kWarps;
  const dim3 grid(static_cast<unsigned>(want < 148 * 2 ? want : 148 * 2));
  return tc05::launch_pdl(add_norm_fwd_ring_kernel<T, V>, grid, dim3(kThreads), kWarps * 2 * row_bytes * stages, st, a, stages,
                          db200_status_ptr());
}

template <typename T, int V, bool RMS>
cudaError_t run_bwd_ring(const BwdArgs& a, unsigned blocks, cudaStream_t st) {
  static bool done[16] = {};
  if (!allow_smem(add_norm_bwd_ring_kernel<T, V, RMS>, done)) return cudaErrorInvalidValue;
  const long long row_bytes = static_cast<long long>(a.cols) * sizeof(T);
  const int stages = ring_stages(3, row_bytes);
  return tc05::launch_pdl(add_norm_bwd_ring_kernel<T, V, RMS>, dim3(blocks), dim3(kThreads), kWarps * 3 * row_bytes * stages, st,
                          a, stages, db200_status_ptr());
}
template <typename T, int V>
cudaError_t run_bwd_ring(const BwdArgs& a, unsigned blocks, cudaStream_t st) {
  return a.mean ? run_bwd_ring<T, V, false>(a, blocks, st) : run_bwd_ring<T, V, true>(a, blocks, st);
}

template <typename T, int TPR, int V, bool VEC>
cudaError_t run_fwd(const FwdArgs& a, cudaStream_t st) {
  constexpr int kRows = kThreads / TPR;
  const long long want = (a.rows + kRows - 1) / kRows;
  const unsigned blocks = static_cast<unsigned>(want < 148 * 16 ? want : 148 * 16);
  return tc05::launch_pdl(add_norm_fwd_kernel<T, TPR, V, VEC>, dim3(blocks), dim3(kThreads), 0, st, a);
}

template <typename T>
cudaError_t pick_fwd(const FwdArgs& a, bool vec, cudaStream_t st) {
  if (!vec) {
    if (a.cols <= 1024) return run_fwd<T, 32, 4, false>(a, st);
    return run_fwd<T, 256, 4, false>(a, st);
  }
  if (a.cols <= 256) return run_fwd_ring<T, 1>(a, st);
  if (a.cols <= 512) return run_fwd_ring<T, 2>(a, st);
  if (a.cols <= 768) return run_fwd_ring<T, 3>(a, st);
  if (a.cols <= 1024) return run_fwd_ring<T, 4>(a, st);
  if (a.cols <= 2048) return run_fwd<T, 256, 1, true>(a, st);
  if (a.cols <= 4096) return run_fwd<T, 256, 2, true>(a, st);
  return run_fwd<T, 256, 4, true>(a, st);
}

template <typename T, int TPR, int V, bool VEC>
cudaError_t run_bwd(const BwdArgs& a, unsigned blocks, cudaStream_t st) {
  return a.mean ? tc05::launch_pdl(add_norm_bwd_kernel<T, TPR, V, VEC, false>, dim3(blocks), dim3(kThreads), 0, st, a)
                : tc05::launch_pdl(add_norm_bwd_kernel<T, TPR, V, VEC, true>, dim3(blocks), dim3(kThreads), 0, st, a);
}

template <typename T>
cudaError_t pick_bwd(const BwdArgs& a, unsigned blocks, bool vec, cudaStream_t st) {
  if (!vec) {
    if (a.cols <= 1024) return run_bwd<T, 32, 4, false>(a, blocks, st);
    return run_bwd<T, 256, 4, false>(a, blocks, st);
  }
  if (a.cols <= 256) return run_bwd_ring<T, 1>(a, blocks, st);
  if (a.cols <= 512) return run_bwd_ring<T, 2>(a, blocks, st);
  if (a.cols <= 768) return run_bwd_ring<T, 3>(a, blocks, st);
  if (a.cols <= 1024) return run_bwd_ring<T, 4>(a, blocks, st);
  if (a.cols <= 2048) return run_bwd<T, 256, 1, true>(a, blocks, st);
  if (a.cols <= 4096) return run_bwd<T, 256, 2, true>(a, blocks, st);
  return run_bwd<T, 256, 4, true>(a, blocks, st);
}

constexpr int kMaxCols = 8192;

}  // namespace

extern "C" int db200_add_norm_fwd(const void* x, long long ldx, const void* residual, long long ldr, const void* gamma,
                                  const void* beta, void* total, void* y, float* mean, float* rstd, long long rows,
                                  int cols, float eps, int dtype, const void* seed_ptr, unsigned long long seed,
                                  unsigned threshold, float scale, void* stream) {
  if (rows <= 0) return 0;
  if (!x || !residual || !gamma || !total || !y || !rstd || cols <= 0 || ldx < cols || ldr < cols || threshold > 65535u)
    return -10;
  if (cols > kMaxCols) return -12;
  const FwdArgs a{x, residual, gamma, beta, ldx, ldr, total, y, mean, rstd, rows, cols, eps,
                  {static_cast<const unsigned long long*>(seed_ptr), seed}, threshold, scale};
  const bool vec = rows::vector_rows(x, ldx, cols) && rows::vector_rows(residual, ldr, cols) &&
                   rows::vector_rows(gamma, cols, cols) && rows::vector_rows(beta, cols, cols) &&
                   rows::vector_rows(total, cols, cols) && rows::vector_rows(y, cols, cols);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t rc = cudaErrorInvalidValue;
  if (dtype == 0) rc = pick_fwd<__nv_bfloat16>(a, vec, st);
  else if (dtype == 1) rc = pick_fwd<__half>(a, vec, st);
  else if (dtype == 2) rc = pick_fwd<float>(a, vec, st);
  else return -11;
  return rc == cudaSuccess ? 0 : -4;
}

// Rows of the partial sums that db200_add_norm_bwd writes: two resident blocks per SM.
extern "C" int db200_add_norm_parts(long long rows, int cols) {
  const int per_block = cols <= 1024 ? kThreads / 32 : 1;
  const long long want = (rows + per_block - 1) / per_block;
  return static_cast<int>(want < 148 * 2 ? (want > 0 ? want : 1) : 148 * 2);
}

extern "C" int db200_add_norm_bwd(const void* dy, const void* total, const void* dtotal, const void* gamma,
                                  const float* mean, const float* rstd, void* dx, void* dresidual, float* parts,
                                  void* dgamma, float* dgamma_acc, void* dbeta, float* dbeta_acc, int has_beta,
                                  long long rows, int cols, int dtype, const void* seed_ptr, unsigned long long seed,
                                  unsigned threshold, float scale, void* stream) {
  if (rows <= 0) return 0;
  if (!dy || !total || !gamma || !rstd || !dx || !parts || cols <= 0 || threshold > 65535u || (!dgamma && !dgamma_acc) ||
      (has_beta && !dbeta && !dbeta_acc) || (has_beta && !mean) || (threshold && !dresidual))
    return -10;
  if (cols > kMaxCols) return -12;
  const int blocks = db200_add_norm_parts(rows, cols);
  float* beta_parts = has_beta ? parts + static_cast<long long>(blocks) * cols : nullptr;
  const BwdArgs a{dy, total, dtotal, gamma, mean, rstd, dx, dresidual, parts, beta_parts, rows, cols,
                  {static_cast<const unsigned long long*>(seed_ptr), seed}, threshold, scale};
  const bool vec = rows::vector_rows(dy, cols, cols) && rows::vector_rows(total, cols, cols) &&
                   rows::vector_rows(dtotal, cols, cols) && rows::vector_rows(gamma, cols, cols) &&
                   rows::vector_rows(dx, cols, cols) && rows::vector_rows(dresidual, cols, cols);
  const SumArgs s{{parts, beta_parts}, {dgamma, dbeta}, {dgamma_acc, dbeta_acc}, blocks, cols};
  const dim3 grid((cols + 31) / 32, has_beta ? 2 : 1);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t rc = cudaErrorInvalidValue;
  if (dtype == 0) {
    rc = pick_bwd<__nv_bfloat16>(a, blocks, vec, st);
    if (rc == cudaSuccess) rc = tc05::launch_pdl(param_grad_kernel<__nv_bfloat16>, grid, dim3(32 * kSumRows), 0, st, s);
  } else if (dtype == 1) {
    rc = pick_bwd<__half>(a, blocks, vec, st);
    if (rc == cudaSuccess) rc = tc05::launch_pdl(param_grad_kernel<__half>, grid, dim3(32 * kSumRows), 0, st, s);
  } else if (dtype == 2) {
    rc = pick_bwd<float>(a, blocks, vec, st);
    if (rc == cudaSuccess) rc = tc05::launch_pdl(param_grad_kernel<float>, grid, dim3(32 * kSumRows), 0, st, s);
  } else {
    return -11;
  }
  return rc == cudaSuccess ? 0 : -4;
}

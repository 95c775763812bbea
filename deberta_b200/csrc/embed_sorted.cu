// Scaled embedding lookup and its gradient by sorted tokens.
//   out[t, :] = scale * table[id[t], :]
//   dtable[v, :] = scale * sum over the tokens t with id[t] = v of dout[t, :]
// The gradient has no atomics: the (id, position) pairs are sorted by id, positions ascending, and every sum is taken in
// an order that depends on the ids alone, so the same call gives the same bits. Three launches:
//   1. sort + fill: the first cluster of eight CTAs sorts (stable, least significant digit first; counters of a warp in
//      its own shared memory, the digit totals of the CTAs read over distributed shared memory), all other clusters
//      clear the dense gradient meanwhile, so the sort hides behind the writes that the call cannot do without.
//   2. sums: a warp adds 16 neighbours of the sorted order (256 columns, all 16 rows in flight). Rows whose tokens lie
//      inside the 16 are written at once; pieces that cross a border go to fp32 partial rows, two at most per tile.
//   3. combine: the block at the tile where a crossing row begins adds its partial rows in order and writes it.
// Up to 256 tokens one launch does it all: a block owns every 592nd table row, lists the tokens of its rows in the order of
// their positions, clears the rows that none names and sums the others (57 tokens of 4096 x 384 fp32 with the lookup: 16.4 us for the three launches, 9.8 us so; 256 of 128100 x 768: 38 us).
// 16384 tokens of 128100 x 768 bf16, lookup and gradient: 70.8 us, of which 42 write the gradient's zeros.
// A token of 15 % of the batch (the mask token) is therefore spread over many warps, not one. Ids out of range and the
// padding id sort behind every other and have no gradient.
#include "kernels.h"
#include "rows.cuh"
#include "tc05.cuh"

#include <cooperative_groups.h>
#include <cuda_runtime.h>

namespace {

namespace cg = cooperative_groups;

// ---- forward ----------------------------------------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kUnroll = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
embed_scaled_kernel(const long long* __restrict__ ids, const T* __restrict__ table, T* __restrict__ out,
                    long long tokens, int cols, long long vocab, float scale) {
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const unsigned groups = (cols + 7) >> 3;
  const long long total = tokens * groups;
  const long long base = static_cast<long long>(blockIdx.x) * (kThreads * kUnroll) + threadIdx.x;
  rows::Raw<T> v[kUnroll];
  long long row[kUnroll];
  int col[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long long i = base + u * kThreads;
    if (i < total) {
      row[u] = total <= 0xffffffffll ? static_cast<unsigned>(i) / groups : i / groups;
      col[u] = static_cast<int>(i - row[u] * groups) * 8;
      long long id = __ldg(ids + row[u]);
      id = id < 0 ? 0 : (id >= vocab ? vocab - 1 : id);  // out-of-range ids are clamped, never dereferenced as given
      rows::load<VEC>(v[u], table + id * cols, col[u], cols);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (base + u * kThreads < total) {
      float f[8];
      rows::unpack(v[u], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= scale;
      rows::store<VEC>(f, out + row[u] * cols, col[u], cols);
    }
  }
}

// ---- sort + fill --------------------------------------------------------------------------------------------------------
constexpr int kSortCtas = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 9;  // of a digit: two passes for vocabularies up to 2^18 - 1
constexpr int kMaxBins = 1 << kMaxBits;

struct SortArgs {
  const long long* ids;
  long long n;
  long long vocab, padding_idx;
  unsigned* key[2];
  unsigned* pos[2];
  int passes, bits;
  uint4* fill;  // or null
  long long fill_bytes;
};

__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
embed_sort_kernel(const SortArgs p) {
  extern __shared__ unsigned warp_hist[];  // [kSortWarps][bins]
  __shared__ unsigned cta_total[kMaxBins];
  __shared__ unsigned offset[kMaxBins];
  __shared__ unsigned scan_sums[kSortWarps];
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (blockIdx.x >= kSortCtas) {
    const long long vecs = p.fill_bytes >> 4;
    const long long step = static_cast<long long>(gridDim.x - kSortCtas) * kSortThreads;
    const long long first = static_cast<long long>(blockIdx.x - kSortCtas) * kSortThreads + tid;
    for (long long i = first; i < vecs; i += step) p.fill[i] = make_uint4(0, 0, 0, 0);
    if (first < (p.fill_bytes & 15)) reinterpret_cast<unsigned char*>(p.fill + vecs)[first] = 0;
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x;
  const int bins = 1 << p.bits;
  // a warp owns a run of neighbouring places, a multiple of 32 long
  const long long run = ((p.n + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31) & ~31ll;
  const long long start = (static_cast<long long>(rank) * kSortWarps + warp) * run;
  const long long end = start + run < p.n ? start + run : p.n;
  unsigned* hist = warp_hist + warp * bins;
  const unsigned below = (1u << lane) - 1u;

  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const unsigned* src_key = p.key[(pass + 1) & 1];
    const unsigned* src_pos = p.pos[(pass + 1) & 1];
    auto key_at = [&](long long i) -> unsigned {
      if (pass > 0) return __ldcg(src_key + i);
      const long long id = p.ids[i];
      return static_cast<unsigned>((id < 0 || id >= p.vocab || id == p.padding_idx) ? p.vocab : id);
    };
    for (int i = tid; i < kSortWarps * bins; i += kSortThreads) warp_hist[i] = 0;
    __syncthreads();
    for (long long i0 = start; i0 < end; i0 += 32) {
      const long long i = i0 + lane;
      const unsigned digit = i < end ? (key_at(i) >> shift) & (bins - 1) : 0xffffffffu;
      const unsigned peers = __match_any_sync(0xffffffffu, digit);
      if (i < end && (peers & below) == 0) hist[digit] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    for (int d = tid; d < bins; d += kSortThreads) {  // counts of the earlier warps of this CTA
      unsigned sum = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = warp_hist[w * bins + d];
        warp_hist[w * bins + d] = sum;
        sum += c;
      }
      cta_total[d] = sum;
    }
    cluster.sync();
    unsigned before = 0, all = 0;
    if (tid < bins) {
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) {
        const unsigned v = cluster.map_shared_rank(cta_total, c)[tid];
        if (c < rank) before += v;
        all += v;
      }
    }
    // exclusive scan of `all` over the digits
    unsigned incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) scan_sums[warp] = incl;
    __syncthreads();
    unsigned lead = 0;
    for (int w = 0; w < warp; ++w) lead += scan_sums[w];
    if (tid < bins) offset[tid] = lead + incl - all + before;
    __syncthreads();
    unsigned* dst_key = p.key[pass & 1];
    unsigned* dst_pos = p.pos[pass & 1];
    for (long long i0 = start; i0 < end; i0 += 32) {
      const long long i = i0 + lane;
      const bool in = i < end;
      const unsigned key = in ? key_at(i) : 0;
      const unsigned digit = in ? (key >> shift) & (bins - 1) : 0xffffffffu;
      const unsigned peers = __match_any_sync(0xffffffffu, digit);
      if (in) {
        const unsigned to = offset[digit] + hist[digit] + __popc(peers & below);
        dst_key[to] = key;
        dst_pos[to] = pass > 0 ? __ldcg(src_pos + i) : static_cast<unsigned>(i);
      }
      __syncwarp();
      if (in && (peers & below) == 0) hist[digit] += __popc(peers);
      __syncwarp();
    }
    __threadfence();  // the next pass reads what all eight CTAs wrote
    cluster.sync();
  }
}

// ---- sums over the sorted order -------------------------------------------------------------------------------------------
constexpr int kTile = 16;     // sorted tokens per warp
constexpr int kSlab = 256;    // columns per warp
constexpr int kAhead = 16;    // rows in flight
constexpr int kSumWarps = 4;

struct SumArgs {
  const unsigned *key, *pos;
  const void* dout;
  long long ld;
  void* grad;        // dense gradient in the table's type, or null:
  float* acc[2];     // fp32 buffers that the sums are added to (either may be null)
  float* part;       // [2 * tiles, part_ld]
  long long part_ld;
  unsigned n, vocab;
  int cols;
  float scale;
};

template <typename T, bool VEC>
__device__ __forceinline__ void emit(const SumArgs& p, unsigned row, int col, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= p.scale;
  const long long at = static_cast<long long>(row) * p.cols;
  if (p.grad) rows::store<VEC>(f, static_cast<T*>(p.grad) + at, col, p.cols);
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    float* acc = b == 0 ? p.acc[0] : p.acc[1];
    if (acc) {
      rows::Raw<float> r;
      float old[8];
      rows::load<VEC>(r, static_cast<const float*>(acc + at), col, p.cols);
      rows::unpack(r, old);
#pragma unroll
      for (int j = 0; j < 8; ++j) old[j] += f[j];
      rows::store<VEC>(old, acc + at, col, p.cols);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kSumWarps * 32)
embed_sum_kernel(const SumArgs p) {
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const int lane = threadIdx.x & 31;
  const unsigned tile = blockIdx.x * kSumWarps + (threadIdx.x >> 5);
  const unsigned first = tile * kTile;
  if (first >= p.n) return;
  const int col = blockIdx.y * kSlab + lane * 8;
  const bool live = col < p.cols;
  const int count = static_cast<int>(p.n - first < kTile ? p.n - first : kTile);
  // past the end: a key that no token has
  const unsigned key = lane < count ? p.key[first + lane] : 0xffffffffu;
  const unsigned pos = lane < count ? p.pos[first + lane] : 0u;
  const unsigned prev = first > 0 ? p.key[first - 1] : 0xffffffffu;
  const unsigned next = first + kTile < p.n ? p.key[first + kTile] : 0xffffffffu;
  float acc[8] = {};
  bool begins = __shfl_sync(0xffffffffu, key, 0) != prev;  // the current piece starts in this tile
  for (int j0 = 0; j0 < count; j0 += kAhead) {
    rows::Raw<T> v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned k = __shfl_sync(0xffffffffu, key, j0 + u);
      const unsigned at = __shfl_sync(0xffffffffu, pos, j0 + u);
      if (live && k < p.vocab) rows::load<VEC>(v[u], static_cast<const T*>(p.dout) + at * p.ld, col, p.cols);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = j0 + u;
      const unsigned k = __shfl_sync(0xffffffffu, key, j);
      const unsigned after = j + 1 < kTile ? __shfl_sync(0xffffffffu, key, (j + 1) & 31) : next;
      if (k >= p.vocab) continue;  // (warp-uniform) padding, out of range, past the end
      if (live) {
        float f[8];
        rows::unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += f[e];
      }
      if (after != k || j + 1 == kTile) {
        const bool ends = after != k;
        if (live) {
          if (begins && ends) {
            emit<T, VEC>(p, k, col, acc);
          } else {
            float* dst = p.part + (2ll * tile + (begins ? 1 : 0)) * p.part_ld + col;
            reinterpret_cast<float4*>(dst)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        begins = true;
      }
    }
  }
}

constexpr int kJoinWarps = 8;
constexpr int kJoinAhead = 8;  // partial rows in flight per warp

template <typename T, bool VEC>
__global__ void __launch_bounds__(kJoinWarps * 32)
embed_join_kernel(const SumArgs p) {
  __shared__ float red[kJoinWarps][kSlab];
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const unsigned tile = blockIdx.x;
  const unsigned first = tile * kTile;
  if (first + kTile >= p.n) return;  // nothing follows the last tile
  const unsigned k = p.key[first + kTile - 1];
  if (k >= p.vocab || p.key[first + kTile] != k) return;                              // ends here
  if (p.key[first] == k && first > 0 && p.key[first - 1] == k) return;                // began in an earlier tile
  // the last tile that holds k: keys are sorted, so its first key tells
  unsigned lo = tile + 1, hi = (p.n - 1) / kTile;  // tile lo's first key is k
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo + 1) / 2;
    if (p.key[mid * kTile] == k) lo = mid; else hi = mid - 1;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.y * kSlab + lane * 8;
  float acc[8] = {};
  // piece 0 is this tile's, piece i the one that tile + i begins with; warp w adds pieces w, w + 8, ...
  const unsigned pieces = lo - tile + 1;
  for (unsigned i0 = warp; i0 < pieces; i0 += kJoinWarps * kJoinAhead) {
    float4 a[kJoinAhead], b[kJoinAhead];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const unsigned i = i0 + u * kJoinWarps;
      a[u] = b[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < pieces && col < p.cols) {
        const long long slot = i == 0 ? 2ll * tile + 1 : 2ll * (tile + i);
        const float4* src = reinterpret_cast<const float4*>(p.part + slot * p.part_ld + col);
        a[u] = src[0];
        b[u] = src[1];
      }
    }
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      acc[0] += a[u].x; acc[1] += a[u].y; acc[2] += a[u].z; acc[3] += a[u].w;
      acc[4] += b[u].x; acc[5] += b[u].y; acc[6] += b[u].z; acc[7] += b[u].w;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) red[warp][e * 32 + lane] = acc[e];
  __syncthreads();
  if (warp == 0 && col < p.cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) acc[e] += red[w][e * 32 + lane];
    }
    emit<T, VEC>(p, k, col, acc);
  }
}

// ---- few tokens: the owner of a table row looks for its tokens -----------------------------------------------------------
constexpr int kSmallTokens = 256;  // (at 512 of a 4096 x 1024 table the three launches are faster: 19 us against 28 us)
constexpr int kSmallThreads = 256;
constexpr int kSmallRows = 8192;  // table rows per block at most
constexpr unsigned kSmallBlocks = 148 * 4;  // (interleaved rows: frequent ids are neighbours in most vocabularies)

struct SmallArgs {
  SumArgs s;             // key and pos unused
  const long long* ids;
  long long padding_idx;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kSmallThreads)
embed_small_kernel(const SmallArgs p) {
  __shared__ unsigned row_of[kSmallTokens];         // tokens of this block's rows, in the order of their positions
  __shared__ unsigned short token_of[kSmallTokens];
  __shared__ unsigned present[kSmallRows / 32];
  __shared__ int warp_count[kSmallThreads / 32];
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned step = gridDim.x;  // this block's rows: blockIdx.x, blockIdx.x + step, ...
  const unsigned nrows = (p.s.vocab - blockIdx.x + step - 1) / step;
  for (unsigned i = tid; i < (nrows + 31) / 32; i += kSmallThreads) present[i] = 0;
  __syncthreads();
  int m = 0;
  for (unsigned base = 0; base < p.s.n; base += kSmallThreads) {
    const unsigned t = base + tid;
    const long long id = t < p.s.n ? p.ids[t] : -1;
    const bool mine = id >= 0 && id < p.s.vocab && id != p.padding_idx && static_cast<unsigned>(id) % step == blockIdx.x;
    const unsigned votes = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) warp_count[warp] = __popc(votes);
    __syncthreads();
    int before = m, all = m;
#pragma unroll
    for (int w = 0; w < kSmallThreads / 32; ++w) {
      if (w < warp) before += warp_count[w];
      all += warp_count[w];
    }
    if (mine) {
      const int at = before + __popc(votes & ((1u << lane) - 1u));
      const unsigned local = static_cast<unsigned>(id) / step;
      row_of[at] = local;
      token_of[at] = static_cast<unsigned short>(t);
      atomicOr(&present[local >> 5], 1u << (local & 31));
    }
    m = all;
    __syncthreads();
  }
  if (p.s.grad) {  // rows that no token names
    const unsigned groups = (p.s.cols + 7) >> 3;
    const unsigned total = nrows * groups;  // (below 2^32: the launcher checks)
    for (unsigned i = tid; i < total; i += kSmallThreads) {
      const unsigned local = i / groups;
      if ((present[local >> 5] >> (local & 31)) & 1u) continue;
      const float zero[8] = {};
      rows::store<VEC>(zero, static_cast<T*>(p.s.grad) + (blockIdx.x + static_cast<long long>(local) * step) * p.s.cols,
                       static_cast<int>(i - local * groups) * 8, p.s.cols);
    }
  }
  // a warp takes (token, 256 columns) pairs; only a row's first token does the work, for all of the row's tokens
  const int slabs = (p.s.cols + kSlab - 1) / kSlab;
  for (int item = warp; item < m * slabs; item += kSmallThreads / 32) {
    const int first = item / slabs;
    const int col = (item - first * slabs) * kSlab + lane * 8;
    const unsigned local = row_of[first];
    bool seen = false;
    for (int base = 0; base < first; base += 32)
      seen |= base + lane < first && row_of[base + lane] == local;
    if (__any_sync(0xffffffffu, seen)) continue;
    float acc[8] = {};
    for (int base = first & ~31; base < m; base += 32) {
      unsigned left = __ballot_sync(0xffffffffu, base + lane >= first && base + lane < m && row_of[base + lane] == local);
      while (left != 0) {
        rows::Raw<T> v[kAhead];
        int count = 0;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (left != 0) {
            const int at = base + __ffs(left) - 1;
            left &= left - 1;
            count = u + 1;
            if (col < p.s.cols) rows::load<VEC>(v[u], static_cast<const T*>(p.s.dout) + token_of[at] * p.s.ld, col, p.s.cols);
          }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (u < count && col < p.s.cols) {
            float f[8];
            rows::unpack(v[u], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += f[e];
          }
        }
      }
    }
    if (col < p.s.cols) emit<T, VEC>(p.s, blockIdx.x + local * step, col, acc);
  }
}

bool small_path(long long tokens, int cols, long long vocab) {
  const long long rows = (vocab + kSmallBlocks - 1) / kSmallBlocks;
  return tokens <= kSmallTokens && rows <= kSmallRows && rows * ((cols + 7) / 8) < (1ll << 32);
}

template <typename T>
cudaError_t small(const SmallArgs& a, bool vec, cudaStream_t st) {
  const dim3 grid(a.s.vocab < kSmallBlocks ? a.s.vocab : kSmallBlocks);
  return vec ? tc05::launch_pdl(embed_small_kernel<T, true>, grid, dim3(kSmallThreads), 0, st, a)
             : tc05::launch_pdl(embed_small_kernel<T, false>, grid, dim3(kSmallThreads), 0, st, a);
}

template <typename T>
cudaError_t gather(const long long* ids, const void* table, void* out, long long tokens, int cols, long long vocab,
                   float scale, cudaStream_t st) {
  const long long vecs = tokens * ((cols + 7) / 8);
  const dim3 grid(static_cast<unsigned>((vecs + kThreads * kUnroll - 1) / (kThreads * kUnroll)));
  auto W = static_cast<const T*>(table);
  auto O = static_cast<T*>(out);
  return rows::vector_rows(table, cols, cols) && rows::vector_rows(out, cols, cols)
             ? tc05::launch_pdl(embed_scaled_kernel<T, true>, grid, dim3(kThreads), 0, st, ids, W, O, tokens, cols, vocab, scale)
             : tc05::launch_pdl(embed_scaled_kernel<T, false>, grid, dim3(kThreads), 0, st, ids, W, O, tokens, cols, vocab, scale);
}

template <typename T>
cudaError_t sums(const SumArgs& s, bool vec, cudaStream_t st) {
  const unsigned tiles = (s.n + kTile - 1) / kTile;
  const unsigned slabs = (s.cols + kSlab - 1) / kSlab;
  const dim3 grid((tiles + kSumWarps - 1) / kSumWarps, slabs), join(tiles, slabs);
  cudaError_t rc = vec ? tc05::launch_pdl(embed_sum_kernel<T, true>, grid, dim3(kSumWarps * 32), 0, st, s)
                       : tc05::launch_pdl(embed_sum_kernel<T, false>, grid, dim3(kSumWarps * 32), 0, st, s);
  if (rc != cudaSuccess || tiles < 2) return rc;
  return vec ? tc05::launch_pdl(embed_join_kernel<T, true>, join, dim3(kJoinWarps * 32), 0, st, s)
             : tc05::launch_pdl(embed_join_kernel<T, false>, join, dim3(kJoinWarps * 32), 0, st, s);
}

constexpr long long kMaxTokens = 1ll << 30;
constexpr int kMaxCols = 1 << 20;

}  // namespace

extern "C" int db200_embed_scaled(const long long* ids, const void* table, void* out, long long tokens, int cols,
                                  long long vocab, float scale, int dtype, void* stream) {
  if (tokens <= 0) return 0;
  if (!ids || !table || !out || cols <= 0 || vocab <= 0) return -10;
  if (tokens > kMaxTokens || cols > kMaxCols || tokens * ((cols + 7) / 8) / (kThreads * kUnroll) >= 0x7fffffffll) return -12;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t rc = cudaErrorInvalidValue;
  if (dtype == 0) rc = gather<__nv_bfloat16>(ids, table, out, tokens, cols, vocab, scale, st);
  else if (dtype == 1) rc = gather<__half>(ids, table, out, tokens, cols, vocab, scale, st);
  else if (dtype == 2) rc = gather<float>(ids, table, out, tokens, cols, vocab, scale, st);
  else return -11;
  return rc == cudaSuccess ? 0 : -4;
}

// Bytes of the workspace of db200_embed_sorted_bwd.
extern "C" long long db200_embed_sorted_workspace(long long tokens, int cols, long long vocab) {
  if (tokens <= 0 || cols <= 0 || small_path(tokens, cols, vocab)) return 0;
  const long long n = (tokens + 3) / 4 * 4, tiles = (tokens + kTile - 1) / kTile;
  return 16 * n + 2 * tiles * ((cols + kSlab - 1) / kSlab * kSlab) * 4;
}

extern "C" int db200_embed_sorted_bwd(const long long* ids, const void* dout, long long ld, long long tokens, int cols,
                                      long long vocab, long long padding_idx, float scale, int dtype, void* grad,
                                      float* acc0, float* acc1, void* workspace, void* stream) {
  if (!dout || !ids || cols <= 0 || vocab <= 0 || ld < cols || (!grad && !acc0 && !acc1) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15) || (reinterpret_cast<uintptr_t>(grad) & 15))
    return -10;
  if (tokens <= 0 || tokens > kMaxTokens || cols > kMaxCols || vocab > 0x7ffffffell) return -12;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  SumArgs s{};
  s.dout = dout;
  s.ld = ld;
  s.grad = grad;
  s.acc[0] = acc0;
  s.acc[1] = acc1;
  s.n = static_cast<unsigned>(tokens);
  s.vocab = static_cast<unsigned>(vocab);
  s.cols = cols;
  s.scale = scale;
  const bool vec = rows::vector_rows(dout, ld, cols) && rows::vector_rows(grad, cols, cols) &&
                   rows::vector_rows(acc0, cols, cols) && rows::vector_rows(acc1, cols, cols);
  cudaError_t rc = cudaErrorInvalidValue;
  if (small_path(tokens, cols, vocab)) {
    const SmallArgs a{s, ids, padding_idx};
    if (dtype == 0) rc = small<__nv_bfloat16>(a, vec, st);
    else if (dtype == 1) rc = small<__half>(a, vec, st);
    else if (dtype == 2) rc = small<float>(a, vec, st);
    else return -11;
    return rc == cudaSuccess ? 0 : -4;
  }
  if (!workspace) return -10;
  const long long n = (tokens + 3) / 4 * 4;
  unsigned* w = static_cast<unsigned*>(workspace);
  SortArgs a{};
  a.ids = ids;
  a.n = tokens;
  a.vocab = vocab;
  a.padding_idx = padding_idx;
  a.key[0] = w; a.key[1] = w + n; a.pos[0] = w + 2 * n; a.pos[1] = w + 3 * n;
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;  // keys reach `vocab`
  a.passes = (bits + kMaxBits - 1) / kMaxBits;
  a.bits = (bits + a.passes - 1) / a.passes;
  const long long size = dtype == 2 ? 4 : 2;
  a.fill = static_cast<uint4*>(grad);
  a.fill_bytes = grad ? vocab * cols * size : 0;
  static bool configured[16] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) return -3;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortWarps * kMaxBins * 4) !=
        cudaSuccess)
      return -3;
    configured[dev] = true;
  }
  // 288 fill CTAs measured best (128100 x 768 bf16: 42 us, 4.7 TB/s of writes; 136 and 1152: 50 to 53 us; 32-byte stores and
  // bulk stores of zeroed shared memory: 42 us as well)
  long long fill_ctas = (a.fill_bytes / 16 + kSortThreads * 8 - 1) / (kSortThreads * 8);
  fill_ctas = (fill_ctas < 288 ? fill_ctas : 288);
  if (a.fill_bytes && fill_ctas == 0) fill_ctas = 1;
  const unsigned grid = kSortCtas * (1 + static_cast<unsigned>((fill_ctas + kSortCtas - 1) / kSortCtas));
  rc = tc05::launch_pdl(embed_sort_kernel, dim3(grid), dim3(kSortThreads),
                                    static_cast<size_t>(kSortWarps) * (1u << a.bits) * 4, st, a);
  if (rc != cudaSuccess) return -4;
  s.key = a.key[(a.passes - 1) & 1];
  s.pos = a.pos[(a.passes - 1) & 1];
  s.part = reinterpret_cast<float*>(w + 4 * n);
  s.part_ld = (cols + kSlab - 1) / kSlab * kSlab;
  if (dtype == 0) rc = sums<__nv_bfloat16>(s, vec, st);
  else if (dtype == 1) rc = sums<__half>(s, vec, st);
  else if (dtype == 2) rc = sums<float>(s, vec, st);
  else return -11;
  return rc == cudaSuccess ? 0 : -4;
}

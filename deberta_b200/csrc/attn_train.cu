// One host entry per direction for attention under dropout: the launches of a training step's forward or backward pass in
// one call (a call from Python costs as much host time as three launches from here), and the last step of the rotary
// backward pass as one kernel.
#include "kernels.h"
#include "tc05.cuh"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

// (posgrad.cu)
extern "C" int db200_posgrad_dual(const void* g, long long ld_g, const void* tab, long long ld_tab, const void* x,
                                  long long ld_x, float* out_f32, long long ld_of, void* out_bf16, long long ld_ob,
                                  const float* acc_in, long long ld_ai, float* d_tab, long long ld_dt, int T, int heads,
                                  int W, void* stream);

namespace {

constexpr int kD = 64;

// dq[t, :] = R(-t) dq_acc[t, :], dk[t, :] = R(-t) dk[t, :]: the query gradient leaves its fp32 accumulator rotated and is
// rounded once (a cast and a rotation in place: 10 + 8 bytes per value against 6 + 4 here). A thread owns four pairs.
__global__ void __launch_bounds__(256)
rotate_back_kernel(const float* __restrict__ dq_acc, __nv_bfloat16* __restrict__ dq, __nv_bfloat16* dk, long long ld,
                   const float* __restrict__ cos_t, const float* __restrict__ sin_t, long long tokens, int S, int heads,
                   int rotary_dim) {
  tc05::pdl_launch_dependents();
  tc05::pdl_wait();
  const int vecs = heads * (kD / 8);  // per token and gradient
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long t = i / (2 * vecs);
  if (t >= tokens) return;
  const int r = static_cast<int>(i - t * (2 * vecs));
  const bool is_k = r >= vecs;
  const int col = (is_k ? r - vecs : r) * 8;
  float f[8];
  __nv_bfloat16* dst = (is_k ? dk : dq) + t * ld + col;
  if (is_k) {
    const uint4 u = *reinterpret_cast<const uint4*>(dst);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
    const float4* src = reinterpret_cast<const float4*>(dq_acc + t * (static_cast<long long>(heads) * kD) + col);
    const float4 a = src[0], b = src[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  const int in_head = col % kD;
  const long long at = (t % S) * rotary_dim + in_head;
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (in_head + 2 * e < rotary_dim) {  // (a rotary dimension is even: pairs are whole)
      const float c = __ldg(cos_t + at + 2 * e), s = __ldg(sin_t + at + 2 * e);
      const float x = f[2 * e], y = f[2 * e + 1];
      f[2 * e] = x * c + y * s;
      f[2 * e + 1] = y * c - x * s;
    }
    w[e] = tc05::pack_bf16(f[2 * e], f[2 * e + 1]);
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// the operands that the attention kernels read: those of a rotary call lie rotated in one buffer
AttnArgs kernel_args(const AttnTrainArgs* t) {
  AttnArgs a = t->a;
  if (t->rotary_dim > 0) {
    const long long H = static_cast<long long>(a.heads) * kD;
    a.q = t->qk_rotated;
    a.k = static_cast<const __nv_bfloat16*>(t->qk_rotated) + H;
    a.ldq = a.ldk = 2 * H;
  }
  return a;
}

}  // namespace

extern "C" int db200_attn_train_fwd(const AttnTrainArgs* t, void* stream) {
  const AttnArgs& o = t->a;
  if (o.B <= 0 || o.S <= 0 || o.heads <= 0) return 0;
  const long long T = static_cast<long long>(o.B) * o.S, H = static_cast<long long>(o.heads) * kD;
  int rc = 0;
  if (t->span2 > 0) {  // first, since it may refuse (-13)
    PosBiasArgs p{};
    p.q = o.q; p.k = o.k; p.ldq = o.ldq; p.ldk = o.ldk;
    p.pos_k = t->pos_k; p.pos_q = t->pos_q; p.ld_pos = H;
    p.lut_c2p = t->lut_c2p; p.lut_p2c = t->lut_p2c; p.lut_c2p_host = t->lut_c2p_host; p.lut_p2c_host = t->lut_p2c_host;
    p.B = o.B; p.S = o.S; p.heads = o.heads; p.span2 = t->span2;
    p.bias = const_cast<void*>(o.bias); p.ldb = o.ldb;
    if ((rc = db200_posbias_tc_fwd(&p, stream))) return rc;
  }
  if (o.doc_ids) {
    if ((rc = db200_attn_doc_tiles(o.doc_ids, const_cast<void*>(o.doc_tiles), o.B, o.S, stream))) return rc;
    if (o.doc_order && (rc = db200_attn_doc_order(o.doc_tiles, const_cast<void*>(o.doc_order), o.B, o.S, stream))) return rc;
  }
  if (t->rotary_dim > 0) {
    __nv_bfloat16* y = static_cast<__nv_bfloat16*>(t->qk_rotated);
    const bool one = o.ldq == o.ldk && static_cast<const __nv_bfloat16*>(o.k) == static_cast<const __nv_bfloat16*>(o.q) + H;
    rc = db200_rotary_bf16(o.q, y, o.ldq, 2 * H, t->cos_t, t->sin_t, T, o.S, one ? 2 * o.heads : o.heads, kD, t->rotary_dim, 0,
                           stream);
    if (!rc && !one)
      rc = db200_rotary_bf16(o.k, y + H, o.ldk, 2 * H, t->cos_t, t->sin_t, T, o.S, o.heads, kD, t->rotary_dim, 0, stream);
    if (rc) return rc;
  }
  const AttnArgs a = kernel_args(t);
  return db200_attn_fwd(&a, stream);
}

extern "C" int db200_attn_train_bwd(const AttnTrainArgs* t, void* stream) {
  const AttnArgs a = kernel_args(t);
  if (a.B <= 0 || a.S <= 0 || a.heads <= 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long T = static_cast<long long>(a.B) * a.S, H = static_cast<long long>(a.heads) * kD;
  if (!t->dq || !aligned16(t->dq) || a.ld_dk != a.ld_dv || (a.ld_dk % 8) || T > 0x7fffffffll) return -10;
  if (t->span2 > 0) {
    if (!t->fold || !t->d_tables || !t->d_tables_out || !t->ranges_c2p || !t->ranges_p2c) return -10;
    if (cudaMemsetAsync(t->d_tables, 0, 2 * static_cast<size_t>(t->span2) * H * 4, st) != cudaSuccess) return -4;
  }
  int rc = db200_attn_delta(a.dout, a.ld_do, a.out, a.ldo, const_cast<float*>(a.delta), a.dq_acc, a.B, a.S, a.heads, stream);
  if (rc) return rc;
  // skipped tiles are never written: with document ids the bias gradient starts from zero
  if (t->span2 > 0 && a.doc_ids &&
      cudaMemsetAsync(a.dbias, 0, static_cast<size_t>(T) * a.heads * a.ldb * 2, st) != cudaSuccess)
    return -4;
  if ((rc = db200_attn_bwd(&a, stream))) return rc;
  if (t->span2 > 0) {
    const long long ld_fold = static_cast<long long>(a.heads) * t->span2;
    // both reductions first: the second finds part of the bias gradient that the first read in the L2 (a product between them
    // cost 43 us at B=32, S=512, 12 heads). Then dQ += dC2P · PosK, dPosK = dC2Pᵀ · Q and dK += dP2C · PosQ, dPosQ = dP2Cᵀ · K
    __nv_bfloat16* fold_p2c = static_cast<__nv_bfloat16*>(t->fold) + T * ld_fold;
    if ((rc = db200_posbias_scatter_ranges(a.dbias, t->ranges_c2p, t->fold, 0, a.B, a.S, static_cast<int>(a.ldb), a.heads,
                                           t->span2, stream)))
      return rc;
    if ((rc = db200_posbias_scatter_ranges(a.dbias, t->ranges_p2c, fold_p2c, 1, a.B, a.S, static_cast<int>(a.ldb), a.heads,
                                           t->span2, stream)))
      return rc;
    if ((rc = db200_posgrad_dual(t->fold, ld_fold, t->pos_k, H, a.q, a.ldq, nullptr, 0, t->dq, a.ld_dk, a.dq_acc, H, t->d_tables,
                                 H, static_cast<int>(T), a.heads, t->span2, stream)))
      return rc;
    if ((rc = db200_posgrad_dual(fold_p2c, ld_fold, t->pos_q, H, a.k, a.ldk, nullptr, 0, a.dk, a.ld_dk, nullptr, 0,
                                 t->d_tables + t->span2 * H, H, static_cast<int>(T), a.heads, t->span2, stream)))
      return rc;
    return db200_cast_f32_bf16(t->d_tables, t->d_tables_out, H, 2ll * t->span2, static_cast<int>(H), stream);
  }
  if (t->rotary_dim <= 0) return db200_cast_f32_bf16(a.dq_acc, t->dq, a.ld_dk, T, static_cast<int>(H), stream);
  const long long vecs = T * 2 * a.heads * (kD / 8);
  if ((vecs + 255) / 256 > 0x7fffffffll) return -12;
  return tc05::launch_pdl(rotate_back_kernel, dim3(static_cast<unsigned>((vecs + 255) / 256)), dim3(256), 0, st, a.dq_acc,
                          static_cast<__nv_bfloat16*>(t->dq), static_cast<__nv_bfloat16*>(a.dk), a.ld_dk, t->cos_t, t->sin_t,
                          T, a.S, a.heads, t->rotary_dim) == cudaSuccess ? 0 : -4;
}

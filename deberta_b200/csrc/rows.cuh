// Eight neighbouring values of a row in the three activation types, for kernels that hold rows in registers: raw
// vectors as they travel (16 bytes, 32 for fp32) and their fp32 values.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace rows {

template <typename T>
struct Raw {  // 16-bit types
  uint4 v;
};
template <>
struct Raw<float> {
  float4 a, b;
};

__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }

__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const Raw<__half>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void unpack(const Raw<float>& r, float (&f)[8]) {
  f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
  f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
}
__device__ __forceinline__ void pack(Raw<__nv_bfloat16>& r, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&v);
  }
  r.v = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(Raw<__half>& r, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<uint32_t*>(&v);
  }
  r.v = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(Raw<float>& r, const float (&f)[8]) {
  r.a = make_float4(f[0], f[1], f[2], f[3]);
  r.b = make_float4(f[4], f[5], f[6], f[7]);
}

// Columns [col, col + 8) of a row of `cols`. VEC: whole aligned vectors (cols and strides multiples of 8, 16-byte
// aligned rows); otherwise value by value, zeros past the end, which a store leaves out.
template <bool VEC, typename T>
__device__ __forceinline__ void load(Raw<T>& r, const T* row, int col, int cols) {
  if constexpr (VEC) {
    r = *reinterpret_cast<const Raw<T>*>(row + col);
  } else {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = col + j < cols ? to_f(row[col + j]) : 0.f;
    pack(r, f);
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store(const float (&f)[8], T* row, int col, int cols) {
  if constexpr (VEC) {
    Raw<T> r;
    pack(r, f);
    *reinterpret_cast<Raw<T>*>(row + col) = r;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols) row[col + j] = from_f<T>(f[j]);
  }
}

inline bool vector_rows(const void* p, long long stride, int cols) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0 && cols % 8 == 0);
}

}  // namespace rows

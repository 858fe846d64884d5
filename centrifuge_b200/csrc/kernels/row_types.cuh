// Element types of the row operators: loads and stores of W consecutive elements as fp32, and the
// dispatch from the host's type codes to template arguments.
#pragma once
#include <cuda_fp16.h>

#include "launch_api.h"
#include "sm100_common.cuh"

namespace cfb {

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// W elements as they lie in memory.  Packs of 16 bytes and less are one access; packs of 32 bytes
// (eight fp32) are one 256-bit access as well: two 128-bit stores of a lane each fill half of a
// 32-byte sector, and a fill of 2.1 GB ran at 4.3 TB/s with them.  These accesses are volatile, so
// code that wants several in flight issues its loads before its stores.
template <typename T, int W>
struct __align__(W * sizeof(T)) Pack {
  T v[W];
};

template <typename T, int W>
__device__ __forceinline__ Pack<T, W> load_pack(const T* p) {
  Pack<T, W> k;
  if constexpr (sizeof(k) == 32) {
    uint32_t* r = reinterpret_cast<uint32_t*>(&k);
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
  } else {
    k = *reinterpret_cast<const Pack<T, W>*>(p);
  }
  return k;
}
template <typename T, int W>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, W>& k) {
  if constexpr (sizeof(k) == 32) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(&k);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
    *reinterpret_cast<Pack<T, W>*>(p) = k;
  }
}
template <typename T, int W>
__device__ __forceinline__ void unpack(const Pack<T, W>& k, float* f) {
#pragma unroll
  for (int i = 0; i < W; ++i) f[i] = to_f32(k.v[i]);
}
template <typename T, int W>
__device__ __forceinline__ void load_f32(const T* p, float* f) {
  unpack<T, W>(load_pack<T, W>(p), f);
}
template <typename T, int W>
__device__ __forceinline__ void store_f32(T* p, const float* f) {
  Pack<T, W> k;
#pragma unroll
  for (int i = 0; i < W; ++i) k.v[i] = from_f32<T>(f[i]);
  store_pack<T, W>(p, k);
}

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// An index outside [0, n) records kErrBounds in the status block; the caller skips the access.
__device__ __forceinline__ bool index_in(long long i, long long n, int* err) {
  if (i >= 0 && i < n) return true;
  if (err) atomicCAS(err, 0, kErrBounds);
  return false;
}

template <typename T>
struct TypeTag {
  using type = T;
};
// f(TypeTag<T>) for a host type code (kBF16, kF16, kF32); -12 for any other.
template <typename F>
int with_type(int code, F&& f) {
  switch (code) {
    case kBF16: return f(TypeTag<__nv_bfloat16>());
    case kF16: return f(TypeTag<__half>());
    case kF32: return f(TypeTag<float>());
    default: return -12;
  }
}
inline int type_bytes(int code) { return code == kF32 ? 4 : 2; }
// Whether rows that start at p, ld elements apart, can be read eight elements at a time.
inline bool rows_of_8(const void* p, long long ld, int code) {
  const int pack = 8 * type_bytes(code);
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % pack == 0 && ld % 8 == 0);
}

inline int launch_status() { return cudaGetLastError() == cudaSuccess ? 0 : -3; }

}  // namespace cfb

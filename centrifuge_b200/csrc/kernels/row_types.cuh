// Element types of the row operators: loads and stores of W consecutive elements as fp32, and the
// dispatch from the host's type codes to template arguments.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

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

// Eight elements of a row in shared memory.
template <typename T>
__device__ __forceinline__ Pack<T, 8> shared_pack(const T* p) {
  Pack<T, 8> k;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
    reinterpret_cast<uint4*>(&k)[i] = reinterpret_cast<const uint4*>(p)[i];
  return k;
}

// Asks the L2 cache for the whole 16-byte pieces of the `bytes` from p.
__device__ __forceinline__ void prefetch_l2(const void* p, int bytes) {
  const uintptr_t at = (reinterpret_cast<uintptr_t>(p) + 15) & ~static_cast<uintptr_t>(15);
  const int n = (bytes - static_cast<int>(at - reinterpret_cast<uintptr_t>(p))) & ~15;
  if (n > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(n) : "memory");
}

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------- pairs of fp32
// sm_100 multiplies and adds two fp32 in one instruction on a 64-bit register pair.  The row
// kernels' arithmetic is a large part of their issue slots, so the wide ones work on pairs.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float s) { return f2(s, s); }
__device__ __forceinline__ float2 halves(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  const float2 t = halves(a);
  return t.x + t.y;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// The N elements of a pack (N even) as N / 2 pairs, and back.
template <typename T, int N>
__device__ __forceinline__ void unpack_f2(const Pack<T, N>& k, F2* f) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&k);
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      f[i] = f2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[i] = f2(to_f32(k.v[2 * i]), to_f32(k.v[2 * i + 1]));
  }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack_f2(const F2* f) {
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 t = halves(f[i]);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      reinterpret_cast<uint32_t*>(&k)[i] = pack_bf16x2(t.x, t.y);
    } else {
      k.v[2 * i] = from_f32<T>(t.x);
      k.v[2 * i + 1] = from_f32<T>(t.y);
    }
  }
  return k;
}
template <typename T, int N>
__device__ __forceinline__ void load_f2(const T* p, F2* f) {
  unpack_f2<T, N>(load_pack<T, N>(p), f);
}
template <typename T, int N>
__device__ __forceinline__ void store_f2(T* p, const F2* f) {
  store_pack<T, N>(p, pack_f2<T, N>(f));
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> zero_pack() {
  Pack<T, N> k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.v[i] = from_f32<T>(0.f);
  return k;
}

// How a team of threads walks the columns of a row: group k of thread t begins at column(t, k) and
// is 2 P columns wide.  Columns from H on are zeros, and are not stored.
//
// WideCols: eight neighbours, for rows of whole aligned groups of eight.
struct WideCols {
  static constexpr int P = 4;
  template <typename T>
  using Raw = Pack<T, 8>;
  static __device__ __forceinline__ int column(int t, int k) { return (t + k * blockDim.x) * 8; }
  template <typename T>
  static __device__ __forceinline__ Raw<T> load(const T* row, int c, int H) {
    return c < H ? load_pack<T, 8>(row + c) : zero_pack<T, 8>();
  }
  template <typename T>
  static __device__ __forceinline__ void unpack(const Raw<T>& k, F2* f) {
    unpack_f2<T, 8>(k, f);
  }
  template <typename T>
  static __device__ __forceinline__ void store(T* row, int c, int H, const F2* f) {
    if (c < H) store_f2<T, 8>(row + c, f);
  }
  // a row in shared memory (the accesses above are of global memory)
  static __device__ __forceinline__ void put(float* row, int c, int H, const F2* f) {
    if (c >= H) return;
#pragma unroll
    for (int i = 0; i < P; ++i) reinterpret_cast<float2*>(row + c)[i] = halves(f[i]);
  }
};
// PairCols: one pair, for teams of NT threads and rows of any width and alignment: neighbours
// (W = 2), or, where not even two elements are aligned (W = 1), the columns c and c + NT, so that
// the arithmetic works on pairs all the same.
template <int W, int NT>
struct PairCols {
  static constexpr int P = 1;
  template <typename T>
  using Raw = F2;
  static __device__ __forceinline__ int column(int t, int k) { return t * W + k * 2 * NT; }
  template <typename T>
  static __device__ __forceinline__ F2 load(const T* row, int c, int H) {
    if constexpr (W == 1)
      return f2(c < H ? to_f32(row[c]) : 0.f, c + NT < H ? to_f32(row[c + NT]) : 0.f);
    F2 f = f2(0.f);
    if (c < H) load_f2<T, 2>(row + c, &f);
    return f;
  }
  template <typename T>
  static __device__ __forceinline__ void unpack(const F2& k, F2* f) {
    f[0] = k;
  }
  template <typename T>
  static __device__ __forceinline__ void store(T* row, int c, int H, const F2* f) {
    if constexpr (W == 1) {
      const float2 t = halves(f[0]);
      if (c < H) row[c] = from_f32<T>(t.x);
      if (c + NT < H) row[c + NT] = from_f32<T>(t.y);
    } else if (c < H) {
      store_f2<T, 2>(row + c, f);
    }
  }
  static __device__ __forceinline__ void put(float* row, int c, int H, const F2* f) {
    store(row, c, H, f);
  }
};

// ---------------------------------------------------------------- sums of several rows
// v[r], summed over the warp, for R rows at once: each exchange halves the number of rows that a
// lane still holds, so that R = 4 takes 6 exchanges instead of 20.  Lane l returns the sum of row
// (l >> (5 - log2 R)).
template <int R>
__device__ __forceinline__ float warp_sums(float* v) {
  const int lane = lane_id();
  int o = 16;
#pragma unroll
  for (int n = R / 2; n > 0; n /= 2, o /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? v[n + i] : v[i];
      const float give = up ? v[i] : v[n + i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  float s = v[0];
#pragma unroll
  for (; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// The same over a team of up to NW warps (a power of two, R * NW <= 32): every thread of the team
// gets all R sums.  red: R * NW floats of shared memory; the caller sees to it that a barrier lies
// between two uses of it.  The team is the block, or, with its number `team` >= 0 in the block,
// exactly NW warps that meet at the block's named barrier 1 + team.
template <int R, int NW>
__device__ __forceinline__ void team_sums(float* v, float* red, int team = -1) {
  constexpr int kShift = R == 4 ? 3 : R == 2 ? 4 : 5;  // lanes of one row after warp_sums
  const int lane = lane_id();
  float s = warp_sums<R>(v);
  if constexpr (NW > 1) {
    const int wp = team >= 0 ? warp_id() % NW : warp_id();
    if ((lane & ((1 << kShift) - 1)) == 0) red[(lane >> kShift) * NW + wp] = s;
    if (team >= 0)
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(NW * 32) : "memory");
    else
      __syncthreads();
    const int at = lane % (R * NW);
    s = team >= 0 || at % NW < static_cast<int>(blockDim.x >> 5) ? red[at] : 0.f;
#pragma unroll
    for (int o = NW / 2; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = __shfl_sync(0xffffffffu, s, r * NW);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = __shfl_sync(0xffffffffu, s, r << kShift);
  }
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
// Whether rows that start at p, ld elements apart, can be read W elements at a time.
inline bool rows_of(int W, const void* p, long long ld, int code) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (W * type_bytes(code)) == 0 && ld % W == 0);
}
inline bool rows_of_8(const void* p, long long ld, int code) { return rows_of(8, p, ld, code); }

// A kernel that is launched behind another one of the same operator: it may start while that one
// ends, and waits for its results itself (after_previous() before it reads them).  Those results
// change during its life, so its pointers to them are not __restrict__: loads of memory that a
// kernel may take for constant can pass the wait or come from a stale cache line.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// In the first kernel: the next one may be put on the SMs from here on.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
inline int launch_status() {
  if (cudaGetLastError() != cudaSuccess) return -3;
  ++cfb_row_launches();
  return 0;
}
template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, int smem, cudaStream_t st,
                  A&&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &attr;
  c.numAttrs = 1;
  if (cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...) != cudaSuccess) {
    cudaGetLastError();  // the error is this launch's, not the next one's
    return -3;
  }
  ++cfb_row_launches();
  return 0;
}


}  // namespace cfb

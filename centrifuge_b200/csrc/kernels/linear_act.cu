// Linear layers with bias, activation and residual on the 5th-generation tensor cores (sm_100a).
//
//   forward   z = x w^T + bias          y = act(z) + resid            x [M, K], w [N, K]
//   dgrad     dz = (dy w) act'(z)       z at the kept rows            dy [M, K], w [K, N]
//   wgrad     dw (+)= dy^T x            dbias (+)= sum of dy's rows   dy [K, M], x [K, N]
//
// bf16 or fp16 operands, products and everything up to the one rounding of an output in fp32; dw and
// dbias are fp32.  Any M, N and K: what TMA copies beyond the operands is zero, and the epilogue
// writes what is inside.  An operand whose rows do not start on 16 bytes is first laid out in a
// workspace with rows that do.
//
// Bound by the tensor cores at a training step's sizes, by latency at small ones.
#include "row_types.cuh"

#include <cudaTypedefs.h>

namespace cfb {

int make_tmap_2d_bf16(CUtensorMap* map, const void* ptr, long long rows, long long cols,
                      long long ld, int box_cols, int box_rows);

// ---------------------------------------------------------------- activations
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + 2^x), 0 for large x
__device__ __forceinline__ float inv_1p_exp2(float x) {
  return __fdividef(1.f, 1.f + exp2_fast(x));
}

constexpr float kLog2e = 1.4426950408889634f;

// The normal distribution's mass below z, and its density times sqrt(2 pi).  With a = |z| the mass
// beyond a is exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.27 a): P is a minimax fit of
// erfcx(a / sqrt 2) / (2 t) of degree six with a relative error of 1.2e-6, so the small values of
// the tail are as exact as the others (1 + erf(z / sqrt 2) loses them).
__device__ __forceinline__ float normal_mass(float z, float& bell) {
  const float a = fabsf(z);
  const float t = __fdividef(1.f, fmaf(0.27f, a, 1.f));
  float p = -0.060966506600379944f;
  p = fmaf(p, t, 0.1590183675289154f);
  p = fmaf(p, t, -0.025057457387447357f);
  p = fmaf(p, t, 0.11830243468284607f);
  p = fmaf(p, t, 0.09249885380268097f);
  p = fmaf(p, t, 0.10852396488189697f);
  p = fmaf(p, t, 0.10767974704504013f);
  bell = exp2_fast(z * z * (-0.5f * kLog2e));
  const float tail = bell * t * p;
  return z < 0.f ? tail : 1.f - tail;
}

// gelu by tanh is z / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kGelu1 = -2.f * 0.7978845608028654f * kLog2e;
constexpr float kGelu3 = kGelu1 * 0.044715f;

template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == kActRelu) return z < 0.f ? 0.f : z;
  if constexpr (ACT == kActSilu) return z * inv_1p_exp2(-kLog2e * z);
  if constexpr (ACT == kActGelu) {
    float bell;
    return z * normal_mass(z, bell);
  }
  if constexpr (ACT == kActGeluTanh) return z * inv_1p_exp2(z * fmaf(kGelu3, z * z, kGelu1));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : z != z ? z : 0.f;
  if constexpr (ACT == kActSilu) {
    const float p = inv_1p_exp2(-kLog2e * z);
    return p * fmaf(z, 1.f - p, 1.f);
  }
  if constexpr (ACT == kActGelu) {
    float bell;
    const float mass = normal_mass(z, bell);
    return fmaf(z * 0.3989422804014327f, bell, mass);
  }
  if constexpr (ACT == kActGeluTanh) {
    // the second term is zero long before |z| = 30, beyond which z^3 may be infinite
    const float c = z != z ? z : fminf(fmaxf(z, -30.f), 30.f);
    const float p = inv_1p_exp2(c * fmaf(kGelu3, c * c, kGelu1));
    const float du = 2.f * 0.7978845608028654f * fmaf(3.f * 0.044715f, c * c, 1.f);
    return p + c * p * (1.f - p) * du;
  }
  return 1.f;
}
// f(ActTag<ACT>): one uniform branch for a whole chunk of columns
template <int ACT>
struct ActTag {
  static constexpr int act = ACT;
};
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case kActRelu: f(ActTag<kActRelu>()); break;
    case kActSilu: f(ActTag<kActSilu>()); break;
    case kActGelu: f(ActTag<kActGelu>()); break;
    case kActGeluTanh: f(ActTag<kActGeluTanh>()); break;
    default: f(ActTag<kActNone>()); break;
  }
}

// ---------------------------------------------------------------- the product
struct LinearArgs {
  int M, N, K;
  int a_mn, b_mn;   // operands [K, M], [K, N] in memory instead of [M, K], [N, K]
  uint32_t idesc;   // instruction descriptor: shape, types and layouts
  void* D;
  long long ldd;
  const void* bias;  // [N]
  const void* R;     // forward: residual [M, N]
  long long ldr;
  void* Z;           // forward: written (or null); dgrad: read at z_rows
  long long ldz;
  const int* z_rows;
  long long n_z;
  int act;
  int add;           // wgrad: add to D
  int vec;           // the outputs, R and Z allow 16-byte accesses
  int* err;
};

// CG CTAs on neighbouring SMs share a tile of CG * 128 rows and BN columns.
template <int CG, int BN>
struct TileShape {
  static constexpr int BM = 128, BK = 64;
  static constexpr int B_ROWS = BN / CG;  // each CTA stages its rows of A and its share of B
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = B_ROWS * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE_BYTES;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int TMEM_COLS = 2 * BN;
};
constexpr int kLinearThreads = 320;  // producer, issuer, eight epilogue warps

// The m-blocks of a group of 16 take turns, so that their rows and the columns at hand stay in L2.
__device__ __forceinline__ void tile_at(int tile, int num_m, int num_n, int& tm, int& tn) {
  constexpr int GROUP = 16;
  const int per_group = GROUP * num_n;
  const int g = tile / per_group, first = g * GROUP;
  const int size = min(num_m - first, GROUP);
  const int r = tile - g * per_group;
  tm = first + r % size;
  tn = r / size;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// 32 neighbouring elements of a row as 16 words, n of them inside (zeros behind).
template <typename T>
__device__ __forceinline__ void load32(const T* p, int n, bool vec, uint32_t* u) {
  if (vec && n >= 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      reinterpret_cast<uint4*>(u)[j] = reinterpret_cast<const uint4*>(p)[j];
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      uint32_t lo = 0, hi = 0;
      if (2 * j < n) lo = s[2 * j];
      if (2 * j + 1 < n) hi = s[2 * j + 1];
      u[j] = lo | (hi << 16);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store32(T* p, int n, bool vec, const float* v) {
  uint32_t u[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) u[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
  if (vec && n >= 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      reinterpret_cast<uint4*>(p)[j] = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
  } else {
    unsigned short* s = reinterpret_cast<unsigned short*>(p);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (2 * j < n) s[2 * j] = static_cast<unsigned short>(u[j]);
      if (2 * j + 1 < n) s[2 * j + 1] = static_cast<unsigned short>(u[j] >> 16);
    }
  }
}

// One row (TMEM lane) of a tile: columns [n0 + first, n0 + last) in chunks of 32, in steps of `step`.
template <typename T, int KIND>
__device__ __forceinline__ void epilogue_rows(const LinearArgs& p, uint32_t taddr, int row, int n0,
                                              int first, int last, int step) {
  const bool live = row < p.M;
  const bool vec = p.vec != 0;
  const T* zrow = nullptr;
  bool z_ok = false;
  if (KIND == kLinearDgrad && live) {
    const long long src = p.z_rows ? p.z_rows[row] : row;
    z_ok = index_in(src, p.n_z, p.err);
    zrow = static_cast<const T*>(p.Z) + (z_ok ? src : 0) * p.ldz;
  }
#pragma unroll 1
  for (int c = first; c < last; c += step) {
    const int col = n0 + c;
    if (col >= p.N) break;  // the same for the whole warp
    const int n = p.N - col;
    uint32_t other[16];  // the residual's or the activation argument's 32 values
    bool have = false;
    if (KIND == kLinearFwd && p.R && live) {
      load32(static_cast<const T*>(p.R) + row * p.ldr + col, n, vec, other);
      have = true;
    }
    if (KIND == kLinearDgrad && z_ok) load32(zrow + col, n, vec, other);
    uint32_t r[32];
    CFB_TMEM_LD32(taddr + c, r);
    tmem_ld_wait();
    if (!live) continue;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
    if constexpr (KIND == kLinearFwd) {
      if (p.bias) {
        uint32_t b[16];
        load32(static_cast<const T*>(p.bias) + col, n,
               (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0, b);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 f = unpack2<T>(b[j]);
          v[2 * j] += f.x;
          v[2 * j + 1] += f.y;
        }
      }
      if (p.Z) store32(static_cast<T*>(p.Z) + row * p.ldz + col, n, vec, v);
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = act_of<decltype(tag)::act>(v[i]);
      });
      if (have) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float2 f = unpack2<T>(other[j]);
          v[2 * j] += f.x;
          v[2 * j + 1] += f.y;
        }
      }
      store32(static_cast<T*>(p.D) + row * p.ldd + col, n, vec, v);
    } else if constexpr (KIND == kLinearDgrad) {
      if (z_ok) {
        with_act(p.act, [&](auto tag) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 f = unpack2<T>(other[j]);
            v[2 * j] *= act_slope<decltype(tag)::act>(f.x);
            v[2 * j + 1] *= act_slope<decltype(tag)::act>(f.y);
          }
        });
      } else {  // a row id outside z: recorded, and a zero row
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
      store32(static_cast<T*>(p.D) + row * p.ldd + col, n, vec, v);
    } else {
      float* d = static_cast<float*>(p.D) + row * p.ldd + col;
      if (vec && n >= 32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float4 o = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          if (p.add) {  // each element once: the same bits as a load, an addition and a store
            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(d + 4 * j),
                         "f"(o.x), "f"(o.y), "f"(o.z), "f"(o.w)
                         : "memory");
          } else {
            reinterpret_cast<float4*>(d)[j] = o;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < n) d[i] = p.add ? d[i] + v[i] : v[i];
      }
    }
  }
}

// Persistent: producer warp 0 (TMA into a ring of stages), issuer warp 1 (tcgen05.mma into one of
// two accumulators), eight epilogue warps (two to a quadrant of the TMEM lanes, each with half of a
// tile's columns).  With CG = 2 both CTAs' copies count on the leader's barriers, and the leader
// issues the products of the pair.  Every wait is bounded.
template <int CG, int BN, typename T, int KIND>
__global__ void __launch_bounds__(kLinearThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const LinearArgs p) {
  using S = TileShape<CG, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE_BYTES);
  uint64_t* empty = full + S::STAGES;
  uint64_t* tfull = empty + S::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const uint32_t crank = CG == 2 ? cluster_ctarank() : 0;
  const bool leader = crank == 0;
  const int group = blockIdx.x / CG, groups = gridDim.x / CG;
  const int num_m = (p.M + CG * S::BM - 1) / (CG * S::BM);
  const int num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int num_kb = (p.K + S::BK - 1) / S::BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&tfull[a]), 1);
      mbar_init(smem_u32(&tempty[a]), 8 * CG);  // the epilogue warps of all CTAs of the tile
    }
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(smem_u32(tmem_slot), S::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), S::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t smem_base = smem_u32(smem);

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; tile < num_tiles && ok; tile += groups) {
        int tm, tn;
        tile_at(tile, num_m, num_n, tm, tn);
        const int m0 = (tm * CG + static_cast<int>(crank)) * S::BM;
        const int n0 = tn * BN + static_cast<int>(crank) * S::B_ROWS;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.err,
                         kErrWaitProducer)) {
            ok = false;
            break;
          }
          uint32_t bar = smem_u32(&full[stage]);
          if (leader) mbar_arrive_expect_tx(bar, CG * S::STAGE_BYTES);
          if (CG == 2) bar = mapa_shared(bar, 0);
          const auto load = [&](uint32_t dst, const CUtensorMap* m, int x, int y) {
            if constexpr (CG == 2) tma_load_2d_pair(dst, m, bar, x, y);
            else tma_load_2d(dst, m, bar, x, y);
          };
          const uint32_t sa = smem_base + stage * S::STAGE_BYTES;
          const uint32_t sb = sa + S::A_BYTES;
          const int k0 = kb * S::BK;
          if (!p.a_mn) {
            load(sa, &tmA, k0, m0);
          } else {
            load(sa, &tmA, m0, k0);
            load(sa + 8192, &tmA, m0 + 64, k0);
          }
          if (!p.b_mn) {
            load(sb, &tmB, k0, n0);
          } else {
#pragma unroll
            for (int c = 0; c < S::B_ROWS / 64; ++c) load(sb + c * 8192, &tmB, n0 + c * 64, k0);
          }
          ++issued;
          if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // a copy may not land after the CTA has given up and left (the leader's barriers count both
      // CTAs' copies)
      if (!ok && leader) tma_drain_ring(full, S::STAGES, issued);
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // K-major: 16 columns of k are 32 bytes on; MN-major: 16 rows of k are 2048 bytes on
      const uint32_t a_step = p.a_mn ? 2048 : 32, a_lbo = p.a_mn ? 8192 : 16;
      const uint32_t b_step = p.b_mn ? 2048 : 32, b_lbo = p.b_mn ? 8192 : 16;
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; tile < num_tiles && ok; tile += groups, ++it) {
        const int acc = it & 1;
        if (!mbar_wait(smem_u32(&tempty[acc]), ((it >> 1) & 1) ^ 1u, abort_flag, p.err,
                       kErrWaitMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(smem_u32(&full[stage]), phase, abort_flag, p.err, kErrWaitMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_base + stage * S::STAGE_BYTES;
          const uint32_t sb = sa + S::A_BYTES;
#pragma unroll
          for (int k = 0; k < S::BK / 16; ++k) {
            const uint64_t ad = sdesc_sw128(sa + k * a_step, a_lbo, 1024);
            const uint64_t bd = sdesc_sw128(sb + k * b_step, b_lbo, 1024);
            const uint32_t accumulate = kb != 0 || k != 0;
            if constexpr (CG == 2) umma_bf16_ss_pair(d, ad, bd, p.idesc, accumulate);
            else umma_bf16_ss(d, ad, bd, p.idesc, accumulate);
          }
          if constexpr (CG == 2) umma_commit_pair_mc(smem_u32(&empty[stage]), 0x3);
          else umma_commit(smem_u32(&empty[stage]));
          if (++stage == S::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if constexpr (CG == 2) umma_commit_pair_mc(smem_u32(&tfull[acc]), 0x3);
        else umma_commit(smem_u32(&tfull[acc]));
      }
      // all products are done before shared memory or TMEM is given up
      if constexpr (CG == 2) umma_commit_pair(smem_u32(drain));
      else umma_commit(smem_u32(drain));
      volatile int never = 0;
      mbar_wait(smem_u32(drain), 0, &never, nullptr, 0);
    }
  } else {
    const int q = warp & 3;  // the quadrant of TMEM lanes that this warp may read
    const int half = (warp - 2) >> 2;
    int it = 0;
    for (int tile = group; tile < num_tiles; tile += groups, ++it) {
      int tm, tn;
      tile_at(tile, num_m, num_n, tm, tn);
      const int acc = it & 1;
      if (!mbar_wait(smem_u32(&tfull[acc]), (it >> 1) & 1, abort_flag, p.err, kErrWaitEpilogue))
        break;
      tc_fence_after();
      const int row = (tm * CG + static_cast<int>(crank)) * S::BM + q * 32 + lane;
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN;
      epilogue_rows<T, KIND>(p, taddr, row, tn * BN, half * 32, BN, 64);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
        else mbar_arrive(smem_u32(&tempty[acc]));
      }
    }
  }

  tc_fence_before();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, S::TMEM_COLS);
    else tmem_dealloc(tmem_base, S::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- layout and column sums
// dst [rows, ld_dst] = src [rows, cols] (2-byte elements)
__global__ void __launch_bounds__(256) relayout_kernel(const unsigned short* __restrict__ src,
                                                       long long ld, int cols,
                                                       unsigned short* __restrict__ dst,
                                                       long long ld_dst, int rows) {
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    const unsigned short* s = src + r * ld;
    unsigned short* d = dst + r * ld_dst;
    for (int c = blockIdx.x * 256 + threadIdx.x; c < cols; c += gridDim.x * 256) d[c] = s[c];
  }
}

// sum[c] (+)= the sum of column c of dy [rows, cols], in a fixed order.  A cluster of eight blocks
// has a slab of columns, each thread W of them in every 256th (W = 8) row; the first block adds the
// eight blocks' sums.  Bound by memory.
template <typename T, int W>
__global__ void __launch_bounds__(256) column_sum_kernel(const T* __restrict__ dy, long long ld,
                                                         int rows, int cols,
                                                         float* __restrict__ sum, int add) {
  constexpr int LANES = W == 8 ? 8 : 32;      // threads across a slab
  constexpr int GROUPS = 256 / LANES;         // rows of a block at a time
  constexpr int SLAB = LANES * W;
  __shared__ float part[GROUPS][SLAB + 1];
  __shared__ float total[SLAB];
  const uint32_t rank = cluster_ctarank();
  const int lane = threadIdx.x % LANES, rg = threadIdx.x / LANES;
  const int slab = blockIdx.x / 8 * SLAB;
  const int c = slab + lane * W;
  float s[W] = {};
  if (c < cols) {
#pragma unroll 4
    for (int r = static_cast<int>(rank) * GROUPS + rg; r < rows; r += 8 * GROUPS) {
      float f[W];
      load_f32<T, W>(dy + r * ld + c, f);
#pragma unroll
      for (int i = 0; i < W; ++i) s[i] += f[i];
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) part[rg][lane * W + i] = s[i];
  __syncthreads();
  if (threadIdx.x < SLAB) {
    float t = 0.f;
    for (int g = 0; g < GROUPS; ++g) t += part[g][threadIdx.x];
    total[threadIdx.x] = t;
  }
  cluster_sync();
  const int col = slab + threadIdx.x;
  if (rank == 0 && threadIdx.x < SLAB && col < cols) {
    float t = 0.f;
    for (int b = 0; b < 8; ++b) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];"
                   : "=f"(v)
                   : "r"(mapa_shared(smem_u32(&total[threadIdx.x]), b))
                   : "memory");
      t += v;
    }
    sum[col] = (add ? sum[col] : 0.f) + t;
  }
  cluster_sync();  // no block leaves while its sums are read
}

}  // namespace cfb

using namespace cfb;

namespace {

constexpr int kMaxDevices = 64;
int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev < kMaxDevices ? dev : -1;
}

template <int CG, int BN, typename T, int KIND>
int launch_linear(const CUtensorMap& ta, const CUtensorMap& tb, const LinearArgs& a,
                  cudaStream_t st) {
  using S = TileShape<CG, BN>;
  auto* kernel = linear_kernel<CG, BN, T, KIND>;
  static bool allowed[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0) return -3;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_BYTES) !=
        cudaSuccess) {
      cudaGetLastError();
      return -3;
    }
    allowed[dev] = true;
  }
  const long long tiles = ((a.M + CG * 128LL - 1) / (CG * 128)) * ((a.N + BN - 1LL) / BN);
  const int groups = static_cast<int>(tiles < 148 / CG ? tiles : 148 / CG);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * CG);
  cfg.blockDim = dim3(kLinearThreads);
  cfg.dynamicSmemBytes = S::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CG;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, ta, tb, a) != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  ++cfb_row_launches();
  return 0;
}

// The tile whose estimated time is least: waves of tiles over the SMs times the time of a tile, in
// units of a 128 x 256 share at full rate.
struct LinearPlan {
  int cg, bn;
};
LinearPlan plan_linear(long long M, long long N) {
  const auto waves = [](long long tiles, int slots) { return (tiles + slots - 1) / slots; };
  const double pair = 0.9 * waves(((M + 255) / 256) * ((N + 255) / 256), 74);
  const double s128 = 0.66 * waves(((M + 127) / 128) * ((N + 127) / 128), 148);
  const double s64 = 0.45 * waves(((M + 127) / 128) * ((N + 63) / 64), 148);
  if (pair <= s128 && pair <= s64) return {2, 256};
  return s128 <= s64 ? LinearPlan{1, 128} : LinearPlan{1, 64};
}

template <typename T, int KIND>
int launch_plan(const LinearPlan& pl, const CUtensorMap& ta, const CUtensorMap& tb,
                const LinearArgs& a, cudaStream_t st) {
  if (pl.cg == 2) return launch_linear<2, 256, T, KIND>(ta, tb, a, st);
  if (pl.bn == 128) return launch_linear<1, 128, T, KIND>(ta, tb, a, st);
  return launch_linear<1, 64, T, KIND>(ta, tb, a, st);
}

// An operand in memory: rows and columns, and whether TMA can read it as it is.
struct Operand {
  const void* p;
  long long ld;
  int rows, cols;
  Operand(const void* p, long long ld, int rows, int cols)  // (a single row's stride says nothing)
      : p(p), ld(rows == 1 ? (cols + 7LL) / 8 * 8 : ld), rows(rows), cols(cols) {}
  bool direct() const { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }
  long long packed_ld() const { return (cols + 7LL) / 8 * 8; }
  long long packed_bytes() const {
    return direct() ? 0 : (packed_ld() * rows * 2 + 255) / 256 * 256;
  }
};
Operand operand_a(const CfbLinear& p) {
  return p.kind == kLinearWgrad ? Operand{p.A, p.lda, p.K, p.M} : Operand{p.A, p.lda, p.M, p.K};
}
Operand operand_b(const CfbLinear& p) {
  return p.kind == kLinearFwd ? Operand{p.B, p.ldb, p.N, p.K} : Operand{p.B, p.ldb, p.K, p.N};
}
// Lays an operand out in the workspace where TMA cannot read it, and moves `work` on.
int lay_out(Operand& o, uint8_t*& work, cudaStream_t st) {
  if (o.direct()) return 0;
  const long long bytes = o.packed_bytes();
  unsigned short* dst = reinterpret_cast<unsigned short*>(work);
  const int x = (o.cols + 1023) / 1024;
  relayout_kernel<<<dim3(x < 64 ? x : 64, o.rows < 65535 ? o.rows : 65535), 256, 0, st>>>(
      static_cast<const unsigned short*>(o.p), o.ld, o.cols, dst, o.packed_ld(), o.rows);
  work += bytes;
  o.p = dst;
  o.ld = o.packed_ld();
  return launch_status();
}

template <typename T>
int launch_column_sum(const CfbLinear& p, cudaStream_t st) {
  const bool wide = p.M % 8 == 0 && rows_of_8(p.A, p.lda, p.type);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(8 * ((p.M + (wide ? 63 : 31)) / (wide ? 64 : 32)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 8;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const T* dy = static_cast<const T*>(p.A);
  const long long ld = p.lda;
  const int rows = p.K, cols = p.M, add = p.add;
  const cudaError_t e =
      wide ? cudaLaunchKernelEx(&cfg, column_sum_kernel<T, 8>, dy, ld, rows, cols, p.dbias, add)
           : cudaLaunchKernelEx(&cfg, column_sum_kernel<T, 1>, dy, ld, rows, cols, p.dbias, add);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  ++cfb_row_launches();
  return 0;
}

}  // namespace

long long cfb_linear_workspace(const CfbLinear* p) {
  return operand_a(*p).packed_bytes() + operand_b(*p).packed_bytes();
}

int cfb_linear(const CfbLinear* p, cudaStream_t st) {
  if (p->type != kBF16 && p->type != kF16) return -12;
  if (p->M == 0 || p->N == 0) {
    if (p->kind != kLinearWgrad || p->M == 0 || !p->dbias) return 0;
  }
  if (p->K == 0) {
    if (p->kind != kLinearWgrad) return -10;
    if (p->add) return 0;  // no rows: nothing to add
    if (p->dbias && cudaMemsetAsync(p->dbias, 0, 4ll * p->M, st) != cudaSuccess) return -3;
    if (p->N > 0 && cudaMemset2DAsync(p->D, 4ll * p->ldd, 0, 4ll * p->N, p->M, st) != cudaSuccess)
      return -3;
    return 0;
  }
  if (p->kind == kLinearWgrad && p->dbias) {
    const int rc = p->type == kBF16 ? launch_column_sum<__nv_bfloat16>(*p, st)
                                    : launch_column_sum<__half>(*p, st);
    if (rc || p->N == 0) return rc;
  }
  if (((p->M + 127LL) / 128) * ((p->N + 63LL) / 64) >= (1LL << 31)) return -11;
  Operand oa = operand_a(*p), ob = operand_b(*p);
  uint8_t* work = static_cast<uint8_t*>(p->work);
  int rc = lay_out(oa, work, st);
  if (rc) return rc;
  rc = lay_out(ob, work, st);
  if (rc) return rc;
  const LinearPlan pl = plan_linear(p->M, p->N);
  LinearArgs a = {};
  a.M = p->M;
  a.N = p->N;
  a.K = p->K;
  a.a_mn = p->kind == kLinearWgrad;
  a.b_mn = p->kind != kLinearFwd;
  a.idesc = idesc_bf16_f32(128 * pl.cg, pl.bn, a.a_mn, a.b_mn);
  if (p->type == kF16) a.idesc &= ~((1u << 7) | (1u << 10));  // f16 operands
  CUtensorMap ta, tb;
  rc = a.a_mn ? make_tmap_2d_bf16(&ta, oa.p, oa.rows, oa.cols, oa.ld, 64, 64)
              : make_tmap_2d_bf16(&ta, oa.p, oa.rows, oa.cols, oa.ld, 64, 128);
  if (rc) return rc * 100 - 1;
  rc = a.b_mn ? make_tmap_2d_bf16(&tb, ob.p, ob.rows, ob.cols, ob.ld, 64, 64)
              : make_tmap_2d_bf16(&tb, ob.p, ob.rows, ob.cols, ob.ld, 64, pl.bn / pl.cg);
  if (rc) return rc * 100 - 2;
  a.D = p->D;
  a.ldd = p->ldd;
  a.bias = p->bias;
  a.R = p->R;
  a.ldr = p->ldr;
  a.Z = p->Z;
  a.ldz = p->ldz;
  a.z_rows = p->z_rows;
  a.n_z = p->n_z;
  a.act = p->act;
  a.add = p->add;
  a.err = p->err;
  const int out_type = p->kind == kLinearWgrad ? kF32 : p->type;
  const int out_width = p->kind == kLinearWgrad ? 4 : 8;
  a.vec = rows_of(out_width, p->D, p->ldd, out_type) && rows_of_8(p->R, p->ldr, p->type) &&
          rows_of_8(p->Z, p->ldz, p->type);
#define CFB_LINEAR(T)                                                                       \
  (p->kind == kLinearFwd     ? launch_plan<T, kLinearFwd>(pl, ta, tb, a, st)               \
   : p->kind == kLinearDgrad ? launch_plan<T, kLinearDgrad>(pl, ta, tb, a, st)             \
                             : launch_plan<T, kLinearWgrad>(pl, ta, tb, a, st))
  return p->type == kBF16 ? CFB_LINEAR(__nv_bfloat16) : CFB_LINEAR(__half);
#undef CFB_LINEAR
}

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
// Bound by the tensor cores at a training step's sizes, by latency at small ones.  16384 x 2048 x 5632
// bf16 (228 us at the measured rate of library products): 254 us without an activation, 277 with gelu
// and z, in bursts of eight calls; the clock falls from 1.9 to 1.6 GHz meanwhile, and in a longer loop
// the power limit makes the last 338.  Of 8192 of its rows (114 us): dgrad 152, wgrad 153 and with dbias
// 168, whose sums are a pass of their own (dealt to the epilogue's warps they cost 22 us).
#include "row_types.cuh"

#include <cudaTypedefs.h>

namespace cfb {

int make_tmap_2d_bf16(CUtensorMap* map, const void* ptr, long long rows, long long cols,
                      long long ld, int box_cols, int box_rows);
int make_tmap_3d_bf16(CUtensorMap* map, const void* ptr, long long rows, long long cols,
                      long long ld, int box_rows, int box_chunks);

// ---------------------------------------------------------------- activations
// On pairs of fp32: an epilogue of 128 x 256 elements has to end while the next tile's products run,
// and its arithmetic is most of it.
__device__ __forceinline__ F2 ex2_2(F2 x) {
  const float2 v = halves(x);
  float lo, hi;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(lo) : "f"(v.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(v.y));
  return f2(lo, hi);
}
__device__ __forceinline__ F2 inv_2(F2 x) {
  const float2 v = halves(x);
  float lo, hi;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(lo) : "f"(v.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(hi) : "f"(v.y));
  return f2(lo, hi);
}
template <typename F>
__device__ __forceinline__ F2 each(F2 x, F&& f) {
  const float2 v = halves(x);
  return f2(f(v.x), f(v.y));
}
// 1 / (1 + 2^x), 0 for large x
__device__ __forceinline__ F2 inv_1p_exp2(F2 x) { return inv_2(ex2_2(x) + f2(1.f)); }

constexpr float kLog2e = 1.4426950408889634f;

// The normal distribution's mass beyond a = |z|, and its density times sqrt(2 pi): exp(-a^2 / 2) t P(t)
// with t = 1 / (1 + 0.27 a), where P is a minimax fit of erfcx(a / sqrt 2) / (2 t) of degree six with a
// relative error of 1.2e-6, so that small values are as exact as the others (1 + erf(z / sqrt 2) loses
// them).  a is cut off at 30, far behind the last one whose mass is not zero.
__device__ __forceinline__ F2 normal_tail(F2 z, F2& a, F2& bell) {
  a = each(z, [](float v) { return fminf(fabsf(v), 30.f); });
  const F2 t = inv_2(fma2(f2(0.27f), a, f2(1.f)));
  F2 p = fma2(f2(-0.060966506600379944f), t, f2(0.1590183675289154f));
  p = fma2(p, t, f2(-0.025057457387447357f));
  p = fma2(p, t, f2(0.11830243468284607f));
  p = fma2(p, t, f2(0.09249885380268097f));
  p = fma2(p, t, f2(0.10852396488189697f));
  p = fma2(p, t, f2(0.10767974704504013f));
  bell = ex2_2(z * z * f2(-0.5f * kLog2e));
  return bell * t * p;
}

// gelu by tanh is z / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kGelu1 = -2.f * 0.7978845608028654f * kLog2e;
constexpr float kGelu3 = kGelu1 * 0.044715f;

template <int ACT>
__device__ __forceinline__ F2 act_of(F2 z) {
  if constexpr (ACT == kActRelu) return each(z, [](float v) { return v < 0.f ? 0.f : v; });
  if constexpr (ACT == kActSilu) return z * inv_1p_exp2(z * f2(-kLog2e));
  if constexpr (ACT == kActGelu) {  // z minus the mass above it, or z times the mass below it
    F2 a, bell;
    const F2 tail = normal_tail(z, a, bell);
    return fma2(a * f2(-1.f), tail, each(z, [](float v) { return fmaxf(v, 0.f); }));
  }
  if constexpr (ACT == kActGeluTanh)
    return z * inv_1p_exp2(z * fma2(f2(kGelu3), z * z, f2(kGelu1)));
  return z;
}
template <int ACT>
__device__ __forceinline__ F2 act_slope(F2 z) {
  if constexpr (ACT == kActRelu)
    return each(z, [](float v) { return v > 0.f ? 1.f : v != v ? v : 0.f; });
  if constexpr (ACT == kActSilu) {
    const F2 p = inv_1p_exp2(z * f2(-kLog2e));
    return p * fma2(z, fma2(p, f2(-1.f), f2(1.f)), f2(1.f));
  }
  if constexpr (ACT == kActGelu) {
    F2 a, bell;
    const F2 tail = normal_tail(z, a, bell);
    const float2 v = halves(z), lo = halves(tail), hi = halves(fma2(tail, f2(-1.f), f2(1.f)));
    return fma2(z * f2(0.3989422804014327f), bell,
                f2(v.x < 0.f ? lo.x : hi.x, v.y < 0.f ? lo.y : hi.y));
  }
  if constexpr (ACT == kActGeluTanh) {
    // the second term is zero long before |z| = 30, beyond which z^3 may be infinite
    const F2 c = each(z, [](float v) { return v != v ? v : fminf(fmaxf(v, -30.f), 30.f); });
    const F2 sq = c * c;
    const F2 p = inv_1p_exp2(c * fma2(f2(kGelu3), sq, f2(kGelu1)));
    constexpr float k = 2.f * 0.7978845608028654f;
    const F2 du = fma2(f2(3.f * 0.044715f * k), sq, f2(k));
    return fma2(c * p * fma2(p, f2(-1.f), f2(1.f)), du, p);
  }
  return f2(1.f);
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
  int a_mn, b_mn;   // operands [K, M], [K, N] in memory instead of [M, K], [N, K] (as template
                    // arguments they made the forward slower: 260 us for 254)
  int a_3d, b_3d;   // ... whose tiles one copy brings: {64 columns, k, groups of 64 columns}
  uint32_t idesc;   // instruction descriptor: shape, types and layouts
  int full;         // units below this are whole tiles, the others pieces of the tiles behind them
  int pieces;       // pieces a tile
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
  int vec;           // what the outputs, R and Z allow: kRows32, kRows16 or kRowsAny
  int* err;
};
// Rows on 32 bytes (every lane reads and writes whole sectors of its row), on 16, or anywhere.
enum { kRowsAny = 0, kRows16 = 1, kRows32 = 2 };

// CG CTAs on neighbouring SMs share a tile of CG * 128 rows and BN columns.
template <int CG, int BN>
struct TileShape {
  static constexpr int BM = 128, BK = 64;
  static constexpr int B_ROWS = BN / CG;  // each CTA stages its rows of A and its share of B
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = B_ROWS * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE_BYTES;
  static constexpr int OUT_BYTES = 4096;  // of each epilogue warp: 32 rows on their way out or in
  static constexpr int SMEM_BYTES =
      STAGES * STAGE_BYTES + 8 * OUT_BYTES + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int TMEM_COLS = 2 * BN;
};
// Three groups of four warps: producer, issuer and two idle; eight epilogue warps.  Of the registers
// that the block is launched with (384 x 168 = 64512) the first group gives up what the other two take:
// 128 x 56 + 256 x 224 = 64512.
constexpr int kLinearThreads = 384, kEpilogueWarp = 4;
constexpr int kFewRegisters = 56, kManyRegisters = 224;
// wgrad: the tensor cores' additions lose 1.1e-9 of the result for each further row (8192 rows:
// 9.1e-6; of one sign, twice that), so that their sum ends after 1024 rows and is added to fp32 sums in
// registers.
constexpr int kSegment = 16;  // blocks of 64 rows

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
// The tile and the columns of a unit of work.
template <int BN>
__device__ __forceinline__ void unit_at(const LinearArgs& p, int unit, int num_m, int num_n, int& tm,
                                        int& n0, int& width) {
  int tn, piece = 0;
  width = BN;
  if (unit >= p.full) {
    const int i = unit - p.full;
    piece = i % p.pieces;
    unit = p.full + i / p.pieces;
    width = BN / p.pieces;
  }
  tile_at(unit, num_m, num_n, tm, tn);
  n0 = tn * BN + piece * width;
}

// 16 pairs as words of two elements of T, and back.
template <typename T>
__device__ __forceinline__ void pack16(const F2* v, uint32_t* u) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float2 h = halves(v[j]);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      u[j] = pack_bf16x2(h.x, h.y);
    } else {
      const __half2 w = __floats2half2_rn(h.x, h.y);
      u[j] = *reinterpret_cast<const uint32_t*>(&w);
    }
  }
}
template <typename T>
__device__ __forceinline__ F2 unpack2(uint32_t u) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&u));
  return f2(h.x, h.y);
}

// ---------------------------------------------------------------- 32 rows x 32 columns of a warp
// In the epilogue a lane has a row, which is how TMEM is read, and 64 bytes of it at a time.  Where
// rows start on 32 bytes, it reads and writes them as whole sectors by 256-bit accesses (stores of 16
// bytes fill half sectors: the forward of 16384 x 2048 x 5632 with z took 323 us with them).
// Elsewhere, and at the last columns, chunks pass through shared memory, where they are written by
// rows and read four lanes (or, element by element, all lanes) to a row, or the other way round; not
// everywhere, since the products need the shared memory's bandwidth themselves.  The 16-byte quarters
// of a row are permuted so that neither way has bank conflicts.
using u16 = unsigned short;
__device__ __forceinline__ uint4* quarter(uint8_t* buf, int row, int j) {
  return reinterpret_cast<uint4*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4));
}
__device__ __forceinline__ u16* element(uint8_t* buf, int row, int c) {
  return reinterpret_cast<u16*>(quarter(buf, row, c >> 3)) + (c & 7);
}
__device__ __forceinline__ void put_row(uint8_t* buf, const uint32_t* u) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *quarter(buf, lane_id(), j) = make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
}
__device__ __forceinline__ void get_row(uint8_t* buf, uint32_t* u) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 q = *quarter(buf, lane_id(), j);
    u[4 * j] = q.x;
    u[4 * j + 1] = q.y;
    u[4 * j + 2] = q.z;
    u[4 * j + 3] = q.w;
  }
}
__device__ __forceinline__ void store_sector(void* p, const uint32_t* u) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]),
               "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
__device__ __forceinline__ void load_sector(const void* p, uint32_t* u) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]),
                 "=r"(u[6]), "=r"(u[7])
               : "l"(p));
}
// The lanes' rows of a chunk (16 words each) to rows [0, rows) and columns [0, cols) of dst.
template <typename T>
__device__ __forceinline__ void chunk_out(uint8_t* buf, const uint32_t* u, T* dst, long long ld,
                                          int rows, int cols, int vec) {
  const int lane = lane_id();
  if (vec == kRows32 && cols >= 32) {
    if (lane < rows) {
      store_sector(dst + lane * ld, u);
      store_sector(dst + lane * ld + 16, u + 8);
    }
    return;
  }
  __syncwarp();  // the chunk before has left the buffer
  put_row(buf, u);
  __syncwarp();
  if (vec != kRowsAny && cols >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2);
      const uint4 v = *quarter(buf, r, lane & 3);
      if (r < rows) reinterpret_cast<uint4*>(dst + r * ld)[lane & 3] = v;
    }
  } else if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (r < rows) reinterpret_cast<u16*>(dst + r * ld)[lane] = *element(buf, r, lane);
  }
}
// A chunk on its way in: `at` is where a lane's own row begins (-1: there is none, zeros come).
template <typename T>
__device__ __forceinline__ void chunk_load(const T* src, long long at, int col, int cols, int vec,
                                           uint32_t* pre) {
  const int lane = lane_id();
  if (vec == kRows32 && cols >= 32) {
    if (at >= 0) {
      load_sector(src + at + col, pre);
      load_sector(src + at + col + 16, pre + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) pre[i] = 0;
    }
  } else if (vec != kRowsAny && cols >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = __shfl_sync(0xffffffffu, at, i * 8 + (lane >> 2));
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row >= 0) v = reinterpret_cast<const uint4*>(src + row + col)[lane & 3];
      reinterpret_cast<uint4*>(pre)[i] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      uint32_t w = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long row = __shfl_sync(0xffffffffu, at, 2 * i + h);
        if (row >= 0 && lane < cols)
          w |= static_cast<uint32_t>(reinterpret_cast<const u16*>(src + row + col)[lane]) << (16 * h);
      }
      pre[i] = w;
    }
  }
}
// ... and what chunk_load brought, as the words of the lane's own row.
__device__ __forceinline__ void chunk_in(uint8_t* buf, int cols, int vec, const uint32_t* pre,
                                         uint32_t* own) {
  const int lane = lane_id();
  if (vec == kRows32 && cols >= 32) {
#pragma unroll
    for (int i = 0; i < 16; ++i) own[i] = pre[i];
    return;
  }
  __syncwarp();  // the chunk before has left buf
  if (vec != kRowsAny && cols >= 32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *quarter(buf, i * 8 + (lane >> 2), lane & 3) = reinterpret_cast<const uint4*>(pre)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      *element(buf, 2 * i, lane) = static_cast<u16>(pre[i]);
      *element(buf, 2 * i + 1, lane) = static_cast<u16>(pre[i] >> 16);
    }
  }
  __syncwarp();
  get_row(buf, own);
}
// 32 fp32 values of each lane's row to dst (added, with `add`); not on 32 bytes through all of a
// warp's buffer.
__device__ __forceinline__ void chunk_out_f32(uint8_t* buf, const float* v, float* dst, long long ld,
                                              int rows, int cols, int vec, bool add) {
  const int lane = lane_id();
  if (vec == kRows32 && cols >= 32) {
    float* d = dst + lane * ld;
    if (lane >= rows) return;
    if (add) {  // each element once: the same bits as a load, an addition and a store but below 1.2e-38
#pragma unroll
      for (int j = 0; j < 8; ++j)
        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(d + 4 * j),
                     "f"(v[4 * j]), "f"(v[4 * j + 1]), "f"(v[4 * j + 2]), "f"(v[4 * j + 3])
                     : "memory");
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) store_sector(d + 8 * j, reinterpret_cast<const uint32_t*>(v) + 8 * j);
    }
    return;
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
        make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      if (r >= rows) continue;
      const float o =
          reinterpret_cast<const float*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4))[lane & 3];
      float* d = dst + r * ld + lane;
      *d = add ? *d + o : o;
    }
  }
}

// The rows of a warp (32 from row0, one a lane) of a unit's columns [n0, n0 + width): every second
// chunk of 32 from `first`.  wait() is for the product; before it the first chunk that is read from
// memory is already asked for.
template <typename T, int KIND, typename F>
__device__ __forceinline__ bool epilogue_rows(const LinearArgs& p, uint32_t taddr, int row0, int n0,
                                              int first, int width, uint8_t* buf, F&& wait) {
  const int vec = p.vec;
  const int row = row0 + lane_id();
  const int rows = p.M - row0;  // may be none
  long long at = -1;            // where the lane's row of `other` begins
  const T* other = static_cast<const T*>(KIND == kLinearFwd ? p.R : p.Z);
  if (row < p.M) {
    if constexpr (KIND == kLinearFwd) {
      at = static_cast<long long>(row) * p.ldr;
    } else {
      const long long src = p.z_rows ? p.z_rows[row] : row;
      if (index_in(src, p.n_z, p.err)) at = src * p.ldz;
    }
  }
  const bool reads = other != nullptr;
  uint32_t pre[16];
  if (reads && n0 + first < p.N && first < width)
    chunk_load(other, at, n0 + first, p.N - n0 - first, vec, pre);
  if (!wait()) return false;
#pragma unroll 1
  for (int c = first; c < width; c += 64) {
    const int col = n0 + c;
    if (col >= p.N) break;  // the same for the whole warp
    const int cols = p.N - col;
    uint32_t own[16], r[32];
    CFB_TMEM_LD32(taddr + c, r);
    if (reads) {
      chunk_in(buf, cols, vec, pre, own);
      if (c + 64 < width && col + 64 < p.N) chunk_load(other, at, col + 64, cols - 64, vec, pre);
    }
    tmem_ld_wait();
    F2 v[16];
    uint32_t u[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = f2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
    if constexpr (KIND == kLinearFwd) {
      if (p.bias) {
        const T* b = static_cast<const T*>(p.bias) + col;
        if (cols >= 32 && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            F2 f[4];
            load_f2<T, 8>(b + 8 * j, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = v[4 * j + i] + f[i];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            v[j] = v[j] + f2(2 * j < cols ? to_f32(b[2 * j]) : 0.f,
                             2 * j + 1 < cols ? to_f32(b[2 * j + 1]) : 0.f);
        }
      }
      if (p.Z) {
        pack16<T>(v, u);
        chunk_out(buf + 2048, u, static_cast<T*>(p.Z) + row0 * p.ldz + col, p.ldz, rows, cols, vec);
      }
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = act_of<decltype(tag)::act>(v[j]);
      });
      if (reads) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = v[j] + unpack2<T>(own[j]);
      }
      pack16<T>(v, u);
    } else {
      with_act(p.act, [&](auto tag) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = v[j] * act_slope<decltype(tag)::act>(unpack2<T>(own[j]));
      });
      pack16<T>(v, u);
      if (at < 0) {  // a row id outside z is recorded, and gives a zero row
#pragma unroll
        for (int j = 0; j < 16; ++j) u[j] = 0;
      }
    }
    chunk_out(buf, u, static_cast<T*>(p.D) + row0 * p.ldd + col, p.ldd, rows, cols, vec);
  }
  return true;
}

// mbar_wait for warps that have nothing else to do for microseconds: polls that the hardware holds for
// up to 20 us take no issue slots from the producer and the issuer.
__device__ __forceinline__ bool mbar_wait_idle(uint32_t bar, uint32_t parity, volatile int* abort,
                                               int* err, int code) {
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000)
        : "memory");
    if (ok) return true;
    if (*abort) return false;
    if (globaltimer_ns() - t0 > local_wait_limit_ns(err)) {
      *abort = 1;
      if (err) atomicCAS(err, 0, code);
      return false;
    }
  }
}

// Persistent: producer warp 0 (TMA into a ring of stages), issuer warp 1 (tcgen05.mma into one of
// two accumulators), eight epilogue warps (two to a quadrant of the TMEM lanes, each with half of a
// tile's chunks of columns).  With CG = 2 both CTAs' copies count on the leader's barriers, and the
// leader issues the products of the pair.  The tiles of the last, partly filled wave are cut into
// pieces of fewer columns.  Every wait is bounded.
template <int CG, int BN, typename T, int KIND>
__global__ void __launch_bounds__(kLinearThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmPiece, const LinearArgs p) {
  using S = TileShape<CG, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* out_area = smem + S::STAGES * S::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(out_area + 8 * S::OUT_BYTES);
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
  const int num_units = p.full + (num_m * num_n - p.full) * p.pieces;
  const int num_kb = (p.K + S::BK - 1) / S::BK;
  // blocks of k that one accumulator takes
  const int segment = KIND == kLinearWgrad ? kSegment : num_kb;

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
  after_previous();  // (an operand that was laid out anew)
  if (warp < kEpilogueWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0 && lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = group; unit < num_units && ok; unit += groups) {
        int tm, n0, width;
        unit_at<BN>(p, unit, num_m, num_n, tm, n0, width);
        const int m0 = (tm * CG + static_cast<int>(crank)) * S::BM;
        const int b_rows = width / CG;
        n0 += static_cast<int>(crank) * b_rows;
        const int b_boxes = (b_rows + 63) / 64;  // MN-major
        const int b_bytes = p.b_mn ? b_boxes * 8192 : b_rows * 128;
        const CUtensorMap* map_b = width == BN ? &tmB : &tmPiece;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.err,
                         kErrWaitProducer)) {
            ok = false;
            break;
          }
          uint32_t bar = smem_u32(&full[stage]);
          if (leader) mbar_arrive_expect_tx(bar, CG * (S::A_BYTES + b_bytes));
          if (CG == 2) bar = mapa_shared(bar, 0);
          const auto load = [&](uint32_t dst, const CUtensorMap* m, int x, int y) {
            if constexpr (CG == 2) tma_load_2d_pair(dst, m, bar, x, y);
            else tma_load_2d(dst, m, bar, x, y);
          };
          const uint32_t sa = smem_base + stage * S::STAGE_BYTES;
          const uint32_t sb = sa + S::A_BYTES;
          const int k0 = kb * S::BK;
          const auto load_3d = [&](uint32_t dst, const CUtensorMap* m, int chunk, int y) {
            if constexpr (CG == 2) tma_load_3d_pair(dst, m, bar, 0, y, chunk);
            else tma_load_3d(dst, m, bar, 0, y, chunk);
          };
          if (!p.a_mn) {
            load(sa, &tmA, k0, m0);
          } else if (p.a_3d) {
            load_3d(sa, &tmA, m0 / 64, k0);
          } else {
            load(sa, &tmA, m0, k0);
            load(sa + 8192, &tmA, m0 + 64, k0);
          }
          if (!p.b_mn) {
            load(sb, map_b, k0, n0);
          } else if (p.b_3d && width == BN) {
            load_3d(sb, &tmB, n0 / 64, k0);
          } else {
            load(sb, map_b, n0, k0);
            if (b_boxes == 2) load(sb + 8192, map_b, n0 + 64, k0);
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
    if (warp == 1 && lane == 0 && leader) {
      // K-major: 16 columns of k are 32 bytes on; MN-major: 16 rows of k are 2048 bytes on
      const uint32_t a_step = p.a_mn ? 2048 : 32, a_lbo = p.a_mn ? 8192 : 16;
      const uint32_t b_step = p.b_mn ? 2048 : 32, b_lbo = p.b_mn ? 8192 : 16;
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = group; unit < num_units && ok; unit += groups) {
        int tm, n0, width;
        unit_at<BN>(p, unit, num_m, num_n, tm, n0, width);
        const uint32_t idesc = (p.idesc & ~(0x3fu << 17)) | (static_cast<uint32_t>(width >> 3) << 17);
        for (int k_seg = 0; k_seg < num_kb && ok; k_seg += segment, ++it) {
          const int k_end = min(num_kb, k_seg + segment);
          const int acc = it & 1;
          if (!mbar_wait(smem_u32(&tempty[acc]), ((it >> 1) & 1) ^ 1u, abort_flag, p.err,
                         kErrWaitMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + acc * BN;
          for (int kb = k_seg; kb < k_end; ++kb) {
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
              const uint32_t accumulate = kb != k_seg || k != 0;
              if constexpr (CG == 2) umma_bf16_ss_pair(d, ad, bd, idesc, accumulate);
              else umma_bf16_ss(d, ad, bd, idesc, accumulate);
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
      }
      // all products are done before shared memory or TMEM is given up
      if constexpr (CG == 2) umma_commit_pair(smem_u32(drain));
      else umma_commit(smem_u32(drain));
      volatile int never = 0;
      mbar_wait(smem_u32(drain), 0, &never, nullptr, 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int q = warp & 3;  // the quadrant of TMEM lanes that this warp may read
    const int half = (warp - kEpilogueWarp) >> 2;
    uint8_t* buf = out_area + (warp - kEpilogueWarp) * S::OUT_BYTES;
    int it = 0;
    bool ok = true;
    const auto wait = [&] {
      ok = mbar_wait_idle(smem_u32(&tfull[it & 1]), (it >> 1) & 1, abort_flag, p.err, kErrWaitEpilogue);
      tc_fence_after();
      return ok;
    };
    const auto release = [&] {  // the accumulator may be written again
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        const uint32_t bar = smem_u32(&tempty[it & 1]);
        if constexpr (CG == 2) mbar_arrive_cluster(mapa_shared(bar, 0));
        else mbar_arrive(bar);
      }
      ++it;
    };
    for (int unit = group; unit < num_units && ok; unit += groups) {
      int tm, n0, width;
      unit_at<BN>(p, unit, num_m, num_n, tm, n0, width);
      const int m0 = (tm * CG + static_cast<int>(crank)) * S::BM;
      const int row0 = m0 + q * 32;
      const auto taddr = [&] {
        return tmem_base + (static_cast<uint32_t>(q * 32) << 16) + (it & 1) * BN;
      };
      if constexpr (KIND != kLinearWgrad) {
        if (!epilogue_rows<T, KIND>(p, taddr(), row0, n0, half * 32, width, buf, wait)) break;
        release();
      } else {
        constexpr int NCH = BN / 64;
        float v[NCH][32];
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) v[i][j] = 0.f;
        for (int k_seg = 0; k_seg < num_kb; k_seg += kSegment) {
          if (!wait()) break;
#pragma unroll
          for (int i = 0; i < NCH; ++i) {
            if (half * 32 + 64 * i >= width) continue;
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              uint32_t r[16];
              CFB_TMEM_LD16(taddr() + half * 32 + 64 * i + h, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[i][h + j] += __uint_as_float(r[j]);
            }
          }
          release();
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
          const int col = n0 + half * 32 + 64 * i;
          if (half * 32 + 64 * i >= width || col >= p.N) continue;
          chunk_out_f32(buf, v[i], static_cast<float*>(p.D) + row0 * p.ldd + col, p.ldd, p.M - row0,
                        p.N - col, p.vec, p.add != 0);
        }
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

// ---------------------------------------------------------------- few tiles
// Issued by lane 0 through a predicate inside, in code that the whole warp runs: the addresses and
// descriptors are then the warp's.  In a branch of lane 0, where they are moved to uniform registers for
// every instruction, a block of four products took 665 clocks, 513 so.  (The kernel of many tiles, whose
// products take as long, gained nothing: 262 us for 254.)
__device__ __forceinline__ void mma_lane0(int lane, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.s32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lane)
      : "memory");
}
// Arrives on `bar` when the products issued before are done.
__device__ __forceinline__ void commit_lane0(int lane, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.eq.s32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(lane)
      : "memory");
}

// One tile of 128 x 128 to a cluster of up to eight CTAs, each with a part of k: an SM takes in about
// 64 bytes of operands a clock, so that a few tiles with a long k leave most of the machine idle (16 x
// 8192 by 2048 x 8192: 45 us with a CTA pair for each 256 columns, 15 so).  Every CTA puts its sums into its
// shared memory; behind a cluster barrier each finishes 128 / splits rows, adding the parts in order
// (the same bits on every run), with accesses to global memory along the rows.
//
// Of rows of A and B that do not exist only the ones up to a multiple of eight are copied; what the
// products make of the rest of a stage is never read.
struct SplitShape {
  static constexpr int BM = 128, BN = 128, BK = 64;
  static constexpr int A_BYTES = BM * BK * 2, STAGE_BYTES = A_BYTES + BN * BK * 2;
  static constexpr int STAGES = 6;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/;
  static constexpr int ROW = BN + 4;  // floats between rows of the sums
};
constexpr int kSplitThreads = 320;  // producer, issuer, eight epilogue warps

template <typename T, int KIND>
__global__ void __launch_bounds__(kSplitThreads, 1)
    linear_split_kernel(const __grid_constant__ CUtensorMap tmA,
                        const __grid_constant__ CUtensorMap tmB, const LinearArgs p, int splits,
                        int a_rows, int b_rows) {
  using S = SplitShape;
  constexpr bool A_MN = KIND == kLinearWgrad, B_MN = KIND != kLinearFwd;
  if (KIND == kLinearWgrad) let_next_start();  // the column sums
  // wgrad: four accumulators, of which each takes 1024 rows at a time (see kSegment), while the epilogue
  // adds the others' to its registers
  constexpr int kAccumulators = KIND == kLinearWgrad ? 4 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * S::STAGE_BYTES);
  uint64_t* empty = full + S::STAGES;
  uint64_t* done = empty + S::STAGES;
  uint64_t* acc_full = done + 1;
  uint64_t* acc_empty = acc_full + kAccumulators;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kAccumulators);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = blockIdx.x / splits;
  const int num_n = (p.N + S::BN - 1) / S::BN;
  const int m0 = tile / num_n * S::BM, n0 = tile % num_n * S::BN;
  const int num_kb = (p.K + S::BK - 1) / S::BK;
  const int kb0 = static_cast<int>(static_cast<long long>(rank) * num_kb / splits);
  const int kb1 = static_cast<int>(static_cast<long long>(rank + 1) * num_kb / splits);
  // segments of k, each with an accumulator for as long as it takes
  const int segments = KIND == kLinearWgrad ? (kb1 - kb0 + kSegment - 1) / kSegment : 1;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bytes = (A_MN ? 2 * 8192 : a_rows * 128) + (B_MN ? 2 * 8192 : b_rows * 128);
  const auto fill = [&](int kb) {  // the copies of block kb0 + kb
    const int stage = kb % S::STAGES, k0 = (kb0 + kb) * S::BK;
    const uint32_t bar = smem_u32(&full[stage]);
    const uint32_t sa = smem_base + stage * S::STAGE_BYTES, sb = sa + S::A_BYTES;
    mbar_arrive_expect_tx(bar, bytes);
    if constexpr (A_MN) {
      tma_load_2d(sa, &tmA, bar, m0, k0);
      tma_load_2d(sa + 8192, &tmA, bar, m0 + 64, k0);
    } else {
      tma_load_2d(sa, &tmA, bar, k0, m0);
    }
    if constexpr (B_MN) {
      tma_load_2d(sb, &tmB, bar, n0, k0);
      tma_load_2d(sb + 8192, &tmB, bar, n0 + 64, k0);
    } else {
      tma_load_2d(sb, &tmB, bar, k0, n0);
    }
  };

  const int blocks = kb1 - kb0, ahead = min(blocks, S::STAGES);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(done), 1);
    *abort_flag = 0;
    fence_mbar_init();
    after_previous();  // (an operand that was laid out anew)
    for (int kb = 0; kb < ahead; ++kb) fill(kb);
  }
  if (threadIdx.x == 64) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (KIND == kLinearWgrad && warp == 3 && lane < kAccumulators) {
    mbar_init(smem_u32(&acc_full[lane]), 1);
    mbar_init(smem_u32(&acc_empty[lane]), 8);  // the epilogue warps
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), S::BN * kAccumulators);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  after_previous();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int kb = ahead;
      for (; kb < blocks; ++kb) {
        ok = mbar_wait(smem_u32(&empty[kb % S::STAGES]), ((kb / S::STAGES) & 1) ^ 1, abort_flag,
                       p.err, kErrWaitProducer);
        if (!ok) break;
        fill(kb);
      }
      if (!ok) tma_drain_ring(full, S::STAGES, kb);
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t a_step = A_MN ? 2048 : 32, a_lbo = A_MN ? 8192 : 16;
    constexpr uint32_t b_step = B_MN ? 2048 : 32, b_lbo = B_MN ? 8192 : 16;
    int stage = 0, kb = 0;
    uint32_t phase = 0;
    bool ready = false, ok = true;
    for (int segment = 0; kb < blocks && ok; ++segment) {
      const int accumulator = segment % kAccumulators;
      if (KIND == kLinearWgrad && segment >= kAccumulators &&
          !mbar_wait(smem_u32(&acc_empty[accumulator]), (segment / kAccumulators & 1) ^ 1, abort_flag, p.err,
                     kErrWaitMma))
        break;
      const uint32_t d = tmem_base + accumulator * S::BN;
      const int end = KIND == kLinearWgrad ? min(blocks, kb + kSegment) : blocks;
      for (bool first = true; kb < end; ++kb, first = false) {
        if (!ready && !mbar_wait(smem_u32(&full[stage]), phase, abort_flag, p.err, kErrWaitMma)) {
          ok = false;
          break;
        }
        __syncwarp();
        tc_fence_after();
        const uint32_t sa = smem_base + stage * S::STAGE_BYTES, sb = sa + S::A_BYTES;
#pragma unroll
        for (int k = 0; k < S::BK / 16; ++k)
          mma_lane0(lane, d, sdesc_sw128(sa + k * a_step, a_lbo, 1024),
                    sdesc_sw128(sb + k * b_step, b_lbo, 1024), p.idesc, !first || k != 0);
        const uint32_t freed = smem_u32(&empty[stage]);
        if (++stage == S::STAGES) {
          stage = 0;
          phase ^= 1;
        }
        ready = kb + 1 < blocks && mbar_try_wait(smem_u32(&full[stage]), phase);
        commit_lane0(lane, freed);
      }
      if (KIND == kLinearWgrad && ok && kb < blocks) commit_lane0(lane, smem_u32(&acc_full[accumulator]));
    }
    commit_lane0(lane, smem_u32(done));
    __syncwarp();
  }
  // What the first turn of the epilogue reads beside the products is on its way while they are formed.
  constexpr int U = 4;  // rows of a warp's turn (eight: 16 x 8192 x 2048 15.7 us for 15.0; two: dgrad slower)
  const int rows = min(S::BM, p.M - m0);
  const bool vec = p.vec != kRowsAny && (n0 + S::BN <= p.N || p.N % 4 == 0);
  const int step = vec ? 1 : 32;  // between a lane's columns (see below)
  const int c = vec ? lane * 4 : lane, col = n0 + c, n = p.N - col;
  const auto get = [&](const auto* from, float* f) {
    using E = typename std::remove_const<typename std::remove_pointer<decltype(from)>::type>::type;
    if (vec) {
      load_f32<E, 4>(from, f);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = 32 * i < n ? to_f32(from[32 * i]) : 0.f;
    }
  };
  const bool reads = KIND == kLinearFwd ? p.R != nullptr : KIND == kLinearDgrad || p.add;
  const auto beside = [&](int r0, float (*g)[4], bool* known) {
    long long src[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + 8 * u * splits;
      src[u] = m0 + r;
      known[u] = r < rows && n > 0;
      if (KIND == kLinearDgrad && known[u] && p.z_rows) src[u] = p.z_rows[src[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (a row id outside z: recorded, and a zero row)
      if (KIND == kLinearDgrad && known[u]) known[u] = index_in(src[u], p.n_z, p.err);
      g[u][0] = g[u][1] = g[u][2] = g[u][3] = 0.f;
      if (!known[u]) continue;
      if constexpr (KIND == kLinearFwd) get(static_cast<const T*>(p.R) + src[u] * p.ldr + col, g[u]);
      else if constexpr (KIND == kLinearDgrad) get(static_cast<const T*>(p.Z) + src[u] * p.ldz + col, g[u]);
      else get(static_cast<const float*>(p.D) + src[u] * p.ldd + col, g[u]);
    }
  };
  const int first = rank + (warp - 2) * splits;  // the warp's first row
  float g[U][4], bias[4] = {0.f, 0.f, 0.f, 0.f};
  bool known[U];
  if (warp >= 2 && reads) beside(first, g, known);
  if (warp >= 2 && KIND == kLinearFwd && p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i * step < n) bias[i] = to_f32(static_cast<const T*>(p.bias)[col + i * step]);
  }
  const int q = warp & 3, c0 = (warp - 2) / 4 * 64;  // (of the epilogue warps)
  const uint32_t from = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + c0;
  constexpr int kHeld = KIND == kLinearWgrad ? 2 : 0;
  float v[kHeld + 1][32];  // wgrad: the sums of the segments before the last
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
#pragma unroll
    for (int i = 0; i < 32; ++i) v[h][i] = 0.f;
  if (KIND == kLinearWgrad && warp >= 2) {
    for (int segment = 0; segment + 1 < segments; ++segment) {
      const int a = segment % kAccumulators;
      if (!mbar_wait_idle(smem_u32(&acc_full[a]), segment / kAccumulators & 1, abort_flag, p.err,
                          kErrWaitEpilogue))
        break;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        uint32_t r[32];
        CFB_TMEM_LD32(from + a * S::BN + h * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[h][i] += __uint_as_float(r[i]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&acc_empty[a]));
    }
  }
  // All products are done (waited for by everyone: the stages become the place of the sums, and TMEM
  // is given up).
  volatile int never = 0;
  const bool ok = mbar_wait_idle(smem_u32(done), 0, &never, p.err, kErrWaitEpilogue) && !*abort_flag;
  tc_fence_after();
  float* sums = reinterpret_cast<float*>(smem);
  if (warp >= 2 && ok) {
    const uint32_t last = from + (segments - 1) % kAccumulators * S::BN;
    uint32_t r[2][32];
    CFB_TMEM_LD32(last, r[0]);
    CFB_TMEM_LD32(last + 32, r[1]);
    tmem_ld_wait();
    float* row = sums + (q * 32 + lane) * S::ROW + c0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h < kHeld) {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[h][i] = __float_as_uint(v[h < kHeld ? h : 0][i] + __uint_as_float(r[h][i]));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<uint4*>(row + h * 32)[i] =
            make_uint4(r[h][4 * i], r[h][4 * i + 1], r[h][4 * i + 2], r[h][4 * i + 3]);
    }
  }
  tc_fence_before();
  if (splits > 1) cluster_sync(); else __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, S::BN * kAccumulators);
  }

  if (warp >= 2 && ok) {
    // The rows are dealt to the CTAs and their warps one by one, four to a turn, whose arithmetic runs
    // together.  A lane has four neighbouring columns, or, where rows do not start on 16 bytes and at
    // the last columns, every 32nd, which keeps the warp's accesses together.
    const auto finish = [&](auto act_tag, auto vec_tag) {
      constexpr int ACT = decltype(act_tag)::act;
      constexpr bool VEC = decltype(vec_tag)::value;
      constexpr int kStep = VEC ? 1 : 32;
      for (int r0 = first; r0 < rows; r0 += 8 * U * splits) {
        if (reads && r0 != first) beside(r0, g, known);
        F2 v[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + 8 * u * splits;
          float f[4] = {0.f, 0.f, 0.f, 0.f};
          if (r < rows && n > 0) {
            const float* mine = sums + r * S::ROW + c;
            if (splits == 1) {
#pragma unroll
              for (int i = 0; i < 4; ++i) f[i] = mine[i * kStep];
            } else {
              for (int s = 0; s < splits; s += 2) {  // (splits is even)
                float q[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t at = mapa_shared(smem_u32(mine), s + h);
                  if constexpr (VEC) {
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(q[h][0]), "=f"(q[h][1]), "=f"(q[h][2]), "=f"(q[h][3])
                                 : "r"(at)
                                 : "memory");
                  } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                      asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                   : "=f"(q[h][i])
                                   : "r"(at + i * kStep * 4)
                                   : "memory");
                  }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = f[i] + q[0][i] + q[1][i];
              }
            }
          }
          v[u][0] = f2(f[0], f[1]);
          v[u][1] = f2(f[2], f[3]);
        }
        const auto put = [&](auto* base, long long ld) {
          using O = typename std::remove_pointer<decltype(base)>::type;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int r = r0 + 8 * u * splits;
            if (r >= rows || n <= 0) continue;
            const float2 a = halves(v[u][0]), b = halves(v[u][1]);
            const float f[4] = {a.x, a.y, b.x, b.y};
            O* to = base + static_cast<long long>(m0 + r) * ld + col;
            if constexpr (VEC) store_f32<O, 4>(to, f);
            else
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (i * kStep < n) to[i * kStep] = from_f32<O>(f[i]);
          }
        };
        if constexpr (KIND == kLinearFwd) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            v[u][0] = v[u][0] + f2(bias[0], bias[1]);
            v[u][1] = v[u][1] + f2(bias[2], bias[3]);
          }
          if (p.Z) put(static_cast<T*>(p.Z), p.ldz);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if constexpr (KIND == kLinearDgrad) {
            v[u][0] = known[u] ? v[u][0] * act_slope<ACT>(f2(g[u][0], g[u][1])) : f2(0.f);
            v[u][1] = known[u] ? v[u][1] * act_slope<ACT>(f2(g[u][2], g[u][3])) : f2(0.f);
          } else {
            v[u][0] = act_of<ACT>(v[u][0]);
            v[u][1] = act_of<ACT>(v[u][1]);
            if (reads) {
              v[u][0] = v[u][0] + f2(g[u][0], g[u][1]);
              v[u][1] = v[u][1] + f2(g[u][2], g[u][3]);
            }
          }
        }
        if constexpr (KIND == kLinearWgrad) put(static_cast<float*>(p.D), p.ldd);
        else put(static_cast<T*>(p.D), p.ldd);
      }
    };
    const auto either = [&](auto act_tag) {
      if (vec) finish(act_tag, std::true_type());
      else finish(act_tag, std::false_type());
    };
    if constexpr (KIND == kLinearWgrad) either(ActTag<kActNone>());
    else with_act(p.act, either);
  }
  if (splits > 1) cluster_sync();  // no CTA leaves while its sums are read
}

// ---------------------------------------------------------------- layout and column sums
// dst [rows, ld_dst] = src [rows, cols] in elements of E (one or two of 2 bytes).
template <typename E>
__global__ void __launch_bounds__(256) relayout_kernel(const E* __restrict__ src, long long ld, int cols,
                                                       E* __restrict__ dst, long long ld_dst, int rows) {
  let_next_start();
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const E* s = src + r * ld;
    E* d = dst + r * ld_dst;
    for (int c0 = threadIdx.x; c0 < cols; c0 += 8 * 256) {
      E v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i * 256 < cols) v[i] = s[c0 + i * 256];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i * 256 < cols) d[c0 + i * 256] = v[i];
    }
  }
}

// sum[c] (+)= the sum of column c of dy [rows, cols], in a fixed order.  A cluster of eight blocks
// has a slab of LANES * W columns, each thread W of them; the first block adds the eight blocks' sums.
// Bound by memory: 8192 x 5632 bf16 in 15 us.  It is launched behind a product of few tiles and may
// start as soon as that has, on the SMs that it leaves idle (16384 rows, 256 x 256: 17.1 us for 20.9);
// but before one of many, which then finds much of dy in the L2 cache (8192 rows, 2048 x 5632: 168 us
// for 180).
template <typename T, int W, int LANES>
__global__ void __launch_bounds__(256) column_sum_kernel(const T* __restrict__ dy, long long ld,
                                                         int rows, int cols,
                                                         float* __restrict__ sum, int add) {
  constexpr int GROUPS = 256 / LANES;  // rows of a block at a time
  constexpr int SLAB = LANES * W;
  __shared__ float part[8][SLAB];  // each warp's sums
  __shared__ float total[SLAB];
  let_next_start();
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
  for (int i = 0; i < W; ++i) {
#pragma unroll
    for (int o = LANES; o < 32; o *= 2) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
    if (lane_id() < LANES) part[warp_id()][lane * W + i] = s[i];
  }
  __syncthreads();
  if (threadIdx.x < SLAB) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += part[w][threadIdx.x];
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
  after_previous();  // (behind a product: what follows the call has to wait for both)
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
int launch_linear(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tp,
                  const LinearArgs& a, bool behind, cudaStream_t st) {
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
  const long long units = a.full + (tiles - a.full) * a.pieces;
  const int groups = static_cast<int>(units < 148 / CG ? units : 148 / CG);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * CG);
  cfg.blockDim = dim3(kLinearThreads);
  cfg.dynamicSmemBytes = S::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (CG > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (behind) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  if (cudaLaunchKernelEx(&cfg, kernel, ta, tb, tp, a) != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  ++cfb_row_launches();
  return 0;
}

// How many clusters of `splits` CTAs of the split kernel run at once: an SM takes one CTA, and a cluster
// does not cross a group of SMs, so fewer than 148 / splits may fit (15 of eight).
int split_clusters(int splits) {
  static int known[4] = {};
  const int at = splits == 8 ? 3 : splits == 4 ? 2 : 1;
  if (known[at] == 0) {
    auto* kernel = linear_split_kernel<__nv_bfloat16, kLinearFwd>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(148 / splits * splits);
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = SplitShape::SMEM_BYTES;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             SplitShape::SMEM_BYTES) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 1;
    }
    known[at] = n;
  }
  return known[at];
}

template <typename T, int KIND>
int launch_split(const CUtensorMap& ta, const CUtensorMap& tb, const LinearArgs& a, int splits,
                 int a_rows, int b_rows, bool behind, cudaStream_t st) {
  auto* kernel = linear_split_kernel<T, KIND>;
  static bool allowed[kMaxDevices] = {};
  const int dev = current_device();
  if (dev < 0) return -3;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             SplitShape::SMEM_BYTES) != cudaSuccess) {
      cudaGetLastError();
      return -3;
    }
    allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(((a.M + 127) / 128) * ((a.N + 127) / 128) * splits);
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = SplitShape::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (splits > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (behind) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  if (cudaLaunchKernelEx(&cfg, kernel, ta, tb, a, splits, a_rows, b_rows) != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  ++cfb_row_launches();
  return 0;
}

// How the output is cut: the tile (a 256 x 256 pair tile, or 128 x bn of one CTA), and the pieces that
// the tiles of the pair's last wave are cut into.
struct LinearPlan {
  int cg, bn;
  long long full;
  int pieces;
  int splits;  // 0, or the parts of k of linear_split_kernel
};
// The least estimated time, in units of a pair tile: waves over the SMs times the time of a tile.  A
// piece of half or a quarter of the columns takes 0.56 or 0.4 of a tile's time (the products of fewer
// columns are bound by shared memory), the tiles of one CTA 0.73 (128 columns, half of the elements of
// a CTA's share of a pair tile) and 0.5 (64 columns).
template <typename F>
LinearPlan plan_linear(long long M, long long N, long long K, F&& clusters) {
  // Where 128 x 128 tiles fill the SMs at most once, each is split over as many CTAs as that leaves,
  // down to four blocks of 64 of k.
  const long long small = ((M + 127) / 128) * ((N + 127) / 128);
  if (small <= 148) {
    int splits = 1;
    while (splits < 8 && small <= clusters(splits * 2) && K >= 2 * splits * 256) splits *= 2;
    return {1, 128, small, 1, splits};
  }
  const auto waves = [](long long units, int slots) { return (units + slots - 1) / slots; };
  const long long pairs = ((M + 255) / 256) * ((N + 255) / 256);
  const long long full = pairs / 74 * 74, rest = pairs - full;
  double best = full / 74 + (rest > 0 ? 1.0 : 0.0);
  LinearPlan plan = {2, 256, pairs, 1, 0};
  const double times[] = {0.56, 0.4};
  for (int i = 0; i < 2 && rest > 0; ++i) {
    const int pieces = 2 << i;
    const double t = full / 74 + times[i] * waves(rest * pieces, 74);
    if (t < best) {
      best = t;
      plan = {2, 256, full, pieces, 0};
    }
  }
  const double singles[] = {0.73, 0.5};
  for (int i = 0; i < 2; ++i) {
    const int bn = 128 >> i;
    const long long tiles = ((M + 127) / 128) * ((N + bn - 1) / bn);
    const double t = singles[i] * waves(tiles, 148);
    if (t < best) {
      best = t;
      plan = {1, bn, tiles, 1, 0};
    }
  }
  return plan;
}

template <typename T, int KIND>
int launch_plan(const LinearPlan& pl, const CUtensorMap& ta, const CUtensorMap& tb,
                const CUtensorMap& tp, const LinearArgs& a, bool behind, cudaStream_t st) {
  if (pl.cg == 2) return launch_linear<2, 256, T, KIND>(ta, tb, tp, a, behind, st);
  if (pl.bn == 128) return launch_linear<1, 128, T, KIND>(ta, tb, tp, a, behind, st);
  return launch_linear<1, 64, T, KIND>(ta, tb, tp, a, behind, st);
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
  const int grid = o.rows < 148 * 16 ? o.rows : 148 * 16;
  if (reinterpret_cast<uintptr_t>(o.p) % 4 == 0 && o.ld % 2 == 0 && o.cols % 2 == 0)
    relayout_kernel<<<grid, 256, 0, st>>>(static_cast<const uint32_t*>(o.p), o.ld / 2, o.cols / 2,
                                          reinterpret_cast<uint32_t*>(work), o.packed_ld() / 2, o.rows);
  else
    relayout_kernel<<<grid, 256, 0, st>>>(static_cast<const unsigned short*>(o.p), o.ld, o.cols,
                                          reinterpret_cast<unsigned short*>(work), o.packed_ld(), o.rows);
  o.p = work;
  work += bytes;
  o.ld = o.packed_ld();
  return launch_status();
}

template <typename T>
int launch_column_sum(const CfbLinear& p, bool behind, cudaStream_t st) {
  const bool wide = p.M % 8 == 0 && rows_of_8(p.A, p.lda, p.type);
  // 64 columns to a slab, or 16 where that would leave SMs without a block
  const int slab = !wide ? 32 : p.M >= 64 * 148 / 8 ? 64 : 16;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(8 * ((p.M + slab - 1) / slab));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 8;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = behind ? 2 : 1;
  const auto launch = [&](auto* kernel) {
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(p.A), p.lda, p.K, p.M, p.dbias, p.add);
  };
  const cudaError_t e = slab == 64   ? launch(column_sum_kernel<T, 8, 8>)
                        : slab == 16 ? launch(column_sum_kernel<T, 8, 2>)
                                     : launch(column_sum_kernel<T, 1, 32>);
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
    const long long pitch = p->M == 1 ? p->N : p->ldd;  // (a single row's stride says nothing)
    if (p->N > 0 && cudaMemset2DAsync(p->D, 4 * pitch, 0, 4ll * p->N, p->M, st) != cudaSuccess)
      return -3;
    return 0;
  }
  const auto column_sum = [&](bool behind) {
    return p->type == kBF16 ? launch_column_sum<__nv_bfloat16>(*p, behind, st)
                            : launch_column_sum<__half>(*p, behind, st);
  };
  if (p->N == 0) return column_sum(false);
  if (((p->M + 127LL) / 128) * ((p->N + 63LL) / 64) >= (1LL << 31)) return -11;
  Operand oa = operand_a(*p), ob = operand_b(*p);
  const LinearPlan pl = plan_linear(p->M, p->N, p->K, split_clusters);
  const bool sums = p->kind == kLinearWgrad && p->dbias;
  if (sums && !pl.splits) {
    const int rc = column_sum(false);
    if (rc) return rc;
  }
  // whether the product follows a kernel of the same call
  const bool behind = (sums && !pl.splits) || !oa.direct() || !ob.direct();
  uint8_t* work = static_cast<uint8_t*>(p->work);
  int rc = lay_out(oa, work, st);
  if (rc) return rc;
  rc = lay_out(ob, work, st);
  if (rc) return rc;
  LinearArgs a = {};
  a.M = p->M;
  a.N = p->N;
  a.K = p->K;
  a.a_mn = p->kind == kLinearWgrad;
  a.b_mn = p->kind != kLinearFwd;
  a.idesc = idesc_bf16_f32(128 * pl.cg, pl.bn, a.a_mn, a.b_mn);
  if (p->type == kF16) a.idesc &= ~((1u << 7) | (1u << 10));  // f16 operands
  const int b_rows = pl.bn / pl.cg;
  // (rows of a K-major operand that a few-tile kernel copies: those there are, in eights)
  const auto rows_of_box = [&](int rows, int box) {
    return pl.splits && rows < box ? (rows + 7) / 8 * 8 : box;
  };
  const int box_a = rows_of_box(p->M, 128), box_b = rows_of_box(p->N, b_rows);
  a.a_3d = a.a_mn && oa.cols % 64 == 0 && !pl.splits;  // (128 columns of a tile)
  a.b_3d = a.b_mn && ob.cols % 64 == 0 && b_rows == 128 && !pl.splits;
  CUtensorMap ta, tb, tp;
  rc = a.a_3d   ? make_tmap_3d_bf16(&ta, oa.p, oa.rows, oa.cols, oa.ld, 64, 2)
       : a.a_mn ? make_tmap_2d_bf16(&ta, oa.p, oa.rows, oa.cols, oa.ld, 64, 64)
                : make_tmap_2d_bf16(&ta, oa.p, oa.rows, oa.cols, oa.ld, 64, box_a);
  if (rc) return rc * 100 - 1;
  rc = a.b_3d   ? make_tmap_3d_bf16(&tb, ob.p, ob.rows, ob.cols, ob.ld, 64, 2)
       : a.b_mn ? make_tmap_2d_bf16(&tb, ob.p, ob.rows, ob.cols, ob.ld, 64, 64)
                : make_tmap_2d_bf16(&tb, ob.p, ob.rows, ob.cols, ob.ld, 64, box_b);
  if (rc) return rc * 100 - 2;
  tp = tb;
  if (pl.pieces > 1 && (!a.b_mn || a.b_3d))
    rc = make_tmap_2d_bf16(&tp, ob.p, ob.rows, ob.cols, ob.ld, 64,
                           a.b_mn ? 64 : b_rows / pl.pieces);
  if (rc) return rc * 100 - 3;
  a.full = static_cast<int>(pl.full);
  a.pieces = pl.pieces;
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
  const auto rows_on = [&](int bytes) {
    return rows_of(bytes / type_bytes(out_type), p->D, p->ldd, out_type) &&
           rows_of(bytes / 2, p->R, p->ldr, p->type) && rows_of(bytes / 2, p->Z, p->ldz, p->type);
  };
  a.vec = rows_on(32) ? kRows32 : rows_on(16) ? kRows16 : kRowsAny;
#define CFB_SPLIT(T)                                                                              \
  (p->kind == kLinearFwd                                                                         \
       ? launch_split<T, kLinearFwd>(ta, tb, a, pl.splits, box_a, box_b, behind, st)             \
   : p->kind == kLinearDgrad                                                                     \
       ? launch_split<T, kLinearDgrad>(ta, tb, a, pl.splits, box_a, box_b, behind, st)           \
       : launch_split<T, kLinearWgrad>(ta, tb, a, pl.splits, box_a, box_b, behind, st))
#define CFB_LINEAR(T)                                                                       \
  (p->kind == kLinearFwd     ? launch_plan<T, kLinearFwd>(pl, ta, tb, tp, a, behind, st)               \
   : p->kind == kLinearDgrad ? launch_plan<T, kLinearDgrad>(pl, ta, tb, tp, a, behind, st)             \
                             : launch_plan<T, kLinearWgrad>(pl, ta, tb, tp, a, behind, st))
  if (pl.splits) rc = p->type == kBF16 ? CFB_SPLIT(__nv_bfloat16) : CFB_SPLIT(__half);
  else rc = p->type == kBF16 ? CFB_LINEAR(__nv_bfloat16) : CFB_LINEAR(__half);
#undef CFB_SPLIT
#undef CFB_LINEAR
  return rc == 0 && sums && pl.splits ? column_sum(true) : rc;
}

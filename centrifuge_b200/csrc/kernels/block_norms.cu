// The norms after and before a block with the block's gate and the residual scale (sm_100a).
//
// With h a block's output, x the residual stream, w1 / w2 the weights of the norm after the block
// and of the norm before the next one, g the gate, a / b the residual and block scales:
//
//   r1 = (mean(h^2) + eps)^-1/2      y = a x + b g (h r1 w1)
//   r2 = (mean(y^2) + eps)^-1/2      n = y r2 w2
//
// and with dy, dn the gradients of y and n, on the kept rows:
//
//   dY  = dy + r2 (w2 dn) - y r2^3 mean(w2 dn y)              dx  = a dY
//   v   = b dY g w1         dh = r1 v - h r1^3 mean(v h)
//   dw2 = sum dn y r2       dw1 = sum b dY g h r1             dg  = b dY w1 h r1
//
// (dg summed over what the gate is broadcast along).  Everything is bound by memory: each row is
// read once, its sums are formed in fp32 and n is computed from y before y is rounded.
//
// The gate is absent, one value for each channel [H], for each token [T, 1] (fp32), or for each
// element [T, H].
#include "row_types.cuh"

namespace cfb {

struct NormRows {
  const void* h;
  long long ld_h;
  const void* x;  // forward: the residual stream; backward: the saved y
  long long ld_x;
  const void* w_post;
  const void* w_pre;  // null: no norm before the next block
  const void* gate;
  long long ld_gate;
  int gate_kind;
  float block_scale, resid_scale;
  int H;
};

// ---------------------------------------------------------------- forward
// A team of up to NW warps (a block; with NW = 1 each of a block's four warps is a team) holds R
// rows in registers: a thread has the same NV groups of W columns of each, so that it unpacks the
// weights once for R rows and the rows share the exchanges of their sums.
//
// Short blocks, dealt by the hardware, with rows in registers; each first asks the L2 cache for the
// rows of the block that will follow it on its SM, so that the loads of a block that waits for its
// sums are already under way.  Measured for 16384 x 2048 bf16 with a channel's gate (floor 41.1 us):
// 44.1 us (46.4 without the request ahead, 86 with one row in registers for two warps, 54 with
// R = 4 rows and eight columns a thread); 8192 x 4096: 46.1 us (51.5); 4096 x 8192: 50.9 us (61.1).
template <typename TH, typename TX, int NW, int NV, int R>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32) block_norms_fwd_kernel(
    NormRows a, float eps, TX* __restrict__ y, TH* __restrict__ n, float* __restrict__ rstd_post,
    float* __restrict__ rstd_pre, int rows) {
  constexpr int W = 8, P = W / 2;
  constexpr int kAhead = 148 * R;  // rows of the blocks in between, at one block an SM
  __shared__ float red[2][R * NW];
  const int team = NW == 1 ? blockIdx.x * 4 + warp_id() : blockIdx.x;
  const int tid = NW == 1 ? lane_id() : threadIdx.x;
  const int nt = NW == 1 ? 32 : blockDim.x;
  const int row0 = team * R;
  if (NW == 1 && row0 >= rows) return;
  const int H = a.H;
  if (NW > 1 && tid < R && row0 + kAhead + tid < rows) {
    const long long row = row0 + kAhead + tid;
    prefetch_l2(static_cast<const TH*>(a.h) + row * a.ld_h, H * static_cast<int>(sizeof(TH)));
    prefetch_l2(static_cast<const TX*>(a.x) + row * a.ld_x, H * static_cast<int>(sizeof(TX)));
  }
  Pack<TH, W> hp[NV][R];
  Pack<TX, W> xp[NV][R];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = c < H && row0 + r < rows;
      hp[k][r] = in ? load_pack<TH, W>(static_cast<const TH*>(a.h) + (row0 + r) * a.ld_h + c)
                    : zero_pack<TH, W>();
      xp[k][r] = in ? load_pack<TX, W>(static_cast<const TX*>(a.x) + (row0 + r) * a.ld_x + c)
                    : zero_pack<TX, W>();
    }
  }
  float ss[R], scale[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    F2 s = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      F2 h[P];
      unpack_f2<TH, W>(hp[k][r], h);
#pragma unroll
      for (int i = 0; i < P; ++i) s = fma2(h[i], h[i], s);
    }
    ss[r] = sum2(s);
  }
  team_sums<R, NW>(ss, red[0]);
  const float inv_h = 1.f / static_cast<float>(H);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float r1 = rsqrtf(ss[r] * inv_h + eps);
    scale[r] = a.block_scale * r1;
    if (row0 + r < rows) {
      if (a.gate_kind == kGateToken)
        scale[r] *= static_cast<const float*>(a.gate)[(row0 + r) * a.ld_gate];
      if (tid == 0) rstd_post[row0 + r] = r1;
    }
  }
  F2 yv[NV][R][P], sq[R];
#pragma unroll
  for (int r = 0; r < R; ++r) sq[r] = f2(0.f);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
    F2 w[P];
    unpack_f2<TH, W>(c < H ? load_pack<TH, W>(static_cast<const TH*>(a.w_post) + c)
                           : zero_pack<TH, W>(), w);
    if (a.gate_kind == kGateChannel && c < H) {
      F2 g[P];
      load_f2<TH, W>(static_cast<const TH*>(a.gate) + c, g);
#pragma unroll
      for (int i = 0; i < P; ++i) w[i] = w[i] * g[i];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      F2 h[P], x[P];
      unpack_f2<TH, W>(hp[k][r], h);
      unpack_f2<TX, W>(xp[k][r], x);
#pragma unroll
      for (int i = 0; i < P; ++i) h[i] = h[i] * w[i];
      if (a.gate_kind == kGateElement && c < H && row0 + r < rows) {
        F2 g[P];
        load_f2<TH, W>(static_cast<const TH*>(a.gate) + (row0 + r) * a.ld_gate + c, g);
#pragma unroll
        for (int i = 0; i < P; ++i) h[i] = h[i] * g[i];
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        yv[k][r][i] = fma2(h[i], f2(scale[r]), x[i] * f2(a.resid_scale));
        sq[r] = fma2(yv[k][r][i], yv[k][r][i], sq[r]);
      }
      if (c < H && row0 + r < rows)
        store_f2<TX, W>(y + static_cast<long long>(row0 + r) * H + c, yv[k][r]);
    }
  }
  if (a.w_pre == nullptr) return;
#pragma unroll
  for (int r = 0; r < R; ++r) ss[r] = sum2(sq[r]);
  team_sums<R, NW>(ss, red[1]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ss[r] = rsqrtf(ss[r] * inv_h + eps);
    if (tid == 0 && row0 + r < rows) rstd_pre[row0 + r] = ss[r];
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
    if (c >= H) continue;
    F2 w[P];
    load_f2<TH, W>(static_cast<const TH*>(a.w_pre) + c, w);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      F2 o[P];
#pragma unroll
      for (int i = 0; i < P; ++i) o[i] = yv[k][r][i] * f2(ss[r]) * w[i];
      if (row0 + r < rows) store_f2<TH, W>(n + static_cast<long long>(row0 + r) * H + c, o);
    }
  }
}

// Rows of other widths and alignments: one row a team, a pair of columns at a time.
template <typename TH, typename TX, int W, int NW, int NV>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32) block_norms_fwd_pairs_kernel(
    NormRows a, float eps, TX* __restrict__ y, TH* __restrict__ n, float* __restrict__ rstd_post,
    float* __restrict__ rstd_pre, int rows) {
  constexpr int NT = NW * 32;
  using C = PairCols<W, NT>;
  __shared__ float red[2][NW];
  const int row = NW == 1 ? blockIdx.x * 4 + warp_id() : blockIdx.x;
  const int tid = NW == 1 ? lane_id() : threadIdx.x;
  if (NW == 1 && row >= rows) return;
  const int H = a.H;
  const TH* h = static_cast<const TH*>(a.h) + row * a.ld_h;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ld_x;
  const TH* gate = static_cast<const TH*>(a.gate);
  if (a.gate_kind == kGateElement) gate += row * a.ld_gate;
  const bool by_column = a.gate_kind == kGateChannel || a.gate_kind == kGateElement;
  F2 hv[NV], xv[NV], s = f2(0.f);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    hv[k] = C::load(h, tid * W + k * 2 * NT, H);
    xv[k] = C::load(x, tid * W + k * 2 * NT, H);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) s = fma2(hv[k], hv[k], s);
  float ss = sum2(s);
  team_sums<1, NW>(&ss, red[0]);
  const float inv_h = 1.f / static_cast<float>(H);
  const float r1 = rsqrtf(ss * inv_h + eps);
  float scale = a.block_scale * r1;
  if (a.gate_kind == kGateToken) scale *= static_cast<const float*>(a.gate)[row * a.ld_gate];
  s = f2(0.f);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = tid * W + k * 2 * NT;
    F2 v = hv[k] * C::load(static_cast<const TH*>(a.w_post), c, H);
    if (by_column) v = v * C::load(gate, c, H);
    xv[k] = fma2(v, f2(scale), xv[k] * f2(a.resid_scale));
    s = fma2(xv[k], xv[k], s);
    C::store(y + static_cast<long long>(row) * H, c, H, xv[k]);
  }
  if (tid == 0) rstd_post[row] = r1;
  if (a.w_pre == nullptr) return;
  ss = sum2(s);
  team_sums<1, NW>(&ss, red[1]);
  const float r2 = rsqrtf(ss * inv_h + eps);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = tid * W + k * 2 * NT;
    C::store(n + static_cast<long long>(row) * H, c, H,
             xv[k] * f2(r2) * C::load(static_cast<const TH*>(a.w_pre), c, H));
  }
  if (tid == 0) rstd_pre[row] = r2;
}

// ---------------------------------------------------------------- backward
// Sum of v over the block.  One barrier: the next call takes another `red`, and comes back to this
// one only after a further barrier.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_add(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  float s = lane_id() < warps ? red[lane_id()] : 0.f;
  return warp_add(s);
}

// One block walks the rows blockIdx.x, + gridDim.x, ...; each thread owns NV groups of W columns of
// every row and keeps the column sums of the weights' gradients in registers:
//   part[block][0] = sum dn y r2,  part[block][1] = sum b dY h r1 (times the token's or element's
// gate; a channel's gate is applied once, when the sums are joined).
template <typename TH, typename TX, int W, int NV>
__global__ void __launch_bounds__(1024) block_norms_bwd_kernel(
    NormRows a, const TX* __restrict__ dy, long long ld_dy, const TH* __restrict__ dn,
    long long ld_dn, const float* __restrict__ rstd_post, const float* __restrict__ rstd_pre,
    const int* __restrict__ row_ids, long long n_rows, TX* __restrict__ dx, TH* __restrict__ dh,
    void* __restrict__ dgate, float* __restrict__ part, int rows, int* err) {
  __shared__ float red[4][32];
  const int H = a.H, tid = threadIdx.x, nt = blockDim.x;
  const bool pre = a.w_pre != nullptr;
  const float inv_h = 1.f / static_cast<float>(H);
  float s_pre[NV][W], s_post[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < W; ++i) s_pre[k][i] = s_post[k][i] = 0.f;

  int turn = 0;
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const long long src = row_ids ? row_ids[r] : r;
    const long long out = static_cast<long long>(r) * H;
    if (!index_in(src, n_rows, err)) {  // out-of-range row id: zero gradients
      float z[W];
#pragma unroll
      for (int i = 0; i < W; ++i) z[i] = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * nt) * W;
        if (c < H) {
          store_f32<TX, W>(dx + out + c, z);
          store_f32<TH, W>(dh + out + c, z);
          if (a.gate_kind == kGateElement) store_f32<TH, W>(static_cast<TH*>(dgate) + out + c, z);
        }
      }
      if (a.gate_kind == kGateToken && tid == 0) static_cast<float*>(dgate)[r] = 0.f;
      continue;
    }
    const TH* h = static_cast<const TH*>(a.h) + src * a.ld_h;
    float d[NV][W], hv[NV][W];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * nt) * W;
      if (c < H) {
        load_f32<TH, W>(h + c, hv[k]);
        if (dy) {
          load_f32<TX, W>(dy + r * ld_dy + c, d[k]);
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) d[k][i] = 0.f;
        }
      }
    }
    if (pre) {
      const TX* y = static_cast<const TX*>(a.x) + src * a.ld_x;
      const float r2 = rstd_pre[src];
      float yv[NV][W];
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * nt) * W;
        if (c < H) {
          float q[W], w[W];
          load_f32<TX, W>(y + c, yv[k]);
          load_f32<TH, W>(dn + r * ld_dn + c, q);
          load_f32<TH, W>(static_cast<const TH*>(a.w_pre) + c, w);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            s_pre[k][i] += q[i] * (yv[k][i] * r2);
            w[i] *= q[i];
            dot += w[i] * yv[k][i];
            d[k][i] += r2 * w[i];
          }
        }
      }
      const float coef = block_sum(dot, red[turn]) * inv_h * r2 * r2 * r2;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) d[k][i] -= yv[k][i] * coef;
    }
    const float r1 = rstd_post[src];
    const float tg = a.gate_kind == kGateToken
                         ? static_cast<const float*>(a.gate)[src * a.ld_gate] : 1.f;
    const TH* gate = static_cast<const TH*>(a.gate);
    if (a.gate_kind == kGateElement) gate += src * a.ld_gate;
    float v[NV][W];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * nt) * W;
      if (c < H) {
        float w[W], g[W], e[W];
        load_f32<TH, W>(static_cast<const TH*>(a.w_post) + c, w);
        const bool by_column = a.gate_kind == kGateChannel || a.gate_kind == kGateElement;
        if (by_column) load_f32<TH, W>(gate + c, g);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          e[i] = a.resid_scale * d[k][i];
          const float t = a.block_scale * d[k][i];
          const float th = t * (hv[k][i] * r1);
          v[k][i] = t * w[i];  // without the token's gate
          if (a.gate_kind == kGateElement) {
            s_post[k][i] += th * g[i];
            w[i] *= th;  // dgate of the element
          } else {
            s_post[k][i] += th * tg;
          }
          if (by_column) v[k][i] *= g[i];
          dot += v[k][i] * hv[k][i];
        }
        store_f32<TX, W>(dx + out + c, e);
        if (a.gate_kind == kGateElement) store_f32<TH, W>(static_cast<TH*>(dgate) + out + c, w);
      }
    }
    dot = block_sum(dot, red[turn + 1]);
    if (a.gate_kind == kGateToken && tid == 0) static_cast<float*>(dgate)[r] = dot * r1;
    const float coef = dot * inv_h * r1 * r1;
    const float scale = tg * r1;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * nt) * W;
      if (c < H) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[k][i] = scale * (v[k][i] - hv[k][i] * coef);
        store_f32<TH, W>(dh + out + c, v[k]);
      }
    }
    turn ^= 2;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
    if (c < H) {
      float* p = part + 2ll * blockIdx.x * H + c;
      if (pre) store_f32<float, W>(p, s_pre[k]);
      store_f32<float, W>(p + H, s_post[k]);
    }
  }
}

// dw_pre, dw_post and a channel gate's gradient from the blocks' column sums, in block order.
// Block: 32 columns x 8 slices of the blocks.
template <typename TH>
__global__ void __launch_bounds__(256) block_norms_join_kernel(
    const float* __restrict__ part, int blocks, int H, const TH* __restrict__ w_post,
    const TH* __restrict__ gate, float* __restrict__ dw_pre, float* __restrict__ dw_post,
    float* __restrict__ dgate, int add) {
  __shared__ float red[2][8][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  float s0 = 0.f, s1 = 0.f;
  if (c < H)
    for (int b = ry; b < blocks; b += 8) {
      if (dw_pre) s0 += part[2ll * b * H + c];
      s1 += part[(2ll * b + 1) * H + c];
    }
  red[0][ry][cx] = s0;
  red[1][ry][cx] = s1;
  __syncthreads();
  if (ry != 0 || c >= H) return;
  s0 = s1 = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    s0 += red[0][k][cx];
    s1 += red[1][k][cx];
  }
  if (dw_pre) dw_pre[c] = (add ? dw_pre[c] : 0.f) + s0;
  const float g = gate ? to_f32(gate[c]) : 1.f;
  dw_post[c] = (add ? dw_post[c] : 0.f) + s1 * g;
  if (dgate) dgate[c] = (add ? dgate[c] : 0.f) + s1 * to_f32(w_post[c]);
}

// f(TypeTag<TH>, TypeTag<TX>): the residual stream has the block's type or fp32.
template <typename F>
int with_types(int type, int resid_type, F&& f) {
  return with_type(type, [&](auto th) {
    using TH = typename decltype(th)::type;
    if (resid_type == type) return f(TypeTag<TH>(), TypeTag<TH>());
    if (resid_type == kF32) return f(TypeTag<TH>(), TypeTag<float>());
    return -12;
  });
}

}  // namespace cfb

using namespace cfb;

namespace {
template <typename TH, typename TX, int NW, int NV, int R>
int launch_fwd(const NormRows& a, float eps, void* y, void* n, float* rstd_post, float* rstd_pre,
               int rows, cudaStream_t st) {
  const int teams = (rows + R - 1) / R;
  const int threads = NW == 1 ? 128 : ((a.H + 8 * NV - 1) / (8 * NV) + 31) / 32 * 32;
  block_norms_fwd_kernel<TH, TX, NW, NV, R>
      <<<NW == 1 ? (teams + 3) / 4 : teams, threads, 0, st>>>(
          a, eps, static_cast<TX*>(y), static_cast<TH*>(n), rstd_post, rstd_pre, rows);
  return launch_status();
}
template <typename TH, typename TX, int W, int NW, int NV>
int launch_fwd_pairs(const NormRows& a, float eps, void* y, void* n, float* rstd_post,
                     float* rstd_pre, int rows, cudaStream_t st) {
  block_norms_fwd_pairs_kernel<TH, TX, W, NW, NV>
      <<<NW == 1 ? (rows + 3) / 4 : rows, NW == 1 ? 128 : NW * 32, 0, st>>>(
          a, eps, static_cast<TX*>(y), static_cast<TH*>(n), rstd_post, rstd_pre, rows);
  return launch_status();
}
// The widest access that all rows of the operator allow.
template <typename F>
int widest(F&& rows_allow) {
  return rows_allow(8) ? 8 : rows_allow(2) ? 2 : 1;
}
}  // namespace

int cfb_block_norms_fwd(const CfbBlockNorms* p, float eps, void* y, void* n, float* rstd_post,
                        float* rstd_pre, int rows, cudaStream_t st) {
  const NormRows a = {p->h, p->ld_h, p->x, p->ld_x, p->w_post, p->w_pre, p->gate, p->ld_gate,
                      p->gate_kind, p->block_scale, p->resid_scale, p->H};
  if (rows == 0 || a.H == 0) return 0;
  if (a.H > kBlockNormsMaxH) return -11;
  const int W = widest([&](int w) {
    return a.H % w == 0 && rows_of(w, a.h, a.ld_h, p->type) &&
           rows_of(w, a.x, a.ld_x, p->resid_type) && rows_of(w, a.w_post, 0, p->type) &&
           rows_of(w, a.w_pre, 0, p->type) && rows_of(w, y, a.H, p->resid_type) &&
           rows_of(w, n, a.H, p->type) &&
           (a.gate_kind == kGateNone || a.gate_kind == kGateToken ||
            rows_of(w, a.gate, a.ld_gate, p->type));
  });
  return with_types(p->type, p->resid_type, [&](auto th, auto tx) {
    using TH = typename decltype(th)::type;
    using TX = typename decltype(tx)::type;
    const int H = a.H;
#define CFB_FWD(NW, NV, R) \
  return launch_fwd<TH, TX, NW, NV, R>(a, eps, y, n, rstd_post, rstd_pre, rows, st)
    if (W == 8) {
      // Several rows a team pay while there are blocks enough, and where a row is 2 bytes an element
      // (an fp32 stream at 8190 x 4096: 63.2 us with one, 64.6 with two).
      if (rows >= 148 * 8 && sizeof(TX) == 2) {
        if (H <= 256) CFB_FWD(1, 1, 4);
        if (H <= 512) CFB_FWD(1, 2, 2);
        if (H <= 1024) CFB_FWD(4, 1, 4);
        if (H <= 2048) CFB_FWD(4, 2, 2);
        if (H <= 4096) CFB_FWD(8, 2, 2);
      }
      if (H <= 256) CFB_FWD(1, 1, 1);
      if (H <= 512) CFB_FWD(1, 2, 1);
      if (H <= 1024) CFB_FWD(4, 1, 1);
      if (H <= 2048) CFB_FWD(4, 2, 1);
      if (H <= 4096) CFB_FWD(8, 2, 1);
      if (H <= 8192) CFB_FWD(16, 2, 1);
      CFB_FWD(32, 2, 1);
    }
#undef CFB_FWD
#define CFB_FWD(NW, NV)                                                                          \
  return W == 2 ? launch_fwd_pairs<TH, TX, 2, NW, NV>(a, eps, y, n, rstd_post, rstd_pre, rows, st) \
                : launch_fwd_pairs<TH, TX, 1, NW, NV>(a, eps, y, n, rstd_post, rstd_pre, rows, st)
    if (H <= 256) CFB_FWD(1, 4);
    if (H <= 512) CFB_FWD(1, 8);
    if (H <= 1024) CFB_FWD(4, 4);
    if (H <= 2048) CFB_FWD(4, 8);
    if (H <= 2560) CFB_FWD(8, 5);
    if (H <= 4096) CFB_FWD(8, 8);
    if (H <= 8192) CFB_FWD(16, 8);
    CFB_FWD(32, 8);
#undef CFB_FWD
  });
}

long long cfb_block_norms_bwd_workspace(int rows, int H) {
  const long long blocks = rows < 148 * 8 ? rows : 148 * 8;
  return 4ll * 2 * blocks * H;  // bytes
}

int cfb_block_norms_bwd(const CfbBlockNorms* p, const void* dy, long long ld_dy, const void* dn,
                        long long ld_dn, const float* rstd_post, const float* rstd_pre,
                        const int* row_ids, long long n_rows, void* dx, void* dh, void* dgate,
                        float* dw_post, float* dw_pre, int add, void* work, int rows, int* err,
                        cudaStream_t st) {
  const NormRows a = {p->h, p->ld_h, p->x, p->ld_x, p->w_post, p->w_pre, p->gate, p->ld_gate,
                      p->gate_kind, p->block_scale, p->resid_scale, p->H};
  const int H = a.H;
  if (H == 0) return 0;
  if (H > kBlockNormsMaxH) return -11;
  const bool by_row = a.gate_kind == kGateToken || a.gate_kind == kGateElement;
  const bool wide = H % 8 == 0 && rows_of_8(a.h, a.ld_h, p->type) &&
                    rows_of_8(a.x, a.ld_x, p->resid_type) && rows_of_8(dy, ld_dy, p->resid_type) &&
                    rows_of_8(dn, ld_dn, p->type) && rows_of_8(a.w_post, 0, p->type) &&
                    rows_of_8(a.w_pre, 0, p->type) && rows_of_8(dx, H, p->resid_type) &&
                    rows_of_8(dh, H, p->type) &&
                    (a.gate_kind == kGateNone || a.gate_kind == kGateToken ||
                     rows_of_8(a.gate, a.ld_gate, p->type)) &&
                    (a.gate_kind != kGateElement || rows_of_8(dgate, H, p->type));
  float* part = static_cast<float*>(work);
  return with_types(p->type, p->resid_type, [&](auto th, auto tx) {
    using TH = typename decltype(th)::type;
    using TX = typename decltype(tx)::type;
    int blocks = 0;
    if (rows > 0) {
      const int W = wide ? 8 : 1;
      const int nv = wide ? (H <= 8192 ? 1 : 2) : (H <= 4096 ? 4 : 16);
      const int threads = ((H + W * nv - 1) / (W * nv) + 31) / 32 * 32;
      auto* kernel = wide ? (nv == 1 ? block_norms_bwd_kernel<TH, TX, 8, 1>
                                     : block_norms_bwd_kernel<TH, TX, 8, 2>)
                          : (nv == 4 ? block_norms_bwd_kernel<TH, TX, 1, 4>
                                     : block_norms_bwd_kernel<TH, TX, 1, 16>);
      const int per_sm = threads >= 1024 ? 1 : threads >= 512 ? 2 : threads >= 256 ? 4 : 8;
      blocks = rows < 148 * per_sm ? rows : 148 * per_sm;
      kernel<<<blocks, threads, 0, st>>>(
          a, static_cast<const TX*>(dy), ld_dy, static_cast<const TH*>(dn), ld_dn, rstd_post,
          rstd_pre, row_ids, n_rows, static_cast<TX*>(dx), static_cast<TH*>(dh),
          by_row ? dgate : nullptr, part, rows, err);
      if (const int rc = launch_status()) return rc;
    } else if (add) {
      return 0;
    }
    const bool channel = a.gate_kind == kGateChannel;
    block_norms_join_kernel<TH><<<(H + 31) / 32, 256, 0, st>>>(
        part, blocks, H, static_cast<const TH*>(a.w_post),
        channel ? static_cast<const TH*>(a.gate) : nullptr, a.w_pre ? dw_pre : nullptr, dw_post,
        channel ? static_cast<float*>(dgate) : nullptr, add);
    return launch_status();
  });
}

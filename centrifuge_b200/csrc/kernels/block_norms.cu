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
// sums are already under way.  The kernel alone, 16384 x 2048 bf16 with a channel's gate (floor 41.1
// us): 44.1 us (46.4 without the request ahead, 86 with one row in registers for two warps, 54 with
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
    hv[k] = C::load(h, C::column(tid, k), H);
    xv[k] = C::load(x, C::column(tid, k), H);
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
    const int c = C::column(tid, k);
    F2 v = hv[k] * C::load(static_cast<const TH*>(a.w_post), c, H);
    if (by_column) v = v * C::load(gate, c, H);
    xv[k] = fma2(v, f2(scale), xv[k] * f2(a.resid_scale));
    s = fma2(xv[k], xv[k], s);
    C::store(y + static_cast<long long>(row) * H, c, H, &xv[k]);
  }
  if (tid == 0) rstd_post[row] = r1;
  if (a.w_pre == nullptr) return;
  ss = sum2(s);
  team_sums<1, NW>(&ss, red[1]);
  const float r2 = rsqrtf(ss * inv_h + eps);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = C::column(tid, k);
    const F2 v = xv[k] * f2(r2) * C::load(static_cast<const TH*>(a.w_pre), c, H);
    C::store(n + static_cast<long long>(row) * H, c, H, &v);
  }
  if (tid == 0) rstd_pre[row] = r2;
}

// ---------------------------------------------------------------- backward
// Blocks walk the rows; a team of NW warps (the block, or, where NW < 8, one of 8 / NW in it) has a
// row, and each thread the same NV groups of columns of every row, whose sums for the weights'
// gradients it keeps in registers:
//   part[block][0] = sum dn y r2,  part[block][1] = sum b dY h r1 (times the token's or element's
// gate; a channel's gate is applied once, when the sums are joined).
// With p = dn y and q = dY h the row sums and the column sums share their products.  While a block
// works, the rows of its next turn are on their way to the L2 cache.
template <typename C, typename TH, typename TX, int NW, int NV>
__global__ void __launch_bounds__(NW < 8 ? 256 : NW * 32, C::P == 1 ? (NW <= 8 ? 3 : NW <= 16 ? 2 : 1) : 1)
    block_norms_bwd_kernel(
    NormRows a, const TX* __restrict__ dy, long long ld_dy, const TH* __restrict__ dn,
    long long ld_dn, const float* __restrict__ rstd_post, const float* __restrict__ rstd_pre,
    const int* __restrict__ row_ids, long long n_rows, TX* __restrict__ dx, TH* __restrict__ dh,
    void* __restrict__ dgate, float* __restrict__ part, int rows, int* err) {
  // A row a turn.  The compiler schedules the loops over the rows of a turn better than the same
  // arithmetic without them (2048 x 8192 with an fp32 stream: 73.6 us a pass, 76.3 without).
  constexpr int P = C::P, R = 1;
  constexpr int kTeams = NW < 8 ? 8 / NW : 1;
  static_assert(!std::is_same<C, WideCols>::value || kTeams == 1 || NV == 1,
                "wide columns step by the block");
  let_next_start();
  __shared__ float red[kTeams][2][R * NW];
  const int H = a.H;
  const int team = kTeams > 1 ? warp_id() / NW : 0;
  const int tid = kTeams > 1 ? threadIdx.x % (NW * 32) : threadIdx.x;
  const int named = kTeams > 1 ? team : -1;
  const bool pre = a.w_pre != nullptr;
  const float inv_h = 1.f / static_cast<float>(H);
  F2 s_pre[NV][P], s_post[NV][P];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) s_pre[k][i] = s_post[k][i] = f2(0.f);

  const int step = gridDim.x * kTeams * R;
  for (int r0 = (blockIdx.x * kTeams + team) * R; r0 < rows; r0 += step) {
    if (tid < R && r0 + step + tid < rows) {  // the next turn's rows
      const long long r = r0 + step + tid;
      const long long src = row_ids ? row_ids[r] : r;
      if (src >= 0 && src < n_rows) {
        prefetch_l2(static_cast<const TH*>(a.h) + src * a.ld_h, H * static_cast<int>(sizeof(TH)));
        if (pre) {
          prefetch_l2(static_cast<const TX*>(a.x) + src * a.ld_x, H * static_cast<int>(sizeof(TX)));
          prefetch_l2(dn + r * ld_dn, H * static_cast<int>(sizeof(TH)));
        }
        if (dy) prefetch_l2(dy + r * ld_dy, H * static_cast<int>(sizeof(TX)));
      }
    }
    long long src[R];
    int width[R];  // H, or 0 where there is no row: everything of it is zero
#pragma unroll
    for (int r = 0; r < R; ++r) {
      src[r] = 0;
      width[r] = 0;
      if (r0 + r < rows) {
        src[r] = row_ids ? row_ids[r0 + r] : r0 + r;
        if (index_in(src[r], n_rows, err)) width[r] = H; else src[r] = 0;
      }
    }
    typename C::template Raw<TH> hp[NV][R];
    typename C::template Raw<TX> yp[NV][R];
    F2 d[NV][R][P];
    float dot[R];
    // dY without the part along y, and the sums for it
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = C::column(tid, k);
        hp[k][r] = C::load(static_cast<const TH*>(a.h) + src[r] * a.ld_h, c, width[r]);
        if (pre) yp[k][r] = C::load(static_cast<const TX*>(a.x) + src[r] * a.ld_x, c, width[r]);
        if (dy) {
          C::template unpack<TX>(C::load(dy + (r0 + r) * ld_dy, c, width[r]), d[k][r]);
        } else {
#pragma unroll
          for (int i = 0; i < P; ++i) d[k][r][i] = f2(0.f);
        }
      }
    if (pre) {
      F2 sum[R];
      float r2[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sum[r] = f2(0.f);
        r2[r] = width[r] ? rstd_pre[src[r]] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = C::column(tid, k);
        F2 w[P];
        C::template unpack<TH>(C::load(static_cast<const TH*>(a.w_pre), c, H), w);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          F2 g[P], y[P];
          C::template unpack<TH>(C::load(dn + (r0 + r) * ld_dn, c, width[r]), g);
          C::template unpack<TX>(yp[k][r], y);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const F2 p = g[i] * y[i];
            s_pre[k][i] = fma2(p, f2(r2[r]), s_pre[k][i]);
            sum[r] = fma2(p, w[i], sum[r]);
            d[k][r][i] = fma2(g[i] * w[i], f2(r2[r]), d[k][r][i]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) dot[r] = sum2(sum[r]);
      team_sums<R, NW>(dot, red[team][0], named);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float coef = -dot[r] * inv_h * r2[r] * r2[r] * r2[r];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          F2 y[P];
          C::template unpack<TX>(yp[k][r], y);
#pragma unroll
          for (int i = 0; i < P; ++i) d[k][r][i] = fma2(y[i], f2(coef), d[k][r][i]);
        }
      }
    }
    float r1[R], tg[R];
    F2 sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[r] = f2(0.f);
      r1[r] = width[r] ? rstd_post[src[r]] : 0.f;
      tg[r] = a.gate_kind == kGateToken && width[r]
                  ? static_cast<const float*>(a.gate)[src[r] * a.ld_gate] : 1.f;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = C::column(tid, k);
      F2 w[P];
      C::template unpack<TH>(C::load(static_cast<const TH*>(a.w_post), c, H), w);
      if (a.gate_kind == kGateChannel) {
        F2 g[P];
        C::template unpack<TH>(C::load(static_cast<const TH*>(a.gate), c, H), g);
#pragma unroll
        for (int i = 0; i < P; ++i) w[i] = w[i] * g[i];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const long long out = static_cast<long long>(r0 + r) * H;
        const int live = r0 + r < rows ? H : 0;  // rows without a source are written as zeros
        F2 e[P], h[P];
        C::template unpack<TH>(hp[k][r], h);
#pragma unroll
        for (int i = 0; i < P; ++i) e[i] = d[k][r][i] * f2(a.resid_scale);
        C::store(dx + out, c, live, e);
        const float br = a.block_scale * r1[r];
        if (a.gate_kind == kGateElement) {
          F2 g[P];
          C::template unpack<TH>(
              C::load(static_cast<const TH*>(a.gate) + src[r] * a.ld_gate, c, width[r]), g);
#pragma unroll
          for (int i = 0; i < P; ++i) e[i] = d[k][r][i] * h[i] * f2(br) * w[i];
          C::store(static_cast<TH*>(dgate) + out, c, live, e);
#pragma unroll
          for (int i = 0; i < P; ++i) d[k][r][i] = d[k][r][i] * g[i];
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const F2 q = d[k][r][i] * h[i];
          s_post[k][i] = fma2(q, f2(br * tg[r]), s_post[k][i]);
          sum[r] = fma2(q, w[i], sum[r]);
          d[k][r][i] = d[k][r][i] * w[i];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) dot[r] = sum2(sum[r]);
    team_sums<R, NW>(dot, red[team][1], named);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long out = static_cast<long long>(r0 + r) * H;
      const int live = r0 + r < rows ? H : 0;
      const float br = a.block_scale * r1[r];
      if (a.gate_kind == kGateToken && tid == 0 && live)
        static_cast<float*>(dgate)[r0 + r] = dot[r] * br;
      const float coef = -dot[r] * inv_h * r1[r] * r1[r];
      const F2 scale = f2(br * tg[r]);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        F2 h[P];
        C::template unpack<TH>(hp[k][r], h);
#pragma unroll
        for (int i = 0; i < P; ++i) h[i] = fma2(h[i], f2(coef), d[k][r][i]) * scale;
        C::store(dh + out, C::column(tid, k), live, h);
      }
    }
    // without the norm before the next block one barrier a turn is left: red[1] would be written
    // again before the slowest warp has read it
    if (!pre && NW > 1) {
      if (kTeams > 1)
        asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(NW * 32) : "memory");
      else
        __syncthreads();
    }
  }

  float* mine = part + 2ll * blockIdx.x * H;
  if constexpr (kTeams > 1) {  // the teams' sums, in the order of the teams
    extern __shared__ float sums[];  // [kTeams][H]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 0 && !pre) continue;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
        C::put(sums + team * H, C::column(tid, k), H, which ? s_post[k] : s_pre[k]);
      __syncthreads();
      for (int c = threadIdx.x; c < H; c += 256) {
        float s = 0.f;
#pragma unroll
        for (int t = 0; t < kTeams; ++t) s += sums[t * H + c];
        mine[which * H + c] = s;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (pre) C::store(mine, C::column(tid, k), H, s_pre[k]);
      C::store(mine + H, C::column(tid, k), H, s_post[k]);
    }
  }
}

// The same for rows of whole aligned groups of eight, of which two at least fit in shared memory:
// each team keeps a ring of kStages rows (h, dn, y, dy) there, filled by bulk copies that its first
// thread issues, so that the loads of the next rows run while a row waits for its sums.  A row's
// stage is free again once every thread has its columns in registers, which the barrier of the
// row's first sum tells.  The weights (the one behind the block times a channel's gate) lie in shared
// memory in fp32, in two planes of the four low and the four high columns of each group of eight,
// so that a thread's two 16-byte reads have no bank conflicts.
//
// Bound by memory over many rows: 8192 kept x 2048 bf16 with a channel's gate take 41 us in the kernel
// alone (66 with loads into registers), 8192 more 31 us more, which is the copy rate; the rest is the
// first rows' latency and the column sums' write.
template <typename TH, typename TX, int NW, int NV>
__global__ void __launch_bounds__(NW < 4 ? 128 : NW * 32, NW < 4 ? 4 : NW <= 16 ? 16 / NW : 1)
    block_norms_bwd_ring_kernel(NormRows a, const TX* __restrict__ dy, long long ld_dy,
                                const TH* __restrict__ dn, long long ld_dn,
                                const float* __restrict__ rstd_post,
                                const float* __restrict__ rstd_pre,
                                const int* __restrict__ row_ids, long long n_rows,
                                TX* __restrict__ dx, TH* __restrict__ dh,
                                void* __restrict__ dgate, float* __restrict__ part, int rows,
                                int stages, int* err) {
  constexpr int P = 4, NT = NW * 32;
  constexpr int kTeams = NW < 4 ? 4 / NW : 1;
  constexpr int kMaxStages = 4;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t full[kTeams][kMaxStages];
  __shared__ float red[kTeams][3][NW];
  __shared__ int abort_flag;
  let_next_start();
  const int H = a.H;
  const int team = threadIdx.x / NT, tid = threadIdx.x % NT;
  const bool pre = a.w_pre != nullptr;
  const float inv_h = 1.f / static_cast<float>(H);
  // a stage: h, dn, y, dy, the element's gate
  const int at_dn = H * static_cast<int>(sizeof(TH)), at_y = 2 * at_dn;
  const int at_dy = at_y + H * static_cast<int>(sizeof(TX));
  const bool element = a.gate_kind == kGateElement;
  const int at_gate = at_dy + H * static_cast<int>(sizeof(TX));
  const int stage_bytes = at_gate + (element ? at_dn : 0);
  uint8_t* ring = ring_all + static_cast<size_t>(team) * stages * stage_bytes;
  float* w_pre = reinterpret_cast<float*>(ring_all + static_cast<size_t>(kTeams) * stages * stage_bytes);
  float* w_post = w_pre + H;
  const auto weights = [&](const float* w, int c, F2* f) {
    const float4 lo = *reinterpret_cast<const float4*>(w + c / 2);
    const float4 hi = *reinterpret_cast<const float4*>(w + H / 2 + c / 2);
    f[0] = f2(lo.x, lo.y);
    f[1] = f2(lo.z, lo.w);
    f[2] = f2(hi.x, hi.y);
    f[3] = f2(hi.z, hi.w);
  };
  if (tid < stages) mbar_init(smem_u32(&full[team][tid]), 1);
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  __syncthreads();

  const int step = gridDim.x * kTeams;
  const int first = blockIdx.x * kTeams + team;
  const auto id_of = [&](int r) { return r < rows ? (row_ids ? row_ids[r] : r) : 0; };
  // Row r, whose row of h and y is src, into stage s.  Of the team's first warp lane 0 copies h,
  // 1 dn, 2 y, 3 dy and 4 the gate, all by the same few instructions.
  const uint8_t* lane_base = static_cast<const uint8_t*>(a.h);
  long long lane_ld = a.ld_h * static_cast<int>(sizeof(TH));
  int lane_at = 0;
  if (tid == 1) {
    lane_base = reinterpret_cast<const uint8_t*>(dn);
    lane_ld = ld_dn * static_cast<int>(sizeof(TH));
    lane_at = at_dn;
  } else if (tid == 2) {
    lane_base = pre ? static_cast<const uint8_t*>(a.x) : nullptr;
    lane_ld = a.ld_x * static_cast<int>(sizeof(TX));
    lane_at = at_y;
  } else if (tid == 3) {
    lane_base = reinterpret_cast<const uint8_t*>(dy);
    lane_ld = ld_dy * static_cast<int>(sizeof(TX));
    lane_at = at_dy;
  } else if (tid == 4) {
    lane_base = element ? static_cast<const uint8_t*>(a.gate) : nullptr;
    lane_ld = a.ld_gate * static_cast<int>(sizeof(TH));
    lane_at = at_gate;
  }
  const int lane_bytes = H * static_cast<int>(tid == 2 || tid == 3 ? sizeof(TX) : sizeof(TH));
  const int row_bytes =
      H * static_cast<int>(sizeof(TH)) * (1 + (pre ? 1 : 0) + (element ? 1 : 0)) +
      H * static_cast<int>(sizeof(TX)) * ((pre ? 1 : 0) + (dy ? 1 : 0));
  const auto fetch = [&](int r, int src, int s) {  // lanes 0 to 4 of the team's first warp
    const uint32_t bar = smem_u32(&full[team][s]);
    const bool ok = src >= 0 && src < n_rows;
    if (tid == 0) {
      if (ok) {
        mbar_arrive_expect_tx(bar, row_bytes);
      } else {  // nothing of it is read
        mbar_arrive(bar);
        if (err) atomicCAS(err, 0, kErrBounds);
      }
    }
    if (ok && lane_base)
      bulk_load(smem_u32(ring + static_cast<size_t>(s) * stage_bytes + lane_at),
                lane_base + ((tid & 1) ? r : src) * lane_ld, lane_bytes, bar);
  };
  int fetch_id = 0;  // the id of the next row to be fetched, read one row ahead
  if (tid < 5) {
    int ids[kMaxStages + 1];
#pragma unroll
    for (int i = 0; i <= kMaxStages; ++i) ids[i] = id_of(first + i * step);
#pragma unroll
    for (int i = 0; i < kMaxStages; ++i)
      if (i < stages && first + i * step < rows) fetch(first + i * step, ids[i], i);
#pragma unroll
    for (int i = 0; i <= kMaxStages; ++i)
      if (i == stages) fetch_id = ids[i];
  }
  // the weights, while the first rows are on their way
  for (int c = threadIdx.x * 8; c < H; c += blockDim.x * 8) {
    const Pack<TH, 8> post = load_pack<TH, 8>(static_cast<const TH*>(a.w_post) + c);
    Pack<TH, 8> gate = post, before = post;
    if (a.gate_kind == kGateChannel) gate = load_pack<TH, 8>(static_cast<const TH*>(a.gate) + c);
    if (pre) before = load_pack<TH, 8>(static_cast<const TH*>(a.w_pre) + c);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = c / 2 + (i & 3) + ((i & 4) ? H / 2 : 0);
      w_post[at] = to_f32(post.v[i]) * (a.gate_kind == kGateChannel ? to_f32(gate.v[i]) : 1.f);
      if (pre) w_pre[at] = to_f32(before.v[i]);
    }
  }
  __syncthreads();

  F2 s_pre[NV][P], s_post[NV][P];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) s_pre[k][i] = s_post[k][i] = f2(0.f);
  // The sum of v over the team, and whether a thread of it gave up a wait.
  const auto team_sum = [&](float v, float* slot, bool& failed) {
    v = warp_add(v);
    if constexpr (NW == 1) {
      failed = __any_sync(0xffffffffu, failed);
      __syncwarp();
      return v;
    } else {
      if (lane_id() == 0) slot[tid / 32] = v;
      int any;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
          "bar.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
          : "=r"(any)
          : "r"(static_cast<int>(failed)), "r"(1 + team), "n"(NT)
          : "memory");
      failed = any != 0;
      if constexpr (NW <= 8) {
        float s = slot[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) s += slot[w];
        return s;
      } else {
        return warp_add(lane_id() < NW ? slot[lane_id()] : 0.f);
      }
    }
  };

  // the row at hand, read one row ahead: its id (-1: out of range), statistics and gate
  int next = -1;
  float r1 = 0.f, r2 = 0.f, tg = 1.f;
  const auto read_row = [&](int id) {
    next = id >= 0 && id < n_rows ? id : -1;
    r1 = r2 = 0.f;
    tg = 1.f;
    if (next < 0) return;
    r1 = rstd_post[next];
    if (pre) r2 = rstd_pre[next];
    if (a.gate_kind == kGateToken) tg = static_cast<const float*>(a.gate)[next * a.ld_gate];
  };
  const int first_id = id_of(first);
  int ahead = id_of(first + step);  // the id of the row after that
  read_row(first_id);

  const auto refill = [&](int r, int s) {
    if (tid >= 5 || r >= rows) return;
    fetch(r, fetch_id, s);
    fetch_id = id_of(r + step);
  };

  int s = 0, phase = 0, turn = 0;
  bool failed = false;
  for (int r = first; r < rows; r += step, ++turn) {
    failed = !mbar_wait(smem_u32(&full[team][s]), phase, &abort_flag, err, kErrWaitProducer);
    const int src = next;
    const float row_r2 = r2, br = a.block_scale * r1, scale = br * tg, c1 = inv_h * r1 * r1;
    read_row(ahead);
    ahead = id_of(r + 2 * step);
    const uint8_t* st = ring + static_cast<size_t>(s) * stage_bytes;
    const int done = s;
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
    const long long out = static_cast<long long>(r) * H;
    if (src < 0) {  // out-of-range row id: zero gradients (the whole team is here)
      F2 zero[P];
#pragma unroll
      for (int i = 0; i < P; ++i) zero[i] = f2(0.f);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * NT) * 8;
        if (c >= H) continue;
        store_f2<TX, 8>(dx + out + c, zero);
        store_f2<TH, 8>(dh + out + c, zero);
        if (element) store_f2<TH, 8>(static_cast<TH*>(dgate) + out + c, zero);
      }
      if (a.gate_kind == kGateToken && tid == 0) static_cast<float*>(dgate)[r] = 0.f;
      team_sum(0.f, red[team][2], failed);  // its barrier alone
      if (failed) break;
      refill(r + stages * step, done);
      continue;
    }
    F2 h[NV][P], d[NV][P];
    F2 sum = f2(0.f);
    Pack<TH, 8> gate[NV];
    if (element) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * NT) * 8;
        if (c < H) gate[k] = shared_pack(reinterpret_cast<const TH*>(st + at_gate) + c);
      }
    }
    if (pre) {
      F2 y[NV][P];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * NT) * 8;
        if (c >= H) continue;
        F2 g[P], w[P];
        unpack_f2<TH, 8>(shared_pack(reinterpret_cast<const TH*>(st) + c), h[k]);
        unpack_f2<TX, 8>(shared_pack(reinterpret_cast<const TX*>(st + at_y) + c), y[k]);
        unpack_f2<TH, 8>(shared_pack(reinterpret_cast<const TH*>(st + at_dn) + c), g);
        if (dy) unpack_f2<TX, 8>(shared_pack(reinterpret_cast<const TX*>(st + at_dy) + c), d[k]);
        weights(w_pre, c, w);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const F2 p = g[i] * y[k][i];
          s_pre[k][i] = fma2(p, f2(row_r2), s_pre[k][i]);
          sum = fma2(p, w[i], sum);
          d[k][i] = fma2(g[i] * w[i], f2(row_r2), dy ? d[k][i] : f2(0.f));
        }
      }
      const float dot = team_sum(sum2(sum), red[team][0], failed);
      if (failed) break;
      refill(r + stages * step, done);
      const F2 coef = f2(-dot * inv_h * row_r2 * row_r2 * row_r2);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) d[k][i] = fma2(y[k][i], coef, d[k][i]);
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (tid + k * NT) * 8;
        if (c >= H) continue;
        unpack_f2<TH, 8>(shared_pack(reinterpret_cast<const TH*>(st) + c), h[k]);
        unpack_f2<TX, 8>(shared_pack(reinterpret_cast<const TX*>(st + at_dy) + c), d[k]);
      }
    }
    sum = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * NT) * 8;
      if (c >= H) continue;
      F2 w[P], e[P];
      weights(w_post, c, w);
#pragma unroll
      for (int i = 0; i < P; ++i) e[i] = d[k][i] * f2(a.resid_scale);
      store_f2<TX, 8>(dx + out + c, e);
      if (element) {
#pragma unroll
        for (int i = 0; i < P; ++i) e[i] = d[k][i] * h[k][i] * f2(br) * w[i];
        store_f2<TH, 8>(static_cast<TH*>(dgate) + out + c, e);
        unpack_f2<TH, 8>(gate[k], e);
#pragma unroll
        for (int i = 0; i < P; ++i) d[k][i] = d[k][i] * e[i];
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const F2 q = d[k][i] * h[k][i];
        s_post[k][i] = fma2(q, f2(scale), s_post[k][i]);
        sum = fma2(q, w[i], sum);
        d[k][i] = d[k][i] * w[i];
      }
    }
    // without the norm before the next block this is the row's only barrier: two slots in turn
    const float dot = team_sum(sum2(sum), red[team][pre ? 1 : turn & 1], failed);
    if (!pre) {
      if (failed) break;
      refill(r + stages * step, done);
    }
    if (a.gate_kind == kGateToken && tid == 0) static_cast<float*>(dgate)[r] = dot * br;
    const F2 coef = f2(-dot * c1);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * NT) * 8;
      if (c >= H) continue;
#pragma unroll
      for (int i = 0; i < P; ++i) h[k][i] = fma2(h[k][i], coef, d[k][i]) * f2(scale);
      store_f2<TH, 8>(dh + out + c, h[k]);
    }
  }
  if (failed && tid == 0) {  // no copy may land in this memory after the block has ended
    volatile int never = 0;
    for (int i = 0; i < stages; ++i)
      if (first + (turn + i) * step < rows)
        mbar_wait(smem_u32(&full[team][(turn + i) % stages]), ((turn + i) / stages) & 1, &never,
                  nullptr, 0);
  }

  float* mine = part + 2ll * blockIdx.x * H;
  if constexpr (kTeams > 1) {  // the teams' sums, in the order of the teams
    float* sums = reinterpret_cast<float*>(ring_all);  // [kTeams][H], in the place of the rows
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 0 && !pre) continue;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
        WideCols::put(sums + team * H, (tid + k * NT) * 8, H, which ? s_post[k] : s_pre[k]);
      __syncthreads();
      for (int c = threadIdx.x; c < H; c += 128) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kTeams; ++i) t += sums[i * H + c];
        mine[which * H + c] = t;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * NT) * 8;
      if (pre) WideCols::store(mine, c, H, s_pre[k]);
      WideCols::store(mine + H, c, H, s_post[k]);
    }
  }
}

// dw_pre (which = 0), dw_post and a channel gate's gradient (which = 1) from the blocks' column sums,
// in block order; which = first + blockIdx.y.  Block: 32 columns x 32 slices of the blocks.  The
// three buffers may be one another (a parameter that is used in two places), so they are not
// __restrict__, and dw_pre has a launch of its own where it is one of the others.
template <typename TH>
__global__ void __launch_bounds__(1024) block_norms_join_kernel(
    const float* part, int blocks, int H, const TH* __restrict__ w_post,
    const TH* __restrict__ gate, float* dw_pre, float* dw_post, float* dgate, int add_pre,
    int add_post, int add_gate, int first) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  const int which = first + blockIdx.y;
  after_previous();
  if (which == 0 && dw_pre == nullptr) return;
  float s = 0.f;
  if (c < H) {
#pragma unroll 8
    for (int b = ry; b < blocks; b += 32) s += part[(2ll * b + which) * H + c];
  }
  red[ry][cx] = s;
  __syncthreads();
  s = warp_add(red[cx][ry]);  // warp ry: the 32 slices of column blockIdx.x * 32 + ry
  const int col = blockIdx.x * 32 + ry;
  if (cx != 0 || col >= H) return;
  if (which == 0) {
    dw_pre[col] = (add_pre ? dw_pre[col] : 0.f) + s;
    return;
  }
  dw_post[col] = (add_post ? dw_post[col] : 0.f) + (gate ? s * to_f32(gate[col]) : s);
  if (dgate) dgate[col] = (add_gate ? dgate[col] : 0.f) + s * to_f32(w_post[col]);
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

namespace {
struct BwdArgs {
  NormRows a;
  const void* dy;
  long long ld_dy;
  const void* dn;
  long long ld_dn;
  const float *rstd_post, *rstd_pre;
  const int* row_ids;
  long long n_rows;
  void *dx, *dh, *dgate;
  float* part;
  int rows;
  int* err;
};
// Launches the kernel and returns the number of its blocks, or a negative status.
template <typename C, typename TH, typename TX, int NW, int NV>
int launch_bwd(const BwdArgs& b, cudaStream_t st) {
  constexpr int kTeams = NW < 8 ? 8 / NW : 1;
  auto* kernel = block_norms_bwd_kernel<C, TH, TX, NW, NV>;
  int threads = NW < 8 ? 256 : NW * 32;
  if (std::is_same<C, WideCols>::value && NW >= 8)  // no more warps than the row needs
    threads = ((b.a.H + 8 * NV - 1) / (8 * NV) + 31) / 32 * 32;
  const int smem = kTeams > 1 ? kTeams * b.a.H * 4 : 0;
  static int per_sm = 0;  // resident blocks of this kernel: the same on every device of this type
  if (per_sm == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, NW < 8 ? 256 : NW * 32,
                                                      kTeams > 1 ? 16384 : 0) != cudaSuccess)
      return -3;
    per_sm = n < 1 ? 1 : n > 8 ? 8 : n;
  }
  const int turns = (b.rows + kTeams - 1) / kTeams;
  const int blocks = turns < 148 * per_sm ? turns : 148 * per_sm;
  kernel<<<blocks, threads, smem, st>>>(
      b.a, static_cast<const TX*>(b.dy), b.ld_dy, static_cast<const TH*>(b.dn), b.ld_dn,
      b.rstd_post, b.rstd_pre, b.row_ids, b.n_rows, static_cast<TX*>(b.dx),
      static_cast<TH*>(b.dh), b.dgate, b.part, b.rows, b.err);
  const int rc = launch_status();
  return rc ? rc : blocks;
}

constexpr int kRingBytes = 220 * 1024;  // shared memory of an SM that the rings may take

// The ring kernel where two rows a team fit; 0 where they do not.
template <typename TH, typename TX, int NW, int NV>
int launch_ring(const BwdArgs& b, cudaStream_t st) {
  constexpr int kTeams = NW < 4 ? 4 / NW : 1;
  // 16 warps of 128 registers are resident on an SM
  constexpr int threads = NW < 4 ? 128 : NW * 32;
  auto* kernel = block_norms_bwd_ring_kernel<TH, TX, NW, NV>;
  const bool element = b.a.gate_kind == kGateElement;
  const int row = b.a.H * static_cast<int>(2 * (sizeof(TH) + sizeof(TX)) +
                                           (element ? sizeof(TH) : 0)) * kTeams;
  const int weights = 8 * b.a.H;
  int per_sm = 512 / threads, stages = 0;
  for (; per_sm > 0; --per_sm) {
    stages = (kRingBytes / per_sm - weights) / row;
    if (stages >= 2) break;
  }
  if (per_sm == 0) return 0;
  if (stages > 4) stages = 4;
  const int smem = stages * row + weights;
  static bool allowed[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes) !=
        cudaSuccess)
      return -3;
    allowed[dev] = true;
  }
  const int turns = (b.rows + kTeams - 1) / kTeams;
  const int blocks = turns < 148 * per_sm ? turns : 148 * per_sm;
  kernel<<<blocks, threads, smem, st>>>(
      b.a, static_cast<const TX*>(b.dy), b.ld_dy, static_cast<const TH*>(b.dn), b.ld_dn,
      b.rstd_post, b.rstd_pre, b.row_ids, b.n_rows, static_cast<TX*>(b.dx),
      static_cast<TH*>(b.dh), b.dgate, b.part, b.rows, stages, b.err);
  const int rc = launch_status();
  return rc ? rc : blocks;
}
}  // namespace

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
  const int W = widest([&](int w) {
    return H % w == 0 && rows_of(w, a.h, a.ld_h, p->type) &&
           rows_of(w, a.x, a.ld_x, p->resid_type) && rows_of(w, dy, ld_dy, p->resid_type) &&
           rows_of(w, dn, ld_dn, p->type) && rows_of(w, a.w_post, 0, p->type) &&
           rows_of(w, a.w_pre, 0, p->type) && rows_of(w, dx, H, p->resid_type) &&
           rows_of(w, dh, H, p->type) &&
           (a.gate_kind == kGateNone || a.gate_kind == kGateToken ||
            rows_of(w, a.gate, a.ld_gate, p->type)) &&
           (a.gate_kind != kGateElement || rows_of(w, dgate, H, p->type));
  });
  float* part = static_cast<float*>(work);
  const BwdArgs b = {a, dy, ld_dy, dn, ld_dn, rstd_post, rstd_pre, row_ids, n_rows, dx, dh,
                     by_row ? dgate : nullptr, part, rows, err};
  return with_types(p->type, p->resid_type, [&](auto th, auto tx) {
    using TH = typename decltype(th)::type;
    using TX = typename decltype(tx)::type;
    const auto launch = [&]() -> int {
#define CFB_BWD(NW, NV) return launch_bwd<WideCols, TH, TX, NW, NV>(b, st)
#define CFB_RING(NW, NV) blocks = launch_ring<TH, TX, NW, NV>(b, st)
      if (W == 8) {
        // A ring of two rows always fits up to 1024 columns, and up to 4096 of two bytes.  Sixteen
        // columns a thread, as few warps as that takes: 8192 x 2048 46.5 us, 51.3 with eight columns
        // in eight warps, 108 with 32 in two; x 2304 59.6 with five warps, 70.4 with eight; x 512 and
        // x 1024, eight columns, 51.2 and 49.0 (of 32768 and 16384 rows), 60.6 and 60.4 with sixteen.
        // With an fp32 stream the ring of two blocks of eight warps ends at 3520 columns, and over
        // 2560 a row takes 16 warps: x 4096 113 us, 149 with eight (x 3400 109 for 93, x 2600 101
        // for 84).
        int blocks = 0;
        if (H <= 256) CFB_RING(1, 1);
        else if (H <= 512) CFB_RING(2, 1);
        else if (H <= 1024) CFB_RING(4, 1);
        if constexpr (sizeof(TH) == 2) {
          if (H > 1024) {
            if (H <= 2048) CFB_RING(4, 2);
            else if (H <= 2560) CFB_RING(5, 2);
            else if (H <= 4096) {
              if constexpr (sizeof(TX) == 4) CFB_RING(16, 1);
              else CFB_RING(8, 2);
            } else if (H <= 8192) CFB_RING(16, 2);
          }
        }
        if (blocks != 0) return blocks;
        // fp32 rows of over 1024 columns: a ring of them leaves room for too few blocks (8192 x 2048:
        // 77.5 us without, 81.0 with; 8192 x 4096: 156, 173)
        if constexpr (sizeof(TH) == 4) {
          if (H <= 2048) CFB_BWD(8, 1);
          if (H <= 4096) CFB_BWD(8, 2);
        }
        if (H <= 8192) CFB_BWD(32, 1);
        CFB_BWD(32, 2);
      }
#undef CFB_RING
#undef CFB_BWD
#define CFB_BWD(NW, NV)                                                     \
  return W == 2 ? launch_bwd<PairCols<2, NW * 32>, TH, TX, NW, NV>(b, st) \
                : launch_bwd<PairCols<1, NW * 32>, TH, TX, NW, NV>(b, st)
      if (H <= 256) CFB_BWD(1, 4);
      if (H <= 1024) CFB_BWD(4, 4);
      if (H <= 2048) CFB_BWD(8, 4);
      if (H <= 2560) CFB_BWD(8, 5);
      if (H <= 4096) CFB_BWD(16, 4);
      if (H <= 8192) CFB_BWD(32, 4);
      CFB_BWD(32, 8);
#undef CFB_BWD
    };
    int blocks = 0;
    if (rows > 0) {
      blocks = launch();
      if (blocks < 0) return blocks;
    } else if (add) {
      return 0;
    }
    // What two gradients share gets the sum of both: dw_pre first, then dw_post, then dgate.
    const bool channel = a.gate_kind == kGateChannel;
    float* pre = a.w_pre ? dw_pre : nullptr;
    float* gate_sum = channel ? static_cast<float*>(dgate) : nullptr;
    const bool post_on_pre = pre != nullptr && dw_post == pre;
    const bool gate_on_pre = pre != nullptr && gate_sum == pre;
    const bool apart = !post_on_pre && !gate_on_pre;
    const auto* w_post = static_cast<const TH*>(a.w_post);
    const auto* gate = channel ? static_cast<const TH*>(a.gate) : nullptr;
    const unsigned columns = (H + 31) / 32;
    const int add_post = add || post_on_pre;
    const int add_gate = add || gate_on_pre || gate_sum == dw_post;
    const int rc = launch_behind(block_norms_join_kernel<TH>, dim3(columns, apart ? 2 : 1),
                                 dim3(1024), 0, st, part, blocks, H, w_post, gate, pre, dw_post,
                                 gate_sum, add, add_post, add_gate, 0);
    if (rc || apart) return rc;
    block_norms_join_kernel<TH><<<columns, 1024, 0, st>>>(part, blocks, H, w_post, gate, pre,
                                                          dw_post, gate_sum, add, add_post,
                                                          add_gate, 1);
    return launch_status();
  });
}

// Layer norm and its gradient over the kept rows (sm_100a).
//
//   mu = mean(x)      r = (mean((x - mu)^2) + eps)^-1/2      n = (x - mu) r      y = n w + b
//
// and with dy the gradient of y, on the kept rows:
//
//   g = dy w      dx = r (g - mean(g) - n mean(g n)) + dres      dw = sum dy n      db = sum dy
//
// Bound by memory: each row is read once and stays in registers for the second sum (the squares are
// of x - mu, so a mean far from zero costs no digits); sums are fp32, each output is rounded once.
#include "row_types.cuh"

namespace cfb {

// ---------------------------------------------------------------- forward
// A team of up to NW warps (a block; with NW = 1 each of a block's four warps is a team) holds R
// rows: a thread has the same NV groups of eight columns of each, so that the weights are unpacked
// once and the rows share the exchanges of their sums.  Short blocks, each of which first asks the
// L2 cache for the rows of the block that will follow it on its SM.  16384 x 2048 bf16: 27 us, 0.76 of
// the measured copy rate; one row a team, four rows, eight or two warps, other columns a thread: 28 to
// 79 us.  Above 4096 columns a 16-bit row takes 16 warps, and above 8192 any row 32, which wait together
// (4096 x 8192 bf16: 37 us, 0.56 of the rate); up to 8192 an fp32 row takes eight (45 to 48 us, 0.86 or
// more).
template <typename TY, typename TX, int NW, int NV, int R>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32) layernorm_fwd_kernel(
    const TX* __restrict__ x, long long ld_x, const TY* __restrict__ w, const TY* __restrict__ b,
    float eps, TY* __restrict__ y, long long ld_y, float* __restrict__ mean,
    float* __restrict__ rstd, int rows, int H) {
  constexpr int W = 8, P = W / 2;
  constexpr int kAhead = 148 * R;
  __shared__ float red[2][R * NW];
  const int team = NW == 1 ? blockIdx.x * 4 + warp_id() : blockIdx.x;
  const int tid = NW == 1 ? lane_id() : threadIdx.x;
  const int nt = NW == 1 ? 32 : blockDim.x;
  const int row0 = team * R;
  if (NW == 1 && row0 >= rows) return;
  if (NW > 1 && tid < R && row0 + kAhead + tid < rows)
    prefetch_l2(x + (row0 + kAhead + tid) * ld_x, H * static_cast<int>(sizeof(TX)));
  Pack<TX, W> xp[NV][R];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
#pragma unroll
    for (int r = 0; r < R; ++r)
      xp[k][r] = c < H && row0 + r < rows ? load_pack<TX, W>(x + (row0 + r) * ld_x + c)
                                          : zero_pack<TX, W>();
  }
  Pack<TY, W> wp[NV], bp[NV];  // on their way while the rows' sums are formed
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
    if (w && c < H) wp[k] = load_pack<TY, W>(w + c);
    if (b && c < H) bp[k] = load_pack<TY, W>(b + c);
  }
  const float inv_h = 1.f / static_cast<float>(H);
  float mu[R], sq[R];
  F2 xv[NV][R][P];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    F2 s = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      unpack_f2<TX, W>(xp[k][r], xv[k][r]);
#pragma unroll
      for (int i = 0; i < P; ++i) s = s + xv[k][r][i];
    }
    mu[r] = sum2(s);
  }
  team_sums<R, NW>(mu, red[0]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mu[r] *= inv_h;
    F2 s = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((tid + k * nt) * W >= H) continue;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        xv[k][r][i] = xv[k][r][i] + f2(-mu[r]);
        s = fma2(xv[k][r][i], xv[k][r][i], s);
      }
    }
    sq[r] = sum2(s);
  }
  team_sums<R, NW>(sq, red[1]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sq[r] = rsqrtf(sq[r] * inv_h + eps);
    if (tid == 0 && row0 + r < rows) {
      mean[row0 + r] = mu[r];
      rstd[row0 + r] = sq[r];
    }
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (tid + k * nt) * W;
    if (c >= H) continue;
    F2 wv[P], bv[P];
    if (w) unpack_f2<TY, W>(wp[k], wv);
    if (b) unpack_f2<TY, W>(bp[k], bv);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (!w) wv[i] = f2(1.f);
      if (!b) bv[i] = f2(0.f);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      F2 o[P];
#pragma unroll
      for (int i = 0; i < P; ++i) o[i] = fma2(xv[k][r][i] * f2(sq[r]), wv[i], bv[i]);
      if (row0 + r < rows) store_f2<TY, W>(y + (row0 + r) * ld_y + c, o);
    }
  }
}

// Rows of other widths and alignments: one row a team, a pair of columns at a time (16384 x 2050 bf16:
// 61 us), or, where rows start anywhere, a column (2049: 87 us).
template <typename TY, typename TX, int W, int NW, int NV>
__global__ void __launch_bounds__(NW == 1 ? 128 : NW * 32) layernorm_fwd_pairs_kernel(
    const TX* __restrict__ x, long long ld_x, const TY* __restrict__ w, const TY* __restrict__ b,
    float eps, TY* __restrict__ y, long long ld_y, float* __restrict__ mean,
    float* __restrict__ rstd, int rows, int H) {
  constexpr int NT = NW * 32;
  using C = PairCols<W, NT>;
  __shared__ float red[2][NW];
  const int row = NW == 1 ? blockIdx.x * 4 + warp_id() : blockIdx.x;
  const int tid = NW == 1 ? lane_id() : threadIdx.x;
  if (NW == 1 && row >= rows) return;
  const TX* xr = x + row * ld_x;
  F2 v[NV], s = f2(0.f);
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = C::load(xr, C::column(tid, k), H);
#pragma unroll
  for (int k = 0; k < NV; ++k) s = s + v[k];
  float mu = sum2(s);
  team_sums<1, NW>(&mu, red[0]);
  const float inv_h = 1.f / static_cast<float>(H);
  mu *= inv_h;
  s = f2(0.f);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = C::column(tid, k);
    const int second = W == 1 ? c + NT : c + 1;
    v[k] = v[k] + f2(-mu);
    const F2 in = f2(c < H ? 1.f : 0.f, second < H ? 1.f : 0.f);
    s = fma2(v[k] * in, v[k], s);
  }
  float sq = sum2(s);
  team_sums<1, NW>(&sq, red[1]);
  const float r = rsqrtf(sq * inv_h + eps);
  if (tid == 0) {
    mean[row] = mu;
    rstd[row] = r;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = C::column(tid, k);
    F2 o = v[k] * f2(r);
    if (w) o = o * C::load(w, c, H);
    if (b) o = o + C::load(b, c, H);
    C::store(y + row * ld_y, c, H, &o);
  }
}

// ---------------------------------------------------------------- backward
struct LnBwd {
  const void* dy;
  long long ld_dy;
  const void* x;
  long long ld_x;
  const float *mean, *rstd;
  const void* w;  // null: ones
  const void* dres;
  long long ld_res;
  const int* row_ids;
  long long n_rows;
  void* dx;
  float* part;  // [blocks][2][H]: sums of dy n and of dy
  int rows, H;
  int* err;
};

// Both of a team's two sums at once, for NW warps that meet at the block's named barrier 1 + team;
// slot: 2 NW floats, of which the caller uses two in turn.  `failed`: whether any thread gave up.
template <int NW>
__device__ __forceinline__ void pair_sums(float& a, float& b, float* slot, int team, bool& failed) {
  float v[2] = {a, b};
  const float s = warp_sums<2>(v);  // lanes 0-15 have the first sum, 16-31 the second
  if constexpr (NW == 1) {
    failed = __any_sync(0xffffffffu, failed);
    __syncwarp();
    a = __shfl_sync(0xffffffffu, s, 0);
    b = __shfl_sync(0xffffffffu, s, 16);
  } else {
    const int wp = warp_id() - team * NW;
    if ((lane_id() & 15) == 0) slot[(lane_id() >> 4) * NW + wp] = s;
    int any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(static_cast<int>(failed)), "r"(1 + team), "n"(NW * 32)
        : "memory");
    failed = any != 0;
    if constexpr (NW <= 8) {
      a = slot[0];
      b = slot[NW];
#pragma unroll
      for (int i = 1; i < NW; ++i) {
        a += slot[i];
        b += slot[NW + i];
      }
    } else {
      a = warp_add(lane_id() < NW ? slot[lane_id()] : 0.f);
      b = warp_add(lane_id() < NW ? slot[NW + lane_id()] : 0.f);
    }
  }
}

// Rows of whole aligned groups of eight, of which two at least fit in shared memory: each team keeps
// a ring of rows (x, dy, dres) there, filled by bulk copies that its first lanes issue, so that the
// loads of the next rows run while a row waits for its sums.  A row's stage is free again once every
// thread has its columns in registers, which the barrier of the row's sums tells.  The weights lie
// in shared memory in fp32, in two planes of the four low and the four high columns of each group.
// 8190 x 4096 with an fp32 stream: 79 us with the join, 0.9 of the measured copy rate; 8192 x 2048 bf16
// 34 us, 0.6: a row is short against the two exchanges of its sums, and the registers hold two blocks.
template <typename TY, typename TX, int NW, int NV>
__global__ void __launch_bounds__(NW < 4 ? 128 : NW * 32, NW < 4 ? 4 : NW <= 16 ? 16 / NW : 1)
    layernorm_bwd_ring_kernel(const LnBwd a, int stages) {
  constexpr int P = 4, NT = NW * 32;
  constexpr int kTeams = NW < 4 ? 4 / NW : 1;
  constexpr int kMaxStages = 4;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t full[kTeams][kMaxStages];
  __shared__ float red[kTeams][2][2 * NW];
  __shared__ int abort_flag;
  let_next_start();
  const int H = a.H, rows = a.rows;
  const int team = threadIdx.x / NT, tid = threadIdx.x % NT;
  const float inv_h = 1.f / static_cast<float>(H);
  const int at_dy = H * static_cast<int>(sizeof(TX));
  const int at_res = at_dy + H * static_cast<int>(sizeof(TY));
  const bool res = a.dres != nullptr;
  const int stage_bytes = at_res + (res ? at_dy : 0);
  uint8_t* ring = ring_all + static_cast<size_t>(team) * stages * stage_bytes;
  float* weights = reinterpret_cast<float*>(ring_all + static_cast<size_t>(kTeams) * stages * stage_bytes);
  if (tid < stages) mbar_init(smem_u32(&full[team][tid]), 1);
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  __syncthreads();

  const int step = gridDim.x * kTeams;
  const int first = blockIdx.x * kTeams + team;
  const auto id_of = [&](int r) { return r < rows ? (a.row_ids ? a.row_ids[r] : r) : 0; };
  // Row r, whose row of x is src, into stage s: lane 0 copies x, 1 dy and 2 dres.
  const uint8_t* lane_base = static_cast<const uint8_t*>(a.x);
  long long lane_ld = a.ld_x * static_cast<int>(sizeof(TX));
  int lane_at = 0, lane_bytes = at_dy;
  if (tid == 1) {
    lane_base = static_cast<const uint8_t*>(a.dy);
    lane_ld = a.ld_dy * static_cast<int>(sizeof(TY));
    lane_at = at_dy;
    lane_bytes = at_res - at_dy;
  } else if (tid == 2) {
    lane_base = static_cast<const uint8_t*>(a.dres);
    lane_ld = a.ld_res * static_cast<int>(sizeof(TX));
    lane_at = at_res;
  }
  const auto fetch = [&](int r, int src, int s) {
    const uint32_t bar = smem_u32(&full[team][s]);
    const bool ok = src >= 0 && src < a.n_rows;
    if (tid == 0) {
      if (ok) {
        mbar_arrive_expect_tx(bar, stage_bytes);
      } else {  // nothing of it is read
        mbar_arrive(bar);
        if (a.err) atomicCAS(a.err, 0, kErrBounds);
      }
    }
    if (ok && lane_base)
      bulk_load(smem_u32(ring + static_cast<size_t>(s) * stage_bytes + lane_at),
                lane_base + (tid ? r : src) * lane_ld, lane_bytes, bar);
  };
  int fetch_id = 0;  // the id of the next row to be fetched, read one row ahead
  if (tid < 3) {
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
  for (int c = threadIdx.x * 8; c < H; c += blockDim.x * 8) {
    Pack<TY, 8> w;
    if (a.w) w = load_pack<TY, 8>(static_cast<const TY*>(a.w) + c);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      weights[c / 2 + (i & 3) + ((i & 4) ? H / 2 : 0)] = a.w ? to_f32(w.v[i]) : 1.f;
  }
  __syncthreads();

  F2 s_w[NV][P], s_b[NV][P];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) s_w[k][i] = s_b[k][i] = f2(0.f);

  // the row at hand, read one row ahead: its id (-1: out of range) and statistics
  int next = -1;
  float mu = 0.f, rs = 0.f;
  const auto read_row = [&](int id) {
    next = id >= 0 && id < a.n_rows ? id : -1;
    mu = next < 0 ? 0.f : a.mean[next];
    rs = next < 0 ? 0.f : a.rstd[next];
  };
  const int first_id = id_of(first);
  int ahead = id_of(first + step);
  read_row(first_id);

  int s = 0, phase = 0, turn = 0;
  bool failed = false;
  TX* dx = static_cast<TX*>(a.dx);
  for (int r = first; r < rows; r += step, ++turn) {
    failed = !mbar_wait(smem_u32(&full[team][s]), phase, &abort_flag, a.err, kErrWaitProducer);
    const int src = next;
    const float row_rs = rs;
    const F2 shift = f2(-mu);
    read_row(ahead);
    ahead = id_of(r + 2 * step);
    const uint8_t* st = ring + static_cast<size_t>(s) * stage_bytes;
    const int done = s;
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
    F2 n[NV][P], g[NV][P];
    Pack<TX, 8> extra[NV];
    F2 sum_g = f2(0.f), sum_gn = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * NT) * 8;
      if (c >= H || src < 0) continue;
      unpack_f2<TX, 8>(shared_pack(reinterpret_cast<const TX*>(st) + c), n[k]);
      unpack_f2<TY, 8>(shared_pack(reinterpret_cast<const TY*>(st + at_dy) + c), g[k]);
      if (res) extra[k] = shared_pack(reinterpret_cast<const TX*>(st + at_res) + c);
      const float4 lo = *reinterpret_cast<const float4*>(weights + c / 2);
      const float4 hi = *reinterpret_cast<const float4*>(weights + H / 2 + c / 2);
      const F2 w[P] = {f2(lo.x, lo.y), f2(lo.z, lo.w), f2(hi.x, hi.y), f2(hi.z, hi.w)};
#pragma unroll
      for (int i = 0; i < P; ++i) {
        n[k][i] = (n[k][i] + shift) * f2(row_rs);
        s_w[k][i] = fma2(g[k][i], n[k][i], s_w[k][i]);
        s_b[k][i] = s_b[k][i] + g[k][i];
        g[k][i] = g[k][i] * w[i];
        sum_g = sum_g + g[k][i];
        sum_gn = fma2(g[k][i], n[k][i], sum_gn);
      }
    }
    float m1 = sum2(sum_g), m2 = sum2(sum_gn);
    pair_sums<NW>(m1, m2, red[team][turn & 1], team, failed);
    if (failed) break;
    if (tid < 3 && r + stages * step < rows) {
      fetch(r + stages * step, fetch_id, done);
      fetch_id = id_of(r + (stages + 1) * step);
    }
    const F2 c0 = f2(-m1 * inv_h), c1 = f2(-m2 * inv_h);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (tid + k * NT) * 8;
      if (c >= H) continue;
      F2 o[P];
#pragma unroll
      for (int i = 0; i < P; ++i) o[i] = f2(0.f);
      if (src >= 0) {
        if (res) unpack_f2<TX, 8>(extra[k], o);
#pragma unroll
        for (int i = 0; i < P; ++i)
          o[i] = fma2(fma2(n[k][i], c1, g[k][i] + c0), f2(row_rs), o[i]);
      }
      store_f2<TX, 8>(dx + static_cast<long long>(r) * H + c, o);
    }
  }
  if (failed && tid == 0) {  // no copy may land in this memory after the block has ended
    volatile int never = 0;
    for (int i = 0; i < stages; ++i)
      if (first + (turn + i) * step < rows)
        mbar_wait(smem_u32(&full[team][(turn + i) % stages]), ((turn + i) / stages) & 1, &never,
                  nullptr, 0);
  }

  float* mine = a.part + 2ll * blockIdx.x * H;
  if constexpr (kTeams > 1) {  // the teams' sums, in the order of the teams
    float* sums = reinterpret_cast<float*>(ring_all);  // [kTeams][H], in the place of the rows
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
        WideCols::put(sums + team * H, (tid + k * NT) * 8, H, which ? s_b[k] : s_w[k]);
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
      WideCols::store(mine, c, H, s_w[k]);
      WideCols::store(mine + H, c, H, s_b[k]);
    }
  }
}

// Any width and alignment: a team of NW warps (the block, or, where NW < 8, one of 8 / NW in it) has
// a row in registers; the rows of its next turn are on their way to the L2 cache.
template <typename C, typename TY, typename TX, int NW, int NV>
__global__ void __launch_bounds__(NW < 8 ? 256 : NW * 32) layernorm_bwd_kernel(const LnBwd a) {
  constexpr int P = C::P;
  constexpr int kTeams = NW < 8 ? 8 / NW : 1;
  __shared__ float red[kTeams][2][2 * NW];
  extern __shared__ float sums[];  // [kTeams][H] where there are several teams
  let_next_start();
  const int H = a.H;
  const int team = kTeams > 1 ? warp_id() / NW : 0;
  const int tid = kTeams > 1 ? threadIdx.x % (NW * 32) : threadIdx.x;
  const float inv_h = 1.f / static_cast<float>(H);
  const TX* x = static_cast<const TX*>(a.x);
  const TY* dy = static_cast<const TY*>(a.dy);
  const TX* dres = static_cast<const TX*>(a.dres);
  F2 s_w[NV][P], s_b[NV][P];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) s_w[k][i] = s_b[k][i] = f2(0.f);
  const int step = gridDim.x * kTeams;
  int turn = 0;
  for (int r = blockIdx.x * kTeams + team; r < a.rows; r += step, ++turn) {
    if (tid == 0 && r + step < a.rows) {
      const long long ahead = a.row_ids ? a.row_ids[r + step] : r + step;
      if (ahead >= 0 && ahead < a.n_rows)
        prefetch_l2(x + ahead * a.ld_x, H * static_cast<int>(sizeof(TX)));
      prefetch_l2(dy + (r + step) * a.ld_dy, H * static_cast<int>(sizeof(TY)));
      if (dres) prefetch_l2(dres + (r + step) * a.ld_res, H * static_cast<int>(sizeof(TX)));
    }
    long long src = a.row_ids ? a.row_ids[r] : r;
    const bool ok = index_in(src, a.n_rows, a.err);
    if (!ok) src = 0;
    const int width = ok ? H : 0;  // without a row everything of it is zero
    const float rs = ok ? a.rstd[src] : 0.f, shift = ok ? -a.mean[src] : 0.f;
    F2 n[NV][P], g[NV][P];
    F2 sum_g = f2(0.f), sum_gn = f2(0.f);
    typename C::template Raw<TX> xr[NV], er[NV];
    typename C::template Raw<TY> gr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = C::column(tid, k);
      xr[k] = C::load(x + src * a.ld_x, c, width);
      gr[k] = C::load(dy + r * a.ld_dy, c, width);
      if (dres) er[k] = C::load(dres + r * a.ld_res, c, width);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = C::column(tid, k);
      F2 w[P];
#pragma unroll
      for (int i = 0; i < P; ++i) w[i] = f2(1.f);
      if (a.w) C::template unpack<TY>(C::load(static_cast<const TY*>(a.w), c, H), w);
      C::template unpack<TX>(xr[k], n[k]);
      C::template unpack<TY>(gr[k], g[k]);
#pragma unroll
      for (int i = 0; i < P; ++i) {  // behind the row's end dy is zero, and so is all that is summed
        n[k][i] = (n[k][i] + f2(shift)) * f2(rs);
        s_w[k][i] = fma2(g[k][i], n[k][i], s_w[k][i]);
        s_b[k][i] = s_b[k][i] + g[k][i];
        g[k][i] = g[k][i] * w[i];
        sum_g = sum_g + g[k][i];
        sum_gn = fma2(g[k][i], n[k][i], sum_gn);
      }
    }
    float m1 = sum2(sum_g), m2 = sum2(sum_gn);
    bool failed = false;
    pair_sums<NW>(m1, m2, red[team][turn & 1], team, failed);
    const F2 c0 = f2(-m1 * inv_h), c1 = f2(-m2 * inv_h);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      F2 o[P];
#pragma unroll
      for (int i = 0; i < P; ++i) o[i] = f2(0.f);
      if (dres) C::template unpack<TX>(er[k], o);
#pragma unroll
      for (int i = 0; i < P; ++i) o[i] = fma2(fma2(n[k][i], c1, g[k][i] + c0), f2(rs), o[i]);
      C::store(static_cast<TX*>(a.dx) + static_cast<long long>(r) * H, C::column(tid, k), H, o);
    }
  }
  float* mine = a.part + 2ll * blockIdx.x * H;
  if constexpr (kTeams > 1) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
        C::put(sums + team * H, C::column(tid, k), H, which ? s_b[k] : s_w[k]);
      __syncthreads();
      for (int c = threadIdx.x; c < H; c += 256) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kTeams; ++i) t += sums[i * H + c];
        mine[which * H + c] = t;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      C::store(mine, C::column(tid, k), H, s_w[k]);
      C::store(mine + H, C::column(tid, k), H, s_b[k]);
    }
  }
}

// dw (blockIdx.y = 0) and db from the blocks' column sums, in block order.  Block: 32 columns x 32
// slices of the blocks.
__global__ void __launch_bounds__(1024) layernorm_join_kernel(const float* part, int blocks, int H,
                                                              float* dw, float* db, int add) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  after_previous();
  float* out = blockIdx.y ? db : dw;
  if (out == nullptr) return;
  float s = 0.f;
  if (c < H) {
#pragma unroll 8
    for (int b = ry; b < blocks; b += 32) s += part[(2ll * b + blockIdx.y) * H + c];
  }
  red[ry][cx] = s;
  __syncthreads();
  s = warp_add(red[cx][ry]);  // warp ry: the 32 slices of column blockIdx.x * 32 + ry
  const int col = blockIdx.x * 32 + ry;
  if (cx == 0 && col < H) out[col] = (add ? out[col] : 0.f) + s;
}

// f(TypeTag<TY>, TypeTag<TX>): the normalised rows have the output's type or fp32.
template <typename F>
int with_row_types(int type, int x_type, F&& f) {
  return with_type(type, [&](auto ty) {
    using TY = typename decltype(ty)::type;
    if (x_type == type) return f(TypeTag<TY>(), TypeTag<TY>());
    if (x_type == kF32) return f(TypeTag<TY>(), TypeTag<float>());
    return -12;
  });
}

}  // namespace cfb

using namespace cfb;

namespace {
struct LnFwd {
  const void* x;
  long long ld_x;
  const void *w, *b;
  float eps;
  void* y;
  long long ld_y;
  float *mean, *rstd;
  int rows, H;
};
template <typename TY, typename TX, int NW, int NV, int R>
int launch_fwd(const LnFwd& a, cudaStream_t st) {
  const int teams = (a.rows + R - 1) / R;
  const int threads = NW == 1 ? 128 : ((a.H + 8 * NV - 1) / (8 * NV) + 31) / 32 * 32;
  layernorm_fwd_kernel<TY, TX, NW, NV, R><<<NW == 1 ? (teams + 3) / 4 : teams, threads, 0, st>>>(
      static_cast<const TX*>(a.x), a.ld_x, static_cast<const TY*>(a.w),
      static_cast<const TY*>(a.b), a.eps, static_cast<TY*>(a.y), a.ld_y, a.mean, a.rstd, a.rows,
      a.H);
  return launch_status();
}
template <typename TY, typename TX, int W, int NW, int NV>
int launch_fwd_pairs(const LnFwd& a, cudaStream_t st) {
  layernorm_fwd_pairs_kernel<TY, TX, W, NW, NV>
      <<<NW == 1 ? (a.rows + 3) / 4 : a.rows, NW == 1 ? 128 : NW * 32, 0, st>>>(
          static_cast<const TX*>(a.x), a.ld_x, static_cast<const TY*>(a.w),
          static_cast<const TY*>(a.b), a.eps, static_cast<TY*>(a.y), a.ld_y, a.mean, a.rstd,
          a.rows, a.H);
  return launch_status();
}
// The widest access that all rows of the operator allow.
template <typename F>
int widest(F&& rows_allow) {
  return rows_allow(8) ? 8 : rows_allow(2) ? 2 : 1;
}

template <typename C, typename TY, typename TX, int NW, int NV>
int launch_bwd(const LnBwd& b, cudaStream_t st) {
  constexpr int kTeams = NW < 8 ? 8 / NW : 1;
  auto* kernel = layernorm_bwd_kernel<C, TY, TX, NW, NV>;
  const int smem = kTeams > 1 ? kTeams * b.H * 4 : 0;
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
  kernel<<<blocks, NW < 8 ? 256 : NW * 32, smem, st>>>(b);
  const int rc = launch_status();
  return rc ? rc : blocks;
}

constexpr int kRingBytes = 220 * 1024;  // shared memory of an SM that the rings may take

// The ring kernel where two rows a team fit; 0 where they do not.
template <typename TY, typename TX, int NW, int NV>
int launch_ring(const LnBwd& b, cudaStream_t st) {
  constexpr int kTeams = NW < 4 ? 4 / NW : 1;
  constexpr int threads = NW < 4 ? 128 : NW * 32;  // 16 warps of 128 registers an SM
  auto* kernel = layernorm_bwd_ring_kernel<TY, TX, NW, NV>;
  const int row = b.H * static_cast<int>(sizeof(TY) + sizeof(TX) * (b.dres ? 2 : 1)) * kTeams;
  const int weights = 4 * b.H;
  int per_sm = 512 / threads, stages = 0;
  for (; per_sm > 0; --per_sm) {
    stages = (kRingBytes / per_sm - weights) / row;
    if (stages >= 2) break;
  }
  if (per_sm == 0) return 0;
  if (stages > 4) stages = 4;
  int smem = stages * row + weights;
  if (kTeams > 1 && smem < kTeams * b.H * 4) smem = kTeams * b.H * 4;  // the teams' sums at the end
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
  kernel<<<blocks, threads, smem, st>>>(b, stages);
  const int rc = launch_status();
  return rc ? rc : blocks;
}
}  // namespace

int cfb_layernorm_fwd(const void* x, int x_type, long long ld_x, const void* w, const void* b,
                      int type, float eps, void* y, long long ld_y, float* mean, float* rstd,
                      int rows, int H, cudaStream_t st) {
  if (rows == 0) return 0;
  if (H == 0) {  // the mean of nothing: all bits set are a NaN
    return cudaMemsetAsync(mean, 0xff, 4ll * rows, st) == cudaSuccess &&
                   cudaMemsetAsync(rstd, 0xff, 4ll * rows, st) == cudaSuccess
               ? 0
               : -3;
  }
  if (H > kLayerNormMaxH) return -11;
  const LnFwd a = {x, ld_x, w, b, eps, y, ld_y, mean, rstd, rows, H};
  const int W = widest([&](int n) {
    return H % n == 0 && rows_of(n, x, ld_x, x_type) && rows_of(n, w, 0, type) &&
           rows_of(n, b, 0, type) && rows_of(n, y, ld_y, type);
  });
  return with_row_types(type, x_type, [&](auto ty, auto tx) {
    using TY = typename decltype(ty)::type;
    using TX = typename decltype(tx)::type;
#define CFB_FWD(NW, NV, R) return launch_fwd<TY, TX, NW, NV, R>(a, st)
    if (W == 8) {
      if (rows >= 148 * 8 && sizeof(TX) == 2) {  // several rows a team pay with blocks enough
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
      if constexpr (sizeof(TY) == 4) {  // (4096 x 8192: 45 us, 67 with 16 warps; 16-bit outputs 39 and 37)
        if (H <= 8192) CFB_FWD(8, 4, 1);
      } else {
        if (H <= 8192) CFB_FWD(16, 2, 1);
      }
      CFB_FWD(32, 2, 1);
    }
#undef CFB_FWD
#define CFB_FWD(NW, NV)                                          \
  return W == 2 ? launch_fwd_pairs<TY, TX, 2, NW, NV>(a, st)     \
                : launch_fwd_pairs<TY, TX, 1, NW, NV>(a, st)
    if (H <= 256) CFB_FWD(1, 4);
    if (H <= 1024) CFB_FWD(4, 4);
    if (H <= 2048) CFB_FWD(4, 8);
    if (H <= 4096) CFB_FWD(8, 8);
    if (H <= 8192) CFB_FWD(16, 8);
    CFB_FWD(32, 8);
#undef CFB_FWD
  });
}

long long cfb_layernorm_bwd_workspace(int rows, int H) {
  const long long blocks = rows < 148 * 8 ? rows : 148 * 8;
  return 4ll * 2 * blocks * H;  // bytes
}

int cfb_layernorm_bwd(const void* dy, int type, long long ld_dy, const void* x, int x_type,
                      long long ld_x, const float* mean, const float* rstd, const void* w,
                      const void* dres, long long ld_res, const int* row_ids, long long n_rows,
                      void* dx, float* dw, float* db, int add, void* work, int rows, int H,
                      int* err, cudaStream_t st) {
  if (H == 0) return 0;
  if (H > kLayerNormMaxH) return -11;
  const int W = widest([&](int n) {
    return H % n == 0 && rows_of(n, x, ld_x, x_type) && rows_of(n, dy, ld_dy, type) &&
           rows_of(n, dres, ld_res, x_type) && rows_of(n, w, 0, type) && rows_of(n, dx, H, x_type);
  });
  float* part = static_cast<float*>(work);
  const LnBwd b = {dy, ld_dy, x, ld_x, mean, rstd, w, dres, ld_res, row_ids,
                   n_rows, dx, part, rows, H, err};
  return with_row_types(type, x_type, [&](auto ty, auto tx) {
    using TY = typename decltype(ty)::type;
    using TX = typename decltype(tx)::type;
    const auto launch = [&]() -> int {
      if (W == 8) {
#define CFB_RING(NW, NV) blocks = launch_ring<TY, TX, NW, NV>(b, st)
        int blocks = 0;
        if (H <= 256) CFB_RING(1, 1);
        else if (H <= 512) CFB_RING(2, 1);
        else if (H <= 1024) CFB_RING(4, 1);
        else if (H <= 2048) CFB_RING(4, 2);
        else if (H <= 4096) CFB_RING(8, 2);
        else if (H <= 8192) CFB_RING(16, 2);
#undef CFB_RING
        if (blocks != 0) return blocks;
        if (H <= 8192) return launch_bwd<WideCols, TY, TX, 32, 1>(b, st);
        return launch_bwd<WideCols, TY, TX, 32, 2>(b, st);
      }
#define CFB_BWD(NW, NV)                                                     \
  return W == 2 ? launch_bwd<PairCols<2, NW * 32>, TY, TX, NW, NV>(b, st) \
                : launch_bwd<PairCols<1, NW * 32>, TY, TX, NW, NV>(b, st)
      if (H <= 256) CFB_BWD(1, 4);
      if (H <= 1024) CFB_BWD(4, 4);
      if (H <= 2048) CFB_BWD(8, 4);
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
    if (!dw && !db) return 0;
    return launch_behind(layernorm_join_kernel, dim3((H + 31) / 32, db ? 2 : 1), dim3(1024), 0, st,
                         part, blocks, H, dw, db, add);
  });
}

// Distillation from a teacher's top logits beside the labels' cross entropy (sm_100a).
//
// A student's logits z (V of them) and temperature tau give q = softmax(z / tau).  The teacher names
// K tokens j with logits t_j:
//
//   without its lse:  p_j = exp(t_j / tau - norm), norm the log of their sum        (sum p = 1)
//     kd = sum p_j (log p_j - log q_j)                 dkd/dz_v = (q_v - p_v) / tau
//   with the lse of all its logits / tau as norm:  left = 1 - sum p is the share of all other tokens,
//     kd += left (log left - log q_rest), q_rest the student's share of them; there, with
//     s_v = q_v / q_rest,                              dkd/dz_v = s_v (q_rest - left) / tau
//
// (Where the list is the whole vocabulary there is no q_rest, the term is left out, and q_v counts
// with the sum of the p alone.)
//
// Beside it ce = lse(z) - z_label, dce/dz = softmax(z) - onehot.  The other tokens' sum is formed
// over them alone (the whole minus the listed would lose it), a row's statistics are
//   stats = (log sum exp(z / tau), the same of the tokens outside the list, q_rest - left (times what
//            makes up for the rounding of a far logarithm before it), norm)
// (without the teacher's lse: (lse, lse, 1, norm)), so that the gradient reads each logit once and
// takes one exponential for either loss.
//
// Bound by memory: the forward reads the logits once, the backward reads and writes them once.
// Exponentials are base 2 with the temperature folded into one multiplication; log q_j uses the same
// rounded factor as the sum, and the terms of the list are formed in 64 bits, since kd is a small
// difference of large logarithms.
#include "row_types.cuh"

namespace cfb {

constexpr float kL2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;
// From here on fp32 has no digits behind the point, and the logarithm of a sum does not say by how much
// it differs from its largest term: a rest that lies so far below the list counts as none, and an
// exponential relative to such a logarithm as zero.  Ordinary logits stay far below; masks do not.
constexpr float kNoDigits = 8388608.f;  // 2^23
// The lowest binary exponent: finite logits below it (masks by the type's lowest value, whose product
// with the temperature may overflow) count as being there.
constexpr float kLowest = -1073741824.f;  // -2^30
__device__ __forceinline__ float exponent(float z, float scale) {
  return fmaxf(__fmul_rn(z, scale), kLowest);  // rounded, as all that uses it
}
// A row is streamed by four warps, seven such blocks to an SM: while some wait for their list or sums,
// others stream.  Of 16384 x 32000 bf16 logits with tail and labels at tau = 2 (161 us at the measured
// copy rate) the forward takes 198 us in bursts of eight calls, and 215 to 223 in a loop, whose power
// takes the clock from 1.97 to 1.64 GHz, since it is bound by issue slots; without tail and labels 177
// and 189; the gradient of 8192 rows (161 us) 177 in both.  When the shape was chosen the first and the
// last were 213 and 181; with eight warps and four blocks an SM 237 and 193, with two and twelve 212 and
// 192, with six blocks of four (more registers) 210 and 185.  At the 56 registers of seven blocks the
// fp32 gradients spill 56 to 152 bytes, and forwards with an exponential of their own up to 88.
constexpr int kThreads = 128;          // the streaming warps'
constexpr int kBlock = kThreads + 32;  // ... and the lister's
constexpr int kBlocksPerSm = 7;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct ListView {
  const void* ids;
  long long ld_ids;
  int ids64;
  const void* top;
  long long ld_top;
  int top_type;
  int K;
  __device__ __forceinline__ long long id(long long row, int j) const {
    const long long at = row * ld_ids + j;
    return ids64 ? static_cast<const long long*>(ids)[at] : static_cast<const int*>(ids)[at];
  }
  __device__ __forceinline__ float logit(long long row, int j) const {
    const long long at = row * ld_top + j;
    if (top_type == kF32) return static_cast<const float*>(top)[at];
    if (top_type == kBF16) return to_f32(static_cast<const __nv_bfloat16*>(top)[at]);
    return to_f32(static_cast<const __half*>(top)[at]);
  }
};

struct DistillArgs {
  const void* z;
  long long ld;
  int V;
  ListView list;
  const float* top_lse;
  const long long* labels;
  float inv_temp;
  double inv_temp64;  // for the teacher's few terms
  int* err;
};

// How exp(z) comes beside exp(z / tau): not wanted or the same; an exponential of its own; the square
// of the other (tau = 2), which halves the exponentials of a kernel that they would bind.
enum { kOneNone = 0, kOneOwn = 1, kOneSquare = 2 };

// The running sums of one thread: of exp2(z c - ref) over the tokens outside the list (or over all),
// over the listed ones, and of exp2(z log2 e - ref1) (or of the squares of the others) over all.
template <int ONE>
struct Sums {
  float max = -INFINITY, ref = kLowest, ref1 = kLowest;
  float rest = 0.f, listed = 0.f, one = 0.f;
  // moves the references to a new maximum
  __device__ __forceinline__ void raise(float m, float c) {
    if (!(m > max)) return;
    max = m;
    const float r = exponent(m, c), f = ex2(ref - r);
    rest *= f;
    listed *= f;
    ref = r;
    if (ONE == kOneOwn) {
      const float r1 = exponent(m, kL2e);
      one *= ex2(ref1 - r1);
      ref1 = r1;
    }
    if (ONE == kOneSquare) one *= f * f;
  }
};

// What the gradient's exponentials relative to a logarithm count from; a far one leaves none of them.
__device__ __forceinline__ float reference(float log_sum) {
  return fabsf(log_sum) >= kNoDigits ? 3e38f : log_sum * kL2e;
}
// A listed logit's or the label's binary exponent, in 64 bits.
__device__ __forceinline__ double listed_exponent(float z, float scale) {
  const double x = static_cast<double>(z) * scale;
  return x < kLowest && z > -INFINITY ? kLowest : x;
}

// Eight logits as they lie in memory: -inf in all places, or in those whose bits are set; the largest.
__device__ __forceinline__ uint32_t ninf2(__nv_bfloat16) { return 0xff80ff80u; }
__device__ __forceinline__ uint32_t ninf2(__half) { return 0xfc00fc00u; }
template <typename T>
__device__ __forceinline__ void set_ninf(Pack<T, 8>& k) {
  uint32_t* u = reinterpret_cast<uint32_t*>(&k);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(k) / 4); ++i)
    if constexpr (sizeof(T) == 4) u[i] = 0xff800000u;
    else u[i] = ninf2(T());
}
template <typename T>
__device__ __forceinline__ void mask_out(Pack<T, 8>& k, uint32_t bits) {
  uint32_t* u = reinterpret_cast<uint32_t*>(&k);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = bits >> i & 1u ? 0xff800000u : u[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = (bits >> (2 * i) & 1u ? 0xffffu : 0u) |
                         (bits >> (2 * i + 1) & 1u ? 0xffff0000u : 0u);
      u[i] = (u[i] & ~m) | (ninf2(T()) & m);
    }
  }
}
template <typename T, int U>
__device__ __forceinline__ float packs_max(const Pack<T, 8>* k) {
  if constexpr (std::is_same<T, float>::value) {
    float m = k[0].v[0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, k[u].v[i]);
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m = reinterpret_cast<const T2*>(&k[0])[0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2(m, reinterpret_cast<const T2*>(&k[u])[i]);
    return fmaxf(to_f32(m.x), to_f32(m.y));
  }
}

// The part of a row that a block has, in columns from v0: single columns up to the first boundary of a
// pack (`head`), packs of eight, and the columns behind them.
template <typename T>
struct Span {
  const T* z;
  int n, head, packs;
  __device__ __forceinline__ Span(const T* at, int n) : z(at), n(n) {
    constexpr int kAlign = 8 * sizeof(T);
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(at) % kAlign);
    head = min(n, odd ? (kAlign - odd) / static_cast<int>(sizeof(T)) : 0);
    packs = (n - head) / 8;
  }
  __device__ __forceinline__ int tail() const { return head + packs * 8; }
  __device__ __forceinline__ Pack<T, 8> pack(int i) const { return load_pack<T, 8>(z + head + i * 8); }
};

// A row to a block (or, split over its columns, to a cluster of up to eight): four warps stream the
// logits, a fifth reads the list, marks its tokens in a bit mask in shared memory for the others, and
// forms the teacher's terms in 64 bits while they work.
template <typename T, bool REST, int ONE>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm) distill_fwd_kernel(
    const DistillArgs p, int splits, int chunk, float* __restrict__ kd, float* __restrict__ ce,
    float* __restrict__ lse, float* __restrict__ stats) {
  constexpr int U = sizeof(T) == 2 ? 4 : 2;  // packs of eight in flight, and as many at work
  constexpr int kWarps = kThreads / 32 + 1;
  extern __shared__ uint32_t dyn[];
  __shared__ float red[kWarps][4];
  __shared__ float joined[5];  // this block's sums of the rest and of the list, behind their maxima, and one
  const int K = p.list.K, tid = threadIdx.x, lane = lane_id();
  const bool lister = tid >= kThreads;
  float* sm_t = reinterpret_cast<float*>(dyn);
  float* sm_z = sm_t + K;
  uint32_t* flags = reinterpret_cast<uint32_t*>(sm_z + K);  // 1: an entry, 2: its token's first; id * 4
  uint32_t* bits = flags + K;
  const long long row = blockIdx.x / splits;
  const int rank = blockIdx.x % splits;
  const int v0 = rank * chunk, n = max(0, min(p.V - v0, chunk));
  const T* z = static_cast<const T*>(p.z) + row * p.ld;
  const T* mine = z + v0;
  const Span<T> span(mine, n);
  const int head = span.head, packs = span.packs;
  const int shift = 8 - head;  // bit of column i (from v0): i + shift, so a pack's bits are a byte
  const float c = p.inv_temp * kL2e;

  constexpr int S = U * kThreads;  // packs of a step
  const auto load = [&](int first, Pack<T, 8>* k) {
    if (first + S <= packs) {
#pragma unroll
      for (int u = 0; u < U; ++u) k[u] = span.pack(first + u * kThreads + tid);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = first + u * kThreads + tid;
        if (at < packs) k[u] = span.pack(at);
        else set_ninf<T>(k[u]);
      }
    }
  };
  Pack<T, 8> now[U];
  long long id0 = -1;  // the list's first ids are on their way with the first logits
  if (!lister) load(0, now);
  else if (lane < K) id0 = p.list.id(row, lane);
  if (REST) {
    for (int i = tid; i < (n + 16 + 31) / 32; i += kBlock) bits[i] = 0;
    __syncthreads();
  }
  if (lister) {
    for (int j = lane; j < K; j += 32) {
      const long long id = j < 32 ? id0 : p.list.id(row, j);
      uint32_t f = 0;
      if (id >= 0 && index_in(id, p.V, p.err)) {
        f = 1;
        const long long i = id - v0;
        if (REST && i >= 0 && i < n) {
          const int b = static_cast<int>(i) + shift;
          const uint32_t bit = 1u << (b & 31);
          if (!(atomicOr(&bits[b >> 5], bit) & bit)) f = 3;
        }
      }
      flags[j] = f | static_cast<uint32_t>(id) << 2;  // (V is below 2^30)
    }
  }
  if (REST) __syncthreads();

  Sums<ONE> s;
  // the teacher's part of the divergence, its shares' sum and normaliser (rank 0's lister)
  double own = 0.0, share = 0.0, norm = 0.0, left = 0.0, log_left = 0.0;
  bool any = false, label_in = false;
  float z_label = 0.f;
  if (!lister) {
    const uint8_t* byte = reinterpret_cast<const uint8_t*>(bits);
    // columns that are no whole pack: before the first and behind the last
    const auto single = [&](int i) {
      const float v = to_f32(mine[i]);
      if (REST && (bits[(i + shift) >> 5] >> ((i + shift) & 31) & 1u)) return;
      s.raise(v, c);
      const float e = ex2(fmaf(v, c, -s.ref));
      s.rest += e;
      if (ONE == kOneOwn) s.one += ex2(fmaf(v, kL2e, -s.ref1));
      if (ONE == kOneSquare) s.one = fmaf(e, e, s.one);
    };
    if (tid < head) single(tid);
    if (tid < n - head - packs * 8) single(head + packs * 8 + tid);
    const auto use = [&](int first, Pack<T, 8>* k) {
      if (REST) {
#pragma unroll
        for (int u = 0; u < U; ++u) {  // (behind the last pack there is nothing left to mask)
          const uint32_t b = byte[min(first + u * kThreads + tid + 1, packs)];
          if (b) mask_out<T>(k[u], b);
        }
      }
      s.raise(packs_max<T, U>(k), c);
      F2 a = f2(0.f), b1 = f2(0.f);
      const F2 cc = f2(c), nr = f2(-s.ref), cl = f2(kL2e), nr1 = f2(-s.ref1);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        F2 v[4];
        unpack_f2<T, 8>(k[u], v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = halves(fma2(v[i], cc, nr));
          const F2 e = f2(ex2(x.x), ex2(x.y));
          a = a + e;
          if (ONE == kOneOwn) {
            const float2 y = halves(fma2(v[i], cl, nr1));
            b1 = b1 + f2(ex2(y.x), ex2(y.y));
          }
          if (ONE == kOneSquare) b1 = fma2(e, e, b1);
        }
      }
      s.rest += sum2(a);
      if (ONE != kOneNone) s.one += sum2(b1);
    };
    constexpr int kUnroll = REST ? 1 : 2;  // two steps with masks spill registers (186 -> 216 us at tau = 1)
#pragma unroll kUnroll
    for (int first = 0; first < packs; first += S) {
      Pack<T, 8> next[U];
      load(first + S, next);
      use(first, now);
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = next[u];
    }
  } else {
    for (int j = lane; j < K; j += 32) {
      const uint32_t f = flags[j];
      if (f & 1) {
        sm_t[j] = p.list.logit(row, j);
        sm_z[j] = to_f32(z[f >> 2]);
      }
    }
    if (REST) {  // the listed tokens, once each
      for (int j = lane; j < K; j += 32) {
        if (!(flags[j] & 2)) continue;
        const float v = sm_z[j];
        s.raise(v, c);
        const float e = ex2(fmaf(v, c, -s.ref));
        s.listed += e;
        if (ONE == kOneOwn) s.one += ex2(fmaf(v, kL2e, -s.ref1));
        if (ONE == kOneSquare) s.one = fmaf(e, e, s.one);
      }
    }
    if (rank == 0) {
      const double inv_temp = p.inv_temp64;
      float hi = -INFINITY;
      for (int j = lane; j < K; j += 32) {
        if (!(flags[j] & 1)) continue;
        any = true;
        hi = fmaxf(hi, sm_t[j]);
      }
      any = __any_sync(0xffffffffu, any);
      if (REST) {
        norm = p.top_lse[row];
      } else {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        if (hi > -INFINITY) {
          double sum = 0.0;
          for (int j = lane; j < K; j += 32)
            if (flags[j] & 1) sum += exp((static_cast<double>(sm_t[j]) - hi) * inv_temp);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          norm = hi * inv_temp + log(sum);
        } else {
          // no entry, or none with a share; a NaN among them stays one
          float bad = 0.f;
          for (int j = lane; j < K; j += 32)
            if ((flags[j] & 1) && sm_t[j] != sm_t[j]) bad = sm_t[j];
          any = __any_sync(0xffffffffu, bad != bad);
          norm = any ? static_cast<double>(NAN) : static_cast<double>(-INFINITY);
        }
      }
      if (any) {
        for (int j = lane; j < K; j += 32) {
          if (!(flags[j] & 1)) continue;
          const double log_p = sm_t[j] * inv_temp - norm;
          const double pj = exp(log_p);
          share += pj;
          if (!(pj == 0.0)) own += pj * (log_p - listed_exponent(sm_z[j], c) * kLn2);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          own += __shfl_xor_sync(0xffffffffu, own, o);
          share += __shfl_xor_sync(0xffffffffu, share, o);
        }
      }
      left = share < 1.0 ? 1.0 - share : share >= 1.0 ? 0.0 : share;
      if (REST) log_left = log(left);
      if (p.labels) {
        const long long label = p.labels[row];
        label_in = label >= 0 && index_in(label, p.V, p.err);
        if (label_in) z_label = to_f32(z[label]);
      }
    }
  }

  // the block's sums: the maximum first, then everything relative to it
  float m = s.max;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s.raise(m, c);
  const float rest = warp_add(s.rest), listed = REST ? warp_add(s.listed) : 0.f;
  const float one = ONE != kOneNone ? warp_add(s.one) : 0.f;
  if (lane == 0) {
    red[warp_id()][0] = m;
    red[warp_id()][1] = rest;
    red[warp_id()][2] = listed;
    red[warp_id()][3] = one;
  }
  __syncthreads();
  if (!lister && splits == 1) return;
  // The rest's sum and the list's keep a maximum each: relative to the other's, one that is 87 logits
  // (times the temperature) below would be lost, and with it all that is to be said of the rest.
  // Lane b: warp b's sums, or block b's, each relative to the largest maximum of them.
  float rest_top, list_top, rest_sum, list_sum, one_sum;
  const auto most = [](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  const auto moved = [](float sum, float from, float to, float scale) {
    return sum * ex2(exponent(from, scale) - exponent(to, scale));
  };
  if (lister) {
    const bool in = lane < kWarps, list_lane = REST && lane == kWarps - 1;
    const float bm = in ? red[lane][0] : -INFINITY, rm = list_lane ? -INFINITY : bm;
    rest_top = most(rm);
    rest_sum = warp_add(moved(in ? red[lane][1] : 0.f, rm, rest_top, c));
    list_top = REST ? red[kWarps - 1][0] : -INFINITY;
    list_sum = REST ? red[kWarps - 1][2] : 0.f;
    const float top = fmaxf(rest_top, list_top);
    one_sum = ONE == kOneNone ? 0.f : warp_add(moved(in ? red[lane][3] : 0.f, bm, top, kL2e));
    // nothing but masks (and -inf): they count one each
    const auto masks = [](float top, float scale) { return top > -INFINITY && __fmul_rn(top, scale) < kLowest; };
    if (masks(top, fmaxf(c, kL2e))) {
      int all = 0, listed = 0;
      for (int i = lane; i < n; i += 32) all += to_f32(mine[i]) > -INFINITY;
      for (int j = lane; REST && j < K; j += 32) listed += (flags[j] & 2) && sm_z[j] > -INFINITY;
      all = __reduce_add_sync(0xffffffffu, all);
      listed = __reduce_add_sync(0xffffffffu, listed);
      if (masks(top, c)) {
        rest_sum = all - listed;
        list_sum = listed;
      }
      if (masks(top, kL2e)) one_sum = all;
    }
  }
  if (splits > 1) {
    if (lister && lane == 0) {
      joined[0] = rest_top;
      joined[1] = rest_sum;
      joined[2] = list_top;
      joined[3] = list_sum;
      joined[4] = one_sum;
    }
    cluster_sync();
    if (lister && rank == 0) {
      const auto peer = [&](int i, float none) {
        if (lane >= splits) return none;
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(v)
                     : "r"(mapa_shared(smem_u32(&joined[i]), lane))
                     : "memory");
        return v;
      };
      const float rm = peer(0, -INFINITY), lm = peer(2, -INFINITY);
      rest_top = most(rm);
      rest_sum = warp_add(moved(peer(1, 0.f), rm, rest_top, c));
      if (REST) {
        list_top = most(lm);
        list_sum = warp_add(moved(peer(3, 0.f), lm, list_top, c));
      }
      one_sum = warp_add(moved(peer(4, 0.f), fmaxf(rm, lm), fmaxf(rest_top, list_top), kL2e));
    }
  }
  if (lister && rank == 0) {
    // the logarithms of the whole, of the rest's sum, and of the labels' sum, a lane each
    const float top = fmaxf(rest_top, list_top);
    const float ref = exponent(top, c), rest_ref = exponent(rest_top, c);
    const float rest_part = REST ? rest_sum * ex2(rest_ref - ref) : rest_sum;
    const double whole = REST ? rest_part + static_cast<double>(list_sum * ex2(exponent(list_top, c) - ref))
                              : static_cast<double>(rest_part);
    const double logs = log(lane == 0 ? whole : static_cast<double>(lane == 1 ? rest_sum : one_sum));
    const double log_all = ref * kLn2 + __shfl_sync(0xffffffffu, logs, 0);
    const double log_rest = REST ? rest_ref * kLn2 + __shfl_sync(0xffffffffu, logs, 1) : log_all;
    const double log_one = exponent(top, kL2e) * kLn2 + __shfl_sync(0xffffffffu, logs, 2);
    if (lane == 0) {
      double loss = any ? own + share * log_all : 0.0;
      double coef = REST || any ? 1.0 : 0.0;
      bool some = true;
      if (REST) {
        // tokens outside the list, not all of them at -inf or masked (a NaN among them stays one)
        some = rest_sum != 0.f && !(rest_sum > 0.f && (rest_ref - ref) * kLn2 < -kNoDigits);
        if (some && !(left == 0.0)) loss += left * (log_left - (log_rest - log_all));
        coef = some ? (share > 1.0 ? share : 1.0) * (rest_part / whole) - left : 0.0;
      }
      kd[row] = static_cast<float>(loss);
      float4 o;
      o.x = static_cast<float>(log_all);
      o.y = some ? static_cast<float>(log_rest) : -INFINITY;
      if (REST && some && fabsf(o.y) > 128.f) {
        // What multiplies the exponentials relative to this logarithm makes up for its rounding, and for
        // that of the gradient's binary exponents: 1e-5 of each term at 128, 7e-2 at 1e6.
        const double t = reference(o.y) * kLn2 - log_rest;
        coef *= fabs(t) < 0.002 ? 1.0 + t + 0.5 * t * t : fabs(t) < 2.0 ? exp(t) : 1.0;
      }
      o.z = static_cast<float>(coef);
      o.w = static_cast<float>(norm);
      reinterpret_cast<float4*>(stats)[row] = o;
      if (p.labels) {
        const double full = ONE == kOneNone ? log_all : log_one;
        lse[row] = static_cast<float>(full);
        ce[row] = label_in ? static_cast<float>(full - listed_exponent(z_label, kL2e) * kLn2) : 0.f;
      }
    }
  }
  if (splits > 1) cluster_sync();  // no block leaves while its sums are read
}

__device__ __forceinline__ F2 exp_of(F2 v, float scale, float off) {
  const float2 x = halves(fma2(v, f2(scale), f2(-off)));
  return f2(ex2(x.x), ex2(x.y));
}
// Slots of the table in which the lister finds a token that is named twice.
__host__ __device__ inline int table_slots(int K) {
  int n = 64;
  while (n < 2 * K) n *= 2;
  return n;
}

enum { kCeNone = 0, kCeOwn = 1, kCeSame = 2 };

// out = dkd dkd/dz + dce dce/dz of a row, its columns dealt to `splits` blocks.  Four warps write the
// whole range as for tokens outside the list; the lister forms the gradients of the listed tokens and
// of the label meanwhile, and writes them over it, from logits that it reads before anything is written
// (out may be the logits).
//
// At a temperature of one (kCeSame) one exponential serves both losses: softmax(z) is exp(z - base)
// times the tokens' share of the whole.
template <typename T, int CE>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm) distill_bwd_kernel(
    const DistillArgs p, const float* __restrict__ stats, const float* __restrict__ lse,
    const float* __restrict__ dkd, const float* __restrict__ dce, const int* __restrict__ row_ids,
    long long n_rows, T* out_all, long long ld_out, int splits, int chunk) {
  constexpr int U = sizeof(T) == 2 ? 4 : 2;
  constexpr int kAlign = 8 * sizeof(T);
  extern __shared__ uint32_t dyn[];
  const int K = p.list.K, tid = threadIdx.x;
  const bool lister = tid >= kThreads;
  const long long r = blockIdx.x / splits;
  const int v0 = (blockIdx.x % splits) * chunk, n = max(0, min(p.V - v0, chunk));
  long long src = row_ids ? row_ids[r] : r;
  const bool ok = src >= 0 && src < n_rows;
  if (!ok) src = 0;
  const T* z = static_cast<const T*>(p.z) + src * p.ld;
  const Span<T> span(z + v0, n);
  T* out = out_all + r * ld_out + v0;
  const bool wide = reinterpret_cast<uintptr_t>(out + span.head) % kAlign == 0;
  const auto load = [&](int first, Pack<T, 8>* k) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = first + u * kThreads + tid;
      if (at < span.packs) k[u] = span.pack(at);
    }
  };
  Pack<T, 8> now[U];
  if (!lister && wide) load(0, now);

  // the row's weights and what they multiply
  const float k = ok ? dkd[r] * p.inv_temp : 0.f;
  long long label = -1;
  float g1 = 0.f;
  if (CE && ok) {
    label = p.labels[src];
    if (label >= 0 && label < p.V) g1 = dce[r];
  }
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  if (k != 0.f) st = reinterpret_cast<const float4*>(stats)[src];
  const float gk = k * st.z;
  const bool spread = gk != 0.f && !(CE == kCeSame && fabsf(st.y) >= kNoDigits);  // also a NaN
  const float c = p.inv_temp * kL2e;
  const float ref = spread ? reference(st.y) : 0.f;
  const float ref1 = CE && g1 != 0.f ? reference(lse[src]) : 0.f;

  if (!lister) {
    const auto stream = [&](auto&& value) {
      const auto one = [&](float v) { return from_f32<T>(halves(value(f2(v))).x); };
      if (wide) {
        if (tid < span.head) out[tid] = one(to_f32(span.z[tid]));
        const int at = span.tail() + tid;
        if (at < n) out[at] = one(to_f32(span.z[at]));
        for (int first = 0; first < span.packs; first += U * kThreads) {
          Pack<T, 8> next[U];
          load(first + U * kThreads, next);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int i = first + u * kThreads + tid;
            if (i < span.packs) {
              F2 v[4];
              unpack_f2<T, 8>(now[u], v);
#pragma unroll
              for (int j = 0; j < 4; ++j) v[j] = value(v[j]);
              store_f2<T, 8>(out + span.head + i * 8, v);
            }
            now[u] = next[u];
          }
        }
      } else {  // packs of the logits and of out have their boundaries at different columns
        for (int i0 = tid; i0 < n; i0 += 8 * kThreads) {
          float v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            v[u] = i0 + u * kThreads < n ? to_f32(span.z[i0 + u * kThreads]) : 0.f;
#pragma unroll
          for (int u = 0; u < 8; u += 2) {
            const float2 g = halves(value(f2(v[u], v[u + 1])));
            if (i0 + u * kThreads < n) out[i0 + u * kThreads] = from_f32<T>(g.x);
            if (i0 + (u + 1) * kThreads < n) out[i0 + (u + 1) * kThreads] = from_f32<T>(g.y);
          }
        }
      }
    };
    // Without a divergence the one exponential is that of the labels' loss.
    const float ec = spread ? c : kL2e, er = spread ? ref : ref1;
    float ge = spread ? gk : g1;
    if (CE == kCeSame && spread && g1 != 0.f) ge = fmaf(g1, ex2(ref - ref1), gk);
    __syncthreads();  // the lister has read its logits
    if (!spread && g1 == 0.f) {
      stream([](F2) { return f2(0.f); });
    } else if (CE == kCeOwn && spread && g1 != 0.f) {
      stream([&](F2 v) {
        return fma2(f2(g1), exp_of(v, kL2e, ref1), f2(ge) * exp_of(v, ec, er));
      });
    } else {
      stream([&](F2 v) { return f2(ge) * exp_of(v, ec, er); });
    }
    __syncthreads();  // what was written above is replaced by the lister
    return;
  }

  // -------------------------------------------------------------- the lister
  const int lane = lane_id();
  if (lane == 0) {  // (recorded once a row)
    index_in(ok ? 0 : -1, 1, p.err);
    if (CE && label >= p.V) index_in(label, p.V, p.err);
  }
  int* sm_id = reinterpret_cast<int*>(dyn);           // -1: no entry
  float* sm_p = reinterpret_cast<float*>(sm_id + K);  // the teacher's logits, then its shares
  float* sm_g = sm_p + K;                             // the student's logits here, then the gradients
  int* table = reinterpret_cast<int*>(sm_g + K);
  const int slots = table_slots(K);
  // (a list without the teacher's lse and without a share says nothing)
  const int entries = k != 0.f && !(st.w == -INFINITY && st.z == 0.f) ? K : 0;
  const auto in_range = [&](long long v) { return v >= v0 && v < v0 + n; };
  for (int i = lane; entries && i < slots; i += 32) table[i] = -1;
  for (int j = lane; j < entries; j += 32) {
    const long long id = p.list.id(src, j);
    int at = -1;
    if (id >= 0 && index_in(id, p.V, p.err)) {
      at = static_cast<int>(id);
      sm_p[j] = p.list.logit(src, j);
      if (in_range(at)) sm_g[j] = to_f32(z[at]);
    }
    sm_id[j] = at;
  }
  const bool labelled = CE && g1 != 0.f;
  const bool label_here = labelled && in_range(label);
  const float z_label = label_here ? to_f32(z[label]) : 0.f;
  __syncthreads();

  // While the others stream.  The differences of two probabilities are formed in 64 bits: where the
  // student agrees with the teacher or the label, little is left of either.
  float whole = 0.f;
  bool twice = false, named = false;
  for (int j = lane; j < entries; j += 32) {
    const int at = sm_id[j];
    float pj = 0.f;
    if (at >= 0) {
      pj = static_cast<float>(exp(sm_p[j] * p.inv_temp64 - st.w));
      unsigned slot = static_cast<unsigned>(at) * 2654435761u;
      for (;; ++slot) {  // (more slots than entries: it ends)
        const int old = atomicCAS(&table[slot & (slots - 1)], -1, at);
        twice = twice || old == at;
        if (old == -1 || old == at) break;
      }
    }
    named = named || (at >= 0 && at == label);
    whole += pj;
    sm_p[j] = pj;
  }
  whole = warp_add(whole);
  // What the teacher's terms add up to: one (without its lse: by its normaliser), or, for a list of the
  // whole vocabulary, what the list's do.
  if (st.y == st.x) whole = 1.f;
  else if (st.y > -INFINITY) whole = fmaxf(whole, 1.f);
  named = __any_sync(0xffffffffu, named);
  twice = __any_sync(0xffffffffu, twice);
  __syncwarp();
  const auto from = [](float log_sum) -> double { return fabsf(log_sum) >= kNoDigits ? INFINITY : log_sum; };
  const double from_all = from(st.x), from1 = labelled ? from(lse[src]) : 0.0;
  for (int j = lane; j < entries; j += 32) {
    const int at = sm_id[j];
    if (at < 0 || !in_range(at)) continue;
    const double v = sm_g[j];
    float share = sm_p[j];
    if (twice) {  // the same token's shares, summed in the list's order by each of its entries
      share = 0.f;
      for (int i = 0; i < K; ++i) share += sm_id[i] == at ? sm_p[i] : 0.f;
    }
    double g = k * (whole * exp(v * p.inv_temp64 - from_all) - share);
    if (labelled) g += g1 * (exp(v - from1) - (at == label ? 1.0 : 0.0));
    sm_g[j] = static_cast<float>(g);
  }
  const bool label_alone = label_here && !named;
  const float label_grad =
      label_alone ? static_cast<float>((spread ? gk * exp2(static_cast<double>(z_label) * c - ref) : 0.0) +
                                       g1 * (exp(z_label - from1) - 1.0))
                  : 0.f;
  __syncthreads();  // the range is written
  for (int j = lane; j < entries; j += 32)
    if (sm_id[j] >= 0 && in_range(sm_id[j])) out[sm_id[j] - v0] = from_f32<T>(sm_g[j]);
  if (label_alone && lane == 0) out[label - v0] = from_f32<T>(label_grad);
}

}  // namespace cfb

using namespace cfb;

namespace {

DistillArgs args_of(const CfbDistill* p) {
  const ListView list = {p->ids, p->ld_ids, p->ids64, p->top, p->ld_top, p->top_type, p->K};
  return {p->z, p->ld, p->V, list, p->top_lse, p->labels,
          static_cast<float>(1.0 / p->temperature), 1.0 / p->temperature, p->err};
}

template <typename T, bool REST, int ONE>
int launch_fwd(const DistillArgs& a, float* kd, float* ce, float* lse, float* stats, int rows,
               int splits, int chunk, cudaStream_t st) {
  auto* kernel = distill_fwd_kernel<T, REST, ONE>;
  const int smem = 12 * a.list.K + (REST ? (chunk + 16 + 31) / 32 * 4 : 0);
  constexpr int kMost = 12 * kDistillMaxTop + 160 * 1024;
  static bool allowed[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  if (smem > kMost) return -11;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) !=
        cudaSuccess) {
      cudaGetLastError();
      return -3;
    }
    allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * splits);
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, a, splits, chunk, kd, ce, lse, stats) != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  ++cfb_row_launches();
  return 0;
}

// Blocks to a row: one where the rows fill `waves` waves of blocks, else up to `most` with at least
// 4096 columns each.
int splits_of(int rows, int V, int waves, int most) {
  int s = 1;
  while (s < most && rows * s < 148 * kBlocksPerSm * waves && V / (2 * s) >= 4096) s *= 2;
  return s;
}
int chunk_of(int V, int splits) { return splits == 1 ? V : (V + splits * 16 - 1) / (splits * 16) * 16; }

}  // namespace

int cfb_distill_fwd(const CfbDistill* p, float* kd, float* ce, float* lse, float* stats, int rows,
                    cudaStream_t st) {
  if (rows == 0) return 0;
  const DistillArgs a = args_of(p);
  const int splits = splits_of(rows, p->V, 1, 8);
  const int chunk = chunk_of(p->V, splits);
  const int one = !p->labels || p->temperature == 1.0 ? kOneNone
                  : p->temperature == 2.0             ? kOneSquare
                                                   : kOneOwn;
  return with_type(p->type, [&](auto tag) {
    using T = typename decltype(tag)::type;
#define CFB_FWD(REST)                                                                            \
  (one == kOneNone                                                                               \
       ? launch_fwd<T, REST, kOneNone>(a, kd, ce, lse, stats, rows, splits, chunk, st)           \
   : one == kOneOwn                                                                              \
       ? launch_fwd<T, REST, kOneOwn>(a, kd, ce, lse, stats, rows, splits, chunk, st)            \
       : launch_fwd<T, REST, kOneSquare>(a, kd, ce, lse, stats, rows, splits, chunk, st))
    return p->top_lse ? CFB_FWD(true) : CFB_FWD(false);
#undef CFB_FWD
  });
}

int cfb_distill_bwd(const CfbDistill* p, const float* stats, const float* lse, const float* dkd,
                    const float* dce, const int* row_ids, long long n_rows, void* out,
                    long long ld_out, int rows, cudaStream_t st) {
  if (rows == 0) return 0;
  const DistillArgs a = args_of(p);
  const int splits = splits_of(rows, p->V, 2, 16);
  const int chunk = chunk_of(p->V, splits);
  const int smem = 12 * p->K + 4 * table_slots(p->K);
  return with_type(p->type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    const unsigned grid = static_cast<unsigned>(rows) * splits;
    const auto launch = [&](auto* kernel) {
      kernel<<<grid, kBlock, smem, st>>>(a, stats, lse, dkd, dce, row_ids, n_rows,
                                         static_cast<T*>(out), ld_out, splits, chunk);
    };
    if (!p->labels) launch(distill_bwd_kernel<T, kCeNone>);
    else if (p->temperature == 1.0) launch(distill_bwd_kernel<T, kCeSame>);
    else launch(distill_bwd_kernel<T, kCeOwn>);
    return launch_status();
  });
}

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
//   stats = (log sum exp(z / tau), the same of the tokens outside the list, q_rest - left, norm)
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
constexpr int kThreads = 256;

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

// The running sums of one thread: of exp2(z c - ref) over the tokens outside the list (or over all),
// over the listed ones, and of exp2(z log2 e - ref1) over all.
struct Sums {
  float max = -INFINITY, ref = 0.f, ref1 = 0.f;
  float rest = 0.f, listed = 0.f, one = 0.f;
  // moves the references to a new maximum
  __device__ __forceinline__ void raise(float m, float c) {
    if (!(m > max)) return;
    const float r = __fmul_rn(m, c), r1 = __fmul_rn(m, kL2e);  // rounded, as all that uses them
    const float f = max == -INFINITY ? 0.f : ex2(ref - r);
    const float f1 = max == -INFINITY ? 0.f : ex2(ref1 - r1);
    rest *= f;
    listed *= f;
    one *= f1;
    max = m;
    ref = r;
    ref1 = r1;
  }
};

// How exp(z) comes beside exp(z / tau): not wanted or the same; an exponential of its own; the square
// of the other (tau = 2), which halves the exponentials of a kernel that they would bind.
enum { kOneNone = 0, kOneOwn = 1, kOneSquare = 2 };

template <typename T, bool REST, int ONE>
__global__ void __launch_bounds__(kThreads) distill_fwd_kernel(const DistillArgs p, int splits,
                                                               int chunk, float* __restrict__ kd,
                                                               float* __restrict__ ce,
                                                               float* __restrict__ lse,
                                                               float* __restrict__ stats) {
  constexpr int U = sizeof(T) == 2 ? 4 : 2;  // packs of eight in flight, and as many at work
  constexpr int kAlign = 8 * sizeof(T);
  extern __shared__ uint32_t dyn[];
  __shared__ float red[kThreads / 32][4];
  __shared__ float joined[4];  // this block's max, rest, listed, one
  const int K = p.list.K, tid = threadIdx.x;
  float* sm_t = reinterpret_cast<float*>(dyn);
  float* sm_z = sm_t + K;
  uint32_t* flags = reinterpret_cast<uint32_t*>(sm_z + K);  // 1: an entry, 2: the first of its token here
  uint32_t* bits = flags + K;
  const long long row = blockIdx.x / splits;
  const int rank = blockIdx.x % splits;
  const int v0 = rank * chunk, n = max(0, min(p.V - v0, chunk));
  const T* z = static_cast<const T*>(p.z) + row * p.ld;
  const T* mine = z + v0;
  const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(mine) % kAlign);
  const int head = min(n, odd ? (kAlign - odd) / static_cast<int>(sizeof(T)) : 0);
  const int packs = (n - head) / 8;
  const int shift = 8 - head;  // bit of column i (from v0): i + shift, so a pack's bits are a byte
  const float c = p.inv_temp * kL2e;

  const auto load = [&](int first, Pack<T, 8>* k) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = first + u * kThreads + tid;
      if (at < packs) k[u] = load_pack<T, 8>(mine + head + at * 8);
    }
  };
  Pack<T, 8> now[U];
  load(0, now);
  if (REST) {
    for (int i = tid; i < (n + 16 + 31) / 32; i += kThreads) bits[i] = 0;
    __syncthreads();
  }
  for (int j = tid; j < K; j += kThreads) {
    const long long id = p.list.id(row, j);
    uint32_t f = 0;
    if (id >= 0) {
      if (id < p.V) {
        f = 1;
        sm_t[j] = p.list.logit(row, j);
        sm_z[j] = to_f32(z[id]);
        const long long i = id - v0;
        if (REST && i >= 0 && i < n) {
          const int b = static_cast<int>(i) + shift;
          const uint32_t bit = 1u << (b & 31);
          if (!(atomicOr(&bits[b >> 5], bit) & bit)) f = 3;
        }
      } else if (p.err) {
        atomicCAS(p.err, 0, kErrBounds);
      }
    }
    flags[j] = f;
  }
  if (REST) __syncthreads();

  Sums s;
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
  for (int first = 0; first < packs; first += U * kThreads) {
    Pack<T, 8> next[U];
    load(first + U * kThreads, next);
    F2 v[U][4];
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = first + u * kThreads + tid;
      if (at < packs) {
        unpack_f2<T, 8>(now[u], v[u]);
        if (REST) {
          const uint32_t b = byte[at + 1];
          if (b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 h = halves(v[u][i]);
              v[u][i] = f2((b >> (2 * i)) & 1u ? -INFINITY : h.x,
                           (b >> (2 * i + 1)) & 1u ? -INFINITY : h.y);
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][i] = f2(-INFINITY);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 h = halves(v[u][i]);
        m = fmaxf(m, fmaxf(h.x, h.y));
      }
      now[u] = next[u];
    }
    s.raise(m, c);
    F2 a = f2(0.f), b1 = f2(0.f);
    const F2 cc = f2(c), nr = f2(-s.ref), cl = f2(kL2e), nr1 = f2(-s.ref1);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = halves(fma2(v[u][i], cc, nr));
        const F2 e = f2(ex2(x.x), ex2(x.y));
        a = a + e;
        if (ONE == kOneOwn) {
          const float2 y = halves(fma2(v[u][i], cl, nr1));
          b1 = b1 + f2(ex2(y.x), ex2(y.y));
        }
        if (ONE == kOneSquare) b1 = fma2(e, e, b1);
      }
    s.rest += sum2(a);
    if (ONE != kOneNone) s.one += sum2(b1);
  }
  if (REST) {  // the listed tokens, once each
    for (int j = tid; j < K; j += kThreads) {
      if (!(flags[j] & 2)) continue;
      const float v = sm_z[j];
      s.raise(v, c);
      s.listed += ex2(fmaf(v, c, -s.ref));
      if (ONE != kOneNone) s.one += ex2(fmaf(v, kL2e, -s.ref1));
    }
  }

  // the block's sums: the maximum first, then everything relative to it
  float m = s.max;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane_id() == 0) red[warp_id()][0] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, red[w][0]);
  s.raise(m, c);
  const float rest = warp_add(s.rest), listed = REST ? warp_add(s.listed) : 0.f;
  const float one = ONE != kOneNone ? warp_add(s.one) : 0.f;
  if (lane_id() == 0) {
    red[warp_id()][1] = rest;
    red[warp_id()][2] = listed;
    red[warp_id()][3] = one;
  }
  __syncthreads();
  if (tid == 0) {
    float t[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w)
#pragma unroll
      for (int i = 0; i < 3; ++i) t[i] += red[w][1 + i];
    joined[0] = m;
#pragma unroll
    for (int i = 0; i < 3; ++i) joined[1 + i] = t[i];
  }
  if (splits > 1) cluster_sync(); else __syncthreads();
  if (rank == 0 && warp_id() == 0) {
    const int lane = lane_id();
    // lane b: block b's sums
    float bm = -INFINITY, br = 0.f, bl = 0.f, bo = 0.f;
    if (lane < splits) {
      const auto peer = [&](int i) {
        if (splits == 1) return joined[i];
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(v)
                     : "r"(mapa_shared(smem_u32(&joined[i]), lane))
                     : "memory");
        return v;
      };
      bm = peer(0);
      br = peer(1);
      bl = peer(2);
      bo = peer(3);
    }
    float top = bm;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = __shfl_sync(0xffffffffu, top, 0);
    const float ref = top == -INFINITY ? 0.f : __fmul_rn(top, c);
    const float ref1 = top == -INFINITY ? 0.f : __fmul_rn(top, kL2e);
    const float f = bm == -INFINITY ? 1.f : ex2(__fmul_rn(bm, c) - ref);  // (sums of nothing are zero)
    const float f1 = bm == -INFINITY ? 1.f : ex2(__fmul_rn(bm, kL2e) - ref1);
    const double rest_sum = warp_add(br * f), list_sum = warp_add(bl * f);
    const double one_sum = warp_add(bo * f1);
    const double log_all = ref + log2(rest_sum + list_sum);  // base 2
    const double log_rest = REST ? ref + log2(rest_sum) : log_all;

    // the teacher's shares
    double norm;
    bool any = false;
    for (int j = lane; j < K; j += 32) any = any || (flags[j] & 1);
    any = __any_sync(0xffffffffu, any);
    const double inv_temp = p.inv_temp64;
    if (REST) {
      norm = p.top_lse[row];
    } else {
      float hi = -INFINITY;
      for (int j = lane; j < K; j += 32)
        if (flags[j] & 1) hi = fmaxf(hi, sm_t[j]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      double sum = 0.0;
      if (hi > -INFINITY) {
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
    double loss = 0.0, share = 0.0;
    if (any) {
      for (int j = lane; j < K; j += 32) {
        if (!(flags[j] & 1)) continue;
        const double log_p = sm_t[j] * inv_temp - norm;
        const double pj = exp(log_p);
        share += pj;
        if (!(pj == 0.0))
          loss += pj * (log_p - (static_cast<double>(sm_z[j]) * c - log_all) * kLn2);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        loss += __shfl_xor_sync(0xffffffffu, loss, o);
        share += __shfl_xor_sync(0xffffffffu, share, o);
      }
    }
    if (lane == 0) {
      double coef = REST || any ? 1.0 : 0.0;
      if (REST) {
        const double left = share < 1.0 ? 1.0 - share : share >= 1.0 ? 0.0 : share;
        const double log_q = (log_rest - log_all) * kLn2;
        const bool some = rest_sum != 0.0;  // tokens outside the list, not all of them at -inf
        if (some && !(left == 0.0)) loss += left * (log(left) - log_q);
        coef = some ? (share > 1.0 ? share : 1.0) * exp(log_q) - left : 0.0;
      }
      kd[row] = static_cast<float>(loss);
      float4 o;
      o.x = static_cast<float>(log_all * kLn2);
      o.y = static_cast<float>(log_rest * kLn2);
      o.z = static_cast<float>(coef);
      o.w = static_cast<float>(norm);
      reinterpret_cast<float4*>(stats)[row] = o;
      if (p.labels) {
        const double full = ONE == kOneNone ? log_all : ref1 + log2(one_sum);
        lse[row] = static_cast<float>(full * kLn2);
        const long long label = p.labels[row];
        float l = 0.f;
        if (label >= 0 && index_in(label, p.V, p.err))
          l = static_cast<float>((full - static_cast<double>(to_f32(z[label])) * kL2e) * kLn2);
        ce[row] = l;
      }
    }
  }
  if (splits > 1) cluster_sync();  // no block leaves while its sums are read
}

// out = dkd dkd/dz + dce dce/dz of a row, its columns dealt to `splits` blocks.  The whole range is
// written as for tokens outside the list; then the listed tokens and the label get their own values,
// from logits that were read before (out may be the logits).
template <typename T, bool CE>
__global__ void __launch_bounds__(kThreads) distill_bwd_kernel(
    const DistillArgs p, const float* __restrict__ stats, const float* __restrict__ lse,
    const float* __restrict__ dkd, const float* __restrict__ dce, const int* __restrict__ row_ids,
    long long n_rows, T* out_all, long long ld_out, int splits, int chunk) {
  constexpr int U = sizeof(T) == 2 ? 4 : 2;
  constexpr int kAlign = 8 * sizeof(T);
  extern __shared__ uint32_t dyn[];
  const int K = p.list.K, tid = threadIdx.x;
  float* sm_z = reinterpret_cast<float*>(dyn);
  float* sm_p = sm_z + K;
  int* sm_id = reinterpret_cast<int*>(sm_p + K);  // -1: not an entry
  const long long r = blockIdx.x / splits;
  const int v0 = (blockIdx.x % splits) * chunk, n = max(0, min(p.V - v0, chunk));
  long long src = row_ids ? row_ids[r] : r;
  const bool ok = index_in(src, n_rows, p.err);
  if (!ok) src = 0;
  const T* z_row = static_cast<const T*>(p.z) + src * p.ld;
  const T* z = z_row + v0;
  T* out = out_all + r * ld_out + v0;
  const float k = ok ? dkd[r] * p.inv_temp : 0.f;
  long long label = -1;
  float g1 = 0.f;
  if (CE && ok) {
    label = p.labels[src];
    if (label >= p.V) {
      index_in(label, p.V, p.err);
      label = -1;
    }
    if (label >= 0) g1 = dce[r];
    if (g1 == 0.f) label = -1;
  }
  const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(z) % kAlign);
  int head = min(n, odd ? (kAlign - odd) / static_cast<int>(sizeof(T)) : 0);
  const bool wide = reinterpret_cast<uintptr_t>(out + head) % kAlign == 0;
  if (k == 0.f && g1 == 0.f) {  // nothing comes from this row
    for (int i = tid; i < n; i += kThreads) out[i] = from_f32<T>(0.f);
    return;
  }
  const float c = p.inv_temp * kL2e;
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  if (k != 0.f) st = reinterpret_cast<const float4*>(stats)[src];
  const float gk = k * st.z;
  const bool spread = gk != 0.f;  // also a NaN
  const float ref = spread ? st.y * kL2e : 0.f;
  const float ref1 = g1 != 0.f ? lse[src] * kL2e : 0.f;
  const float all = st.x * kL2e;
  // the list, and the logits at it
  const int entries = k != 0.f ? K : 0;
  for (int j = tid; j < entries; j += kThreads) {
    const long long id = p.list.id(src, j);
    int at = -1;
    sm_p[j] = 0.f;
    if (id >= 0 && id < p.V) {
      at = static_cast<int>(id);
      sm_z[j] = to_f32(z_row[id]);
      const double pj = exp(p.list.logit(src, j) * p.inv_temp64 - st.w);
      sm_p[j] = static_cast<float>(pj);
    } else if (id >= p.V && p.err) {
      atomicCAS(p.err, 0, kErrBounds);
    }
    sm_id[j] = at;
  }
  float z_label = 0.f;
  if (CE && label >= 0) z_label = to_f32(z_row[label]);

  const auto value = [&](float v) {
    float g = spread ? gk * ex2(fmaf(v, c, -ref)) : 0.f;
    if (CE && g1 != 0.f) g = fmaf(g1, ex2(fmaf(v, kL2e, -ref1)), g);
    return g;
  };
  if (wide) {
    const int packs = (n - head) / 8;
    const int tail = head + packs * 8;
    float edge = 0.f;
    if (tid < head) edge = to_f32(z[tid]);
    if (tid >= 32 && tid - 32 < n - tail) edge = to_f32(z[tail + tid - 32]);
    Pack<T, 8> now[U];
    const auto load = [&](int first, Pack<T, 8>* d) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = first + u * kThreads + tid;
        if (at < packs) d[u] = load_pack<T, 8>(z + head + at * 8);
      }
    };
    load(0, now);
    __syncthreads();  // the listed logits are read before anything is written
    for (int first = 0; first < packs; first += U * kThreads) {
      Pack<T, 8> next[U];
      load(first + U * kThreads, next);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = first + u * kThreads + tid;
        if (at < packs) {
          F2 v[4];
          unpack_f2<T, 8>(now[u], v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            F2 g = f2(0.f);
            if (spread) {
              const float2 x = halves(fma2(v[i], f2(c), f2(-ref)));
              g = f2(gk) * f2(ex2(x.x), ex2(x.y));
            }
            if (CE) {
              const float2 y = halves(fma2(v[i], f2(kL2e), f2(-ref1)));
              if (g1 != 0.f) g = fma2(f2(g1), f2(ex2(y.x), ex2(y.y)), g);
            }
            v[i] = g;
          }
          store_f2<T, 8>(out + head + at * 8, v);
        }
        now[u] = next[u];
      }
    }
    if (tid < head) out[tid] = from_f32<T>(value(edge));
    if (tid >= 32 && tid - 32 < n - tail) out[tail + tid - 32] = from_f32<T>(value(edge));
  } else {
    __syncthreads();
    for (int i0 = tid; i0 < n; i0 += 8 * kThreads) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i0 + u * kThreads < n ? to_f32(z[i0 + u * kThreads]) : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i0 + u * kThreads < n) out[i0 + u * kThreads] = from_f32<T>(value(v[u]));
    }
  }
  __syncthreads();  // what was written above is replaced below
  const auto in_range = [&](long long v) { return v >= v0 && v < v0 + n; };
  const float soft_label = CE && label >= 0 ? ex2(fmaf(z_label, kL2e, -ref1)) : 0.f;
  for (int j = tid; j < entries; j += kThreads) {
    const int id = sm_id[j];
    if (id < 0 || !in_range(id)) continue;
    float share = 0.f, whole = 0.f;  // a token named twice: both threads form the same sum
    for (int i = 0; i < K; ++i) {
      whole += sm_p[i];
      share += sm_id[i] == id ? sm_p[i] : 0.f;
    }
    // what the teacher's terms add up to: one, but for a list of the whole vocabulary
    if (st.y > -INFINITY) whole = fmaxf(whole, 1.f);
    float g = k * fmaf(whole, ex2(fmaf(sm_z[j], c, -all)), -share);
    if (CE && g1 != 0.f) g += g1 * (ex2(fmaf(sm_z[j], kL2e, -ref1)) - (id == label ? 1.f : 0.f));
    out[id - v0] = from_f32<T>(g);
  }
  if (CE && label >= 0 && tid == kThreads - 1 && in_range(label)) {
    bool listed = false;
    for (int i = 0; i < entries; ++i) listed = listed || sm_id[i] == label;
    if (!listed) {
      const float g = spread ? gk * ex2(fmaf(z_label, c, -ref)) : 0.f;
      out[label - v0] = from_f32<T>(g + g1 * (soft_label - 1.f));
    }
  }
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
  cfg.blockDim = dim3(kThreads);
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

// Blocks to a row: one where there are rows enough for the SMs, else up to `most` with at least
// `least` columns each.
int splits_of(int rows, int V, int least, int most) {
  int s = 1;
  while (s < most && rows * s < 148 * 4 && V / (2 * s) >= least) s *= 2;
  return s;
}
int chunk_of(int V, int splits) { return splits == 1 ? V : (V + splits * 16 - 1) / (splits * 16) * 16; }

}  // namespace

int cfb_distill_fwd(const CfbDistill* p, float* kd, float* ce, float* lse, float* stats, int rows,
                    cudaStream_t st) {
  if (rows == 0) return 0;
  const DistillArgs a = args_of(p);
  const int splits = splits_of(rows, p->V, 4096, 8);
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
  const int splits = splits_of(rows, p->V, 4096, 16);
  const int chunk = chunk_of(p->V, splits);
  const int smem = 12 * p->K;
  return with_type(p->type, [&](auto tag) {
    using T = typename decltype(tag)::type;
    const unsigned grid = static_cast<unsigned>(rows) * splits;
    if (p->labels)
      distill_bwd_kernel<T, true><<<grid, kThreads, smem, st>>>(
          a, stats, lse, dkd, dce, row_ids, n_rows, static_cast<T*>(out), ld_out, splits, chunk);
    else
      distill_bwd_kernel<T, false><<<grid, kThreads, smem, st>>>(
          a, stats, lse, dkd, dce, row_ids, n_rows, static_cast<T*>(out), ld_out, splits, chunk);
    return launch_status();
  });
}

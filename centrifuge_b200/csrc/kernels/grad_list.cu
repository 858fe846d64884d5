// Global gradient norm over a list of tensors, and clipping (sm_100a).
//
//   norm  = extra_scale * sqrt(sum over the tensors of sum g^2)
//   out_i = g_i * extra_scale * min(1, max_norm / (norm + 1e-6))
//
// A model's gradients are hundreds of tensors between one element and hundreds of millions, of
// mixed types.  The whole list travels in the kernel's parameters (no table in device memory to
// fill, so a captured graph holds all it needs), every tensor is cut into chunks of kListChunk
// elements, and the chunks of all tensors are dealt to the blocks: two or three launches for up to
// 1024 tensors, whatever their sizes.  Bound by memory: one read for the norm, and, where something
// is written, one read and one write; the second pass takes the chunks in reverse, so that what the
// first read last still lies in the L2 cache.
//
// Squares are summed in fp32 within a chunk's share of a thread (128 values), and a block's shares in
// fp64.  Each block writes its sum rounded to fp32, which is what ranks exchange (the rounding, 2^-25
// of the norm at most, is below that of the norm itself); these are joined in fp64, in a fixed order.
// So a sum of squares above 3.4e38 may be infinite, and one below 1.2e-38 loses bits.
#include "row_types.cuh"

namespace cfb {

constexpr int kListChunk = 32768;  // elements

template <int CAP>
struct GradList {
  static constexpr int kCap = CAP;
  const void* ptr[CAP];
  void* out[CAP];
  long long numel[CAP];
  int first[CAP];  // index of the tensor's first chunk
  uint8_t type[CAP], out_type[CAP];
  int count, chunks;
};

// The tensor that chunk c lies in.
template <int CAP>
__device__ __forceinline__ int tensor_of(const GradList<CAP>& l, int c) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (l.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum_f64(double v) {
  __shared__ double red[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane_id() == 0) red[warp_id()] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += red[i];
  return v;
}

// Sum of squares of the n elements at p.
template <typename T>
__device__ __forceinline__ float chunk_sumsq(const T* p, int n) {
  constexpr int W = 16 / sizeof(T);
  const int tid = threadIdx.x;
  // elements before the first 16-byte boundary, whole vectors, and the rest
  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T));
  if (head > n) head = n;
  const int vecs = (n - head) / W;
  float s = 0.f;
#pragma unroll 8
  for (int i = tid; i < vecs; i += 256) {
    float f[W];
    load_f32<T, W>(p + head + i * W, f);
#pragma unroll
    for (int k = 0; k < W; ++k) s += f[k] * f[k];
  }
  const int rest = head + vecs * W;
  if (tid < head) s += to_f32(p[tid]) * to_f32(p[tid]);
  if (rest + tid < n) s += to_f32(p[rest + tid]) * to_f32(p[rest + tid]);
  return s;
}

template <int CAP>
__global__ void __launch_bounds__(256) grad_list_sumsq_kernel(const __grid_constant__ GradList<CAP> l,
                                                              float* __restrict__ partial) {
  let_next_start();
  double sum = 0.0;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    const long long at = static_cast<long long>(c - l.first[t]) * kListChunk;
    const int n = static_cast<int>(min(l.numel[t] - at, static_cast<long long>(kListChunk)));
    float s;
    if (l.type[t] == kF32)
      s = chunk_sumsq(static_cast<const float*>(l.ptr[t]) + at, n);
    else if (l.type[t] == kBF16)
      s = chunk_sumsq(static_cast<const __nv_bfloat16*>(l.ptr[t]) + at, n);
    else
      s = chunk_sumsq(static_cast<const __half*>(l.ptr[t]) + at, n);
    sum += static_cast<double>(s);
  }
  sum = block_sum_f64(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = static_cast<float>(sum);
}

template <typename TI, typename TO>
__device__ __forceinline__ void chunk_scale(const TI* p, TO* o, int n, float k) {
  const int tid = threadIdx.x;
  int done = 0;
  if (reinterpret_cast<uintptr_t>(p) % (8 * sizeof(TI)) == 0 &&
      reinterpret_cast<uintptr_t>(o) % (8 * sizeof(TO)) == 0) {
    constexpr int U = 4;  // packs in flight
    const int vecs = n / 8;
    for (int i = tid; i < vecs; i += 256 * U) {
      Pack<TI, 8> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * 256 < vecs) v[u] = load_pack<TI, 8>(p + (i + u * 256) * 8);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * 256 >= vecs) break;
        float f[8];
        unpack<TI, 8>(v[u], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= k;
        store_f32<TO, 8>(o + (i + u * 256) * 8, f);
      }
    }
    done = vecs * 8;
  }
#pragma unroll 8
  for (int i = done + tid; i < n; i += 256) o[i] = from_f32<TO>(to_f32(p[i]) * k);
}

template <typename TI>
__device__ __forceinline__ void chunk_scale_to(const TI* p, void* o, int type, long long at, int n,
                                               float k) {
  if (type == kF32)
    chunk_scale(p, static_cast<float*>(o) + at, n, k);
  else if (type == kBF16)
    chunk_scale(p, static_cast<__nv_bfloat16*>(o) + at, n, k);
  else
    chunk_scale(p, static_cast<__half*>(o) + at, n, k);
}

// The norm from the partial sums; every thread of the block gets it.
__device__ __forceinline__ float joined_norm(const float* partial, int n_partial,
                                             float extra_scale) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n_partial; i += 256) s += static_cast<double>(partial[i]);
  s = block_sum_f64(s);
  return static_cast<float>(sqrt(s) * static_cast<double>(extra_scale));
}
// What the elements are multiplied by.
__device__ __forceinline__ float clip_factor(float norm, float max_norm, float extra_scale) {
  if (!(max_norm > 0.f)) return extra_scale;
  const float c = max_norm / (norm + 1e-6f);
  return (c >= 1.f ? 1.f : c) * extra_scale;  // a norm that is no number leaves none in the output
}

__global__ void __launch_bounds__(256) grad_list_norm_kernel(const float* partial, int n_partial,
                                                             float extra_scale, float* norm) {
  after_previous();
  const float v = joined_norm(partial, n_partial, extra_scale);
  if (threadIdx.x == 0) *norm = v;
}

// One chunk a block: the hardware's dealing of short blocks keeps more of the memory busy than 1184
// blocks that loop (1.1 G elements bf16 -> fp32: 987 us in all against 1380).  The norm comes from a
// launch of its own, or, with n_partial, from the partial sums.
template <int CAP>
__global__ void __launch_bounds__(256) grad_list_scale_kernel(
    const __grid_constant__ GradList<CAP> l, const float* partial, int n_partial, float max_norm,
    float extra_scale, float* norm, int in_place) {
  after_previous();
  const float v = n_partial > 0 ? joined_norm(partial, n_partial, extra_scale) : *norm;
  if (n_partial > 0 && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float k = clip_factor(v, max_norm, extra_scale);
  if (in_place && k == 1.f) return;
  const int c = l.chunks - 1 - static_cast<int>(blockIdx.x);
  if (c < 0) return;
  const int t = tensor_of(l, c);
  const long long at = static_cast<long long>(c - l.first[t]) * kListChunk;
  const int n = static_cast<int>(min(l.numel[t] - at, static_cast<long long>(kListChunk)));
  if (l.type[t] == kF32)
    chunk_scale_to(static_cast<const float*>(l.ptr[t]) + at, l.out[t], l.out_type[t], at, n, k);
  else if (l.type[t] == kBF16)
    chunk_scale_to(static_cast<const __nv_bfloat16*>(l.ptr[t]) + at, l.out[t], l.out_type[t], at,
                   n, k);
  else
    chunk_scale_to(static_cast<const __half*>(l.ptr[t]) + at, l.out[t], l.out_type[t], at, n, k);
}

constexpr int kSmallList = 128;   // 3.9 KB of parameters
constexpr int kLargeList = 1024;  // 30 KB of parameters

// Tensors [begin, end) of the list as kernel parameters.
template <int CAP>
GradList<CAP> pack_list(const CfbTensorRef* refs, int begin, int end) {
  GradList<CAP> l;
  l.count = end - begin;
  long long chunks = 0;
  for (int i = 0; i < l.count; ++i) {
    const CfbTensorRef& r = refs[begin + i];
    l.ptr[i] = r.ptr;
    l.out[i] = r.out;
    l.numel[i] = r.numel;
    l.type[i] = static_cast<uint8_t>(r.type);
    l.out_type[i] = static_cast<uint8_t>(r.out_type);
    l.first[i] = static_cast<int>(chunks);
    chunks += (r.numel + kListChunk - 1) / kListChunk;
  }
  l.chunks = static_cast<int>(chunks);
  return l;
}

// f(list) for each group of tensors that one launch takes.
template <typename F>
int each_group(const CfbTensorRef* refs, int count, F&& f) {
  if (count <= kSmallList) return f(pack_list<kSmallList>(refs, 0, count), 0);
  for (int b = 0, g = 0; b < count; b += kLargeList, ++g) {
    const int e = b + kLargeList < count ? b + kLargeList : count;
    if (const int rc = f(pack_list<kLargeList>(refs, b, e), g)) return rc;
  }
  return 0;
}

}  // namespace cfb

using namespace cfb;

int cfb_grad_list_groups(int count) { return count <= kLargeList ? 1 : (count + kLargeList - 1) / kLargeList; }

int cfb_grad_list_sumsq(const CfbTensorRef* refs, int count, float* partial, int per_group,
                        cudaStream_t st) {
  if (count <= 0 || per_group <= 0) return -11;
  return each_group(refs, count, [&](const auto& l, int g) {
    grad_list_sumsq_kernel<<<per_group, 256, 0, st>>>(l, partial + static_cast<long long>(g) * per_group);
    return launch_status();
  });
}

int cfb_grad_list_scale(const CfbTensorRef* refs, int count, const float* partial, int n_partial,
                        float max_norm, float extra_scale, float* norm, int in_place,
                        cudaStream_t st) {
  if (count <= 0 || n_partial <= 0) return -11;
  // Where there are few blocks each of them joins the partial sums itself, which saves a launch;
  // with many that costs each of them more than the launch does.
  long long chunks = 0;
  for (int i = 0; i < count; ++i) chunks += (refs[i].numel + kListChunk - 1) / kListChunk;
  const bool joined = chunks > 148 * 8;
  if (joined)
    if (const int rc = launch_behind(grad_list_norm_kernel, dim3(1), dim3(256), 0, st, partial,
                                     n_partial, extra_scale, norm))
      return rc;
  return each_group(refs, count, [&](const auto& l, int g) {
    constexpr int kCap = std::remove_reference_t<decltype(l)>::kCap;
    const dim3 grid(l.chunks > 0 ? l.chunks : 1);
    const int sums = joined ? 0 : n_partial;
    if (joined || g > 0) {  // thousands of blocks that wait would be in the way of the ones before
      grad_list_scale_kernel<kCap><<<grid, 256, 0, st>>>(l, partial, sums, max_norm, extra_scale,
                                                         norm, in_place);
      return launch_status();
    }
    return launch_behind(grad_list_scale_kernel<kCap>, grid, dim3(256), 0, st, l, partial, sums,
                         max_norm, extra_scale, norm, in_place);
  });
}

// Scaled embedding lookup and its gradient by sorted tokens (sm_100a).
//
//   forward    out[r] = scale * table[ids[r]]
//   gradient   dtable[v] (+)= scale * sum over the rows r of token v of dy[r]
//
// Both are bound by memory.  The forward gives each row to one warp.  The gradient has to sum rows
// of equal tokens in one fixed order, whatever the scheduling and however uneven the tokens are
// (text repeats a few tokens very often, a padded batch has one token in a third of its rows):
//
//   1. sort_tokens_kernel   a stable counting sort of the rows by token.  Each block owns a range of
//                           tokens, reads all the tokens, and so knows both where its range begins
//                           in the sorted order and which rows are in it: one launch, no exchange
//                           between blocks.
//   2. embed_grad_kernel    chunks of kChunk sorted positions, one block each (and per slab of
//                           columns): a run of equal tokens that lies inside a chunk is summed and
//                           written by that block alone; a run that crosses a chunk's border leaves
//                           a partial sum.  A token in half of the rows is so spread over as many
//                           blocks as any other rows.
//   3. embed_join_kernel    the chunk in which a crossing run begins adds the partial sums up in
//                           chunk order and writes the table row.
//
// No atomics on floating values anywhere: two runs give the same bits.
#include "row_types.cuh"

namespace cfb {

constexpr int kChunk = 32;      // sorted positions of one block of the gradient
constexpr int kMaxSpan = 1024;  // tokens of one block of the sort

template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(256) scaled_embed_fwd_kernel(
    const TI* __restrict__ table, long long ld, long long V, const void* __restrict__ ids,
    int ids32, TO* __restrict__ out, long long ld_out, int rows, int H, float scale, int* err) {
  const int row = blockIdx.x * 8 + warp_id();
  if (row >= rows) return;
  const long long tok = ids32 ? static_cast<const int*>(ids)[row]
                              : static_cast<const long long*>(ids)[row];
  TO* d = out + row * ld_out;
  float f[W];
  if (!index_in(tok, V, err)) {  // token id outside the vocabulary: zero embedding
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = 0.f;
    for (int c = lane_id() * W; c < H; c += 32 * W) store_f32<TO, W>(d + c, f);
    return;
  }
  const TI* s = table + tok * ld;
#pragma unroll 4
  for (int c = lane_id() * W; c < H; c += 32 * W) {
    load_f32<TI, W>(s + c, f);
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] *= scale;
    store_f32<TO, W>(d + c, f);
  }
}

// The token of gradient row r, or -1 for a row without one: a padding token, or (recorded in the
// status block by the block that is told to) a row id outside ids or a token outside the table.
__device__ __forceinline__ int row_token(int r, const void* ids, int ids32, long long n_ids,
                                         const int* id_rows, long long V, long long pad, int* err) {
  const long long i = id_rows ? id_rows[r] : r;
  if (!index_in(i, n_ids, err)) return -1;
  const long long tok = ids32 ? static_cast<const int*>(ids)[i]
                              : static_cast<const long long*>(ids)[i];
  if (tok == pad && pad >= 0) return -1;
  return index_in(tok, V, err) ? static_cast<int>(tok) : -1;
}

// Block b places the rows of tokens [b * span, (b + 1) * span) at their sorted positions.  Each of
// the 32 warps takes a contiguous part of the rows; hist[w][t] first counts the rows of token t in
// part w and then, after the scan, is the next position of such a row.
__global__ void __launch_bounds__(1024) sort_tokens_kernel(
    const void* __restrict__ ids, int ids32, long long n_ids, const int* __restrict__ id_rows,
    int rows, long long V, long long pad, int span, int* __restrict__ order,
    int* __restrict__ stok, int* __restrict__ n_valid, int* err) {
  extern __shared__ int hist[];  // [32][span]
  __shared__ int warp_sums[32];
  __shared__ int below;
  const int tid = threadIdx.x, lane = lane_id(), wp = warp_id();
  const long long lo = static_cast<long long>(blockIdx.x) * span;
  const long long hi = min(V, lo + span);
  if (blockIdx.x != 0) err = nullptr;  // one block reports
  for (int i = tid; i < 32 * span; i += 1024) hist[i] = 0;
  if (tid == 0) below = 0;
  __syncthreads();

  const int part = (rows + 1023) / 1024 * 32;
  const int r0 = min(rows, wp * part), r1 = min(rows, r0 + part);
  int less = 0;
#pragma unroll 4
  for (int r = r0 + lane; r < r1; r += 32) {
    const int tok = row_token(r, ids, ids32, n_ids, id_rows, V, pad, err);
    less += (tok >= 0 && tok < lo);
    if (tok >= lo && tok < hi) atomicAdd(&hist[wp * span + static_cast<int>(tok - lo)], 1);
  }
  less = __reduce_add_sync(0xffffffffu, less);
  if (lane == 0) atomicAdd(&below, less);
  __syncthreads();

  // exclusive scan over (token, warp); thread t owns token lo + t (span <= 1024)
  int tot = 0;
  if (tid < span)
    for (int w = 0; w < 32; ++w) {
      const int c = hist[w * span + tid];
      hist[w * span + tid] = tot;
      tot += c;
    }
  int inc = tot;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) warp_sums[wp] = inc;
  __syncthreads();
  if (wp == 0) {
    const int s = warp_sums[lane];
    int x = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += t;
    }
    warp_sums[lane] = x - s;
    if (lane == 31 && blockIdx.x == gridDim.x - 1) *n_valid = below + x;
  }
  __syncthreads();
  const int first = below + warp_sums[wp] + inc - tot;
  if (tid < span)
    for (int w = 0; w < 32; ++w) hist[w * span + tid] += first;
  __syncthreads();

  for (int r = r0 + lane; r - lane < r1; r += 32) {
    int key = -1;
    if (r < r1) {
      const int tok = row_token(r, ids, ids32, n_ids, id_rows, V, pad, nullptr);
      if (tok >= lo && tok < hi) key = static_cast<int>(tok - lo);
    }
    if (__ballot_sync(0xffffffffu, key >= 0) == 0) continue;
    const unsigned same = __match_any_sync(0xffffffffu, key);
    const int rank = __popc(same & ((1u << lane) - 1));
    int* next = &hist[wp * span + max(key, 0)];
    const int at = *next + rank;
    __syncwarp();
    if (key >= 0) {
      order[at] = r;
      stok[at] = static_cast<int>(lo) + key;
      if (rank == 0) *next = at + __popc(same);
    }
    __syncwarp();
  }
}

// Adds (or, without ACC, writes) W columns of a run's sum to its table row.
template <int W>
__device__ __forceinline__ void write_run(float* dst, const float* acc, float scale, int add) {
  float o[W];
  if (add) load_f32<float, W>(dst, o);
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] = (add ? o[i] : 0.f) + scale * acc[i];
  store_f32<float, W>(dst, o);
}

// Chunk blockIdx.x of the sorted rows, columns (blockIdx.y * blockDim.x + thread) * W.
// part[chunk][0]: the sum of the rows of a run that began in an earlier chunk;
// part[chunk][1]: of a run that begins here and goes on in the next chunk.
template <typename T, int W>
__global__ void __launch_bounds__(256) embed_grad_kernel(
    const T* __restrict__ dy, long long ld, const int* __restrict__ order,
    const int* __restrict__ stok, const int* __restrict__ n_valid, float* __restrict__ dtable,
    long long ld_t, float* __restrict__ part, int H, float scale, int add) {
  constexpr int U = sizeof(T) == 4 && W == 8 ? 4 : 8;  // rows in flight
  __shared__ int s_row[kChunk];
  __shared__ int s_tok[kChunk + 2];  // with the tokens before and behind the chunk (-1: none)
  const int n = *n_valid;
  const int p0 = blockIdx.x * kChunk;
  if (p0 >= n) return;
  const int m = min(kChunk, n - p0);
  if (threadIdx.x < m) s_row[threadIdx.x] = order[p0 + threadIdx.x];
  for (int i = threadIdx.x; i < m + 2; i += blockDim.x) {
    const int p = p0 + i - 1;
    s_tok[i] = p >= 0 && p < n ? stok[p] : -1;
  }
  __syncthreads();
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * W;
  if (c >= H) return;
  const bool from_before = s_tok[0] == s_tok[1];
  float acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0.f;
  int begin = 0;  // first row of the run that acc sums
  for (int j = 0; j < m; j += U) {
    Pack<T, W> k[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u < m) k[u] = load_pack<T, W>(dy + s_row[j + u] * ld + c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= m) break;
      float f[W];
      unpack<T, W>(k[u], f);
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] += f[i];
      const int tok = s_tok[j + u + 1];
      const bool goes_on = s_tok[j + u + 2] == tok;
      if (goes_on && j + u + 1 < m) continue;
      const bool head = begin == 0 && from_before;
      if (head || goes_on) {
        const long long slot = 2ll * blockIdx.x + (head ? 0 : 1);
        store_f32<float, W>(part + slot * H + c, acc);
      } else {
        write_run<W>(dtable + tok * ld_t + c, acc, scale, add);
      }
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] = 0.f;
      begin = j + u + 1;
    }
  }
}

// The run that begins in chunk blockIdx.x and goes on behind it: its partial sums in chunk order.
template <int W>
__global__ void __launch_bounds__(256) embed_join_kernel(
    const int* __restrict__ stok, const int* __restrict__ n_valid, float* __restrict__ dtable,
    long long ld_t, const float* __restrict__ part, int H, float scale, int add) {
  const int n = *n_valid;
  const int p0 = blockIdx.x * kChunk, p1 = p0 + kChunk;
  if (p1 >= n) return;
  const int tok = stok[p1 - 1];
  if (stok[p1] != tok || (p0 > 0 && stok[p0 - 1] == tok)) return;
  int lo = p1, hi = n;  // the first position behind the run
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (stok[mid] == tok) lo = mid + 1; else hi = mid;
  }
  const int last = (lo - 1) / kChunk;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * W;
  if (c >= H) return;
  float acc[W], f[W];
  load_f32<float, W>(part + (2ll * blockIdx.x + 1) * H + c, acc);
#pragma unroll 4
  for (int k = blockIdx.x + 1; k <= last; ++k) {
    load_f32<float, W>(part + 2ll * k * H + c, f);
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] += f[i];
  }
  write_run<W>(dtable + tok * ld_t + c, acc, scale, add);
}

template <int W>
__global__ void __launch_bounds__(256) zero_rows_kernel(float* __restrict__ t, long long ld,
                                                        long long V, int H) {
  float z[W];
#pragma unroll
  for (int i = 0; i < W; ++i) z[i] = 0.f;
  for (long long r = blockIdx.x * 8ll + warp_id(); r < V; r += gridDim.x * 8ll)
    for (int c = lane_id() * W; c < H; c += 32 * W) store_f32<float, W>(t + r * ld + c, z);
}

}  // namespace cfb

using namespace cfb;

int cfb_scaled_embedding_fwd(const void* table, int type, long long ld, long long V,
                             const void* ids, int ids32, void* out, int out_type,
                             long long ld_out, int rows, int H, float scale, int* err,
                             cudaStream_t st) {
  if (rows == 0 || H == 0) return 0;
  const bool wide = H % 8 == 0 && rows_of_8(table, ld, type) && rows_of_8(out, ld_out, out_type);
  return with_type(type, [&](auto ti) {
    return with_type(out_type, [&](auto to) {
      using TI = typename decltype(ti)::type;
      using TO = typename decltype(to)::type;
      auto* kernel = wide ? scaled_embed_fwd_kernel<TI, TO, 8> : scaled_embed_fwd_kernel<TI, TO, 1>;
      kernel<<<(rows + 7) / 8, 256, 0, st>>>(static_cast<const TI*>(table), ld, V, ids, ids32,
                                             static_cast<TO*>(out), ld_out, rows, H, scale, err);
      return launch_status();
    });
  });
}

long long cfb_scaled_embedding_bwd_workspace(int rows, int H) {
  const long long chunks = (rows + kChunk - 1) / kChunk;
  return 4ll * (8 + 2ll * ((rows + 3) / 4 * 4) + 2 * chunks * H);  // bytes
}

int cfb_scaled_embedding_bwd(const void* dy, int type, long long ld, const void* ids, int ids32,
                             long long n_ids, const int* id_rows, long long pad, float* dtable,
                             long long ld_t, long long V, int rows, int H, float scale, int add,
                             void* work, int* err, cudaStream_t st) {
  if (V <= 0 || V > INT32_MAX) return -11;
  if (H == 0) return 0;
  const bool wide = H % 8 == 0 && rows_of_8(dy, ld, type) && rows_of_8(dtable, ld_t, kF32);
  if (!add) {
    const long long blocks = (V + 7) / 8 < 148 * 16 ? (V + 7) / 8 : 148 * 16;
    if (wide)
      zero_rows_kernel<8><<<blocks, 256, 0, st>>>(dtable, ld_t, V, H);
    else
      zero_rows_kernel<1><<<blocks, 256, 0, st>>>(dtable, ld_t, V, H);
  }
  if (rows == 0) return launch_status();
  const int padded = (rows + 3) / 4 * 4;
  int* n_valid = static_cast<int*>(work);
  int* order = n_valid + 8;  // the partial sums behind it begin on a 32-byte border
  int* stok = order + padded;
  float* part = reinterpret_cast<float*>(stok + padded);
  // one block for each SM where the vocabulary allows, ranges of whole warps
  long long span = ((V + 147) / 148 + 31) / 32 * 32;
  if (span > kMaxSpan) span = kMaxSpan;
  const int smem = static_cast<int>(32 * span * sizeof(int));
  if (cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           32 * kMaxSpan * static_cast<int>(sizeof(int))) != cudaSuccess)
    return -3;
  sort_tokens_kernel<<<static_cast<unsigned>((V + span - 1) / span), 1024, smem, st>>>(
      ids, ids32, n_ids, id_rows, rows, V, pad, static_cast<int>(span), order, stok, n_valid, err);
  const int W = wide ? 8 : 1;
  const int need = (H + W - 1) / W;
  const int threads = need >= 256 ? 256 : (need + 31) / 32 * 32;
  const dim3 grid((rows + kChunk - 1) / kChunk, (need + threads - 1) / threads);
  return with_type(type, [&](auto t) {
    using T = typename decltype(t)::type;
    auto* grad = wide ? embed_grad_kernel<T, 8> : embed_grad_kernel<T, 1>;
    grad<<<grid, threads, 0, st>>>(static_cast<const T*>(dy), ld, order, stok, n_valid, dtable,
                                   ld_t, part, H, scale, add);
    auto* join = wide ? embed_join_kernel<8> : embed_join_kernel<1>;
    join<<<grid, threads, 0, st>>>(stok, n_valid, dtable, ld_t, part, H, scale, add);
    return launch_status();
  });
}

// Scaled embedding lookup and its gradient by sorted tokens (sm_100a).
//
//   forward    out[r] = scale * table[ids[r]]
//   gradient   dtable[v] (+)= scale * sum over the rows r of token v of dy[r]
//
// Both are bound by memory.  The forward gives each row to one warp.  The gradient has to sum rows
// of equal tokens in one fixed order, whatever the scheduling and however uneven the tokens are
// (text repeats a few tokens very often, a padded batch has one token in a third of its rows):
//
//   1. sort_tokens_kernel   a stable counting sort of the rows by token.  Each block owns the tokens
//                           with one remainder, reads all the tokens, and so knows both where its
//                           tokens begin in the sorted order and which rows they are in: one launch,
//                           no exchange between blocks.  (A text's frequent tokens have neighbouring
//                           ids; by ranges one block would have had half of all rows.)
//   2. embed_grad_kernel    chunks of sorted positions, a warp each (and per slab of columns): a run
//                           of equal tokens that lies inside a chunk is summed and written by that
//                           warp alone; a run that crosses a chunk's border leaves a partial sum.
//                           A token in half of the rows is so spread over as many warps as any
//                           other rows.  Where the gradient replaces the table, further blocks
//                           clear the rows of the tokens that do not occur meanwhile.
//   3. embed_join_kernel    the chunk in which a crossing run begins adds the partial sums up in
//                           chunk order and writes the table row.
//
// Measured, 8192 kept of 16384 rows x 2048 bf16, 32000 tokens of text, the table replaced: 55 us a
// pass (8 us sort, 45 us sums and clearing at 296 MB, the join; 45 us is all of it at the copy rate);
// 8192 rows x 4096 of 128256 tokens: 314 us (2.17 GB, 332 us at the copy rate).
//
// A handful of rows takes one launch instead (embed_grad_few_kernel).  Every element of the table is
// written by one thread, once: two runs give the same bits.
#include "row_types.cuh"

namespace cfb {

constexpr int kMaxSpan = 1024;  // tokens of one block of the sort
constexpr int kKeyRows = 32768; // rows whose keys a block of the sort holds in shared memory
// Table rows that one block clears: the gradient measured above took 63.5 us with 8 and 61 with 4,
// before the steps that made it 55.
constexpr int kClear = 4;
// Up to here one launch does it all (a row id fits 8 bits).  256 rows x 1024 of 3000 tokens: 8 us for
// 12 sorted, x 4096 and most of one token 20 for 20.
constexpr int kFewRows = 256;
// Rows of a token that one warp sums there by itself; of more the block's four warps have a quarter
// each.  128 rows of 3000 tokens, us for none / 24 / 64 / any by itself: x 256 text 5.4 / 3.3 / 3.3 /
// 3.3, nine tenths one token 4.7 / 4.5 / 4.5 / 8.3; 256 rows x 1024, a fifth one token 8.3 (none), 6.2,
// 6.9, 6.9; x 4096, nine tenths 15.7, 14.2, 14.1, 22.3 (128 rows).
constexpr int kWarpRun = 24;

constexpr int kAhead = 128;     // blocks of the gradient that request rows during the sort
constexpr int kAheadBytes = 32 << 20;  // and what they request: the rate of the memory times the sort

// Sorted positions of one warp of the gradient: few where few rows would leave SMs idle, more where
// there are enough, since every chunk border costs a partial sum.  us a pass with 8 / 16 / 32: 1000
// rows x 4096 added to 32000 tokens 16.7 / 22.8, 2000 x 1024 15.8 / 21.8; replacing, x 2048 of 32000
// tokens of text, 4000 rows 49.4 / 48.3 / 49.4, 8192 rows 55.9 / 52.0 / 52.3 (x 512: 21.8 / 21.2 /
// 22.7), 16384 rows 73.5 / 65.5 / 63.8, 32768 rows 109.5 / 92.3 / 87.5.
inline int chunk_rows(int rows) { return rows >= 32768 ? 32 : rows >= 2048 ? 16 : 8; }

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

// Clears a table row of H columns, in stores of 256 bits between the first and the last boundary of
// 32 bytes in it, wherever the row begins.  (28386 x 1124, 128 MB: 32.9 us a pass with stores of four
// bytes, now 29.2.)
template <int W>
__device__ __forceinline__ void clear_row(float* t, int H) {
  const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int lane = lane_id();
  int lo = 0, hi = H;  // W = 8: whole packs of aligned rows
  if constexpr (W == 1) {
    lo = min(H, static_cast<int>(-(reinterpret_cast<uintptr_t>(t) >> 2) & 7));
    hi = lo + (H - lo) / 8 * 8;
    if (lane < lo) t[lane] = 0.f;
    if (lane < H - hi) t[hi + lane] = 0.f;
  }
#pragma unroll 4
  for (int c = lo + lane * 8; c < hi; c += 256) store_f32<float, 8>(t + c, z);
}

// Block b of 2^shift places the rows of the tokens t 2^shift + b at their sorted positions, which are
// by block and t.  Each of the 32 warps takes a contiguous part of the rows; hist[w][t] first counts
// the rows of the block's token t in part w and then, after the scan, is the next position of such a
// row.  A thread has eight tokens in flight; up to kKeyRows rows the second pass finds which of them
// are of the block in shared memory.
__global__ void __launch_bounds__(1024) sort_tokens_kernel(
    const void* __restrict__ ids, int ids32, unsigned n_ids, const int* __restrict__ id_rows,
    int rows, int V, int pad, int shift, int span, int* __restrict__ order,
    int* __restrict__ stok, int* __restrict__ n_valid, uint32_t* __restrict__ absent, int* err) {
  constexpr int U = 8;
  extern __shared__ int hist[];  // [32][span], and a 16-bit key for each of up to kKeyRows rows
  uint16_t* keys = reinterpret_cast<uint16_t*>(hist + 32 * span);  // 1 + t, 0: not ours
  const bool keep = rows <= kKeyRows;
  __shared__ int warp_sums[32];
  __shared__ int below;
  let_next_start();
  const int tid = threadIdx.x, lane = lane_id(), wp = warp_id();
  const int me = blockIdx.x, mask = (1 << shift) - 1;
  const int mine = (V - me + mask) >> shift;  // tokens of this block
  const int part = (rows + 1023) / 1024 * 32;
  const int r0 = min(rows, wp * part), r1 = min(rows, r0 + part);
  int tok[U];
  // Tokens as 32-bit numbers, -1 for a row without one: every comparison below is unsigned.
  const auto read = [&](int base, bool report) {
    int id[U];
    int2 t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = base + u * 32 + lane;
      id[u] = r < r1 ? (id_rows ? id_rows[r] : r) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t[u] = make_int2(-1, 0);
      if (static_cast<unsigned>(id[u]) < n_ids) {
        if (ids32)
          t[u].x = static_cast<const int*>(ids)[id[u]];
        else
          t[u] = static_cast<const int2*>(ids)[id[u]];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = t[u].y == 0 && static_cast<unsigned>(t[u].x) < static_cast<unsigned>(V);
      const bool padding = pad >= 0 && t[u].y == 0 && t[u].x == pad;
      tok[u] = ok && !padding ? t[u].x : -1;
      if (report && base + u * 32 + lane < r1 && !ok && !padding) atomicCAS(err, 0, kErrBounds);
    }
  };
  const bool report = blockIdx.x == 0 && err;  // one block does
  read(r0, report);  // under way while the counts are cleared
  for (int i = tid * 4; i < 32 * span; i += 4096)
    *reinterpret_cast<int4*>(hist + i) = make_int4(0, 0, 0, 0);
  if (tid == 0) below = 0;
  __syncthreads();

  int less = 0;
  for (int base = r0; base < r1; base += 32 * U) {
    if (base != r0) read(base, report);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int owner = tok[u] >= 0 ? tok[u] & mask : INT32_MAX;
      less += owner < me;
      if (owner == me) atomicAdd(&hist[wp * span + (tok[u] >> shift)], 1);
      const int r = base + u * 32 + lane;
      if (keep && r < r1) keys[r] = static_cast<uint16_t>(owner == me ? (tok[u] >> shift) + 1 : 0);
    }
  }
  less = __reduce_add_sync(0xffffffffu, less);
  if (lane == 0 && less) atomicAdd(&below, less);
  __syncthreads();

  // exclusive scan over (token, warp); thread t has the block's token t (span <= 1024)
  int count[32];
  int tot = 0;
  if (tid < span) {
#pragma unroll
    for (int w = 0; w < 32; ++w) count[w] = hist[w * span + tid];
#pragma unroll
    for (int w = 0; w < 32; ++w) tot += count[w];
  }
  if (tid < span) {  // tokens without a row, a bit each
    const uint32_t none = __ballot_sync(0xffffffffu, tot == 0 && tid < mine);
    if (lane == 0) absent[(me * span + tid) / 32] = none;
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
  if (tid < span) {
    int at = below + warp_sums[wp] + inc - tot;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      hist[w * span + tid] = at;
      at += count[w];
    }
  }
  __syncthreads();

  for (int base = r0; base < r1; base += 32 * U) {
    if (!keep) read(base, false);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = base + u * 32 + lane;
      int key = -1;
      if (keep)
        key = r < r1 ? static_cast<int>(keys[r]) - 1 : -1;
      else if (tok[u] >= 0 && (tok[u] & mask) == me)
        key = tok[u] >> shift;
      if (__ballot_sync(0xffffffffu, key >= 0) == 0) continue;
      const unsigned same = __match_any_sync(0xffffffffu, key);
      const int rank = __popc(same & ((1u << lane) - 1));
      int* next = &hist[wp * span + max(key, 0)];
      const int at = *next + rank;
      __syncwarp();
      if (key >= 0) {
        order[at] = r;
        stok[at] = (key << shift) + me;
        if (rank == 0) *next = at + __popc(same);
      }
      __syncwarp();
    }
  }
}

// A lane's columns of a slab of rows: eight neighbours (W = 8), or four columns 32 apart (W = 1).
// Loads are made without a branch, columns behind the row from its first one, and what is not wanted
// of a batch is set to zero without one: a load behind a branch, or one whose value is used behind
// one, is waited for before the next is made (115 rows of one token, 256 wide: 31 us, now 8).
template <int W>
struct SlabCols {
  static constexpr int N = W == 8 ? 8 : 4;
  static constexpr int kSlab = 32 * N;
  int c, H;
  __device__ __forceinline__ SlabCols(int slab, int H_) : c(slab * kSlab + lane_id() * W), H(H_) {}
  template <typename T>
  __device__ __forceinline__ Pack<T, N> load(const T* row) const {
    Pack<T, N> k;
    if constexpr (W == 8 && sizeof(k) == 16) {
      uint32_t* u = reinterpret_cast<uint32_t*>(&k);
      asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
                   : "l"(row + (c < H ? c : 0)));
      return k;
    } else if constexpr (W == 8) {
      return load_pack<T, 8>(row + (c < H ? c : 0));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) k.v[i] = row[c + 32 * i < H ? c + 32 * i : 0];
      return k;
    }
  }
  // The same into shared memory, on its way until the thread waits for its cp.async groups.
  template <typename T>
  __device__ __forceinline__ void fetch(const T* row, Pack<T, N>* to) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(*to) / 16); ++i)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to) + i * 16),
                   "l"(reinterpret_cast<const uint8_t*>(row + (c < H ? c : 0)) + i * 16)
                   : "memory");
  }
  // The same, zeros where it is not wanted.
  template <typename T>
  __device__ __forceinline__ Pack<T, N> load_if(bool wanted, const T* row) const {
    Pack<T, N> k = load(row);
#pragma unroll
    for (int i = 0; i < N; ++i) k.v[i] = wanted ? k.v[i] : from_f32<T>(0.f);
    return k;
  }
  __device__ __forceinline__ void store(float* row, const float* f) const {
    if constexpr (W == 8) {
      if (c < H) store_f32<float, 8>(row + c, f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + 32 * i < H) row[c + 32 * i] = f[i];
    }
  }
  // Adds a run's sum to its table row, or writes it there.  No other thread has these elements, so
  // the additions of the reduction instructions happen once each and in no order that could vary;
  // unlike a load and a store they do not make the warp wait for the table.  (They take subnormal
  // numbers, below 1.2e-38, as zeros.)
  __device__ __forceinline__ void write_run(float* row, const float* acc, float scale,
                                            int add) const {
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = scale * acc[i];
    if (!add) {
      store(row, o);
    } else if constexpr (W == 8) {
      if (c < H)
#pragma unroll
        for (int i = 0; i < N; i += 4)
          asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(row + c + i),
                       "f"(o[i]), "f"(o[i + 1]), "f"(o[i + 2]), "f"(o[i + 3])
                       : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + 32 * i < H) atomicAdd(row + c + 32 * i, o[i]);
    }
  }
};

// One warp: sorted positions [chunk * per, + per) (per <= 32), one slab of columns.
// part[chunk][0]: the sum of the rows of a run that began in an earlier chunk;
// part[chunk][1]: of a run that begins here and goes on in the next chunk.
template <typename T, int W>
__global__ void __launch_bounds__(128, 8) embed_grad_kernel(
    const T* __restrict__ dy, long long ld, const int* order,
    const int* stok, const int* n_valid,
    const uint32_t* absent, float* __restrict__ dtable, long long ld_t,
    float* __restrict__ part, int rows, int H, int slabs, int per, int sum_blocks, int shift,
    int span, int vocab, float scale, int add) {
  using S = SlabCols<W>;
  constexpr int N = S::N;
  // Rows in flight: with whole packs they go to shared memory, each lane's to a place of its own,
  // since the branches at the ends of runs would have loads into registers wait for each other
  // (8192 kept of 16384 x 2048: 61 us a pass with four rows in registers, 58 with 16 in shared memory).
  constexpr bool kStaged = W == 8;
  constexpr int U = !kStaged ? 4 : sizeof(T) == 2 ? 16 : 8;
  __shared__ Pack<T, N> stage[kStaged ? 4 : 1][kStaged ? U : 1][32];
  // blocks that sum and blocks that clear in turn, as long as there are both: the ones wait for
  // their rows, the others keep the memory busy
  const int clear_blocks = static_cast<int>(gridDim.x) - sum_blocks;
  const int both = 2 * min(sum_blocks, clear_blocks);
  const int b = blockIdx.x;
  const bool sums = b < both ? b % 2 == 0 : sum_blocks > clear_blocks;
  const int block = b < both ? b / 2 : b - both / 2;
  // The sort leaves the memory idle: the first blocks ask the L2 cache for what it can bring in
  // meanwhile.  (8192 kept of 16384 x 2048: 58 -> 55 us a pass, added to the table 35 -> 30.)
  const long long bytes = static_cast<long long>(H) * sizeof(T);
  if (b < kAhead && bytes <= 65536) {
    const int some = min(rows, kAheadBytes / static_cast<int>(bytes));
    for (int r = b * 128 + threadIdx.x; r < some; r += kAhead * 128)
      prefetch_l2(dy + r * ld, static_cast<int>(bytes));
  }
  after_previous();
  let_next_start();
  if (!sums) {  // clear what does not occur of kClear neighbouring tokens
#pragma unroll
    for (int i = 0; i < kClear / 4; ++i) {
      const int token = block * kClear + i * 4 + warp_id();
      const int place = (token & ((1 << shift) - 1)) * span + (token >> shift);
      if (token < vocab && (absent[place / 32] >> (place % 32) & 1))
        clear_row<W>(dtable + token * ld_t, H);
    }
    return;
  }
  const int item = block * 4 + warp_id();
  const int chunk = item / slabs;
  const int p0 = chunk * per;
  const int lane = lane_id();
  // all loads at once; what lies behind the last valid row was never written, and is not used
  const int n = *n_valid;
  int my_row = lane < per && p0 + lane < rows ? order[p0 + lane] : 0;
  const int my_tok = lane < per && p0 + lane < rows ? stok[p0 + lane] : -1;
  const int before = p0 > 0 && p0 <= rows ? stok[p0 - 1] : -1;
  const int after = p0 + per < rows ? stok[p0 + per] : -1;
  if (p0 >= n) return;
  const int m = min(per, n - p0);
  if (lane >= m) my_row = 0;  // a row that is there: the loads below ask no further
  const int behind = p0 + per < n ? after : -1;
  const bool from_before = before == __shfl_sync(0xffffffffu, my_tok, 0);
  const S cols(item % slabs, H);
  F2 acc[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) acc[i] = f2(0.f);
  bool head = from_before;  // acc sums the run that began before the chunk
#pragma unroll 1
  for (int j = 0; j < m; j += U) {
    Pack<T, N> k[kStaged ? 1 : U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = __shfl_sync(0xffffffffu, my_row, (j + u) & 31);  // 0 behind the last one
      if constexpr (kStaged) {
        if (j + u < m) cols.fetch(dy + row * ld, &stage[warp_id()][u][lane]);
      } else {
        k[u] = cols.load(dy + row * ld);
      }
    }
    if constexpr (kStaged)
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
#pragma unroll(kStaged ? 1 : U)
    for (int u = 0; u < U; ++u) {
      if (j + u >= m) break;
      F2 f[N / 2];
      if constexpr (kStaged)
        unpack_f2<T, N>(stage[warp_id()][u][lane], f);
      else
        unpack_f2<T, N>(k[u], f);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) acc[i] = acc[i] + f[i];
      const int tok = __shfl_sync(0xffffffffu, my_tok, j + u);
      const bool last = j + u + 1 == m;
      const int next = __shfl_sync(0xffffffffu, my_tok, (j + u + 1) & 31);
      const bool goes_on = (last ? behind : next) == tok;
      if (goes_on && !last) continue;
      float sum[N];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        sum[2 * i] = halves(acc[i]).x;
        sum[2 * i + 1] = halves(acc[i]).y;
        acc[i] = f2(0.f);
      }
      if (head || goes_on) {
        cols.store(part + (2ll * chunk + (head ? 0 : 1)) * H, sum);
      } else {
        cols.write_run(dtable + tok * ld_t, sum, scale, add);
      }
      head = false;
    }
  }
}

// The runs that begin in chunks 8 blockIdx.x .. + 8 and go on behind their chunk: their partial sums
// in chunk order.  A warp has a chunk, and sums a run of up to eight more chunks by itself; of a
// longer run, of which a block can only have one, eight warps take a contiguous share of the chunks
// each, and the shares are added in their order.
template <int W>
__global__ void __launch_bounds__(256) embed_join_kernel(
    const int* stok, const int* n_valid, float* __restrict__ dtable,
    long long ld_t, const float* part, int rows, int H, int per, float scale,
    int add) {
  using S = SlabCols<W>;
  constexpr int N = S::N;
  constexpr int U = 8;  // partial sums in flight
  __shared__ float share[8][32 * N];
  __shared__ int long_chunk;
  after_previous();
  const int wp = warp_id(), lane = lane_id();
  const int chunk = blockIdx.x * 8 + wp;
  const int p0 = chunk * per, p1 = p0 + per;
  const S cols(blockIdx.y, H);
  float acc[N];
  // the sum of part[k][0] over [k0, k1) added to acc
  const auto add_parts = [&](int k0, int k1) {
#pragma unroll 1
    for (int k = k0; k < k1; k += U) {
      Pack<float, N> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = cols.load_if(k + u < k1, part + 2ll * min(k + u, k1 - 1) * H);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += v[u].v[i];
    }
  };
  if (threadIdx.x == 0) long_chunk = -1;
  __syncthreads();
  if (p1 < rows) {
    // all loads at once; what lies behind the last valid row is not used
    const int n = *n_valid;
    const int tok = stok[p1 - 1], before = p0 > 0 ? stok[p0 - 1] : -1;
    const int q = p1 + lane * per;  // the first rows of the 32 chunks behind
    const int ahead = q < rows ? stok[q] : -1;
    const int more = __popc(__ballot_sync(0xffffffffu, q < n && ahead == tok));
    if (more > 8 && before != tok) {
      if (lane == 0) long_chunk = chunk;
    } else if (more > 0 && before != tok) {
      unpack<float, N>(cols.load(part + (2ll * chunk + 1) * H), acc);
      add_parts(chunk + 1, chunk + 1 + more);
      cols.write_run(dtable + tok * ld_t, acc, scale, add);
    }
  }
  __syncthreads();
  const int from = long_chunk;
  if (from < 0) return;
  const int n = *n_valid, tok = stok[(from + 1) * per];
  int chunks = 0;
  for (int k = from + 1;; k += 256) {
    const long long p = static_cast<long long>(k + threadIdx.x) * per;
    const int more = __syncthreads_count(p < n && stok[p] == tok);
    chunks += more;
    if (more < 256) break;
  }
  const int each = (chunks + 7) / 8;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  if (wp == 0) unpack<float, N>(cols.load(part + (2ll * from + 1) * H), acc);
  add_parts(from + 1 + wp * each, from + 1 + min(chunks, (wp + 1) * each));
#pragma unroll
  for (int i = 0; i < N; ++i) share[wp][i * 32 + lane] = acc[i];
  __syncthreads();
  if (wp != 0) return;
#pragma unroll
  for (int w = 1; w < 8; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += share[w][i * 32 + lane];
  cols.write_run(dtable + tok * ld_t, acc, scale, add);
}

// Up to kFewRows rows.  Blocks [0, row_blocks): a warp for each row and slab, which does nothing
// unless the row is the first of its token, and then sums that token's rows in row order; runs of
// over kWarpRun rows are left to all four warps of the block, a quarter each, and the quarters are
// added in their order (the warps of a block have different rows and so different tokens).  The
// blocks behind them clear the table rows of tokens that do not occur, kClear each.
template <typename T, int W>
__global__ void __launch_bounds__(128, 6) embed_grad_few_kernel(
    const T* __restrict__ dy, long long ld, const void* __restrict__ ids, int ids32,
    long long n_ids, const int* __restrict__ id_rows, long long pad, float* __restrict__ dtable,
    long long ld_t, long long V, int rows, int H, int slabs, int row_blocks, float scale, int add,
    int* err) {
  using S = SlabCols<W>;
  constexpr int N = S::N;
  constexpr int U = sizeof(T) == 4 && W == 8 ? 4 : 8;
  __shared__ int tok[kFewRows];
  __shared__ uint8_t list[4][kFewRows];  // for each warp the rows of its token, in row order
  __shared__ int found[4];
  __shared__ float share[4][32 * N];
  __shared__ uint32_t present;
  const int tid = threadIdx.x, wp = warp_id(), lane = lane_id();
  if (tid == 0) present = 0;
  for (int r = tid; r < rows; r += 128)
    tok[r] = row_token(r, ids, ids32, n_ids, id_rows, V, pad, blockIdx.x == 0 ? err : nullptr);
  __syncthreads();
  if (static_cast<int>(blockIdx.x) >= row_blocks) {
    const long long lo = (static_cast<long long>(blockIdx.x) - row_blocks) * kClear;
    for (int r = tid; r < rows; r += 128)
      if (tok[r] >= lo && tok[r] < lo + kClear) atomicOr(&present, 1u << (tok[r] - lo));
    __syncthreads();
    for (int t = wp; t < kClear; t += 4)
      if (lo + t < V && !(present >> t & 1)) clear_row<W>(dtable + (lo + t) * ld_t, H);
    return;
  }
  const int item = blockIdx.x * 4 + wp;
  const int r = item % rows, slab = item / rows;
  const int mine = slab < slabs ? tok[r] : -1;
  bool first = mine >= 0;
  for (int q = lane; q < r; q += 32) first = first && tok[q] != mine;
  int n = 0;
  if (__all_sync(0xffffffffu, first)) {
    for (int base = r / 32 * 32; base < rows; base += 32) {
      const int q = base + lane;
      const bool hit = q >= r && q < rows && tok[q] == mine;
      const unsigned hits = __ballot_sync(0xffffffffu, hit);
      if (hit) list[wp][n + __popc(hits & ((1u << lane) - 1))] = static_cast<uint8_t>(q);
      n += __popc(hits);
    }
  }
  if (lane == 0) found[wp] = n;
  float acc[N];
  // acc: the sum of the rows [from, to) of the list of warp w
  const auto sum_rows = [&](const S& cols, int w, int from, int to) {
    F2 sum[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) sum[i] = f2(0.f);
#pragma unroll 1
    for (int j = from; j < to; j += U) {
      Pack<T, N> k[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        k[u] = cols.load_if(j + u < to, dy + list[w][min(j + u, to - 1)] * ld);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        F2 f[N / 2];
        unpack_f2<T, N>(k[u], f);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) sum[i] = sum[i] + f[i];
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      acc[2 * i] = halves(sum[i]).x;
      acc[2 * i + 1] = halves(sum[i]).y;
    }
  };
  __syncwarp();
  if (n > 0 && n <= kWarpRun) {
    const S cols(slab, H);
    sum_rows(cols, wp, 0, n);
    cols.write_run(dtable + mine * ld_t, acc, scale, add);
  }
  __syncthreads();
  for (int w = 0; w < 4; ++w) {
    const int all = found[w];
    if (all <= kWarpRun) continue;
    const int quarter = (all + 3) / 4, other = blockIdx.x * 4 + w;
    const S cols(other / rows, H);
    sum_rows(cols, w, min(all, wp * quarter), min(all, (wp + 1) * quarter));
#pragma unroll
    for (int i = 0; i < N; ++i) share[wp][i * 32 + lane] = acc[i];
    __syncthreads();
    if (wp == 0) {
#pragma unroll
      for (int k = 1; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += share[k][i * 32 + lane];
      cols.write_run(dtable + tok[other % rows] * ld_t, acc, scale, add);
    }
    __syncthreads();
  }
}

template <int W>
__global__ void __launch_bounds__(256) clear_table_kernel(float* __restrict__ t, long long ld,
                                                          long long V, int H) {
  for (long long r = blockIdx.x * 8ll + warp_id(); r < V; r += gridDim.x * 8ll)
    clear_row<W>(t + r * ld, H);
}

}  // namespace cfb

using namespace cfb;

int cfb_scaled_embedding_fwd(const void* table, int type, long long ld, long long V,
                             const void* ids, int ids32, void* out, int out_type,
                             long long ld_out, int rows, int H, float scale, int* err,
                             cudaStream_t st) {
  if (H > kEmbedMaxH) return -11;
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

// 32-bit words: the number of sorted rows, their order, their tokens, the bits of absent tokens, and
// the partial sums, each from a 32-byte border on
static long long words_of_8(long long n) { return (n + 7) / 8 * 8; }

// Blocks of the sort (a power of two) and the places each has for its tokens (whole warps).
struct SortPlan {
  int shift, span;
  long long words() const { return (static_cast<long long>(span) << shift) / 32; }
};
static SortPlan sort_plan(long long V) {
  int shift = 7;  // 128 blocks, or as many as keep the tokens of one under kMaxSpan
  while (((V - 1) >> shift) + 1 > kMaxSpan) ++shift;
  return {shift, static_cast<int>((((V - 1) >> shift) + 32) / 32 * 32)};
}

long long cfb_scaled_embedding_bwd_workspace(long long V, int rows, int H) {
  if (rows <= kFewRows) return 0;
  const int per = chunk_rows(rows);
  const long long chunks = (rows + per - 1) / per;
  return 4 * (8 + 2 * words_of_8(rows) + words_of_8(sort_plan(V).words()) + 2 * chunks * H);
}

int cfb_scaled_embedding_bwd(const void* dy, int type, long long ld, const void* ids, int ids32,
                             long long n_ids, const int* id_rows, long long pad, float* dtable,
                             long long ld_t, long long V, int rows, int H, float scale, int add,
                             void* work, int* err, cudaStream_t st) {
  if (V < 0 || V > (1ll << 30) || (V == 0 && rows > 0) || H > kEmbedMaxH || pad > INT32_MAX)
    return -11;
  if (H == 0 || V == 0) return 0;
  const bool wide = H % 8 == 0 && rows_of_8(dy, ld, type) && rows_of_8(dtable, ld_t, kF32);
  if (rows == 0) {
    if (add) return 0;
    auto* clear = wide ? clear_table_kernel<8> : clear_table_kernel<1>;
    clear<<<static_cast<unsigned>((V + 7) / 8), 256, 0, st>>>(dtable, ld_t, V, H);
    return launch_status();
  }
  const int slab = wide ? SlabCols<8>::kSlab : SlabCols<1>::kSlab;
  const int slabs = (H + slab - 1) / slab;
  if (rows <= kFewRows) {
    const int row_blocks = (rows * slabs + 3) / 4;
    const unsigned blocks =
        row_blocks + (add ? 0 : static_cast<unsigned>((V + kClear - 1) / kClear));
    return with_type(type, [&](auto t) {
      using T = typename decltype(t)::type;
      auto* kernel = wide ? embed_grad_few_kernel<T, 8> : embed_grad_few_kernel<T, 1>;
      kernel<<<blocks, 128, 0, st>>>(static_cast<const T*>(dy), ld, ids, ids32, n_ids, id_rows,
                                     pad, dtable, ld_t, V, rows, H, slabs, row_blocks, scale, add,
                                     err);
      return launch_status();
    });
  }
  int* n_valid = static_cast<int*>(work);
  int* order = n_valid + 8;
  int* stok = order + words_of_8(rows);
  uint32_t* absent = reinterpret_cast<uint32_t*>(stok + words_of_8(rows));
  const SortPlan plan = sort_plan(V);
  float* part = reinterpret_cast<float*>(absent + words_of_8(plan.words()));
  const int smem = static_cast<int>(32 * plan.span * sizeof(int)) +
                   (rows <= kKeyRows ? (rows + 1) / 2 * 4 : 0);
  static bool allowed[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return -3;
  if (!allowed[dev]) {
    if (cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             32 * kMaxSpan * 4 + kKeyRows * 2) != cudaSuccess)
      return -3;
    allowed[dev] = true;
  }
  sort_tokens_kernel<<<1u << plan.shift, 1024, smem, st>>>(
      ids, ids32, static_cast<unsigned>(n_ids < INT32_MAX ? n_ids : INT32_MAX), id_rows, rows,
      static_cast<int>(V), static_cast<int>(pad), plan.shift, plan.span,
      order, stok, n_valid, absent, err);
  if (const int rc = launch_status()) return rc;
  const int per = chunk_rows(rows);
  const int chunks = (rows + per - 1) / per;
  return with_type(type, [&](auto t) {
    using T = typename decltype(t)::type;
    const int sums = static_cast<int>((static_cast<long long>(chunks) * slabs + 3) / 4);
    const int clears = add ? 0 : static_cast<int>((V + kClear - 1) / kClear);
    if (const int rc = launch_behind(wide ? embed_grad_kernel<T, 8> : embed_grad_kernel<T, 1>,
                                     dim3(sums + clears), dim3(128), 0, st,
                                     static_cast<const T*>(dy), ld, order, stok, n_valid, absent,
                                     dtable, ld_t, part, rows, H, slabs, per, sums, plan.shift,
                                     plan.span, static_cast<int>(V), scale, add))
      return rc;
    return launch_behind(wide ? embed_join_kernel<8> : embed_join_kernel<1>,
                         dim3((chunks + 7) / 8, slabs), dim3(256), 0, st, stok, n_valid, dtable,
                         ld_t, part, rows, H, per, scale, add);
  });
}

// Embedding lookup with scaling, and its table gradient by sorted tokens.
//
//   out[n, :]  = scale * table[id_n, :]
//   grad[r, :] = scale * sum over n ascending with id_n = r of dout[n, :]
//
// Both are bound by memory: the lookup reads a row and writes a row per token, the gradient
// reads the tokens' rows and writes the whole table's. (Of 32,768 tokens of 1152 bf16 channels over
// 32,768 rows, half of them padding and the others' ids as frequent as their cube roots fall: lookup
// 23 us, gradient 60 us, of which its sort takes 34 beside clearing the table, and the sum 21 for twice the rows
// that it needs: the padding tokens', which sort last, are read and dropped.) Ids outside the table select its last
// row in both (the host wrappers reject them), so no access can leave it.
//
// The gradient takes no atomics on values. Few tokens: every block owns a few table rows, lists
// the tokens that select them in ascending order and sums their rows. Many tokens: the ids are
// sorted, stably, by a radix sort of at most 10 bits a pass, and the sorted tokens are cut into
// chunks of equal length, so that a frequent row costs no block more than a rare one: a wave
// sums the runs of its chunk, stores the runs that end inside it, and leaves a partial row for
// one that goes on, which a second kernel sums in ascending order.
#include "cond_common.h"

namespace {
using namespace sihc_cond;

// Up to so many tiles the scattering blocks add the counts up themselves, past them one block does for all
// (whole gradients of 64 channels: 16, 32 and 64 tiles 33, 49 and 92 us, with that block 38, 56 and 107).
constexpr int OWN_SCAN = 64;
// Up to so many tokens the rows' tokens are listed by scanning all ids (1152 bf16 channels, 1001 rows: 256 and
// 1024 tokens 4.7 and 5.9 us, by the sort 19.5 and 21.5; 32,768 rows: 1024 tokens 24 and 36, 2048 more than
// 40 and 36). A row that all tokens select is then summed by one block, whose threads add token after token: 256, 512
// and 1024 tokens of one id 42, 82 and 160 us, by the sort 25, 26 and 31 (32,768 rows: 50, 94 and 183; 38, 40 and
// 45). The line is drawn for spread ids; a prompt padded without a padding row is on the wrong side of it.
constexpr int FEW_TOKENS = 1024;
constexpr int FEW_ROWS = 8;  // table rows of a block there, at most

template <typename I>
__device__ __forceinline__ uint32_t id_at(const I* ids, int64_t n, uint32_t rows) {
  const uint64_t id = uint64_t(int64_t(ids[n]));  // a negative id is larger than any row
  return id < rows ? uint32_t(id) : rows - 1u;
}

// ------------------------------------------------------------------------------- lookup
// 32,768 rows of 1152 bf16 channels from 32,768: 23.5 us, 6.4 TB/s of the rows read (in part from the caches)
// and written. UNROLL vectors a thread, a block apart, so that a thread's ids, then its rows, are in flight together;
// the last vector of a row that V does not divide moves back to end with it.
template <typename T, typename I, int V, int UNROLL>
__global__ __launch_bounds__(256) void k_embed(const T* __restrict__ table, const I* __restrict__ ids,
                                               T* __restrict__ out, int64_t items, uint32_t rows, int C, int vecs,
                                               float scale) {
  const int64_t first = int64_t(blockIdx.x) * (256 * UNROLL) + threadIdx.x;
  const T* from[UNROLL];
  int64_t to[UNROLL];
#pragma unroll
  for (int k = 0; k < UNROLL; ++k) {
    const int64_t i = min(first + k * 256, items - 1);  // (threads past the end repeat the last vector)
    const int64_t n = items <= 0x7fffffff ? int64_t(uint32_t(i) / uint32_t(vecs)) : i / vecs;
    const int c = min(int(i - n * vecs) * V, C - V);
    from[k] = table + int64_t(id_at(ids, n, rows)) * C + c;
    to[k] = n * C + c;
  }
  Vec<T, V> row[UNROLL];
#pragma unroll
  for (int k = 0; k < UNROLL; ++k) row[k] = load<T, V>(from[k]);
#pragma unroll
  for (int k = 0; k < UNROLL; ++k) {
    float v[V];
    row[k].to(v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= scale;
    store<T, V>(out + to[k], Vec<T, V>::of(v));
  }
}

// ------------------------------------------------------------------- gradient, few tokens
// Latency: 256 fp32 tokens of 1152 channels over 1001 rows 4.8 us, half of it the scan of the ids. Each thread
// owns an ascending run of the ids, so a prefix sum of the threads' matches lists the
// block's tokens in ascending order.
template <typename T, typename I, int V>
__global__ __launch_bounds__(256) void k_embed_grad_few(const T* __restrict__ grad, const I* __restrict__ ids,
                                                        T* __restrict__ out, int tokens, uint32_t rows, int C, int vecs,
                                                        float scale, int64_t padding, int per_block,
                                                        uint32_t first_row) {
  __shared__ uint32_t list[FEW_TOKENS];  // token << 3 | row of the block
  __shared__ int wave_total[4];
  const int tid = int(threadIdx.x);
  const uint32_t r0 = first_row + blockIdx.x * uint32_t(per_block);
  const int per = (tokens + 255) / 256, begin = min(tokens, tid * per), end = min(tokens, begin + per);
  uint32_t found[FEW_TOKENS / 256];
  int count = 0;
#pragma unroll
  for (int k = 0; k < FEW_TOKENS / 256; ++k) {
    found[k] = ~0u;
    if (begin + k < end) {
      const uint32_t id = id_at(ids, begin + k, rows);
      if (id - r0 < uint32_t(per_block) && int64_t(id) != padding) {
        found[k] = uint32_t(begin + k) << 3 | (id - r0);
        ++count;
      }
    }
  }
  int before = count;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(before, d);
    if ((tid & 63) >= d) before += o;
  }
  if ((tid & 63) == 63) wave_total[tid >> 6] = before;
  __syncthreads();
  int total = 0;
  before -= count;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < (tid >> 6)) before += wave_total[w];
    total += wave_total[w];
  }
#pragma unroll
  for (int k = 0; k < FEW_TOKENS / 256; ++k)
    if (found[k] != ~0u) list[before++] = found[k];
  __syncthreads();
  const int here = min(per_block, int(rows - r0));
  for (int item = tid; item < here * vecs; item += 256) {
    const int row = item / vecs, c = min((item - row * vecs) * V, C - V);
    float sum[V] = {};
    auto add = [&](int k0, auto n) {  // n tokens' rows in flight, the block's other rows' among them
      constexpr int N = decltype(n)::value;
      uint32_t at[N];
      Vec<T, V> v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) at[j] = list[min(k0 + j, total - 1)];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = load<T, V>(grad + int64_t(at[j] >> 3) * C + c);
      __builtin_amdgcn_sched_barrier(0);  // (the loads would be taken apart to save registers)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool own = int(at[j] & 7u) == row && (N == 8 || k0 + j < total);
        float f[V];
        v[j].to(f);
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += own ? f[e] : 0.f;
      }
    };
    int k = 0;
    for (; k + 8 <= total; k += 8) add(k, IC<8>{});
    for (; k < total; k += 2) add(k, IC<2>{});
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] *= scale;
    store<T, V>(out + (int64_t(r0) + row) * C + c, Vec<T, V>::of(sum));
  }
}

// ------------------------------------------------------------------------------ the sort
// Keys of the first pass come from the ids: padding tokens get the key `rows`, which sorts last.
template <typename I>
struct IdKeys {
  const I* ids;
  uint32_t rows;
  int64_t padding;
  __device__ __forceinline__ u32x2 operator()(int64_t n) const {
    const uint32_t id = id_at(ids, n, rows);
    return u32x2{int64_t(id) == padding ? rows : id, uint32_t(n)};
  }
};
struct PairKeys {
  const u32x2* pairs;
  __device__ __forceinline__ u32x2 operator()(int64_t n) const { return pairs[n]; }
};

// n16 vectors and what is left of `bytes`, by `blocks` blocks.
__device__ __forceinline__ void clear(u32x4* p, int64_t bytes, int64_t block, int64_t blocks) {
  const int64_t n16 = bytes / 16;
#pragma unroll 4
  for (int64_t i = block * 256 + threadIdx.x; i < n16; i += blocks * 256) p[i] = u32x4{};
  if (block == 0 && threadIdx.x < (bytes & 15)) reinterpret_cast<uint8_t*>(p + n16)[threadIdx.x] = 0;
}

// One pass of a sort of 32,768 tokens: count 3.7 us (14.0 beside the clearing of 75 MB, 5.4 TB/s), scatter 7.5,
// most of it launch and latency.
// hist[tile][digit]: keys of the tile (256 x STEPS keys) with that digit. Blocks past the tiles clear the table's
// gradient, of which a sort of few blocks leaves the memory's time free.
template <typename K, int STEPS>
__global__ __launch_bounds__(256) void k_sort_count(K keys, uint32_t* __restrict__ hist, int64_t n, int shift, int bins,
                                                    int tiles, u32x4* __restrict__ table, int64_t table_bytes,
                                                    uint32_t* __restrict__ crossing) {
  __shared__ uint32_t h[1024];
  if (blockIdx.x == 0 && threadIdx.x == 0) *crossing = 0;
  if (int(blockIdx.x) >= tiles) return clear(table, table_bytes, blockIdx.x - tiles, gridDim.x - tiles);
  for (int b = int(threadIdx.x); b < bins; b += 256) h[b] = 0;
  __syncthreads();
  const int64_t base = int64_t(blockIdx.x) * (256 * STEPS);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int64_t i = base + k * 256 + threadIdx.x;
    if (i < n) atomicAdd(&h[(keys(i).x >> shift) & uint32_t(bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = int(threadIdx.x); b < bins; b += 256) hist[int64_t(blockIdx.x) * bins + b] = h[b];
}

// Where each tile's keys of each digit go: start[tile][digit] = keys of smaller digits + keys of
// this digit in earlier tiles. One block; a thread owns one digit.
__global__ __launch_bounds__(1024) void k_sort_scan(uint32_t* __restrict__ hist, int tiles, int bins) {
  __shared__ uint32_t wave_total[16];
  const int b = int(threadIdx.x), wave = b >> 6;
  uint32_t total = 0;
  auto each_tile = [&](auto f) {  // f(count) is the new value; 8 tiles' counts are in flight at a time
    if (b < bins)
      for (int t0 = 0; t0 < tiles; t0 += 8) {
        uint32_t c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = hist[int64_t(min(t0 + k, tiles - 1)) * bins + b];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (t0 + k < tiles) hist[int64_t(t0 + k) * bins + b] = f(c[k]);
      }
  };
  each_tile([&](uint32_t c) {
    const uint32_t had = total;
    total += c;
    return had;
  });
  uint32_t before = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(before, d);
    if ((b & 63) >= d) before += o;
  }
  if ((b & 63) == 63) wave_total[wave] = before;
  __syncthreads();
  before -= total;
  for (int w = 0; w < wave; ++w) before += wave_total[w];
  each_tile([&](uint32_t c) { return c + before; });
}

// The same for one tile, by every block for itself: bin b of a thread, b < bins <= 1024.
__device__ __forceinline__ void own_scan(const uint32_t* hist, uint32_t* at, int tile, int tiles, int bins) {
  __shared__ uint32_t wave_total[4];
  const int tid = int(threadIdx.x), wave = tid >> 6;
  const int per = (bins + 255) / 256;  // adjacent bins of a thread
  uint32_t total[4] = {}, earlier[4] = {}, all = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < per && tid * per + k < bins)
      for (int t0 = 0; t0 < tiles; t0 += 16) {  // 16 tiles' counts in flight at a time
        uint32_t c[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) c[j] = hist[int64_t(min(t0 + j, tiles - 1)) * bins + tid * per + k];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (t0 + j < tile) earlier[k] += c[j];
          if (t0 + j < tiles) total[k] += c[j];
        }
      }
#pragma unroll
  for (int k = 0; k < 4; ++k) all += total[k];
  uint32_t before = all;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(before, d);
    if ((tid & 63) >= d) before += o;
  }
  if ((tid & 63) == 63) wave_total[wave] = before;
  __syncthreads();
  before -= all;
  for (int w = 0; w < wave; ++w) before += wave_total[w];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < per && tid * per + k < bins) {
      at[tid * per + k] = before + earlier[k];
      before += total[k];
    }
  __syncthreads();
}

// Stable scatter of a tile: a wave takes 64 keys at a time in ascending order; a key's place among
// its equals is the waves before, the wave's steps before, and the lanes before (a ballot a bit).
template <typename K, int STEPS>
__global__ __launch_bounds__(256) void k_sort_scatter(K keys, const uint32_t* __restrict__ start,
                                                      u32x2* __restrict__ out, int64_t n, int shift, int bits,
                                                      int tiles) {
  __shared__ uint32_t count[4][1024], own[1024];
  const int tid = int(threadIdx.x), wave = tid >> 6, lane = tid & 63, bins = 1 << bits;
  for (int b = tid; b < 4 * 1024; b += 256) (&count[0][0])[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t(blockIdx.x) * 4 + wave) * (64 * STEPS);
  u32x2 key[STEPS];
  uint32_t rank[STEPS];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int64_t i = base + k * 64 + lane;
    key[k] = i < n ? keys(i) : u32x2{0, 0};
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const bool valid = base + k * 64 + lane < n;
    const uint32_t d = (key[k].x >> shift) & uint32_t(bins - 1);
    uint64_t same = __ballot(valid);
    for (int bit = 0; bit < bits; ++bit) {
      const uint64_t set = __ballot((d >> bit) & 1u);
      same &= (d >> bit) & 1u ? set : ~set;
    }
    const int below = __popcll(same & ((uint64_t(1) << lane) - 1));
    uint32_t had = 0;
    if (valid) had = count[wave][d];
    rank[k] = had + uint32_t(below);
    __builtin_amdgcn_wave_barrier();  // (the counters are this wave's own: LDS keeps its order)
    if (valid && below == 0) count[wave][d] = had + uint32_t(__popcll(same));
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  const bool counts = tiles <= OWN_SCAN;  // `start` holds the counts
  if (counts) own_scan(start, own, int(blockIdx.x), tiles, bins);
  for (int b = tid; b < bins; b += 256) {
    uint32_t at = counts ? own[b] : start[int64_t(blockIdx.x) * bins + b];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t c = count[w][b];
      count[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < STEPS; ++k)
    if (base + k * 64 + lane < n) out[count[wave][(key[k].x >> shift) & uint32_t(bins - 1)] + rank[k]] = key[k];
}

// ----------------------------------------------------------------- gradient, sorted tokens
// One wave: CHUNK (8 or 32) sorted tokens x 64 vectors of the row, 8 of them in flight. partial[chunk][0]:
// the run that the chunk before began; [1]: the run that begins here and goes on in the next chunk. A run
// through the whole chunk is [0].
template <typename T, int V, int CHUNK>
__global__ __launch_bounds__(256) void k_embed_grad(const T* __restrict__ grad, const u32x2* __restrict__ sorted,
                                                    T* __restrict__ out, float* __restrict__ partial,
                                                    uint32_t* __restrict__ crossing, int64_t n, int64_t chunks,
                                                    uint32_t rows, int C, int slices, float scale) {
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t chunk = item / slices;
  if (chunk >= chunks) return;
  const int lane = int(threadIdx.x & 63), cb = (int(item - chunk * slices) * 64 + lane) * V;
  const bool on = cb < C;
  const int c = min(cb, C - V);
  const int64_t first = chunk * CHUNK;
  const int here = int(min(int64_t(CHUNK), n - first));
  const u32x2 mine = sorted[first + min(lane, here - 1)];  // (lanes past CHUNK repeat the last)
  const uint32_t prev = first ? sorted[first - 1].x : ~0u;
  const uint32_t next = first + here < n ? sorted[first + here].x : ~0u;
  float sum[V] = {};
  bool head = __shfl(mine.x, 0) == prev;  // the run began before this chunk
  for (int k0 = 0; k0 < here; k0 += 8) {
    Vec<T, V> v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = min(k0 + j, here - 1);
      v[j] = load<T, V>(grad + int64_t(__shfl(mine.y, k)) * C + c);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = k0 + j;
      if (k >= here) break;
      const uint32_t row = __shfl(mine.x, k);
      float f[V];
      v[j].to(f);
#pragma unroll
      for (int e = 0; e < V; ++e) sum[e] += f[e];
      const bool last = k + 1 == here;
      const uint32_t after = last ? next : __shfl(mine.x, min(k + 1, 63));
      if (after == row && !last) continue;
      const bool goes_on = last && after == row;
      if (goes_on && !head && row < rows && cb == 0) crossing[1 + atomicAdd(crossing, 1u)] = uint32_t(chunk);
      if (on && row < rows) {
        if (head || goes_on) {
          float* p = partial + (chunk * 2 + (head ? 0 : 1)) * C + c;
#pragma unroll
          for (int e = 0; e < V; ++e) p[e] = sum[e];
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) sum[e] *= scale;
          store<T, V>(out + int64_t(row) * C + c, Vec<T, V>::of(sum));
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) sum[e] = 0.f;
      head = false;
    }
  }
}

// The runs that cross chunks, of the listed chunks in which they begin: their partial rows of this chunk
// and the following ones are summed, 256 channels a block (blockIdx.y), in ascending order; of a long
// run by 4 thread rows over ascending quarters of the run's chunks, then the quarters in order.
template <typename T>
__global__ __launch_bounds__(256) void k_embed_grad_runs(const u32x2* __restrict__ sorted,
                                                         const float* __restrict__ partial,
                                                         const uint32_t* __restrict__ crossing, T* __restrict__ out,
                                                         int64_t n, int C, float scale, int CHUNK) {
  __shared__ float quarter[4][64];
  const int lane = int(threadIdx.x & 63), q = int(threadIdx.x >> 6);
  const int listed = int(crossing[0]);
  for (int item = int(blockIdx.x); item < listed; item += int(gridDim.x)) {
    const int64_t chunk = crossing[1 + item];
    const uint32_t row = sorted[(chunk + 1) * CHUNK].x;
    int64_t parts = 1;  // chunks after this one that the run reaches: 64 of their ends at a time
    for (;; parts += 64) {
      const int64_t end = (chunk + 1 + parts + lane) * CHUNK;
      const uint64_t stops = __ballot(end >= n || sorted[min(end, n - 1)].x != row);
      if (stops) {
        parts += __builtin_ctzll(stops);
        break;
      }
    }
    const int64_t last = chunk + parts, each = (parts + 3) / 4;
    const float* own = partial + (chunk * 2 + 1) * C;
    for (int base = int(blockIdx.y) * 256; base < C; base += int(gridDim.y) * 256) {
      if (parts <= 16) {
        const int c = base + int(threadIdx.x);
        if (c >= C) continue;
        float sum = own[c];
#pragma unroll 4
        for (int64_t k = chunk + 1; k <= last; ++k) sum += partial[k * 2 * C + c];
        out[int64_t(row) * C + c] = from_f32<T>(scale * sum);
        continue;
      }
      for (int c0 = base; c0 < min(C, base + 256); c0 += 64) {
        const int c = min(c0 + lane, C - 1);
        float sum = q == 0 ? own[c] : 0.f;
        const int64_t begin = chunk + 1 + q * each, end = min(last + 1, begin + each);
#pragma unroll 8
        for (int64_t k = begin; k < end; ++k) sum += partial[k * 2 * C + c];
        quarter[q][lane] = sum;
        __syncthreads();
        if (q == 0 && c0 + lane < C)
          out[int64_t(row) * C + c] =
              from_f32<T>(scale * (((quarter[0][lane] + quarter[1][lane]) + quarter[2][lane]) + quarter[3][lane]));
        __syncthreads();
      }
    }
  }
}

// ---------------------------------------------------------------------------------- host
// The widest vector of a row, at most 16 bytes and the row.
int row_vec(int C, int elem) {
  for (int v : {8, 4, 2})
    if (v * elem <= 16 && v <= C) return v;
  return 1;
}
template <typename F>
int by_vec(int v, F&& f) {
  switch (v) {
    case 8: return f(IC<8>{});
    case 4: return f(IC<4>{});
    case 2: return f(IC<2>{});
    default: return f(IC<1>{});
  }
}
template <typename F>
int by_id(int id_bits, F&& f) {
  return id_bits == 32 ? f(int32_t{}) : f(int64_t{});
}

struct SortPlan {
  int passes, bits;  // of at most 10 bits each
  int steps;         // keys a thread sorts in one pass
  int chunk;         // sorted tokens a wave sums
  int64_t tiles, chunks;
  size_t pairs_bytes, hist_bytes, list_bytes, partial_bytes;  // two pair arrays, counts, runs, partial rows
  size_t total() const { return 2 * pairs_bytes + hist_bytes + list_bytes + partial_bytes; }
};
SortPlan sort_plan(int64_t tokens, int64_t rows, int C) {
  SortPlan p{};
  int bits = 1;
  while ((int64_t(1) << bits) < rows + 1) ++bits;
  p.passes = (bits + 9) / 10;
  p.bits = (bits + p.passes - 1) / p.passes;
  // (whole gradients of 64 channels: 32,768 tokens 48 us by 4 steps, 65 by 16; 131,072: 111, 96)
  p.steps = tokens <= 1024 * OWN_SCAN ? 4 : 16;
  p.tiles = ceil_div(tokens, 256 * p.steps);
  // short chunks where long ones would leave most of the card idle (bf16, 1152 channels, 32,768 rows, the whole
  // gradient: 4,096 tokens 39 us by chunks of 8, 46 of 32; 16,384: 49, 48; 32,768: 70, 58; 256 channels alike)
  p.chunk = tokens <= 16384 ? 8 : 32;
  p.chunks = ceil_div(tokens, p.chunk);
  p.pairs_bytes = size_t(ceil_div(tokens * 8, 256)) * 256;
  p.hist_bytes = size_t(ceil_div(p.tiles * (int64_t(4) << p.bits), 256)) * 256;
  p.list_bytes = size_t(ceil_div((p.chunks + 1) * 4, 256)) * 256;
  p.partial_bytes = size_t(p.chunks) * 2 * size_t(C) * 4;
  return p;
}

int check_sizes(const char* what, int64_t tokens, int64_t rows, int C, int id_bits, int dtype) {
  if (tokens < 0 || tokens >= SIHC_MAX_TOKENS || rows <= 0 || rows >= SIHC_MAX_TOKENS || C <= 0 || C > (1 << 24))
    return fail(SIHC_ERR_INVALID, "%s: bad sizes", what);
  if (id_bits != 32 && id_bits != 64) return fail(SIHC_ERR_INVALID, "%s: ids of %d bits (32 or 64)", what, id_bits);
  if (!valid_dtype(dtype)) return fail(SIHC_ERR_INVALID, "%s: bad dtype %d", what, dtype);
  return SIHC_OK;
}

}  // namespace

extern "C" {

int sihc_embedding(const void* table, const void* ids, void* out, int64_t tokens, int64_t rows, int channels,
                   float scale, int id_bits, int dtype, void* stream) {
  const char* what = "sihc_embedding";
  if (int rc = check_sizes(what, tokens, rows, channels, id_bits, dtype)) return rc;
  if (tokens == 0) return SIHC_OK;
  if (!table || !ids || !out) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_id(id_bits, [&](auto i) {
      using I = decltype(i);
      return by_vec(row_vec(channels, int(sizeof(T))), [&](auto v) {
        constexpr int V = decltype(v)::value;
        if constexpr (V * sizeof(T) <= 16) {
          const int vecs = int(ceil_div(channels, V));
          const int64_t items = tokens * vecs;
          auto launch = [&](auto unroll) {
            constexpr int U = decltype(unroll)::value;
            const int64_t blocks = ceil_div(items, 256 * U);
            if (blocks > MOST_LAUNCHED / 256) return fail(SIHC_ERR_INVALID, "%s: tensor too large", what);
            hipLaunchKernelGGL((k_embed<T, I, V, U>), dim3(unsigned(blocks)), dim3(256), 0,
                               static_cast<hipStream_t>(stream), static_cast<const T*>(table),
                               static_cast<const I*>(ids), static_cast<T*>(out), items, uint32_t(rows), channels, vecs,
                               scale);
            return check_launch(what);
          };
          // several vectors a thread once that leaves 4 blocks to a CU (8,192 rows of 1152 bf16 channels: 6.8 us,
          // one vector a thread 7.1; 2,048: 4.0 and 3.8)
          return items >= 256 * 4 * 1024 ? launch(IC<4>{}) : launch(IC<1>{});
        }
        return check_launch(what);
      });
    });
  });
}

size_t sihc_embedding_backward_workspace_size(int64_t tokens, int64_t rows, int channels) {
  if (check_sizes("sihc_embedding_backward", tokens, rows, channels, 32, SIHC_DTYPE_F32) || tokens <= FEW_TOKENS) return 0;
  return sort_plan(tokens, rows, channels).total();
}

int sihc_embedding_backward(const void* grad, const void* ids, void* grad_table, int64_t tokens, int64_t rows,
                            int channels, float scale, int64_t padding, int id_bits, int dtype, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* what = "sihc_embedding_backward";
  if (int rc = check_sizes(what, tokens, rows, channels, id_bits, dtype)) return rc;
  if (!grad_table || (tokens && (!grad || !ids))) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  if (grad_table == grad || grad_table == ids) return fail(SIHC_ERR_INVALID, "%s: an output is one of the inputs", what);
  const size_t need = sihc_embedding_backward_workspace_size(tokens, rows, channels);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SIHC_ERR_INVALID, "%s: workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  if (need && !aligned(workspace, 16)) return fail(SIHC_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_id(id_bits, [&](auto i) {
      using I = decltype(i);
      return by_vec(row_vec(channels, int(sizeof(T))), [&](auto v) {
        constexpr int V = decltype(v)::value;
        if constexpr (V * sizeof(T) <= 16) {
          const int vecs = int(ceil_div(channels, V));
          const T* g = static_cast<const T*>(grad);
          const I* id = static_cast<const I*>(ids);
          T* out = static_cast<T*>(grad_table);
          if (tokens <= FEW_TOKENS) {
            // about two vectors a thread: more rows would follow one another (64 fp32 tokens of 1152 channels:
            // one row 5.0 us, 8 rows 7.7)
            const int per_block = std::max(1, std::min(FEW_ROWS, 512 / vecs));
            // (134 million narrow rows are more blocks than one launch takes)
            const int64_t step = MOST_LAUNCHED / 256 * per_block;
            int rc = SIHC_OK;
            for (int64_t r = 0; r < rows && !rc; r += step) {
              hipLaunchKernelGGL((k_embed_grad_few<T, I, V>), dim3(unsigned(ceil_div(std::min(step, rows - r), per_block))),
                                 dim3(256), 0, st, g, id, out, int(tokens), uint32_t(rows), channels, vecs, scale, padding,
                                 per_block, uint32_t(r));
              rc = check_launch(what);
            }
            return rc;
          }
          const SortPlan p = sort_plan(tokens, rows, channels);
          char* w = static_cast<char*>(workspace);
          u32x2* pairs[2] = {reinterpret_cast<u32x2*>(w), reinterpret_cast<u32x2*>(w + p.pairs_bytes)};
          uint32_t* hist = reinterpret_cast<uint32_t*>(w + 2 * p.pairs_bytes);
          uint32_t* crossing = reinterpret_cast<uint32_t*>(w + 2 * p.pairs_bytes + p.hist_bytes);
          float* partial = reinterpret_cast<float*>(w + 2 * p.pairs_bytes + p.hist_bytes + p.list_bytes);
          const int64_t bytes = rows * channels * int64_t(sizeof(T));
          if (!aligned(out, 16)) return fail(SIHC_ERR_INVALID, "%s: grad_table must be 16-byte aligned", what);
          const unsigned tiles = unsigned(p.tiles), clearing = unsigned(std::min<int64_t>(ceil_div(bytes, 16384) + 1, 2048));
          auto tiled_pass = [&](auto keys, auto n, u32x2* to, int shift) {
            using K = decltype(keys);
            constexpr int STEPS = decltype(n)::value;
            hipLaunchKernelGGL((k_sort_count<K, STEPS>), dim3(tiles + (shift ? 0 : clearing)), dim3(256), 0, st, keys, hist,
                               tokens, shift, 1 << p.bits, int(tiles), reinterpret_cast<u32x4*>(out), bytes, crossing);
            if (p.tiles > OWN_SCAN)
              hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, st, hist, int(tiles), 1 << p.bits);
            hipLaunchKernelGGL((k_sort_scatter<K, STEPS>), dim3(tiles), dim3(256), 0, st, keys, hist, to, tokens, shift,
                               p.bits, int(tiles));
          };
          auto pass = [&](auto keys, u32x2* to, int shift) {
            if (p.steps == 4) tiled_pass(keys, IC<4>{}, to, shift);
            else tiled_pass(keys, IC<16>{}, to, shift);
          };
          pass(IdKeys<I>{id, uint32_t(rows), padding}, pairs[0], 0);
          for (int k = 1; k < p.passes; ++k) pass(PairKeys{pairs[(k + 1) & 1]}, pairs[k & 1], k * p.bits);
          const u32x2* sorted = pairs[(p.passes - 1) & 1];
          const int slices = int(ceil_div(vecs, 64));
          const int64_t blocks = ceil_div(p.chunks * slices, 4);
          if (blocks > MOST_LAUNCHED / 256) return fail(SIHC_ERR_INVALID, "%s: tensor too large", what);
          auto sum = [&](auto chunk) {
            hipLaunchKernelGGL((k_embed_grad<T, V, decltype(chunk)::value>), dim3(unsigned(blocks)), dim3(256), 0, st, g,
                               sorted, out, partial, crossing, tokens, p.chunks, uint32_t(rows), channels, slices, scale);
          };
          if (p.chunk == 8) sum(IC<8>{});
          else sum(IC<32>{});
          const unsigned listed = unsigned(std::min<int64_t>(p.chunks, 1024)),
                         columns = unsigned(std::min<int64_t>(ceil_div(channels, 256), 64));
          hipLaunchKernelGGL(k_embed_grad_runs<T>, dim3(listed, columns), dim3(256), 0, st, sorted, partial, crossing, out,
                             tokens, channels, scale, p.chunk);
        }
        return check_launch(what);
      });
    });
  });
}

}  // extern "C"

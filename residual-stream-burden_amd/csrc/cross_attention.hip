// Cross attention to states of another length, and its gradients.
//
//   S = scale q k^T over the first lengths[b] keys, P = softmax(S), O = P v
//   dV = P^T dO;  dP = dO V^T;  dS = P (dP - rowsum(dO O));  dQ = scale dS K;  dK = scale dS^T Q
//
// Every product runs on the matrix cores in 32 x 32 tiles (bf16 32x32x16, fp32 32x32x2, fp32 sums).
// A wave owns 32 rows of one side, one a lane pair, as the columns of its tiles: queries in the
// forward and the query gradient, keys in the key and value gradients. The other side passes
// through LDS in pieces that the block's waves share. The tile of scores then has its own row's
// 32 values in the registers of two lanes, 16 each, so that the softmax needs one exchange per
// tile, and the probabilities are already laid out as an operand of the next product, whose
// contraction runs over them in the order the registers have (the other operand is read in the
// same order). Transposed operands are read from LDS by the transposing load.
//
// The query rows of all heads that share a key head are one list of rows (head by head), so shared
// heads fill tiles together, and their key gradients are one sum.
//
// What bounds it, at 4 images, 16 heads of 64 over 4 key heads, 4,096 rows over up to 2,048 keys (bf16): the
// matrix and vector instructions between them. A training pass takes 570 us, half the rate of a large matrix
// product, because a wave's exponentials and its products share one SIMD and its tiles leave it one to two
// other waves to run beside. (Traced, where launches of this case are slower: the forward 172, the query
// gradient 204, the key and value gradients 319, their parts' sum 8.) At 256 rows over 256 keys (64 images,
// 16 heads of 72) the blocks live for a few pieces only, and their loads' latency bounds them: 198 us a
// training pass, 2.4 times the time of the bytes (traced 64, 75 and 78). One row over 4,096 keys (8 images, 16
// heads of 128 over 4): 17 us of 67 MB, and 4.5 us to join.
//
// Rounding: probabilities and score gradients enter their products in the inputs' type (a bf16 gradient is
// then 1.4 times as far from the exact one as its own rounding puts it: two products' operands are rounded,
// and fp32 operands would take eight times the matrix time); scores, statistics, sums and the row sums of
// dO O stay in fp32.
#include "cond_common.h"

namespace {
using namespace sihc_cond;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int PIECE = 64;  // rows of the other side in LDS at a time
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void *q, *k, *v, *grad, *out, *low;
  void *o, *o_low, *dq, *dk, *dv;
  const int32_t* lengths;
  float2* stats;
  float* delta;  // [batch, heads, queries] rowsum(dO O)
  int64_t qs[3], ks[3], vs[3];
  int64_t batch;
  int queries, keys, heads, shared, each, dim;
  int64_t rows;   // query rows of a key head: each * queries
  int64_t tiles;  // blocks of a key head (in the forward, of one part of its keys)
  int cluster;       // (unit_of)
  int splits;        // parts of a key head's keys (forward) or query rows (key and value gradients)
  int64_t span;      // keys or rows of a part, a multiple of PIECE
  float* part_o;     // where there are several: [splits][batch, key head][rows][dim] sums (forward), or
                     // [splits][2][batch, keys, key heads, dim] (gradients of keys and values)
  float2* part_s;    // (forward) their bases and sums of powers
  float scale;
  bool fast;               // (Piece)
  uint32_t magic;  // r / queries is the high word of r * magic, shifted right (0: r shifted right)
  int shift;
};

// ------------------------------------------------------------------------------ fragments
template <typename T, int DP>
struct Lds {  // a piece in LDS: rows of DP channels (zeros past dim), padded against bank conflicts
  static constexpr int STRIDE = DP + 16 / int(sizeof(T));
  static constexpr int SIZE = PIECE * STRIDE + 32;  // (the last row's reads may run past its end)
};
template <int DP>
constexpr int d_tiles() { return (DP + 31) / 32; }

// A wave's own 32 rows as the right operand of a product over channels.
template <typename T, int DP>
struct Own;
template <int DP>
struct Own<bf16, DP> { bf16x8 v[DP / 16]; };
template <int DP>
struct Own<float, DP> { f32x4 v[DP / 8]; };

// n elements of a row from p, as far as the row's `left` go, zeros past them.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_some(const T* p, int left) {
  if (left >= N) return load<T, N>(p);
  T e[N] = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < left) e[i] = p[i];
  Vec<T, N> v;
  __builtin_memcpy(&v.raw, e, sizeof(e));
  return v;
}
// The loads are apart from their use, so that those of several tensors are in flight together: heads of
// whole vectors load without branches, from places that exist, and take their zeros in own().
template <typename T, int DP>
struct OwnLoads {
  static constexpr int N = 16 / int(sizeof(T));  // 8 or 4: the lane's channels of one step
  static constexpr int STEPS = DP / (2 * N);
  Vec<T, N> v[STEPS];
  __device__ __forceinline__ OwnLoads(const T* row, bool valid, int dim, int half) {
    if (dim % N == 0) {
#pragma unroll
      for (int k = 0; k < STEPS; ++k) v[k] = load<T, N>(row + min(k * 2 * N + half * N, dim - N));
    } else {
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const int c = k * 2 * N + half * N;
        v[k] = valid ? load_some<T, N>(row + c, dim - c) : Vec<T, N>::zero();
      }
    }
  }
  __device__ __forceinline__ Own<T, DP> own(bool valid, int dim, int half) const {
    Own<T, DP> out;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const u32x4 w = !valid || k * 2 * N + half * N >= dim ? u32x4{} : v[k].raw;
      __builtin_memcpy(&out.v[k], &w, 16);
    }
    return out;
  }
};

// acc[r, own] + sum over channels of piece[r, c] own[c], r one of 32 rows from `piece`.
template <int DP>
__device__ __forceinline__ f32x16 rows_product(const bf16* piece, const Own<bf16, DP>& own, int lane, int half,
                                               f32x16 acc = f32x16{}) {
  const bf16* p = piece + lane * Lds<bf16, DP>::STRIDE + half * 8;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(p + k * 16), own.v[k], acc, 0, 0, 0);
  return acc;
}
template <int DP>
__device__ __forceinline__ f32x16 rows_product(const float* piece, const Own<float, DP>& own, int lane, int half,
                                               f32x16 acc = f32x16{}) {
  const float* p = piece + lane * Lds<float, DP>::STRIDE + half * 4;
#pragma unroll
  for (int k = 0; k < DP / 8; ++k) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p + k * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], own.v[k][j], acc, 0, 0, 0);
  }
  return acc;
}
// Row of a tile that register i of a lane's half holds.
__device__ __forceinline__ constexpr int row_of(int i, int half) { return (i / 4) * 8 + half * 4 + i % 4; }

// A tile of probabilities or score gradients as the right operand of a product over its rows.
template <typename T>
struct Tile;
template <>
struct Tile<bf16> {
  bf16x8 v[2];  // registers 0..7 and 8..15
  __device__ __forceinline__ explicit Tile(const f32x16& p) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = static_cast<__bf16>(p[k * 8 + i]);
  }
  // Sum of the lane's 16 values as rounded: the weights that the values are multiplied by.
  __device__ __forceinline__ float add_to(float sum) const {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair ones = __builtin_bit_cast(pair, 0x3f803f80u);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        sum = __builtin_amdgcn_fdot2_f32_bf16(pair{v[k][i], v[k][i + 1]}, ones, sum, false);
    return sum;
  }
};
template <>
struct Tile<float> {
  f32x16 v;
  __device__ __forceinline__ explicit Tile(const f32x16& p) : v(p) {}
  __device__ __forceinline__ float add_to(float sum) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += v[i];
    return sum;
  }
};

// acc[t][c, own] += sum over the 32 rows r from `piece` of piece[r, 32 t + c] p[r, own].
template <int DP>
__device__ __forceinline__ void columns_product(f32x16* acc, const bf16* piece, const Tile<bf16>& p, int lane, int half) {
  constexpr int S = Lds<bf16, DP>::STRIDE;
  typedef __attribute__((address_space(3))) s16x4* LdsPtr;
  const int j = lane & 15;
  const bf16* at = piece + (half * 4 + j / 4) * S + (lane & 16) + (j % 4) * 4;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int t = 0; t < d_tiles<DP>(); ++t) {
      const bf16* low = at + k * 16 * S + t * 32;
      const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)low);
      const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(low + 8 * S));
      const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
      acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, p.v[k], acc[t], 0, 0, 0);
    }
  }
}
template <int DP>
__device__ __forceinline__ void columns_product(f32x16* acc, const float* piece, const Tile<float>& p, int lane, int half) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int t = 0; t < d_tiles<DP>(); ++t)
      acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(piece[row_of(i, half) * Lds<float, DP>::STRIDE + t * 32 + lane], p.v[i],
                                                    acc[t], 0, 0, 0);
}

// PIECE rows on their way to LDS: loaded into registers while the piece before is worked on. Heads of
// whole 16-byte vectors whose rows lie within 32-bit offsets of `base` (Args::fast) load without
// branches, from places that exist, so that all loads are in flight at once; others are loaded when
// they are stored. offset(r) is the byte offset of row r of the piece; rows past `valid` and channels
// past dim are zeros.
template <typename T, int DP, int THREADS>
struct Piece {
  static constexpr int N = 16 / int(sizeof(T)), VECS = DP / N, COUNT = (PIECE * VECS + THREADS - 1) / THREADS;
  static constexpr bool HELD = COUNT <= 16;  // (fp32 pieces of one wave would fill its registers)
  Vec<T, N> v[COUNT];
  template <typename Offset>
  __device__ __forceinline__ void fetch(const void* base, Offset offset, int valid, int dim) {
    const char* from = static_cast<const char*>(base);
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
      const int i = int(threadIdx.x) + k * THREADS, r = i / VECS, c = (i - r * VECS) * N;
      const uint32_t at = offset(min(r, valid - 1)) + uint32_t(min(c, dim - N)) * uint32_t(sizeof(T));
      v[k] = load<T, N>(reinterpret_cast<const T*>(from + at));
    }
  }
  // (the zeros are put in here: in fetch() they would wait for the loads)
  __device__ __forceinline__ void commit(T* lds, int valid, int dim) const {
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
      const int i = int(threadIdx.x) + k * THREADS, r = i / VECS, c = (i - r * VECS) * N;
      const u32x4 w = r >= valid || c >= dim ? u32x4{} : v[k].raw;
      if (PIECE * VECS % THREADS == 0 || r < PIECE) *reinterpret_cast<u32x4*>(lds + r * Lds<T, DP>::STRIDE + c) = w;
    }
  }
  template <typename Row>
  __device__ static void copy(T* lds, Row row, int valid, int dim) {
    constexpr int UNROLL = HELD ? 1 : 4;  // (4 loads in flight where this is the only way in)
#pragma unroll UNROLL
    for (int i = int(threadIdx.x); i < PIECE * VECS; i += THREADS) {
      const int r = i / VECS, c = (i - r * VECS) * N;
      Vec<T, N> v;
      if (!HELD && dim % N == 0) {
        v = load<T, N>(row(min(r, valid - 1)) + min(c, dim - N));
        if (r >= valid || c >= dim) v = Vec<T, N>::zero();
      } else {
        v = r < valid ? load_some<T, N>(row(r) + c, dim - c) : Vec<T, N>::zero();
      }
      *reinterpret_cast<u32x4*>(lds + r * Lds<T, DP>::STRIDE + c) = v.raw;
    }
  }
};

// A wave's 32 rows of sums, times f, to `to` + the rows' offsets (each lane's own). They pass through the
// wave's part of LDS (32 rows of a piece), so that a store writes whole 16-byte vectors of adjacent
// channels: straight from the registers it would write 8 bytes of each of 64 rows. Every wave of the
// block calls it, with `rows` in use by none.
template <typename T, int DP, typename TO>
__device__ __forceinline__ void store_rows(TO* to, int64_t offset, bool valid, T* rows, const f32x16* acc, float f, int dim,
                                           int lane, int half) {
  constexpr int N = 16 / int(sizeof(TO)), VECS = DP / N;
  if constexpr (sizeof(TO) == sizeof(T)) {
    constexpr int S = Lds<T, DP>::STRIDE;
#pragma unroll
    for (int t = 0; t < d_tiles<DP>(); ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        if (t * 32 + (i / 4) * 8 >= DP) continue;
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = acc[t][i + j] * f;
        const Vec<T, 4> v = Vec<T, 4>::of(e);
        __builtin_memcpy(rows + lane * S + t * 32 + row_of(i, half), &v.raw, sizeof(v.raw));
      }
    __syncthreads();
    const int lane64 = half * 32 + lane, mine = valid ? 1 : 0;
    for (int i = lane64; i < 32 * VECS; i += 64) {
      const int r = i / VECS, c = (i - r * VECS) * N;
      const int64_t at = (int64_t(__shfl(int(offset >> 32), r)) << 32) | uint32_t(__shfl(int(offset), r));
      if (!__shfl(mine, r) || c >= dim) continue;
      Vec<T, N> v;
      __builtin_memcpy(&v.raw, rows + r * S + c, 16);
      if (c + N <= dim) {
        store<T, N>(to + at + c, v);
      } else {
        T e[N];
        __builtin_memcpy(e, &v.raw, 16);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (c + j < dim) to[at + c + j] = e[j];
      }
    }
    __syncthreads();
  } else if (valid) {  // fp32 parts of bf16 inputs: 16 bytes from each lane
#pragma unroll
    for (int t = 0; t < d_tiles<DP>(); ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int c = t * 32 + row_of(i, half);
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = acc[t][i + j] * f;
        if (c + 4 <= dim) {
          store<TO, 4>(to + offset + c, Vec<TO, 4>::of(e));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < dim) to[offset + c + j] = e[j];
        }
      }
  }
}

// ------------------------------------------------------------------------------ addresses
struct Unit {  // what a block works on
  int64_t b, tile;
  int split;
  int g;    // key head
  int len;  // keys of the batch row
};
// Blocks of a key head share its keys (or its queries), and neighbouring heads the lines at the ends of
// their rows' pieces, so `cluster` heads go to one XCD, whose L2 they meet in; the clusters go to the
// XCDs in turn, so that the rows of the batch, of different lengths, are spread over all of them.
// Heads of many blocks are spread themselves: what they share is small against their work.
__device__ __forceinline__ Unit unit_of(const Args& a) {
  const int64_t block = blockIdx.x, parts = a.batch * a.shared * a.splits;
  int64_t part = block / a.tiles;
  Unit u;
  u.tile = block - part * a.tiles;
  const int64_t round = 8 * a.cluster, whole = parts - parts % round;  // (the last parts: in order)
  if (a.tiles < 8 && block < whole * a.tiles) {
    const int64_t i = block >> 3, in = i / a.tiles, row = in / a.cluster;  // of this XCD: part and round
    part = row * round + (block & 7) * a.cluster + (in - row * a.cluster);
    u.tile = i - in * a.tiles;
  }
  // (parts of the sums are the slowest, so that neighbours are of one batch row and other heads)
  const int64_t heads = a.batch * a.shared;
  u.split = int(part / heads);
  const int64_t bg = part - u.split * heads;
  u.b = bg / a.shared;
  u.g = int(bg - u.b * a.shared);
  u.len = a.lengths ? min(max(a.lengths[u.b], 0), a.keys) : a.keys;
  return u;
}
struct QueryRow {
  int head, query;
};
__device__ __forceinline__ QueryRow query_row(const Args& a, const Unit& u, int64_t r) {
  const uint32_t h = uint32_t(r) / uint32_t(a.queries);
  return {u.g * a.each + int(h), int(uint32_t(r) - h * uint32_t(a.queries))};
}
// r / queries, without a division.
__device__ __forceinline__ uint32_t fast_query_head(const Args& a, uint32_t r) {
  return a.magic ? uint32_t((uint64_t(r) * a.magic) >> 32) >> a.shift : r >> a.shift;
}
template <typename T>
__device__ __forceinline__ const T* q_at(const Args& a, const Unit& u, QueryRow r) {
  return static_cast<const T*>(a.q) + u.b * a.qs[0] + r.query * a.qs[1] + r.head * a.qs[2];
}
__device__ __forceinline__ int64_t packed_q(const Args& a, const Unit& u, QueryRow r) {
  return ((u.b * a.queries + r.query) * a.heads + r.head) * a.dim;
}
__device__ __forceinline__ int64_t stat_at(const Args& a, const Unit& u, QueryRow r) {
  return (u.b * a.heads + r.head) * a.queries + r.query;
}
template <typename T>
__device__ __forceinline__ const T* k_at(const Args& a, const Unit& u, int64_t key) {
  return static_cast<const T*>(a.k) + u.b * a.ks[0] + key * a.ks[1] + u.g * a.ks[2];
}
template <typename T>
__device__ __forceinline__ const T* v_at(const Args& a, const Unit& u, int64_t key) {
  return static_cast<const T*>(a.v) + u.b * a.vs[0] + key * a.vs[1] + u.g * a.vs[2];
}

// What a value loses when it is stored (an infinity or NaN loses nothing that could be added back).
template <typename T>
__device__ __forceinline__ float lost(float v) {
  const float d = v - to_f32(from_f32<T>(v));
  return fabsf(d) < INFINITY ? d : 0.f;
}

// Where a wave's 32 rows lie in the two pieces' LDS (SIZE is not less than 64 rows).
template <typename T, int DP>
__device__ __forceinline__ int wave_rows() { return int(threadIdx.x >> 6) * 32 * Lds<T, DP>::STRIDE; }

// Blocks of several waves are compiled for two waves on a SIMD where their tiles fit 256 registers, three where
// they fit 168 or nearly: the softmax of one wave then runs beside the products of another. bf16 forwards over
// heads of 64 and 80 channels spill 3 and 7 registers for the third wave (16 and 32 bytes a lane; fp32 ones of 96
// 6, some query gradients 1), and all forwards keep 26 to 62 scalars in lanes of vector registers: both ways of
// loading a piece live in one kernel.
// -------------------------------------------------------------------------------- forward
constexpr int forward_waves(int bytes, bool halves, int NW) {  // waves of a SIMD; bytes of a head's row
  return NW == 1 || bytes > 384 ? 1 : halves && bytes <= 160 ? 3 : 2;
}
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, forward_waves(sizeof(T) * DP, sizeof(T) == 2, NW)) void k_attend(Args a) {
  __shared__ __attribute__((aligned(16))) T lds[2 * Lds<T, DP>::SIZE];
  T *const lds_k = lds, *const lds_v = lds + Lds<T, DP>::SIZE, *const mine = lds + wave_rows<T, DP>();
  const Unit u = unit_of(a);
  const int lane = int(threadIdx.x & 31), half = int(threadIdx.x >> 5 & 1), wave = int(threadIdx.x >> 6);
  const int64_t r = u.tile * (NW * 32) + wave * 32 + lane;
  const bool valid = r < a.rows;
  const QueryRow qr = query_row(a, u, valid ? r : 0);
  const float c = a.scale * LOG2E;
  f32x16 o[d_tiles<DP>()] = {};
  float top = -INFINITY, sum = 0.f;  // sum: of the keys of this lane's half
  const int begin = int(u.split * a.span), end = int(min(int64_t(u.len), begin + a.span));
  Piece<T, DP, NW * 64> pk, pv;
  const bool fast = pk.HELD && a.fast;
  auto fetch = [&](int k0) {
    const int here = min(PIECE, end - k0);
    const uint32_t ks = uint32_t(a.ks[1]) * uint32_t(sizeof(T)), vs = uint32_t(a.vs[1]) * uint32_t(sizeof(T));
    pk.fetch(k_at<T>(a, u, k0), [&](int i) { return uint32_t(i) * ks; }, here, a.dim);
    pv.fetch(v_at<T>(a, u, k0), [&](int i) { return uint32_t(i) * vs; }, here, a.dim);
  };
  Own<T, DP> q;
  if (begin < end) {
    const OwnLoads<T, DP> lq(q_at<T>(a, u, qr), valid, a.dim, half);
    if (fast) fetch(begin);
    q = lq.own(valid, a.dim, half);
  }
  for (int k0 = begin; k0 < end; k0 += PIECE) {
    const int here = min(PIECE, end - k0);
    __syncthreads();
    if (fast) {
      pk.commit(lds_k, here, a.dim);
      pv.commit(lds_v, here, a.dim);
    } else {
      Piece<T, DP, NW * 64>::copy(lds_k, [&](int i) { return k_at<T>(a, u, k0 + i); }, here, a.dim);
      Piece<T, DP, NW * 64>::copy(lds_v, [&](int i) { return v_at<T>(a, u, k0 + i); }, here, a.dim);
    }
    __syncthreads();
    if (fast && k0 + PIECE < end) fetch(k0 + PIECE);
    // Scores under the base of earlier pieces need no maximum as long as their powers stay small: a base
    // is a scale, and sums keep their digits under any. The first piece, and one whose powers grow
    // past 2^40, take their maximum as the new base, on scores computed again. (So values may be as large as
    // 2^128 / 2^40 over the pieces' number before a sum overflows whose quotient would not.)
    bool anew = __any(top == -INFINITY);
    for (;;) {
      asm volatile("" ::: "memory");  // (operands are read in every turn, not held across them)
      f32x16 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = rows_product<DP>(lds_k + t * 32 * Lds<T, DP>::STRIDE, q, lane, half);
      if (anew) {
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (t * 32 + row_of(i, half) < here) most = fmaxf(most, s[t][i] * c);
        most = fmaxf(most, __shfl_xor(most, 32));
        const float now = fmaxf(top, most), keep = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - now);
        top = now;
        sum *= keep;
#pragma unroll
        for (int t = 0; t < d_tiles<DP>(); ++t) o[t] *= keep;
      }
      const float base = top == -INFINITY ? 0.f : top;  // (every score so far is -inf)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], c, -base));
      if (here < PIECE) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (t * 32 + row_of(i, half) >= here) s[t][i] = 0.f;
      }
      const Tile<T> p0(s[0]), p1(s[1]);
      const float more = p1.add_to(p0.add_to(0.f));
      if (!anew && __any(more > 0x1p40f)) {
        anew = true;
        continue;
      }
      sum += more;
      columns_product<DP>(o, lds_v, p0, lane, half);
      columns_product<DP>(o, lds_v + 32 * Lds<T, DP>::STRIDE, p1, lane, half);
      break;
    }
  }
  sum += __shfl_xor(sum, 32);
  __syncthreads();
  if (a.splits > 1) {
    const int64_t row = ((int64_t(u.split) * a.batch + u.b) * a.shared + u.g) * a.rows + r;
    if (valid && half == 0) a.part_s[row] = {top, sum};
    store_rows<T, DP>(a.part_o, row * a.dim, valid, mine, o, 1.f, a.dim, lane, half);  // (zeros past the length)
    return;
  }
  const float inverse = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // (NaN stays NaN)
  if (valid && a.stats && half == 0) a.stats[stat_at(a, u, qr)] = {top == -INFINITY ? 0.f : top, inverse};
  store_rows<T, DP>(static_cast<T*>(a.o), packed_q(a, u, qr), valid, mine, o, inverse, a.dim, lane, half);
  if (sizeof(T) == 2 && a.o_low) {
#pragma unroll
    for (int t = 0; t < d_tiles<DP>(); ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][i] = lost<T>(o[t][i] * inverse);
    store_rows<T, DP>(static_cast<T*>(a.o_low), packed_q(a, u, qr), valid, mine, o, 1.f, a.dim, lane, half);
  }
}

// The parts of a row, brought under their largest score and summed: a block a row, of 8 groups of 32 lanes
// that take every eighth part, 4 channels a lane, and whose sums are added in order. Latency: 4.4 us for 128
// rows of 32 parts of 128 channels.
template <typename T>
__global__ __launch_bounds__(256) void k_attend_join(Args a, int64_t total) {
  __shared__ f32x4 lds_o[8][32];
  __shared__ float lds_sum[8];
  const int64_t row = blockIdx.x;
  const int lane = int(threadIdx.x & 31), group = int(threadIdx.x >> 5);
  const int64_t bg = row / a.rows;
  Unit u;
  u.b = bg / a.shared;
  u.g = int(bg - u.b * a.shared);
  const QueryRow qr = query_row(a, u, row - bg * a.rows);
  float top = -INFINITY;
  for (int s = int(threadIdx.x & 63); s < a.splits; s += 64) top = fmaxf(top, a.part_s[s * total + row].x);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  f32x4 o = {};
  const int c = min(lane * 4, max(a.dim - 4, 0)), n = min(4, a.dim);
#pragma unroll 4
  for (int s = group; s < a.splits; s += 8) {
    const float2 p = a.part_s[s * total + row];
    const float worth = __builtin_amdgcn_exp2f(p.x - base);
    sum += worth * p.y;
    const float* from = a.part_o + (s * total + row) * a.dim + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(worth, from[min(e, n - 1)], o[e]);
  }
  lds_o[group][lane] = o;
  if (lane == 0) lds_sum[group] = sum;
  __syncthreads();
  if (group) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    o += lds_o[k][lane];
    sum += lds_sum[k];
  }
  const float inverse = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  T* to = static_cast<T*>(a.o) + packed_q(a, u, qr) + c;
  T* low = a.o_low ? static_cast<T*>(a.o_low) + packed_q(a, u, qr) + c : nullptr;
  if (lane * 4 < a.dim)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) {
        to[e] = from_f32<T>(o[e] * inverse);
        if (sizeof(T) == 2 && low) low[e] = from_f32<T>(lost<T>(o[e] * inverse));
      }
  if (a.stats && lane == 0) a.stats[stat_at(a, u, qr)] = {base, inverse};
}

// The statistics of a row as a gradient's kernel takes them: bf16 folds the sum into the exponent, whose
// rounding (2^-24 of about 10) is far below the inputs'; fp32 keeps the factor.
template <typename T>
__device__ __forceinline__ float2 exponent(float2 st) {
  return sizeof(T) == 2 ? float2{st.x - __builtin_amdgcn_logf(st.y), 1.f} : st;  // (log2; no key: +inf, P = 0)
}
template <typename T>
__device__ __forceinline__ float probability(float s, float c, float2 st) {
  const float p = __builtin_amdgcn_exp2f(fmaf(s, c, -st.x));
  return sizeof(T) == 2 ? p : p * st.y;
}

// ------------------------------------------------------------------ gradient of the queries
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW > 1 && sizeof(T) * DP <= 320 ? 2 : 1) void k_attend_dq(Args a) {
  __shared__ __attribute__((aligned(16))) T lds[2 * Lds<T, DP>::SIZE];
  T *const lds_k = lds, *const lds_v = lds + Lds<T, DP>::SIZE, *const mine = lds + wave_rows<T, DP>();
  const Unit u = unit_of(a);
  const int lane = int(threadIdx.x & 31), half = int(threadIdx.x >> 5 & 1), wave = int(threadIdx.x >> 6);
  const int64_t r = u.tile * (NW * 32) + wave * 32 + lane;
  const bool valid = r < a.rows;
  const QueryRow qr = query_row(a, u, valid ? r : 0);
  // everything that the row needs, and the first piece, in flight together
  const OwnLoads<T, DP> lq(q_at<T>(a, u, qr), valid, a.dim, half);
  const OwnLoads<T, DP> lg(static_cast<const T*>(a.grad) + packed_q(a, u, qr), valid, a.dim, half);
  const OwnLoads<T, DP> lo(static_cast<const T*>(a.out) + packed_q(a, u, qr), valid, a.dim, half);
  const OwnLoads<T, DP> ll(static_cast<const T*>(sizeof(T) == 2 ? a.low : a.out) + packed_q(a, u, qr), valid, a.dim, half);
  float2 st = valid ? a.stats[stat_at(a, u, qr)] : float2{0.f, 0.f};
  const float c = a.scale * LOG2E;
  Piece<T, DP, NW * 64> pk, pv;
  const bool fast = pk.HELD && a.fast;
  const int begin = int(u.split * a.span), end = int(min(int64_t(u.len), begin + a.span));
  auto fetch = [&](int k0) {
    const int here = min(PIECE, end - k0);
    const uint32_t ks = uint32_t(a.ks[1]) * uint32_t(sizeof(T)), vs = uint32_t(a.vs[1]) * uint32_t(sizeof(T));
    pk.fetch(k_at<T>(a, u, k0), [&](int i) { return uint32_t(i) * ks; }, here, a.dim);
    pv.fetch(v_at<T>(a, u, k0), [&](int i) { return uint32_t(i) * vs; }, here, a.dim);
  };
  if (fast && begin < end) fetch(begin);
  const Own<T, DP> q = lq.own(valid, a.dim, half), g = lg.own(valid, a.dim, half);
  float delta = 0.f;
  {
    // dP - delta is small where one key has most of a row, so delta is summed over the output as it was
    // before its rounding
    const Own<T, DP> o = lo.own(valid, a.dim, half), low = ll.own(valid, a.dim, half);
    constexpr int N = 16 / int(sizeof(T));
#pragma unroll
    for (int k = 0; k < DP / (2 * N); ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float whole = sizeof(T) == 2 ? float(o.v[k][i]) + float(low.v[k][i]) : float(o.v[k][i]);
        delta = fmaf(float(g.v[k][i]), whole, delta);
      }
    delta += __shfl_xor(delta, 32);
  }
  st = exponent<T>(st);
  if (valid && half == 0 && u.split == 0) a.delta[stat_at(a, u, qr)] = delta;
  f32x16 minus_delta;  // where dP starts from, so that P times it is dS
#pragma unroll
  for (int i = 0; i < 16; ++i) minus_delta[i] = -delta;
  f32x16 dq[d_tiles<DP>()] = {};
  for (int k0 = begin; k0 < end; k0 += PIECE) {
    const int here = min(PIECE, end - k0);
    __syncthreads();
    if (fast) {
      pk.commit(lds_k, here, a.dim);
      pv.commit(lds_v, here, a.dim);
    } else {
      Piece<T, DP, NW * 64>::copy(lds_k, [&](int i) { return k_at<T>(a, u, k0 + i); }, here, a.dim);
      Piece<T, DP, NW * 64>::copy(lds_v, [&](int i) { return v_at<T>(a, u, k0 + i); }, here, a.dim);
    }
    __syncthreads();
    if (fast && k0 + PIECE < end) fetch(k0 + PIECE);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const T* kp = lds_k + t * 32 * Lds<T, DP>::STRIDE;
      f32x16 s = rows_product<DP>(kp, q, lane, half);
      const f32x16 dp = rows_product<DP>(lds_v + t * 32 * Lds<T, DP>::STRIDE, g, lane, half, minus_delta);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = probability<T>(s[i], c, st) * dp[i];
      if (here < PIECE) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t * 32 + row_of(i, half) >= here) s[i] = 0.f;
      }
      columns_product<DP>(dq, kp, Tile<T>(s), lane, half);
    }
  }
  __syncthreads();
  if (a.splits > 1) {
    float* part = a.part_o + u.split * (a.batch * a.queries * a.heads * a.dim);
    store_rows<T, DP>(part, packed_q(a, u, qr), valid, mine, dq, a.scale, a.dim, lane, half);
    return;
  }
  store_rows<T, DP>(static_cast<T*>(a.dq), packed_q(a, u, qr), valid, mine, dq, a.scale, a.dim, lane, half);
}

// --------------------------------------------------------- gradients of the keys and values
constexpr int keys_waves(int bytes, bool halves, int NW) { return NW > 1 && bytes <= (halves ? 192 : 256) ? 2 : 1; }
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, keys_waves(sizeof(T) * DP, sizeof(T) == 2, NW)) void k_attend_dkv(Args a) {
  __shared__ __attribute__((aligned(16))) T lds[2 * Lds<T, DP>::SIZE];
  T *const lds_q = lds, *const lds_g = lds + Lds<T, DP>::SIZE, *const mine = lds + wave_rows<T, DP>();
  __shared__ __attribute__((aligned(16))) float lds_top[PIECE], lds_inverse[PIECE], lds_delta[PIECE];
  const Unit u = unit_of(a);
  const int lane = int(threadIdx.x & 31), half = int(threadIdx.x >> 5 & 1), wave = int(threadIdx.x >> 6);
  const int64_t key = u.tile * (NW * 32) + wave * 32 + lane;
  const bool valid = key < u.len;
  const OwnLoads<T, DP> lk(k_at<T>(a, u, valid ? key : 0), valid, a.dim, half);
  const OwnLoads<T, DP> lv(v_at<T>(a, u, valid ? key : 0), valid, a.dim, half);
  const Own<T, DP> k = lk.own(valid, a.dim, half), v = lv.own(valid, a.dim, half);
  f32x16 dk[d_tiles<DP>()] = {}, dv[d_tiles<DP>()] = {};
  const float c = a.scale * LOG2E;
  if (u.tile * (NW * 32) < u.len) {
    Piece<T, DP, NW * 64> pq, pg;
    const bool fast = pq.HELD && a.fast;
    float2 st = {0.f, 0.f};  // the statistics of the row that this thread stages
    float delta = 0.f;
    const T* grad = static_cast<const T*>(a.grad);
    const void* q0 = q_at<T>(a, u, {u.g * a.each, 0});
    const void* g0 = grad + packed_q(a, u, {u.g * a.each, 0});
    const uint32_t size = sizeof(T), qt = uint32_t(a.qs[1]) * size, qh = uint32_t(a.qs[2]) * size,
                   gt = uint32_t(a.heads * a.dim) * size, gh = uint32_t(a.dim) * size;
    auto fetch = [&](int64_t r0) {
      const int here = int(min(int64_t(PIECE), a.rows - r0));
      auto offset = [&](int i, uint32_t token, uint32_t head) {
        const uint32_t r = uint32_t(r0) + uint32_t(i), h = fast_query_head(a, r);
        return (r - h * uint32_t(a.queries)) * token + h * head;
      };
      pq.fetch(q0, [&](int i) { return offset(i, qt, qh); }, here, a.dim);
      pg.fetch(g0, [&](int i) { return offset(i, gt, gh); }, here, a.dim);
    };
    // the statistics of the piece's row that this thread stages, from a row that exists
    auto fetch_stats = [&](int64_t r0) {
      const int64_t at = stat_at(a, u, query_row(a, u, min(r0 + int(threadIdx.x), a.rows - 1)));
      st = a.stats[at];
      delta = a.delta[at];
    };
    const int64_t begin = u.split * a.span, end = min(a.rows, begin + a.span);
    if (begin < end) {
      if (fast) fetch(begin);
      fetch_stats(begin);
    }
    for (int64_t r0 = begin; r0 < end; r0 += PIECE) {
      const int here = int(min(int64_t(PIECE), end - r0));
      __syncthreads();
      if (fast) {
        pq.commit(lds_q, here, a.dim);
        pg.commit(lds_g, here, a.dim);
      } else {
        Piece<T, DP, NW * 64>::copy(lds_q, [&](int i) { return q_at<T>(a, u, query_row(a, u, r0 + i)); }, here, a.dim);
        Piece<T, DP, NW * 64>::copy(
            lds_g, [&](int i) { return grad + packed_q(a, u, query_row(a, u, r0 + i)); }, here, a.dim);
      }
      if (threadIdx.x < PIECE) {
        // (a row past the end: no probability)
        const bool in = int(threadIdx.x) < here;
        const float2 e = exponent<T>(in ? st : float2{0.f, 0.f});
        lds_top[threadIdx.x] = e.x;
        lds_inverse[threadIdx.x] = e.y;
        lds_delta[threadIdx.x] = in ? -delta : 0.f;
      }
      __syncthreads();
      if (r0 + PIECE < end) {
        if (fast) fetch(r0 + PIECE);
        fetch_stats(r0 + PIECE);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const T *qp = lds_q + t * 32 * Lds<T, DP>::STRIDE, *gp = lds_g + t * 32 * Lds<T, DP>::STRIDE;
        f32x16 dp;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const f32x4 d = *reinterpret_cast<const f32x4*>(lds_delta + t * 32 + row_of(i, half));
#pragma unroll
          for (int j = 0; j < 4; ++j) dp[i + j] = d[j];
        }
        f32x16 s = rows_product<DP>(qp, k, lane, half);
        dp = rows_product<DP>(gp, v, lane, half, dp);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int row = t * 32 + row_of(i, half);
          const f32x4 top = *reinterpret_cast<const f32x4*>(lds_top + row);
          f32x4 inverse = {};
          if (sizeof(T) == 4) inverse = *reinterpret_cast<const f32x4*>(lds_inverse + row);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[i + j] = probability<T>(s[i + j], c, {top[j], inverse[j]});
            dp[i + j] *= s[i + j];
          }
        }
        columns_product<DP>(dv, gp, Tile<T>(s), lane, half);
        columns_product<DP>(dk, qp, Tile<T>(dp), lane, half);
      }
    }
  }
  if (!valid) {  // past the length: the sums of this lane's column mean nothing
#pragma unroll
    for (int t = 0; t < d_tiles<DP>(); ++t) dk[t] = dv[t] = f32x16{};
  }
  const bool row = key < a.keys;
  const int64_t at = ((u.b * a.keys + key) * a.shared + u.g) * a.dim;
  __syncthreads();
  if (a.splits > 1) {
    const int64_t all = a.batch * a.keys * a.shared * a.dim;
    store_rows<T, DP>(a.part_o + 2 * u.split * all, at, row, mine, dk, a.scale, a.dim, lane, half);
    store_rows<T, DP>(a.part_o + (2 * u.split + 1) * all, at, row, mine, dv, 1.f, a.dim, lane, half);
    return;
  }
  store_rows<T, DP>(static_cast<T*>(a.dk), at, row, mine, dk, a.scale, a.dim, lane, half);
  store_rows<T, DP>(static_cast<T*>(a.dv), at, row, mine, dv, 1.f, a.dim, lane, half);
}

// Parts of one tensor's gradient (blockIdx.y: of two), added in ascending order: out[i] = sum over s of
// part[s * tensors * n + i].
template <typename T>
__global__ __launch_bounds__(256) void k_attend_sum(const float* __restrict__ part, T* __restrict__ first,
                                                    T* __restrict__ second, int64_t n, int splits) {
  const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4, stride = n * gridDim.y;
  if (i >= n) return;
  const float* from = part + blockIdx.y * n + i;
  T* to = (blockIdx.y ? second : first) + i;
  if (n % 4 == 0) {
    f32x4 sum = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) sum += *reinterpret_cast<const f32x4*>(from + s * stride);
    const float e[4] = {sum[0], sum[1], sum[2], sum[3]};
    store<T, 4>(to, Vec<T, 4>::of(e));
    return;
  }
  for (int j = 0; j < 4 && i + j < n; ++j) {
    float sum = 0.f;
    for (int s = 0; s < splits; ++s) sum += from[s * stride + j];
    to[j] = from_f32<T>(sum);
  }
}

// ---------------------------------------------------------------------------------- host
int check_args(const char* what, const sihc_attention* a) {
  if (!a) return fail(SIHC_ERR_INVALID, "%s: null sizes", what);
  if (!valid_dtype(a->dtype)) return fail(SIHC_ERR_INVALID, "%s: bad dtype %d", what, a->dtype);
  if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->dim <= 0)
    return fail(SIHC_ERR_INVALID, "%s: bad sizes", what);
  if (a->heads % a->kv_heads)
    return fail(SIHC_ERR_INVALID, "%s: %d query heads do not share %d key heads", what, a->heads, a->kv_heads);
  if (a->dim > SIHC_MAX_HEAD_DIM)
    return fail(SIHC_ERR_INVALID, "%s: heads of %d channels (at most %d)", what, a->dim, SIHC_MAX_HEAD_DIM);
  // row lists and tiles are counted in int32; stats and packed offsets in int64
  const int64_t rows = int64_t(a->queries) * (a->heads / a->kv_heads);
  if (rows >= SIHC_MAX_TOKENS || a->keys >= SIHC_MAX_TOKENS ||
      a->batch > (0x7fffffff >> 8) / (rows / 32 + a->keys / 32 + 2) / a->kv_heads)
    return fail(SIHC_ERR_INVALID, "%s: tensor too large", what);
  return SIHC_OK;
}
Args args_of(const sihc_attention* s) {
  Args a{};
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = s->q_stride[i];
    a.ks[i] = s->k_stride[i];
    a.vs[i] = s->v_stride[i];
  }
  a.batch = s->batch;
  a.queries = s->queries;
  a.keys = s->keys;
  a.heads = s->heads;
  a.shared = s->kv_heads;
  a.each = s->heads / s->kv_heads;
  a.dim = s->dim;
  a.rows = int64_t(a.each) * a.queries;
  a.scale = s->scale;
  a.cluster = 1;
  // as long as every XCD takes 16 clusters (64 x 16 heads of 72 channels, 256 rows over up to 256 keys:
  // forward and gradients 237 us by single heads, 224 by 2, 215 by 4, 227 by 8)
  for (int n : {4, 2})
    if (s->kv_heads % n == 0 && s->batch * s->kv_heads / n >= 128) {
      a.cluster = n;
      break;
    }
  a.splits = 1;
  a.span = int64_t(1) << 40;
  // Rows of whole vectors, and offsets within an image's queries, and within a piece of keys, below 2^31.
  const int64_t size = s->dtype == SIHC_DTYPE_F32 ? 4 : 2, most = (int64_t(1) << 31) / size - s->dim;
  auto within = [&](int64_t tokens, int64_t token, int64_t heads, int64_t head) {
    return token >= 0 && head >= 0 && (token == 0 || tokens <= most / token) && (head == 0 || heads <= most / head) &&
           tokens * token + heads * head < most;
  };
  a.fast = s->dim * size % 16 == 0 && within(s->queries, s->q_stride[1], s->heads, s->q_stride[2]) &&
           within(s->queries, int64_t(s->heads) * s->dim, s->heads, s->dim) &&
           within(PIECE, s->k_stride[1], 0, 0) && within(PIECE, s->v_stride[1], 0, 0);
  // r / queries for r < 2^31 (Granlund and Montgomery 1994, as in sihc_kernels.hip): with 2^l the next
  // power of two, magic = ceil(2^(31 + l) / queries) is exact; powers of two are a shift.
  int l = 0;
  while ((int64_t(1) << l) < a.queries) ++l;
  if (a.queries > 0 && (int64_t(1) << l) != a.queries) {
    a.magic = uint32_t(((uint64_t(1) << (31 + l)) + uint64_t(a.queries) - 1) / uint64_t(a.queries));
    a.shift = l - 1;
  } else {
    a.shift = l;
  }
  return a;
}
// Parts of `length` keys or rows for `blocks` blocks of one wave: none where `full` of them fill the card or
// `length` is `alone` at most, otherwise for about `target` blocks, of at least `least`.
struct Parts {
  int count;
  int64_t span;  // a multiple of PIECE
};
Parts parts_of(int64_t length, int64_t blocks, int64_t full, int64_t target, int64_t alone, int64_t least) {
  Parts p{1, ceil_div(std::max<int64_t>(length, 1), PIECE) * PIECE};
  if (blocks <= 0 || blocks >= full || length <= alone) return p;
  const int64_t most = std::min<int64_t>({ceil_div(target, blocks), ceil_div(length, least), int64_t(256)});
  p.span = ceil_div(ceil_div(length, most), PIECE) * PIECE;
  p.count = int(ceil_div(length, p.span));
  return p;
}
int64_t row_count(const sihc_attention* s) { return int64_t(s->queries) * (s->heads / s->kv_heads); }
int64_t row_blocks(const sihc_attention* s) { return s->batch * s->kv_heads * ceil_div(row_count(s), 32); }
// fp32 products take 8 times the time of bf16 ones, so parts of one piece are worth their joining where those
// of bf16 are not (8 heads of 64, one query over 128 keys: 9.2 us in two parts, 8.4 in one).
int64_t alone(const sihc_attention* s) { return s->dtype == SIHC_DTYPE_F32 ? PIECE : 2 * PIECE; }
// Few query rows: the keys in parts, for the forward (one query over 4,096 keys, 4 key heads of 128: batches of
// 8, 32, 64 and 128 take 24, 52, 106 and 203 us in parts for 1024 blocks, 175, 177, 180 and 190 in one) and
// for the gradient of the queries (32 queries over 2,048 keys, 8 heads of 64: all gradients of batches of 1,
// 16, 32, 48 18, 54, 90 and 135 us in parts for 512 blocks, 57, 84, 108 and 141 in one).
Parts forward_parts(const sihc_attention* s) { return parts_of(s->keys, row_blocks(s), 512, 1024, alone(s), PIECE); }
Parts dq_parts(const sihc_attention* s) { return parts_of(s->keys, row_blocks(s), 512, 512, alone(s), PIECE); }
// Few keys and many query rows: the rows in parts, for the gradients of keys and values (4 x 16 heads x
// 4,096 rows over 2,048 keys and 4 key heads, 1024 waves of 32 keys: 463 us in one part, 329 in two,
// 338 in four; 8 x 16 heads of 72, 256 rows over 256 keys: all gradients 42 us in parts of 128 rows, 30 in one).
Parts dkv_parts(const sihc_attention* s) {
  return parts_of(row_count(s), s->batch * s->kv_heads * ceil_div(s->keys, 32), 2048, 2048, 2 * alone(s), 2 * alone(s));
}
int64_t query_rows(const sihc_attention* s) { return s->batch * s->heads * int64_t(s->queries); }
// Calls f(T, DP): the smallest compiled width of a head.
template <typename F>
int by_width(const sihc_attention* s, F&& f) {
  return by_dtype(s->dtype, [&](auto t) {
    if (s->dim <= 32) return f(t, IC<32>{});
    if (s->dim <= 64) return f(t, IC<64>{});
    if (s->dim <= 80) return f(t, IC<80>{});
    if (s->dim <= 96) return f(t, IC<96>{});
    return f(t, IC<128>{});
  });
}
// Calls f(NW) with the waves of a block over `rows` rows of its own side: four share the other side's pieces
// (4 x 16 heads of 72, 256 rows over 256 keys: forward 15.3 us, by blocks of one wave 17.8, gradients 27 and
// 33) unless there is work for one alone (64 x 16 heads of 72, 32 rows: 33 and 22).
template <typename F>
int by_waves(int64_t rows, F&& f) {
  return rows <= 32 ? f(IC<1>{}) : f(IC<4>{});
}

}  // namespace

extern "C" {

size_t sihc_cross_attention_workspace_size(const sihc_attention* s) {
  if (check_args("sihc_cross_attention", s)) return 0;
  const int splits = forward_parts(s).count;
  return splits > 1 ? size_t(splits) * size_t(query_rows(s)) * size_t(s->dim + 2) * 4 : 0;
}

int sihc_cross_attention(const sihc_attention* s, const void* q, const void* k, const void* v, const int32_t* lengths,
                         void* out, float* stats, void* low, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "sihc_cross_attention";
  if (int rc = check_args(what, s)) return rc;
  if (s->batch == 0 || s->queries == 0) return SIHC_OK;
  if (!q || !out || (s->keys && (!k || !v))) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  const size_t need = sihc_cross_attention_workspace_size(s);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SIHC_ERR_INVALID, "%s: workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  if (!aligned(stats, 8) || !aligned(workspace, 16))
    return fail(SIHC_ERR_INVALID, "%s: misaligned workspace or stats", what);
  Args a = args_of(s);
  const int64_t total = query_rows(s);
  const Parts parts = forward_parts(s);
  a.splits = parts.count;
  a.span = parts.span;
  if (a.splits > 1) {
    a.part_s = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(a.part_s + a.splits * total);
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.lengths = lengths;
  a.o = out;
  a.o_low = low;
  a.stats = reinterpret_cast<float2*>(stats);
  return by_width(s, [&](auto t, auto dp) {
    using T = decltype(t);
    return by_waves(a.rows, [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      a.tiles = ceil_div(a.rows, NW * 32);
      hipLaunchKernelGGL((k_attend<T, decltype(dp)::value, NW>),
                         dim3(unsigned(a.tiles * a.batch * a.shared * a.splits)), dim3(NW * 64), 0,
                         static_cast<hipStream_t>(stream), a);
      if (a.splits > 1)
        hipLaunchKernelGGL(k_attend_join<T>, dim3(unsigned(total)), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a, total);
      return check_launch(what);
    });
  });
}

static size_t delta_bytes(const sihc_attention* s) { return size_t(ceil_div(query_rows(s) * 4, 256)) * 256; }

size_t sihc_cross_attention_backward_workspace_size(const sihc_attention* s) {
  if (check_args("sihc_cross_attention_backward", s)) return 0;
  // the two gradients' parts follow one another
  const int q = dq_parts(s).count, kv = dkv_parts(s).count;
  const size_t q_bytes = q > 1 ? size_t(q) * size_t(query_rows(s)) * size_t(s->dim) * 4 : 0;
  const size_t kv_bytes =
      kv > 1 ? size_t(kv) * 2 * size_t(s->batch) * size_t(s->keys) * size_t(s->kv_heads) * size_t(s->dim) * 4 : 0;
  const size_t sums = std::max(q_bytes, kv_bytes);
  return delta_bytes(s) + sums;
}

int sihc_cross_attention_backward(const sihc_attention* s, const void* grad, const void* q, const void* k,
                                  const void* v, const int32_t* lengths, const void* out, const float* stats,
                                  const void* low, void* grad_q, void* grad_k, void* grad_v, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* what = "sihc_cross_attention_backward";
  if (int rc = check_args(what, s)) return rc;
  if (s->batch == 0) return SIHC_OK;
  if (s->queries && (!grad || !q || !out || !stats || !grad_q || (s->dtype == SIHC_DTYPE_BF16 && !low)))
    return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  if (s->keys && (!k || !v || !grad_k || !grad_v)) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  for (const void* in : {grad, q, k, v, out, low})
    for (const void* to : {grad_q, grad_k, grad_v})
      if (in && in == to) return fail(SIHC_ERR_INVALID, "%s: an output is one of the inputs", what);
  const size_t need = sihc_cross_attention_backward_workspace_size(s);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SIHC_ERR_INVALID, "%s: workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  if (!aligned(workspace, 16) || !aligned(stats, 8))
    return fail(SIHC_ERR_INVALID, "%s: misaligned workspace or stats", what);
  Args a = args_of(s);
  a.q = q;
  a.k = k;
  a.v = v;
  a.grad = grad;
  a.out = out;
  a.low = low;
  a.dq = grad_q;
  a.dk = grad_k;
  a.dv = grad_v;
  a.lengths = lengths;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.delta = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_width(s, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    int rc = SIHC_OK;
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes(s));
    auto sum = [&](void* first, void* second, int64_t n) {
      if (a.splits > 1)
        hipLaunchKernelGGL(k_attend_sum<T>, dim3(unsigned(ceil_div(n, 1024)), second ? 2 : 1), dim3(256), 0, st, a.part_o,
                           static_cast<T*>(first), static_cast<T*>(second), n, a.splits);
    };
    if (a.queries) {
      const Parts parts = dq_parts(s);
      a.splits = parts.count;
      a.span = parts.span;
      rc = by_waves(a.rows, [&](auto nw) {
        constexpr int NW = decltype(nw)::value;
        a.tiles = ceil_div(a.rows, NW * 32);
        hipLaunchKernelGGL((k_attend_dq<T, DP, NW>), dim3(unsigned(a.tiles * a.batch * a.shared * a.splits)),
                           dim3(NW * 64), 0, st, a);
        sum(grad_q, nullptr, query_rows(s) * a.dim);
        return check_launch(what);
      });
    }
    if (rc || !a.keys) return rc;
    const Parts parts = dkv_parts(s);
    a.splits = parts.count;
    a.span = parts.span;
    return by_waves(a.keys, [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      a.tiles = ceil_div(a.keys, NW * 32);
      hipLaunchKernelGGL((k_attend_dkv<T, DP, NW>), dim3(unsigned(a.tiles * a.batch * a.shared * a.splits)),
                         dim3(NW * 64), 0, st, a);
      sum(grad_k, grad_v, a.batch * a.keys * a.shared * a.dim);
      return check_launch(what);
    });
  });
}

}  // extern "C"

// Projections with their epilogue, and their gradients.
//
//   h = x W^T + b;  u = h | silu(h) | silu(h_a) h_b (h = [h_a, h_b]);  y = residual + gate u
//   du = gate dy;  dgate = sum over the image's rows of dy u;  dh = du act'(h);  db = sum over rows of dh
//   dx = dh W;  dW = dh^T x
//
// Every product runs on the matrix cores in 32 x 32 tiles (bf16 32x32x16, fp32 32x32x2, fp32 sums).
// A block owns a tile of the result; pieces of both operands, BK of the contraction at a time, pass
// through two buffers in LDS: while one is worked on, the next piece is stored from registers to the
// other one and the loads of the piece after it are under way, so that a piece costs one barrier and a
// load has a whole piece's products to arrive. An operand whose contraction runs across its rows lies in
// LDS as it is in memory, and is read by the transposing load. The result passes through LDS once more,
// a wave's own 32 rows at a time, so that the epilogue has 8 adjacent channels of a row and reads and
// writes whole vectors. With SwiGLU a block's columns alternate between 32 rows of W_a and their 32 of
// W_b, so that both halves of a channel meet in one wave. Which tile, and in how many parts the
// contraction is cut, is what the measured costs of the tiles promise the least time for (make_plan).
// Small products and few rows have a kernel without LDS buffers or parts (small_product).
//
// What bounds it (bf16, one MI355X, long runs). At 8,192 cubed 1,150 to 1,240 TFLOP/s; the library's products take 0.72
// (both operands in rows), 0.82 (dx) and 1.01 (dW) of these times, so that the card's power is not the bound: the tiles' waves are
// not fed without a pause. At 16,384 x 768 to a SwiGLU of 2,048: 120 us without and 135 with what the backward
// needs of h (168 MB more), 760 TFLOP/s, where every tile of 256 x 256 starts and ends within 12 pieces; dx 106
// (970 TFLOP/s), dW 99 and 11 to join its 4 parts, the slopes between them 83 for 369 MB. At 16,384 x 1,152 to 1,152 with gate
// and residual 67 us (650 TFLOP/s; the library's product alone 60): 4.5 tiles of 128 x 128 a CU. Two rows
// of 1,152 to 6,912: 6 us of 16 MB, a launch and two loads' latency.
#include "cond_common.h"

#include <atomic>

namespace {
using namespace sihc_cond;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int V = 8;  // adjacent channels of a thread in every epilogue

// ------------------------------------------------------------------------------- row vectors
// n <= V channels of a row from p as fp32, zeros past them (WHOLE: there are V).
template <bool WHOLE = false, typename T>
__device__ __forceinline__ void get(const T* p, int left, float* o) {
  if (WHOLE || left >= V) {
    load_f32<T, V>(p, o);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < left ? to_f32(p[i]) : 0.f;
  }
}
template <bool WHOLE = false, typename T>
__device__ __forceinline__ void put(T* p, int left, const float* v) {
  constexpr int PIECE = 16 / int(sizeof(T));
  if (WHOLE || left >= V) {
#pragma unroll
    for (int i = 0; i < V; i += PIECE) store(p + i, Vec<T, PIECE>::of(v + i));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) p[i] = from_f32<T>(v[i]);
  }
}
// N elements of a row from p, as far as the row's `left` go, zeros past them.
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

// h as the backward has it. In bf16 with an activation that is 20 bits, the upper 16 where a bf16 would be and
// 4 beside it, those of 8 channels in one word: rounded to 16 bits, h would put the gradients of a SwiGLU 1.75
// times as far from the exact ones as their own rounding does (with 20: 1.42, from the rounding of dh as an
// operand). `low` is [rows, parts of h, words_of(outer)].
__host__ __device__ constexpr int words_of(int outer) { return (outer + V - 1) / V; }
template <typename T, bool WHOLE>
__device__ __forceinline__ void put_kept(void* h, uint32_t* low, int64_t at, int left, const float* v) {
  if (sizeof(T) == 4 || !low) {
    put<WHOLE>(static_cast<T*>(h) + at, left, v);
    return;
  }
  uint16_t high[V];
  uint32_t rest = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // To nearest, ties to even, at most 2^-12 of the value; what would round to infinity, and what is not finite, is cut
    // (an arithmetic NaN has bit 22). Cutting all of them would shift every value towards zero, and so the sums over rows.
    uint32_t bits = __float_as_uint(v[i]);
    if (fabsf(v[i]) < 0x1.fffp127f) bits += 0x7ff + (bits >> 12 & 1);
    high[i] = uint16_t(bits >> 16);
    rest |= (bits >> 12 & 0xfu) << (4 * i);
  }
  uint16_t* to = static_cast<uint16_t*>(h) + at;
  if (WHOLE || left >= V) {
    typedef u32x4 words __attribute__((aligned(2)));
    words w;
    __builtin_memcpy(&w, high, 16);
    *reinterpret_cast<words*>(to) = w;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) to[i] = high[i];
  }
  *low = rest;
}
// A value of h from its upper 16 bits, as a float, and channel i's 4 of the word beside it.
__device__ __forceinline__ float kept(float high, uint32_t rest, int i) {
  const uint32_t nibble = i < 3 ? rest << (12 - 4 * i) : rest >> (4 * i - 12);
  return __uint_as_float(__float_as_uint(high) | (nibble & 0xf000u));
}

// ---------------------------------------------------------------------------------- epilogue
struct Epilogue {
  const void *bias, *gate, *residual;
  void *y, *h;         // the result; h as the backward wants it, or null
  uint32_t* low;       // (put_kept)
  float* part;         // [splits][rows][columns] sums instead of the result, or null
  int64_t gate_stride;
  int rows, outer, act, rows_per_gate;
  uint32_t magic;  // row / rows_per_gate is the high word of row * magic, shifted (magic 0: the row itself)
  int shift;
};
__device__ __forceinline__ int image_of(const Epilogue& e, int row) {
  return e.magic ? int(__umulhi(uint32_t(row), e.magic) >> e.shift) : row;
}
// Off by at most (2 |v| + 8) 2^-24 of its value, nearly all of it for negative v, where the exponential's argument is
// rounded as a multiple of log2(e); 0 below -88.7, where the exponential passes fp32.
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// V channels of a row as they are in memory, on their way while something else is done.
template <typename T>
struct Row {
  static constexpr int N = V * int(sizeof(T)) / 16;
  u32x4 raw[N];
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(const T* p, int left) {
    if (WHOLE || left >= V) {
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = load<T, V / N>(p + i * (V / N)).raw;
    } else {
      T e[V] = {};
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < left) e[i] = p[i];
      __builtin_memcpy(raw, e, sizeof(e));
    }
  }
  __device__ __forceinline__ void to(float* o) const {
    T e[V];
    __builtin_memcpy(e, raw, sizeof(e));
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f32(e[i]);
  }
};
// What the epilogue reads for channels col .. col + V - 1: the bias once, gate and residual for each row.
template <typename T, bool SWIGLU>
struct Bias {
  Row<T> a, b;
  __device__ __forceinline__ Bias(const Epilogue& e, int col) {
    if (!e.bias || col >= e.outer) return;
    a.template fetch<false>(static_cast<const T*>(e.bias) + col, e.outer - col);
    if constexpr (SWIGLU) b.template fetch<false>(static_cast<const T*>(e.bias) + e.outer + col, e.outer - col);
  }
};
template <typename T>
struct Rest {
  Row<T> gate, residual;
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(const Epilogue& e, int row, int col) {
    const int left = e.outer - col;
    if (e.gate)
      gate.template fetch<WHOLE>(static_cast<const T*>(e.gate) + image_of(e, row) * e.gate_stride + col, left);
    if (e.residual)
      residual.template fetch<WHOLE>(static_cast<const T*>(e.residual) + int64_t(row) * e.outer + col, left);
  }
};

// Channels col .. col + V - 1 of row `row` from the products: a of W's first rows, b (SwiGLU) of its second.
template <typename T, bool SWIGLU, bool WHOLE>
__device__ __forceinline__ void finish(const Epilogue& e, const Bias<T, SWIGLU>& bias, const Rest<T>& rest, int row,
                                       int col, float* a, float* b) {
  const int left = e.outer - col;
  float t[V];
  if (e.bias) {
    bias.a.to(t);
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] += t[i];
    if constexpr (SWIGLU) {
      bias.b.to(t);
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] += t[i];
    }
  }
  if (e.h) {
    const int64_t first = int64_t(row) * (SWIGLU ? 2 : 1);
    uint32_t* low = e.low ? e.low + first * words_of(e.outer) + col / V : nullptr;
    put_kept<T, WHOLE>(e.h, low, first * e.outer + col, left, a);
    if constexpr (SWIGLU)
      put_kept<T, WHOLE>(e.h, low ? low + words_of(e.outer) : nullptr, (first + 1) * e.outer + col, left, b);
  }
  if constexpr (SWIGLU) {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = a[i] * sigmoid(a[i]) * b[i];
  } else if (e.act == SIHC_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] *= sigmoid(a[i]);
  }
  if (e.gate) {
    rest.gate.to(t);
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] *= t[i];
  }
  if (e.residual) {
    rest.residual.to(t);
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] += t[i];
  }
  put<WHOLE>(static_cast<T*>(e.y) + int64_t(row) * e.outer + col, left, a);
}

// ---------------------------------------------------------------------------------- products
// c[m, n] = sum over k of a[m, k] b[n, k]; an operand is [rows, contraction], or transposed.
struct Gemm {
  const void *a, *b;
  int64_t lda, ldb;
  int m, n, k;      // (SwiGLU: n is the result's channels, half of b's rows)
  int steps;        // pieces of a part of the contraction
  int tiles_m, tiles_n;
  Epilogue e;
};

template <typename T> struct Matrix;
template <>
struct Matrix<bf16> {
  static constexpr int STEP = 16;  // contraction of one fragment
  using Frag = bf16x8;
  static __device__ __forceinline__ f32x16 multiply(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Matrix<float> {
  static constexpr int STEP = 8;
  using Frag = f32x4;
  static __device__ __forceinline__ f32x16 multiply(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};
__device__ __forceinline__ constexpr int row_of(int i, int half) { return (i / 4) * 8 + half * 4 + i % 4; }

template <typename T, int BM_, int BN_, int BK_, int WAVES_M_, int WAVES_N_, int PER_SIMD_>
struct Config {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, PER_SIMD = PER_SIMD_;
  static constexpr int THREADS = WAVES_M * WAVES_N * 64;
  static constexpr int MT = BM / WAVES_M / 32, NT = BN / WAVES_N / 32;  // a wave's tiles
  static constexpr int PER_CU = PER_SIMD * 256 / THREADS;               // blocks of a CU at a time
};

// ROWS rows of an operand, BK of the contraction: in registers on their way, and in LDS.
template <typename T, int ROWS, int BK, int THREADS, bool TRANSPOSED, bool SWIGLU>
struct Piece {
  static constexpr int N = 16 / int(sizeof(T));
  // padded: 16 rows of 16 bytes, or 4 rows of 64 (transposing loads), fall into different banks
  static constexpr int STRIDE = TRANSPOSED ? ROWS + 64 / int(sizeof(T)) : BK + N;
  static constexpr int SIZE = (TRANSPOSED ? BK : ROWS) * STRIDE;
  // Vectors of a row that adjacent threads take: all of BK, or (transposed) a run of ROWS, one after another.
  static constexpr int RUN = std::max(64, THREADS * N / BK);
  static constexpr int VECS = (TRANSPOSED ? RUN : BK) / N, RUNS = TRANSPOSED ? ROWS / RUN : 1;
  static constexpr int LINES = TRANSPOSED ? BK : ROWS, STEP = THREADS / VECS, COUNT = RUNS * LINES / STEP;
  static_assert(THREADS % VECS == 0 && LINES % STEP == 0 && ROWS % (TRANSPOSED ? RUN : 1) == 0, "every thread has the same vectors");

  const T* base;
  int64_t offset[TRANSPOSED ? 1 : COUNT];
  int64_t ld;
  int line, at;  // the thread's first row in the piece and its place in the row
  int left;      // (transposed) rows of the operand from its place on
  Vec<T, N> v[COUNT];

  __device__ __forceinline__ Piece(const void* p, int64_t ld_, int first, int rows, int outer) : ld(ld_) {
    base = static_cast<const T*>(p);
    line = int(threadIdx.x) / VECS;
    at = (int(threadIdx.x) % VECS) * N;
    if constexpr (TRANSPOSED) {
      left = rows - first - at;
      offset[0] = first + at;
    } else {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        const int r = line + i * STEP;
        int64_t row;
        if constexpr (SWIGLU)
          row = min(first + r / 64 * 32 + r % 32, rows - 1) + int64_t(r / 32 % 2) * outer;
        else
          row = min(first + r, rows - 1);
        offset[i] = row * ld + at;
      }
    }
  }
  // Whether piece k0 of a contraction that ends at k needs no care.
  __device__ __forceinline__ static bool whole(int k0, int k, int first, int rows) {
    return k0 + BK <= k && (!TRANSPOSED || first + ROWS <= rows);
  }
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(int k0, int k) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      if constexpr (TRANSPOSED) {
        const int row = k0 + line + i / RUNS * STEP, run = i % RUNS * RUN;
        const T* p = base + offset[0] + int64_t(row) * ld + run;
        if constexpr (WHOLE)
          v[i] = load<T, N>(p);
        else
          v[i] = row < k && left > run ? load_some<T, N>(p, left - run) : Vec<T, N>::zero();
      } else {
        if constexpr (WHOLE)
          v[i] = load<T, N>(base + offset[i] + k0);
        else
          v[i] = k0 + at < k ? load_some<T, N>(base + offset[i] + k0, k - k0 - at) : Vec<T, N>::zero();
      }
    }
  }
  __device__ __forceinline__ void commit(T* lds) const {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      *reinterpret_cast<u32x4*>(lds + (line + i / RUNS * STEP) * STRIDE + at + i % RUNS * RUN) = v[i].raw;
  }
  // The lane's part of rows `row` .. row + 31 at step s of the piece.
  static __device__ __forceinline__ typename Matrix<T>::Frag fragment(const T* lds, int row, int s) {
    const int lane = int(threadIdx.x) & 63, half = lane >> 5;
    if constexpr (!TRANSPOSED) {
      return *reinterpret_cast<const typename Matrix<T>::Frag*>(lds + (row + (lane & 31)) * STRIDE +
                                                                s * Matrix<T>::STEP + half * (Matrix<T>::STEP / 2));
    } else if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4* LdsPtr;
      const int j = lane & 15;
      const T* p = lds + (s * 16 + half * 8 + j / 4) * STRIDE + row + (lane & 16) + (j % 4) * 4;
      const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)p);
      const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p + 4 * STRIDE));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      f32x4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = lds[(s * 8 + half * 4 + j) * STRIDE + row + (lane & 31)];
      return f;
    }
  }
};

template <typename T, typename C, bool TA, bool TB, bool SWIGLU>
struct Layout {
  using A = Piece<T, C::BM, C::BK, C::THREADS, TA, false>;
  using B = Piece<T, C::BN, C::BK, C::THREADS, TB, SWIGLU>;
  static constexpr int BUFFER = A::SIZE + B::SIZE;  // elements
  static constexpr int STRIP = C::NT * 32 + 8;      // a row of a wave's strip in the epilogue (fp32)
  static constexpr size_t BYTES = std::max(size_t(2) * BUFFER * sizeof(T),
                                           size_t(C::THREADS / 64) * 32 * STRIP * sizeof(float));
};

template <typename T, typename C, bool TA, bool TB, bool SWIGLU>
__global__ __launch_bounds__(C::THREADS, C::PER_SIMD) void gemm_kernel(const Gemm g) {
  using L = Layout<T, C, TA, TB, SWIGLU>;
  using A = typename L::A;
  using B = typename L::B;
  extern __shared__ __align__(16) char lds_bytes[];
  T* lds = reinterpret_cast<T*>(lds_bytes);
  constexpr int COLUMNS = SWIGLU ? C::BN / 2 : C::BN;  // the result's

  // Tiles of one part, 8 rows of tiles at a time: neighbours on an XCD share rows and columns.
  const int tiles = g.tiles_m * g.tiles_n;
  const int block = xcd_block(blockIdx.x, gridDim.x), part = block / tiles, tile = block - part * tiles;
  const int band = tile / (8 * g.tiles_n), in = tile - band * 8 * g.tiles_n;
  const int high = min(8, g.tiles_m - band * 8);
  const int m0 = (band * 8 + in % high) * C::BM, n0 = in / high * COLUMNS;
  const int from = part * g.steps * C::BK, k = min(g.k, from + g.steps * C::BK);

  A a(g.a, g.lda, m0, g.m, 0);
  B b(g.b, g.ldb, n0, g.n, g.n);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WAVES_N * C::MT * 32, wn = wave % C::WAVES_N * C::NT * 32;
  auto fetch = [&](int k0) {
    if (A::whole(k0, k, m0, g.m)) a.template fetch<true>(k0, k);
    else a.template fetch<false>(k0, k);
    if (B::whole(k0, k, n0, g.n)) b.template fetch<true>(k0, k);
    else b.template fetch<false>(k0, k);
  };
  f32x16 acc[C::MT][C::NT] = {};
  fetch(from);
  a.commit(lds);
  b.commit(lds + A::SIZE);
  if (from + C::BK < k) fetch(from + C::BK);
  __syncthreads();
  int buffer = 0;
  for (int k0 = from; k0 < k; k0 += C::BK, buffer ^= 1) {
    T* next = lds + (buffer ^ 1) * L::BUFFER;
    const T *pa = lds + buffer * L::BUFFER, *pb = pa + A::SIZE;
    if (k0 + C::BK < k) {
      a.commit(next);
      b.commit(next + A::SIZE);
      if (k0 + 2 * C::BK < k) fetch(k0 + 2 * C::BK);
    }
#pragma unroll
    for (int s = 0; s < C::BK / Matrix<T>::STEP; ++s) {
      typename Matrix<T>::Frag fa[C::MT], fb[C::NT];
#pragma unroll
      for (int i = 0; i < C::MT; ++i) fa[i] = A::fragment(pa, wm + i * 32, s);
#pragma unroll
      for (int j = 0; j < C::NT; ++j) fb[j] = B::fragment(pb, wn + j * 32, s);
#pragma unroll
      for (int i = 0; i < C::MT; ++i)
#pragma unroll
        for (int j = 0; j < C::NT; ++j) acc[i][j] = Matrix<T>::multiply(fa[i], fb[j], acc[i][j]);
    }
    __syncthreads();
  }

  // a strip of 32 rows at a time through the wave's own LDS
  const int lane = threadIdx.x & 63;
  float* strip = reinterpret_cast<float*>(lds_bytes) + wave * 32 * L::STRIP;
  constexpr int WIDE = SWIGLU ? C::NT * 16 : C::NT * 32;  // the result's channels of a wave
  constexpr int GROUPS = WIDE / V, ROWS = 64 / GROUPS, PASSES = (32 + ROWS - 1) / ROWS;  // (three tiles: 60 lanes)
  const int c = lane % GROUPS * V, col = n0 + (SWIGLU ? wn / 2 : wn) + c;
  const Bias<T, SWIGLU> bias(g.e, col);
  auto leave = [&](auto whole, const Rest<T>& rest, int r, int row) {
    constexpr bool WHOLE = decltype(whole)::value != 0;
    float p[V], q[V];
    const float* from_strip = strip + r * L::STRIP + (SWIGLU ? c / 32 * 64 + c % 32 : c);
#pragma unroll
    for (int x = 0; x < V; ++x) p[x] = from_strip[x];
    if constexpr (SWIGLU)
#pragma unroll
      for (int x = 0; x < V; ++x) q[x] = from_strip[32 + x];
    if (g.e.part) {
      float* to = g.e.part + (int64_t(part) * g.m + row) * (SWIGLU ? 2 : 1) * g.n + col;
      put<WHOLE>(to, g.n - col, p);
      if constexpr (SWIGLU) put<WHOLE>(to + g.n, g.n - col, q);
    } else {
      finish<T, SWIGLU, WHOLE>(g.e, bias, rest, row, col, p, q);
    }
  };
  const bool inside = m0 + C::BM <= g.m && n0 + COLUMNS <= g.n;  // (the block's tile: no test for a row or a channel)
  const int r0 = lane / GROUPS;
  // two strips side by side, so that both have their loads under way; four would be too much code
  constexpr int STRIPS = C::MT <= 2 ? 2 : 1;
#pragma unroll STRIPS
  for (int i = 0; i < C::MT; ++i) {
    const int row0 = m0 + wm + i * 32;
    Rest<T> rest[PASSES];
    if (inside && !g.e.part)
#pragma unroll
      for (int r = 0; r < PASSES; ++r) rest[r].template fetch<true>(g.e, min(row0 + r0 + r * ROWS, g.m - 1), col);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int x = 0; x < C::MT; ++x)
      if (x == i)
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) strip[row_of(r, lane >> 5) * L::STRIP + j * 32 + (lane & 31)] = acc[x][j][r];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (inside) {
#pragma unroll
      for (int r = 0; r < PASSES; ++r)
        if ((32 % ROWS == 0 || r0 + r * ROWS < 32) && (64 % GROUPS == 0 || lane < GROUPS * ROWS))
          leave(IC<1>{}, rest[r], r0 + r * ROWS, row0 + r0 + r * ROWS);
    } else {
#pragma unroll 1
      for (int r = r0; r < 32; r += ROWS) {
        if (row0 + r >= g.m || col >= g.n || lane >= GROUPS * ROWS) break;
        if (!g.e.part) rest[0].template fetch<false>(g.e, row0 + r, col);
        leave(IC<0>{}, rest[0], r, row0 + r);
      }
    }
  }
}

// Small products and few rows: a block owns 32 x 32 of the result (SwiGLU: of both halves; 16 x 32 where there
// are no more rows), its waves a run of the contraction each, in 16 x 16 tiles (bf16 16x16x32, fp32 16x16x4).
// Operands go from memory straight to the matrix cores' registers, 64 adjacent bytes of a row for four lanes;
// (transposed) two adjacent elements a lane, one for each of its tiles. The waves' sums meet in LDS, in
// the waves' order: one launch, and no wait but for the loads of the next piece.
constexpr int SMALL = 32;       // columns of a block, and its rows
constexpr int most_waves(bool swiglu, bool transposed) { return swiglu || transposed ? 8 : 16; }  // (their registers)
template <typename T>
constexpr int SMALL_PIECE = 128 / int(sizeof(T));  // of the contraction, in two steps

// TILES tiles of 16 rows of an operand, a piece of the contraction. Row `lane` of tile t is 16 t + lane,
// or (transposed) 2 lane + t.
template <typename T, bool TRANSPOSED, int TILES>
struct Direct {
  using Frag = typename Matrix<T>::Frag;
  static constexpr int N = 16 / int(sizeof(T)), STEP = 4 * N;
  const T* base;
  int64_t ld;
  int64_t offset[TILES];
  int first;   // the lane's place in a step
  bool whole;  // (transposed) the tiles' rows all exist
  Frag f[2][TILES];
  // rows `row` .. of `rows`, which start at row `shift` of the operand
  __device__ __forceinline__ Direct(const void* p, int64_t ld_, int row, int rows, int64_t shift)
      : base(static_cast<const T*>(p)), ld(ld_) {
    const int lane = int(threadIdx.x) & 15;
    first = (int(threadIdx.x) >> 4 & 3) * N;
    whole = row + 16 * TILES <= rows;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      offset[t] = TRANSPOSED ? shift + min(row + TILES * lane + t, rows - 1)
                             : (shift + min(row + 16 * t + lane, rows - 1)) * ld + first;
  }
  __device__ __forceinline__ void fetch(int k0, int k) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int from = k0 + s * STEP, left = k - from - first;
      T e[TILES][N];
      if constexpr (!TRANSPOSED) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          Vec<T, N> v;
          if (k0 + 2 * STEP <= k) v = load<T, N>(base + offset[t] + from);
          else v = left > 0 ? load_some<T, N>(base + offset[t] + from, left) : Vec<T, N>::zero();
          __builtin_memcpy(e[t], &v.raw, 16);
        }
      } else if (k0 + 2 * STEP <= k && whole) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const Vec<T, TILES> v = load<T, TILES>(base + int64_t(from + first + i) * ld + offset[0]);
          T pair[TILES];
          __builtin_memcpy(pair, &v.raw, sizeof(pair));
#pragma unroll
          for (int t = 0; t < TILES; ++t) e[t][i] = pair[t];
        }
      } else {
        __builtin_memset(e, 0, sizeof(e));
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i < left)
#pragma unroll
            for (int t = 0; t < TILES; ++t) e[t][i] = base[int64_t(from + first + i) * ld + offset[t]];
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) __builtin_memcpy(&f[s][t], e[t], 16);
    }
  }
};
__device__ __forceinline__ f32x4 multiply16(const bf16x8& a, const bf16x8& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 multiply16(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

template <typename T, bool TA, bool TB, bool SWIGLU, int TILES_M>
__device__ __forceinline__ void small_product(const Gemm& g, int block, int blocks, float* lds) {
  constexpr int HALVES = SWIGLU ? 2 : 1, ROWS = 16 * TILES_M, STRIDE = SMALL + 4, TILE = ROWS * STRIDE;
  constexpr int PIECE = SMALL_PIECE<T>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int tile = xcd_block(block, blocks), m0 = tile / g.tiles_n * ROWS, n0 = tile % g.tiles_n * SMALL;
  const int from = min(g.k, wave * g.steps * PIECE), k = min(g.k, from + g.steps * PIECE);
  using A = Direct<T, TA, TILES_M>;
  using B = Direct<T, TB, 2>;
  A a(g.a, g.lda, m0, g.m, 0);
  B b(g.b, g.ldb, n0, g.n, 0), c(g.b, g.ldb, n0, g.n, SWIGLU ? g.n : 0);
  f32x4 acc[HALVES][TILES_M][2] = {};
  if (from < k) {
    a.fetch(from, k);
    b.fetch(from, k);
    if constexpr (SWIGLU) c.fetch(from, k);
    for (int k0 = from; k0 < k; k0 += PIECE) {
      const A now_a = a;
      const B now_b = b, now_c = c;
      if (k0 + PIECE < k) {
        a.fetch(k0 + PIECE, k);
        b.fetch(k0 + PIECE, k);
        if constexpr (SWIGLU) c.fetch(k0 + PIECE, k);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < TILES_M; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            acc[0][i][j] = multiply16(now_a.f[s][i], now_b.f[s][j], acc[0][i][j]);
            if constexpr (SWIGLU) acc[1][i][j] = multiply16(now_a.f[s][i], now_c.f[s][j], acc[1][i][j]);
          }
    }
  }
  // a thread's V channels of a row
  const int r = int(threadIdx.x) / (SMALL / V), cc = int(threadIdx.x) % (SMALL / V) * V, row = m0 + r, col = n0 + cc;
  const bool owns = int(threadIdx.x) < ROWS * SMALL / V && row < g.m && col < g.n;
  Rest<T> rest;
  if (owns) rest.template fetch<false>(g.e, row, col);
  const Bias<T, SWIGLU> bias(g.e, owns ? col : g.n);
#pragma unroll
  for (int h = 0; h < HALVES; ++h)
#pragma unroll
    for (int i = 0; i < TILES_M; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int at = (lane >> 4) * 4 + x;  // of tile i's rows
          lds[(wave * HALVES + h) * TILE + (TA ? TILES_M * at + i : 16 * i + at) * STRIDE +
              (TB ? 2 * (lane & 15) + j : 16 * j + (lane & 15))] = acc[h][i][j][x];
        }
  __syncthreads();
  if (!owns) return;
  float p[V] = {}, q[V] = {};
  for (int w = 0; w < waves; ++w) {
    const float* t = lds + w * HALVES * TILE + r * STRIDE + cc;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] += t[i];
      if constexpr (SWIGLU) q[i] += t[TILE + i];
    }
  }
  finish<T, SWIGLU, false>(g.e, bias, rest, row, col, p, q);
}
template <typename T, bool TA, bool TB, bool SWIGLU, int TILES_M>
__global__ __launch_bounds__(64 * most_waves(SWIGLU, TA || TB)) void small_kernel(const Gemm g) {
  extern __shared__ __align__(16) char lds_bytes[];
  small_product<T, TA, TB, SWIGLU, TILES_M>(g, blockIdx.x, gridDim.x, reinterpret_cast<float*>(lds_bytes));
}

// The result from the parts' sums, in their order.
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(256) void join_kernel(const Epilogue e, int splits) {
  const int groups = (e.outer + V - 1) / V;
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / groups;
  if (row >= e.rows) return;
  const int col = int(i - row * groups) * V, left = e.outer - col;
  const int64_t wide = (SWIGLU ? 2 : 1) * int64_t(e.outer), all = int64_t(e.rows) * wide;
  const float* p = e.part + row * wide + col;
  float a[V] = {}, b[V] = {};
  const Bias<T, SWIGLU> bias(e, col);
  Rest<T> rest;
  rest.template fetch<false>(e, int(row), col);
#pragma unroll 2
  for (int s = 0; s < splits; ++s) {
    float t[V];
    get(p + s * all, left, t);
#pragma unroll
    for (int x = 0; x < V; ++x) a[x] += t[x];
    if constexpr (SWIGLU) {
      get(p + s * all + e.outer, left, t);
#pragma unroll
      for (int x = 0; x < V; ++x) b[x] += t[x];
    }
  }
  finish<T, SWIGLU, false>(e, bias, rest, int(row), col, a, b);
}

// ------------------------------------------------------------------------------ dh and its sums
struct Slopes {
  const void *grad, *h, *gate;
  const uint32_t* low;
  void *dh;            // null where dh is the gradient itself
  void* dgate;         // the gate's gradient, where a chunk's sum is all of it
  float *bias_part, *gate_part;
  int64_t gate_stride;
  int outer, act, rows_per_gate, chunks;  // chunks of an image's rows
  bool gate_of_row;    // every row has a gate of its own: no sums of it, and images matter no more
};
constexpr int CHUNK = 64;  // rows whose sums are one partial row

// A block: 256 channels (32 threads of V) by 8 rows at a time, over one chunk of one image.
// (A row at a time: two a thread, and three waves a SIMD for them, took 98 us instead of 80 for 16,384 rows of
// a SwiGLU of 2,048, 369 MB. An image of few rows leaves row lanes idle and a partial row of every sum: a SwiGLU of 768
// over 16,384 rows takes 29 us with its sums at 64 rows a gate, 46 at 8, 77 at 4, 155 at 2, and 35 at one, which has no sums.)
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(256, 4) void slopes_kernel(const Slopes s) {
  __shared__ float lds[8][32 * V + 4];
  const int across = threadIdx.x & 31, down = threadIdx.x >> 5;
  const int blocks = (s.outer + 32 * V - 1) / (32 * V);
  const unsigned at = unsigned(xcd_block(int(blockIdx.x), int(gridDim.x)));  // a row's blocks on one XCD
  const int chunk = int(at / unsigned(blocks)), col0 = int(at % unsigned(blocks)) * 32 * V, col = col0 + across * V;
  const int image = chunk / s.chunks, first = (chunk - image * s.chunks) * CHUNK;
  const int count = min(CHUNK, s.rows_per_gate - first), left = s.outer - col;
  const int64_t row0 = int64_t(image) * s.rows_per_gate + first;
  const int wide = SWIGLU ? 2 : 1;
  float sums[3][V] = {}, gate[V];
  if (left > 0) {
    if (s.gate && !s.gate_of_row) get(static_cast<const T*>(s.gate) + image * s.gate_stride + col, left, gate);
#pragma unroll 1
    for (int r = down; r < count; r += 8) {
      float g[V], a[V], b[V], gate_grad[V];
      const int64_t row = row0 + r;
      if (s.gate_of_row) get(static_cast<const T*>(s.gate) + row * s.gate_stride + col, left, gate);
      get(static_cast<const T*>(s.grad) + row * s.outer + col, left, g);
      if (s.h) {
        const T* h = static_cast<const T*>(s.h) + row * wide * s.outer + col;
        get(h, left, a);
        if constexpr (SWIGLU) get(h + s.outer, left, b);
        if (sizeof(T) == 2 && s.low) {
          const uint32_t* low = s.low + row * wide * words_of(s.outer) + col / V;
          const uint32_t rest_a = low[0], rest_b = SWIGLU ? low[words_of(s.outer)] : 0;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            a[i] = kept(a[i], rest_a, i);
            if constexpr (SWIGLU) b[i] = kept(b[i], rest_b, i);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float u = a[i], slope = 1.f;
        if (SWIGLU || s.act == SIHC_ACT_SILU) {
          const float sigma = sigmoid(a[i]);
          u = a[i] * sigma;
          slope = sigma * (1.f + a[i] * (1.f - sigma));
        }
        float du = g[i];
        if (s.gate) {
          gate_grad[i] = g[i] * (SWIGLU ? u * b[i] : u);
          sums[2][i] += gate_grad[i];
          du *= gate[i];
        }
        if constexpr (SWIGLU) {
          a[i] = du * b[i] * slope;
          b[i] = du * u;
          sums[1][i] += b[i];
        } else {
          a[i] = du * slope;
        }
        sums[0][i] += a[i];
      }
      if (s.gate_of_row && s.dgate) put(static_cast<T*>(s.dgate) + row * s.outer + col, left, gate_grad);
      if (s.dh) {
        T* dh = static_cast<T*>(s.dh) + row * wide * s.outer + col;
        put(dh, left, a);
        if constexpr (SWIGLU) put(dh + s.outer, left, b);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k == 1 && !SWIGLU) continue;
    float* part = k == 2 ? s.gate_part : s.bias_part;
    const bool whole = k == 2 && s.dgate && !s.gate_of_row;
    if (!part && !whole) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) lds[down][across * V + i] = sums[k][i];
    __syncthreads();
    const int c = col0 + int(threadIdx.x);
    if (c < s.outer) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += lds[i][threadIdx.x];
      if (whole) static_cast<T*>(s.dgate)[int64_t(chunk) * s.outer + c] = from_f32<T>(v);
      else part[k == 2 ? int64_t(chunk) * s.outer + c : (int64_t(chunk) * wide + k) * s.outer + c] = v;
    }
  }
}
// out[r, :] = sum over `parts` rows of part[r * parts + i, :]: 32 columns a block, 8 threads each.
struct Sums {
  const float* part;
  void* out;
  int columns, parts;
  int64_t blocks;
};
// (threads past 256 take no part)
template <typename T>
__device__ __forceinline__ void add_up(const Sums& s, unsigned block, float (*lds)[33]) {
  const int across = threadIdx.x & 31, down = threadIdx.x >> 5;
  const int blocks = (s.columns + 31) / 32;
  const int64_t r = block / unsigned(blocks);
  const int c = int(block % unsigned(blocks)) * 32 + across;
  float v = 0.f;
  if (c < s.columns && down < 8) {
    const float* p = s.part + r * s.parts * s.columns + c;
#pragma unroll 8
    for (int i = down; i < s.parts; i += 8) v += p[int64_t(i) * s.columns];
  }
  if (down < 8) lds[down][across] = v;
  __syncthreads();
  if (down || c >= s.columns) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += lds[i][across];
  static_cast<T*>(s.out)[r * s.columns + c] = from_f32<T>(v);
}
// Two such sums in one launch, the second's blocks after the first's.
template <typename T>
__global__ __launch_bounds__(256) void sums_kernel(const Sums first, const Sums second) {
  __shared__ float lds[8][33];
  const bool other = blockIdx.x >= first.blocks;
  add_up<T>(other ? second : first, other ? blockIdx.x - unsigned(first.blocks) : blockIdx.x, lds);
}
// What follows the slopes of a small backward, in one launch: dx and dW as small products, and both sums.
template <typename T>
__global__ __launch_bounds__(64 * most_waves(false, true)) void small_backward_kernel(const Gemm dx, const Gemm dw,
                                                                                      int dx_blocks, int dw_blocks,
                                                                                      const Sums first,
                                                                                      const Sums second) {
  extern __shared__ __align__(16) char lds_bytes[];
  float* lds = reinterpret_cast<float*>(lds_bytes);
  int block = blockIdx.x;
  if (block < dx_blocks) return small_product<T, false, true, false, 2>(dx, block, dx_blocks, lds);
  block -= dx_blocks;
  if (block < dw_blocks) return small_product<T, true, true, false, 2>(dw, block, dw_blocks, lds);
  block -= dw_blocks;
  const bool other = block >= first.blocks;
  add_up<T>(other ? second : first, unsigned(other ? block - int(first.blocks) : block),
            reinterpret_cast<float(*)[33]>(lds));
}

// ---------------------------------------------------------------------------------- host
constexpr int CUS = 256, MOST_LDS = 160 * 1024;

// The tiles, the largest first, and what they take by measurement, with rows and with transposed operands: the
// time of a piece (of a full CU's, for each block in it; of a block alone on its CU) and of a tile's start and
// end, in microseconds. (fp32 takes the same either way: 4,096 cubed 1.02 ms with rows, dx 1.03, dW 1.05.)
struct Cost {
  double piece, alone, tile;
};
template <typename T, int SIZE> struct Tiles;
template <> struct Tiles<bf16, 0> : Config<bf16, 256, 256, 64, 2, 4, 2> {
  static constexpr Cost COST[2]{{1.75, 1.75, 9.0}, {1.75, 1.75, 8.7}};
};
template <> struct Tiles<bf16, 1> : Config<bf16, 256, 192, 64, 4, 2, 2> {
  static constexpr Cost COST[2]{{1.33, 1.33, 10.0}, {1.3, 1.3, 7.5}};
};
template <> struct Tiles<bf16, 2> : Config<bf16, 256, 128, 64, 4, 2, 2> {
  static constexpr Cost COST[2]{{1.1, 1.1, 4.5}, {1.05, 1.05, 5.2}};
};
template <> struct Tiles<bf16, 3> : Config<bf16, 128, 128, 64, 2, 2, 2> {
  static constexpr Cost COST[2]{{0.62, 0.72, 2.6}, {0.7, 0.8, 3.0}};
};
template <> struct Tiles<bf16, 4> : Config<bf16, 64, 64, 64, 2, 1, 2> {
  static constexpr Cost COST[2]{{0.21, 0.5, 3.5}, {0.28, 0.55, 3.5}};
};
template <> struct Tiles<float, 0> : Config<float, 128, 128, 32, 2, 2, 2> {
  static constexpr Cost COST[2]{{2.1, 2.3, 4.0}, {2.1, 2.3, 4.0}};
};
template <> struct Tiles<float, 1> : Config<float, 64, 64, 32, 2, 1, 2> {
  static constexpr Cost COST[2]{{0.6, 1.6, 4.0}, {0.6, 1.6, 4.0}};
};
template <typename T>
constexpr int SIZES = sizeof(T) == 2 ? 5 : 2;
// Calls f(tile, its number) for every tile that the product can have: SwiGLU wants pairs of a wave's tiles.
template <typename T, bool SWIGLU, int SIZE = 0, typename F>
void each_tile(F&& f) {
  if constexpr (SIZE < SIZES<T>) {
    if constexpr (!SWIGLU || Tiles<T, SIZE>::NT % 2 == 0) f(Tiles<T, SIZE>{}, SIZE);
    each_tile<T, SWIGLU, SIZE + 1>(f);
  }
}

struct Plan {
  int size, splits, steps, tiles_m, tiles_n;  // size -1: small_kernel, whose waves are the splits
  int64_t blocks;
};
constexpr double NOT_LAUNCHED = 1e15;  // of more threads than a launch has: the plan only where there is no other, to be refused
// small_kernel's: a piece where the CU is full, one that a wave waits for, start and end.
constexpr Cost SMALL_COST{0.22, 2.0, 3.2};
// The tile and the parts of the contraction that promise the least time: every CU's blocks one after
// another, and the parts' sums through memory (at 8 TB/s, for they are still in a cache) and a launch.
template <typename T, bool SWIGLU>
Plan make_plan(int64_t m, int64_t n, int64_t k, bool transposed) {
  Plan best{};
  double least = 1e30;
  each_tile<T, SWIGLU>([&](auto tile, int size) {
    using C = decltype(tile);
    const int64_t tm = ceil_div(m, C::BM), tn = ceil_div(n, SWIGLU ? C::BN / 2 : C::BN), pieces = ceil_div(k, C::BK);
    for (int splits = 1; splits <= 32 && splits <= pieces; ++splits) {
      const int64_t steps = ceil_div(pieces, splits), blocks = tm * tn * splits;
      if (ceil_div(pieces, steps) != splits) continue;
      const int64_t each = ceil_div(blocks, CUS), rounds = ceil_div(each, C::PER_CU);
      const Cost cost = C::COST[transposed];
      double us = std::max(double(each) * cost.piece, double(rounds) * cost.alone) * double(steps) +
                  double(rounds) * cost.tile;
      if (splits > 1) us += 5.0 + double(m) * double(n) * (SWIGLU ? 2 : 1) * 4.0 * (splits + 1) / 8e6;
      if (blocks * C::THREADS > MOST_LAUNCHED) us += NOT_LAUNCHED;
      if (us < least) {
        least = us;
        best = Plan{size, splits, int(steps), int(tm), int(tn), blocks};
      }
      if (blocks > 8 * CUS) break;  // (more parts only add to the sums)
    }
  });
  const int64_t tm = ceil_div(m, SMALL), tn = ceil_div(n, SMALL), pieces = ceil_div(k, SMALL_PIECE<T>);
  const int64_t each = ceil_div(tm * tn, CUS);
  for (int waves = 4; waves <= most_waves(SWIGLU, transposed); waves *= 2) {
    if (waves > 4 && pieces <= waves / 2) break;
    const int64_t steps = ceil_div(pieces, waves), rounds = ceil_div(each * waves, 16);
    const double us = std::max(double(each * pieces) * SMALL_COST.piece * (SWIGLU ? 1.5 : 1.0),
                               double(rounds * steps) * SMALL_COST.alone) + SMALL_COST.tile +
                      (tm * tn * 64 * waves > MOST_LAUNCHED ? NOT_LAUNCHED : 0.0);
    if (us < least) {
      least = us;
      best = Plan{-1, waves, int(steps), int(tm), int(tn), tm * tn};
    }
  }
  return best;
}
// A call asks for the same plan several times, and a program for few of them: a thread keeps the last ones.
template <typename T, bool SWIGLU>
Plan plan_of(int64_t m, int64_t n, int64_t k, bool transposed) {
  struct Kept {
    int64_t m = -1, n = 0, k = 0;
    bool transposed = false;
    Plan plan{};
  };
  thread_local Kept kept[64];
  Kept& e = kept[uint64_t((m * 31 + n) * 31 + k * 2 + transposed) * 0x9E3779B97F4A7C15u >> 58];
  if (e.m != m || e.n != n || e.k != k || e.transposed != transposed)
    e = Kept{m, n, k, transposed, make_plan<T, SWIGLU>(m, n, k, transposed)};
  return e.plan;
}
Plan plan_for(int dtype, int64_t m, int64_t n, int64_t k, bool swiglu, bool transposed) {
  if (dtype == SIHC_DTYPE_BF16)
    return swiglu ? plan_of<bf16, true>(m, n, k, transposed) : plan_of<bf16, false>(m, n, k, transposed);
  return swiglu ? plan_of<float, true>(m, n, k, transposed) : plan_of<float, false>(m, n, k, transposed);
}
size_t part_bytes(const Plan& p, int64_t m, int64_t n, bool swiglu) {
  return p.size >= 0 && p.splits > 1 ? size_t(p.splits) * size_t(m) * size_t(n) * (swiglu ? 2 : 1) * sizeof(float) : 0;
}

// More dynamic LDS than a launch may have by itself, once for a kernel on every device.
template <typename K>
int allow(K kernel, size_t bytes, std::atomic<uint64_t>& allowed, const char* what) {
  if (bytes <= 65536) return SIHC_OK;
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) device = 64;
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return SIHC_OK;
  const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, MOST_LDS);
  if (err != hipSuccess) return fail(SIHC_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return SIHC_OK;
}
template <typename T, typename C, bool TA, bool TB, bool SWIGLU>
int start(const Gemm& g, int64_t blocks, hipStream_t stream, const char* what) {
  using L = Layout<T, C, TA, TB, SWIGLU>;
  const auto kernel = &gemm_kernel<T, C, TA, TB, SWIGLU>;
  static_assert(L::BYTES <= MOST_LDS, "a CU's LDS");
  static std::atomic<uint64_t> allowed{0};
  if (blocks * C::THREADS > MOST_LAUNCHED) return fail(SIHC_ERR_INVALID, "%s: too many rows for a launch", what);
  if (const int rc = allow(kernel, L::BYTES, allowed, what)) return rc;
  kernel<<<unsigned(blocks), C::THREADS, L::BYTES, stream>>>(g);
  return check_launch(what);
}
// g.e, g.a, g.b and the sizes given; `part`: the parts' sums.
template <typename T, bool TA, bool TB, bool SWIGLU>
int product(Gemm g, float* part, hipStream_t stream, const char* what) {
  const Plan p = plan_of<T, SWIGLU>(g.m, g.n, g.k, TA || TB);
  g.steps = p.steps;
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.e.part = p.size >= 0 && p.splits > 1 ? part : nullptr;
  g.e.rows = g.m;
  g.e.outer = g.n;
  if (const uint32_t d = uint32_t(g.e.rows_per_gate); d > 1) {  // exact below 2^31
    int log = 0;
    while ((uint64_t(1) << log) < d) ++log;
    g.e.magic = uint32_t((uint64_t(1) << (31 + log)) / d + 1);
    g.e.shift = log - 1;
  }
  if (p.size < 0) {
    if (p.blocks * 64 * p.splits > MOST_LAUNCHED)
      return fail(SIHC_ERR_INVALID, "%s: too many rows for a launch", what);
    auto launch = [&](auto tiles) {
      constexpr int TILES_M = decltype(tiles)::value;
      const size_t lds = size_t(p.splits) * (SWIGLU ? 2 : 1) * 16 * TILES_M * (SMALL + 4) * sizeof(float);
      const auto kernel = &small_kernel<T, TA, TB, SWIGLU, TILES_M>;
      static std::atomic<uint64_t> allowed{0};
      if (const int rc = allow(kernel, lds, allowed, what)) return rc;
      kernel<<<unsigned(p.blocks), unsigned(64 * p.splits), lds, stream>>>(g);
      return check_launch(what);
    };
    return g.m <= 16 ? launch(IC<1>{}) : launch(IC<2>{});
  }
  int rc = SIHC_OK;
  each_tile<T, SWIGLU>([&](auto tile, int size) {
    if (size == p.size) rc = start<T, decltype(tile), TA, TB, SWIGLU>(g, p.blocks, stream, what);
  });
  if (rc || p.splits == 1) return rc;
  const int64_t threads = int64_t(g.m) * ceil_div(g.n, V);
  if (threads > MOST_LAUNCHED) return fail(SIHC_ERR_INVALID, "%s: too many rows for a launch", what);
  join_kernel<T, SWIGLU><<<unsigned(ceil_div(threads, 256)), 256, 0, stream>>>(g.e, p.splits);
  return check_launch(what);
}

int check(const sihc_linear* l, const char* what) {
  if (!l) return fail(SIHC_ERR_INVALID, "%s: null sizes", what);
  if (!valid_dtype(l->dtype)) return fail(SIHC_ERR_INVALID, "%s: bad dtype %d", what, l->dtype);
  if (l->act != SIHC_ACT_NONE && l->act != SIHC_ACT_SILU && l->act != SIHC_ACT_SWIGLU)
    return fail(SIHC_ERR_INVALID, "%s: bad activation %d", what, l->act);
  if (l->rows < 0 || l->rows > (int64_t(1) << 30) || l->inner < 1 || l->outer < 1 || l->inner > (1 << 24) ||
      l->outer > (1 << 24))
    return fail(SIHC_ERR_INVALID, "%s: at most 2^30 rows of 1..2^24 channels", what);
  if (l->rows_per_gate < 1 || l->rows % l->rows_per_gate)
    return fail(SIHC_ERR_INVALID, "%s: %lld rows of %lld a gate", what, (long long)l->rows, (long long)l->rows_per_gate);
  return SIHC_OK;
}
int64_t align(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

// What the backward keeps in its workspace, in this order; sizes in bytes.
struct Space {
  int64_t dh, bias, gate, part;
  int64_t chunks, images;
  int64_t total() const { return dh + bias + gate + part; }
};
Space space_of(const sihc_linear* l, bool gated) {
  Space s{};
  const bool swiglu = l->act == SIHC_ACT_SWIGLU;
  const int64_t wide = (swiglu ? 2 : 1) * int64_t(l->outer), size = l->dtype == SIHC_DTYPE_BF16 ? 2 : 4;
  const int64_t each = gated && l->rows_per_gate > 1 ? l->rows_per_gate : l->rows;
  s.images = l->rows / each;
  s.chunks = ceil_div(each, CHUNK);
  if (l->act != SIHC_ACT_NONE || gated) s.dh = align(l->rows * wide * size);
  s.bias = align(s.images * s.chunks * wide * 4);
  if (gated && l->rows_per_gate > CHUNK) s.gate = align(s.images * s.chunks * l->outer * 4);
  const Plan dx = plan_for(l->dtype, l->rows, l->inner, wide, false, true);
  const Plan dw = plan_for(l->dtype, wide, l->inner, l->rows, false, true);
  s.part = align(int64_t(std::max(part_bytes(dx, l->rows, l->inner, false), part_bytes(dw, wide, l->inner, false))));
  return s;
}
}  // namespace

extern "C" size_t sihc_linear_act_workspace_size(const sihc_linear* l) {
  if (check(l, "linear_act") || l->rows == 0) return 0;
  const bool swiglu = l->act == SIHC_ACT_SWIGLU;
  return part_bytes(plan_for(l->dtype, l->rows, l->outer, l->inner, swiglu, false), l->rows, l->outer, swiglu);
}

extern "C" int sihc_linear_act(const sihc_linear* l, const void* x, const void* weight, const void* bias,
                               const void* gate, const void* residual, void* y, void* h, uint32_t* low,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(l, "linear_act")) return rc;
  if (l->rows == 0) return SIHC_OK;
  if (!x || !weight || !y || (low && !h)) return fail(SIHC_ERR_INVALID, "linear_act: null pointer");
  if (low && (l->dtype != SIHC_DTYPE_BF16 || l->act == SIHC_ACT_NONE))
    return fail(SIHC_ERR_INVALID, "linear_act: more bits of h are for bf16 with an activation");
  for (const void* in : {x, weight, bias, gate})
    if (in && (in == y || in == h)) return fail(SIHC_ERR_INVALID, "linear_act: an output is one of the inputs");
  const size_t need = sihc_linear_act_workspace_size(l);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SIHC_ERR_INVALID, "linear_act: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  Gemm g{};
  g.a = x;
  g.b = weight;
  g.lda = g.ldb = l->inner;
  g.m = int(l->rows);
  g.n = l->outer;
  g.k = l->inner;
  g.e = Epilogue{bias, gate, residual, y, h, low, nullptr, l->gate_stride, 0, 0, l->act, int(l->rows_per_gate), 0, 0};
  return by_dtype(l->dtype, [&](auto t) {
    using T = decltype(t);
    float* part = static_cast<float*>(workspace);
    return l->act == SIHC_ACT_SWIGLU ? product<T, false, false, true>(g, part, hipStream_t(stream), "linear_act")
                                     : product<T, false, false, false>(g, part, hipStream_t(stream), "linear_act");
  });
}

extern "C" size_t sihc_linear_act_backward_workspace_size(const sihc_linear* l, int gated) {
  if (check(l, "linear_act_backward") || l->rows == 0) return 0;
  return size_t(space_of(l, gated != 0).total());
}

extern "C" int sihc_linear_act_backward(const sihc_linear* l, const void* grad, const void* x, const void* weight,
                                        const void* h, const uint32_t* low, const void* gate, void* dx, void* dweight,
                                        void* dbias, void* dgate, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(l, "linear_act_backward")) return rc;
  const bool swiglu = l->act == SIHC_ACT_SWIGLU, gated = gate != nullptr;
  const int wide = (swiglu ? 2 : 1) * l->outer, images = int(l->rows / l->rows_per_gate);
  const hipStream_t on = hipStream_t(stream);
  if (dgate && !gated) return fail(SIHC_ERR_INVALID, "linear_act_backward: no gate, no gradient of it");
  const char* what = "linear_act_backward";
  auto sums_of = [](const float* part, void* out, int64_t rows, int columns, int64_t parts) {
    return Sums{part, out, columns, int(parts), out ? rows * ceil_div(columns, 32) : 0};
  };
  auto sum = [&](const Sums& first, const Sums& second) {
    const int64_t blocks = first.blocks + second.blocks;
    if (blocks * 256 > MOST_LAUNCHED) return fail(SIHC_ERR_INVALID, "%s: too many rows for a launch", what);
    if (blocks == 0) return int(SIHC_OK);
    return by_dtype(l->dtype, [&](auto t) {
      sums_kernel<decltype(t)><<<unsigned(blocks), 256, 0, on>>>(first, second);
      return check_launch(what);
    });
  };
  if (l->rows == 0)  // sums over nothing
    return sum(sums_of(nullptr, dweight, wide, l->inner, 0), sums_of(nullptr, dbias, 1, wide, 0));
  if (!grad || !x || !weight || ((gated || l->act != SIHC_ACT_NONE) && !h) ||
      (l->dtype == SIHC_DTYPE_BF16 && l->act != SIHC_ACT_NONE && !low))
    return fail(SIHC_ERR_INVALID, "linear_act_backward: null pointer");
  for (const void* out : {static_cast<const void*>(dx), static_cast<const void*>(dweight),
                          static_cast<const void*>(dbias), static_cast<const void*>(dgate)})
    for (const void* in : {grad, x, weight, h, gate})
      if (out && out == in) return fail(SIHC_ERR_INVALID, "linear_act_backward: an output is one of the inputs");
  const Space s = space_of(l, gated);
  if (!workspace || workspace_bytes < size_t(s.total()))
    return fail(SIHC_ERR_INVALID, "linear_act_backward: workspace of %zu bytes, %lld needed", workspace_bytes,
                (long long)s.total());
  char* at = static_cast<char*>(workspace);
  void* dh = s.dh ? at : nullptr;
  const bool gate_summed = dgate && s.gate;  // (else a chunk has all of an image)
  float* bias_part = reinterpret_cast<float*>(at + s.dh);
  float* gate_part = reinterpret_cast<float*>(at + s.dh + s.bias);
  float* part = reinterpret_cast<float*>(at + s.dh + s.bias + s.gate);
  return by_dtype(l->dtype, [&](auto t) {
    using T = decltype(t);
    if (dh || dbias) {
      Slopes v{};
      v.grad = grad;
      v.h = dh ? h : nullptr;
      v.gate = gate;
      v.low = l->act == SIHC_ACT_NONE ? nullptr : low;
      v.dh = dh;
      v.dgate = gate_summed ? nullptr : dgate;
      v.bias_part = dbias ? bias_part : nullptr;
      v.gate_part = gate_summed ? gate_part : nullptr;
      v.gate_stride = l->gate_stride;
      v.outer = l->outer;
      v.act = l->act;
      v.gate_of_row = gated && l->rows_per_gate == 1;
      v.rows_per_gate = int(gated && !v.gate_of_row ? l->rows_per_gate : l->rows);
      v.chunks = int(s.chunks);
      const int64_t blocks = s.images * s.chunks * ceil_div(l->outer, 32 * V);
      if (blocks * 256 > MOST_LAUNCHED) return fail(SIHC_ERR_INVALID, "%s: too many rows for a launch", what);
      if (swiglu) slopes_kernel<T, true><<<unsigned(blocks), 256, 0, on>>>(v);
      else slopes_kernel<T, false><<<unsigned(blocks), 256, 0, on>>>(v);
      if (const int rc = check_launch(what)) return rc;
    }
    const void* slopes = dh ? dh : grad;
    const Sums bias_sums = sums_of(bias_part, dbias, 1, wide, s.images * s.chunks);
    const Sums gate_sums = sums_of(gate_part, gate_summed ? dgate : nullptr, images, l->outer, s.chunks);
    auto gradient = [&](const void* b, void* out, int m, int k) {
      Gemm g{};
      g.a = slopes;
      g.b = b;
      g.lda = wide;
      g.ldb = l->inner;
      g.m = m;
      g.n = l->inner;
      g.k = k;
      g.e = Epilogue{nullptr, nullptr, nullptr, out, nullptr, nullptr, nullptr, 0, 0, 0, SIHC_ACT_NONE, 1, 0, 0};
      return g;
    };
    Gemm gx = gradient(weight, dx, int(l->rows), wide), gw = gradient(x, dweight, wide, int(l->rows));
    if (dx && dweight) {
      const Plan px = plan_of<T, false>(gx.m, gx.n, gx.k, true), pw = plan_of<T, false>(gw.m, gw.n, gw.k, true);
      if (px.size < 0 && pw.size < 0) {
        // one launch has one number of waves: a product that wants fewer has more of them, each with less
        const int waves = std::max(px.splits, pw.splits);
        auto place = [&](Gemm& g, const Plan& p) {
          g.steps = int(ceil_div(ceil_div(g.k, SMALL_PIECE<T>), waves));
          g.tiles_m = p.tiles_m;
          g.tiles_n = p.tiles_n;
          g.e.rows = g.m;
          g.e.outer = g.n;
        };
        place(gx, px);
        place(gw, pw);
        const int64_t blocks = px.blocks + pw.blocks + bias_sums.blocks + gate_sums.blocks;
        if (blocks * 64 * waves > MOST_LAUNCHED) return fail(SIHC_ERR_INVALID, "%s: too many rows for a launch", what);
        const size_t lds = size_t(waves) * SMALL * (SMALL + 4) * sizeof(float);
        small_backward_kernel<T><<<unsigned(blocks), unsigned(64 * waves), lds, on>>>(
            gx, gw, int(px.blocks), int(pw.blocks), bias_sums, gate_sums);
        return check_launch(what);
      }
    }
    if (const int rc = sum(bias_sums, gate_sums)) return rc;
    if (dx)
      if (const int rc = product<T, false, true, false>(gx, part, on, what)) return rc;
    if (dweight)
      if (const int rc = product<T, true, true, false>(gw, part, on, what)) return rc;
    return int(SIHC_OK);
  });
}

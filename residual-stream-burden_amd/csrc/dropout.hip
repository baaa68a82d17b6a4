// Dropout whose mask is never stored, with a residual.
//
//   keep_i = word_i >= threshold;  y = residual + (keep ? x scale : 0);  dx = keep ? dy scale : 0
//
// Word i is part i % 4 of the block that the Philox 4x32 generator of 10 rounds (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) gives for the counter (i / 4, stream)
// under the key: a function of the element's place alone, so the backward and a recomputed forward
// have the same mask. The key is read from the device, so a replayed graph follows its tensor.
//
// A round is two products of 32 x 32 bits, quarter-rate instructions: 20 for 4 elements, hidden behind the
// memory that bounds it. 18.9 million bf16 elements: 19 us with a residual (113 MB, 5.9 TB/s), 16.5 without (75 MB).
#include "cond_common.h"

#include <cmath>

namespace {
using namespace sihc_cond;

struct Words { uint32_t w[4]; };
__device__ __forceinline__ Words philox(uint64_t block, uint64_t stream, uint64_t key) {
  uint32_t c0 = uint32_t(block), c1 = uint32_t(block >> 32), c2 = uint32_t(stream), c3 = uint32_t(stream >> 32);
  uint32_t k0 = uint32_t(key), k1 = uint32_t(key >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t a = uint64_t(0xD2511F53u) * c0, b = uint64_t(0xCD9E8D57u) * c2;
    c0 = uint32_t(b >> 32) ^ c1 ^ k0;
    c2 = uint32_t(a >> 32) ^ c3 ^ k1;
    c1 = uint32_t(b);
    c3 = uint32_t(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

constexpr int V = 8;  // elements of a thread: two blocks of the generator

template <typename T, bool RESIDUAL>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* residual, T* y, int64_t count,
                                                      uint32_t threshold, float scale, const uint64_t* key,
                                                      uint64_t stream, int64_t first) {
  const int64_t i = first + (int64_t(blockIdx.x) * 256 + threadIdx.x) * V;
  if (i >= count) return;
  const uint64_t k = *key;
  float v[V], r[V] = {};
  const bool whole = i + V <= count;
  if (whole) {
    load_f32<T, V>(x + i, v);
    if constexpr (RESIDUAL) load_f32<T, V>(residual + i, r);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i + j < count) {
        v[j] = to_f32(x[i + j]);
        if constexpr (RESIDUAL) r[j] = to_f32(residual[i + j]);
      }
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const Words w = philox(uint64_t(i / 4 + half), stream, k);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = half * 4 + j;
      v[e] = (w.w[j] >= threshold ? v[e] * scale : 0.f) + r[e];
    }
  }
  if (whole) {
    constexpr int PIECE = 16 / int(sizeof(T));
#pragma unroll
    for (int j = 0; j < V; j += PIECE) store(y + i + j, Vec<T, PIECE>::of(v + j));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i + j < count) y[i + j] = from_f32<T>(v[j]);
  }
}
}  // namespace

extern "C" int sihc_dropout(const void* x, const void* residual, void* y, int64_t count, double p, const int64_t* key,
                            int64_t stream_id, int dtype, void* stream) {
  if (!valid_dtype(dtype)) return fail(SIHC_ERR_INVALID, "dropout: bad dtype %d", dtype);
  if (!(p >= 0.0 && p < 1.0)) return fail(SIHC_ERR_INVALID, "dropout: p must lie in [0, 1)");
  if (count < 0 || stream_id < 0) return fail(SIHC_ERR_INVALID, "dropout: negative count or stream");
  if (count == 0) return SIHC_OK;
  if (!x || !y || !key) return fail(SIHC_ERR_INVALID, "dropout: null pointer");
  // (rounding up to 2^32 would drop nothing: the largest threshold keeps one value of 2^32)
  const uint32_t threshold = uint32_t(std::min(std::nearbyint(p * 4294967296.0), 4294967295.0));
  const float scale = float(1.0 / (1.0 - p));
  const int64_t most = MOST_LAUNCHED * V;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    for (int64_t first = 0; first < count; first += most) {
      const unsigned blocks = unsigned(ceil_div(std::min(most, count - first), 256 * V));
      const T *from = static_cast<const T*>(x), *add = static_cast<const T*>(residual);
      if (add)
        dropout_kernel<T, true><<<blocks, 256, 0, hipStream_t(stream)>>>(
            from, add, static_cast<T*>(y), count, threshold, scale, reinterpret_cast<const uint64_t*>(key),
            uint64_t(stream_id), first);
      else
        dropout_kernel<T, false><<<blocks, 256, 0, hipStream_t(stream)>>>(
            from, add, static_cast<T*>(y), count, threshold, scale, reinterpret_cast<const uint64_t*>(key),
            uint64_t(stream_id), first);
      if (const int rc = check_launch("dropout")) return rc;
    }
    return int(SIHC_OK);
  });
}

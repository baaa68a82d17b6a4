// Norms of query and key heads with the rotation by the token's positions, and their gradients.
//
//   hat = x r, r = 1 / sqrt(mean x^2 + eps);  n = w hat;  y = R n
//   dn = R^T dy;  dw = sum dn hat;  dx = r (w dn - hat mean(w dn hat))
//
// R turns the pairs (2i, 2i + 1) of each axis' run of channels by position times
// theta^(-2i / width); channels past the runs stay. Without weights there is no norm: y = R x.
//
// A wave owns a few tokens. Its lanes first take the sine and cosine of one pair each, once for
// all heads, into the wave's own part of LDS. Then groups of LPH lanes take a head each, 8 channels
// a lane, so that a head is read once and its statistics are a few moves between lanes.
//
// What bounds it (bf16, one MI355X): memory, with the vector instructions close behind. 16,384 tokens of 32 heads of 72
// take 41 us (151 MB, 3.7 TB/s) forward and 71 backward (226 MB, 3.2 TB/s, two loads of two heads ahead, at the 128
// registers of four waves a SIMD: more loads leave three waves, which took 83 to 109); 32,768 of 20 heads of 128 take 76 (336 MB, 4.4
// TB/s) and 123 (503 MB, 4.1). In fp32 69 and 103, 143 and 231. A head of 72 fills 9 of its 16 lanes. Heads past 128
// channels, 32 lanes each, spill 6 registers (fp32 10) in the backward. Two images of 256 tokens: 8 us, four loads' latency
// in a row.
//
// The angle is a product in 64 bits, in turns, whose whole turns are dropped before it is rounded to
// fp32: a position of 2^31 still has its angle to 2^-24 of a turn.
#include "cond_common.h"

#include <cmath>
#include <cstring>

namespace {
using namespace sihc_cond;

constexpr int V = 8;       // channels of a lane
constexpr int UNROLL = 4;   // heads of a lane whose loads are in flight together
constexpr int BACKWARD = 2;  // (in the backward: two inputs each, and four waves a SIMD)
constexpr int MAX_PAIRS = SIHC_MAX_ROTARY_DIM / 2;
constexpr int MAX_GROUP = 8;  // tokens of a wave

struct Args {
  const void *x[2], *grad[2], *weight[2], *positions;
  void* y[2];
  float* part;         // [blocks][2][dim] sums of the weights' gradients
  int64_t stride[2][3];
  int64_t position_batch;  // positions between two sequences, 0 where all share them
  int heads[2];
  int dim, tokens, total, axes, turned, group;
  bool float_positions, w_f32;
  float eps, sign;
  float share, least;  // 1 / dim; the smallest sum of squares that is taken as it is
  double rate[MAX_PAIRS];  // turns of a pair per position
  uint8_t axis[MAX_PAIRS];
};

template <typename T>
struct Chunk {  // a lane's 8 channels as they are in memory
  static constexpr int N = V * int(sizeof(T)) / 16;
  u32x4 raw[N];
  __device__ __forceinline__ void get(const T* p, int left) {
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = u32x4{};
    if (left >= V) {
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = load<T, V / N>(p + i * (V / N)).raw;
    } else if (left > 0) {
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
  // (past the caches: 75.6 us instead of 81.5 for 168 MB each way)
  __device__ __forceinline__ static void put(T* p, const float* v, int left) {
    typedef u32x4 words __attribute__((aligned(2)));
    if (left >= V) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        __builtin_nontemporal_store(Vec<T, V / N>::of(v + i * (V / N)).raw, reinterpret_cast<words*>(p + i * (V / N)));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < left) p[i] = from_f32<T>(v[i]);
    }
  }
};

// Sum over the LPH lanes of a head, in each of them.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (LPH >= 2) v += moved<0xb1>(v);
  if constexpr (LPH >= 4) v += moved<0x4e>(v);
  if constexpr (LPH >= 8) v += moved<0x141>(v);
  if constexpr (LPH >= 16) v += moved<0x140>(v);
  if constexpr (LPH >= 32) v += __shfl_xor(v, 16);
  return v;
}
template <int LPH>
__device__ __forceinline__ float head_max(float v) {
#pragma unroll
  for (int k = 1; k < LPH; k *= 2) v = fmaxf(v, __shfl_xor(v, k));
  return v;
}

// What a head's values are multiplied by before their squares are summed: 1 where fp32 has the squares.
struct Scale {
  bool any, large, small;  // of the wave's heads; of the lane's
  __device__ __forceinline__ float of() const { return large ? 0x1p-70f : small ? 0x1p100f : 1.f; }
};
// 1 / sqrt(mean x^2 + eps) of a head's scaled values. Where squares leave the range of fp32, all lanes of the wave scale
// their heads by a power of two: 256 values of 2^128 2^-70 have a sum of 2^124, and the least value of all, 2^-149, a
// square of 2^-98. The root and the scale stay two factors, for their product may be too large for fp32 or subnormal.
template <int LPH>
__device__ __forceinline__ float reciprocal_rms(float* x, const Args& a, Scale& scale) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) sum += x[i] * x[i];
  sum = head_sum<LPH>(sum);
  float r = rsqrtf(sum * a.share + a.eps);
  const bool odd = !(sum < 0x1p125f && sum >= a.least);
  scale = Scale{__any(odd) != 0, false, false};
  if (__builtin_expect(scale.any, 0)) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) most = fmaxf(most, fabsf(x[i]));
    most = head_max<LPH>(most);
    scale.large = odd && most >= 1.f;
    scale.small = odd && !(most >= 1.f);
    const float s = scale.of();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] *= s;
      sum += x[i] * x[i];
    }
    sum = head_sum<LPH>(sum);
    if (odd) r = rsqrtf(sum * a.share + a.eps * s * s);
  }
  return r;
}

// A lane's pairs turned by their angles, if not WHOLE (every channel turns) then those of its `turns` first pairs: the
// others stay as they are, for an infinite value times a sine of 0 would be its neighbour's NaN. (WHOLE is the kernels'
// parameter: choosing pair by pair takes 117 us for the training pass of 16,384 tokens of 32 heads of 72 in place of
// 115, a branch on it in the kernels 125.)
template <bool WHOLE>
__device__ __forceinline__ void turn(float* v, const float2* angle, int turns) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float c = angle[i].x, s = angle[i].y, a = v[2 * i], b = v[2 * i + 1];
    const bool turned = WHOLE || i < turns;
    v[2 * i] = turned ? a * c - b * s : a;
    v[2 * i + 1] = turned ? a * s + b * c : b;
  }
}

// Pair p of a token's angles: its cosine and sine, 1 and 0 where nothing turns (a norm's weights are multiplied by them).
__device__ __forceinline__ float2 angle_of(const Args& a, int64_t at, double rate, int axis, bool turns) {
  if (!turns) return make_float2(1.f, 0.f);
  const double position = a.float_positions ? double(static_cast<const float*>(a.positions)[at + axis])
                                            : double(static_cast<const int32_t*>(a.positions)[at + axis]);
  const double turned = position * rate;
  float s, c;
  sincospif(float(2.0 * (turned - rint(turned))), &s, &c);
  return make_float2(c, s * a.sign);
}

// What a lane keeps over the tokens of its wave.
struct Lane {
  int first, left;      // its channels of a head: the first, how many there are from it on
  int turns;            // how many pairs turn from its first on (fewer than one: none)
  int sub;              // its head among those of a pass
  float2* angles;       // the wave's angles in LDS: [group][pairs]
  int pairs;
  double rate[2];
  int axis[2];
};
template <int LPH>
__device__ __forceinline__ Lane lane_of(const Args& a, float2* lds) {
  Lane l;
  const int lane = threadIdx.x & 63;
  l.sub = lane / LPH;
  l.first = (lane % LPH) * V;
  l.left = a.dim - l.first;
  l.turns = a.turned - l.first / 2;
  l.pairs = LPH * V / 2;  // (whole chunks: those past dim have no turn)
  l.angles = lds + (threadIdx.x >> 6) * a.group * l.pairs;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int p = min(lane % (LPH * V / 2) + 64 * k, MAX_PAIRS - 1);
    l.rate[k] = a.rate[p];
    l.axis[k] = a.axis[p];
  }
  return l;
}
// Tokens first .. first + count - 1: their angles into LDS, as many tokens at a time as fill the wave.
template <int LPH>
__device__ __forceinline__ void take_angles(const Args& a, const Lane& l, int first, int count) {
  constexpr int PAIRS = LPH * V / 2, AT_ONCE = PAIRS < 64 ? 64 / PAIRS : 1;
  const int lane = threadIdx.x & 63;
  for (int t0 = 0; t0 < count; t0 += AT_ONCE) {
    const int t = t0 + lane / (PAIRS < 64 ? PAIRS : 64);
    if (t >= count) break;
    const int token = first + t, b = token / a.tokens, n = token - b * a.tokens;
    const int64_t at = (int64_t(b) * a.position_batch + n) * a.axes;
#pragma unroll
    for (int k = 0; k < (PAIRS + 63) / 64; ++k) {
      const int p = lane % (PAIRS < 64 ? PAIRS : 64) + 64 * k;
      l.angles[t * PAIRS + p] = angle_of(a, at, l.rate[k], l.axis[k], p < a.turned);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wave's own LDS traffic is in order
}

template <typename T>
__device__ __forceinline__ const T* head_at(const Args& a, const void* x, int side, int token, int head) {
  const int b = token / a.tokens, n = token - b * a.tokens;
  return static_cast<const T*>(x) + int64_t(b) * a.stride[side][0] + int64_t(n) * a.stride[side][1] +
         int64_t(head) * a.stride[side][2];
}
__device__ __forceinline__ int64_t packed_at(const Args& a, int side, int token, int head) {
  return (int64_t(token) * a.heads[side] + head) * a.dim;
}
__device__ __forceinline__ void weights_of(const Args& a, int side, const Lane& l, bool f32, bool bf, float* w) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = l.first + i;
    w[i] = c >= a.dim ? 0.f
           : f32      ? static_cast<const float*>(a.weight[side])[c]
                      : to_f32(static_cast<const bf16*>(a.weight[side])[c]);
  }
}
// A wave's work is its tokens' heads, the queries' and then the keys', COUNT * 64 / LPH of them a batch: one
// a pass for each group of LPH lanes. fetch(side, base) loads a batch, work(side, base) computes and
// stores it; the next batch's loads leave before a batch is worked on.
template <int LPH, bool ONE, int COUNT, typename Fetch, typename Keep, typename Work>
__device__ __forceinline__ void each_batch(const Args& a, int count, Fetch fetch, Keep keep, Work work) {
  constexpr int STEP = COUNT * (64 / LPH);
  int side = 0, base = 0;
  while (true) {
    keep();
    const int now = side, from = base, items = a.heads[side] * (ONE ? 1 : count);
    base += STEP;
    if (base >= items) {
      ++side;
      base = 0;
    }
    const bool more = side < 2 && a.heads[side] > 0;
    if (more) fetch(side, base);
    work(now, from);
    if (!more) break;
  }
}
// Item `item` of a side's heads: its token of the group and its head.
struct Item {
  int t, token, head;
  bool valid;
};
template <bool ONE>
__device__ __forceinline__ Item item_of(const Args& a, int side, int first, int count, int item) {
  const int heads = a.heads[side];
  Item i;
  i.t = ONE ? 0 : min(item / heads, count - 1);  // (past the end: a lane that takes part in the sums alone)
  i.token = first + i.t;
  i.head = item - i.t * heads;
  i.valid = item < heads * (ONE ? 1 : count);
  return i;
}

template <typename T, int LPH, bool NORM, bool ONE, bool WHOLE>
__global__ __launch_bounds__(256) void heads_kernel(const Args a) {
  constexpr int SUB = 64 / LPH;
  extern __shared__ float2 lds[];
  const Lane l = lane_of<LPH>(a, lds);
  const int waves = blockDim.x >> 6;
  const int wave = xcd_block(blockIdx.x, gridDim.x) * waves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = wave * a.group;
  if (first >= a.total) return;
  const int count = min(a.group, a.total - first);
  Chunk<T> next[UNROLL], in[UNROLL];
  auto fetch = [&](int side, int base) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const Item i = item_of<ONE>(a, side, first, count, base + u * SUB + l.sub);
      next[u].get(head_at<T>(a, a.x[side], side, i.token, i.head) + l.first, i.valid ? l.left : 0);
    }
  };
  fetch(0, 0);
  take_angles<LPH>(a, l, first, count);
  float w[V];
  // One token: its angles stay in registers, and the weights in them: n_0 c - n_1 s = x_0 (w_0 c) - x_1 (w_1 s).
  float2 angle[V / 2];
  float first_of[V], second_of[V];
  auto take_weights = [&](int side) {
    if constexpr (NORM) weights_of(a, side, l, a.w_f32, !a.w_f32, w);
    if constexpr (ONE) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        angle[i] = l.angles[l.first / 2 + i];
        if constexpr (NORM) {
          first_of[2 * i] = w[2 * i] * angle[i].x;
          first_of[2 * i + 1] = w[2 * i] * angle[i].y;
          second_of[2 * i] = -w[2 * i + 1] * angle[i].y;
          second_of[2 * i + 1] = w[2 * i + 1] * angle[i].x;
        }
      }
    }
  };
  auto keep = [&] {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) in[u] = next[u];
  };
  each_batch<LPH, ONE, UNROLL>(a, count, fetch, keep, [&](int side, int base) {
    if (base == 0) take_weights(side);
    const int items = a.heads[side] * (ONE ? 1 : count);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (base + u * SUB >= items) break;
      const Item item = item_of<ONE>(a, side, first, count, base + u * SUB + l.sub);
      float v[V];
      in[u].to(v);
      if constexpr (NORM && ONE) {
        Scale scale;
        const float r = reciprocal_rms<LPH>(v, a, scale);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float x = v[i] * r, y = v[i + 1] * r;
          const bool turned = WHOLE || i / 2 < l.turns;
          v[i] = turned ? x * first_of[i] + y * second_of[i] : x * first_of[i];
          v[i + 1] = turned ? x * first_of[i + 1] + y * second_of[i + 1] : y * second_of[i + 1];
        }
      } else {
        if constexpr (NORM) {
          Scale scale;
          const float r = reciprocal_rms<LPH>(v, a, scale);
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] *= r * w[i];
        }
        if constexpr (!ONE) {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) angle[i] = l.angles[item.t * l.pairs + l.first / 2 + i];
        }
        turn<WHOLE>(v, angle, l.turns);
      }
      if (item.valid)
        Chunk<T>::put(static_cast<T*>(a.y[side]) + packed_at(a, side, item.token, item.head) + l.first, v, l.left);
    }
  });
}

template <typename T, int LPH, bool ONE, bool WHOLE>
__global__ __launch_bounds__(256, 4) void heads_backward_kernel(const Args a) {
  constexpr int SUB = 64 / LPH;
  extern __shared__ float2 lds[];
  const Lane l = lane_of<LPH>(a, lds);
  const int waves = blockDim.x >> 6, groups = (a.total + a.group - 1) / a.group;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float dw[2][V] = {};
  // every wave takes a run of groups of tokens
  const int all = gridDim.x * waves, id = xcd_block(blockIdx.x, gridDim.x) * waves + wave;
  const int64_t from = int64_t(groups) * id / all, to = int64_t(groups) * (id + 1) / all;
  for (int group = int(from); group < int(to); ++group) {
    const int first = group * a.group, count = min(a.group, a.total - first);
    take_angles<LPH>(a, l, first, count);
    float2 angle[V / 2];
    if constexpr (ONE) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) angle[i] = l.angles[l.first / 2 + i];
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      if (a.heads[side] == 0) continue;
      float w[V];
      weights_of(a, side, l, a.w_f32, !a.w_f32, w);
      const int items = a.heads[side] * (ONE ? 1 : count);
      for (int base = 0; base < items; base += BACKWARD * SUB) {
        Chunk<T> in[BACKWARD], grad[BACKWARD];
#pragma unroll
        for (int u = 0; u < BACKWARD; ++u) {
          const Item i = item_of<ONE>(a, side, first, count, base + u * SUB + l.sub);
          const int left = i.valid ? l.left : 0;
          in[u].get(head_at<T>(a, a.x[side], side, i.token, i.head) + l.first, left);
          grad[u].get(static_cast<const T*>(a.grad[side]) + packed_at(a, side, i.token, i.head) + l.first, left);
        }
#pragma unroll
        for (int u = 0; u < BACKWARD; ++u) {
          if (base + u * SUB >= items) break;
          const Item item = item_of<ONE>(a, side, first, count, base + u * SUB + l.sub);
          float x[V], g[V];
          in[u].to(x);
          grad[u].to(g);
          if constexpr (!ONE) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) angle[i] = l.angles[item.t * l.pairs + l.first / 2 + i];
          }
          turn<WHOLE>(g, angle, l.turns);  // (the angles are taken backwards)
          Scale scale;
          const float rms = reciprocal_rms<LPH>(x, a, scale), r = item.valid ? rms : 0.f;  // (0 / 0 without eps)
          float dot = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            x[i] *= r;
            const float t = g[i] * x[i];
            dw[side][i] += t;
            dot += w[i] * t;
          }
          dot = head_sum<LPH>(dot) * a.share;
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] = r * (w[i] * g[i] - x[i] * dot);
          if (__builtin_expect(scale.any, 0)) {
            const float s = scale.of();
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] *= s;
          }
          if (item.valid)
            Chunk<T>::put(static_cast<T*>(a.y[side]) + packed_at(a, side, item.token, item.head) + l.first, g, l.left);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // the block's sums: over a wave's heads by moves, over its waves in LDS
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);  // [waves][2][LPH * V]
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = dw[side][i];
#pragma unroll
      for (int k = LPH; k < 64; k *= 2) v += __shfl_xor(v, k);
      if (l.sub == 0) sums[(wave * 2 + side) * LPH * V + l.first + i] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += blockDim.x) {
    const int side = i / a.dim, c = i - side * a.dim;
    float v = 0.f;
    for (int k = 0; k < waves; ++k) v += sums[(k * 2 + side) * LPH * V + c];
    a.part[int64_t(blockIdx.x) * 2 * a.dim + i] = v;
  }
}

// The weights' gradients from the blocks' sums: 8 columns a block, 32 threads each.
template <typename W>
__global__ __launch_bounds__(256) void weights_kernel(const float* part, W* dq, W* dk, int dim, int parts) {
  __shared__ float lds[32][9];
  const int c = threadIdx.x & 7, row = threadIdx.x >> 3, column = blockIdx.x * 8 + c;
  float v = 0.f;
  if (column < 2 * dim)
#pragma unroll 8
    for (int i = row; i < parts; i += 32) v += part[int64_t(i) * 2 * dim + column];
  lds[row][c] = v;
  __syncthreads();
  if (threadIdx.x >= 8 || column >= 2 * dim) return;
  v = 0.f;
  for (int i = 0; i < 32; ++i) v += lds[i][c];
  W* to = column < dim ? dq : dk;
  if (to) to[column < dim ? column : column - dim] = from_f32<W>(v);
}

// ---------------------------------------------------------------------------------- host
constexpr int BACKWARD_BLOCKS = 1024;  // four of four waves on every CU

int lanes_of(int dim) {
  int lanes = 1;
  while (lanes * V < dim) lanes *= 2;
  return lanes;
}
int check(const sihc_heads* h, const void* k, const void* q_weight, const void* k_weight, const char* what) {
  if (!h) return fail(SIHC_ERR_INVALID, "%s: null sizes", what);
  if (!valid_dtype(h->dtype) || !valid_dtype(h->w_dtype)) return fail(SIHC_ERR_INVALID, "%s: bad dtype", what);
  if (h->w_dtype != h->dtype && h->w_dtype != SIHC_DTYPE_F32)
    return fail(SIHC_ERR_INVALID, "%s: weights of the heads' type or fp32", what);
  if (h->position_dtype != SIHC_POSITION_I32 && h->position_dtype != SIHC_POSITION_F32)
    return fail(SIHC_ERR_INVALID, "%s: positions are int32 or fp32", what);
  if (h->batch < 0 || h->tokens < 0 || h->heads < 1 || h->kv_heads < 0)
    return fail(SIHC_ERR_INVALID, "%s: bad sizes", what);
  if (h->dim < 1 || h->dim > SIHC_MAX_ROTARY_DIM)
    return fail(SIHC_ERR_INVALID, "%s: heads of 1..%d channels", what, SIHC_MAX_ROTARY_DIM);
  if (h->heads > (1 << 20) || h->kv_heads > (1 << 20)) return fail(SIHC_ERR_INVALID, "%s: too many heads", what);
  if (h->tokens > INT32_MAX - 64 || (h->tokens && h->batch > (INT32_MAX - 64) / h->tokens))
    return fail(SIHC_ERR_INVALID, "%s: at most 2^31 - 64 tokens", what);
  if (h->axes < 0 || h->axes > SIHC_MAX_AXES) return fail(SIHC_ERR_INVALID, "%s: 0..%d axes", what, SIHC_MAX_AXES);
  int sum = 0;
  for (int i = 0; i < h->axes; ++i) {
    if (h->widths[i] < 0 || h->widths[i] > h->dim || h->widths[i] % 2)
      return fail(SIHC_ERR_INVALID, "%s: axis %d turns %d channels of %d", what, i, h->widths[i], h->dim);
    sum += h->widths[i];
  }
  if (sum > h->dim) return fail(SIHC_ERR_INVALID, "%s: the axes turn %d channels of %d", what, sum, h->dim);
  if (!(h->theta > 0.0) || !std::isfinite(h->theta)) return fail(SIHC_ERR_INVALID, "%s: theta must be positive", what);
  if (!(h->eps >= 0.f)) return fail(SIHC_ERR_INVALID, "%s: eps must not be negative", what);
  if ((h->kv_heads != 0) != (k != nullptr)) return fail(SIHC_ERR_INVALID, "%s: keys go with kv_heads", what);
  if (k ? (q_weight == nullptr) != (k_weight == nullptr) : k_weight != nullptr)
    return fail(SIHC_ERR_INVALID, "%s: weights of both sides or of none", what);
  return SIHC_OK;
}
Args args_of(const sihc_heads* h) {
  Args a{};
  const int64_t* strides[2] = {h->q_stride, h->k_stride};
  for (int s = 0; s < 2; ++s)
    for (int i = 0; i < 3; ++i) a.stride[s][i] = strides[s][i];
  a.position_batch = h->position_batch_stride;
  a.heads[0] = h->heads;
  a.heads[1] = h->kv_heads;
  a.dim = h->dim;
  a.tokens = int(h->tokens);
  a.total = int(h->batch * h->tokens);
  a.axes = h->axes;
  a.float_positions = h->position_dtype == SIHC_POSITION_F32;
  a.w_f32 = h->w_dtype == SIHC_DTYPE_F32;
  a.eps = h->eps;
  a.sign = h->inverse ? -1.f : 1.f;
  a.share = 1.f / float(h->dim);
  a.least = h->eps < 0x1p-90f ? 0x1p-90f : 0.f;  // (a larger eps hides what smaller squares lose)
  for (int i = 0; i < h->axes; ++i) a.turned += h->widths[i] / 2;
  // Tokens of a wave: one where a token's heads fill 4 passes, else as many as do.
  const int sub = 64 / lanes_of(h->dim), heads = h->heads + h->kv_heads;
  a.group = std::max(1, std::min(MAX_GROUP, 4 * sub / heads));
  return a;
}
void take_rates(const sihc_heads* h, Args& a) {
  // (a program has few of them: a thread keeps the last)
  struct Kept {
    double theta = 0.0;
    int axes = -1, widths[SIHC_MAX_AXES] = {};
    double rate[MAX_PAIRS] = {};
    uint8_t axis[MAX_PAIRS] = {};
  };
  thread_local Kept kept;
  if (kept.theta != h->theta || kept.axes != h->axes || std::memcmp(kept.widths, h->widths, sizeof(kept.widths))) {
    const double log = std::log2(h->theta);
    int pair = 0;
    for (int i = 0; i < h->axes; ++i)
      for (int c = 0; c < h->widths[i]; c += 2, ++pair) {
        kept.rate[pair] = std::exp2(-double(c) / double(h->widths[i]) * log) / 6.283185307179586476925;
        kept.axis[pair] = uint8_t(i);
      }
    kept.theta = h->theta;
    kept.axes = h->axes;
    std::memcpy(kept.widths, h->widths, sizeof(kept.widths));
  }
  std::memcpy(a.rate, kept.rate, sizeof(a.rate));
  std::memcpy(a.axis, kept.axis, sizeof(a.axis));
}
template <typename F>
int by_lanes(int lanes, F&& f) {
  switch (lanes) {
    case 1: return f(IC<1>{});
    case 2: return f(IC<2>{});
    case 4: return f(IC<4>{});
    case 8: return f(IC<8>{});
    case 16: return f(IC<16>{});
    default: return f(IC<32>{});
  }
}
// Calls f with a constant for every truth value.
template <typename F>
void choose(F&& f) { f(); }
template <typename F, typename... Rest>
void choose(F&& f, bool first, Rest... rest) {
  if (first) choose([&](auto... others) { f(std::true_type{}, others...); }, rest...);
  else choose([&](auto... others) { f(std::false_type{}, others...); }, rest...);
}
int64_t backward_blocks(const Args& a) {
  return std::min<int64_t>(BACKWARD_BLOCKS, ceil_div(ceil_div(a.total, a.group), 4));
}
}  // namespace

extern "C" int sihc_qk_norm_rotary(const sihc_heads* h, const void* q, const void* k, const void* q_weight,
                                   const void* k_weight, const void* positions, void* q_out, void* k_out,
                                   void* stream) {
  if (const int rc = check(h, k, q_weight, k_weight, "qk_norm_rotary")) return rc;
  Args a = args_of(h);
  if (a.total == 0) return SIHC_OK;
  take_rates(h, a);
  if (!q || !q_out || (k && !k_out) || (a.turned && !positions))
    return fail(SIHC_ERR_INVALID, "qk_norm_rotary: null pointer");
  for (const void* in : {q, k, q_weight, k_weight, positions})
    if (in && (in == q_out || in == k_out))
      return fail(SIHC_ERR_INVALID, "qk_norm_rotary: an output is one of the inputs");
  a.x[0] = q;
  a.x[1] = k;
  a.weight[0] = q_weight;
  a.weight[1] = k_weight;
  a.positions = positions;
  a.y[0] = q_out;
  a.y[1] = k_out;
  const int64_t groups = ceil_div(a.total, a.group);
  const int waves = groups >= 2048 ? 4 : 1;  // few tokens: a wave a block, over more CUs
  if (ceil_div(groups, waves) * waves * 64 > MOST_LAUNCHED)
    return fail(SIHC_ERR_INVALID, "qk_norm_rotary: too many tokens for a launch");
  return by_dtype(h->dtype, [&](auto t) {
    using T = decltype(t);
    return by_lanes(lanes_of(h->dim), [&](auto lanes) {
      constexpr int LPH = decltype(lanes)::value;
      const size_t lds = size_t(waves) * a.group * (LPH * V / 2) * sizeof(float2);
      const dim3 grid{unsigned(ceil_div(groups, waves))}, block{unsigned(waves * 64)};
      choose([&](auto norm, auto one, auto whole) {
        heads_kernel<T, LPH, decltype(norm)::value, decltype(one)::value, decltype(whole)::value>
            <<<grid, block, lds, hipStream_t(stream)>>>(a);
      }, q_weight != nullptr, a.group == 1, 2 * a.turned == a.dim);
      return check_launch("qk_norm_rotary");
    });
  });
}

extern "C" size_t sihc_qk_norm_rotary_backward_workspace_size(const sihc_heads* h) {
  if (!h || check(h, h->kv_heads ? h : nullptr, nullptr, nullptr, "qk_norm_rotary_backward")) return 0;
  const Args a = args_of(h);
  return size_t(backward_blocks(a)) * 2 * size_t(a.dim) * sizeof(float);
}

extern "C" int sihc_qk_norm_rotary_backward(const sihc_heads* h, const void* grad_q, const void* grad_k,
                                            const void* q, const void* k, const void* q_weight,
                                            const void* k_weight, const void* positions, void* dq, void* dk,
                                            void* dq_weight, void* dk_weight, void* workspace,
                                            size_t workspace_bytes, void* stream) {
  if (const int rc = check(h, k, q_weight, k_weight, "qk_norm_rotary_backward")) return rc;
  Args a = args_of(h);
  take_rates(h, a);
  a.sign = -a.sign;
  if (!q_weight || !dq_weight || (k && !dk_weight))
    return fail(SIHC_ERR_INVALID, "qk_norm_rotary_backward: the weights and their gradients are needed");
  if (a.total && (!q || !grad_q || !dq || (k && (!grad_k || !dk)) || (a.turned && !positions) || !workspace))
    return fail(SIHC_ERR_INVALID, "qk_norm_rotary_backward: null pointer");
  for (const void* in : {grad_q, grad_k, q, k, q_weight, k_weight, positions})
    if (in && (in == dq || in == dk || in == dq_weight || in == dk_weight))
      return fail(SIHC_ERR_INVALID, "qk_norm_rotary_backward: an output is one of the inputs");
  const int64_t blocks = backward_blocks(a);
  if (workspace_bytes < size_t(blocks) * 2 * size_t(a.dim) * sizeof(float))
    return fail(SIHC_ERR_INVALID, "qk_norm_rotary_backward: workspace of %zu bytes is too small", workspace_bytes);
  a.x[0] = q;
  a.x[1] = k;
  a.grad[0] = grad_q;
  a.grad[1] = grad_k;
  a.weight[0] = q_weight;
  a.weight[1] = k_weight;
  a.positions = positions;
  a.y[0] = dq;
  a.y[1] = dk;
  a.part = static_cast<float*>(workspace);
  if (a.total) {
    const int rc = by_dtype(h->dtype, [&](auto t) {
      using T = decltype(t);
      return by_lanes(lanes_of(h->dim), [&](auto lanes) {
        constexpr int LPH = decltype(lanes)::value;
        const size_t lds = 4 * std::max(size_t(a.group) * (LPH * V / 2) * sizeof(float2), size_t(2 * LPH * V) * 4);
        const dim3 grid{unsigned(blocks)}, block{256};
        choose([&](auto one, auto whole) {
          heads_backward_kernel<T, LPH, decltype(one)::value, decltype(whole)::value>
              <<<grid, block, lds, hipStream_t(stream)>>>(a);
        }, a.group == 1, 2 * a.turned == a.dim);
        return check_launch("qk_norm_rotary_backward");
      });
    });
    if (rc) return rc;
  }
  return by_dtype(h->w_dtype, [&](auto w) {
    using W = decltype(w);
    weights_kernel<W><<<unsigned(ceil_div(2 * a.dim, 8)), 256, 0, hipStream_t(stream)>>>(
        a.part, static_cast<W*>(dq_weight), static_cast<W*>(dk_weight), a.dim, a.total ? int(blocks) : 0);
    return check_launch("qk_norm_rotary_backward (weights)");
  });
}

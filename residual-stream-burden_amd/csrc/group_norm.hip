// Group norm with an activation over a channels-last tensor [batch, pixels, channels], and its
// gradients. For one image and group of n = pixels x channels/groups elements, in fp32:
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), h = (x - m) r, u = w h + b, y = act(u)
//   g  = dy act'(u);  db[c] = sum g;  dw[c] = sum g h          (sums over images and pixels)
//   dx = r (w g - mean(w g) - h mean(w g h))
//
// Both directions are bound by memory: forward x in and y out, backward x and dy in and dx out.
//
// Whole slices: a block owns the channels of one or a few groups of one image and holds all of their
// pixels in registers, so that the statistics and the result take one pass over memory. 64 images of
// 32 x 32 x 1152 bf16 channels in 32 groups: forward 80 us, 3.8 TB/s of 302 MB; gradients 154 us, 2.9 TB/s
// of 453 MB. What bounds them: a block's loads, sums, exponentials and stores follow one another and
// its registers leave one or two blocks to a CU, so the memory idles where the blocks of a CU meet in
// the same phase.
//
// Whole rows, twice: where a slice does not fit a block's registers, and where images are so large that
// slices of a few groups read too short pieces of a pixel, the pixels pass in whole rows, once for the
// moments and once for the result. 64 images of 64 x 64 x 1152: 343 us, 3.5 TB/s of the 1.2 GB in and
// out (5.3 TB/s with the second reading); by slices 392. Their gradients 570 us, 3.2 TB/s of the 1.8 GB in and out
// (5.3 TB/s with the second reading of x and dy).
//
// What this is not made for: images of one pixel ([rows, channels]). A block then holds one slice of a row, and the
// weights' gradients are one chain of sums over the images: 262,144 rows of 1152 channels 5.8 ms and 13 ms.
//
// A mean is subtracted before squares are summed (over the block's own elements, or about a middle value of
// a thread's own, then about the threads' and the chunks' means), so neither a large mean nor a value far from
// the others costs digits. Channel sums are added in a fixed
// order, without atomics.
#include "cond_common.h"

namespace {
using namespace sihc_cond;

struct Shape {
  int64_t batch, pixels;
  int C, groups, per_group;  // channels, groups, channels of a group
  int slice_groups, W;       // groups and channels of a block's slice
  int threads;               // of a block
  int lanes, rows;           // vectors of a slice's pixel; pixels a block loads at once
  // rows of whole pixels (the streaming kernels): an image in chunks, a pixel in `widths` of W channels
  int widths, chunks;
  int64_t span;  // pixels of a chunk
  float eps;
  bool silu;
};

// A rounded product: where a group has one element, its gradient less its mean is exactly zero.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// The vectors that a thread holds are worked on one after another, and converted anew in each phase:
// interleaved, or kept from one phase to the next, their fp32 values would not fit its registers.
template <typename T, int V>
__device__ __forceinline__ void convert(Vec<T, V>& held, float* v) {
  asm volatile("" : "+v"(held.raw));
  held.to(v);
}
// A thread's Place::reach, for one phase: kept from one phase to the next, the comparisons with it would
// take the scalar registers.
__device__ __forceinline__ int for_phase(int reach) {
  asm volatile("" : "+v"(reach));
  return reach;
}
__device__ __forceinline__ void one_vector() { __builtin_amdgcn_sched_barrier(0); }

struct Place {
  int64_t b;
  int slice, lane, row, group;  // group: of the slice
  bool on;
  int reach;  // pixels from this thread's first on (0 for a thread without pixels)
};
// Of block `block` among `blocks`; neighbouring slices share lines, so they go to one XCD.
template <int V>
__device__ __forceinline__ Place place(const Shape& s, int block, int blocks) {
  Place p;
  const int slices = s.groups / s.slice_groups;
  const int64_t at = xcd_block(block, blocks);
  p.b = at / slices;
  p.slice = int(at - p.b * slices);
  p.row = int(threadIdx.x) / s.lanes;
  p.lane = int(threadIdx.x) - p.row * s.lanes;
  p.on = p.row < s.rows;
  p.group = p.on ? p.lane * V / s.per_group : 0;
  p.reach = p.on ? int(s.pixels) - p.row : 0;
  return p;
}

// Threads of a block, at most, and the blocks of 1024 threads on a CU that a kernel is compiled for: two
// where what a thread holds, and works with beside it, fits 64 registers, so that one loads while
// the other computes.
constexpr int MOST_THREADS = 1024, MIDDLE = 512, MIDDLE_VECTORS = 20;
constexpr int large_blocks(int held, int V, bool backward) {
  return (backward ? held + 4 * V <= 22 : held + 2 * V <= 28) ? 2 : 1;
}
[[maybe_unused]] constexpr int simd_waves(int TB, int held, int V, bool backward) {
  return TB == MIDDLE ? 4 : TB < MOST_THREADS ? 1 : 4 * large_blocks(held, V, backward);
}
template <typename T, int V>
constexpr int words() { return V * int(sizeof(T)) < 4 ? 1 : V * int(sizeof(T)) / 4; }

// Sums of two values over the threads of each group of the slice, for every thread its own group's.
// lds: 2 x TB floats, not in use since the last barrier but one. of: the groups' sums, where there are several.
template <int TB>
__device__ __forceinline__ float2 two_sums(float2 v, const Shape& s, int group, float* lds, float2* of) {
  const int tid = int(threadIdx.x), wave = tid >> 6, lane = tid & 63;
  float2 out = {0.f, 0.f};
  if (s.slice_groups == 1) {
    v = {wave_sum(v.x), wave_sum(v.y)};
    if (lane == 0) {
      lds[wave] = v.x;
      lds[TB + wave] = v.y;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TB / 64; ++k) {
      out.x += lds[k];
      out.y += lds[TB + k];
    }
    return out;
  }
  lds[tid] = v.x;
  lds[TB + tid] = v.y;
  __syncthreads();
  const int span = s.lanes / s.slice_groups, count = s.rows * span;
  for (int g = wave; g < s.slice_groups; g += TB / 64) {
    float2 t = {0.f, 0.f};
    for (int i = lane; i < count; i += 64) {
      const int at = (i / span) * s.lanes + g * span + i % span;
      t.x += lds[at];
      t.y += lds[TB + at];
    }
    t = {wave_sum(t.x), wave_sum(t.y)};
    if (lane == 0) of[g] = t;
  }
  __syncthreads();
  return of[group];
}

// Sums of the V elements of a vector and of their squares. bf16: two elements an instruction, the
// products exact and the sums fp32.
template <typename T, int V>
__device__ __forceinline__ void add_moments(const Vec<T, V>& v, float2& sum) {
  if constexpr (sizeof(T) == 2 && V >= 2) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    constexpr uint32_t ONES = 0x3f803f80u;
    uint32_t w[V / 2];
    __builtin_memcpy(w, &v.raw, sizeof(w));
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const pair x = __builtin_bit_cast(pair, w[k]);
      sum.x = __builtin_amdgcn_fdot2_f32_bf16(x, __builtin_bit_cast(pair, ONES), sum.x, false);
      sum.y = __builtin_amdgcn_fdot2_f32_bf16(x, x, sum.y, false);
    }
  } else {
    float f[V];
    v.to(f);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sum.x += f[e];
      sum.y = fmaf(f[e], f[e], sum.y);
    }
  }
}

// u sigmoid(u) from u and -u log2(e).
__device__ __forceinline__ float silu(float u, float minus_u2) {
  return u * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(minus_u2));
}
constexpr float LOG2E = 1.4426950408889634f;

// Whole slices, one a block. The variance is first taken from the sums of x and of x^2; where that loses
// digits (a mean above 8 deviations, or any fp32 input) from the squares about the mean. stats:
// [batch, groups] of (mean, rstd), may be null.
template <typename T, typename TW, int V, int NV, int TB>
__global__ __launch_bounds__(TB, (simd_waves(TB, NV * words<T, V>(), V, false))) void k_group_norm(
    const T* __restrict__ x, const TW* __restrict__ weight, const TW* __restrict__ bias, T* __restrict__ y,
    float2* __restrict__ stats, Shape s) {
  __shared__ float lds[2][2 * TB];
  __shared__ float2 sums[TB];
  const Place p = place<V>(s, int(blockIdx.x), int(gridDim.x));
  const int64_t at = (p.b * s.pixels + p.row) * s.C + p.slice * s.W + p.lane * V, step = int64_t(s.rows) * s.C;
  Vec<T, V> held[NV];
  int reach = for_phase(p.reach);
#pragma unroll
  for (int k = 0; k < NV; ++k) held[k] = k * s.rows < reach ? load<T, V>(x + at + k * step) : Vec<T, V>::zero();
  const float inverse_n = 1.f / (float(s.pixels) * float(s.per_group));
  float2 sum = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) add_moments(held[k], sum);
  sum = two_sums<TB>(p.on ? sum : float2{0.f, 0.f}, s, p.group, lds[0], sums);
  const float mean = sum.x * inverse_n;
  float var = sum.y * inverse_n - mean * mean;
  // The same answer for every thread of the block, which meet at barriers below: each works out every group's from
  // the same sums by the same instructions, and takes its own group's from nowhere else.
  bool lost = sizeof(T) == 4 || (s.slice_groups == 1 && !(mean * mean <= 64.f * var));
  for (int g = 0; sizeof(T) == 2 && s.slice_groups > 1 && g < s.slice_groups; ++g) {
    const float m = sums[g].x * inverse_n, v = sums[g].y * inverse_n - m * m;
    lost |= !(m * m <= 64.f * v);
  }
  if (lost) {
    float2 squares = {0.f, 0.f};
    reach = for_phase(p.reach);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      one_vector();
      if (k * s.rows < reach) {
        float v[V];
        convert(held[k], v);
#pragma unroll
        for (int e = 0; e < V; ++e) squares.x += (v[e] - mean) * (v[e] - mean);
      }
    }
    var = two_sums<TB>(squares, s, p.group, lds[1], sums).x * inverse_n;
  }
  const float rstd = 1.f / sqrtf(var + s.eps);
  if (stats && p.row == 0 && p.on && p.lane * V % s.per_group == 0)
    stats[p.b * s.groups + p.slice * s.slice_groups + p.group] = {mean, rstd};
  // u = (x - shift) a + d. bf16: shift = 0, a = weight rstd, d = bias - mean a, whose rounding is far below
  // the output's; fp32: the mean is subtracted first.
  const int c = p.on ? p.slice * s.W + p.lane * V : 0;
  float a[V], d[V];
  load_f32<TW, V>(weight + c, a);
  load_f32<TW, V>(bias + c, d);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    a[e] *= rstd;
    if (sizeof(T) == 2) d[e] = fmaf(-mean, a[e], d[e]);
  }
  T* dst = y + at;
  reach = for_phase(p.reach);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    one_vector();
    if (k * s.rows < reach) {
      float v[V];
      convert(held[k], v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u = fmaf(sizeof(T) == 4 ? v[e] - mean : v[e], a[e], d[e]);
        v[e] = s.silu ? silu(u, -LOG2E * u) : u;
      }
      store<T, V>(dst, Vec<T, V>::of(v));
    }
    dst += step;
  }
}

// ----------------------------------------------------------------------- whole rows, twice
// Rows pass in 16-byte vectors whatever the groups' width, the second time in reverse, so that the
// last-level cache still has part of what it reads. A block takes a chunk of an image's pixels; a thread
// holds V channels and walks the chunk's pixels, AHEAD of them loaded at once.
struct Stream {
  int64_t b, first;  // image, first pixel of the chunk
  int chunk, row, c, pixels;
  bool on;
};
template <int V>
__device__ __forceinline__ Stream stream_of(const Shape& s, int block) {
  Stream p;
  const int width = block % s.widths;
  const int64_t unit = block / s.widths;
  p.b = unit / s.chunks;
  p.chunk = int(unit - p.b * s.chunks);
  p.row = int(threadIdx.x) / s.lanes;
  p.c = width * s.W + (int(threadIdx.x) - p.row * s.lanes) * V;
  p.first = p.chunk * s.span;
  p.pixels = int(min(s.span, s.pixels - p.first));
  p.on = p.row < s.rows && p.c < s.C;
  return p;
}
constexpr int AHEAD = 4;

// One reading: 604 MB (64 images of 64 x 64 x 1152) in 136 us, 4.4 TB/s, the rest of the time the blocks' own sums.
// part: [batch, chunks, groups] of (mean, squares about it) of the chunk's pixels. A thread sums about the median
// of its channel's first three values, so that neither a mean nor a single value far from the others costs
// digits; the block then takes the mean of the threads' means, and their squares about that.
template <typename T, int V>
__global__ __launch_bounds__(1024) void k_norm_moments(const T* __restrict__ x, float2* __restrict__ part, Shape s) {
  extern __shared__ float lds[];  // [2][rows][W]: the threads' means, and squares about them
  const Stream p = stream_of<V>(s, int(blockIdx.x));
  const int tid = int(threadIdx.x), size = s.rows * s.W, groups = s.W / s.per_group, first_group = p.c / s.W * groups;
  const int64_t at = (p.b * s.pixels + p.first + p.row) * s.C + p.c, step = int64_t(s.rows) * s.C;
  const int cl = p.c % s.W;
  float shift[V] = {}, sum[V] = {}, squares[V] = {};
  int count = 0;
  if (p.on && p.row < p.pixels) {
    count = (p.pixels - p.row + s.rows - 1) / s.rows;
    for (int k0 = 0; k0 < count; k0 += AHEAD) {
      Vec<T, V> v[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) v[j] = load<T, V>(x + at + min(k0 + j, count - 1) * step);
      if (k0 == 0) {
        float f[3][V];
#pragma unroll
        for (int j = 0; j < 3; ++j) v[j].to(f[j]);
#pragma unroll
        for (int e = 0; e < V; ++e) shift[e] = __builtin_amdgcn_fmed3f(f[0][e], f[1][e], f[2][e]);
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (k0 + j >= count) break;
        float f[V];
        v[j].to(f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = f[e] - shift[e];
          sum[e] += d;
          squares[e] = fmaf(d, d, squares[e]);
        }
      }
    }
  }
  if (p.on) {
    const float inverse = count ? 1.f / float(count) : 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      lds[p.row * s.W + cl + e] = fmaf(sum[e], inverse, shift[e]);
      lds[size + p.row * s.W + cl + e] = fmaxf(squares[e] - sum[e] * (sum[e] * inverse), 0.f);
    }
  }
  __syncthreads();
  // (row r holds `each` pixels, or one more)
  const int each = p.pixels / s.rows, more = p.pixels - each * s.rows, used = min(s.rows, p.pixels);
  const float n = float(p.pixels) * float(s.per_group), inverse_n = 1.f / n;
  for (int g = tid >> 6; g < groups; g += int(blockDim.x) >> 6) {
    if (first_group + g >= s.groups) break;
    float mean = 0.f, a = 0.f, d = 0.f;
    for (int r = 0; r < used; ++r)
      for (int k = tid & 63; k < s.per_group; k += 64)
        mean = fmaf(float(each + (r < more)) * inverse_n, lds[r * s.W + g * s.per_group + k], mean);
    mean = wave_sum(mean);
    for (int r = 0; r < used; ++r)
      for (int k = tid & 63; k < s.per_group; k += 64) {
        const float off = lds[r * s.W + g * s.per_group + k] - mean, count = float(each + (r < more));
        a = fmaf(count, off, a);
        d += fmaf(count * off, off, lds[size + r * s.W + g * s.per_group + k]);
      }
    a = wave_sum(a);  // (what rounding left of the mean)
    d = wave_sum(d);
    if ((tid & 63) == 0)
      part[(p.b * s.chunks + p.chunk) * s.groups + first_group + g] = {fmaf(a, inverse_n, mean),
                                                                       fmaxf(d - a * (a * inverse_n), 0.f)};
  }
}

// stats: [batch, groups] of (mean, rstd) from the chunks' moments; a wave a group.
__global__ __launch_bounds__(256) void k_norm_stats(const float2* __restrict__ part, float2* __restrict__ stats,
                                                    float2* __restrict__ out, Shape s) {
  const int64_t i = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= s.batch * s.groups) return;
  const int64_t b = i / s.groups;
  const float2* from = part + b * s.chunks * s.groups + (i - b * s.groups);
  const int lane = int(threadIdx.x & 63);
  float mean = 0.f, squares = 0.f;
  for (int k = lane; k < s.chunks; k += 64)
    mean += float(min(s.span, s.pixels - k * s.span)) / float(s.pixels) * from[int64_t(k) * s.groups].x;
  mean = wave_sum(mean);
  for (int k = lane; k < s.chunks; k += 64) {
    const float2 p = from[int64_t(k) * s.groups];
    squares += p.y + float(min(s.span, s.pixels - k * s.span)) * float(s.per_group) * (p.x - mean) * (p.x - mean);
  }
  squares = wave_sum(squares);
  if (lane) return;
  const float2 st = {mean, 1.f / sqrtf(squares / (float(s.pixels) * float(s.per_group)) + s.eps)};
  stats[i] = st;
  if (out) out[i] = st;
}

template <typename T, typename TW, int V>
__global__ __launch_bounds__(1024) void k_norm_apply(const T* __restrict__ x, const TW* __restrict__ weight,
                                                     const TW* __restrict__ bias, const float2* __restrict__ stats,
                                                     T* __restrict__ y, Shape s) {
  const Stream p = stream_of<V>(s, int(gridDim.x) - 1 - int(blockIdx.x));
  if (!p.on || p.row >= p.pixels) return;
  const int64_t at = (p.b * s.pixels + p.first + p.row) * s.C + p.c, step = int64_t(s.rows) * s.C;
  float a[V], d[V], mean[V];
  load_f32<TW, V>(weight + p.c, a);
  load_f32<TW, V>(bias + p.c, d);
#pragma unroll
  for (int e = 0; e < V; ++e) {  // u = (x - mean) a + d, as k_group_norm
    const float2 st = stats[p.b * s.groups + (p.c + e) / s.per_group];
    a[e] *= st.y;
    mean[e] = st.x;
    if (sizeof(T) == 2) d[e] = fmaf(-st.x, a[e], d[e]);
  }
  const int count = (p.pixels - p.row + s.rows - 1) / s.rows;
  for (int k0 = 0; k0 < count; k0 += AHEAD) {
    Vec<T, V> v[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v[j] = load<T, V>(x + at + min(k0 + j, count - 1) * step);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (k0 + j >= count) break;
      float f[V];
      v[j].to(f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u = fmaf(sizeof(T) == 4 ? f[e] - mean[e] : f[e], a[e], d[e]);
        f[e] = s.silu ? silu(u, -LOG2E * u) : u;
      }
      store<T, V>(y + at + (k0 + j) * step, Vec<T, V>::of(f));
    }
  }
}

// Sums over the block's rows of each channel's two values, left in channel[2][W]. lds: 2 x rows x W floats,
// then 2 x W for `channel`.
template <int V, int TB>
__device__ __forceinline__ float* channel_sums(const float* sg, const float* sh, const Place& p, const Shape& s,
                                               float* lds) {
  const int tid = int(threadIdx.x), size = s.rows * s.W;
  float* channel = lds + 2 * size;
  if (p.on)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      lds[p.row * s.W + p.lane * V + e] = sg[e];
      lds[size + p.row * s.W + p.lane * V + e] = sh[e];
    }
  __syncthreads();
  // the threads' first step adds rows a stride apart, the second the strides, in ascending order
  const int stride = max(1, min(s.rows, TB / (2 * s.W)));
  for (int i = tid; i < 2 * s.W * stride; i += TB) {
    const int which = i / (s.W * stride), rest = i - which * s.W * stride, first = rest / s.W, k = rest - first * s.W;
    float sum = 0.f;
    for (int r = first; r < s.rows; r += stride) sum += lds[which * size + r * s.W + k];
    lds[which * size + first * s.W + k] = sum;  // (of these rows, which no other thread reads)
  }
  __syncthreads();
  for (int i = tid; i < 2 * s.W; i += TB) {
    const int which = i / s.W, k = i - which * s.W;
    float sum = 0.f;
    for (int r = 0; r < stride; ++r) sum += lds[which * size + r * s.W + k];
    channel[i] = sum;
  }
  __syncthreads();
  return channel;
}

// h and g = dy act'(u) of an element.
__device__ __forceinline__ void element(float x, float dy, float2 st, float w, float b, bool act, float& h, float& g) {
  h = (x - st.x) * st.y;
  g = dy;
  if (act) {
    const float u = fmaf(h, w, b), q = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * u));
    g *= q * fmaf(u, 1.f - q, 1.f);
  }
}

// The means of w g and of w g h over a group, from its channels' sums; one wave a group.
template <typename TW, int TB>
__device__ __forceinline__ void group_means(const TW* weight, const float* channel, const Place& p, const Shape& s,
                                            float2* means) {
  const int tid = int(threadIdx.x);
  const float inverse_n = 1.f / (float(s.pixels) * float(s.per_group));
  for (int g = tid >> 6; g < s.slice_groups; g += TB / 64) {
    float a = 0.f, d = 0.f;
    for (int k = tid & 63; k < s.per_group; k += 64) {
      const float wk = to_f32(weight[p.slice * s.W + g * s.per_group + k]);
      a += wk * channel[g * s.per_group + k];
      d += wk * channel[s.W + g * s.per_group + k];
    }
    a = wave_sum(a);
    d = wave_sum(d);
    if ((tid & 63) == 0) means[g] = {a * inverse_n, d * inverse_n};
  }
  __syncthreads();
}

// Whole slices, one a block. g takes the registers that dy came in, as fp32, so that the second pass needs
// no exponentials; part: [batch][2][C] sums over the pixels of g and of g h.
template <typename T, typename TW, int V, int NV, int TB>
__global__ __launch_bounds__(TB, (simd_waves(TB, NV * (words<T, V>() + V), V, true))) void k_group_norm_grad(
    const T* __restrict__ dy, const T* __restrict__ x, const TW* __restrict__ weight, const TW* __restrict__ bias,
    const float2* __restrict__ stats, T* __restrict__ dx, float* __restrict__ part, Shape s) {
  extern __shared__ float lds[];
  __shared__ float2 means[TB];
  const int tid = int(threadIdx.x);
  const Place p = place<V>(s, int(blockIdx.x), int(gridDim.x));
  const int64_t at = (p.b * s.pixels + p.row) * s.C + p.slice * s.W + p.lane * V, step = int64_t(s.rows) * s.C;
  Vec<T, V> hx[NV], hg[NV];
  int reach = for_phase(p.reach);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const bool in = k * s.rows < reach;
    hx[k] = in ? load<T, V>(x + at + k * step) : Vec<T, V>::zero();
    hg[k] = in ? load<T, V>(dy + at + k * step) : Vec<T, V>::zero();
  }
  const int c = p.on ? p.slice * s.W + p.lane * V : 0;
  const float2 st = stats[p.b * s.groups + p.slice * s.slice_groups + p.group];
  float g[NV][V], w[V], sg[V] = {}, sh[V] = {};
  load_f32<TW, V>(weight + c, w);
  {
    float b[V];
    load_f32<TW, V>(bias + c, b);
    reach = for_phase(p.reach);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      one_vector();
      if (k * s.rows < reach) {
        float xv[V], gv[V];
        convert(hx[k], xv);
        hg[k].to(gv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float h;
          element(xv[e], gv[e], st, w[e], b[e], s.silu, h, g[k][e]);
          sg[e] += g[k][e];
          sh[e] = fmaf(g[k][e], h, sh[e]);
        }
      }
    }
  }
  const float* channel = channel_sums<V, TB>(sg, sh, p, s, lds);
  for (int i = tid; i < 2 * s.W; i += TB) {
    const int which = i / s.W;
    part[(p.b * 2 + which) * s.C + p.slice * s.W + i - which * s.W] = channel[i];
  }
  group_means<TW, TB>(weight, channel, p, s, means);
  // dx = rstd (w g - mean_g - h mean_gh), h = (x - mean) rstd
  const float2 m = means[p.group];
  T* dst = dx + at;
  reach = for_phase(p.reach);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    one_vector();
    if (k * s.rows < reach) {
      float xv[V];
      convert(hx[k], xv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = (xv[e] - st.x) * st.y;
        xv[e] = st.y * (rounded_product(w[e], g[k][e]) - m.x - h * m.y);
      }
      store<T, V>(dst, Vec<T, V>::of(xv));
    }
    dst += step;
  }
}

// Whole rows, as the forward's: the channels' sums of g and g h over a chunk, part [batch, chunks][2][C].
template <typename T, typename TW, int V, bool DX>
__global__ __launch_bounds__(1024) void k_norm_grad_rows(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const TW* __restrict__ weight, const TW* __restrict__ bias,
                                                        const float2* __restrict__ stats, const float2* __restrict__ means,
                                                        T* __restrict__ dx, float* __restrict__ part, Shape s) {
  extern __shared__ float lds[];  // [2][rows][W]
  const Stream p = stream_of<V>(s, DX ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x));
  const bool on = p.on && p.row < p.pixels;
  if (DX && !on) return;
  const int64_t at = (p.b * s.pixels + p.first + p.row) * s.C + p.c, step = int64_t(s.rows) * s.C;
  const int tid = int(threadIdx.x), size = s.rows * s.W, cl = p.c % s.W;
  float w[V] = {}, b[V] = {}, sg[V] = {}, sh[V] = {};
  float2 st[V] = {}, m[V] = {};
  if (on) {
    load_f32<TW, V>(weight + p.c, w);
    load_f32<TW, V>(bias + p.c, b);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int64_t group = p.b * s.groups + (p.c + e) / s.per_group;
      st[e] = stats[group];
      if (DX) m[e] = means[group];
    }
    const int count = (p.pixels - p.row + s.rows - 1) / s.rows;
    constexpr int N = AHEAD / 2;
    for (int k0 = 0; k0 < count; k0 += N) {
      Vec<T, V> vx[N], vg[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        vx[j] = load<T, V>(x + at + min(k0 + j, count - 1) * step);
        vg[j] = load<T, V>(dy + at + min(k0 + j, count - 1) * step);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (k0 + j >= count) break;
        float f[V], g0[V];
        vx[j].to(f);
        vg[j].to(g0);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float h, g;
          element(f[e], g0[e], st[e], w[e], b[e], s.silu, h, g);
          if (DX) {
            f[e] = st[e].y * (rounded_product(w[e], g) - m[e].x - h * m[e].y);
          } else {
            sg[e] += g;
            sh[e] = fmaf(g, h, sh[e]);
          }
        }
        if (DX) store<T, V>(dx + at + (k0 + j) * step, Vec<T, V>::of(f));
      }
    }
  }
  if constexpr (!DX) {
    if (p.on)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        lds[p.row * s.W + cl + e] = sg[e];
        lds[size + p.row * s.W + cl + e] = sh[e];
      }
    __syncthreads();
    const int c0 = p.c - cl;  // of the block's width (a thread past the rows has its own c, of the same width)
    for (int i = tid; i < 2 * s.W; i += int(blockDim.x)) {
      const int which = i / s.W, k = i - which * s.W;
      if (c0 + k >= s.C) continue;
      float sum = 0.f;
      for (int r = 0; r < s.rows; ++r) sum += lds[which * size + r * s.W + k];
      part[((p.b * s.chunks + p.chunk) * 2 + which) * s.C + c0 + k] = sum;
    }
  }
}

// One image: the channels' sums over its chunks, total [batch][2][C], and the groups' means of w g and w g h.
template <typename TW>
__global__ __launch_bounds__(1024) void k_norm_grad_means(const float* __restrict__ part, const TW* __restrict__ weight,
                                                          float* __restrict__ total, float2* __restrict__ means, Shape s) {
  const int64_t b = blockIdx.x;
  float* sums = total + b * 2 * s.C;
  for (int i = int(threadIdx.x); i < 2 * s.C; i += 1024) {
    float sum = 0.f;
#pragma unroll 8
    for (int k = 0; k < s.chunks; ++k) sum += part[(b * s.chunks + k) * 2 * s.C + i];
    sums[i] = sum;
  }
  __threadfence_block();
  __syncthreads();
  const float inverse_n = 1.f / (float(s.pixels) * float(s.per_group));
  for (int g = int(threadIdx.x) >> 6; g < s.groups; g += 16) {
    float a = 0.f, d = 0.f;
    for (int k = int(threadIdx.x) & 63; k < s.per_group; k += 64) {
      const int c = g * s.per_group + k;
      const float wk = to_f32(weight[c]);
      a += wk * sums[c];
      d += wk * sums[s.C + c];
    }
    a = wave_sum(a);
    d = wave_sum(d);
    if ((threadIdx.x & 63) == 0) means[b * s.groups + g] = {a * inverse_n, d * inverse_n};
  }
}

// out[c] = sum over the parts, in ascending order; 4 thread rows take a quarter of them each.
template <typename TW>
__global__ __launch_bounds__(256) void k_channel_sums(const float* __restrict__ part, TW* __restrict__ dw,
                                                      TW* __restrict__ db, int64_t parts, int C) {
  __shared__ float quarter[4][64];
  const int lane = int(threadIdx.x & 63), q = int(threadIdx.x >> 6), which = int(blockIdx.y);
  const int c = min(int(blockIdx.x) * 64 + lane, C - 1);
  const int64_t each = (parts + 3) / 4, begin = q * each, end = min(parts, begin + each);
  float sum = 0.f;
#pragma unroll 8
  for (int64_t k = begin; k < end; ++k) sum += part[(k * 2 + which) * C + c];
  quarter[q][lane] = sum;
  __syncthreads();
  if (q == 0 && int(blockIdx.x) * 64 + lane < C)
    (which ? dw : db)[c] = from_f32<TW>(((quarter[0][lane] + quarter[1][lane]) + quarter[2][lane]) + quarter[3][lane]);
}

// ---------------------------------------------------------------------------------- host
// The register words a thread holds, at most.
constexpr int WORDS = 80;
// Images from so many bytes on pass in whole rows though their slices fit (64 images of 64 x 64 x 1152,
// 9.4 MB each: 343 us, by slices 392; of 32 x 32 x 1152, 2.4 MB: 106 and 80, the gradients 168 and 154).
constexpr int64_t STREAM_FROM = int64_t(4) << 20;
struct Plan {
  Shape s;
  bool whole;  // one slice a block; else whole rows
  int V, NV;
};
// The widest vector of at most 16 bytes that divides a group, so that each lies in one group.
int vec_of(int per_group, int elem) {
  for (int v : {8, 4, 2})
    if (v * elem <= 16 && per_group % v == 0) return v;
  return 1;
}
// Vectors of a pixel that a block takes in whole rows, at most: LDS holds two sums of each channel.
int most_lanes(int V) { return V >= 4 ? 512 : MOST_THREADS; }
// backward: a block holds x and the output's gradient, and that in fp32.
Plan plan(int64_t batch, int64_t pixels, int C, int groups, float eps, bool silu, int elem, bool backward) {
  Plan p{};
  Shape& s = p.s;
  s.batch = batch;
  s.pixels = pixels;
  s.C = C;
  s.groups = groups;
  s.per_group = C / groups;
  s.eps = eps;
  s.silu = silu;
  p.V = vec_of(s.per_group, elem);
  // whole groups until a pixel's piece is a line of 128 bytes, as long as the slice fits and the grid fills
  // the card (64 x 32 x 32 x 1152, 36 channels a group: pieces of 72 bytes 88 us, writing 1.17 times the
  // output, of 144 bytes 82 us and 1.00)
  const int most = WORDS / (std::max(1, p.V * elem / 4) + (backward ? p.V : 0));
  auto vectors = [&](int g, int threads) {
    const int lanes = g * s.per_group / p.V;
    return lanes > threads ? int64_t(1) << 40 : ceil_div(pixels, threads / lanes);
  };
  s.slice_groups = 1;
  for (int g = 2; g <= groups; ++g) {
    if (groups % g || g * s.per_group / p.V > MOST_THREADS) continue;
    if (vectors(g, MOST_THREADS) > most || s.slice_groups * s.per_group * elem >= 128 || batch * (groups / g) < 512) break;
    s.slice_groups = g;
  }
  // small slices: blocks of 256 threads, several to a CU (256 x 4 x 4 x 1152: 24 us, by 1024 threads 50; 64 x 7 x 7
  // x 136: 17.6 and 18.9)
  s.threads = vectors(s.slice_groups, 256) <= std::min(8, most) ? 256 : MOST_THREADS;
  // forward: two blocks of 512 threads to a CU where the grid has them and a thread's 20 vectors hold the slice (32
  // images of 32 x 32 x 768: 22 us, by 1024 threads 26; 128 of 16 x 16 x 1152: 29 and 35; fp32, 64 of 32 x 32 x
  // 512: 45 and 56; by twice as many shorter vectors, 64 of 32 x 32 x 1152, 79 and 78; the gradients hold too much)
  if (!backward && p.V * elem >= 8 && s.threads == MOST_THREADS &&
      vectors(s.slice_groups, MIDDLE) <= std::min(MIDDLE_VECTORS, most) && batch * (groups / s.slice_groups) >= 512)
    s.threads = MIDDLE;
  s.W = s.slice_groups * s.per_group;
  s.lanes = s.W / p.V;
  s.rows = s.threads / s.lanes;
  p.NV = int(std::min<int64_t>(ceil_div(pixels, s.rows), most + 1));
  p.whole = p.NV <= most && pixels * C * elem < STREAM_FROM;
  if (p.whole) return p;
  // whole rows: 16-byte vectors where a pixel's fit a block, else whole groups of them
  p.V = vec_of(C, elem);
  int threads = most_lanes(p.V);
  s.W = C;
  s.widths = 1;
  if (C / p.V > threads) {
    p.V = vec_of(s.per_group, elem);
    threads = most_lanes(p.V);
    s.W = std::max(1, threads * p.V / s.per_group) * s.per_group;
    s.widths = int(ceil_div(C, s.W));
  }
  s.lanes = s.W / p.V;
  s.rows = std::max(1, 512 / s.lanes);
  s.threads = int(ceil_div(int64_t(s.rows) * s.lanes, 64) * 64);
  // 32 pixels a thread, fewer for 32 chunks of an image (64 images of 64 x 64 x 1152: forward 380 us by 8
  // pixels, 368 by 16, 352 by 32; one image 20, 21 and 24; its results do not depend on the batch)
  const int64_t steps = std::max<int64_t>(4, std::min<int64_t>(32, pixels / (int64_t(s.rows) * 32)));
  s.span = steps * s.rows;
  s.chunks = int(ceil_div(pixels, s.span));
  return p;
}

int check_sizes(const char* what, int64_t batch, int64_t pixels, int C, int groups, int act, int dtype, int w_dtype) {
  // (channels are counted in int32, two sums of each)
  if (batch < 0 || pixels < 0 || C <= 0 || C > (1 << 24) || (pixels && batch > SIHC_MAX_TOKENS / pixels))
    return fail(SIHC_ERR_INVALID, "%s: bad sizes", what);
  if (groups <= 0 || C % groups) return fail(SIHC_ERR_INVALID, "%s: %d channels are not %d groups", what, C, groups);
  const int V = vec_of(C / groups, dtype == SIHC_DTYPE_F32 ? 4 : 2);
  if (C / groups / V > most_lanes(V))
    return fail(SIHC_ERR_INVALID, "%s: groups of %d channels are too wide", what, C / groups);
  if (act != SIHC_ACT_NONE && act != SIHC_ACT_SILU) return fail(SIHC_ERR_INVALID, "%s: bad activation %d", what, act);
  if (!valid_dtype(dtype) || !valid_dtype(w_dtype)) return fail(SIHC_ERR_INVALID, "%s: bad dtype", what);
  if (w_dtype != dtype && w_dtype != SIHC_DTYPE_F32)
    return fail(SIHC_ERR_INVALID, "%s: weights must be fp32 or share the input's type", what);
  return SIHC_OK;
}
// The chunks of a pass that leaves no sums: short, their length changes no result (64 x 64 x 64 x 1152, 32 steps
// in the chunks of the moments: the forward 341 us by 4 steps, 353 by 8, 367 by 32; one image 21, 21 and 31).
Shape short_chunks(Shape s) {
  s.span = AHEAD * s.rows;
  // (longer ones where an image's would pass what a launch takes)
  while (ceil_div(s.pixels, s.span) * s.widths * s.threads > MOST_LAUNCHED) s.span *= 2;
  s.chunks = int(ceil_div(s.pixels, s.span));
  return s;
}
int elem_size(int dtype) { return dtype == SIHC_DTYPE_F32 ? 4 : 2; }
// Images whose blocks a launch takes, for the widest of the launches of a direction; 0: not one.
int64_t images_of_launch(const Plan& p) {
  const Shape& s = p.s;
  int64_t most = 0;
  if (p.whole) {
    most = int64_t(s.groups / s.slice_groups) * s.threads;
  } else {
    const int64_t sums = int64_t(s.chunks) * s.widths * s.threads,
                  result = int64_t(short_chunks(s).chunks) * s.widths * s.threads;
    most = std::max({sums, result, int64_t(s.groups) * 64, int64_t(1024)});  // (a wave a group, a block an image)
  }
  return MOST_LAUNCHED / most;
}
// Calls f(first image, images) for as many images at a time as a launch takes: a million rows of few channels are
// a million images of one pixel.
template <typename F>
int by_images(const char* what, const Plan& p, F&& f) {
  const int64_t step = images_of_launch(p);
  if (step == 0) return fail(SIHC_ERR_INVALID, "%s: tensor too large", what);
  int rc = SIHC_OK;
  for (int64_t b = 0; b < p.s.batch && !rc; b += step) rc = f(b, std::min(step, p.s.batch - b));
  return rc;
}
template <typename P>
P* advanced(P* p, int64_t elements, int size) {  // (the element type is known by its size alone)
  using Byte = std::conditional_t<std::is_const_v<P>, const char, char>;
  return p ? static_cast<P*>(static_cast<Byte*>(p) + elements * size) : nullptr;
}

// Calls f(T, TW, V, NV, TB) with NV the smallest compiled count of at least p.NV vectors, or, for whole
// rows, rows(T, TW, V).
template <bool BACKWARD, typename F, typename R>
int by_plan(const Plan& p, int dtype, int w_dtype, F&& f, R&& rows) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto with = [&](auto tw, auto v) {
      if (!p.whole) return rows(t, tw, v);
      constexpr int V = decltype(v)::value, MOST = WORDS / (words<T, V>() + (BACKWARD ? V : 0));
      int rc = SIHC_OK;
      auto attempt = [&](auto nv, auto tb) {
        constexpr int NV = decltype(nv)::value;
        if constexpr (NV <= MOST) {
          if (p.s.threads == decltype(tb)::value && p.NV <= NV) {
            rc = f(t, tw, v, nv, tb);
            return true;
          }
        }
        return false;
      };
      constexpr IC<256> small{};
      constexpr IC<1024> large{};
      if constexpr (!BACKWARD && V * sizeof(T) >= 8) {
        constexpr IC<MIDDLE> middle{};
        if (attempt(IC<8>{}, middle) || attempt(IC<14>{}, middle) || attempt(IC<MIDDLE_VECTORS>{}, middle))
          return rc;
      }
      if (attempt(IC<1>{}, small) || attempt(IC<2>{}, small) || attempt(IC<4>{}, small) || attempt(IC<6>{}, small) ||
          attempt(IC<8>{}, small) ||
          attempt(IC<4>{}, large) || attempt(IC<7>{}, large) || attempt(IC<10>{}, large) || attempt(IC<14>{}, large) ||
          attempt(IC<20>{}, large) || attempt(IC<28>{}, large) || attempt(IC<40>{}, large) || attempt(IC<80>{}, large) ||
          attempt(IC<MOST>{}, large))
        return rc;
      return fail(SIHC_ERR_INVALID, "group norm: internal plan");
    };
    auto by_v = [&](auto tw) {
      switch (p.V) {
        case 8:
          if constexpr (sizeof(T) == 2) return with(tw, IC<8>{});
        case 4: return with(tw, IC<4>{});
        case 2: return with(tw, IC<2>{});
        default: return with(tw, IC<1>{});
      }
    };
    return w_dtype == SIHC_DTYPE_F32 ? by_v(float{}) : by_v(T{});
  });
}

}  // namespace

extern "C" {

size_t sihc_group_norm_workspace_size(int64_t batch, int64_t pixels, int channels, int groups, int dtype) {
  if (check_sizes("sihc_group_norm", batch, pixels, channels, groups, SIHC_ACT_NONE, dtype, dtype) || batch == 0 ||
      pixels == 0)
    return 0;
  const Plan p = plan(batch, pixels, channels, groups, 0.f, false, elem_size(dtype), false);
  return p.whole ? 0 : size_t(batch) * size_t(p.s.chunks + 1) * size_t(groups) * 8;  // the chunks' moments, the statistics
}

int sihc_group_norm(const void* x, const void* weight, const void* bias, void* y, float* stats, int64_t batch,
                    int64_t pixels, int channels, int groups, float eps, int act, int dtype, int w_dtype,
                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "sihc_group_norm";
  if (int rc = check_sizes(what, batch, pixels, channels, groups, act, dtype, w_dtype)) return rc;
  if (batch == 0 || pixels == 0) return SIHC_OK;
  if (!x || !weight || !bias || !y) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  const size_t need = sihc_group_norm_workspace_size(batch, pixels, channels, groups, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SIHC_ERR_INVALID, "%s: workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
  if (!aligned(workspace, 8) || !aligned(stats, 8)) return fail(SIHC_ERR_INVALID, "%s: misaligned workspace or stats", what);
  const Plan all = plan(batch, pixels, channels, groups, eps, act == SIHC_ACT_SILU, elem_size(dtype), false);
  const void* const whole_x = x;
  void* const whole_y = y;
  float2* const whole_stats = reinterpret_cast<float2*>(stats);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_images(what, all, [&](int64_t first, int64_t images) {
    Plan p = all;
    p.s.batch = images;
    const int64_t element = first * pixels * channels;
    const void* x = advanced(whole_x, element, elem_size(dtype));
    void* y = advanced(whole_y, element, elem_size(dtype));
    float2* stats = whole_stats ? whole_stats + first * groups : nullptr;
    const int64_t blocks = images * (p.whole ? groups / p.s.slice_groups : p.s.chunks * p.s.widths);
    const dim3 grid(static_cast<unsigned>(blocks)), threads(static_cast<unsigned>(p.s.threads));
    return by_plan<false>(
        p, dtype, w_dtype,
        [&](auto t, auto tw, auto v, auto nv, auto tb) {
          using T = decltype(t);
          using TW = decltype(tw);
          constexpr int V = decltype(v)::value, NV = decltype(nv)::value, TB = decltype(tb)::value;
          hipLaunchKernelGGL((k_group_norm<T, TW, V, NV, TB>), grid, threads, 0, st, static_cast<const T*>(x),
                             static_cast<const TW*>(weight), static_cast<const TW*>(bias), static_cast<T*>(y), stats, p.s);
          return check_launch(what);
        },
        [&](auto t, auto tw, auto v) {
          using T = decltype(t);
          using TW = decltype(tw);
          constexpr int V = decltype(v)::value;
          float2 *part = static_cast<float2*>(workspace), *own = part + images * p.s.chunks * groups;
          const unsigned lds = 2u * unsigned(p.s.rows) * unsigned(p.s.W) * 4u;
          hipLaunchKernelGGL((k_norm_moments<T, V>), grid, threads, lds, st, static_cast<const T*>(x), part, p.s);
          hipLaunchKernelGGL(k_norm_stats, dim3(unsigned(ceil_div(images * groups, 4))), dim3(256), 0, st, part, own,
                             stats, p.s);
          const Shape s = short_chunks(p.s);
          hipLaunchKernelGGL((k_norm_apply<T, TW, V>), dim3(unsigned(images * s.chunks * s.widths)), threads, 0, st,
                             static_cast<const T*>(x), static_cast<const TW*>(weight), static_cast<const TW*>(bias), own,
                             static_cast<T*>(y), s);
          return check_launch(what);
        });
  });
}

size_t sihc_group_norm_backward_workspace_size(int64_t batch, int64_t pixels, int channels, int groups, int dtype) {
  if (check_sizes("sihc_group_norm_backward", batch, pixels, channels, groups, SIHC_ACT_NONE, dtype, dtype) ||
      batch == 0 || pixels == 0)
    return 0;
  const Plan p = plan(batch, pixels, channels, groups, 0.f, false, elem_size(dtype), true);
  // the images' channel sums; whole rows: and the chunks', and the groups' means
  const size_t rows = size_t(batch) * 2 * size_t(channels) * 4;
  return p.whole ? rows : rows * size_t(p.s.chunks + 1) + size_t(batch) * size_t(groups) * 8;
}

int sihc_group_norm_backward(const void* grad, const void* x, const void* weight, const void* bias, const float* stats,
                             void* grad_x, void* grad_weight, void* grad_bias, int64_t batch, int64_t pixels,
                             int channels, int groups, int act, int dtype, int w_dtype, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* what = "sihc_group_norm_backward";
  if (int rc = check_sizes(what, batch, pixels, channels, groups, act, dtype, w_dtype)) return rc;
  if (!grad_weight || !grad_bias) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool empty = batch == 0 || pixels == 0;
  int64_t parts = 0;
  if (!empty) {
    if (!grad || !x || !weight || !bias || !stats || !grad_x) return fail(SIHC_ERR_INVALID, "%s: null pointer", what);
    for (const void* in : {grad, x, weight, bias, static_cast<const void*>(stats)})
      for (const void* out : {grad_x, grad_weight, grad_bias})
        if (in == out) return fail(SIHC_ERR_INVALID, "%s: an output is one of the inputs", what);
    const size_t need = sihc_group_norm_backward_workspace_size(batch, pixels, channels, groups, dtype);
    if (!workspace || workspace_bytes < need)
      return fail(SIHC_ERR_INVALID, "%s: workspace of %zu bytes required, got %zu", what, need, workspace_bytes);
    if (!aligned(workspace, 8) || !aligned(stats, 8))
      return fail(SIHC_ERR_INVALID, "%s: misaligned workspace or stats", what);
    const Plan all = plan(batch, pixels, channels, groups, 0.f, act == SIHC_ACT_SILU, elem_size(dtype), true);
    parts = batch;
    const void *const whole_grad = grad, *const whole_x = x;
    void* const whole_grad_x = grad_x;
    const int rc = by_images(what, all, [&](int64_t first, int64_t images) {
      Plan p = all;
      p.s.batch = images;
      const int64_t element = first * pixels * channels;
      const void *grad = advanced(whole_grad, element, elem_size(dtype)), *x = advanced(whole_x, element, elem_size(dtype));
      void* grad_x = advanced(whole_grad_x, element, elem_size(dtype));
      const float2* st2 = reinterpret_cast<const float2*>(stats) + first * groups;
      float* total = static_cast<float*>(workspace) + first * 2 * channels;  // every image's; the rest is used again
      const int64_t blocks = images * (p.whole ? groups / p.s.slice_groups : p.s.chunks * p.s.widths);
      const dim3 grid(static_cast<unsigned>(blocks)), threads(static_cast<unsigned>(p.s.threads));
      return by_plan<true>(
          p, dtype, w_dtype,
          [&](auto t, auto tw, auto v, auto nv, auto tb) {
            using T = decltype(t);
            using TW = decltype(tw);
            constexpr int V = decltype(v)::value, NV = decltype(nv)::value, TB = decltype(tb)::value;
            const unsigned lds = 2u * unsigned(p.s.rows + 1) * unsigned(p.s.W) * 4u;
            hipLaunchKernelGGL((k_group_norm_grad<T, TW, V, NV, TB>), grid, threads, lds, st, static_cast<const T*>(grad),
                               static_cast<const T*>(x), static_cast<const TW*>(weight), static_cast<const TW*>(bias),
                               st2, static_cast<T*>(grad_x), total, p.s);
            return check_launch(what);
          },
          [&](auto t, auto tw, auto v) {
            using T = decltype(t);
            using TW = decltype(tw);
            constexpr int V = decltype(v)::value;
            float* part = static_cast<float*>(workspace) + batch * 2 * channels;
            float2* means = reinterpret_cast<float2*>(part + images * p.s.chunks * 2 * channels);
            const unsigned lds = 2u * unsigned(p.s.rows) * unsigned(p.s.W) * 4u;
            auto pass = [&](auto dx) {
              constexpr bool DX = decltype(dx)::value;
              const Shape s = DX ? short_chunks(p.s) : p.s;
              hipLaunchKernelGGL((k_norm_grad_rows<T, TW, V, DX>), dim3(unsigned(images * s.chunks * s.widths)), threads,
                                 DX ? 0 : lds, st, static_cast<const T*>(grad), static_cast<const T*>(x),
                                 static_cast<const TW*>(weight), static_cast<const TW*>(bias), st2, means,
                                 static_cast<T*>(grad_x), part, s);
            };
            pass(std::false_type{});
            hipLaunchKernelGGL(k_norm_grad_means<TW>, dim3(unsigned(images)), dim3(1024), 0, st, part,
                               static_cast<const TW*>(weight), total, means, p.s);
            pass(std::true_type{});
            return check_launch(what);
          });
    });
    if (rc) return rc;
  }
  auto sums = [&](auto tw) {
    using TW = decltype(tw);
    hipLaunchKernelGGL(k_channel_sums<TW>, dim3(unsigned(ceil_div(channels, 64)), 2), dim3(256), 0, st,
                       static_cast<const float*>(workspace), static_cast<TW*>(grad_weight),
                       static_cast<TW*>(grad_bias), parts, channels);
  };
  if (w_dtype == SIHC_DTYPE_F32) sums(float{});
  else sums(bf16{});
  return check_launch(what);
}

}  // extern "C"

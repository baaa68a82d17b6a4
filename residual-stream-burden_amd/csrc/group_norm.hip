// Group norm with an activation over a channels-last tensor [batch, pixels, channels], and its
// gradients. For one image and group of n = pixels x channels/groups elements, in fp32:
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), h = (x - m) r, u = w h + b, y = act(u)
//   g  = dy act'(u);  db[c] = sum g;  dw[c] = sum g h          (sums over images and pixels)
//   dx = r (w g - mean(w g) - h mean(w g h))
//
// Both directions are bound by memory: forward x in and y out, backward x and dy in and dx out. A
// block owns a slice: the channels of one or a few groups of one image, whose pixels it holds in
// registers, so that the statistics and the result take one pass over memory. Where a slice is
// too large for a block's registers it is cut into chunks of pixels: one launch leaves each
// chunk's statistics, a second reads the chunks again and applies them. A mean is subtracted
// before squares are summed (over the block's own elements, then over the chunks' means), so a
// large mean costs no digits. Channel sums are added in a fixed order, without atomics.
#include "cond_common.h"

namespace {
using namespace sihc_cond;

constexpr int THREADS = 1024;

struct Shape {
  int64_t batch, pixels;
  int C, groups, per_group;  // channels, groups, channels of a group
  int slice_groups, W;       // groups and channels of a block's slice
  int lanes, rows;           // vectors of a slice's pixel; pixels a block loads at once
  int chunks;                // blocks that share a slice
  int64_t chunk_pixels;
  float eps;
  bool silu;
};

// A rounded product: where a group has one element, its gradient less its mean is exactly zero.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// What a launch does: all of it, or the two halves of a slice in chunks.
enum { WHOLE, STATS, APPLY };

// Sum of v over the threads of each group of the slice, left in out[group] (and visible to all).
__device__ __forceinline__ void group_sums(float v, const Shape& s, float* scratch, float* out) {
  const int tid = int(threadIdx.x);
  __syncthreads();  // earlier readers of scratch and out are done
  if (s.slice_groups == 1) {
    const float t = wave_sum(v);
    if ((tid & 63) == 0) scratch[tid >> 6] = t;
    __syncthreads();
    if (tid < 64) {
      const float sum = wave_sum(tid < int(blockDim.x >> 6) ? scratch[tid] : 0.f);
      if (tid == 0) out[0] = sum;
    }
  } else {
    scratch[tid] = v;
    __syncthreads();
    const int wave = tid >> 6, lane = tid & 63, waves = int(blockDim.x >> 6), span = s.lanes / s.slice_groups;
    for (int g = wave; g < s.slice_groups; g += waves) {
      float t = 0.f;
      for (int k = lane; k < s.rows * span; k += 64) t += scratch[(k / span) * s.lanes + g * span + k % span];
      t = wave_sum(t);
      if (lane == 0) out[g] = t;
    }
  }
  __syncthreads();
}

// The vectors that a thread holds are worked on one after another, and converted anew in each phase:
// interleaved, or kept from one phase to the next, their fp32 values would not fit its registers.
template <typename T, int V>
__device__ __forceinline__ void convert(Vec<T, V>& held, float* v) {
  asm volatile("" : "+v"(held.raw));
  held.to(v);
}
__device__ __forceinline__ void one_vector() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __expf(-u)); }

struct Place {
  int64_t b;
  int slice, chunk, lane, row, group;  // group: of the slice
  bool on;
  int64_t first;  // first pixel of the chunk
  int pixels;     // pixels of the chunk
};
template <int V>
__device__ __forceinline__ Place place(const Shape& s) {
  Place p;
  const int slices = s.groups / s.slice_groups;
  const int64_t block = xcd_block(int(blockIdx.x), int(gridDim.x));
  const int64_t unit = block / s.chunks;
  p.chunk = int(block - unit * s.chunks);
  p.b = unit / slices;
  p.slice = int(unit - p.b * slices);
  p.row = int(threadIdx.x) / s.lanes;
  p.lane = int(threadIdx.x) - p.row * s.lanes;
  p.on = p.row < s.rows;
  p.group = p.on ? p.lane * V / s.per_group : 0;
  p.first = p.chunk * s.chunk_pixels;
  p.pixels = int(min(s.chunk_pixels, s.pixels - p.first));
  return p;
}

// The mean and the sum of squares about it of a group from its chunks' (chunks x [mean, squares]).
__device__ __forceinline__ float2 merge(const float2* part, const Shape& s, int stride) {
  float mean = 0.f, squares = 0.f;
  for (int k = 0; k < s.chunks; ++k) {
    const float n = float(min(s.chunk_pixels, s.pixels - k * s.chunk_pixels)) / float(s.pixels);
    mean += n * part[int64_t(k) * stride].x;
  }
  for (int k = 0; k < s.chunks; ++k) {
    const float n = float(min(s.chunk_pixels, s.pixels - k * s.chunk_pixels)) * float(s.per_group);
    const float2 p = part[int64_t(k) * stride];
    squares += p.y + n * (p.x - mean) * (p.x - mean);
  }
  return {mean, squares};
}

// stats: [batch, groups] of (mean, rstd), may be null. part: [batch, chunks, groups] of (mean, squares).
template <typename T, typename TW, int V, int NV, int MODE>
__global__ __launch_bounds__(THREADS) void k_group_norm(const T* __restrict__ x, const TW* __restrict__ weight,
                                                        const TW* __restrict__ bias, T* __restrict__ y,
                                                        float2* __restrict__ stats, float2* __restrict__ part,
                                                        Shape s) {
  __shared__ float scratch[THREADS], sums[THREADS], sums2[THREADS];
  const Place p = place<V>(s);
  const int c = p.slice * s.W + p.lane * V;
  const int64_t at = (p.b * s.pixels + p.first + p.row) * s.C + c;
  const T* src = x + at;
  const int64_t step = int64_t(s.rows) * s.C;
  Vec<T, V> held[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    held[k] = p.on && k * s.rows + p.row < p.pixels ? load<T, V>(src + k * step) : Vec<T, V>::zero();
  }
  float mean, rstd;
  if constexpr (MODE != APPLY) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      one_vector();
      float v[V];
      convert(held[k], v);
#pragma unroll
      for (int e = 0; e < V; ++e) sum += v[e];
    }
    group_sums(p.on ? sum : 0.f, s, scratch, sums);
    const float n = float(p.pixels) * float(s.per_group);
    mean = sums[p.group] / n;
    float squares = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      one_vector();
      if (p.on && k * s.rows + p.row < p.pixels) {
        float v[V];
        convert(held[k], v);
#pragma unroll
        for (int e = 0; e < V; ++e) squares += (v[e] - mean) * (v[e] - mean);
      }
    }
    group_sums(squares, s, scratch, sums2);
    if constexpr (MODE == STATS) {
      if (int(threadIdx.x) < s.slice_groups) {
        const int g = p.slice * s.slice_groups + int(threadIdx.x);
        part[(p.b * s.chunks + p.chunk) * s.groups + g] = {sums[threadIdx.x] / n, sums2[threadIdx.x]};
      }
      return;
    }
    rstd = 1.f / sqrtf(sums2[p.group] / n + s.eps);
    if (stats && int(threadIdx.x) < s.slice_groups)
      stats[p.b * s.groups + p.slice * s.slice_groups + int(threadIdx.x)] = {
          sums[threadIdx.x] / n, 1.f / sqrtf(sums2[threadIdx.x] / n + s.eps)};
  } else {
    if (int(threadIdx.x) < s.slice_groups) {
      const int g = p.slice * s.slice_groups + int(threadIdx.x);
      const float2 m = merge(part + p.b * s.chunks * s.groups + g, s, s.groups);
      sums[threadIdx.x] = m.x;
      sums2[threadIdx.x] = 1.f / sqrtf(m.y / (float(s.pixels) * float(s.per_group)) + s.eps);
      if (stats && p.chunk == 0) stats[p.b * s.groups + g] = {m.x, sums2[threadIdx.x]};
    }
    __syncthreads();
    mean = sums[p.group];
    rstd = sums2[p.group];
  }
  if (!p.on) return;
  float w[V], b[V];
  load_f32<TW, V>(weight + c, w);
  load_f32<TW, V>(bias + c, b);
  T* dst = y + at;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    one_vector();
    if (k * s.rows + p.row < p.pixels) {
      float v[V];
      convert(held[k], v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u = fmaf((v[e] - mean) * rstd, w[e], b[e]);
        v[e] = s.silu ? u * sigmoid(u) : u;
      }
      store<T, V>(dst, Vec<T, V>::of(v));
    }
    dst += step;
  }
}

// part: [batch * chunks][2][C] sums over the chunk's pixels of g and of g h.
template <typename T, typename TW, int V, int NV, int MODE>
__global__ __launch_bounds__(THREADS) void k_group_norm_grad(const T* __restrict__ dy, const T* __restrict__ x,
                                                             const TW* __restrict__ weight,
                                                             const TW* __restrict__ bias,
                                                             const float2* __restrict__ stats, T* __restrict__ dx,
                                                             float* __restrict__ part, Shape s) {
  extern __shared__ float lds[];  // [rows][W], twice the slice's channel sums
  const Place p = place<V>(s);
  const int tid = int(threadIdx.x), c = p.slice * s.W + p.lane * V;
  const int64_t at = (p.b * s.pixels + p.first + p.row) * s.C + c, step = int64_t(s.rows) * s.C;
  Vec<T, V> hx[NV], hg[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const bool in = p.on && k * s.rows + p.row < p.pixels;
    hx[k] = in ? load<T, V>(x + at + k * step) : Vec<T, V>::zero();
    hg[k] = in ? load<T, V>(dy + at + k * step) : Vec<T, V>::zero();
  }
  const float2 st = stats[p.b * s.groups + p.slice * s.slice_groups + p.group];
  float w[V] = {}, b[V] = {};
  if (p.on) {
    load_f32<TW, V>(weight + c, w);
    load_f32<TW, V>(bias + c, b);
  }
  // h and g of an element
  auto element = [&](float xv, float gv, int e, float& h, float& g) {
    h = (xv - st.x) * st.y;
    g = gv;
    if (s.silu) {
      const float u = fmaf(h, w[e], b[e]), q = sigmoid(u);
      g *= q * (1.f + u * (1.f - q));
    }
  };
  float* channel = lds + s.rows * s.W;  // [2][W]
  if constexpr (MODE != APPLY) {
    float sg[V] = {}, sh[V] = {};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      one_vector();
      if (k * s.rows + p.row < p.pixels) {
        float xv[V], gv[V];
        convert(hx[k], xv);
        convert(hg[k], gv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float h, g;
          element(xv[e], gv[e], e, h, g);
          sg[e] += g;
          sh[e] += g * h;
        }
      }
    }
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if (p.on)
#pragma unroll
        for (int e = 0; e < V; ++e) lds[p.row * s.W + p.lane * V + e] = which ? sh[e] : sg[e];
      __syncthreads();
      for (int k = tid; k < s.W; k += THREADS) {
        float sum = 0.f;
        for (int r = 0; r < s.rows; ++r) sum += lds[r * s.W + k];
        channel[which * s.W + k] = sum;
        part[((p.b * s.chunks + p.chunk) * 2 + which) * s.C + p.slice * s.W + k] = sum;
      }
    }
    if constexpr (MODE == STATS) return;
    __syncthreads();
  } else {
    for (int k = tid; k < 2 * s.W; k += THREADS) {
      const int which = k / s.W, cc = k - which * s.W;
      float sum = 0.f;
      for (int q = 0; q < s.chunks; ++q)
        sum += part[((p.b * s.chunks + q) * 2 + which) * s.C + p.slice * s.W + cc];
      channel[k] = sum;
    }
    __syncthreads();
  }
  // the two group means
  __shared__ float means[2][THREADS];
  const float inv_n = 1.f / (float(s.pixels) * float(s.per_group));
  for (int g = tid >> 6; g < s.slice_groups; g += THREADS / 64) {
    float a = 0.f, d = 0.f;
    for (int k = tid & 63; k < s.per_group; k += 64) {
      const float wk = to_f32(weight[p.slice * s.W + g * s.per_group + k]);
      a += wk * channel[g * s.per_group + k];
      d += wk * channel[s.W + g * s.per_group + k];
    }
    a = wave_sum(a);
    d = wave_sum(d);
    if ((tid & 63) == 0) {
      means[0][g] = a * inv_n;
      means[1][g] = d * inv_n;
    }
  }
  __syncthreads();
  if (!p.on) return;
  const float ma = means[0][p.group], md = means[1][p.group];
  T* dst = dx + at;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    one_vector();
    if (k * s.rows + p.row < p.pixels) {
      float xv[V], gv[V];
      convert(hx[k], xv);
      convert(hg[k], gv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float h, g;
        element(xv[e], gv[e], e, h, g);
        xv[e] = st.y * (rounded_product(w[e], g) - ma - h * md);
      }
      store<T, V>(dst, Vec<T, V>::of(xv));
    }
    dst += step;
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
// The register words a thread holds of a tensor, at most; NV vectors of V elements.
constexpr int WORDS = 64;
struct Plan {
  Shape s;
  int V, NV;
};
// The widest vector of at most 16 bytes that divides a group, so that each lies in one group.
int vec_of(int per_group, int elem) {
  for (int v : {8, 4, 2})
    if (v * elem <= 16 && per_group % v == 0) return v;
  return 1;
}
// arrays: tensors a block holds (1 forward, 2 backward).
Plan plan(int64_t batch, int64_t pixels, int C, int groups, float eps, bool silu, int elem, int arrays) {
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
  // whole groups until a pixel's piece is a line of 128 bytes, as long as the slice fits
  const int word_vec = std::max(1, p.V * elem / 4), most = WORDS / arrays / word_vec;
  auto vectors = [&](int g) {
    const int lanes = g * s.per_group / p.V;
    return lanes > THREADS ? int64_t(1) << 40 : ceil_div(pixels, THREADS / lanes);
  };
  s.slice_groups = 1;
  for (int g = 1; g <= groups; ++g) {
    if (groups % g || g * s.per_group / p.V > THREADS) continue;
    if (g > 1 && (vectors(g) > most || s.slice_groups * s.per_group * elem >= 128)) break;
    s.slice_groups = g;
  }
  s.W = s.slice_groups * s.per_group;
  s.lanes = s.W / p.V;
  s.rows = THREADS / s.lanes;
  const int64_t need = vectors(s.slice_groups);
  s.chunks = int(ceil_div(need, most));
  s.chunk_pixels = ceil_div(pixels, s.chunks);
  p.NV = int(ceil_div(s.chunk_pixels, s.rows));
  return p;
}

int check_sizes(const char* what, int64_t batch, int64_t pixels, int C, int groups, int act, int dtype, int w_dtype) {
  if (batch < 0 || pixels < 0 || C <= 0 || (pixels && batch > SIHC_MAX_TOKENS / pixels))
    return fail(SIHC_ERR_INVALID, "%s: bad sizes", what);
  if (groups <= 0 || C % groups) return fail(SIHC_ERR_INVALID, "%s: %d channels are not %d groups", what, C, groups);
  if (C / groups / vec_of(C / groups, dtype == SIHC_DTYPE_F32 ? 4 : 2) > THREADS)
    return fail(SIHC_ERR_INVALID, "%s: groups of %d channels are too wide", what, C / groups);
  if (act != SIHC_ACT_NONE && act != SIHC_ACT_SILU) return fail(SIHC_ERR_INVALID, "%s: bad activation %d", what, act);
  if (!valid_dtype(dtype) || !valid_dtype(w_dtype)) return fail(SIHC_ERR_INVALID, "%s: bad dtype", what);
  if (w_dtype != dtype && w_dtype != SIHC_DTYPE_F32)
    return fail(SIHC_ERR_INVALID, "%s: weights must be fp32 or share the input's type", what);
  return SIHC_OK;
}
int elem_size(int dtype) { return dtype == SIHC_DTYPE_F32 ? 4 : 2; }

// Calls f<T, TW, V, NV> with NV the smallest compiled count of at least p.NV vectors.
template <int ARRAYS, typename F>
int by_plan(const Plan& p, int dtype, int w_dtype, F&& f) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto with = [&](auto tw, auto v) {
      constexpr int V = decltype(v)::value, words = V * int(sizeof(T)) / 4 > 0 ? V * int(sizeof(T)) / 4 : 1;
      int rc = SIHC_ERR_INVALID;
      auto attempt = [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        if constexpr (NV * words * ARRAYS <= WORDS) {
          if (p.NV <= NV) {
            rc = f(t, tw, v, nv);
            return true;
          }
        }
        return false;
      };
      if (attempt(IC<1>{}) || attempt(IC<2>{}) || attempt(IC<4>{}) || attempt(IC<8>{}) || attempt(IC<16>{}) ||
          attempt(IC<32>{}) || attempt(IC<64>{}))
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
  if (batch <= 0 || pixels <= 0 || channels <= 0 || groups <= 0 || channels % groups || !valid_dtype(dtype)) return 0;
  const Plan p = plan(batch, pixels, channels, groups, 0.f, false, elem_size(dtype), 1);
  return p.s.chunks > 1 ? size_t(batch) * size_t(p.s.chunks) * size_t(groups) * 8 : 0;
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
  const Plan p = plan(batch, pixels, channels, groups, eps, act == SIHC_ACT_SILU, elem_size(dtype), 1);
  const int64_t blocks = batch * (groups / p.s.slice_groups) * p.s.chunks;
  if (blocks > 0x7fffffff) return fail(SIHC_ERR_INVALID, "%s: tensor too large", what);
  const dim3 grid(static_cast<unsigned>(blocks));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_plan<1>(p, dtype, w_dtype, [&](auto t, auto tw, auto v, auto nv) {
    using T = decltype(t);
    using TW = decltype(tw);
    constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
    auto launch = [&](auto mode) {
      hipLaunchKernelGGL((k_group_norm<T, TW, V, NV, decltype(mode)::value>), grid, dim3(THREADS), 0, st,
                         static_cast<const T*>(x), static_cast<const TW*>(weight), static_cast<const TW*>(bias),
                         static_cast<T*>(y), reinterpret_cast<float2*>(stats), static_cast<float2*>(workspace), p.s);
    };
    if (p.s.chunks == 1) {
      launch(IC<WHOLE>{});
    } else {
      launch(IC<STATS>{});
      launch(IC<APPLY>{});
    }
    return check_launch(what);
  });
}

size_t sihc_group_norm_backward_workspace_size(int64_t batch, int64_t pixels, int channels, int groups, int dtype) {
  if (batch <= 0 || pixels <= 0 || channels <= 0 || groups <= 0 || channels % groups || !valid_dtype(dtype)) return 0;
  const Plan p = plan(batch, pixels, channels, groups, 0.f, false, elem_size(dtype), 2);
  return size_t(batch) * size_t(p.s.chunks) * 2 * size_t(channels) * 4;
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
    const Plan p = plan(batch, pixels, channels, groups, 0.f, act == SIHC_ACT_SILU, elem_size(dtype), 2);
    const int64_t blocks = batch * (groups / p.s.slice_groups) * p.s.chunks;
    if (blocks > 0x7fffffff) return fail(SIHC_ERR_INVALID, "%s: tensor too large", what);
    parts = batch * p.s.chunks;
    const dim3 grid(static_cast<unsigned>(blocks));
    const unsigned lds = unsigned(p.s.rows + 2) * unsigned(p.s.W) * 4u;
    const int rc = by_plan<2>(p, dtype, w_dtype, [&](auto t, auto tw, auto v, auto nv) {
      using T = decltype(t);
      using TW = decltype(tw);
      constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
      auto launch = [&](auto mode) {
        hipLaunchKernelGGL((k_group_norm_grad<T, TW, V, NV, decltype(mode)::value>), grid, dim3(THREADS), lds, st,
                           static_cast<const T*>(grad), static_cast<const T*>(x), static_cast<const TW*>(weight),
                           static_cast<const TW*>(bias), reinterpret_cast<const float2*>(stats),
                           static_cast<T*>(grad_x), static_cast<float*>(workspace), p.s);
      };
      if (p.s.chunks == 1) {
        launch(IC<WHOLE>{});
      } else {
        launch(IC<STATS>{});
        launch(IC<APPLY>{});
      }
      return check_launch(what);
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

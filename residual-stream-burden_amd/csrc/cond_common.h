// What the conditioning kernels (embedding.hip, group_norm.hip, cross_attention.hip) and the body kernels
// (linear.hip, head_norm.hip, dropout.hip) share:
// element types, unaligned row vectors, block order and the host's error reporting.
#ifndef SIHC_COND_COMMON_H
#define SIHC_COND_COMMON_H

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "sihc_hip.h"

// Stores the message sihc_last_error() returns on this thread; defined in sihc_kernels.hip.
__attribute__((visibility("hidden"))) int sihc_record_error(int code, const char* message);

namespace sihc_cond {

template <int N>
using IC = std::integral_constant<int, N>;

struct bf16 {  // bfloat16 storage (the upper 16 bits of an IEEE fp32)
  uint16_t bits;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __uint_as_float(uint32_t(v.bits) << 16); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) {  // to nearest, ties to even
  return bf16{__builtin_bit_cast(uint16_t, static_cast<__bf16>(v))};
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = u32x4; };
template <> struct Raw<8> { using type = u32x2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// V adjacent elements of T in the words of one load, which promises only the alignment of the
// element: gfx950 takes global accesses at any byte address, so rows may start anywhere.
template <typename T, int V>
struct Vec {
  static constexpr int BYTES = V * int(sizeof(T));
  using R = typename Raw<BYTES>::type;
  R raw;
  __device__ __forceinline__ void to(float* o) const {
    T e[V];
    __builtin_memcpy(e, &raw, BYTES);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f32(e[i]);
  }
  __device__ __forceinline__ static Vec of(const float* v) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(v[i]);
    Vec out;
    __builtin_memcpy(&out.raw, e, BYTES);
    return out;
  }
  __device__ __forceinline__ static Vec zero() {
    Vec out;
    __builtin_memset(&out.raw, 0, BYTES);
    return out;
  }
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  using R = typename Vec<T, V>::R;
  typedef R RU __attribute__((aligned(sizeof(T))));
  Vec<T, V> v;
  v.raw = *reinterpret_cast<const RU*>(p);
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& v) {
  using R = typename Vec<T, V>::R;
  typedef R RU __attribute__((aligned(sizeof(T))));
  *reinterpret_cast<RU*>(p) = v.raw;
}

// V adjacent elements as fp32, in loads of at most 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* p, float* o) {
  constexpr int PIECE = V * int(sizeof(T)) > 16 ? 16 / int(sizeof(T)) : V;
#pragma unroll
  for (int k = 0; k < V; k += PIECE) load<T, PIECE>(p + k).to(o + k);
}

// Sum over a wave, in every lane: within rows of 16 lanes by data-parallel moves (quad permutations
// and mirrors), then across the rows.
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += moved<0xb1>(v);   // quad_perm [1,0,3,2]
  v += moved<0x4e>(v);   // quad_perm [2,3,0,1]
  v += moved<0x141>(v);  // row_half_mirror
  v += moved<0x140>(v);  // row_mirror
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Logical index of this workgroup among n: the hardware deals workgroups to the 8 XCDs in turn, and
// this gives each XCD a contiguous run, so that neighbours meet in its L2.
__device__ __forceinline__ int xcd_block(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7, i = b >> 3;
  return x < r ? x * (q + 1) + i : r * (q + 1) + (x - r) * q + i;
}

// ---------------------------------------------------------------------------------- host
inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return sihc_record_error(code, buf);
}
inline int check_launch(const char* what) {
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(SIHC_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(err));
  return SIHC_OK;
}
inline bool valid_dtype(int dtype) { return dtype == SIHC_DTYPE_F32 || dtype == SIHC_DTYPE_BF16; }
inline bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Threads of a launch: HIP takes fewer than 2^32 in a dimension (a block of 256 less, for counts rounded up to one).
constexpr int64_t MOST_LAUNCHED = (int64_t(1) << 32) - 256;
// Calls f with the element type of a dtype code.
template <typename F>
int by_dtype(int dtype, F&& f) {
  return dtype == SIHC_DTYPE_F32 ? f(float{}) : f(bf16{});
}

}  // namespace sihc_cond
#endif

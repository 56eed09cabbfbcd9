// What the attention kernels share: matrix instructions by type, exchanges between lane rows, transposed reads of LDS.
#pragma once
#include "fr_common.h"

namespace fr {
namespace {

template <typename T> struct Attn;
template <> struct Attn<bf16_t> {
  typedef bf16x4 vec4;
  typedef bf16x8 vec8;
  static constexpr float kRaise = 0.f;
  static __device__ __forceinline__ f32x4 mma16(vec8 a, vec8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Attn<f16_t> {
  typedef f16x4 vec4;
  typedef f16x8 vec8;
  static constexpr float kRaise = 7.f;
  static __device__ __forceinline__ f32x4 mma16(vec8 a, vec8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

typedef short i16x4 __attribute__((ext_vector_type(4)));

// A group of 16 lanes reads a 4 x 16 matrix of 16-bit elements, lane l the four from column 4 (l % 4) of row (l / 4) % 4 at `at`; lane l gets
// column l % 16, rows 0 .. 3.
template <typename T>
__device__ __forceinline__ typename Attn<T>::vec4 read_transposed(const T* at) {
  const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)at);
  return __builtin_bit_cast(typename Attn<T>::vec4, v);
}

template <typename V4>
__device__ __forceinline__ auto join8(V4 a, V4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

#if defined(__HIP_DEVICE_COMPILE__)  // buffer resources exist in the device pass only
// `bytes` from a pointer that all lanes share: loads behind them are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform_buffer(const void* p, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const uint64_t there = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32))) << 32 |
                         static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(there), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}
#endif

// Over the lanes that differ in bit 4 (5) of their number: of the two values, in both lanes.
__device__ __forceinline__ float max_over_16(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float max_over_32(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float sum_over_16(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}
__device__ __forceinline__ float sum_over_32(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// Of the lanes up to this one; over the wavefront, in every lane.
__device__ __forceinline__ int sum_up_to(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  const int lane = threadIdx.x & 63;
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31), r2 = __builtin_amdgcn_readlane(v, 47);
  return v + (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
}
__device__ __forceinline__ int sum_of_all(int v) {
  v += partner_i32<1>(v);
  v += partner_i32<2>(v);
  v += partner_i32<4>(v);
  v += partner_i32<8>(v);
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) + (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}

// The lengths of up to kHeldLengths sequences stay in a wavefront's lanes; of more, a launch of one workgroup writes what lies in front of each (prefix_of) to the
// workspace first, where place_in finds a place again.  us, with that launch / every wavefront going over all lengths: packed, 300 sequences of 8 rows 23 / 27, 1100 of
// 64 205 / 609, 4000 of 20 306 / 2492; paged, 300 of up to 2000 keys 143 / 138, 1100 of up to 600 190 / 199, 4000 of up to 600 549 / 681.
constexpr int kHeldLengths = 256, kPlanThreads = 1024;

// to[i] = the sum of value(0) .. value(i - 1), to[count] of all; by one workgroup of kPlanThreads.
template <typename F>
__device__ __forceinline__ void prefix_of(int count, F value, int* to) {
  __shared__ int of_wave[kPlanThreads / kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int before = 0;
  for (int b0 = 0; b0 < count; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x, mine = b < count ? value(b) : 0, sum = sum_up_to(mine);
    if (lane == 63) of_wave[wave] = sum;
    __syncthreads();
    int front = before, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / kWave; ++w) front += w < wave ? of_wave[w] : 0, all += of_wave[w];
    if (b < count) to[b] = front + sum - mine;
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) to[count] = before;
}
// The i with to[i] <= place < to[i + 1], -1: none.
__device__ __forceinline__ int place_in(const int* to, int count, int place) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (to[mid] <= place) lo = mid;
    else hi = mid;
  }
  return count > 0 && to[lo] <= place && place < to[lo + 1] ? lo : -1;
}

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }

constexpr float kLog2e = 1.4426950408889634f;

// A term is exp2((score - maximum) * scale + kRaise), scale with log2(e) in it.  A running maximum that lags behind the scores by up to kLag factors of 2 leaves the results
// as they are - every term and the sum carry the same 2^(lag + kRaise) - and the output rows need not be rescaled for each new maximum.  The terms, rounded to the inputs' type, are the
// second product's operand, and the sum is theirs, in fp32.  bf16 has fp32's range.  In fp16 terms may reach 2^15, which kRaise makes use of: with the largest term at 2^7 or above,
// those from 2^-21 of it on keep 11 bits, and smaller ones, subnormal, are off by 2^-32 of it at most.  Without the raise that was 2^-25: of 131071 keys 25 octaves below
// another nothing was left, 0.4 % of the result.
// The difference comes first, or the maximum's product is known not to be large: score * scale - maximum * scale is off by 2^-24 of the products, which
// makes a term of any size of scores beyond 2^25 factors of 2.
constexpr float kLag = 8.f;

// Joins the parts of a head's keys: rows of DP sums, the softmax's maxima and sums, each `pitch` floats from part to part.  The
// workgroup's 256 threads are groups of DP / 4, four dimensions to a thread.  Not wide: a head to a group.  wide: one head for all groups, which share its
// parts - for few heads, where a part after the other is a round trip to memory each (one row of 32 heads, 31 parts: 21 -> 5 us).
template <int DP>
struct JoinShape {
  static constexpr int kThreads = 256, kLanes = DP / 4, kGroups = kThreads / kLanes;
  static int64_t blocks(int64_t heads, bool wide) { return wide ? heads : (heads + kGroups - 1) / kGroups; }
};
template <typename T, int DP>
__device__ __forceinline__ void join_parts(bool wide, bool live, int parts, const float* rows, int64_t row_pitch, const float* tops, const float* sums,
                                           int64_t pitch, float scale, T* out, int dim) {
  typedef JoinShape<DP> S;
  __shared__ float joined[S::kGroups][DP];
  __shared__ float weight_of[S::kGroups];
  const int group = threadIdx.x / S::kLanes, d = threadIdx.x % S::kLanes * 4;
  live = live && group < S::kGroups;
  float top = -INFINITY, weight = 0.f;
  if (wide) {
    for (int p = threadIdx.x & 63; p < parts; p += kWave) top = fmaxf(top, tops[p * pitch]);
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, kWave));
  } else if (live) {
#pragma unroll 8
    for (int p = 0; p < parts; ++p) top = fmaxf(top, tops[p * pitch]);
  }
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (live) {
#pragma unroll 8
    for (int p = wide ? group : 0; p < parts; p += wide ? S::kGroups : 1) {
      const float t = tops[p * pitch], by = t == -INFINITY ? 0.f : exp2_of((t - top) * scale);
      weight += by * sums[p * pitch];
      x += *reinterpret_cast<const f32x4*>(rows + p * row_pitch + d) * by;
    }
  }
  if (!wide) {
    if (live && d < dim) {
      typename Attn<T>::vec4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(weight == 0.f ? 0.f : x[e] / weight);
      *reinterpret_cast<typename Attn<T>::vec4*>(out + d) = y;
    }
    return;
  }
  if (live) {
    *reinterpret_cast<f32x4*>(&joined[group][d]) = x;
    if (d == 0) weight_of[group] = weight;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < dim; i += S::kThreads) {
    float sum = 0.f, total = 0.f;
#pragma unroll
    for (int r = 0; r < S::kGroups; ++r) sum += joined[r][i], total += weight_of[r];
    out[i] = static_cast<T>(total == 0.f ? 0.f : sum / total);  // no key at all: zeros
  }
}

}  // namespace
}  // namespace fr

// Rotary positions of queries and keys, and the keys' and values' way into a paged cache.
//
// Pair i of the first `turned` dimensions of a head, at position p, is turned by the angle p * freq[i]:
//   (a, b) -> (a cos - b sin, b cos + a sin) * factor,  pairs (i, i + turned / 2) or, interleaved, (2 i, 2 i + 1); the rest of a head stays.
// A frequency comes as turns per position in units of 2^-64 turn, rounded: position * frequency in wrapping 64-bit integers is the angle's part
// within a turn, off by |position| * 2^-65 turn at most (2^-25, what the next rounding takes, at 2^40), where a 32-bit product of position and radians is off by
// half a radian at 10^7.  The part, signed, is rounded to 32 bits (1.9e-7 radian at most) and goes to sincospi.
//
// Bound by memory: everything is read once and written once (keys twice with a cache): 8192 tokens of 32 and 8 heads of 128 dimensions into a cache 39.6 us, 5.5 TB/s.  The
// angles of a token are computed once, by one thread each, and shared by its heads through LDS.  Rows that 16-byte accesses cannot read go element by element.
#include "fr_memory.h"

namespace fr {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 4;     // of a workgroup, at most
constexpr int kRotMaxPairs = 256;

template <typename T, int VEC>
struct RotVec {
  typedef T type __attribute__((ext_vector_type(VEC)));
};
template <typename T>
struct RotVec<T, 1> {
  typedef T type;
};

// `tokens` tokens to a workgroup.  Items of a token: per head of q and k, turned / 2 / VEC pieces of VEC pairs and
// (dim - turned) / VEC pieces that stay; per head of v dim / VEC pieces.
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(fr_rotary_args a, int tokens) {
  typedef typename RotVec<T, VEC>::type vec;
  __shared__ float2 turn[kRotTokens][kRotMaxPairs];
  __shared__ int64_t cache_at[kRotTokens][2];  // of k and v, -1: not kept
  const int tid = threadIdx.x, pairs = static_cast<int>(a.turned / 2), dim = static_cast<int>(a.dim);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens;
  const int live = static_cast<int>(a.T - first < tokens ? a.T - first : tokens);
  for (int i = tid; i < live * pairs; i += kRotThreads) {
    const int t = i / pairs, p = i - t * pairs;
    const uint64_t at = a.positions_i64 ? static_cast<uint64_t>(reinterpret_cast<const int64_t*>(a.positions)[first + t])
                                        : static_cast<uint64_t>(static_cast<int64_t>(reinterpret_cast<const int32_t*>(a.positions)[first + t]));
    const int64_t part = static_cast<int64_t>(at * reinterpret_cast<const uint64_t*>(a.turns)[p]);  // of a turn, in 2^-64
    float s, c;
    sincospif(static_cast<float>(part) * 0x1p-63f, &s, &c);
    turn[t][p] = make_float2(c * static_cast<float>(a.factor), s * static_cast<float>(a.factor));
  }
  if (tid < live) {
    int64_t k_at = -1, v_at = -1;
    if (a.slots) {
      const int64_t slot = a.slots_i64 ? reinterpret_cast<const int64_t*>(a.slots)[first + tid]
                                       : static_cast<int64_t>(reinterpret_cast<const int32_t*>(a.slots)[first + tid]);
      if (slot >= 0 && slot < a.pages * a.page_size) {
        const int64_t page = slot / a.page_size, in = slot - page * a.page_size;
        k_at = page * a.k_cache_page + in * a.k_cache_slot;
        v_at = page * a.v_cache_page + in * a.v_cache_slot;
      }
    }
    cache_at[tid][0] = k_at;
    cache_at[tid][1] = v_at;
  }
  __syncthreads();
  const int turning = pairs / VEC, staying = (dim - static_cast<int>(a.turned)) / VEC, whole = dim / VEC;
  const int per_head = turning + staying, heads = static_cast<int>(a.heads), kv_heads = static_cast<int>(a.kv_heads);
  const int of_qk = (heads + kv_heads) * per_head, items = of_qk + (a.slots ? kv_heads * whole : 0);
  for (int i = tid; i < live * items; i += kRotThreads) {
    const int t = i / items, j = i - t * items;
    const int64_t token = first + t;
    if (j >= of_qk) {
      const int h = (j - of_qk) / whole, at = (j - of_qk - h * whole) * VEC;
      if (cache_at[t][1] < 0) continue;
      const T* from = reinterpret_cast<const T*>(a.v) + token * a.v_token + h * a.v_head + at;
      T* to = reinterpret_cast<T*>(a.v_cache) + cache_at[t][1] + h * a.v_cache_head + at;
      *reinterpret_cast<vec*>(to) = *reinterpret_cast<const vec*>(from);
      continue;
    }
    const int head = j / per_head, piece = j - head * per_head;
    const bool key = head >= heads;
    const int h = key ? head - heads : head;
    const T* from = key ? reinterpret_cast<const T*>(a.k) + token * a.k_token + h * a.k_head : reinterpret_cast<const T*>(a.q) + token * a.q_token + h * a.q_head;
    T* to = key ? reinterpret_cast<T*>(a.k_out) + token * a.k_out_token + h * a.k_out_head
                : reinterpret_cast<T*>(a.q_out) + token * a.q_out_token + h * a.q_out_head;
    T* kept = key && cache_at[t][0] >= 0 ? reinterpret_cast<T*>(a.k_cache) + cache_at[t][0] + h * a.k_cache_head : nullptr;
    if (piece >= turning) {
      const int at = static_cast<int>(a.turned) + (piece - turning) * VEC;
      if (to == from && !kept) continue;
      const vec v = *reinterpret_cast<const vec*>(from + at);
      if (to != from) *reinterpret_cast<vec*>(to + at) = v;
      if (kept) *reinterpret_cast<vec*>(kept + at) = v;
      continue;
    }
    const int at0 = INTERLEAVED ? piece * 2 * VEC : piece * VEC, at1 = INTERLEAVED ? at0 + VEC : at0 + pairs;
    const vec v0 = *reinterpret_cast<const vec*>(from + at0), v1 = *reinterpret_cast<const vec*>(from + at1);
    float x[2 * VEC], y[2 * VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (VEC == 1) x[0] = static_cast<float>(v0), x[1] = static_cast<float>(v1);
      else x[e] = static_cast<float>(v0[e]), x[VEC + e] = static_cast<float>(v1[e]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int p0 = INTERLEAVED ? 2 * e : e, p1 = INTERLEAVED ? p0 + 1 : VEC + e;
      const float2 w = turn[t][piece * VEC + e];
      y[p0] = __builtin_fmaf(x[p0], w.x, -(x[p1] * w.y));
      y[p1] = __builtin_fmaf(x[p1], w.x, x[p0] * w.y);
    }
    vec o0, o1;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (VEC == 1) o0 = static_cast<T>(y[0]), o1 = static_cast<T>(y[1]);
      else o0[e] = static_cast<T>(y[e]), o1[e] = static_cast<T>(y[VEC + e]);
    }
    *reinterpret_cast<vec*>(to + at0) = o0;
    *reinterpret_cast<vec*>(to + at1) = o1;
    if (kept) {
      *reinterpret_cast<vec*>(kept + at0) = o0;
      *reinterpret_cast<vec*>(kept + at1) = o1;
    }
  }
}

// The call on its tokens from the t-th on.
fr_rotary_args tokens_from(fr_rotary_args a, int64_t t) {
  auto on = [](const void* p, int64_t bytes) { return p ? static_cast<const char*>(p) + bytes : nullptr; };
  auto on_out = [](void* p, int64_t bytes) { return p ? static_cast<char*>(p) + bytes : nullptr; };
  a.q = on(a.q, t * a.q_token * 2), a.k = on(a.k, t * a.k_token * 2), a.v = on(a.v, t * a.v_token * 2);
  a.q_out = on_out(a.q_out, t * a.q_out_token * 2), a.k_out = on_out(a.k_out, t * a.k_out_token * 2);
  a.positions = on(a.positions, t * (a.positions_i64 ? 8 : 4)), a.slots = on(a.slots, t * (a.slots_i64 ? 8 : 4));
  a.T -= t;
  return a;
}

template <typename T>
int launch_rotary(const fr_rotary_args& a, bool wide, hipStream_t st) {
  // As many tokens as give every thread an item, where there are tokens enough for every CU: 8192 tokens of 12 and 4 heads of 64 dimensions 14.5 us one by one,
  // 11.7 four together; 32 and 8 heads of 128, which have 448 items a token, 39.6 and 43.5; 64 tokens 4.3 and 7.1.
  const int64_t vec = wide ? 8 : 1, items = ((a.heads + a.kv_heads) * (a.dim - a.turned / 2) + (a.slots ? a.kv_heads * a.dim : 0)) / vec;
  const int64_t fill = items < kRotThreads ? kRotThreads / (items > 0 ? items : 1) : 1;
  const int tokens = a.T < 2048 ? 1 : static_cast<int>(fill < kRotTokens ? fill : kRotTokens);
  // More tokens than the workgroups of a launch take: one launch after the other.
  const int64_t most = kMostBlocks256 * tokens;
  for (int64_t t = 0; t < a.T; t += most) {
    const fr_rotary_args b = t == 0 ? a : tokens_from(a, t);
    const int64_t count = b.T < most ? b.T : most;
    const dim3 grid(static_cast<unsigned>(ceil_div(count, tokens))), block(kRotThreads);
    if (wide && a.interleaved) hipLaunchKernelGGL((rotary_kernel<T, 8, true>), grid, block, 0, st, b, tokens);
    else if (wide) hipLaunchKernelGGL((rotary_kernel<T, 8, false>), grid, block, 0, st, b, tokens);
    else if (a.interleaved) hipLaunchKernelGGL((rotary_kernel<T, 1, true>), grid, block, 0, st, b, tokens);
    else hipLaunchKernelGGL((rotary_kernel<T, 1, false>), grid, block, 0, st, b, tokens);
    const int rc = check_launch("rotary_kernel");
    if (rc != FR_OK) return rc;
  }
  return FR_OK;
}

// Rows of heads that 16-byte accesses can read: address and strides.
bool rot_wide(const void* p, int64_t s0, int64_t s1, int64_t s2 = 0) {
  return aligned16(p) && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0;
}

// Results that lie where another workgroup, or another thread, still reads or writes: all but queries and keys turned in place.
int check_rotary_memory(const fr_rotary_args& a) {
  const Box in[3] = {Box(a.q, a.T, a.q_token, a.heads, a.q_head, a.dim), Box(a.k, a.T, a.k_token, a.kv_heads, a.k_head, a.dim),
                     Box(a.v, a.slots ? a.T : 0, a.v_token, a.kv_heads, a.v_head, a.dim)};
  const int64_t pages = a.slots ? a.pages : 0;
  const Box out[4] = {Box(a.q_out, a.T, a.q_out_token, a.heads, a.q_out_head, a.dim), Box(a.k_out, a.T, a.k_out_token, a.kv_heads, a.k_out_head, a.dim),
                      Box(a.k_cache, pages, a.k_cache_page, a.page_size, a.k_cache_slot, a.kv_heads, a.k_cache_head, a.dim, 1),
                      Box(a.v_cache, pages, a.v_cache_page, a.page_size, a.v_cache_slot, a.kv_heads, a.v_cache_head, a.dim, 1)};
  static const char* const in_name[3] = {"q", "k", "v"};
  static const char* const out_name[4] = {"turned q", "turned k", "k_cache", "v_cache"};
  for (int i = 0; i < 4; ++i) {
    FR_REQUIRE(!meets_itself(out[i]), FR_E_SHAPE, "fr_rotary: %s: places that share memory", out_name[i]);
    for (int j = 0; j < 3; ++j)
      FR_REQUIRE((i == j && is_same(out[i], in[j])) || !meets(out[i], in[j]), FR_E_SHAPE, "fr_rotary: %s and %s share memory", out_name[i], in_name[j]);
    for (int j = 0; j < i; ++j) FR_REQUIRE(!meets(out[i], out[j]), FR_E_SHAPE, "fr_rotary: %s and %s share memory", out_name[i], out_name[j]);
  }
  return FR_OK;
}

}  // namespace
}  // namespace fr

extern "C" int fr_rotary(const fr_rotary_args* args, void* stream) {
  using namespace fr;
  FR_REQUIRE(args, FR_E_NULL, "fr_rotary: null pointer");
  const fr_rotary_args& a = *args;
  FR_REQUIRE(a.T >= 0 && a.T <= 0x7fffffff, FR_E_SHAPE, "fr_rotary: %lld tokens", (long long)a.T);
  FR_REQUIRE(a.heads >= 1 && a.kv_heads >= 1 && a.heads <= 4096 && a.kv_heads <= 4096, FR_E_SHAPE, "fr_rotary: %lld and %lld heads: 1 to 4096",
             (long long)a.heads, (long long)a.kv_heads);
  FR_REQUIRE(a.dim >= 1 && a.dim <= 1024, FR_E_SHAPE, "fr_rotary: head size %lld outside [1, 1024]", (long long)a.dim);
  FR_REQUIRE(a.turned >= 0 && a.turned % 2 == 0 && a.turned <= a.dim && a.turned <= 2 * kRotMaxPairs, FR_E_SHAPE,
             "fr_rotary: %lld turned dimensions of %lld: an even number, at most %d", (long long)a.turned, (long long)a.dim, 2 * kRotMaxPairs);
  FR_REQUIRE(a.dtype == FR_F16 || a.dtype == FR_BF16, FR_E_DTYPE, "fr_rotary: dtype %lld not in {f16, bf16}", (long long)a.dtype);
  FR_REQUIRE(!a.slots || (a.pages >= 0 && a.page_size >= 1 && a.page_size <= 0x7fffffff && a.pages <= 0x7fffffff), FR_E_SHAPE,
             "fr_rotary: %lld pages of %lld", (long long)a.pages, (long long)a.page_size);
  if (a.T == 0) return FR_OK;
  FR_REQUIRE(a.q && a.k && a.q_out && a.k_out && a.positions && (a.turns || a.turned == 0), FR_E_NULL, "fr_rotary: null pointer");
  FR_REQUIRE(!a.slots || (a.v && (a.pages == 0 || (a.k_cache && a.v_cache))), FR_E_NULL, "fr_rotary: null pointer");
  bool wide = a.dim % 8 == 0 && a.turned % 16 == 0 && rot_wide(a.q, a.q_token, a.q_head) && rot_wide(a.k, a.k_token, a.k_head) &&
              rot_wide(a.q_out, a.q_out_token, a.q_out_head) && rot_wide(a.k_out, a.k_out_token, a.k_out_head);
  if (a.slots)
    wide = wide && rot_wide(a.v, a.v_token, a.v_head) && rot_wide(a.k_cache, a.k_cache_page, a.k_cache_slot, a.k_cache_head) &&
           rot_wide(a.v_cache, a.v_cache_page, a.v_cache_slot, a.v_cache_head);
  const int rc = check_rotary_memory(a);
  if (rc != FR_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FR_BF16 ? launch_rotary<bf16_t>(a, wide, st) : launch_rotary<f16_t>(a, wide, st);
}

// Routing with scores, a bias for balance and groups of experts: one wavefront per token.
//
//   score   s = softmax(l) or sigmoid(l) over the E logits of a token
//   choice  c = s + bias, or l itself where there is no bias (both scores rise with the logit)
//   group   E / groups consecutive experts; its worth is its largest c, with a bias the sum of its two largest
//   result  the topk experts of largest c in the kept groups of largest worth; weights s (/ their sum) * scale
//
// Ties go to the lower index.  With a bias the order depends on sums of rounded scores, so scores and choices are 64-bit floats there: 32 bits
// would swap experts whose choices differ by less than a rounding, which happens every few hundred tokens of 256 experts.  Without one the
// logits themselves decide and 32 bits lose nothing.
#include "gating_core.h"

namespace fr {
namespace {

constexpr int kGroupWaves = 4;  // tokens of a workgroup at a time

// Order-preserving keys, every real value above 0, which serves as "not a candidate".
struct Key32 {
  unsigned hi;
  static constexpr bool kWide = false;
};
struct Key64 {
  unsigned hi, lo;
  static constexpr bool kWide = true;
};
__device__ __forceinline__ Key32 key_of(float v) { return Key32{float_key(v)}; }
__device__ __forceinline__ Key64 key_of(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  const uint64_t k = (b >> 63) ? ~b : (b | 0x8000000000000000ull);
  return Key64{static_cast<unsigned>(k >> 32), static_cast<unsigned>(k)};
}
__device__ __forceinline__ bool above(Key32 a, Key32 b) { return a.hi > b.hi; }
__device__ __forceinline__ bool above(Key64 a, Key64 b) { return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo); }

// Largest value and sum over a wavefront, in every lane.
__device__ __forceinline__ double shfl_xor_f64(double v, int s) { return __shfl_xor(v, s, kWave); }
__device__ __forceinline__ float wave_max(float v) { return group_max<64>(v); }
__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) v = fmax(v, shfl_xor_f64(v, s));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) { return group_sum<64>(v); }
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) v += shfl_xor_f64(v, s);
  return v;
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ double lane_of(double v, int lane) { return __shfl(v, lane, kWave); }

// A NaN is the lowest value: no comparison holds for it, and an expert that has one is chosen last.  (+ 0: -0 and +0 are the same value.)
template <typename S>
__device__ __forceinline__ S ordered(S v) { return v == v ? v + S(0) : -static_cast<S>(INFINITY); }

// S: float without a bias, double with one.  Expert of lane l's value i: l + 64 i.
template <typename T, typename S, int VPL>
__global__ __launch_bounds__(kGroupWaves * kWave) void gating_grouped_kernel(const T* __restrict__ logits, int64_t M, int E, int64_t ld,
                                                                             const float* __restrict__ bias, int groups, int kept, int topk,
                                                                             int sigmoid, int renorm, float scale, float* __restrict__ w_out,
                                                                             int32_t* __restrict__ id_out) {
  typedef decltype(key_of(S(0))) Key;
  __shared__ S choice_of[kGroupWaves][VPL * kWave];
  __shared__ S worth_of[kGroupWaves][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int size = E / groups;
  int per = kWave;  // lanes that share a group: a power of two, groups * per <= 64
  while (per * groups > kWave) per >>= 1;
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * kGroupWaves + wave; token < M; token += static_cast<int64_t>(gridDim.x) * kGroupWaves) {
    const T* row = logits + token * ld;
    S x[VPL], score[VPL];
    Key key[VPL];
    S top = -static_cast<S>(INFINITY);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 64 * i;
      x[i] = e < E ? ordered(static_cast<S>(static_cast<float>(row[e]))) : -static_cast<S>(INFINITY);
      top = x[i] > top ? x[i] : top;
    }
    // Scores of all experts where the order or the whole softmax's sum needs them; without a bias those of the chosen ones follow from
    // their logits below.  The largest logits' terms are 1, infinite ones among them: they share the row, and so do all experts of a row of
    // nothing but -infinity.
    S all = 0;
    if (!sigmoid) top = wave_max(top);
    if (sizeof(S) == 8 && sigmoid) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) score[i] = S(1) / (S(1) + exp(-x[i]));
    } else if (!sigmoid && (sizeof(S) == 8 || !renorm)) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        score[i] = lane + 64 * i >= E ? S(0) : (x[i] == top ? S(1) : exp(x[i] - top));
        all += score[i];
      }
      all = wave_sum(all);
#pragma unroll
      for (int i = 0; i < VPL; ++i) score[i] /= all;
    }
    S choice[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 64 * i;
      choice[i] = x[i];
      if constexpr (sizeof(S) == 8) choice[i] = e < E ? ordered(score[i] + static_cast<S>(bias[e])) : x[i];
      key[i] = key_of(choice[i]);
      if (e >= E) key[i] = Key{};
    }
    if (kept < groups) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) choice_of[wave][lane + 64 * i] = choice[i];
      __builtin_amdgcn_wave_barrier();
      const int g = lane / per;
      S first = -static_cast<S>(INFINITY), second = first;
      if (g < groups)
        for (int j = lane % per; j < size; j += per) {
          const S c = choice_of[wave][g * size + j];
          second = c > first ? first : (c > second ? c : second);
          first = c > first ? c : first;
        }
      for (int s = 1; s < per; s <<= 1) {
        const S f = __shfl_xor(first, s, kWave), n = __shfl_xor(second, s, kWave);
        const S low = f > first ? first : f, high = f > first ? f : first, next = n > second ? n : second;
        first = high;
        second = low > next ? low : next;
      }
      S worth = first;
      if constexpr (sizeof(S) == 8) worth = size > 1 ? ordered(first + second) : first;
      if (g < groups && lane % per == 0) worth_of[wave][g] = worth;
      __builtin_amdgcn_wave_barrier();
      int ahead = 0;
      for (int o = 0; o < groups; ++o) {
        const S w = worth_of[wave][o];
        ahead += (w > worth || (w == worth && o < g)) ? 1 : 0;
      }
      const uint64_t keep = __ballot(g < groups && ahead < kept);
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = lane + 64 * i;
        if (e < E && !((keep >> (e / size * per)) & 1)) key[i] = Key{};
      }
      __builtin_amdgcn_wave_barrier();  // the next token's choices come after this one's have been read
    }
    S mine = 0;  // lane j: of choice j the score, without a bias the logit, and the expert
    int mine_id = 0;
    for (int j = 0; j < topk; ++j) {
      Key best = key[0];
      S s = sizeof(S) == 8 ? score[0] : x[0];
      int slot = 0;
#pragma unroll
      for (int i = 1; i < VPL; ++i)
        if (above(key[i], best)) best = key[i], s = sizeof(S) == 8 ? score[i] : x[i], slot = i;
      uint64_t who = __ballot(best.hi == group_max_key<64>(best.hi));
      if (who & (who - 1)) {  // more than one lane
        if constexpr (Key::kWide) {
          const bool in = (who >> lane) & 1;
          const unsigned lo = group_max_key<64>(in ? best.lo : 0u);
          who = __ballot(in && best.lo == lo);
        }
        if (who & (who - 1)) {  // equal choices: the lowest expert; slots rise with it faster than lanes
          unsigned e = ((who >> lane) & 1) ? ~static_cast<unsigned>(lane + 64 * slot) : 0u;
          who = __ballot(e == group_max_key<64>(e));
        }
      }
      const int winner = __ffsll(static_cast<unsigned long long>(who)) - 1;
      const int won_slot = __builtin_amdgcn_readlane(slot, winner);
      const S won = lane_of(s, winner);
      if (lane == j) mine = won, mine_id = winner + 64 * won_slot;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (lane == winner && i == won_slot) key[i] = Key{};
    }
    // Weights in 64 bits: sigmoids far below zero, whose quotients count, are nothing in 32.
    double w = static_cast<double>(mine);
    if constexpr (sizeof(S) == 4) {
      if (sigmoid) w = 1.0 / (1.0 + exp(-w));
      else w = static_cast<double>(mine == top ? 1.f : __builtin_expf(mine - top)) / (renorm ? 1.0 : static_cast<double>(all));
    }
    if (renorm) {
      double sum = 0.0;
      for (int j = 0; j < topk; ++j) sum += __shfl(w, j, kWave);
      w = sum > 0.0 ? w / sum : 0.0;  // chosen scores that are all zero: no expert counts
    }
    if (lane < topk) {
      w_out[token * topk + lane] = static_cast<float>(w * static_cast<double>(scale));
      id_out[token * topk + lane] = mine_id;
    }
  }
}

template <typename T, typename S, int VPL>
void launch_grouped(const void* logits, int64_t M, int E, int64_t ld, const float* bias, int groups, int kept, int topk, int sigmoid, int renorm,
                    float scale, float* w, int32_t* ids, hipStream_t st) {
  int64_t blocks = ceil_div(M, kGroupWaves);
  if (blocks > 4096) blocks = 4096;  // the rest is the in-kernel token loop
  hipLaunchKernelGGL((gating_grouped_kernel<T, S, VPL>), dim3(static_cast<unsigned>(blocks)), dim3(kGroupWaves * kWave), 0, st,
                     static_cast<const T*>(logits), M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids);
}

template <typename T, typename S>
int dispatch_grouped(const void* logits, int64_t M, int E, int64_t ld, const float* bias, int groups, int kept, int topk, int sigmoid, int renorm,
                     float scale, float* w, int32_t* ids, hipStream_t st) {
  if (E <= 64) launch_grouped<T, S, 1>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);
  else if (E <= 128) launch_grouped<T, S, 2>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);
  else if (E <= 256) launch_grouped<T, S, 4>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);
  else if (E <= 512) launch_grouped<T, S, 8>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);
  else launch_grouped<T, S, 16>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);
  return check_launch("gating_grouped_kernel");
}

template <typename T>
int dispatch_scores(const void* logits, int64_t M, int E, int64_t ld, const float* bias, int groups, int kept, int topk, int sigmoid, int renorm,
                    float scale, float* w, int32_t* ids, hipStream_t st) {
  return bias ? dispatch_grouped<T, double>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st)
              : dispatch_grouped<T, float>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);
}

}  // namespace
}  // namespace fr

extern "C" int fr_gating_grouped(const void* logits, int logits_dtype, int64_t M, int64_t E, int64_t ld, const float* bias, int groups, int kept,
                                 int topk, int scoring, int renormalize, float scale, float* weights_out, int32_t* ids_out, void* stream) {
  using namespace fr;
  FR_REQUIRE(M >= 0, FR_E_SHAPE, "fr_gating_grouped: M=%lld < 0", (long long)M);
  FR_REQUIRE(E >= 1 && E <= 1024, FR_E_SHAPE, "fr_gating_grouped: E=%lld outside [1, 1024]", (long long)E);
  FR_REQUIRE(groups >= 1 && groups <= 64 && E % groups == 0, FR_E_SHAPE, "fr_gating_grouped: %d groups: 1 to 64 that divide E=%lld", groups, (long long)E);
  FR_REQUIRE(kept >= 1 && kept <= groups, FR_E_SHAPE, "fr_gating_grouped: %d kept groups of %d", kept, groups);
  FR_REQUIRE(topk >= 1 && topk <= 64 && topk <= E / groups * kept, FR_E_SHAPE, "fr_gating_grouped: topk=%d outside [1, 64] or more than the kept groups hold", topk);
  FR_REQUIRE(scoring == FR_SCORE_SOFTMAX || scoring == FR_SCORE_SIGMOID, FR_E_SHAPE, "fr_gating_grouped: scoring %d", scoring);
  FR_REQUIRE(ld >= E || M <= 1, FR_E_SHAPE, "fr_gating_grouped: row stride %lld < E", (long long)ld);
  if (M == 0) return FR_OK;
  FR_REQUIRE(logits && weights_out && ids_out, FR_E_NULL, "fr_gating_grouped: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int sig = scoring == FR_SCORE_SIGMOID;
  switch (logits_dtype) {
    case FR_F32: return dispatch_scores<float>(logits, M, (int)E, ld, bias, groups, kept, topk, sig, renormalize, scale, weights_out, ids_out, st);
    case FR_F16: return dispatch_scores<f16_t>(logits, M, (int)E, ld, bias, groups, kept, topk, sig, renormalize, scale, weights_out, ids_out, st);
    case FR_BF16: return dispatch_scores<bf16_t>(logits, M, (int)E, ld, bias, groups, kept, topk, sig, renormalize, scale, weights_out, ids_out, st);
    default: return fail(FR_E_DTYPE, "fr_gating_grouped: logits dtype %d not in {f16, bf16, f32}", logits_dtype);
  }
}

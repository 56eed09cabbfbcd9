// Routing with scores, a bias for balance and groups of experts: a wavefront per token, or four tokens to a wavefront.
//
//   score   s = softmax(l) or sigmoid(l) over the E logits of a token
//   choice  c = s + bias, or l itself where there is no bias (both scores rise with the logit)
//   group   E / groups consecutive experts; its worth is its largest c, with a bias the sum of its two largest
//   result  the topk experts of largest c in the kept groups of largest worth; weights s (/ their sum) * scale
//
// Ties go to the lower index.  With a bias the order depends on sums of rounded scores, so the order is that of 64-bit scores and choices there: 32 bits
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

template <int S>
__device__ __forceinline__ double partner_f64(double v) {
  return __hiloint2double(partner_i32<S>(__double2hiint(v)), partner_i32<S>(__double2loint(v)));
}

// A NaN is the lowest value: no comparison holds for it, and an expert that has one is chosen last.  (+ 0: -0 and +0 are the same value.)
template <typename S>
__device__ __forceinline__ S ordered(S v) { return v == v ? v + S(0) : -static_cast<S>(INFINITY); }

// One token by a wavefront.  S: float without a bias, double with one.  Expert of lane l's value i: l + 64 i.  choice_of (VPL * 64 values) and worth_of (64) are
// the wavefront's own.
template <typename T, typename S, int VPL>
__device__ __forceinline__ void gate_grouped_token(const T* __restrict__ logits, int64_t token, int E, int64_t ld, const float* __restrict__ bias, int groups, int kept,
                                                   int topk, int sigmoid, int renorm, float scale, float* __restrict__ w_out, int32_t* __restrict__ id_out,
                                                   S* choice_of, S* worth_of) {
  typedef decltype(key_of(S(0))) Key;
  const int lane = threadIdx.x & 63, size = E / groups;
  int per = kWave;  // lanes that share a group: a power of two, groups * per <= 64
  while (per * groups > kWave) per >>= 1;
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
    for (int i = 0; i < VPL; ++i) choice_of[lane + 64 * i] = choice[i];
    __builtin_amdgcn_wave_barrier();
    const int g = lane / per;
    S first = -static_cast<S>(INFINITY), second = first;
    if (g < groups)
      for (int j = lane % per; j < size; j += per) {
        const S c = choice_of[g * size + j];
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
    if (g < groups && lane % per == 0) worth_of[g] = worth;
    __builtin_amdgcn_wave_barrier();
    int ahead = 0;
    for (int o = 0; o < groups; ++o) {
      const S w = worth_of[o];
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

template <typename T, typename S, int VPL>
__global__ __launch_bounds__(kGroupWaves * kWave) void gating_grouped_kernel(const T* __restrict__ logits, int64_t M, int E, int64_t ld,
                                                                             const float* __restrict__ bias, int groups, int kept, int topk,
                                                                             int sigmoid, int renorm, float scale, float* __restrict__ w_out,
                                                                             int32_t* __restrict__ id_out) {
  __shared__ S choice_of[kGroupWaves][VPL * kWave];
  __shared__ S worth_of[kGroupWaves][kWave];
  const int wave = threadIdx.x >> 6;
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * kGroupWaves + wave; token < M; token += static_cast<int64_t>(gridDim.x) * kGroupWaves)
    gate_grouped_token<T, S, VPL>(logits, token, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w_out, id_out, choice_of[wave], worth_of[wave]);
}

// Several tokens to a wavefront: 16 lanes (a DPP row) own a token, lane l experts l * VPL .. + VPL - 1, so that a group of experts is a lane or a few lanes
// next to each other and every cross-lane step serves four tokens.
//
// Choices are 32-bit floats here, and the selection runs on unsigned keys: the choice in units of 2^-23 (256 experts) of the span of the candidates' choices,
// the expert's index in the bits below.  The largest key below the previous winner is the largest key minus the winner modulo 2^32.  That is
// the order of the 64-bit choices wherever neighbours - the choices drawn, one more than asked for, and the last kept and the first dropped group - lie
// further apart than both can be off: a sigmoid 2^-21 (exponential, sum and reciprocal, an ulp each where they weigh: 2^-22), a softmax (VPL + 8) 2^-24 (its sum), the
// sum with the bias half an ulp, the key a unit.  Where they do not, more are drawn until the next one does, and their exact choices, which the weights' sigmoids
// give, are ranked (a softmax's are not: it takes all experts' exponentials).  A token whose groups lie too close, or with choices that are not finite among those drawn, is
// done again by the whole wavefront in 64 bits.  Without a bias 16-bit logits' order keys fit beside the index as they are: exact.  The
// weights are computed in 64 bits from the chosen experts' logits.
// Bound by vector instructions, and by the memory's latency for few tokens.
template <typename T, int VPL, bool BIASED>
__global__ __launch_bounds__(kGroupWaves * kWave) void gating_grouped_rows_kernel(const T* __restrict__ logits, int64_t M, int E, int64_t ld,
                                                                                  const float* __restrict__ bias, int groups, int kept, int topk,
                                                                                  int sigmoid, int renorm, float scale, float* __restrict__ w_out,
                                                                                  int32_t* __restrict__ id_out) {
  typedef std::conditional_t<BIASED, double, float> S;
  constexpr int kPiece = VPL * sizeof(T) < 16 ? VPL : 16 / sizeof(T);  // logits of a load
  constexpr int kWhole = (VPL * 16 + kWave - 1) / kWave;               // values per lane where the wavefront does one token
  constexpr int kIndexBits = VPL == 4 ? 6 : VPL == 8 ? 7 : VPL == 16 ? 8 : 9, kBits = 31 - kIndexBits;
  constexpr unsigned kMask = VPL * 16 - 1;
  static_assert(kMask == (1u << kIndexBits) - 1, "an index's bits");
  constexpr bool kExact = !BIASED && sizeof(T) == 2;
  typedef T piece __attribute__((ext_vector_type(kPiece)));
  __shared__ S choice_of[kGroupWaves][kWhole * kWave];
  __shared__ S worth_of[kGroupWaves][kWave];
  const int lane = threadIdx.x & 63, l = lane & 15, wave = threadIdx.x >> 6;
  const bool grouped = kept < groups;
  const float error = sigmoid ? 0x1p-21f : (VPL + 8) * 0x1p-24f;
  const int per = grouped ? 16 / groups : 1;  // lanes of a group, a power of two
  const int have = E - l * VPL;  // of the lane's experts, those that there are
  f32x4 b[BIASED ? VPL / 4 : 1];
  if constexpr (BIASED) {
#pragma unroll
    for (int i = 0; i < VPL / 4; ++i) b[i] = *reinterpret_cast<const f32x4*>(bias + (4 * i < have ? l * VPL + 4 * i : 0));
  }
  for (int64_t token0 = (static_cast<int64_t>(blockIdx.x) * kGroupWaves + wave) * 4; token0 < M; token0 += static_cast<int64_t>(gridDim.x) * kGroupWaves * 4) {
    const int64_t token = token0 + (lane >> 4);
    const bool live = token < M;
    const T* row = logits + (live ? token : M - 1) * ld;
    float x[VPL], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; i += kPiece) {
      const piece v = *reinterpret_cast<const piece*>(row + (i < have ? l * VPL + i : 0));  // E is a multiple of kPiece
#pragma unroll
      for (int e = 0; e < kPiece; ++e) x[i + e] = fmaxf(static_cast<float>(v[e]), -INFINITY);  // no NaN
    }
    if (E < 16 * VPL) {
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i >= have) x[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = fmaxf(top, x[i]);
    top = group_max<16>(top);
    float all = 0.f;
    float c[VPL], first = -INFINITY, second = -INFINITY;
    {
      if (BIASED && sigmoid) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) c[i] = __builtin_amdgcn_rcpf(1.f + __expf(-x[i]));
      } else if (!sigmoid && (BIASED || !renorm)) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          c[i] = x[i] == top ? 1.f : __expf(x[i] - top);
          if (i >= have) c[i] = 0.f;
          all += c[i];
        }
        all = group_sum<16>(all);
        const float by = 1.f / all;
#pragma unroll
        for (int i = 0; i < VPL; ++i) c[i] *= by;
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i) c[i] = BIASED ? fmaxf(c[i] + b[i / 4][i % 4], -INFINITY) : x[i];
      if (BIASED && E < 16 * VPL) {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          if (i >= have) c[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        second = fmaxf(second, fminf(first, c[i]));
        first = fmaxf(first, c[i]);
      }
    }
    bool sure = true, in = true;
    if (grouped) {
      auto merge = [&](float f, float n) {
        second = fmaxf(fmaxf(second, n), fminf(first, f));
        first = fmaxf(first, f);
      };
      if (per > 1) merge(partner_f32<1>(first), partner_f32<1>(second));
      if (per > 2) merge(partner_f32<2>(first), partner_f32<2>(second));
      if (per > 4) merge(partner_f32<4>(first), partner_f32<4>(second));
      const float worth = BIASED ? fmaxf(first + second, -INFINITY) : first;
      const int g = l & -per;  // its first lane
      int ahead = 0;
      auto against = [&](int w, int other) {
        const float v = __int_as_float(w);
        ahead += (v > worth || (v == worth && other < g)) ? 1 : 0;
      };
      const int bits = __float_as_int(worth);
#define FR_AGAINST(n_) \
  if ((n_ & (per - 1)) == 0) against(__builtin_amdgcn_update_dpp(0, bits, 0x120 + n_, 0xF, 0xF, true), __builtin_amdgcn_update_dpp(0, g, 0x120 + n_, 0xF, 0xF, true));
      FR_AGAINST(1) FR_AGAINST(2) FR_AGAINST(3) FR_AGAINST(4) FR_AGAINST(5) FR_AGAINST(6) FR_AGAINST(7) FR_AGAINST(8)
      FR_AGAINST(9) FR_AGAINST(10) FR_AGAINST(11) FR_AGAINST(12) FR_AGAINST(13) FR_AGAINST(14) FR_AGAINST(15)
#undef FR_AGAINST
      in = ahead < kept;
      if constexpr (BIASED) {
        const float low = -group_max<16>(in ? -worth : -INFINITY), high = group_max<16>(in ? -INFINITY : worth);
        const float size = group_max<16>(fmaxf(fabsf(first), fabsf(second)));
        sure = low - high > 4.f * (error + 0x1p-23f * size);  // infinite ones: not sure
      }
    }
    unsigned key[VPL], apart = 0;  // winners that lie closer are not sure
    if constexpr (kExact) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) key[i] = in && i < have ? (float_key(c[i] + 0.f) & ~kMask) | (kMask - (l * VPL + i)) : 0u;
    } else {
      constexpr float kLowest = -1e30f;  // masks; their span would leave the others no bits
      float most = -INFINITY, least = INFINITY;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (in && c[i] > kLowest) most = fmaxf(most, c[i]), least = fminf(least, c[i]);
      most = group_max<16>(most);
      least = -group_max<16>(-least);
      const int e = kBits - __builtin_amdgcn_frexp_expf(most - least);
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const unsigned units = static_cast<unsigned>(ldexpf(c[i] - least, e)) + 1;
        key[i] = in && c[i] > kLowest ? units << kIndexBits | (kMask - (l * VPL + i)) : 0u;
      }
      const float off = BIASED ? ldexpf(error + 0x1p-24f * fmaxf(fabsf(most), fabsf(least)), e) : 0.f;
      apart = 3 + static_cast<unsigned>(2.f * fminf(off, 1e9f));
      sure = sure && most - least < 1e30f;
    }
    // Lane j of a token's 16 draws place j.  More than topk are drawn until a distance says that no other can belong to them; where one of the distances in
    // front says nothing, the drawn ones' exact choices are ranked below.
    unsigned before = 0u, mine = 0u;
    int drawn = 0;  // 0: not known yet
    bool rank = false;
    for (int j = 0; j <= 16; ++j) {
      unsigned best = 0u;
#pragma unroll
      for (int i = 0; i < VPL; ++i) best = max(best, key[i] - before);
      const unsigned won = group_max_key<16>(best) + before;
      const bool far = kExact || (before >> kIndexBits) - (won >> kIndexBits) > apart;
      if (j < topk) {
        if (won == 0u) sure = false;  // the choices that are left are not finite
        rank = rank || (j > 0 && !far);
      } else if (drawn == 0 && (far || won == 0u)) {
        drawn = j;
      }
      if (l == j) mine = won;
      before = won;
      if (j + 1 >= topk && (kExact || __all(drawn > 0 || !sure || !live))) break;
    }
    if (kExact) drawn = topk;
    rank = rank || drawn > topk;
    sure = sure && drawn > 0 && !(rank && BIASED && !sigmoid);  // (an exact softmax takes all experts)
    const int id = static_cast<int>(kMask - (mine & kMask));
    const bool chosen = l < drawn && sure;
    double w = 0.0, exact = 0.0;
    if (chosen) {
      const float v = ordered(static_cast<float>(row[id]));
      const double d = static_cast<double>(v);
      if (sigmoid) w = 1.0 / (1.0 + exp(-d));
      else w = v == top ? 1.0 : exp(d - static_cast<double>(top));
      if (!sigmoid && !renorm) w /= static_cast<double>(all);
      exact = d;
      if constexpr (BIASED) exact = w + static_cast<double>(bias[id]);
    }
    int at = l;
    if (!kExact && __any(rank && sure && live)) {
      at = 0;
      const int low = __double2loint(exact), high = __double2hiint(exact), who = chosen ? id : -1;
#define FR_RANK(n_)                                                                                                                               \
  {                                                                                                                                               \
    const double o = __hiloint2double(__builtin_amdgcn_update_dpp(0, high, 0x120 + n_, 0xF, 0xF, true), __builtin_amdgcn_update_dpp(0, low, 0x120 + n_, 0xF, 0xF, true)); \
    const int other = __builtin_amdgcn_update_dpp(0, who, 0x120 + n_, 0xF, 0xF, true);                                                           \
    at += other >= 0 && (o > exact || (o == exact && other < id)) ? 1 : 0;                                                                        \
  }
      FR_RANK(1) FR_RANK(2) FR_RANK(3) FR_RANK(4) FR_RANK(5) FR_RANK(6) FR_RANK(7) FR_RANK(8) FR_RANK(9) FR_RANK(10) FR_RANK(11) FR_RANK(12)
      FR_RANK(13) FR_RANK(14) FR_RANK(15)
#undef FR_RANK
    }
    const bool kept_place = chosen && at < topk;
    if (renorm) {
      double sum = kept_place ? w : 0.0;
      sum += partner_f64<1>(sum);
      sum += partner_f64<2>(sum);
      sum += partner_f64<4>(sum);
      sum += partner_f64<8>(sum);
      w = sum > 0.0 ? w / sum : 0.0;
    }
    if (kept_place && live) {
      w_out[token * topk + at] = static_cast<float>(w * static_cast<double>(scale));
      id_out[token * topk + at] = id;
    }
    for (uint64_t again = __ballot(l == 0 && live && !sure); again; again &= again - 1)
      gate_grouped_token<T, S, kWhole>(logits, token0 + (__ffsll(static_cast<unsigned long long>(again)) - 1) / 16, E, ld, bias, groups, kept, topk, sigmoid, renorm,
                                       scale, w_out, id_out, choice_of[wave], worth_of[wave]);
  }
}

// Whether the calls' sizes and addresses suit gating_grouped_rows_kernel, with VPL logits to a lane.  us, a wavefront per token / this: 16384 tokens, 256 experts in 8 groups,
// sigmoid and bias 32.1 / 15.4, 7 tokens 6.8 / 6.2; 16384 of 64 experts, softmax and bias 17.8 / 10.7, of 512 60.6 / 30.6, of 256 without bias 18.6 / 10.7; but 7 of 64
// experts in 8 groups 4.2 / 4.6.  Other sizes, a wavefront per token, us for 7, 1031 and 16384 tokens: 8 or 16 experts 2.9, 3.2, 8.7; 60 in 4 groups 4.1, 4.6, 14.4; 160 in 8 groups 6.3,
// 7.2, 27.7; the best 32 of 256 13.1, 15.2, 62.7 (sigmoid and bias).  Without a bias and groups topk_softmax does the softmax's job too: 16384 tokens of 8 experts 2.6 us for 7.8 here, of
// 64 4.3 / 5.4, of 256 7.1 / 7.9, but 64 tokens of 128 5.2 / 3.9 and of 256 6.4 / 4.6 (bf16).
template <typename T, int VPL>
bool rows_fit(const void* logits, int64_t M, int E, int64_t ld, const float* bias, int groups, int kept, int topk, int sigmoid, int renorm) {
  constexpr int piece = VPL * sizeof(T) < 16 ? VPL : 16 / sizeof(T);
  if (topk > 16 || E % piece != 0 || (M > 1 && ld % piece != 0) || reinterpret_cast<uintptr_t>(logits) % (piece * sizeof(T)) != 0) return false;
  if (bias && (E % 4 != 0 || !aligned16(bias))) return false;
  if (bias && !sigmoid && !renorm) return false;  // the weights are the whole softmax's, whose sum is 32 bits there
  if (kept == groups) return true;
  const int size = E / groups;
  return E == 16 * VPL && size % VPL == 0 && 16 % groups == 0;
}

template <typename T, int VPL>
void launch_rows(const void* logits, int64_t M, int E, int64_t ld, const float* bias, int groups, int kept, int topk, int sigmoid, int renorm,
                 float scale, float* w, int32_t* ids, hipStream_t st) {
  int64_t blocks = ceil_div(M, kGroupWaves * 4);
  if (blocks > 2048) blocks = 2048;  // the rest is the in-kernel token loop
  const dim3 grid(static_cast<unsigned>(blocks)), block(kGroupWaves * kWave);
  const T* const x = static_cast<const T*>(logits);
  if (bias) hipLaunchKernelGGL((gating_grouped_rows_kernel<T, VPL, true>), grid, block, 0, st, x, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids);
  else hipLaunchKernelGGL((gating_grouped_rows_kernel<T, VPL, false>), grid, block, 0, st, x, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids);
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
#define FR_ROWS(vpl_)                                                                                          \
  if (E <= 16 * vpl_ && rows_fit<T, vpl_>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm)) { \
    launch_rows<T, vpl_>(logits, M, E, ld, bias, groups, kept, topk, sigmoid, renorm, scale, w, ids, st);     \
    return check_launch("gating_grouped_rows_kernel");                                                       \
  }
  if (E > 16) {
    FR_ROWS(4) else FR_ROWS(8) else FR_ROWS(16) else FR_ROWS(32)
  }
#undef FR_ROWS
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

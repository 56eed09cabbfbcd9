// Attention of packed prompts: softmax(scale Q K^T + mask) V per sequence, in one pass over the keys with a running maximum and sum.
//
// A workgroup takes 128 rows of one sequence and key head, a row being a token's query head that shares the key head: the heads of a token lie next
// to each other, so a tile of few tokens is still a whole one and its keys are read once for all of them.  Four wavefronts of 32 rows; keys in
// blocks of 64, through LDS in two buffers, the next block's loads in flight while one is worked on.
//   S^T [64 keys, 32 rows] = K Q^T on 32x32x16 matrix instructions: Q stays in registers.  A lane's accumulators are 32 scores of one row: maximum
//   and sum need one exchange with the lane that has the other 32, and rescaling is a factor per lane.
//   O^T [dim, 32 rows] += V^T P^T: the accumulators, rounded, are the second operand as they are, if the keys of V^T are taken in the same
//   order; transposed reads of LDS give four keys of a dimension at a time.
// Bound by the matrix instructions and, nearly as long, the exponentials beside them; two workgroups to a CU cover for one another.
//
// Tiles of all sequences are taken in the order of their place in the sequence, last ones first: with a causal mask these have the most keys.
#include "attention_core.h"

namespace fr {
namespace {

constexpr int kAttThreads = 256, kAttWaves = 4, kAttRows = 32, kAttTile = kAttWaves * kAttRows, kAttKeys = 64;

__device__ __forceinline__ int64_t att_clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }
// Rows [*begin, *end) of sequence b of the cumulative lengths cu, inside [0, all] whatever they say; b = B: the rows behind the last one.
__device__ __forceinline__ void att_range(const int32_t* cu, int64_t b, int64_t B, int64_t all, int64_t* begin, int64_t* end) {
  *begin = att_clamp(cu[b], 0, all);
  *end = b == B ? all : att_clamp(cu[b + 1], *begin, all);
}

// Tile `nth` of the tiles in descending order of their place: its sequence (-1: none) and place.
__device__ __forceinline__ void att_place(const fr_attention_args& a, int64_t nth, int64_t* seq, int* place) {
  const int lane = threadIdx.x & 63;
  const int64_t share = a.heads / a.kv_heads, count = a.B + (a.fill ? 1 : 0);
  const int32_t* cu = reinterpret_cast<const int32_t*>(a.cu_q);
  auto tiles_of = [&](int64_t b) -> int {
    if (b >= count) return 0;
    int64_t begin, end;
    att_range(cu, b, a.B, a.rows, &begin, &end);
    return static_cast<int>(((end - begin) * share + kAttTile - 1) / kAttTile);
  };
  const int mine = tiles_of(lane);  // of the first 64 sequences, most often all
  auto total = [&](auto f) {
    int v = f(mine);
    for (int64_t b = lane + kWave; b < count; b += kWave) v += f(tiles_of(b));
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) v += __shfl_xor(v, s, kWave);
    return v;
  };
  *seq = -1;
  int lo = 0, hi = static_cast<int>((a.rows * share + kAttTile - 1) / kAttTile);  // tiles at places >= lo: more than nth; >= hi: not
  if (total([&](int t) { return t; }) <= nth) return;
  if (count == 1) {
    *seq = 0;
    *place = tiles_of(0) - 1 - static_cast<int>(nth);
    return;
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (total([&](int t) { return t > mid ? t - mid : 0; }) > nth) lo = mid;
    else hi = mid;
  }
  int left = static_cast<int>(nth) - total([&](int t) { return t > lo + 1 ? t - lo - 1 : 0; });  // which of the sequences with a tile there
  for (int64_t b0 = 0; b0 < count; b0 += kWave) {
    const uint64_t has = __ballot((b0 ? tiles_of(b0 + lane) : mine) > lo);
    const int n = __popcll(has);
    if (left < n) {
      const int before = __popcll(has & ((1ull << lane) - 1));
      const uint64_t hit = __ballot(((has >> lane) & 1) && before == left);
      if (!hit) return;
      *seq = b0 + __ffsll(static_cast<unsigned long long>(hit)) - 1;
      *place = lo;
      return;
    }
    left -= n;
  }
}

template <int DP>
struct AttShape {
  static constexpr int kChunks = DP / 8;                               // 16-byte pieces of a row
  static constexpr int kLoads = kAttKeys * kChunks / kAttThreads;      // pieces of a block that a thread loads
  static constexpr int kSteps = DP / 16, kTiles = DP / 32;
  // Rows lie in LDS with their pieces exchanged: K so that 8 rows' pieces of one place meet in no bank, V so that the four rows of a
  // transposed read, 32 elements each, do not.
  static __device__ __forceinline__ int k_at(int row, int chunk) { return row * DP + (chunk ^ (row & 7)) * 8; }
  static __device__ __forceinline__ int v_at(int row, int chunk) {
    return row * DP + (chunk ^ (DP % 128 == 0 ? (row & 3) << 2 : ((row >> 1) & 1) << 2)) * 8;
  }
};

// A 16-bit float that is infinite or not a number, in either half of a word.
template <typename T>
__device__ __forceinline__ bool not_finite(unsigned w) {
  constexpr unsigned e = sizeof(T) == 2 && __is_same(T, bf16_t) ? 0x7F80u : 0x7C00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

template <typename T, int DP>
__global__ __launch_bounds__(kAttThreads, DP <= 128 ? 2 : 1) void attention_kernel(fr_attention_args a) {
  typedef typename Attn<T>::vec8 vec8;
  typedef typename Attn<T>::vec4 vec4;
  typedef AttShape<DP> S;
  __shared__ __attribute__((aligned(16))) T shared[2][2][kAttKeys * DP];  // buffer; K, V
  __shared__ int odd[4];  // a block with masked keys has values that are not finite
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, low = lane & 31;
  const int kv_heads = static_cast<int>(a.kv_heads), share = static_cast<int>(a.heads / a.kv_heads), dim = static_cast<int>(a.dim);
  // Workgroups go to the eight XCDs in turn: those of a key head to one of them, whose L2 then holds its keys once.
  int kv;
  int64_t nth;
  if (kv_heads % 8 == 0) {
    const int64_t i = blockIdx.x / 8;
    kv = static_cast<int>(blockIdx.x % 8) * (kv_heads / 8) + static_cast<int>(i % (kv_heads / 8));
    nth = i / (kv_heads / 8);
  } else {
    kv = blockIdx.x % kv_heads;
    nth = blockIdx.x / kv_heads;
  }
  int64_t seq;
  int place = 0;
  att_place(a, nth, &seq, &place);
  if (seq < 0) return;
  seq = __builtin_amdgcn_readfirstlane(static_cast<int>(seq));
  place = __builtin_amdgcn_readfirstlane(place);
  int64_t q_begin, q_end, k_begin = 0, k_end = 0;
  att_range(reinterpret_cast<const int32_t*>(a.cu_q), seq, a.B, a.rows, &q_begin, &q_end);
  if (seq < a.B) att_range(reinterpret_cast<const int32_t*>(a.cu_k), seq, a.B, a.keys, &k_begin, &k_end);
  const int n = static_cast<int>(q_end - q_begin), m = static_cast<int>(k_end - k_begin);
  const int64_t rows = static_cast<int64_t>(n) * share, row0 = static_cast<int64_t>(place) * kAttTile;
  if (row0 >= rows) return;
  // the lane's row: token and query head; keys up to `limit` are seen
  const int64_t row = row0 + wave * kAttRows + low;
  const bool live = row < rows;
  const int token = static_cast<int>((live ? row : rows - 1) / share);
  const int head = kv * share + static_cast<int>((live ? row : rows - 1) - static_cast<int64_t>(token) * share);
  const int limit = a.causal ? m - n + token : m - 1;
  // of the wavefront's first row and of the workgroup's first and last
  const int64_t last_row = row0 + kAttTile < rows ? row0 + kAttTile - 1 : rows - 1;
  const int wave_first = a.causal ? __builtin_amdgcn_readfirstlane(limit) : m - 1;
  const int wave_last = row0 + wave * kAttRows >= rows ? -1 : (a.causal ? __builtin_amdgcn_readlane(limit, 31) : m - 1);
  const int group_first = a.causal ? m - n + static_cast<int>(row0 / share) : m - 1;
  const int group_last = a.causal ? m - n + static_cast<int>(last_row / share) : m - 1;
  const int blocks = group_last < 0 ? 0 : (group_last + kAttKeys) / kAttKeys;
  const int masked_from = group_first < 0 ? 0 : (group_first + 1) / kAttKeys;  // blocks from here on have keys that a row does not see

  vec8 q[S::kSteps];
  {
    const T* from = reinterpret_cast<const T*>(a.q) + (q_begin + token) * a.q_row + head * a.q_head;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      const int d = s * 16 + half * 8;
      q[s] = d < dim ? *reinterpret_cast<const vec8*>(from + d) : vec8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  const float scale = static_cast<float>(a.scale) * kLog2e, lag = kLag / scale;
  const T* const kc = reinterpret_cast<const T*>(a.k) + k_begin * a.k_row + kv * a.k_head;
  const T* const vc = reinterpret_cast<const T*>(a.v) + k_begin * a.v_row + kv * a.v_head;
  if (threadIdx.x < 4) odd[threadIdx.x] = 0;
  __syncthreads();

  vec8 kr[S::kLoads], vr[S::kLoads];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * kAttThreads + threadIdx.x, r = k0 + at / S::kChunks, d = at % S::kChunks * 8;
      const bool in = r < m && d < dim;  // behind the last key: zeros, not what lies there
      kr[i] = in ? *reinterpret_cast<const vec8*>(kc + r * a.k_row + d) : vec8{0, 0, 0, 0, 0, 0, 0, 0};
      vr[i] = in ? *reinterpret_cast<const vec8*>(vc + r * a.v_row + d) : vec8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  };
  auto keep = [&](int block) {
    T* const to = shared[block & 1][0];
    T* const vt = shared[block & 1][1];
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * kAttThreads + threadIdx.x;
      *reinterpret_cast<vec8*>(to + S::k_at(at / S::kChunks, at % S::kChunks)) = kr[i];
      *reinterpret_cast<vec8*>(vt + S::v_at(at / S::kChunks, at % S::kChunks)) = vr[i];
    }
    if (a.causal && block >= masked_from) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const i32x4 w = __builtin_bit_cast(i32x4, vr[i]);
        bad = bad || not_finite<T>(w[0]) || not_finite<T>(w[1]) || not_finite<T>(w[2]) || not_finite<T>(w[3]);
      }
      if (bad) odd[(block - masked_from) & 3] = 1;
    }
  };

  f32x16 o[S::kTiles];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float top = -INFINITY, sum = 0.f;  // unscaled, in both halves, lagging; the sum of the lane's own keys

  if (blocks > 0) {
    load(0);
    keep(0);
  }
  __syncthreads();
  for (int block = 0; block < blocks; ++block) {
    const int k0 = block * kAttKeys;
    if (block + 1 < blocks) load(k0 + kAttKeys);
    const T* const kt = shared[block & 1][0];
    const T* const vt = shared[block & 1][1];
    if (k0 <= wave_last) {
      f32x16 st[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[t][r] = 0.f;
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          st[t] = Attn<T>::mma32(*reinterpret_cast<const vec8*>(kt + S::k_at(t * 32 + low, s * 2 + half)), q[s], st[t]);
      if (k0 + kAttKeys - 1 > wave_first || k0 + kAttKeys > m) {
        const int mine = (limit < m ? limit : m - 1) - k0 - 4 * half;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (t * 32 + 8 * (r / 4) + r % 4 > mine) st[t][r] = -INFINITY;
      }
      float high = st[0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) high = fmaxf(high, st[t][r]);
      if (__any(high > top + lag)) {
        high = max_over_32(high);
        const float now = fmaxf(top, high), by = top == -INFINITY ? 0.f : exp2_of((top - now) * scale);
        sum *= by;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[t][r] *= by;
        top = now;
      }
      const float from = top == -INFINITY ? 0.f : top * scale;
      vec8 p[4];  // 16 keys each, to 8 or 11 bits: the second product's operand
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = exp2_of(st[t][r] * scale - from);
          sum += e;
          p[t * 2 + r / 8][r % 8] = static_cast<T>(e);
        }
      auto values = [&](int s, int t) {
        const int r = s * 16 + half * 4 + ((lane & 15) >> 2), chunk = t * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), rest = (lane & 1) * 4;
        return join8(read_transposed<T>(vt + S::v_at(r, chunk) + rest), read_transposed<T>(vt + S::v_at(r + 8, chunk) + rest));
      };
      if (a.causal && block >= masked_from && odd[(block - masked_from) & 3]) {
        // A masked key's term is zero, but its product with a value that is not finite is not: keys one at a time, added where they are seen.
#pragma unroll
        for (int s = 0; s < 4; ++s)
          for (int key = 0; key < 16; ++key)
#pragma unroll
            for (int t = 0; t < S::kTiles; ++t) {
              vec8 v = values(s, t);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (half != ((key >> 2) & 1) || e != 4 * (key >> 3) + (key & 3)) v[e] = 0;
              f32x16 c;
#pragma unroll
              for (int r = 0; r < 16; ++r) c[r] = 0.f;
              c = Attn<T>::mma32(v, p[s], c);
              const bool sees = k0 + s * 16 + key <= limit;
#pragma unroll
              for (int r = 0; r < 16; ++r) o[t][r] += sees ? c[r] : 0.f;
            }
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int t = 0; t < S::kTiles; ++t) o[t] = Attn<T>::mma32(values(s, t), p[s], o[t]);
      }
    }
    if (block + 1 < blocks) keep(block + 1);
    __syncthreads();
  }

  sum = sum_over_32(sum);
  const float by = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no key: zeros
  if (live) {
    T* const to = reinterpret_cast<T*>(a.out) + (q_begin + token) * a.out_row + head * a.out_head + half * 4;
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = t * 32 + r * 8;
        vec4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(o[t][r * 4 + e] * by);
        if (d < dim) *reinterpret_cast<vec4*>(to + d) = y;
      }
  }
}

template <typename T, int DP>
int launch_attention(const fr_attention_args& a, hipStream_t st) {
  // every sequence's last tile may be a part of one; the rows behind the last sequence are one more
  const int64_t tiles = ceil_div(a.rows * (a.heads / a.kv_heads), kAttTile) + a.B + (a.fill ? 1 : 0) - 1;
  hipLaunchKernelGGL((attention_kernel<T, DP>), dim3(static_cast<unsigned>(tiles * a.kv_heads)), dim3(kAttThreads), 0, st, a);
  return check_launch("attention_kernel");
}

template <typename T>
int dispatch_attention(const fr_attention_args& a, hipStream_t st) {
  if (a.dim <= 64) return launch_attention<T, 64>(a, st);
  if (a.dim <= 128) return launch_attention<T, 128>(a, st);
  if (a.dim <= 192) return launch_attention<T, 192>(a, st);
  return launch_attention<T, 256>(a, st);
}

}  // namespace
}  // namespace fr

extern "C" int fr_attention(const fr_attention_args* args, void* stream) {
  using namespace fr;
  FR_REQUIRE(args, FR_E_NULL, "fr_attention: null pointer");
  const fr_attention_args& a = *args;
  FR_REQUIRE(a.heads >= 1 && a.kv_heads >= 1 && a.heads % a.kv_heads == 0 && a.heads <= 65536, FR_E_SHAPE, "fr_attention: %lld heads over %lld key heads",
             (long long)a.heads, (long long)a.kv_heads);
  FR_REQUIRE(a.dim >= 8 && a.dim <= 256 && a.dim % 8 == 0, FR_E_SHAPE, "fr_attention: head size %lld: a multiple of 8 up to 256", (long long)a.dim);
  FR_REQUIRE(a.rows >= 0 && a.rows < (int64_t(1) << 30) && a.keys >= 0 && a.keys < (int64_t(1) << 30), FR_E_SHAPE, "fr_attention: %lld rows, %lld keys: below 2^30",
             (long long)a.rows, (long long)a.keys);
  FR_REQUIRE(a.B >= 0 && a.B <= (1 << 20) && (a.rows + a.B * kAttTile) * a.heads < (int64_t(1) << 37), FR_E_SHAPE, "fr_attention: %lld sequences, %lld rows of %lld heads",
             (long long)a.B, (long long)a.rows, (long long)a.heads);
  FR_REQUIRE(a.dtype == FR_F16 || a.dtype == FR_BF16, FR_E_DTYPE, "fr_attention: dtype %lld not in {f16, bf16}", (long long)a.dtype);
  FR_REQUIRE(a.scale >= 1e-20 && a.scale <= 1e20, FR_E_SHAPE, "fr_attention: scale %g outside [1e-20, 1e20]", a.scale);
  if (a.rows == 0 || (a.B == 0 && !a.fill)) return FR_OK;
  FR_REQUIRE(a.q && a.out && a.cu_q && a.cu_k && (a.keys == 0 || (a.k && a.v)), FR_E_NULL, "fr_attention: null pointer");
  const int64_t strides = a.q_row | a.q_head | a.k_row | a.k_head | a.v_row | a.v_head | a.out_row | a.out_head;
  FR_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out) && strides % 8 == 0, FR_E_ALIGN,
             "fr_attention: q, k, v and out: 16-byte aligned, strides multiples of 8 elements");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FR_BF16 ? dispatch_attention<bf16_t>(a, st) : dispatch_attention<f16_t>(a, st);
}

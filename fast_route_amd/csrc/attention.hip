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

constexpr int kAttThreads = 256, kAttWaves = 4, kAttRows = 32, kAttTile = kAttWaves * kAttRows;

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
  static constexpr int kKeys = DP <= 128 ? 64 : 32;                 // of a block: four buffers of it let two workgroups share a CU
  static constexpr int kGroups = kKeys / 32;                        // of 32 keys
  static constexpr int kChunks = DP / 8;                            // 16-byte pieces of a row
  static constexpr int kRow = DP * 2, kBlock = kKeys * kRow;        // bytes
  static constexpr int kLoads = kKeys * kChunks / kAttThreads;      // pieces of a block that a thread loads
  static constexpr int kSteps = DP / 16, kTiles = DP / 32;
  // Rows lie in LDS with their pieces exchanged: K so that 8 rows' pieces of one place meet in no bank, V so that the four rows of a
  // transposed read, 32 elements each, do not.
  static constexpr bool kWide = DP % 128 == 0;
  static constexpr int kValueBases = kWide ? 4 : 2;
  static __device__ __forceinline__ int k_piece(int row, int chunk) { return chunk ^ (row & 7); }
  static __device__ __forceinline__ int v_piece(int row, int chunk) { return chunk ^ (kWide ? (row & 3) << 2 : ((row >> 1) & 1) << 2); }
};

// A 16-bit float that is infinite or not a number, in either half of a word.
template <typename T>
__device__ __forceinline__ bool not_finite(unsigned w) {
  constexpr unsigned e = __is_same(T, bf16_t) ? 0x7F80u : 0x7C00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// The wavefront's rows one by one, keys to lanes and then dimensions to lanes, fp32: no product of a masked key is formed.
template <typename T, int DP>
__device__ void attention_rows(const fr_attention_args& a, const T* kc, const T* vc, int64_t row0, int64_t rows, int64_t q_begin, int n, int m, int kv, int share) {
  typedef typename Attn<T>::vec8 vec8;
  const int lane = threadIdx.x & 63, dim = static_cast<int>(a.dim);
  const float scale = static_cast<float>(a.scale) * kLog2e;
  for (int i = 0; i < kAttRows && row0 + i < rows; ++i) {
    const int token = static_cast<int>((row0 + i) / share), head = kv * share + static_cast<int>(row0 + i - static_cast<int64_t>(token) * share);
    const int count = a.causal ? (m - n + token + 1 < 0 ? 0 : m - n + token + 1) : m;
    const T* q = reinterpret_cast<const T*>(a.q) + (q_begin + token) * a.q_row + head * a.q_head;
    auto score = [&](int key) {
      float s = 0.f;
      for (int d = 0; d < dim; d += 8) {
        const vec8 x = *reinterpret_cast<const vec8*>(q + d), y = *reinterpret_cast<const vec8*>(kc + key * a.k_row + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(static_cast<float>(x[e]), static_cast<float>(y[e]), s);
      }
      return s * scale;
    };
    float top = -INFINITY, sum = 0.f, acc[DP / kWave];
    for (int key = lane; key < count; key += kWave) top = fmaxf(top, score(key));
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, kWave));
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int d = 0; d < DP / kWave; ++d) acc[d] = 0.f;
    for (int k0 = 0; k0 < count; k0 += kWave) {
      const float p = k0 + lane < count ? exp2_of(score(k0 + lane) - from) : 0.f;
      sum += p;
      for (int j = 0; j < kWave && k0 + j < count; ++j) {
        const float pj = __shfl(p, j, kWave);
#pragma unroll
        for (int d = 0; d < DP / kWave; ++d)
          if (d * kWave + lane < dim) acc[d] = __builtin_fmaf(pj, static_cast<float>(vc[(k0 + j) * a.v_row + d * kWave + lane]), acc[d]);
      }
    }
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) sum += __shfl_xor(sum, s, kWave);
    T* to = reinterpret_cast<T*>(a.out) + (q_begin + token) * a.out_row + head * a.out_head;
#pragma unroll
    for (int d = 0; d < DP / kWave; ++d)
      if (d * kWave + lane < dim) to[d * kWave + lane] = static_cast<T>(sum == 0.f ? 0.f : acc[d] / sum);
  }
}

template <typename T, int DP>
__global__ __launch_bounds__(kAttThreads, 2) void attention_kernel(fr_attention_args a) {
#if defined(__HIP_DEVICE_COMPILE__)  // buffer resources and loads to LDS exist in the device pass only
  typedef typename Attn<T>::vec8 vec8;
  typedef typename Attn<T>::vec4 vec4;
  typedef AttShape<DP> S;
  __shared__ __attribute__((aligned(16))) char shared[4 * S::kBlock];  // K in two buffers, V in two
  __shared__ int odd;  // a block with masked keys has values that are not finite
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
  const int64_t rows = static_cast<int64_t>(n) * share, row0 = static_cast<int64_t>(place) * kAttTile, wave_row0 = row0 + wave * kAttRows;
  if (row0 >= rows) return;
  // the lane's row: token and query head; keys up to `limit` are seen
  const bool live = wave_row0 + low < rows;
  const int64_t row = live ? wave_row0 + low : rows - 1;
  const int token = static_cast<int>(row / share), head = kv * share + static_cast<int>(row - static_cast<int64_t>(token) * share);
  const int limit = a.causal ? m - n + token : m - 1;
  // of the wavefront's first and last row and of the workgroup's
  const int64_t last_row = row0 + kAttTile < rows ? row0 + kAttTile - 1 : rows - 1;
  const int wave_first = __builtin_amdgcn_readfirstlane(limit), wave_last = wave_row0 >= rows ? -1 : __builtin_amdgcn_readlane(limit, 31);
  const int group_first = a.causal ? m - n + static_cast<int>(row0 / share) : m - 1;
  const int group_last = a.causal ? m - n + static_cast<int>(last_row / share) : m - 1;
  const int blocks = group_last < 0 ? 0 : group_last / S::kKeys + 1;

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
  if (threadIdx.x == 0) odd = 0;
  if (dim < DP) {  // the dimensions that there are not stay zero: no load goes there
    for (int i = threadIdx.x; i < 4 * S::kBlock / 16; i += kAttThreads) reinterpret_cast<i32x4*>(shared)[i] = i32x4{0, 0, 0, 0};
  }
  // Where this thread's pieces of a block come from: bytes from the block's first row.
  int k_from[S::kLoads], v_from[S::kLoads];
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) {
    const int at = i * kAttThreads + threadIdx.x, r = at / S::kChunks, kd = S::k_piece(r, at % S::kChunks) * 8, vd = S::v_piece(r, at % S::kChunks) * 8;
    k_from[i] = kd < dim ? (r * static_cast<int>(a.k_row) + kd) * 2 : -1;  // -1: behind every resource's end
    v_from[i] = vd < dim ? (r * static_cast<int>(a.v_row) + vd) * 2 : -1;
  }
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto load = [&](int block) {
    const int k0 = block * S::kKeys, there = m - k0 < S::kKeys ? m - k0 : S::kKeys;
    const __amdgpu_buffer_rsrc_t kr = uniform_buffer(kc + k0 * a.k_row, ((there - 1) * static_cast<int>(a.k_row) + dim) * 2);
    const __amdgpu_buffer_rsrc_t vr = uniform_buffer(vc + k0 * a.v_row, ((there - 1) * static_cast<int>(a.v_row) + dim) * 2);
    char* const kt = shared + (block & 1) * S::kBlock;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_ptr)(kt + (i * kAttThreads + wave * kWave) * 16), 16, k_from[i], 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_ptr)(kt + 2 * S::kBlock + (i * kAttThreads + wave * kWave) * 16), 16, v_from[i], 0, 0, 0);
    }
  };
  // What this lane reads of a block's rows: see k_piece and v_piece.
  int k_at[4], v_at[S::kValueBases];
#pragma unroll
  for (int j = 0; j < 4; ++j) k_at[j] = low * S::kRow + S::k_piece(low, 2 * j + half) * 16;
#pragma unroll
  for (int j = 0; j < S::kValueBases; ++j) {
    const int r = half * 4 + ((lane & 15) >> 2);
    v_at[j] = 2 * S::kBlock + r * S::kRow + S::v_piece(r, j * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
  }

  f32x16 o[S::kTiles];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float top = -INFINITY, sum = 0.f;  // unscaled, in both halves, lagging; the sum of the lane's own keys

  __syncthreads();
  if (blocks > 0) load(0);
  for (int block = 0; block < blocks; ++block) {
    const int k0 = block * S::kKeys;
    const char* const buffer = shared + (block & 1) * S::kBlock;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the block is there, and the one before it has been read
    if (block + 1 < blocks) load(block + 1);
    if (k0 + S::kKeys > m) {  // behind the last key: zeros, whatever lies there
      for (int i = threadIdx.x; i < (S::kKeys - (m - k0)) * S::kChunks; i += kAttThreads)
        *reinterpret_cast<i32x4*>(const_cast<char*>(buffer) + 2 * S::kBlock + ((m - k0) * S::kChunks + i) * 16) = i32x4{0, 0, 0, 0};
      __syncthreads();
    }
    if (a.causal && k0 + S::kKeys - 1 > group_first) {
      bool bad = false;
      for (int i = threadIdx.x; i < S::kBlock / 16; i += kAttThreads) {
        const i32x4 w = *reinterpret_cast<const i32x4*>(buffer + 2 * S::kBlock + i * 16);
        bad = bad || not_finite<T>(w[0]) || not_finite<T>(w[1]) || not_finite<T>(w[2]) || not_finite<T>(w[3]);
      }
      if (bad) odd = 1;
    }
    if (k0 > wave_last) continue;
    f32x16 st[S::kGroups];
#pragma unroll
    for (int t = 0; t < S::kGroups; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[t][r] = 0.f;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
      for (int t = 0; t < S::kGroups; ++t)
        st[t] = Attn<T>::mma32(*reinterpret_cast<const vec8*>(buffer + k_at[s & 3] + (s >> 2) * 128 + t * 32 * S::kRow), q[s], st[t]);
    if (k0 + S::kKeys - 1 > wave_first) {
      const int mine = limit - k0 - 4 * half;
#pragma unroll
      for (int t = 0; t < S::kGroups; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * 32 + 8 * (r / 4) + r % 4 > mine) st[t][r] = -INFINITY;
    }
    float high = st[0][0];
#pragma unroll
    for (int t = 0; t < S::kGroups; ++t)
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
    vec8 p[2 * S::kGroups];  // 16 keys each, to 8 or 11 bits: the second product's operand
#pragma unroll
    for (int t = 0; t < S::kGroups; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = exp2_of(__builtin_fmaf(st[t][r], scale, -from));
        sum += e;
        p[t * 2 + r / 8][r % 8] = static_cast<T>(e);
      }
#pragma unroll
    for (int s = 0; s < 2 * S::kGroups; ++s)
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) {
        const char* const at = buffer + v_at[t % S::kValueBases] + t / S::kValueBases * (S::kValueBases * 64) + s * 16 * S::kRow;
        const vec8 v = join8(read_transposed<T>(reinterpret_cast<const T*>(at)), read_transposed<T>(reinterpret_cast<const T*>(at + 8 * S::kRow)));
        o[t] = Attn<T>::mma32(v, p[s], o[t]);
      }
  }

  __syncthreads();
  if (odd) {
    attention_rows<T, DP>(a, kc, vc, wave_row0, rows, q_begin, n, m, kv, share);
    return;
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
#endif
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
  FR_REQUIRE(a.k_row >= 0 && a.k_row < (1 << 23) && a.v_row >= 0 && a.v_row < (1 << 23), FR_E_SHAPE, "fr_attention: keys %lld and values %lld elements apart: below 2^23",
             (long long)a.k_row, (long long)a.v_row);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FR_BF16 ? dispatch_attention<bf16_t>(a, st) : dispatch_attention<f16_t>(a, st);
}

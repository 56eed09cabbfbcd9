// Attention of packed prompts: softmax(scale Q K^T + mask) V per sequence, in one pass over the keys with a running maximum and sum.
//
// A workgroup takes 128 rows of one sequence and key head, a row being a token's query head that shares the key head: the heads of a token lie next
// to each other, so a tile of few tokens is still a whole one and its keys are read once for all of them.  Four wavefronts of 32 rows; keys in
// blocks of 64 (32 from 129 dimensions on), straight to LDS in two buffers, the next block's loads in flight while one is worked on, one barrier a block.
//   S^T [keys, rows] = K Q^T on 16x16x32 matrix instructions: Q stays in registers.  A lane's accumulators are the scores of two rows with every
//   fourth run of four keys: the maximum needs no exchange until it moves (kLag), and rescaling is a factor per lane.
//   O^T [dim, rows] += V^T P^T: the accumulators, rounded, are the second operand as they are, if the keys of V^T are taken in the same
//   order; transposed reads of LDS give four keys of a dimension at a time.
// 16x16x32 and not 32x32x16 (a register of accumulators read per 32 flops more): the part runs under its power limit, and the clock is 1.92 in place of 1.72 GHz; 8192
// rows without a mask 993 us against 1033.  A prompt of 16384 rows, 32 heads over 8 of 128 dimensions: 2.0 ms, 1.08 to 1.12 PFLOP/s (a matrix product 8192^3 reaches 1.47); 64
// dimensions 0.98, 192 1.14, 256 1.04; 80 and 96, which are computed as 128, 0.74 and 0.88.
// Bound by the matrix instructions (48 % of the cycles) and the vector instructions between them (an exponential, a multiply-add, half
// a maximum and half a conversion per score: 770 cycles beside 1090 in a wavefront's block of 128 dimensions, and a block takes 1880): a SIMD hardly runs the two at once.
// Tried and taken back: the next block's scores computed beside this one's exponentials in one wavefront (3 % slower, and no faster with the order fixed by hand);
// eight wavefronts whose halves take turns, products beside exponentials, with a barrier between the turns (10 % slower, 64 dimensions 27 %).
//
// Short sequences: about 6 us of a workgroup go by before its first product (lengths, search, first loads), 24 prompts of 512 rows 119 us, 0.43 PFLOP/s.  Tiles of all
// sequences are taken in the order of their place in the sequence, last ones first: with a causal mask these have the most keys.  Few tiles over many
// keys are split along the keys as well and joined by a second launch.
#include "attention_core.h"
#include "fr_memory.h"

namespace fr {
namespace {

constexpr int kAttThreads = 256, kAttWaves = 4, kAttRows = 32, kAttTile = kAttWaves * kAttRows;

__device__ __forceinline__ int64_t att_clamp(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }
// Rows [*begin, *end) of sequence b of the cumulative lengths cu, inside [0, all] whatever they say; b = B: the rows behind the last one, B + 1: in front of
// the first.
__device__ __forceinline__ void att_range(const int32_t* cu, int64_t b, int64_t B, int64_t all, int64_t* begin, int64_t* end) {
  *begin = b > B ? 0 : att_clamp(cu[b], 0, all);
  *end = b > B ? att_clamp(cu[0], 0, all) : b == B ? all : att_clamp(cu[b + 1], *begin, all);
}
constexpr int kAttOutside = 2;  // of those two

struct AttPlace {
  int tile;                  // of the sequence, -1: none
  int q_begin, n, k_begin, m;  // its rows and keys
};

__device__ __forceinline__ int att_tiles_of(const fr_attention_args& a, int b) {
  int64_t begin, end;
  att_range(reinterpret_cast<const int32_t*>(a.cu_q), b, a.B, a.rows, &begin, &end);
  return (static_cast<int>(end - begin) * static_cast<int>(a.heads / a.kv_heads) + kAttTile - 1) / kAttTile;
}

// Tile `nth` of the tiles in descending order of their place.  The sequences' tiles stay in the lanes, four times 64: a search step is a
// handful of instructions there and a round trip to L2 beyond (96 sequences of 128 rows: 6.7 us of a workgroup's 16 when only 64 did).  More sequences: one after the
// other, found in what attention_plan_kernel wrote.
constexpr int kAttHeld = kHeldLengths / kWave;
__device__ __forceinline__ AttPlace att_place(const fr_attention_args& a, int nth) {
  const int lane = threadIdx.x & 63;
  const int count = static_cast<int>(a.B + (a.fill ? kAttOutside : 0));
  AttPlace p = {-1, 0, 0, 0, 0};
  int seq = 0, lo = 0;
  struct Rows { int begin, n; };
  auto range = [](const void* cu, int b, int64_t B, int64_t all) -> Rows {
    int64_t begin, end;
    att_range(reinterpret_cast<const int32_t*>(cu), b, B, all, &begin, &end);
    return Rows{static_cast<int>(begin), static_cast<int>(end - begin)};
  };
  Rows mine_q = {0, 0}, mine_k = {0, 0};  // of sequence `lane`
  if (a.plan) {
    const int* const plan = reinterpret_cast<const int*>(a.plan);
    seq = place_in(plan, count, nth);
    if (seq < 0) return p;
    lo = plan[seq + 1] - 1 - nth;
    mine_q = range(a.cu_q, seq, a.B, a.rows);
    if (seq < a.B) mine_k = range(a.cu_k, seq, a.B, a.keys);
  } else {
    if (lane < count) mine_q = range(a.cu_q, lane, a.B, a.rows);
    if (lane < a.B) mine_k = range(a.cu_k, lane, a.B, a.keys);
    const int share = static_cast<int>(a.heads / a.kv_heads);
    int mine[kAttHeld];  // tiles of sequences lane + 64 j
#pragma unroll
    for (int j = 0; j < kAttHeld; ++j) {
      const int b = lane + j * kWave;
      mine[j] = j == 0 ? (mine_q.n * share + kAttTile - 1) / kAttTile : (b < count ? att_tiles_of(a, b) : 0);
    }
    auto total = [&](auto f) {
      int v = f(mine[0]);
      if (count > kWave) {
#pragma unroll
        for (int j = 1; j < kAttHeld; ++j) v += f(mine[j]);
      }
      return sum_of_all(v);
    };
    if (count == 1) {
      lo = __builtin_amdgcn_readfirstlane(mine[0]) - 1 - nth;
      if (lo < 0) return p;
    } else {
      if (total([](int t) { return t; }) <= nth) return p;
      int hi = (static_cast<int>(a.rows) * share + kAttTile - 1) / kAttTile;  // tiles at places >= lo: more than nth; >= hi: not
      for (int step = 1; lo + step < hi; step <<= 1) {                        // most sequences are short beside all of them
        if (total([&](int t) { return t > lo + step ? t - lo - step : 0; }) <= nth) {
          hi = lo + step;
          break;
        }
        lo += step;
      }
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (total([&](int t) { return t > mid ? t - mid : 0; }) > nth) lo = mid;
        else hi = mid;
      }
      int left = nth - total([&](int t) { return t > lo + 1 ? t - lo - 1 : 0; });  // which of the sequences with a tile there
      seq = -1;
#pragma unroll
      for (int j = 0; j < kAttHeld; ++j) {
        const uint64_t has = __ballot(mine[j] > lo);
        const int there = __popcll(has);
        if (seq < 0 && left < there) {
          const uint64_t hit = __ballot(((has >> lane) & 1) && __popcll(has & ((1ull << lane) - 1)) == left);
          if (!hit) return p;
          seq = j * kWave + __ffsll(static_cast<unsigned long long>(hit)) - 1;
        }
        left -= there;
      }
      if (seq < 0) return p;
      if (seq >= kWave) {
        mine_q = range(a.cu_q, seq, a.B, a.rows);
        mine_k = seq < a.B ? range(a.cu_k, seq, a.B, a.keys) : Rows{0, 0};
      }
    }
  }
  p.tile = __builtin_amdgcn_readfirstlane(lo);
  const int l = __builtin_amdgcn_readfirstlane(seq & 63);
  p.q_begin = __builtin_amdgcn_readlane(mine_q.begin, l);
  p.n = __builtin_amdgcn_readlane(mine_q.n, l);
  p.k_begin = __builtin_amdgcn_readlane(mine_k.begin, l);
  p.m = __builtin_amdgcn_readlane(mine_k.n, l);
  return p;
}

__global__ __launch_bounds__(kPlanThreads) void attention_plan_kernel(fr_attention_args a) {
  prefix_of(static_cast<int>(a.B + (a.fill ? kAttOutside : 0)), [&](int b) { return att_tiles_of(a, b); }, reinterpret_cast<int*>(a.plan));
}

template <int DP>
struct AttShape {
  static constexpr int kKeys = DP <= 128 ? 64 : 32;                 // of a block: four buffers of it let two workgroups share a CU
  static constexpr int kGroups = kKeys / 32;                        // of 32 keys
  static constexpr int kChunks = DP / 8;                            // 16-byte pieces of a row
  static constexpr int kRow = DP * 2, kBlock = kKeys * kRow;        // bytes
  static constexpr int kLoads = kKeys * kChunks / kAttThreads;      // pieces of a block that a thread loads
  static constexpr int kSteps = DP / 32, kTiles = DP / 16;
  // Rows lie in LDS with their pieces exchanged, so that 16 rows' pieces of one place (K) and eight rows' 32 bytes of one place (V: lanes 0 .. 31 of a
  // transposed read, or 0 .. 15 and 32 .. 47) meet in no bank of the 64; rows of an odd multiple of 128 bytes alternate between their
  // halves by themselves.  (256 dimensions: 8 rows of K, registers being short, and lanes 0 .. 31 of V, a load's rows being eight.)
  static constexpr bool kWide = DP % 128 == 0;
  static constexpr int kKeyBases = DP == 128 ? 4 : 2, kValueBases = kWide ? 8 : 4;
  static __device__ __forceinline__ int k_piece(int row, int chunk) { return chunk ^ (DP == 128 ? row & 15 : kWide ? row & 7 : (row >> 1) & 7); }
  static __device__ __forceinline__ int v_piece(int row, int chunk) {
    return chunk ^ (DP == 256 ? (row & 7) << 1 : kWide ? (row & 3) << 1 | ((row >> 2 ^ row >> 3) & 1) << 3 : ((row >> 1) & 1) << 1 | ((row >> 2 ^ row >> 3) & 1) << 2);
  }
};

// A maximum that is finite and whose product with the scale, in factors of 2, is more than kFar.  (Looked at where a maximum moves: a prompt of 16384 rows 1980 us for 1974.
// The difference first for all scores, by a branch in each block: 1990, 256 dimensions 1168 for 1146.)
constexpr float kFar = 0x1p20f;
__device__ __forceinline__ bool too_far(float top, float scale) { return fabsf(top) * scale > kFar && fabsf(top) != INFINITY; }
// A 16-bit float that is infinite or not a number, in either half of a word.
template <typename T>
__device__ __forceinline__ bool not_finite(unsigned w) {
  constexpr unsigned e = __is_same(T, bf16_t) ? 0x7F80u : 0x7C00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// Results of a part of the keys: [part][row][head] rows of DP sums, then as many maxima and sums of the softmax.
template <int DP>
struct AttPart {
  float *rows, *tops, *sums;
  __device__ __forceinline__ AttPart(const fr_attention_args& a, int part, int64_t row, int head) {
    const int64_t all = a.rows * a.heads, at = part * all + row * a.heads + head;
    float* const to = reinterpret_cast<float*>(a.workspace);
    rows = to + at * DP;
    tops = to + a.parts * all * DP + at;
    sums = to + a.parts * all * (DP + 1) + at;
  }
};

// The wavefront's rows one by one over keys k_first .. k_last - 1, keys to lanes and then dimensions to lanes, fp32: no product of a masked key is formed.
template <typename T, int DP>
__device__ void attention_rows(const fr_attention_args& a, const T* kc, const T* vc, int row0, int rows, AttPlace at, int kv, int share, int part, int k_first,
                               int k_last) {
  typedef typename Attn<T>::vec8 vec8;
  const int lane = threadIdx.x & 63, dim = static_cast<int>(a.dim);
  const float scale = static_cast<float>(a.scale) * kLog2e;
  for (int i = 0; i < kAttRows && row0 + i < rows; ++i) {
    const int token = (row0 + i) / share, head = kv * share + (row0 + i - token * share);
    const int seen = a.causal ? at.m - at.n + token + 1 : at.m, count = seen < k_last ? seen : k_last;
    const T* q = reinterpret_cast<const T*>(a.q) + (at.q_begin + token) * a.q_row + head * a.q_head;
    auto score = [&](int key) {
      float s = 0.f;
      for (int d = 0; d < dim; d += 8) {
        const vec8 x = *reinterpret_cast<const vec8*>(q + d), y = *reinterpret_cast<const vec8*>(kc + key * a.k_row + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(static_cast<float>(x[e]), static_cast<float>(y[e]), s);
      }
      return s;
    };
    float top = -INFINITY, sum = 0.f, acc[DP / kWave];
    for (int key = k_first + lane; key < count; key += kWave) top = fmaxf(top, score(key));
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) top = fmaxf(top, __shfl_xor(top, s, kWave));
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int d = 0; d < DP / kWave; ++d) acc[d] = 0.f;
    for (int k0 = k_first; k0 < count; k0 += kWave) {
      const float p = k0 + lane < count ? exp2_of(__builtin_fmaf(score(k0 + lane) - from, scale, Attn<T>::kRaise)) : 0.f;
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
    if (a.parts > 1) {
      const AttPart<DP> to(a, part, at.q_begin + token, head);
#pragma unroll
      for (int d = 0; d < DP / kWave; ++d) to.rows[d * kWave + lane] = d * kWave + lane < dim ? acc[d] : 0.f;
      if (lane == 0) to.tops[0] = top, to.sums[0] = sum;
      continue;
    }
    T* to = reinterpret_cast<T*>(a.out) + (at.q_begin + token) * a.out_row + head * a.out_head;
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
  __shared__ int odd;  // a block with masked keys has values that are not finite, or scores are too far from zero
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4, low = lane & 15;
  const int kv_heads = static_cast<int>(a.kv_heads), share = static_cast<int>(a.heads / a.kv_heads), dim = static_cast<int>(a.dim);
  // Workgroups go to the eight XCDs in turn: those of a key head to one of them, whose L2 then holds its keys once.
  int kv, item;
  if (kv_heads % 8 == 0) {
    const int i = blockIdx.x / 8;
    kv = blockIdx.x % 8 * (kv_heads / 8) + i % (kv_heads / 8);
    item = i / (kv_heads / 8);
  } else {
    kv = blockIdx.x % kv_heads;
    item = blockIdx.x / kv_heads;
  }
  const int parts = static_cast<int>(a.parts), part = item % parts;
  const AttPlace at = att_place(a, item / parts);
  if (at.tile < 0) return;
  const int n = at.n, m = at.m, q_begin = at.q_begin;
  const int rows = n * share, row0 = at.tile * kAttTile, wave_row0 = row0 + wave * kAttRows;
  if (row0 < 0 || row0 >= rows) return;
  // the lane's two rows, 16 apart: token and query head; keys up to `limit` are seen
  int token[2], head[2], limit[2];
  bool live[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wave_row0 + 16 * i + low;
    live[i] = r < rows;
    token[i] = (live[i] ? r : rows - 1) / share;
    head[i] = kv * share + (live[i] ? r : rows - 1) - token[i] * share;
    limit[i] = a.causal ? m - n + token[i] : m - 1;
  }
  // of the wavefront's first and last row and of the workgroup's
  const int last_row = row0 + kAttTile < rows ? row0 + kAttTile - 1 : rows - 1;
  const int wave_first = __builtin_amdgcn_readfirstlane(limit[0]), wave_last = wave_row0 >= rows ? -1 : __builtin_amdgcn_readlane(limit[1], 15);
  const int group_first = a.causal ? m - n + row0 / share : m - 1;
  const int group_last = a.causal ? m - n + last_row / share : m - 1;
  const int all_blocks = group_last < 0 ? 0 : group_last / S::kKeys + 1;
  // 2^30 / 32 blocks times 32 parts: 32 bits
  const int first = static_cast<int>(static_cast<unsigned>(all_blocks) * part / parts), blocks = static_cast<int>(static_cast<unsigned>(all_blocks) * (part + 1) / parts);

  const float scale = static_cast<float>(a.scale) * kLog2e, lag = kLag / scale;
  const T* const kc = reinterpret_cast<const T*>(a.k) + at.k_begin * a.k_row + kv * a.k_head;
  const T* const vc = reinterpret_cast<const T*>(a.v) + at.k_begin * a.v_row + kv * a.v_head;
  if (threadIdx.x == 0) odd = 0;
  if (dim < DP) {  // the dimensions that there are not stay zero: no load goes there
    for (int i = threadIdx.x; i < 4 * S::kBlock / 16; i += kAttThreads) reinterpret_cast<i32x4*>(shared)[i] = i32x4{0, 0, 0, 0};
    __syncthreads();
  }
  // Where this thread's pieces of a block come from: bytes from the block's first row; where the pieces of a load are whole rows, from the
  // load's, one register for all loads (their pieces are exchanged alike).  Rows behind the last key and dimensions that there are
  // not lie behind the resource's end: dropped.
  constexpr bool kRows = kAttThreads % S::kChunks == 0;
  constexpr int kOffsets = kRows ? 1 : S::kLoads, kStep = kRows ? kAttThreads / S::kChunks : 0;
  int k_from[kOffsets], v_from[kOffsets];
#pragma unroll
  for (int i = 0; i < kOffsets; ++i) {
    const int at = i * kAttThreads + threadIdx.x, r = at / S::kChunks, kd = S::k_piece(r, at % S::kChunks) * 8, vd = S::v_piece(r, at % S::kChunks) * 8;
    k_from[i] = kd < dim ? (r * static_cast<int>(a.k_row) + kd) * 2 : -1;
    v_from[i] = vd < dim ? (r * static_cast<int>(a.v_row) + vd) * 2 : -1;
  }
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto load = [&](const T* from, int row, const int (&offset)[kOffsets], char* to, int block) {
    const int k0 = block * S::kKeys, there = m - k0 < S::kKeys ? m - k0 : S::kKeys;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int left = there - i * kStep;
      const __amdgpu_buffer_rsrc_t r = uniform_buffer(from + static_cast<int64_t>(k0 + i * kStep) * row, left > 0 ? ((left - 1) * row + dim) * 2 : 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(to + (block & 1) * S::kBlock + (i * kAttThreads + wave * kWave) * 16), 16, offset[kRows ? 0 : i], 0, 0, 0);
    }
  };
  auto load_k = [&](int block) { load(kc, static_cast<int>(a.k_row), k_from, shared, block); };
  auto load_v = [&](int block) { load(vc, static_cast<int>(a.v_row), v_from, shared + 2 * S::kBlock, block); };
  if (first < blocks) {
    load_k(first);
    load_v(first);
  }
  vec8 q[2][S::kSteps];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const T* from = reinterpret_cast<const T*>(a.q) + (q_begin + token[i]) * a.q_row + head[i] * a.q_head;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      const int d = s * 32 + quarter * 8;
      q[i][s] = d < dim ? *reinterpret_cast<const vec8*>(from + d) : vec8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  // What this lane reads of a block's rows: see k_piece and v_piece.
  int k_at[S::kKeyBases], v_at[S::kValueBases];
#pragma unroll
  for (int j = 0; j < S::kKeyBases; ++j) k_at[j] = low * S::kRow + S::k_piece(low, 4 * j + quarter) * 16;
#pragma unroll
  for (int j = 0; j < S::kValueBases; ++j) {
    const int r = quarter * 4 + (low >> 2);
    v_at[j] = 2 * S::kBlock + r * S::kRow + S::v_piece(r, j * 2 + ((low & 3) >> 1)) * 16 + (low & 1) * 8;
  }

  f32x4 o[2][S::kTiles];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) o[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top[2] = {-INFINITY, -INFINITY};  // unscaled, in all four lanes of a row, lagging
  f32x4 sum[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  const T one = static_cast<T>(1.f);
  const vec8 ones = {one, one, one, one, one, one, one, one};

  for (int block = first; block < blocks; ++block) {
    const int k0 = block * S::kKeys;
    const char* const buffer = shared + (block & 1) * S::kBlock;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the block is there, and the one before it has been read
    if (block + 1 < blocks) {
      load_k(block + 1);
      load_v(block + 1);
    }
    if (a.causal || k0 + S::kKeys > m) {
      char* const values = shared + 2 * S::kBlock + (block & 1) * S::kBlock;
      if (k0 + S::kKeys > m) {  // behind the last key: zeros, whatever lies there
        for (int i = threadIdx.x; i < (S::kKeys - (m - k0)) * S::kChunks; i += kAttThreads)
          *reinterpret_cast<i32x4*>(values + ((m - k0) * S::kChunks + i) * 16) = i32x4{0, 0, 0, 0};
        __syncthreads();
      }
      if (a.causal && k0 + S::kKeys - 1 > group_first) {
        bool bad = false;
        for (int i = threadIdx.x; i < S::kBlock / 16; i += kAttThreads) {
          const i32x4 w = *reinterpret_cast<const i32x4*>(values + i * 16);
          bad = bad || not_finite<T>(w[0]) || not_finite<T>(w[1]) || not_finite<T>(w[2]) || not_finite<T>(w[3]);
        }
        if (bad) odd = 1;
      }
    }
    if (k0 > wave_last) continue;
    __builtin_amdgcn_s_setprio(1);  // in front of the other workgroup's exponentials: 0.5 %
    f32x4 st[2][2 * S::kGroups];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < 2 * S::kGroups; ++t) st[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
      for (int t = 0; t < 2 * S::kGroups; ++t) {
        const vec8 k = *reinterpret_cast<const vec8*>(buffer + k_at[s % S::kKeyBases] + s / S::kKeyBases * (S::kKeyBases * 64) + t * 16 * S::kRow);
#pragma unroll
        for (int i = 0; i < 2; ++i) st[i][t] = Attn<T>::mma16(k, q[i][s], st[i][t]);
      }
    __builtin_amdgcn_s_setprio(0);
    if (k0 + S::kKeys - 1 > wave_first) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int mine = limit[i] - k0 - 4 * quarter;
#pragma unroll
        for (int t = 0; t < 2 * S::kGroups; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t * 16 + r > mine) st[i][t][r] = -INFINITY;
      }
    }
    float high[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      high[i] = st[i][0][0];
#pragma unroll
      for (int t = 0; t < 2 * S::kGroups; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) high[i] = fmaxf(high[i], st[i][t][r]);
    }
    if (__any(high[0] > top[0] + lag || high[1] > top[1] + lag)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float now = fmaxf(top[i], max_over_32(max_over_16(high[i]))), by = top[i] == -INFINITY ? 0.f : exp2_of((top[i] - now) * scale);
        sum[i] *= by;
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) o[i][t] *= by;
        top[i] = now;
      }
      // exp2(score * scale - maximum * scale) is off by 2^-24 of the products: row by row, the difference first, where that is more than 2^-4
      if (too_far(top[0], scale) || too_far(top[1], scale)) odd = 1;
    }
    vec8 p[2][S::kGroups];  // 32 keys each, to 8 or 11 bits: the second product's operand
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float from = top[i] == -INFINITY ? 0.f : __builtin_fmaf(top[i], scale, -Attn<T>::kRaise);
#pragma unroll
      for (int t = 0; t < 2 * S::kGroups; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = exp2_of(__builtin_fmaf(st[i][t][r], scale, -from));
          p[i][t / 2][t % 2 * 4 + r] = static_cast<T>(e);
        }
    }
#pragma unroll
    for (int s = 0; s < S::kGroups; ++s) {
      // the terms' sum, as they are rounded, in every register of a row's lanes: on the matrix unit, which has the time the vector unit has not
#pragma unroll
      for (int i = 0; i < 2; ++i) sum[i] = Attn<T>::mma16(ones, p[i][s], sum[i]);
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) {
        const char* const at = buffer + v_at[t % S::kValueBases] + t / S::kValueBases * (S::kValueBases * 32) + s * 32 * S::kRow;
        const vec8 v = join8(read_transposed<T>(reinterpret_cast<const T*>(at)), read_transposed<T>(reinterpret_cast<const T*>(at + 16 * S::kRow)));
#pragma unroll
        for (int i = 0; i < 2; ++i) o[i][t] = Attn<T>::mma16(v, p[i][s], o[i][t]);
      }
    }
  }

  __syncthreads();
  if (odd) {
    attention_rows<T, DP>(a, kc, vc, wave_row0, rows, at, kv, share, part, first * S::kKeys, blocks * S::kKeys < m ? blocks * S::kKeys : m);
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float all = sum[i][0];
    if (parts > 1) {
      if (live[i]) {
        const AttPart<DP> to(a, part, q_begin + token[i], head[i]);
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) *reinterpret_cast<f32x4*>(to.rows + t * 16 + quarter * 4) = o[i][t];
        if (quarter == 0) to.tops[0] = top[i], to.sums[0] = all;
      }
      continue;
    }
    const float by = all == 0.f ? 0.f : 1.f / all;  // a row that sees no key: zeros
    T* const to = reinterpret_cast<T*>(a.out) + (q_begin + token[i]) * a.out_row + head[i] * a.out_head + (quarter & 1) * 16 + (quarter >> 1) * 8;
#pragma unroll
    for (int t = 0; t < S::kTiles; t += 2) {
      // four dimensions of two tiles to eight of one: lanes of odd quarters exchange with those of even ones
      typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
      vec4 y[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[j][e] = static_cast<T>(o[i][t + j][e] * by);
      const u32x2 lo = __builtin_bit_cast(u32x2, y[0]), hi = __builtin_bit_cast(u32x2, y[1]);
      const auto w0 = __builtin_amdgcn_permlane16_swap(lo[0], hi[0], false, false), w1 = __builtin_amdgcn_permlane16_swap(lo[1], hi[1], false, false);
      const int d = t * 16 + (quarter & 1) * 16 + (quarter >> 1) * 8;
      if (live[i] && d < dim) *reinterpret_cast<u32x4_t*>(to + t * 16) = u32x4_t{w0[0], w1[0], w0[1], w1[1]};
    }
  }
#endif
}

template <typename T, int DP>
__global__ __launch_bounds__(kAttThreads) void attention_join_kernel(fr_attention_args a, int wide) {
  typedef JoinShape<DP> J;
  const int64_t all = a.rows * a.heads, at = wide ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * J::kGroups + threadIdx.x / J::kLanes;
  const int64_t row = (at < all ? at : all - 1) / a.heads, head = (at < all ? at : all - 1) - row * a.heads;
  const int32_t* const cu = reinterpret_cast<const int32_t*>(a.cu_q);
  const bool live = at < all && (a.fill || (row < att_clamp(cu[a.B], 0, a.rows) && row >= cu[0]));  // of a sequence
  if (wide && !live) return;
  const AttPart<DP> from(a, 0, row, static_cast<int>(head));
  join_parts<T, DP>(wide, live, static_cast<int>(a.parts), from.rows, all * DP, from.tops, from.sums, all, static_cast<float>(a.scale) * kLog2e,
                    reinterpret_cast<T*>(a.out) + row * a.out_row + head * a.out_head, static_cast<int>(a.dim));
}

int att_dim(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }

// Workgroups of a part: every sequence's last tile may be a part of one; the rows in front of the first sequence and behind the last one are two more.
int64_t att_tiles(int64_t B, int64_t rows, int64_t share, bool fill) { return ceil_div(rows * share, kAttTile) + B + (fill ? kAttOutside : 0) - 1; }

// Parts that the keys are split into: as many as fill the chip's 512 places for workgroups where the tiles do not, none of less than kAttPartKeys keys
// of a sequence of average length (the lengths themselves are on the device).  509 rows over 8192 keys, 16 heads over 2 of 64: one part 117 us, eight 44.  At 768
// places 512 rows over 8704 keys take 109 us for 88; parts of 512 keys and more: a row over 8000 keys 22.5 us for 17.3.  All of these are of equal sequences: the average says
// little where one has most of the keys (512 rows over 66048 keys, 32 heads over 8: 620 us; beside seven prompts of 100 rows, which take 13 alone, 1960).
constexpr int64_t kAttPlaces = 512, kAttPartKeys = 256, kAttMostParts = 32;
int64_t att_parts(int64_t B, int64_t rows, int64_t keys, int64_t heads, int64_t kv_heads) {
  if (B < 1 || rows < 1) return 1;
  const int64_t groups = (ceil_div(rows * (heads / kv_heads), kAttTile) + B - 1) * kv_heads;
  int64_t parts = kAttPlaces / groups;
  const int64_t useful = keys / B / kAttPartKeys;
  parts = parts < useful ? parts : useful;
  return parts < 1 ? 1 : (parts > kAttMostParts ? kAttMostParts : parts);
}

int64_t att_part_bytes(int64_t parts, int64_t rows, int64_t heads, int64_t dim) { return parts == 1 ? 0 : round_up(parts * rows * heads * (att_dim(dim) + 2) * 4, 16); }
int64_t att_plan_bytes(int64_t B) { return B + kAttOutside <= kHeldLengths ? 0 : round_up((B + kAttOutside + 1) * 4, 16); }

template <typename T, int DP>
int launch_attention(const fr_attention_args& a, hipStream_t st) {
  if (a.plan) {
    hipLaunchKernelGGL(attention_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    const int rc = check_launch("attention_plan_kernel");
    if (rc != FR_OK) return rc;
  }
  const int64_t tiles = att_tiles(a.B, a.rows, a.heads / a.kv_heads, a.fill != 0);
  hipLaunchKernelGGL((attention_kernel<T, DP>), dim3(static_cast<unsigned>(tiles * a.parts * a.kv_heads)), dim3(kAttThreads), 0, st, a);
  const int rc = check_launch("attention_kernel");
  if (rc != FR_OK || a.parts == 1) return rc;
  typedef JoinShape<DP> J;
  static_assert(J::kThreads == kAttThreads, "join_parts' workgroups");
  const bool wide = a.rows * a.heads <= 4096;
  hipLaunchKernelGGL((attention_join_kernel<T, DP>), dim3(static_cast<unsigned>(J::blocks(a.rows * a.heads, wide))), dim3(kAttThreads), 0, st, a, wide);
  return check_launch("attention_join_kernel");
}

template <typename T>
int dispatch_attention(const fr_attention_args& a, hipStream_t st) {
  switch (att_dim(a.dim)) {
    case 64: return launch_attention<T, 64>(a, st);
    case 128: return launch_attention<T, 128>(a, st);
    case 192: return launch_attention<T, 192>(a, st);
    default: return launch_attention<T, 256>(a, st);
  }
}

int check_attention_sizes(int64_t B, int64_t rows, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
  FR_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 65536, FR_E_SHAPE, "fr_attention: %lld heads over %lld key heads", (long long)heads,
             (long long)kv_heads);
  FR_REQUIRE(dim >= 8 && dim <= 256 && dim % 8 == 0, FR_E_SHAPE, "fr_attention: head size %lld: a multiple of 8 up to 256", (long long)dim);
  FR_REQUIRE(rows >= 0 && rows < (int64_t(1) << 30) && keys >= 0 && keys < (int64_t(1) << 30), FR_E_SHAPE, "fr_attention: %lld rows, %lld keys: below 2^30",
             (long long)rows, (long long)keys);
  FR_REQUIRE(B >= 0 && B <= (1 << 20) && (rows + B + kAttTile) * heads < (int64_t(1) << 31), FR_E_SHAPE,
             "fr_attention: %lld sequences, %lld rows of %lld heads: up to 2^20 sequences, (rows + sequences + 128) times heads below 2^31", (long long)B, (long long)rows, (long long)heads);
  FR_REQUIRE(att_tiles(B, rows, heads / kv_heads, true) * kv_heads <= kMostBlocks256, FR_E_SHAPE,
             "fr_attention: %lld sequences, %lld rows of %lld heads over %lld: rows times heads / 128 and sequences times key heads, together, up to 2^24", (long long)B, (long long)rows,
             (long long)heads, (long long)kv_heads);
  return FR_OK;
}

}  // namespace
}  // namespace fr

extern "C" int64_t fr_attention_workspace_bytes(int64_t B, int64_t rows, int64_t keys, int64_t heads, int64_t kv_heads, int64_t dim) {
  using namespace fr;
  if (check_attention_sizes(B, rows, keys, heads, kv_heads, dim) != FR_OK) return -1;
  return att_part_bytes(att_parts(B, rows, keys, heads, kv_heads), rows, heads, dim) + att_plan_bytes(B);
}

extern "C" int fr_attention(const fr_attention_args* args, void* stream) {
  using namespace fr;
  FR_REQUIRE(args, FR_E_NULL, "fr_attention: null pointer");
  fr_attention_args a = *args;
  const int rc = check_attention_sizes(a.B, a.rows, a.keys, a.heads, a.kv_heads, a.dim);
  if (rc != FR_OK) return rc;
  FR_REQUIRE(a.dtype == FR_F16 || a.dtype == FR_BF16, FR_E_DTYPE, "fr_attention: dtype %lld not in {f16, bf16}", (long long)a.dtype);
  FR_REQUIRE(a.scale >= 1e-20 && a.scale <= 1e20, FR_E_SHAPE, "fr_attention: scale %g outside [1e-20, 1e20]", a.scale);
  if (a.rows == 0 || (a.B == 0 && !a.fill)) return FR_OK;
  FR_REQUIRE(a.q && a.out && a.cu_q && a.cu_k && (a.keys == 0 || (a.k && a.v)), FR_E_NULL, "fr_attention: null pointer");
  const int64_t strides = a.q_row | a.q_head | a.k_row | a.k_head | a.v_row | a.v_head | a.out_row | a.out_head;
  FR_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out) && strides % 8 == 0, FR_E_ALIGN,
             "fr_attention: q, k, v and out: 16-byte aligned, strides multiples of 8 elements");
  FR_REQUIRE(a.k_row >= 0 && a.k_row < (1 << 23) && a.v_row >= 0 && a.v_row < (1 << 23), FR_E_SHAPE, "fr_attention: keys %lld and values %lld elements apart: below 2^23",
             (long long)a.k_row, (long long)a.v_row);
  const int64_t need = fr_attention_workspace_bytes(a.B, a.rows, a.keys, a.heads, a.kv_heads, a.dim);
  FR_REQUIRE(need == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= need), FR_E_WORKSPACE,
             "fr_attention: workspace of %lld bytes, %lld needed", (long long)a.workspace_bytes, (long long)need);
  const Box q(a.q, a.rows, a.q_row, a.heads, a.q_head, a.dim), out(a.out, a.rows, a.out_row, a.heads, a.out_head, a.dim);
  FR_REQUIRE(!meets_itself(out), FR_E_SHAPE, "fr_attention: out: rows that share memory");
  FR_REQUIRE(is_same(out, q) || !meets(out, q), FR_E_SHAPE, "fr_attention: out shares memory with q, and is not q itself");
  FR_REQUIRE(!meets(out, Box(a.k, a.keys, a.k_row, a.kv_heads, a.k_head, a.dim)) && !meets(out, Box(a.v, a.keys, a.v_row, a.kv_heads, a.v_head, a.dim)), FR_E_SHAPE,
             "fr_attention: out shares memory with k or v");
  a.parts = att_parts(a.B, a.rows, a.keys, a.heads, a.kv_heads);
  a.plan = att_plan_bytes(a.B) ? static_cast<char*>(a.workspace) + att_part_bytes(a.parts, a.rows, a.heads, a.dim) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FR_BF16 ? dispatch_attention<bf16_t>(a, st) : dispatch_attention<f16_t>(a, st);
}

// The MXFP4 mixture-of-experts layer for up to 32 tokens: a stream of the hit experts' weights past a few token rows.
//
// The token rows are the columns of the matrix instruction, whatever expert they go to: column m is token m, so nothing is sorted, and the
// products of all experts meet in one set of sums.  An expert's weights are read once, straight into registers, by the one wavefront that
// multiplies them; its operand for the token rows is read at 16 bytes per token and fragment, lanes behind the last token repeat it.
//
//   front   gating (a wavefront per token or several tokens to one), hidden states to MXFP4
//   gateup  a workgroup per 32 activated features and hit expert, K cut over its four wavefronts (where K is short and the workgroups are many: a
//           wavefront each); SiLU * up, quantised from fp32
//   down    a workgroup per 32 output features and part of the experts' K tiles, cut over its eight wavefronts; the routed weight and the sum
//           over experts in registers, the parts added in order by the workgroup that comes last
//
// For so few tokens that every gateup workgroup can gate and quantise for itself, front is left out: two launches.
#include "gating_core.h"
#include "mxfp4_core.h"
#include "mxfp4_few.h"

namespace fr {
namespace {

constexpr int kFewThreads = 256, kFewWaves = 4;
constexpr int kDownThreads = 512, kDownWaves = 8;

struct MxFew {
  const void* x;
  const void* logits;
  int logits_dtype, M, E, topk, renorm;
  int h_tiles, act_tiles, act_blocks, H;  // K tiles of either product, blocks of 32 activated features, output features
  const unsigned char *w1, *w2;
  int64_t w1_stride, w2_stride;           // bytes of an expert's
  float* topk_w;                          // [M, topk]
  int32_t* ids;
  unsigned char *xq, *act;                // operands: hidden states, activated rows of each hit expert; a row group each
  float* parts;                           // [H / 32][splits][M][32]
  int* arrived;                           // [H / 32], zero before `down`
  int splits;
  void* out;
};

// Tokens t0 .. t1 - 1 of the batch by this workgroup's wavefronts, 64 / G of them at a time each.
template <typename LT, int G, int VPL>
__device__ __forceinline__ void few_gate_as(const LT* logits, int t0, int t1, int waves, int E, int topk, int renorm, float* w, int32_t* ids) {
  constexpr int PER = kWave / G;
  const int lane = threadIdx.x & 63;
  for (int base = t0 + static_cast<int>(threadIdx.x >> 6) * PER; base < t1; base += waves * PER) {
    const int token = base + lane / G;
    const bool live = token < t1;
    const LT* row = logits + static_cast<int64_t>(live ? token : t0) * E;
    gate_token<G, VPL>([&](int e) { return to_float(row[e]); }, live, E, topk, renorm, w + token * topk, ids + token * topk);
  }
}
template <typename LT>
__device__ __forceinline__ void few_gate_typed(const LT* logits, int t0, int t1, int waves, int E, int topk, int renorm, float* w, int32_t* ids) {
  if (E <= 8) few_gate_as<LT, 8, 1>(logits, t0, t1, waves, E, topk, renorm, w, ids);
  else if (E <= 16) few_gate_as<LT, 16, 1>(logits, t0, t1, waves, E, topk, renorm, w, ids);
  else if (E <= 32) few_gate_as<LT, 32, 1>(logits, t0, t1, waves, E, topk, renorm, w, ids);
  else if (E <= 64) few_gate_as<LT, 64, 1>(logits, t0, t1, waves, E, topk, renorm, w, ids);
  else if (E <= 128) few_gate_as<LT, 64, 2>(logits, t0, t1, waves, E, topk, renorm, w, ids);
  else few_gate_as<LT, 64, 4>(logits, t0, t1, waves, E, topk, renorm, w, ids);
}
__device__ __forceinline__ void few_gate(const MxFew& a, int t0, int t1, int waves, float* w, int32_t* ids) {
  if (a.logits_dtype == FR_F32) few_gate_typed(static_cast<const float*>(a.logits), t0, t1, waves, a.E, a.topk, a.renorm, w, ids);
  else if (a.logits_dtype == FR_BF16) few_gate_typed(static_cast<const bf16_t*>(a.logits), t0, t1, waves, a.E, a.topk, a.renorm, w, ids);
  else few_gate_typed(static_cast<const f16_t*>(a.logits), t0, t1, waves, a.E, a.topk, a.renorm, w, ids);
}
// tokens a wavefront gates at a time
__host__ __device__ __forceinline__ int few_gate_tokens(int E) { return E <= 8 ? 8 : E <= 16 ? 4 : E <= 32 ? 2 : 1; }

// A block of 32 elements by four lanes, eight each: their codes; *byte: the block's scale byte.
template <typename T>
__device__ __forceinline__ unsigned few_quant8(const T* from, bool live, unsigned* byte) {
  typedef typename MxVec8<T>::type vec8;
  vec8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (live) v = *reinterpret_cast<const vec8*>(from);
  float f[8];
  unsigned amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = static_cast<float>(v[i]);
    const unsigned m = magnitude(f[i]);
    amax = amax > m ? amax : m;
  }
  unsigned o = static_cast<unsigned>(partner_i32<1>(static_cast<int>(amax)));
  amax = amax > o ? amax : o;
  o = static_cast<unsigned>(partner_i32<2>(static_cast<int>(amax)));
  amax = amax > o ? amax : o;
  *byte = mx_scale_byte(amax);
  return mx_pack8(f, *byte);
}

// Blocks gate_blocks ..: a K tile of all token rows each.  Rows of 256 elements are 32 chunks of 8, a thread each.
template <typename T>
__global__ __launch_bounds__(kFewThreads) void mx_few_front_kernel(MxFew a, int gate_blocks) {
  if (static_cast<int>(blockIdx.x) < gate_blocks) {
    const int per = few_gate_tokens(a.E) * kFewWaves, t0 = blockIdx.x * per;
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < a.H / kMxRows; i += kFewThreads) a.arrived[i] = 0;
    few_gate(a, t0, min(t0 + per, a.M), kFewWaves, a.topk_w, a.ids);
    return;
  }
  const int t = blockIdx.x - gate_blocks, chunk = threadIdx.x & 31, b = chunk >> 2;
  const int k = t * kMxTileK + chunk * 8;
  for (int m = threadIdx.x >> 5; m < a.M; m += kFewThreads / 32) {
    unsigned byte;
    const unsigned o = few_quant8<T>(static_cast<const T*>(a.x) + static_cast<int64_t>(m) * a.H + k, k < a.H, &byte);
    unsigned char* u = a.xq + static_cast<int64_t>(t) * kMxUnit;
    *reinterpret_cast<unsigned*>(u + mx_code_at(m, b) + (chunk & 3) * 4) = o;
    if ((chunk & 3) == 0) u[mx_scale_at(m, b)] = static_cast<unsigned char>(byte);
  }
}

// The hit experts, in order, from the pairs' ids in LDS; all threads, `present` 256 flags.  An id outside [0, E) (a token of NaN
// logits) is no pair.
struct FewHits {
  unsigned long long mask[4];
};
__device__ __forceinline__ void few_present(const int32_t* ids, int n, int E, unsigned char* present, FewHits& hits, int threads) {
  const int tid = threadIdx.x;
  if (tid < 256) present[tid] = 0;
  __syncthreads();
  for (int p = tid; p < n; p += threads)
    if (static_cast<unsigned>(ids[p]) < static_cast<unsigned>(E)) present[ids[p]] = 1;
  __syncthreads();
  if (tid < 256) {
    const unsigned long long m = __ballot(present[tid] != 0);
    if ((tid & 63) == 0) hits.mask[tid >> 6] = m;
  }
  __syncthreads();
}
__device__ __forceinline__ int few_hit_count(const FewHits& hits) {
  return __popcll(hits.mask[0]) + __popcll(hits.mask[1]) + __popcll(hits.mask[2]) + __popcll(hits.mask[3]);
}
// the index-th hit expert (index < few_hit_count, the same in all lanes)
__device__ __forceinline__ int few_hit(const FewHits& hits, int index) {
  for (int w = 0; w < 4; ++w) {
    unsigned long long m = hits.mask[w];
    const int c = __popcll(m);
    if (index < c) {
      for (; index > 0; --index) m &= m - 1;
      return __builtin_amdgcn_readfirstlane(w * 64 + __ffsll(m) - 1);
    }
    index -= c;
  }
  return 0;
}

// A lane's four fragments of K tile k of token row col and their scales.  Rows that the workgroup quantised for itself lie in LDS a tile at
// a time, block after block, the scales behind.
constexpr int kFewRow = 144;  // bytes of a token's K tile in LDS: 128 of codes, 8 of scales, 8 that spread the banks
template <bool OWN>
__device__ __forceinline__ int few_token_rows(const unsigned char* rows, int tiles, int k, int col, int half, mx_frag (&xf)[4]) {
  if constexpr (OWN) {
    const unsigned char* row = rows + (col * tiles + k) * kFewRow;
#pragma unroll
    for (int s = 0; s < 4; ++s) xf[s] = *reinterpret_cast<const mx_frag*>(row + half * 64 + s * 16);
    return *reinterpret_cast<const int*>(row + 128 + half * 4);
  } else {
    const unsigned char* u = rows + static_cast<int64_t>(k) * kMxUnit;
#pragma unroll
    for (int s = 0; s < 4; ++s) xf[s] = *reinterpret_cast<const mx_frag*>(u + s * 1024 + (col + 32 * half) * 16);
    return *reinterpret_cast<const int*>(u + kMxScales + (col + 32 * half) * 4);
  }
}

// SHARED: the workgroup's four wavefronts cut K of one block of 32 activated features, else each has a block to
// itself.
constexpr int kGateupRing = 3;  // K tiles of weights on their way to a wavefront's registers
template <typename T, bool SHARED, bool ROUTE, bool NT>
__global__ __launch_bounds__(kFewThreads) void mx_few_gateup_kernel(MxFew a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ int32_t ids[kFewPairs];
  __shared__ float weights[ROUTE ? kFewPairs : 1];
  __shared__ unsigned char present[256];
  __shared__ FewHits hits;
  __shared__ unsigned tokens_of;  // bit m: token m goes to this workgroup's expert
  extern __shared__ __attribute__((aligned(16))) unsigned char few_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = a.M * a.topk, index = blockIdx.y, blk = SHARED ? blockIdx.x : blockIdx.x * kFewWaves + wave;
  if (tid == 0) tokens_of = 0;
  if constexpr (ROUTE) {
    few_gate(a, 0, a.M, kFewWaves, weights, ids);
  } else {
    for (int p = tid; p < n; p += kFewThreads) ids[p] = a.ids[p];
  }
  __syncthreads();
  few_present(ids, n, a.E, present, hits, kFewThreads);
  if constexpr (ROUTE) {
    if (blockIdx.x == 0 && index == 0) {
      for (int p = tid; p < n; p += kFewThreads) {
        a.topk_w[p] = weights[p];
        a.ids[p] = ids[p];
      }
      for (int i = tid; i < a.H / kMxRows; i += kFewThreads) a.arrived[i] = 0;
    }
  }
  if (index >= few_hit_count(hits)) return;
  const int expert = few_hit(hits, index);
  const int half = lane >> 5;
  const bool stream = blk < a.act_blocks;  // behind the last activated feature: zeros up to a whole K tile
  const int pitch = a.h_tiles * kMxUnit;
  const unsigned char* const w0 = a.w1 + expert * a.w1_stride + static_cast<int64_t>(stream ? blk : 0) * 2 * pitch;
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(w0), 0, -1, 0x00020000);
  const int k0 = SHARED ? wave * a.h_tiles / kFewWaves : 0, k1 = !stream ? k0 : SHARED ? (wave + 1) * a.h_tiles / kFewWaves : a.h_tiles;
  mx_frag wf[kGateupRing][2][4];
  int ws[kGateupRing][2];
  auto load_w = [&](int k, int p) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        wf[p][j][s] = __builtin_bit_cast(mx_frag, __builtin_amdgcn_raw_buffer_load_b128(wr, lane * 16 + s * 1024, j * pitch + k * kMxUnit, NT ? 2 : 0));
      ws[p][j] = __builtin_amdgcn_raw_buffer_load_b32(wr, lane * 4 + kMxScales, j * pitch + k * kMxUnit, NT ? 2 : 0);
    }
  };
#pragma unroll
  for (int p = 0; p < kGateupRing; ++p)
    if (k0 + p < k1) load_w(k0 + p, p);
  for (int p = tid; p < n; p += kFewThreads)
    if (ids[p] == expert) atomicOr(&tokens_of, 1u << (p / a.topk));
  __syncthreads();
  if constexpr (ROUTE) {
    // the expert's tokens, all their chunks of 8 elements over the threads
    const int chunks = a.h_tiles * 32, all = __popc(tokens_of) * chunks;
    for (int i = tid; i < all; i += kFewThreads) {
      const int r = i / chunks, c = i - r * chunks, t = c >> 5, b = (c & 31) >> 2;
      unsigned left = tokens_of;
      for (int q = 0; q < r; ++q) left &= left - 1;
      const int m = __ffs(left) - 1;
      unsigned byte;
      const unsigned o = few_quant8<T>(static_cast<const T*>(a.x) + static_cast<int64_t>(m) * a.H + c * 8, c * 8 < a.H, &byte);
      unsigned char* row = few_lds + (m * a.h_tiles + t) * kFewRow;
      *reinterpret_cast<unsigned*>(row + b * 16 + (c & 3) * 4) = o;
      if ((c & 3) == 0) row[128 + b] = static_cast<unsigned char>(byte);
    }
    __syncthreads();
  }
  // the lane's token; one that goes elsewhere reads a row that is read anyway (a hit expert has a token)
  const bool mine = tokens_of >> (lane & 31) & 1;
  const int col = mine ? lane & 31 : __ffs(tokens_of) - 1;
  f32x16 acc[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
  for (int kk = k0; kk < k1; kk += kGateupRing) {
#pragma unroll
    for (int p = 0; p < kGateupRing; ++p) {
      const int k = kk + p;
      if (k < k1) {
        mx_frag xf[4];
        const int xs = few_token_rows<ROUTE>(ROUTE ? few_lds : a.xq, a.h_tiles, k, col, half, xf);
        mx_each<0, 4>([&](auto S) {
          constexpr int s = decltype(S)::value;
          acc[0] = mx_mfma<s>(wf[p][0][s], ws[p][0], xf[s], xs, acc[0]);
          acc[1] = mx_mfma<s>(wf[p][1][s], ws[p][1], xf[s], xs, acc[1]);
        });
        if (k + kGateupRing < k1) load_w(k + kGateupRing, p);
      }
    }
  }
  if constexpr (SHARED) {  // the wavefronts' sums meet in the first one
    f32x4* const red = reinterpret_cast<f32x4*>(few_lds);
    __syncthreads();  // the token rows have been read
    if (wave > 0) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          red[((wave - 1) * 8 + j * 4 + q) * 64 + lane] = f32x4{acc[j][q * 4], acc[j][q * 4 + 1], acc[j][q * 4 + 2], acc[j][q * 4 + 3]};
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int v = 0; v < kFewWaves - 1; ++v)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 t = red[(v * 8 + j * 4 + q) * 64 + lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][q * 4 + r] += t[r];
        }
  }
  float v[16];
  unsigned amax = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    v[r] = mx_silu_mul(acc[0][r], acc[1][r]);
    const unsigned m = magnitude(v[r]);
    amax = amax > m ? amax : m;
  }
  const unsigned byte = mx_scale_byte(mx_pair_max(amax));
  unsigned char* const act = a.act + (static_cast<int64_t>(index) * a.act_tiles + (blk >> 3)) * kMxUnit;
  if (mine) {
    *reinterpret_cast<uint2*>(act + mx_code_at(lane & 31, blk & 7) + half * 8) = uint2{mx_pack8(v, byte), mx_pack8(v + 8, byte)};
    if (half == 0) act[mx_scale_at(lane & 31, blk & 7)] = static_cast<unsigned char>(byte);
  }
#endif
}

constexpr int kDownRing = 4;
constexpr int kDownLane = 17;  // floats of a lane's sums in LDS: 16 and one that spreads the banks
constexpr int kDownLds = kDownWaves * 64 * kDownLane * 4;
template <typename T, bool NT>
__global__ __launch_bounds__(kDownThreads) void mx_few_down_kernel(MxFew a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ int32_t ids[kFewPairs];
  __shared__ float weights[kFewPairs];
  __shared__ unsigned char present[256];
  __shared__ FewHits hits;
  __shared__ int last;
  extern __shared__ __attribute__((aligned(16))) unsigned char few_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = a.M * a.topk, unit = blockIdx.x, split = blockIdx.y, tiles = a.act_tiles;
  for (int p = tid; p < n; p += kDownThreads) {
    ids[p] = a.ids[p];
    weights[p] = a.topk_w[p];
  }
  __syncthreads();
  few_present(ids, n, a.E, present, hits, kDownThreads);
  // K tiles of all hit experts in a row; this wavefront's part of them
  const int total = few_hit_count(hits) * tiles, parts = a.splits * kDownWaves, part = split * kDownWaves + wave;
  const int i0 = static_cast<int>(static_cast<int64_t>(part) * total / parts), i1 = static_cast<int>(static_cast<int64_t>(part + 1) * total / parts);
  const int half = lane >> 5, pitch = tiles * kMxUnit;
  const int col = min(lane & 31, a.M - 1);
  f32x16 sum, acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) sum[r] = acc[r] = 0.f;
  mx_frag wf[kDownRing][4], xf[kDownRing][4];
  int ws[kDownRing], xs[kDownRing];
  // next tile to load: its expert's index, K tile, expert
  int li = i0 / tiles, lk = i0 - li * tiles, le = i0 < i1 ? few_hit(hits, li) : 0;
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(a.act, 0, -1, 0x00020000);
  auto load = [&](int p) {
    const unsigned char* w = a.w2 + le * a.w2_stride + static_cast<int64_t>(unit) * pitch;
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(w), 0, -1, 0x00020000);
#pragma unroll
    for (int s = 0; s < 4; ++s) wf[p][s] = __builtin_bit_cast(mx_frag, __builtin_amdgcn_raw_buffer_load_b128(wr, lane * 16 + s * 1024, lk * kMxUnit, NT ? 2 : 0));
    ws[p] = __builtin_amdgcn_raw_buffer_load_b32(wr, lane * 4 + kMxScales, lk * kMxUnit, NT ? 2 : 0);
    const int at = li * pitch + lk * kMxUnit;  // below 2^31, see mx_few_fits
#pragma unroll
    for (int s = 0; s < 4; ++s) xf[p][s] = __builtin_bit_cast(mx_frag, __builtin_amdgcn_raw_buffer_load_b128(xr, (col + 32 * half) * 16 + s * 1024, at, 0));
    xs[p] = __builtin_amdgcn_raw_buffer_load_b32(xr, (col + 32 * half) * 4 + kMxScales, at, 0);
    if (++lk == tiles) {
      lk = 0;
      ++li;
      if (li * tiles < i1) le = few_hit(hits, li);
    }
  };
#pragma unroll
  for (int p = 0; p < kDownRing; ++p)
    if (i0 + p < i1) load(p);
  int ck = i0 % tiles, ci = i0 / tiles;  // tile being multiplied
  auto flush = [&]() {  // an expert's part of the sums, weighted, to those of its tokens
    const int e = few_hit(hits, ci);
    float w = 0.f;
    bool mine = false;
    for (int j = 0; j < a.topk; ++j)
      if (ids[col * a.topk + j] == e) {
        w += weights[col * a.topk + j];
        mine = true;
      }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      sum[r] += mine ? acc[r] * w : 0.f;
      acc[r] = 0.f;
    }
  };
  for (int ii = i0; ii < i1; ii += kDownRing) {
#pragma unroll
    for (int p = 0; p < kDownRing; ++p) {
      const int i = ii + p;
      if (i < i1) {
        mx_each<0, 4>([&](auto S) {
          constexpr int s = decltype(S)::value;
          acc = mx_mfma<s>(wf[p][s], ws[p], xf[p][s], xs[p], acc);
        });
        if (i + kDownRing < i1) load(p);
        if (++ck == tiles || i + 1 == i1) {
          flush();
          ck = 0;
          ++ci;
        }
      }
    }
  }
  float* const red = reinterpret_cast<float*>(few_lds);
  const int outs = a.M * 32;
  float* const mine = a.parts + (static_cast<int64_t>(unit) * a.splits + split) * outs;
#pragma unroll
  for (int r = 0; r < 16; ++r) red[(wave * 64 + lane) * kDownLane + r] = sum[r];
  __syncthreads();
  for (int o = tid; o < outs; o += kDownThreads) {
    const int m = o >> 5, f = o & 31;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWaves; ++w) s += red[(w * 64 + m + 32 * (f >> 4)) * kDownLane + (f & 15)];
    if (a.splits == 1) static_cast<T*>(a.out)[static_cast<int64_t>(m) * a.H + unit * 32 + f] = static_cast<T>(s);
    else __hip_atomic_store(mine + o, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.splits == 1) return;
  // The part that comes last adds all of them, in order.  XCDs have an L2 each: the parts are written through and read past it, an access
  // at a time (agent scope), and every wavefront's stores have been acknowledged before the barrier ahead of the count.  Fences, which
  // write back and invalidate the whole L2 for a few KB, took 40 us here.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) last = __hip_atomic_fetch_add(a.arrived + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.splits - 1;
  __syncthreads();
  if (!last) return;
  for (int o = tid; o < outs; o += kDownThreads) {
    const int m = o >> 5, f = o & 31;
    float s = 0.f;
    for (int p = 0; p < a.splits; ++p)
      s += __hip_atomic_load(a.parts + (static_cast<int64_t>(unit) * a.splits + p) * outs + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    static_cast<T*>(a.out)[static_cast<int64_t>(m) * a.H + unit * 32 + f] = static_cast<T>(s);
  }
#endif
}

constexpr int kLinearRing = 4;
// The product of a matrix with up to 32 U token rows: a workgroup per 32 output features, K cut over its eight wavefronts.
// OWN (U = 1): the workgroup quantises the rows into LDS itself, else xq is the operand.
struct MxFewLinear {
  const void* x;
  int64_t ldx;
  const unsigned char *xq, *w;
  int M, K, k_tiles;
  int64_t N;
  void* out;
};
template <typename T, int U, bool OWN, bool NT>
__global__ __launch_bounds__(kDownThreads) void mx_few_linear_kernel(MxFewLinear a) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(16))) unsigned char few_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = blockIdx.x;
  const int half = lane >> 5;
  const int k0 = wave * a.k_tiles / kDownWaves, k1 = (wave + 1) * a.k_tiles / kDownWaves;
  const __amdgpu_buffer_rsrc_t wr =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(a.w + unit * a.k_tiles * kMxUnit), 0, -1, 0x00020000);
  mx_frag wf[kLinearRing][4];
  int ws[kLinearRing];
  auto load_w = [&](int k, int p) {
#pragma unroll
    for (int s = 0; s < 4; ++s) wf[p][s] = __builtin_bit_cast(mx_frag, __builtin_amdgcn_raw_buffer_load_b128(wr, lane * 16 + s * 1024, k * kMxUnit, NT ? 2 : 0));
    ws[p] = __builtin_amdgcn_raw_buffer_load_b32(wr, lane * 4 + kMxScales, k * kMxUnit, NT ? 2 : 0);
  };
#pragma unroll
  for (int p = 0; p < kLinearRing; ++p)
    if (k0 + p < k1) load_w(k0 + p, p);
  if constexpr (OWN) {
    const int per = a.k_tiles * 32, chunks = a.M * per;
    for (int c = tid; c < chunks; c += kDownThreads) {
      const int m = c / per, i = c - m * per, b = (i & 31) >> 2;
      unsigned byte;
      const unsigned o = few_quant8<T>(static_cast<const T*>(a.x) + m * a.ldx + i * 8, i * 8 < a.K, &byte);
      unsigned char* row = few_lds + (m * a.k_tiles + (i >> 5)) * kFewRow;
      *reinterpret_cast<unsigned*>(row + b * 16 + (i & 3) * 4) = o;
      if ((i & 3) == 0) row[128 + b] = static_cast<unsigned char>(byte);
    }
    __syncthreads();
  }
  f32x16 acc[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[u][r] = 0.f;
  for (int kk = k0; kk < k1; kk += kLinearRing) {
#pragma unroll
    for (int p = 0; p < kLinearRing; ++p) {
      const int k = kk + p;
      if (k < k1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          mx_frag xf[4];
          const int col = min(lane & 31, a.M - 1 - u * 32);  // lanes behind the last row repeat it (a row group has one at least)
          const int xs = few_token_rows<OWN>(OWN ? few_lds : a.xq + static_cast<int64_t>(u) * a.k_tiles * kMxUnit, a.k_tiles, k, col, half, xf);
          mx_each<0, 4>([&](auto S) {
            constexpr int s = decltype(S)::value;
            acc[u] = mx_mfma<s>(wf[p][s], ws[p], xf[s], xs, acc[u]);
          });
        }
        if (k + kLinearRing < k1) load_w(k + kLinearRing, p);
      }
    }
  }
  float* const red = reinterpret_cast<float*>(few_lds);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    __syncthreads();  // the token rows, or the last row group's sums, have been read
#pragma unroll
    for (int r = 0; r < 16; ++r) red[(wave * 64 + lane) * kDownLane + r] = acc[u][r];
    __syncthreads();
    for (int o = tid; o < min(a.M - u * 32, 32) * 32; o += kDownThreads) {
      const int m = o >> 5, f = o & 31;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kDownWaves; ++w) s += red[(w * 64 + m + 32 * (f >> 4)) * kDownLane + (f & 15)];
      if (unit * 32 + f < a.N) static_cast<T*>(a.out)[(m + u * 32) * a.N + unit * 32 + f] = static_cast<T>(s);
    }
  }
#endif
}

// Parts a unit's K tiles are cut into: enough workgroups for the card, as long as a wavefront has four tiles - the parts meet in memory, which
// takes longer than a few tiles more.
int few_splits(int64_t M, int64_t H, int64_t F, int E, int topk) {
  const int64_t n = M * topk, experts = n < E ? n : E;
  const int64_t card = 256 / (H / kMxRows), work = experts * mx_tiles(F) / (4 * kDownWaves);
  const int64_t s = card < work ? card : work;
  return static_cast<int>(s < 1 ? 1 : s > 8 ? 8 : s);
}

constexpr int kGateupLds = (kFewWaves - 1) * 8 * 64 * 16;
constexpr int kRouteLds = 56 * 1024;  // with the kernels' static arrays below the limit that needs no set-up
// Every gateup workgroup gates all tokens and quantises its expert's rows: a launch of 4 us less for up to 6 us more in each workgroup.  Two launches /
// three, us: H = 1024, F = 3584, 8 experts, top-2, 1 token 15.5 / 18.6, 2 15.0 / 17.9, 5 25.1 / 25.9; H = 4096, F = 14336 4 96 / 97, 8 133 / 125;
// H = 2048, F = 1408, 64 experts, top-6 1 19.0 / 20.3, 4 26.3 / 23.2.
bool few_routes(int64_t M, int64_t H, int E) { return M <= (E <= 32 ? 4 : 2) && M * mx_tiles(H) * kFewRow <= kRouteLds; }

// Every workgroup of the linear product quantises the rows.
bool few_quantises(int64_t M, int64_t K) { return M <= 4 && M * mx_tiles(K) * kFewRow <= kRouteLds; }

}  // namespace

bool mx_few_fits(int64_t M, int64_t F, int E, int topk) {
  const int64_t n = M * topk, experts = n < E ? n : E;
  return M >= 1 && M <= kFewTokens && n <= kFewPairs && experts * mx_tiles(F) * kMxUnit < (int64_t(1) << 31);
}

int64_t mx_few_workspace(void* ws, int64_t M, int64_t H, int64_t F, int E, int topk, MxFewScratch* s) {
  MxBump b{static_cast<unsigned char*>(ws)};
  const int64_t n = M * topk, experts = n < E ? n : E;
  s->topk_w = b.take<float>(n);
  s->ids = b.take<int32_t>(n);
  s->arrived = b.take<int>(H / kMxRows);
  s->parts = b.take<float>(static_cast<int64_t>(few_splits(M, H, F, E, topk)) * M * H);
  s->xq = b.take<unsigned char>(mx_tiles(H) * kMxUnit);
  s->act = b.take<unsigned char>(experts * mx_tiles(F) * kMxUnit);
  return b.at;
}

namespace {
template <typename T, bool NT>
int launch_few(const MxFew& a, hipStream_t st) {
  const int n = a.M * a.topk, experts = n < a.E ? n : a.E;
  const dim3 threads(kFewThreads), shared(static_cast<unsigned>(a.act_tiles * 8), static_cast<unsigned>(experts));
  if (few_routes(a.M, a.H, a.E)) {
    const int rows = a.M * a.h_tiles * kFewRow, lds = rows > kGateupLds ? rows : kGateupLds;
    hipLaunchKernelGGL((mx_few_gateup_kernel<T, true, true, NT>), shared, threads, lds, st, a);
  } else {
    const int gate_blocks = static_cast<int>(ceil_div(static_cast<int64_t>(a.M), int64_t(few_gate_tokens(a.E)) * kFewWaves));
    hipLaunchKernelGGL((mx_few_front_kernel<T>), dim3(static_cast<unsigned>(gate_blocks + a.h_tiles)), threads, 0, st, a, gate_blocks);
    const int rc = check_launch("mx_few_front_kernel");
    if (rc != FR_OK) return rc;
    const dim3 apart(static_cast<unsigned>(a.act_tiles * 8 / kFewWaves), static_cast<unsigned>(experts));
    // A block per wavefront where K is short: no sums to join.  H = 1024, F = 3584, 8 experts, 5 tokens 10.3 -> 7.8 us; H = 2048, F = 1408,
    // 64 experts, 32 tokens 25.6 -> 20.5.
    const bool alone = a.h_tiles <= 8 && static_cast<int64_t>(a.act_blocks) * experts >= 512;
    if (alone) hipLaunchKernelGGL((mx_few_gateup_kernel<T, false, false, NT>), apart, threads, 0, st, a);
    else hipLaunchKernelGGL((mx_few_gateup_kernel<T, true, false, NT>), shared, threads, kGateupLds, st, a);
  }
  const int rc = check_launch("mx_few_gateup_kernel");
  if (rc != FR_OK) return rc;
  const dim3 down(static_cast<unsigned>(a.H / kMxRows), static_cast<unsigned>(a.splits));
  hipLaunchKernelGGL((mx_few_down_kernel<T, NT>), down, dim3(kDownThreads), kDownLds, st, a);
  return check_launch("mx_few_down_kernel");
}
}  // namespace

int mx_few_layer(const void* x, int dtype, const void* w1, const void* w2, const void* logits, int logits_dtype, int64_t M, int64_t H,
                 int64_t F, int E, int topk, int renorm, void* out, void* workspace, hipStream_t st) {
  MxFewScratch s;
  mx_few_workspace(workspace, M, H, F, E, topk, &s);
  MxFew a = {};
  a.x = x;
  a.logits = logits;
  a.logits_dtype = logits_dtype;
  a.M = static_cast<int>(M);
  a.E = E;
  a.topk = topk;
  a.renorm = renorm;
  a.h_tiles = static_cast<int>(mx_tiles(H));
  a.act_tiles = static_cast<int>(mx_tiles(F));
  a.act_blocks = static_cast<int>(F / kMxBlock);
  a.H = static_cast<int>(H);
  a.w1 = static_cast<const unsigned char*>(w1);
  a.w2 = static_cast<const unsigned char*>(w2);
  a.w1_stride = mx_groups(2 * F) * a.h_tiles * kMxUnit;
  a.w2_stride = mx_groups(H) * a.act_tiles * kMxUnit;
  a.topk_w = s.topk_w;
  a.ids = s.ids;
  a.xq = s.xq;
  a.act = s.act;
  a.parts = s.parts;
  a.arrived = s.arrived;
  a.splits = few_splits(M, H, F, E, topk);
  a.out = out;
  const int64_t n = M * topk, experts = n < E ? n : E;
  if (mx_streams(experts * (a.w1_stride + a.w2_stride))) return dtype == FR_BF16 ? launch_few<bf16_t, true>(a, st) : launch_few<f16_t, true>(a, st);
  return dtype == FR_BF16 ? launch_few<bf16_t, false>(a, st) : launch_few<f16_t, false>(a, st);
}

bool mx_few_linear_fits(int64_t M, int64_t N) { return M <= 32 || (M <= 128 && mx_groups(N) <= 512); }

int64_t mx_few_linear_workspace(int64_t M, int64_t K) { return few_quantises(M, K) ? 0 : mx_groups(M) * mx_tiles(K) * kMxUnit; }

namespace {
template <typename T, bool NT>
void launch_few_linear(const MxFewLinear& a, bool own, hipStream_t st) {
  const int rows = own ? a.M * a.k_tiles * kFewRow : 0, lds = rows > kDownLds ? rows : kDownLds;
  const dim3 grid(static_cast<unsigned>(mx_groups(a.N))), threads(kDownThreads);
  if (own) hipLaunchKernelGGL((mx_few_linear_kernel<T, 1, true, NT>), grid, threads, lds, st, a);
  else if (a.M <= 32) hipLaunchKernelGGL((mx_few_linear_kernel<T, 1, false, NT>), grid, threads, lds, st, a);
  else if (a.M <= 64) hipLaunchKernelGGL((mx_few_linear_kernel<T, 2, false, NT>), grid, threads, lds, st, a);
  else if (a.M <= 96) hipLaunchKernelGGL((mx_few_linear_kernel<T, 3, false, NT>), grid, threads, lds, st, a);
  else hipLaunchKernelGGL((mx_few_linear_kernel<T, 4, false, NT>), grid, threads, lds, st, a);
}
}  // namespace

int mx_few_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* w, int64_t N, void* out, void* workspace,
                  hipStream_t st) {
  MxFewLinear a = {};
  a.x = x;
  a.ldx = ldx;
  a.xq = static_cast<const unsigned char*>(workspace);
  a.w = static_cast<const unsigned char*>(w);
  a.M = static_cast<int>(M);
  a.K = static_cast<int>(K);
  a.k_tiles = static_cast<int>(mx_tiles(K));
  a.N = N;
  a.out = out;
  const bool own = few_quantises(M, K);
  if (!own) {
    const int rc = mx_quant_tiled(x, dtype, M, K, ldx, mx_groups(M), MxGather{}, false, workspace, st);
    if (rc != FR_OK) return rc;
  }
  if (mx_streams(mx_groups(N) * a.k_tiles * kMxUnit)) dtype == FR_BF16 ? launch_few_linear<bf16_t, true>(a, own, st) : launch_few_linear<f16_t, true>(a, own, st);
  else dtype == FR_BF16 ? launch_few_linear<bf16_t, false>(a, own, st) : launch_few_linear<f16_t, false>(a, own, st);
  return check_launch("mx_few_linear_kernel");
}

}  // namespace fr

// Products of MXFP4 operands on gfx950: a matrix (linear) and the two grouped products of the mixture-of-experts layer.
//
//   C[m, f] = sum_k X[m, k] W[f, k],   both operands e2m1 codes with a power-of-two scale per 32 elements of k, fp32 sums.
//
// A workgroup of four wavefronts computes a token tile of up to kMxMaxUnits row groups (32 rows each) x 256 weight rows, or 128 where
// workgroups are few: a wavefront holds J = 2 units of weight rows, or one, against all token rows.
#include "mxfp4_few.h"

namespace fr {
namespace {

constexpr int kMxThreads = 256;
// MX_PART: the down product, K cut over workgroups; MX_PAST: a linear product whose whole lines are written past the caches.  (A flag of the
// call would not do: the compiler makes one plain store of both kinds.)
enum { MX_LINEAR = 0, MX_SILU = 1, MX_DOWN = 2, MX_PART = 3, MX_PAST = 4 };
template <int EPI>
constexpr bool kMxLinear = EPI == MX_LINEAR || EPI == MX_PAST;
template <int EPI>
constexpr bool kMxPairs = EPI == MX_DOWN || EPI == MX_PART;  // results are weighted rows of pairs

// What a workgroup multiplies: row groups group .. group + units - 1 of an expert's.
struct MxSpan {
  int group, units, expert;
};

struct MxArgs {
  const unsigned char* x;  // operand of the token rows
  const unsigned char* w;  // operand(s) of the weights
  int64_t w_stride;        // bytes of an expert's weights
  int k_tiles;
  int w_groups;            // row groups of an expert's weights
  int f_tiles;             // tiles of 4 J weight row groups
  // grouped: the tile list; else tiles of kMxMaxUnits row groups out of x_groups
  const int* tile_count;
  const MxTile* tiles;
  int x_groups;
  // MX_SILU: operand of the activated rows, its tiles along K, blocks of 32 activated features
  unsigned char* act;
  int act_tiles, act_blocks;
  // MX_DOWN, MX_PART: rows of the pairs
  const int32_t* sorted;
  const float* topk_w;
  int n_pairs;
  float* rows;             // [slices][n_pairs, N]; MX_DOWN: one slice
  // MX_LINEAR, MX_PAST
  void* out;
  int64_t ldo;
  int64_t M;
  int N;               // columns of rows / out
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// A lane holds 16 consecutive features of a row and feature unit, so its stores fill lines in instructions of 64 scattered 16-byte pieces.  Where a
// wavefront has 64 features they are turned in LDS (32 rows of 64 features, a row group at a time) and leave as whole lines: 8192 x 12288 x 4096 213 -> 206 us,
// down product of 64 experts, H = 2048, F = 1408, 8192 tokens 207 -> 174, of 8, H = 4096, F = 14336, 16384 1112 -> 1067; K slices would lose, 50 tokens on 8
// experts, H = 1024, F = 3584 6.7 -> 7.3.  A product larger than the caches keep goes past them, 206 -> 191 (286 in pieces).
// A product whose N is no multiple of 8 is stored value by value: 4096 x 12287 x 4096 254 us, 12288 99.
template <int EPI, int J>
constexpr bool kMxTurned = J == 2 && (kMxLinear<EPI> || EPI == MX_DOWN);
template <int EPI>
constexpr int kMxTurnPieces = kMxPairs<EPI> ? 16 : 8;  // 16-byte pieces of a row: fp32, or a 2-byte type
template <int EPI>
constexpr int kMxTurnPitch = kMxTurnPieces<EPI> * 16 + 16;

template <typename T, int EPI, int U, int J>
__device__ __forceinline__ void mx_epilogue(const MxArgs& a, const MxSpan& t, int f, int wave, int lane, unsigned char* lds, f32x16 (&acc)[U][J]);

// Token rows through LDS (every wavefront reads all of them), weights from memory to registers (no other wavefront reads them).  A
// ring of kMxSlots K tiles of token rows and two of weights are under way.  All loads are spread between the MFMAs, a row
// group's two at a time: issued in one run per K tile they held up the MFMAs behind them (8 experts, H = 4096, F = 14336, 16384 tokens: gate/up
// 1966 -> 1830 us, down 1048 -> 1003).
//
// 128 x 256 outputs and two workgroups per CU, whose prologues and epilogues meet the other's MFMAs.  256 x 256 by one workgroup
// of four wavefronts moves a third less through L1 but stalls more: 2098 / 1039 us.  A stream of these MFMAs alone reaches 6.4 PFLOP/s (the
// part lowers its clock to 1.67 GHz for it); without any load, on data that is there, this loop reaches 5.1 to 5.5.
constexpr int kMxSlots = 4;
template <typename T, int EPI, int U, int J, bool NT>
__device__ __forceinline__ void mx_tile(const MxArgs& a, const MxSpan& t, int f, unsigned char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) void* lptr_t;
  constexpr int SLOT = U * 4096 + 1024, RING = 2, AUX = NT ? 2 : 0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wg = min((f * 4 + wave) * J, a.w_groups - 1), wg1 = min(wg + 1, a.w_groups - 1);
  const int pitch = a.k_tiles * kMxUnit;
  // the workgroup's K tiles: all of them, or slice blockIdx.y of gridDim.y
  const int k_first = EPI == MX_PART ? static_cast<int>(blockIdx.y) * a.k_tiles / static_cast<int>(gridDim.y) : 0;
  const int k_end = EPI == MX_PART ? (static_cast<int>(blockIdx.y) + 1) * a.k_tiles / static_cast<int>(gridDim.y) : a.k_tiles;
  const int last = k_end - k_first - 1;
  const unsigned char* const w0 = a.w + t.expert * a.w_stride + static_cast<int64_t>(wg) * pitch + k_first * kMxUnit;
  const unsigned char* const x0 = a.x + static_cast<int64_t>(t.group) * pitch + k_first * kMxUnit;
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(x0), 0, -1, 0x00020000);
  // a K tile of token rows: wavefront w takes fragment w of every row group and a copy of all their scales
  const int code_off = lane * 16, scale_off = min(lane >> 4, U - 1) * pitch + kMxScales + (lane & 15) * 16;
  f32x16 acc[U][J];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[u][j][r] = 0.f;
  mx_frag wf[RING][J][4], xf[U];  // weights of K tile k in part k % RING
  int ws[RING][J], xs[2][U];
  auto load_x1 = [&](int k, int u) {  // u == U: the scales
    const int kc = min(k, last);
    unsigned char* slot = lds + (k & (kMxSlots - 1)) * SLOT;
    if (u < U) __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lptr_t)(slot + u * 4096 + wave * 1024), 16, code_off, u * pitch + kc * kMxUnit + wave * 1024, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lptr_t)(slot + U * 4096), 16, scale_off, kc * kMxUnit, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto load_x = [&](int k) {
#pragma unroll
    for (int u = 0; u <= U; ++u) load_x1(k, u);
  };
  const __amdgpu_buffer_rsrc_t r0 = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(w0), 0, -1, 0x00020000);
  const int d01 = (wg1 - wg) * pitch;
  auto load_w1 = [&](int k, int s, int p, int j) {
    const int kc = min(k, last);
    wf[p][j][s] = __builtin_bit_cast(mx_frag, __builtin_amdgcn_raw_buffer_load_b128(r0, lane * 16 + s * 1024, (j ? d01 : 0) + kc * kMxUnit, AUX));
  };
  auto load_w = [&](int k, int s, int p) {
#pragma unroll
    for (int j = 0; j < J; ++j) load_w1(k, s, p, j);
  };
  auto load_ws = [&](int k, int p) {
    const int kc = min(k, last);
#pragma unroll
    for (int j = 0; j < J; ++j) ws[p][j] = __builtin_amdgcn_raw_buffer_load_b32(r0, lane * 4 + kMxScales, (j ? d01 : 0) + kc * kMxUnit, AUX);
  };
  auto read_x = [&](int k, int s, int u) {
    return *reinterpret_cast<const mx_frag*>(lds + (k & (kMxSlots - 1)) * SLOT + u * 4096 + s * 1024 + lane * 16);
  };
  auto read_xs = [&](int k, int u) { return *reinterpret_cast<const int*>(lds + (k & (kMxSlots - 1)) * SLOT + U * 4096 + u * 256 + lane * 4); };
  load_x(0);
  load_x(1);
  load_x(2);
#pragma unroll
  for (int p = 0; p < RING; ++p) {
    if (p < RING - 1) load_ws(p, p);
#pragma unroll
    for (int s = 0; s < (p < RING - 1 ? 4 : 3); ++s) load_w(p, s, p);
  }
  __builtin_amdgcn_sched_barrier(0);
  // K tile 0 of the token rows has landed: 2 (U + 1) + 8 J loads are newer, of which J, of K tile 1, are waited for too
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * (U + 1) + 5 * J * RING - 3 * J) : "memory");
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    xf[u] = read_x(0, 0, u);
    xs[0][u] = read_xs(0, u);
  }
  for (int k0 = 0; k0 <= last; k0 += RING) {
#pragma unroll
    for (int p = 0; p < RING; ++p) {
      const int k = k0 + p;
      if (p == 0 || k <= last) {
        mx_each<0, 4>([&](auto S) {
          constexpr int s = decltype(S)::value;
          if constexpr (s == 3) {
            // K tile k + 1 of the token rows has landed, everybody's loads of it behind the barrier (this wavefront has issued U + 1 of
            // k + 2 and 9 J of weights since, the oldest 2 J of them fragment 3 and scales of K tile k, which the MFMAs below need); and slot
            // (k + 3) & 3, that of k - 1, has been read by everybody.
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(U + 1 + 7 * J) : "memory");
            __builtin_amdgcn_s_barrier();
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < J; ++j) acc[u][j] = mx_mfma<s>(wf[p][j][s], ws[p][j], xf[u], xs[p & 1][u], acc[u][j]);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (s < 3) xf[u] = read_x(k, s + 1, u);
            else {
              xf[u] = read_x(k + 1, 0, u);
              xs[(p + 1) & 1][u] = read_xs(k + 1, u);
              load_x1(k + 3, u);
            }
            // weights of the step before: its fragments are free
#pragma unroll
            for (int j = u; j < J; j += U) {
              if constexpr (s > 0) {
                load_w1(k + RING, s - 1, p, j);
              } else {
                load_w1(k + RING - 1, 3, (p + RING - 1) % RING, j);
                if (j == J - 1) load_ws(k + RING - 1, (p + RING - 1) % RING);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if constexpr (s == 3) load_x1(k + 3, U);
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load of this workgroup's is under way to LDS
  if constexpr (kMxTurned<EPI, J>) __syncthreads();  // nor does any wavefront still read there: it is the epilogue's
  mx_epilogue<T, EPI, U, J>(a, t, f, wave, lane, lds + wave * (32 * kMxTurnPitch<EPI>), acc);
#endif
}

// acc[u][j]: the lane's 16 consecutive features of token row `lane % 32` of row group u.
template <typename T, int EPI, int U, int J>
__device__ __forceinline__ void mx_epilogue(const MxArgs& a, const MxSpan& t, int f, int wave, int lane, unsigned char* lds, f32x16 (&acc)[U][J]) {
  const int wg = (f * 4 + wave) * J, col = lane & 31, half = lane >> 5;
  if constexpr (EPI == MX_SILU) {
    const int blk = f * 4 + wave;  // of 32 activated features; the operand's last K tile is filled up with zeros
    const bool pad = blk >= a.act_blocks;
    unsigned char* unit = a.act + (static_cast<int64_t>(t.group) * a.act_tiles + (blk >> 3)) * kMxUnit;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const f32x16 g = acc[u][0], up = acc[u][1];
      float v[16];
      unsigned amax = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        v[r] = pad ? 0.f : mx_silu_mul(g[r], up[r]);
        const unsigned m = magnitude(v[r]);
        amax = amax > m ? amax : m;
      }
      const unsigned byte = mx_scale_byte(mx_pair_max(amax));
      const uint2 o = {mx_pack8(v, byte), mx_pack8(v + 8, byte)};
      *reinterpret_cast<uint2*>(unit + mx_code_at(col, blk & 7) + half * 8) = o;
      if (half == 0) unit[mx_scale_at(col, blk & 7)] = static_cast<unsigned char>(byte);
      unit += static_cast<int64_t>(a.act_tiles) * kMxUnit;
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      constexpr int PIECES = kMxTurnPieces<EPI>, PITCH = kMxTurnPitch<EPI>;
      const int64_t slot = static_cast<int64_t>(t.group + u) * kMxRows + col;
      u32x4* const turn = reinterpret_cast<u32x4*>(lds + col * PITCH + half * (PIECES * 4));  // + j * PIECES / 2: the lane's pieces of unit j
      // rows of the group from LDS to `to(row)`, the address of their 64 features or null
      auto turned = [&](auto to) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < PIECES / 2; ++i) {
          const int r = i * (64 / PIECES) + lane / PIECES;
          const u32x4 v = *reinterpret_cast<const u32x4*>(lds + r * PITCH + lane % PIECES * 16);
          u32x4* const row = to(r);
          if (row) {
            if constexpr (EPI == MX_PAST) __builtin_nontemporal_store(v, row + lane % PIECES);
            else row[lane % PIECES] = v;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      };
      if constexpr (kMxPairs<EPI>) {
        // Weighted rows stay in fp32 until the pairs are summed.
        const bool whole = kMxTurned<EPI, J> && wg + 1 < a.w_groups;
        const int pair = a.sorted[slot];
        const bool live = pair < a.n_pairs;
        const float s = live ? a.topk_w[pair] : 0.f;
        float* const rows = a.rows + (EPI == MX_PART ? static_cast<int64_t>(blockIdx.y) * a.n_pairs * a.N : 0) + wg * 32;
        if (live) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            if (wg + j < a.w_groups) {
              u32x4* const row = whole ? turn + j * (PIECES / 2) : reinterpret_cast<u32x4*>(rows + static_cast<int64_t>(pair) * a.N + j * 32 + half * 16);
#pragma unroll
              for (int r = 0; r < 16; r += 4)
                row[r / 4] = __builtin_bit_cast(u32x4, f32x4{acc[u][j][r] * s, acc[u][j][r + 1] * s, acc[u][j][r + 2] * s, acc[u][j][r + 3] * s});
            }
          }
        }
        if (whole)
          turned([&](int r) {
            const int p = __shfl(pair, r);
            return p < a.n_pairs ? reinterpret_cast<u32x4*>(rows + static_cast<int64_t>(p) * a.N) : nullptr;
          });
      } else {
        typedef T vec8 __attribute__((ext_vector_type(8)));
        const bool whole = kMxTurned<EPI, J> && (wg + 2) * 32 <= a.N && (a.ldo & 7) == 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const f32x16 v = acc[u][j];
          const int c = (wg + j) * 32 + half * 16;
          vec8 o[2];
#pragma unroll
          for (int r = 0; r < 16; ++r) o[r >> 3][r & 7] = static_cast<T>(v[r]);
          if (whole) {
            turn[j * (PIECES / 2)] = __builtin_bit_cast(u32x4, o[0]);
            turn[j * (PIECES / 2) + 1] = __builtin_bit_cast(u32x4, o[1]);
          } else if (slot < a.M) {
            T* row = static_cast<T*>(a.out) + slot * a.ldo + c;
            if (c + 16 <= a.N && (a.ldo & 7) == 0) {
              *reinterpret_cast<vec8*>(row) = o[0];
              *reinterpret_cast<vec8*>(row + 8) = o[1];
            } else {
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (c + r < a.N) row[r] = o[r >> 3][r & 7];
            }
          }
        }
        if (whole)
          turned([&](int r) {
            const int64_t m = static_cast<int64_t>(t.group + u) * kMxRows + r;
            return m < a.M ? reinterpret_cast<u32x4*>(static_cast<T*>(a.out) + m * a.ldo + wg * 32) : nullptr;
          });
      }
    }
  }
}

template <typename T, int EPI, int J, bool NT>
__device__ __forceinline__ void mx_tile_of(const MxArgs& a, const MxSpan& t, int f, unsigned char* lds) {
  if (t.units == 4) mx_tile<T, EPI, 4, J, NT>(a, t, f, lds);
  else if (t.units == 3) mx_tile<T, EPI, 3, J, NT>(a, t, f, lds);
  else if (t.units == 2) mx_tile<T, EPI, 2, J, NT>(a, t, f, lds);
  else mx_tile<T, EPI, 1, J, NT>(a, t, f, lds);
}

// Blocks behind the last activated feature, up to a whole K tile: zero codes, scales of 1.
__device__ __forceinline__ void mx_fill(const MxArgs& a, const MxSpan& t, int f) {
  const int lane = threadIdx.x & 63, blk = f * 4 + (threadIdx.x >> 6), col = lane & 31;
  for (int u = 0; u < t.units; ++u) {
    unsigned char* unit = a.act + (static_cast<int64_t>(t.group + u) * a.act_tiles + (blk >> 3)) * kMxUnit;
    *reinterpret_cast<uint2*>(unit + mx_code_at(col, blk & 7) + (lane >> 5) * 8) = uint2{0, 0};
    if (lane < 32) unit[mx_scale_at(col, blk & 7)] = 127;
  }
}

template <typename T, int EPI, int J, bool NT>
__global__ __launch_bounds__(kMxThreads, 2) void mx_gemm_kernel(MxArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char mx_lds[];
  // workgroups b, b + 8, .. share an XCD and its L2: an XCD takes a consecutive part of the walk
  const int tiles = kMxLinear<EPI> ? (a.x_groups + kMxMaxUnits - 1) / kMxMaxUnits : a.tile_count[0];
  const int total = tiles * a.f_tiles, per = (total + 7) / 8;
  const int i = blockIdx.x >> 3, lin = (blockIdx.x & 7) * per + i;
  if (i >= per || lin >= total) return;
  const int guess = lin / a.f_tiles;  // a tile of the chunk that lin belongs to
  MxTile e;
  if constexpr (kMxLinear<EPI>) {
    e.first = e.expert = e.index0 = 0;
    e.count = a.x_groups;
    e.n = tiles;
    e.chunk0 = guess / kMxChunk * kMxChunk;
    e.chunk_n = min(kMxChunk, tiles - e.chunk0);
  } else {
    e = a.tiles[guess];
  }
  const int q = lin - e.chunk0 * a.f_tiles, f = q / e.chunk_n, i0 = e.chunk0 - e.index0 + q - f * e.chunk_n;
  const int base = e.count / e.n, rem = e.count - base * e.n;  // the first rem tiles are a row group taller
  const MxSpan t = {e.first + i0 * base + min(i0, rem), base + (i0 < rem ? 1 : 0), e.expert};
  if constexpr (EPI == MX_SILU) {
    if (f * 4 >= a.act_blocks) return mx_fill(a, t, f);
  }
  // a tile alone on its weights reads them past the caches if the call streams them; those that share a weight tile meet in L2
  if (NT && e.chunk_n == 1) mx_tile_of<T, EPI, J, true>(a, t, f, mx_lds);
  else mx_tile_of<T, EPI, J, false>(a, t, f, mx_lds);
}

constexpr int64_t kMxNarrowBelow = 128;  // workgroups, see launch_mx_gemm
constexpr int kMxLds = kMxSlots * (kMxMaxUnits * 4096 + 1024);
static_assert(kMxThreads / 64 * 32 * kMxTurnPitch<MX_DOWN> <= kMxLds, "the epilogue's rows lie in the ring");

// More than 64 KB of LDS needs the kernel's limit raised, once per device (a set-up call, not stream work).
template <typename T, int EPI, int J, bool NT>
int mx_allow_lds() {
  constexpr int kMaxDevices = 64;
  static bool set[kMaxDevices] = {};  // a race between threads sets the same limit twice
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess || dev < 0 || dev >= kMaxDevices) return fail(FR_E_LAUNCH, "mxfp4 product: device %d (%s)", dev, hipGetErrorString(e));
  if (set[dev]) return FR_OK;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_gemm_kernel<T, EPI, J, NT>), hipFuncAttributeMaxDynamicSharedMemorySize, kMxLds);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    return fail(FR_E_LAUNCH, "mxfp4 product: %d bytes of LDS: %s", kMxLds, hipGetErrorString(e));
  }
  set[dev] = true;
  return FR_OK;
}

template <typename T, int EPI, int J, bool NT>
int launch_mx_gemm_as(const MxArgs& a, dim3 grid, hipStream_t st) {
  const int rc = mx_allow_lds<T, EPI, J, NT>();
  if (rc != FR_OK) return rc;
  hipLaunchKernelGGL((mx_gemm_kernel<T, EPI, J, NT>), grid, dim3(kMxThreads), kMxLds, st, a);
  return check_launch("mx_gemm_kernel");
}
template <typename T, int EPI, int J>
int launch_mx_gemm_wide(MxArgs a, int64_t tiles, int64_t matrices, hipStream_t st, int slices) {
  if (EPI != MX_SILU) a.f_tiles = static_cast<int>(ceil_div(static_cast<int64_t>(a.w_groups), int64_t(4 * J)));
  const int64_t wgs = 8 * ceil_div(tiles * a.f_tiles, int64_t(8));
  FR_REQUIRE(wgs < (int64_t(1) << 31), FR_E_SHAPE, "mxfp4 product: %lld workgroups", (long long)wgs);
  const dim3 grid(static_cast<unsigned>(wgs), static_cast<unsigned>(slices));
  if (mx_streams(matrices * a.w_groups * a.k_tiles * kMxUnit)) return launch_mx_gemm_as<T, EPI, J, true>(a, grid, st);
  return launch_mx_gemm_as<T, EPI, J, false>(a, grid, st);
}

// tiles: token tiles, at most; likely: token tiles with even loads; matrices: weight matrices that the call reads, at most.  Where tiles of 256 weight rows
// would leave half of the CUs without a workgroup, tiles of 128: twice the workgroups, and twice the LDS reads per MFMA.  H = 4096, F = 14336, 8 experts,
// 256 tokens (128 workgroups) down 72 -> 55 us; 200 x 12288 x 4096 (96) 16.0 -> 12.6; but 509 (192) 19.7 -> 21.0, 600 tokens (256) 77 -> 81.
template <typename T, int EPI>
int launch_mx_gemm(const MxArgs& a, int64_t tiles, int64_t likely, int64_t matrices, hipStream_t st, int slices = 1) {
  if constexpr (EPI == MX_LINEAR || EPI == MX_DOWN) {
    if (likely * ceil_div(static_cast<int64_t>(a.w_groups), int64_t(8)) <= kMxNarrowBelow) return launch_mx_gemm_wide<T, EPI, 1>(a, tiles, matrices, st, slices);
  }
  return launch_mx_gemm_wide<T, EPI, 2>(a, tiles, matrices, st, slices);
}

// out[m, :] = sum over the token's pairs and their slices, in order, of weighted rows [slices][n, H]; a pair without an expert (a
// token row of NaN logits) has no row.  Bound by memory: each row is read once, past the caches, two of a token's under way together.  64 experts, H = 2048,
// top-6, 8192 tokens one / two / four at a time 99 / 96 / 96 us, two past the caches 73 (435 MB, 6.0 TB/s); H = 4096, top-2, 16384 129 / 113 / 128, 111.
template <typename T>
__global__ __launch_bounds__(kMxThreads) void mx_combine_kernel(const float* __restrict__ rows, int slices, int64_t n, const int32_t* __restrict__ ids,
                                                                int E, int topk, int64_t M, int H, T* __restrict__ out) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const int per = H / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kMxThreads + threadIdx.x;
  if (i >= M * per) return;
  const int64_t m = i / per;
  const int c = static_cast<int>(i - m * per) * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  int j = 0, v = 0;  // next pair of the token and slice
  while (j < topk) {
    f32x4 q[2];
    bool has[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t p = m * topk + min(j, topk - 1);  // a pair without an expert has memory, but no row in it
      has[u] = j < topk && static_cast<unsigned>(ids[p]) < static_cast<unsigned>(E);
      q[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(rows + (v * n + p) * H + c));
      if (++v == slices) {
        v = 0;
        ++j;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!has[u]) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] += q[u][r];
    }
  }
  vec4 o;
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(s[r]);
  *reinterpret_cast<vec4*>(out + i * 4) = o;
}

// ---- workspaces ------------------------------------------------------------------------------------------------
struct MxLayer {
  float* topk_w;
  int32_t *topk_ids, *sorted, *expert_ids, *npost;
  void* align_ws;
  int64_t align_bytes, groups, tile_limit, bytes;
  int* tile_count;
  MxTile* tiles;
  unsigned char *x, *act;
  int slices;   // of the down product's K
  float* rows;  // [slices][n, H]
};

// K slices of the down product: where its workgroups are few (a narrow layer, few rows) more of them, of four K tiles at least, as long
// as their fp32 rows, written and read, stay below a tenth of the weights' bytes or 16 MB.  H = 1024, F = 3584, 8 experts, 100 tokens: down
// 11.4 -> 7.3 us; H = 4096, F = 14336, 40 tokens 57.7 -> 47.0.
int mx_slices(int64_t n, int64_t H, int64_t F, int E) {
  if (n == 0) return 1;
  const int64_t experts = n < E ? n : E, tiles = experts * ceil_div(ceil_div(n, experts), int64_t(kMxMaxUnits) * kMxRows);
  const int64_t wgs = tiles * ceil_div(H, 8 * kMxRows);
  int64_t s = 512 / wgs;
  if (s > mx_tiles(F) / 4) s = mx_tiles(F) / 4;
  const int64_t weights = experts * H * F * 17 / 32, most = weights / 10 > (16 << 20) ? weights / 10 : 16 << 20;
  if (s > most / (n * H * 8)) s = most / (n * H * 8);
  return static_cast<int>(s < 1 ? 1 : s > 8 ? 8 : s);
}

MxLayer mx_layer(void* ws, int64_t M, int64_t H, int64_t F, int E, int topk) {
  MxLayer l;
  MxBump b{static_cast<unsigned char*>(ws)};
  const int64_t n = M * topk;
  // groups of 32 slots: each holds a pair, and every expert fills up one at most
  l.groups = n < (n + int64_t(E) * (kMxRows - 1)) / kMxRows ? n : (n + int64_t(E) * (kMxRows - 1)) / kMxRows;
  const int64_t experts = n < E ? n : E;
  l.tile_limit = l.groups / kMxMaxUnits + experts;  // an expert has a lower tile than the limit at most once
  l.topk_w = b.take<float>(n);
  l.topk_ids = b.take<int32_t>(n);
  l.sorted = b.take<int32_t>(n + int64_t(E) * (kMxRows - 1));
  l.expert_ids = b.take<int32_t>(n + E);
  l.npost = b.take<int32_t>(1);
  l.align_bytes = fr_moe_align_workspace_bytes(n, E);
  l.align_ws = b.take<unsigned char>(l.align_bytes);
  l.tile_count = b.take<int>(1);
  l.tiles = b.take<MxTile>(l.tile_limit);
  l.x = b.take<unsigned char>(l.groups * mx_tiles(H) * kMxUnit);
  l.act = b.take<unsigned char>(l.groups * mx_tiles(F) * kMxUnit);
  l.slices = mx_slices(n, H, F, E);
  l.rows = b.take<float>(l.slices * n * H);
  l.bytes = b.at;
  return l;
}

int check_mx_layer(const char* who, int64_t M, int64_t H, int64_t F, int E, int topk) {
  FR_REQUIRE(M >= 0 && M <= (int64_t(1) << 24), FR_E_SHAPE, "%s: M=%lld outside [0, 2^24]", who, (long long)M);
  FR_REQUIRE(H >= 32 && F >= 32 && H % 32 == 0 && F % 32 == 0 && H <= (1 << 20) && F <= (1 << 20), FR_E_SHAPE,
             "%s: H=%lld and F=%lld must be multiples of 32 up to 2^20", who, (long long)H, (long long)F);
  FR_REQUIRE(E >= 1 && E <= 256, FR_E_SHAPE, "%s: E=%d outside [1, 256]", who, E);
  FR_REQUIRE(topk >= 1 && topk <= E, FR_E_SHAPE, "%s: topk=%d outside [1, E=%d]", who, topk, E);
  FR_REQUIRE(M * topk <= (int64_t(1) << 24), FR_E_SHAPE, "%s: M*topk=%lld above 2^24", who, (long long)(M * topk));
  return FR_OK;
}

}  // namespace
}  // namespace fr

extern "C" int64_t fr_linear_mxfp4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  using namespace fr;
  if (M < 0 || N < 1 || K < 0 || M > (int64_t(1) << 24) || N > (int64_t(1) << 24) || K > (int64_t(1) << 20)) return -1;
  return mx_few_linear_fits(M, N) ? mx_few_linear_workspace(M, K) : mx_groups(M) * mx_tiles(K) * kMxUnit;
}

extern "C" int fr_linear_mxfp4(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* w_tiled, int64_t N, void* out,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace fr;
  FR_REQUIRE(M >= 0 && M <= (int64_t(1) << 24), FR_E_SHAPE, "fr_linear_mxfp4: M=%lld outside [0, 2^24]", (long long)M);
  FR_REQUIRE(K >= 32 && K % 32 == 0 && K <= (1 << 20), FR_E_SHAPE, "fr_linear_mxfp4: K=%lld must be a multiple of 32 up to 2^20", (long long)K);
  FR_REQUIRE(N >= 1 && N <= (1 << 24), FR_E_SHAPE, "fr_linear_mxfp4: N=%lld outside [1, 2^24]", (long long)N);
  FR_REQUIRE(dtype == FR_BF16 || dtype == FR_F16, FR_E_DTYPE, "fr_linear_mxfp4: dtype %d not in {f16, bf16}", dtype);
  if (M == 0) return FR_OK;
  FR_REQUIRE(x && w_tiled && out, FR_E_NULL, "fr_linear_mxfp4: null pointer");
  FR_REQUIRE(ldx >= K && ldx % 8 == 0 && aligned16(x) && aligned16(w_tiled) && aligned16(out), FR_E_ALIGN,
             "fr_linear_mxfp4: 16-byte alignment, ldx %% 8 == 0, ldx >= K");
  const int64_t need = fr_linear_mxfp4_workspace_bytes(M, N, K);
  FR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), FR_E_WORKSPACE, "fr_linear_mxfp4: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  FR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, FR_E_ALIGN, "fr_linear_mxfp4: workspace must be 256-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (mx_few_linear_fits(M, N)) return mx_few_linear(x, dtype, M, K, ldx, w_tiled, N, out, workspace, st);
  const int64_t groups = mx_groups(M);
  // x is read past the caches where it and the result would not both stay: 8192 x 4096 in, 12288 features out 24 -> 17.5 us
  int rc = mx_quant_tiled(x, dtype, M, K, ldx, groups, MxGather{}, mx_streams(2 * M * (K + N)), workspace, st);
  if (rc != FR_OK) return rc;
  MxArgs a = {};
  a.x = static_cast<const unsigned char*>(workspace);
  a.w = static_cast<const unsigned char*>(w_tiled);
  a.k_tiles = static_cast<int>(mx_tiles(K));
  a.w_groups = static_cast<int>(mx_groups(N));
  a.x_groups = static_cast<int>(groups);
  a.out = out;
  a.ldo = N;
  a.M = M;
  a.N = static_cast<int>(N);
  const int64_t token_tiles = ceil_div(groups, int64_t(kMxMaxUnits));
  if (mx_streams(2 * M * N))  // tiles enough for 256 weight rows
    return dtype == FR_BF16 ? launch_mx_gemm_wide<bf16_t, MX_PAST, 2>(a, token_tiles, 1, st, 1) : launch_mx_gemm_wide<f16_t, MX_PAST, 2>(a, token_tiles, 1, st, 1);
  return dtype == FR_BF16 ? launch_mx_gemm<bf16_t, MX_LINEAR>(a, token_tiles, token_tiles, 1, st)
                          : launch_mx_gemm<f16_t, MX_LINEAR>(a, token_tiles, token_tiles, 1, st);
}

extern "C" int64_t fr_moe_mxfp4_workspace_bytes(int64_t M, int64_t H, int64_t F, int E, int topk) {
  using namespace fr;
  if (check_mx_layer("fr_moe_mxfp4_workspace_bytes", M, H, F, E, topk) != FR_OK) return -1;
  MxFewScratch few;
  return mx_few_fits(M, F, E, topk) ? mx_few_workspace(nullptr, M, H, F, E, topk, &few) : mx_layer(nullptr, M, H, F, E, topk).bytes;
}

extern "C" int fr_fused_moe_mxfp4(const void* x, int dtype, const void* w1_tiled, const void* w2_tiled, const void* logits, int logits_dtype,
                                  int64_t M, int64_t H, int64_t F, int E, int topk, int renormalize, void* out, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  using namespace fr;
  int rc = check_mx_layer("fr_fused_moe_mxfp4", M, H, F, E, topk);
  if (rc != FR_OK) return rc;
  FR_REQUIRE(dtype == FR_BF16 || dtype == FR_F16, FR_E_DTYPE, "fr_fused_moe_mxfp4: dtype %d not in {f16, bf16}", dtype);
  FR_REQUIRE(logits_dtype == FR_F32 || logits_dtype == FR_BF16 || logits_dtype == FR_F16, FR_E_DTYPE,
             "fr_fused_moe_mxfp4: logits dtype %d not in {f32, f16, bf16}", logits_dtype);
  if (M == 0) return FR_OK;
  FR_REQUIRE(x && w1_tiled && w2_tiled && logits && out, FR_E_NULL, "fr_fused_moe_mxfp4: null pointer");
  FR_REQUIRE(aligned16(x) && aligned16(w1_tiled) && aligned16(w2_tiled) && aligned16(out), FR_E_ALIGN, "fr_fused_moe_mxfp4: 16-byte alignment");
  const int64_t need = fr_moe_mxfp4_workspace_bytes(M, H, F, E, topk);
  FR_REQUIRE(workspace && workspace_bytes >= need, FR_E_WORKSPACE, "fr_fused_moe_mxfp4: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  FR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, FR_E_ALIGN, "fr_fused_moe_mxfp4: workspace must be 256-byte aligned");
  if (mx_few_fits(M, F, E, topk))
    return mx_few_layer(x, dtype, w1_tiled, w2_tiled, logits, logits_dtype, M, H, F, E, topk, renormalize, out, workspace, static_cast<hipStream_t>(stream));
  const MxLayer l = mx_layer(workspace, M, H, F, E, topk);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t n = M * topk, experts = n < E ? n : E, likely = experts * ceil_div(ceil_div(n, experts), int64_t(kMxMaxUnits) * kMxRows);
  if (route_align_fits(M, E, topk, false)) {
    rc = route_align_small(logits, logits_dtype, M, E, topk, renormalize, kMxRows, l.topk_w, l.topk_ids, l.sorted, l.expert_ids, l.npost, nullptr, 0,
                           nullptr, nullptr, st);
  } else {
    rc = fr_gating_topk(logits, logits_dtype, M, E, E, topk, renormalize, l.topk_w, l.topk_ids, stream);
    if (rc == FR_OK) rc = fr_moe_align(l.topk_ids, FR_I32, n, E, kMxRows, l.sorted, l.expert_ids, l.npost, l.align_ws, l.align_bytes, stream);
  }
  if (rc != FR_OK) return rc;
  MxGather g;
  g.sorted = l.sorted;
  g.expert_ids = l.expert_ids;
  g.npost = l.npost;
  g.topk = topk;
  g.tile_count = l.tile_count;
  g.tiles = l.tiles;
  rc = mx_quant_tiled(x, dtype, n, H, H, l.groups, g, false, l.x, st);
  if (rc != FR_OK) return rc;
  MxArgs a = {};
  a.tile_count = l.tile_count;
  a.tiles = l.tiles;
  a.sorted = l.sorted;
  a.topk_w = l.topk_w;
  a.n_pairs = static_cast<int>(n);
  a.act_tiles = static_cast<int>(mx_tiles(F));
  a.act_blocks = static_cast<int>(F / kMxBlock);
  // gate and up
  a.x = l.x;
  a.act = l.act;
  a.w = static_cast<const unsigned char*>(w1_tiled);
  a.k_tiles = static_cast<int>(mx_tiles(H));
  a.w_groups = static_cast<int>(2 * F / kMxRows);
  a.w_stride = static_cast<int64_t>(a.w_groups) * a.k_tiles * kMxUnit;
  a.f_tiles = 2 * a.act_tiles;  // whole units of activated features: the last ones are filled up with zeros
  rc = launch_mx_gemm<bf16_t, MX_SILU>(a, l.tile_limit, likely, experts, st);
  if (rc != FR_OK) return rc;
  // down
  a.x = l.act;
  a.w = static_cast<const unsigned char*>(w2_tiled);
  a.k_tiles = a.act_tiles;
  a.w_groups = static_cast<int>(H / kMxRows);
  a.w_stride = static_cast<int64_t>(a.w_groups) * a.k_tiles * kMxUnit;
  a.rows = l.rows;
  a.N = static_cast<int>(H);
  rc = l.slices > 1 ? launch_mx_gemm<bf16_t, MX_PART>(a, l.tile_limit, likely, experts, st, l.slices)
                    : launch_mx_gemm<bf16_t, MX_DOWN>(a, l.tile_limit, likely, experts, st);
  if (rc != FR_OK) return rc;
  const dim3 grid(static_cast<unsigned>(ceil_div(M * (H / 4), int64_t(kMxThreads))));
  if (dtype == FR_BF16)
    hipLaunchKernelGGL((mx_combine_kernel<bf16_t>), grid, dim3(kMxThreads), 0, st, l.rows, l.slices, n, l.topk_ids, E, topk, M, (int)H, static_cast<bf16_t*>(out));
  else
    hipLaunchKernelGGL((mx_combine_kernel<f16_t>), grid, dim3(kMxThreads), 0, st, l.rows, l.slices, n, l.topk_ids, E, topk, M, (int)H, static_cast<f16_t*>(out));
  return check_launch("mx_combine_kernel");
}

// MXFP4 on gfx950: the format, and the memory layout that the matrix instructions read.
//
// Format (OCP microscaling): 32 consecutive elements of a row share a scale 2^(b - 127), held in the byte b; an element is e2m1
// (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives).  b = floor(log2(largest magnitude)) - 2 + 127, at least 0, so that the
// largest magnitude lies in [4, 8) units: elements are rounded to the nearest value, ties to the even code, and what exceeds
// 6 becomes 6.  A block of zeros has b = 127.  A block that holds an infinity or a NaN has b = 255, which stands for NaN: all
// 32 elements come back as NaN, and so does every product they enter.
//
// Layout of an operand matrix [rows, K] in units of 32 rows x 256 elements (4352 bytes): a row group's units one after the
// other along K, then the next row group's.  v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 rows x 64 elements per operand: lane l
// holds the 16 bytes of one block of row l % 32 and that block's scale, one byte of a register chosen by the instruction.  A
// unit therefore is four fragments of 1 KB - fragment s: lane l's 16 bytes at 16 l - and 256 bytes of scales - lane l's dword,
// byte s for fragment s.  Lane half l / 32 takes blocks 4 (l / 32) .. + 3 of the unit's eight, one per fragment: the order of blocks
// along K is free as long as both operands have the same, and this one lets 128 consecutive elements' scales be whole dwords.
// Any load of a fragment by a wavefront is 1 KB of consecutive memory, a row group's stream along K is one run.  Rows and K
// are filled up with zero codes and scales of 1.
//
// Weight rows inside a unit are permuted: the instruction leaves a lane rows (r & 3) + 8 (r >> 2) + 4 (l / 32), r = 0 .. 15, of
// its column; row m of a unit of weights is output feature weight_row(m), so that these are 16 consecutive features.
#pragma once
#include <type_traits>

#include "fr_common.h"

namespace fr {

constexpr int kMxBlock = 32;           // elements that share a scale
constexpr int kMxRows = 32;            // rows of a unit
constexpr int kMxTileK = 256;          // elements of a unit's rows
constexpr int kMxScales = 4096;        // offset of a unit's scales
constexpr int kMxUnit = 4096 + 256;    // bytes of a unit

inline __host__ __device__ int64_t mx_groups(int64_t rows) { return (rows + kMxRows - 1) / kMxRows; }
inline __host__ __device__ int64_t mx_tiles(int64_t K) { return (K + kMxTileK - 1) / kMxTileK; }

// where block b (of 8) of row r lies in a unit: its 16 bytes of codes, its scale byte
__device__ __forceinline__ int mx_code_at(int r, int b) { return (b & 3) * 1024 + (r + 32 * (b >> 2)) * 16; }
__device__ __forceinline__ int mx_scale_at(int r, int b) { return kMxScales + (r + 32 * (b >> 2)) * 4 + (b & 3); }
__device__ __forceinline__ int weight_row(int m) { return 16 * ((m >> 2) & 1) + (m & 3) + 4 * (m >> 3); }

// bits of |v|: as integers they order finite values, then infinity, then NaN
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// scale byte of a block whose largest magnitude has these bits
__device__ __forceinline__ unsigned mx_scale_byte(unsigned amax) {
  const int e = static_cast<int>(amax >> 23);
  return amax == 0 ? 127u : e == 255 ? 255u : static_cast<unsigned>(e > 2 ? e - 2 : 0);
}
// the scale as a float: 2^(b - 127), NaN for 255
__device__ __forceinline__ float mx_scale_value(unsigned b) {
  return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7FC00000u : b << 23);
}
// Eight elements of a block as codes; v_cvt_scalef32_pk_fp4_f32 divides by the scale, rounds to nearest even and saturates.  A block
// without a finite scale has zero codes.
__device__ __forceinline__ unsigned mx_pack8(const float* v, unsigned b) {
  const float s = mx_scale_value(b == 255 ? 127 : b);
  unsigned o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], s, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], s, 3);
  return b == 255 ? 0u : o;
}

template <typename T> struct MxVec8;
template <> struct MxVec8<bf16_t> { typedef bf16x8 type; };
template <> struct MxVec8<f16_t> { typedef f16x8 type; };

// f(integral_constant<0>) .. f(integral_constant<N - 1>): the instruction's scale byte is part of its encoding
template <int I, int N, typename F>
__device__ __forceinline__ void mx_each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    mx_each<I + 1, N>(f);
  }
}

typedef unsigned mx_frag __attribute__((ext_vector_type(4)));  // a lane's block of 32 codes

// acc[r] += sum over 64 elements of w . x with both operands' scales, fragment S of their units
template <int S>
__device__ __forceinline__ f32x16 mx_mfma(mx_frag w, int ws, mx_frag x, int xs, f32x16 acc) {
  const i32x8 a = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3]), 0, 0, 0, 0};
  const i32x8 b = {static_cast<int>(x[0]), static_cast<int>(x[1]), static_cast<int>(x[2]), static_cast<int>(x[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 4, 4, S, ws, S, xs);  // 4: e2m1
}

// largest |v| bits over the 32 elements of a block held by a lane and its partner in the other half of the wavefront
__device__ __forceinline__ unsigned mx_pair_max(unsigned v) {
  const unsigned o = static_cast<unsigned>(partner_i32<32>(static_cast<int>(v)));
  return v > o ? v : o;
}

// Weights that a call reads once and that are more than the memory-side cache (256 MB) may keep from one call to the next are read past the
// caches: 8 experts, H = 4096, F = 14336, 40 tokens gate/up 91.7 -> 85.4 us, down 47.0 -> 43.9; but H = 1024, F = 3584 (17 MB), 50 tokens
// 7.9 -> 9.0, 10.6 -> 15.1.
inline bool mx_streams(int64_t weight_bytes) { return weight_bytes > (int64_t(128) << 20); }

// A token tile of the grouped product.  Its expert's run is `count` row groups from `first` on, cut into tiles index0 .. index0 + n - 1 of heights
// as equal as whole groups allow; tiles chunk0 .. chunk0 + chunk_n - 1 are walked together over the feature tiles (they share
// weight tiles).  Any tile's entry says where every tile of its expert lies: a workgroup looks at one entry.
struct MxTile {
  int first, count, expert, index0, n, chunk0, chunk_n;
};
constexpr int kMxChunk = 8;      // tiles walked together, at most
constexpr int kMxMaxUnits = 4;   // row groups of a tile, at most

// ---- launches (mxfp4_quant.hip, mxfp4_gemm.hip) ----------------------------------------------------------------

// Rows of x [*, K] (row stride ldx) as an operand of `groups` row groups.  sorted == nullptr: row m of the operand is row m of x, zeros
// from `rows` on.  Else slot m holds pair sorted[m] of token sorted[m] / topk, nothing where sorted[m] >= rows (the number of
// pairs), and only the first npost[0] slots exist; workgroup 0 also writes the tile list of the experts' runs (expert_ids: of each
// group of 32 slots), its length first.
struct MxGather {
  const int32_t* sorted = nullptr;
  const int32_t* expert_ids = nullptr;
  const int32_t* npost = nullptr;
  int topk = 1;
  int* tile_count = nullptr;
  MxTile* tiles = nullptr;
};
// nt: x is read past the caches.
int mx_quant_tiled(const void* x, int dtype, int64_t rows, int64_t K, int64_t ldx, int64_t groups, const MxGather& g, bool nt, void* out,
                   hipStream_t st);

}  // namespace fr

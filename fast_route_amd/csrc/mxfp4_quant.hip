// MXFP4 rows: quantisation, the way back, and the layout of operands for the matrix instructions (mxfp4_core.h).
//
// All of it is bound by memory: four lanes share a block of 32 elements, each reads 16 bytes of it, the block's largest magnitude comes from two
// quad permutes, and the codes go out as 4 bytes per lane - a wavefront reads and writes consecutive memory.
#include "mxfp4_core.h"

namespace fr {
namespace {

constexpr int kMxThreads = 256;
constexpr int kMxChunks = 4;  // 8-element chunks per thread: their loads are in flight together

__device__ __forceinline__ unsigned quad_max(unsigned v) {
  unsigned o = static_cast<unsigned>(partner_i32<1>(static_cast<int>(v)));
  v = v > o ? v : o;
  o = static_cast<unsigned>(partner_i32<2>(static_cast<int>(v)));
  return v > o ? v : o;
}

// Eight elements of a block (of which the lane's quad holds all): their codes; *byte: the block's scale byte.
template <typename T>
__device__ __forceinline__ unsigned quant8(const typename MxVec8<T>::type& v, unsigned* byte) {
  float f[8];
  unsigned amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = static_cast<float>(v[i]);
    const unsigned m = magnitude(f[i]);
    amax = amax > m ? amax : m;
  }
  *byte = mx_scale_byte(quad_max(amax));
  return mx_pack8(f, *byte);
}

// Values of more than the memory-side cache are read and written past the caches (NT, see mx_streams): 28672 x 4096 quantisation 65 -> 46 us, the
// way back 45 -> 42; 16384 x 4096 33 -> 28, 26 -> 25; but 8192 x 4096 quantisation 13.8 -> 15.0.
template <bool NT, typename V>
__device__ __forceinline__ V load_values(const V* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

// Chunk c of a row: elements 8 c .. 8 c + 7.  `chunks` = rows * K / 8; rows contiguous (per_row == 0) or ldx apart.
template <typename T, bool NT>
__global__ __launch_bounds__(kMxThreads) void mx_quant_rows_kernel(const T* __restrict__ x, int64_t chunks, int64_t per_row, int64_t ldx,
                                                                   unsigned* __restrict__ codes, unsigned char* __restrict__ scales) {
  typedef typename MxVec8<T>::type vec8;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kMxThreads * kMxChunks) + threadIdx.x;
  vec8 v[kMxChunks];
#pragma unroll
  for (int c = 0; c < kMxChunks; ++c) {
    const int64_t at = first + c * kMxThreads;
    v[c] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
    if (at < chunks) {
      int64_t from = at * 8;
      if (per_row) from = at / per_row * ldx + at % per_row * 8;
      v[c] = load_values<NT>(reinterpret_cast<const vec8*>(x + from));
    }
  }
#pragma unroll
  for (int c = 0; c < kMxChunks; ++c) {
    const int64_t at = first + c * kMxThreads;
    unsigned byte;
    const unsigned o = quant8<T>(v[c], &byte);  // a quad is whole: chunks is a multiple of 4
    if (at < chunks) {
      codes[at] = o;
      if ((at & 3) == 0) scales[at >> 2] = static_cast<unsigned char>(byte);
    }
  }
}

template <typename T, bool NT>
__global__ __launch_bounds__(kMxThreads) void mx_dequant_rows_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                                     int64_t chunks, T* __restrict__ out) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef T vec8 __attribute__((ext_vector_type(8)));
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kMxThreads * kMxChunks) + threadIdx.x;
  unsigned q[kMxChunks], b[kMxChunks];
#pragma unroll
  for (int c = 0; c < kMxChunks; ++c) {
    const int64_t at = first + c * kMxThreads;
    q[c] = at < chunks ? codes[at] : 0u;
    b[c] = at < chunks ? scales[at >> 2] : 127u;
  }
#pragma unroll
  for (int c = 0; c < kMxChunks; ++c) {
    const int64_t at = first + c * kMxThreads;
    const float s = mx_scale_value(b[c]), t = b[c] == 255 ? 1.f : s;
    f32x2 p[4];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[c], t, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[c], t, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[c], t, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[c], t, 3);
    vec8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = static_cast<T>(b[c] == 255 ? s : p[i >> 1][i & 1]);
    if (at < chunks) {
      vec8* const to = reinterpret_cast<vec8*>(out + at * 8);
      if constexpr (NT) __builtin_nontemporal_store(o, to);
      else *to = o;
    }
  }
}

// Weights [matrices, rows, K] as codes and scales to units; gate_up: rows are `rows / 2` gate rows, then as many up rows, and units of
// 32 gate and 32 up rows alternate.  A workgroup per unit, a block per thread; bound by memory: 8 experts, H = 4096, F = 14336 205 us (gate and up) and
// 107 (down), 4.8 TB/s read and written.
__global__ __launch_bounds__(kMxThreads) void mx_tile_weights_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                                     int64_t rows, int64_t K, int64_t groups, int64_t tiles, int gate_up,
                                                                     unsigned char* __restrict__ out) {
  const int64_t unit = blockIdx.x;  // (matrix, group, tile)
  const int64_t t = unit % tiles, g = unit / tiles % groups, m = unit / tiles / groups;
  const int row = threadIdx.x >> 3, b = threadIdx.x & 7;
  const int64_t half = gate_up ? rows / 2 : rows;
  const int64_t r = gate_up ? (g >> 1) * kMxRows + weight_row(row) : g * kMxRows + weight_row(row);
  const int64_t k = t * kMxTileK + b * kMxBlock;
  u32x4_t c = {0, 0, 0, 0};
  unsigned char s = 127;
  if (r < half && k < K) {
    const int64_t from = m * rows + r + ((gate_up && (g & 1)) ? half : 0);
    c = *reinterpret_cast<const u32x4_t*>(codes + (from * K + k) / 2);
    s = scales[(from * K + k) / kMxBlock];
  }
  unsigned char* u = out + unit * kMxUnit;
  *reinterpret_cast<u32x4_t*>(u + mx_code_at(row, b)) = c;
  u[mx_scale_at(row, b)] = s;
}

// The tile list of the experts' runs (one workgroup; E <= kMxThreads): an expert's groups of 32 slots, which are consecutive, are cut into as
// few tiles of at most kMxMaxUnits as hold them, of heights that differ by one at most.
__device__ void mx_tile_list(const MxGather& g) {
  __shared__ int first[kMxThreads], count[kMxThreads], sum[kMxThreads];
  const int e = threadIdx.x, nb = g.npost[0] / kMxRows;
  first[e] = 0;
  count[e] = 0;
  __syncthreads();
  for (int b = e; b < nb; b += kMxThreads) {
    const int id = g.expert_ids[b];
    if (b == 0 || g.expert_ids[b - 1] != id) first[id] = b;
    atomicAdd(&count[id], 1);
  }
  __syncthreads();
  const int n = (count[e] + kMxMaxUnits - 1) / kMxMaxUnits;
  sum[e] = n;
  __syncthreads();
  for (int d = 1; d < kMxThreads; d <<= 1) {
    const int below = e >= d ? sum[e - d] : 0;
    __syncthreads();
    sum[e] += below;
    __syncthreads();
  }
  const int at = sum[e] - n;
  if (e == kMxThreads - 1) g.tile_count[0] = sum[e];
  if (n == 0) return;
  const int chunks = (n + kMxChunk - 1) / kMxChunk;
  for (int i = 0; i < n; ++i) {
    const int c = static_cast<int>((static_cast<int64_t>(i + 1) * chunks - 1) / n);  // chunk c: tiles [c n / chunks, (c + 1) n / chunks)
    const int c0 = static_cast<int>(static_cast<int64_t>(c) * n / chunks), c1 = static_cast<int>(static_cast<int64_t>(c + 1) * n / chunks);
    g.tiles[at + i] = MxTile{first[e], count[e], e, at, n, at + c0, c1 - c0};
  }
}

// A unit per workgroup: wavefront w takes rows 16 (w & 1) .. + 15 and blocks 4 (w >> 1) .. + 3; a quad's four scales are one dword.
template <typename T, bool GATHER, bool NT>
__global__ __launch_bounds__(kMxThreads) void mx_quant_tiled_kernel(const T* __restrict__ x, int64_t rows, int64_t K, int64_t ldx, int64_t tiles,
                                                                    MxGather g, unsigned char* __restrict__ out) {
  typedef typename MxVec8<T>::type vec8;
  int64_t unit = blockIdx.x;
  if constexpr (GATHER) {
    if (unit == 0) {
      mx_tile_list(g);
      return;
    }
    --unit;
  }
  const int64_t group = unit / tiles, t = unit - group * tiles;
  if (GATHER && group * kMxRows >= g.npost[0]) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // A load instruction of a wavefront takes 64 bytes of 16 rows where rows are gathered, 128 of 8 where they are not (8192 x 4096, rows past the
  // caches: 17.5 against 20.5 us; gathered 49152 x 2048 36 against 33).
  constexpr int kRows = GATHER ? 16 : 8, kBlocks = 16 / kRows, kSets = 16 / kRows;
  const int row = (wave & 1) * 16 + lane / (4 * kBlocks), part = lane & 3, b0 = (wave >> 1) * 4 + (lane >> 2) % kBlocks;
  vec8 v[4];
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    int64_t src = group * kMxRows + row + i * kRows;
    bool live = src < rows;
    if constexpr (GATHER) {
      const int id = g.sorted[src];
      live = id < rows;
      src = live ? id / g.topk : 0;
    }
    const T* from = x + src * ldx;
#pragma unroll
    for (int j = 0; j < 4 / kSets; ++j) {
      const int64_t k = t * kMxTileK + (b0 + j * kBlocks) * kMxBlock + part * 8;
      vec8& to = v[i * (4 / kSets) + j];
      to = vec8{0, 0, 0, 0, 0, 0, 0, 0};
      if (live && k < K) to = load_values<NT>(reinterpret_cast<const vec8*>(from + k));
    }
  }
  unsigned char* u = out + unit * kMxUnit;
#pragma unroll
  for (int i = 0; i < kSets; ++i) {
    const int r = row + i * kRows;
    unsigned packed = 0;
#pragma unroll
    for (int j = 0; j < 4 / kSets; ++j) {
      unsigned byte;
      const unsigned o = quant8<T>(v[i * (4 / kSets) + j], &byte);
      *reinterpret_cast<unsigned*>(u + mx_code_at(r, b0 + j * kBlocks) + part * 4) = o;
      packed |= byte << (8 * kBlocks * j);
    }
    if constexpr (kBlocks == 2) packed |= __shfl_xor(packed, 4) << 8;  // the other block's of each two
    if (lane % (4 * kBlocks) == 0) *reinterpret_cast<unsigned*>(u + mx_scale_at(r, b0)) = packed;
  }
}

}  // namespace

int mx_quant_tiled(const void* x, int dtype, int64_t rows, int64_t K, int64_t ldx, int64_t groups, const MxGather& g, bool nt, void* out,
                   hipStream_t st) {
  const int64_t tiles = mx_tiles(K), wgs = groups * tiles + (g.sorted ? 1 : 0);
  FR_REQUIRE(wgs < (int64_t(1) << 31), FR_E_SHAPE, "mxfp4 operand: %lld units", (long long)wgs);
  const dim3 grid(static_cast<unsigned>(wgs)), block(kMxThreads);
  unsigned char* o = static_cast<unsigned char*>(out);
#define FR_QT(T_, G_, NT_) hipLaunchKernelGGL((mx_quant_tiled_kernel<T_, G_, NT_>), grid, block, 0, st, static_cast<const T_*>(x), rows, K, ldx, tiles, g, o)
  if (dtype == FR_BF16) {
    if (g.sorted) FR_QT(bf16_t, true, false);
    else if (nt) FR_QT(bf16_t, false, true);
    else FR_QT(bf16_t, false, false);
  } else {
    if (g.sorted) FR_QT(f16_t, true, false);
    else if (nt) FR_QT(f16_t, false, true);
    else FR_QT(f16_t, false, false);
  }
#undef FR_QT
  return check_launch("mx_quant_tiled_kernel");
}

}  // namespace fr

extern "C" int fr_quant_mxfp4_rows(const void* x, int dtype, int64_t rows, int64_t K, int64_t ldx, void* codes_out, void* scales_out,
                                   void* stream) {
  using namespace fr;
  FR_REQUIRE(rows >= 0, FR_E_SHAPE, "fr_quant_mxfp4_rows: rows=%lld < 0", (long long)rows);
  FR_REQUIRE(K > 0 && K % kMxBlock == 0 && K < (int64_t(1) << 30), FR_E_SHAPE, "fr_quant_mxfp4_rows: K=%lld must be a positive multiple of 32", (long long)K);
  FR_REQUIRE(dtype == FR_BF16 || dtype == FR_F16, FR_E_DTYPE, "fr_quant_mxfp4_rows: dtype %d not in {f16, bf16}", dtype);
  if (rows == 0) return FR_OK;
  FR_REQUIRE(x && codes_out && scales_out, FR_E_NULL, "fr_quant_mxfp4_rows: null pointer");
  FR_REQUIRE(ldx >= K && ldx % 8 == 0 && aligned16(x) && aligned16(codes_out), FR_E_ALIGN, "fr_quant_mxfp4_rows: 16-byte alignment, ldx %% 8 == 0, ldx >= K");
  FR_REQUIRE(rows < (int64_t(1) << 40) / K, FR_E_SHAPE, "fr_quant_mxfp4_rows: %lld rows of %lld elements", (long long)rows, (long long)K);
  const int64_t chunks = rows * (K / 8), per_row = ldx == K ? 0 : K / 8;
  const dim3 grid(static_cast<unsigned>(ceil_div(chunks, int64_t(kMxThreads) * kMxChunks))), block(kMxThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  unsigned* q = static_cast<unsigned*>(codes_out);
  unsigned char* s = static_cast<unsigned char*>(scales_out);
  const bool nt = mx_streams(chunks * (16 + 4));
#define FR_QR(T_, NT_) hipLaunchKernelGGL((mx_quant_rows_kernel<T_, NT_>), grid, block, 0, st, static_cast<const T_*>(x), chunks, per_row, ldx, q, s)
  if (dtype == FR_BF16) {
    if (nt) FR_QR(bf16_t, true);
    else FR_QR(bf16_t, false);
  } else {
    if (nt) FR_QR(f16_t, true);
    else FR_QR(f16_t, false);
  }
#undef FR_QR
  return check_launch("mx_quant_rows_kernel");
}

extern "C" int fr_dequant_mxfp4_rows(const void* codes, const void* scales, int64_t rows, int64_t K, int out_dtype, void* out, void* stream) {
  using namespace fr;
  FR_REQUIRE(rows >= 0, FR_E_SHAPE, "fr_dequant_mxfp4_rows: rows=%lld < 0", (long long)rows);
  FR_REQUIRE(K > 0 && K % kMxBlock == 0 && K < (int64_t(1) << 30), FR_E_SHAPE, "fr_dequant_mxfp4_rows: K=%lld must be a positive multiple of 32", (long long)K);
  FR_REQUIRE(out_dtype == FR_BF16 || out_dtype == FR_F16 || out_dtype == FR_F32, FR_E_DTYPE, "fr_dequant_mxfp4_rows: dtype %d not in {f16, bf16, f32}", out_dtype);
  if (rows == 0) return FR_OK;
  FR_REQUIRE(codes && scales && out, FR_E_NULL, "fr_dequant_mxfp4_rows: null pointer");
  FR_REQUIRE(aligned16(codes) && aligned16(out), FR_E_ALIGN, "fr_dequant_mxfp4_rows: 16-byte alignment");
  FR_REQUIRE(rows < (int64_t(1) << 40) / K, FR_E_SHAPE, "fr_dequant_mxfp4_rows: %lld rows of %lld elements", (long long)rows, (long long)K);
  const int64_t chunks = rows * (K / 8);
  const dim3 grid(static_cast<unsigned>(ceil_div(chunks, int64_t(kMxThreads) * kMxChunks))), block(kMxThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned* q = static_cast<const unsigned*>(codes);
  const unsigned char* s = static_cast<const unsigned char*>(scales);
  const bool nt = mx_streams(chunks * ((out_dtype == FR_F32 ? 32 : 16) + 4));
#define FR_DR(T_)                                                                                                                       \
  do {                                                                                                                                  \
    if (nt) hipLaunchKernelGGL((mx_dequant_rows_kernel<T_, true>), grid, block, 0, st, q, s, chunks, static_cast<T_*>(out));           \
    else hipLaunchKernelGGL((mx_dequant_rows_kernel<T_, false>), grid, block, 0, st, q, s, chunks, static_cast<T_*>(out));             \
  } while (0)
  if (out_dtype == FR_BF16) FR_DR(bf16_t);
  else if (out_dtype == FR_F16) FR_DR(f16_t);
  else FR_DR(float);
#undef FR_DR
  return check_launch("mx_dequant_rows_kernel");
}

extern "C" int64_t fr_mxfp4_tiled_bytes(int64_t matrices, int64_t rows, int64_t K) {
  using namespace fr;
  if (matrices < 0 || rows < 0 || K < 0 || matrices > (int64_t(1) << 20) || rows > (int64_t(1) << 30) || K > (int64_t(1) << 30)) return -1;
  const int64_t units = mx_groups(rows) * mx_tiles(K);
  if (matrices > 0 && units >= (int64_t(1) << 31) / matrices) return -1;
  return matrices * units * kMxUnit;
}

extern "C" int fr_mxfp4_tile_weights(const void* codes, const void* scales, int64_t matrices, int64_t rows, int64_t K, int gate_up, void* out,
                                     void* stream) {
  using namespace fr;
  FR_REQUIRE(matrices >= 1 && rows >= 1, FR_E_SHAPE, "fr_mxfp4_tile_weights: %lld matrices of %lld rows", (long long)matrices, (long long)rows);
  FR_REQUIRE(K > 0 && K % kMxBlock == 0, FR_E_SHAPE, "fr_mxfp4_tile_weights: K=%lld must be a positive multiple of 32", (long long)K);
  FR_REQUIRE(!gate_up || rows % (2 * kMxRows) == 0, FR_E_SHAPE, "fr_mxfp4_tile_weights: %lld gate and up rows are no multiple of 64", (long long)rows);
  FR_REQUIRE(fr_mxfp4_tiled_bytes(matrices, rows, K) >= 0, FR_E_SHAPE, "fr_mxfp4_tile_weights: %lld x %lld x %lld is too large",
             (long long)matrices, (long long)rows, (long long)K);
  FR_REQUIRE(codes && scales && out, FR_E_NULL, "fr_mxfp4_tile_weights: null pointer");
  FR_REQUIRE(aligned16(codes) && aligned16(out), FR_E_ALIGN, "fr_mxfp4_tile_weights: 16-byte alignment");
  const int64_t groups = mx_groups(rows), tiles = mx_tiles(K);
  hipLaunchKernelGGL(mx_tile_weights_kernel, dim3(static_cast<unsigned>(matrices * groups * tiles)), dim3(kMxThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<const unsigned char*>(codes), static_cast<const unsigned char*>(scales), rows, K, groups, tiles, gate_up,
                     static_cast<unsigned char*>(out));
  return check_launch("mx_tile_weights_kernel");
}

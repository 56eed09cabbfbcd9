// Attention of one query row per sequence over its pages: every key and value is read once, 4 flops per byte and query head that
// shares it, so the cache's way from memory bounds it.
//
// A workgroup takes the query heads of one key head (up to 16, the columns of a matrix instruction) and a part of one sequence's keys; its
// four wavefronts take runs of 32 keys in turn, each with a running maximum and sum of its own.
//   S^T [32 keys, 16 heads] = K Q^T: rows of K are the first operand as they lie in memory, straight to registers.
//   O^T [dim, 16 heads] += V^T P^T: S^T's accumulators hold, per lane, 2 x 4 consecutive keys of one head, which is the second
//   operand's place for them if V^T's keys are taken in the same order: V goes through LDS (of the wavefront's own, no barrier), where
//   transposed reads give 4 consecutive keys of a dimension.
// A run's 16 KB (128 dimensions) are asked for before the run in front is worked on, in registers.
//
// The keys of all sequences are split into parts of equal length on the device, since the lengths are there: with `slots` places per key head,
// the length is the smallest multiple of 128 that gives every sequence its parts.  Parts of a sequence that has one go to the output, others
// to fp32 rows with their maxima and sums, which a second launch joins.
#include "attention_core.h"

namespace fr {
namespace {

constexpr int kPagThreads = 256, kPagWaves = 4, kPagRun = 32, kPagHeads = 16;
constexpr int kPagStep = kPagRun * kPagWaves;

__device__ __forceinline__ int64_t pag_length(const fr_paged_args& a, int64_t b) {
  const int64_t cap = a.table_pages * a.page_size, n = reinterpret_cast<const int32_t*>(a.lengths)[b];
  return n < 0 ? 0 : (n > cap ? cap : n);
}
__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) v += __shfl_xor(v, s, kWave);
  return v;
}
// Keys of a part: sum over b of max(1, ceil(length / part)) <= total / part + B <= slots.
__device__ __forceinline__ int64_t pag_part(const fr_paged_args& a) {
  int64_t total = 0;
  for (int64_t b = threadIdx.x & 63; b < a.B; b += kWave) total += pag_length(a, b);
  total = wave_sum_i64(total);
  const int64_t spare = a.slots - a.B;
  if (spare <= 0) return int64_t(1) << 40;  // a part each
  const int64_t per = (total + spare - 1) / spare;
  return per < kPagStep ? kPagStep : (per + kPagStep - 1) / kPagStep * kPagStep;
}
__device__ __forceinline__ int pag_parts(int64_t length, int64_t part) { return length <= part ? 1 : static_cast<int>((length + part - 1) / part); }

// Sequence and part of a slot (sequence -1: none).
__device__ __forceinline__ void pag_place(const fr_paged_args& a, int64_t part, int64_t slot, int64_t* seq, int* at, int* of) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  *seq = -1;
  for (int64_t b0 = 0; b0 < a.B; b0 += kWave) {
    const int64_t b = b0 + lane;
    const int n = b < a.B ? pag_parts(pag_length(a, b), part) : 0;
    int sum = n;
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) {
      const int below = __shfl_up(sum, s, kWave);
      sum += lane >= s ? below : 0;
    }
    const int64_t mine = before + sum;
    const uint64_t hit = __ballot(n > 0 && slot < mine && slot >= mine - n);
    if (hit) {
      const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      *seq = b0 + l;
      *of = __shfl(n, l, kWave);
      *at = static_cast<int>(slot - (before + __shfl(sum, l, kWave) - *of));
      return;
    }
    before += __shfl(sum, 63, kWave);
  }
}

template <int DP>
struct PagShape {
  static constexpr int kChunks = DP / 8;                  // 16-byte pieces of a row
  static constexpr int kLoads = kPagRun * kChunks / kWave;  // of a run's V rows
  static constexpr int kSteps = DP / 32, kTiles = DP / 16;
  // Rows of V lie in LDS with their pieces exchanged in pairs, so that a transposed read's four rows, 16 elements each, meet in no bank.
  static constexpr int kMask = DP % 128 == 0 ? 7 : 3;
  static __device__ __forceinline__ int at(int row, int chunk) { return row * DP + (chunk ^ ((row & kMask) << 1)) * 8; }
};

// ALIGNED: pages are multiples of 16 keys, so 16 consecutive keys from a multiple of 16 on share a page.
template <typename T, int DP, bool ALIGNED>
__global__ __launch_bounds__(kPagThreads) void paged_attention_kernel(fr_paged_args a) {
  typedef typename Attn<T>::vec8 vec8;
  typedef PagShape<DP> S;
  __shared__ __attribute__((aligned(16))) char shared[kPagWaves * kPagRun * DP * sizeof(T)];
  __shared__ float max_of[kPagWaves][kPagHeads], sum_of[kPagWaves][kPagHeads];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = static_cast<int>(a.heads / a.kv_heads), tiles = (share + kPagHeads - 1) / kPagHeads, columns = static_cast<int>(a.kv_heads) * tiles;
  const int64_t slot = blockIdx.x / columns;
  const int column = blockIdx.x % columns, kv = column / tiles, head0 = (column % tiles) * kPagHeads;
  const int heads = share - head0 < kPagHeads ? share - head0 : kPagHeads;  // of the columns, in use

  const int64_t part = pag_part(a);
  int64_t seq;
  int nth = 0, parts = 0;
  pag_place(a, part, slot, &seq, &nth, &parts);
  if (seq < 0) return;
  seq = __builtin_amdgcn_readfirstlane(static_cast<int>(seq));
  const int64_t length = pag_length(a, seq);
  const int64_t begin = parts > 1 ? nth * part : 0;
  const int first = __builtin_amdgcn_readfirstlane(static_cast<int>(begin));
  const int last = __builtin_amdgcn_readfirstlane(static_cast<int>(length < begin + part ? length : begin + part));
  const int dim = static_cast<int>(a.dim);
  const int32_t* table = reinterpret_cast<const int32_t*>(a.table) + seq * a.table_row;
  const T* kc = reinterpret_cast<const T*>(a.k_cache) + kv * a.k_cache_head;
  const T* vc = reinterpret_cast<const T*>(a.v_cache) + kv * a.v_cache_head;
  const int quarter = lane >> 4, low = lane & 15;

  // Q^T, the second operand: column = lane % 16
  vec8 q[S::kSteps];
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    q[s] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
    const int d = s * 32 + quarter * 8;
    if (low < heads && d < dim)
      q[s] = *reinterpret_cast<const vec8*>(reinterpret_cast<const T*>(a.q) + seq * a.q_row + (kv * share + head0 + low) * a.q_head + d);
  }
  const float scale = static_cast<float>(a.scale) * kLog2e;

  auto page_of = [&](int key) { return a.page_shift >= 0 ? key >> static_cast<int>(a.page_shift) : key / static_cast<int>(a.page_size); };
  // Where key `key`'s row lies, -1 behind the last key and in a page that there is not: such keys take no part, their rows are zeros.
  auto row_of = [&](int key, int64_t page_stride, int64_t slot_stride) -> int64_t {
    if (key >= last) return -1;
    const int p = page_of(key);
    const int64_t page = table[p];
    if (page < 0 || page >= a.pages) return -1;
    return page * page_stride + (key - p * static_cast<int>(a.page_size)) * slot_stride;
  };
  vec8 k[2][S::kSteps], v[S::kLoads];
  bool whole = false;  // the run in the registers: no key of it is left out
  auto load = [&](int base) {
    if (ALIGNED && base + kPagRun <= last) {
      int64_t page[2];
      int in[2];
      whole = true;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p = page_of(base + 16 * t);
        page[t] = table[p];
        in[t] = base + 16 * t - p * static_cast<int>(a.page_size);
        whole = whole && page[t] >= 0 && page[t] < a.pages;
      }
      if (whole) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const T* from = kc + page[t] * a.k_cache_page + in[t] * a.k_cache_slot + (low * a.k_cache_slot + quarter * 8);
#pragma unroll
          for (int s = 0; s < S::kSteps; ++s) k[t][s] = (s + 1) * 32 <= dim || s * 32 + quarter * 8 < dim ? *reinterpret_cast<const vec8*>(from + s * 32) : vec8{0, 0, 0, 0, 0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
          const int at = i * kWave + lane, row = at / S::kChunks, d = at % S::kChunks * 8, t = i * kWave / S::kChunks >= 16 ? 1 : 0;  // a load's rows are in one half
          const T* from = vc + page[t] * a.v_cache_page + in[t] * a.v_cache_slot + ((row - 16 * t) * a.v_cache_slot + d);
          v[i] = dim == DP || d < dim ? *reinterpret_cast<const vec8*>(from) : vec8{0, 0, 0, 0, 0, 0, 0, 0};
        }
        return;
      }
    }
    whole = false;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t from = row_of(base + 16 * t + low, a.k_cache_page, a.k_cache_slot);
#pragma unroll
      for (int s = 0; s < S::kSteps; ++s) {
        const int d = s * 32 + quarter * 8;
        k[t][s] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
        if (from >= 0 && d < dim) k[t][s] = *reinterpret_cast<const vec8*>(kc + from + d);
      }
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * kWave + lane, row = at / S::kChunks, d = at % S::kChunks * 8;
      const int64_t from = row_of(base + row, a.v_cache_page, a.v_cache_slot);
      v[i] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
      if (from >= 0 && d < dim) v[i] = *reinterpret_cast<const vec8*>(vc + from + d);
    }
  };

  T* const vl = reinterpret_cast<T*>(shared) + wave * kPagRun * DP;
  f32x4 o[S::kTiles];
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;  // of column lane % 16: the maximum (lagging) in all four lanes, the sum of the lane's own keys
  int base = first + wave * kPagRun;
  if (base < last) load(base);
  for (; base < last; base += kPagStep) {
    f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) st[t] = Attn<T>::mma16(k[t][s], q[s], st[t]);
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * kWave + lane;
      *reinterpret_cast<vec8*>(vl + S::at(at / S::kChunks, at % S::kChunks)) = v[i];
    }
    const bool all_seen = whole;
    if (base + kPagStep < last) load(base + kPagStep);
    float p[2][4], high = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) p[t][r] = st[t][r] * scale;
    if (!all_seen) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row_of(base + 16 * t + quarter * 4 + r, 0, 0) < 0) p[t][r] = -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) high = fmaxf(high, p[t][r]);
    if (__any(high > top + kLag)) {
      high = max_over_32(max_over_16(high));
      const float now = fmaxf(top, high), by = top == -INFINITY ? 0.f : exp2_of(top - now);
      sum *= by;
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) o[t] *= by;
      top = now;
    }
    const float from = top == -INFINITY ? 0.f : top;
    vec8 pt;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = exp2_of(p[t][r] - from);
        sum += e;
        pt[t * 4 + r] = static_cast<T>(e);  // to 8 or 11 bits: the second product's operand
      }
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) {
      const int chunk = 2 * t + ((lane & 3) >> 1), rest = (lane & 1) * 4, row = quarter * 4 + (low >> 2);
      const auto lo = read_transposed<T>(vl + S::at(row, chunk) + rest), hi = read_transposed<T>(vl + S::at(row + 16, chunk) + rest);
      o[t] = Attn<T>::mma16(join8(lo, hi), pt, o[t]);
    }
  }
  sum = sum_over_32(sum_over_16(sum));

  // The four wavefronts' rows in one: fp32, over V's place in LDS.
  if (quarter == 0) max_of[wave][low] = top, sum_of[wave][low] = sum;
  __syncthreads();
  float all = -INFINITY, total = 0.f;
#pragma unroll
  for (int w = 0; w < kPagWaves; ++w) all = fmaxf(all, max_of[w][low]);
#pragma unroll
  for (int w = 0; w < kPagWaves; ++w) total += max_of[w][low] == -INFINITY ? 0.f : sum_of[w][low] * exp2_of(max_of[w][low] - all);
  float by = top == -INFINITY ? 0.f : exp2_of(top - all);
  if (parts == 1) by = total == 0.f ? 0.f : by / total;  // no key at all: zeros
  float* const rows = reinterpret_cast<float*>(shared);  // [wave][head][dimension]
#pragma unroll
  for (int t = 0; t < S::kTiles; ++t) *reinterpret_cast<f32x4*>(&rows[(wave * kPagHeads + low) * DP + t * 16 + quarter * 4]) = o[t] * by;
  float* const to_part = reinterpret_cast<float*>(a.workspace) + (slot * columns + column) * (kPagHeads * (DP + 2));
  if (parts > 1 && wave == 0 && quarter == 0) {
    to_part[kPagHeads * DP + low] = all;
    to_part[kPagHeads * (DP + 1) + low] = total;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * (DP / 4); i += kPagThreads) {
    const int h = i / (DP / 4), d = i % (DP / 4) * 4;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kPagWaves; ++w) x += *reinterpret_cast<const f32x4*>(&rows[(w * kPagHeads + h) * DP + d]);
    if (parts > 1) {
      *reinterpret_cast<f32x4*>(to_part + h * DP + d) = x;
    } else if (d < dim) {
      typename Attn<T>::vec4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(x[e]);
      *reinterpret_cast<typename Attn<T>::vec4*>(reinterpret_cast<T*>(a.out) + seq * a.out_row + (kv * share + head0 + h) * a.out_head + d) = y;
    }
  }
}

// Joins the parts of a sequence's head: a workgroup each, threads of a dimension and of every kPagThreads / DP-th part.
template <typename T, int DP>
__global__ __launch_bounds__(kPagThreads) void paged_join_kernel(fr_paged_args a) {
  constexpr int kLanes = DP / 4, kAtOnce = kPagThreads / kLanes;  // threads of a row, four dimensions each
  __shared__ float rows[kAtOnce][DP];
  __shared__ float weight_of[kAtOnce];
  const int64_t seq = blockIdx.x / a.heads;
  const int head = static_cast<int>(blockIdx.x % a.heads), share = static_cast<int>(a.heads / a.kv_heads), tiles = (share + kPagHeads - 1) / kPagHeads;
  const int columns = static_cast<int>(a.kv_heads) * tiles, kv = head / share, in = head % share;
  const int column = kv * tiles + in / kPagHeads, h = in % kPagHeads;
  const int64_t part = pag_part(a);
  const int parts = pag_parts(pag_length(a, seq), part);
  if (parts == 1) return;
  int64_t slot = 0;
  for (int64_t b = threadIdx.x & 63; b < seq; b += kWave) slot += pag_parts(pag_length(a, b), part);
  slot = wave_sum_i64(slot);
  const int64_t pitch = static_cast<int64_t>(columns) * (kPagHeads * (DP + 2));
  const float* from = reinterpret_cast<const float*>(a.workspace) + (slot * columns + column) * (kPagHeads * (DP + 2));
  const float* tops = from + kPagHeads * DP + h;
  float all = -INFINITY;
  for (int p = threadIdx.x & 63; p < parts; p += kWave) all = fmaxf(all, tops[p * pitch]);
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) all = fmaxf(all, __shfl_xor(all, s, kWave));
  const int mine = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  float weight = 0.f;
  if (mine < kAtOnce)
    for (int p = mine; p < parts; p += kAtOnce) {
      const float top = tops[p * pitch], by = top == -INFINITY ? 0.f : exp2_of(top - all);
      weight += by * tops[p * pitch + kPagHeads];
      x += *reinterpret_cast<const f32x4*>(from + p * pitch + h * DP + d) * by;
    }
  if (mine < kAtOnce) {
    *reinterpret_cast<f32x4*>(&rows[mine][d]) = x;
    if (d == 0) weight_of[mine] = weight;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.dim; i += kPagThreads) {
    float sum = 0.f, total = 0.f;
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) sum += rows[r][i], total += weight_of[r];
    reinterpret_cast<T*>(a.out)[seq * a.out_row + head * a.out_head + i] = static_cast<T>(total == 0.f ? 0.f : sum / total);
  }
}

int pag_dim(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }

int64_t pag_columns(int64_t heads, int64_t kv_heads) { return kv_heads * ceil_div(heads / kv_heads, kPagHeads); }

// Places for parts, per key head and 16 of its query heads: one per sequence and, where a sequence may be longer than a part's least, enough more that
// about kPagGroups workgroups share the keys.
constexpr int64_t kPagGroups = 1024;
int64_t pag_slots(int64_t B, int64_t heads, int64_t kv_heads, int64_t most) {
  if (most <= kPagStep) return B;
  const int64_t spare = ceil_div(kPagGroups, pag_columns(heads, kv_heads)), useful = B * ceil_div(most, kPagStep);
  return B + (spare < useful ? spare : useful);
}

template <typename T, int DP>
int launch_paged(const fr_paged_args& a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.slots * pag_columns(a.heads, a.kv_heads))), block(kPagThreads);
  if (a.page_size % 16 == 0) hipLaunchKernelGGL((paged_attention_kernel<T, DP, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_attention_kernel<T, DP, false>), grid, block, 0, st, a);
  int rc = check_launch("paged_attention_kernel");
  if (rc != FR_OK || a.slots == a.B) return rc;
  hipLaunchKernelGGL((paged_join_kernel<T, DP>), dim3(static_cast<unsigned>(a.B * a.heads)), block, 0, st, a);
  return check_launch("paged_join_kernel");
}

template <typename T>
int dispatch_paged(const fr_paged_args& a, hipStream_t st) {
  switch (pag_dim(a.dim)) {
    case 64: return launch_paged<T, 64>(a, st);
    case 128: return launch_paged<T, 128>(a, st);
    case 192: return launch_paged<T, 192>(a, st);
    default: return launch_paged<T, 256>(a, st);
  }
}

int check_paged_sizes(int64_t B, int64_t heads, int64_t kv_heads, int64_t dim, int64_t most) {
  FR_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 65536, FR_E_SHAPE, "fr_paged_attention: %lld heads over %lld key heads",
             (long long)heads, (long long)kv_heads);
  FR_REQUIRE(dim >= 8 && dim <= 256 && dim % 8 == 0, FR_E_SHAPE, "fr_paged_attention: head size %lld: a multiple of 8 up to 256", (long long)dim);
  FR_REQUIRE(most >= 0 && most <= (int64_t(1) << 30), FR_E_SHAPE, "fr_paged_attention: a table of %lld keys: up to 2^30", (long long)most);
  FR_REQUIRE(B >= 0 && B <= (1 << 20) && B * heads <= (1 << 26), FR_E_SHAPE, "fr_paged_attention: %lld rows of %lld heads", (long long)B, (long long)heads);
  return FR_OK;
}

}  // namespace
}  // namespace fr

extern "C" int64_t fr_paged_attention_workspace_bytes(int64_t B, int64_t heads, int64_t kv_heads, int64_t dim, int64_t most) {
  using namespace fr;
  if (check_paged_sizes(B, heads, kv_heads, dim, most) != FR_OK) return -1;
  const int64_t slots = pag_slots(B, heads, kv_heads, most);
  return slots == B ? 0 : slots * pag_columns(heads, kv_heads) * kPagHeads * (pag_dim(dim) + 2) * 4;
}

extern "C" int fr_paged_attention(const fr_paged_args* args, void* stream) {
  using namespace fr;
  FR_REQUIRE(args, FR_E_NULL, "fr_paged_attention: null pointer");
  fr_paged_args a = *args;
  FR_REQUIRE(a.page_size >= 1 && a.page_size <= (1 << 20) && a.table_pages >= 0 && a.table_pages <= (1 << 30) && a.pages >= 0, FR_E_SHAPE,
             "fr_paged_attention: tables of %lld pages of %lld keys", (long long)a.table_pages, (long long)a.page_size);
  const int64_t most = a.table_pages * a.page_size;
  const int rc = check_paged_sizes(a.B, a.heads, a.kv_heads, a.dim, most);
  if (rc != FR_OK) return rc;
  FR_REQUIRE(a.dtype == FR_F16 || a.dtype == FR_BF16, FR_E_DTYPE, "fr_paged_attention: dtype %lld not in {f16, bf16}", (long long)a.dtype);
  FR_REQUIRE(a.scale >= 1e-20 && a.scale <= 1e20, FR_E_SHAPE, "fr_paged_attention: scale %g outside [1e-20, 1e20]", a.scale);
  if (a.B == 0) return FR_OK;
  FR_REQUIRE(a.q && a.out && a.lengths && (most == 0 || (a.table && (a.pages == 0 || (a.k_cache && a.v_cache)))), FR_E_NULL, "fr_paged_attention: null pointer");
  const int64_t strides = a.q_row | a.q_head | a.k_cache_page | a.k_cache_slot | a.k_cache_head | a.v_cache_page | a.v_cache_slot | a.v_cache_head | a.out_row | a.out_head;
  FR_REQUIRE(aligned16(a.q) && aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.out) && strides % 8 == 0, FR_E_ALIGN,
             "fr_paged_attention: q, out and the cache: 16-byte aligned, strides multiples of 8 elements");
  a.slots = pag_slots(a.B, a.heads, a.kv_heads, most);
  const int64_t need = fr_paged_attention_workspace_bytes(a.B, a.heads, a.kv_heads, a.dim, most);
  FR_REQUIRE(need == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= need), FR_E_WORKSPACE,
             "fr_paged_attention: workspace of %lld bytes, %lld needed", (long long)a.workspace_bytes, (long long)need);
  a.page_shift = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctzll(a.page_size) : -1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FR_BF16 ? dispatch_paged<bf16_t>(a, st) : dispatch_paged<f16_t>(a, st);
}

// Attention of one query row per sequence over its pages: every key and value is read once, a flop per byte and query head that
// shares it (4 D of each for a key, its value and a head), so the cache's way from memory bounds it.
//
// A wavefront takes the query heads of one key head (up to 16, the columns of a matrix instruction: a "column") and a part of one sequence's keys,
// in runs of 32 with a running maximum and sum:
//   S^T [32 keys, 16 heads] = K Q^T: rows of K are the first operand as they lie in memory, straight to registers.
//   O^T [dim, 16 heads] += V^T P^T: S^T's accumulators hold, per lane, 2 x 4 consecutive keys of one head, which is the second
//   operand's place for them if V^T's keys are taken in the same order: V goes through LDS (of the wavefront's own, no barrier), where
//   transposed reads give 4 consecutive keys of a dimension.
// A run's 16 KB (128 dimensions) are asked for before the run in front is worked on, in registers.  The four wavefronts of a workgroup take the same keys of
// four columns where there are so many, whose rows lie next to each other in memory (64 rows of up to 16384 keys, 8 key heads: 492 us with a key head to a
// workgroup, where a cache whose heads come first took 461); with fewer columns they share a part's keys and join their rows in LDS.
//
// The keys of all sequences are cut into parts of equal length on the device, since the lengths are there (every wavefront adds them up in its lanes, of more than 256 sequences a
// launch in front), and the workgroups, as many as the chip holds at a time, take the parts in turn.  Parts of a sequence that has one go to the output,
// others to fp32 rows with their maxima and sums, which a second launch joins.
#pragma once
#include "attention_core.h"

namespace fr {
namespace {

constexpr int kPagThreads = 256, kPagWaves = 4, kPagRun = 32, kPagHeads = 16;
constexpr int kPagHeld = kHeldLengths / kWave;  // times 64 lengths stay in the lanes

__device__ __forceinline__ int pag_length(const fr_paged_args& a, int b) {
  const int64_t cap = a.table_pages * a.page_size;
  const int n = reinterpret_cast<const int32_t*>(a.lengths)[b];
  return n < 0 ? 0 : (n > cap ? static_cast<int>(cap) : n);
}
__device__ __forceinline__ int pag_units(int n, int unit) { return static_cast<int>((static_cast<unsigned>(n) + unit - 1) / unit); }
// Parts of `per` units each, one at least.
__device__ __forceinline__ int pag_parts(int units, int per) { return units <= per ? 1 : static_cast<int>((static_cast<unsigned>(units) + per - 1) / per); }
// Units of a part where all sequences have `total`: with `slots` places as many as give every sequence its parts - the sum over b of max(1, ceil(units / per)) is at most
// total / per + B <= slots -, and `least` where there are more places than that takes.
__device__ __forceinline__ int pag_per(const fr_paged_args& a, int total) {
  const int spare = static_cast<int>(a.slots - a.B), need = static_cast<int>((static_cast<unsigned>(total) + spare - 1) / spare);
  return need < static_cast<int>(a.least) ? static_cast<int>(a.least) : need;
}

// The parts of all sequences, counted in units of `unit` keys.  Three forms: a part each (slots == B); the lengths in the lanes; what paged_plan_kernel wrote: the
// places in front of each sequence and, behind them, the units of a part.
struct PagPlan {
  const fr_paged_args& a;
  int lane, count, unit, per;  // units of a part
  bool each;
  int held[kPagHeld];  // lengths of sequences lane + 64 j
  __device__ __forceinline__ const int* plan() const { return reinterpret_cast<const int*>(a.plan); }
  __device__ __forceinline__ int parts(int n) const { return each ? 1 : pag_parts(pag_units(n, unit), per); }
  __device__ __forceinline__ PagPlan(const fr_paged_args& args, int keys) : a(args), lane(threadIdx.x & 63), count(static_cast<int>(args.B)), unit(keys), per(1) {
    // (In front of the branches, which would put a wait for arguments before it: a launch's first loads are 0.3 us each.  Few sequences: one load.)
#pragma unroll
    for (int j = 0; j < kPagHeld; ++j) held[j] = j == 0 || j * kWave < count ? (lane + j * kWave < count ? pag_length(a, lane + j * kWave) : 0) : 0;
    each = a.slots == a.B;
    if (each) return;
    if (a.plan) {
      per = __builtin_amdgcn_readfirstlane(plan()[count + 1]);
      return;
    }
    int sum = 0;
#pragma unroll
    for (int j = 0; j < kPagHeld; ++j) sum += pag_units(held[j], unit);
    per = pag_per(a, sum_of_all(sum));
  }
  // Sequence, part, number of parts and length of place `slot`; false behind the last one.
  __device__ __forceinline__ bool place(int slot, int* seq, int* nth, int* of, int* n) const {
    if (each || a.plan) {
      const int b = each ? (slot < count ? slot : -1) : place_in(plan(), count, slot);
      if (b < 0) return false;
      *seq = __builtin_amdgcn_readfirstlane(b);
      *n = __builtin_amdgcn_readfirstlane(pag_length(a, b));
      *of = parts(*n);
      *nth = each ? 0 : __builtin_amdgcn_readfirstlane(slot - plan()[b]);
      return true;
    }
    int before = 0;
#pragma unroll 1  // unrolled, 64 dimensions take 138 registers: three workgroups to a CU for four, 103 us for 82 (three rows of 131071 keys)
    for (int j = 0; j * kWave < count; ++j) {
      const int len = j == 0 ? held[0] : j == 1 ? held[1] : j == 2 ? held[2] : held[3];
      const int mine = lane + j * kWave < count ? parts(len) : 0, sum = before + sum_up_to(mine);
      const uint64_t hit = __ballot(slot < sum && slot >= sum - mine);
      if (hit) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
        *seq = j * kWave + l;
        *of = __builtin_amdgcn_readlane(mine, l);
        *nth = slot - (__builtin_amdgcn_readlane(sum, l) - *of);
        *n = __builtin_amdgcn_readlane(len, l);
        return true;
      }
      before = __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
  }
  // Places of the sequences in front of `seq`, which the lanes may differ in.
  __device__ __forceinline__ int in_front(int seq) const {
    if (a.plan) return plan()[seq];
    const int first = __builtin_amdgcn_readfirstlane(seq);  // the lowest
    int sum = 0;
#pragma unroll
    for (int j = 0; j < kPagHeld; ++j)
      if (j == 0 || j * kWave < first) sum += lane + j * kWave < first ? parts(held[j]) : 0;
    sum = sum_of_all(sum);
    for (int b = first; __any(b < seq); ++b) sum += b < seq ? parts(pag_length(a, b)) : 0;
    return sum;
  }
};

// Results of a part of the keys, by place and column: for the heads that a column has, rows of DP sums and behind them the softmax's maxima and sums (next to the rows: in
// arrays of their own 8 rows of up to 8192 keys, 256 dimensions, took 36.2 us for 35.3), whole 16 bytes together.
__host__ __device__ __forceinline__ int pag_column_heads(int share) { return share < kPagHeads ? share : kPagHeads; }
__host__ __device__ __forceinline__ int pag_column_floats(int share, int padded) { return pag_column_heads(share) * padded + (2 * pag_column_heads(share) + 3) / 4 * 4; }
template <int DP>
struct PagPart {
  float *rows, *tops, *sums;
  __device__ __forceinline__ PagPart(const fr_paged_args& a, int64_t at, int share)  // at: place * columns + column
      : rows(reinterpret_cast<float*>(a.workspace) + at * pag_column_floats(share, DP)), tops(rows + pag_column_heads(share) * DP), sums(tops + pag_column_heads(share)) {}
};

// Loads of a cache that the memory-side cache does not hold go past the caches (pag_past).
template <bool NT, typename V>
__device__ __forceinline__ V pag_load(const V* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

template <int DP>
struct PagShape {
  static constexpr int kChunks = DP / 8;                  // 16-byte pieces of a row
  static constexpr int kLoads = kPagRun * kChunks / kWave;  // of a run's V rows
  static constexpr int kSteps = DP / 32, kTiles = DP / 16;
  // Rows of V lie in LDS with their pieces exchanged in pairs, so that a transposed read's four rows, 16 elements each, meet in no bank.
  static constexpr int kMask = DP % 128 == 0 ? 7 : 3;
  // K through LDS too: a load instruction then takes whole rows, where the product's operand takes 64 bytes of 16 (64 rows of up to 16384 keys: 476 us
  // against 460, past the caches 500 against 415; with 64 dimensions, a row being 128 bytes, 82 against 92, registers for three workgroups in place of four).
  static constexpr bool kKeysToo = DP == 128;
  static __device__ __forceinline__ int k_at(int row, int chunk) { return kPagRun * DP + row * DP + (chunk ^ (row & 15)) * 8; }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * DP + (chunk ^ ((row & kMask) << 1)) * 8; }
};

// ALIGNED: pages are multiples of 16 keys, so 16 consecutive keys from a multiple of 16 on share a page.  SHARED: wavefronts that share a part's keys;
// 4 / SHARED columns to a workgroup.
template <typename T, int DP, bool ALIGNED, int SHARED, bool NT>
__global__ __launch_bounds__(kPagThreads, DP <= 64 ? 4 : DP <= 128 ? 2 : 1) void paged_attention_kernel(fr_paged_args a) {
  typedef typename Attn<T>::vec8 vec8;
  typedef typename Attn<T>::vec4 vec4;
  typedef PagShape<DP> S;
  constexpr int kStep = kPagRun * SHARED, kColumns = kPagWaves / SHARED, kSlice = (S::kKeysToo ? 2 : 1) * kPagRun * DP;
  __shared__ __attribute__((aligned(16))) char shared[kPagWaves * kSlice * sizeof(T)];
  __shared__ float max_of[kPagWaves][kPagHeads], sum_of[kPagWaves][kPagHeads];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = static_cast<int>(a.heads / a.kv_heads), tiles = (share + kPagHeads - 1) / kPagHeads, columns = static_cast<int>(a.kv_heads) * tiles;
  const int groups = columns / kColumns;
  const PagPlan plan(a, kStep);
  const int dim = static_cast<int>(a.dim), quarter = lane >> 4, low = lane & 15;
  const float scale = static_cast<float>(a.scale) * kLog2e;
  T* const vl = reinterpret_cast<T*>(shared) + wave * kSlice;  // the wavefront's V rows, and K rows
  for (int item = blockIdx.x;; item += gridDim.x) {
    const int slot = item / groups, column = (item - slot * groups) * kColumns + wave / SHARED;
    const int kv = column / tiles, head0 = (column - kv * tiles) * kPagHeads;
    const int heads = share - head0 < kPagHeads ? share - head0 : kPagHeads;  // of the columns of the matrix instruction, in use
    int seq, nth, parts, length;
    if (!plan.place(slot, &seq, &nth, &parts, &length)) return;
    const int first = parts > 1 ? nth * plan.per * kStep : 0;
    const int last = parts > 1 && length - first > plan.per * kStep ? first + plan.per * kStep : length;
    const int32_t* table = reinterpret_cast<const int32_t*>(a.table) + seq * a.table_row;
    const T* kc = reinterpret_cast<const T*>(a.k_cache) + kv * a.k_cache_head;
    const T* vc = reinterpret_cast<const T*>(a.v_cache) + kv * a.v_cache_head;

    // Q^T, the second operand: column = lane % 16
    vec8 q[S::kSteps];
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
      q[s] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
      const int d = s * 32 + quarter * 8;
      if (low < heads && d < dim)
        q[s] = *reinterpret_cast<const vec8*>(reinterpret_cast<const T*>(a.q) + seq * a.q_row + (kv * share + head0 + low) * a.q_head + d);
    }

    auto page_of = [&](int key) { return a.page_shift >= 0 ? key >> static_cast<int>(a.page_shift) : key / static_cast<int>(a.page_size); };
    // Where key `key`'s row lies, -1 behind the last key and in a page that there is not: such keys take no part, their rows are zeros.
    auto row_of = [&](int key, int64_t page_stride, int64_t slot_stride) -> int64_t {
      if (key >= last) return -1;
      const int p = page_of(key);
      const int64_t page = table[p];
      if (page < 0 || page >= a.pages) return -1;
      return page * page_stride + (key - p * static_cast<int>(a.page_size)) * slot_stride;
    };
    vec8 k[S::kLoads], v[S::kLoads];  // K: in the order of V's rows, or as the product takes them, 16 keys after the other
    static_assert(S::kLoads == 2 * S::kSteps, "as many registers either way");
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
          const vec8 none = {0, 0, 0, 0, 0, 0, 0, 0};
          if constexpr (!S::kKeysToo) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const T* from = kc + page[t] * a.k_cache_page + in[t] * a.k_cache_slot + (low * a.k_cache_slot + quarter * 8);
#pragma unroll
              for (int s = 0; s < S::kSteps; ++s) k[t * S::kSteps + s] = dim == DP || s * 32 + quarter * 8 < dim ? pag_load<NT>(reinterpret_cast<const vec8*>(from + s * 32)) : none;
            }
          }
#pragma unroll
          for (int i = 0; i < S::kLoads; ++i) {
            const int at = i * kWave + lane, row = at / S::kChunks, d = at % S::kChunks * 8, t = i * kWave / S::kChunks >= 16 ? 1 : 0;  // a load's rows are in one half
            const bool in_row = dim == DP || d < dim;
            if constexpr (S::kKeysToo) {
              const T* from = kc + page[t] * a.k_cache_page + in[t] * a.k_cache_slot + ((row - 16 * t) * a.k_cache_slot + d);
              k[i] = in_row ? pag_load<NT>(reinterpret_cast<const vec8*>(from)) : none;
            }
            const T* from = vc + page[t] * a.v_cache_page + in[t] * a.v_cache_slot + ((row - 16 * t) * a.v_cache_slot + d);
            v[i] = in_row ? pag_load<NT>(reinterpret_cast<const vec8*>(from)) : none;
          }
          return;
        }
      }
      whole = false;
      if constexpr (!S::kKeysToo) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int64_t from = row_of(base + 16 * t + low, a.k_cache_page, a.k_cache_slot);
#pragma unroll
          for (int s = 0; s < S::kSteps; ++s) {
            const int d = s * 32 + quarter * 8;
            k[t * S::kSteps + s] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
            if (from >= 0 && d < dim) k[t * S::kSteps + s] = *reinterpret_cast<const vec8*>(kc + from + d);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int at = i * kWave + lane, row = at / S::kChunks, d = at % S::kChunks * 8;
        if constexpr (S::kKeysToo) {
          const int64_t from = row_of(base + row, a.k_cache_page, a.k_cache_slot);
          k[i] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
          if (from >= 0 && d < dim) k[i] = *reinterpret_cast<const vec8*>(kc + from + d);
        }
        const int64_t from = row_of(base + row, a.v_cache_page, a.v_cache_slot);
        v[i] = vec8{0, 0, 0, 0, 0, 0, 0, 0};
        if (from >= 0 && d < dim) v[i] = *reinterpret_cast<const vec8*>(vc + from + d);
      }
    };

    f32x4 o[S::kTiles];
#pragma unroll
    for (int t = 0; t < S::kTiles; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;  // of column lane % 16: the maximum (lagging) in all four lanes, the sum of the lane's own keys
    int base = first + wave % SHARED * kPagRun;
    if (base < last) load(base);
    for (; base < last; base += kStep) {
      f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      if constexpr (!S::kKeysToo) {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
          for (int t = 0; t < 2; ++t) st[t] = Attn<T>::mma16(k[t * S::kSteps + s], q[s], st[t]);
      }
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int at = i * kWave + lane;
        if constexpr (S::kKeysToo) *reinterpret_cast<vec8*>(vl + S::k_at(at / S::kChunks, at % S::kChunks)) = k[i];
        *reinterpret_cast<vec8*>(vl + S::at(at / S::kChunks, at % S::kChunks)) = v[i];
      }
      const bool all_seen = whole;
      if (base + kStep < last) load(base + kStep);
      if constexpr (S::kKeysToo) {
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s)
#pragma unroll
          for (int t = 0; t < 2; ++t) st[t] = Attn<T>::mma16(*reinterpret_cast<const vec8*>(vl + S::k_at(t * 16 + low, s * 4 + quarter)), q[s], st[t]);
      }
      float p[2][4], high = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[t][r] = st[t][r];
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
      if (__any((high - top) * scale > kLag)) {
        high = max_over_32(max_over_16(high));
        const float now = fmaxf(top, high), by = top == -INFINITY ? 0.f : exp2_of((top - now) * scale);
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
          const T e = static_cast<T>(exp2_of(__builtin_fmaf(p[t][r] - from, scale, Attn<T>::kRaise)));  // to 8 or 11 bits: the second product's operand
          sum += static_cast<float>(e);
          pt[t * 4 + r] = e;
        }
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) {
        const int chunk = 2 * t + ((lane & 3) >> 1), rest = (lane & 1) * 4, row = quarter * 4 + (low >> 2);
        const auto lo = read_transposed<T>(vl + S::at(row, chunk) + rest), hi = read_transposed<T>(vl + S::at(row + 16, chunk) + rest);
        o[t] = Attn<T>::mma16(join8(lo, hi), pt, o[t]);
      }
    }
    sum = sum_over_32(sum_over_16(sum));

    const PagPart<DP> to_part(a, static_cast<int64_t>(slot) * columns + column, share);
    T* const to_out = reinterpret_cast<T*>(a.out) + seq * a.out_row + (kv * share + head0) * a.out_head;
    auto put = [&](int h, int d, const f32x4& x) {  // four dimensions of a head of the column
      if (parts > 1) {
        *reinterpret_cast<f32x4*>(to_part.rows + h * DP + d) = x;
      } else if (d < dim) {
        vec4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = static_cast<T>(x[e]);
        *reinterpret_cast<vec4*>(to_out + h * a.out_head + d) = y;
      }
    };
    auto put_sums = [&](float all, float total) {
      if (parts > 1 && quarter == 0 && low < heads) {
        to_part.tops[low] = all;
        to_part.sums[low] = total;
      }
    };
    if constexpr (SHARED == 1) {
      put_sums(top, sum);
      const float by = parts > 1 ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);  // no key at all: zeros
      if (low < heads) {
#pragma unroll
        for (int t = 0; t < S::kTiles; ++t) put(low, t * 16 + quarter * 4, o[t] * by);
      }
    } else {
      // The wavefronts' rows in one: fp32, over V's place in LDS.
      const int mate = wave / SHARED * SHARED;
      if (quarter == 0) max_of[wave][low] = top, sum_of[wave][low] = sum;
      __syncthreads();
      float all = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < SHARED; ++w) all = fmaxf(all, max_of[mate + w][low]);
#pragma unroll
      for (int w = 0; w < SHARED; ++w)  // (a wavefront without a key has the sum 0, one whose scores are no numbers a NaN, which stays)
        total += sum_of[mate + w][low] * (max_of[mate + w][low] == -INFINITY ? 0.f : exp2_of((max_of[mate + w][low] - all) * scale));
      float by = top == -INFINITY ? 0.f : exp2_of((top - all) * scale);
      if (parts == 1) by = total == 0.f ? 0.f : by / total;
      float* const rows = reinterpret_cast<float*>(shared);  // [wave][head][dimension]
#pragma unroll
      for (int t = 0; t < S::kTiles; ++t) *reinterpret_cast<f32x4*>(&rows[(wave * kPagHeads + low) * DP + t * 16 + quarter * 4]) = o[t] * by;
      if (wave == mate) put_sums(all, total);
      __syncthreads();
      for (int i = (wave - mate) * kWave + lane; i < heads * (DP / 4); i += SHARED * kWave) {
        const int h = i / (DP / 4), d = i % (DP / 4) * 4;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < SHARED; ++w) x += *reinterpret_cast<const f32x4*>(&rows[((mate + w) * kPagHeads + h) * DP + d]);
        put(h, d, x);
      }
      __syncthreads();  // the next part's values come after this one's rows have been read
    }
  }
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(fr_paged_args a, int unit) {
  __shared__ int of_wave[kPlanThreads / kWave];
  const int count = static_cast<int>(a.B);
  int sum = 0;
  for (int b = threadIdx.x; b < count; b += kPlanThreads) sum += pag_units(pag_length(a, b), unit);
  sum = sum_of_all(sum);
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = sum;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) total += of_wave[w];
  const int per = pag_per(a, total);
  int* const to = reinterpret_cast<int*>(a.plan);
  prefix_of(count, [&](int b) { return pag_parts(pag_units(pag_length(a, b), unit), per); }, to);
  if (threadIdx.x == 0) to[count + 1] = per;
}

// Joins the parts of a sequence's heads (join_parts); `unit`: the keys that the parts were counted in.
template <typename T, int DP>
__global__ __launch_bounds__(kPagThreads) void paged_join_kernel(fr_paged_args a, int unit, int wide) {
  typedef JoinShape<DP> J;
  const int share = static_cast<int>(a.heads / a.kv_heads), tiles = (share + kPagHeads - 1) / kPagHeads;
  const int64_t at = wide ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * J::kGroups + threadIdx.x / J::kLanes, all = a.B * a.heads;
  const int seq = static_cast<int>((at < all ? at : all - 1) / a.heads), head = static_cast<int>((at < all ? at : all - 1) - seq * a.heads);
  const PagPlan plan(a, unit);
  const int parts = plan.parts(pag_length(a, seq));
  const int kv = head / share, in = head - kv * share, columns = static_cast<int>(a.kv_heads) * tiles;
  const int64_t pitch = static_cast<int64_t>(columns) * pag_column_floats(share, DP);
  const PagPart<DP> from(a, static_cast<int64_t>(plan.in_front(seq)) * columns + kv * tiles + in / kPagHeads, share);
  const int at_head = in % kPagHeads;
  if (wide && parts == 1) return;
  join_parts<T, DP>(wide, at < all && parts > 1, parts, from.rows + at_head * DP, pitch, from.tops + at_head, from.sums + at_head, pitch, static_cast<float>(a.scale) * kLog2e,
                    reinterpret_cast<T*>(a.out) + seq * a.out_row + head * a.out_head, static_cast<int>(a.dim));
}

int pag_dim(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }

int64_t pag_columns(int64_t heads, int64_t kv_heads) { return kv_heads * ceil_div(heads / kv_heads, kPagHeads); }

// How a call is cut: wavefronts that share a part's keys, places for parts (per group of columns), the least units of a part.
struct PagCut {
  int shared;
  int64_t groups, slots, least;
};
int64_t pag_places(int64_t dim) { return dim <= 64 ? 1024 : dim <= 128 ? 512 : 256; }  // workgroups that the chip holds, by their registers: four, two or one to a CU
PagCut pag_cut(int64_t B, int64_t heads, int64_t kv_heads, int64_t dim, int64_t most) {
  const int64_t columns = pag_columns(heads, kv_heads);
  PagCut c;
  c.shared = columns % 4 == 0 ? 1 : columns % 2 == 0 ? 2 : 4;
  c.groups = columns * c.shared / kPagWaves;
  const int64_t unit = kPagRun * c.shared, useful = B * ceil_div(most, unit), once = pag_places(dim) / c.groups;
  c.slots = B;
  c.least = 1;
  // A part each where a second launch takes longer: a run after the other is 1.9 us, joining 4 us.  us, a part each / split: one row of 128 keys 12.1 / 10.5, of 256
  // 19.6 / 10.5; 32 rows of 256 20.6 / 16.0; but 128 rows of 256 26.5 / 29.9, of 512 45.6 / 50.2.
  if (most <= 64 || (most <= 512 && B * c.groups >= 256)) return c;
  // Few sequences: a part to each workgroup that the chip holds.  Many: eight times as many, taken in turn, none of less than 256 or 512 keys (32 rows of up to
  // 2048 keys, 32 key heads: 512 keys 122 us, 256 92, 128 97; 256 rows of up to 300, which fill the chip by themselves: 42, 57, 46).  64 rows of up to 16384
  // keys, parts for one / two / four / eight times the places: 591, 515, 494, 487 us.
  int64_t spare;
  if (4 * B <= once) {
    spare = once - B;
  } else {
    spare = ceil_div(8 * pag_places(dim), c.groups);
    c.least = (B * c.groups < pag_places(dim) ? 256 : 512) / unit;
  }
  c.slots = B + (spare < useful ? spare : useful);
  return c;
}

int64_t pag_part_bytes(int64_t B, int64_t slots, int64_t heads, int64_t kv_heads, int64_t dim) {
  return slots == B ? 0 : slots * pag_columns(heads, kv_heads) * pag_column_floats(static_cast<int>(heads / kv_heads), static_cast<int>(pag_dim(dim))) * 4;
}
int64_t pag_plan_bytes(int64_t B, int64_t slots) { return slots == B || B <= kHeldLengths ? 0 : round_up((B + 2) * 4, 16); }

// Whether keys and values are read past the caches: where the pages are more than the memory-side cache's 256 MB, so that what a call reads is most likely no longer there
// from the last step, however little it is.  us, past them / not: 64 rows of up to 16384 keys (2.6 GB) 421 / 462, three of 131071 (0.4 GB) 82 / 88, 32 rows (0.45 GB) 85 / 95.
// Small reads of a pool of 2.6 GB, other pages each time (16 sets in turn): 134 MB 36.7 / 39.0 and 36.2 / 39.9, 34 MB 19.9 / 20.8 and 17.9 / 18.8, 268 MB 58.2 / 63.4; the same
// pages again and again, which a layer among others does not do: 134 MB 34.8 / 32.7 and 34.3 / 32.0, 34 MB 17.0 / 16.9 and 16.4 / 15.5, 268 MB 56.5 / 53.4.  Pages of 139 MB in
// all, again and again: 35.4 / 32.5.
bool pag_past(const fr_paged_args& a) { return a.pages * a.page_size * a.kv_heads * a.dim * 2 * 2 > (int64_t(256) << 20); }

template <typename T, int DP, bool ALIGNED, bool NT>
int launch_paged(const fr_paged_args& a, const PagCut& c, hipStream_t st) {
  if (a.plan) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a, kPagRun * c.shared);
    const int rc = check_launch("paged_plan_kernel");
    if (rc != FR_OK) return rc;
  }
  const int64_t items = a.slots * c.groups;
  const dim3 grid(static_cast<unsigned>(items < pag_places(DP) ? items : pag_places(DP))), block(kPagThreads);
  if (c.shared == 1) hipLaunchKernelGGL((paged_attention_kernel<T, DP, ALIGNED, 1, NT>), grid, block, 0, st, a);
  else if (c.shared == 2) hipLaunchKernelGGL((paged_attention_kernel<T, DP, ALIGNED, 2, NT>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_attention_kernel<T, DP, ALIGNED, 4, NT>), grid, block, 0, st, a);
  int rc = check_launch("paged_attention_kernel");
  if (rc != FR_OK || a.slots == a.B) return rc;
  typedef JoinShape<DP> J;
  static_assert(J::kThreads == kPagThreads, "join_parts' workgroups");
  const bool wide = a.B * a.heads <= 1024;  // (more sequences have few parts each, most often one)
  hipLaunchKernelGGL((paged_join_kernel<T, DP>), dim3(static_cast<unsigned>(J::blocks(a.B * a.heads, wide))), block, 0, st, a, kPagRun * c.shared, wide);
  return check_launch("paged_join_kernel");
}

template <typename T, int DP>
int launch_paged_pages(const fr_paged_args& a, const PagCut& c, hipStream_t st) {
  if (a.page_size % 16 != 0) return launch_paged<T, DP, false, false>(a, c, st);
  return pag_past(a) ? launch_paged<T, DP, true, true>(a, c, st) : launch_paged<T, DP, true, false>(a, c, st);
}

template <typename T>
int dispatch_paged(const fr_paged_args& a, const PagCut& c, hipStream_t st) {
  switch (pag_dim(a.dim)) {
    case 64: return launch_paged_pages<T, 64>(a, c, st);
    case 128: return launch_paged_pages<T, 128>(a, c, st);
    case 192: return launch_paged_pages<T, 192>(a, c, st);
    default: return launch_paged_pages<T, 256>(a, c, st);
  }
}

}  // namespace

// A call of checked arguments on rows of T; in a translation unit per type (paged_attention_inst_*.hip).
template <typename T>
int paged_attention_run(const fr_paged_args& a, int64_t groups, int shared, hipStream_t st) {
  PagCut c;
  c.groups = groups;
  c.shared = shared;
  return dispatch_paged<T>(a, c, st);
}
extern template int paged_attention_run<bf16_t>(const fr_paged_args&, int64_t, int, hipStream_t);
extern template int paged_attention_run<f16_t>(const fr_paged_args&, int64_t, int, hipStream_t);

}  // namespace fr

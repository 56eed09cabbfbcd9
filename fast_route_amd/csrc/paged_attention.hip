// Attention of single tokens over a paged cache: sizes, checks and the entry points.  The kernels: paged_attention_kernel.h.
#include "paged_attention_kernel.h"
#include "fr_memory.h"

namespace fr {
namespace {

int check_paged_sizes(int64_t B, int64_t heads, int64_t kv_heads, int64_t dim, int64_t most) {
  FR_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 65536, FR_E_SHAPE, "fr_paged_attention: %lld heads over %lld key heads",
             (long long)heads, (long long)kv_heads);
  FR_REQUIRE(dim >= 8 && dim <= 256 && dim % 8 == 0, FR_E_SHAPE, "fr_paged_attention: head size %lld: a multiple of 8 up to 256", (long long)dim);
  FR_REQUIRE(most >= 0 && most <= (int64_t(1) << 30), FR_E_SHAPE, "fr_paged_attention: a table of %lld keys: up to 2^30", (long long)most);
  // (256 dimensions: four heads to a workgroup of the joining launch, kMostBlocks256 of them)
  FR_REQUIRE(B >= 0 && B <= (1 << 20) && B * heads <= 4 * kMostBlocks256 && B * ceil_div(most, kPagRun) < (int64_t(1) << 31), FR_E_SHAPE,
             "fr_paged_attention: %lld rows of %lld heads, %lld keys each: up to 2^20 rows, rows times heads below 2^26 - 3, rows times keys below 2^36", (long long)B, (long long)heads, (long long)most);
  return FR_OK;
}

}  // namespace
}  // namespace fr

extern "C" int64_t fr_paged_attention_workspace_bytes(int64_t B, int64_t heads, int64_t kv_heads, int64_t dim, int64_t most) {
  using namespace fr;
  if (check_paged_sizes(B, heads, kv_heads, dim, most) != FR_OK) return -1;
  const int64_t slots = pag_cut(B, heads, kv_heads, dim, most).slots;
  return pag_part_bytes(B, slots, heads, kv_heads, dim) + pag_plan_bytes(B, slots);
}

extern "C" int fr_paged_attention(const fr_paged_args* args, void* stream) {
  using namespace fr;
  FR_REQUIRE(args, FR_E_NULL, "fr_paged_attention: null pointer");
  fr_paged_args a = *args;
  FR_REQUIRE(a.page_size >= 1 && a.page_size <= (1 << 30) && a.table_pages >= 0 && a.table_pages <= (1 << 30) && a.pages >= 0, FR_E_SHAPE,
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
  const PagCut cut = pag_cut(a.B, a.heads, a.kv_heads, a.dim, most);
  a.slots = cut.slots;
  a.least = cut.least;
  a.plan = nullptr;
  const int64_t need = fr_paged_attention_workspace_bytes(a.B, a.heads, a.kv_heads, a.dim, most);
  FR_REQUIRE(need == 0 || (a.workspace && aligned16(a.workspace) && a.workspace_bytes >= need), FR_E_WORKSPACE,
             "fr_paged_attention: workspace of %lld bytes, %lld needed", (long long)a.workspace_bytes, (long long)need);
  const Box q(a.q, a.B, a.q_row, a.heads, a.q_head, a.dim), out(a.out, a.B, a.out_row, a.heads, a.out_head, a.dim);
  FR_REQUIRE(!meets_itself(out), FR_E_SHAPE, "fr_paged_attention: out: rows that share memory");
  FR_REQUIRE(is_same(out, q) || !meets(out, q), FR_E_SHAPE, "fr_paged_attention: out shares memory with q, and is not q itself");
  FR_REQUIRE(!meets(out, Box(a.k_cache, a.pages, a.k_cache_page, a.page_size, a.k_cache_slot, a.kv_heads, a.k_cache_head, a.dim, 1)) &&
                 !meets(out, Box(a.v_cache, a.pages, a.v_cache_page, a.page_size, a.v_cache_slot, a.kv_heads, a.v_cache_head, a.dim, 1)),
             FR_E_SHAPE, "fr_paged_attention: out shares memory with the cache");
  if (pag_plan_bytes(a.B, a.slots)) a.plan = static_cast<char*>(a.workspace) + pag_part_bytes(a.B, a.slots, a.heads, a.kv_heads, a.dim);
  a.page_shift = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctzll(a.page_size) : -1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FR_BF16 ? paged_attention_run<bf16_t>(a, cut.groups, cut.shared, st) : paged_attention_run<f16_t>(a, cut.groups, cut.shared, st);
}

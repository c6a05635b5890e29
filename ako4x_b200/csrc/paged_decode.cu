// Paged decode: the entry points, and the kernels for bf16 queries.
#include "paged_decode.cuh"

int ako::paged::run_bf16(const Params& p, const Plan& pl, int64_t dim, bool fp8, cudaStream_t st) {
  return fp8 ? launch_dim<__nv_bfloat16, true>(p, pl, dim, st) : launch_dim<__nv_bfloat16, false>(p, pl, dim, st);
}

namespace {

using namespace ako::paged;

bool sizes_ok(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_pages, int64_t page_size, int64_t window) {
  const int64_t most = 0x7fffffffLL;
  return batch >= 0 && batch < most && q_heads > 0 && kv_heads > 0 && q_heads <= (1 << 16) && q_heads % kv_heads == 0 && page_size >= 1 &&
         page_size < most && max_pages >= 0 && max_pages < most && window >= 0 && (dim == 64 || dim == 128 || dim == 256);
}

// A stride in units of `unit` elements, if it fits.
bool set_stride(uint32_t& to, int64_t elements, int64_t unit) {
  to = (uint32_t)(elements / unit);
  return elements >= 0 && elements % unit == 0 && elements / unit <= 0xffffffffLL;
}
bool set_cache(Cache& c, const ako4x_kv_cache* in, bool fp8, int64_t kv_heads, int64_t page_size) {
  const int64_t unit = fp8 ? 16 : 8;                // elements of 16 bytes
  c.data = (const uint4*)in->data;
  c.scale = in->scale;
  if (!in->data || ((uintptr_t)in->data & 15)) return false;
  if (!set_stride(c.page, in->page_stride, unit) || !set_stride(c.slot, in->slot_stride, unit) || !set_stride(c.head, in->head_stride, unit))
    return false;
  if ((page_size - 1) * (int64_t)c.slot > 0xffffffffLL) return false;   // 64 GB in a page
  if (!fp8) return true;
  if (!in->scale || ((uintptr_t)in->scale & 3)) return false;
  if (!set_stride(c.scale_page, in->scale_page_stride, 1) || !set_stride(c.scale_slot, in->scale_slot_stride, 1) ||
      !set_stride(c.scale_head, in->scale_head_stride, 1))
    return false;
  return (page_size - 1) * (int64_t)c.scale_slot + (kv_heads - 1) * (int64_t)c.scale_head <= 0xffffffffLL;
}

}  // namespace

extern "C" size_t ako4x_paged_decode_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                     int64_t max_pages, int64_t page_size, int64_t window) {
  if (batch == 0 || !sizes_ok(batch, q_heads, kv_heads, dim, max_pages, page_size, window)) return 0;
  return std::max(plan_for(batch, q_heads, kv_heads, dim, max_pages, page_size, window, false).total,
                  plan_for(batch, q_heads, kv_heads, dim, max_pages, page_size, window, true).total);
}

extern "C" int ako4x_paged_decode(const void* q, const ako4x_kv_cache* k_cache, const ako4x_kv_cache* v_cache,
                                  const int32_t* block_table, const int32_t* seq_lens, float sm_scale, int64_t window, void* o,
                                  float* lse, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t num_pages,
                                  int64_t page_size, int64_t max_pages, int dtype, int cache_dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (batch < 0 || num_pages < 0 || num_pages > 0x7fffffffLL) return AKO4X_EINVAL;
  if (dtype != AKO4X_BF16 && dtype != AKO4X_FP16) return AKO4X_EUNSUPPORTED_SHAPE;
  if (cache_dtype != dtype && cache_dtype != AKO4X_E4M3) return AKO4X_EUNSUPPORTED_SHAPE;
  if (!sizes_ok(batch, q_heads, kv_heads, dim, max_pages, page_size, window)) return AKO4X_EUNSUPPORTED_SHAPE;
  if (batch == 0) return AKO4X_OK;
  if (!q || !k_cache || !v_cache || !seq_lens || !o || !lse || (max_pages > 0 && !block_table)) return AKO4X_EINVAL;
  if ((((uintptr_t)q | (uintptr_t)o) & 15) || (((uintptr_t)block_table | (uintptr_t)seq_lens | (uintptr_t)lse) & 3)) return AKO4X_EINVAL;
  const bool fp8 = cache_dtype == AKO4X_E4M3;
  Params p = {};
  if ((!set_cache(p.k, k_cache, fp8, kv_heads, page_size) || !set_cache(p.v, v_cache, fp8, kv_heads, page_size)) && num_pages > 0)
    return AKO4X_EINVAL;
  p.same_strides = p.k.page == p.v.page && p.k.slot == p.v.slot;
  const Plan pl = plan_for(batch, q_heads, kv_heads, dim, max_pages, page_size, window, fp8);
  if (pl.total && (!workspace || workspace_bytes < pl.total)) return AKO4X_EWORKSPACE;
  if (pl.whole_rows && batch * pl.unit_ctas > 0x7fffffffLL) return AKO4X_ETOOLARGE;
  if ((uintptr_t)workspace & 15) return AKO4X_EINVAL;
  unsigned char* ws = (unsigned char*)workspace;
  p.q = q;
  p.table = block_table;
  p.lens = seq_lens;
  p.o = o;
  p.lse = lse;
  p.cut = (int2*)ws;
  p.part_ml = (float*)(ws + pl.ml);
  p.part_acc = (float*)(ws + pl.acc);
  p.scale_log2 = sm_scale * AKO_LOG2E;
  p.batch = (int)batch;
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.group = (int)(q_heads / kv_heads);
  p.head_blocks = pl.head_blocks;
  p.per_cta = pl.per_cta;
  p.unit_ctas = pl.unit_ctas;
  p.num_pages = (int)num_pages;
  p.page_size = (int)page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)page_size) : -1;
  p.max_pages = (int)max_pages;
  p.window = (int)std::min<int64_t>(window, 0x7fffffff);
  p.shares = pl.shares;
  p.whole_rows = pl.whole_rows;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == AKO4X_BF16 ? run_bf16(p, pl, dim, fp8, st) : run_fp16(p, pl, dim, fp8, st);
}

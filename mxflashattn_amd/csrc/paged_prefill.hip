// Host side of the paged prefill (prefill_kernels.h): argument checks, launch shape and
// workspace layout behind the package entry points of mxfa_package.h.
#include "mxfa_package.h"
#include "prefill_kernels.h"

namespace mxfa {

int launch_prefill_64(const PrefillParams &p, int items, bool bf16, int cache, hipStream_t st);
int launch_prefill_128(const PrefillParams &p, int items, bool bf16, int cache, hipStream_t st);
int launch_prefill_256(const PrefillParams &p, int items, bool bf16, int cache, hipStream_t st);

namespace {

bool al(const void *ptr, uintptr_t n) { return ((uintptr_t)ptr & (n - 1)) == 0; }

// Fewest keys of a piece.
constexpr int kLeastKeys = 256;

// Pieces per kv head that a call's keys are cut into, 0 where no row tile is ever cut.
// Two workgroups' worth per CU.
int target_of(int batch, int rows_q, int gq, int hkv, int hd, int64_t max_len, int num_cus) {
  if (max_len <= kLeastKeys) return 0;
  const int target = (2 * num_cus + hkv - 1) / hkv;
  const int64_t tiles = ((int64_t)rows_q * gq + kPrefillRows - 1) / kPrefillRows;
  // One sequence: its tiles all span the same keys, W / target or fewer from here on.
  if (batch == 1 && tiles >= target) return 0;
  return target;
}

struct Layout {
  size_t o, lse, desc, total;  // byte offsets
  size_t bytes;
};

// The pieces of tiles that are cut: at most two per piece aimed at (a tile is cut into
// ceil(span / most) < 2 span / most pieces, and most >= W / target).
Layout layout(int target, int hkv, int hd) {
  const size_t slots = (size_t)2 * target * hkv, rows = kPrefillRows;
  Layout w;
  w.o = 0;
  w.lse = slots * rows * hd * 4;
  w.desc = w.lse + slots * rows * 4;
  w.total = w.desc + slots * 16;
  w.bytes = target ? w.total + 16 : 0;
  return w;
}

bool sizes_fit(int batch, int rows_q, int q_heads, int kv_heads, int head_dim, int page_size,
               int block_table_width) {
  return batch > 0 && rows_q >= 0 && q_heads > 0 && kv_heads > 0 && head_dim > 0 &&
         page_size > 0 && block_table_width > 0;
}

}  // namespace
}  // namespace mxfa

using namespace mxfa;

extern "C" {

int mxfa_package_prefill_workspace_size(int batch, int rows_q, int q_heads, int kv_heads,
                                        int head_dim, int page_size, int block_table_width,
                                        int num_cus, size_t *bytes) {
  if (!bytes || num_cus <= 0 || !sizes_fit(batch, rows_q, q_heads, kv_heads, head_dim, page_size,
                                           block_table_width))
    return MXFA_EINVAL;
  const int target = target_of(batch, rows_q, q_heads / kv_heads, kv_heads, head_dim,
                               (int64_t)block_table_width * page_size, num_cus);
  *bytes = layout(target, kv_heads, head_dim).bytes;
  return MXFA_OK;
}

int mxfa_package_prefill_launch(
    const void *q, int64_t q_stride_t, int64_t q_stride_h, int rows_q,
    const int32_t *cu_seqlens_q, const void *k_cache, const void *v_cache,
    int64_t cache_stride_page, int64_t cache_stride_token, int64_t cache_stride_head,
    const float *k_scales, int64_t ks_stride_page, int64_t ks_stride_head, const float *v_scales,
    int64_t vs_stride_page, int64_t vs_stride_head, const float *k_scale, const float *v_scale,
    const int32_t *block_table, int64_t bt_stride, const int32_t *seqlens, void *out,
    int64_t out_stride_t, int64_t out_stride_h, void *workspace, size_t workspace_bytes,
    float scale, int causal, int window_left, float softcap, const float *sinks,
    const float *alibi_slopes, int batch, int q_heads, int kv_heads, int head_dim, int page_size,
    int block_table_width, int num_pages, int dtype, int cache_dtype, int num_cus, void *stream) {
  if (num_cus <= 0 || !sizes_fit(batch, rows_q, q_heads, kv_heads, head_dim, page_size,
                                 block_table_width) || num_pages <= 0)
    return MXFA_EINVAL;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MXFA_EUNSUPPORTED;
  if (q_heads % kv_heads || q_heads / kv_heads > 16 || kv_heads > 65535) return MXFA_EUNSUPPORTED;
  if (page_size > 4096 || (page_size & (page_size - 1))) return MXFA_EUNSUPPORTED;
  if (dtype != MXFA_DTYPE_F16 && dtype != MXFA_DTYPE_BF16) return MXFA_EUNSUPPORTED;
  int cache;
  if (cache_dtype == dtype) cache = kCache16;
  else if (cache_dtype == MXFA_DTYPE_FP8_E4M3) cache = kCacheE4m3;
  else if (cache_dtype == MXFA_PACKAGE_DTYPE_INT8) cache = kCacheInt8;
  else return MXFA_EUNSUPPORTED;
  const int esz = cache == kCache16 ? 2 : 1;
  const int64_t max_len = (int64_t)block_table_width * page_size;
  if (batch > kPrefillMaxBatch || max_len > 1 << 30) return MXFA_EUNSUPPORTED;
  if (rows_q == 0) return MXFA_OK;
  if (!q || !cu_seqlens_q || !k_cache || !v_cache || !block_table || !seqlens || !out)
    return MXFA_EINVAL;
  if (!al(q, 16) || !al(k_cache, 16) || !al(v_cache, 16) || !al(out, 8) || !al(cu_seqlens_q, 4) ||
      !al(block_table, 4) || !al(seqlens, 4) || !al(k_scales, 4) || !al(v_scales, 4) ||
      !al(k_scale, 4) || !al(v_scale, 4) || !al(sinks, 4) || !al(alibi_slopes, 4))
    return MXFA_EINVAL;
  if (((q_stride_t | q_stride_h) & 7) || ((out_stride_t | out_stride_h) & 3) || q_stride_t < 0 ||
      q_stride_h < 0 || out_stride_t < 0 || out_stride_h < 0)
    return MXFA_EINVAL;
  const int64_t lines = (cache_stride_page | cache_stride_token | cache_stride_head) * esz;
  if ((lines & 15) || cache_stride_page < 0 || cache_stride_token < 0 || cache_stride_head < 0 ||
      bt_stride < 0 || ks_stride_page < 0 || ks_stride_head < 0 || vs_stride_page < 0 ||
      vs_stride_head < 0)
    return MXFA_EINVAL;
  // Rows of the output are written by different workgroups: none may share memory.
  const bool heads_apart = q_heads == 1 || out_stride_h >= head_dim;
  if (rows_q > 1 ? !(heads_apart && out_stride_t >= (q_heads - 1) * out_stride_h + head_dim) &&
                       !(out_stride_t >= head_dim &&
                         out_stride_h >= (rows_q - 1) * out_stride_t + head_dim)
                 : !heads_apart)
    return MXFA_EINVAL;
  if (window_left < -1 || !(softcap >= 0.f) || isinf(softcap)) return MXFA_EINVAL;
  const int gq = q_heads / kv_heads, rows = kPrefillRows;
  const int target = target_of(batch, rows_q, gq, kv_heads, head_dim, max_len, num_cus);
  const Layout w = layout(target, kv_heads, head_dim);
  if (w.bytes && (!workspace || !al(workspace, 16) || workspace_bytes < w.bytes))
    return MXFA_EWORKSPACE;
  if ((int64_t)rows_q * gq > 0x7fffff00) return MXFA_EUNSUPPORTED;
  // Items (row tiles and pieces) of a kv head: no sequence's rows fill more than one tile in
  // part, and cutting adds at most W / most <= target.
  const int64_t items =
      (int64_t)rows_q * gq / rows + (batch < rows_q ? batch : rows_q) + target;
  if (items * kv_heads > 0x7fffffff || (int64_t)2 * target * kv_heads > 0x7fffffff)
    return MXFA_EUNSUPPORTED;
  PrefillParams p{};
  p.q = (const char *)q;
  p.q_st = q_stride_t * 2;
  p.q_sh = q_stride_h * 2;
  p.k = (const char *)k_cache;
  p.v = (const char *)v_cache;
  p.sp = cache_stride_page * esz;
  p.st = cache_stride_token * esz;
  p.sh = cache_stride_head * esz;
  p.ks = cache == kCache16 ? nullptr : k_scales;
  p.vs = cache == kCache16 ? nullptr : v_scales;
  p.ks_sp = ks_stride_page;
  p.ks_sh = ks_stride_head;
  p.vs_sp = vs_stride_page;
  p.vs_sh = vs_stride_head;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.seqlens = seqlens;
  p.cu = cu_seqlens_q;
  p.out = (char *)out;
  p.o_st = out_stride_t * 2;
  p.o_sh = out_stride_h * 2;
  p.sinks = sinks;
  p.alibi = alibi_slopes;
  p.scale = scale;
  p.softcap = softcap;
  p.causal = causal != 0;
  // A window over every position that a table holds hides nothing (and stays clear of the end
  // of 32 bits).
  p.window_left = window_left < max_len ? window_left : -1;
  p.batch = batch;
  p.rows_q = rows_q;
  p.hkv = kv_heads;
  p.gq = gq;
  p.ps_log2 = __builtin_ctz((unsigned)page_size);
  p.max_len = (int)max_len;
  p.num_pages = num_pages;
  // A window's keys, its tokens' windows together (and a tile's worth ahead of them).
  const int64_t span = (int64_t)p.window_left + rows / gq + 1 + kPrefillKeys;
  p.span = (int)(p.window_left < 0 || span > max_len ? max_len : span);
  const auto mul = [](int d) {
    return d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d);
  };
  p.hkv_mul = mul(kv_heads);
  p.gq_mul = mul(gq);
  p.target = target;
  p.least = kLeastKeys;
  p.max_slots = 2 * target;
  p.uniform = page_size >= 16 && cache_stride_page * esz < (int64_t)1 << 32 &&
              cache_stride_token * esz < (int64_t)1 << 24 &&
              (int64_t)page_size * cache_stride_token * esz < (int64_t)1 << 32;
  char *ws = (char *)workspace;
  if (target) {
    p.ws_o = (float *)(ws + w.o);
    p.ws_lse = (float *)(ws + w.lse);
    p.ws_desc = (int4 *)(ws + w.desc);
    p.ws_total = (int *)(ws + w.total);
  }
  const bool bf16 = dtype == MXFA_DTYPE_BF16;
  hipStream_t st = (hipStream_t)stream;
  switch (head_dim) {
    case 64: return launch_prefill_64(p, (int)items, bf16, cache, st);
    case 128: return launch_prefill_128(p, (int)items, bf16, cache, st);
    default: return launch_prefill_256(p, (int)items, bf16, cache, st);
  }
}

}  // extern "C"

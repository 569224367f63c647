// The paged KV cache in 8 bits with one scale for each token and kv head: the write
// (quantising rows of K and V as they go to their slots) and reading pages back.
//
// A row x of HD elements is stored as codes c and a scale s, both by 32-bit arithmetic:
//   s = max(max_i |x_i| / TOP, 2^-126),  c_i = x_i / s to the nearest, ties to even,
// TOP = 448 (e4m3fn) or 127 (int8). The floor keeps s a normal number, so a row of zeros
// has codes 0 and no division by zero. A row with an infinity or a NaN has no such scale:
// it gets s = NaN and codes 0, and so reads back as NaN. Read back, element i is c_i * s,
// rounded once to the output's type.
//
// Both kernels are bound by memory (2 bytes read, 1 written an element, or the reverse)
// and small calls by the latency of their dependent loads: slot, row; or offsets, page,
// row. One thread moves 16 bytes of the 16-bit side of K and of V.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mxfa_device.h"
#include "mxfa_mi355x.h"
#include "mxfa_package.h"

namespace mxfa {
namespace {

constexpr int kQuantThreads = 256;

struct QuantParams {
  const uint16_t *k, *v;
  int64_t s_t, s_h;  // source strides (token, head), elements
  uint8_t *kc, *vc;
  int64_t c_sp, c_st, c_sh;  // cache strides, bytes
  float *ks, *vs;
  int64_t ks_sp, ks_sh, vs_sp, vs_sh;  // scale strides, elements (page, head; token: 1)
  const int64_t *slots;
  int rows, hkv, frags, lanes_log2;  // rows of tokens; 8-element fragments of a row; lanes of one
  int ps_log2, num_pages;
};

// Largest |x| of packed 16-bit elements as its bits: magnitudes order as integers, above
// all finite ones infinity, above it NaN.
__device__ __forceinline__ uint32_t pair_top(uint32_t w, uint32_t top) {
  const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
  return max(top, max(a, b));
}

template <typename T>
__device__ __forceinline__ uint32_t row_top(const uint4 w, int lanes) {
  uint32_t top = pair_top(w.x, pair_top(w.y, pair_top(w.z, pair_top(w.w, 0u))));
  for (int d = lanes >> 1; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  return top;
}

template <typename T, bool kInt8>
__device__ __forceinline__ float row_scale(uint32_t top) {
  const float s = fmaxf(__fdiv_rn(Elem<T>::lo(top), kInt8 ? 127.f : 448.f), 0x1p-126f);
  const bool finite = std::is_same_v<T, BF16> ? top < 0x7f80u : top < 0x7c00u;
  return finite ? s : __builtin_nanf("");
}

// x / s correctly rounded from y = 1 / s correctly rounded: with q = x y off by an ulp at
// most, the residual x - q s is exact in one fma, and q plus the residual times y rounds to
// the quotient's nearest (Markstein's theorem). Exact where the residual is no subnormal
// number, so for |x| of 2^-100 or more; below that (s is then the larger by far, see kFastScale)
// the quotient is so small that its code is 0 either way.
__device__ __forceinline__ float quotient(float x, float s, float y) {
  const float q = x * y;
  return __builtin_fmaf(__builtin_fmaf(-q, s, x), y, q);
}
// Rows of smaller scales take the division itself. Three instructions an element instead of
// ten: 16384 rows of 8 x 128, bf16 to e4m3fn, 28.7 -> 20.7 us on MI355X (102 MB, 4.9 TB/s; a
// large copy reaches 4.8).
constexpr float kFastScale = 0x1p-60f;

// Four codes of x / s. No quotient needs a clamp: |x| <= TOP s (1 + 2^-23), which rounds to
// TOP or less.
template <bool kInt8>
__device__ __forceinline__ uint32_t quad_codes(float a, float b, float c, float d) {
  if constexpr (kInt8) {
    const auto one = [&](float x) { return (uint32_t)(int)__builtin_rintf(x); };
    const uint32_t lo = __builtin_amdgcn_perm(one(b), one(a), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(one(d), one(c), 0x04000c0cu);
    return lo | hi;
  } else {
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  }
}

template <typename T, bool kInt8>
__device__ __forceinline__ uint2 row_codes(const uint4 w, float s) {
  using E = Elem<T>;
  float x[8] = {E::lo(w.x), E::hi(w.x), E::lo(w.y), E::hi(w.y),
                E::lo(w.z), E::hi(w.z), E::lo(w.w), E::hi(w.w)};
  if (s >= kFastScale) {
    const float y = __fdiv_rn(1.f, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = quotient(x[i], s, y);
  } else {
    // (s = NaN: codes 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s != s ? 0.f : __fdiv_rn(x[i], s);
  }
  return make_uint2(quad_codes<kInt8>(x[0], x[1], x[2], x[3]),
                    quad_codes<kInt8>(x[4], x[5], x[6], x[7]));
}

// A group of 2^lanes_log2 lanes (the power of two at or above HD / 8) takes one row of one
// head, K and V, so its largest element is a few exchanges inside the wave.
// I = uint32_t (calls of fewer rows x heads than 2^31 less a step): divisions in 32 bits.
template <typename T, bool kInt8, typename I>
__global__ __launch_bounds__(kQuantThreads) void quantize_and_cache_kernel(QuantParams p) {
  const int lanes = 1 << p.lanes_log2;
  const int f = threadIdx.x & (lanes - 1);
  const I total = (I)p.rows * (I)p.hkv;
  const I step = (I)gridDim.x * (I)(kQuantThreads >> p.lanes_log2);
  for (I i = (I)blockIdx.x * (I)(kQuantThreads >> p.lanes_log2) +
             (I)(threadIdx.x >> p.lanes_log2);
       i < total; i += step) {
    const int r = (int)(i / (I)p.hkv), h = (int)(i - (I)r * (I)p.hkv);
    // The row's loads go out with the slot's: they do not depend on it.
    const int64_t slot = p.slots[r];
    uint4 wk = make_uint4(0u, 0u, 0u, 0u), wv = wk;
    if (f < p.frags) {
      const int64_t src = (int64_t)r * p.s_t + (int64_t)h * p.s_h + f * 8;
      wk = *reinterpret_cast<const uint4 *>(p.k + src);
      wv = *reinterpret_cast<const uint4 *>(p.v + src);
    }
    const int64_t page = slot >> p.ps_log2;
    if (slot < 0 || page >= p.num_pages) continue;  // the same for the whole group
    const int off = (int)(slot & ((1 << p.ps_log2) - 1));
    const float ks = row_scale<T, kInt8>(row_top<T>(wk, lanes));
    const float vs = row_scale<T, kInt8>(row_top<T>(wv, lanes));
    if (f < p.frags) {
      const int64_t dst = page * p.c_sp + (int64_t)off * p.c_st + (int64_t)h * p.c_sh + f * 8;
      *reinterpret_cast<uint2 *>(p.kc + dst) = row_codes<T, kInt8>(wk, ks);
      *reinterpret_cast<uint2 *>(p.vc + dst) = row_codes<T, kInt8>(wv, vs);
    }
    if (f == 0) {
      p.ks[page * p.ks_sp + (int64_t)h * p.ks_sh + off] = ks;
      p.vs[page * p.vs_sp + (int64_t)h * p.vs_sh + off] = vs;
    }
  }
}

struct GatherParams {
  const uint8_t *kc, *vc;
  int64_t c_sp, c_st, c_sh;  // bytes
  const float *ks, *vs;      // per row, or null
  int64_t ks_sp, ks_sh, vs_sp, vs_sh;
  const float *k_scale, *v_scale;  // per cache, or null
  const int32_t *bt;
  int64_t bt_stride;
  const int32_t *cu;
  uint16_t *ko, *vo;
  int64_t o_st, o_sh;  // elements
  int batch, btw, total, hkv, frags;  // frags: 8-element fragments of a row
  int ps_log2, num_pages;
};

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  return (uint32_t)Elem<T>::narrow(a) | ((uint32_t)Elem<T>::narrow(b) << 16);
}

// Eight codes times s: the 32-bit product, then one rounding. (The empty statement keeps the
// two apart: joined in one instruction, fp16's would round the exact product, bf16's not.)
template <typename T, bool kInt8>
__device__ __forceinline__ uint4 read_codes(uint2 c, float s) {
  const uint32_t in[2] = {c.x, c.y};
  uint32_t out[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float x[4];
    if constexpr (kInt8) {
      const int w = (int)in[j];
      x[0] = (float)((w << 24) >> 24);
      x[1] = (float)((w << 16) >> 24);
      x[2] = (float)((w << 8) >> 24);
      x[3] = (float)(w >> 24);
    } else {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)in[j], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)in[j], true);
      x[0] = lo[0];
      x[1] = lo[1];
      x[2] = hi[0];
      x[3] = hi[1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] *= s;
      if constexpr (std::is_same_v<T, F16>) asm("" : "+v"(x[i]));
    }
    out[2 * j] = pack_pair<T>(x[0], x[1]);
    out[2 * j + 1] = pack_pair<T>(x[2], x[3]);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// A block takes kGatherRows consecutive rows: threads 0.. find each row's sequence (a binary
// search of the offsets) and place, in LDS, then all threads move the rows, 16 bytes of the
// narrower side of K and of V each, their loads all out before the first store. Against a
// thread that searched for its own eight codes: 16 sequences of 1k-8k int8 rows, 8 x 128,
// 138 -> 95 us on MI355X (437 MB, 4.6 TB/s).
// kBits 16: the cache holds T itself; 8: codes (kInt8 or e4m3fn).
constexpr int kGatherRows = 16;

template <typename T, int kBits, bool kInt8>
__global__ __launch_bounds__(kQuantThreads) void gather_cache_kernel(GatherParams p) {
  __shared__ int64_t s_page[kGatherRows];  // -1: a row of no sequence
  __shared__ int s_off[kGatherRows];
  const int r0 = blockIdx.x * kGatherRows;
  const int rows = min(kGatherRows, p.total - r0);
  if ((int)threadIdx.x < rows) {
    const int r = r0 + threadIdx.x;
    // The last sequence that starts at or before row r.
    int lo = 0, n = p.batch;
    while (n > 1) {
      const int half = n >> 1;
      const bool right = p.cu[lo + half] <= r;
      lo = right ? lo + half : lo;
      n = right ? n - half : half;
    }
    const int pos = r - p.cu[lo];
    const int pidx = pos >> p.ps_log2;
    int64_t page = -1;
    if (pos >= 0 && r < p.cu[lo + 1] && pidx < p.btw)
      page = min(max(p.bt[(int64_t)lo * p.bt_stride + pidx], 0), p.num_pages - 1);
    s_page[threadIdx.x] = page;
    s_off[threadIdx.x] = pos & ((1 << p.ps_log2) - 1);
  }
  __syncthreads();
  constexpr int kElems = kBits == 16 ? 8 : 16;  // of a thread's 16 bytes
  const int frags = p.frags / (kElems / 8);     // of a row
  const int units = p.hkv * frags;              // of a token
  const int all = rows * units;
  constexpr int kAhead = 4;
  for (int i0 = threadIdx.x; i0 < all; i0 += kAhead * kQuantThreads) {
    uint4 ck[kAhead], cv[kAhead];
    float ks[kAhead], vs[kAhead];
    int64_t dst[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = min(i0 + a * kQuantThreads, all - 1);
      const int row = i / units, u = i - row * units;
      const int h = u / frags, f = u - h * frags;
      const int64_t page = s_page[row];
      const int off = s_off[row];
      dst[a] = page < 0 || i0 + a * kQuantThreads >= all
                   ? -1
                   : (int64_t)(r0 + row) * p.o_st + (int64_t)h * p.o_sh + f * kElems;
      const int64_t at = max(page, (int64_t)0);
      const int64_t src = at * p.c_sp + (int64_t)off * p.c_st + (int64_t)h * p.c_sh + f * 16;
      ck[a] = load_stream16(p.kc + src);
      cv[a] = load_stream16(p.vc + src);
      if constexpr (kBits == 8) {
        ks[a] = p.ks   ? p.ks[at * p.ks_sp + (int64_t)h * p.ks_sh + off]
                : p.k_scale ? p.k_scale[0]
                            : 1.f;
        vs[a] = p.vs   ? p.vs[at * p.vs_sp + (int64_t)h * p.vs_sh + off]
                : p.v_scale ? p.v_scale[0]
                            : 1.f;
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (dst[a] < 0) continue;
      uint4 *const k = reinterpret_cast<uint4 *>(p.ko + dst[a]);
      uint4 *const v = reinterpret_cast<uint4 *>(p.vo + dst[a]);
      if constexpr (kBits == 16) {
        *k = ck[a];
        *v = cv[a];
      } else {
        k[0] = read_codes<T, kInt8>(make_uint2(ck[a].x, ck[a].y), ks[a]);
        k[1] = read_codes<T, kInt8>(make_uint2(ck[a].z, ck[a].w), ks[a]);
        v[0] = read_codes<T, kInt8>(make_uint2(cv[a].x, cv[a].y), vs[a]);
        v[1] = read_codes<T, kInt8>(make_uint2(cv[a].z, cv[a].w), vs[a]);
      }
    }
  }
}

bool al(const void *ptr, uintptr_t n) { return ((uintptr_t)ptr & (n - 1)) == 0; }

int log2_of(int v) {
  if (v <= 0 || (v & (v - 1))) return -1;
  return __builtin_ctz((unsigned)v);
}

unsigned blocks_for(int64_t threads) {
  const int64_t b = (threads + kQuantThreads - 1) / kQuantThreads;
  return (unsigned)(b > 65536 ? 65536 : b);
}

}  // namespace
}  // namespace mxfa

using namespace mxfa;

extern "C" {

int mxfa_package_quantize_and_cache_launch(
    const void *key, const void *value, int64_t kv_stride_token, int64_t kv_stride_head,
    void *k_cache, void *v_cache, int64_t cache_stride_page, int64_t cache_stride_token,
    int64_t cache_stride_head, float *k_scales, int64_t ks_stride_page, int64_t ks_stride_head,
    float *v_scales, int64_t vs_stride_page, int64_t vs_stride_head, const int64_t *slot_mapping,
    int num_tokens, int kv_heads, int head_dim, int page_size, int num_pages, int dtype,
    int cache_dtype, void *stream) {
  if (num_tokens < 0 || kv_heads <= 0 || num_pages <= 0 || page_size <= 0) return MXFA_EINVAL;
  const int ps = log2_of(page_size);
  if (ps < 0 || head_dim <= 0 || head_dim % 16 || head_dim > 512) return MXFA_EUNSUPPORTED;
  if (dtype != MXFA_DTYPE_F16 && dtype != MXFA_DTYPE_BF16) return MXFA_EUNSUPPORTED;
  if (cache_dtype != MXFA_DTYPE_FP8_E4M3 && cache_dtype != MXFA_PACKAGE_DTYPE_INT8)
    return MXFA_EUNSUPPORTED;
  if (num_tokens == 0) return MXFA_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scales || !v_scales || !slot_mapping)
    return MXFA_EINVAL;
  if (!al(key, 16) || !al(value, 16) || !al(k_cache, 16) || !al(v_cache, 16) ||
      !al(k_scales, 4) || !al(v_scales, 4) || !al(slot_mapping, 8))
    return MXFA_EINVAL;
  if (k_cache == v_cache || k_scales == v_scales) return MXFA_EINVAL;
  if (((kv_stride_token | kv_stride_head) & 7) || kv_stride_token < 0 || kv_stride_head < 0 ||
      ((cache_stride_page | cache_stride_token | cache_stride_head) & 15) ||
      cache_stride_page < 0 || cache_stride_token < 0 || cache_stride_head < 0 ||
      ks_stride_page < 0 || ks_stride_head < 0 || vs_stride_page < 0 || vs_stride_head < 0)
    return MXFA_EINVAL;
  QuantParams p{};
  p.k = (const uint16_t *)key;
  p.v = (const uint16_t *)value;
  p.s_t = kv_stride_token;
  p.s_h = kv_stride_head;
  p.kc = (uint8_t *)k_cache;
  p.vc = (uint8_t *)v_cache;
  p.c_sp = cache_stride_page;
  p.c_st = cache_stride_token;
  p.c_sh = cache_stride_head;
  p.ks = k_scales;
  p.vs = v_scales;
  p.ks_sp = ks_stride_page;
  p.ks_sh = ks_stride_head;
  p.vs_sp = vs_stride_page;
  p.vs_sh = vs_stride_head;
  p.slots = slot_mapping;
  p.rows = num_tokens;
  p.hkv = kv_heads;
  p.frags = head_dim / 8;
  while ((1 << p.lanes_log2) < p.frags) ++p.lanes_log2;
  p.ps_log2 = ps;
  p.num_pages = num_pages;
  const unsigned blocks = blocks_for(((int64_t)num_tokens * kv_heads) << p.lanes_log2);
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kQuantThreads), 0, (hipStream_t)stream, p);
  };
  const bool i8 = cache_dtype == MXFA_PACKAGE_DTYPE_INT8;
  const auto pick = [&](auto type, auto codes) {
    using T = decltype(type);
    constexpr bool kInt8 = decltype(codes)::value;
    if ((int64_t)num_tokens * kv_heads < ((int64_t)1 << 31) - ((int64_t)1 << 24))
      go(quantize_and_cache_kernel<T, kInt8, uint32_t>);
    else
      go(quantize_and_cache_kernel<T, kInt8, int64_t>);
  };
  if (dtype == MXFA_DTYPE_BF16)
    i8 ? pick(BF16{}, std::true_type{}) : pick(BF16{}, std::false_type{});
  else
    i8 ? pick(F16{}, std::true_type{}) : pick(F16{}, std::false_type{});
  return hipGetLastError() == hipSuccess ? MXFA_OK : MXFA_ELAUNCH;
}

int mxfa_package_gather_cache_launch(
    const void *k_cache, const void *v_cache, int64_t cache_stride_page,
    int64_t cache_stride_token, int64_t cache_stride_head, const float *k_scales,
    int64_t ks_stride_page, int64_t ks_stride_head, const float *v_scales, int64_t vs_stride_page,
    int64_t vs_stride_head, const float *k_scale, const float *v_scale,
    const int32_t *block_table, int64_t bt_stride, const int32_t *cu_seqlens, void *k_out,
    void *v_out, int64_t out_stride_token, int64_t out_stride_head, int batch,
    int block_table_width, int total, int kv_heads, int head_dim, int page_size, int num_pages,
    int dtype, int cache_dtype, void *stream) {
  if (batch <= 0 || block_table_width <= 0 || total < 0 || kv_heads <= 0 || num_pages <= 0 ||
      page_size <= 0)
    return MXFA_EINVAL;
  const int ps = log2_of(page_size);
  if (ps < 0 || head_dim <= 0 || head_dim % 16 || head_dim > 512) return MXFA_EUNSUPPORTED;
  if (dtype != MXFA_DTYPE_F16 && dtype != MXFA_DTYPE_BF16) return MXFA_EUNSUPPORTED;
  const bool wide = cache_dtype == dtype, i8 = cache_dtype == MXFA_PACKAGE_DTYPE_INT8;
  if (!wide && !i8 && cache_dtype != MXFA_DTYPE_FP8_E4M3) return MXFA_EUNSUPPORTED;
  if (total == 0) return MXFA_OK;
  if (!k_cache || !v_cache || !block_table || !cu_seqlens || !k_out || !v_out) return MXFA_EINVAL;
  if (!al(k_cache, 16) || !al(v_cache, 16) || !al(k_out, 16) || !al(v_out, 16) ||
      !al(k_scales, 4) || !al(v_scales, 4) || !al(k_scale, 4) || !al(v_scale, 4) ||
      !al(block_table, 4) || !al(cu_seqlens, 4))
    return MXFA_EINVAL;
  const int64_t lines =
      (cache_stride_page | cache_stride_token | cache_stride_head) * (wide ? 2 : 1);
  if ((lines & 15) || cache_stride_page < 0 || cache_stride_token < 0 || cache_stride_head < 0 ||
      ks_stride_page < 0 || ks_stride_head < 0 || vs_stride_page < 0 || vs_stride_head < 0 ||
      bt_stride < 0)
    return MXFA_EINVAL;
  // Rows of the outputs are written by different threads: none may share memory.
  if (k_out == v_out) return MXFA_EINVAL;
  if (((out_stride_token | out_stride_head) & 7) || (kv_heads > 1 && out_stride_head < head_dim) ||
      (total > 1 && out_stride_token < (kv_heads - 1) * out_stride_head + head_dim))
    return MXFA_EINVAL;
  GatherParams p{};
  const int esz = wide ? 2 : 1;
  p.kc = (const uint8_t *)k_cache;
  p.vc = (const uint8_t *)v_cache;
  p.c_sp = cache_stride_page * esz;
  p.c_st = cache_stride_token * esz;
  p.c_sh = cache_stride_head * esz;
  p.ks = wide ? nullptr : k_scales;
  p.vs = wide ? nullptr : v_scales;
  p.ks_sp = ks_stride_page;
  p.ks_sh = ks_stride_head;
  p.vs_sp = vs_stride_page;
  p.vs_sh = vs_stride_head;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.bt = block_table;
  p.bt_stride = bt_stride;
  p.cu = cu_seqlens;
  p.ko = (uint16_t *)k_out;
  p.vo = (uint16_t *)v_out;
  p.o_st = out_stride_token;
  p.o_sh = out_stride_head;
  p.batch = batch;
  p.btw = block_table_width;
  p.total = total;
  p.hkv = kv_heads;
  p.frags = head_dim / 8;
  p.ps_log2 = ps;
  p.num_pages = num_pages;
  const unsigned blocks = (unsigned)(((int64_t)total + kGatherRows - 1) / kGatherRows);
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kQuantThreads), 0, (hipStream_t)stream, p);
  };
  if (dtype == MXFA_DTYPE_BF16)
    wide ? go(gather_cache_kernel<BF16, 16, false>)
         : i8 ? go(gather_cache_kernel<BF16, 8, true>) : go(gather_cache_kernel<BF16, 8, false>);
  else
    wide ? go(gather_cache_kernel<F16, 16, false>)
         : i8 ? go(gather_cache_kernel<F16, 8, true>) : go(gather_cache_kernel<F16, 8, false>);
  return hipGetLastError() == hipSuccess ? MXFA_OK : MXFA_ELAUNCH;
}

}  // extern "C"

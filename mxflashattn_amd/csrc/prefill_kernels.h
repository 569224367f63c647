// Attention of a chunk of new tokens over a paged KV cache, for MI355X (gfx950).
//
// Sequence b has n_b query tokens, rows [cu[b], cu[b+1]) of the packed q, and L_b
// keys in its pages, the chunk's own among them; token t sits at position
// L_b - n_b + t. For query head h of kv head h / GQ:
//   x_j = cap(scale * ks_j * q.k_j) - slope_h * |pos - j|    over the keys j it sees
//   out = sum_j e^(x_j - m) vs_j v_j / (sum_j e^(x_j - m) + e^(sink_h - m)),  m = max_j x_j
// (ks, vs: the scales of an 8-bit cache's rows, 1 otherwise), one pass over the keys
// with the running maximum and sum of each row.
//
// Rows. The GQ query heads of a kv head share its keys, so row r of a sequence is
// token r / GQ, head r % GQ: a workgroup takes kRows consecutive rows of one kv head,
// 32 per wave, and reads each key once for all of them.
//
// Products, both on v_mfma_f32_32x32x16 and transposed, so that a lane holds one row's
// scores and P never changes lanes:
//   S^T[32 keys][32 rows] = K[32 x HD] . Q^T: lane l holds row l % 32 and, of each block
//     of eight keys, keys 4 (l / 32) .. + 3;
//   O^T[32 dims][32 rows] = V^T . P^T: the registers of S^T are, in order, the operand
//     P^T of a product whose k index runs over the same keys in the same order, and
//     ds_read_b64_tr_b16 reads V's rows from LDS transposed in that order.
// A row's maximum is then 31 comparisons in a lane and one swap of the wave's halves.
//
// Tiles of 64 keys go through LDS, two buffers each of K and V, rows of HD elements whose
// 16-byte chunks are permuted within the row (swizzle_k, swizzle_v) so that neither operand
// read meets a bank conflict. An 8-bit cache is widened exactly on
// its way into LDS, once for the whole workgroup; its scales join the scores (ks) and the
// weights (vs, ahead of P's one rounding) in 32 bits.
//
// Few rows and many keys: a row tile's keys are cut into pieces of about W / target keys,
// W the sum over all row tiles of the keys they span, so that about `target` workgroups
// per kv head share the work; a second launch joins the pieces. Every workgroup finds its
// tile and piece itself from the lengths on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "mxfa_device.h"
#include "mxfa_mi355x.h"

namespace mxfa {

constexpr int kPrefillKeys = 64;        // keys of a tile
constexpr int kPrefillMaxBatch = 16000;
constexpr float kPrefillLog2e = 1.4426950408889634f;
// A row's reference maximum moves only when a score passes it by this (base 2), so
// weights stay below 2^8 and most tiles leave the accumulators as they are.
constexpr float kPrefillRescaleLog2 = 8.0f;

// What the cache holds: q's 16-bit type, or 8 bits.
enum : int { kCache16 = 0, kCacheE4m3 = 1, kCacheInt8 = 2 };

struct PrefillParams {
  const char *q;
  int64_t q_st, q_sh;  // bytes (token, head)
  const char *k, *v;
  int64_t sp, st, sh;  // cache strides, bytes (page, token, head)
  const float *ks, *vs;     // 8-bit caches: scales [page][head][token], or null
  int64_t ks_sp, ks_sh, vs_sp, vs_sh;  // their strides, elements
  const float *k_scale, *v_scale;      // one scale for the whole cache, or null
  const int32_t *bt;
  int64_t bt_stride;
  const int32_t *seqlens;
  const int32_t *cu;  // first query row of each sequence, batch + 1
  char *out;
  int64_t o_st, o_sh;  // bytes
  const float *sinks, *alibi;  // per query head, or null
  float scale;         // score scale (base e)
  float softcap;       // 0: none
  int causal, window_left;
  int batch, rows_q, hkv, gq, ps_log2, max_len, num_pages;
  int target;          // pieces per kv head that the keys are cut into (0: none)
  int least;           // fewest keys of a piece
  float *ws_o, *ws_lse;  // pieces: [slot][kv head][kRows][HD], [slot][kv head][kRows]
  int4 *ws_desc;         // [slot][kv head]: pieces (0 but for a tile's first), batch, tile
  int *ws_total;         // slots in use
  int max_slots;
  int uniform;  // pages of 16 tokens or more (and rows within 32-bit offsets of each other)
};

// Waves of a workgroup, 32 rows each: eight, two per SIMD; at head dim 256, whose
// accumulators alone are 128 registers, four with all of a SIMD's registers each.
template <int HD>
constexpr int kPrefillWaves = 4;
template <int HD>
constexpr int kPrefillRows = 32 * kPrefillWaves<HD>;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

template <typename T>
struct Prod32;
template <>
struct Prod32<F16> {
  static __device__ __forceinline__ float add_pair(uint32_t w, float l) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2v, w),
                                  __builtin_bit_cast(f16x2v, 0x3c003c00u), l, false);
  }
  static __device__ __forceinline__ f32x16 run(const uint4 &a, const uint4 &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const f16x2v v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct Prod32<BF16> {
  static __device__ __forceinline__ float add_pair(uint32_t w, float l) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, w),
                                           __builtin_bit_cast(bf16x2v, 0x3f803f80u), l, false);
  }
  static __device__ __forceinline__ f32x16 run(const uint4 &a, const uint4 &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const bf16x2v v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};

// Four 8-bit codes (one word) as two packed pairs of T, exactly.
template <typename T, int kCache>
__device__ __forceinline__ uint2 widen_codes(uint32_t w) {
  if constexpr (kCache == kCacheE4m3) {
    if constexpr (std::is_same_v<T, BF16>)
      return make_uint2(
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)));
    else
      return make_uint2(
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)));
  } else {
    const int s = (int)w;
    return make_uint2(Prod32<T>::pack((float)((s << 24) >> 24), (float)((s << 16) >> 24)),
                      Prod32<T>::pack((float)((s << 8) >> 24), (float)(s >> 24)));
  }
}

// Where row r's 16-byte chunk c lies in its LDS row: c ^ swizzle(r). LDS serves 256 bytes
// a clock, each 16-byte column of them once: 16 lanes of a b128 read (16 rows' same K chunk)
// and 32 of a transposed b64 read (four rows' four V chunks) then take a clock each. (With
// permutations within 128 bytes half of LDS's busy cycles were conflicts.)
template <int HD>
__device__ __forceinline__ int swizzle_k(int r) {
  return HD == 64 ? (r >> 1) & 7 : r & 15;
}
template <int HD>
__device__ __forceinline__ int swizzle_v(int r) {
  return HD == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
}

// Byte offset of a pointer into LDS.
__device__ __forceinline__ uint32_t lds_offset(const char *ptr) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)ptr;
}

// 16 bytes a lane from base + off (base the same in the whole wave) to LDS at `lds` + 16 *
// lane, with no register in between. The compiler does not see the load: the caller waits
// for it (vmcnt) ahead of the barrier that hands the data over. (The builtin for it makes
// the compiler wait at the next LDS read, of the other buffer.)
__device__ __forceinline__ void load_to_lds(const char *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}

// What one sequence asks for: its query rows and keys, held to those that exist.
struct PrefillSeq {
  int start, n, len, tiles, span;
};

template <int kRows>
__device__ __forceinline__ PrefillSeq prefill_seq(const PrefillParams &p, int b) {
  PrefillSeq s;
  s.start = min(max(p.cu[b], 0), p.rows_q);
  const int end = min(max(p.cu[b + 1], s.start), p.rows_q);
  s.n = end - s.start;
  s.len = min(max(p.seqlens[b], 0), p.max_len);
  s.tiles = (int)(((int64_t)s.n * p.gq + kRows - 1) / kRows);
  // Keys that one row tile spans, at most: with a window its tokens' windows together.
  s.span = p.window_left < 0
               ? s.len
               : (int)min((int64_t)s.len, (int64_t)p.window_left + kRows / p.gq + 1 + kPrefillKeys);
  return s;
}

struct PrefillItem {
  int b, tile, piece, pieces, slot;
};

template <int kThreads>
struct PrefillScan {
  int64_t work[kThreads / 64];
  int items[kThreads / 64], slots[kThreads / 64];
  PrefillItem item;
};

// The row tile and piece of item `index`, in LDS for the whole workgroup; b = -1 past the
// last. Tiles of a sequence in falling order: with the causal mask the later ones see more
// keys, and the longest work goes out first.
template <int kRows, int kThreads>
__device__ __forceinline__ PrefillItem prefill_find(const PrefillParams &p, int index,
                                                    PrefillScan<kThreads> &s, bool tell) {
  constexpr int kWaves = kThreads / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = threadIdx.x * per, b1 = min(b0 + per, p.batch);
  int most = 0x7fffffff;
  if (p.target > 0) {
    int64_t work = 0;
    for (int b = b0; b < b1; ++b) {
      const PrefillSeq q = prefill_seq<kRows>(p, b);
      work += (int64_t)q.tiles * q.span;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) work += __shfl_xor(work, d);
    if (lane == 0) s.work[wave] = work;
    __syncthreads();
    work = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) work += s.work[w];
    const int64_t each = (work + p.target - 1) / p.target;
    most = (int)min(max(each, (int64_t)p.least), (int64_t)0x7fffffff);
  }
  int items = 0, slots = 0;
  for (int b = b0; b < b1; ++b) {
    const PrefillSeq q = prefill_seq<kRows>(p, b);
    const int pieces = q.span > most ? (q.span + most - 1) / most : 1;
    items += q.tiles * pieces;
    slots += pieces > 1 ? q.tiles * pieces : 0;
  }
  int items_in = items, slots_in = slots;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(items_in, d), c = __shfl_up(slots_in, d);
    if (lane >= d) {
      items_in += a;
      slots_in += c;
    }
  }
  if (lane == 63) {
    s.items[wave] = items_in;
    s.slots[wave] = slots_in;
  }
  if (threadIdx.x == 0) s.item.b = -1;
  __syncthreads();
  int items_at = items_in - items, slots_at = slots_in - slots, slots_all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    items_at += w < wave ? s.items[w] : 0;
    slots_at += w < wave ? s.slots[w] : 0;
    slots_all += s.slots[w];
  }
  if (index >= items_at && index < items_at + items) {
    for (int b = b0; b < b1; ++b) {
      const PrefillSeq q = prefill_seq<kRows>(p, b);
      const int pieces = q.span > most ? (q.span + most - 1) / most : 1;
      const int here = q.tiles * pieces;
      if (index < items_at + here) {
        const int local = index - items_at;
        s.item.b = b;
        s.item.tile = q.tiles - 1 - local / pieces;
        s.item.piece = local % pieces;
        s.item.pieces = pieces;
        s.item.slot = slots_at + local;
        break;
      }
      items_at += here;
      slots_at += pieces > 1 ? here : 0;
    }
  }
  if (tell && p.target > 0 && threadIdx.x == 0) *p.ws_total = min(slots_all, p.max_slots);
  __syncthreads();
  return s.item;
}

// One row tile (and piece of its keys) of one kv head.
//
// kUniform (pages of 16 tokens or more): the rows that a wave stages at a time lie in one
// page, so page ids and row addresses are scalars, and a 16-bit cache's rows go to LDS
// without passing through registers (a lane loads the chunk that belongs where its 16
// bytes land). Page ids are read a tile ahead of the loads, those a tile ahead of the math.
template <int HD, typename T, int kCache, bool kExtras, bool kUniform>
__global__ __launch_bounds__(kPrefillWaves<HD> * 64) void paged_prefill_kernel(PrefillParams p) {
  constexpr int kThreads = kPrefillWaves<HD> * 64;
  constexpr int kRows = kPrefillRows<HD>;
  constexpr int KT = kPrefillKeys;
  constexpr int kRowBytes = HD * 2;              // of a row in LDS
  constexpr bool kWide = kCache == kCache16;
  constexpr int kLoadBytes = kWide ? HD * 2 : HD;  // of a row in the cache
  constexpr int kLoads = kLoadBytes / 16;          // its 16-byte loads
  constexpr int kPass = kThreads / kLoads;         // rows that one load of every thread covers
  constexpr int kPer = kPass >= KT ? 1 : KT / kPass;
  constexpr int NQ = HD / 16;                      // product steps over the head dim
  constexpr int ND = HD / 32;                      // 32-dim blocks of the output
  // An fp16 call on an 8-bit cache holds V as bf16 and P as the sum of two bf16 (16 bits
  // of precision): vs times a weight may lie below fp16's range.
  constexpr bool kSplitP = !kWide && std::is_same_v<T, F16>;
  using TV = std::conditional_t<kSplitP, BF16, T>;

  __shared__ __align__(16) char lds_k[2][KT * kRowBytes];
  __shared__ __align__(16) char lds_v[2][KT * kRowBytes];
  __shared__ __align__(16) float lds_ks[kWide ? 1 : 2][KT], lds_vs[kWide ? 1 : 2][KT];
  __shared__ PrefillScan<kThreads> scan;

  const int kvh = blockIdx.x % p.hkv;
  const PrefillItem it =
      prefill_find<kRows, kThreads>(p, blockIdx.x / p.hkv, scan, blockIdx.x == 0);
  if (it.b < 0) return;
  if (it.pieces > 1 && it.slot >= p.max_slots) return;
  const PrefillSeq sq = prefill_seq<kRows>(p, it.b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, half = lane >> 5;
  const int gq = p.gq;
  const int rows = sq.n * gq;  // of the sequence, per kv head
  const int first_pos = sq.len - sq.n;

  // Keys of the tile, then of the piece, in tiles of KT.
  const int t_first = it.tile * kRows / gq;
  const int t_last = min(sq.n - 1, (it.tile * kRows + kRows - 1) / gq);
  const int k_end = max(0, p.causal ? min(sq.len, first_pos + t_last + 1) : sq.len);
  const int k_begin =
      p.window_left >= 0 ? max(0, first_pos + t_first - p.window_left) / KT * KT : 0;
  const int all = k_end > k_begin ? (k_end - k_begin + KT - 1) / KT : 0;
  const int j0 = (int)((int64_t)all * it.piece / it.pieces);
  const int j1 = (int)((int64_t)all * (it.piece + 1) / it.pieces);

  // This lane's row, and the wave's rows.
  const int row_w = it.tile * kRows + wave * 32;
  const int row = row_w + col;
  const bool live = row < rows;
  const int tok = min(row, rows - 1) / gq, head = min(row, rows - 1) % gq;
  const int pos = first_pos + tok;
  const bool wave_live = row_w < rows;
  const int pos_lo = first_pos + row_w / gq;
  const int pos_hi = first_pos + min(row_w + 31, rows - 1) / gq;
  const int lim = p.causal ? min(pos, sq.len - 1) : sq.len - 1;  // last key the row sees
  const int from = p.window_left >= 0 ? pos - p.window_left : 0;  // and the first

  uint4 qf[NQ];
  {
    const char *src = p.q + (int64_t)(sq.start + tok) * p.q_st +
                      (int64_t)(kvh * gq + head) * p.q_sh + half * 16;
#pragma unroll
    for (int i = 0; i < NQ; ++i)
      qf[i] = live ? *reinterpret_cast<const uint4 *>(src + i * 32) : make_uint4(0u, 0u, 0u, 0u);
  }
  // Scores are kept as products; c takes them to base 2 in one multiply-add with the
  // reference. c > 0: a negative scale's sign goes to q, and a scale of zero zeroes q.
  float c = p.scale * kPrefillLog2e;
  if (!kWide && p.k_scale) c *= p.k_scale[0];
  {
    const uint32_t keep = c == 0.f ? 0u : 0xffffffffu, flip = c < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < NQ; ++i)
      qf[i] = make_uint4((qf[i].x ^ flip) & keep, (qf[i].y ^ flip) & keep,
                         (qf[i].z ^ flip) & keep, (qf[i].w ^ flip) & keep);
    c = c == 0.f ? 1.f : fabsf(c);
  }
  const float cs = kExtras ? 1.f : c;  // what is left to multiply scores by at the exponent
  const float v_scale = !kWide && p.v_scale ? p.v_scale[0] : 1.f;
  const bool capped = kExtras && p.softcap > 0.f;
  const float slope = kExtras && p.alibi ? p.alibi[kvh * gq + head] * kPrefillLog2e : 0.f;

  // Staging: thread (row, chunk) of each pass; a wave's rows follow each other.
  constexpr int kWaveRows = 64 / kLoads;
  constexpr bool kDirect = kWide && kUniform;
  const int s_row = threadIdx.x / kLoads, s_chunk = threadIdx.x % kLoads;
  const int w_row = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kWaveRows;
  const int ps_mask = (1 << p.ps_log2) - 1;
  const int last_page = (p.max_len - 1) >> p.ps_log2;
  const int32_t *bt = p.bt + (int64_t)it.b * p.bt_stride;
  const int64_t head_off = (int64_t)kvh * p.sh;
  // Byte offsets of this lane from its wave's first row (kUniform). A pass of eight rows
  // (head dim 256) swaps K's chunk halves every other time.
  static_assert(!kDirect || kPass % 16 == 0 || (HD == 256 && kPass % 8 == 0), "swizzle_k");
  const uint32_t lane_row = (uint32_t)(s_row & (kWaveRows - 1)) * (uint32_t)p.st;
  const uint32_t k_off = lane_row + (kDirect ? (s_chunk ^ swizzle_k<HD>(s_row)) : s_chunk) * 16;
  const uint32_t k_off_odd =
      kPass % 16 == 0 ? k_off : lane_row + (s_chunk ^ swizzle_k<HD>(s_row + kPass)) * 16;
  const uint32_t v_off = lane_row + (kDirect ? (s_chunk ^ swizzle_v<HD>(s_row)) : s_chunk) * 16;
  uint4 rk[kDirect ? 1 : kPer], rv[kDirect ? 1 : kPer];
  float rks = 0.f, rvs = 0.f;  // 8-bit: the scales of the tile's key threadIdx.x
  int pg[kPer], pg_scale = 0;  // page ids of the tile to load next

  // Page ids as the table has them, of keys that may lie past the sequence: the index is
  // held to the table's row here, the id to the cache where it is used.
  auto find_pages = [&](int j) {
    const int key0 = k_begin + j * KT;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int r = u * kPass + (kUniform ? w_row : s_row);
      const int at = min((key0 + min(r, KT - 1)) >> p.ps_log2, last_page);
      if constexpr (kUniform)
        pg[u] = ((const __attribute__((address_space(4))) int32_t *)bt)[at];
      else
        pg[u] = bt[at];
    }
    if constexpr (!kWide) {
      if (threadIdx.x < KT) pg_scale = bt[min((key0 + (int)threadIdx.x) >> p.ps_log2, last_page)];
    }
  };
  auto page_off = [&](int page) -> int64_t {
    return (int64_t)min(max(page, 0), p.num_pages - 1) * p.sp;
  };
  auto load_tile = [&](int j, int buf) {
    const int key0 = k_begin + j * KT;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if constexpr (kUniform) {
        if (kPass * kPer > KT && u * kPass + w_row >= KT) break;
        const int64_t off = page_off(pg[u]) +
                            (int64_t)((key0 + u * kPass + w_row) & ps_mask) * p.st + head_off;
        if constexpr (kDirect) {
          const uint32_t at = (u * kPass + w_row) * kRowBytes;
          load_to_lds(p.k + off, u & 1 ? k_off_odd : k_off, lds_offset(lds_k[buf]) + at);
          load_to_lds(p.v + off, v_off, lds_offset(lds_v[buf]) + at);
        } else {
          rk[u] = *reinterpret_cast<const uint4 *>(p.k + off + k_off);
          rv[u] = *reinterpret_cast<const uint4 *>(p.v + off + v_off);
        }
      } else {
        const int r = min(s_row + u * kPass, KT - 1);
        const int64_t off = page_off(pg[u]) + (int64_t)((key0 + r) & ps_mask) * p.st + head_off +
                            s_chunk * 16;
        rk[u] = *reinterpret_cast<const uint4 *>(p.k + off);
        rv[u] = *reinterpret_cast<const uint4 *>(p.v + off);
      }
    }
    if constexpr (!kWide) {
      if (threadIdx.x < KT) {
        const int key = key0 + threadIdx.x;
        const int64_t page = min(max(pg_scale, 0), p.num_pages - 1);
        rks = p.ks ? p.ks[page * p.ks_sp + (int64_t)kvh * p.ks_sh + (key & ps_mask)] : 1.f;
        rvs = p.vs ? p.vs[page * p.vs_sp + (int64_t)kvh * p.vs_sh + (key & ps_mask)] : 1.f;
      }
    }
  };
  // The tile into LDS (kDirect: it is on its way there; this thread's loads are waited for).
  // V rows at or past the sequence's end become zeros, whatever their memory holds; their
  // keys are masked.
  auto store_tile = [&](int j, int buf) {
    const int valid = sq.len - (k_begin + j * KT);  // rows of the tile that exist
    if constexpr (kDirect) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (valid < KT) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          const int r = s_row + u * kPass;
          if (r >= valid && r < KT)
            *reinterpret_cast<uint4 *>(lds_v[buf] + r * kRowBytes + s_chunk * 16) =
                make_uint4(0u, 0u, 0u, 0u);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int r = s_row + u * kPass;
        const uint4 wk = rk[u];
        const bool there = r < valid;
        const uint4 wv = make_uint4(there ? rv[u].x : 0u, there ? rv[u].y : 0u,
                                    there ? rv[u].z : 0u, there ? rv[u].w : 0u);
        const int sk = swizzle_k<HD>(r), sv = swizzle_v<HD>(r);
        if (r < KT) {
          char *dk = lds_k[buf] + r * kRowBytes, *dv = lds_v[buf] + r * kRowBytes;
          if constexpr (kWide) {
            *reinterpret_cast<uint4 *>(dk + (s_chunk ^ sk) * 16) = wk;
            *reinterpret_cast<uint4 *>(dv + (s_chunk ^ sv) * 16) = wv;
          } else {
            const uint2 k0 = widen_codes<T, kCache>(wk.x), k1 = widen_codes<T, kCache>(wk.y);
            const uint2 k2 = widen_codes<T, kCache>(wk.z), k3 = widen_codes<T, kCache>(wk.w);
            const uint2 v0 = widen_codes<TV, kCache>(wv.x), v1 = widen_codes<TV, kCache>(wv.y);
            const uint2 v2 = widen_codes<TV, kCache>(wv.z), v3 = widen_codes<TV, kCache>(wv.w);
            *reinterpret_cast<uint4 *>(dk + ((2 * s_chunk) ^ sk) * 16) =
                make_uint4(k0.x, k0.y, k1.x, k1.y);
            *reinterpret_cast<uint4 *>(dk + ((2 * s_chunk + 1) ^ sk) * 16) =
                make_uint4(k2.x, k2.y, k3.x, k3.y);
            *reinterpret_cast<uint4 *>(dv + ((2 * s_chunk) ^ sv) * 16) =
                make_uint4(v0.x, v0.y, v1.x, v1.y);
            *reinterpret_cast<uint4 *>(dv + ((2 * s_chunk + 1) ^ sv) * 16) =
                make_uint4(v2.x, v2.y, v3.x, v3.y);
          }
        }
      }
      if constexpr (!kWide) {
        if (threadIdx.x < KT) {
          // A V row without a scale (NaN: it held an infinity or a NaN) takes its key's score
          // along instead, so that it reaches the rows that see the key and no other (a
          // weight of zero times NaN would).
          const bool whole = fabsf(rvs) < INFINITY;
          lds_ks[buf][threadIdx.x] = whole ? rks : __builtin_nanf("");
          lds_vs[buf][threadIdx.x] = whole && (int)threadIdx.x < valid ? rvs : 0.f;
        }
      }
    }
  };

  float m = -INFINITY, l = 0.f;
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  auto compute = [&](int buf, int key0) {
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
      const int r = kb * 32 + col;
      const char *base = lds_k[buf] + r * kRowBytes;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const uint4 a = *reinterpret_cast<const uint4 *>(
            base + (((2 * i + half) ^ swizzle_k<HD>(r)) * 16));
        s[kb] = Prod32<T>::run(a, qf[i], s[kb]);
      }
    }
    // Scores: keys kb * 32 + 8 (i / 4) + 4 half + i % 4 of the tile.
    if constexpr (!kWide) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 f =
              *reinterpret_cast<const float4 *>(&lds_ks[buf][kb * 32 + 8 * g + 4 * half]);
          s[kb][4 * g] *= f.x;
          s[kb][4 * g + 1] *= f.y;
          s[kb][4 * g + 2] *= f.z;
          s[kb][4 * g + 3] *= f.w;
        }
    }
    if constexpr (kExtras) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x = s[kb][i] * c;
          if (capped) {
            // cap * tanh(x / cap) = cap * (1 - 2 / (e^(2 x / cap) + 1)), in base 2
            const float e = fast_exp2(x * (2.f / p.softcap));
            x = p.softcap * kPrefillLog2e * (1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f));
          }
          const int key = key0 + kb * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
          x -= slope * (float)abs(pos - key);
          s[kb][i] = x;
        }
    }
    // Tiles with keys that some row of the wave does not see.
    const bool full = key0 + KT - 1 <= (p.causal ? min(pos_lo, sq.len - 1) : sq.len - 1) &&
                      (p.window_left < 0 || key0 >= pos_hi - p.window_left);
    if (!full) {
      const int hi = lim - key0 - 4 * half, lo = from - key0 - 4 * half;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = kb * 32 + 8 * (i >> 2) + (i & 3);
          s[kb][i] = (k <= hi && k >= lo) ? s[kb][i] : -INFINITY;
        }
    }
    float mt = s[0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[0][i]);
#pragma unroll
    for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[1][i]);
    mt *= cs;
    if (__builtin_amdgcn_ballot_w64(mt > m + kPrefillRescaleLog2) != 0) {  // wave-uniform
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt),
                                                       false, false);
      const float mm = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      const float mn = mm > m + kPrefillRescaleLog2 ? mm : m;
      const float f = mn == m ? 1.f : fast_exp2(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
      m = mn;
    }
    const float mr = m == -INFINITY ? 0.f : m;  // no key seen yet: the scores here are -inf too
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[kb][i] = fast_exp2(__builtin_fmaf(s[kb][i], cs, -mr));
        if constexpr (!kWide) l += s[kb][i];
      }
    if constexpr (!kWide) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 f =
              *reinterpret_cast<const float4 *>(&lds_vs[buf][kb * 32 + 8 * g + 4 * half]);
          s[kb][4 * g] *= f.x;
          s[kb][4 * g + 1] *= f.y;
          s[kb][4 * g + 2] *= f.z;
          s[kb][4 * g + 3] *= f.w;
        }
    }
    // P rounded once (the 16-bit products take no more), eight keys per operand register set.
    uint4 pf[4], pl[kSplitP ? 4 : 1];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      uint32_t w[4], x[4];
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const float a = s[st >> 1][8 * (st & 1) + 2 * jj], b = s[st >> 1][8 * (st & 1) + 2 * jj + 1];
        w[jj] = Prod32<TV>::pack(a, b);
        if constexpr (kSplitP)
          x[jj] = Prod32<TV>::pack(a - Elem<BF16>::lo(w[jj]), b - Elem<BF16>::hi(w[jj]));
        // The sum of the rounded weights: the output is then a mean of V rows, and a pair
        // takes one instruction. (8-bit rows: the weights carry vs; summed above.)
        if constexpr (kWide) l = Prod32<T>::add_pair(w[jj], l);
      }
      pf[st] = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (kSplitP) pl[st] = make_uint4(x[0], x[1], x[2], x[3]);
    }
    // V^T operand: lane l reads dims 16 ((l / 16) % 2) + 4 (l % 4) .. of key
    // 4 (l / 32) + (l / 4) % 4 and receives dim l % 32 of four keys.
    const int v_key = 4 * half + ((lane >> 2) & 3);
    const int v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);  // within the 32-dim block
#pragma unroll
    for (int st = 0; st < 4; ++st) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = st * 16 + 8 * u + v_key;
          const int byte = (d * 32 + v_dim) * 2;
          const int at =
              r * kRowBytes + (((byte >> 4) ^ swizzle_v<HD>(r)) << 4) + (byte & 15);
          typedef __attribute__((address_space(3))) s16x4v LdsVec;
          const s16x4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec *)(lds_v[buf] + at));
          const uint2 y = __builtin_bit_cast(uint2, x);
          w[2 * u] = y.x;
          w[2 * u + 1] = y.y;
        }
        const uint4 a = make_uint4(w[0], w[1], w[2], w[3]);
        o[d] = Prod32<TV>::run(a, pf[st], o[d]);
        if constexpr (kSplitP) o[d] = Prod32<TV>::run(a, pl[st], o[d]);
      }
    }
  };

  if (j0 < j1) {
    find_pages(j0);
    load_tile(j0, 0);
    find_pages(j0 + 1);
  }
  for (int j = j0; j < j1; ++j) {
    const int buf = (j - j0) & 1;
    // One barrier a tile: past it the tile's rows are there, and every wave is done with
    // the other buffer, which the next tile's loads then fill.
    store_tile(j, buf);
    if (!kDirect && j + 1 < j1) {
      load_tile(j + 1, buf ^ 1);
      find_pages(j + 2);
    }
    __syncthreads();
    if (kDirect && j + 1 < j1) {
      load_tile(j + 1, buf ^ 1);
      find_pages(j + 2);
    }
    const int key0 = k_begin + j * KT;
    const bool seen = wave_live && key0 <= (p.causal ? pos_hi : sq.len - 1) &&
                      (p.window_left < 0 || key0 + KT - 1 >= pos_lo - p.window_left);
    if (seen) compute(buf, key0);
  }

  const auto lw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false,
                                                   false);
  l = __uint_as_float(lw[0]) + __uint_as_float(lw[1]);
  if (it.pieces > 1) {
    const int64_t at = (int64_t)it.slot * p.hkv + kvh;
    if (threadIdx.x == 0)
      p.ws_desc[at] = make_int4(it.piece == 0 ? it.pieces : 0, it.b, it.tile, 0);
    const int r = wave * 32 + col;
    if (half == 0) p.ws_lse[at * kRows + r] = l > 0.f ? m + __log2f(l) : (l == 0.f ? -INFINITY : l);
    const float inv = l == 0.f ? 0.f : v_scale / l;
    float *dst = p.ws_o + (at * kRows + r) * HD + 4 * half;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4 *>(dst + d * 32 + 8 * g) =
            make_float4(o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv,
                        o[d][4 * g + 3] * inv);
    return;
  }
  if (!live) return;
  // No key seen: zeros (l = 0; a sink alone leaves zeros too).
  float den = l;
  if (p.sinks) den += fast_exp2(p.sinks[kvh * gq + head] * kPrefillLog2e - m);
  const float inv = l == 0.f ? 0.f : v_scale / den;
  char *dst = p.out + (int64_t)(sq.start + tok) * p.o_st + (int64_t)(kvh * gq + head) * p.o_sh +
              8 * half;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2 *>(dst + d * 64 + 16 * g) =
          make_uint2(Prod32<T>::pack(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                     Prod32<T>::pack(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
}

// Joins the pieces of one row tile: workgroup (slot, kv head; part) where the slot holds a
// tile's first piece, a thread for four dims of every kParts * kJoinRows-th row.
constexpr int kPrefillJoinThreads = 256;
constexpr int kPrefillJoinParts = 4;

template <int HD, typename T>
__global__ __launch_bounds__(kPrefillJoinThreads) void paged_prefill_join_kernel(PrefillParams p) {
  constexpr int kRows = kPrefillRows<HD>;
  constexpr int kJoinRows = kPrefillJoinThreads / (HD / 4);
  const int at = blockIdx.x;  // slot * hkv + kv head
  const int slot = at / p.hkv, kvh = at - slot * p.hkv;
  if (slot >= *p.ws_total) return;
  const int4 d = p.ws_desc[at];
  const int pieces = d.x;
  if (pieces <= 1 || slot + pieces > p.max_slots || d.y < 0 || d.y >= p.batch) return;
  const PrefillSeq sq = prefill_seq<kRows>(p, d.y);
  const int chunk = threadIdx.x % (HD / 4);
  const int rows = min(kRows, sq.n * p.gq - d.z * kRows);
  for (int r = blockIdx.y * kJoinRows + threadIdx.x / (HD / 4); r < rows;
       r += kPrefillJoinParts * kJoinRows) {
    const int row = d.z * kRows + r;
    const int tok = row / p.gq, head = kvh * p.gq + row % p.gq;
    float m = -INFINITY;
    for (int i = 0; i < pieces; ++i)
      m = fmaxf(m, p.ws_lse[(at + (int64_t)i * p.hkv) * kRows + r]);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < pieces; ++i) {
      const int64_t a = (at + (int64_t)i * p.hkv) * kRows + r;
      const float lse = p.ws_lse[a];
      const float w = lse == -INFINITY ? 0.f : fast_exp2(lse - m);
      const float4 x = *reinterpret_cast<const float4 *>(p.ws_o + a * HD + 4 * chunk);
      sum += w;
      acc.x += w * x.x;
      acc.y += w * x.y;
      acc.z += w * x.z;
      acc.w += w * x.w;
    }
    float den = sum;
    if (p.sinks) den += fast_exp2(p.sinks[head] * kPrefillLog2e - m);
    const float inv = sum == 0.f ? 0.f : 1.f / den;
    *reinterpret_cast<uint2 *>(p.out + (int64_t)(sq.start + tok) * p.o_st +
                               (int64_t)head * p.o_sh + 8 * chunk) =
        make_uint2(Prod32<T>::pack(acc.x * inv, acc.y * inv),
                   Prod32<T>::pack(acc.z * inv, acc.w * inv));
  }
}

// Launches of one head dim (prefill_hd*.hip).
template <int HD, typename T, int kCache>
int launch_prefill_t(const PrefillParams &p, int items, hipStream_t st) {
  const dim3 grid((unsigned)(items * p.hkv)), block(kPrefillWaves<HD> * 64);
  const bool extras = p.softcap > 0.f || p.alibi;
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, p); };
  if (p.uniform)
    extras ? go(paged_prefill_kernel<HD, T, kCache, true, true>)
           : go(paged_prefill_kernel<HD, T, kCache, false, true>);
  else
    extras ? go(paged_prefill_kernel<HD, T, kCache, true, false>)
           : go(paged_prefill_kernel<HD, T, kCache, false, false>);
  if (hipGetLastError() != hipSuccess) return MXFA_ELAUNCH;
  if (p.target == 0) return MXFA_OK;
  hipLaunchKernelGGL((paged_prefill_join_kernel<HD, T>),
                     dim3((unsigned)(p.max_slots * p.hkv), kPrefillJoinParts),
                     dim3(kPrefillJoinThreads), 0, st, p);
  return hipGetLastError() == hipSuccess ? MXFA_OK : MXFA_ELAUNCH;
}

template <int HD>
int launch_prefill_hd(const PrefillParams &p, int items, bool bf16, int cache, hipStream_t st) {
  if (bf16) {
    if (cache == kCache16) return launch_prefill_t<HD, BF16, kCache16>(p, items, st);
    if (cache == kCacheE4m3) return launch_prefill_t<HD, BF16, kCacheE4m3>(p, items, st);
    return launch_prefill_t<HD, BF16, kCacheInt8>(p, items, st);
  }
  if (cache == kCache16) return launch_prefill_t<HD, F16, kCache16>(p, items, st);
  if (cache == kCacheE4m3) return launch_prefill_t<HD, F16, kCacheE4m3>(p, items, st);
  return launch_prefill_t<HD, F16, kCacheInt8>(p, items, st);
}

}  // namespace mxfa

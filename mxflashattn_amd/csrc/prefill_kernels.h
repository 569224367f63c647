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
// Tiles of 64 keys go through LDS, two buffers each of K and V, K 32 keys ahead of V: the
// scores of the next 32 keys are computed among the exponentials of these. LDS rows hold HD
// elements, their 16-byte chunks permuted (swizzle_k, swizzle_v) so that neither operand read
// meets a bank conflict. A 16-bit cache's rows go straight to LDS (pages of 16 tokens or more);
// an 8-bit cache is widened exactly on its way there, once for the whole workgroup, and its
// scales join the scores (ks) and the weights (vs, ahead of P's one rounding) in 32 bits.
//
// Bound (MI355X): a chunk of 4096 tokens on 32k keys, 32q/8kv HD 128 bf16, takes 1.88 ms, 1.10
// PFLOP/s where a large library product reaches 1.20; the matrix unit is busy 57 % of the
// cycles, and without the loads of keys the loop would take 20 % less. Two chunks of a layer
// over int8 rows run at 0.65 PFLOP/s: a wave issues some 330 vector instructions for 64 keys
// against 115 (widening, two scales a key).
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
#include <utility>

#include "mxfa_device.h"
#include "mxfa_mi355x.h"

// A kernel's parts are lambdas; none may become a call.
#define MXFA_INLINE __attribute__((always_inline))

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
  uint32_t hkv_mul, gq_mul;  // div_by
  int span;                  // keys that one row tile spans, at most
  int target;          // pieces per kv head that the keys are cut into (0: none)
  int least;           // fewest keys of a piece
  float *ws_o, *ws_lse;  // pieces: [slot][kv head][kRows][HD], [slot][kv head][kRows]
  int4 *ws_desc;         // [slot][kv head]: pieces (0 but for a tile's first), batch, tile
  int *ws_total;         // slots in use
  int max_slots;
  int uniform;  // pages of 16 tokens or more, strides that 32-bit offsets reach over
};

// Waves of a workgroup, 32 rows each. Two workgroups of four share a CU where one of eight
// would fit: they are not in step, so one's exponentials meet the other's products, and the
// last workgroups of a call leave less of the chip idle (six prompts of 300-1500 tokens,
// 32q/8kv HD 128: 90.8 us against 112.6; a long chunk, before rows went straight to LDS,
// 2661 against 2369).
constexpr int kPrefillWaves = 4;
constexpr int kPrefillRows = 32 * kPrefillWaves;
// Workgroups per CU, as far as the registers of their waves (one per SIMD each) reach: the
// accumulators are HD / 2 registers, q HD / 4.
template <int HD, typename T, int kCache, bool kExtras, bool kUniform>
constexpr int kPrefillOccupancy =
    HD == 256 || (HD == 128 && kExtras && (kCache != kCache16 || !kUniform)) ? 1
    : HD == 64 && kCache == kCache16 && !kExtras                             ? 3
                                                                             : 2;

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

// A pointer that is the same in every lane, as a scalar.
__device__ __forceinline__ const char *uniform_pointer(const char *ptr) {
  const uint64_t x = (uint64_t)ptr;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (const char *)(((uint64_t)hi << 32) | lo);
}

// 16 bytes a lane from base + off (base the same in the whole wave) to LDS at `lds` + 16 *
// lane, with no register in between. The compiler does not see the load: the caller waits
// for it (vmcnt) ahead of the barrier that hands the data over. (The builtin for it makes
// the compiler wait at the next LDS read, of the other buffer. It keeps nothing in m0.)
__device__ __forceinline__ void load_to_lds(const char *base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory");
}

// The same where `on` is ~0; no load where it is 0. (A branch amid the products makes the
// compiler copy their accumulators.)
__device__ __forceinline__ void load_to_lds_if(const char *base, uint32_t off, uint32_t lds,
                                               uint64_t on) {
  uint64_t all;
  asm volatile("s_mov_b32 m0, %1\n\ts_and_saveexec_b64 %0, %4\n\t"
               "global_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, %0"
               : "=&s"(all)
               : "s"(lds), "v"(off), "s"(base), "s"(on)
               : "memory", "scc");
}

// f(std::integral_constant<int, I>) for I = 0 .. N-1, unrolled at compile time.
template <typename F, int... I>
__device__ __forceinline__ void static_unroll_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_unroll(F &&f) {
  static_unroll_impl(f, std::make_integer_sequence<int, N>{});
}

// x / d for 0 <= x < 2^31 and 1 <= d < 2^16 by m = ceil(2^32 / d) (0 for d = 1): x m / 2^32
// passes x / d by less than a half, so the quotient is one too many at most.
__device__ __forceinline__ int div_by(int x, int d, uint32_t m) {
  const uint32_t q = m ? __umulhi((uint32_t)x, m) : (uint32_t)x;
  return (int)(q - (q * (uint32_t)d > (uint32_t)x ? 1u : 0u));
}

// A wave's fold of values with identity 0, in every lane.
template <typename T, typename F>
__device__ __forceinline__ T wave_fold(T x, F f) {
  const auto with = [&](int y) { x = f(x, __builtin_bit_cast(T, y)); };
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kDppRowShr0 + 1, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kDppRowShr0 + 2, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kDppRowShr0 + 4, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kDppRowShr0 + 8, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kDppRowBcast15, 0xa, 0xf, false));
  with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kDppRowBcast31, 0xc, 0xf, false));
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ float wave_sum(float x) {
  return wave_fold(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ int wave_sum(int x) {
  return wave_fold(x, [](int a, int b) { return a + b; });
}

// What one sequence asks for: its query rows and keys, held to those that exist.
struct PrefillSeq {
  int start, n, len;
};

__device__ __forceinline__ PrefillSeq prefill_seq(const PrefillParams &p, int b) {
  PrefillSeq s;
  s.start = min(max(p.cu[b], 0), p.rows_q);
  const int end = min(max(p.cu[b + 1], s.start), p.rows_q);
  s.n = end - s.start;
  s.len = min(max(p.seqlens[b], 0), p.max_len);
  return s;
}
__device__ __forceinline__ int prefill_tiles(const PrefillParams &p, const PrefillSeq &q) {
  return (int)((uint32_t)(q.n * p.gq + kPrefillRows - 1) / kPrefillRows);  // (a call's rows: int)
}
// At most 32 rows in a call whose tiles may be cut: all waves on one row tile.
__device__ __forceinline__ bool prefill_few(const PrefillParams &p, const PrefillSeq &q) {
  return p.target > 0 && q.n * p.gq <= 32;
}
// What a row tile costs, in keys: four waves on their own keys take half of a tile's time.
__device__ __forceinline__ int prefill_cost(const PrefillParams &p, const PrefillSeq &q) {
  const int span = min(q.len, p.span);
  return prefill_few(p, q) ? (span + 1) / 2 : span;
}
__device__ __forceinline__ int prefill_pieces(int cost, int most) {
  return cost > most ? (cost + most - 1) / most : 1;
}
// Keys (at their cost) of a piece: W / target, a little more so that 32-bit sums of W keep
// the pieces of cut tiles within 2 * target.
__device__ __forceinline__ int prefill_most(const PrefillParams &p, float work) {
  if (p.target <= 0) return 0x7fffffff;
  return max(p.least, (int)fminf(work * 1.001f / (float)p.target + 1.f, 2e9f));
}

struct PrefillItem {
  int b, tile, piece, pieces, slot;
  PrefillSeq seq;
};

struct PrefillScan {
  float work[kPrefillWaves];
  int items[kPrefillWaves], slots[kPrefillWaves];
  int b, tile, piece, pieces, slot;
};

// The row tile and piece of item `index`; b = -1 past the last.
//
// Up to 64 sequences (one a lane, every wave for itself): the last tile of every sequence,
// then the last but one of every sequence that has it, and so on. With the causal mask a
// sequence's later tiles see more keys, so the longest work goes out first and the end of
// the call is made of short pieces.
// More: sequence by sequence, in falling order too, through a scan in LDS.
__device__ __forceinline__ PrefillItem prefill_find(const PrefillParams &p, int index,
                                                    PrefillScan &s, bool tell) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (p.batch <= 64) {
    const PrefillSeq q = prefill_seq(p, min(lane, p.batch - 1));
    const int tiles = lane < p.batch ? prefill_tiles(p, q) : 0;
    int pieces = 1;
    if (p.target > 0) {
      const int cost = prefill_cost(p, q);
      const int most = prefill_most(p, wave_sum((float)tiles * (float)cost));
      if (__builtin_amdgcn_ballot_w64(cost > most) != 0) pieces = prefill_pieces(cost, most);
    }
    const int cut = pieces > 1 ? tiles * pieces : 0;
    const int slots = wave_scan_incl(cut);
    if (tell && p.target > 0 && threadIdx.x == 0)
      *p.ws_total = min(__builtin_amdgcn_readlane(slots, 63), p.max_slots);
    if (index >= wave_sum(tiles * pieces)) return {-1, 0, 0, 1, 0, {0, 0, 0}};
    // The round: the largest d whose items of earlier rounds are at most `index`, 64
    // candidates at a time.
    int lo = 0, before = 0;
    int hi = wave_fold(tiles, [](int a, int b) { return max(a, b); });
    while (hi - lo > 1) {  // items before round lo <= index < items before round hi
      const int step = (hi - lo + 63) >> 6, d = lo + lane * step;
      int items = 0;
#pragma unroll 4
      for (int b = 0; b < p.batch; ++b)
        items += __builtin_amdgcn_readlane(pieces, b) * min(__builtin_amdgcn_readlane(tiles, b), d);
      const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(items <= index)) - 1;
      before = __builtin_amdgcn_readlane(items, at);
      lo += at * step;
      hi = min(hi, lo + step);
    }
    const int here = tiles > lo ? pieces : 0;
    const int upto = wave_scan_incl(here);
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > index - before);
    const int b = past ? __builtin_ctzll(past) : 0;
    const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, b); };
    const int piece = index - before - (of(upto) - of(here));
    return {b, of(tiles) - 1 - lo, piece, of(pieces),
            of(slots) - of(cut) + lo * of(pieces) + piece, {of(q.start), of(q.n), of(q.len)}};
  }
  const int per = (p.batch + kPrefillWaves * 64 - 1) / (kPrefillWaves * 64);
  const int b0 = threadIdx.x * per, b1 = min(b0 + per, p.batch);
  int most = 0x7fffffff;
  if (p.target > 0) {
    float work = 0.f;
    for (int b = b0; b < b1; ++b) {
      const PrefillSeq q = prefill_seq(p, b);
      work += (float)prefill_tiles(p, q) * (float)prefill_cost(p, q);
    }
    work = wave_sum(work);
    if (lane == 0) s.work[wave] = work;
    __syncthreads();
    work = 0.f;
#pragma unroll
    for (int w = 0; w < kPrefillWaves; ++w) work += s.work[w];
    most = prefill_most(p, work);
  }
  int items = 0, slots = 0;
  for (int b = b0; b < b1; ++b) {
    const PrefillSeq q = prefill_seq(p, b);
    const int pieces = prefill_pieces(prefill_cost(p, q), most);
    const int here = prefill_tiles(p, q) * pieces;
    items += here;
    slots += pieces > 1 ? here : 0;
  }
  const int items_in = wave_scan_incl(items), slots_in = wave_scan_incl(slots);
  if (lane == 63) {
    s.items[wave] = items_in;
    s.slots[wave] = slots_in;
  }
  if (threadIdx.x == 0) s.b = -1;
  __syncthreads();
  int items_at = items_in - items, slots_at = slots_in - slots, slots_all = 0;
#pragma unroll
  for (int w = 0; w < kPrefillWaves; ++w) {
    items_at += w < wave ? s.items[w] : 0;
    slots_at += w < wave ? s.slots[w] : 0;
    slots_all += s.slots[w];
  }
  if (index >= items_at && index < items_at + items) {
    for (int b = b0; b < b1; ++b) {
      const PrefillSeq q = prefill_seq(p, b);
      const int pieces = prefill_pieces(prefill_cost(p, q), most);
      const int tiles = prefill_tiles(p, q), here = tiles * pieces;
      if (index < items_at + here) {
        const int local = index - items_at;
        s.b = b;
        s.tile = tiles - 1 - local / pieces;
        s.piece = local % pieces;
        s.pieces = pieces;
        s.slot = slots_at + local;
        break;
      }
      items_at += here;
      slots_at += pieces > 1 ? here : 0;
    }
  }
  if (tell && p.target > 0 && threadIdx.x == 0) *p.ws_total = min(slots_all, p.max_slots);
  __syncthreads();
  // The same in every lane: scalars, and so is what follows from them.
  const auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int b = uniform(s.b);
  const PrefillSeq q = prefill_seq(p, max(b, 0));
  return {b, uniform(s.tile), uniform(s.piece), uniform(s.pieces), uniform(s.slot),
          {uniform(q.start), uniform(q.n), uniform(q.len)}};
}

// One row tile (and piece of its keys) of one kv head.
//
// kUniform (pages of 16 tokens or more): the rows that a wave stages at a time lie in one
// page, so page ids and row addresses are scalars, and a 16-bit cache's rows go to LDS
// without passing through registers (a lane loads the chunk that belongs where its 16
// bytes land). Page ids are read a tile ahead of the loads, those a tile ahead of the math.
template <int HD, typename T, int kCache, bool kExtras, bool kUniform>
__global__ __launch_bounds__(kPrefillWaves * 64, (kPrefillOccupancy<HD, T, kCache, kExtras, kUniform>))
void paged_prefill_kernel(PrefillParams p) {
  constexpr int kRows = kPrefillRows;
  constexpr int KT = kPrefillKeys;
  constexpr int kRowBytes = HD * 2;              // of a row in LDS
  constexpr bool kWide = kCache == kCache16;
  constexpr int kLoadBytes = kWide ? HD * 2 : HD;  // of a row in the cache
  constexpr int kLoads = kLoadBytes / 16;          // its 16-byte loads
  constexpr int kWaveRows = 64 / kLoads;           // rows that one load of a wave covers
  constexpr int kWaveKeys = KT / kPrefillWaves;    // rows that a wave stages
  constexpr int kPer = kWaveKeys / kWaveRows;      // loads of them
  constexpr int NQ = HD / 16;                      // product steps over the head dim
  constexpr int ND = HD / 32;                      // 32-dim blocks of the output
  // An fp16 call on an 8-bit cache holds V as bf16 and P as the sum of two bf16 (16 bits
  // of precision): vs times a weight may lie below fp16's range.
  constexpr bool kSplitP = !kWide && std::is_same_v<T, F16>;
  using TV = std::conditional_t<kSplitP, BF16, T>;

  __shared__ __align__(16) char lds_k[2][KT * kRowBytes];
  __shared__ __align__(16) char lds_v[2][KT * kRowBytes];
  __shared__ __align__(16) float lds_ks[kWide ? 1 : 2][KT], lds_vs[kWide ? 1 : 2][KT];
  __shared__ PrefillScan scan;
  __shared__ float few_m[kPrefillWaves][32], few_l[kPrefillWaves][32];

  const int item = div_by(blockIdx.x, p.hkv, p.hkv_mul), kvh = blockIdx.x - item * p.hkv;
  const PrefillItem it = prefill_find(p, item, scan, blockIdx.x == 0);
  if (it.b < 0) return;
  if (it.pieces > 1 && it.slot >= p.max_slots) return;
  const PrefillSeq sq = it.seq;
  const bool few = prefill_few(p, sq);
  // The wave's number and what follows from it are scalars.
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int gq = p.gq;
  const int rows = sq.n * gq;  // of the sequence, per kv head
  const int first_pos = sq.len - sq.n;
  // The tile's first row: token t_first, head r_first; row r of the tile is then
  // token_of(r_first + r) tokens on (numbers below 2^8, divided exactly).
  const int t_first = div_by(it.tile * kRows, gq, p.gq_mul);
  const int r_first = it.tile * kRows - t_first * gq;
  const uint32_t small = (p.gq_mul >> 16) + 1;  // 2^16 / gq, or a little more
  const auto token_of = [&](int r) { return gq == 1 ? r : (int)((uint32_t)r * small >> 16); };

  // Keys that some row of the tile sees, [k_first, k_end), then tiles of KT of them, then the
  // piece's.
  const int t_last = min(sq.n - 1, t_first + token_of(r_first + kRows - 1));
  const int k_end = max(0, p.causal ? min(sq.len, first_pos + t_last + 1) : sq.len);
  const int k_first = p.window_left >= 0 ? max(0, first_pos + t_first - p.window_left) : 0;
  const int k_begin = k_first / KT * KT;
  const int all = k_end > k_begin ? (k_end - k_begin + KT - 1) / KT : 0;
  int j0 = 0, j1 = all;
  if (it.pieces > 1) {
    j0 = (int)((int64_t)all * it.piece / it.pieces);
    j1 = (int)((int64_t)all * (it.piece + 1) / it.pieces);
  }

  // This lane's row, and the wave's rows.
  const int in_tile = few ? 0 : wave * 32;
  const int row_w = it.tile * kRows + in_tile;
  const bool live = row_w + col < rows;
  const int ahead = token_of(r_first + in_tile + col);  // tokens from t_first on
  const int tok = live ? t_first + ahead : sq.n - 1;
  const int head = live ? r_first + in_tile + col - ahead * gq : gq - 1;
  const int pos = first_pos + tok;
  // Keys that all of the wave's rows see, [all_from, all_to], and the last that any does.
  const int pos_lo = first_pos + t_first + token_of(r_first + in_tile);
  const int pos_hi = first_pos + min(t_first + token_of(r_first + in_tile + 31), sq.n - 1);
  const int all_to = p.causal ? min(pos_lo, sq.len - 1) : sq.len - 1;
  const int all_from = p.window_left < 0 ? 0 : pos_hi - p.window_left;
  const int any_to = row_w >= rows ? -1
                                   : min(p.causal ? pos_hi : sq.len - 1, k_begin + j1 * KT - 1);
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
  const uint32_t keep = c == 0.f ? 0u : 0xffffffffu, flip = c < 0.f ? 0x80008000u : 0u;
  c = c == 0.f ? 1.f : fabsf(c);
  const auto sign_q = [&]() MXFA_INLINE {  // (once the first keys' loads are out)
#pragma unroll
    for (int i = 0; i < NQ; ++i)
      qf[i] = make_uint4((qf[i].x ^ flip) & keep, (qf[i].y ^ flip) & keep,
                         (qf[i].z ^ flip) & keep, (qf[i].w ^ flip) & keep);
  };
  const float cs = kExtras ? 1.f : c;  // what is left to multiply scores by at the exponent
  const float v_scale = !kWide && p.v_scale ? p.v_scale[0] : 1.f;
  const bool capped = kExtras && p.softcap > 0.f;
  const float slope = kExtras && p.alibi ? p.alibi[kvh * gq + head] * kPrefillLog2e : 0.f;

  // Staging: a wave brings kWaveKeys = 16 consecutive rows (kUniform: of one page), a lane
  // 16 bytes of every kWaveRows-th of them.
  static_assert(kPer >= 1 && kWaveKeys == 16, "whole loads, rows of one page");
  constexpr bool kDirect = kWide && kUniform;
  const int l_row = lane / kLoads, l_chunk = lane % kLoads;
  const int w_row = wave * kWaveKeys;
  const int ps_mask = (1 << p.ps_log2) - 1;
  const int last_page = (p.max_len - 1) >> p.ps_log2;
  const int32_t *bt = p.bt + (int64_t)it.b * p.bt_stride;
  const int64_t head_off = (int64_t)kvh * p.sh;
  const uint32_t st = (uint32_t)p.st;  // kUniform: below 2^24
  // Byte offset of this lane from the first of the rows that a load covers (kUniform).
  const uint32_t lane_off = (uint32_t)l_row * st;
  uint4 rk[kDirect ? 1 : kPer], rv[kDirect ? 1 : kPer];
  // K's stage j holds the keys that come 32 behind V's tile j: the second half of tile j and
  // the first of tile j + 1.
  constexpr int kAhead = KT / 2;
  float rks = 0.f, rvk = 0.f, rvs = 0.f;  // 8-bit: scales of stage row `lane` (vs at K's key too)
  // Page ids of the rows to load next: one for the wave's rows of K and of V (kUniform: K's in
  // the lower half's lanes of pg_k, V's in the upper's), else one for each of this lane's.
  // They are vector loads, a tile ahead, which the wait for that tile's rows covers: a scalar
  // load in flight makes every wait for an LDS read wait for it too (64 keys of a wave alone
  // on its SIMD: 3460 cycles, 2260 without the loads).
  constexpr int kPages = kUniform ? 1 : kPer;
  int pg_k[kPages], pg_v[kPages], pg_ks = 0, pg_vs = 0;

  // As the table has them, of keys that may lie before or past the sequence: the index is
  // held to the table's row here, the id to the cache where it is used.
  auto page_at = [&](int key) MXFA_INLINE { return min(max(key, 0) >> p.ps_log2, last_page); };
  auto find_pages = [&](int j) MXFA_INLINE {
    const int key0 = k_begin + j * KT;
    if constexpr (kUniform) {
      pg_k[0] = bt[page_at(key0 + w_row + (half ? 0 : kAhead))];
    } else {
#pragma unroll
      for (int u = 0; u < kPages; ++u) {
        const int r = w_row + u * kWaveRows + l_row;
        pg_k[u] = bt[page_at(key0 + kAhead + r)];
        pg_v[u] = bt[page_at(key0 + r)];
      }
    }
    if constexpr (!kWide) {
      if (wave == 0) {
        pg_ks = bt[page_at(key0 + kAhead + lane)];
        pg_vs = bt[page_at(key0 + lane)];
      }
    }
  };
  // Offset in the cache of key's row of this head.
  auto row_off = [&](int key, int page) MXFA_INLINE -> int64_t {
    page = min(max(page, 0), p.num_pages - 1);
    if constexpr (kUniform)  // page and token strides within 32 bits, a page's rows too
      return (int64_t)((uint64_t)(uint32_t)page * (uint32_t)p.sp) +
             (head_off + (uint32_t)(key & ps_mask) * st);
    return (int64_t)page * p.sp + (int64_t)(key & ps_mask) * p.st + head_off;
  };
  auto load_rows = [&](const char *side, int key0, const int (&pg)[kPages], auto is_k, char *lds,
                       uint4 (&reg)[kDirect ? 1 : kPer]) MXFA_INLINE {
    if constexpr (kUniform) {
      const int page = __builtin_amdgcn_readlane(pg[0], decltype(is_k)::value ? 0 : 32);
      const char *src = uniform_pointer(side + row_off(key0 + w_row, page));
      uint32_t at = lds_offset(lds) + w_row * kRowBytes;
      static_unroll<kPer>([&](auto uc) {
        constexpr int u = decltype(uc)::value;
        // The lane whose 16 bytes land at chunk l_chunk of the LDS row loads the chunk that
        // belongs there.
        const int r = u * kWaveRows + l_row;  // of the wave's 16, which start a multiple of 16
        const int from = !kDirect ? l_chunk
                         : decltype(is_k)::value ? l_chunk ^ swizzle_k<HD>(r)
                                                 : l_chunk ^ swizzle_v<HD>(r);
        if constexpr (kDirect)
          load_to_lds(src, lane_off + from * 16, at);
        else
          reg[u] = *reinterpret_cast<const uint4 *>(src + lane_off + from * 16);
        src += kWaveRows * st;
        at += kWaveRows * kRowBytes;
      });
    } else {
#pragma unroll
      for (int u = 0; u < kPer; ++u)
        reg[u] = *reinterpret_cast<const uint4 *>(
            side + row_off(key0 + w_row + u * kWaveRows + l_row, pg[u]) + l_chunk * 16);
    }
  };
  auto load_k_scales = [&](int key0, int id) MXFA_INLINE {
    if constexpr (!kWide) {
      if (wave == 0) {
        const int off = (key0 + lane) & ps_mask;
        const int64_t page = min(max(id, 0), p.num_pages - 1);
        rks = p.ks ? p.ks[page * p.ks_sp + (int64_t)kvh * p.ks_sh + off] : 1.f;
        rvk = p.vs ? p.vs[page * p.vs_sp + (int64_t)kvh * p.vs_sh + off] : 1.f;
      }
    }
  };
  auto load_k = [&](int j, int buf) MXFA_INLINE {
    const int key0 = k_begin + j * KT + kAhead;
    load_rows(p.k, key0, pg_k, std::true_type{}, lds_k[buf], rk);
    load_k_scales(key0, pg_ks);
  };
  auto load_v = [&](int j, int buf) MXFA_INLINE {
    const int key0 = k_begin + j * KT;
    load_rows(p.v, key0, kUniform ? pg_k : pg_v, std::false_type{}, lds_v[buf], rv);
    if constexpr (!kWide) {
      if (wave == 0) {
        const int64_t page = min(max(pg_vs, 0), p.num_pages - 1);
        rvs = p.vs ? p.vs[page * p.vs_sp + (int64_t)kvh * p.vs_sh + ((key0 + lane) & ps_mask)]
                   : 1.f;
      }
    }
  };
  auto load_tile = [&](int j, int buf) MXFA_INLINE {
    load_k(j, buf);
    load_v(j, buf);
  };
  // 16 loaded bytes of a row into its LDS row, an 8-bit cache's widened.
  auto put = [&](auto type, char *dst, const uint4 &w, int sw) MXFA_INLINE {
    using TR = decltype(type);
    if constexpr (kWide) {
      *reinterpret_cast<uint4 *>(dst + (l_chunk ^ sw) * 16) = w;
    } else {
      const uint2 a = widen_codes<TR, kCache>(w.x), b = widen_codes<TR, kCache>(w.y);
      const uint2 c = widen_codes<TR, kCache>(w.z), d = widen_codes<TR, kCache>(w.w);
      *reinterpret_cast<uint4 *>(dst + ((2 * l_chunk) ^ sw) * 16) = make_uint4(a.x, a.y, b.x, b.y);
      *reinterpret_cast<uint4 *>(dst + ((2 * l_chunk + 1) ^ sw) * 16) =
          make_uint4(c.x, c.y, d.x, d.y);
    }
  };
  // Rows from registers to LDS; of V, zeros outside rows [lo, hi).
  auto store_rows = [&](const uint4 (&reg)[kDirect ? 1 : kPer], char *lds, auto type, auto is_k,
                        int lo, int hi) MXFA_INLINE {
    if constexpr (!kDirect) {
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int r = w_row + u * kWaveRows + l_row;
        uint4 w = reg[u];
        if constexpr (!decltype(is_k)::value) {
          const bool there = r >= lo && r < hi;
          w = make_uint4(there ? w.x : 0u, there ? w.y : 0u, there ? w.z : 0u, there ? w.w : 0u);
        }
        const int sw = decltype(is_k)::value ? swizzle_k<HD>(r) : swizzle_v<HD>(r);
        put(type, lds + r * kRowBytes, w, sw);
      }
    }
  };
  auto store_k = [&](int buf) MXFA_INLINE {
    store_rows(rk, lds_k[buf], T{}, std::true_type{}, 0, KT);
    // A V row without a scale (NaN: it held an infinity or a NaN) takes its key's score along
    // instead, so that it reaches the rows that see the key and no other (a weight of zero
    // times NaN would).
    if constexpr (!kWide) {
      if (wave == 0) lds_ks[buf][lane] = fabsf(rvk) < INFINITY ? rks : __builtin_nanf("");
    }
  };
  // The loaded rows into LDS (kDirect: they are on their way there; this wave's are waited
  // for). V rows that no row of the tile sees (past its last key, ahead of its windows) become
  // zeros, whatever their memory holds: a weight of zero times a NaN is a NaN.
  auto store_tile = [&](int j, int buf) MXFA_INLINE {
    const int lo = k_first - (k_begin + j * KT), hi = k_end - (k_begin + j * KT);
    if constexpr (kDirect) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (hi < KT || lo > 0) {  // at the ends of the tile's keys
        int r = w_row + l_row;
        asm volatile("" : "+v"(r));  // nothing of this is worth registers in the loop
        for (int u = 0; u < kPer; ++u, r += kWaveRows)
          if (r < lo || r >= hi)
            *reinterpret_cast<uint4 *>(lds_v[buf] + r * kRowBytes + l_chunk * 16) =
                make_uint4(0u, 0u, 0u, 0u);
      }
    } else {
      store_k(buf);
      store_rows(rv, lds_v[buf], TV{}, std::false_type{}, lo, hi);
      if constexpr (!kWide) {
        if (wave == 0) lds_vs[buf][lane] = fabsf(rvs) < INFINITY ? rvs : 0.f;
      }
    }
  };

  float m = -INFINITY, l = 0.f;
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  // K operand of the 32 keys in rows r0.. of buffer buf, dims 16 i ..; up to eight are read
  // ahead of their products.
  constexpr int kReads = !kWide ? (NQ < 4 ? NQ : 4) : NQ < 8 ? NQ : 8;
  uint4 kf[kReads];
  // LDS addresses of the lane's operands, kept in registers where they fit (kUnroll): buffer
  // and row are then the reads' constant offsets.
  constexpr bool kUnroll = kUniform && !kExtras && HD < 256 && !(kSplitP && HD == 128);
  uint32_t k_at[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    k_at[i] = lds_offset(lds_k[0]) + col * kRowBytes + (((2 * i + half) ^ swizzle_k<HD>(col)) * 16);
    if constexpr (kUnroll) asm("" : "+v"(k_at[i]));
  }
  auto read_k = [&](int buf, int r0, int i) MXFA_INLINE {
    typedef const __attribute__((address_space(3))) u32x4_t LdsVec;
    const u32x4_t x =
        *(LdsVec *)(uintptr_t)(k_at[i] + buf * (KT * kRowBytes) + r0 * kRowBytes);
    kf[i % kReads] = make_uint4(x.x, x.y, x.z, x.w);
  };
  // The scales of an 8-bit cache's rows: scores keys 8 (i / 4) + 4 half + i % 4 of the 32.
  auto scale_scores = [&](int buf, int r0, f32x16 &s) MXFA_INLINE {
    if constexpr (!kWide) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 f = *reinterpret_cast<const float4 *>(&lds_ks[buf][r0 + 8 * g + 4 * half]);
        s[4 * g] *= f.x;
        s[4 * g + 1] *= f.y;
        s[4 * g + 2] *= f.z;
        s[4 * g + 3] *= f.w;
      }
    }
  };
  const auto largest = [&](const f32x16 &s) MXFA_INLINE {
    float x = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) x = fmaxf(x, s[i]);
    return x;
  };
  // Options and masks; top: the lane's largest score.
  auto limit = [&](int key0, f32x16 &s, float &top) MXFA_INLINE {
    if constexpr (kExtras) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x = s[i] * c;
        if (capped) {
          // cap * tanh(x / cap) = cap * (1 - 2 / (e^(2 x / cap) + 1)), in base 2
          const float e = fast_exp2(x * (2.f / p.softcap));
          x = p.softcap * kPrefillLog2e * (1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f));
        }
        const int key = key0 + 8 * (i >> 2) + 4 * half + (i & 3);
        x -= slope * (float)abs(pos - key);
        s[i] = x;
      }
      top = largest(s);
    }
    // Keys that some row of the wave does not see.
    if (key0 + 31 > all_to || key0 < all_from) {
      const int hi = lim - key0 - 4 * half, lo = from - key0 - 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int k = 8 * (i >> 2) + (i & 3);
        s[i] = (k <= hi && k >= lo) ? s[i] : -INFINITY;
      }
      top = largest(s);
    }
  };
  // Moves the reference where a score passed it by more than kPrefillRescaleLog2.
  auto refer = [&](float top) MXFA_INLINE {
    top *= cs;
    if (__builtin_amdgcn_ballot_w64(top > m + kPrefillRescaleLog2) != 0) {  // wave-uniform
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top),
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
  };
  // Weights of 32 keys (V rows r0.. of buffer buf), rounded once (the 16-bit products take no
  // more): eight keys per operand register set. Score i's part of it: pairs are packed and
  // summed as they come.
  uint32_t pf[8], pl[kSplitP ? 8 : 1];
  float mr;  // the reference; 0 where no key is seen yet (the scores are -inf then)
  // 8-bit: V's scales of the lane's keys, all read ahead, or (fp16, where the split weights
  // take the registers) four keys ahead.
  constexpr int kScales = 2;
  float4 vsc[kScales];
  auto read_vs = [&](int buf, int r0, int g) MXFA_INLINE {
    vsc[g % kScales] = *reinterpret_cast<const float4 *>(&lds_vs[buf][r0 + 8 * g + 4 * half]);
  };
  auto weigh_start = [&](int buf, int r0) MXFA_INLINE {
    mr = m == -INFINITY ? 0.f : m;
    if constexpr (!kWide) {
#pragma unroll
      for (int g = 0; g < kScales - 1; ++g) read_vs(buf, r0, g);
    }
  };
  auto weigh = [&](auto ic, int buf, int r0, f32x16 &s) MXFA_INLINE {
    constexpr int i = decltype(ic)::value;
    s[i] = fast_exp2(__builtin_fmaf(s[i], cs, -mr));
    if constexpr (!kWide) {
      if constexpr (i % 4 == 0 && i < 12) read_vs(buf, r0, i / 4 + 1);
      l += s[i];
      const float4 f = vsc[(i >> 2) % kScales];
      s[i] *= (i & 3) == 0 ? f.x : (i & 3) == 1 ? f.y : (i & 3) == 2 ? f.z : f.w;
    }
    if constexpr (i & 1) {
      pf[i >> 1] = Prod32<TV>::pack(s[i - 1], s[i]);
      if constexpr (kSplitP)
        pl[i >> 1] = Prod32<TV>::pack(s[i - 1] - Elem<BF16>::lo(pf[i >> 1]),
                                      s[i] - Elem<BF16>::hi(pf[i >> 1]));
      // The sum of the rounded weights: the output is then a mean of V rows, and a pair
      // takes one instruction. (8-bit rows: the weights carry vs; summed above.)
      if constexpr (kWide) l = Prod32<T>::add_pair(pf[i >> 1], l);
    }
  };
  // V^T operand: lane l reads dims 16 ((l / 16) % 2) + 4 (l % 4) .. of key
  // 4 (l / 32) + (l / 4) % 4 and receives dim l % 32 of four keys.
  const int v_key = 4 * half + ((lane >> 2) & 3);
  const int v_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);  // within the 32-dim block
  uint32_t v_at[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int byte = (d * 32 + v_dim) * 2;
    v_at[d] = lds_offset(lds_v[0]) + v_key * kRowBytes +
              (((byte >> 4) ^ swizzle_v<HD>(v_key)) << 4) + (byte & 15);
    if constexpr (kUnroll) asm("" : "+v"(v_at[d]));
  }
  auto read_v = [&](int buf, int r0, int d) MXFA_INLINE {
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t at = v_at[d] + buf * (KT * kRowBytes) + (r0 + 8 * u) * kRowBytes;
      typedef __attribute__((address_space(3))) s16x4v LdsVec;
      const s16x4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec *)(uintptr_t)at);
      const uint2 y = __builtin_bit_cast(uint2, x);
      w[2 * u] = y.x;
      w[2 * u + 1] = y.y;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  // The loop runs the scores of 32 keys ahead of their weights: the next keys' products fill
  // the matrix unit while these keys' exponentials go through the VALU, a few after each
  // product. The order is written out (sched_barrier): left to itself the compiler issues
  // the products in a row, and a wave issues in order.
  float top = -INFINITY;
  auto first_scores = [&](int buf, int r0, f32x16 &s) MXFA_INLINE {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      read_k(buf, r0, i);
      s = Prod32<T>::run(kf[i % kReads], qf[i], s);
    }
    scale_scores(buf, r0, s);
    if constexpr (!kExtras) top = largest(s);
  };
  // The weights of cur's keys and their part of the output, and nxt's scores.
  // between(slot): work after the slot-th product of NQ + 2 ND.
  const auto nothing = [](auto) MXFA_INLINE {};
  auto advance = [&](int buf, int r0, f32x16 &cur, f32x16 &nxt, auto between) MXFA_INLINE {
#pragma unroll
    for (int i = 0; i < kReads; ++i) read_k(buf, r0, i);
    weigh_start(buf, r0);
    uint4 vf[ND];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) nxt[i] = 0.f;
    static_unroll<NQ>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      nxt = Prod32<T>::run(kf[i % kReads], qf[i], nxt);
      if constexpr (i + kReads < NQ) read_k(buf, r0, i + kReads);
      static_unroll<16 / NQ>([&](auto jc) {
        weigh(std::integral_constant<int, i * (16 / NQ) + decltype(jc)::value>{}, buf, r0, cur);
      });
      if constexpr (i >= NQ / 2) {  // the first V operands, in the second half's shadow
        static_unroll<2 * ND / NQ>([&](auto jc) {
          constexpr int d = (i - NQ / 2) * (2 * ND / NQ) + decltype(jc)::value;
          vf[d] = read_v(buf, r0, d);
        });
      }
      between(ic);
      __builtin_amdgcn_sched_barrier(0);
    });
    uint4 vn[ND];
    static_unroll<2 * ND>([&](auto ic) {
      constexpr int st = decltype(ic)::value / ND, d = decltype(ic)::value % ND;
      const uint4 a = st ? vn[d] : vf[d];
      o[d] = Prod32<TV>::run(
          a, make_uint4(pf[4 * st], pf[4 * st + 1], pf[4 * st + 2], pf[4 * st + 3]), o[d]);
      if constexpr (kSplitP)
        o[d] = Prod32<TV>::run(
            a, make_uint4(pl[4 * st], pl[4 * st + 1], pl[4 * st + 2], pl[4 * st + 3]), o[d]);
      if constexpr (st == 0) vn[d] = read_v(buf, r0 + 16, d);
      between(std::integral_constant<int, NQ + decltype(ic)::value>{});
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (st == 0 && d == ND - 1) scale_scores(buf, r0, nxt);
    });
    if constexpr (!kExtras) top = largest(nxt);
  };
  auto step = [&](int key0, int buf, int r0, f32x16 &cur, f32x16 &nxt, auto between) MXFA_INLINE {
    if (key0 <= any_to) {  // some row of the wave sees some of the 32 keys
      limit(key0, cur, top);
      refer(top);
      // (past the last keys, products that nobody looks at)
      advance(buf, r0, cur, nxt, between);
    }
  };
  // Rows straight to LDS: a wave's 2 kPer loads of the next tile go out one by one among the
  // first step's products. (All at once they hold the wave up: the CU takes 64 bytes a clock,
  // 512 clocks for a tile of the four waves.)
  auto spread_load = [&](int j, int buf, bool more) MXFA_INLINE {
    const int key0 = k_begin + j * KT + w_row;
    const int page_k = __builtin_amdgcn_readlane(pg_k[0], 0);
    const int page_v = __builtin_amdgcn_readlane(pg_k[0], 32);
    const char *const src_k = uniform_pointer(p.k + row_off(key0 + kAhead, page_k));
    const char *const src_v = uniform_pointer(p.v + row_off(key0, page_v));
    const uint32_t to_k = lds_offset(lds_k[buf]) + w_row * kRowBytes;
    const uint32_t to_v = lds_offset(lds_v[buf]) + w_row * kRowBytes;
    const uint32_t half_on = __builtin_amdgcn_readfirstlane(more ? 0xffffffffu : 0u);
    const uint64_t on = (uint64_t)half_on << 32 | half_on;
    return [=](auto slot) MXFA_INLINE {
      constexpr int s = decltype(slot)::value;
      constexpr bool is_k = s < NQ;
      constexpr int apart = is_k ? NQ / kPer : 2 * ND / kPer, i = is_k ? s : s - NQ;
      if constexpr (i % apart == 0 && i / apart < kPer) {
        constexpr int u = i / apart;
        const int r = u * kWaveRows + l_row;
        const int from = is_k ? l_chunk ^ swizzle_k<HD>(r) : l_chunk ^ swizzle_v<HD>(r);
        load_to_lds_if((is_k ? src_k : src_v) + u * kWaveRows * st, lane_off + from * 16,
                       (is_k ? to_k : to_v) + u * kWaveRows * kRowBytes, on);
      }
    };
  };
  if constexpr (!kDirect) sign_q();  // (later, the unsigned q would take registers too)
  if (few) {
    // Few rows: the four waves share them and each takes a quarter of the piece's keys, 32 at
    // a time through its own quarter of the K and V buffers, with no barrier; rows come
    // through registers, the next 32 keys' loads in flight during the math. (One wave on all
    // keys is bound by the time of a step: 31 sequences of one token on 1k-8k int8 keys beside
    // a chunk of 1024, 32q/8kv HD 128, 179 us against 128.)
    constexpr int kFew = 32 / kWaveRows;
    constexpr int kFewPages = kUniform ? 1 : kFew;  // (kUniform: of 16 rows, in each half)
    char *const own_k = lds_k[wave >> 1] + (wave & 1) * 32 * kRowBytes;
    char *const own_v = lds_v[wave >> 1] + (wave & 1) * 32 * kRowBytes;
    const int buf = wave >> 1, r0 = (wave & 1) * 32;
    const int blocks = 2 * (j1 - j0);
    const int i1 = blocks * (wave + 1) / kPrefillWaves;
    const int base = k_begin + j0 * KT;
    uint4 fk[kFew], fv[kFew];
    int pages[kFewPages], page_s = 0;
    float fks = 1.f, fvs = 1.f;
    auto few_pages = [&](int i) MXFA_INLINE {
      const int key0 = base + 32 * i;
#pragma unroll
      for (int u = 0; u < kFewPages; ++u) {
        if constexpr (kUniform)
          pages[u] = bt[page_at(key0 + 16 * half)];
        else
          pages[u] = bt[page_at(key0 + u * kWaveRows + l_row)];
      }
      if constexpr (!kWide) page_s = bt[page_at(key0 + (lane & 31))];
    };
    auto few_load = [&](int i) MXFA_INLINE {
      const int key0 = base + 32 * i;
#pragma unroll
      for (int u = 0; u < kFew; ++u) {
        const int r = u * kWaveRows;
        int64_t off;
        if constexpr (kUniform)
          off = row_off(key0 + r, __builtin_amdgcn_readlane(pages[0], r < 16 ? 0 : 32)) + lane_off;
        else
          off = row_off(key0 + r + l_row, pages[u]);
        off += l_chunk * 16;
        fk[u] = load_stream16(p.k + off);
        fv[u] = load_stream16(p.v + off);
      }
      if constexpr (!kWide) {
        const int64_t page = min(max(page_s, 0), p.num_pages - 1);
        const int at = (key0 + (lane & 31)) & ps_mask;
        fks = p.ks ? p.ks[page * p.ks_sp + (int64_t)kvh * p.ks_sh + at] : 1.f;
        fvs = p.vs ? p.vs[page * p.vs_sp + (int64_t)kvh * p.vs_sh + at] : 1.f;
      }
    };
    int i = blocks * wave / kPrefillWaves;
    if (i < i1) {
      few_pages(i);
      few_load(i);
      few_pages(i + 1);
    }
    if constexpr (kDirect) sign_q();
    for (; i < i1; ++i) {
      const int key0 = base + 32 * i;
#pragma unroll
      for (int u = 0; u < kFew; ++u) {
        const int r = u * kWaveRows + l_row;
        const bool there = key0 + r >= k_first && key0 + r < k_end;
        put(T{}, own_k + r * kRowBytes, fk[u], swizzle_k<HD>(r));
        const uint4 w = fv[u];
        put(TV{}, own_v + r * kRowBytes,
            make_uint4(there ? w.x : 0u, there ? w.y : 0u, there ? w.z : 0u, there ? w.w : 0u),
            swizzle_v<HD>(r));
      }
      if constexpr (!kWide) {
        if (lane < 32) {
          const bool whole = fabsf(fvs) < INFINITY;
          lds_ks[buf][r0 + lane] = whole ? fks : __builtin_nanf("");
          lds_vs[buf][r0 + lane] = whole ? fvs : 0.f;
        }
      }
      if (i + 1 < i1) {
        few_load(i + 1);
        few_pages(i + 2);
      }
      f32x16 s;
      first_scores(buf, r0, s);
      limit(key0, s, top);
      refer(top);
      weigh_start(buf, r0);
      static_unroll<16>([&](auto ic) { weigh(ic, buf, r0, s); });
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const uint4 a = read_v(buf, r0 + 16 * st, d);
          o[d] = Prod32<TV>::run(
              a, make_uint4(pf[4 * st], pf[4 * st + 1], pf[4 * st + 2], pf[4 * st + 3]), o[d]);
          if constexpr (kSplitP)
            o[d] = Prod32<TV>::run(
                a, make_uint4(pl[4 * st], pl[4 * st + 1], pl[4 * st + 2], pl[4 * st + 3]), o[d]);
        }
    }
  } else if (j0 < j1) {
    f32x16 sa, sb;
    // K's stage before the first holds the first 32 keys. Loads go out as their pages come.
    find_pages(j0 - 1);
    int pg_0[kPages];
#pragma unroll
    for (int u = 0; u < kPages; ++u) pg_0[u] = pg_k[u];
    const int pg_s0 = pg_ks;
    find_pages(j0);
    load_rows(p.k, k_begin + j0 * KT - kAhead, pg_0, std::true_type{}, lds_k[1], rk);
    load_k_scales(k_begin + j0 * KT - kAhead, pg_s0);
    load_v(j0, 0);
    if constexpr (!kDirect) store_k(1);
    load_k(j0, 0);
    if constexpr (kDirect) sign_q();
    find_pages(j0 + 1);
    if constexpr (kDirect) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    first_scores(1, kAhead, sa);
    auto tile = [&](int j, auto bc) MXFA_INLINE {
      const int buf = bc, key0 = k_begin + j * KT;
      // One barrier a tile: past it V of tile j and K 32 keys on are in LDS, and every wave is
      // done with the other buffers, which the next loads fill.
      store_tile(j, buf);
      if (!kDirect && j + 1 < j1) {
        load_tile(j + 1, buf ^ 1);
        find_pages(j + 2);
      }
      __syncthreads();
      if constexpr (kDirect) {
        const auto loads = spread_load(j + 1, buf ^ 1, j + 1 < j1);
        find_pages(j + 2);
        // (A wave without work in the step: apart from the step's condition, or the compiler
        // joins the two and copies accumulators.)
        int first = key0;
        asm("" : "+s"(first));
        if (first > any_to) static_unroll<NQ + 2 * ND>(loads);
        step(key0, buf, 0, sa, sb, loads);
      } else {
        step(key0, buf, 0, sa, sb, nothing);
      }
      step(key0 + 32, buf, 32, sb, sa, nothing);
    };
    if constexpr (kUnroll) {
      // Two tiles a round: the buffers are then constants, and part of the LDS reads' offsets.
      for (int j = j0; j < j1; j += 2) {
        tile(j, std::integral_constant<int, 0>{});
        if (j + 1 < j1) tile(j + 1, std::integral_constant<int, 1>{});
      }
    } else {  // (the staging registers leave no room for that)
      for (int j = j0; j < j1; ++j) tile(j, (j - j0) & 1);
    }
  }

  const auto lw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false,
                                                   false);
  l = __uint_as_float(lw[0]) + __uint_as_float(lw[1]);
  if (few) {
    // The four waves' rows: references and sums, then the accumulators as [4 dims][row] through
    // the K (waves 0, 1) and V (2, 3) buffers; thread (part, row) then joins HD / 8 dims of a
    // row in wave order.
    __syncthreads();
    float4 *const mine = reinterpret_cast<float4 *>(wave < 2 ? lds_k[0] : lds_v[0]) +
                         (wave & 1) * (HD / 4) * 32;
    if (half == 0) {
      few_m[wave][col] = m;
      few_l[wave][col] = l;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        mine[(d * 8 + 2 * g + half) * 32 + col] =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    __syncthreads();
    const int r = threadIdx.x & 31, part = threadIdx.x >> 5;
    if (r >= rows) return;
    float mm = -INFINITY, ll = 0.f, f[kPrefillWaves];
#pragma unroll
    for (int w = 0; w < kPrefillWaves; ++w) mm = fmaxf(mm, few_m[w][r]);
#pragma unroll
    for (int w = 0; w < kPrefillWaves; ++w) {
      // A wave that saw no key has the reference -inf and no sum; one that saw only NaN too,
      // and its NaN sum stays.
      f[w] = few_m[w][r] == -INFINITY ? 1.f : fast_exp2(few_m[w][r] - mm);
      ll += f[w] * few_l[w][r];
    }
    const int64_t at = (int64_t)it.slot * p.hkv + kvh;
    float inv;
    if (it.pieces > 1) {
      if (threadIdx.x == 0)
        p.ws_desc[at] = make_int4(it.piece == 0 ? it.pieces : 0, it.b, it.tile, 0);
      if (part == 0)
        p.ws_lse[at * kRows + r] = ll > 0.f ? mm + __log2f(ll) : (ll == 0.f ? -INFINITY : ll);
      inv = ll == 0.f ? 0.f : v_scale / ll;
    } else {
      float den = ll;
      if (p.sinks) den += fast_exp2(p.sinks[kvh * gq + r - token_of(r) * gq] * kPrefillLog2e - mm);
      inv = ll == 0.f ? 0.f : v_scale / den;
    }
    char *const dst = p.out + (int64_t)(sq.start + token_of(r)) * p.o_st +
                      (int64_t)(kvh * gq + r - token_of(r) * gq) * p.o_sh;
#pragma unroll
    for (int cc = 0; cc < HD / 32; ++cc) {
      const int chunk = part * (HD / 32) + cc;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPrefillWaves; ++w) {
        const float4 x = (reinterpret_cast<const float4 *>(w < 2 ? lds_k[0] : lds_v[0]) +
                          (w & 1) * (HD / 4) * 32)[chunk * 32 + r];
        acc.x += f[w] * x.x;
        acc.y += f[w] * x.y;
        acc.z += f[w] * x.z;
        acc.w += f[w] * x.w;
      }
      acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (it.pieces > 1)
        *reinterpret_cast<float4 *>(p.ws_o + (at * kRows + r) * HD + 4 * chunk) = acc;
      else
        *reinterpret_cast<uint2 *>(dst + 8 * chunk) =
            make_uint2(Prod32<T>::pack(acc.x, acc.y), Prod32<T>::pack(acc.z, acc.w));
    }
    return;
  }
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
// tile's first piece, a thread for four dims of kPer rows, in one pass with the running
// reference and sum of each, kAhead pieces' loads at a time (16 heads on one kv head, some 200
// tokens on up to 6k keys, 20 pieces a tile: 65.3 us with a piece's loads at a time, 45.6).
constexpr int kPrefillJoinThreads = 256;
constexpr int kPrefillJoinParts = 4;

template <int HD, typename T>
__global__ __launch_bounds__(kPrefillJoinThreads) void paged_prefill_join_kernel(PrefillParams p) {
  constexpr int kRows = kPrefillRows;
  constexpr int kTogether = kPrefillJoinThreads / (HD / 4);  // rows
  constexpr int kPer = kRows / kPrefillJoinParts / kTogether;
  constexpr int kAhead = 16 / kPer;
  const int at = blockIdx.x;  // slot * hkv + kv head
  const int slot = div_by(at, p.hkv, p.hkv_mul), kvh = at - slot * p.hkv;
  if (slot >= *p.ws_total) return;
  const int4 d = p.ws_desc[at];
  const int pieces = d.x;
  if (pieces <= 1 || slot + pieces > p.max_slots || d.y < 0 || d.y >= p.batch) return;
  const PrefillSeq sq = prefill_seq(p, d.y);
  const int chunk = threadIdx.x % (HD / 4);
  const int rows = min(kRows, sq.n * p.gq - d.z * kRows);
  if ((int)blockIdx.y * (kTogether * kPer) >= rows) return;
  const int r0 = blockIdx.y * (kTogether * kPer) + threadIdx.x / (HD / 4);
  float m[kPer], sum[kPer];
  float4 acc[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    m[u] = -INFINITY;
    sum[u] = 0.f;
    acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int i = 0; i < pieces; i += kAhead) {
    float lse[kAhead][kPer];
    float4 x[kAhead][kPer];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int64_t first = (at + (int64_t)min(i + a, pieces - 1) * p.hkv) * kRows;
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int64_t r = first + min(r0 + u * kTogether, rows - 1);
        lse[a][u] = p.ws_lse[r];
        x[a][u] = *reinterpret_cast<const float4 *>(p.ws_o + r * HD + 4 * chunk);
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (i + a >= pieces) break;
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const float top = fmaxf(m[u], lse[a][u]);
        // No key seen so far, or none in the piece: weight 0. (A NaN stays one.)
        const float f = m[u] == -INFINITY ? 0.f : fast_exp2(m[u] - top);
        const float w = lse[a][u] == -INFINITY ? 0.f : fast_exp2(lse[a][u] - top);
        m[u] = top;
        sum[u] = sum[u] * f + w;
        acc[u].x = acc[u].x * f + w * x[a][u].x;
        acc[u].y = acc[u].y * f + w * x[a][u].y;
        acc[u].z = acc[u].z * f + w * x[a][u].z;
        acc[u].w = acc[u].w * f + w * x[a][u].w;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int r = r0 + u * kTogether;
    if (r >= rows) continue;
    const int row = d.z * kRows + r;
    const int tok = div_by(row, p.gq, p.gq_mul), head = kvh * p.gq + row - tok * p.gq;
    float den = sum[u];
    if (p.sinks) den += fast_exp2(p.sinks[head] * kPrefillLog2e - m[u]);
    const float inv = sum[u] == 0.f ? 0.f : 1.f / den;
    *reinterpret_cast<uint2 *>(p.out + (int64_t)(sq.start + tok) * p.o_st +
                               (int64_t)head * p.o_sh + 8 * chunk) =
        make_uint2(Prod32<T>::pack(acc[u].x * inv, acc[u].y * inv),
                   Prod32<T>::pack(acc[u].z * inv, acc[u].w * inv));
  }
}

// Launches of one head dim (prefill_hd*.hip).
template <int HD, typename T, int kCache>
int launch_prefill_t(const PrefillParams &p, int items, hipStream_t st) {
  const dim3 grid((unsigned)(items * p.hkv)), block(kPrefillWaves * 64);
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

// Attention over rows = (token, query head of a K/V head's group): what packed prompts
// (attn_packed.hip) and a batch's new tokens behind a shared prefix (attn_prefix.hip) have in common.
//
// For one K/V head and a range of keys, each row i keeps the running maximum top of its scores, the sum of its softmax and
// the output O = sum_j 2^(c s_ij - mu) v_j, c = scale * log2 e, mu = c top:
//   S^T = K · Q^T and O^T += V^T · P^T on 16x16x32 MFMAs, keys in BN-key tiles through a ring of LDS
//   tiles filled by LDS-DMA, V^T fragments by transpose reads of the key-major tile. A lane holds
//   one row (lane % 16) and 4 keys of every 16, so the scores of a 32-key unit are its P^T operand
//   as they are: keys 4 g + i and 16 + 4 g + i (g = lane / 16), the order of the V^T reads.
//   The heads of a group are rows of one tile: K and V are read once for all of them.
//   The maximum moves only when a score exceeds it by more than 8 (log2 units), and only then do
//   the four lanes of a row exchange anything; sums are exchanged once at the end.
// Bound by the matrix cores and the exponentials' vector instructions where rows are many (one prompt of 8192
// tokens, 32/8 heads of 128, bf16: 479 to 498 us on different cards, 1.10 to 1.15 PFLOP/s, matrix cores busy 52% and
// vector ALU 32% of the cycles at 1.9 GHz), by the bytes of K and V where they are few (32 single tokens against 4000 keys
// each: 96 us and 5 of joining, 5.2 TB/s).
#pragma once

#include <type_traits>

#include "attn.h"

namespace rows {

// What a work-group's rows attend to: a range of a packed sequence's keys; of the prefix, for rows of the
// whole batch; of one sequence's own cache; prefix and cache one after the other (WHOLE: nothing to join).
enum Mode { PACKED = 0, PREFIX = 1, OWN = 2, WHOLE = 3 };

// Work on one tile of rows of one packed sequence (mi355_attn_packed_plan writes them).
struct PackedTile {
  int32_t q0, q_len;        // the sequence's first token in q and its tokens
  int32_t k0, k_len;        // ... in k / v
  int32_t row0;             // first row of the tile: token row0 / G, head row0 % G of the group
  int32_t k_begin, k_stop;  // the range of its keys, of which it takes what its rows see
  int32_t slot;             // first row of its partial result; -1: the range is all there is
};
static_assert(sizeof(PackedTile) == 32, "plan entry");

// Division of n < 2^31 by a fixed d >= 1: with 2^(l - 1) < d <= 2^l and mul = ceil(2^(31 + l) / d), which
// exceeds the quotient by less than d / d, floor(n / d) = floor(n mul / 2^(31 + l)), since n (mul d - 2^(31 + l)) <
// 2^31 d <= 2^(31 + l). Two instructions for the compiler's twenty-five.
struct Div {
  uint32_t mul, shift;  // d = 1: mul 0
};
inline Div make_div(int64_t d) {
  if (d <= 1) return Div{0u, 0u};
  uint32_t l = 0;
  while ((int64_t(1) << l) < d) ++l;
  return Div{static_cast<uint32_t>(((uint64_t(1) << (31 + l)) + d - 1) / d), l - 1};
}
MI355_DEVINL int quotient(int n, Div d) {
  return d.mul == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), d.mul) >> d.shift);
}

struct Args {
  const void *q, *k, *v;
  void* o;                // PACKED: output
  int64_t qb, qt, qh;     // strides in elements: batch (not PACKED), token, head
  int64_t kb, kt, kh;     // batch (OWN), token, head
  int64_t vb, vt, vh;
  int64_t ob, ot, oh;
  float c;                // scale * log2(e)
  int32_t G, H, Hkv;      // query heads of a K/V head, query heads, K/V heads
  Div by_G, by_Hkv;
  // PACKED
  const PackedTile* tiles;
  int32_t causal;
  int64_t slots;          // partial rows of a K/V head: row (h slots + slot + i) of part / ml
  // PREFIX / OWN / WHOLE: rows of a sequence are its n_q tokens' heads
  int32_t B, n_q;
  int32_t keys;           // PREFIX: prefix keys; OWN, WHOLE: keys a cache has room for
  const int32_t* lens;    // OWN, WHOLE: keys in each cache (clamped to [0, keys])
  const void *pk, *pv;    // WHOLE: the prefix, its token and head strides and keys (k, v: the caches)
  int64_t pkt, pkh, pvt, pvh;
  int32_t pkeys;
  int32_t chunk;          // keys of a split
  int32_t splits, row_tiles;
  Div by_n_q, by_splits, by_row_tiles;
  int32_t part0;          // first split's index in part / ml
  float* part;            // partial rows [HD], unnormalised; PREFIX / OWN: [splits][B n_q H]
  float* ml;              // their mu (-inf: no key seen) and sum
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

MI355_DEVINL f32x4 mma32(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
MI355_DEVINL f32x4 mma32(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// sum of a fragment's probabilities, as rounded
MI355_DEVINL float prob_sum(f16x8 f, float acc) {
  const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_fdot2(f16x2{f[2 * r], f[2 * r + 1]}, one, acc, false);
  return acc;
}
MI355_DEVINL float prob_sum(bf16x8 f, float acc) {
  const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{f[2 * r], f[2 * r + 1]}, one, acc, false);
  return acc;
}
// A fragment of probabilities as two terms: what is left of each after its lower bits are cut off, and those. The
// second is positive where the first is (at least the type's least number; in all off by at most 2^-21 of the
// probability or 2^-24 in fp16, 2^-15 of it in bf16), so that both have an infinite v's product with its sign.
MI355_DEVINL void two_terms(const float (&e)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int r = 0; r < 8; r += 2) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(e[r], e[r + 1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      hi[r + i] = h[i];
      lo[r + i] = static_cast<_Float16>(__builtin_amdgcn_fmed3f(e[r + i] - static_cast<float>(h[i]), 0x1p-24f, e[r + i]));
    }
  }
}
MI355_DEVINL void two_terms(const float (&e)[8], bf16x8& hi, bf16x8& lo) {
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float h = __uint_as_float(__float_as_uint(e[r]) & 0xffff0000u);
    hi[r] = static_cast<__bf16>(h);
    lo[r] = static_cast<__bf16>(__builtin_amdgcn_fmed3f(e[r] - h, 0x1p-126f, e[r]));
  }
}
// reductions over the four lanes l, l ^ 16, l ^ 32, l ^ 48 of a row
MI355_DEVINL float row_maximum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_maximum(vmax(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
MI355_DEVINL float row_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// buffer_dma_lds16 (common.h) for a resource that the vector ALU may have written just before, as it does with a
// range that depends on a length from memory: five wait states before the load reads it.
MI355_DEVINL void buffer_dma_lds16_after_valu(u32x4 rsrc, uint32_t voffset, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voffset), "s"(rsrc),
               "s"(__builtin_amdgcn_readfirstlane(lds_addr))
               : "memory", "m0");
}

// XOR of a row's 16-byte chunks (NCH per row) by its low 4 bits. 16 lanes are served together: of a
// K fragment read (16 rows, 4 neighbouring chunks) rows 0-3 and 12-15 at one chunk with rows 4-11 at
// the next, of a V transpose read 4 rows at 2 neighbouring chunks. Row pitches of 2, 6 and 10 chunks
// keep those apart by themselves.
template <int NCH>
MI355_DEVINL int swz(int r) {
  const int r0 = r & 1, r1 = (r >> 1) & 1, r2 = (r >> 2) & 1, r3 = (r >> 3) & 1;
  if constexpr (NCH % 16 == 0)
    return r2 | (r0 << 1) | (r1 << 2) | ((r2 ^ r3) << 3);
  else if constexpr (NCH % 8 == 0)
    return r2 | ((r0 ^ r2 ^ r3) << 1) | (r1 << 2);
  else if constexpr (NCH % 4 == 0)
    return r2 | ((r1 ^ r2 ^ r3) << 1);
  else
    return 0;
}

// 16-byte chunks of LDS that a body needs
template <int HD, int NW, int BN, bool OWN_KEYS>
constexpr int lds_chunks() { return 2 * BN * (HD / 8) * (OWN_KEYS ? NW : 2); }

// What waves with the same rows leave for each other: maximum and sum of each row, and of all whether one has a NaN.
template <int NW, int QW>
struct Joined {
  float ml[NW][QW][2];
  uint32_t flags[NW];
};

// Scores whose product with c is so large that its rounding, 2^-24 of it, shifts a probability by a factor of 2 and
// more; fp16 probabilities would overflow from 2^28 on.
constexpr float FAR = 0x1p24f;

enum Pass { GIVEN = 0, CLEAN = 1, UP = 2, DOWN = 3 };

// The work of one work-group: NW waves of QG groups of 16 rows.
//   OWN_KEYS = false: each wave has rows of its own, the waves share tiles of BN keys (double-buffered).
//   OWN_KEYS = true, for at most 16 QG rows: the waves have the same rows and keys of their own, tile w,
//     w + NW .. of the range, in one buffer each for K and V, and are joined through LDS at the end.
// TERMS: the probabilities enter P · V as that many terms of the input type. One where tiles have rows enough to be matrix
// work (packed tiles of 64 and 128 rows, prefix tiles of 128), as in the framework's other attention kernels: against 64
// bits the outputs are then off by 1.1 to 1.4 times their own rounding (8 pieces of prompts, fp16: 2.9e-4 of the norm
// beside 2.1e-4). Two terms would cost the pieces half of their speed and 64 x 4 tokens behind 8192 keys 60 -> 71 us. Two
// where K and V are waited for (up to 32 rows, prefix tiles up to 64): it costs nothing there, and the error is the rounding's.
// A key that a row does not see has probability 0, but its v row is in the tile: 0 · inf and 0 · NaN leave NaN in rows
// that do not see it. Where that may have happened (a NaN beside keys that not all rows see: true is returned) the
// work-group goes through its keys again (AGAIN: three passes, but if V has no such element at those keys), with
//   CLEAN: infinities and NaN of V as 0, for the outputs; then, with K = 0 (every key that a row sees counts 1), for
//   the outputs that such elements reach: UP: V = 1 for inf and NaN, 0 else, and inf is added where anything is left,
//   DOWN: V = 1 for -inf and NaN, and -inf is added.
// (2048 tokens, 32/8 heads of 128, bf16, all of which see a NaN: 71 us instead of 65.)
template <typename T, int HD, int NW, int QG, int BN, bool OWN_KEYS, int TERMS, int MODE, bool AGAIN>
MI355_DEVINL bool sweep_rows(const Args& p, u32x4* lds, Joined<NW, 16 * QG>* join, const unsigned block, const int pass) {
  constexpr int RING = OWN_KEYS ? 1 : 2;
  using frag = typename Mfma<T>::frag;
  typedef T frag4 __attribute__((ext_vector_type(4)));
  static_assert(HD % 16 == 0 && BN % 32 == 0, "shape");
  constexpr int QW = 16 * QG, BM = OWN_KEYS ? QW : NW * QW;
  constexpr int LW = OWN_KEYS ? 1 : NW;  // waves that load a tile
  constexpr int NCH = HD / 8, ROWB = HD * 2;
  // MFMA steps of S^T, 32 elements each; of HD 16, 48 and 80 the last one's upper half is zeros in both
  // operands. (A 16x16x16 MFMA for it, accumulating onto the 16x16x32 right before it, lost two of its four
  // results: the compiler leaves no wait states between the two.)
  constexpr int KS = (HD + 31) / 32;
  constexpr bool HALF = HD % 32 != 0;
  constexpr int DT = HD / 16, KT = BN / 16;
  static_assert(BN * NCH % 64 == 0, "whole blocks of loads");
  constexpr int BLK = BN * NCH / 64, LPW = (BLK + LW - 1) / LW, TILE = BN * NCH;

  int tid = threadIdx.x;
  if constexpr (AGAIN) asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;

  // the work-group's rows [row0, nrows) of a sequence (or of the batch), its K/V head and keys
  int h, row0, nrows, k_begin, k_end, k_off, split = 0, b = 0;
  const T *Qb, *Kb, *Vb;
  int64_t out_tok = 0, slot = -1;
  if constexpr (MODE == PACKED) {
    const int entry = quotient(static_cast<int>(block), p.by_Hkv);
    h = static_cast<int>(block) - entry * p.Hkv;
    const PackedTile t = p.tiles[entry];
    row0 = t.row0;
    nrows = t.q_len * p.G;
    k_begin = t.k_begin;
    // key j is seen by token i when j < i + k_off (causal), j < k_len
    k_off = p.causal ? t.k_len - t.q_len + 1 : 0x40000000;
    const int last = (row0 + BM < nrows ? row0 + BM : nrows) - 1;
    const int lim = quotient(last, p.by_G) + k_off;
    k_end = lim < t.k_stop ? lim : t.k_stop;
    k_end = k_end > k_begin ? k_end : k_begin;
    if (t.slot >= 0) slot = h * p.slots + t.slot;
    Qb = static_cast<const T*>(p.q) + t.q0 * p.qt;
    Kb = static_cast<const T*>(p.k) + t.k0 * p.kt + h * p.kh;
    Vb = static_cast<const T*>(p.v) + t.k0 * p.vt + h * p.vh;
    out_tok = t.q0;
  } else if constexpr (MODE == WHOLE) {
    b = quotient(static_cast<int>(block), p.by_Hkv);
    h = static_cast<int>(block) - b * p.Hkv;
    row0 = k_begin = 0;
    nrows = p.n_q * p.G;
    const int given = p.lens[b];
    k_end = given < 0 ? 0 : (given < p.keys ? given : p.keys);
    k_off = k_end - p.n_q + 1;
    Qb = static_cast<const T*>(p.q) + b * p.qb;
    Kb = static_cast<const T*>(p.k) + b * p.kb + h * p.kh;
    Vb = static_cast<const T*>(p.v) + b * p.vb + h * p.vh;
  } else {
    const int x = quotient(static_cast<int>(block), p.by_Hkv), y = quotient(x, p.by_splits);
    h = static_cast<int>(block) - x * p.Hkv;
    split = x - y * p.splits;
    b = quotient(y, p.by_row_tiles);
    row0 = (y - b * p.row_tiles) * BM;
    k_begin = split * p.chunk;
    Qb = static_cast<const T*>(p.q);
    Kb = static_cast<const T*>(p.k) + h * p.kh;
    Vb = static_cast<const T*>(p.v) + h * p.vh;
    int len = p.keys;
    if constexpr (MODE == OWN) {
      nrows = p.n_q * p.G;
      const int given = p.lens[b];
      len = given < 0 ? 0 : (given < p.keys ? given : p.keys);
      k_off = len - p.n_q + 1;
      Qb += b * p.qb;
      Kb += b * p.kb;
      Vb += b * p.vb;
    } else {
      nrows = p.B * p.n_q * p.G;
      k_off = 0x40000000;
    }
    if (k_begin >= len) return false;  // (the combining kernel does not read this split)
    k_end = k_begin + p.chunk < len ? k_begin + p.chunk : len;
  }
  Kb = uniform_ptr(Kb + static_cast<int64_t>(k_begin) * p.kt);
  Vb = uniform_ptr(Vb + static_cast<int64_t>(k_begin) * p.vt);
  int n_keys = __builtin_amdgcn_readfirstlane(k_end - k_begin);  // keys from here on are counted from k_begin
  k_off = __builtin_amdgcn_readfirstlane(k_off);
  int64_t kt = p.kt, vt = p.vt;
  const int row_w = OWN_KEYS ? row0 : row0 + wave * QW;
  const int lwave = OWN_KEYS ? 0 : wave;
  if constexpr (OWN_KEYS) lds += wave * 2 * TILE;
  const bool idle = row_w >= nrows;    // no row of this wave is real: it only loads

  // token (of the batch in PREFIX) of a row, and its offset in q
  const auto q_of = [&](int r) MI355_LAMBDA_INLINE {
    const int t = quotient(r, p.by_G), hh = h * p.G + (r - t * p.G);
    if constexpr (MODE == PREFIX) {
      const int bb = quotient(t, p.by_n_q);
      return bb * p.qb + (t - bb * p.n_q) * p.qt + hh * p.qh;
    } else {
      return t * p.qt + hh * p.qh;
    }
  };
  // keys [0, lim) of the work-group's range are seen by row r
  int lim_off = k_off - k_begin;
  const auto lim_of = [&](int r) MI355_LAMBDA_INLINE {
    const int lim = quotient(r, p.by_G) + lim_off;
    return lim < n_keys ? lim : n_keys;
  };

  // row r's output, or its partial result
  const bool direct = MODE == WHOLE || (MODE == PACKED && slot < 0);
  const auto out_of = [&](int r) MI355_LAMBDA_INLINE {
    const int t = quotient(r, p.by_G), hh = h * p.G + (r - t * p.G);
    return static_cast<T*>(p.o) + (MODE == WHOLE ? b * p.ob : out_tok * p.ot) + t * p.ot + hh * p.oh;
  };
  const auto part_of = [&](int r) MI355_LAMBDA_INLINE {
    if constexpr (MODE == PACKED) {
      return slot + (r - row0);
    } else {
      const int t = quotient(r, p.by_G), hh = h * p.G + (r - t * p.G);
      return (static_cast<int64_t>(p.part0 + split) * p.B * p.n_q + (MODE == OWN ? static_cast<int64_t>(b) * p.n_q : 0) + t) * p.H + hh;
    }
  };

  // Q^T fragments: lane (row l16 of group n, slice g) holds elements 32 s + 8 g ..
  frag qf[QG][KS];
  const bool upper = HALF && g >= 2;
  const auto lower_half = [&](u32x4 v) MI355_LAMBDA_INLINE { return upper ? u32x4{0u, 0u, 0u, 0u} : v; };
#pragma unroll
  for (int n = 0; n < QG; ++n) {
    const int r = row_w + 16 * n + l16;
    const bool real = r < nrows;
    const T* src = Qb + q_of(real ? r : nrows - 1);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bool half = HALF && s == KS - 1;
      const u32x4 v = *reinterpret_cast<const u32x4*>(src + 32 * s + 8 * (half ? g & 1 : g));
      qf[n][s] = __builtin_bit_cast(frag, half ? lower_half(v) : v);
    }
  }
  // What the sweep over the keys goes by. Loads: lane i of block blk lands at chunk 64 blk + i of the tile,
  // so it fetches the logical chunk that the swizzle places there; rows past the last key read as zeros.
  int lim[QG], lim_first, lim_last;
  uint32_t kstride, vstride, kcap, vcap, koff[LPW], voff[LPW];
  const auto bind = [&]() MI355_LAMBDA_INLINE {
#pragma unroll
    for (int n = 0; n < QG; ++n) lim[n] = lim_of(row_w + 16 * n + l16 < nrows ? row_w + 16 * n + l16 : nrows - 1);
    lim_first = MODE == PREFIX ? n_keys : __builtin_amdgcn_readfirstlane(lim[0]);
    lim_last = MODE == PREFIX ? n_keys : lim_of(row_w + QW - 1 < nrows ? row_w + QW - 1 : nrows - 1);
    kstride = static_cast<uint32_t>(kt) * sizeof(T);
    vstride = static_cast<uint32_t>(vt) * sizeof(T);
    kcap = 0xffffffffu / kstride;
    vcap = 0xffffffffu / vstride;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int at = (lwave + i * LW) * 64 + lane, row = at / NCH, ch = (at % NCH) ^ swz<NCH>(row);
      koff[i] = static_cast<uint32_t>(row) * kstride + ch * 16;
      voff[i] = static_cast<uint32_t>(row) * vstride + ch * 16;
    }
  };
  // WHOLE: the prefix in the place of the cache, and back
  const T *const own_k = Kb, *const own_v = Vb;
  const int own_keys = n_keys;
  const auto bind_part = [&](int part) MI355_LAMBDA_INLINE {
    if constexpr (MODE == WHOLE) {
      const T* pk = uniform_ptr(static_cast<const T*>(p.pk) + h * p.pkh);
      const T* pv = uniform_ptr(static_cast<const T*>(p.pv) + h * p.pvh);
      Kb = part == 0 ? pk : own_k;
      Vb = part == 0 ? pv : own_v;
      n_keys = part == 0 ? p.pkeys : own_keys;
      kt = part == 0 ? p.pkt : p.kt;
      vt = part == 0 ? p.pvt : p.vt;
      lim_off = part == 0 ? 0x40000000 : k_off;
    }
    bind();
  };
  auto issue_k = [&](int j, int st) MI355_LAMBDA_INLINE {
    const uint32_t key = static_cast<uint32_t>(j) * BN, rem = static_cast<uint32_t>(n_keys) - key;
    const u32x4 kr = buffer_rsrc(reinterpret_cast<const char*>(Kb) + static_cast<uint64_t>(key) * kstride,
                                 rem > kcap ? 0xffffffffu : rem * kstride);
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int blk = lwave + i * LW;
      if (BLK % LW != 0 && blk >= BLK) break;
      const uint32_t to = lds_addr_of(&lds[st * TILE + blk * 64]);
      if (OWN_KEYS && i == 0) buffer_dma_lds16_after_valu(kr, koff[i], to);
      else buffer_dma_lds16(kr, koff[i], 0, to);
    }
  };
  auto issue_v = [&](int j, int st) MI355_LAMBDA_INLINE {
    const uint32_t key = static_cast<uint32_t>(j) * BN, rem = static_cast<uint32_t>(n_keys) - key;
    const u32x4 vr = buffer_rsrc(reinterpret_cast<const char*>(Vb) + static_cast<uint64_t>(key) * vstride,
                                 rem > vcap ? 0xffffffffu : rem * vstride);
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int blk = lwave + i * LW;
      if (BLK % LW != 0 && blk >= BLK) break;
      const uint32_t to = lds_addr_of(&lds[(RING + st) * TILE + blk * 64]);
      if (OWN_KEYS && i == 0) buffer_dma_lds16_after_valu(vr, voff[i], to);
      else buffer_dma_lds16(vr, voff[i], 0, to);
    }
  };

  // byte offsets of a lane's fragments in a tile; what the swizzle makes non-additive in registers
  constexpr int KV = NCH % 16 == 0 ? 4 : NCH % 8 == 0 ? 2 : 1;
  constexpr int VV = NCH % 16 == 0 ? 8 : NCH % 8 == 0 ? 4 : NCH % 4 == 0 ? 2 : 1;
  const char* const ldsb = reinterpret_cast<const char*>(lds);
  uint32_t k_at[KV], v_at[VV];
  const int ve = (lane >> 2) & 3, vq = lane & 3;
#pragma unroll
  for (int i = 0; i < KV; ++i) k_at[i] = l16 * ROWB + ((4 * i + g) ^ swz<NCH>(l16)) * 16;
#pragma unroll
  for (int i = 0; i < VV; ++i)
    v_at[i] = (4 * g + ve) * ROWB + ((2 * i + (vq >> 1)) ^ swz<NCH>(4 * g + ve)) * 16 + (vq & 1) * 8;
  auto kfrag = [&](int st, int kt, int s) MI355_LAMBDA_INLINE {
    if (HALF && s == KS - 1)  // (rows of 2, 6, 10 chunks: no swizzle)
      return __builtin_bit_cast(frag, lower_half(*reinterpret_cast<const u32x4*>(
          ldsb + st * TILE * 16 + (16 * kt + l16) * ROWB + s * 64 + (g & 1) * 16)));
    return __builtin_bit_cast(frag, *reinterpret_cast<const u32x4*>(
        ldsb + st * TILE * 16 + 16 * kt * ROWB + s / KV * (KV * 64) + k_at[s % KV]));
  };
  auto vfrag = [&](int st, int t, int dt) MI355_LAMBDA_INLINE {
    const char* base = ldsb + (RING + st) * TILE * 16 + 32 * t * ROWB + dt / VV * (VV * 32) + v_at[dt % VV];
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(base));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(base + 16 * ROWB));
    return __builtin_bit_cast(frag, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  };

  f32x4 o[QG][DT];
  float top[QG], gate[QG], lsum[QG];  // running max, the score (log2 domain) that moves it, row sum
  uint32_t far = 0;                   // bit n: a row of group n has had a maximum of FAR or more

  constexpr bool F16 = std::is_same_v<T, _Float16>;
  constexpr uint32_t LOWEST = 0x00010001u << (F16 ? 10 : 7), EXP = 0x80008000u - LOWEST, ONES = F16 ? 0x3c003c00u : 0x3f803f80u;
  const auto all_ones = [](uint32_t sign) MI355_LAMBDA_INLINE { return (sign >> 15 & 0x00010001u) * 0xffffu; };
  // halves of all ones where an exponent has all bits set: adding the lowest carries into the sign's place
  const auto not_finite = [&](uint32_t w) MI355_LAMBDA_INLINE { return all_ones((w & EXP) + LOWEST); };
  // this wave's part of a tile as `pass` has it, K and V
  const auto pass_k = [&](int st) MI355_LAMBDA_INLINE {
#pragma nounroll
    for (int blk = lwave; blk < BLK && pass > CLEAN; blk += LW) lds[st * TILE + 64 * blk + lane] = u32x4{0u, 0u, 0u, 0u};
  };
  const auto pass_v = [&](int st) MI355_LAMBDA_INLINE {
#pragma nounroll
    for (int blk = lwave; blk < BLK; blk += LW) {
      u32x4 w = lds[(RING + st) * TILE + 64 * blk + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t bad = not_finite(w[e]), nan = all_ones((w[e] & (LOWEST - 0x00010001u)) + 0x7fff7fffu);
        const uint32_t one = bad & (nan | (pass == UP ? ~all_ones(w[e]) : all_ones(w[e])));
        w[e] = pass == CLEAN ? w[e] & ~bad : one & ONES;
      }
      lds[(RING + st) * TILE + 64 * blk + lane] = w;
    }
  };

  // scores_done: the tile's K has been read; need_v: its V is about to be
  auto tile = [&](const int j, const int st, auto&& scores_done, auto&& need_v) MI355_LAMBDA_INLINE {
    const int k0 = j * BN;
    f32x4 s[QG][KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int n = 0; n < QG; ++n) s[n][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const frag kf = kfrag(st, kt, x);
#pragma unroll
        for (int n = 0; n < QG; ++n) s[n][kt] = mma32(kf, qf[n][x], s[n][kt]);
      }
    }
    scores_done();
    if (k0 + BN > lim_first) {  // the tile crosses a row's last key
#pragma unroll
      for (int n = 0; n < QG; ++n) {
        const int rel = lim[n] - k0 - 4 * g;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * kt + i >= rel) s[n][kt][i] = NEG_INF;
      }
    }
#pragma unroll
    for (int n = 0; n < QG; ++n) {
      float mx = s[n][0][0];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = vmax(mx, s[n][kt][i]);
      if (__builtin_amdgcn_ballot_w64(mx * p.c > gate[n]) != 0) {
        mx = row_maximum(mx);
        const bool grow = mx * p.c > gate[n];
        const float t2 = grow ? mx : top[n];
        const float m1 = top[n] * p.c, m2 = t2 * p.c;
        const bool far1 = __builtin_fabsf(m1) >= FAR, far2 = __builtin_fabsf(m2) >= FAR;
        if (__builtin_amdgcn_ballot_w64(far2) != 0) far |= 1u << n;
        if (__builtin_amdgcn_ballot_w64(gate[n] != NEG_INF) != 0) {  // (sums and outputs are 0 before the first maximum)
          float by = m1 - m2;
          if ((far >> n) & 1)
            by = far1 ? (far2 ? (top[n] - t2) * p.c : __builtin_fmaf(top[n], p.c, -m2)) : far2 ? __builtin_fmaf(-t2, p.c, m1) : by;
          const float alpha = gate[n] == NEG_INF ? 1.f : fast_exp2(by);
          lsum[n] *= alpha;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][t][i] *= alpha;
        }
        top[n] = t2;
        gate[n] = grow ? mx * p.c + 8.f : gate[n];
      }
    }
    float mu[QG];
#pragma unroll
    for (int n = 0; n < QG; ++n) {
      mu[n] = top[n] * p.c;
      if ((far >> n) & 1) {  // rows whose maximum is: it is taken off before the product
        const bool is = __builtin_fabsf(mu[n]) >= FAR;
        const float off = is ? top[n] : 0.f;
        mu[n] = is ? 0.f : mu[n];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][kt][i] -= off;
      }
    }
    frag pf[TERMS][QG][KT / 2];
#pragma unroll
    for (int t = 0; t < KT / 2; ++t)
#pragma unroll
      for (int n = 0; n < QG; ++n) {
        float e[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          e[r] = fast_exp2(__builtin_fmaf(s[n][2 * t + r / 4][r % 4], p.c, -mu[n]));
          if constexpr (TERMS == 1) pf[0][n][t][r] = from_f32<T>(e[r]);
        }
        if constexpr (TERMS == 2) {
          two_terms(e, pf[0][n][t], pf[1][n][t]);
          lsum[n] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        } else {
          lsum[n] = prob_sum(pf[0][n][t], lsum[n]);
        }
      }
    need_v();
#pragma unroll
    for (int t = 0; t < KT / 2; ++t)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const frag vf = vfrag(st, t, dt);
#pragma unroll
        for (int n = 0; n < QG; ++n)
#pragma unroll
          for (int x = 0; x < TERMS; ++x) o[n][dt] = mma32(vf, pf[x][n][t], o[n][dt]);
      }
  };

  const auto sweep = [&]() MI355_LAMBDA_INLINE {
#pragma unroll
    for (int n = 0; n < QG; ++n) {
#pragma unroll
      for (int t = 0; t < DT; ++t) o[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      top[n] = 0.f;
      gate[n] = NEG_INF;
      lsum[n] = 0.f;
    }
    far = 0;
    if constexpr (OWN_KEYS) {
      // K of the next tile is requested as soon as this one's has been read, V likewise, so that one of
      // them is always in flight: of the 2 LPW newest loads the older LPW have to be there.
      static_assert(LPW < 64, "vmcnt");
      constexpr int OLDER = (LPW & 15) | (LPW >> 4) << 14 | 7 << 4 | 15 << 8;  // vmcnt(LPW)
      constexpr int READ = 15 | 3 << 14 | 7 << 4;                              // lgkmcnt(0)
      for (int part = MODE == WHOLE ? 0 : 1; part < 2; ++part) {
        bind_part(part);
        const int n_kt = (n_keys + BN - 1) / BN;
        const int n_mine = n_kt < (lim_last + BN - 1) / BN ? n_kt : (lim_last + BN - 1) / BN;
        if (wave < n_mine) {
          issue_k(wave, 0);
          issue_v(wave, 0);
        }
        for (int j = wave; j < n_mine; j += NW) {
          const bool more = j + NW < n_mine;
          __builtin_amdgcn_s_waitcnt(OLDER);
          if constexpr (AGAIN) pass_k(0);
          tile(j, 0,
               [&]() MI355_LAMBDA_INLINE {
                 __builtin_amdgcn_s_waitcnt(READ);
                 if (more) issue_k(j + NW, 0);
               },
               [&]() MI355_LAMBDA_INLINE {
                 if (more) __builtin_amdgcn_s_waitcnt(OLDER);
                 else __builtin_amdgcn_s_waitcnt(0);
                 if constexpr (AGAIN) pass_v(0);
               });
          __builtin_amdgcn_s_waitcnt(READ);
          if (more) issue_v(j + NW, 0);
        }
      }
    } else {
      bind();
      const int n_kt = (n_keys + BN - 1) / BN;
      const auto issue = [&](int j, int st) MI355_LAMBDA_INLINE {
        issue_k(j, st);
        issue_v(j, st);
      };
      const auto nothing = []() MI355_LAMBDA_INLINE {};
      if (n_kt > 0) issue(0, 0);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      auto step = [&](const int j, const int st) MI355_LAMBDA_INLINE {
        if (j + 1 < n_kt) issue(j + 1, st ^ 1);
        if constexpr (AGAIN) {
          pass_k(st);
          pass_v(st);
          __syncthreads();
        }
        if (!idle && j * BN < lim_last) tile(j, st, nothing, nothing);
        // this wave's loads of tile j + 1 have landed and its reads of tile j are done
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
      };
      int j = 0;
      for (; j + 2 <= n_kt; j += 2) {
        step(j, 0);
        step(j + 1, 1);
      }
      if (j < n_kt) step(j, 0);
    }
  };

  // 4 elements of a row whose output (or partial result) starts at dst (part); whether one is NaN
  const auto put = [&](T* dst, float* part, int d, f32x4 v, float inv, bool sees, bool& nan) MI355_LAMBDA_INLINE {
    frag4* const out = reinterpret_cast<frag4*>(dst + d);
    f32x4* const some = reinterpret_cast<f32x4*>(part + d);
    if (AGAIN && pass > CLEAN) {
      const float add = pass == UP ? -NEG_INF : NEG_INF;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (v[e] == 0.f || (direct && !sees)) continue;
        if (direct) (*out)[e] = from_f32<T>(to_f32((*out)[e]) + add);
        else (*some)[e] += add;
      }
      return;
    }
    if (direct) {
      // no key seen: zeros; keys seen, all with a score of -inf: 0 / 0, as softmax's
      frag4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = sees ? v[e] * inv : 0.f;
        w[e] = from_f32<T>(v[e]);
      }
      *out = w;
    } else {
      *some = v;
    }
    if constexpr (MODE != PREFIX && !AGAIN) {
      const float m = vmax(vmax(v[0], v[1]), vmax(v[2], v[3]));
      nan |= m != m;
    }
  };
  const auto put_ml = [&](int r, float m, float sum) MI355_LAMBDA_INLINE {
    if (direct || AGAIN) return;
    const int64_t at = part_of(r);
    p.ml[2 * at] = m;
    p.ml[2 * at + 1] = sum;
  };
  // writes what the sweep has left; whether there is a NaN among what this thread wrote
  const auto results = [&]() MI355_LAMBDA_INLINE {
    bool nan = false;
    if constexpr (OWN_KEYS) {
      // The waves' rows meet in LDS: each wave's outputs where its tiles were, its maxima and sums beside.
      static_assert(QW * HD * 4 <= 2 * TILE * 16, "a wave's outputs fit its tiles");
      f32x4* const mine = reinterpret_cast<f32x4*>(lds);
#pragma unroll
      for (int n = 0; n < QG; ++n) {
        const float sum = row_sum(lsum[n]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) mine[(16 * n + l16) * (HD / 4) + 4 * dt + g] = o[n][dt];
        if (g == 0) {
          // (a sum that is not 0 without a maximum is NaN's)
          join->ml[wave][16 * n + l16][0] = gate[n] == NEG_INF && sum == 0.f ? NEG_INF : top[n] * p.c;
          join->ml[wave][16 * n + l16][1] = sum;
        }
      }
      __syncthreads();
      const f32x4* const all = reinterpret_cast<const f32x4*>(lds - wave * 2 * TILE);
      const int real = nrows - row0 < QW ? nrows - row0 : QW;
      for (int at = tid; at < real * (HD / 4); at += NW * 64) {
        const int x = at / (HD / 4), d = at % (HD / 4);
        float m = NEG_INF, sum = 0.f;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) m = vmax(m, join->ml[w][x][0]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float mw = join->ml[w][x][0];
          if (mw == NEG_INF) continue;  // no finite score there
          const float f = fast_exp2(mw - m);
          sum = __builtin_fmaf(join->ml[w][x][1], f, sum);
          const f32x4 ow = all[w * 2 * TILE + x * (HD / 4) + d];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(ow[e], f, v[e]);
        }
        T* const dst = direct ? out_of(row0 + x) : nullptr;
        float* const part = direct ? nullptr : p.part + part_of(row0 + x) * HD;
        put(dst, part, 4 * d, v, 1.0f / sum, lim_of(row0 + x) > 0 || (MODE == WHOLE && p.pkeys > 0), nan);
        if (d == 0) put_ml(row0 + x, m, sum);
      }
    } else {
      // each lane holds runs of 4 of its row's elements
#pragma unroll
      for (int n = 0; n < QG; ++n) {
        const int r = row_w + 16 * n + l16;
        const float sum = row_sum(lsum[n]);
        if (r < nrows) {
          T* const dst = direct ? out_of(r) : nullptr;
          float* const part = direct ? nullptr : p.part + part_of(r) * HD;
          const float inv = 1.0f / sum;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) put(dst, part, 16 * dt + 4 * g, o[n][dt], inv, lim[n] > 0, nan);
          if (g == 0) put_ml(r, gate[n] == NEG_INF && sum == 0.f ? NEG_INF : top[n] * p.c, sum);
        }
      }
    }
    return nan;
  };
  // Whether any thread of the work-group says so; nothing but LDS is waited for, the outputs above are still on their
  // way. (Where the waves share tiles, those have all been read.)
  const auto any_wave = [&](bool mine) MI355_LAMBDA_INLINE {
    uint32_t* const flags = OWN_KEYS ? join->flags : reinterpret_cast<uint32_t*>(lds);
    const bool any = __builtin_amdgcn_ballot_w64(mine) != 0;
    if (lane == 0) flags[wave] = any;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) all |= flags[w];
    return __builtin_amdgcn_readfirstlane(all) != 0;
  };
  // keys that every row sees; from there on (of the work-group's keys) those that only some do
  const int first = lim_of(row0) > 0 ? lim_of(row0) : 0;
  if (AGAIN && pass == CLEAN) {
    bool leak = false;
    for (int at = tid; at < (n_keys - first) * NCH; at += NW * 64) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(Vb + (first + at / NCH) * vt + at % NCH * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) leak |= not_finite(w[e]) != 0;
    }
    if (!any_wave(leak)) return false;
    __syncthreads();  // the flags have been read
  }
  sweep();
  const bool nan = results();
  if constexpr (AGAIN) return pass < DOWN;
  return MODE != PREFIX && first < n_keys && any_wave(nan);
}

// ... from its kernel's arguments, ARGS bytes of which come before p
template <typename T, int HD, int NW, int QG, int BN, bool OWN_KEYS, int TERMS, int MODE, int ARGS = 0>
MI355_DEVINL void attn_rows(const Args& p, u32x4* lds, const unsigned block) {
  __shared__ Joined<NW, 16 * QG> own_join;
  Joined<NW, 16 * QG>* const join = OWN_KEYS ? &own_join : nullptr;
  bool more = sweep_rows<T, HD, NW, QG, BN, OWN_KEYS, TERMS, MODE, false>(p, lds, join, block, GIVEN);
  if constexpr (MODE != PREFIX) {
#pragma nounroll
    for (int pass = CLEAN; more; ++pass) {
      __syncthreads();  // what the waves have in LDS has been read
      // The arguments once more from memory: the compiler would keep all that the sweeps share in registers throughout.
      auto args = reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr());
      unsigned same = block;
      asm volatile("" : "+s"(args), "+s"(same));
      struct Words { uint64_t v[sizeof(Args) / 8]; } words;
      static_assert(sizeof(words) == sizeof(Args), "8-byte words");
#pragma unroll
      for (size_t i = 0; i < sizeof(Args) / 8; ++i)
        words.v[i] = reinterpret_cast<const __attribute__((address_space(4))) uint64_t*>(args + ARGS)[i];
      more = sweep_rows<T, HD, NW, QG, BN, OWN_KEYS, TERMS, MODE, true>(__builtin_bit_cast(Args, words), lds, join, same, pass);
    }
  }
}

}  // namespace rows

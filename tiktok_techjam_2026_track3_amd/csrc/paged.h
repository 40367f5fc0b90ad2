// A K/V cache in pages, held in e4m3 with one scale for each block of 16 tokens and head, and the batch of sequences
// that lives in it: what paged_append.hip writes and attn_paged.hip reads.
//
//   K, V     [pages][kv_heads][page][head_dim] bytes   token p of a sequence: row p % page of page table[b][p / page]
//   scales   [pages][kv_heads][page / 16] fp32, powers of two   value = scale * e4m3
//
// Pages are head-major, so that a head's 16 tokens are one run of 16 head_dim bytes. Power-of-two scales cost e4m3
// nothing (its steps are relative) and make what happens when a later token raises its block's scale exact: bytes move
// to smaller exponents, and only those that fall below e4m3's least normal value are rounded again.
#pragma once

#include "common.h"

namespace paged {

constexpr int BLOCK = 16;  // tokens that share a scale: the rows of one 16x16x32 MFMA operand

struct Cache {
  uint8_t *k, *v;
  float *ks, *vs;
  int32_t pages, kv_heads, head_dim;
  int32_t page_shift;  // page = 2^page_shift tokens
};

// Sequences of a batch and their newest tokens. Everything that is read on the device is checked there: no value of
// it makes an access leave its tensor.
struct Batch {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;     // tokens in the cache, the new ones among them, last
  const int32_t* offsets;  // [B + 1] first new token of each sequence; NULL: sequence b's are b * most ..
  int32_t B, width, most, tokens;
};

struct Sequence {
  int32_t first, n;  // its new tokens are first .. first + n
  int32_t len;       // tokens with them
  int32_t cut;       // rows behind them that the offsets give it beyond `most`: left out, as if len did not count them either
};

MI355_DEVINL Sequence sequence_of(const Batch& p, int b) {
  Sequence s;
  s.len = p.lens[b];
  if (p.offsets == nullptr) {
    s.first = b * p.most;
    s.n = p.most;
    s.cut = 0;
  } else {
    const int lo = p.offsets[b], hi = p.offsets[b + 1];
    s.first = lo < 0 ? 0 : (lo < p.tokens ? lo : p.tokens);
    const int end = hi < s.first ? s.first : (hi < p.tokens ? hi : p.tokens);
    s.n = end - s.first < p.most ? end - s.first : p.most;
    s.cut = end - s.first - s.n;
    s.len = s.len < -0x7fffffff + s.cut ? -0x7fffffff : s.len - s.cut;
  }
  return s;
}

// Rows that no sequence has, of a new output: those behind the last one's, those before the first one's, and what is cut
// off each. First of those behind:
MI355_DEVINL int64_t tail_of(const Batch& p) {
  if (p.offsets == nullptr) return static_cast<int64_t>(p.B) * p.most;
  const int end = p.offsets[p.B];
  return end < 0 ? 0 : end;
}

// Zeros (zero(t), by all lanes of a wave) for the rows [from, to) that no sequence has, shared out by the waves of `workers`
// work-groups of 256. Offsets that decrease may have given them to another sequence, so each row is looked for.
template <typename Zero>
MI355_DEVINL void zero_rows(const Batch& p, int64_t from, int64_t to, int64_t worker, int64_t workers, Zero zero) {
  const int lane = threadIdx.x & 63;
  for (int64_t t = from + 4 * worker + (threadIdx.x >> 6); t < to; t += 4 * workers) {
    bool has = false;
    for (int b = lane; b < p.B && !has; b += 64) {
      const Sequence s = sequence_of(p, b);
      has = t >= s.first && t - s.first < s.n;
    }
    if (__ballot(has) == 0) zero(t);
  }
}

// The sizes of a call, as both entry points take them.
struct Sizes {
  int64_t B, most, tokens, heads, kv_heads, head_dim, pages, page, width, table_stride;
};

// What both refuse.
inline int check(int dtype, const Sizes& z) {
  const auto [B, most, tokens, heads, kv_heads, head_dim, pages, page, width, table_stride] = z;
  if (dtype != MI355_F16 && dtype != MI355_BF16) return MI355_E_BAD_DTYPE;
  switch (head_dim) {
    case 16: case 32: case 48: case 64: case 80: case 96: case 128: case 192: case 256: break;
    default: return MI355_E_HEAD_DIM;
  }
  constexpr int64_t MOST = int64_t(1) << 30;
  for (const int64_t n : {B, most, tokens, pages, width, table_stride})
    if (n < 0 || n >= MOST) return MI355_E_BAD_SIZE;
  if (B > (1 << 20) || heads < 1 || heads > 65535 || kv_heads < 1 || heads % kv_heads) return MI355_E_BAD_SIZE;
  if (page < BLOCK || page > 1024 || (page & (page - 1)) || width * page >= MOST) return MI355_E_BAD_SIZE;
  return MI355_OK;
}

inline Cache cache_of(const Sizes& z, const uint8_t* k, const uint8_t* v, const float* ks, const float* vs) {
  return Cache{const_cast<uint8_t*>(k), const_cast<uint8_t*>(v), const_cast<float*>(ks), const_cast<float*>(vs),
               static_cast<int32_t>(z.pages), static_cast<int32_t>(z.kv_heads), static_cast<int32_t>(z.head_dim),
               __builtin_ctzll(static_cast<uint64_t>(z.page))};
}

inline Batch batch_of(const Sizes& z, const int32_t* table, const int32_t* lens, const int32_t* offsets) {
  return Batch{table, z.table_stride, lens, offsets, static_cast<int32_t>(z.B), static_cast<int32_t>(z.width),
               static_cast<int32_t>(z.most), static_cast<int32_t>(z.tokens)};
}

}  // namespace paged

// Attention of each sequence's newest tokens over its pages of an e4m3 cache (paged.h), heads grouped:
//   O[i, h] = sum_j softmax_j(scale Q[i, h] · K[j, h / G]) V[j, h / G],  j <= the token's own position.
//
// Rows = (token, query head of a K/V head's group), 16 to a group. A wave takes its keys 32 at a time, straight from
// memory into registers, without LDS:
//   S^T = K · Q^T on 16x16x32 MFMAs. A lane (key l % 16, slice g = l / 16) loads 16 bytes of its key and converts them,
//     two to an instruction, into the type of q: exact, e4m3 has 4 significant bits. The scale of the block multiplies
//     the scores in fp32. Which dims make up an MFMA's 32 is free as long as Q is read alike: 64 c + 16 g + ..
//   O^T += V^T · P^T: the scores of 32 keys leave a lane with those of its row at keys 4 g + i and 16 + 4 g + i, which
//     is a P^T operand as it is. For V^T a lane loads the run of dims that it has of the same eight keys; byte pairs of
//     two keys are put together (v_perm) and converted. Output row m of MFMA e is dim m * run + e: a free choice again.
// A probability times its block's V scale is split into two bf16 terms, off by at most 2^-16 of it; V is exact in bf16
// whatever the type of q, so fp16 needs no range for scales. Statistics and sums are fp32.
// Four waves share a range of keys and are joined through LDS; ranges of a sequence are joined by a second launch.
#include "paged.h"

namespace {

using paged::BLOCK;

constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float LOG2E = 1.4426950408889634f;
constexpr int64_t MIN_CHUNK = 256;  // least keys of a work-group's range

struct PagedArgs {
  paged::Cache cache;
  paged::Batch batch;
  const void* q;
  void* o;
  int64_t qt, qh, ot, oh;
  float scale;
  int32_t heads, G, row_tiles;
  int32_t target;    // work-groups to aim at
  int32_t zero_tail, split;
  int64_t slots;     // partial rows that the workspace has
  float* part;       // [work-group][rows][head_dim], unnormalised
  float* ml;         // [work-group][rows]{maximum, sum}
};

MI355_DEVINL f32x4 mma32(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
MI355_DEVINL f32x4 mma32(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
MI355_DEVINL float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// reductions over the four lanes l, l ^ 16, l ^ 32, l ^ 48 of a row
MI355_DEVINL float row_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
MI355_DEVINL float row_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// e4m3 bytes 2 word, 2 word + 1 of w as two elements, exactly
template <typename T, bool WORD>
MI355_DEVINL uint32_t two_of(uint32_t w) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, WORD));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, WORD));
}

// 0x80 in each byte of w that is a NaN, one bit lower ones aside
MI355_DEVINL uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// How a batch's keys are shared out: `chunk` keys to a work-group.
struct Shares {
  int chunk, index, b;  // range `index` of sequence b
  int first;            // ranges of the sequences before b
};

MI355_DEVINL int keys_of(const PagedArgs& p, int b) {  // keys that exist of a sequence
  const int64_t room = static_cast<int64_t>(p.batch.width) << p.cache.page_shift;
  const int len = p.batch.lens[b];
  return len < 0 ? 0 : (len < room ? len : static_cast<int>(room));
}

MI355_DEVINL int ranges_of(int keys, int chunk) { return keys > chunk ? (keys + chunk - 1) / chunk : 1; }

// Keys to a range: those of the batch, times its row tiles and heads, over the work-groups aimed at; whole steps of
// 128 (32 for each wave).
MI355_DEVINL int chunk_of(const PagedArgs& p, int lane) {
  if (!p.split) return 0x7fffffff;
  int64_t sum = 0;
  for (int b0 = 0; b0 < p.batch.B; b0 += 64) sum += b0 + lane < p.batch.B ? keys_of(p, b0 + lane) : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
  int64_t chunk = (sum * p.row_tiles * p.cache.kv_heads + p.target - 1) / p.target;
  chunk = (chunk + 127) & ~int64_t(127);
  chunk = chunk < MIN_CHUNK ? MIN_CHUNK : chunk;
  return chunk < 0x40000000 ? static_cast<int>(chunk) : 0x40000000;
}

// The sequence that range x of the whole batch belongs to; b = -1: there is none.
MI355_DEVINL Shares share_of(const PagedArgs& p, int x, int lane) {
  Shares s{chunk_of(p, lane), 0, -1, 0};
  if (!p.split) {
    s.b = x < p.batch.B ? x : -1;
    s.first = x;
    return s;
  }
  int before = 0;
  for (int b0 = 0; b0 < p.batch.B; b0 += 64) {
    const int mine = b0 + lane < p.batch.B ? ranges_of(keys_of(p, b0 + lane), s.chunk) : 0;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off);
      if (lane >= off) upto += v;
    }
    const uint64_t hit = __ballot(x < before + upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      s.b = b0 + l;
      s.first = before + __builtin_amdgcn_readlane(upto - mine, l);
      s.index = x - s.first;
      return s;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return s;
}

// DW: dwords that a lane has of a V row, head_dim / 64 rounded up to 1, 2, 3 or 4 (dims behind head_dim are loaded from
// its start: Q is 0 there, and those output rows are not stored). NR: groups of 16 rows.
template <typename T, int DW, int NR>
__global__ __launch_bounds__(256) void attn_paged_few(PagedArgs p) {
  using frag = typename Mfma<T>::frag;
  constexpr int DP = 64 * DW, KS = 2 * DW, ME = 4 * DW, ROWS = 16 * NR;
  __shared__ float lds_o[2][ROWS * DP];
  __shared__ float lds_ml[4][ROWS][2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const int hd = p.cache.head_dim, G = p.G;
  const int kvh = p.cache.kv_heads;

  // the work-group's head, row tile and range
  const int w = blockIdx.x;
  const int h = w % kvh, tile = (w / kvh) % p.row_tiles;
  const Shares share = share_of(p, w / kvh / p.row_tiles, lane);
  if (share.b < 0) return;
  const int b = __builtin_amdgcn_readfirstlane(share.b);
  const paged::Sequence s = paged::sequence_of(p.batch, b);
  if (p.zero_tail && b == p.batch.B - 1 && share.index == 0 && tile == 0) {  // rows that no sequence has
    for (int64_t t = s.first + s.n; t < p.batch.tokens; ++t)
      for (int i = tid; i < G * hd; i += 256)
        static_cast<T*>(p.o)[t * p.ot + (h * G + i / hd) * p.oh + i % hd] = T(0.0f);
  }
  const int row0 = tile * ROWS, nrows = s.n * G;
  if (row0 >= nrows) return;
  const int keys = keys_of(p, b);
  const int ranges = ranges_of(keys, share.chunk);
  // token i of the n sees positions up to len - n + i; lim(r): how many keys row r sees, were there room for all
  const int64_t see0 = static_cast<int64_t>(s.len) - s.n + 1;
  const auto lim = [&](int r) MI355_LAMBDA_INLINE {
    const int64_t n = see0 + r / G;
    return static_cast<int>(n < 0 ? 0 : n);
  };
  const int last = row0 + ROWS < nrows ? row0 + ROWS - 1 : nrows - 1;
  const int sees = lim(last) < keys ? lim(last) : keys;  // by the tile's last row
  const int fewest = lim(row0);                          // by its first
  const int64_t range0 = static_cast<int64_t>(share.index) * share.chunk;
  const int64_t range1 = range0 + share.chunk < sees ? range0 + share.chunk : sees;
  // the wave's keys: a quarter of the range, in whole units of 32
  const int64_t quarter = ranges > 1 ? share.chunk / 4 : ((sees + 127) / 128) * 32;
  const int k0 = __builtin_amdgcn_readfirstlane(static_cast<int>(range0 + wave * quarter < range1 ? range0 + wave * quarter : range1));
  const int k1 = __builtin_amdgcn_readfirstlane(static_cast<int>(range0 + (wave + 1) * quarter < range1 ? range0 + (wave + 1) * quarter : range1));

  frag qf[NR][KS];
  int limit[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = row0 + 16 * n + l16 < nrows ? row0 + 16 * n + l16 : nrows - 1;
    limit[n] = lim(r);
    const int t = r / G;
    const T* src = static_cast<const T*>(p.q) + (s.first + static_cast<int64_t>(t)) * p.qt + (h * G + r - t * G) * p.qh;
#pragma unroll
    for (int c = 0; c < DW; ++c) {
      const int d = 64 * c + 16 * g;
      const bool real = d < hd;
      const u32x4 a = *reinterpret_cast<const u32x4*>(src + (real ? d : 0));
      const u32x4 z = *reinterpret_cast<const u32x4*>(src + (real ? d + 8 : 0));
      qf[n][2 * c] = __builtin_bit_cast(frag, real ? a : u32x4{0u, 0u, 0u, 0u});
      qf[n][2 * c + 1] = __builtin_bit_cast(frag, real ? z : u32x4{0u, 0u, 0u, 0u});
    }
  }

  f32x4 acc[NR][ME];
  float top[NR], sum[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    top[n] = NEG_INF;
    sum[n] = 0.0f;
#pragma unroll
    for (int e = 0; e < ME; ++e) acc[n][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // offsets within a block of 16 keys
  uint32_t k_at[DW], v_at[4];
#pragma unroll
  for (int c = 0; c < DW; ++c) k_at[c] = l16 * hd + (64 * c + 16 * g < hd ? 64 * c + 16 * g : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) v_at[i] = (4 * g + i) * hd + (l16 * 4 * DW < hd ? l16 * 4 * DW : 0);

  struct Unit {
    u32x4 k[2][DW];
    uint32_t v[2][4][DW];
  };

  // lane l knows block l of a window of 64: its page, and the factors of its scores and V (a page that does not
  // exist: NaN for the rows that see its keys, and page 0 is read in its place)
  int page = 0;
  float kf = 0.0f, vf = 1.0f;
  const auto window = [&](int from) MI355_LAMBDA_INLINE {
    const int at = from + lane * BLOCK;
    page = 0;
    kf = 0.0f;
    vf = 1.0f;
    if (at < k1) {
      const int id = p.batch.table[b * p.batch.table_stride + (at >> p.cache.page_shift)];
      const bool ok = id >= 0 && id < p.cache.pages;
      page = ok ? id : 0;
      const int64_t si = ((static_cast<int64_t>(page) * kvh + h) << (p.cache.page_shift - 4)) + ((at & ((1 << p.cache.page_shift) - 1)) >> 4);
      kf = ok ? p.cache.ks[si] * p.scale : __builtin_nanf("");
      vf = ok ? p.cache.vs[si] : 1.0f;
    }
  };
  const auto block_at = [&](int at, int l) MI355_LAMBDA_INLINE {  // byte offset of the block at key `at`, lane l's
    const int id = __builtin_amdgcn_readlane(page, l);
    return (((static_cast<int64_t>(id) * kvh + h) << p.cache.page_shift) + (at & ((1 << p.cache.page_shift) - 1))) * hd;
  };
  const auto load = [&](Unit& u, int at, int l) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t base = block_at(at + BLOCK * t, l + t);
      const uint8_t* kb = p.cache.k + base;
      const uint8_t* vb = p.cache.v + base;
#pragma unroll
      for (int c = 0; c < DW; ++c) u.k[t][c] = *reinterpret_cast<const u32x4*>(kb + k_at[c]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DW; ++c) u.v[t][i][c] = *reinterpret_cast<const uint32_t*>(vb + v_at[i] + 4 * c);
    }
  };
  const auto compute = [&](Unit& u, int at, int l) MI355_LAMBDA_INLINE {
    f32x4 sc[NR][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int n = 0; n < NR; ++n) sc[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < DW; ++c) {
        const u32x4 x = u.k[t][c];
        const u32x4 lo = {two_of<T, false>(x[0]), two_of<T, true>(x[0]), two_of<T, false>(x[1]), two_of<T, true>(x[1])};
        const u32x4 hi = {two_of<T, false>(x[2]), two_of<T, true>(x[2]), two_of<T, false>(x[3]), two_of<T, true>(x[3])};
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          sc[n][t] = mma32(__builtin_bit_cast(frag, lo), qf[n][2 * c], sc[n][t]);
          sc[n][t] = mma32(__builtin_bit_cast(frag, hi), qf[n][2 * c + 1], sc[n][t]);
        }
      }
    }
    const float kf2[2] = {__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kf), l)),
                          __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kf), l + 1))};
    const float vf2[2] = {__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vf), l)),
                          __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vf), l + 1))};
    const bool partial = at + 32 > fewest || at + 32 > k1;  // some row does not see all of the keys
    bool nans = false;
    uint32_t is_nan[2][4][DW];
    if (partial) {
      // Keys that no row sees: V to zeros. NaN in V that only some rows see: to zeros as well, and back below.
      bool mine = false;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool seen = at + BLOCK * t + 4 * g + i < k1;
#pragma unroll
          for (int c = 0; c < DW; ++c) {
            u.v[t][i][c] = seen ? u.v[t][i][c] : 0u;
            is_nan[t][i][c] = nan_bytes(u.v[t][i][c]);
            mine = mine || is_nan[t][i][c] != 0;
          }
        }
      nans = __ballot(mine) != 0;
      if (nans) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < DW; ++c) u.v[t][i][c] &= ~((is_nan[t][i][c] >> 7) * 0xffu);
      }
    }
    bf16x8 hi[NR], lo[NR], seen_by[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float x[8], most = NEG_INF;
#pragma unroll
      for (int r = 0; r < 8; ++r) x[r] = sc[n][r >> 2][r & 3] * kf2[r >> 2];
      if (partial) {
        const int stop = limit[n] < k1 ? limit[n] : k1;
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = at + BLOCK * (r >> 2) + 4 * g + (r & 3) < stop ? x[r] : NEG_INF;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) most = fmaxf(most, x[r]);
      // the maximum moves only when a score exceeds it by more than 5 (natural units: probabilities up to 2^7.3)
      if (__ballot(most > top[n] + 5.0f)) {
        const float now = fmaxf(top[n], row_max(most));
        const float keep = top[n] == NEG_INF ? 0.0f : fast_exp2((top[n] - now) * LOG2E);
        top[n] = now;
        sum[n] *= keep;
#pragma unroll
        for (int e = 0; e < ME; ++e) acc[n][e] *= keep;
      }
      const float ref = top[n] == NEG_INF ? 0.0f : top[n];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float e = fast_exp2((x[r] - ref) * LOG2E);
        sum[n] += e;
        e *= vf2[r >> 2];
        if (partial) {
          const int stop = limit[n] < k1 ? limit[n] : k1;
          const bool seen = at + BLOCK * (r >> 2) + 4 * g + (r & 3) < stop;
          e = seen ? e : 0.0f;
          seen_by[n][r] = static_cast<__bf16>(seen ? 1.0f : 0.0f);
        }
        const float cut = __uint_as_float(__float_as_uint(e) & 0xffff0000u);
        hi[n][r] = static_cast<__bf16>(cut);
        lo[n][r] = static_cast<__bf16>(e - cut);
      }
    }
    const auto pairs_of = [&](const uint32_t (&a)[2][4][DW], int c, int half, int t, int i) MI355_LAMBDA_INLINE {
      return __builtin_amdgcn_perm(a[t][i + 1][c], a[t][i][c], half ? 0x07030602u : 0x05010400u);
    };
#pragma unroll
    for (int c = 0; c < DW; ++c)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pr[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) pr[k] = pairs_of(u.v, c, half, k >> 1, (k & 1) * 2);
        const u32x4 even = {two_of<__bf16, false>(pr[0]), two_of<__bf16, false>(pr[1]), two_of<__bf16, false>(pr[2]), two_of<__bf16, false>(pr[3])};
        const u32x4 odd = {two_of<__bf16, true>(pr[0]), two_of<__bf16, true>(pr[1]), two_of<__bf16, true>(pr[2]), two_of<__bf16, true>(pr[3])};
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          f32x4& a0 = acc[n][4 * c + 2 * half];
          f32x4& a1 = acc[n][4 * c + 2 * half + 1];
          a0 = mma32(__builtin_bit_cast(bf16x8, even), hi[n], a0);
          a1 = mma32(__builtin_bit_cast(bf16x8, odd), hi[n], a1);
          a0 = mma32(__builtin_bit_cast(bf16x8, even), lo[n], a0);
          a1 = mma32(__builtin_bit_cast(bf16x8, odd), lo[n], a1);
        }
      }
    if (nans) {  // outputs that a NaN reaches: counts of those that a row sees, in each dim
#pragma unroll
      for (int c = 0; c < DW; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pr[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) pr[k] = pairs_of(is_nan, c, half, k >> 1, (k & 1) * 2);
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            u32x4 one;  // 1.0 where the byte is set
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t w2 = odd ? pr[k] >> 16 : pr[k];
              one[k] = ((w2 >> 7) & 1) * 0x3f80u | ((w2 >> 15) & 1) * 0x3f800000u;
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              const f32x4 hits = mma32(__builtin_bit_cast(bf16x8, one), seen_by[n], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int i = 0; i < 4; ++i)
                acc[n][4 * c + 2 * half + odd][i] = hits[i] > 0.0f ? __builtin_nanf("") : acc[n][4 * c + 2 * half + odd][i];
            }
          }
        }
    }
  };

  for (int from = k0; from < k1; from += 64 * BLOCK) {
    window(from);
    const int stop = k1 < from + 64 * BLOCK ? k1 : from + 64 * BLOCK;
    Unit one, two;
    load(one, from, 0);
    for (int at = from; at < stop; at += 64) {
      const int l = (at - from) >> 4;
      if (at + 32 < stop) load(two, at + 32, l + 2);
      compute(one, at, l);
      if (at + 32 >= stop) break;
      if (at + 64 < stop) load(one, at + 64, l + 4);
      compute(two, at + 32, l + 2);
    }
  }

  // the four waves' results: factors of a row from their maxima, then pairs of waves added up in LDS
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    sum[n] = row_sum(sum[n]);
    if (g == 0) {
      lds_ml[wave][16 * n + l16][0] = top[n];
      lds_ml[wave][16 * n + l16][1] = sum[n];
    }
  }
  __syncthreads();
  float all_top[NR], all_sum[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float m = NEG_INF;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, lds_ml[k][16 * n + l16][0]);
    const auto factor = [&](float t) MI355_LAMBDA_INLINE { return t == NEG_INF ? 1.0f : fast_exp2((t - m) * LOG2E); };
    float z = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) z += lds_ml[k][16 * n + l16][1] * factor(lds_ml[k][16 * n + l16][0]);
    all_top[n] = m;
    all_sum[n] = z;
    const float f = factor(top[n]);
#pragma unroll
    for (int e = 0; e < ME; ++e) acc[n][e] *= f;
  }
  const auto put = [&](float* dst) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < ME; ++e) *reinterpret_cast<f32x4*>(dst + ((n * ME + e) * 64 + lane) * 4) = acc[n][e];
  };
  const auto add = [&](const float* src) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < ME; ++e) acc[n][e] += *reinterpret_cast<const f32x4*>(src + ((n * ME + e) * 64 + lane) * 4);
  };
  if (wave >= 2) put(lds_o[wave - 2]);
  __syncthreads();
  if (wave < 2) add(lds_o[wave]);
  __syncthreads();
  if (wave == 1) put(lds_o[0]);
  __syncthreads();
  if (wave != 0) return;
  add(lds_o[0]);

  // lane (row l16, g) has dims 16 DW g + 4 DW i + e of its row
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int r = row0 + 16 * n + l16;
    if (r >= nrows) continue;
    if (ranges > 1) {
      const int64_t at = static_cast<int64_t>(w) * ROWS + 16 * n + l16;
      if (g == 0) {
        p.ml[2 * at] = all_top[n];
        p.ml[2 * at + 1] = all_sum[n];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * DW * g + 4 * DW * i;
        if (d < hd)
#pragma unroll
          for (int c = 0; c < DW; ++c)
            *reinterpret_cast<f32x4*>(p.part + at * hd + d + 4 * c) =
                f32x4{acc[n][4 * c][i], acc[n][4 * c + 1][i], acc[n][4 * c + 2][i], acc[n][4 * c + 3][i]};
      }
    } else {
      // no key: zeros; keys whose scores were all -inf, and keys behind the table's end: NaN
      float inv = all_sum[n] > 0.0f ? 1.0f / all_sum[n] : (all_sum[n] == 0.0f && limit[n] == 0 ? 0.0f : __builtin_nanf(""));
      if (limit[n] > keys) inv = __builtin_nanf("");
      const int t = r / G;
      T* dst = static_cast<T*>(p.o) + (s.first + static_cast<int64_t>(t)) * p.ot + (h * G + r - t * G) * p.oh;
      typedef T V4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 16 * DW * g + 4 * DW * i;
        if (d < hd)
#pragma unroll
          for (int c = 0; c < DW; ++c)
            *reinterpret_cast<V4*>(dst + d + 4 * c) =
                V4{from_f32<T>(acc[n][4 * c][i] * inv), from_f32<T>(acc[n][4 * c + 1][i] * inv),
                   from_f32<T>(acc[n][4 * c + 2][i] * inv), from_f32<T>(acc[n][4 * c + 3][i] * inv)};
      }
    }
  }
}

// Joins the ranges of the sequences that have several: a work-group for each row (token, head).
template <typename T>
__global__ __launch_bounds__(256) void attn_paged_join(PagedArgs p, int rows_of_tile) {
  __shared__ float lds[8 * 256];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kvh = p.cache.kv_heads, hd = p.cache.head_dim, G = p.G;
  const int head = blockIdx.x % p.heads, i = (blockIdx.x / p.heads) % p.batch.most, b = blockIdx.x / p.heads / p.batch.most;
  const int keys = keys_of(p, b);
  const int chunk = chunk_of(p, lane);
  const int ranges = ranges_of(keys, chunk);
  if (ranges == 1) return;
  const paged::Sequence s = paged::sequence_of(p.batch, b);
  if (i >= s.n) return;
  int64_t first = 0;
  for (int b0 = 0; b0 < b; b0 += 64) first += b0 + lane < b ? ranges_of(keys_of(p, b0 + lane), chunk) : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) first += __shfl_xor(first, off);
  const int h = head / G, r = i * G + head - h * G, tile = r / rows_of_tile;
  // ranges that the tile's last row reaches have partial results; the others' are zeros without keys
  const auto slot = [&](int c) MI355_LAMBDA_INLINE {  // (in the workspace, whatever lens has become since)
    const int64_t at = (((first + c) * p.row_tiles + tile) * kvh + h) * rows_of_tile + (r - tile * rows_of_tile);
    return at < p.slots ? at : p.slots - 1;
  };
  float m = NEG_INF;
  for (int c = lane; c < ranges; c += 64) m = fmaxf(m, p.ml[2 * slot(c)]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  const auto factor = [&](float t) MI355_LAMBDA_INLINE { return t == NEG_INF ? 1.0f : fast_exp2((t - m) * LOG2E); };
  float z = 0.0f;
  for (int c = lane; c < ranges; c += 64) z += p.ml[2 * slot(c) + 1] * factor(p.ml[2 * slot(c)]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) z += __shfl_xor(z, off);
  // quarters of dims side by side, eight groups of 32 threads walk the ranges
  const int quads = hd / 4, grp = tid >> 5, q0 = tid & 31;
  for (int q = q0; q < quads; q += 32) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int c = grp; c < ranges; c += 8) {
      const int64_t at = slot(c);
      a += *reinterpret_cast<const f32x4*>(p.part + at * hd + 4 * q) * factor(p.ml[2 * at]);
    }
    *reinterpret_cast<f32x4*>(lds + grp * 256 + 4 * q) = a;
  }
  __syncthreads();
  const int64_t sees = static_cast<int64_t>(s.len) - s.n + i + 1;
  float inv = z > 0.0f ? 1.0f / z : (z == 0.0f && sees <= 0 ? 0.0f : __builtin_nanf(""));
  if (sees > keys) inv = __builtin_nanf("");
  for (int d = tid; d < hd; d += 256) {
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) a += lds[k * 256 + d];
    static_cast<T*>(p.o)[(s.first + static_cast<int64_t>(i)) * p.ot + head * p.oh + d] = from_f32<T>(a * inv);
  }
}

struct Launch {
  int nr;              // groups of 16 rows
  int64_t row_tiles, target, grid, ws;
  bool split;
};

Launch launch_of(int64_t B, int64_t most, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t width, int64_t page) {
  Launch l{};
  const int64_t rows = most * (heads / kv_heads);
  // two groups of 16 rows at head dims whose outputs leave registers for them
  l.nr = rows > 16 && head_dim <= 128 ? 2 : 1;
  l.row_tiles = (rows + 16 * l.nr - 1) / (16 * l.nr);
  l.target = 4 * 256;  // work-groups: four a CU
  l.split = width * page > MIN_CHUNK;
  const int64_t whole = B * l.row_tiles * kv_heads;
  l.grid = whole + (l.split ? l.target : 0);
  l.ws = l.split ? l.grid * 16 * l.nr * (head_dim + 2) * 4 : 0;
  return l;
}

template <typename T, int DW>
int launch_rows(const PagedArgs& p, const Launch& l, hipStream_t s) {
  const uint32_t grid = static_cast<uint32_t>(l.grid);
  if constexpr (DW <= 2) {
    if (l.nr == 2)
      attn_paged_few<T, DW, 2><<<grid, 256, 0, s>>>(p);
    else
      attn_paged_few<T, DW, 1><<<grid, 256, 0, s>>>(p);
  } else {
    attn_paged_few<T, DW, 1><<<grid, 256, 0, s>>>(p);
  }
  if (const hipError_t e = hipGetLastError(); e != hipSuccess) return static_cast<int>(e);
  if (!l.split) return MI355_OK;
  attn_paged_join<T><<<static_cast<uint32_t>(p.heads) * p.batch.most * p.batch.B, 256, 0, s>>>(p, 16 * l.nr);
  return static_cast<int>(hipGetLastError());
}

template <typename T>
int launch_dim(const PagedArgs& p, const Launch& l, hipStream_t s) {
  switch ((p.cache.head_dim + 63) / 64) {
    case 1: return launch_rows<T, 1>(p, l, s);
    case 2: return launch_rows<T, 2>(p, l, s);
    case 3: return launch_rows<T, 3>(p, l, s);
    default: return launch_rows<T, 4>(p, l, s);
  }
}

int check_all(int dtype, int64_t B, int64_t most, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
              int64_t pages, int64_t page, int64_t width) {
  if (const int st = paged::check(dtype, B, most, tokens, heads, kv_heads, head_dim, pages, page, width)) return st;
  if (B * most >= (int64_t(1) << 30) || B * most * heads >= (int64_t(1) << 23)) return MI355_E_BAD_SIZE;  // 2^31 threads
  return MI355_OK;
}

}  // namespace

extern "C" int64_t mi355_attn_paged_workspace_bytes(int64_t B, int64_t most, int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim, int64_t page, int64_t width) {
  if (const int st = check_all(MI355_F16, B, most, 0, heads, kv_heads, head_dim, 0, page, width)) return st;
  return launch_of(B, most, heads, kv_heads, head_dim, width, page).ws;
}

extern "C" int mi355_attn_paged(int dtype, const void* Q, const uint8_t* cache_k, const uint8_t* cache_v,
                                const float* k_scale, const float* v_scale, const int32_t* table, int64_t table_stride,
                                const int32_t* lens, const int32_t* offsets, void* O, int64_t B, int64_t most,
                                int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                int64_t page, int64_t width, const int64_t* q_strides, const int64_t* o_strides,
                                float scale, int zero_tail, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int st = check_all(dtype, B, most, tokens, heads, kv_heads, head_dim, pages, page, width)) return st;
  if (B * most == 0 || tokens == 0) return MI355_OK;
  if (!Q || !O || !lens || !q_strides || !o_strides || !cache_k || !cache_v || !k_scale || !v_scale || (width > 0 && !table))
    return MI355_E_NULL_POINTER;
  if (pages < 1) return MI355_E_BAD_SIZE;
  if (!offsets && B * most > tokens) return MI355_E_BAD_SIZE;
  if (!(scale > 0.0f) || scale > 1e30f) return MI355_E_UNSUPPORTED;
  if (!aligned16(Q) || (reinterpret_cast<uintptr_t>(O) & 7u) || !aligned16(cache_k) || !aligned16(cache_v) ||
      q_strides[0] % 8 || q_strides[1] % 8 || o_strides[0] % 4 || o_strides[1] % 4)
    return MI355_E_ALIGNMENT;
  const Launch l = launch_of(B, most, heads, kv_heads, head_dim, width, page);
  if (l.ws > 0 && (!workspace || workspace_bytes < l.ws || !aligned16(workspace))) return MI355_E_BAD_SIZE;
  PagedArgs p{};
  p.cache = paged::Cache{const_cast<uint8_t*>(cache_k), const_cast<uint8_t*>(cache_v), const_cast<float*>(k_scale),
                         const_cast<float*>(v_scale), static_cast<int32_t>(pages), static_cast<int32_t>(kv_heads),
                         static_cast<int32_t>(head_dim), __builtin_ctzll(static_cast<uint64_t>(page))};
  p.batch = paged::Batch{table, table_stride, lens, offsets, static_cast<int32_t>(B), static_cast<int32_t>(width),
                         static_cast<int32_t>(most), static_cast<int32_t>(tokens)};
  p.q = Q;
  p.o = O;
  p.qt = q_strides[0];
  p.qh = q_strides[1];
  p.ot = o_strides[0];
  p.oh = o_strides[1];
  p.scale = scale;
  p.heads = static_cast<int32_t>(heads);
  p.G = static_cast<int32_t>(heads / kv_heads);
  p.row_tiles = static_cast<int32_t>(l.row_tiles);
  p.target = static_cast<int32_t>(l.target);
  p.zero_tail = zero_tail;
  p.split = l.split;
  p.slots = l.ws ? l.grid * 16 * l.nr : 0;
  p.part = static_cast<float*>(workspace);
  p.ml = p.part + (l.ws ? l.grid * 16 * l.nr * head_dim : 0);
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == MI355_F16 ? launch_dim<_Float16>(p, l, s) : launch_dim<__bf16>(p, l, s);
}

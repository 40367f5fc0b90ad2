// Attention of each sequence's newest tokens over its pages of an e4m3 cache (paged.h), heads grouped:
//   O[i, h] = sum_j softmax_j(scale Q[i, h] · K[j, h / G]) V[j, h / G],  j <= the token's own position.
//
// Rows = (token, query head of a K/V head's group), 16 to a group. A wave takes its keys 32 at a time. Up to 32 rows
// (Few) K and V go straight from memory into registers, more rows (Many) share what is converted through LDS:
//   S^T = K · Q^T on 16x16x32 MFMAs. A lane (key l % 16, slice g = l / 16) loads 16 bytes of its key and converts them,
//     two to an instruction, into the type of q: exact, e4m3 has 4 significant bits. The scale of the block multiplies
//     the scores in fp32. Which dims make up an MFMA's 32 is free as long as Q is read alike: 64 c + 16 g + ..
//     (16x16x128 MFMAs take K's bytes as they come, with q as two or three e4m3 terms; but they do not keep 24 bits of
//     a sum: 2^-14 to 2^-17 of sum |q k| was lost where these lose 2^-24.)
//   O^T += V^T · P^T: the scores of 32 keys leave a lane with those of its row at keys 4 g + i and 16 + 4 g + i, which
//     is a P^T operand as it is. For V^T a lane loads the run of dims that it has of the same eight keys; byte pairs of
//     two keys are put together (v_perm) and converted, the block's scale applied by the conversion. Output row m of
//     MFMA e is dim m * run + e: a free choice again.
// Bound by the bytes of K and V up to 32 rows, by instruction issue (matrix and vector) above.
// The maximum moves only when a score exceeds it by more than 7 (log2 units; LIFT), and only then do the four lanes of a row
// exchange anything. Statistics and sums are fp32.
//
// Work is dealt out evenly: the units of 32 keys of all (sequence, K/V head, tile of rows), in this order, are cut into
// as many equal runs as there are work-groups. A work-group's first and last job may be parts of one; those leave partial
// results, and a second launch joins them. So lengths that differ, and one long sequence, fill the GPU alike.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace {

using paged::BLOCK;

constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 7.0f;
// fp16 probabilities that are rounded once are held as 2^8 times what they are beside the running maximum, which uses the type's
// upper range: those down to 2^-22 of it keep all their bits and 2^-33 is half the smallest step (without: 2^-14 and 2^-25, so
// that what 10000 keys far below a sink weigh together was lost). The factor is in numerator and denominator. They stay
// below 2^15 as the maximum moves at 2^14; a product's rounding to fp32 adds at most 1 to the exponent where it is not FAR.
constexpr float LIFT = 8.0f, LIFTED_SLACK = 14.0f;
// Products of scores and scale so large that fma(s, a, -top) may come out above SLACK by a factor that matters: the
// rounding of top is 2^-24 of it. Then the product is rounded before the difference is taken, like top was.
constexpr float FAR = 0x1p24f;
constexpr int UNIT = 32;

// What a work-group leaves for the second launch: a job whose first part it has.
struct alignas(16) Head {
  paged::Sequence s;
  int32_t h, tile, parts;  // parts: work-groups after it that have more of the job; 0: there is nothing to join
};

struct PagedArgs {
  paged::Cache cache;
  paged::Batch batch;
  const void* q;
  void* o;
  int64_t qt, qh, ot, oh;
  float scale;
  int32_t heads, G;
  int32_t row_tiles;   // tiles of a sequence of `most` tokens
  int32_t groups;      // work-groups that share the work; 0: one for each (sequence, head, tile)
  int32_t least;       // least units of a work-group
  int32_t zero_tail;
  float* part;         // [2 groups][rows][head_dim], unnormalised: of a work-group's first job (0) and last (1)
  float* ml;           // [2 groups][rows]{maximum, sum}
  Head* joins;         // [groups]
};

MI355_DEVINL f32x4 mma32(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
MI355_DEVINL f32x4 mma32(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// IEEE maximum (NaN-propagating): gfx950 v_maximum3_f32, no operand canonicalisation needed
MI355_DEVINL float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
MI355_DEVINL float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// reductions over the four lanes l, l ^ 16, l ^ 32, l ^ 48 of a row
MI355_DEVINL float row_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
MI355_DEVINL float row_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
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

// e4m3 bytes 2 word, 2 word + 1 of w, times a power of two, as two elements
template <typename T, bool WORD>
MI355_DEVINL uint32_t two_of(uint32_t w, float scale) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, WORD));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, WORD));
}

// DW dwords at `at`; AUX: cache policy of the load (0, or PAST: not kept)
constexpr int PAST = 2;
template <int DW, int AUX>
MI355_DEVINL void run_of(uint32_t (&v)[DW], __amdgpu_buffer_rsrc_t src, uint32_t at) {
  if constexpr (DW == 1) {
    v[0] = __builtin_amdgcn_raw_buffer_load_b32(src, at, 0, AUX);
  } else if constexpr (DW == 2) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(src, at, 0, AUX);
    v[0] = x[0], v[1] = x[1];
  } else if constexpr (DW == 3) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b96(src, at, 0, AUX);
    v[0] = x[0], v[1] = x[1], v[2] = x[2];
  } else {
    const auto x = __builtin_amdgcn_raw_buffer_load_b128(src, at, 0, AUX);
    v[0] = x[0], v[1] = x[1], v[2] = x[2], v[3] = x[3];
  }
}

// 0x80 in each byte of w that is a NaN, and w with zeros for those
MI355_DEVINL uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
MI355_DEVINL uint32_t without(uint32_t w, uint32_t nans) { return w & ~((nans >> 7) * 0xffu); }

MI355_DEVINL float lane_of(float v, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l)); }

MI355_DEVINL int keys_of(const PagedArgs& p, int len) {  // keys that exist of a sequence
  const int64_t room = static_cast<int64_t>(p.batch.width) << p.cache.page_shift;
  return len < 0 ? 0 : (len < room ? len : static_cast<int>(room));
}

// A sequence as a job's rows see it.
struct Rows {
  paged::Sequence s;
  int nrows, keys;
  int64_t see0;  // row r sees keys below see0 + r / G, were there room for all
  MI355_DEVINL int lim(int r, int G) const {
    const int64_t n = see0 + r / G;
    return static_cast<int>(n < 0 ? 0 : n);
  }
  // keys that rows below `stop` see
  MI355_DEVINL int sees(int stop, int G) const {
    const int last = lim((stop < nrows ? stop : nrows) - 1, G);
    return last < keys ? last : keys;
  }
  // units of the tile that ends before row `stop`; one where it sees nothing, to write its zeros
  MI355_DEVINL int units(int stop, int G) const {
    const int n = sees(stop, G);
    return n > 0 ? (n + UNIT - 1) / UNIT : 1;
  }
  // What a row's outputs are multiplied by. No key: zeros. Keys whose scores were all -inf, and a key that it sees
  // behind the table's end: NaN.
  MI355_DEVINL float inverse(float sum, int limit) const {
    if (limit > keys) return __builtin_nanf("");
    return sum > 0.0f ? 1.0f / sum : (sum == 0.0f && limit == 0 ? 0.0f : __builtin_nanf(""));
  }
};

MI355_DEVINL Rows rows_of(const PagedArgs& p, paged::Sequence s) {
  Rows r;
  r.s = s;
  r.nrows = s.n * p.G;
  r.keys = keys_of(p, s.len);
  r.see0 = static_cast<int64_t>(s.len) - s.n + 1;
  return r;
}

// Sequence b's, of which lane b of `near` has the numbers if b < 64.
MI355_DEVINL Rows rows_at(const PagedArgs& p, const paged::Sequence& near, int b) {
  if (b >= 64) return rows_of(p, paged::sequence_of(p.batch, b));
  return rows_of(p, paged::Sequence{static_cast<int32_t>(__builtin_amdgcn_readlane(near.first, b)),
                                    static_cast<int32_t>(__builtin_amdgcn_readlane(near.n, b)),
                                    static_cast<int32_t>(__builtin_amdgcn_readlane(near.len, b)), 0});
}

MI355_DEVINL int64_t quotient(int64_t n, int64_t d) {  // of what is not negative, mostly of 32 bits
  if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// units of all tiles of `rows` rows of a sequence, for one head
MI355_DEVINL int64_t all_units(const Rows& r, int rows, int G) {
  int64_t n = 0;
  for (int row0 = 0; row0 < r.nrows; row0 += rows) n += r.units(row0 + rows, G);
  return n;
}

MI355_DEVINL int64_t first_lane(int64_t v) {  // of the wave, in scalar registers
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// Work-groups that a CU's registers hold.
constexpr int per_cu(int64_t dw, int64_t nr, bool many) { return dw > 2 ? 1 : many ? 2 : dw == 1 ? 5 - nr : 4 - nr; }

// A wave's rows: NR groups of 16, their queries, statistics and outputs.
// DW: dwords that a lane has of a V row, head_dim / 64 rounded up to 1, 2, 3 or 4 (dims behind head_dim are loaded from
// its start: Q is 0 there, and those output rows are not stored).
// TERMS: a probability enters P·V as that many. Two bf16 terms, off by at most 2^-16 of it, where K and V are waited for
// and they cost nothing; where rows are many enough to be matrix work, where a second term is as many MFMAs again, one of
// the type of q: half a step of it in numerator and denominator alike (bf16 pieces of prompts 0.0023 of the output's norm off,
// 0.0017 with its rounding alone).
template <typename T, int DW, int NR, int TERMS>
struct Tile {
  using TP = std::conditional_t<TERMS == 1, T, __bf16>;  // type of P and V
  using frag = typename Mfma<T>::frag;
  using pfrag = typename Mfma<TP>::frag;
  static constexpr int KS = 2 * DW, ME = 4 * DW;  // MFMAs of S^T (32 dims each) and of O^T (16) for a group
  static constexpr bool LIFTED = TERMS == 1 && __is_same(T, _Float16);
  static constexpr float GATE = LIFTED ? LIFTED_SLACK : SLACK;  // a score this far above `top` moves it
  typedef T V4 __attribute__((ext_vector_type(4)));

  frag qf[NR][KS];
  int limit[NR];  // keys that the lane's rows see
  f32x4 acc[NR][ME];
  float top[NR], sum[NR];  // top: what probabilities are relative to, in log2 units (the maximum then, less LIFT)
  bool far;                // a row's maximum is

  MI355_DEVINL void start(const PagedArgs& p, const Rows& rows, int h, int row0, int lane) {
    const int l16 = lane & 15, g = lane >> 4, hd = p.cache.head_dim;
    far = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = row0 + 16 * n + l16 < rows.nrows ? row0 + 16 * n + l16 : rows.nrows - 1;
      limit[n] = rows.lim(r, p.G);
      const int t = r / p.G;
      const T* src = static_cast<const T*>(p.q) + (rows.s.first + static_cast<int64_t>(t)) * p.qt + (h * p.G + r - t * p.G) * p.qh;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = 64 * (k >> 1) + 16 * g + 8 * (k & 1);
        const u32x4 v = *reinterpret_cast<const u32x4*>(src + (d < hd ? d : 0));
        qf[n][k] = __builtin_bit_cast(frag, d < hd ? v : u32x4{0u, 0u, 0u, 0u});
      }
      top[n] = NEG_INF;
      sum[n] = 0.0f;
#pragma unroll
      for (int e = 0; e < ME; ++e) acc[n][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // 16 bytes of K as the operands of MFMAs 2 c and 2 c + 1
  static MI355_DEVINL u32x4 k_operand(uint32_t x, uint32_t y) {
    return u32x4{two_of<T, false>(x, 1.0f), two_of<T, true>(x, 1.0f), two_of<T, false>(y, 1.0f), two_of<T, true>(y, 1.0f)};
  }

  // Row n's lane sees key `at` + 16 (r / 4) + 4 g + r % 4 of a unit where that offset less 4 g is below this.
  MI355_DEVINL int seen_below(int n, int at, int k1, int g) const { return (limit[n] < k1 ? limit[n] : k1) - at - 4 * g; }

  // Scores of a unit that some row does not see whole: scaled, -inf where not seen.
  MI355_DEVINL void mask(f32x4 (&sc)[NR][2], float (&a)[2], int at, int k1, int g) const {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int stop = seen_below(n, at, k1, g);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        sc[n][r >> 2][r & 3] = BLOCK * (r >> 2) + (r & 3) < stop ? sc[n][r >> 2][r & 3] * a[r >> 2] : NEG_INF;
    }
    a[0] = a[1] = 1.0f;
  }

  // Probabilities of a unit from its scores (a: their factors, in log2 units), and what they do to the statistics.
  MI355_DEVINL void softmax(const f32x4 (&sc)[NR][2], const float (&a)[2], pfrag (&hi)[NR], pfrag (&lo)[NR]) {
    float most[NR];
    bool moves = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const auto four = [&](const f32x4& x) MI355_LAMBDA_INLINE { return vmax(vmax(vmax(x[0], x[1]), x[2]), x[3]); };
      most[n] = vmax(four(sc[n][0]) * a[0], four(sc[n][1]) * a[1]);
      moves = moves || most[n] - top[n] > GATE;
    }
    if (__ballot(moves)) {  // (a row's statistics are its own: neither this nor `far` is another's to change)
      bool beyond = false;
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float high = row_max(most[n]);
        // (far ones have steps too wide to be lifted exactly)
        const float to = LIFTED && __builtin_fabsf(high) < FAR ? high - LIFT : high;
        const float now = high - top[n] > GATE ? to : top[n];
        const float keep = top[n] == NEG_INF ? 0.0f : fast_exp2(top[n] - now);
        top[n] = now;
        beyond = beyond || (__builtin_fabsf(now) >= FAR && now != NEG_INF);
        sum[n] *= keep;
#pragma unroll
        for (int e = 0; e < ME; ++e) acc[n][e] *= keep;
      }
      far = __ballot(beyond) != 0;
    }
    const auto rest = [&](auto some_far) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float ref = top[n] == NEG_INF ? 0.0f : top[n];
        const bool rounded = decltype(some_far)::value && __builtin_fabsf(ref) >= FAR;
        float e[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float s = sc[n][r >> 2][r & 3], f = a[r >> 2];
          e[r] = fast_exp2(rounded ? s * f - ref : __builtin_fmaf(s, f, -ref));
        }
        if constexpr (TERMS == 1) {
#pragma unroll
          for (int r = 0; r < 8; ++r) hi[n][r] = static_cast<TP>(e[r]);
          sum[n] = prob_sum(hi[n], sum[n]);
        } else {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            sum[n] += e[r];
            const float cut = __uint_as_float(__float_as_uint(e[r]) & 0xffff0000u);
            hi[n][r] = static_cast<TP>(cut);
            lo[n][r] = static_cast<TP>(e[r] - cut);
          }
        }
      }
    };
    if (far)
      rest(std::true_type{});
    else
      rest(std::false_type{});
  }

  // Outputs e: += V^T · P^T
  MI355_DEVINL void add(int e, u32x4 v, const pfrag (&hi)[NR], const pfrag (&lo)[NR]) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      acc[n][e] = mma32(__builtin_bit_cast(pfrag, v), hi[n], acc[n][e]);
      if constexpr (TERMS == 2) acc[n][e] = mma32(__builtin_bit_cast(pfrag, v), lo[n], acc[n][e]);
    }
  }

  // Outputs e of a unit that some row does not see whole, whose V had NaN (zeros by now: 0 · NaN would be NaN in rows that
  // do not see it): NaN where a row sees one. count: V^T with 1 for each. MFMAs count what a row sees.
  MI355_DEVINL void inject(int e, u32x4 count, int at, int k1, int g) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      int stop = seen_below(n, at, k1, g);
      asm volatile("" : "+v"(stop));  // (worked out here, not kept in registers for all e)
      pfrag seen;
#pragma unroll
      for (int r = 0; r < 8; ++r) seen[r] = static_cast<TP>(BLOCK * (r >> 2) + (r & 3) < stop ? 1.0f : 0.0f);
      const f32x4 hits = mma32(__builtin_bit_cast(pfrag, count), seen, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][e][i] += hits[i] > 0.0f ? __builtin_nanf("") : 0.0f;
    }
  }
  // Two elements of V^T with 1 for each NaN, of an output and the next one: from bytes with 0x80 for each, pairs of two keys
  static MI355_DEVINL void count(uint32_t w, uint32_t& even, uint32_t& odd) {
    constexpr uint32_t one = __is_same(TP, _Float16) ? 0x3c00u : 0x3f80u;
    even = ((w >> 7) & 1) * one | ((w >> 15) & 1) * (one << 16);
    odd = ((w >> 23) & 1) * one | (w >> 31) * (one << 16);
  }

  // The rows' outputs, or with slot >= 0 partial results of a tile of `rows_of_tile` rows from `tile0` on. top and
  // sum are the row's. Lane (row l16, g) has dims 16 DW g + 4 DW i + e of its row.
  MI355_DEVINL void write(const PagedArgs& p, const Rows& rows, int h, int row0, int tile0, int rows_of_tile, int64_t slot, int lane) {
    const int l16 = lane & 15, g = lane >> 4, hd = p.cache.head_dim;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = row0 + 16 * n + l16;
      if (r >= rows.nrows) continue;
      if (slot >= 0) {
        const int64_t at = slot * rows_of_tile + (r - tile0);
        if (g == 0) {
          p.ml[2 * at] = top[n];
          p.ml[2 * at + 1] = sum[n];
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
        const float inv = rows.inverse(sum[n], limit[n]);
        const int t = r / p.G;
        T* dst = static_cast<T*>(p.o) + (rows.s.first + static_cast<int64_t>(t)) * p.ot + (h * p.G + r - t * p.G) * p.oh;
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
};

// 64 blocks of a sequence's keys from `from` on, one to a lane: where it is in the pools, and the factors of its scores
// (in log2 units) and V. A page that does not exist: NaN for the rows that see its keys, and page 0 is read in its place. Blocks
// behind `stop`: likewise page 0, with zeros.
struct Window {
  int from;
  uint32_t lo, hi;  // byte offset
  float kf, vf;
  MI355_DEVINL void fill(const PagedArgs& p, int b, int h, int at0, int stop, int lane) {
    const int at = at0 + lane * BLOCK, shift = p.cache.page_shift;
    from = at0;
    int64_t row = 0;
    kf = vf = 0.0f;
    if (at < stop) {
      const int id = p.batch.table[b * p.batch.table_stride + (at >> shift)];
      const bool ok = id >= 0 && id < p.cache.pages;
      row = ((static_cast<int64_t>(ok ? id : 0) * p.cache.kv_heads + h) << shift) + (at & ((1 << shift) - 1));
      kf = ok ? p.cache.ks[row / BLOCK] * (p.scale * LOG2E) : __builtin_nanf("");
      vf = ok ? p.cache.vs[row / BLOCK] : 0.0f;
    }
    row *= p.cache.head_dim;
    lo = static_cast<uint32_t>(row);
    hi = static_cast<uint32_t>(row >> 32);
  }
  MI355_DEVINL int64_t offset(int at) const {
    const int l = (at - from) >> 4;
    const uint64_t a = static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, l)), b = static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, l));
    return static_cast<int64_t>(a | (b << 32));
  }
  // The block with key `at`, of K or V
  MI355_DEVINL __amdgpu_buffer_rsrc_t block(const PagedArgs& p, const uint8_t* pool, int at) const {
    return raw_rsrc(uniform_ptr(pool + offset(at)), BLOCK * p.cache.head_dim);
  }
  MI355_DEVINL float k_factor(int at) const { return lane_of(kf, (at - from) >> 4); }
  MI355_DEVINL float v_factor(int at) const { return lane_of(vf, (at - from) >> 4); }
};

// Up to 16 NR rows: the four waves have the same rows and a quarter of the keys each, and are joined through LDS. K and V
// are waited for; a unit's bytes are requested as soon as the registers of those before it are free. 64 sequences of 0.9k to
// 9k keys (8 K/V heads of 128, 655 MB) 116 us and 5 of the join, 5.4 TB/s in all; 200000 keys of one 71 and 5. Operands
// through LDS or a second unit in flight gave nothing: the bytes on their way already cover the latency.
template <typename T, int DW, int NR, int AUX>
struct Few {
  using Own = Tile<T, DW, NR, 2>;
  using TP = typename Own::TP;
  using pfrag = typename Own::pfrag;
  static constexpr int ME = Own::ME, ROWS = 16 * NR;
  struct Lds {
    float o[2][16 * NR * 64 * DW];
    float ml[4][16 * NR][2];
  };

  // One job, or a part of one: units [u0, u1) of its tile's keys. slot < 0: the rows' outputs, otherwise partial results.
  static MI355_DEVINL void run(const PagedArgs& p, Lds& lds, const Rows& rows, int b, int h, int tile, int u0, int u1,
                               int64_t slot) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, l16 = lane & 15, hd = p.cache.head_dim, row0 = tile * ROWS;
    const int sees = rows.sees(row0 + ROWS, p.G), each = (u1 - u0 + 3) / 4 * UNIT;
    int k1 = u1 * UNIT < sees ? u1 * UNIT : sees, k0 = u0 * UNIT + wave * each;
    k1 = __builtin_amdgcn_readfirstlane(k0 + each < k1 ? k0 + each : k1);
    k0 = __builtin_amdgcn_readfirstlane(k0);
    const int first = rows.lim(row0, p.G), fewest = __builtin_amdgcn_readfirstlane(first < k1 ? first : k1);
    Own own;
    own.start(p, rows, h, row0, lane);

    // offsets within a block of 16 keys
    uint32_t k_at[DW], v_at[4];
#pragma unroll
    for (int c = 0; c < DW; ++c) k_at[c] = l16 * hd + (64 * c + 16 * g < hd ? 64 * c + 16 * g : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) v_at[i] = (4 * g + i) * hd + (l16 * 4 * DW < hd ? l16 * 4 * DW : 0);
    u32x4 ku[2][DW];
    uint32_t vu[2][4][DW];
    float ka[2], va[2];
    Window win;
    const auto load_k = [&](int at) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto src = win.block(p, p.cache.k, at + BLOCK * t);
#pragma unroll
        for (int c = 0; c < DW; ++c) ku[t][c] = __builtin_amdgcn_raw_buffer_load_b128(src, k_at[c], 0, AUX);
        ka[t] = win.k_factor(at + BLOCK * t);
      }
    };
    const auto load_v = [&](int at) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto src = win.block(p, p.cache.v, at + BLOCK * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) run_of<DW, AUX>(vu[t][i], src, v_at[i]);
        va[t] = win.v_factor(at + BLOCK * t);
      }
    };
    // byte pairs of two keys for outputs 4 c + 2 half and the next one
    const auto pair_of = [&](const uint32_t (&v)[2][4][DW], int x, int k) MI355_LAMBDA_INLINE {
      return __builtin_amdgcn_perm(v[k >> 1][(k & 1) * 2 + 1][x >> 1], v[k >> 1][(k & 1) * 2][x >> 1], x & 1 ? 0x07030602u : 0x05010400u);
    };

    for (int w0 = k0; w0 < k1; w0 += 64 * BLOCK) {
      win.fill(p, b, h, w0, k1, lane);
      const int stop = k1 < w0 + 64 * BLOCK ? k1 : w0 + 64 * BLOCK;
      load_k(w0);
      __builtin_amdgcn_sched_barrier(0);  // (K first, as in the loop: it waits for K, not for V)
      load_v(w0);
      __builtin_amdgcn_sched_barrier(0);
      for (int at = w0; at < stop; at += UNIT) {
        const int next = at + UNIT < stop ? at + UNIT : at;
        f32x4 sc[NR][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int n = 0; n < NR; ++n) sc[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2 * DW; ++k) {
            const u32x4 x = Own::k_operand(ku[t][k >> 1][2 * (k & 1)], ku[t][k >> 1][2 * (k & 1) + 1]);
#pragma unroll
            for (int n = 0; n < NR; ++n) sc[n][t] = mma32(__builtin_bit_cast(typename Own::frag, x), own.qf[n][k], sc[n][t]);
          }
        }
        float a[2] = {ka[0], ka[1]};
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        if (at + UNIT > fewest) {  // some row does not see all of the keys
          own.mask(sc, a, at, k1, g);
          uint32_t any = 0;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int c = 0; c < DW; ++c) {
                vu[t][i][c] = BLOCK * t + i < k1 - at - 4 * g ? vu[t][i][c] : 0u;
                any |= nan_bytes(vu[t][i][c]);
              }
          if (__ballot(any != 0)) {
            uint32_t nans[2][4][DW];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < DW; ++c) {
                  nans[t][i][c] = nan_bytes(vu[t][i][c]);
                  vu[t][i][c] = without(vu[t][i][c], nans[t][i][c]);
                }
#pragma unroll
            for (int x = 0; x < 2 * DW; ++x) {
              u32x4 even, odd;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t a2, b2;
                Own::count(pair_of(nans, x, k), a2, b2);
                even[k] = a2;
                odd[k] = b2;
              }
              own.inject(2 * x, even, at, k1, g);
              own.inject(2 * x + 1, odd, at, k1, g);
            }
          }
        }
        pfrag hi[NR], lo[NR];
        own.softmax(sc, a, hi, lo);
#pragma unroll
        for (int x = 0; x < 2 * DW; ++x) {
          u32x4 even, odd;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t pr = pair_of(vu, x, k);
            even[k] = two_of<TP, false>(pr, va[k >> 1]);
            odd[k] = two_of<TP, true>(pr, va[k >> 1]);
          }
          own.add(2 * x, even, hi, lo);
          own.add(2 * x + 1, odd, hi, lo);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(next);
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // the four waves' results: factors of a row from their maxima, then pairs of waves added up in LDS
#pragma unroll
    for (int n = 0; n < NR; ++n) own.sum[n] = row_sum(own.sum[n]);
    if (g == 0)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        lds.ml[wave][16 * n + l16][0] = own.top[n];
        lds.ml[wave][16 * n + l16][1] = own.sum[n];
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float m = NEG_INF;
#pragma unroll
      for (int k = 0; k < 4; ++k) m = fmaxf(m, lds.ml[k][16 * n + l16][0]);
      const auto factor = [&](float t) MI355_LAMBDA_INLINE { return t == NEG_INF ? 1.0f : fast_exp2(t - m); };
      float z = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) z += lds.ml[k][16 * n + l16][1] * factor(lds.ml[k][16 * n + l16][0]);
      const float f = factor(own.top[n]);
      own.top[n] = m;
      own.sum[n] = z;
#pragma unroll
      for (int e = 0; e < ME; ++e) own.acc[n][e] *= f;
    }
    const auto put = [&](float* dst) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < ME; ++e) *reinterpret_cast<f32x4*>(dst + ((n * ME + e) * 64 + lane) * 4) = own.acc[n][e];
    };
    const auto add = [&](const float* src) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < ME; ++e) own.acc[n][e] += *reinterpret_cast<const f32x4*>(src + ((n * ME + e) * 64 + lane) * 4);
    };
    if (wave >= 2) put(lds.o[wave - 2]);
    __syncthreads();
    if (wave < 2) add(lds.o[wave]);
    __syncthreads();
    if (wave == 1) put(lds.o[0]);
    __syncthreads();
    if (wave == 0) add(lds.o[0]);
    __syncthreads();  // (the next job's waves write there again)
    if (wave == 0) own.write(p, rows, h, row0, row0, ROWS, slot, lane);
  }
};

template <int N, typename F>
MI355_DEVINL void for_each(F f) {  // f(0) .. f(N - 1), as constants
  if constexpr (N > 0) {
    for_each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// More rows: each wave has 16 NR of its own. A unit's K and V are converted once for the four of them, a quarter by
// each, into LDS, as the operands that the lanes read: 16 bytes each, one after the other, so without conflicts. Two
// buffers: while unit i is worked on, unit i + 1 is converted and unit i + 3 requested; one barrier a unit. Each wave on its
// own (as in Few) converted all of K and V four times: two pieces of 1024 tokens against 12000 keys (32/8 heads of 128)
// 1039 us, so 350, 14 of them the join: 870 TFLOP/s, matrix cores busy 36% of the time and the vector ALU 48%,
// hardly at once with the two waves that a SIMD's registers hold. The scores of unit i + 1 beside the softmax of unit i (more registers, one wave a SIMD) were slower.
// fp16: V's scales are taken relative to the largest up to their own block, so that V fits the type; blocks down to
// 2^-21 of that are exact. (Up to their own: a later block's scale is not to touch rows that do not see it.)
template <typename T, int DW, int NR>
struct Many {
  using Own = Tile<T, DW, NR, 1>;
  using pfrag = typename Own::pfrag;
  static constexpr int ME = Own::ME, ROWS = 64 * NR;
  static constexpr bool RELATIVE = __is_same(T, _Float16);
  struct Lds {
    u32x4 k[2][4 * DW][64];  // [buffer][MFMA of S^T: (tile of 16 keys, 32 dims)][lane]
    u32x4 v[2][4 * DW][64];  // [buffer][output e][lane]
    u32x4 nans[2][4 * DW][64];  // 1 for each NaN of V, where flag says that a wave found one
    int flag[2][4];
  };
  // A wave's part of a unit: of its 2 DW pieces of K (16 keys, 64 dims) and 2 DW of V (16 keys, four outputs) those with
  // number wave + 4 s, as bytes.
  struct Stage {
    uint32_t r[DW][4];
    float vs[2];
  };

  static MI355_DEVINL void run(const PagedArgs& p, Lds& lds, const Rows& rows, int b, int h, int tile, int u0, int u1,
                               int64_t slot) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, l16 = lane & 15, hd = p.cache.head_dim, row0 = tile * ROWS + wave * 16 * NR;
    const bool active = row0 < rows.nrows;
    const int all = rows.sees(tile * ROWS + ROWS, p.G), k0 = u0 * UNIT;
    const int stop = __builtin_amdgcn_readfirstlane(u1 * UNIT < all ? u1 * UNIT : all);  // keys that any row sees
    const int mine = active ? rows.sees(row0 + 16 * NR, p.G) : 0, first = rows.lim(tile * ROWS, p.G);
    const int k1 = __builtin_amdgcn_readfirstlane(mine < stop ? mine : stop);        // ... that the wave's rows see
    const int all_see = __builtin_amdgcn_readfirstlane(first < stop ? first : stop);  // ... that all rows see
    Own own;
    if (active) own.start(p, rows, h, row0, lane);

    Window win, ahead;  // blocks of the units worked on, and those after them
    // half t of a lane's operand (the keys of tile t)
    const auto put = [&](u32x4 (&to)[64], int t, uint32_t a, uint32_t b) MI355_LAMBDA_INLINE {
      *(reinterpret_cast<u32x2*>(&to[lane]) + t) = u32x2{a, b};
    };
    // whether slot s of a wave is a piece of K: for all waves, none, or the first 2 DW - 4 s
    const auto is_k = [&](auto s) MI355_LAMBDA_INLINE {
      constexpr int left = 2 * DW - 4 * decltype(s)::value;
      return left >= 4 ? true : left <= 0 ? false : wave < left;
    };
    const auto load = [&](Stage& st, int at) MI355_LAMBDA_INLINE {
      const bool now = at - win.from < 64 * BLOCK;
      Window w;
      w.from = now ? win.from : ahead.from;
      w.lo = now ? win.lo : ahead.lo;
      w.hi = now ? win.hi : ahead.hi;
      w.vf = now ? win.vf : ahead.vf;
      for_each<DW>([&](auto s) MI355_LAMBDA_INLINE {
        constexpr int S = decltype(s)::value;
        const int piece = wave + 4 * S;
        if (is_k(s)) {
          const int t = piece / DW, c = piece - t * DW;
          const auto src = w.block(p, p.cache.k, at + BLOCK * t);
          const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(src, l16 * hd + (64 * c + 16 * g < hd ? 64 * c + 16 * g : 0), 0, 0);
          st.r[S][0] = x[0], st.r[S][1] = x[1], st.r[S][2] = x[2], st.r[S][3] = x[3];
        } else {
          const int t = (piece - 2 * DW) / DW, c = piece - 2 * DW - t * DW;
          const auto src = w.block(p, p.cache.v, at + BLOCK * t);
          const uint32_t run = (l16 * 4 * DW < hd ? l16 * 4 * DW : 0) + 4 * c;
          for_each<4>([&](auto i) MI355_LAMBDA_INLINE {
            constexpr int I = decltype(i)::value;
            st.r[S][I] = __builtin_amdgcn_raw_buffer_load_b32(src, (4 * g + I) * hd + run, 0, 0);
          });
        }
      });
      const auto scale = [&](int k) MI355_LAMBDA_INLINE {  // as the conversions take it: the exponent alone
        const float v = w.v_factor(k);
        return RELATIVE ? __uint_as_float(__float_as_uint(v) & 0x7f800000u) : v;
      };
      st.vs[0] = scale(at);
      st.vs[1] = scale(at + BLOCK);
    };
    constexpr float LEAST = 0x1p-118f;  // least scale of a block
    float v_top = LEAST, v_of[2][2] = {}, v_acc = LEAST;  // RELATIVE: largest V scale so far, of the buffers' blocks, of the outputs
    // A unit that goes into buffer `buf`, where some row does not see all of its keys: zeros for V that no row sees and for
    // NaN, whose places are noted.
    const auto sanitize = [&](Stage& st, int at, auto buffer) MI355_LAMBDA_INLINE {
      constexpr int buf = decltype(buffer)::value;
      if (at + UNIT <= all_see) return;
      bool found = false;
      for_each<DW>([&](auto s) MI355_LAMBDA_INLINE {
        constexpr int S = decltype(s)::value;
        if (is_k(s)) return;
        const int piece = wave + 4 * S - 2 * DW, t = piece / DW, e = 4 * (piece - t * DW);
        uint32_t nans[4], any = 0;
        for_each<4>([&](auto i) MI355_LAMBDA_INLINE {
          constexpr int I = decltype(i)::value;
          const uint32_t v = BLOCK * t + I < stop - at - 4 * g ? st.r[S][I] : 0u;
          nans[I] = nan_bytes(v);
          st.r[S][I] = without(v, nans[I]);
          any |= nans[I];
        });
        found = found || __ballot(any != 0) != 0;
        for_each<2>([&](auto half) MI355_LAMBDA_INLINE {
          constexpr int H = decltype(half)::value;
          const uint32_t sel = H ? 0x07030602u : 0x05010400u;
          uint32_t even[2], odd[2];
          Own::count(__builtin_amdgcn_perm(nans[1], nans[0], sel), even[0], odd[0]);
          Own::count(__builtin_amdgcn_perm(nans[3], nans[2], sel), even[1], odd[1]);
          put(lds.nans[buf][e + 2 * H], t, even[0], even[1]);
          put(lds.nans[buf][e + 2 * H + 1], t, odd[0], odd[1]);
        });
      });
      if (lane == 0) lds.flag[buf][wave] = found;
    };
    const auto convert = [&](Stage& st, auto buffer) MI355_LAMBDA_INLINE {
      constexpr int buf = decltype(buffer)::value;
      float vs[2] = {st.vs[0], st.vs[1]};
      if constexpr (RELATIVE) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          v_of[buf][t] = v_top = fmaxf(v_top, vs[t]);
          vs[t] *= __uint_as_float((260u << 23) - __float_as_uint(v_top));  // 64 / v_top: powers of two
        }
      }
      for_each<DW>([&](auto s) MI355_LAMBDA_INLINE {
        constexpr int S = decltype(s)::value;
        int piece = wave + 4 * S;
        if (is_k(s)) {
          lds.k[buf][2 * piece][lane] = Own::k_operand(st.r[S][0], st.r[S][1]);
          lds.k[buf][2 * piece + 1][lane] = Own::k_operand(st.r[S][2], st.r[S][3]);
        } else {
          piece -= 2 * DW;
          const int t = piece / DW, e = 4 * (piece - t * DW);
          const float f = t ? vs[1] : vs[0];
          for_each<2>([&](auto half) MI355_LAMBDA_INLINE {
            constexpr int H = decltype(half)::value;
            const uint32_t sel = H ? 0x07030602u : 0x05010400u;
            const uint32_t a = __builtin_amdgcn_perm(st.r[S][1], st.r[S][0], sel), b = __builtin_amdgcn_perm(st.r[S][3], st.r[S][2], sel);
            put(lds.v[buf][e + 2 * H], t, two_of<T, false>(a, f), two_of<T, false>(b, f));
            put(lds.v[buf][e + 2 * H + 1], t, two_of<T, true>(a, f), two_of<T, true>(b, f));
          });
        }
      });
    };
    const auto barrier = [&]() MI355_LAMBDA_INLINE { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const int n = u1 - u0;
    const auto key = [&](int i) MI355_LAMBDA_INLINE { return k0 + (i < n ? i : n - 1) * UNIT; };
    const auto fence = [&]() MI355_LAMBDA_INLINE { __builtin_amdgcn_sched_barrier(0); };
    // MFMAs with this many of the region's other instructions after each
    const auto spread = [&](auto count, auto others) MI355_LAMBDA_INLINE {
      for_each<decltype(count)::value>([&](auto) MI355_LAMBDA_INLINE {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x6 | 0x200 | 0x20, decltype(others)::value, 0);  // ALU, LDS writes, loads
      });
      fence();
    };
    const auto relative_to = [&](float v) MI355_LAMBDA_INLINE {
      if (v == v_acc) return;
      const float keep = v_acc / v;
      v_acc = v;
#pragma unroll
      for (int m = 0; m < NR; ++m)
#pragma unroll
        for (int e = 0; e < ME; ++e) own.acc[m][e] *= keep;
    };
    u32x4 operand[4 * DW];
    const auto read = [&](const u32x4 (&from)[4 * DW][64]) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int e = 0; e < 4 * DW; ++e) operand[e] = from[e][lane];
      fence();
    };
    // Unit i, and the conversion of unit i + 1 from st. Operands are read well before their MFMAs, K's at once, V's
    // before the softmax; the conversion and the next loads go between the MFMAs.
    const auto step = [&](int i, auto buffer, Stage& st) MI355_LAMBDA_INLINE {
      constexpr int buf = decltype(buffer)::value;
      using Next = std::integral_constant<int, 1 - buf>;
      const int at = k0 + i * UNIT;
      read(lds.k[buf]);
      sanitize(st, key(i + 1), Next{});
      if (at < k1) {
        f32x4 sc[NR][2];
#pragma unroll
        for (int m = 0; m < NR; ++m) sc[m][0] = sc[m][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 2 * DW; ++k)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int m = 0; m < NR; ++m)
              sc[m][t] = mma32(__builtin_bit_cast(typename Own::frag, operand[2 * DW * t + k]), own.qf[m][k], sc[m][t]);
        convert(st, Next{});
        spread(std::integral_constant<int, 4 * DW * NR>{}, std::integral_constant<int, 3>{});
        read(lds.v[buf]);
        float a[2] = {win.k_factor(at), win.k_factor(at + BLOCK)};
        if (at + UNIT > all_see) {
          own.mask(sc, a, at, k1, g);
          if (lds.flag[buf][0] | lds.flag[buf][1] | lds.flag[buf][2] | lds.flag[buf][3])
#pragma unroll
            for (int e = 0; e < ME; ++e) own.inject(e, lds.nans[buf][e][lane], at, k1, g);
        }
        pfrag hi[NR], lo[NR];
        // the SIMD's other wave has its matrix instructions first meanwhile
        __builtin_amdgcn_s_setprio(0);
        own.softmax(sc, a, hi, lo);
        __builtin_amdgcn_s_setprio(1);
        if constexpr (RELATIVE) {
          if (v_of[buf][0] != v_of[buf][1]) {  // the unit's first block has another factor: it comes alone
            relative_to(v_of[buf][0]);
            pfrag one[NR];
#pragma unroll
            for (int m = 0; m < NR; ++m)
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                one[m][r] = r < 4 ? hi[m][r] : T(0.0f);
                hi[m][r] = r < 4 ? T(0.0f) : hi[m][r];
              }
#pragma unroll
            for (int e = 0; e < ME; ++e) own.add(e, operand[e], one, lo);
          }
          relative_to(v_of[buf][1]);
        }
        fence();
#pragma unroll
        for (int e = 0; e < ME; ++e) own.add(e, operand[e], hi, lo);
        load(st, key(i + 3));
        spread(std::integral_constant<int, ME * NR>{}, std::integral_constant<int, 4>{});
      } else {
        convert(st, Next{});
        load(st, key(i + 3));
      }
      barrier();
    };

    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    Stage even, odd;
    win.fill(p, b, h, k0, stop, lane);
    ahead.fill(p, b, h, k0 + 64 * BLOCK, stop, lane);
    load(even, key(0));
    fence();  // (loads stay in order: waits are for the older ones)
    load(odd, key(1));
    fence();
    sanitize(even, key(0), Even{});
    convert(even, Even{});
    load(even, key(2));
    fence();
    barrier();
    for (int i = 0; i < n; i += 2) {
      if (k0 + i * UNIT >= win.from + 64 * BLOCK) {
        win = ahead;
        ahead.fill(p, b, h, win.from + 64 * BLOCK, stop, lane);
      }
      step(i, Even{}, odd);
      if (i + 1 < n) step(i + 1, Odd{}, even);
    }
    if (!active) return;
    if constexpr (RELATIVE) {
      const float back = v_acc / 64.0f;
#pragma unroll
      for (int m = 0; m < NR; ++m)
#pragma unroll
        for (int e = 0; e < ME; ++e) own.acc[m][e] *= back;
    }
#pragma unroll
    for (int m = 0; m < NR; ++m) own.sum[m] = row_sum(own.sum[m]);
    own.write(p, rows, h, row0, tile * ROWS, ROWS, slot, lane);
  }
};

// Zeros for rows that no sequence has, shared out by work-group. i0, step: which elements are the thread's.
template <typename T>
MI355_DEVINL void zero_row(const PagedArgs& p, int64_t t, int i0, int step) {
  for (int i = i0; i < p.heads * p.cache.head_dim; i += step)
    static_cast<T*>(p.o)[t * p.ot + (i / p.cache.head_dim) * p.oh + i % p.cache.head_dim] = T(0.0f);
}
template <typename T>
MI355_DEVINL void zero_behind(const PagedArgs& p) {
  for (int64_t t = paged::tail_of(p.batch) + blockIdx.x; t < p.batch.tokens; t += gridDim.x) zero_row<T>(p, t, threadIdx.x, 256);
}
template <typename T>
MI355_DEVINL void zero_between(const PagedArgs& p, int64_t from, int64_t to, int64_t worker, int64_t workers) {
  paged::zero_rows(p.batch, from, to, worker, workers,
                   [&](int64_t t) MI355_LAMBDA_INLINE { zero_row<T>(p, t, threadIdx.x & 63, 64); });
}
// ... what is before the lanes' sequences, if b0 is 0, or cut off them: sequence b0 + l is lane l's
template <typename T>
MI355_DEVINL void zero_of_lanes(const PagedArgs& p, const paged::Sequence& s, int b0) {
  if (b0 == 0) zero_between<T>(p, 0, __builtin_amdgcn_readfirstlane(s.first), blockIdx.x, gridDim.x);
  for (uint64_t left = __ballot(s.cut > 0); left; left &= left - 1) {
    const int l = __builtin_ctzll(left);
    const int64_t from = static_cast<int64_t>(__shfl(s.first, l)) + __shfl(s.n, l);
    zero_between<T>(p, from, from + __shfl(s.cut, l), blockIdx.x, gridDim.x);
  }
}

// A launch of its own for them where the kernel's registers are all taken: two groups of many rows at head dims above 192
// spill more with it inside (two of 1024 tokens against up to 8192 keys of 256 dims, bf16 874 us, so 832).
constexpr bool zeros_inside(int dw, bool many) { return !(many && dw > 3); }

template <typename T>
__global__ __launch_bounds__(256) void attn_paged_zero(PagedArgs p) {
  const int lane = threadIdx.x & 63;
  zero_behind<T>(p);
  for (int b0 = 0; b0 < p.batch.B; b0 += 64)
    zero_of_lanes<T>(p, b0 + lane < p.batch.B ? paged::sequence_of(p.batch, b0 + lane) : paged::Sequence{0, 0, 0, 0}, b0);
}

template <typename T, int DW, int NR, bool MANY, int AUX>
__global__ __launch_bounds__(256, (per_cu(DW, NR, MANY))) void attn_paged_kernel(PagedArgs p) {
  using K = std::conditional_t<MANY, Many<T, DW, NR>, Few<T, DW, NR, AUX>>;
  __shared__ typename K::Lds lds;
  const int lane = threadIdx.x & 63, kvh = p.cache.kv_heads, G = p.G;

  const bool zeros = zeros_inside(DW, MANY) && p.zero_tail;
  if (zeros) zero_behind<T>(p);  // (others where their sequence is met)

  // the work-group's run of units: [x, x + left) of all, or one job whole
  int b = 0, h, tile, u0, w = blockIdx.x;
  int64_t each = 0, left;
  Rows rows;
  Head head{{0, 0, 0, 0}, 0, 0, 0};
  paged::Sequence near{0, 0, 0, 0};  // lane l has sequence l
  if (p.groups == 0) {
    const int heads = p.batch.B * kvh;  // (later tiles see more keys: they come first)
    tile = p.row_tiles - 1 - w / heads;
    h = w % heads % kvh;
    b = w % heads / kvh;
    const paged::Sequence s = paged::sequence_of(p.batch, b);
    if (zeros) {
      const int worker = tile * kvh + h, workers = p.row_tiles * kvh;
      if (b == 0) zero_between<T>(p, 0, s.first, worker, workers);
      const int64_t from = static_cast<int64_t>(s.first) + s.n;
      zero_between<T>(p, from, from + s.cut, worker, workers);
    }
    rows = rows_of(p, s);
    if (tile * K::ROWS >= rows.nrows) return;
    u0 = 0;
    left = rows.units((tile + 1) * K::ROWS, G);
  } else {
    // work-groups of one XCD (every eighth) have neighbouring runs: jobs there share keys
    w = blockIdx.x % 8 * (p.groups / 8) + blockIdx.x / 8;
    // units of the sequences for one head, 64 at a time: of the lane's, and up to it
    int64_t mine = 0, upto;
    const auto scan = [&](int b0) MI355_LAMBDA_INLINE {
      paged::Sequence s{0, 0, 0, 0};
      if (b0 + lane < p.batch.B) s = paged::sequence_of(p.batch, b0 + lane);
      mine = b0 + lane < p.batch.B ? all_units(rows_of(p, s), K::ROWS, G) : 0;
      upto = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int64_t v = __shfl_up(upto, off);
        if (lane >= off) upto += v;
      }
      return s;
    };
    near = scan(0);
    if (zeros) zero_of_lanes<T>(p, near, 0);
    const int64_t mine0 = mine, upto0 = upto;
    int64_t total = first_lane(__shfl(upto, 63));
    for (int b0 = 64; b0 < p.batch.B; b0 += 64) {
      const paged::Sequence s = scan(b0);
      if (zeros) zero_of_lanes<T>(p, s, b0);
      total += first_lane(__shfl(upto, 63));
    }
    total *= kvh;
    each = quotient(total + p.groups - 1, p.groups);
    each = each > p.least ? each : p.least;
    const int64_t x = w * each;
    left = x + each < total ? each : total - x;
    if (left <= 0) {
      if (threadIdx.x == 0) p.joins[w] = head;
      return;
    }
    // the sequence with unit x, and the unit within it
    int64_t rest = x, per_head = 1;
    mine = mine0;
    upto = upto0;
    for (;;) {
      const uint64_t hit = __ballot(rest < upto * kvh);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        b += l;
        per_head = first_lane(__shfl(mine, l));
        rest -= (first_lane(__shfl(upto, l)) - per_head) * kvh;
        break;
      }
      rest -= first_lane(__shfl(upto, 63)) * kvh;
      b += 64;
      if (b >= p.batch.B) {  // (there is one)
        if (threadIdx.x == 0) p.joins[w] = head;
        return;
      }
      scan(b);
    }
    rows = rows_at(p, near, b);
    h = static_cast<int>(quotient(rest, per_head));
    tile = 0;
    rest -= h * per_head;
    while (rest >= rows.units((tile + 1) * K::ROWS, G)) rest -= rows.units(++tile * K::ROWS, G);
    u0 = static_cast<int>(rest);
  }
  for (;;) {
    const int all = rows.units((tile + 1) * K::ROWS, G);
    const int u1 = all - u0 < left ? all : u0 + static_cast<int>(left);
    const bool whole = u0 == 0 && u1 == all;
    if (u0 == 0 && !whole) head = Head{rows.s, h, tile, static_cast<int32_t>(quotient(all - u1 + each - 1, each))};
    K::run(p, lds, rows, b, h, tile, u0, u1, whole ? -1 : 2 * static_cast<int64_t>(w) + (u0 == 0));
    left -= u1 - u0;
    if (left <= 0) break;
    u0 = 0;
    if (++tile * K::ROWS < rows.nrows) continue;
    tile = 0;
    if (++h < kvh) continue;
    h = 0;
    do  // (there is one with rows: units are left)
      rows = ++b < p.batch.B ? rows_at(p, near, b) : Rows{};
    while (rows.nrows == 0 && b < p.batch.B);
    if (rows.nrows == 0) break;
  }
  if (p.groups == 0) return;
  if (threadIdx.x == 0) p.joins[w] = head;
}

// Joins the parts of the jobs that several work-groups had: a work-group with a first part (blockIdx.x) and a row of its
// job's tile, whose parts its runs of LANES lanes share (SPLIT: few rows have many parts), or a row for each run (tiles of
// many rows have few). Several parts of a run are requested at a time; lanes have runs of four dims. 64 parts of 32 rows of
// 128 dims 5 us, 2 of 128 rows of 450 tiles (67 MB) 15.
template <typename T, bool SPLIT, int LANES>
__global__ __launch_bounds__(256) void attn_paged_join(PagedArgs p, int rows_of_tile) {
  constexpr int AHEAD = SPLIT ? 8 : 4, RUNS = 256 / LANES, STEP = SPLIT ? RUNS : 1;
  __shared__ float lds[RUNS][4 * LANES];
  __shared__ float lds_m[4], lds_z[RUNS];
  const int w = blockIdx.x, hd = p.cache.head_dim, G = p.G;
  const int lane = threadIdx.x % LANES, run = threadIdx.x / LANES, wave = threadIdx.x >> 6;
  const int in_tile = SPLIT ? blockIdx.y : blockIdx.y * RUNS + run;
  const Head j = p.joins[w];
  if (j.parts == 0) return;
  const Rows rows = rows_of(p, j.s);
  const int r = j.tile * rows_of_tile + in_tile, in_ws = in_tile < rows_of_tile ? in_tile : 0;
  // part 0: the work-group's last job; part k: the first one of the k-th after it
  const auto slot = [&](int k) MI355_LAMBDA_INLINE {
    const int64_t s = k == 0 ? 2 * static_cast<int64_t>(w) + 1 : 2 * (static_cast<int64_t>(w) + k);
    return s * rows_of_tile + in_ws;
  };
  const int parts = (j.parts < p.groups - w ? j.parts : p.groups - 1 - w) + 1;
  const int first = SPLIT ? run : 0, d4 = 4 * lane < hd ? 4 * lane : 0;
  f32x4 v[AHEAD];
  float top[AHEAD], sum[AHEAD];
  const auto fetch = [&](int k0) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      if (k0 + STEP * x >= parts) break;
      const int64_t at = slot(k0 + STEP * x);
      v[x] = *reinterpret_cast<const f32x4*>(p.part + at * hd + d4);
      top[x] = p.ml[2 * at];
      sum[x] = p.ml[2 * at + 1];
    }
  };
  fetch(first);  // (under way while the maximum is made)
  float m = NEG_INF;
  for (int k = SPLIT ? static_cast<int>(threadIdx.x) : lane; k < parts; k += SPLIT ? 256 : LANES) m = fmaxf(m, p.ml[2 * slot(k)]);
#pragma unroll
  for (int off = SPLIT ? 32 : LANES / 2; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  if constexpr (SPLIT) {
    if ((threadIdx.x & 63) == 0) lds_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(lds_m[0], lds_m[1]), fmaxf(lds_m[2], lds_m[3]));
  }
  const auto factor = [&](float t) MI355_LAMBDA_INLINE { return t == NEG_INF ? 1.0f : fast_exp2(t - m); };
  float z = 0.0f;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = first; k0 < parts; k0 += STEP * AHEAD) {
    if (k0 != first) fetch(k0);
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      if (k0 + STEP * x >= parts) break;
      const float f = factor(top[x]);
      z += sum[x] * f;
      a += v[x] * f;
    }
  }
  if constexpr (SPLIT) {
    *reinterpret_cast<f32x4*>(&lds[run][4 * lane]) = a;
    if (lane == 0) lds_z[run] = z;
    __syncthreads();
    if (run != 0) return;
    z = 0.0f;
    a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < RUNS; ++k) {
      z += lds_z[k];
      a += *reinterpret_cast<const f32x4*>(&lds[k][4 * lane]);
    }
  }
  if (r >= rows.nrows || in_tile >= rows_of_tile || 4 * lane >= hd) return;
  const float inv = rows.inverse(z, rows.lim(r, G));
  const int t = r / G;
  typedef T V4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<V4*>(static_cast<T*>(p.o) + (rows.s.first + static_cast<int64_t>(t)) * p.ot + (j.h * G + r - t * G) * p.oh + 4 * lane) =
      V4{from_f32<T>(a[0] * inv), from_f32<T>(a[1] * inv), from_f32<T>(a[2] * inv), from_f32<T>(a[3] * inv)};
}

struct Launch {
  bool many, past;
  int nr, rows;               // groups of 16 rows of a wave, rows of a tile
  int64_t row_tiles, groups, least, grid, ws;
};

Launch launch_of(const paged::Sizes& z) {
  Launch l{};
  const int64_t rows = z.most * (z.heads / z.kv_heads), dw = (z.head_dim + 63) / 64;
  l.many = rows > 32;
  // Groups of 16 rows of a wave. Few rows: as many as there are, where registers allow two. Many: two, which share each operand
  // that is read; above head dim 128 such a wave has the SIMD for itself, and short tiles leave waves idle: only for
  // enough rows (us of 16 sequences of 4096 keys, 32 heads of 192 / of 256, one group then two: 64 rows 94 112 / 112 177, 128
  // rows 154 125 / 191 185, 256 rows 299 231 / 368 336; two of 1024 tokens against 8192 keys 1085 734 / 1229 999).
  l.nr = l.many ? (dw <= 2 || rows > 64 * (dw - 2) ? 2 : 1) : (rows > 16 && dw <= 2 ? 2 : 1);
  l.rows = 16 * l.nr * (l.many ? 4 : 1);
  l.row_tiles = (rows + l.rows - 1) / l.rows;
  const int64_t jobs = z.B * z.kv_heads * l.row_tiles;
  // Sharing the work out evenly takes two work-groups a CU (one above head dim 128, whose registers allow no more: with
  // two 16 sequences of 8192 keys of 256 dims 102 us instead of 92; three or four where they are allowed: 200000 keys
  // of one sequence 92 us instead of 86), partial results and a second launch. A work-group for each job instead where
  // the longest that the table allows is short, or jobs fill the GPU. Measured (us, shared out / a job each; bf16, 8 K/V heads of 128, groups of 4, K and V in the last-level cache
  // but for the largest): one new token, sequences of one length, then of 10 to 100% of it: 2 sequences of 1024 keys 14.5 / 11.3, 2048
  // 17.4 / 16.7, 4096 18.6 / 27.2; 8: 2048 20.2 / 17.8 and 21.0 / 14.8, 4096 25.1 / 28.5 and 21.7 / 23.6; 16: 4096 33.7 / 29.0 and
  // 23.9 / 26.6, 8192 51.4 / 54.4 and 32.1 / 47.1; 64: 4096 110 / 98 and 56 / 59, 8192 201 / 187 and 110 / 130. Many rows: a
  // prompt of 2048 121 / 69, 8192 684 / 554; 512 tokens against 2048 63 / 63, 4096 75 / 117; 1024 against 16384 (256 jobs) 298 / 452;
  // 2048 against 16384 (512) 550 / 507.
  const int64_t room = z.width * z.page;
  // Few rows read K and V once. Where the tables allow more of them than the last-level cache holds (256 MiB), they are loaded
  // as what is not kept (us, so / as what is): 64 sequences of up to 9000 keys (655 MB) 121 / 129, 200000 keys (409 MB) 79.4 / 86.0,
  // 128 sequences of 2048 keys (537 MB) 91.5 / 97.6; 1024 keys (268 MB, in that cache) 50.1 / 43.4.
  l.past = !l.many && z.B * room * z.kv_heads * z.head_dim * 2 > int64_t(320) << 20;
  // (More than 1024 sequences fill the GPU by themselves, and each work-group would go through all their lengths: 1100 of
  // up to 300 keys in wide tables, one K/V head, 53.1 / 21.7; 4000 of up to 4000 keys 468 / 411.)
  const bool better = l.many ? room <= 2048 || (jobs >= 512 && jobs * 32 >= room) : room <= (jobs >= 128 ? 4096 : 2048);
  const bool each = jobs < (int64_t(1) << 23) && (z.B > 1024 || better);  // (a launch has fewer than 2^31 threads)
  constexpr int64_t CUS = 256;  // (not asked for: the workspace's size follows, which is known without a device)
  l.groups = each ? 0 : CUS * (dw > 2 ? 1 : 2);
  l.least = 8;
  l.grid = l.groups ? l.groups : jobs;
  l.ws = l.groups * (2 * l.rows * (z.head_dim + 2) * 4 + static_cast<int64_t>(sizeof(Head)));
  return l;
}

template <typename T, int DW, int NR, bool MANY>
int launch(const PagedArgs& p, const Launch& l, hipStream_t s) {
  const auto grid = static_cast<uint32_t>(l.grid);
  if constexpr (!zeros_inside(DW, MANY))
    if (p.zero_tail) attn_paged_zero<T><<<256, 256, 0, s>>>(p);
  if constexpr (!MANY)
    if (l.past) attn_paged_kernel<T, DW, NR, false, PAST><<<grid, 256, 0, s>>>(p);
  if (!l.past) attn_paged_kernel<T, DW, NR, MANY, 0><<<grid, 256, 0, s>>>(p);
  if (const hipError_t e = hipGetLastError(); e != hipSuccess || l.groups == 0) return static_cast<int>(e);
  const int64_t rows = std::min<int64_t>(l.rows, p.batch.most * static_cast<int64_t>(p.G));
  constexpr int LANES = DW == 1 ? 16 : DW == 2 ? 32 : 64, PER = MANY ? 256 / LANES : 1;
  const dim3 grid_of_join(static_cast<uint32_t>(l.groups), static_cast<uint32_t>((rows + PER - 1) / PER));
  attn_paged_join<T, !MANY, LANES><<<grid_of_join, 256, 0, s>>>(p, l.rows);
  return static_cast<int>(hipGetLastError());
}

template <typename T, int DW>
int launch_rows(const PagedArgs& p, const Launch& l, hipStream_t s) {
  if constexpr (DW <= 2) {
    if (l.many) return launch<T, DW, 2, true>(p, l, s);
    if (l.nr == 2) return launch<T, DW, 2, false>(p, l, s);
  } else {
    if (l.many && l.nr == 2) return launch<T, DW, 2, true>(p, l, s);
    if (l.many) return launch<T, DW, 1, true>(p, l, s);
  }
  return launch<T, DW, 1, false>(p, l, s);
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

// Few enough rows that 32 bits count them: by how many tokens there are, or by how many `most` allows.
int check_all(int dtype, const paged::Sizes& z) {
  if (const int st = paged::check(dtype, z)) return st;
  constexpr int64_t MOST = int64_t(1) << 23;
  const int64_t allowed = z.B * z.most;
  if (allowed < MOST && allowed * z.heads < MOST) return MI355_OK;
  return z.tokens * z.heads < MOST && z.most <= (1 << 20) ? MI355_OK : MI355_E_BAD_SIZE;
}

}  // namespace

extern "C" int64_t mi355_attn_paged_workspace_bytes(const int64_t* sizes) {
  if (!sizes) return MI355_E_NULL_POINTER;
  const paged::Sizes z = *reinterpret_cast<const paged::Sizes*>(sizes);
  if (const int st = check_all(MI355_F16, z)) return st;
  return launch_of(z).ws;
}

extern "C" int mi355_attn_paged(int dtype, const void* Q, const uint8_t* cache_k, const uint8_t* cache_v,
                                const float* k_scale, const float* v_scale, const int32_t* table, const int32_t* lens,
                                const int32_t* offsets, void* O, const int64_t* sizes, const int64_t* strides, float scale,
                                int zero_tail, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!sizes || !strides) return MI355_E_NULL_POINTER;
  const paged::Sizes z = *reinterpret_cast<const paged::Sizes*>(sizes);
  if (const int st = check_all(dtype, z)) return st;
  if (z.B * z.most == 0 || z.tokens == 0) return MI355_OK;
  if (!Q || !O || !lens || !cache_k || !cache_v || !k_scale || !v_scale || (z.width > 0 && !table)) return MI355_E_NULL_POINTER;
  if (z.pages < 1) return MI355_E_BAD_SIZE;
  if (!offsets && z.B * z.most > z.tokens) return MI355_E_BAD_SIZE;
  if (!(scale > 0.0f) || scale > 1e30f) return MI355_E_UNSUPPORTED;
  if (!aligned16(Q) || (reinterpret_cast<uintptr_t>(O) & 7u) || !aligned16(cache_k) || !aligned16(cache_v) ||
      strides[0] % 8 || strides[1] % 8 || strides[2] % 4 || strides[3] % 4)
    return MI355_E_ALIGNMENT;
  const Launch l = launch_of(z);
  if (l.ws > 0 && (!workspace || workspace_bytes < l.ws || !aligned16(workspace))) return MI355_E_BAD_SIZE;
  PagedArgs p{};
  p.cache = paged::cache_of(z, cache_k, cache_v, k_scale, v_scale);
  p.batch = paged::batch_of(z, table, lens, offsets);
  p.q = Q;
  p.o = O;
  p.qt = strides[0];
  p.qh = strides[1];
  p.ot = strides[2];
  p.oh = strides[3];
  p.scale = scale;
  p.heads = static_cast<int32_t>(z.heads);
  p.G = static_cast<int32_t>(z.heads / z.kv_heads);
  p.row_tiles = static_cast<int32_t>(l.row_tiles);
  p.groups = static_cast<int32_t>(l.groups);
  p.least = static_cast<int32_t>(l.least);
  p.zero_tail = zero_tail && (offsets || z.tokens > z.B * z.most);
  p.part = static_cast<float*>(workspace);
  p.ml = p.part + l.groups * 2 * l.rows * z.head_dim;
  p.joins = reinterpret_cast<Head*>(p.ml + l.groups * 2 * l.rows * 2);
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == MI355_F16 ? launch_dim<_Float16>(p, l, s) : launch_dim<__bf16>(p, l, s);
}

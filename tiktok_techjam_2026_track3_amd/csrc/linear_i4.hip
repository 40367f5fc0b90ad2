// Projection of a few rows with 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k] + b[n] with
// W[n, k] = s[n, k / GROUP] (q[n, k] - z[n, k / GROUP]), q in 0 .. 15, two to a byte (even k low).
//
// Bound by the weights' bytes: every 4-bit value is read once, straight into the registers of the
// lane that multiplies it, and rows of x ride along as the other operand of 16x16x32 MFMAs (A = x:
// 16 rows, B = weights: 16 features; a lane holds one feature, lane % 16, so its scale and zero are
// one scalar each, and D[m][n] of 4 rows of x). A wave takes R tiles of 16 features, for which it
// loads x once, or holds its k of x in registers and walks tiles of features (linear_i4_held, up to 16 rows);
// the waves of a work-group take contiguous ranges of k and add up through LDS.
//   Nibbles become operands without conversions: put into the top mantissa bits of 16 (shift, and-or),
//   q is the number 16 + q. A group's sum is then corrected in fp32, sum x q' - (16 + z) sum x, with
//   sum x from MFMAs against ones (shared by the R tiles); at most 31 : 15 + z in size, so that nothing is lost
//   to the larger operands. Subtracting in 16 bits before the product (packed, fp16 only) took 11 vector
//   instructions for 8 weights, this takes 8, which is what a CU can spend on them at 5 TB/s.
//   A lane's 16 bytes are 32 neighbouring k. For GROUP 128 the four lanes of a feature hold the
//   whole group and each word is one MFMA's operand as it is; for 32 and 64 the words change
//   places between the four lanes (4 lane swaps) so that one MFMA's 32 k are neighbours.
// 16 x 16384 x 4096 (bf16, group 128) 12.5 us, 2.9 TB/s (linear_i4_held; 17.4 with x from L2 for every two tiles),
// 7 x 4096 x 16384 (group 64; linear_i4_kernel, bound by what a CU can have in flight of the 360 kB of x and weights
// that it takes in: one work-group alone takes as long) 17.3 us, 1 x 12288 x 4096 (linear_i4_few) 7.9 us, 3.3 TB/s.
#include "common.h"

namespace {

// most features of a wave of linear_i4_few
constexpr int MAX_FEW = 32;

struct I4Args {
  const void* x;
  const uint8_t* w;
  const void* scale;
  const uint8_t* zero;  // nullable: 8
  const float* bias;    // nullable
  void* y;
  int64_t ldx, ldy;
  int32_t M, N, K;
};

template <typename T>
struct Nib;
template <>
struct Nib<_Float16> {
  using vec = f16x8;
  static constexpr uint32_t SIXTEEN = 0x4c004c00u;
  static constexpr int SHIFT = 6;  // of a nibble's lowest bit, 16's mantissa is 10 bits long
};
template <>
struct Nib<__bf16> {
  using vec = bf16x8;
  static constexpr uint32_t SIXTEEN = 0x41804180u;
  static constexpr int SHIFT = 3;  // ... 7 bits
};
MI355_DEVINL f32x4 mma_i4(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
MI355_DEVINL f32x4 mma_i4(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// 8 nibbles of a word, 16 + q each: elements 0 4 1 5 2 6 3 7
template <typename T>
MI355_DEVINL typename Nib<T>::vec nibbles(uint32_t w) {
  constexpr int SH = Nib<T>::SHIFT;
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = ((4 * i < SH ? w << (SH - 4 * i) : w >> (4 * i - SH)) & (0x000f000fu << SH)) | Nib<T>::SIXTEEN;
  return __builtin_bit_cast(typename Nib<T>::vec, r);
}
// 8 elements in the order 0 4 1 5 2 6 3 7
MI355_DEVINL u32x4 nibble_order(u32x4 v) {
  return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
               __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// A 4 x 4 transposition over (lane / 16, word): word m of lanes j becomes word j of lanes m.
MI355_DEVINL u32x4 transposed(u32x4 w) {
  const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{c[0], c[1], e[0], e[1]};
}

// BYTES bytes from any address, into words (one or two wide loads; nothing waits for them here)
template <int BYTES, int N>
MI355_DEVINL void load_words(const void* src, uint32_t (&dst)[N]) {
  static_assert(N == (BYTES + 3) / 4 && BYTES % 4 != 3, "words");
  struct Words { uint32_t v[BYTES < 4 ? 1 : BYTES / 4]; } __attribute__((packed, aligned(1)));
  struct Half { uint16_t v; } __attribute__((packed, aligned(1)));
  if constexpr (BYTES >= 4) {
    const Words w = *static_cast<const Words*>(src);
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) dst[i] = w.v[i];
  }
  if constexpr (BYTES % 4 == 2) dst[N - 1] = reinterpret_cast<const Half*>(static_cast<const uint8_t*>(src) + BYTES - 2)->v;
  if constexpr (BYTES % 4 == 1) dst[N - 1] = static_cast<const uint8_t*>(src)[BYTES - 1];
}
// group j's -(16 + z) and scale
template <int N>
MI355_DEVINL float minus_zero(const I4Args& p, const uint32_t (&z)[N], int j) {
  const uint32_t v = p.zero != nullptr ? z[j / 4] >> (8 * (j % 4)) & 255u : 8u;
  return -16.f - static_cast<float>(v);
}
template <typename T, int N>
MI355_DEVINL float scale_of(const uint32_t (&s)[N], int j) {
  const uint16_t v = static_cast<uint16_t>(s[j / 2] >> (16 * (j % 2)));
  return to_f32(__builtin_bit_cast(T, v));
}

// MT tiles of 16 rows of x, R tiles of 16 features. Steps of 128 k in batches of 4, whose weights, scales and
// zero points are loaded a batch ahead. The last batch of K starts early enough to be whole, what it repeats
// counts with a scale of 0, so that nothing in the loop branches: behind a branch that loads, the compiler waits
// for every load in flight (128 x 8192 x 4096, group 64, 50 us so, now 41). SHORT: K below 512, a batch reaches past it.
template <typename T, int GROUP, int MT, int R, int NW, bool SHORT, typename TO>
__global__ __launch_bounds__(64 * NW) void linear_i4_kernel(I4Args p) {
  using vec = typename Nib<T>::vec;
  constexpr int GP = 128 / GROUP;           // groups of a step
  constexpr int U = 4;                      // steps of a batch
  constexpr int XU = MT == 4 && R == 1 ? 1 : 2;  // steps whose x is in flight
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * R), m0 = blockIdx.y * (16 * MT);
  const int groups = p.K / GROUP, steps = (p.K + 127) / 128;
  const int per = ((steps + NW - 1) / NW + U - 1) / U * U;
  const int s_begin = wave * per, s_end = s_begin + per < steps ? s_begin + per : steps;
  const uint8_t* const zeros = p.zero != nullptr ? p.zero : static_cast<const uint8_t*>(p.scale);  // (not used)
  const uint8_t* wrow[R];
  const T* srow[R];
  const uint8_t* zrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    // features past the last: any real one's, not stored
    const int64_t f = n0 + 16 * r + l16 < p.N ? n0 + 16 * r + l16 : p.N - 1;
    wrow[r] = p.w + f * (p.K / 2);
    srow[r] = static_cast<const T*>(p.scale) + f * groups;
    zrow[r] = zeros + f * groups;
  }
  const T* xrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + l16 < p.M ? m0 + 16 * t + l16 : p.M - 1;
    xrow[t] = static_cast<const T*>(p.x) + m * p.ldx;
  }
  f32x4 total[R][MT];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) total[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  vec ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.0f);

  struct Batch {
    u32x4 w[U][R];
    uint32_t s[R][U * GP / 2], z[R][U * GP / 4];  // as they are in memory
  };
  const auto first_k = [&](int s0) MI355_LAMBDA_INLINE {  // of the batch at step s0
    const int k = s0 * 128;
    return SHORT || k < p.K - 128 * U ? k : p.K - 128 * U;
  };
  auto fetch = [&](int s0, Batch& d) MI355_LAMBDA_INLINE {
    const int k0 = first_k(s0), at = k0 / GROUP;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        int k = k0 + 128 * u + 32 * g;
        if (SHORT) k = k < p.K ? k : p.K - 32;
        d.w[u][r] = *reinterpret_cast<const u32x4*>(wrow[r] + k / 2);
      }
      if constexpr (!SHORT) {
        load_words<U * GP * 2>(srow[r] + at, d.s[r]);
        load_words<U * GP>(zrow[r] + at, d.z[r]);
      } else {
#pragma unroll
        for (int i = 0; i < U * GP; ++i) {
          const int gi = i < groups ? i : groups - 1;
          const uint32_t sv = __builtin_bit_cast(uint16_t, srow[r][gi]), zv = zrow[r][gi];
          d.s[r][i / 2] = i % 2 ? d.s[r][i / 2] | sv << 16 : sv;
          d.z[r][i / 4] = i % 4 ? d.z[r][i / 4] | zv << (8 * (i % 4)) : zv;
        }
      }
    }
  };
  typedef u32x4 Rows[XU][4][MT];
  auto fetch_x = [&](Rows& x, int k0, int u0) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int u = 0; u < XU; ++u)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        int k = k0 + 128 * (u0 + u) + (GROUP == 128 ? 32 * g + 8 * m : 32 * m + 8 * g);
        if (SHORT) k = k < p.K ? k : p.K - 8;
#pragma unroll
        for (int t = 0; t < MT; ++t) x[u][m][t] = *reinterpret_cast<const u32x4*>(xrow[t] + k);
      }
  };
  const auto batch = [&](int s0, const Batch& cur, Rows& x) MI355_LAMBDA_INLINE {
    const int k0 = first_k(s0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && u % XU == 0) fetch_x(x, k0, u);
      u32x4 wu[R];
#pragma unroll
      for (int r = 0; r < R; ++r) wu[r] = GROUP == 128 ? cur.w[u][r] : transposed(cur.w[u][r]);
#pragma unroll
      for (int i = 0; i < GP; ++i) {
        f32x4 acc[R][MT], sum[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int m = i * 4 / GP; m < (i + 1) * 4 / GP; ++m) {
          vec xo[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            xo[t] = __builtin_bit_cast(vec, nibble_order(x[u % XU][m][t]));
            sum[t] = mma_i4(xo[t], ones, sum[t]);
          }
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const vec wv = nibbles<T>(wu[r][m]);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[r][t] = mma_i4(xo[t], wv, acc[r][t]);
          }
        }
        const int j = u * GP + i, k = k0 + j * GROUP;
        const bool counts = SHORT ? k < p.K : k >= s0 * 128;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float z = minus_zero(p, cur.z[r], j), sf = counts ? scale_of<T>(cur.s[r], j) : 0.f;
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              total[r][t][e] = __builtin_fmaf(__builtin_fmaf(sum[t][e], z, acc[r][t][e]), sf, total[r][t][e]);
        }
      }
    }
  };
  if (s_begin < s_end) {
    Batch cur, nxt;
    Rows x;
    int s0 = s_begin;
    fetch(s0, cur);
    for (; s0 + U < s_end; s0 += U) {
      fetch_x(x, first_k(s0), 0);
      fetch(s0 + U, nxt);
      batch(s0, cur, x);
      cur = nxt;
    }
    fetch_x(x, first_k(s0), 0);
    batch(s0, cur, x);
  }

  __shared__ f32x4 part[NW][R * MT][64];
#pragma unroll
  for (int i = 0; i < R * MT; ++i) part[wave][i][lane] = total[i / MT][i % MT];
  __syncthreads();
  // wave w adds up tiles w, w + NW ..
#pragma unroll
  for (int i = 0; i < R * MT; ++i) {
    if (i % NW != wave) continue;
    const int r = i / MT, t = i % MT, n = n0 + 16 * r + l16;
    f32x4 v = part[0][i][lane];
#pragma unroll
    for (int y = 1; y < NW; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += part[y][i][lane][e];
    if (n < p.N) {
      const float b = p.bias != nullptr ? p.bias[n] : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = m0 + 16 * t + 4 * g + e;
        if (row < p.M) static_cast<TO*>(p.y)[row * p.ldy + n] = from_f32<TO>(v[e] + b);
      }
    }
  }
}

// Up to 16 rows of x and S steps of 128 k for each of 8 waves: a wave holds its x (and up to 4 sums of it) in
// registers and walks tiles of 16 features, whose weights, scales and zero points are requested before the
// waves meet over the tile before (two and three tiles ahead gained nothing: 16 x 16384 x 4096 12.8, 15.0,
// 15.8 us), and no load of which is behind a branch. The last waves of K start early enough to be whole; what they
// repeat counts with a scale of 0.
template <typename T, int GROUP, int S, typename TO>
__global__ __launch_bounds__(512) void linear_i4_held(I4Args p, int per) {
  using vec = typename Nib<T>::vec;
  constexpr int GP = 128 / GROUP, NW = 8;
  constexpr bool HOLD = S * GP <= 4;      // sums of x in registers too
  __shared__ f32x4 part[2][NW][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int groups = p.K / GROUP, tiles = (p.N + 15) / 16;
  // the wave's k: [begin, begin + 128 S), of which those before `from` are another wave's
  const int from = wave * S * 128, begin = from < p.K - S * 128 ? from : p.K - S * 128;
  const int t0 = blockIdx.x * per, t1 = t0 + per < tiles ? t0 + per : tiles;
  struct Tile {
    u32x4 w[S];
    uint32_t s[(S * GP + 1) / 2], z[(S * GP + 3) / 4];  // as they are in memory
    float bias;
  };
  // (where there are none: bytes that are there, 2 a group and 64 or more a feature, not used)
  const uint8_t* const zeros = p.zero != nullptr ? p.zero : static_cast<const uint8_t*>(p.scale);
  const float* const biases = p.bias != nullptr ? p.bias : reinterpret_cast<const float*>(p.w);
  auto fetch = [&](int t, Tile& d) MI355_LAMBDA_INLINE {
    const int64_t f = t * 16 + l16 < p.N ? t * 16 + l16 : p.N - 1;
    const uint8_t* wrow = p.w + f * (p.K / 2) + (begin + 32 * g) / 2;
#pragma unroll
    for (int u = 0; u < S; ++u) d.w[u] = *reinterpret_cast<const u32x4*>(wrow + 64 * u);
    load_words<S * GP * 2>(static_cast<const uint16_t*>(p.scale) + f * groups + begin / GROUP, d.s);
    load_words<S * GP>(zeros + f * groups + begin / GROUP, d.z);
    d.bias = biases[f];
  };
  Tile d;
  fetch(t0, d);
  vec x[S][4];
  {
    const T* row = static_cast<const T*>(p.x) + static_cast<int64_t>(l16 < p.M ? l16 : p.M - 1) * p.ldx;
#pragma unroll
    for (int u = 0; u < S; ++u)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        x[u][m] = __builtin_bit_cast(vec, *reinterpret_cast<const u32x4*>(row + begin + u * 128 + 32 * m + 8 * g));
      }
  }
  vec ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.0f);
  f32x4 sx[HOLD ? S * GP : 1];
#pragma unroll
  for (int u = 0; u < S; ++u) {
    u32x4 v[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) v[m] = nibble_order(__builtin_bit_cast(u32x4, x[u][m]));
    if constexpr (GROUP == 128) {  // x, once, instead of the weights (loaded in that order it took 0.4 us longer)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x4 c = transposed(u32x4{v[0][e], v[1][e], v[2][e], v[3][e]});
#pragma unroll
        for (int m = 0; m < 4; ++m) v[m][e] = c[m];
      }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) x[u][m] = __builtin_bit_cast(vec, v[m]);
  }
  auto sum_of = [&](int u, int i) MI355_LAMBDA_INLINE {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = i * 4 / GP; m < (i + 1) * 4 / GP; ++m) s = mma_i4(x[u][m], ones, s);
    return s;
  };
  if constexpr (HOLD) {
#pragma unroll
    for (int u = 0; u < S; ++u)
#pragma unroll
      for (int i = 0; i < GP; ++i) sx[u * GP + i] = sum_of(u, i);
  }
  auto work = [&](int t) MI355_LAMBDA_INLINE {
    const float b0 = p.bias != nullptr && wave == 0 ? d.bias : 0.f;
    f32x4 total = {b0, b0, b0, b0};
#pragma unroll
    for (int u = 0; u < S; ++u) {
      const u32x4 w = GROUP == 128 ? d.w[u] : transposed(d.w[u]);
#pragma unroll
      for (int i = 0; i < GP; ++i) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = i * 4 / GP; m < (i + 1) * 4 / GP; ++m) acc = mma_i4(x[u][m], nibbles<T>(w[m]), acc);
        const f32x4 s = HOLD ? sx[HOLD ? u * GP + i : 0] : sum_of(u, i);
        const int j = u * GP + i;
        const float z = minus_zero(p, d.z, j), sf = begin + j * GROUP >= from ? scale_of<T>(d.s, j) : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] = __builtin_fmaf(__builtin_fmaf(s[e], z, acc[e]), sf, total[e]);
      }
    }
    part[(t - t0) & 1][wave][lane] = total;
  };
  auto finish = [&](int t) MI355_LAMBDA_INLINE {
    __syncthreads();
    if (((t - t0) & 7) != wave) return;
    f32x4 v = part[(t - t0) & 1][0][lane];
#pragma unroll
    for (int y = 1; y < NW; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += part[(t - t0) & 1][y][lane][e];
    const int n = t * 16 + l16;
    if (n < p.N) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 4 * g + e;
        if (row < p.M) static_cast<TO*>(p.y)[row * p.ldy + n] = from_f32<TO>(v[e]);
      }
    }
  };
  for (int t = t0; t < t1 - 1; ++t) {
    work(t);
    fetch(t + 1, d);
    finish(t);
  }
  work(t1 - 1);
  finish(t1 - 1);
}

// Up to 4 rows of x on the vector ALUs. The MFMA kernels above load x for 16 rows however few are real; here
// a wave holds its k of every row in registers (32 neighbouring k a lane, CH chunks of 2048) and walks
// features, whose weights, scales and zero points it reads as whole lines: 16, 2 and 1 bytes a lane. KW waves
// share a feature's k. 4 features at a time: q x in packed dot products, the zero point as above, and one
// exchange that adds up 64 lanes for 4 features together (2.5 instructions a sum instead of 7).
template <typename T>
MI355_DEVINL float dot2(uint32_t a, uint32_t b, float c);
template <>
MI355_DEVINL float dot2<_Float16>(uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
}
template <>
MI355_DEVINL float dot2<__bf16>(uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
}
template <int CTRL>
MI355_DEVINL float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, false));
}
// Sums over the wave of 4 values a lane: lanes 16 i .. get the sum of value 0, 2, 1, 3 for i = 0 .. 3.
MI355_DEVINL float wave_sum4(float v0, float v1, float v2, float v3) {
  const auto u = [](float x) MI355_LAMBDA_INLINE { return __float_as_uint(x); };
  const auto f = [](uint32_t x) MI355_LAMBDA_INLINE { return __uint_as_float(x); };
  const auto a = __builtin_amdgcn_permlane32_swap(u(v0), u(v1), false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(u(v2), u(v3), false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(u(f(a[0]) + f(a[1])), u(f(b[0]) + f(b[1])), false, false);
  return dpp_add<0x121>(dpp_add<0x122>(dpp_add<0x124>(dpp_add<0x128>(f(c[0]) + f(c[1])))));  // row_ror 8 4 2 1
}

template <typename T, int GROUP, int M, int CH, int KW, typename TO>
__global__ __launch_bounds__(KW == 8 ? 512 : 256) void linear_i4_few(I4Args p, int per_wave) {
  constexpr int SH = Nib<T>::SHIFT, F = 4, NW = KW == 8 ? 8 : 4;
  __shared__ float part[NW][MAX_FEW][M];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % KW, wg_features = per_wave * (NW / KW);
  const int n_wave = blockIdx.x * wg_features + wave / KW * per_wave;  // first feature of this wave
  const int groups = p.K / GROUP;
  const uint8_t* wp[CH];
  int at[CH];
  bool in[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k0 = (kw * CH + c) * 2048 + lane * 32;
    in[c] = k0 < p.K;
    const int k = in[c] ? k0 : 0;  // (lanes past K: x = 0)
    wp[c] = p.w + k / 2;
    at[c] = k / GROUP;
  }
  const uint8_t* const zeros = p.zero != nullptr ? p.zero : static_cast<const uint8_t*>(p.scale);  // (not used)
  struct Four {
    u32x4 w[F][CH];
    uint16_t s[F][CH];
    uint8_t z[F][CH];
  };
  auto fetch = [&](int n, Four& d) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      const int64_t f = n + i < p.N ? n + i : p.N - 1;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        d.w[i][c] = *reinterpret_cast<const u32x4*>(wp[c] + f * (p.K / 2));
        d.s[i][c] = static_cast<const uint16_t*>(p.scale)[f * groups + at[c]];
        d.z[i][c] = zeros[f * groups + at[c]];
      }
    }
  };
  Four cur, nxt;
  fetch(n_wave, cur);
  uint32_t x[CH][M][16];
  float sx[CH][M];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k = in[c] ? (kw * CH + c) * 2048 + lane * 32 : 0;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const T* row = static_cast<const T*>(p.x) + static_cast<int64_t>(m < p.M ? m : 0) * p.ldx + k;
      sx[c][m] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 v = *reinterpret_cast<const u32x4*>(row + 8 * i);
        if (!in[c]) v = u32x4{0u, 0u, 0u, 0u};
        v = nibble_order(v);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[c][m][4 * i + e] = v[e];
      }
    }
  }
  const T one1 = static_cast<T>(1.0f);
  const uint32_t one = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, one1)) * 0x10001u;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) sx[c][m] = dot2<T>(x[c][m][i], one, sx[c][m]);

  auto work = [&](int n, const Four& cur) MI355_LAMBDA_INLINE {
    float v[F][M];
#pragma unroll
    for (int i = 0; i < F; ++i) {
#pragma unroll
      for (int m = 0; m < M; ++m) v[i][m] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float d[M];
#pragma unroll
        for (int m = 0; m < M; ++m) d[m] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = cur.w[i][c][j];
            const uint32_t q = ((4 * e < SH ? w << (SH - 4 * e) : w >> (4 * e - SH)) & (0x000f000fu << SH)) | Nib<T>::SIXTEEN;
#pragma unroll
            for (int m = 0; m < M; ++m) d[m] = dot2<T>(q, x[c][m][4 * j + e], d[m]);
          }
        const float z = -16.f - (p.zero != nullptr ? static_cast<float>(cur.z[i][c]) : 8.f);
        const float s = in[c] ? to_f32(__builtin_bit_cast(T, cur.s[i][c])) : 0.f;
#pragma unroll
        for (int m = 0; m < M; ++m) v[i][m] = __builtin_fmaf(__builtin_fmaf(sx[c][m], z, d[m]), s, v[i][m]);
      }
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const float sum = wave_sum4(v[0][m], v[1][m], v[2][m], v[3][m]);
      const int g = lane >> 4, i = g == 1 ? 2 : g == 2 ? 1 : g;
      if ((lane & 15) == 0) part[wave][n + i][m] = sum;
    }
  };
  int n = 0;
  for (; n + F < per_wave; n += F) {
    fetch(n_wave + n + F, nxt);
    work(n, cur);
    cur = nxt;
  }
  work(n, cur);
  __syncthreads();
  for (int i = threadIdx.x; i < wg_features * M; i += 64 * NW) {
    const int f = i % wg_features, m = i / wg_features, n = blockIdx.x * wg_features + f;
    if (n >= p.N || m >= p.M) continue;
    float v = p.bias != nullptr ? p.bias[n] : 0.f;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) sum += part[f / per_wave * KW + w][f % per_wave][m];
    static_cast<TO*>(p.y)[m * p.ldy + n] = from_f32<TO>(sum + v);
  }
}

template <typename T, int GROUP, int M, int CH, int KW, typename TO>
int launch_few(const I4Args& a, hipStream_t s) {
  // enough waves for the CUs (8 each), several groups of 4 features a wave beyond that: each wave loads x
  // (1024 to 4096 waves: 2 x 4096 x 16384 18.6, 13.4, 11.9, 13.3, 13.2 us, 1 x 65536 x 2048 19.7, 18.4, 15.8, 17.8, 16.2)
  const int64_t waves = static_cast<int64_t>(a.N) * KW / 2048;
  const int per_wave = static_cast<int>(waves < 8 ? 4 : waves >= MAX_FEW ? MAX_FEW : waves / 4 * 4);
  constexpr int NW = KW == 8 ? 8 : 4;
  const int64_t wg = per_wave * (NW / KW);
  hipLaunchKernelGGL((linear_i4_few<T, GROUP, M, CH, KW, TO>), dim3(static_cast<unsigned>((a.N + wg - 1) / wg)), dim3(64 * NW), 0, s, a, per_wave);
  return static_cast<int>(hipGetLastError());
}
template <typename T, int GROUP, int S, typename TO>
int launch_held(const I4Args& a, hipStream_t s) {
  // a work-group a CU (two: 16 x 16384 x 4096 21 us)
  const int tiles = (a.N + 15) / 16, per = (tiles + 255) / 256;
  hipLaunchKernelGGL((linear_i4_held<T, GROUP, S, TO>), dim3(static_cast<unsigned>((tiles + per - 1) / per)), dim3(512), 0, s, a, per);
  return static_cast<int>(hipGetLastError());
}
template <typename T, int GROUP, int MT, int R, int NW, bool SHORT, typename TO>
int launch_one(const I4Args& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.N + 16 * R - 1) / (16 * R)), static_cast<unsigned>((a.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((linear_i4_kernel<T, GROUP, MT, R, NW, SHORT, TO>), grid, dim3(64 * NW), 0, s, a);
  return static_cast<int>(hipGetLastError());
}
template <typename T, int GROUP, int MT, typename TO>
int launch_tiles(const I4Args& a, hipStream_t s) {
  if (a.K < 512) return launch_one<T, GROUP, MT, 1, 4, true, TO>(a, s);
  if constexpr (MT == 1) {  // (K > HELD_K)
    // Two tiles a wave halve the loads of x, where that leaves every CU work-groups (16 x 12288 x 11008 40 us
    // with two, 42 with one, 16 x 16384 x 12288, group 64, 47 and 63)
    if ((a.N + 15) / 16 >= 768) return launch_one<T, GROUP, MT, 2, 4, false, TO>(a, s);
    return launch_one<T, GROUP, MT, 1, 8, false, TO>(a, s);
  } else {
    if constexpr (GROUP != 32) {
      // (32 x 8192 x 8192 28.8, 64 x 12288 x 4096 42 us with two tiles a wave, 36.2 and 51.1 with one; 64 rows and
      // two tiles at group 128 take all 512 registers and 4 more in scratch, at one wave a SIMD)
      if ((a.N + 15) / 16 >= 512) return launch_one<T, GROUP, MT, 2, 4, false, TO>(a, s);
    }
    return launch_one<T, GROUP, MT, 1, 4, false, TO>(a, s);
  }
}
template <typename T, int GROUP, typename TO>
int launch_mt(const I4Args& a, hipStream_t s) {
  constexpr int HELD_K = GROUP == 32 ? 6144 : 8192;  // what 8 waves' registers hold
  // linear_i4_few: one row (us, against linear_i4_held: 1 x 12288 x 4096 7.9 / 8.8, 1 x 4096 x 8192 6.3 / 8.9; below
  // 512 k most of a wave would idle), two from a k where linear_i4_held's tiles are few and large (2 x 4096 x 8192
  // 6.8 / 9.1, but 2 x 12288 x 4096 9.4 / 8.5), four where it does not hold x (against linear_i4_kernel: 4 x 4096 x
  // 16384 13.6 / 17; but 4 x 12288 x 8192 18.4 / 17.8 held).
  if (a.K >= 512 && a.K <= 16384) {
    if (a.M == 1) {
      if (a.K <= 2048) return launch_few<T, GROUP, 1, 1, 1, TO>(a, s);
      if (a.K <= 4096) return launch_few<T, GROUP, 1, 2, 1, TO>(a, s);
      if (a.K <= 8192) return launch_few<T, GROUP, 1, 2, 2, TO>(a, s);
      return launch_few<T, GROUP, 1, 2, 4, TO>(a, s);
    }
    if (a.M == 2 && a.K > 4096)
      return a.K <= 8192 ? launch_few<T, GROUP, 2, 1, 4, TO>(a, s) : launch_few<T, GROUP, 2, 1, 8, TO>(a, s);
    if (a.M <= 4 && a.K > 8192) return launch_few<T, GROUP, 4, 1, 8, TO>(a, s);
  }
  if (a.M <= 16) {
    if (a.K < 128 || a.K > HELD_K) return launch_tiles<T, GROUP, 1, TO>(a, s);
    if (a.K <= 1024) return launch_held<T, GROUP, 1, TO>(a, s);
    if (a.K <= 2048) return launch_held<T, GROUP, 2, TO>(a, s);
    if (a.K <= 4096) return launch_held<T, GROUP, 4, TO>(a, s);
    if (a.K <= 6144) return launch_held<T, GROUP, 6, TO>(a, s);
    if constexpr (GROUP != 32) return launch_held<T, GROUP, 8, TO>(a, s);
  }
  if (a.M <= 32) return launch_tiles<T, GROUP, 2, TO>(a, s);
  return launch_tiles<T, GROUP, 4, TO>(a, s);
}
template <typename T, typename TO>
int launch_group(const I4Args& a, int64_t group, hipStream_t s) {
  if (group == 32) return launch_mt<T, 32, TO>(a, s);
  if (group == 64) return launch_mt<T, 64, TO>(a, s);
  return launch_mt<T, 128, TO>(a, s);
}

}  // namespace

extern "C" int mi355_linear_i4(int dtype, int out_dtype, const void* X, int64_t ldx, const uint8_t* Wq,
                               const void* scale, const uint8_t* zero, const float* bias, void* Y,
                               int64_t ldy, int64_t M, int64_t N, int64_t K, int64_t group, void* stream) {
  if (M < 0 || N < 0 || K < 0 || M > (int64_t(1) << 20) || N > (int64_t(1) << 26) || K > (int64_t(1) << 26))
    return MI355_E_BAD_SIZE;
  if (dtype != MI355_F16 && dtype != MI355_BF16) return MI355_E_BAD_DTYPE;
  if (out_dtype != dtype && out_dtype != MI355_F32) return MI355_E_BAD_DTYPE;
  if (group != 32 && group != 64 && group != 128) return MI355_E_UNSUPPORTED;
  if (K % group != 0) return MI355_E_BAD_SIZE;
  if (M == 0 || N == 0) return MI355_OK;
  if (!Y || (K > 0 && (!X || !Wq || !scale))) return MI355_E_NULL_POINTER;
  if (ldx < K || ldy < N) return MI355_E_BAD_SIZE;
  if (ldx % 8 || !aligned16(X) || !aligned16(Wq)) return MI355_E_ALIGNMENT;
  const I4Args a{X, Wq, scale, zero, bias, Y, ldx, ldy, static_cast<int32_t>(M), static_cast<int32_t>(N), static_cast<int32_t>(K)};
  const auto s = static_cast<hipStream_t>(stream);
  if (dtype == MI355_F16)
    return out_dtype == MI355_F32 ? launch_group<_Float16, float>(a, group, s) : launch_group<_Float16, _Float16>(a, group, s);
  return out_dtype == MI355_F32 ? launch_group<__bf16, float>(a, group, s) : launch_group<__bf16, __bf16>(a, group, s);
}

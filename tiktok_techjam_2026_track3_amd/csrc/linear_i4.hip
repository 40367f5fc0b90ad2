// Projection of a few rows with 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k] + b[n] with
// W[n, k] = s[n, k / GROUP] (q[n, k] - z[n, k / GROUP]), q in 0 .. 15, two to a byte (even k low).
//
// Bound by the weights' bytes: every 4-bit value is read once, straight into the registers of the
// lane that multiplies it, and rows of x ride along as the other operand of 16x16x32 MFMAs (A = x:
// 16 rows, B = weights: 16 features; a lane holds one feature, lane % 16, so its scale and zero are
// one scalar each, and D[m][n] of 4 rows of x). A wave takes R tiles of 16 features, for which it
// loads x once; the waves of a work-group take contiguous ranges of k and add up through LDS.
//   Nibbles become operands without conversions: put into the top mantissa bits of 16 (shift, and-or),
//   q is the number 16 + q. A group's sum is then corrected in fp32, sum x q' - (16 + z) sum x, with
//   sum x from MFMAs against ones (shared by the R tiles); at most 31 : 15 + z in size, so that nothing is lost
//   to the larger operands. Subtracting in 16 bits before the product (packed, fp16 only) took 11 vector
//   instructions for 8 weights, this takes 8, which is what a CU can spend on them at 5 TB/s.
//   A lane's 16 bytes are 32 neighbouring k. For GROUP 128 the four lanes of a feature hold the
//   whole group and each word is one MFMA's operand as it is; for 32 and 64 the words change
//   places between the four lanes (4 lane swaps) so that one MFMA's 32 k are neighbours.
// 16 x 16384 x 4096 (bf16, group 128) 16.1 us, 2.2 TB/s: without the loads of x, which every work-group takes from
// L2, it took 11; 7 x 4096 x 16384 (group 64) 18 us. 1 x 12288 x 4096 (linear_i4_few) 8 us, 3.2 TB/s.
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

// N consecutive values from any address of their type (one or two wide loads where they line up)
template <int N, typename V>
MI355_DEVINL void load_run(const V* src, V (&dst)[N]) {
  struct Run { V v[N]; } __attribute__((packed, aligned(1)));
  const Run run = *reinterpret_cast<const Run*>(src);
#pragma unroll
  for (int i = 0; i < N; ++i) dst[i] = run.v[i];
}

// MT tiles of 16 rows of x, R tiles of 16 features. Steps of 128 k in batches of 4, whose weights are
// loaded a batch ahead; a feature's scales and zero points of a batch are neighbours and loaded together.
template <typename T, int GROUP, int MT, int R, int NW, typename TO>
__global__ __launch_bounds__(64 * NW) void linear_i4_kernel(I4Args p) {
  using vec = typename Nib<T>::vec;
  constexpr int GP = 128 / GROUP;           // groups of a step
  constexpr int U = 4;                      // steps of a batch
  constexpr int XU = MT == 1 ? 2 : 1;       // steps whose x is in flight
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * R), m0 = blockIdx.y * (16 * MT);
  const int groups = p.K / GROUP, steps = (p.K + 127) / 128;
  const int per = ((steps + NW - 1) / NW + U - 1) / U * U;
  const int s_begin = wave * per, s_end = s_begin + per < steps ? s_begin + per : steps;
  const uint8_t* wrow[R];
  const T* srow[R];
  const uint8_t* zrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    // features past the last: any real one's, not stored
    const int64_t f = n0 + 16 * r + l16 < p.N ? n0 + 16 * r + l16 : p.N - 1;
    wrow[r] = p.w + f * (p.K / 2);
    srow[r] = static_cast<const T*>(p.scale) + f * groups;
    zrow[r] = p.zero + f * groups;  // (read only where there are any)
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
    T s[R][U * GP];
    uint8_t z[R][U * GP];
  };
  // (steps past the wave's range load its last one again; k past K, the row's last ones)
  auto fetch = [&](int s0, Batch& d) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u < s_end ? s0 + u : s_end - 1;
      int k = s * 128 + 32 * g;
      if constexpr (GROUP != 128) k = k < p.K ? k : p.K - 32;
#pragma unroll
      for (int r = 0; r < R; ++r) d.w[u][r] = *reinterpret_cast<const u32x4*>(wrow[r] + k / 2);
    }
    const int at = s0 * GP;
    if (at + U * GP <= groups) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        load_run(srow[r] + at, d.s[r]);
        if (p.zero != nullptr) load_run(zrow[r] + at, d.z[r]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < U * GP; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int gi = at + i < groups ? at + i : groups - 1;
          d.s[r][i] = srow[r][gi];
          if (p.zero != nullptr) d.z[r][i] = zrow[r][gi];
        }
    }
    if (p.zero == nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < U * GP; ++i) d.z[r][i] = 8;
    }
  };
  Batch cur;
  if (s_begin < s_end) fetch(s_begin, cur);
  for (int s0 = s_begin; s0 < s_end; s0 += U) {
    u32x4 x[XU][4][MT];
    auto fetch_x = [&](int s1) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int u = 0; u < XU; ++u) {
        const int s = s1 + u < s_end ? s1 + u : s_end - 1;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          int k = s * 128 + (GROUP == 128 ? 32 * g + 8 * m : 32 * m + 8 * g);
          if constexpr (GROUP != 128) k = k < p.K ? k : p.K - 8;
#pragma unroll
          for (int t = 0; t < MT; ++t) x[u][m][t] = *reinterpret_cast<const u32x4*>(xrow[t] + k);
        }
      }
    };
    fetch_x(s0);
    Batch nxt;
    if (s0 + U < s_end) fetch(s0 + U, nxt);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= s_end) break;
      if (u > 0 && u % XU == 0) fetch_x(s0 + u);
      u32x4 wu[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        wu[r] = cur.w[u][r];
        if constexpr (GROUP != 128) {
          // word m of lanes j becomes word j of lanes m: a 4 x 4 transposition over (lane / 16, word)
          auto a = __builtin_amdgcn_permlane32_swap(wu[r][0], wu[r][2], false, false);
          auto b = __builtin_amdgcn_permlane32_swap(wu[r][1], wu[r][3], false, false);
          auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
          auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
          wu[r] = u32x4{c[0], c[1], e[0], e[1]};
        }
      }
#pragma unroll
      for (int i = 0; i < GP; ++i) {
        if (GROUP != 128 && (s0 + u) * GP + i >= groups) break;  // past K
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
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float z = -16.f - static_cast<float>(cur.z[r][u * GP + i]), sf = to_f32(cur.s[r][u * GP + i]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              total[r][t][e] = __builtin_fmaf(__builtin_fmaf(sum[t][e], z, acc[r][t][e]), sf, total[r][t][e]);
        }
      }
    }
    cur = nxt;
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

// Up to 4 rows of x on the vector ALUs. The MFMA kernel above loads x for 16 rows however few are real; here
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
  uint32_t x[CH][M][16];
  float sx[CH][M];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int k0 = (kw * CH + c) * 2048 + lane * 32;
    in[c] = k0 < p.K;
    const int k = in[c] ? k0 : 0;  // (lanes past K: x = 0)
    wp[c] = p.w + k / 2;
    at[c] = k / GROUP;
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

  struct Four {
    u32x4 w[F][CH];
    T s[F][CH];
    uint8_t z[F][CH];
  };
  auto fetch = [&](int n, Four& d) MI355_LAMBDA_INLINE {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      const int64_t f = n + i < p.N ? n + i : p.N - 1;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        d.w[i][c] = *reinterpret_cast<const u32x4*>(wp[c] + f * (p.K / 2));
        d.s[i][c] = static_cast<const T*>(p.scale)[f * groups + at[c]];
        d.z[i][c] = p.zero != nullptr ? p.zero[f * groups + at[c]] : uint8_t(8);
      }
    }
  };
  Four cur;
  fetch(n_wave, cur);
  for (int n = 0; n < per_wave; n += F) {
    Four nxt;
    if (n + F < per_wave) fetch(n_wave + n + F, nxt);
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
        const float z = -16.f - static_cast<float>(cur.z[i][c]), s = in[c] ? to_f32(cur.s[i][c]) : 0.f;
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
    cur = nxt;
  }
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
template <typename T, int GROUP, int M, typename TO>
int launch_few_k(const I4Args& a, hipStream_t s) {
  if (a.K <= 2048) return launch_few<T, GROUP, M, 1, 1, TO>(a, s);
  if constexpr (M == 1) {
    if (a.K <= 4096) return launch_few<T, GROUP, M, 2, 1, TO>(a, s);
    if (a.K <= 8192) return launch_few<T, GROUP, M, 2, 2, TO>(a, s);
    return launch_few<T, GROUP, M, 2, 4, TO>(a, s);
  } else {
    if (a.K <= 4096) return launch_few<T, GROUP, M, 1, 2, TO>(a, s);
    if (a.K <= 8192) return launch_few<T, GROUP, M, 1, 4, TO>(a, s);
    return launch_few<T, GROUP, M, 1, 8, TO>(a, s);
  }
}

template <typename T, int GROUP, int MT, int R, int NW, typename TO>
int launch_one(const I4Args& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.N + 16 * R - 1) / (16 * R)), static_cast<unsigned>((a.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((linear_i4_kernel<T, GROUP, MT, R, NW, TO>), grid, dim3(64 * NW), 0, s, a);
  return static_cast<int>(hipGetLastError());
}
template <typename T, int GROUP, int MT, typename TO>
int launch_nw(const I4Args& a, hipStream_t s) {
  [[maybe_unused]] const int64_t tiles = (a.N + 15) / 16, steps = (a.K + 127) / 128;
  if constexpr (MT == 1 && GROUP != 32) {
    // Two tiles a wave halve the loads of x: where two tiles a wave leave every CU work-groups (16 x 16384 x 4096
    // 16.7 us with two, 22.9 with one; 8 x 12288 x 4096 14.0 and 13.7; 7 x 4096 x 16384 38 and 19)
    if (a.M > 4 && tiles >= 768) return launch_one<T, GROUP, MT, 2, 4, TO>(a, s);
  }
  if constexpr (MT == 1) {
    return steps > 16 ? launch_one<T, GROUP, MT, 1, 8, TO>(a, s) : launch_one<T, GROUP, MT, 1, 4, TO>(a, s);
  } else {
    if constexpr (GROUP != 32) {
      // (32 x 8192 x 8192 27.8, 64 x 12288 x 4096 45.0 us with two tiles a wave, 36.2 and 51.1 with one)
      if (tiles >= 512) return launch_one<T, GROUP, MT, 2, 4, TO>(a, s);
    }
    return launch_one<T, GROUP, MT, 1, 4, TO>(a, s);
  }
}
template <typename T, int GROUP, typename TO>
int launch_mt(const I4Args& a, hipStream_t s) {
  // Up to four rows: linear_i4_few (against the MFMA kernel, us: 1 x 12288 x 4096 7.7 / 11.5, 2 x 9.4 / 11.7,
  // 4 x 12.9 / 13.0; 1 x 4096 x 16384, group 64, 10.2 / 17.3, 2 x 11.9 / 17.6, 4 x 15.6 / 18.7;
  // 4 x 11008 x 4096, group 32, 12.3 / 17.2; eight rows 18.4 / 14.4). Below 512 k most of a wave would idle.
  if (a.K >= 512 && a.K <= 16384) {
    if (a.M == 1) return launch_few_k<T, GROUP, 1, TO>(a, s);
    if (a.M == 2) return launch_few_k<T, GROUP, 2, TO>(a, s);
    if (a.M <= 4) return launch_few_k<T, GROUP, 4, TO>(a, s);
  }
  if (a.M <= 16) return launch_nw<T, GROUP, 1, TO>(a, s);
  if (a.M <= 32) return launch_nw<T, GROUP, 2, TO>(a, s);
  return launch_nw<T, GROUP, 4, TO>(a, s);
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

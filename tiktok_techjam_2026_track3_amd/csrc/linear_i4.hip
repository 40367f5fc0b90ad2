// Projection of a few rows with 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k] + b[n] with
// W[n, k] = s[n, k / GROUP] (q[n, k] - z[n, k / GROUP]), q in 0 .. 15, two to a byte (even k low).
//
// Bound by the weights' bytes: every 4-bit value is read once, straight into the registers of the
// lane that multiplies it, and rows of x ride along as the other operand of 16x16x32 MFMAs (A = x:
// 16 rows, B = weights: 16 features; a lane holds one feature, lane % 16, so its scale and zero are
// one scalar each, and D[m][n] of 4 rows of x). A work-group takes 16 features; its waves take
// contiguous ranges of k and add up through LDS.
//   Nibbles become operands without conversions: (w >> 4 i) & 0x000f000f put into the mantissa of
//   1024 (fp16) or 128 (bf16) is the number 1024 + q or 128 + q. fp16 subtracts 1024 + z, exactly
//   (packed); bf16 has no packed subtraction, so its sum over a group is corrected in fp32 by
//   (128 + z) sum x, with sum x from MFMAs against ones. x up to 2^119 is safe there (143 x GROUP
//   products are added up before the correction).
//   A lane's 16 bytes are 32 neighbouring k. For GROUP 128 the four lanes of a feature hold the
//   whole group and each word is one MFMA's operand as it is; for 32 and 64 the words change
//   places between the four lanes (4 lane swaps) so that one MFMA's 32 k are neighbours.
#include "common.h"

namespace {

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
  static constexpr uint32_t MAGIC = 0x64006400u;
};
template <>
struct Nib<__bf16> {
  using vec = bf16x8;
  static constexpr uint32_t MAGIC = 0x43004300u;
};
MI355_DEVINL f32x4 mma_i4(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
MI355_DEVINL f32x4 mma_i4(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// 8 nibbles of a word as an operand: elements 0 4 1 5 2 6 3 7
template <typename T>
MI355_DEVINL typename Nib<T>::vec nibbles(uint32_t w, f16x2 zz) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t two = ((w >> (4 * i)) & 0x000f000fu) | Nib<T>::MAGIC;
    if constexpr (__is_same(T, _Float16)) two = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, two) - zz);
    r[i] = two;
  }
  return __builtin_bit_cast(typename Nib<T>::vec, r);
}
// 8 elements in the order 0 4 1 5 2 6 3 7
MI355_DEVINL u32x4 nibble_order(u32x4 v) {
  return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
               __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// MT tiles of 16 rows of x
template <typename T, int GROUP, int MT, int NW, typename TO>
__global__ __launch_bounds__(64 * NW) void linear_i4_kernel(I4Args p) {
  using vec = typename Nib<T>::vec;
  constexpr int GP = 128 / GROUP;  // groups of a 128-k step
  constexpr int U = 4;             // steps whose loads are in flight
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, feature = n0 + l16 < p.N ? n0 + l16 : p.N - 1;
  const int m0 = blockIdx.y * (16 * MT);
  const int groups = p.K / GROUP;
  const uint8_t* wrow = p.w + static_cast<int64_t>(feature) * (p.K / 2);
  const T* srow = static_cast<const T*>(p.scale) + static_cast<int64_t>(feature) * groups;
  const uint8_t* zrow = p.zero != nullptr ? p.zero + static_cast<int64_t>(feature) * groups : nullptr;
  const int steps = (p.K + 127) / 128, per = (steps + NW - 1) / NW;
  const int s_begin = wave * per, s_end = s_begin + per < steps ? s_begin + per : steps;

  struct Step {
    u32x4 w;
    float s[GP];
    float z[GP];
  };
  auto fetch = [&](int s, Step& d) MI355_LAMBDA_INLINE {
    const int k = s * 128 + 32 * g;
    d.w = s < s_end && k < p.K ? *reinterpret_cast<const u32x4*>(wrow + k / 2) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < GP; ++i) {
      const int at = s * GP + i;
      const bool in = s < s_end && at < groups;
      d.s[i] = in ? to_f32(srow[at]) : 0.f;
      d.z[i] = in && zrow != nullptr ? static_cast<float>(zrow[at]) : 8.f;
    }
  };
  f32x4 total[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) total[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  vec ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.0f);

  auto compute = [&](int s, const Step& d) MI355_LAMBDA_INLINE {
    u32x4 w = d.w;
    if constexpr (GROUP != 128) {
      // words of the lanes g' become word g' of the lanes: a 4 x 4 transposition over (lane / 16, word)
      auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
      auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
      w = u32x4{c[0], c[1], e[0], e[1]};
    }
    f32x4 acc[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int i = m * GP / 4;  // the MFMA's group in the step
      if (m * GP % 4 == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const _Float16 z1 = static_cast<_Float16>(1024.f + d.z[i]);
      const vec wv = nibbles<T>(w[m], f16x2{z1, z1});
      const int k = s * 128 + (GROUP == 128 ? 32 * g + 8 * m : 32 * m + 8 * g);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        u32x4 xv = {0u, 0u, 0u, 0u};
        const int row = m0 + 16 * t + l16;
        if (row < p.M && k < p.K) xv = *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.x) + row * p.ldx + k);
        const vec xo = __builtin_bit_cast(vec, nibble_order(xv));
        acc[t] = mma_i4(xo, wv, acc[t]);
        if constexpr (__is_same(T, __bf16)) sum[t] = mma_i4(xo, ones, sum[t]);
      }
      if ((m + 1) * GP % 4 == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = acc[t][e];
            if constexpr (__is_same(T, __bf16)) v = __builtin_fmaf(sum[t][e], -128.f - d.z[i], v);
            total[t][e] = __builtin_fmaf(v, d.s[i], total[t][e]);
          }
      }
    }
  };
  Step cur[U], nxt[U];
#pragma unroll
  for (int u = 0; u < U; ++u) fetch(s_begin + u, cur[u]);
  for (int s = s_begin; s < s_end; s += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(s + U + u, nxt[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < s_end) compute(s + u, cur[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = nxt[u];
  }

  __shared__ f32x4 part[NW][MT][64];
  if constexpr (NW > 1) {
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = total[t];
    __syncthreads();
  }
  // wave t' adds up tiles t', t' + NW ..
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if (t % NW != wave) continue;
    f32x4 v = total[t];
    if constexpr (NW > 1) {
      v = part[0][t][lane];
#pragma unroll
      for (int w = 1; w < NW; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += part[w][t][lane][e];
    }
    if (n0 + l16 < p.N) {
      const float b = p.bias != nullptr ? p.bias[n0 + l16] : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = m0 + 16 * t + 4 * g + e;
        if (row < p.M) static_cast<TO*>(p.y)[row * p.ldy + n0 + l16] = from_f32<TO>(v[e] + b);
      }
    }
  }
}

template <typename T, int GROUP, int MT, typename TO>
int launch_nw(const I4Args& a, hipStream_t s) {
  const int64_t tiles = (a.N + 15) / 16, my = (a.M + 16 * MT - 1) / (16 * MT), steps = (a.K + 127) / 128;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(my));
  // waves that share a work-group's sum: as many as leave each 4 steps, until the CUs are full
  if (steps > 16 && tiles * my < 1024)
    hipLaunchKernelGGL((linear_i4_kernel<T, GROUP, MT, 8, TO>), grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((linear_i4_kernel<T, GROUP, MT, 4, TO>), grid, dim3(256), 0, s, a);
  return static_cast<int>(hipGetLastError());
}
template <typename T, int GROUP, typename TO>
int launch_mt(const I4Args& a, hipStream_t s) {
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
  if (M < 0 || N < 0 || K < 0 || M > (int64_t(1) << 20) || N > (int64_t(1) << 30) || K > (int64_t(1) << 30))
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

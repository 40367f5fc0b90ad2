// Rotation of pairs of a head's elements by position * frequency (rotary positions):
//   y1 = a (x1 cos t - x2 sin t),  y2 = a (x2 cos t + x1 sin t),  t = position * f_j,
// j-th pair (x_j, x_{j + rot / 2}) or (x_2j, x_2j+1); elements behind the first rot are copied. fp32, rounded once.
// Bound by the bytes of x and y: a thread computes the angles of its pairs once and walks over several heads with them, the
// loads of four under way and those of the first while it computes (4096 tokens of 16 heads of 64 in fp32 9.1 -> 8.0 us).
// 8192 tokens of 40 heads of 128 in bf16 28.3 us, 5.9 TB/s read and written; 5 tokens 3.6 us of the GPU.
#include "rotary.h"

namespace {

struct RotaryArgs {
  const void* x;
  void* y;
  const void* positions;
  const uint64_t* freqs;
  int64_t n1;            // tokens in a batch row
  int64_t tokens;        // all of them
  int64_t ps0, ps1;      // strides of positions: batch row, token
  int64_t xs0, xs1, xs2, ys0, ys1, ys2;
  int32_t heads, per, units, pair_units, rot;  // heads a thread takes; units of 2 VEC elements a head, of pairs first
  int32_t long_positions;
  float amplitude, sign;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// A thread: VEC pairs of a token in `per` heads. The two halves of a unit's elements are VEC neighbours at first and at
// second; pairs that are neighbours come as one run of 2 VEC, like the elements that are copied.
// AHEAD: heads whose loads a thread has under way, the first of them while it computes the angles.
// PAST: 16-byte stores past the L2s, for outputs larger than those (PAST_CACHES).
template <typename T, int VEC, bool INTERLEAVED, int AHEAD, bool PAST>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  const int unit = static_cast<int>(threadIdx.x) % p.units;
  const int local = static_cast<int>(threadIdx.x) / p.units, tpb = 256 / p.units;
  if (local >= tpb) return;
  const int h0 = blockIdx.y * p.per, h1 = h0 + p.per < p.heads ? h0 + p.per : p.heads;
  const bool pairs = unit < p.pair_units;
  const int first = INTERLEAVED || !pairs ? unit * 2 * VEC : unit * VEC;
  const int second = INTERLEAVED || !pairs ? first + VEC : first + p.rot / 2;
  uint64_t f[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = pairs ? p.freqs[unit * VEC + i] : 0;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * tpb + local; t < p.tokens; t += static_cast<int64_t>(gridDim.x) * tpb) {
    const int64_t b = t / p.n1, s = t - b * p.n1;
    const int64_t at = b * p.ps0 + s * p.ps1;
    const int64_t position = p.long_positions ? static_cast<const int64_t*>(p.positions)[at]
                                              : static_cast<const int32_t*>(p.positions)[at];
    const T* x = static_cast<const T*>(p.x) + b * p.xs0 + s * p.xs1;
    T* y = static_cast<T*>(p.y) + b * p.ys0 + s * p.ys1;
    Vec<T, VEC> u[AHEAD][2];
    const auto fetch = [&](int h) MI355_LAMBDA_INLINE {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const T* row = x + (h + k < h1 ? h + k : h) * p.xs2;
        u[k][0] = *reinterpret_cast<const Vec<T, VEC>*>(row + first);
        u[k][1] = *reinterpret_cast<const Vec<T, VEC>*>(row + second);
      }
    };
    fetch(h0);
    float si[VEC], co[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sincos_of_turn(position, f[i], si[i], co[i]);
      si[i] *= p.sign * p.amplitude;
      co[i] *= p.amplitude;
    }
    for (int h = h0; h < h1; h += AHEAD) {
      if (h != h0) fetch(h);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (h + k >= h1) break;
        if (pairs) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            T& a = INTERLEAVED ? u[k][2 * i / VEC].v[2 * i % VEC] : u[k][0].v[i];
            T& c = INTERLEAVED ? u[k][(2 * i + 1) / VEC].v[(2 * i + 1) % VEC] : u[k][1].v[i];
            const float xa = to_f32(a), xc = to_f32(c);
            a = from_f32<T>(__builtin_fmaf(xa, co[i], -xc * si[i]));
            c = from_f32<T>(__builtin_fmaf(xc, co[i], xa * si[i]));
          }
        }
        T* row = y + (h + k) * p.ys2;
        if constexpr (PAST) {
          __builtin_nontemporal_store(__builtin_bit_cast(u32x4, u[k][0]), reinterpret_cast<u32x4*>(row + first));
          __builtin_nontemporal_store(__builtin_bit_cast(u32x4, u[k][1]), reinterpret_cast<u32x4*>(row + second));
        } else {
          *reinterpret_cast<Vec<T, VEC>*>(row + first) = u[k][0];
          *reinterpret_cast<Vec<T, VEC>*>(row + second) = u[k][1];
        }
      }
    }
  }
}

// Outputs of this many bytes and more are stored past the L2s, which hold 32 MiB together and would be written back at the
// kernel's end. Measured (us, past them / through them): 84 MB (8192 tokens, 40 heads of 128) 28.3 / 37.4, 16.8 MB 9.1 / 9.0,
// 9.6 MB 9.9 / 8.2. (x past them as well: 35.0 and 17.6 where it is in the last-level cache from before.)
constexpr int64_t PAST_CACHES = int64_t(32) << 20;

template <typename T, int VEC>
int launch(RotaryArgs& p, int64_t head_dim, bool interleaved, hipStream_t s) {
  p.units = static_cast<int32_t>(head_dim / (2 * VEC));
  p.pair_units = p.rot / (2 * VEC);
  const int64_t tpb = 256 / p.units, rows = (p.tokens + tpb - 1) / tpb;
  // heads a thread takes: as many as leave four work-groups a CU, up to 8
  p.per = 8;
  while (p.per > 1 && rows * ((p.heads + p.per - 1) / p.per) < 1024) p.per /= 2;
  const dim3 grid(static_cast<uint32_t>(rows < (1 << 20) ? rows : (1 << 20)), static_cast<uint32_t>((p.heads + p.per - 1) / p.per));
  const bool past = sizeof(T) * VEC == 16 && p.tokens * p.heads * head_dim * static_cast<int64_t>(sizeof(T)) >= PAST_CACHES;
  constexpr bool WHOLE = sizeof(T) * VEC == 16;
  if (past && interleaved)
    rotary_kernel<T, VEC, true, 4, WHOLE><<<grid, 256, 0, s>>>(p);
  else if (past)
    rotary_kernel<T, VEC, false, 4, WHOLE><<<grid, 256, 0, s>>>(p);
  else if (p.per >= 4 && interleaved)
    rotary_kernel<T, VEC, true, 4, false><<<grid, 256, 0, s>>>(p);
  else if (p.per >= 4)
    rotary_kernel<T, VEC, false, 4, false><<<grid, 256, 0, s>>>(p);
  else if (interleaved)
    rotary_kernel<T, VEC, true, 1, false><<<grid, 256, 0, s>>>(p);
  else
    rotary_kernel<T, VEC, false, 1, false><<<grid, 256, 0, s>>>(p);
  return static_cast<int>(hipGetLastError());
}

template <typename T>
int launch_vec(RotaryArgs& p, int64_t head_dim, bool interleaved, int vec, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch<T, 8>(p, head_dim, interleaved, s);
  return vec == 4 ? launch<T, 4>(p, head_dim, interleaved, s) : launch<T, 1>(p, head_dim, interleaved, s);
}

}  // namespace

extern "C" int mi355_rotary(int dtype, const void* X, void* Y, const void* positions, int positions_64,
                            const uint64_t* frequencies, float amplitude, const int64_t* sizes, const int64_t* strides,
                            int interleaved, int inverse, void* stream) {
  if (!sizes || !strides) return MI355_E_NULL_POINTER;
  const int64_t n0 = sizes[0], n1 = sizes[1], heads = sizes[2], head_dim = sizes[3], rot_dim = sizes[4];
  const int64_t *position_strides = strides, *x_strides = strides + 2, *y_strides = strides + 5;
  if (n0 < 0 || n1 < 0 || heads < 0 || n0 > (int64_t(1) << 31) || n1 > (int64_t(1) << 31) || n0 * n1 > (int64_t(1) << 31) ||
      heads > 65535)
    return MI355_E_BAD_SIZE;
  if (head_dim < 2 || head_dim > 512 || head_dim % 2 || rot_dim < 2 || rot_dim > head_dim || rot_dim % 2) return MI355_E_HEAD_DIM;
  if (dtype != MI355_F32 && dtype != MI355_F16 && dtype != MI355_BF16) return MI355_E_BAD_DTYPE;
  if (n0 * n1 * heads == 0) return MI355_OK;
  if (!X || !Y || !positions || !frequencies) return MI355_E_NULL_POINTER;
  RotaryArgs p{};
  p.x = X;
  p.y = Y;
  p.positions = positions;
  p.freqs = frequencies;
  p.n1 = n1;
  p.tokens = n0 * n1;
  p.ps0 = position_strides[0];
  p.ps1 = position_strides[1];
  p.xs0 = x_strides[0];
  p.xs1 = x_strides[1];
  p.xs2 = x_strides[2];
  p.ys0 = y_strides[0];
  p.ys1 = y_strides[1];
  p.ys2 = y_strides[2];
  p.heads = static_cast<int32_t>(heads);
  p.rot = static_cast<int32_t>(rot_dim);
  p.long_positions = positions_64;
  p.amplitude = amplitude;
  p.sign = inverse ? -1.0f : 1.0f;
  // the widest unit that every run of elements starts at a multiple of
  const auto fits = [&](int64_t vec) {
    const int64_t bytes = vec * (dtype == MI355_F32 ? 4 : 2);
    bool ok = rot_dim % (2 * vec) == 0 && head_dim % (2 * vec) == 0 && reinterpret_cast<uintptr_t>(X) % bytes == 0 &&
              reinterpret_cast<uintptr_t>(Y) % bytes == 0;
    for (int i = 0; i < 3; ++i) ok = ok && x_strides[i] % vec == 0 && y_strides[i] % vec == 0;
    return ok;
  };
  const auto s = static_cast<hipStream_t>(stream);
  const int vec = dtype != MI355_F32 && fits(8) ? 8 : fits(4) ? 4 : 1;
  if (dtype == MI355_F32) return launch_vec<float>(p, head_dim, interleaved, vec, s);
  if (dtype == MI355_F16) return launch_vec<_Float16>(p, head_dim, interleaved, vec, s);
  return launch_vec<__bf16>(p, head_dim, interleaved, vec, s);
}

// New tokens' K and V into the pages of an e4m3 cache, K rotated by its position on the way, and the queries of the same
// tokens rotated in the same launch.
//
// A work-group has a block of 16 positions of one sequence. It computes the angles of the block's new tokens once,
// into LDS; then a wave takes a K/V head's rows at a time: rotate, largest magnitude of all, scale, convert, store;
// the queries are rotated by all threads. For a block with older tokens the scale can only grow; when it does, the
// wave converts their bytes to the new one. Nothing else writes that block and head, so there are no atomics.
//   scale = the least power of two with max|x| <= 448 scale (448: e4m3's largest), at least 2^-118;
//   byte = e4m3(x / scale), nearest, ties to even; infinities and NaN are held as NaN and do not count for the scale.
// Bound by bytes in long prompts (16 bits in, 8 out, the queries in and out: 11 700 tokens of 32 query and 8 K/V heads of 128
// 52 us, 4.7 TB/s), by the chain of its loads (lengths, page, old scale) for single tokens (64 sequences 5.9 us of the GPU).
#include "paged.h"
#include "rotary.h"

namespace {

using paged::BLOCK;
constexpr int AHEAD = 4;  // rows of queries whose loads a thread has under way

struct AppendArgs {
  paged::Cache cache;
  paged::Batch batch;
  const void *k, *v, *q;
  void* qo;
  int64_t kt, kh, vt, vh, qt, qh, ot, oh;  // token and head strides in elements
  const uint64_t* freqs;                   // NULL: no rotation
  float amplitude;
  int32_t rot, interleaved, heads, blocks, slices, zero_tail;
};

MI355_DEVINL float wave_max(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}

// four floats as e4m3 bytes
MI355_DEVINL uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// Rotates 8 elements of a token's head: four pairs (a_i, b_i), a the first four and b the last four of x, or
// neighbours where interleaved.
template <bool INTERLEAVED>
MI355_DEVINL void rotate8(float (&x)[8], const float2* cs) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float& a = x[INTERLEAVED ? 2 * i : i];
    float& b = x[INTERLEAVED ? 2 * i + 1 : 4 + i];
    const float a0 = a, b0 = b;
    a = __builtin_fmaf(a0, cs[i].x, -b0 * cs[i].y);
    b = __builtin_fmaf(b0, cs[i].x, a0 * cs[i].y);
  }
}

// The two runs of 4 elements that unit c of a head's row has: for pairs across half the rotated part, they are apart.
template <bool INTERLEAVED>
MI355_DEVINL void runs_of(int c, int rot, int& first, int& second) {
  if (!INTERLEAVED && c < rot / 8) {
    first = 4 * c;
    second = 4 * c + rot / 2;
  } else {
    first = 8 * c;
    second = first + 4;
  }
}

// PAST: past the caches (PAST_CACHES)
template <bool PAST, typename V>
MI355_DEVINL V load(const void* at) {
  if constexpr (PAST) return __builtin_nontemporal_load(static_cast<const V*>(at));
  return *static_cast<const V*>(at);
}
template <bool PAST, typename V>
MI355_DEVINL void store(V v, void* at) {
  if constexpr (PAST)
    __builtin_nontemporal_store(v, static_cast<V*>(at));
  else
    *static_cast<V*>(at) = v;
}

template <typename T>
MI355_DEVINL void load8(const T* row, int first, int second, float (&x)[8]) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  const V4 a = *reinterpret_cast<const V4*>(row + first), b = *reinterpret_cast<const V4*>(row + second);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = to_f32(static_cast<T>(a[i]));
    x[4 + i] = to_f32(static_cast<T>(b[i]));
  }
}

// UNITS: units of 8 elements that a lane has at most. A wave takes 64 / (head_dim / 8) rows of a head at a time (lanes that
// are left over idle), so that a lane's unit of a row is the same in all of them.
template <typename T, int UNITS, bool INTERLEAVED, bool PAST>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs p) {
  extern __shared__ float2 angles[];  // [16][rot / 2] of the new tokens
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x % p.slices, at = blockIdx.x / p.slices;
  const int b = at / p.blocks, nth = at % p.blocks;
  const paged::Sequence s = paged::sequence_of(p.batch, b);
  if (p.zero_tail) {  // rows that no sequence has: those behind all by every work-group, a sequence's by its own
    const auto zero = [&](int64_t t, int i0, int step) MI355_LAMBDA_INLINE {
      for (int i = i0; i < p.heads * p.cache.head_dim; i += step)
        static_cast<T*>(p.qo)[t * p.ot + (i / p.cache.head_dim) * p.oh + i % p.cache.head_dim] = T(0.0f);
    };
    for (int64_t t = paged::tail_of(p.batch) + blockIdx.x; t < p.batch.tokens; t += gridDim.x) zero(t, tid, 256);
    const int worker = nth * p.slices + slice, workers = p.blocks * p.slices;
    const auto of_wave = [&](int64_t t) MI355_LAMBDA_INLINE { zero(t, lane, 64); };
    if (b == 0 && s.first > 0) paged::zero_rows(p.batch, 0, s.first, worker, workers, of_wave);
    if (s.cut > 0) paged::zero_rows(p.batch, s.first + s.n, static_cast<int64_t>(s.first) + s.n + s.cut, worker, workers, of_wave);
  }
  const int64_t begin = static_cast<int64_t>(s.len) - s.n;  // position of the first new token
  const int64_t block = (begin >> 4) + nth;                 // (floor: positions can be negative)
  const int64_t base = block * BLOCK;
  const int t0 = begin > base ? static_cast<int>(begin - base) : 0;
  const int64_t left = s.len - base;
  const int t1 = left < BLOCK ? static_cast<int>(left) : BLOCK;  // new tokens t0 .. t1 of the block
  if (t1 <= t0) return;
  const int hd = p.cache.head_dim, hu = hd / 8, half = p.rot / 2, nt = t1 - t0;
  const int64_t token0 = s.first + (base - begin);  // token of the block's position 0 (t0 and later ones exist)

  if (p.freqs != nullptr) {
    for (int i = tid; i < nt * half; i += 256) {
      const int t = i / half, j = i - t * half;
      float si, co;
      sincos_of_turn(base + t0 + t, p.freqs[j], si, co);
      angles[t * half + j] = make_float2(co * p.amplitude, si * p.amplitude);
    }
    __syncthreads();
  }

  // the page that holds the block
  int page = -1;
  if (block >= 0 && (base >> p.cache.page_shift) < p.batch.width) page = p.batch.table[b * p.batch.table_stride + (base >> p.cache.page_shift)];
  if (page >= 0 && page < p.cache.pages) {
    const int per = 64 / hu, row0 = lane / hu, c = lane - row0 * hu;
    const int in_page = static_cast<int>(base & ((1 << p.cache.page_shift) - 1));
    for (int item = wave + 4 * slice; item < 2 * p.cache.kv_heads; item += 4 * p.slices) {
      const bool is_v = item >= p.cache.kv_heads;
      const int h = is_v ? item - p.cache.kv_heads : item;
      const T* src = is_v ? static_cast<const T*>(p.v) + h * p.vh : static_cast<const T*>(p.k) + h * p.kh;
      const int64_t ts = is_v ? p.vt : p.kt;
      const int64_t head = static_cast<int64_t>(page) * p.cache.kv_heads + h;
      uint8_t* dst = (is_v ? p.cache.v : p.cache.k) + ((head << p.cache.page_shift) + in_page) * hd;
      float* scale = (is_v ? p.cache.vs : p.cache.ks) + ((head << p.cache.page_shift) + in_page) / BLOCK;
      const float old = t0 > 0 ? *scale : 0.0f;
      const bool turn = !is_v && p.freqs != nullptr;
      const int rot = turn ? p.rot : 0;
      float x[UNITS][8], top = 0.0f;
      int first, second;
      runs_of<INTERLEAVED>(c, rot, first, second);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int t = row0 + per * u;
        if (row0 < per && t < nt) {
          load8(src + (token0 + t0 + t) * ts, first, second, x[u]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[u][e] = 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int t = row0 + per * u;
        if (c < rot / 8 && row0 < per && t < nt) rotate8<INTERLEAVED>(x[u], angles + t * half + 4 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = __builtin_fabsf(x[u][e]);
          top = m < __builtin_huge_valf() && m > top ? m : top;
        }
      }
      top = fmaxf(wave_max(top), 0x1p-110f);
      // 448 = 1.75 * 2^8: the exponent of `top` less 8, and one more where its mantissa is over 1.75
      const uint32_t bits = __float_as_uint(top);
      const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased
      float s_new = __uint_as_float(static_cast<uint32_t>(e) << 23);
      const bool grows = t0 > 0 && s_new > old;
      s_new = s_new > old ? s_new : old;
      const float inv = 1.0f / s_new;
      if (grows) {
        const float ratio = old * inv;
        for (int i = lane; i < t0 * hu; i += 64) {
          uint32_t* w = reinterpret_cast<uint32_t*>(dst) + 2 * i;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[r], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[r], true);
            w[r] = to_e4m3(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int t = row0 + per * u;
        if (row0 < per && t < nt) {
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {  // (an infinity to NaN: inf - inf)
            const float w = x[u][k] * inv;
            y[k] = __builtin_fabsf(w) < __builtin_huge_valf() ? w : w - w;
          }
          uint8_t* row = dst + (t0 + t) * hd;
          *reinterpret_cast<uint32_t*>(row + first) = to_e4m3(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint32_t*>(row + second) = to_e4m3(y[4], y[5], y[6], y[7]);
        }
      }
      if (lane == 0) *scale = s_new;
    }
  }

  if (p.q != nullptr) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    const int per = 256 / hu, row0 = tid / hu, c = tid - row0 * hu;
    if (row0 >= per) return;
    int first, second;
    runs_of<INTERLEAVED>(c, p.rot, first, second);
    const bool turn = c < p.rot / 8;
    // rows (token, head) of the block's new tokens, heads fastest: AHEAD of them under way
    const int rows = nt * p.heads, step = per * p.slices;
    for (int row = row0 + per * slice; row < rows; row += AHEAD * step) {
      V4 a[AHEAD], b4[AHEAD];
      int t[AHEAD], h[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int r = row + k * step < rows ? row + k * step : row;
        t[k] = r / p.heads;
        h[k] = r - t[k] * p.heads;
        const T* src = static_cast<const T*>(p.q) + (token0 + t0 + t[k]) * p.qt + h[k] * p.qh;
        a[k] = load<PAST, V4>(src + first);
        b4[k] = load<PAST, V4>(src + second);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (row + k * step >= rows) break;
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = to_f32(static_cast<T>(a[k][i]));
          x[4 + i] = to_f32(static_cast<T>(b4[k][i]));
        }
        if (turn) rotate8<INTERLEAVED>(x, angles + t[k] * half + 4 * c);
        T* dst = static_cast<T*>(p.qo) + (token0 + t0 + t[k]) * p.ot + h[k] * p.oh;
        store<PAST>(V4{from_f32<T>(x[0]), from_f32<T>(x[1]), from_f32<T>(x[2]), from_f32<T>(x[3])}, dst + first);
        store<PAST>(V4{from_f32<T>(x[4]), from_f32<T>(x[5]), from_f32<T>(x[6]), from_f32<T>(x[7])}, dst + second);
      }
    }
  }
}

// Queries of this many bytes and more are loaded and stored past the L2s, which hold 32 MiB together: 24 prompts of 33 to 2011
// tokens (32/8 heads of 128, 130 MB) 59.3 -> 51.9 us. (K and V too: 57.4.) What goes into the cache's pages stays
// in them for the attention.
constexpr int64_t PAST_CACHES = int64_t(32) << 20;

template <typename T, int UNITS>
int launch(const AppendArgs& p, hipStream_t s) {
  const uint32_t grid = static_cast<uint32_t>(p.batch.B) * p.blocks * p.slices;
  const size_t lds = p.freqs ? size_t(BLOCK) * (p.rot / 2) * sizeof(float2) : 0;
  const bool past = p.q && int64_t(p.batch.tokens) * p.heads * p.cache.head_dim * 2 >= PAST_CACHES;
  if (p.interleaved && past)
    paged_append_kernel<T, UNITS, true, true><<<grid, 256, lds, s>>>(p);
  else if (p.interleaved)
    paged_append_kernel<T, UNITS, true, false><<<grid, 256, lds, s>>>(p);
  else if (past)
    paged_append_kernel<T, UNITS, false, true><<<grid, 256, lds, s>>>(p);
  else
    paged_append_kernel<T, UNITS, false, false><<<grid, 256, lds, s>>>(p);
  return static_cast<int>(hipGetLastError());
}

template <typename T>
int launch_dim(const AppendArgs& p, hipStream_t s) {
  if (p.cache.head_dim <= 64) return launch<T, 2>(p, s);
  if (p.cache.head_dim <= 128) return launch<T, 4>(p, s);
  return launch<T, 8>(p, s);
}

}  // namespace

extern "C" int mi355_paged_append(int dtype, const void* K, const void* V, const void* Q, void* Q_out, uint8_t* cache_k,
                                  uint8_t* cache_v, float* k_scale, float* v_scale, const int32_t* table,
                                  const int32_t* lens, const int32_t* offsets, const int64_t* sizes, const int64_t* strides,
                                  const uint64_t* frequencies, int64_t rot_dim, int interleaved, float amplitude,
                                  int zero_tail, void* stream) {
  if (!sizes || !strides) return MI355_E_NULL_POINTER;
  const paged::Sizes z = *reinterpret_cast<const paged::Sizes*>(sizes);
  if (const int st = paged::check(dtype, z)) return st;
  if (z.B * z.most == 0 || z.tokens == 0) return MI355_OK;
  if (!K || !V || !lens || (z.pages > 0 && (!cache_k || !cache_v || !k_scale || !v_scale)) || (z.width > 0 && !table))
    return MI355_E_NULL_POINTER;
  if (Q && (!Q_out || !frequencies)) return MI355_E_NULL_POINTER;
  if (!offsets && z.B * z.most > z.tokens) return MI355_E_BAD_SIZE;
  if (frequencies && (rot_dim < 8 || rot_dim > z.head_dim || rot_dim % 8)) return MI355_E_HEAD_DIM;
  const auto even = [](const void* base, const int64_t* st) {
    return aligned16(base) && st[0] % 8 == 0 && st[1] % 8 == 0;
  };
  if (!even(K, strides) || !even(V, strides + 2) || (Q && (!even(Q, strides + 4) || !even(Q_out, strides + 6))) ||
      !aligned16(cache_k) || !aligned16(cache_v))
    return MI355_E_ALIGNMENT;
  AppendArgs p{};
  p.cache = paged::cache_of(z, cache_k, cache_v, k_scale, v_scale);
  p.batch = paged::batch_of(z, table, lens, offsets);
  p.k = K;
  p.v = V;
  p.q = Q;
  p.qo = Q_out;
  p.kt = strides[0];
  p.kh = strides[1];
  p.vt = strides[2];
  p.vh = strides[3];
  if (Q) {
    p.qt = strides[4];
    p.qh = strides[5];
    p.ot = strides[6];
    p.oh = strides[7];
  }
  p.freqs = frequencies;
  p.amplitude = amplitude;
  p.rot = frequencies ? static_cast<int32_t>(rot_dim) : 0;
  p.interleaved = interleaved;
  p.heads = static_cast<int32_t>(z.heads);
  p.zero_tail = Q && zero_tail && (offsets || z.tokens > z.B * z.most);
  p.blocks = static_cast<int32_t>((z.most + 2 * BLOCK - 2) / BLOCK);
  // work-groups that share a block's heads: enough for 8192 of them, 32 a CU, no more than heads can use
  const int64_t groups = z.B * p.blocks;
  const int64_t slices = (8192 + groups - 1) / groups, useful = (2 * z.kv_heads + 3) / 4;
  p.slices = static_cast<int32_t>(slices < useful ? slices : useful);
  if (groups * p.slices >= (int64_t(1) << 23)) return MI355_E_BAD_SIZE;  // 2^31 threads
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == MI355_F16 ? launch_dim<_Float16>(p, s) : launch_dim<__bf16>(p, s);
}

// Attention of a batch's new tokens against a prefix that all sequences share and their own caches.
//
// The softmax over prefix ++ own cache is split over ranges of keys: attn_rows_kernel computes each
// range's unnormalised output, maximum and sum, for the prefix with the rows of the whole batch (its
// K and V are read once for all sequences, and as many tiles of rows share them as matrix rows), for
// the own caches with one sequence's rows; combine_splits joins a row's ranges:
//   M = max mu_s, o = sum_s 2^(mu_s - M) O_s / sum_s 2^(mu_s - M) l_s.
#include <algorithm>

#include "attn_rows.h"

namespace {

struct Shape {
  int64_t B, n_q, H, Hkv, hd, prefix, room;
  int64_t rows() const { return B * n_q * H; }
};

// How the work is split: work-groups of the prefix (tile rows) and of the caches, and their splits.
struct Split {
  int prefix_rows, own_rows;
  int64_t prefix_chunk, own_chunk, prefix_splits, own_splits;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Split split_of(const Shape& s) {
  Split d{};
  const int64_t G = s.H / s.Hkv, pr = s.B * s.n_q * G, orows = s.n_q * G;
  d.prefix_rows = pr <= 16 ? 16 : pr <= 32 ? 32 : pr <= 64 ? 64 : 128;
  d.own_rows = orows <= 16 ? 16 : 32;
  const auto chunk = [](int64_t keys, int64_t groups, int64_t want, int64_t least) {
    const int64_t splits = std::max<int64_t>(1, want / std::max<int64_t>(1, groups));
    return std::max(least, ceil_div(ceil_div(keys, splits), 64) * 64);
  };
  d.prefix_chunk = chunk(s.prefix, ceil_div(pr, d.prefix_rows) * s.Hkv, d.prefix_rows <= 32 ? 1280 : 512, 128);
  d.own_chunk = chunk(s.room, s.B * ceil_div(orows, d.own_rows) * s.Hkv, 1280, 128);
  d.prefix_splits = ceil_div(s.prefix, d.prefix_chunk);
  d.own_splits = ceil_div(s.room, d.own_chunk);
  return d;
}

int check(const Shape& s) {
  if (s.B < 0 || s.n_q < 0 || s.H <= 0 || s.Hkv <= 0 || s.H % s.Hkv != 0 || s.H > 65535 || s.prefix < 0 ||
      s.room < 0 || s.prefix >= (int64_t(1) << 30) || s.room >= (int64_t(1) << 30) || s.B > 65535 ||
      s.n_q > 65535 || s.B * s.n_q * s.H >= (int64_t(1) << 30))
    return MI355_E_BAD_SIZE;
  switch (s.hd) {
    case 16: case 32: case 48: case 64: case 80: case 96: case 128: case 192: case 256: break;
    default: return MI355_E_HEAD_DIM;
  }
  return MI355_OK;
}

struct CombineArgs {
  const float *part, *ml;
  void* o;
  int64_t ob, ot, oh;
  int64_t rows;
  int32_t n_q, H, hd;
  int32_t prefix_splits, own_chunk, prefix, room;
  const int32_t* lens;
};

// A wave per row: lane x holds elements 4 x .. of hd <= 256.
template <typename T>
__global__ __launch_bounds__(256) void combine_splits(CombineArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int head = static_cast<int>(row % p.H);
  const int64_t bt = row / p.H;
  const int b = static_cast<int>(bt / p.n_q), t = static_cast<int>(bt % p.n_q);
  const int given = p.lens[b];
  const int len = given < 0 ? 0 : (given < p.room ? given : p.room);
  const int seen = len - p.n_q + t + 1;  // own keys of this token
  const int splits = p.prefix_splits + (seen > 0 ? (seen + p.own_chunk - 1) / p.own_chunk : 0);
  typedef T t4 __attribute__((ext_vector_type(4)));
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = NEG_INF, l = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float ms = p.ml[2 * (s * p.rows + row)], ls = p.ml[2 * (s * p.rows + row) + 1];
    if (ms == NEG_INF) continue;  // no finite score there
    const float m2 = vmax(m, ms);
    const float a = m == NEG_INF ? 0.f : fast_exp2(m - m2), w = fast_exp2(ms - m2);
    l = __builtin_fmaf(l, a, ls * w);
    if (4 * lane < p.hd) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p.part + (s * p.rows + row) * p.hd + 4 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(acc[e], a, x[e] * w);
    }
    m = m2;
  }
  if (4 * lane >= p.hd) return;
  const bool none = p.prefix == 0 && seen <= 0;  // no key: zeros (no finite score: 0 / 0)
  t4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(none ? 0.f : acc[e] / l);
  *reinterpret_cast<t4*>(static_cast<T*>(p.o) + b * p.ob + t * p.ot + head * p.oh + 4 * lane) = w;
}

template <typename T, int HD, int MODE>
int launch_rows(const rows::Args& a, int tile_rows, int64_t blocks, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(blocks));
  if (tile_rows == 16)
    hipLaunchKernelGGL((rows::attn_rows_kernel<T, HD, 1, 1, 32, 2, 1, 2, MODE>), grid, dim3(64), 0, s, a);
  else if (tile_rows == 32)
    hipLaunchKernelGGL((rows::attn_rows_kernel<T, HD, 1, 2, 32, 2, 1, 2, MODE>), grid, dim3(64), 0, s, a);
  else if constexpr (MODE == rows::PREFIX) {
    if (tile_rows == 64)
      hipLaunchKernelGGL((rows::attn_rows_kernel<T, HD, 4, 1, HD <= 128 ? 64 : 32, 2, 1, 2, MODE>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((rows::attn_rows_kernel<T, HD, 4, 2, HD <= 128 ? 64 : 32, 2, HD <= 128 ? 2 : 1, 1, MODE>), grid, dim3(256), 0, s, a);
  }
  return static_cast<int>(hipGetLastError());
}

template <typename T, int HD>
int launch_hd(rows::Args a, const rows::Args& own, const Shape& s, const Split& d, hipStream_t st) {
  const int64_t G = s.H / s.Hkv;
  if (s.prefix > 0) {
    a.chunk = static_cast<int32_t>(d.prefix_chunk);
    a.splits = static_cast<int32_t>(d.prefix_splits);
    a.row_tiles = static_cast<int32_t>(ceil_div(s.B * s.n_q * G, d.prefix_rows));
    const int e = launch_rows<T, HD, rows::PREFIX>(a, d.prefix_rows, s.Hkv * d.prefix_splits * a.row_tiles, st);
    if (e) return e;
  }
  if (s.room > 0) {
    rows::Args w = own;
    w.chunk = static_cast<int32_t>(d.own_chunk);
    w.splits = static_cast<int32_t>(d.own_splits);
    w.row_tiles = static_cast<int32_t>(ceil_div(s.n_q * G, d.own_rows));
    w.part0 = static_cast<int32_t>(d.prefix_splits);
    return launch_rows<T, HD, rows::OWN>(w, d.own_rows, s.Hkv * d.own_splits * w.row_tiles * s.B, st);
  }
  return MI355_OK;
}

template <typename T>
int launch(const rows::Args& a, const rows::Args& own, const CombineArgs& c, const Shape& s, const Split& d, hipStream_t st) {
  int e = MI355_E_HEAD_DIM;
  switch (s.hd) {
    case 16: e = launch_hd<T, 16>(a, own, s, d, st); break;
    case 32: e = launch_hd<T, 32>(a, own, s, d, st); break;
    case 48: e = launch_hd<T, 48>(a, own, s, d, st); break;
    case 64: e = launch_hd<T, 64>(a, own, s, d, st); break;
    case 80: e = launch_hd<T, 80>(a, own, s, d, st); break;
    case 96: e = launch_hd<T, 96>(a, own, s, d, st); break;
    case 128: e = launch_hd<T, 128>(a, own, s, d, st); break;
    case 192: e = launch_hd<T, 192>(a, own, s, d, st); break;
    case 256: e = launch_hd<T, 256>(a, own, s, d, st); break;
  }
  if (e) return e;
  hipLaunchKernelGGL((combine_splits<T>), dim3(static_cast<unsigned>(ceil_div(c.rows, 4))), dim3(256), 0, st, c);
  return static_cast<int>(hipGetLastError());
}

}  // namespace

extern "C" int64_t mi355_attn_shared_prefix_workspace_bytes(int64_t B, int64_t n_q, int64_t heads,
                                                            int64_t kv_heads, int64_t head_dim,
                                                            int64_t prefix_len, int64_t room) {
  const Shape s{B, n_q, heads, kv_heads, head_dim, prefix_len, room};
  const int e = check(s);
  if (e) return e;
  const Split d = split_of(s);
  return (d.prefix_splits + d.own_splits) * s.rows() * (head_dim + 2) * 4;
}

extern "C" int mi355_attn_shared_prefix(int dtype, const void* Q, const void* K_prefix, const void* V_prefix,
                                        const void* K_own, const void* V_own, const int32_t* own_lens,
                                        void* O, int64_t B, int64_t n_q, int64_t heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t prefix_len, int64_t room,
                                        const int64_t* q_strides, const int64_t* kp_strides,
                                        const int64_t* vp_strides, const int64_t* ko_strides,
                                        const int64_t* vo_strides, const int64_t* o_strides, float scale,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  const Shape s{B, n_q, heads, kv_heads, head_dim, prefix_len, room};
  const int e = check(s);
  if (e) return e;
  if (dtype != MI355_F16 && dtype != MI355_BF16) return MI355_E_BAD_DTYPE;
  if (!(scale > 0.f) || scale > 1e30f) return MI355_E_UNSUPPORTED;
  if (s.rows() == 0) return MI355_OK;
  if (!Q || !O || !own_lens || !q_strides || !kp_strides || !vp_strides || !ko_strides || !vo_strides ||
      !o_strides || !workspace || (prefix_len > 0 && (!K_prefix || !V_prefix)) || (room > 0 && (!K_own || !V_own)))
    return MI355_E_NULL_POINTER;
  const Split d = split_of(s);
  if (workspace_bytes < (d.prefix_splits + d.own_splits) * s.rows() * (head_dim + 2) * 4) return MI355_E_BAD_SIZE;
  // token strides of K and V: rows that do not overlap, whose tiles' offsets fit 32 bits
  for (const int64_t t : {prefix_len > 0 ? kp_strides[0] : head_dim, prefix_len > 0 ? vp_strides[0] : head_dim,
                          room > 0 ? ko_strides[1] : head_dim, room > 0 ? vo_strides[1] : head_dim})
    if (t < head_dim || t > (int64_t(1) << 24)) return MI355_E_BAD_SIZE;
  for (int i = 0; i < 3; ++i) {
    if (q_strides[i] % 8 || ko_strides[i] % 8 || vo_strides[i] % 8) return MI355_E_ALIGNMENT;
    if (i < 2 && (kp_strides[i] % 8 || vp_strides[i] % 8)) return MI355_E_ALIGNMENT;
    if (o_strides[i] % 4) return MI355_E_ALIGNMENT;
  }
  if (!aligned16(Q) || !aligned16(K_prefix) || !aligned16(V_prefix) || !aligned16(K_own) || !aligned16(V_own) ||
      !aligned16(workspace) || (reinterpret_cast<uintptr_t>(O) & 7u) || (reinterpret_cast<uintptr_t>(own_lens) & 3u))
    return MI355_E_ALIGNMENT;
  const int64_t G = heads / kv_heads;
  if (kv_heads * d.prefix_splits * ceil_div(B * n_q * G, d.prefix_rows) > 0x7fffffffLL ||
      kv_heads * d.own_splits * ceil_div(n_q * G, d.own_rows) * B > 0x7fffffffLL)
    return MI355_E_BAD_SIZE;
  rows::Args a{};
  a.q = Q;
  a.qb = q_strides[0]; a.qt = q_strides[1]; a.qh = q_strides[2];
  a.c = scale * 1.4426950408889634f;
  a.G = static_cast<int32_t>(G);
  a.H = static_cast<int32_t>(heads);
  a.Hkv = static_cast<int32_t>(kv_heads);
  a.B = static_cast<int32_t>(B);
  a.n_q = static_cast<int32_t>(n_q);
  a.part = static_cast<float*>(workspace);
  a.ml = a.part + (d.prefix_splits + d.own_splits) * s.rows() * head_dim;
  rows::Args own = a;
  a.k = K_prefix; a.v = V_prefix;
  a.kt = kp_strides[0]; a.kh = kp_strides[1];
  a.vt = vp_strides[0]; a.vh = vp_strides[1];
  a.keys = static_cast<int32_t>(prefix_len);
  own.k = K_own; own.v = V_own;
  own.kb = ko_strides[0]; own.kt = ko_strides[1]; own.kh = ko_strides[2];
  own.vb = vo_strides[0]; own.vt = vo_strides[1]; own.vh = vo_strides[2];
  own.keys = static_cast<int32_t>(room);
  own.lens = own_lens;
  CombineArgs c{};
  c.part = a.part;
  c.ml = a.ml;
  c.o = O;
  c.ob = o_strides[0]; c.ot = o_strides[1]; c.oh = o_strides[2];
  c.rows = s.rows();
  c.n_q = a.n_q;
  c.H = a.H;
  c.hd = static_cast<int32_t>(head_dim);
  c.prefix_splits = static_cast<int32_t>(d.prefix_splits);
  c.own_chunk = static_cast<int32_t>(d.own_chunk);
  c.prefix = static_cast<int32_t>(prefix_len);
  c.room = static_cast<int32_t>(room);
  c.lens = own_lens;
  const auto st = static_cast<hipStream_t>(stream);
  return dtype == MI355_F16 ? launch<_Float16>(a, own, c, s, d, st) : launch<__bf16>(a, own, c, s, d, st);
}

// Attention of a batch's new tokens against a prefix that all sequences share and their own caches.
//
// The softmax over prefix ++ own cache is split over ranges of keys: attn_rows_kernel computes each
// range's unnormalised output, maximum and sum, for the prefix with the rows of the whole batch (its
// K and V are read once for all sequences, and as many tiles of rows share them as matrix rows), for
// the own caches with one sequence's rows; combine_splits joins a row's ranges:
//   M = max mu_s, o = sum_s 2^(mu_s - M) O_s / sum_s 2^(mu_s - M) l_s.
// Bound by bytes: K and V of the prefix once, of the caches as far as they are filled (16 sequences, 32/8 heads of
// 128, behind 65521 keys with caches of up to 4096: 84 us, 4.4 TB/s, 6 of them the join; 64 behind 8192 with up to
// 1024: 51 us, 3.3 TB/s, where the caches' lengths leave CUs idle at the end).
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
  bool whole;  // neither is split, nothing to join
};

// most splits of the prefix or of a cache, and of both together for one wave to join
constexpr int64_t MAX_SPLITS = 512;
// most work-groups (and rows, each joined by one) of a launch, which has at most 2^32 - 1 threads
constexpr int64_t MAX_BLOCKS = 0xffffffffLL / 256;
constexpr int WAVE_SPLITS = 32;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Split split_of(const Shape& s) {
  Split d{};
  const int64_t G = s.H / s.Hkv, pr = s.B * s.n_q * G, orows = s.n_q * G;
  d.prefix_rows = pr <= 16 ? 16 : pr <= 32 ? 32 : pr <= 64 ? 64 : 128;
  d.own_rows = orows <= 16 && d.prefix_rows != 32 ? 16 : 32;
  // Few keys for few work-groups: the joining launch (4 us and its place in the stream) costs more than reading the
  // prefix for every sequence (4 sequences, 8/2 heads of 64, behind 300 + 128 keys: 6.3 against 9.6 us).
  d.whole = orows <= 32 && s.prefix + s.room <= 1024 && s.B * s.Hkv <= 512;
  if (d.whole) {
    d.own_rows = orows <= 16 ? 16 : 32;
    return d;
  }
  // As many ranges as fill the work-groups that run at once (two a CU), half of them where the prefix has 64 rows
  // and more: there the waves share tiles (16 sequences, 32/8 heads of 128, behind 65521 keys: 88 us with one a
  // CU, 91 with two, 98 with four). With 128 rows (matrix work) each range writes 128 partial rows a head, so ranges are longer still where the caches
  // run beside them for long enough, at 40 keys of a range for each us of half-full caches at 5 TB/s (64
  // sequences, 32/8 heads of 128, behind 8192 keys, caches of up to 1024: 52 us with at least 1024 keys, 56 with
  // 256; 128 sequences behind 2048, up to 512: 43 and 49; but 27 and 33 with caches of 16; 24 x 4 tokens, 16/16
  // heads of 64, behind 2047, up to 777: 22 and 17).
  const auto chunk = [](int64_t keys, int64_t groups, int64_t want, int64_t least) {
    const int64_t splits = std::min(MAX_SPLITS, std::max<int64_t>(1, want / std::max<int64_t>(1, groups)));
    return std::max<int64_t>(least, ceil_div(ceil_div(keys, splits), 64) * 64);
  };
  const bool matrix = d.prefix_rows == 128;
  const int64_t beside = s.B * s.room * s.Hkv * s.hd * 4 / 250000;
  d.prefix_chunk = chunk(s.prefix, ceil_div(pr, d.prefix_rows) * s.Hkv, d.prefix_rows >= 64 ? 256 : 512,
                         matrix ? std::min<int64_t>(1024, std::max<int64_t>(256, beside / 64 * 64)) : 256);
  d.own_chunk = chunk(s.room, s.B * ceil_div(orows, d.own_rows) * s.Hkv, 512, 256);
  d.prefix_splits = ceil_div(s.prefix, d.prefix_chunk);
  d.own_splits = ceil_div(s.room, d.own_chunk);
  return d;
}

int check(const Shape& s) {
  if (s.B < 0 || s.n_q < 0 || s.H <= 0 || s.Hkv <= 0 || s.H % s.Hkv != 0 || s.H > 65535 || s.prefix < 0 ||
      s.room < 0 || s.prefix >= (int64_t(1) << 30) || s.room >= (int64_t(1) << 30) || s.B > 65535 ||
      s.n_q > 65535 || s.B * s.n_q * s.H > MAX_BLOCKS)
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

// W waves a row, W divides 4 rows' worth of them: first each lane takes splits of its own (maximum, then
// weights 2^(mu_s - M), left in LDS), then lanes of 4 elements each add up the weighted outputs, as many
// splits at a time as the waves have lanes for, and what they hold is added up through LDS.
template <typename T, int W>
__global__ __launch_bounds__(256) void combine_splits(CombineArgs p) {
  constexpr int RPG = 4 / W, NT = 64 * W;  // rows of a work-group, threads of a row
  __shared__ float weight[RPG][W == 1 ? WAVE_SPLITS : 2 * MAX_SPLITS];
  __shared__ float red[RPG][2][W];
  __shared__ f32x4 sums[RPG][NT];
  const int slot = threadIdx.x / NT, tid = threadIdx.x % NT, lane = threadIdx.x & 63, wave = tid >> 6;
  const int64_t given_row = static_cast<int64_t>(blockIdx.x) * RPG + slot;
  const int64_t row = given_row < p.rows ? given_row : p.rows - 1;  // (computed twice, stored once)
  const int head = static_cast<int>(row % p.H);
  const int64_t bt = row / p.H;
  const int b = static_cast<int>(bt / p.n_q), t = static_cast<int>(bt % p.n_q);
  const int given = p.lens[b];
  const int len = given < 0 ? 0 : (given < p.room ? given : p.room);
  const int seen = len - p.n_q + t + 1;  // own keys of this token
  const int splits = p.prefix_splits + (seen > 0 ? (seen + p.own_chunk - 1) / p.own_chunk : 0);
  float m = NEG_INF;
  for (int s = tid; s < splits; s += NT) m = vmax(m, p.ml[2 * (s * p.rows + row)]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = vmax(m, __shfl_xor(m, off));
  if constexpr (W > 1) {
    if (lane == 0) red[slot][0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = vmax(m, red[slot][0][i]);
  }
  float l = 0.f;
  for (int s = tid; s < splits; s += NT) {
    const float ms = p.ml[2 * (s * p.rows + row)], ls = p.ml[2 * (s * p.rows + row) + 1];
    const float w = fast_exp2(ms - m);
    weight[slot][s] = ms == NEG_INF ? NEG_INF : w;  // -inf: nothing there counts
    l = ms == NEG_INF ? l : __builtin_fmaf(ls, w, l);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off);
  if constexpr (W > 1) {
    if (lane == 0) red[slot][1][wave] = l;
  }
  __syncthreads();
  if constexpr (W > 1) {
    l = red[slot][1][0];
#pragma unroll
    for (int i = 1; i < W; ++i) l += red[slot][1][i];
  }
  const int per = p.hd / 4, at_once = NT / per, mine = tid / per, x = tid % per;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (mine < at_once) {
    const float* src = p.part + row * p.hd + 4 * x;
    const int64_t pitch = p.rows * p.hd;
    for (int s0 = mine; s0 < splits; s0 += 4 * at_once) {
      f32x4 v[4];
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = s0 + i * at_once;
        w[i] = s < splits ? weight[slot][s] : NEG_INF;
        v[i] = *reinterpret_cast<const f32x4*>(src + (s < splits ? s : s0) * pitch);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = w[i] == NEG_INF ? acc[e] : __builtin_fmaf(v[i][e], w[i], acc[e]);
    }
  }
  sums[slot][tid] = acc;
  __syncthreads();
  if (mine != 0 || given_row >= p.rows) return;
  for (int i = 1; i < at_once; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += sums[slot][i * per + x][e];
  const bool none = p.prefix == 0 && seen <= 0;  // no key: zeros (no finite score: 0 / 0)
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(none ? 0.f : acc[e] / l);
  *reinterpret_cast<t4*>(static_cast<T*>(p.o) + b * p.ob + t * p.ot + head * p.oh + 4 * x) = w;
}

// Both kinds of range in one launch, the prefix's (matrix work, where the batch is large) first, so that the
// caches' (memory) run beside them. PR, OR: rows of a prefix and of a cache work-group.
template <typename T, int HD, int PR, int OR>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_rows_prefix(rows::Args a, rows::Args own, unsigned n_prefix) {
  constexpr bool SPLIT = PR <= 32;  // few rows: the waves share out the keys
  constexpr int BN = SPLIT || HD > 128 ? 32 : 64, QG = SPLIT ? PR / 16 : PR / 64;
  constexpr int CHUNKS = rows::lds_chunks<HD, 4, 32, true>() > rows::lds_chunks<HD, 4, BN, SPLIT>()
                             ? rows::lds_chunks<HD, 4, 32, true>() : rows::lds_chunks<HD, 4, BN, SPLIT>();
  __shared__ u32x4 lds[CHUNKS];
  if (blockIdx.x < n_prefix)
    rows::attn_rows<T, HD, 4, QG, BN, SPLIT, PR <= 64 ? 2 : 1, rows::PREFIX>(a, lds, blockIdx.x);
  else
    rows::attn_rows<T, HD, 4, OR / 16, 32, true, 2, rows::OWN, sizeof(rows::Args)>(own, lds, blockIdx.x - n_prefix);
}

template <typename T, int HD, int PR, int OR>
void launch_one(const rows::Args& a, const rows::Args& own, int64_t n_prefix, int64_t n_own, hipStream_t st) {
  hipLaunchKernelGGL((attn_rows_prefix<T, HD, PR, OR>), dim3(static_cast<unsigned>(n_prefix + n_own)), dim3(256), 0, st,
                     a, own, static_cast<unsigned>(n_prefix));
}

// A work-group per sequence and K/V head goes through the prefix and the sequence's cache itself.
template <typename T, int HD, int OR>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_rows_whole(rows::Args p) {
  __shared__ u32x4 lds[rows::lds_chunks<HD, 4, 32, true>()];
  rows::attn_rows<T, HD, 4, OR / 16, 32, true, 2, rows::WHOLE>(p, lds, blockIdx.x);
}

template <typename T, int HD>
int launch_whole(const rows::Args& own, const Split& d, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(own.B * own.Hkv));
  if (d.own_rows == 16)
    hipLaunchKernelGGL((attn_rows_whole<T, HD, 16>), grid, dim3(256), 0, st, own);
  else
    hipLaunchKernelGGL((attn_rows_whole<T, HD, 32>), grid, dim3(256), 0, st, own);
  return static_cast<int>(hipGetLastError());
}

template <typename T, int HD>
int launch_hd(const rows::Args& a, const rows::Args& own, const Split& d, hipStream_t st) {
  if (d.whole) return launch_whole<T, HD>(own, d, st);
  const int64_t np = static_cast<int64_t>(a.Hkv) * a.splits * a.row_tiles;
  const int64_t no = static_cast<int64_t>(a.Hkv) * own.splits * own.row_tiles * own.B;
  if (np + no == 0) return MI355_OK;  // no prefix and no caches: only the zeros
  if (d.prefix_rows <= 16) launch_one<T, HD, 16, 16>(a, own, np, no, st);
  else if (d.prefix_rows == 32) launch_one<T, HD, 32, 32>(a, own, np, no, st);
  else if (d.prefix_rows == 64 && d.own_rows == 16) launch_one<T, HD, 64, 16>(a, own, np, no, st);
  else if (d.prefix_rows == 64) launch_one<T, HD, 64, 32>(a, own, np, no, st);
  else if (d.own_rows == 16) launch_one<T, HD, 128, 16>(a, own, np, no, st);
  else launch_one<T, HD, 128, 32>(a, own, np, no, st);
  return static_cast<int>(hipGetLastError());
}

template <typename T>
int launch(const rows::Args& a, const rows::Args& own, const CombineArgs& c, const Shape& s, const Split& d, hipStream_t st) {
  int e = MI355_E_HEAD_DIM;
  switch (s.hd) {
    case 16: e = launch_hd<T, 16>(a, own, d, st); break;
    case 32: e = launch_hd<T, 32>(a, own, d, st); break;
    case 48: e = launch_hd<T, 48>(a, own, d, st); break;
    case 64: e = launch_hd<T, 64>(a, own, d, st); break;
    case 80: e = launch_hd<T, 80>(a, own, d, st); break;
    case 96: e = launch_hd<T, 96>(a, own, d, st); break;
    case 128: e = launch_hd<T, 128>(a, own, d, st); break;
    case 192: e = launch_hd<T, 192>(a, own, d, st); break;
    case 256: e = launch_hd<T, 256>(a, own, d, st); break;
  }
  if (e || d.whole) return e;
  if (d.prefix_splits + d.own_splits <= WAVE_SPLITS)
    hipLaunchKernelGGL((combine_splits<T, 1>), dim3(static_cast<unsigned>(ceil_div(c.rows, 4))), dim3(256), 0, st, c);
  else
    hipLaunchKernelGGL((combine_splits<T, 4>), dim3(static_cast<unsigned>(c.rows)), dim3(256), 0, st, c);
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
      !o_strides || (prefix_len > 0 && (!K_prefix || !V_prefix)) || (room > 0 && (!K_own || !V_own)))
    return MI355_E_NULL_POINTER;
  const Split d = split_of(s);
  const int64_t need = (d.prefix_splits + d.own_splits) * s.rows() * (head_dim + 2) * 4;
  if (need > 0 && !workspace) return MI355_E_NULL_POINTER;
  if (workspace_bytes < need) return MI355_E_BAD_SIZE;
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
  if (kv_heads * d.prefix_splits * ceil_div(B * n_q * G, d.prefix_rows) +
      kv_heads * d.own_splits * ceil_div(n_q * G, d.own_rows) * B > MAX_BLOCKS)
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
  a.by_G = rows::make_div(a.G);
  a.by_Hkv = rows::make_div(a.Hkv);
  a.by_n_q = rows::make_div(n_q);
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
  own.pk = K_prefix; own.pv = V_prefix;
  own.pkt = kp_strides[0]; own.pkh = kp_strides[1];
  own.pvt = vp_strides[0]; own.pvh = vp_strides[1];
  own.pkeys = a.keys;
  own.o = O;
  own.ob = o_strides[0]; own.ot = o_strides[1]; own.oh = o_strides[2];
  a.chunk = static_cast<int32_t>(d.prefix_chunk);
  a.splits = static_cast<int32_t>(d.prefix_splits);
  a.row_tiles = static_cast<int32_t>(ceil_div(B * n_q * G, d.prefix_rows));
  own.chunk = static_cast<int32_t>(d.own_chunk);
  own.splits = static_cast<int32_t>(d.own_splits);
  own.row_tiles = static_cast<int32_t>(ceil_div(n_q * G, d.own_rows));
  own.part0 = a.splits;
  for (rows::Args* x : {&a, &own}) {
    x->by_splits = rows::make_div(x->splits);
    x->by_row_tiles = rows::make_div(x->row_tiles);
  }
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

// Attention over packed sequences of different lengths with grouped query heads: the plan (host), the
// launches of attn_rows_kernel over its tiles, and the joining of tiles whose keys it split.
#include <algorithm>
#include <vector>

#include "attn_rows.h"

namespace {

bool packed_head_dim(int64_t hd) {
  switch (hd) {
    case 16: case 32: case 48: case 64: case 80: case 96: case 128: case 192: case 256: return true;
    default: return false;
  }
}

constexpr int64_t MAX_TOKENS = int64_t(1) << 30;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows of a tile. Sequences of up to 32 rows (a token or a few) take NARROW ones, whose keys four waves
// share out; the others WIDE ones of four waves of two groups of 16 rows, or HALF ones of one group where WIDE
// ones leave CUs without work: fewer than two a CU, above head dim 64 counting the ranges that their keys are
// split into. Measured (us, WIDE / HALF; bf16, 32/8 heads of 128 but where noted; from card to card up to 4% either way):
// 8192 tokens 479 / 553; 24 prompts of 33-2011 (32/4) 157 / 169; 512 tokens against 8192 keys 81 / 103; 2048 against
// 16384 (8/2) 150 / 176; 4 x 100 against 3000 44 / 43; 3 x 700 (16/4) 30 / 22; 1000 34 / 30; heads of 64, 16/16: 8
// pieces of 200-512 against up to 5500 keys (fp16) 85 / 70, 300 against 6000 27 / 24. WIDE tiles take 32 keys at a time
// (64, two work-groups a CU then: 8192 tokens 531 beside 498, the 24 prompts 172 beside 154), HALF ones 64 up to head
// dim 64 (32: the pieces 104 beside 70).
constexpr int WIDE = 128, HALF = 64, NARROW = 32;
// Least keys of a range of a WIDE or HALF tile: its partial rows are 4 bytes an element, twice.
constexpr int64_t WIDE_KEYS = 512;

// What a plan starts with: its sizes; tiles of 128 or 64 rows, then of 32, then the joins.
struct Counts {
  int64_t wide, narrow, joins, slots;
};

// A tile whose keys were split: its ranges' partial rows follow each other, `rows` (the tile's) apart.
struct Join {
  int32_t q0, q_len, k_len, row0, rows, slot, splits, pad;
};
static_assert(sizeof(Join) == sizeof(rows::PackedTile), "plan entry");

// Work-groups a CU that the registers have to leave room for: what the first sweep takes by itself, which the ones
// over V that is not finite must not exceed.
template <int HD, int QG, bool OWN_KEYS>
constexpr int waves() {
  if (HD > 128) return 1;
  if (OWN_KEYS) return HD > 96 ? 2 : HD > 64 ? 3 : 4;
  return QG == 1 ? (HD > 96 ? 4 : 5) : HD > 64 ? 3 : 4;
}

template <typename T, int HD, int QG, int BN, bool OWN_KEYS>
__global__ __launch_bounds__(256, (waves<HD, QG, OWN_KEYS>())) void attn_rows_packed(rows::Args p) {
  __shared__ u32x4 lds[rows::lds_chunks<HD, 4, BN, OWN_KEYS>()];
  rows::attn_rows<T, HD, 4, QG, BN, OWN_KEYS, OWN_KEYS ? 2 : 1, rows::PACKED>(p, lds, blockIdx.x);
}

template <typename T, int HD>
int launch_hd(const rows::Args& a, const Counts& n, int wide_rows, hipStream_t s) {
  if (n.wide > 0) {
    const dim3 grid(static_cast<unsigned>(n.wide * a.Hkv));
    if (wide_rows == WIDE)
      hipLaunchKernelGGL((attn_rows_packed<T, HD, 2, 32, false>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((attn_rows_packed<T, HD, 1, HD <= 64 ? 64 : 32, false>), grid, dim3(256), 0, s, a);
  }
  if (n.narrow > 0) {
    rows::Args b = a;
    b.tiles += n.wide;
    hipLaunchKernelGGL((attn_rows_packed<T, HD, 2, 32, true>), dim3(static_cast<unsigned>(n.narrow * a.Hkv)), dim3(256), 0, s, b);
  }
  return static_cast<int>(hipGetLastError());
}

struct JoinArgs {
  const Join* joins;
  const float *part, *ml;
  void* o;
  int64_t ot, oh, slots;
  int32_t G, Hkv, hd, causal;
};

// A wave per row: o = sum_s 2^(mu_s - M) O_s / sum_s 2^(mu_s - M) l_s over the tile's ranges s. Lanes take
// ranges of their own for M and the sum, then 4 elements each, as many ranges at a time as that leaves.
template <typename T>
__global__ __launch_bounds__(256) void join_tiles(JoinArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = static_cast<int>(blockIdx.x % static_cast<unsigned>(p.Hkv));
  const Join j = p.joins[blockIdx.x / static_cast<unsigned>(p.Hkv)];
  const int i = blockIdx.y * 4 + wave, r = j.row0 + i;
  if (i >= j.rows || r >= j.q_len * p.G) return;
  const int t = r / p.G;
  const bool none = p.causal && t + j.k_len - j.q_len < 0;  // no key: zeros (no finite score: 0 / 0)
  const int64_t first = h * p.slots + j.slot + i;
  float m = NEG_INF, l = 0.f;
  for (int s = lane; s < j.splits; s += 64) m = vmax(m, p.ml[2 * (first + static_cast<int64_t>(s) * j.rows)]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = vmax(m, __shfl_xor(m, off));
  for (int s = lane; s < j.splits; s += 64) {
    const float* ml = p.ml + 2 * (first + static_cast<int64_t>(s) * j.rows);
    l = ml[0] == NEG_INF ? l : __builtin_fmaf(ml[1], fast_exp2(ml[0] - m), l);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off);
  const int per = p.hd / 4, at_once = 64 / per, mine = lane / per, x = lane % per;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (mine < at_once) {
    for (int s0 = mine; s0 < j.splits; s0 += 4 * at_once) {
      f32x4 v[4];
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int s = s0 + k * at_once;
        const int64_t at = first + static_cast<int64_t>(s < j.splits ? s : s0) * j.rows;
        w[k] = s < j.splits ? p.ml[2 * at] : NEG_INF;
        v[k] = *reinterpret_cast<const f32x4*>(p.part + at * p.hd + 4 * x);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[e] = w[k] == NEG_INF ? acc[e] : __builtin_fmaf(v[k][e], fast_exp2(w[k] - m), acc[e]);
    }
  }
  // the lanes of one element, at_once of them, per lanes apart
  f32x4 sum = acc;
  for (int k = 1; k < at_once; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += __shfl(acc[e], (lane + k * per) & 63);
  if (mine != 0) return;
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(none ? 0.f : sum[e] / l);
  *reinterpret_cast<t4*>(static_cast<T*>(p.o) + (static_cast<int64_t>(j.q0) + t) * p.ot +
                         (h * p.G + r - t * p.G) * p.oh + 4 * x) = w;
}

template <typename T>
int launch(const rows::Args& a, int64_t hd, const Counts& n, int wide_rows, hipStream_t s) {
  int e = MI355_E_HEAD_DIM;
  switch (hd) {
    case 16: e = launch_hd<T, 16>(a, n, wide_rows, s); break;
    case 32: e = launch_hd<T, 32>(a, n, wide_rows, s); break;
    case 48: e = launch_hd<T, 48>(a, n, wide_rows, s); break;
    case 64: e = launch_hd<T, 64>(a, n, wide_rows, s); break;
    case 80: e = launch_hd<T, 80>(a, n, wide_rows, s); break;
    case 96: e = launch_hd<T, 96>(a, n, wide_rows, s); break;
    case 128: e = launch_hd<T, 128>(a, n, wide_rows, s); break;
    case 192: e = launch_hd<T, 192>(a, n, wide_rows, s); break;
    case 256: e = launch_hd<T, 256>(a, n, wide_rows, s); break;
  }
  if (e || n.joins == 0) return e;
  const JoinArgs j{reinterpret_cast<const Join*>(a.tiles + n.wide + n.narrow), a.part, a.ml, a.o, a.ot, a.oh,
                   a.slots, a.G, a.Hkv, static_cast<int32_t>(hd), a.causal};
  const int most = n.wide > 0 ? wide_rows : NARROW;
  hipLaunchKernelGGL((join_tiles<T>), dim3(static_cast<unsigned>(n.joins * a.Hkv), most / 4), dim3(256), 0, s, j);
  return static_cast<int>(hipGetLastError());
}

bool fits(const Counts& n, int64_t kv_heads) {
  const int64_t most = 0xffffffffLL / 256;  // a launch has at most 2^32 - 1 threads
  return n.wide >= 0 && n.narrow >= 0 && n.joins >= 0 && n.slots >= 0 && n.wide <= most / kv_heads &&
         n.narrow <= most / kv_heads && n.joins <= most / kv_heads && n.slots <= 0x7fffffffLL;
}

}  // namespace

extern "C" int mi355_attn_packed_plan(const int32_t* q_lens, const int32_t* k_lens, int64_t n_seqs,
                                      int64_t heads, int64_t kv_heads, int64_t head_dim, int causal,
                                      int32_t* plan, int64_t capacity, int64_t* counts,
                                      int32_t* tile_rows) {
  if (n_seqs < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads > 65535 || capacity < 0)
    return MI355_E_BAD_SIZE;
  if (!packed_head_dim(head_dim)) return MI355_E_HEAD_DIM;
  if (!counts || !tile_rows || (n_seqs > 0 && (!q_lens || !k_lens))) return MI355_E_NULL_POINTER;
  const int64_t G = heads / kv_heads;
  int64_t tq = 0, tk = 0, wide = 0, wide_ranges = 0, few = 0, few_keys = 0;
  for (int64_t i = 0; i < n_seqs; ++i) {
    if (q_lens[i] < 0 || k_lens[i] < 0) return MI355_E_BAD_SIZE;
    tq += q_lens[i];
    tk += k_lens[i];
    if (tq >= MAX_TOKENS || tk >= MAX_TOKENS || q_lens[i] * G >= MAX_TOKENS) return MI355_E_BAD_SIZE;
    if (q_lens[i] * G > NARROW) {
      const int64_t tiles = ceil_div(q_lens[i] * G, WIDE);
      wide += tiles;
      wide_ranges += tiles * std::max<int64_t>(1, k_lens[i] / WIDE_KEYS);
    } else if (q_lens[i] > 0) {
      ++few;
      few_keys = std::max<int64_t>(few_keys, k_lens[i]);
    }
  }
  const int wide_rows = (head_dim > 64 ? wide_ranges : wide) * kv_heads >= 512 ? WIDE : HALF;
  // A few short sequences of few rows beside others take the others' tiles, which saves a launch.
  const int64_t narrow = wide > 0 && few * kv_heads <= 256 && few_keys <= 512 ? 0 : NARROW;
  struct Ref {
    int64_t keys;
    rows::PackedTile t;
  };
  std::vector<Ref> lists[2];  // wide, narrow
  std::vector<Join> joins;
  Counts n{};
  try {
    // Tiles, then ranges of their keys where the tiles alone leave CUs idle: as many as fill the work-groups
    // that run at once (two a CU), each of a like share of all keys, but not so short that writing and
    // reading a range's partial rows outweighs reading its keys.
    int64_t keys_of[2] = {0, 0}, tiles_of[2] = {0, 0};
    const auto visit = [&](auto&& each) {
      int64_t q0 = 0, k0 = 0;
      for (int64_t i = 0; i < n_seqs; ++i) {
        const int64_t total = q_lens[i] * G;
        const int which = total > narrow ? 0 : 1, rows = which ? NARROW : wide_rows;
        for (int64_t r = 0; r < total; r += rows) {
          const int64_t last = std::min(r + rows, total) - 1;
          int64_t keys = k_lens[i];
          if (causal) keys = std::max<int64_t>(0, std::min<int64_t>(keys, last / G + k_lens[i] - q_lens[i] + 1));
          rows::PackedTile t{};
          t.q0 = static_cast<int32_t>(q0);
          t.q_len = q_lens[i];
          t.k0 = static_cast<int32_t>(k0);
          t.k_len = k_lens[i];
          t.row0 = static_cast<int32_t>(r);
          each(which, rows, keys, t, std::min<int64_t>(rows, total - r));
        }
        q0 += q_lens[i];
        k0 += k_lens[i];
      }
    };
    visit([&](int which, int, int64_t keys, const rows::PackedTile&, int64_t) {
      keys_of[which] += keys;
      ++tiles_of[which];
    });
    int64_t chunk[2];
    for (int w = 0; w < 2; ++w) {
      const int64_t at_once = 512, least = w ? 256 : WIDE_KEYS;
      const int64_t share = ceil_div(ceil_div(keys_of[w] * kv_heads, at_once), 64) * 64;
      chunk[w] = tiles_of[w] * kv_heads >= at_once ? MAX_TOKENS : std::max(least, share);
    }
    visit([&](int which, int, int64_t keys, rows::PackedTile t, int64_t real) {
      const int64_t splits = std::max<int64_t>(1, ceil_div(keys, chunk[which]));
      const int64_t each = ceil_div(ceil_div(keys, splits), 64) * 64;
      const int64_t used = std::max<int64_t>(1, each > 0 ? ceil_div(keys, each) : 1);
      if (used > 1) joins.push_back({t.q0, t.q_len, t.k_len, t.row0, static_cast<int32_t>(real), static_cast<int32_t>(n.slots), static_cast<int32_t>(used), 0});
      for (int64_t s = 0; s < used; ++s) {
        t.k_begin = static_cast<int32_t>(s * each);
        t.k_stop = static_cast<int32_t>(std::min(keys, (s + 1) * each));
        t.slot = -1;
        if (used > 1) {
          t.slot = static_cast<int32_t>(n.slots);
          n.slots += real;
          if (n.slots > 0x7fffffffLL) return;
        }
        lists[which].push_back({t.k_stop - t.k_begin, t});
      }
    });
  } catch (...) {  // (out of memory)
    return MI355_E_BAD_SIZE;
  }
  n.wide = static_cast<int64_t>(lists[0].size());
  n.narrow = static_cast<int64_t>(lists[1].size());
  n.joins = static_cast<int64_t>(joins.size());
  if (!fits(n, kv_heads)) return MI355_E_BAD_SIZE;
  *tile_rows = wide_rows;
  counts[0] = n.wide;
  counts[1] = n.narrow;
  counts[2] = n.joins;
  counts[3] = n.slots;
  if (!plan) return MI355_OK;  // sizes only
  if (capacity < n.wide + n.narrow + n.joins) return MI355_E_BAD_SIZE;
  auto* out = reinterpret_cast<rows::PackedTile*>(plan);
  for (auto& list : lists) {  // longest first, so that no long one is left for the end
    std::sort(list.begin(), list.end(), [](const Ref& a, const Ref& b) {
      return a.keys != b.keys ? a.keys > b.keys : a.t.q0 != b.t.q0 ? a.t.q0 < b.t.q0
             : a.t.row0 != b.t.row0 ? a.t.row0 < b.t.row0 : a.t.k_begin < b.t.k_begin;
    });
    for (const Ref& r : list) *out++ = r.t;
  }
  for (const Join& j : joins) *reinterpret_cast<Join*>(out++) = j;
  return MI355_OK;
}

extern "C" int mi355_attn_packed(int dtype, const void* Q, const void* K, const void* V, void* O,
                                 int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 const int64_t* q_strides, const int64_t* k_strides,
                                 const int64_t* v_strides, const int64_t* o_strides, float scale,
                                 int causal, const int32_t* plan, const int64_t* counts,
                                 int32_t tile_rows, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads > 65535) return MI355_E_BAD_SIZE;
  if (dtype != MI355_F16 && dtype != MI355_BF16) return MI355_E_BAD_DTYPE;
  if (!packed_head_dim(head_dim)) return MI355_E_HEAD_DIM;
  if (tile_rows != WIDE && tile_rows != HALF) return MI355_E_UNSUPPORTED;
  if (!(scale > 0.f) || scale > 1e30f) return MI355_E_UNSUPPORTED;
  if (!counts) return MI355_E_NULL_POINTER;
  const Counts n{counts[0], counts[1], counts[2], counts[3]};
  if (!fits(n, kv_heads)) return MI355_E_BAD_SIZE;
  if (n.wide + n.narrow == 0) return MI355_OK;
  if (!Q || !O || !plan || !q_strides || !k_strides || !v_strides || !o_strides || (n.joins > 0 && !workspace))
    return MI355_E_NULL_POINTER;
  const int64_t part_rows = n.slots * kv_heads;
  if (n.joins > 0 && workspace_bytes < part_rows * (head_dim + 2) * 4) return MI355_E_BAD_SIZE;
  // (without keys in any sequence there may be no K and V: nothing of them is read)
  for (const int64_t* st : {k_strides, v_strides})
    if (st[0] < head_dim || st[0] > (int64_t(1) << 24)) return MI355_E_BAD_SIZE;
  for (const int64_t* st : {q_strides, k_strides, v_strides})
    if (st[0] % 8 || st[1] % 8) return MI355_E_ALIGNMENT;
  if (o_strides[0] % 4 || o_strides[1] % 4) return MI355_E_ALIGNMENT;
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(O) & 7u))
    return MI355_E_ALIGNMENT;
  rows::Args a{};
  a.q = Q; a.k = K; a.v = V; a.o = O;
  a.qt = q_strides[0]; a.qh = q_strides[1];
  a.kt = k_strides[0]; a.kh = k_strides[1];
  a.vt = v_strides[0]; a.vh = v_strides[1];
  a.ot = o_strides[0]; a.oh = o_strides[1];
  a.c = scale * 1.4426950408889634f;
  a.G = static_cast<int32_t>(heads / kv_heads);
  a.H = static_cast<int32_t>(heads);
  a.Hkv = static_cast<int32_t>(kv_heads);
  a.by_G = rows::make_div(a.G);
  a.by_Hkv = rows::make_div(a.Hkv);
  a.tiles = reinterpret_cast<const rows::PackedTile*>(plan);
  a.causal = causal != 0;
  a.slots = n.slots;
  a.part = static_cast<float*>(workspace);
  a.ml = a.part + part_rows * head_dim;
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == MI355_F16 ? launch<_Float16>(a, head_dim, n, tile_rows, s) : launch<__bf16>(a, head_dim, n, tile_rows, s);
}

// Attention over packed sequences of different lengths with grouped query heads: the plan (host) and
// the launch of attn_rows_kernel over its tiles.
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

// Rows of a work-group: LARGE tiles (4 waves of 32 rows), SMALL ones (a wave of 32 rows).
constexpr int LARGE = 128, SMALL = 32;

template <typename T, int HD>
int launch_hd(const rows::Args& a, int64_t blocks, int tile_rows, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(blocks));
  if (tile_rows == LARGE)
    hipLaunchKernelGGL((rows::attn_rows_kernel<T, HD, 4, 2, HD <= 128 ? 64 : 32, 2, HD <= 128 ? 2 : 1, 1, rows::PACKED>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((rows::attn_rows_kernel<T, HD, 1, 2, 32, 2, 1, 1, rows::PACKED>), grid, dim3(64), 0, s, a);
  return static_cast<int>(hipGetLastError());
}

template <typename T>
int launch(const rows::Args& a, int64_t hd, int64_t blocks, int tile_rows, hipStream_t s) {
  switch (hd) {
    case 16: return launch_hd<T, 16>(a, blocks, tile_rows, s);
    case 32: return launch_hd<T, 32>(a, blocks, tile_rows, s);
    case 48: return launch_hd<T, 48>(a, blocks, tile_rows, s);
    case 64: return launch_hd<T, 64>(a, blocks, tile_rows, s);
    case 80: return launch_hd<T, 80>(a, blocks, tile_rows, s);
    case 96: return launch_hd<T, 96>(a, blocks, tile_rows, s);
    case 128: return launch_hd<T, 128>(a, blocks, tile_rows, s);
    case 192: return launch_hd<T, 192>(a, blocks, tile_rows, s);
    case 256: return launch_hd<T, 256>(a, blocks, tile_rows, s);
    default: return MI355_E_HEAD_DIM;
  }
}

}  // namespace

extern "C" int mi355_attn_packed_plan(const int32_t* q_lens, const int32_t* k_lens, int64_t n_seqs,
                                      int64_t heads, int64_t kv_heads, int64_t head_dim, int causal,
                                      int32_t* tiles, int64_t capacity, int64_t* n_tiles,
                                      int32_t* tile_rows) {
  if (n_seqs < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads > 65535 || capacity < 0)
    return MI355_E_BAD_SIZE;
  if (!packed_head_dim(head_dim)) return MI355_E_HEAD_DIM;
  if (!n_tiles || !tile_rows || (n_seqs > 0 && (!q_lens || !k_lens))) return MI355_E_NULL_POINTER;
  const int64_t G = heads / kv_heads;
  int64_t tq = 0, tk = 0, large = 0;
  for (int64_t i = 0; i < n_seqs; ++i) {
    if (q_lens[i] < 0 || k_lens[i] < 0) return MI355_E_BAD_SIZE;
    tq += q_lens[i];
    tk += k_lens[i];
    if (tq >= MAX_TOKENS || tk >= MAX_TOKENS || q_lens[i] * G >= MAX_TOKENS) return MI355_E_BAD_SIZE;
    large += (q_lens[i] * G + LARGE - 1) / LARGE;
  }
  // large tiles once they give every CU two work-groups
  const int rows = large * kv_heads >= 512 ? LARGE : SMALL;
  int64_t count = 0;
  for (int64_t i = 0; i < n_seqs; ++i) count += (q_lens[i] * G + rows - 1) / rows;
  *tile_rows = rows;
  *n_tiles = count;
  if (count * kv_heads > 0x7fffffffLL) return MI355_E_BAD_SIZE;
  if (!tiles) return MI355_OK;  // sizes only
  if (capacity < count) return MI355_E_BAD_SIZE;
  // longest key range first, so that no long tile is left for the end
  struct Ref { int64_t keys; rows::PackedTile t; };
  std::vector<Ref> list;
  try {
    list.reserve(static_cast<size_t>(count));
  } catch (...) {
    return MI355_E_BAD_SIZE;
  }
  int64_t q0 = 0, k0 = 0;
  for (int64_t i = 0; i < n_seqs; ++i) {
    const int64_t n = q_lens[i] * G;
    for (int64_t r = 0; r < n; r += rows) {
      const int64_t last = std::min(r + rows, n) - 1;
      int64_t keys = k_lens[i];
      if (causal) keys = std::max<int64_t>(0, std::min<int64_t>(keys, last / G + k_lens[i] - q_lens[i] + 1));
      rows::PackedTile t{};
      t.q0 = static_cast<int32_t>(q0);
      t.q_len = q_lens[i];
      t.k0 = static_cast<int32_t>(k0);
      t.k_len = k_lens[i];
      t.row0 = static_cast<int32_t>(r);
      list.push_back({keys, t});
    }
    q0 += q_lens[i];
    k0 += k_lens[i];
  }
  std::sort(list.begin(), list.end(), [](const Ref& a, const Ref& b) {
    return a.keys != b.keys ? a.keys > b.keys : a.t.q0 != b.t.q0 ? a.t.q0 < b.t.q0 : a.t.row0 < b.t.row0;
  });
  for (int64_t i = 0; i < count; ++i) reinterpret_cast<rows::PackedTile*>(tiles)[i] = list[i].t;
  return MI355_OK;
}

extern "C" int mi355_attn_packed(int dtype, const void* Q, const void* K, const void* V, void* O,
                                 int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 const int64_t* q_strides, const int64_t* k_strides,
                                 const int64_t* v_strides, const int64_t* o_strides, float scale,
                                 int causal, const int32_t* tiles, int64_t n_tiles, int32_t tile_rows,
                                 void* stream) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads > 65535 || n_tiles < 0 ||
      n_tiles * kv_heads > 0x7fffffffLL)
    return MI355_E_BAD_SIZE;
  if (dtype != MI355_F16 && dtype != MI355_BF16) return MI355_E_BAD_DTYPE;
  if (!packed_head_dim(head_dim)) return MI355_E_HEAD_DIM;
  if (tile_rows != LARGE && tile_rows != SMALL) return MI355_E_UNSUPPORTED;
  if (!(scale > 0.f) || scale > 1e30f) return MI355_E_UNSUPPORTED;
  if (n_tiles == 0) return MI355_OK;
  if (!Q || !O || !tiles || !q_strides || !k_strides || !v_strides || !o_strides) return MI355_E_NULL_POINTER;
  // (without keys in any sequence there may be no K and V: nothing of them is read)
  for (const int64_t* st : {k_strides, v_strides})
    if (st[0] < head_dim || st[0] > (int64_t(1) << 24)) return MI355_E_BAD_SIZE;
  for (const int64_t* st : {q_strides, k_strides, v_strides})
    if (st[0] % 8 || st[1] % 8) return MI355_E_ALIGNMENT;
  if (o_strides[0] % 4 || o_strides[1] % 4) return MI355_E_ALIGNMENT;
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || (reinterpret_cast<uintptr_t>(O) & 7u)) return MI355_E_ALIGNMENT;
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
  a.tiles = reinterpret_cast<const rows::PackedTile*>(tiles);
  a.causal = causal != 0;
  const auto s = static_cast<hipStream_t>(stream);
  return dtype == MI355_F16 ? launch<_Float16>(a, head_dim, n_tiles * kv_heads, tile_rows, s)
                            : launch<__bf16>(a, head_dim, n_tiles * kv_heads, tile_rows, s);
}

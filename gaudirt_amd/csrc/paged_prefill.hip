// Chunked / prefix-shared paged prefill attention for gfx950 (bf16 MFMA).
//
// A sequence contributes a chunk of consecutive query rows at positions
// prefix .. prefix + rows - 1; row i attends keys [left_i, prefix + i] of its
// request (causal; left_i = prefix + i - window + 1 with a sliding window).
// The chunk's own K/V rows are already in the pool (the store runs first), so
// every key is read through the block table.
//
// Work decomposition. A workgroup of eight waves owns one (sequence, kv head,
// tile of rows), or with a work list (prefill_schedule.hpp) a range of such a
// tile's keys, whose partial result prefill_merge_kernel combines. The GQA group is folded into the tile: its 256 "query rows"
// (128 at head_dim 256) are (row, head) pairs, so one K/V tile serves every
// head of the group. Each wave computes 32 query rows (two 16-column MFMA
// tiles; one, 16 rows, at head_dim 256) against the keys of a step (64 at
// head_dim 128, 32 at head_dim 64 and 256):
//   S^T[key][qrow] = K . Q^T      v_mfma_f32_16x16x32_bf16, K from LDS
//   O[qrow][dim]  += P . V        P straight from S^T's registers, V read
//                                 transposed from LDS (ds_read_b64_tr_b16)
// A step's K and V tiles are shared by the eight waves through LDS: 16-byte
// buffer->LDS loads issued by the whole workgroup, XOR-swizzled by token,
// double-buffered so the next tile streams in while the current one is used.
// Online softmax runs in log2 units with a lazily re-based running maximum.
//
// Numerics versus the reference (the tile chain of
// src/bridge/paged_attention_tiles.cpp:57-195): fp32 scores times scale,
// probabilities rounded to bf16 before P.V (relative to the running maximum),
// fp32 accumulation, one normalisation at the end by the sum of those bf16
// probabilities, bf16 output.
#include "prefill_kernel.hpp"

#include <algorithm>
#include <cstring>
#include <new>
#include <type_traits>
#include <vector>

namespace gk {
namespace {

// ---------------------------------------------------------------------------
// Merge of the items that a work list splits
// ---------------------------------------------------------------------------
struct PrefillMergeArgs {
  const int32_t* merges;  // PrefillMerge records
  int32_t part_slots, group, q_heads;
  DivMagic group_div;
  const float* part_o;
  const float* part_ml;
  uint16_t* out;
  int64_t out_stride;
};

// Bound by reading the partials (from the last-level cache mostly) and, for few
// of them, by the launch: 8 us for 256 partials of 128 KiB (4.2 TB/s), 15 us for
// 496 (4.4 TB/s), 7 us for 258 of 64 KiB. One wave per (split item, kv head, 16 query rows, 32
// dims): the partials are read as the pieces' lanes stored them, 1 KiB a load,
// the loads of up to eight parts in one memory round trip.
template <int D>
__global__ __launch_bounds__(64) void prefill_merge_kernel(PrefillMergeArgs a) {
  constexpr int kTiles = prefill_tile_qrows(D) / 16, NO = D / 16, CC = 2, kGroups = NO / CC;
  constexpr int kRowBytes = 16 * CC * 2 + 16;
  __shared__ __attribute__((aligned(16))) char lds[16 * kRowBytes];
  const int lane = threadIdx.x, q = lane >> 4, c16 = lane & 15;
  const int mi = blockIdx.x / (kTiles * kGroups), rest = blockIdx.x % (kTiles * kGroups);
  const int t = rest / kGroups, cg = rest % kGroups, kvh = blockIdx.y;
  const int32_t* rec = a.merges + (int64_t)mi * kPrefillMergeWords;
  const int first_row = scalar_load(rec, 0), nr = scalar_load(rec, 1), slot = scalar_load(rec, 2),
            parts = scalar_load(rec, 3);
  if ((int)fast_div((uint32_t)(16 * t), a.group_div) >= nr) return;
  const int64_t tile0 = ((int64_t)kvh * a.part_slots + slot) * kTiles + t;  // part p: + p kTiles
  f32x4_t m_run, l_run{0.f, 0.f, 0.f, 0.f}, acc[CC];
#pragma unroll
  for (int r = 0; r < 4; ++r) m_run[r] = -INFINITY;
#pragma unroll
  for (int c = 0; c < CC; ++c) acc[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto merge_parts = [&](auto batch) {
    constexpr int BATCH = decltype(batch)::value;
    for (int p0 = 0; p0 < parts; p0 += BATCH) {
      f32x4_t mp[BATCH], lp[BATCH], op[BATCH][CC];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int64_t tile = tile0 + (int64_t)min(p0 + u, parts - 1) * kTiles;
        mp[u] = *reinterpret_cast<const f32x4_t*>(a.part_ml + tile * 32 + 4 * q);
        lp[u] = *reinterpret_cast<const f32x4_t*>(a.part_ml + tile * 32 + 16 + 4 * q);
        const f32x4_t* po = reinterpret_cast<const f32x4_t*>(a.part_o) + (tile * NO + cg * CC) * 64 + lane;
#pragma unroll
        for (int c = 0; c < CC; ++c) op[u][c] = po[c * 64];
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // Parts past the last (clamped duplicates) weigh nothing. A part
          // without a visible key has no output: its slot is not read into
          // the sum.
          const float mu = p0 + u < parts ? mp[u][r] : -INFINITY;
          const float mn = fmaxf(m_run[r], mu);
          const float fa = m_run[r] == -INFINITY ? 0.f : fast_exp2(m_run[r] - mn);
          const float fb = mu == -INFINITY ? 0.f : fast_exp2(mu - mn);
          l_run[r] = l_run[r] * fa + (mu == -INFINITY ? 0.f : lp[u][r] * fb);
#pragma unroll
          for (int c = 0; c < CC; ++c) acc[c][r] = acc[c][r] * fa + (mu == -INFINITY ? 0.f : op[u][c][r] * fb);
          m_run[r] = mn;
        }
      }
    }
  };
  if (parts <= 4) merge_parts(std::integral_constant<int, 4>{});
  else merge_parts(std::integral_constant<int, 8>{});
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float inv = l_run[r] > 0.f ? 1.f / l_run[r] : 0.f;
    __bf16* dst = reinterpret_cast<__bf16*>(lds + (4 * q + r) * kRowBytes) + c16;
#pragma unroll
    for (int c = 0; c < CC; ++c) dst[16 * c] = (__bf16)(acc[c][r] * inv);
  }
  // The wave's own LDS operations complete in order: 16 rows x 4 pieces of 16 bytes.
  static_assert(CC == 2, "one 16-byte piece per lane");
  const int ql = lane >> 2, part = lane & 3;
  const uint4 v = *reinterpret_cast<const uint4*>(lds + ql * kRowBytes + part * 16);
  const int qr = 16 * t + ql, row = (int)fast_div((uint32_t)qr, a.group_div), head = qr - row * a.group;
  if (row < nr)
    *reinterpret_cast<uint4*>(a.out + (int64_t)(first_row + row) * a.out_stride +
                              (int64_t)(kvh * a.group + head) * D + cg * (16 * CC) + part * 8) = v;
}

template <int D, int MODE>
void launch_mode(const PrefillArgs& a, int score, dim3 grid, hipStream_t stream) {
  if (score == kScoreBias) prefill_kernel<D, kScoreBias, MODE, PrefillArgs><<<grid, kPrefillWaves * 64, 0, stream>>>(a);
  else if (score == kScoreCapBias) prefill_kernel<D, kScoreCapBias, MODE, PrefillArgs><<<grid, kPrefillWaves * 64, 0, stream>>>(a);
  else if (score == kScoreCap) prefill_kernel<D, kScoreCap, MODE, PrefillArgs><<<grid, kPrefillWaves * 64, 0, stream>>>(a);
  else prefill_kernel<D, kScorePlain, MODE, PrefillArgs><<<grid, kPrefillWaves * 64, 0, stream>>>(a);
}

template <int D>
void launch(const PrefillArgs& a, int score, int block_size, dim3 grid, hipStream_t stream) {
  constexpr int keys = prefill_keys<D>();
  if (block_size >= keys) launch_mode<D, kStepBlocks>(a, score, grid, stream);
  else if (block_size >= keys / PrefillShape<D>::NI) launch_mode<D, kLoadBlocks>(a, score, grid, stream);
  else launch_mode<D, kKeyBlocks>(a, score, grid, stream);
}

}  // namespace

namespace {

int launch_prefill(const gk_prefill_params* p, const PrefillArgs& a, int64_t workgroups, hipStream_t stream) {
  const dim3 grid((unsigned)workgroups);
  const int score = p->softcap > 0.f ? (a.slopes ? kScoreCapBias : kScoreCap) : a.slopes ? kScoreBias : kScorePlain;
  if (p->head_dim == 64) launch<64>(a, score, p->block_size, grid, stream);
  else if (p->head_dim == 128) launch<128>(a, score, p->block_size, grid, stream);
  else launch<256>(a, score, p->block_size, grid, stream);
  return hip_status(hipGetLastError(), "gk_paged_prefill launch");
}

// Workspace of a work list: the partial outputs, then (base, sum) of every row.
size_t list_output_bytes(const gk_prefill_params* p, const gk_prefill_list* list) {
  return (size_t)p->kv_heads * list->part_slots * prefill_tile_qrows(p->head_dim) * p->head_dim * sizeof(float);
}
size_t list_workspace_bytes(const gk_prefill_params* p, const gk_prefill_list* list) {
  return list_output_bytes(p, list) +
         (size_t)p->kv_heads * list->part_slots * prefill_tile_qrows(p->head_dim) * 2 * sizeof(float);
}

}  // namespace

int device_cus();

int paged_prefill(const gk_prefill_params* p, hipStream_t stream) {
  if (int rc = check_prefill(p, false, "gk_paged_prefill")) return rc;
  if (p->seqs == 0 || p->max_rows == 0) return GK_OK;
  PrefillArgs a = prefill_args(p);
  a.seq_request = p->seq_request;
  a.seq_first_row = p->seq_first_row;
  a.seq_rows = p->seq_rows;
  a.seq_prefix = p->seq_prefix;
  a.seqs = p->seqs;
  a.tiles = (p->max_rows + a.rows_per_tile - 1) / a.rows_per_tile;
  a.tiles_div = div_magic((uint32_t)a.tiles);
  a.seqs_div = div_magic((uint32_t)a.seqs);
  const int64_t items = (int64_t)a.tiles * p->kv_heads * p->seqs;
  if (items > (int64_t)1 << 30) return fail(GK_ERR_INVALID_ARGUMENT, "gk_paged_prefill: too many rows");
  return launch_prefill(p, a, items, stream);
}

int paged_prefill_listed(const gk_prefill_params* p, const gk_prefill_list* list, const float* slopes, void* workspace,
                         size_t workspace_bytes, hipStream_t stream) {
  if (int rc = check_prefill(p, true, "gk_paged_prefill")) return rc;
  if (!list || list->struct_size != sizeof(gk_prefill_list))
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_paged_prefill_listed: struct_size does not match this library's gk_prefill_list");
  if (list->item_count < 0 || list->merge_count < 0 || list->part_slots < 0 || list->part_slots > (1 << 20) ||
      list->merge_count > (1 << 20))
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_paged_prefill_listed: list counts out of range");
  if (list->item_count == 0) return GK_OK;
  if (!list->items || !list->row_request || (list->merge_count && !list->merges))
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_paged_prefill_listed: null pointer");
  if (list->part_slots && (!workspace || workspace_bytes < list_workspace_bytes(p, list) ||
                           (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(GK_ERR_WORKSPACE, "gk_paged_prefill_listed: workspace too small or not 16-byte aligned (" +
                                      std::to_string(list_workspace_bytes(p, list)) + " bytes needed)");
  PrefillArgs a = prefill_args(p);
  a.slopes = slopes;
  a.items = list->items;
  a.item_count = list->item_count;
  a.row_request = list->row_request;
  int classes = kXcds;
  while (p->kv_heads % classes) classes /= 2;
  a.class_shift = log2_int(classes);
  a.class_heads = p->kv_heads / classes;
  a.class_xcds = kXcds / classes;
  a.class_heads_div = div_magic((uint32_t)a.class_heads);
  a.part_slots = list->part_slots;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + list_output_bytes(p, list));
  const int64_t per_xcd = ((int64_t)list->item_count + a.class_xcds - 1) / a.class_xcds * a.class_heads;
  if (per_xcd * kXcds > (int64_t)1 << 30)
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_paged_prefill_listed: too many items");
  if (int rc = launch_prefill(p, a, per_xcd * kXcds, stream)) return rc;
  if (!list->merge_count) return GK_OK;
  PrefillMergeArgs m{};
  m.merges = list->merges;
  m.part_slots = list->part_slots;
  m.group = a.group;
  m.q_heads = p->q_heads;
  m.group_div = a.group_div;
  m.part_o = a.part_o;
  m.part_ml = a.part_ml;
  m.out = a.out;
  m.out_stride = a.out_stride;
  const int waves = prefill_tile_qrows(p->head_dim) / 16 * (p->head_dim / 32);
  const dim3 grid((unsigned)(list->merge_count * waves), (unsigned)p->kv_heads);
  if (p->head_dim == 64) prefill_merge_kernel<64><<<grid, 64, 0, stream>>>(m);
  else if (p->head_dim == 128) prefill_merge_kernel<128><<<grid, 64, 0, stream>>>(m);
  else prefill_merge_kernel<256><<<grid, 64, 0, stream>>>(m);
  return hip_status(hipGetLastError(), "gk_paged_prefill_listed merge launch");
}

int prefill_list_build(const int32_t* seq_first_row, const int32_t* seq_rows, const int32_t* seq_prefix, int32_t seqs,
                       int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t sliding_window, bool cut,
                       int32_t* words, int64_t capacity, gk_prefill_list* list) {
  if (!list || list->struct_size != sizeof(gk_prefill_list))
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_prefill_list_build: struct_size does not match this library's gk_prefill_list");
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
      q_heads / kv_heads > 128)
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_prefill_list_build: invalid head geometry");
  if (seqs < 0 || seqs > 65535 || capacity < 0 || (seqs && (!seq_first_row || !seq_rows || !seq_prefix)))
    return fail(GK_ERR_INVALID_ARGUMENT, "gk_prefill_list_build: invalid sequences");
  int64_t rows = 0;
  for (int32_t s = 0; s < seqs; ++s) {
    if (seq_rows[s] < 0 || seq_prefix[s] < 0 || seq_first_row[s] < 0 ||
        (int64_t)seq_prefix[s] + seq_rows[s] > INT32_MAX - 64)
      return fail(GK_ERR_INVALID_ARGUMENT, "gk_prefill_list_build: invalid sequences");
    rows += seq_rows[s];
  }
  if (rows > (1 << 20)) return fail(GK_ERR_INVALID_ARGUMENT, "gk_prefill_list_build: too many rows");
  try {
    std::vector<PrefillSeq> in(seqs);
    for (int32_t s = 0; s < seqs; ++s)
      in[s] = {seq_first_row[s], seq_rows[s], seq_prefix[s]};
    const int group = q_heads / kv_heads;
    const PrefillWorkList work =
        cut ? prefill_work_list(in.data(), seqs, group, kv_heads, head_dim, sliding_window, device_cus())
            : prefill_whole_list(in.data(), seqs, group, head_dim, sliding_window);
    list->item_count = (int32_t)work.items.size();
    list->merge_count = (int32_t)work.merges.size();
    list->part_slots = work.slots;
    const int64_t item_words = (int64_t)work.items.size() * kPrefillItemWords,
                  merge_words = (int64_t)work.merges.size() * kPrefillMergeWords;
    if (!words || capacity < item_words + merge_words)
      return fail(GK_ERR_WORKSPACE, "gk_prefill_list_build: the list needs " + std::to_string(item_words + merge_words) +
                                        " words");
    if (item_words) std::memcpy(words, work.items.data(), item_words * sizeof(int32_t));
    if (merge_words) std::memcpy(words + item_words, work.merges.data(), merge_words * sizeof(int32_t));
    return GK_OK;
  } catch (const std::bad_alloc&) {
    return fail(GK_ERR_OUT_OF_MEMORY, "gk_prefill_list_build: out of host memory");
  }
}

}  // namespace gk

extern "C" int gk_paged_prefill(const gk_prefill_params* params, hipStream_t stream) {
  gk::clear_error();
  return gk::paged_prefill(params, stream);
}

extern "C" int gk_prefill_list_build(const int32_t* seq_first_row, const int32_t* seq_rows, const int32_t* seq_prefix,
                                     int32_t seqs, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                     int32_t sliding_window, int32_t* words, int64_t capacity, gk_prefill_list* list) {
  gk::clear_error();
  return gk::prefill_list_build(seq_first_row, seq_rows, seq_prefix, seqs, q_heads, kv_heads, head_dim, sliding_window,
                                true, words, capacity, list);
}

extern "C" int gk_prefill_list_build_uncut(const int32_t* seq_first_row, const int32_t* seq_rows,
                                           const int32_t* seq_prefix, int32_t seqs, int32_t q_heads, int32_t kv_heads,
                                           int32_t head_dim, int32_t sliding_window, int32_t* words, int64_t capacity,
                                           gk_prefill_list* list) {
  gk::clear_error();
  return gk::prefill_list_build(seq_first_row, seq_rows, seq_prefix, seqs, q_heads, kv_heads, head_dim, sliding_window,
                                false, words, capacity, list);
}

extern "C" size_t gk_prefill_list_workspace_bytes(const gk_prefill_params* params, const gk_prefill_list* list) {
  return params && list && params->struct_size == sizeof(gk_prefill_params) &&
                 list->struct_size == sizeof(gk_prefill_list) && params->kv_heads > 0 && list->part_slots > 0
             ? gk::list_workspace_bytes(params, list)
             : 0;
}

extern "C" int gk_paged_prefill_listed(const gk_prefill_params* params, const gk_prefill_list* list, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  gk::clear_error();
  return gk::paged_prefill_listed(params, list, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int gk_paged_prefill_alibi(const gk_prefill_params* params, const gk_prefill_list* list,
                                      const float* slopes, void* workspace, size_t workspace_bytes,
                                      hipStream_t stream) {
  gk::clear_error();
  if (!slopes) return gk::fail(GK_ERR_INVALID_ARGUMENT, "gk_paged_prefill_alibi: null slopes");
  return gk::paged_prefill_listed(params, list, slopes, workspace, workspace_bytes, stream);
}

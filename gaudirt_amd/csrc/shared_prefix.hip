// Attention of a batch whose requests share a long prefix, the prefix attended
// once for all rows of a group.
//
// A decode step of R rows behind one prefix of P tokens reads, row by row, R
// times the same K/V; the rows' queries against those keys are one matrix
// product. Here a group's (row, head) pairs of a kv head are the columns of a
// tile, so the prefix is read once per tile (256 columns; 64 rows of four heads)
// and its work moves from HBM to the matrix cores:
//   o_i = sum_p 2^(m_p - M) acc_p / sum_p 2^(m_p - M) l_p,  M = max_p m_p
// over the partials p = (m, l, acc) of the prefix's key ranges (the tile's) and
// of the row's own keys' (its own). Two launches:
//  1. the attention: workgroups of the prefill kernel's tiles (eight waves on
//     one K/V tile in LDS) over the prefixes and over runs of many rows, beside
//     workgroups of eight independent waves (shared_worker.hpp) that stream the
//     rows' own keys. Both kinds fill the GPU together: the plan
//     (shared_schedule.hpp) gives the workers as many CUs as their bytes need
//     while the other CUs multiply.
//  2. the merge, one workgroup per (row, head).
// Measured, whole call, against every row by itself (us): 64 rows of 32 q / 8 kv
// heads behind 4096 shared tokens, 32 to 1023 of their own (head_dim 128, 164 MB
// once each) 36.8 / 175, of which the first launch ~30 and the merge 4.0-4.6; 256
// rows behind 32000 (515 MB, 136 GFLOP) 171-176 / 4110, tiles at 1.2 PFLOP/s on 24
// of a kv head's 32 CUs beside workers on the other eight, merge 7.1; 48 rows of
// 16 q / 8 kv heads at head_dim 256 with a window (753 MB) 135 / 256, 5.6 TB/s
// over the call, 6.5 in the steady part.
#include "shared_worker.hpp"

#include <cstring>
#include <new>
#include <string>

namespace gk {

int device_cus();

namespace {

struct SharedMergeArgs {
  const int32_t* merges;  // SharedMerge records
  const float* part_o;
  const float* part_ml;
  int64_t part_cols;
  int32_t group;
  DivMagic group_div;
  uint16_t* out;
  int64_t out_stride;
};

// One (row, head) a workgroup: a part's head_dim floats on D / 4 lanes, four
// parts a lane in one memory round trip, the lanes' states joined in LDS.
template <int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void shared_merge_kernel(SharedMergeArgs a) {
  constexpr int L = D / 4, SUBS = WAVES * 64 / L, UNROLL = 4;
  __shared__ f32x4_t s_o[SUBS][L];
  __shared__ float s_m[SUBS], s_l[SUBS];
  const int sub = threadIdx.x / L, at = threadIdx.x % L;
  const int head = blockIdx.x, kvh = (int)fast_div((uint32_t)head, a.group_div), j = head - kvh * a.group;
  const int32_t* rec = a.merges + (int64_t)blockIdx.y * kSharedMergeWords;
  const int pre_col = scalar_load(rec, 0), pre_parts = scalar_load(rec, 1), pre_stride = scalar_load(rec, 2),
            own_col = scalar_load(rec, 3), own_parts = scalar_load(rec, 4), own_stride = scalar_load(rec, 5),
            row = scalar_load(rec, 6);
  const int parts = pre_parts + own_parts;
  const int64_t col0 = (int64_t)kvh * a.part_cols + j;
  float m_run = -INFINITY, l_run = 0.f;
  f32x4_t acc{0.f, 0.f, 0.f, 0.f};
  for (int p0 = sub; p0 < parts; p0 += SUBS * UNROLL) {
    float m[UNROLL], l[UNROLL];
    f32x4_t o[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int p = min(p0 + u * SUBS, parts - 1);
      const int64_t col = col0 + (p < pre_parts ? pre_col + (int64_t)p * pre_stride
                                                : own_col + (int64_t)(p - pre_parts) * own_stride);
      m[u] = a.part_ml[2 * col];
      l[u] = a.part_ml[2 * col + 1];
      o[u] = *reinterpret_cast<const f32x4_t*>(a.part_o + col * D + 4 * at);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      // A part without a visible key has no output to read, nor have the
      // repeats of the last part.
      if (p0 + u * SUBS >= parts || m[u] == -INFINITY) continue;
      const float mn = fmaxf(m_run, m[u]);
      const float fa = m_run == -INFINITY ? 0.f : fast_exp2(m_run - mn), fb = fast_exp2(m[u] - mn);
      l_run = l_run * fa + l[u] * fb;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = acc[i] * fa + o[u][i] * fb;
      m_run = mn;
    }
  }
  if constexpr (SUBS > 1) {
    s_o[sub][at] = acc;
    if (at == 0) {
      s_m[sub] = m_run;
      s_l[sub] = l_run;
    }
    __syncthreads();
    if (sub) return;
    float mm = -INFINITY;
#pragma unroll
    for (int s = 0; s < SUBS; ++s) mm = fmaxf(mm, s_m[s]);
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    l_run = 0.f;
#pragma unroll
    for (int s = 0; s < SUBS; ++s) {
      const float f = s_m[s] == -INFINITY ? 0.f : fast_exp2(s_m[s] - mm);
      l_run += s_l[s] * f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += s_o[s][at][i] * f;
    }
  }
  const float inv = l_run > 0.f ? 1.f / l_run : 0.f;
  uint2 v;
  v.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  v.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<uint2*>(a.out + (int64_t)row * a.out_stride + (int64_t)head * D + 4 * at) = v;
}

template <int D, int MODE>
void launch_mode(const SharedArgs& a, bool softcap, dim3 grid, hipStream_t stream) {
  if (softcap) prefill_kernel<D, kScoreCap, MODE, SharedArgs><<<grid, kPrefillWaves * 64, 0, stream>>>(a);
  else prefill_kernel<D, kScorePlain, MODE, SharedArgs><<<grid, kPrefillWaves * 64, 0, stream>>>(a);
}

template <int D>
void launch(const SharedArgs& a, bool softcap, int block_size, dim3 grid, hipStream_t stream) {
  constexpr int keys = shared_step_keys(D);
  if (block_size >= keys) launch_mode<D, kStepBlocks>(a, softcap, grid, stream);
  else if (block_size >= keys / PrefillShape<D, keys>::NI) launch_mode<D, kLoadBlocks>(a, softcap, grid, stream);
  else launch_mode<D, kKeyBlocks>(a, softcap, grid, stream);
}

size_t output_bytes(const gk_prefill_params* p, const gk_shared_prefix_list* list) {
  return (size_t)p->kv_heads * list->part_cols * p->head_dim * sizeof(float);
}
size_t workspace_bytes_of(const gk_prefill_params* p, const gk_shared_prefix_list* list) {
  return output_bytes(p, list) + (size_t)p->kv_heads * list->part_cols * 2 * sizeof(float);
}

}  // namespace

int shared_prefix_list_build(const int32_t* run_first_row, const int32_t* run_rows, const int32_t* run_pos,
                             const int32_t* run_group, const int32_t* run_request, int32_t runs,
                             const int32_t* group_prefix, int32_t groups, int32_t q_heads, int32_t kv_heads,
                             int32_t head_dim, int32_t sliding_window, int32_t* words, int64_t capacity,
                             gk_shared_prefix_list* list) {
  const char* const name = "gk_shared_prefix_list_build";
  const auto bad = [&](const char* what) { return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": " + what); };
  if (!list || list->struct_size != sizeof(gk_shared_prefix_list))
    return bad("struct_size does not match this library's gk_shared_prefix_list");
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
      q_heads / kv_heads > 128)
    return bad("invalid head geometry (GQA group at most 128)");
  if (runs <= 0 || runs > 65535 || groups <= 0 || groups > 65535 || capacity < 0 || !run_first_row || !run_rows ||
      !run_pos || !run_group || !group_prefix)
    return bad("invalid runs or groups");
  int64_t rows = 0;
  for (int32_t i = 0; i < runs; ++i) {
    const int32_t g = run_group[i];
    if (g < 0 || g >= groups || (i && g < run_group[i - 1])) return bad("runs are not in the order of their groups");
    if (run_rows[i] <= 0 || run_first_row[i] < 0 || group_prefix[g] < 0 || run_pos[i] < group_prefix[g] ||
        (int64_t)run_pos[i] + run_rows[i] > INT32_MAX - 64)
      return bad("a run's rows must lie behind its group's prefix");
    if (run_request && run_request[i] < 0) return bad("negative request");
    rows += run_rows[i];
  }
  if (rows > 65535) return bad("too many rows");
  try {
    std::vector<SharedRun> in(runs);
    for (int32_t i = 0; i < runs; ++i)
      in[i] = {run_first_row[i], run_rows[i], run_pos[i], run_group[i], run_request ? run_request[i] : -1};
    const SharedPlan plan =
        shared_plan(in.data(), runs, group_prefix, q_heads / kv_heads, kv_heads, head_dim, sliding_window, device_cus());
    if (plan.cols > INT32_MAX) return bad("too many partial results");
    int64_t total = 0;
    const auto reserve = [&](int64_t count) {
      const int64_t at = total;
      total += (count + 3) / 4 * 4;
      return (int32_t)at;
    };
    list->rows = (int32_t)plan.row_map.size();
    list->tile_count = (int32_t)plan.tiles.size();
    list->workers = (int32_t)plan.workers.size();
    list->worker_groups = plan.worker_groups;
    list->part_cols = plan.cols;
    list->can_store = plan.stores;
    list->q_heads = q_heads;
    list->kv_heads = kv_heads;
    list->head_dim = head_dim;
    list->sliding_window = sliding_window > 0 ? sliding_window : -1;
    list->map_at = reserve(list->rows);
    list->position_at = reserve(list->rows);
    list->merges_at = reserve(int64_t{kSharedMergeWords} * list->rows);
    list->tiles_at = reserve(int64_t{kSharedTileWords} * list->tile_count);
    list->workers_at = reserve(int64_t{kSharedWorkerWords} * list->workers);
    list->segments_at = reserve(int64_t{kSharedSegmentWords} * (int64_t)plan.segs.size());
    if (total > INT32_MAX) return bad("too much work");
    list->word_count = (int32_t)total;
    if (!words || capacity < total)
      return fail(GK_ERR_WORKSPACE, std::string(name) + ": the list needs " + std::to_string(total) + " words");
    std::memset(words, 0, total * sizeof(int32_t));
    const auto put = [&](int32_t at, const auto& v) {
      if (!v.empty()) std::memcpy(words + at, v.data(), v.size() * sizeof(v[0]));
    };
    put(list->map_at, plan.row_map);
    put(list->position_at, plan.row_position);
    put(list->merges_at, plan.merges);
    put(list->tiles_at, plan.tiles);
    put(list->workers_at, plan.workers);
    put(list->segments_at, plan.segs);
    return GK_OK;
  } catch (const std::bad_alloc&) {
    return fail(GK_ERR_OUT_OF_MEMORY, std::string(name) + ": out of host memory");
  }
}

int shared_prefix_attention(const gk_prefill_params* p, const gk_shared_prefix_list* list, void* workspace,
                            size_t workspace_bytes, hipStream_t stream) {
  const char* const name = "gk_shared_prefix_attention";
  if (int rc = check_prefill(p, true, name)) return rc;
  if (!list || list->struct_size != sizeof(gk_shared_prefix_list))
    return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": struct_size does not match this library's gk_shared_prefix_list");
  if (list->q_heads != p->q_heads || list->kv_heads != p->kv_heads || list->head_dim != p->head_dim ||
      list->sliding_window != (p->sliding_window > 0 ? p->sliding_window : -1))
    return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": the list was built for other heads or another window");
  if (list->rows < 0 || list->rows > 65535 || list->tile_count < 0 || list->workers < 0 || list->worker_groups < 0 ||
      list->worker_groups != (list->workers + kSharedWaves - 1) / kSharedWaves || list->part_cols < 0 ||
      list->part_cols > INT32_MAX)
    return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": list counts out of range");
  if (list->rows == 0) return GK_OK;
  if (!list->words || !list->row_request || (reinterpret_cast<uintptr_t>(list->words) & 15))
    return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": null or misaligned list");
  if (list->new_key) {
    if (!list->can_store || !list->new_value)
      return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": this list cannot store, or new_value is null");
    if (int rc = check_kv_store(list->new_key, list->new_value, list->new_kv_row_stride, list->new_kv_row_stride, p->pool,
                                p->kv_heads, p->head_dim))
      return rc;
  }
  const size_t need = workspace_bytes_of(p, list);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(GK_ERR_WORKSPACE, std::string(name) + ": workspace too small or not 16-byte aligned (" +
                                      std::to_string(need) + " bytes needed)");
  SharedArgs a{};
  static_cast<PrefillArgs&>(a) = prefill_args(p);
  a.items = list->words + list->tiles_at;
  a.tile_count = list->tile_count;
  a.item_count = list->tile_count + list->worker_groups;
  a.workers = list->workers;
  a.worker_list = list->words + list->workers_at;
  a.segs = list->words + list->segments_at;
  a.row_map = list->words + list->map_at;
  a.row_position = list->words + list->position_at;
  a.row_request = list->row_request;
  a.new_key = static_cast<const uint16_t*>(list->new_key);
  a.new_value = static_cast<const uint16_t*>(list->new_value);
  a.new_stride = list->new_kv_row_stride;
  a.pool_out = static_cast<uint16_t*>(const_cast<void*>(p->pool));
  a.part_cols = list->part_cols;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + output_bytes(p, list));
  int classes = kXcds;
  while (p->kv_heads % classes) classes /= 2;
  a.class_shift = log2_int(classes);
  a.class_heads = p->kv_heads / classes;
  a.class_xcds = kXcds / classes;
  a.class_heads_div = div_magic((uint32_t)a.class_heads);
  const int64_t per_xcd = ((int64_t)a.item_count + a.class_xcds - 1) / a.class_xcds * a.class_heads;
  if (per_xcd * kXcds > (int64_t)1 << 30) return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + ": too many items");
  const dim3 grid((unsigned)(per_xcd * kXcds));
  const bool softcap = p->softcap > 0.f;
  if (p->head_dim == 64) launch<64>(a, softcap, p->block_size, grid, stream);
  else if (p->head_dim == 128) launch<128>(a, softcap, p->block_size, grid, stream);
  else launch<256>(a, softcap, p->block_size, grid, stream);
  if (int rc = hip_status(hipGetLastError(), "gk_shared_prefix_attention launch")) return rc;
  SharedMergeArgs m{};
  m.merges = list->words + list->merges_at;
  m.part_o = a.part_o;
  m.part_ml = a.part_ml;
  m.part_cols = a.part_cols;
  m.group = a.group;
  m.group_div = a.group_div;
  m.out = a.out;
  m.out_stride = a.out_stride;
  const dim3 mgrid((unsigned)p->q_heads, (unsigned)list->rows);
  const auto merge = [&](auto waves) {
    constexpr int W = decltype(waves)::value;
    if (p->head_dim == 64) shared_merge_kernel<64, W == 8 ? 4 : W><<<mgrid, (W == 8 ? 4 : W) * 64, 0, stream>>>(m);
    else if (p->head_dim == 128) shared_merge_kernel<128, W><<<mgrid, W * 64, 0, stream>>>(m);
    else shared_merge_kernel<256, W><<<mgrid, W * 64, 0, stream>>>(m);
  };
  // Few (row, head) pairs have many parts each and leave CUs idle: more waves take a pair's parts side by side. Many
  // pairs fill the GPU by themselves. One / four / eight waves (us): head_dim 128, 32 pairs 21.4 / 7.0 / 5.2, 256 pairs
  // 13.4 / 5.7 / 5.5, 512 4.2 / 3.9 / 4.0, 1024 5.6 / 5.2 / 5.2, 2048 6.0 / 6.0 / 7.3, 8192 6.4 / 10.0 / 15.6; head_dim
  // 256, 128 pairs 30.3 / 10.3 / 7.0, 1024 6.4 / 5.9 / 5.6, 2048 5.7 / 5.9 / 7.4; head_dim 64, where four waves hold 16
  // parts already, 56 pairs 11.4 / 4.7 / 5.0, 896 4.0 / 4.0 / 5.3, 1792 4.3 / 4.8 / 7.1.
  const int64_t pairs = (int64_t)list->rows * p->q_heads;
  if (pairs <= 512) merge(std::integral_constant<int, 8>{});
  else if (pairs <= 1024) merge(std::integral_constant<int, 4>{});
  else merge(std::integral_constant<int, 1>{});
  return hip_status(hipGetLastError(), "gk_shared_prefix_attention merge launch");
}

}  // namespace gk

extern "C" int gk_shared_prefix_list_build(const int32_t* run_first_row, const int32_t* run_rows,
                                           const int32_t* run_pos, const int32_t* run_group,
                                           const int32_t* run_request, int32_t runs,
                                           const int32_t* group_prefix, int32_t groups, int32_t q_heads,
                                           int32_t kv_heads, int32_t head_dim, int32_t sliding_window, int32_t* words,
                                           int64_t capacity, gk_shared_prefix_list* list) {
  gk::clear_error();
  return gk::shared_prefix_list_build(run_first_row, run_rows, run_pos, run_group, run_request, runs, group_prefix,
                                      groups, q_heads, kv_heads, head_dim, sliding_window, words, capacity, list);
}

extern "C" size_t gk_shared_prefix_workspace_bytes(const gk_prefill_params* params, const gk_shared_prefix_list* list) {
  return params && list && params->struct_size == sizeof(gk_prefill_params) &&
                 list->struct_size == sizeof(gk_shared_prefix_list) && params->kv_heads > 0 && params->head_dim > 0 &&
                 list->part_cols > 0
             ? gk::workspace_bytes_of(params, list)
             : 0;
}

extern "C" int gk_shared_prefix_attention(const gk_prefill_params* params, const gk_shared_prefix_list* list,
                                          void* workspace, size_t workspace_bytes, hipStream_t stream) {
  gk::clear_error();
  return gk::shared_prefix_attention(params, list, workspace, workspace_bytes, stream);
}

// Work plan of a shared-prefix attention launch: which keys every workgroup and
// every one-wave worker takes, and where its partial results go. Plain host
// C++, built once per attention plan from lengths that the plan's owner has on
// the host; the CPU tests compile it with g++.
//
// Rows come in groups whose rows hold the same slots for the group's first
// `prefix` tokens. The group's columns, (row, head) pairs of one kv head, attend
// those keys together: in tiles of up to prefill_tile_qrows columns (eight waves
// on one K/V tile in LDS) or, where columns are few and keys many, as one wave's
// columns. Behind the prefix every run of rows (consecutive positions of one
// request) attends its own keys. Both kinds of work are cut along their keys; each
// piece leaves an unnormalised partial, and a second launch joins a row's partials.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

#include "prefill_schedule.hpp"

namespace gk {

// A worker is one wave: at most shared_columns columns (two 16-column tiles; one
// at head_dim 256, where two spill 77 registers), tiles of shared_tile_keys keys.
constexpr int shared_columns(int head_dim) { return head_dim > 128 ? 16 : 32; }
constexpr int shared_step_keys(int head_dim) { return head_dim > 128 ? 32 : 64; }  // of a workgroup's tile
constexpr int shared_tile_keys(int head_dim) { return head_dim > 128 ? 16 : 32; }
constexpr int kSharedWaves = 8;  // workers of a workgroup

struct SharedRun {
  int32_t first_row, rows, pos, group, request;  // request: its block-table row; -1: only the device knows
};

// A tile of a workgroup: compact rows first .. first + rows - 1, keys
// [key_lo, key_hi) in `steps` steps of shared_step_keys from key0 on. pos >= 0:
// the rows are the batch rows from batch_row on, at positions pos, pos + 1, ...
// (behind all of the tile's keys, whatever they are, where no row's window starts
// among them); else rows and positions are looked up.
struct SharedTile {
  int32_t first, rows, key_lo, key_hi, key0, steps, col, batch_row, pos, request, pad[2];
};
constexpr int kSharedTileWords = 12;
// A stretch of one worker's keys: `cols` columns of the compact rows from `first`
// on, key tiles tile0 .. tile0 + tiles - 1; rows and positions as a tile's. From
// key new_pos on, keys are the run's new tokens: those of the batch rows from
// new_row on (INT32_MAX: none).
struct SharedSegment {
  int32_t first, cols, tile0, tiles, key_lo, key_hi, col, batch_row, pos, new_pos, new_row, request;
};
constexpr int kSharedSegmentWords = 12;
// A worker's first segment, and where its others stand among the segments.
struct SharedWorker {
  SharedSegment first;
  int32_t next, end, pad[2];
};
constexpr int kSharedWorkerWords = 16;
// Where a row's partials are: columns pre_col + p pre_stride (p < pre_parts) of
// its prefix, own_col + p own_stride of its own keys, one column a head.
struct SharedMerge {
  int32_t pre_col, pre_parts, pre_stride, own_col, own_parts, own_stride, batch_row, pad;
};
constexpr int kSharedMergeWords = 8;

struct SharedPlan {
  std::vector<int32_t> row_map, row_position;
  std::vector<SharedWorker> workers;
  std::vector<SharedMerge> merges;   // one per compact row
  std::vector<SharedTile> tiles;     // longest first
  std::vector<SharedSegment> segs;
  int64_t cols = 0;                  // partial columns of one kv head
  int32_t worker_groups = 0;         // workgroups of workers
  bool stores = true;                // workers see every new token: they can store it
};

// What the split weighs, in microseconds. A worker's key tile takes `key_tile`
// while few workers run; under load latency and bandwidth add up like the sides
// of a right angle. Measured against the share of a kv head's CUs that workers
// get, whole call (us): 64 rows of 32 to 1023 own keys behind 4096, 32 q / 8 kv
// heads: 3 of 32 CUs 128, 8 65, 12 54, 16 49, 22 42, 27 39, 28 42; 256 rows of 16
// to 700 behind 32000: 6 187, 8 177, 9 191, 16 212, 19 271; 48 rows of 16 q / 8
// kv heads at head_dim 256 with a window: 8 243, 16 170, 22 145, 28 129.
struct SharedCost {
  double step;        // a tile's step with all its waves busy, a quarter of it whatever the columns
  double tile_start;  // a workgroup's start and end
  double key_tile;    // a worker's key tile
  double bytes;       // of a worker's key tile
};
inline SharedCost shared_cost(int head_dim) {
  if (head_dim == 64) return {1.2, 5.0, 1.8, 32 * 64 * 4.0};
  if (head_dim == 128) return {1.95, 6.0, 2.35, 32 * 128 * 4.0};
  return {1.8, 6.0, 2.35, 16 * 256 * 4.0};
}
constexpr double kSharedBandwidth = 6.3e6;  // bytes a microsecond
constexpr double kSegmentTiles = 2.0;       // a segment's start and end, in key tiles

// Work of one kv head before it is cut.
struct SharedWork {
  int32_t first, rows, key_lo, key_hi;  // compact rows and their keys
  int32_t run;                          // compact row of the run whose own keys these are; -1: its group's prefix
  int32_t units;                        // steps of a tile, key tiles of a worker
  int32_t start;                        // first key, aligned
};

inline SharedPlan shared_plan(const SharedRun* runs, int count, const int32_t* group_prefix, int group, int kv_heads,
                              int head_dim, int window, int cus) {
  SharedPlan plan;
  const int tile_cols = prefill_tile_qrows(head_dim), tile_rows = tile_cols / group;
  const int step_keys = shared_step_keys(head_dim), key_tile = shared_tile_keys(head_dim);
  const int columns = shared_columns(head_dim), slots = std::max(1, cus / kv_heads);
  // Prefixes of few columns, in keys a CU: what decides who attends them. Workers stream at HBM's rate, but each
  // leaves a partial of every column; a tile's workgroup leaves one and streams at two thirds of the rate. Whole call,
  // tile / worker (us), head_dim 128: 375 keys a CU, 8 columns 17.1 / 19.4, 12 17.7 / 23.2; 1000 keys, 8 columns 28.6
  // / 29.6, 16 29.7 / 33.5, 32 32.7 / 42.3; 750 keys, 4 columns 33.8 / 26.6; 1500 keys, 2 columns 50.2 / 40.1, 3000
  // keys, 4 columns 120 / 72, 16 columns 124 / 84. head_dim 256: 375 keys, 2 columns 23.0 / 25.8, 16 23.7 / 36.4;
  // 1500, 6 columns 92 / 81. head_dim 64: 375 keys, 21 columns 15.2 / 17.5; 3000, 7 columns 86 / 41.
  int64_t few_keys = 0;
  for (int i = 0; i < count;) {
    const int g = runs[i].group;
    int rows = 0, low = INT32_MAX;
    for (; i < count && runs[i].group == g; ++i) {
      rows += runs[i].rows;
      low = std::min(low, runs[i].pos);
    }
    if (rows % tile_rows && rows % tile_rows * group <= columns)
      few_keys += std::max(0, group_prefix[g] - (window > 0 ? std::max(0, low - window + 1) : 0));
  }
  const int64_t few_a_cu = few_keys / slots;
  const int prefix_columns = few_a_cu <= 512 ? 0 : few_a_cu <= 1024 ? columns / 4 : columns;  // of a worker, at most
  std::vector<SharedWork> wide, narrow;
  std::vector<int32_t> row_request;  // of compact rows
  const auto add = [&](int first, int rows, int lo, int hi, int run) {
    // Own keys are a worker's up to the columns of two, which streams them twice at most.
    if (lo >= hi) return;
    const bool own = run >= 0;
    SharedWork w{first, rows, lo, hi, run, 0, 0};
    const bool tile = group > columns || rows * group > (own ? 2 * columns : prefix_columns);
    if (tile) {
      w.start = lo / step_keys * step_keys;
      w.units = (hi - w.start + step_keys - 1) / step_keys;
      wide.push_back(w);
      plan.stores = plan.stores && !own;
      return;
    }
    const int most = columns / group;  // rows of a worker
    w.start = lo / key_tile * key_tile;
    for (int r = 0; r < rows; r += most) {
      w.first = first + r;
      w.rows = std::min(most, rows - r);
      if (own) w.key_hi = hi - (rows - r - w.rows);  // the slice's last row's own key
      w.units = (w.key_hi - w.start + key_tile - 1) / key_tile;
      narrow.push_back(w);
    }
  };
  // Rows in the order of their runs; a group's rows are side by side.
  for (int i = 0; i < count;) {
    const int g = runs[i].group, first = (int)plan.row_map.size(), prefix = group_prefix[g];
    for (; i < count && runs[i].group == g; ++i) {
      const SharedRun& run = runs[i];
      const int at = (int)plan.row_map.size();
      for (int r = 0; r < run.rows; ++r) {
        plan.row_map.push_back(run.first_row + r);
        plan.row_position.push_back(run.pos + r);
        row_request.push_back(run.request);
        plan.merges.push_back({0, 0, 0, 0, 0, 0, run.first_row + r, 0});
      }
      for (int r = 0; r < run.rows; r += tile_rows) {
        const int nr = std::min(tile_rows, run.rows - r), pos = run.pos + r;
        add(at + r, nr, std::max(prefix, window > 0 ? pos - window + 1 : 0), pos + nr, at);
      }
    }
    const int rows = (int)plan.row_map.size() - first;
    for (int r = 0; r < rows; r += tile_rows) {
      const int nr = std::min(tile_rows, rows - r);
      int lo = 0;
      if (window > 0) {
        lo = INT32_MAX;
        for (int k = 0; k < nr; ++k) lo = std::min(lo, std::max(0, plan.row_position[first + r + k] - window + 1));
      }
      add(first + r, nr, lo, prefix, -1);
    }
  }

  // Pieces of at most `most` steps: the fewest steps with which one round of
  // `room` workgroups holds all pieces; whole where there are more tiles than that.
  const auto tile_pieces = [&](int room) {
    int lo = 4, hi = 4;
    for (const auto& w : wide) hi = std::max(hi, w.units);
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      int64_t sum = 0;
      for (const auto& w : wide) sum += (w.units + mid - 1) / mid;
      if (sum <= room) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };

  // How many of a kv head's CUs take workers: the number with which both kinds
  // of work, side by side, end soonest.
  const SharedCost cost = shared_cost(head_dim);
  int64_t key_tiles = 0;
  for (const auto& w : narrow) key_tiles += w.units;
  int best = narrow.empty() ? 0 : slots;
  if (!narrow.empty() && !wide.empty()) {
    double steps = 0;
    for (const auto& w : wide) {
      const int waves = (w.rows * group + tile_cols / 8 - 1) / (tile_cols / 8);
      steps = std::max(steps, cost.step * (0.25 + 0.75 * waves / 8));
    }
    const double bandwidth = key_tiles * cost.bytes * kv_heads / kSharedBandwidth;
    double best_time = 1e30;
    const int stride = std::max(1, slots / 32);
    for (int a = stride; a < slots || a == stride; a += stride) {
      const double workers = double(a) * kSharedWaves;
      const double latency = cost.key_tile * (key_tiles + kSegmentTiles * std::max<double>(workers, narrow.size())) / workers;
      const double busy = std::sqrt(latency * latency + bandwidth * bandwidth);
      const int room = std::max(1, slots - a), most = tile_pieces(room);
      int64_t pieces = 0;
      for (const auto& w : wide) pieces += (w.units + most - 1) / most;
      const double beside = double((pieces + room - 1) / room) * (most * steps + cost.tile_start);
      const double time = std::max(busy, beside);
      if (time < best_time) {
        best_time = time;
        best = a;
      }
    }
  }
  // Two key tiles a worker at least: each segment costs a partial and a start.
  int workers = (int)std::min<int64_t>(int64_t{best} * kSharedWaves, std::max<int64_t>(1, (key_tiles + 1) / 2));
  if (narrow.empty()) workers = 0;
  const int tile_slots = std::max(1, slots - (workers + kSharedWaves - 1) / kSharedWaves);

  // A record's pos (SharedTile).
  const auto position = [&](const SharedWork& w) {
    const int row0 = plan.row_map[w.first], pos0 = plan.row_position[w.first];
    bool rows_follow = true, positions_follow = true;
    for (int r = 1; r < w.rows; ++r) {
      rows_follow = rows_follow && plan.row_map[w.first + r] == row0 + r;
      positions_follow = positions_follow && plan.row_position[w.first + r] == pos0 + r;
    }
    const bool see_all = window <= 0 && w.run < 0;
    return !rows_follow ? -1 : positions_follow ? pos0 : see_all ? w.key_hi : -1;
  };
  const auto place = [&](const SharedWork& w, int parts) {
    // Columns of the work's parts, a multiple of 16 each.
    const int stride = (w.rows * group + 15) / 16 * 16;
    const int64_t col = plan.cols;
    plan.cols += int64_t{stride} * parts;
    for (int r = 0; r < w.rows; ++r) {
      SharedMerge& m = plan.merges[w.first + r];
      const int32_t at = (int32_t)(col + int64_t{r} * group);
      if (w.run >= 0) m.own_col = at, m.own_parts = parts, m.own_stride = stride;
      else m.pre_col = at, m.pre_parts = parts, m.pre_stride = stride;
    }
    return col;
  };

  if (!wide.empty()) {
    const int most = tile_pieces(tile_slots);
    for (const auto& w : wide) {
      const int parts = (w.units + most - 1) / most, pos = position(w);
      const int64_t col = place(w, parts);
      const int stride = (w.rows * group + 15) / 16 * 16;
      for (int p = 0, done = 0; p < parts; ++p) {
        const int end = (int)(int64_t{w.units} * (p + 1) / parts);
        plan.tiles.push_back({w.first, w.rows, w.key_lo, w.key_hi, w.start + done * step_keys, end - done,
                              (int32_t)(col + int64_t{p} * stride), plan.row_map[w.first], pos, row_request[w.first], {0, 0}});
        done = end;
      }
    }
    std::stable_sort(plan.tiles.begin(), plan.tiles.end(), [](const SharedTile& a, const SharedTile& b) {
      if (a.steps != b.steps) return a.steps > b.steps;
      return a.key0 < b.key0;  // pieces of one key range together: they read the same K/V
    });
  }

  // Workers: all key tiles end to end, each piece after one position that stands
  // for its start and end, in equal shares: the smallest with which the workers
  // suffice.
  if (workers) {
    std::vector<int32_t> piece_ends, pieces_of, worker_segs;  // key tiles where each piece ends; pieces of each work
    int64_t share = std::max<int64_t>(3, (key_tiles + (int64_t)narrow.size() + workers - 1) / workers);
    for (;; share += std::max<int64_t>(1, share / 64)) {
      piece_ends.clear();
      pieces_of.clear();
      worker_segs.assign(1, 0);
      int64_t room = share;
      for (const auto& w : narrow) {
        int pieces = 0;
        for (int done = 0; done < w.units; ++pieces) {
          if (room < 2) {
            worker_segs.push_back((int32_t)piece_ends.size());
            room = share;
          }
          int take = (int)std::min<int64_t>(w.units - done, room - 1);
          if (w.units - done - take == 1) ++take;  // no piece of one tile
          done += take;
          room -= take + 1;
          piece_ends.push_back(done);
        }
        pieces_of.push_back(pieces);
      }
      worker_segs.push_back((int32_t)piece_ends.size());
      if ((int)worker_segs.size() - 1 <= workers) break;
    }
    size_t at = 0, worker = 0;
    for (size_t i = 0; i < narrow.size(); ++i) {
      const SharedWork& w = narrow[i];
      const int pos = position(w);
      const int64_t col = place(w, pieces_of[i]);
      const int stride = (w.rows * group + 15) / 16 * 16;
      for (int p = 0, done = 0; p < pieces_of[i]; ++p, ++at) {
        const SharedSegment seg{w.first, w.rows * group, w.start / key_tile + done, piece_ends[at] - done, w.key_lo,
                                w.key_hi, (int32_t)(col + int64_t{p} * stride), plan.row_map[w.first], pos,
                                w.run < 0 ? INT32_MAX : plan.row_position[w.run],
                                w.run < 0 ? 0 : plan.row_map[w.run], row_request[w.first]};
        done = piece_ends[at];
        if ((int32_t)at == worker_segs[worker]) {
          plan.workers.push_back({seg, (int32_t)plan.segs.size(), (int32_t)plan.segs.size(), {0, 0}});
          ++worker;
        } else {
          plan.segs.push_back(seg);
          plan.workers.back().end = (int32_t)plan.segs.size();
        }
      }
    }
    plan.worker_groups = ((int)plan.workers.size() + kSharedWaves - 1) / kSharedWaves;
  }
  return plan;
}

}  // namespace gk

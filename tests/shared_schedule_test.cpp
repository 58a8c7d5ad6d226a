// CPU checks of gaudirt_amd/csrc/shared_schedule.hpp: for many sets of groups,
// runs, head geometries and windows, every (row, visible key) is attended
// exactly once by the pieces that the row's merge record names, every piece
// stays inside the keys of the row whose block table it reads, partial columns
// are distinct, and workers hold whole segments in order. Prints OK on success.
#include <cstdio>
#include <map>
#include <random>
#include <vector>

#include "shared_schedule.hpp"

namespace {

int failures = 0;
void expect(bool ok, const char* what, int trial) {
  if (!ok && failures++ < 10) std::printf("trial %d: %s\n", trial, what);
}

struct Piece {
  int first, rows, lo, hi;  // compact rows; keys the piece's steps or tiles reach
};

void check(const std::vector<gk::SharedRun>& runs, const std::vector<int32_t>& prefix, int group, int kv_heads, int d,
           int window, int trial) {
  const auto plan = gk::shared_plan(runs.data(), (int)runs.size(), prefix.data(), group, kv_heads, d, window, 256);
  std::vector<gk::SharedRun> row_run;
  for (const auto& run : runs)
    for (int r = 0; r < run.rows; ++r) row_run.push_back({run.first_row + r, 1, run.pos + r, run.group, run.request});
  const size_t rows = row_run.size();
  expect(plan.row_map.size() == rows && plan.row_position.size() == rows && plan.merges.size() == rows, "row count", trial);
  for (size_t i = 0; i < rows; ++i)
    expect(plan.row_map[i] == row_run[i].first_row && plan.row_position[i] == row_run[i].pos &&
               plan.merges[i].batch_row == row_run[i].first_row,
           "a compact row", trial);
  std::vector<char> used(plan.cols, 0);
  std::map<int64_t, Piece> pieces;  // by first partial column
  const auto add = [&](int first, int n, int lo, int hi, int col, int batch_row) {
    expect(first >= 0 && n > 0 && first + n <= (int)rows && lo < hi, "a piece's rows and keys", trial);
    expect(batch_row == plan.row_map[first], "the row whose block table a piece reads", trial);
    expect(lo >= 0 && hi <= row_run[first + n - 1].pos + 1, "a piece reads behind its rows", trial);
    const int width = (n * group + 15) / 16 * 16;
    expect(col >= 0 && col + width <= plan.cols, "a partial column out of range", trial);
    for (int c = col; c < col + width && c < plan.cols; ++c) {
      expect(!used[c], "two pieces share a partial column", trial);
      used[c] = 1;
    }
    pieces[col] = {first, n, lo, hi};
  };
  const int step = gk::shared_step_keys(d), tile = gk::shared_tile_keys(d);
  for (size_t i = 0; i < plan.tiles.size(); ++i) {
    const auto& t = plan.tiles[i];
    expect(t.steps > 0 && t.key0 % step == 0, "a tile's steps", trial);
    expect(t.rows * group <= gk::prefill_tile_qrows(d), "a tile's columns", trial);
    expect(t.request == row_run[t.first].request, "a tile's request", trial);
    for (int r = 0; t.pos >= 0 && r < t.rows; ++r)
      expect(plan.row_map[t.first + r] == t.batch_row + r &&
                 (t.pos + r == row_run[t.first + r].pos ||
                  (window <= 0 && std::min(t.pos + r, row_run[t.first + r].pos) >= t.key_hi - 1)),
             "a tile's rows and positions", trial);
    expect(i == 0 || plan.tiles[i - 1].steps >= t.steps, "tiles are not longest first", trial);
    add(t.first, t.rows, std::max(t.key_lo, t.key0), std::min(t.key_hi, t.key0 + t.steps * step), t.col, t.batch_row);
  }
  const auto segment = [&](const gk::SharedSegment& s) {
    expect(s.tiles > 0 && s.cols > 0 && s.cols <= gk::shared_columns(d) && s.cols % group == 0, "a segment", trial);
    add(s.first, s.cols / group, std::max(s.key_lo, s.tile0 * tile), std::min(s.key_hi, (s.tile0 + s.tiles) * tile), s.col,
        s.batch_row);
    expect(s.request == row_run[s.first].request, "a segment's request", trial);
    // New tokens: the run's rows, seen by a run's own segments only.
    if (s.new_pos != INT32_MAX) {
      const gk::SharedRun* run = nullptr;
      for (const auto& x : runs)
        if (s.batch_row >= x.first_row && s.batch_row < x.first_row + x.rows) run = &x;
      expect(run && s.new_pos == run->pos && s.new_row == run->first_row && s.key_hi <= run->pos + run->rows &&
                 s.key_lo >= std::min(prefix[run->group], run->pos),
             "a segment's new tokens", trial);
    } else {
      expect(s.key_hi <= prefix[row_run[s.first].group], "an own segment without its new tokens", trial);
    }
    if (s.pos < 0) return;
    for (int r = 0; r < s.cols / group && s.first + r < (int)rows; ++r) {
      const int pos = row_run[s.first + r].pos;
      expect(plan.row_map[s.first + r] == s.batch_row + r, "a segment's rows do not follow each other", trial);
      expect(s.pos + r == pos || (window <= 0 && std::min(s.pos + r, pos) >= s.key_hi - 1), "a segment's positions", trial);
    }
  };
  int32_t at = 0;
  for (const auto& w : plan.workers) {
    expect(w.next == at && w.end >= w.next, "a worker's segments", trial);
    segment(w.first);
    for (at = w.next; at < w.end && at < (int32_t)plan.segs.size(); ++at) segment(plan.segs[at]);
  }
  expect(at == (int32_t)plan.segs.size(), "segments without a worker", trial);
  expect(((int)plan.workers.size() + 7) / 8 == plan.worker_groups, "worker groups", trial);
  if (plan.tiles.empty())
    expect(plan.worker_groups <= std::max(1, 256 / kv_heads), "more workers than fit the GPU at once", trial);
  // Every row: its visible keys, each once.
  size_t named = 0;
  for (size_t i = 0; i < rows; ++i) {
    const auto& m = plan.merges[i];
    const int pos = row_run[i].pos, left = window > 0 ? std::max(0, pos - window + 1) : 0;
    std::vector<std::pair<int, int>> ranges;
    const auto parts = [&](int col, int count, int stride) {
      for (int p = 0; p < count; ++p) {
        const int64_t c = (int64_t)col + (int64_t)p * stride;
        auto found = pieces.upper_bound(c);
        expect(found != pieces.begin(), "a merge record names no piece", trial);
        if (found == pieces.begin()) return;
        --found;
        const Piece& q = found->second;
        expect(c - found->first == (int64_t)((int)i - q.first) * group && (int)i >= q.first && (int)i < q.first + q.rows,
               "a merge record names another row's columns", trial);
        ranges.push_back({std::max(q.lo, left), std::min(q.hi, pos + 1)});
        ++named;
      }
    };
    parts(m.pre_col, m.pre_parts, m.pre_stride);
    parts(m.own_col, m.own_parts, m.own_stride);
    std::sort(ranges.begin(), ranges.end());
    int reached = left;
    for (const auto& r : ranges) {
      if (r.first >= r.second) continue;  // no key of this piece is visible to the row
      expect(r.first == reached, "a key is attended twice, or not at all", trial);
      reached = r.second;
    }
    expect(reached == pos + 1, "the row's last key", trial);
  }
  size_t total = 0;
  for (const auto& p : pieces) total += p.second.rows;
  expect(named == total, "a piece that no merge record names", trial);
}

}  // namespace

int main() {
  std::mt19937 rng(7);
  const auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  const int geometry[][3] = {{4, 8, 128}, {8, 8, 128}, {4, 2, 128}, {7, 2, 64}, {2, 8, 256}, {1, 8, 128}, {3, 8, 128},
                             {4, 8, 64},  {128, 1, 128}, {33, 1, 64}, {17, 2, 256}, {128, 1, 256}, {16, 24, 128}};
  for (int trial = 0; trial < 3000; ++trial) {
    const auto& g = geometry[pick(0, 12)];
    const int groups = pick(1, 6);
    std::vector<int32_t> prefix;
    std::vector<gk::SharedRun> runs;
    int row = pick(0, 3);
    for (int k = 0; k < groups; ++k) {
      prefix.push_back(pick(0, 3) ? pick(0, trial % 3 ? 700 : 9000) : 0);
      const int count = pick(1, trial % 5 ? 5 : 60);
      for (int i = 0; i < count; ++i) {
        const int n = pick(0, 2) ? 1 : pick(1, trial % 7 ? 8 : 150);
        runs.push_back({row, n, prefix[k] + (pick(0, 2) ? pick(0, 900) : 0), k, trial % 2 ? (int)runs.size() : -1});
        row += n + (pick(0, 9) == 0);
      }
    }
    const int window = pick(0, 2) ? -1 : pick(1, 2000);
    check(runs, prefix, g[0], g[1], g[2], window, trial);
  }
  if (failures) {
    std::printf("%d failures\n", failures);
    return 1;
  }
  std::printf("OK\n");
  return 0;
}

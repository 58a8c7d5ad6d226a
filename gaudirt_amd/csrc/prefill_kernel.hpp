// The prefill attention kernel: its tile shapes, arguments and body. Launched by
// paged_prefill.hip (causal chunks) and shared_prefix.hip (tiles of a group's
// rows over their shared prefix, beside one-wave workers for the rows' own keys).
#pragma once

#include "gk_mfma.hpp"
#include "prefill_schedule.hpp"
#include "shared_schedule.hpp"
#include "work_order.hpp"

#include <type_traits>

namespace gk {
namespace {

// Waves per workgroup (each owns 16 * kNT query rows). Eight, one workgroup
// per CU (two waves per SIMD): each K/V tile is loaded into LDS once for 256
// query rows instead of twice for two 128-row workgroups (C4, 64-key steps,
// same box: 180.0 -> 174.1 us with four -> eight waves; 168.8 us together with
// the early V reads below).
constexpr int kPrefillWaves = 8;
// 16-column query tiles per wave. Two at head_dim 64 and 128: three fit in 256
// VGPRs only without the early V reads, and four spill; both also quantise
// C4's rows badly (48- or 64-row tiles of 512-row chunks leave a partial round
// of workgroups). One at head_dim 256, whose output accumulators alone take 64
// VGPRs per tile: with two, every head_dim 256 instance spills 536-588 bytes
// per lane; four waves of two tiles (one wave per SIMD, accumulators in AGPRs,
// no spills) measured 163.6-164.7 -> 227.4-227.5 us on C4's shapes at head_dim
// 256: the second wave of a SIMD matters more than halving the operand reads.
constexpr int kNT = 2;
constexpr int kQrowsPerWave = 16 * kNT;
template <int D>
constexpr int prefill_nt() { return D > 128 ? 1 : kNT; }
static_assert(prefill_tile_qrows(64) == kPrefillWaves * 16 * prefill_nt<64>() &&
                  prefill_tile_qrows(128) == kPrefillWaves * 16 * prefill_nt<128>() &&
                  prefill_tile_qrows(256) == kPrefillWaves * 16 * prefill_nt<256>(),
              "the schedule's row tiles are the kernel's");
// Keys per step: 64 at head_dim 128 (half the per-step barriers, cross-lane
// maxima, re-base checks and load setup of 32-key steps: C4 178.1 -> 166.8
// us); 32 at head_dim 64, whose 64-key form needs 130 VGPRs and so would drop
// from four waves per SIMD to three, and at head_dim 256, where a 64-key K
// and V tile pair takes 64 KiB of LDS per stage.
template <int D>
constexpr int prefill_keys() { return prefill_step_keys(D); }
// K/V pipeline depth. Two: three and four stages measured the same on C4 (the
// kernel is bound by its instruction stream, not by load latency).
constexpr int kStages = 2;
constexpr float kLazyRescale = 8.f;
// XCDs of an MI355X: consecutive workgroups of a launch go to consecutive XCDs.
constexpr int kXcds = 8;

struct PrefillArgs {
  const uint16_t* query;
  int64_t q_stride;
  const uint16_t* pool;
  int64_t slots;
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t block_shift;
  const int32_t* seq_request;
  const int32_t* seq_first_row;
  const int32_t* seq_rows;
  const int32_t* seq_prefix;
  int32_t q_heads, kv_heads, group, rows_per_tile;
  int32_t tiles, seqs;  // row tiles per sequence; sequences
  float score_scale;   // scale * log2(e), or scale / softcap when capping
  float softcap_log2;  // softcap * log2(e) when capping
  int32_t window;
  uint16_t* out;
  int64_t out_stride;
  DivMagic tiles_div, seqs_div, group_div;  // division by tiles, seqs and group (work_order.hpp)
  // Work list (prefill_schedule.hpp) instead of the sequence arrays when not null.
  const int32_t* items;
  const int32_t* row_request;  // block-table row of each query row
  int32_t item_count;
  // XCD x serves the kv heads h with h % classes == x % classes, classes =
  // gcd(kv_heads, 8): class_heads = kv_heads / classes heads on class_xcds =
  // 8 / classes XCDs (class_shift = log2 classes).
  int32_t class_shift, class_heads, class_xcds;
  DivMagic class_heads_div;
  int32_t part_slots;          // partial slots of one kv head
  float* part_o;               // [kv head, slot][wave][query tile][16-dim chunk][lane] x 4 output rows
  float* part_ml;              // [kv head, slot][wave][query tile][2][16]: base (log2 units), sum
  const float* slopes;         // [q_heads] distance slopes (kScoreBias)
};

// Arguments of a shared-prefix launch (shared_prefix.hip): items are
// SharedTile records of compact rows, behind them the workgroups of one-wave
// workers; every result is a partial, rows of head_dim floats per column.
struct SharedArgs : PrefillArgs {
  const int32_t* row_map;       // batch row of each compact row
  const int32_t* row_position;
  const int32_t* worker_list;   // SharedWorker records
  const int32_t* segs;          // SharedSegment records
  int32_t tile_count, workers;
  int64_t part_cols;            // columns of one kv head
  // The new tokens' rows, which the workers then store (null: stored before).
  const uint16_t* new_key;
  const uint16_t* new_value;
  int64_t new_stride;
  uint16_t* pool_out;
};

template <int D, int KEYS = prefill_keys<D>()>
struct PrefillShape {
  static constexpr int NC = D / 32;                 // 32-dim k chunks of Q.K
  static constexpr int CPR = D / 8;                 // 16-byte chunks per head row
  static constexpr int NO = D / 16;                 // 16-dim output chunks
  static constexpr int TILE = KEYS * D * 2;  // bytes of one K or V tile
  static constexpr int NI = TILE / 1024;            // 1 KiB load instructions per tile
};

// How a step's slots are found (the MODE template argument):
//  kStepBlocks  blocks of at least a step's keys: one scalar block-table entry per step;
//  kLoadBlocks  blocks of >= 64 / (D / 8) keys (one load instruction's): one
//               scalar entry per load instruction;
//  kKeyBlocks   shorter blocks, down to the token-granular map (block 1): each
//               lane reads its own key's entry with a vector load.
constexpr int kStepBlocks = 0, kLoadBlocks = 1, kKeyBlocks = 2;

// Of the 16 lanes that hold a tile's columns (every 16-lane row holds the same).
__device__ __forceinline__ int columns_min(int x) {
  x = min(x, __builtin_amdgcn_mov_dpp(x, kDppQuadXor1, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_mov_dpp(x, kDppQuadXor2, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_mov_dpp(x, kDppRowHalfMirror, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_mov_dpp(x, kDppRowMirror, 0xf, 0xf, false));
  return __builtin_amdgcn_readfirstlane(x);
}

// The workgroups behind the tiles of a shared-prefix launch (shared_worker.hpp).
template <int D, int SCORE>
__device__ __forceinline__ void shared_worker(const SharedArgs& a, char* lds, int kvh, int worker);
constexpr int kWorkerEntries = 64;  // block-table entries of a worker's tile in LDS (a lane each), two tiles
constexpr int shared_worker_lds(int head_dim) {
  return kSharedWaves * (2 * shared_tile_keys(head_dim) * head_dim * 2 + 2 * kWorkerEntries * 4);
}

// Args: PrefillArgs, or SharedArgs for the tiles of a shared-prefix launch.
template <int D, int SCORE, int MODE, class Args>
__global__ __launch_bounds__(kPrefillWaves * 64, 1) void prefill_kernel(Args a) {
  constexpr bool SHARED = std::is_same_v<Args, SharedArgs>;
  constexpr int kKeys = SHARED ? shared_step_keys(D) : prefill_keys<D>();
  using S = PrefillShape<D, kKeys>;
  // Room between a base and the maximum that set it. A causal tile takes it above the base (a re-base when a score
  // exceeds the base by it: probabilities of up to 2^8), a shared one below (the base lies that far above the
  // maximum: up to 1), so that its unnormalised sums overflow only where the values' own sum does. Powers of two: the
  // results are the same.
  constexpr float kAbove = SHARED ? 0.f : kLazyRescale;
  [[maybe_unused]] constexpr float kBelow = kLazyRescale;
  static_assert(!SHARED || !score_biased(SCORE), "a shared tile's rows keep no distances");
  constexpr bool LOG2 = score_capped(SCORE);  // scores in log2 units before the maxima, not raw products
  // This head dimension's query tiles per wave (in place of the namespace's).
  constexpr int kNT = prefill_nt<D>(), kQrowsPerWave = 16 * kNT;
  static_assert(kKeys == 32 || kKeys == 64, "a step is one or two 32-key halves");
  constexpr int kKG = kKeys / 16;  // 16-key groups per step (Q.K tiles)
  constexpr int kKH = kKeys / 32;  // 32-key halves per step (P.V k chunks)
  // Load instructions per wave per K (or V) tile; wave w issues instructions w, w + waves, ...
  constexpr int LPW = (S::NI + kPrefillWaves - 1) / kPrefillWaves;
  constexpr int NE = MODE == kStepBlocks ? 1 : LPW;  // block-table entries per wave (per lane) per step
  constexpr int KPL = kKeys / S::NI;                 // keys of one load instruction
  constexpr bool CLAMPED = MODE != kStepBlocks;      // entries of keys outside [key_begin, key_end) clamped
  static_assert(MODE != kKeyBlocks || kStages == 2, "per-lane entries rely on the step's full drain");
  // kStages K/V stages. The direct loads are asm statements the compiler does
  // not track, so one array serves every stage; reads are ordered by the
  // explicit vmcnt wait and the barrier of each step.
  // A region of its own (after the stages) holds, after the step loop, each
  // wave's output rows in bf16 (rows padded by 16 bytes so that the four
  // q-groups' rows of a write fall on different banks), read back as 16-byte
  // pieces for the global stores. Being separate from the stages, a wave
  // starts its output as soon as its own last step ends, with no barrier
  // (132 KiB at head_dim 128, one workgroup per CU either way).
  constexpr int kOutRowBytes = 2 * D + 16;
  constexpr int kKvBytes = kStages * 2 * S::TILE,
                kOutBytes = kPrefillWaves * kQrowsPerWave * kOutRowBytes;
  // (Shared tiles leave partials, which need no output rows here.)
  constexpr int kLdsBytes = !SHARED                          ? kKvBytes + kOutBytes
                            : kKvBytes > shared_worker_lds(D) ? kKvBytes
                                                              : shared_worker_lds(D);
  __shared__ __attribute__((aligned(16))) char lds[kLdsBytes];
  auto kv = reinterpret_cast<char(*)[2][S::TILE]>(lds);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform (LDS bases of the direct loads)
  const int q = lane >> 4, c16 = lane & 15;
  // Work item (row tile, sequence, kv head), row tiles fastest, kv heads
  // slowest. Workgroup b runs on XCD b % 8, so b is mapped to items with each
  // XCD taking one contiguous eighth of that order: the workgroups sharing a
  // kv head's K/V (every row tile of every sequence, which share the prefix)
  // run under one L2 instead of fetching it into all eight. Inside its share
  // an XCD takes the row tiles highest first (heavy_first_item).
  //
  // The prologue is a chain of scalar loads: the arguments, the sequence's
  // fields, its first block-table entry, then the first K/V tile. Each link is
  // a memory round trip, so every argument is materialised in one batch at the
  // top and the four sequence fields are loaded together ahead of the
  // early-exit test (the compiler would otherwise fetch the sequence pointers
  // after the work-item arithmetic and the fields one by one: six round trips
  // before the first K/V load instead of three).
  // A work list's record holds all of that in one load.
  const int g = a.group;
  const auto div_group = [&](int x) { return (int)fast_div((uint32_t)x, a.group_div); };
  int kvh, request, first_row, nr, pos_lo, key_begin, kb0, nsteps, slot = -1;
  // Shared tiles: the keys that their rows share; the batch row and position of the first row (SharedTile).
  [[maybe_unused]] int key_lo = 0, key_hi = 0, batch_row0 = 0, pos0 = 0;
  if constexpr (SHARED) {
    asm volatile("" ::"s"(a.items), "s"(a.row_request), "s"(a.item_count), "s"(a.class_shift), "s"(a.class_heads),
                 "s"(a.class_xcds), "s"(a.class_heads_div.mul), "s"(a.class_heads_div.shift), "s"(a.block_tables),
                 "s"(a.query), "s"(a.pool), "s"(a.group), "s"(a.bt_stride), "s"(a.block_shift), "s"(a.window),
                 "s"(a.q_stride), "s"(a.slots), "s"(a.kv_heads), "s"(a.group_div.mul), "s"(a.group_div.shift),
                 "s"(a.row_map), "s"(a.row_position), "s"(a.tile_count), "s"(a.workers), "s"(a.worker_list),
                 "s"(a.segs));
    const int xcd = blockIdx.x % kXcds, j = blockIdx.x / kXcds;
    const int jl = (int)fast_div((uint32_t)j, a.class_heads_div);
    const int li = jl * a.class_xcds + (xcd >> a.class_shift);
    kvh = (xcd & ((1 << a.class_shift) - 1)) + ((j - jl * a.class_heads) << a.class_shift);
    if (li >= a.item_count) return;
    if (li >= a.tile_count) {
      const int worker = (li - a.tile_count) * kPrefillWaves + wave;
      if (worker < a.workers) shared_worker<D, SCORE>(a, lds, kvh, worker);
      return;
    }
    const int32_t* rec = a.items + (int64_t)li * kSharedTileWords;
    first_row = scalar_load(rec, 0);
    nr = scalar_load(rec, 1);
    key_lo = scalar_load(rec, 2);
    key_hi = scalar_load(rec, 3);
    kb0 = scalar_load(rec, 4);
    nsteps = scalar_load(rec, 5);
    slot = scalar_load(rec, 6);
    batch_row0 = scalar_load(rec, 7);
    pos0 = scalar_load(rec, 8);
    request = scalar_load(rec, 9);
    if (request < 0) request = scalar_load(a.row_request, batch_row0);
    key_begin = max(key_lo, kb0);
    pos_lo = 0;
  } else if (a.items) {
    asm volatile("" ::"s"(a.items), "s"(a.row_request), "s"(a.item_count), "s"(a.class_shift), "s"(a.class_heads),
                 "s"(a.class_xcds), "s"(a.class_heads_div.mul), "s"(a.class_heads_div.shift), "s"(a.part_slots),
                 "s"(a.block_tables), "s"(a.query), "s"(a.pool), "s"(a.out), "s"(a.group), "s"(a.bt_stride),
                 "s"(a.block_shift), "s"(a.window), "s"(a.q_stride), "s"(a.slots), "s"(a.kv_heads),
                 "s"(a.group_div.mul), "s"(a.group_div.shift));
    // Item j of this XCD: the list is dealt out over the XCDs of the class,
    // longest items first, the class's kv heads side by side.
    const int xcd = blockIdx.x % kXcds, j = blockIdx.x / kXcds;
    const int jl = (int)fast_div((uint32_t)j, a.class_heads_div);
    const int li = jl * a.class_xcds + (xcd >> a.class_shift);
    kvh = (xcd & ((1 << a.class_shift) - 1)) + ((j - jl * a.class_heads) << a.class_shift);
    if (li >= a.item_count) return;
    const int32_t* rec = a.items + (int64_t)li * kPrefillItemWords;
    first_row = scalar_load(rec, 0);
    nr = scalar_load(rec, 1);
    pos_lo = scalar_load(rec, 2);
    const int key0 = scalar_load(rec, 3);
    nsteps = scalar_load(rec, 4);
    slot = scalar_load(rec, 5);
    request = scalar_load(a.row_request, first_row);
    // The list may be made for a wider window than the call's: steps that lie
    // before every row's window are skipped.
    const int left = a.window > 0 ? max(0, pos_lo - a.window + 1) : 0;
    kb0 = max(key0, left & ~(kKeys - 1));
    nsteps -= (kb0 - key0) / kKeys;
    key_begin = max(left, kb0);
    if (nsteps <= 0) {
      // No visible key in this piece (never a whole item): an empty partial,
      // whose output the merge does not read into its sums.
      if (slot >= 0 && lane < 16) {
        float* ml = a.part_ml + (((int64_t)kvh * a.part_slots + slot) * kPrefillWaves + wave) * (kNT * 32);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          ml[nt * 32 + lane] = -INFINITY;
          ml[nt * 32 + 16 + lane] = 0.f;
        }
      }
      return;
    }
  } else {
    asm volatile("" ::"s"(a.seq_rows), "s"(a.seq_prefix), "s"(a.seq_first_row), "s"(a.seq_request),
                 "s"(a.block_tables), "s"(a.query), "s"(a.pool), "s"(a.out), "s"(a.tiles), "s"(a.seqs),
                 "s"(a.rows_per_tile), "s"(a.group), "s"(a.bt_stride), "s"(a.block_shift), "s"(a.window),
                 "s"(a.q_stride), "s"(a.slots), "s"(a.kv_heads), "s"(gridDim.x), "s"(a.tiles_div.mul),
                 "s"(a.tiles_div.shift), "s"(a.seqs_div.mul), "s"(a.seqs_div.shift), "s"(a.group_div.mul),
                 "s"(a.group_div.shift));
    const int nitems = gridDim.x, xcd = blockIdx.x % kXcds, per_xcd = nitems / kXcds, extra = nitems % kXcds;
    // Divisions by runtime values go through the host's multiply-shift pairs.
    const auto div_tiles = [&](int x) { return (int)fast_div((uint32_t)x, a.tiles_div); };
    const int item = heavy_first_item(xcd * per_xcd + min(xcd, extra), per_xcd + (xcd < extra), a.tiles,
                                      (int)blockIdx.x / kXcds, div_tiles);
    const int item_seq = div_tiles(item), tile = item - item_seq * a.tiles;
    kvh = (int)fast_div((uint32_t)item_seq, a.seqs_div);
    const int seq = item_seq - kvh * a.seqs;
    const int rows = a.seq_rows[seq], prefix = a.seq_prefix[seq], seq_first = a.seq_first_row[seq];
    request = a.seq_request[seq];
    asm volatile("" ::"s"(rows), "s"(prefix), "s"(seq_first), "s"(request));
    const int r0 = tile * a.rows_per_tile;
    if (r0 >= rows) return;
    nr = min(a.rows_per_tile, rows - r0);
    first_row = seq_first + r0;
    pos_lo = prefix + r0;
    key_begin = a.window > 0 ? max(0, pos_lo - a.window + 1) : 0;
    kb0 = key_begin & ~(kKeys - 1);
    nsteps = (pos_lo + nr - kb0 + kKeys - 1) / kKeys;
  }
  const int32_t* __restrict__ bt = a.block_tables + (int64_t)request * a.bt_stride;
  // Keys of this workgroup: [key_begin, key_end), a whole item's or a piece's.
  const int key_end = min(SHARED ? key_hi : pos_lo + nr, kb0 + nsteps * kKeys);

  // This lane's query rows (one per 16-column tile): qrow = (row, head).
  int qpos[kNT], qleft[kNT];
  bool qvalid[kNT];
  bf16x8_t qb[kNT][S::NC];
  [[maybe_unused]] float slope[kNT];
  // Smallest query position and largest window start over this wave's valid rows.
  int wave_pos_min = pos_lo + div_group(wave * kQrowsPerWave);
  int wave_left_max =
      a.window > 0 ? pos_lo + min(nr - 1, div_group(wave * kQrowsPerWave + kQrowsPerWave - 1)) - a.window + 1 : 0;
  auto load_queries = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int qr = wave * kQrowsPerWave + nt * 16 + c16;
      const int row = div_group(qr), head = qr - row * g;
      qvalid[nt] = row < nr;
      int batch_row = first_row + row;
      if constexpr (SHARED) {
        // The rows share the keys [key_lo, key_hi) of the tile; their positions (and windows) are their own.
        const int at = min(row, nr - 1);
        int pos = pos0 + at;
        batch_row = batch_row0 + at;
        if (pos0 < 0) {
          batch_row = a.row_map[first_row + at];
          pos = a.row_position[first_row + at];
        }
        qpos[nt] = qvalid[nt] ? min(pos, key_hi - 1) : -1;
        qleft[nt] = a.window > 0 ? max(key_lo, pos - a.window + 1) : key_lo;
      } else {
        qpos[nt] = qvalid[nt] ? pos_lo + row : -1;
        qleft[nt] = a.window > 0 ? qpos[nt] - a.window + 1 : 0;
      }
      const uint16_t* src = a.query + (int64_t)batch_row * a.q_stride + (int64_t)(kvh * g + head) * D;
      if constexpr (score_biased(SCORE))
        slope[nt] = qvalid[nt] ? fminf(a.slopes[kvh * g + head], kMostSlope) * (LOG2 ? kLog2e : kLog2e / a.score_scale) : 0.f;
#pragma unroll
      for (int c = 0; c < S::NC; ++c) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (qvalid[nt]) v = load16(src + (4 * c + q) * 8);
        qb[nt][c] = __builtin_bit_cast(bf16x8_t, v);
      }
    }

    if constexpr (SHARED) {
      int low = INT32_MAX, left = 0;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        low = min(low, qvalid[nt] ? qpos[nt] : INT32_MAX);
        left = max(left, qvalid[nt] ? qleft[nt] : 0);
      }
      wave_pos_min = columns_min(low);
      wave_left_max = -columns_min(-left);
    }
  };
  // (A shared tile's come behind its first K and V tiles: a chain of round trips less before those.)
  if constexpr (!SHARED) load_queries();

  // At d 128 the row sums of the bf16 probabilities run on one more MFMA per
  // half step against an all-ones operand, in the output layout (rows 4q + r).
  // At d 64 the registers would drop the kernel from four waves per SIMD to
  // three, which costs more than it saves: each lane sums its query row on the
  // VALU (component 0 of l_run).
  constexpr bool kMfmaSum = D >= 128;
  // Step loop (below): at d 64 two groups of waves alternate between MFMA and
  // softmax phases (C4 shapes: 113.7 -> 104.8 us); at d 128 the same order
  // measured 158.9 -> 181.0 us, with or without the phase offset, so d 128
  // keeps one barrier per step with every wave in Q.K -> softmax -> P.V order.
  // (A shared tile has its CU to itself and few steps: there a step of 64 keys
  // and one barrier, whose loads have a whole step to arrive, serve head_dim 64
  // too.)
  constexpr bool kPingPong = D < 128 && !SHARED;
  f32x4_t o[kNT][S::NO];
  float m_run[kNT];
  // Without softcap the re-base check compares the raw score maximum with
  // (m_run + kLazyRescale) / scale, kept per tile and updated at each re-base:
  // the step's maximum is scaled only when a re-base is due.
  float m_thr[kNT];
  const float inv_scale = 1.f / a.score_scale;
  // The base the probabilities are formed against: m_run, or 0 while the row
  // has no maximum yet (kept with m_run, so a step does not select it).
  float m_base[kNT];
  f32x4_t l_run[kNT];
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
    for (int c = 0; c < S::NO; ++c) o[nt][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[nt] = -INFINITY;
    m_thr[nt] = -INFINITY;
    m_base[nt] = 0.f;
    l_run[nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const uint16_t* kbase = a.pool + (int64_t)kvh * a.slots * D;
  const uint16_t* vbase = kbase + (int64_t)a.kv_heads * a.slots * D;
  const uint32_t region = (uint32_t)(a.slots * D * 2);
  // The unrolled d 128 loop passes the resources to the direct-load asm as
  // words made uniform with readfirstlane (the compiler keeps the opaque
  // resource in VGPRs there); d 64 keeps the builtin resource (1.8% faster).
  auto make_rsrc = [&](const uint16_t* base) {
    if constexpr (D < 128 && !SHARED) return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, region, kBufferDword3);
    else return buffer_words(base, region);
  };
  using Rsrc = decltype(make_rsrc(kbase));
  const Rsrc krs = make_rsrc(kbase), vrs = make_rsrc(vbase);
  const int shift = a.block_shift, bmask = (1 << shift) - 1;

  // Block-table entries of the step at key tb (scalar loads, or per-lane
  // vector loads for kKeyBlocks, fetched a step ahead: the loop's wait before
  // its closing barrier covers them). With CLAMPED a key outside
  // [key_begin, key_end) takes the entry of the nearest such key.
  struct Entries {
    int e[NE];
  };
  auto entry_of = [&](int tb) __attribute__((always_inline)) {
    Entries en;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      int key = tb;
      if constexpr (MODE == kLoadBlocks) key += (wave + k * kPrefillWaves) * KPL;
      if constexpr (MODE == kKeyBlocks) key += (wave + k * kPrefillWaves) * KPL + lane / S::CPR;
      if constexpr (CLAMPED) key = min(max(key, key_begin), key_end - 1);
      if constexpr (MODE == kKeyBlocks) en.e[k] = bt[key >> shift];
      else en.e[k] = scalar_load(bt, key >> shift);
    }
    return en;
  };
  // Byte offsets of this wave's direct loads for the step at tb, the same for
  // its K and its V tile. Steps are kKeys-aligned. Piece p = 64 ins + lane of
  // load instruction ins (wave ins % waves): token p / CPR, stored chunk
  // p % CPR holding the token's chunk (p % CPR) ^ swz(token, D / 8). A token
  // outside [key_begin, key_end) reads the row of the nearest token inside:
  // every row read is a stored token, so the masked keys' V rows are finite
  // and their zero probabilities contribute exactly zero (no zeroing pass).
  // The clamped token stays in the block of the entry used for it: blocks of
  // kKeys or more hold the whole step, shorter blocks whole load instructions
  // or (kKeyBlocks) the lane's own token, and clamping is monotone.
  struct Offsets {
    uint32_t v[LPW];
  };
  auto offsets_of = [&](int tb, const Entries& en) __attribute__((always_inline)) {
    Offsets of{};
    // One block holds the whole step: the clamped key's offset in the step
    // stays in [0, kKeys) (the first step starts at or below key_begin, the
    // last holds key_end - 1), so the slot is a scalar base plus that offset.
    const int lo = key_begin - tb, hi = key_end - 1 - tb;
    const uint32_t step_slot = ((uint32_t)en.e[0] << shift) + (uint32_t)(tb & bmask);
#pragma unroll
    for (int k = 0; k < LPW; ++k) {
      const int ins = wave + k * kPrefillWaves;
      if (S::NI % kPrefillWaves != 0 && ins >= S::NI) break;  // wave-uniform
      const int p = ins * 64 + lane, tt = p / S::CPR, pc = p % S::CPR;
      uint32_t slot;
      if constexpr (MODE == kStepBlocks) {
        slot = step_slot + (uint32_t)min(max(tt, lo), hi);
      } else {
        const int key = min(max(tb + tt, key_begin), key_end - 1);
        slot = (uint32_t)((en.e[k] << shift) | (key & bmask));
      }
      of.v[k] = slot * (2 * D) + ((pc ^ swz(tt, D / 8)) << 4);
    }
    return of;
  };
  auto issue = [&](const Offsets& of, Rsrc rs, char* tile) __attribute__((always_inline)) {
    // Per-lane entries are vector loads of the previous step, already complete
    // (the loop waits for every load before its closing barrier); say so to
    // the compiler.
    if constexpr (MODE == kKeyBlocks) wait_vmem_visible();
    const uint32_t base = lds_addr(tile);
#pragma unroll
    for (int k = 0; k < LPW; ++k) {
      const int ins = wave + k * kPrefillWaves;
      if (S::NI % kPrefillWaves != 0 && ins >= S::NI) break;  // wave-uniform
      if constexpr (D < 128 && !SHARED) lds_dma16(base + ins * 1024, rs, of.v[k]);
      else lds_dma16_w(base + ins * 1024, rs, of.v[k]);
    }
  };

  // Scores of the current step and probabilities of the previous one.
  f32x4_t sc[kKG][kNT];
  bf16x8_t pa[kKH][kNT];

  // A distance bias's part inside the step (slope times the key's offset): the
  // scores' accumulators start from it where the registers hold it, else the
  // softmax adds it, one instruction a score. Starting / adding (us): head_dim 64,
  // 8 x 512 rows on 2048 tokens, 32 heads 139.8 / 144.4, 2 x 1000 on 16000 453.6 /
  // 466.8; head_dim 256, 16 heads 196.1 / 197.8, 581.7 / 585.0; head_dim 128, where
  // starting spills 38 registers, 266 / 175.
  constexpr bool kBiasFirst = SCORE == kScoreBias && D != 128;
  [[maybe_unused]] f32x4_t inside[kKG][kNT];
  if constexpr (kBiasFirst) {
#pragma unroll
    for (int h = 0; h < kKG; ++h)
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) inside[h][nt] = bias4(slope[nt], 0.f, h);
  }

  // S^T = K.Q^T into sc: lane (q, c16) gets qrow c16 (+16 nt), keys tb + 16h + 4q + r.
  auto scores = [&](const char* kt) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < kKG; ++h) {
      const int tt = 16 * h + c16;
      bf16x8_t kr[S::NC];
#pragma unroll
      for (int c = 0; c < S::NC; ++c)
        kr[c] = *reinterpret_cast<const bf16x8_t*>(kt + tt * (2 * D) + (((4 * c + q) ^ swz(tt, D / 8)) << 4));
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        if constexpr (kBiasFirst) sc[h][nt] = inside[h][nt];
        else sc[h][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < S::NC; ++c) sc[h][nt] = mfma32(kr[c], qb[nt][c], sc[h][nt]);
      }
    }
  };

  // V operand c of P . V for the 32-key half hh of the V tile vt: keys
  // 32hh + 4q + (c16 >> 2) and 32hh + 16 + 4q + (c16 >> 2), dims
  // 16c + 4 (c16 & 3), read transposed.
  auto read_v = [&](const char* vt, int hh, int c) __attribute__((always_inline)) {
    const int lc = 2 * c + ((c16 & 3) >> 1);
    const int t0 = 32 * hh + 4 * q + (c16 >> 2), t1 = t0 + 16;
    const bf16x4_t v0 = lds_read_tr4(vt + t0 * (2 * D) + ((lc ^ swz(t0, D / 8)) << 4) + ((c16 & 1) << 3));
    const bf16x4_t v1 = lds_read_tr4(vt + t1 * (2 * D) + ((lc ^ swz(t1, D / 8)) << 4) + ((c16 & 1) << 3));
    return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // O[qrow][dim] += P . V with pa and the V tile vt, and the row sums. The
  // first half's operands come from vfirst when the caller read them earlier.
  auto accumulate = [&](const char* vt, const bf16x8_t* vfirst, int nfirst = S::NO) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < S::NO; ++c) {
#pragma unroll
      for (int hh = 0; hh < kKH; ++hh) {
        const bf16x8_t v = (hh == 0 && vfirst && c < nfirst) ? vfirst[c] : read_v(vt, hh, c);
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) o[nt][c] = mfma32(pa[hh][nt], v, o[nt][c]);
      }
    }
    if constexpr (kMfmaSum) {
      const bf16x8_t ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f,
                             (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
#pragma unroll
      for (int hh = 0; hh < kKH; ++hh)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) l_run[nt] = mfma32(pa[hh][nt], ones, l_run[nt]);
    }
  };

  // Online softmax of the step at tb: mask sc, form pa, re-base o and l_run.
  // A step whose keys every valid query row of this wave sees (below the
  // causal diagonal, inside the window) needs no per-element mask. Without
  // softcap the scale folds into the exponent: masked scores become -inf in
  // place (the same registers on both paths), the row maximum is taken on raw
  // scores (scale > 0), and p = exp2(fma(s, scale, -max)).
  auto softmax = [&](int tb) __attribute__((always_inline)) {
    const bool full = tb + kKeys - 1 <= wave_pos_min && tb >= wave_left_max;
    // With a distance bias the scores hold its part inside the step from the start
    // or get it here; the rest, the same for all of a lane's keys, joins the maximum
    // and the exponent's base.
    if constexpr (!LOG2 && (SCORE != kScoreBias || kBiasFirst)) mfma_results_ready(sc);
    // Mask, and each tile's row maximum over this lane's 4 kKG scores.
    float mx[kNT];
    [[maybe_unused]] float bias0[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      if constexpr (LOG2) {
#pragma unroll
        for (int h = 0; h < kKG; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[h][nt][r] = soft_cap(sc[h][nt][r] * a.score_scale, a.softcap_log2);
      }
      if constexpr (SCORE == kScoreCapBias) {
        const float distance = (float)(tb + 4 * q - qpos[nt]);
#pragma unroll
        for (int h = 0; h < kKG; ++h) sc[h][nt] += bias4(slope[nt], distance, h);
      }
      if constexpr (SCORE == kScoreBias) {
        bias0[nt] = slope[nt] * (float)(tb + 4 * q - qpos[nt]);
        if constexpr (!kBiasFirst) {
#pragma unroll
          for (int h = 0; h < kKG; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[h][nt][r] = __builtin_fmaf(slope[nt], (float)(16 * h + r), sc[h][nt][r]);
        }
      }
      if (!full) {
#pragma unroll
        for (int h = 0; h < kKG; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = tb + 16 * h + 4 * q + r;
            sc[h][nt][r] = (key <= qpos[nt] && key >= qleft[nt]) ? sc[h][nt][r] : -INFINITY;
          }
      }
      float t[4 * kKG];
#pragma unroll
      for (int i = 0; i < 4 * kKG; ++i) t[i] = sc[i >> 2][nt][i & 3];
      mx[nt] = tree_max(t);  // log2 units with softcap, raw scores without
      if constexpr (SCORE == kScoreBias) mx[nt] += bias0[nt];
    }
    // The probabilities of both tiles are formed right away against the
    // running maxima, before the cross-lane reduction of the steps' maxima,
    // which only decides afterwards whether a (rare) re-base is due; that
    // recomputes them against the new maximum. Same values as re-basing
    // first. Empty asm uses keep them above the re-base branch, which the
    // compiler would otherwise sink them into, behind the reduction (C4 shapes
    // at head_dim 64: 107.2 -> 105.4 us). One branch serves both tiles, so the
    // common path of a step is one basic block (head_dim 128: 156.3 ->
    // 154.9 us against a branch per tile).
    auto probabilities = [&](int nt, float base) __attribute__((always_inline)) {
      float ps[4 * kKG];
      if constexpr (SCORE == kScoreBias) base = __builtin_fmaf(-bias0[nt], a.score_scale, base);
#pragma unroll
      for (int i = 0; i < 4 * kKG; ++i) {
        if constexpr (LOG2) ps[i] = fast_exp2(sc[i >> 2][nt][i & 3] - base);
        else ps[i] = fast_exp2(__builtin_fmaf(sc[i >> 2][nt][i & 3], a.score_scale, -base));
      }
#pragma unroll
      for (int i = 0; i < 4 * kKG; ++i) pa[i >> 3][nt][i & 7] = (__bf16)ps[i];
      if constexpr (!kMfmaSum) {
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * kKG; ++i) l += ps[i];
        return l;
      }
      return 0.f;
    };
    float lsum[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      lsum[nt] = probabilities(nt, m_base[nt]);
#pragma unroll
      for (int hh = 0; hh < kKH; ++hh) {
        const auto w = __builtin_bit_cast(u32x4_t, pa[hh][nt]);
        asm volatile("" ::"v"(w[0]), "v"(w[1]), "v"(w[2]), "v"(w[3]));
      }
    }
#pragma unroll
    for (int nt = 0; nt + 1 < kNT; nt += 2) col4_max2(mx[nt], mx[nt + 1]);
    if constexpr (kNT % 2) mx[kNT - 1] = col4_max(mx[kNT - 1]);
    bool any = false;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) any = any || (mx[nt] > (LOG2 ? m_run[nt] + kAbove : m_thr[nt]));
    if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        if (!__builtin_amdgcn_ballot_w64(mx[nt] > (LOG2 ? m_run[nt] + kAbove : m_thr[nt]))) continue;
        float top = LOG2 ? mx[nt] : mx[nt] * a.score_scale;
        if constexpr (SHARED) top += kBelow;
        if constexpr (SCORE == kScoreBias) top = base_above(top, bias0[nt] * a.score_scale);
        const float m_new = fmaxf(m_run[nt], top);
        const float alpha = m_run[nt] == -INFINITY ? 0.f : fast_exp2(m_run[nt] - m_new);
        m_run[nt] = m_new;
        m_thr[nt] = (m_new + kAbove) * inv_scale;
        m_base[nt] = m_new == -INFINITY ? 0.f : m_new;
        if constexpr (!kMfmaSum) l_run[nt][0] *= alpha;
        // o rows are qrows 4q + r; qrow h's factor lives in lanes with c16 == h.
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float f = __int_as_float(__builtin_amdgcn_ds_bpermute((4 * q + r) << 2, __float_as_int(alpha)));
#pragma unroll
          for (int c = 0; c < S::NO; ++c) o[nt][c][r] *= f;
          if constexpr (kMfmaSum) l_run[nt][r] *= f;
        }
        lsum[nt] = probabilities(nt, m_base[nt]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
      if constexpr (!kMfmaSum) l_run[nt][0] += lsum[nt];
  };

  static_assert(kStages == 2, "K and V alternate between two stages");
  // The steps' keys ascend; with a distance bias they descend from the rows' own
  // keys, where a positive slope leaves the largest scores: ascending, the
  // maximum would rise by the slope's 64 keys at every step, and every step
  // re-base (eight 512-row chunks on a 2048-token prefix, 32 heads' slopes from
  // 0.84 to 2^-8: 214 us).
  auto step_key = [&](int step) __attribute__((always_inline)) {
    return kb0 + (score_biased(SCORE) ? nsteps - 1 - step : step) * kKeys;
  };
  if constexpr (!kPingPong) {
    // One barrier per step: before it each wave waits for its own loads of
    // the current stage; after it every wave's loads of the stage have landed
    // and every wave has finished the previous step, whose stage is refilled
    // with the next step. The first half's V operands are read before the
    // softmax, their LDS latency behind its arithmetic.
    Entries e_next{};
    {
      const Offsets first = offsets_of(step_key(0), entry_of(step_key(0)));
      issue(first, krs, kv[0][0]);
      issue(first, vrs, kv[0][1]);
    }
    if (1 < nsteps) e_next = entry_of(step_key(1));
    if (__builtin_expect(div_group(wave * kQrowsPerWave) >= nr, 0)) {
      // All rows of this wave lie past the tile's last: it only loads its share
      // and keeps step, and the other wave of its SIMD has the matrix cores and
      // the LDS to itself (256 workgroups of 64 steps, half the waves active:
      // head_dim 128 113.9 -> 82.6 us, with softcap 189.8 -> 120.0; three
      // quarters 116.6 -> 110.6. A branch inside the loop below instead cost full
      // tiles 2%).
      for (int step = 0; step < nsteps; ++step) {
        wait_vmem<0>();
        __syncthreads();
        wait_vmem_visible();
        if (step + 1 < nsteps) {
          const int next = (step + 1) & 1;
          const Offsets of = offsets_of(step_key(step + 1), e_next);
          issue(of, krs, kv[next][0]);
          issue(of, vrs, kv[next][1]);
          if (step + 2 < nsteps) e_next = entry_of(step_key(step + 2));
        }
      }
      return;
    }
    if constexpr (SHARED) load_queries();
    // The loop is unrolled over the two stages, so that every LDS address of a
    // step is a per-lane offset plus an immediate (stage, 16-key group, half):
    // ~44 fewer VALU instructions per wave and step (C4: 148.6 -> 138.0 us).
    // The lambdas are forced inline (with three call sites the compiler made
    // the softmax a real call with a stack frame) and the buffer resources go
    // to the direct-load asm as scalar words (make_rsrc).
    auto body = [&](int step, auto stage) __attribute__((always_inline)) {
      constexpr int cur = decltype(stage)::value, next = cur ^ 1;
      const int tb = step_key(step);
      wait_vmem<0>();
      __syncthreads();
      // Every load of this wave has landed; tell the compiler. Its wait-count
      // model does not see the asm direct loads or waits, so it still counts
      // the query loads before the loop (and, with per-lane entries, the entry
      // loads) as outstanding, and would put an s_waitcnt vmcnt(0) before
      // their first use in the step: after this step's direct loads, which it
      // would then wait for (C4: 185.2 -> 183.9 us).
      wait_vmem_visible();
      if (step + 1 < nsteps) {
        const Offsets of = offsets_of(step_key(step + 1), e_next);
        issue(of, krs, kv[next][0]);
        issue(of, vrs, kv[next][1]);
        if (step + 2 < nsteps) e_next = entry_of(step_key(step + 2));
      }
      scores(kv[cur][0]);
      if constexpr (D <= 128) {
        bf16x8_t vfirst[S::NO];
#pragma unroll
        for (int c = 0; c < S::NO; ++c) vfirst[c] = read_v(kv[cur][1], 0, c);
        softmax(tb);
        accumulate(kv[cur][1], vfirst);
      } else {
        // head_dim 256: half the V operands are read early (32 VGPRs; C4's
        // shapes at head_dim 256, same box: none 162.7-164.2 us, a quarter
        // 160.5-162.8, half 158.2-158.7, all 164.9-166.0).
        constexpr int NF = S::NO / 2;
        bf16x8_t vfirst[NF];
#pragma unroll
        for (int c = 0; c < NF; ++c) vfirst[c] = read_v(kv[cur][1], 0, c);
        softmax(tb);
        accumulate(kv[cur][1], vfirst, NF);
      }
    };
    int step = 0;
    for (; step + 1 < nsteps; step += 2) {
      body(step, std::integral_constant<int, 0>{});
      body(step + 1, std::integral_constant<int, 1>{});
    }
    if (step < nsteps) body(step, std::integral_constant<int, 0>{});
  } else {
    // Two groups of waves, one wave of each on every SIMD (waves w and w + 4
    // share a SIMD), take turns between the matrix cores and the vector ALU.
    // A wave's work per step is an MFMA phase M(i) (scores of step i, then
    // P.V of step i - 1) and a VALU phase S(i) (the softmax of step i), run as
    // M(0) S(0) M(1) S(1) ... M(n) with a barrier after each phase. The
    // second group passes one barrier before its first phase and the first
    // group one after its last, so the second runs every phase one barrier
    // interval later: between two barriers one wave of each SIMD is in an
    // MFMA phase while the other is in a softmax phase.
    //
    // LDS: a wave's iteration i reads K(i) (stage i % 2) and V(i - 1) (stage
    // (i - 1) % 2). At its start each wave issues its share of the direct
    // loads of K(i + 1) and V(i), into the stages that both groups last read
    // in iteration i - 1, and waits for them before the barrier that ends
    // interval 2i + 1 (the first group's second barrier of the iteration, the
    // second group's first), after which the first group reads them.
    const bool lead = wave < kPrefillWaves / 2;
    Entries e_next = entry_of(step_key(0));
    Offsets off_v = offsets_of(step_key(0), e_next);  // offsets of the step whose V is issued next
    issue(off_v, krs, kv[0][0]);
    if (1 < nsteps) e_next = entry_of(step_key(1));
    wait_vmem<0>();
    __syncthreads();
    wait_vmem_visible();  // as in the other loop: the query (and entry) loads have landed
    if (!lead) __syncthreads();
    for (int i = 0; i <= nsteps; ++i) {
      const int tb = step_key(i);
      if (i + 1 < nsteps) {
        const Offsets off_k = offsets_of(step_key(i + 1), e_next);
        issue(off_k, krs, kv[(i + 1) & 1][0]);
        issue(off_v, vrs, kv[i & 1][1]);
        off_v = off_k;
        if (i + 2 < nsteps) e_next = entry_of(step_key(i + 2));
      } else if (i + 1 == nsteps) {
        issue(off_v, vrs, kv[i & 1][1]);
      }
      if (i < nsteps) scores(kv[i & 1][0]);
      if (i > 0) accumulate(kv[(i - 1) & 1][1], nullptr);
      if (!lead) wait_vmem<0>();
      __syncthreads();
      if (i < nsteps) softmax(tb);
      if (lead) wait_vmem<0>();
      __syncthreads();
      wait_vmem_visible();
    }
    if (lead) __syncthreads();
  }

  if constexpr (SHARED) {
    // Unnormalised rows of head_dim floats, (base, sum) pairs beside them.
    const int64_t col0 = (int64_t)kvh * a.part_cols + slot;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int t = wave * kNT + nt;
      if (div_group(16 * t) >= nr) break;
      float* po = a.part_o + (col0 + 16 * t + 4 * q) * D + c16;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < S::NO; ++c) po[r * D + 16 * c] = o[nt][c][r];
      float* ml = a.part_ml + (col0 + 16 * t) * 2;
      if (lane < 16) ml[2 * lane] = m_run[nt];
      if constexpr (kMfmaSum) {
        if (c16 == 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r) ml[2 * (4 * q + r) + 1] = l_run[nt][r];
        }
      } else {
        const float l = col4_sum(l_run[nt][0]);
        if (lane < 16) ml[2 * lane + 1] = l;
      }
    }
    return;
  }
  if (slot >= 0) {
    // A piece: its accumulators, bases and sums as they stand in registers
    // (1 KiB stores; the merge kernel reads them back in the same layout).
    const int64_t pslot = (int64_t)kvh * a.part_slots + slot;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int t = wave * kNT + nt;  // 16-row tile of the workgroup
      if (div_group(16 * t) >= nr) break;
      f32x4_t* po = reinterpret_cast<f32x4_t*>(a.part_o) + ((pslot * (kPrefillWaves * kNT) + t) * S::NO) * 64 + lane;
#pragma unroll
      for (int c = 0; c < S::NO; ++c) po[c * 64] = o[nt][c];
      float* ml = a.part_ml + (pslot * (kPrefillWaves * kNT) + t) * 32;
      if (lane < 16) ml[lane] = m_run[nt];
      if constexpr (kMfmaSum) {
        if (c16 == 0) *reinterpret_cast<f32x4_t*>(ml + 16 + 4 * q) = l_run[nt];
      } else {
        const float l = col4_sum(l_run[nt][0]);
        if (lane < 16) ml[16 + lane] = l;
      }
    }
    return;
  }
  // Normalise into bf16 rows in LDS: o row 4q + r of tile nt, its sum in
  // l_run[nt][r] (MFMA sums) or in lane c16 == 4q + r after the cross-row sum
  // (VALU sums). Then each wave stores its own rows as 16-byte pieces: the
  // wave's LDS operations complete in order, so it reads back what it wrote.
  // (Stored straight from the MFMA layout, a lane's values are 2-byte
  // elements 32 bytes apart: 64 narrow stores per lane.)
  char* rows_lds = lds + kKvBytes + wave * kQrowsPerWave * kOutRowBytes;
#pragma unroll
  for (int nt = 0; nt < kNT; ++nt) {
    float l = 0.f;
    if constexpr (!kMfmaSum) l = col4_sum(l_run[nt][0]);
    // The hardware reciprocal (within one fp32 ulp, far below the bf16
    // rounding that follows) instead of a full division; every row sum is at
    // least 1 (the row's maximum contributes at least 1).
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float lr = kMfmaSum ? l_run[nt][r]
                                : __int_as_float(__builtin_amdgcn_ds_bpermute((4 * q + r) << 2, __float_as_int(l)));
      const float inv = lr > 0.f ? __builtin_amdgcn_rcpf(lr) : 0.f;
      __bf16* dst = reinterpret_cast<__bf16*>(rows_lds + (nt * 16 + 4 * q + r) * kOutRowBytes) + c16;
#pragma unroll
      for (int c = 0; c < S::NO; ++c) dst[16 * c] = (__bf16)(o[nt][c][r] * inv);
    }
  }
  constexpr int kPieces = kQrowsPerWave * D / 8;  // 16-byte pieces of the wave's rows
  static_assert(kPieces % 64 == 0, "whole pieces per lane");
#pragma unroll
  for (int i = 0; i < kPieces / 64; ++i) {
    const int piece = i * 64 + lane, ql = piece / (D / 8), part = piece % (D / 8);
    const int qr = wave * kQrowsPerWave + ql;
    const int row = div_group(qr), head = qr - row * g;
    const uint4 v = *reinterpret_cast<const uint4*>(rows_lds + ql * kOutRowBytes + part * 16);
    if (row < nr)
      *reinterpret_cast<uint4*>(a.out + (int64_t)(first_row + row) * a.out_stride + (int64_t)(kvh * g + head) * D +
                                part * 8) = v;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Checks of gk_prefill_params for the entry point `name`; `listed`: its sequence arrays are not read.
inline int check_prefill(const gk_prefill_params* p, bool listed, const char* name) {
  const auto bad = [&](int code, const char* what) { return fail(code, std::string(name) + ": " + what); };
  if (!p) return bad(GK_ERR_INVALID_ARGUMENT, "null parameters");
  if (p->struct_size != sizeof(gk_prefill_params))
    return bad(GK_ERR_INVALID_ARGUMENT, "struct_size does not match this library's gk_prefill_params");
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return bad(GK_ERR_UNSUPPORTED, "head dimension must be 64, 128 or 256");
  if (p->q_heads <= 0 || p->kv_heads <= 0 || p->q_heads % p->kv_heads || p->q_heads / p->kv_heads > 128)
    return bad(GK_ERR_INVALID_ARGUMENT, "invalid head geometry (GQA group at most 128)");
  if (!is_pow2(p->block_size) || p->block_size > (1 << 20))
    return bad(GK_ERR_UNSUPPORTED, "block_size must be a power of two of at most 2^20");
  if (p->seqs < 0 || p->seqs > 65535 || p->max_rows < 0 || p->slots <= 0)
    return bad(GK_ERR_INVALID_ARGUMENT, "sequence count, rows or slots out of range");
  if (p->slots > (int64_t)(UINT32_MAX / 2) / p->head_dim)
    return bad(GK_ERR_UNSUPPORTED, "one kv head's K or V region must stay below 4 GiB");
  if (!(p->scale > 0.f) || !(p->scale < INFINITY) || !(p->softcap >= 0.f) || !(p->softcap < INFINITY))
    return bad(GK_ERR_INVALID_ARGUMENT, "invalid scale or softcap");
  if (!listed && (p->seqs == 0 || p->max_rows == 0)) return GK_OK;
  if (!p->query || !p->pool || !p->block_tables || !p->out ||
      (!listed && (!p->seq_request || !p->seq_first_row || !p->seq_rows || !p->seq_prefix)))
    return bad(GK_ERR_INVALID_ARGUMENT, "null pointer");
  const auto misaligned = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) != 0; };
  if (misaligned(p->query) || misaligned(p->pool) || misaligned(p->out) || (p->q_row_stride & 7) ||
      (p->out_row_stride & 7) || p->q_row_stride < (int64_t)p->q_heads * p->head_dim ||
      p->out_row_stride < (int64_t)p->q_heads * p->head_dim)
    return bad(GK_ERR_INVALID_ARGUMENT, "query/pool/out must be 16-byte aligned with full rows");
  return GK_OK;
}

// The arguments that do not depend on where the work comes from.
inline PrefillArgs prefill_args(const gk_prefill_params* p) {
  PrefillArgs a{};
  a.query = static_cast<const uint16_t*>(p->query);
  a.q_stride = p->q_row_stride;
  a.pool = static_cast<const uint16_t*>(p->pool);
  a.slots = p->slots;
  a.block_tables = p->block_tables;
  a.bt_stride = p->bt_stride;
  a.block_shift = log2_int(p->block_size);
  a.q_heads = p->q_heads;
  a.kv_heads = p->kv_heads;
  a.group = p->q_heads / p->kv_heads;
  a.rows_per_tile = prefill_tile_qrows(p->head_dim) / a.group;
  const bool softcap = p->softcap > 0.f;
  a.score_scale = softcap ? p->scale / p->softcap : p->scale * kLog2e;
  a.softcap_log2 = p->softcap * kLog2e;
  a.window = p->sliding_window > 0 ? p->sliding_window : 0;
  a.out = static_cast<uint16_t*>(p->out);
  a.out_stride = p->out_row_stride;
  a.group_div = div_magic((uint32_t)a.group);
  return a;
}

}  // namespace
}  // namespace gk

// One-wave workers of a shared-prefix launch: a list of segments, each up to 32
// (row, head) columns over a stretch of keys, a partial per segment.
//
// Per-tile arithmetic is the short-context decode kernel's: S^T = K . Q^T on
// 16 x 16 MFMA tiles, a re-base at every new running maximum, probabilities
// rounded to bf16 (relative to that maximum, as in every kernel of this
// library), P . V from a transposed LDS read, sums and accumulators in fp32. A
// second 16-column tile, where a segment has one, uses the same K and V
// registers. A wave keeps one stage: the next K tile is issued once this one is
// in registers, the next V tile after P . V, so that a tile's bytes are in
// flight at almost any time, and the eight waves of a CU cover each other's
// waits (2048 waves keep 32 MiB in flight; HBM at its rate needs a third).
//
// A tile's block-table entries come to LDS with a direct load of their own, one
// a key, two tiles ahead: the vector load counter then orders everything, and
// one code path serves every page size.
#pragma once

#include "decode_common.hpp"
#include "prefill_kernel.hpp"

namespace gk {
namespace {

// lds_dma16_w for rows that one worker reads once (GK_KV_LOAD_POLICY).
__device__ __forceinline__ void lds_dma16_once_w(uint32_t lds, u32x4_t rsrc, uint32_t voffset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen " GK_KV_LOAD_POLICY " lds" ::"s"(lds),
      "v"(voffset), "s"(rsrc)
      : "memory");
}

// 4 bytes per lane, HBM -> LDS (lds_dma16_w's narrow form; the s_nop also
// covers a resource word that a readfirstlane has just made).
__device__ __forceinline__ void lds_dma4_w(uint32_t lds, u32x4_t rsrc, uint32_t voffset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 4\n\t"
      "buffer_load_dword %1, %2, 0 offen lds" ::"s"(lds),
      "v"(voffset), "s"(rsrc)
      : "memory");
}

// A segment's record (SharedSegment) in scalar registers.
struct SegmentWords {
  int first, ncols, tile0, ntiles, key_lo, key_hi, col, batch_row, pos, new_pos, new_row, request;
};
__device__ __forceinline__ SegmentWords load_segment(const int32_t* rec) {
  return {scalar_load(rec, 0), scalar_load(rec, 1), scalar_load(rec, 2), scalar_load(rec, 3), scalar_load(rec, 4),
          scalar_load(rec, 5), scalar_load(rec, 6), scalar_load(rec, 7), scalar_load(rec, 8), scalar_load(rec, 9),
          scalar_load(rec, 10), scalar_load(rec, 11)};
}

// NT: 16-column tiles of the segment. `meanwhile` runs once its first loads are on their way.
template <int D, int SCORE, int NT, class Meanwhile>
__device__ __forceinline__ void shared_segment(const SharedArgs& a, char* kt, int32_t* entries, int kvh,
                                               const SegmentWords& seg, const int32_t* bt, Meanwhile meanwhile) {
  const int ncols = seg.ncols, tile0 = seg.tile0, ntiles = seg.ntiles, key_lo = seg.key_lo, key_hi = seg.key_hi;
  using S = MfmaShape<D>;
  constexpr bool LOG2 = SCORE != kScorePlain;
  constexpr int TS = S::TS, LOADS = S::LOADS, CPR = S::CPR;
  static_assert(TS == shared_tile_keys(D) && 16 * NT <= shared_columns(D), "the plan's tiles are the worker's");
  const int lane = threadIdx.x & 63, q = lane >> 4, c16 = lane & 15;
  const int g = a.group, shift = a.block_shift, bmask = (1 << shift) - 1;
  char* const vt = kt + S::TILE;
  const int tile_end = tile0 + ntiles;
  const int key_begin = max(key_lo, tile0 * TS), key_end = min(key_hi, tile_end * TS);

  // Entry of lane's key of tile t (lanes past the tile repeat its last key), keys outside
  // [key_begin, key_end) the nearest one's.
  const u32x4_t ers = buffer_words(bt, (uint32_t)min((int64_t)UINT32_MAX, a.bt_stride * 4));
  auto issue_entries = [&](int t) __attribute__((always_inline)) {
    const int key = min(max(t * TS + min(lane, TS - 1), key_begin), key_end - 1);
    lds_dma4_w(lds_addr(entries + (t & 1) * kWorkerEntries), ers, (uint32_t)(key >> shift) * 4u);
  };
  issue_entries(tile0);
  issue_entries(tile0 + 1);

  // The columns' rows: positions, windows and queries.
  int qpos[NT], qleft[NT];
  bf16x8_t qb[NT][S::NC];
  int low = INT32_MAX, left = 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int j = nt * 16 + c16;
    const bool valid = j < ncols;
    const int row = (int)fast_div((uint32_t)min(j, ncols - 1), a.group_div), head = min(j, ncols - 1) - row * g;
    int batch_row = seg.batch_row + row, pos = seg.pos + row;
    if (seg.pos < 0) {
      batch_row = a.row_map[seg.first + row];
      pos = a.row_position[seg.first + row];
    }
    qpos[nt] = min(pos, key_end - 1);
    qleft[nt] = a.window > 0 ? max(key_begin, pos - a.window + 1) : key_begin;
    low = min(low, qpos[nt]);
    left = max(left, qleft[nt]);
    const uint16_t* src = a.query + (int64_t)batch_row * a.q_stride + (int64_t)(kvh * g + head) * D;
#pragma unroll
    for (int c = 0; c < S::NC; ++c) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (valid) v = load16(src + (4 * c + q) * 8);
      qb[nt][c] = __builtin_bit_cast(bf16x8_t, v);
    }
  }
  const int pos_min = columns_min(low), left_max = -columns_min(-left);

  // New tokens among the segment's keys: their rows come from the caller's
  // tensors, not from the pool, where this wave stores them. Lanes 0 .. 2 CPR - 1
  // (and again the lanes after them) hold the pieces of a token's key and value;
  // those of the first new token are fetched ahead.
  const int new_lo = max(key_begin, a.new_key ? seg.new_pos : INT32_MAX);
  const bool key_lane = (lane & (2 * CPR - 1)) < CPR;
  const int chunk = lane & (CPR - 1);
  auto new_piece = [&](int key) __attribute__((always_inline)) {
    const uint16_t* src = key_lane ? a.new_key : a.new_value;
    return *reinterpret_cast<const u32x4_t*>(src + (int64_t)(seg.new_row + (key - seg.new_pos)) * a.new_stride +
                                             (int64_t)kvh * D + chunk * 8);
  };
  u32x4_t ahead{0u, 0u, 0u, 0u};
  if (new_lo < key_end) ahead = new_piece(new_lo);

  const uint32_t region = (uint32_t)(a.slots * D * 2);
  const uint16_t* kbase = a.pool + (int64_t)kvh * a.slots * D;
  const u32x4_t krs = buffer_words(kbase, region), vrs = buffer_words(kbase + (int64_t)a.kv_heads * a.slots * D, region);
  struct Offsets {
    uint32_t v[LOADS];
  };
  // Byte offsets of this lane's pieces of tile t, whose entries are in LDS.
  auto offsets_of = [&](int t) __attribute__((always_inline)) {
    Offsets of;
    const int32_t* e = entries + (t & 1) * kWorkerEntries;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int s = i * 64 + lane, tt = s / CPR, pc = s % CPR;
      const int key = min(max(t * TS + tt, key_begin), key_end - 1);
      const uint32_t slot = ((uint32_t)e[tt] << shift) | (uint32_t)(key & bmask);
      of.v[i] = slot * (uint32_t)(2 * D) + ((pc ^ swz(tt, D / 8)) << 4);
    }
    return of;
  };
  auto issue = [&](const Offsets& of, u32x4_t rs, char* tile) __attribute__((always_inline)) {
    const uint32_t base = lds_addr(tile);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) lds_dma16_once_w(base + i * 1024, rs, of.v[i]);
  };

  f32x4_t o[NT][S::NO];
  float m_run[NT], l_run[NT], m_thr[NT], m_base[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < S::NO; ++c) o[nt][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m_run[nt] = m_thr[nt] = -INFINITY;
    l_run[nt] = m_base[nt] = 0.f;
  }
  const float inv_scale = 1.f / a.score_scale;

  // Everything so far has landed, the entries among it; the compiler's wait
  // counts do not see the direct loads below.
  wait_vmem<0>();
  wait_vmem_visible();
  Offsets next = offsets_of(tile0);
  issue(next, krs, kt);
  issue(next, vrs, vt);
  meanwhile();
  for (int t = tile0; t < tile_end; ++t) {
    const int tb = t * TS;
    const bool more = t + 1 < tile_end;
    // In flight: (entries of t + 1,) K, V of t, in this order.
    if (tb + TS > new_lo && new_lo < key_end) {
      wait_vmem<0>();
      for (int key = max(tb, new_lo); key < min(tb + TS, key_end); ++key) {
        u32x4_t v = ahead;
        if (key != new_lo) v = new_piece(key);
        const int tt = key - tb;
        *reinterpret_cast<u32x4_t*>(kt + (key_lane ? 0 : S::TILE) + tt * (2 * D) + ((chunk ^ swz(tt, D / 8)) << 4)) = v;
        const int32_t entry = entries[(t & 1) * kWorkerEntries + tt];
        const int64_t slot = ((int64_t)entry << shift) | (key & bmask);
        if (entry >= 0 && slot < a.slots && lane < 2 * CPR)
          __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(
                                             a.pool_out + ((int64_t)(key_lane ? kvh : a.kv_heads + kvh) * a.slots + slot) * D + chunk * 8));
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else {
      wait_vmem<LOADS>();
    }
    bf16x8_t kr[S::TG][S::NC];
#pragma unroll
    for (int h = 0; h < S::TG; ++h) {
      const int tt = 16 * h + c16;
#pragma unroll
      for (int c = 0; c < S::NC; ++c)
        kr[h][c] = *reinterpret_cast<const bf16x8_t*>(kt + tt * (2 * D) + (((4 * c + q) ^ swz(tt, D / 8)) << 4));
    }
    if (more) next = offsets_of(t + 1);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) {
      issue_entries(t + 2);
      issue(next, krs, kt);
    }
    f32x4_t sc[NT][S::TG];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < S::TG; ++h) {
        sc[nt][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < S::NC; ++c) sc[nt][h] = mfma32(kr[h][c], qb[nt][c], sc[nt][h]);
      }
    if constexpr (!LOG2) {
      if constexpr (NT == 1) mfma_results_ready(sc[0]);
      else mfma_results_ready(sc);
    }
    const bool full = tb >= left_max && tb + TS - 1 <= pos_min;
    float mx[NT];
    bool any = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (LOG2 || !full) {
#pragma unroll
        for (int h = 0; h < S::TG; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float s = sc[nt][h][r];
            if constexpr (SCORE == kScoreCap) s = soft_cap(s * a.score_scale, a.softcap_log2);
            const int key = tb + 16 * h + 4 * q + r;
            sc[nt][h][r] = (key >= qleft[nt] && key <= qpos[nt]) ? s : -INFINITY;
          }
      }
      float v[4 * S::TG];
#pragma unroll
      for (int i = 0; i < 4 * S::TG; ++i) v[i] = sc[nt][i >> 2][i & 3];
      mx[nt] = tree_max(v);
    }
    if constexpr (NT == 2) {
      // The swaps read the asm maxima two slots after them at the earliest (tests/test_shared_asm_waits.py).
      asm volatile("s_nop 1" : "+v"(mx[0]), "+v"(mx[1]));
      col4_max2(mx[0], mx[1]);
    } else {
      asm volatile("s_nop 1" : "+v"(mx[0]));
      mx[0] = col4_max(mx[0]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) any = any || mx[nt] > (LOG2 ? m_run[nt] + kDecodeRescaleSlack : m_thr[nt]);
    if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m_new = fmaxf(m_run[nt], LOG2 ? mx[nt] : mx[nt] * a.score_scale);
        const float alpha = m_run[nt] == -INFINITY ? 0.f : fast_exp2(m_run[nt] - m_new);
        l_run[nt] *= alpha;
        m_run[nt] = m_new;
        m_thr[nt] = (m_new + kDecodeRescaleSlack) * inv_scale;
        m_base[nt] = m_new == -INFINITY ? 0.f : m_new;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float f = __int_as_float(__builtin_amdgcn_ds_bpermute((4 * q + r) << 2, __float_as_int(alpha)));
#pragma unroll
          for (int c = 0; c < S::NO; ++c) o[nt][c][r] *= f;
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < S::TG; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = LOG2 ? fast_exp2(sc[nt][h][r] - m_base[nt])
                               : fast_exp2(__builtin_fmaf(sc[nt][h][r], a.score_scale, -m_base[nt]));
          sc[nt][h][r] = p;
          l_run[nt] += p;
        }

    // In flight: V of t, entries of t + 2, K of t + 1.
    if (more) wait_vmem<LOADS + 1>();
    else wait_vmem<0>();
    if (tb < key_begin || tb + TS > key_end) {
      // A masked key weighs zero, but its row may hold an infinity.
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int s = i * 64 + lane, key = tb + s / CPR;
        if (key < key_begin || key >= key_end) *reinterpret_cast<uint4*>(vt + s * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (TS == 32) {
      bf16x8_t pa[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          pa[nt][r] = (__bf16)sc[nt][0][r];
          pa[nt][4 + r] = (__bf16)sc[nt][S::TG - 1][r];
        }
#pragma unroll
      for (int c = 0; c < S::NO; ++c) {
        const int lc = 2 * c + ((c16 & 3) >> 1);
        const int t0 = 4 * q + (c16 >> 2), t1 = t0 + 16;
        const bf16x4_t v0 = lds_read_tr4(vt + t0 * (2 * D) + ((lc ^ swz(t0, D / 8)) << 4) + ((c16 & 1) << 3));
        const bf16x4_t v1 = lds_read_tr4(vt + t1 * (2 * D) + ((lc ^ swz(t1, D / 8)) << 4) + ((c16 & 1) << 3));
        const bf16x8_t v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][c] = mfma32(pa[nt], v, o[nt][c]);
      }
    } else {
      bf16x4_t pa[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) pa[nt][r] = (__bf16)sc[nt][0][r];
#pragma unroll
      for (int c = 0; c < S::NO; ++c) {
        const int lc = 2 * c + ((c16 & 3) >> 1);
        const int t0 = 4 * q + (c16 >> 2);
        const bf16x4_t v = lds_read_tr4(vt + t0 * (2 * D) + ((lc ^ swz(t0, D / 8)) << 4) + ((c16 & 1) << 3));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][c] = mfma16(pa[nt], v, o[nt][c]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) issue(next, vrs, vt);
  }

  // The partial: unnormalised rows of head_dim floats, (base, sum) beside them.
  const int64_t col0 = (int64_t)kvh * a.part_cols + seg.col;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float l = col4_sum(l_run[nt]);
    if (lane < 16 && 16 * nt + lane < ncols) {
      float* ml = a.part_ml + (col0 + 16 * nt + lane) * 2;
      ml[0] = m_run[nt];
      ml[1] = l;
    }
    float* po = a.part_o + (col0 + 16 * nt + 4 * q) * D + c16;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (16 * nt + 4 * q + r < ncols) {
#pragma unroll
        for (int c = 0; c < S::NO; ++c) po[r * D + 16 * c] = o[nt][c][r];
      }
  }
}

template <int D, int SCORE>
__device__ __forceinline__ void shared_worker(const SharedArgs& a, char* lds, int kvh, int worker) {
  using S = MfmaShape<D>;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  char* kt = lds + wave * (2 * S::TILE);
  int32_t* entries = reinterpret_cast<int32_t*>(lds + kSharedWaves * 2 * S::TILE) + wave * 2 * kWorkerEntries;
  // The next segment's record, and the request behind it, come while a segment runs.
  const int32_t* rec = a.worker_list + (int64_t)worker * kSharedWorkerWords;
  SegmentWords seg = load_segment(rec), next;
  int at = scalar_load(rec, kSharedSegmentWords), next_request = 0;
  const auto request_of = [&](const SegmentWords& s) {
    return s.request >= 0 ? s.request : scalar_load(a.row_request, s.batch_row);
  };
  int request = request_of(seg);
  const int end = scalar_load(rec, kSharedSegmentWords + 1);
  for (;;) {
    const bool more = at < end;
    next = more ? load_segment(a.segs + (int64_t)at * kSharedSegmentWords) : seg;
    const auto meanwhile = [&] { next_request = request_of(next); };
    const int32_t* bt = a.block_tables + (int64_t)request * a.bt_stride;
    if (shared_columns(D) == 16 || seg.ncols <= 16)
      shared_segment<D, SCORE, 1>(a, kt, entries, kvh, seg, bt, meanwhile);
    else
      shared_segment<D, SCORE, shared_columns(D) / 16>(a, kt, entries, kvh, seg, bt, meanwhile);
    if (!more) return;
    seg = next;
    request = next_request;
    ++at;
  }
}

}  // namespace
}  // namespace gk

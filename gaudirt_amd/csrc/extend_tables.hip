// Block tables, token map and slots of a scheduler step, made on the GPU from
// the sequences' lengths.
//
// Sequence s holds prefix_s tokens and gets length_s more. With page size P it
// needs n_s = ceil((prefix_s + length_s) / P) - ceil(prefix_s / P) new pages,
// which come from the free list in batch order: the exclusive sum of the n is
// where a sequence's pages start, the exclusive sum of the lengths where its
// rows do. A sequence with a parent starts from the parent's first prefix_s
// tokens (whole pages): its entries are copies of the parent's, and a third
// sum, of those tokens, numbers the copies.
//
// One launch. Every workgroup makes the three sums for itself, in LDS (a few
// bytes a sequence from L2 and one scan), so nothing waits for another workgroup;
// then all threads share the rows, pages and copied tokens, whose sequence a
// binary search finds. What bounds a decode step is the launch and that chain of
// round trips; the code is kept small for it (rows four at a time, with 64-bit
// indexes, were slower: most of such a call is the code's own way into the
// instruction caches). Kernel and whole call (us): 256 sequences of one new token
// 5.3 / 6.7; 64 children of an 8192-token parent 7.3 a call; 48 prompts of up to
// 32000 tokens, 13 MB written, 10.5 / 10.1, the write at copy rate being 2.7.
#include "gk_common.hpp"

#include <algorithm>

namespace gk {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kSmallBatch = 1024;
constexpr int kMaxBatch = GK_EXTEND_MAX_BATCH;

struct ExtendArgs {
  int32_t* tables;
  int32_t* mapping;  // or null
  int32_t requests, pages, context;
  const void* seq_requests;
  const void* prefixes;
  const void* lengths;
  const void* parents;  // or null; the type of seq_requests
  const void* free_pages;
  const int32_t* free_head;
  int32_t requests64, lengths64, pages64;
  int64_t free_count;
  int32_t batch, shift, max_rows;
  int64_t slots;
  int32_t* out_locations;
  int32_t* out_requests;
  int32_t* out_positions;
  void* out_lengths;
  int32_t* counts;
};

// Element i of an int32 or int64 vector, without a branch on the type (a load
// whose value a branch converts is waited for there, one after the other).
__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  const int32_t* w = static_cast<const int32_t*>(p) + (i << is64);
  const int32_t low = w[0], high = w[is64];
  return is64 ? (int64_t)((uint64_t)(uint32_t)high << 32 | (uint32_t)low) : (int64_t)low;
}

// Sums that end at INT32_MAX instead of passing it: a batch whose sum gets there is refused.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, (uint32_t)INT32_MAX); }

struct Sums {
  uint32_t rows, pages, copies;
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
  return {add_sat(a.rows, b.rows), add_sat(a.pages, b.pages), add_sat(a.copies, b.copies)};
}
// The sum of the lanes up to this one, with DPP shifts (a source outside the row reads 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ Sums shifted(const Sums& a) {
  const auto move = [](uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, ROWS == 0xf);
  };
  return {move(a.rows), move(a.pages), move(a.copies)};
}
__device__ __forceinline__ Sums wave_inclusive(Sums x) {
  x = x + shifted<0x111, 0xf>(x);  // row_shr:1
  x = x + shifted<0x112, 0xf>(x);  // row_shr:2
  x = x + shifted<0x114, 0xf>(x);  // row_shr:4
  x = x + shifted<0x118, 0xf>(x);  // row_shr:8
  x = x + shifted<0x142, 0xa>(x);  // row_bcast:15, rows 1 and 3
  x = x + shifted<0x143, 0xc>(x);  // row_bcast:31, rows 2 and 3
  return x;
}

// The last s < n with first[s] <= x (first[0] = 0 <= x < first[n]): the sequence that owns x, empty ones passed over.
// `top`: the largest power of two below n, or 0.
__device__ __forceinline__ int owner(const int32_t* first, int n, int top, int x) {
  int s = 0;
  for (int step = top; step; step >>= 1) {
    const int mid = s + step;
    s = mid < n && first[mid] <= x ? mid : s;
  }
  return s;
}

template <int MAX>
__global__ __launch_bounds__(kThreads) void extend_tables_kernel(ExtendArgs a) {
  // A sequence's table row, its parent's and the page that its first new token may continue as well, where the LDS has
  // room for them (8192 sequences leave them in memory): known before the sums are.
  constexpr bool kInLds = MAX <= kSmallBatch;
  constexpr int kExtra = kInLds ? MAX : 1;
  __shared__ int32_t s_row[MAX + 1], s_page[MAX + 1], s_copy[MAX + 1], s_prefix[MAX];
  __shared__ int32_t s_request[kExtra], s_parent[kExtra], s_last[kExtra];
  __shared__ Sums s_wave[kWaves];
  __shared__ uint32_t s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1 << a.shift;
  // Table and map elements, tokens of a row and slots stay below 2^31 (checked on the host or below): 32-bit indexes.
  const auto pages_of = [&](int tokens) { return (int)(((uint32_t)tokens + (uint32_t)(P - 1)) >> a.shift); };
  const int head = a.free_head ? *a.free_head : 0;
  const int copy_shift = a.mapping ? 0 : a.shift;  // copies are numbered by token with a map, else by page
  if (tid == 0) s_bad = UINT32_MAX;
  __syncthreads();

  // A thread's sequences, their sums and the first one that cannot be right:
  // (index << 3 | code), the smallest over the batch.
  constexpr int kPer = MAX / kThreads;  // sequences of a thread
  const int s0 = tid * kPer;
  uint32_t bad = UINT32_MAX;
  Sums mine{0, 0, 0};
  [[maybe_unused]] int32_t last[kInLds ? kPer : 1];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int s = s0 + u;
    if (s >= a.batch) break;
    const int64_t request = load_index(a.seq_requests, a.requests64, s), prefix = load_index(a.prefixes, a.lengths64, s),
                  length = load_index(a.lengths, a.lengths64, s),
                  parent = a.parents ? load_index(a.parents, a.requests64, s) : -1;
    const int64_t room = min((int64_t)a.pages << a.shift, (int64_t)(a.mapping ? a.context : INT32_MAX));
    int code = 0;
    if (request < 0 || request >= a.requests || parent >= a.requests) code = 1;
    else if (prefix < 0 || length < 0 || prefix > room || length > room - prefix) code = 2;
    else if (parent >= 0 && ((prefix & (P - 1)) || parent == request)) code = 3;
    if (code) {
      bad = min(bad, (uint32_t)s << 3 | (uint32_t)code);
    } else {
      mine = mine + Sums{(uint32_t)length, (uint32_t)(pages_of((int)(prefix + length)) - pages_of((int)prefix)),
                         parent >= 0 ? (uint32_t)prefix >> copy_shift : 0u};
    }
    if constexpr (kInLds) {
      s_request[s] = (int32_t)(code ? 0 : request);
      s_parent[s] = (int32_t)(code ? -1 : parent);
      last[u] = !code && (prefix & (P - 1)) ? a.tables[(int)request * a.pages + ((int)prefix >> a.shift)] : -1;
    }
    s_prefix[s] = (int32_t)(code ? 0 : prefix);
    s_row[s] = code ? 0 : (int32_t)length;  // kept for the second pass
    s_copy[s] = !code && parent >= 0;
  }
  const Sums scan = wave_inclusive(mine);
  if (lane == 63) s_wave[wave] = scan;
  __syncthreads();
  Sums at{0, 0, 0}, total{0, 0, 0};
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at = at + s_wave[w];
    total = total + s_wave[w];
  }
  const Sums below{(uint32_t)__shfl_up((int)scan.rows, 1), (uint32_t)__shfl_up((int)scan.pages, 1),
                   (uint32_t)__shfl_up((int)scan.copies, 1)};
  if (lane) at = at + below;
  const int64_t free_left = head >= 0 && head <= a.free_count ? a.free_count - head : 0;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int s = s0 + u;
    if (s >= a.batch) break;
    const int length = s_row[s], prefix = s_prefix[s];
    if constexpr (kInLds) s_last[s] = last[u];
    const Sums one{(uint32_t)length, (uint32_t)(pages_of(prefix + length) - pages_of(prefix)),
                   s_copy[s] ? (uint32_t)prefix >> copy_shift : 0u};
    s_row[s] = (int32_t)at.rows;
    s_page[s] = (int32_t)at.pages;
    s_copy[s] = (int32_t)at.copies;
    at = at + one;
    if (at.rows > (uint32_t)a.max_rows) bad = min(bad, (uint32_t)s << 3 | 4u);
    else if ((int64_t)at.pages > free_left) bad = min(bad, (uint32_t)s << 3 | 5u);
  }
  if (tid == 0) {
    s_row[a.batch] = (int32_t)total.rows;
    s_page[a.batch] = (int32_t)total.pages;
    s_copy[a.batch] = (int32_t)total.copies;
  }
  if (bad != UINT32_MAX) atomicMin(&s_bad, bad);
  __syncthreads();
  const uint32_t first_bad = s_bad;
  const bool ok = first_bad == UINT32_MAX;
  const int rows = ok ? s_row[a.batch] : 0, pages = ok ? s_page[a.batch] : 0;
  const int copies = ok ? s_copy[a.batch] : 0;
  if (blockIdx.x == 0) {
    for (int s = tid; s < a.batch; s += kThreads) {
      const int64_t was = load_index(a.prefixes, a.lengths64, s);
      const int64_t now = ok ? (int64_t)s_prefix[s] + (s_row[s + 1] - s_row[s]) : was;
      if (a.lengths64) static_cast<int64_t*>(a.out_lengths)[s] = now;
      else static_cast<int32_t*>(a.out_lengths)[s] = (int32_t)now;
    }
    if (tid == 0) {
      a.counts[0] = rows;
      a.counts[1] = head + pages;
      a.counts[2] = ok ? 0 : (int32_t)(first_bad & 7u);
      a.counts[3] = ok ? -1 : (int32_t)(first_bad >> 3);
    }
  }
  const auto request_of = [&](int s) {
    if constexpr (kInLds) return s_request[s];
    else return (int32_t)load_index(a.seq_requests, a.requests64, s);
  };
  const auto parent_of = [&](int s) {
    if constexpr (kInLds) return s_parent[s];
    else return (int32_t)load_index(a.parents, a.requests64, s);
  };
  // A page of the free list, -1 where it lies outside the pool.
  const auto page_at = [&](int i) {
    const int64_t page = load_index(a.free_pages, a.pages64, (int64_t)head + i);
    return page >= 0 && page < (a.slots >> a.shift) ? (int32_t)page : -1;
  };
  const int threads = gridDim.x * kThreads, thread = blockIdx.x * kThreads + tid;
  const int top = a.batch > 1 ? 1 << (31 - __builtin_clz(a.batch - 1)) : 0;

  // Rows: slot, request and position of every new token; rows behind the last are no tokens.
  for (int row = thread; row < a.max_rows; row += threads) {
    int32_t slot = -1, request = 0, position = 0;
    if (row < rows) {
      const int s = owner(s_row, a.batch, top, row), prefix = s_prefix[s], held = pages_of(prefix);
      request = request_of(s);
      position = prefix + (row - s_row[s]);
      const int entry = position >> a.shift;
      int32_t page;
      if (entry >= held) page = page_at(s_page[s] + entry - held);
      else if constexpr (kInLds) page = s_last[s];  // the one page that cached tokens share with new ones
      else page = a.tables[request * a.pages + entry];
      if (page >= 0 && page < a.slots >> a.shift) slot = (page << a.shift) + (position & (P - 1));
      if (a.mapping) a.mapping[request * a.context + position] = slot;
    }
    a.out_locations[row] = slot;
    a.out_requests[row] = request;
    a.out_positions[row] = position;
  }
  // New pages into the tables, from the last workgroup on: the first ones have the rows.
  for (int i = threads - 1 - thread; i < pages; i += threads) {
    const int s = owner(s_page, a.batch, top, i);
    a.tables[request_of(s) * a.pages + pages_of(s_prefix[s]) + (i - s_page[s])] = page_at(i);
  }
  // The parents' tokens and pages into their children's rows, by the workgroups without rows where there are others.
  const int busy = min((rows + kThreads - 1) / kThreads, (int)gridDim.x / 2);
  if ((int)blockIdx.x < busy) return;
  const int copiers = threads - busy * kThreads;
  for (int64_t i = thread - busy * kThreads; i < copies; i += copiers) {
    const int s = owner(s_copy, a.batch, top, (int)i), t = ((int)i - s_copy[s]) << copy_shift;
    const int request = request_of(s), parent = parent_of(s);
    if (a.mapping) a.mapping[request * a.context + t] = a.mapping[parent * a.context + t];
    if (!(t & (P - 1))) a.tables[request * a.pages + (t >> a.shift)] = a.tables[parent * a.pages + (t >> a.shift)];
  }
}

}  // namespace

int extend_block_tables(const gk_extend_params* p, hipStream_t stream) {
  const char* const name = "gk_extend_block_tables: ";
  const auto bad = [&](const char* what) { return fail(GK_ERR_INVALID_ARGUMENT, std::string(name) + what); };
  if (!p) return bad("null parameters");
  if (p->struct_size != sizeof(gk_extend_params)) return bad("struct_size does not match this library's gk_extend_params");
  if (p->batch < 0 || p->batch > kMaxBatch) return bad("at most 8192 sequences");
  if (p->requests <= 0 || p->pages <= 0 || (int64_t)p->requests * p->pages > INT32_MAX) return bad("invalid table size");
  if (p->mapping && (p->context <= 0 || (int64_t)p->requests * p->context > INT32_MAX)) return bad("invalid map size");
  if (!is_pow2(p->page_size) || p->page_size > (1 << 20)) return bad("page_size must be a power of two of at most 2^20");
  if (p->slots <= 0 || p->slots > INT32_MAX || p->free_count < 0 || p->free_count > INT32_MAX || p->max_rows < 0 ||
      p->max_rows > (1 << 30))
    return bad("slots, free pages or rows out of range");
  if (!p->block_tables || !p->counts || (p->batch && (!p->seq_requests || !p->prefixes || !p->lengths || !p->out_lengths)) ||
      (p->free_count && !p->free_pages) ||
      (p->max_rows && (!p->out_locations || !p->out_requests || !p->out_positions)))
    return bad("null pointer");
  // Workgroups read these inputs while others write the outputs.
  const auto overlap = [](const void* in, int64_t in_bytes, const void* out, int64_t out_bytes) {
    const uintptr_t i = reinterpret_cast<uintptr_t>(in), o = reinterpret_cast<uintptr_t>(out);
    return in && i < o + (uint64_t)out_bytes && o < i + (uint64_t)in_bytes;
  };
  const int64_t length_bytes = (p->lengths_int64 ? int64_t{8} : int64_t{4}) * p->batch;
  if (overlap(p->free_head, 4, p->counts, 16) || overlap(p->prefixes, length_bytes, p->out_lengths, length_bytes) ||
      overlap(p->lengths, length_bytes, p->out_lengths, length_bytes))
    return bad("counts overlap free_head, or out_lengths the lengths");
  ExtendArgs a{};
  a.tables = p->block_tables;
  a.mapping = p->mapping;
  a.requests = p->requests;
  a.pages = p->pages;
  a.context = p->context;
  a.seq_requests = p->seq_requests;
  a.prefixes = p->prefixes;
  a.lengths = p->lengths;
  a.parents = p->parents;
  a.free_pages = p->free_pages;
  a.free_head = p->free_head;
  a.requests64 = p->requests_int64;
  a.lengths64 = p->lengths_int64;
  a.pages64 = p->pages_int64;
  a.free_count = p->free_count;
  a.batch = p->batch;
  a.shift = log2_int(p->page_size);
  a.max_rows = p->max_rows;
  a.slots = p->slots;
  a.out_locations = p->out_locations;
  a.out_requests = p->out_requests;
  a.out_positions = p->out_positions;
  a.out_lengths = p->out_lengths;
  a.counts = p->counts;
  // A thread a row, and 512 workgroups at most (two a CU), as many as copies get, whose number the host does not know.
  // 256 / 512 / 1024 workgroups (us, whole call): 64 children of an 8192-token parent 9.3 / 7.5 / 10.1, a decode step of
  // 256 sequences 7.0 / 7.0 / 8.0, 48 new prompts of up to 32000 tokens - / 10.4 / 12.5.
  const int64_t wanted = ((int64_t)p->max_rows + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)std::max<int64_t>(p->parents ? 512 : 1, std::min<int64_t>(wanted, 512));
  if (p->batch <= kSmallBatch) extend_tables_kernel<kSmallBatch><<<grid, kThreads, 0, stream>>>(a);
  else extend_tables_kernel<kMaxBatch><<<grid, kThreads, 0, stream>>>(a);
  return hip_status(hipGetLastError(), "gk_extend_block_tables launch");
}

}  // namespace gk

extern "C" int gk_extend_block_tables(const gk_extend_params* params, hipStream_t stream) {
  gk::clear_error();
  return gk::extend_block_tables(params, stream);
}

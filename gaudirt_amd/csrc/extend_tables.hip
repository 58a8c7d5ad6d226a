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
// One launch. Every workgroup makes the three sums for itself, in LDS (8 bytes a
// sequence from L2 and one scan: 1.5 us for 1024 sequences), so nothing waits
// for another workgroup; then all threads share the rows, pages and copied
// tokens, four in a row each, whose sequence a binary search finds. What bounds
// it is the launch and that chain of round trips for a decode step, writing the
// map for long prompts.
#include "gk_common.hpp"

#include <algorithm>

namespace gk {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kPerThread = 4;  // consecutive rows, pages or tokens of a thread
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

__device__ __forceinline__ int64_t load_index(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// Sums that end at INT32_MAX instead of passing it: a batch whose sum gets there is refused.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, (uint32_t)INT32_MAX); }

struct Sums {
  uint32_t rows, pages, copies;
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) {
  return {add_sat(a.rows, b.rows), add_sat(a.pages, b.pages), add_sat(a.copies, b.copies)};
}
__device__ __forceinline__ Sums shift_up(const Sums& a, int n) {
  return {(uint32_t)__shfl_up((int)a.rows, n), (uint32_t)__shfl_up((int)a.pages, n), (uint32_t)__shfl_up((int)a.copies, n)};
}

// Last s with first[s] <= x (first[0] = 0 <= x < first[n]): the sequence that owns x, empty ones passed over.
__device__ __forceinline__ int owner(const int32_t* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int MAX>
__global__ __launch_bounds__(kThreads) void extend_tables_kernel(ExtendArgs a) {
  __shared__ int32_t s_row[MAX + 1], s_page[MAX + 1], s_copy[MAX + 1], s_prefix[MAX];
  __shared__ Sums s_wave[kWaves];
  __shared__ uint32_t s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = 1 << a.shift;
  const int head = a.free_head ? *a.free_head : 0;
  const int copy_shift = a.mapping ? 0 : a.shift;  // copies are numbered by token with a map, else by page
  if (tid == 0) s_bad = UINT32_MAX;
  __syncthreads();

  // A thread's sequences, their sums and the first one that cannot be right:
  // (index << 3 | code), the smallest over the batch.
  const int per = (a.batch + kThreads - 1) / kThreads, s0 = min(a.batch, tid * per), s1 = min(a.batch, s0 + per);
  uint32_t bad = UINT32_MAX;
  Sums mine{0, 0, 0};
  for (int s = s0; s < s1; ++s) {
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
      const int64_t held = (prefix + P - 1) >> a.shift;
      mine = mine + Sums{(uint32_t)length, (uint32_t)(((prefix + length + P - 1) >> a.shift) - held),
                         parent >= 0 ? (uint32_t)prefix >> copy_shift : 0u};
    }
    s_prefix[s] = (int32_t)(code ? 0 : prefix);
    s_row[s] = code ? 0 : (int32_t)length;  // kept for the second pass
    s_copy[s] = !code && parent >= 0;
  }
  Sums scan = mine;
#pragma unroll
  for (int n = 1; n < 64; n <<= 1) {
    const Sums below = shift_up(scan, n);
    if (lane >= n) scan = scan + below;
  }
  if (lane == 63) s_wave[wave] = scan;
  __syncthreads();
  Sums at = shift_up(scan, 1), total{0, 0, 0};
  if (lane == 0) at = Sums{0, 0, 0};
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at = at + s_wave[w];
    total = total + s_wave[w];
  }
  const int64_t free_left = head >= 0 && head <= a.free_count ? a.free_count - head : 0;
  for (int s = s0; s < s1; ++s) {
    const int length = s_row[s], prefix = s_prefix[s];
    const Sums one{(uint32_t)length,
                   (uint32_t)((((int64_t)prefix + length + P - 1) >> a.shift) - (((int64_t)prefix + P - 1) >> a.shift)),
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
  // A page of the free list, -1 where it lies outside the pool.
  const auto page_at = [&](int i) {
    const int64_t page = load_index(a.free_pages, a.pages64, (int64_t)head + i);
    return page >= 0 && page < (a.slots >> a.shift) ? (int32_t)page : -1;
  };
  const int64_t threads = (int64_t)gridDim.x * kThreads, thread = (int64_t)blockIdx.x * kThreads + tid;

  // Rows: slot, request and position of every new token; rows behind the last are no tokens.
  for (int64_t r0 = thread * kPerThread; r0 < a.max_rows; r0 += threads * kPerThread) {
    const int n = (int)min((int64_t)kPerThread, a.max_rows - r0);
    int s = r0 < rows ? owner(s_row, a.batch, (int)r0) : 0;
    int last_entry = -1, last_page = -1, last_seq = -1;
    int64_t request = 0;
    for (int k = 0; k < n; ++k) {
      const int r = (int)r0 + k;
      int32_t slot = -1, position = 0, where = 0;
      if (r < rows) {
        while (r >= s_row[s + 1]) ++s;
        const int prefix = s_prefix[s], held = (int)(((int64_t)prefix + P - 1) >> a.shift);
        position = prefix + (r - s_row[s]);
        const int entry = position >> a.shift;
        if (s != last_seq) request = load_index(a.seq_requests, a.requests64, s);
        if (s != last_seq || entry != last_entry)
          last_page = entry < held ? a.tables[request * a.pages + entry] : page_at(s_page[s] + entry - held);
        last_seq = s;
        last_entry = entry;
        slot = last_page >= 0 ? (int32_t)(((int64_t)last_page << a.shift) + (position & (P - 1))) : -1;
        where = (int32_t)request;
        if (a.mapping) a.mapping[request * a.context + position] = slot;
      }
      a.out_locations[r] = slot;
      a.out_requests[r] = where;
      a.out_positions[r] = position;
    }
  }
  // New pages into the tables.
  for (int64_t p = thread; p < pages; p += threads) {
    const int s = owner(s_page, a.batch, (int)p);
    const int held = (int)(((int64_t)s_prefix[s] + P - 1) >> a.shift);
    const int64_t request = load_index(a.seq_requests, a.requests64, s);
    a.tables[request * a.pages + held + ((int)p - s_page[s])] = page_at((int)p);
  }
  // The parents' tokens and pages into their children's rows.
  for (int64_t c0 = thread * kPerThread; c0 < copies; c0 += threads * kPerThread) {
    const int n = (int)min((int64_t)kPerThread, copies - c0);
    int s = owner(s_copy, a.batch, (int)c0), last_seq = -1;
    int64_t request = 0, parent = 0;
    for (int k = 0; k < n; ++k) {
      const int c = (int)c0 + k;
      while (c >= s_copy[s + 1]) ++s;
      if (s != last_seq) {
        request = load_index(a.seq_requests, a.requests64, s);
        parent = load_index(a.parents, a.requests64, s);
        last_seq = s;
      }
      const int t = (c - s_copy[s]) << copy_shift;
      if (a.mapping) a.mapping[request * a.context + t] = a.mapping[parent * a.context + t];
      if (!(t & (P - 1))) a.tables[request * a.pages + (t >> a.shift)] = a.tables[parent * a.pages + (t >> a.shift)];
    }
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
  // Enough threads for the rows; a map's copies, whose number the host does not know, get a whole GPU's.
  const int64_t wanted = ((int64_t)p->max_rows + kThreads * kPerThread - 1) / (kThreads * kPerThread);
  const unsigned grid = p->parents ? 256u : (unsigned)std::max<int64_t>(1, std::min<int64_t>(wanted, 512));
  if (p->batch <= kSmallBatch) extend_tables_kernel<kSmallBatch><<<grid, kThreads, 0, stream>>>(a);
  else extend_tables_kernel<kMaxBatch><<<grid, kThreads, 0, stream>>>(a);
  return hip_status(hipGetLastError(), "gk_extend_block_tables launch");
}

}  // namespace gk

extern "C" int gk_extend_block_tables(const gk_extend_params* params, hipStream_t stream) {
  gk::clear_error();
  return gk::extend_block_tables(params, stream);
}

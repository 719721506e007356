// A step's tables, made on the device from the sequences' lengths.
//
// The pages of all sequences come from one stack of free ones.  In one call each
// sequence b is cut to keep_b tokens, its pages behind them go back, and it takes
// pages for new_b more:
//
//   held = ceil(len / P), left = ceil(keep / P), need = ceil((keep + new) / P) - left
//   top = n_free + sum(held - left)
//   served: (need = 0 or sum_{c <= b} need_c <= top) and sum_{c <= b} new_c <= rows
//
// and row_start is the sum of the served sequences' new tokens.  Pages go back
// so that the first sequence's first one is on top, and are taken from the top in
// the same order: a step that keeps nothing of the last one's drafts gets the
// same pages again.
//
// tables_kernel is one workgroup: it moves a few kilobytes, so what bounds it is
// its chain of dependent loads (lengths, the entries that go back, the stack, the
// entries that are taken) and three sums over the sequences.  Each thread holds
// up to four sequences in registers; where a page or a row belongs is found by
// bisection in LDS.  The rows' positions, slots and masks follow in the same
// launch where they are few, in rows_kernel where they are many.
#include "draft.h"
#include "kvcache.h"

namespace {

constexpr int kThreads = 1024, kEach = 4, kMost = kThreads * kEach;  // sequences

struct TablesArgs {
  int32_t* table;  // [B][width]
  int32_t* lengths;
  int32_t* free;  // a stack of n_pages, of which n_free[0] are free
  int32_t* n_free;
  const int32_t* add;    // new tokens
  const int32_t* keep;   // null: all
  const int32_t* first;  // [B]: where a sequence's tree begins; null: at its kept length
  int width, n_pages, log_size, B, rows, max_new, max_len;
  int32_t* row_start;
  int32_t* kv_len;
  int32_t* base;
  int32_t* positions;
  int64_t* slots;
  int32_t* mask;           // [rows][words]; null without parents
  const int32_t* parents;  // [B or 1][nodes]
  int64_t ldp;             // 0: one tree for all
  int nodes, words;
};

// Row r of the step, whose sequences' first rows and lengths are `start` (B + 1)
// and `len`.
__device__ __forceinline__ void row_of(const TablesArgs& a, const int32_t* start, const int32_t* len, int r) {
  int32_t position = -1;
  int64_t slot = -1;
  int32_t* mask = a.mask ? a.mask + (int64_t)r * a.words : nullptr;
  if (r < start[a.B]) {
    const int b = lz_last_at(start, a.B, r), place = len[b] - start[b + 1] + r;
    const LzPages pg{a.table, a.width, a.n_pages, a.log_size};
    const int page = pg.page_of(b, place);
    position = place;
    if (page >= 0) slot = ((int64_t)page << a.log_size) + (place & ((1 << a.log_size) - 1));
    if (mask) {
      const int base = a.base[b], depth = lz_node_depth(a.parents + b * a.ldp, a.nodes, (int)((uint32_t)place - (uint32_t)base), mask,
                                                              a.words);
      if (depth >= 0) position = base + depth;
    }
  } else if (mask) {
    for (int w = 0; w < a.words; ++w) mask[w] = 0;
  }
  a.positions[r] = position;
  a.slots[r] = slot;
}

// Sums over the workgroup, in place: x becomes the sum of the threads before
// this one; returns the sum of all.  `sums`: a value a wave and one more.
__device__ __forceinline__ int64_t sum_before(int64_t& x, int64_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t z = __shfl_up(y, o, 64);
    if (lane >= o) y += z;
  }
  __syncthreads();  // the last sums have been read
  if (lane == 63) sums[wave] = y;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const int64_t z = sums[w];
    before += w < wave ? z : 0;
    all += z;
  }
  x = before + y - x;
  return all;
}

// `rows`: of the step, to be described here.
__global__ void __launch_bounds__(kThreads) tables_kernel(TablesArgs a, int rows) {
  __shared__ int32_t start[kMost + 1], len[kMost], left[kMost], gone[kMost + 1], taken[kMost + 1];
  __shared__ int64_t sums[kThreads / 64];
  const int tid = threadIdx.x;
  const int64_t cap = (int64_t)a.width << a.log_size;
  const int up = (1 << a.log_size) - 1;
  auto pages = [&](int64_t n) { return (int)((n + up) >> a.log_size); };

  int keep[kEach], add[kEach], need[kEach];
  int64_t back = 0, asked_pages = 0, asked = 0;
  const int free0 = min(max(a.n_free[0], 0), a.n_pages);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = tid * kEach + i;
    keep[i] = add[i] = need[i] = 0;
    if (b >= a.B) continue;
    const int now = (int)min((int64_t)max(a.lengths[b], 0), cap);
    keep[i] = a.keep ? min(max(a.keep[b], 0), now) : now;
    const int n = a.add[b];
    const int64_t total = (int64_t)keep[i] + n;
    if (n > 0 && n <= a.max_new && n <= a.rows && total <= min((int64_t)a.max_len, cap)) {
      add[i] = n;
      need[i] = pages(total) - pages(keep[i]);
    }
    left[b] = pages(keep[i]);
    gone[b] = pages(now) - left[b];
    back += gone[b];
    asked_pages += need[i];
    asked += add[i];
  }
  int64_t back_before = back;
  const int64_t all_back = sum_before(back_before, sums);
  const int64_t top = min(free0 + all_back, (int64_t)a.n_pages);
  sum_before(asked_pages, sums);
  sum_before(asked, sums);
  int64_t pages_here = 0, rows_here = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    asked_pages += need[i];
    asked += add[i];
    if ((need[i] > 0 && asked_pages > top) || asked > a.rows) add[i] = need[i] = 0;
    pages_here += need[i];
    rows_here += add[i];
  }
  int64_t page_at = pages_here, row_at = rows_here;
  const int64_t all_taken = sum_before(page_at, sums), all_rows = sum_before(row_at, sums);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = tid * kEach + i;
    if (b >= a.B) break;
    const int n = gone[b];
    gone[b] = (int)back_before;
    taken[b] = (int)page_at;
    start[b] = (int)row_at;
    len[b] = keep[i] + add[i];
    back_before += n;
    page_at += need[i];
    row_at += add[i];
    a.base[b] = a.first ? a.first[b] : keep[i];
    a.lengths[b] = a.kv_len[b] = len[b];
    a.row_start[b] = start[b];
  }
  if (tid == 0) {
    start[a.B] = a.row_start[a.B] = (int)all_rows;
    a.n_free[0] = (int)(top - all_taken);
  }
  __syncthreads();

  for (int x = tid; x < (int)all_back; x += kThreads) {
    const int b = lz_last_at(gone, a.B, x);
    int32_t* entry = a.table + (int64_t)b * a.width + left[b] + (x - gone[b]);
    const int64_t at = free0 + all_back - 1 - x;
    if (at < a.n_pages) a.free[at] = *entry;
    *entry = -1;
  }
  __syncthreads();
  for (int x = tid; x < (int)all_taken; x += kThreads) {
    const int b = lz_last_at(taken, a.B, x);
    a.table[(int64_t)b * a.width + left[b] + (x - taken[b])] = a.free[top - 1 - x];
  }
  if (rows == 0) return;  // the same for all
  __syncthreads();
  for (int r = tid; r < rows; r += kThreads) row_of(a, start, len, r);
}

__global__ void __launch_bounds__(256) rows_kernel(TablesArgs a) {
  __shared__ int32_t start[kMost + 1], len[kMost];
  for (int i = threadIdx.x; i <= a.B; i += 256) {
    start[i] = a.row_start[i];
    if (i < a.B) len[i] = a.kv_len[i];
  }
  __syncthreads();
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < a.rows) row_of(a, start, len, r);
}

}  // namespace

LZ_EXPORT int lz_cache_tables(int32_t* table, int64_t width, int32_t* lengths, int32_t* free, int64_t pages,
                              int32_t* n_free, int64_t page_size, const int32_t* add, const int32_t* keep,
                              const int32_t* first, const int32_t* parents, int64_t ldp, int64_t nodes, int64_t B,
                              int64_t rows, int64_t max_new, int64_t max_len, int32_t* row_start, int32_t* kv_len,
                              int32_t* base, int32_t* positions, int64_t* slots, int32_t* mask, int64_t words,
                              void* stream) {
  LZ_REQUIRE(lz_page_size_ok(page_size), "lz_cache_tables: page size %lld (a power of two, 16 to 1024)", (long long)page_size);
  LZ_REQUIRE(B > 0 && B <= kMost, "lz_cache_tables: %lld sequences (1 to %d)", (long long)B, kMost);
  LZ_REQUIRE(width > 0 && width * page_size <= INT32_MAX && B * width <= INT32_MAX - 1024 && pages > 0 && pages <= INT32_MAX - 1024 && rows >= 0 &&
                 rows <= INT32_MAX - 1024 && max_new >= 0 && max_new <= INT32_MAX && max_len >= 0 && max_len <= INT32_MAX,
             "lz_cache_tables: bad shape");
  LZ_REQUIRE((mask == nullptr) == (parents == nullptr), "lz_cache_tables: a mask and no parents, or the reverse");
  LZ_REQUIRE(!parents || (nodes > 0 && nodes <= (1 << 20) && words >= lz_cdiv(nodes, 32) && words <= (1 << 20) &&
                          (ldp == 0 || ldp >= nodes)),
             "lz_cache_tables: trees of %lld nodes in %lld mask words", (long long)nodes, (long long)words);
  LZ_REQUIRE(table && lengths && free && n_free && add && row_start && kv_len && base && (rows == 0 || (positions && slots)),
             "lz_cache_tables: bad arguments");
  TablesArgs a{table, lengths, free, n_free, add, keep, first, (int)width, (int)pages, lz_log2(page_size), (int)B,
               (int)rows, (int)max_new, (int)max_len, row_start, kv_len, base, positions, slots, mask, parents, ldp,
               (int)nodes, (int)words};
  const bool few = rows <= 2 * kThreads;
  tables_kernel<<<1, kThreads, 0, lz_stream(stream)>>>(a, few ? (int)rows : 0);
  if (!few) rows_kernel<<<(uint32_t)lz_cdiv(rows, 256), 256, 0, lz_stream(stream)>>>(a);
  return lz_check_launch("lz_cache_tables");
}

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
// (new_b that by itself passes max_new, max_len, the table or `rows` counts as 0
// in these sums: it could not be served in any order and holds up nobody)
// and row_start is the sum of the served sequences' new tokens.  Pages go back
// so that the first sequence's first one is on top, and are taken from the top in
// the same order: a step that keeps nothing of the last one's drafts gets the
// same pages again.
//
// tables_kernel is one workgroup: it moves a few kilobytes, so what bounds it is
// its chain of dependent loads (lengths, the entries that go back, the stack, the
// entries that are taken, the rows' pages) and four sums over the sequences, each
// of which threads hold up to four of in registers: 256 are one wave's, which needs
// no barrier for them.  Where a page or a row belongs is found by bisection in LDS,
// and trees are walked in LDS where they fit (64 x 24 nodes: 7.3 us a call, from
// memory 9.4).  The rows' positions, slots and masks follow in the same launch
// where they are few, in rows_kernel where they are many.
#include "draft.h"
#include "kvcache.h"

namespace {

constexpr int kThreads = 1024, kEach = 4, kMost = kThreads * kEach;  // sequences
constexpr int kTrees = 8192;  // parents that LDS holds

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
// and `len`; base and parents: a.base and a.parents, or copies.
__device__ __forceinline__ void row_of(const TablesArgs& a, const int32_t* start, const int32_t* len, const int32_t* bases,
                                       const int32_t* parents, int r) {
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
      const int base = bases[b];
      const int depth =
          lz_node_depth(parents + b * a.ldp, a.nodes, (int)((uint32_t)place - (uint32_t)base), mask, a.words);
      if (depth >= 0) position = base + depth;
    }
  } else if (mask) {
    for (int w = 0; w < a.words; ++w) mask[w] = 0;
  }
  a.positions[r] = position;
  a.slots[r] = slot;
}

// Sums that stop at INT32_MAX (what sequences ask for together may be any number).
__device__ __forceinline__ int add_up(int x, int y) {
  const uint32_t z = (uint32_t)x + (uint32_t)y;
  return z > (uint32_t)INT32_MAX ? INT32_MAX : (int)z;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_shifted(int x) {
  return add_up(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false));
}

// x becomes the sum of the threads up to this one, of the wave (`waves` 1) or the
// workgroup; returns the sum of all.  `sums`: a value a wave.
__device__ __forceinline__ int sum_up_to(int& x, int* sums, int waves) {
  x = add_shifted<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8, row_bcast 15, 31
  x = add_shifted<0x112, 0xf>(x);
  x = add_shifted<0x114, 0xf>(x);
  x = add_shifted<0x118, 0xf>(x);
  x = add_shifted<0x142, 0xa>(x);
  x = add_shifted<0x143, 0xc>(x);
  if (waves == 1) return __builtin_amdgcn_readlane(x, 63);
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // the last sums have been read
  if ((threadIdx.x & 63) == 63) sums[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before = add_up(before, w < wave ? sums[w] : 0);
    all = add_up(all, sums[w]);
  }
  x = add_up(x, before);
  return all;
}

struct TablesLds {
  int32_t start[kMost + 1], len[kMost], base[kMost], left[kMost], gone[kMost], taken[kMost], parents[kTrees];
  int sums[kThreads / 64];
  int all_back, all_taken, top, free0;
};

// The sequences of this thread: what they ask for and get.  `waves`: that hold
// any sequences, 1 or all of the workgroup's.
__device__ __forceinline__ void deal(const TablesArgs& a, TablesLds& s, int waves) {
  const int tid = threadIdx.x;
  const int64_t cap = (int64_t)a.width << a.log_size;
  const int up = (1 << a.log_size) - 1;
  auto pages = [&](int64_t n) { return (int)((n + up) >> a.log_size); };
  int now[kEach], keep[kEach], add[kEach], need[kEach], first[kEach];
  const int free0 = min(max(a.n_free[0], 0), a.n_pages);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = tid * kEach + i;
    now[i] = b < a.B ? a.lengths[b] : 0;
    keep[i] = b < a.B && a.keep ? a.keep[b] : INT32_MAX;
    add[i] = b < a.B ? a.add[b] : 0;
    first[i] = b < a.B && a.first ? a.first[b] : 0;
  }
  int back = 0, asked_pages = 0, asked = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    now[i] = (int)min((int64_t)max(now[i], 0), cap);
    keep[i] = min(max(keep[i], 0), now[i]);
    const int64_t total = (int64_t)keep[i] + add[i];
    if (!(add[i] > 0 && add[i] <= a.max_new && add[i] <= a.rows && total <= min((int64_t)a.max_len, cap))) add[i] = 0;
    need[i] = add[i] ? pages(total) - pages(keep[i]) : 0;
    back += pages(now[i]) - pages(keep[i]);
    asked_pages += need[i];
    asked = add_up(asked, add[i]);
  }
  int back_at = back, pages_at = asked_pages, rows_at = asked;
  const int all_back = sum_up_to(back_at, s.sums, waves);
  const int top = (int)min((int64_t)free0 + all_back, (int64_t)a.n_pages);
  sum_up_to(pages_at, s.sums, waves);
  sum_up_to(rows_at, s.sums, waves);
  // the sums up to each of this thread's, from the last one back (a sum that was cut
  // off is over a.rows, which is 2^28 at most, without this thread's up to 2^30)
  int taken = 0, rows = 0, over_pages = pages_at, over_rows = rows_at;
#pragma unroll
  for (int i = kEach - 1; i >= 0; --i) {
    const int p = over_pages, r = over_rows;
    over_pages -= need[i];
    over_rows = r == INT32_MAX ? r : r - add[i];
    if ((need[i] > 0 && p > top) || r > a.rows) add[i] = need[i] = 0;
    taken += need[i];
    rows += add[i];
  }
  int taken_at = taken, row_at = rows;
  const int all_taken = sum_up_to(taken_at, s.sums, waves), all_rows = sum_up_to(row_at, s.sums, waves);
  taken_at -= taken;
  row_at -= rows;
  back_at -= back;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = tid * kEach + i;
    if (b >= a.B) break;
    s.left[b] = pages(keep[i]);
    s.gone[b] = back_at;
    s.taken[b] = taken_at;
    s.start[b] = row_at;
    s.len[b] = keep[i] + add[i];
    s.base[b] = a.first ? first[i] : keep[i];
    back_at += pages(now[i]) - pages(keep[i]);
    taken_at += need[i];
    row_at += add[i];
    a.lengths[b] = a.kv_len[b] = s.len[b];
    a.row_start[b] = s.start[b];
    a.base[b] = s.base[b];
  }
  if (tid == 0) {
    s.start[a.B] = a.row_start[a.B] = all_rows;
    a.n_free[0] = top - all_taken;
    s.all_back = all_back;
    s.all_taken = all_taken;
    s.top = top;
    s.free0 = free0;
  }
}

// `rows`: of the step, to be described here.
__global__ void __launch_bounds__(kThreads) tables_kernel(TablesArgs a, int rows) {
  __shared__ TablesLds s;
  const int tid = threadIdx.x;
  const bool one_wave = a.B <= 64 * kEach;
  const int trees = rows > 0 && a.parents ? (a.ldp ? a.B : 1) * a.nodes : 0;
  const bool near = trees > 0 && trees <= kTrees;
  if (one_wave) {
    if (tid < 64) deal(a, s, 1);
    else if (near)
      for (int i = tid - 64; i < trees; i += kThreads - 64) s.parents[i] = a.parents[i];
  } else {
    deal(a, s, kThreads / 64);
    if (near)
      for (int i = tid; i < trees; i += kThreads) s.parents[i] = a.parents[i];
  }
  __syncthreads();

  const int all_back = s.all_back, top = s.top;
  for (int x = tid; x < all_back; x += kThreads) {
    const int b = lz_last_at(s.gone, a.B, x);
    int32_t* entry = a.table + (int64_t)b * a.width + s.left[b] + (x - s.gone[b]);
    const int64_t at = (int64_t)s.free0 + all_back - 1 - x;
    if (at < a.n_pages) a.free[at] = *entry;
    *entry = -1;
  }
  if (all_back) __syncthreads();  // the same for all
  for (int x = tid; x < s.all_taken; x += kThreads) {
    const int b = lz_last_at(s.taken, a.B, x);
    a.table[(int64_t)b * a.width + s.left[b] + (x - s.taken[b])] = a.free[top - 1 - x];
  }
  if (rows == 0) return;
  if (s.all_taken) __syncthreads();
  for (int r = tid; r < rows; r += kThreads) row_of(a, s.start, s.len, s.base, near ? s.parents : a.parents, r);
}

__global__ void __launch_bounds__(256) rows_kernel(TablesArgs a) {
  __shared__ int32_t start[kMost + 1], len[kMost];
  for (int i = threadIdx.x; i <= a.B; i += 256) {
    start[i] = a.row_start[i];
    if (i < a.B) len[i] = a.kv_len[i];
  }
  __syncthreads();
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < a.rows) row_of(a, start, len, a.base, a.parents, r);
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
                 rows <= (1 << 28) && max_new >= 0 && max_new <= INT32_MAX && max_len >= 0 && max_len <= INT32_MAX,
             "lz_cache_tables: bad shape");
  LZ_REQUIRE((mask == nullptr) == (parents == nullptr), "lz_cache_tables: a mask and no parents, or the reverse");
  LZ_REQUIRE(!parents || (nodes > 0 && nodes <= kMostNodes && words >= lz_cdiv(nodes, 32) && words <= (1 << 20) &&
                          (ldp == 0 || ldp == nodes)),
             "lz_cache_tables: trees of %lld nodes (1 to %d) in %lld mask words", (long long)nodes, kMostNodes, (long long)words);
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

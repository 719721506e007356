// The paged key/value cache as the kernels see it.
//
// A layer's keys and values are [pages][KV][page size][hd] each, in the
// model's type or as e4m3 with one exponent e per (page, kv head, token): the
// value is the stored number times 2^e.  Page ids are multiplied out in 64
// bits (a layer's pages may pass 2^31 elements).  What the device tables say
// is not trusted: an id outside [0, pages), a position outside the page table
// or a row outside row_start's ranges is left out, never an address.
#pragma once
#include "lz_common.h"

#define LZ_E4M3 8  // float8_e4m3fn storage of a cache, beside LZ_F32, LZ_BF16 and LZ_F16

struct LzPages {
  const int32_t* table;  // [B][width] page ids
  int width;
  int pages;
  int log_size;  // page size = 1 << log_size

  // The page that holds position p of sequence b, or -1.
  __host__ __device__ __forceinline__ int page_of(int b, int p) const {
    const int i = p >> log_size;
    if (p < 0 || i >= width) return -1;
    const int id = table[(int64_t)b * width + i];
    return id >= 0 && id < pages ? id : -1;
  }
};

// The sequence b with start[b] <= r < start[b + 1], or -1.  Sequences of one
// length (single tokens above all) are hit by the first guess, whose two
// loads are independent; other batches bisect.
__host__ __device__ __forceinline__ int lz_seq_of_row(const int32_t* __restrict__ start, int B, int rows, int r) {
  const int g = (int)((int64_t)r * B / rows);
  if (start[g] <= r && r < start[g + 1]) return g;
  int lo = 0, hi = B;  // the last b with start[b] <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= r) lo = mid;
    else hi = mid;
  }
  return start[lo] <= r && r < start[lo + 1] ? lo : -1;
}

// The sequence of a row and its place, for kernels whose rows are of many
// sequences.  Where the first guess serves (no more rows than sequences, or
// one sequence) it costs one round of loads; elsewhere the workgroup copies
// the tables into LDS in one round and bisects there (8736 rows of 16 prompts,
// bisected in memory and so: 13.4 and 12.4 us to write in e4m3, 6.1 and 5.4 to
// read back; 30000 cached tokens of four sequences 43.3 and 40.0).
struct LzSeqs {
  static constexpr int kMost = 1024;  // sequences that LDS holds
  int32_t start[kMost + 1], len[kMost];

  // With the whole workgroup.  kv_len may be null.
  __device__ __forceinline__ void load(const int32_t* row_start, const int32_t* kv_len, int B, int rows, int tid) {
    if (rows <= B || B == 1 || B > kMost) return;  // the same for all
    for (int i = tid; i <= B; i += 256) {
      start[i] = row_start[i];
      if (kv_len && i < B) len[i] = kv_len[i];
    }
    __syncthreads();
  }
  // (sequence or -1, rows before its first or, with kv_len, its length minus
  // the row that comes after its last: the row's position is row - or + that)
  __device__ __forceinline__ int find(const int32_t* row_start, const int32_t* kv_len, int B, int rows, int r,
                                      int& base) const {
    if (rows <= B || B == 1 || B > kMost) {
      const int g = (int)((int64_t)r * B / rows);
      const int s0 = row_start[g], s1 = row_start[g + 1], l = kv_len ? kv_len[g] : 0;
      if (s0 <= r && r < s1) {
        base = kv_len ? l - s1 : -s0;
        return g;
      }
      const int b = lz_seq_of_row(row_start, B, rows, r);
      if (b >= 0) base = kv_len ? kv_len[b] - row_start[b + 1] : -row_start[b];
      return b;
    }
    const int b = lz_seq_of_row(start, B, rows, r);
    if (b >= 0) base = kv_len ? len[b] - start[b + 1] : -start[b];
    return b;
  }
};

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float lz_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

static inline bool lz_page_size_ok(int64_t n) { return n >= 16 && n <= 1024 && (n & (n - 1)) == 0; }
static inline int lz_log2(int64_t n) {
  int k = 0;
  while ((int64_t(1) << (k + 1)) <= n) ++k;
  return k;
}

// The checks that every entry point makes of a cache layer; LZ_OK or a status.
int lz_check_pages(const char* what, const void* k, const void* v, const void* k_exp, const void* v_exp, int cache_dtype,
                   int dtype, int64_t pages, int64_t page_size, const void* table, int64_t width, int64_t B, int64_t KV,
                   int64_t hd);

// RUN(T, HD, is e4m3) for the call's types and head dim.
#define LZ_CACHE_CASES(dtype, cache, hd, RUN)                         \
  do {                                                                \
    const bool e8 = (cache) == LZ_E4M3;                               \
    if ((dtype) == LZ_BF16) { LZ_CACHE_HD(uint16_t, e8, hd, RUN); }   \
    else if ((dtype) == LZ_F16) { LZ_CACHE_HD(_Float16, e8, hd, RUN); } \
    else { LZ_CACHE_HD(float, e8, hd, RUN); }                         \
  } while (0)
#define LZ_CACHE_HD(T, e8, hd, RUN)                 \
  do {                                              \
    if ((hd) == 32) { if (e8) RUN(T, 32, true); else RUN(T, 32, false); }        \
    else if ((hd) == 64) { if (e8) RUN(T, 64, true); else RUN(T, 64, false); }   \
    else { if (e8) RUN(T, 128, true); else RUN(T, 128, false); }                 \
  } while (0)

// Writing a paged key/value cache, reading it back, and moving the tokens that
// are kept of a draft.
//
// lz_kv_write takes the rows of a fused QKV product, rotates q and k at each
// row's own position (NeoX half split: y1 = x1 c1 - x2 s1, y2 = x2 c2 + x1 s2,
// as lz_rope), writes the rotated q out and k and v into the sequence's pages.
// The rotation is formed in fp32, each product and sum rounded on its own
// (this file is built without contraction), and rounded to the storage type
// once; lz_rope rounds every step to the activation type, as the reference's
// separate operations do, which costs a factor 1.7 in error and would move
// about 2 % of the e4m3 values by a step.
//
// e4m3 storage: e is the smallest integer with max |x| <= 448 * 2^e over a
// (token, head)'s hd values, so x * 2^-e is exact and each value is rounded
// once, by at most half a step of e4m3 (2^-4 of a normal value).  A power of
// two costs no precision against max/448 as a factor (e4m3's steps are
// relative) and makes the way back exact in bf16: four significant bits.  e is
// kept in -120..119 (448 * 2^119 is the largest finite value of that form), and
// in -15..7 for fp16 rows, so that every stored value is an fp16 number (a
// multiple of 2^-24 up to 57344); larger inputs become the largest value.  All
// zeros take e = 0.  An infinity or NaN is stored as NaN and left out of the
// maximum.
#include <type_traits>

#include "kvcache.h"

namespace {

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void load(float (&x)[N], const T* p) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = Elem<T>::load(e, i);
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[N]) {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < N; ++i) Elem<T>::store(e, i, x[i]);
    *reinterpret_cast<uint4*>(p) = w;
  }
};

// Four floats to four e4m3 bytes (round to nearest even; |x| <= 448, or not
// finite: NaN).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// CAP: finite values past 448 / inv become that.
template <int N, bool CAP>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&x)[N], float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = x[4 * i + e] * inv;
      if constexpr (CAP)
        if (fabsf(x[4 * i + e]) < INFINITY) y[e] = fminf(fmaxf(y[e], -448.f), 448.f);
    }
    w[i] = pack_e4m3(y[0], y[1], y[2], y[3]);
  }
  if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// The exponent of a group's largest finite magnitude (see above).
template <bool kHalf>
__device__ __forceinline__ int exponent_of(float amax) {
  if (amax == 0.f) return 0;
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);  // 448 = 1.75 * 2^8
  return kHalf ? min(max(e, -15), 7) : min(max(e, -120), 119);
}

struct WriteArgs {
  const void* qkv;
  int64_t ld;
  const void* cos;
  const void* sin;
  void* q;
  int64_t ldq;
  void* k;
  void* v;
  int8_t* k_exp;
  int8_t* v_exp;
  LzPages pg;
  const int32_t* row_start;
  const int32_t* kv_len;
  int rows, positions, B, H, KV;
  const int32_t* turn;  // kTurn: the position that each row is rotated to
};

// One thread per (row, head, 16 bytes of its lower half and the same of its
// upper half): a head is HD / 2 / N neighbouring lanes.  kTurn: a drafted token's
// position is its depth in its tree, not the place where it is cached.
template <typename T, int HD, bool k8, bool kTurn>
__global__ void __launch_bounds__(256) kv_write_kernel(WriteArgs a) {
  __shared__ LzSeqs seqs;
  seqs.load(a.row_start, a.kv_len, a.B, a.rows, threadIdx.x);
  constexpr int N = Vec<T>::N, kLanes = HD / 2 / N;
  const int heads = a.H + 2 * a.KV, per_row = heads * kLanes;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const int row = (int)(idx / (uint32_t)per_row);
  if (row >= a.rows) return;  // whole heads: HD / 2 / N divides both 64 and per_row
  const int rem = (int)(idx - (uint32_t)row * (uint32_t)per_row);
  const int head = rem / kLanes, i = (rem - head * kLanes) * N;

  float lo[N], hi[N];
  const T* x = static_cast<const T*>(a.qkv) + row * a.ld + (int64_t)head * HD + i;
  Vec<T>::load(lo, x);
  Vec<T>::load(hi, x + HD / 2);
  int base = 0;
  const int b = seqs.find(a.row_start, a.kv_len, a.B, a.rows, row, base);
  if (b < 0) return;
  const int pos = base + row, turn = kTurn ? a.turn[row] : pos;
  const bool there = turn >= 0 && turn < a.positions;
  if (head < a.H + a.KV) {
    if (there) {
      const T* cp = static_cast<const T*>(a.cos) + (int64_t)turn * HD + i;
      const T* sp = static_cast<const T*>(a.sin) + (int64_t)turn * HD + i;
      float c1[N], c2[N], s1[N], s2[N];
      Vec<T>::load(c1, cp);
      Vec<T>::load(c2, cp + HD / 2);
      Vec<T>::load(s1, sp);
      Vec<T>::load(s2, sp + HD / 2);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float u = lo[e], w = hi[e];
        lo[e] = u * c1[e] + -w * s1[e];
        hi[e] = w * c2[e] + u * s2[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) lo[e] = hi[e] = 0.f;
    }
    if (head < a.H) {
      T* q = static_cast<T*>(a.q) + row * a.ldq + (int64_t)head * HD + i;
      Vec<T>::store(q, lo);
      Vec<T>::store(q + HD / 2, hi);
      return;
    }
  }
  const int page = there ? a.pg.page_of(b, pos) : -1;
  if (page < 0) return;
  const bool is_k = head < a.H + a.KV;
  const int g = head - a.H - (is_k ? 0 : a.KV);
  const int64_t token = (((int64_t)page * a.KV + g) << a.pg.log_size) + (pos & ((1 << a.pg.log_size) - 1));
  if constexpr (!k8) {
    T* dst = static_cast<T*>(is_k ? a.k : a.v) + token * HD + i;
    Vec<T>::store(dst, lo);
    Vec<T>::store(dst + HD / 2, hi);
  } else {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float u = fabsf(lo[e]), w = fabsf(hi[e]);
      amax = u < INFINITY ? fmaxf(amax, u) : amax;
      amax = w < INFINITY ? fmaxf(amax, w) : amax;
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    const int e = exponent_of<std::is_same<T, _Float16>::value>(amax);
    const float inv = lz_pow2(-e);
    uint8_t* dst = static_cast<uint8_t*>(is_k ? a.k : a.v) + token * HD + i;
    if (amax * inv > 448.f) {  // the exponent is at its limit
      store_e4m3<N, true>(dst, lo, inv);
      store_e4m3<N, true>(dst + HD / 2, hi, inv);
    } else {
      store_e4m3<N, false>(dst, lo, inv);
      store_e4m3<N, false>(dst + HD / 2, hi, inv);
    }
    if (i == 0) (is_k ? a.k_exp : a.v_exp)[token] = (int8_t)e;
  }
}

struct ReadArgs {
  const void* k;
  const void* v;
  const int8_t* k_exp;
  const int8_t* v_exp;
  LzPages pg;
  const int32_t* start;
  void* k_out;
  void* v_out;
  int rows, B, KV;
};

struct KeepArgs {
  void* k;
  void* v;
  int8_t* k_exp;
  int8_t* v_exp;
  const int64_t* slots;      // [rows]: page * page size + place in it, -1 without one
  const int32_t* row_start;
  const int32_t* kept;       // [B][ldk]
  const int32_t* counts;
  int64_t ldk, slots_all;    // slots of a layer
  int rows, layers, KV, log_size, nodes;
};

// Moves the kept nodes of each sequence to its first slots of the step: node
// kept[j]'s keys and values to slot j.  One thread per (layer, keys or values, kv
// head, 16 bytes of a token), and gridDim.y for the sequences: it goes over the
// nodes in their order, eight at a time, all of which it reads before it writes.
// kept ascends, so kept[j] >= j: what a thread still has to read lies behind what
// it has written, and no other thread touches its bytes.
//
// The eight are not in flight together: as compiled each one's 16 bytes go to
// scratch (144 bytes a thread) and wait for the load, and that chain of loads
// bounds it (32 sequences of up to 32 nodes, 32 layers of 8 heads of 128 in bf16:
// 10.7 us for 22 MB; a trial that kept them in registers, with a vector type for
// uint4 and loads that no branch surrounds, took 6.6).  Whether a node moves stands apart in moves[]: with -1 in
// to[] for it and `continue` in place of the condition, hipcc of ROCm 7.2 held to[]
// in one run of registers, wrote a comparison's operand into those of to[0] ahead
// of a branch, and a token went to place slots_all.
template <bool k8>
__global__ void __launch_bounds__(256) kv_keep_kernel(KeepArgs a, int chunks) {
  constexpr int kAhead = 8;
  const int b = blockIdx.y;
  int node[kAhead];  // fetched beside the counts that say which of them there are
#pragma unroll
  for (int i = 0; i < kAhead; ++i) node[i] = a.kept[b * a.ldk + min(i, a.nodes - 1)];
  const int lo = min(max(a.row_start[b], 0), a.rows), hi = min(max(a.row_start[b + 1], lo), a.rows), n = hi - lo;
  const int count = min(min(a.counts[b], n), a.nodes);
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t per_layer = 2u * (uint32_t)a.KV * (uint32_t)chunks;
  const uint32_t layer = idx / per_layer, rem = idx - layer * per_layer;
  if (layer >= (uint32_t)a.layers) return;
  const int side = rem >= per_layer / 2, at = (int)(rem - side * (per_layer / 2));
  const int g = at / chunks, c = at - g * chunks;
  const int64_t token = (int64_t)layer * a.slots_all * a.KV;  // of the layer's first page and head
  char* x = static_cast<char*>(side ? a.v : a.k) + (token * chunks + c) * 16;
  int8_t* e = k8 ? (side ? a.v_exp : a.k_exp) + token : nullptr;
  const int mask = (1 << a.log_size) - 1;
  auto place = [&](int64_t slot) {  // of this head, in tokens
    return ((((slot >> a.log_size) * a.KV + g) << a.log_size) + (slot & mask));
  };
  for (int j0 = 0; j0 < count; j0 += kAhead) {
    // nodes, their slots, their tokens
    if (j0 > 0)
#pragma unroll
      for (int i = 0; i < kAhead; ++i) node[i] = a.kept[b * a.ldk + min(j0 + i, a.nodes - 1)];
    int64_t from[kAhead], to[kAhead];
    bool moves[kAhead];
    uint4 w[kAhead];
    int8_t we[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      from[i] = a.slots[lo + min(max(node[i], 0), n - 1)];
      to[i] = a.slots[lo + min(j0 + i, count - 1)];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      moves[i] = j0 + i < count && node[i] >= 0 && node[i] < n && node[i] != j0 + i && (uint64_t)from[i] < (uint64_t)a.slots_all &&
                 (uint64_t)to[i] < (uint64_t)a.slots_all;
      if (moves[i]) {  // the same for the workgroup
        const int64_t src = place(from[i]);
        w[i] = *reinterpret_cast<const uint4*>(x + src * chunks * 16);
        if (k8) we[i] = e[src];
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (moves[i]) {
        const int64_t dst = place(to[i]);
        *reinterpret_cast<uint4*>(x + dst * chunks * 16) = w[i];
        if (k8 && c == 0) e[dst] = we[i];
      }
  }
}

// One thread per 16 bytes of an output row, keys and values alike.
template <typename T, int HD, bool k8>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
  __shared__ LzSeqs seqs;
  seqs.load(a.start, nullptr, a.B, a.rows, threadIdx.x);
  constexpr int N = Vec<T>::N, kLanes = HD / N;
  const int per_row = a.KV * kLanes;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const int row = (int)(idx / (uint32_t)per_row);
  if (row >= a.rows) return;
  const int rem = (int)(idx - (uint32_t)row * (uint32_t)per_row);
  const int g = rem / kLanes, i = (rem - g * kLanes) * N;
  int base = 0;
  const int b = seqs.find(a.start, nullptr, a.B, a.rows, row, base);
  const int pos = base + row;
  const int page = b < 0 ? -1 : a.pg.page_of(b, pos);
  const int64_t token = (((int64_t)page * a.KV + g) << a.pg.log_size) + (pos & ((1 << a.pg.log_size) - 1));
  const int64_t out = ((int64_t)row * a.KV + g) * HD + i;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    T* dst = static_cast<T*>(side ? a.v_out : a.k_out) + out;
    const void* src = side ? a.v : a.k;
    if (page < 0) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    } else if constexpr (!k8) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(static_cast<const T*>(src) + token * HD + i);
    } else {
      uint32_t w[N / 4];
      const uint8_t* p = static_cast<const uint8_t*>(src) + token * HD + i;
#pragma unroll
      for (int j = 0; j < N / 4; ++j) w[j] = reinterpret_cast<const uint32_t*>(p)[j];
      const float unit = lz_pow2((side ? a.v_exp : a.k_exp)[token]);
      float x[N];
#pragma unroll
      for (int j = 0; j < N / 4; ++j) {
        x[4 * j] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 0) * unit;
        x[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 1) * unit;
        x[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 2) * unit;
        x[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[j], 3) * unit;
      }
      Vec<T>::store(dst, x);
    }
  }
}

}  // namespace

int lz_check_pages(const char* what, const void* k, const void* v, const void* k_exp, const void* v_exp, int cache_dtype,
                int dtype, int64_t pages, int64_t page_size, const void* table, int64_t width, int64_t B, int64_t KV,
                int64_t hd) {
  LZ_REQUIRE(dtype == LZ_BF16 || dtype == LZ_F16 || dtype == LZ_F32, "%s: bad dtype %d", what, dtype);
  LZ_REQUIRE(cache_dtype == dtype || cache_dtype == LZ_E4M3, "%s: a cache of dtype %d with rows of dtype %d", what,
             cache_dtype, dtype);
  LZ_REQUIRE(hd == 32 || hd == 64 || hd == 128, "%s: head dim %lld (32, 64 or 128)", what, (long long)hd);
  LZ_REQUIRE(lz_page_size_ok(page_size), "%s: page size %lld (a power of two, 16 to 1024)", what, (long long)page_size);
  LZ_REQUIRE(pages > 0 && pages <= INT32_MAX && width > 0 && width * page_size <= INT32_MAX && B > 0 && B < INT32_MAX &&
                 KV > 0 && KV <= 65536,
             "%s: bad shape", what);
  LZ_REQUIRE(k && v && table && lz_aligned16(k) && lz_aligned16(v), "%s: pages must be 16-byte aligned", what);
  LZ_REQUIRE(cache_dtype != LZ_E4M3 || (k_exp && v_exp && lz_aligned16(k_exp) && lz_aligned16(v_exp)),
             "%s: an e4m3 cache needs its exponents, 16-byte aligned", what);
  return LZ_OK;
}

static int write(const char* what, const void* qkv, int64_t ld, int dtype, int64_t rows, const void* cos_t,
                 const void* sin_t, int64_t positions, void* q_out, int64_t ldq, void* k, void* v, void* k_exp, void* v_exp,
                 int cache_dtype, int64_t pages, int64_t page_size, const int32_t* table, int64_t width,
                 const int32_t* row_start, const int32_t* kv_len, const int32_t* turn, int64_t B, int64_t H, int64_t KV,
                 int64_t hd, void* stream) {
  if (int rc = lz_check_pages(what, k, v, k_exp, v_exp, cache_dtype, dtype, pages, page_size, table, width, B, KV,
                           hd))
    return rc;
  const int esz = lz_esize(dtype);
  LZ_REQUIRE(rows >= 0 && rows <= INT32_MAX && H > 0 && H <= 65536 && positions > 0 && positions <= INT32_MAX,
             "%s: bad shape", what);
  LZ_REQUIRE(ld >= (H + 2 * KV) * hd && ldq >= H * hd, "%s: row strides shorter than the rows", what);
  LZ_REQUIRE(rows == 0 || (qkv && q_out && cos_t && sin_t && row_start && kv_len && lz_aligned16(qkv) &&
                           lz_aligned16(q_out) && lz_aligned16(cos_t) && lz_aligned16(sin_t) && ld * esz % 16 == 0 &&
                           ldq * esz % 16 == 0),
             "%s: rows and tables must be 16-byte aligned", what);
  if (rows == 0) return LZ_OK;
  const int64_t threads = rows * (H + 2 * KV) * (hd * esz / 32);
  LZ_REQUIRE(threads <= (int64_t)UINT32_MAX - 255, "%s: too many rows", what);
  WriteArgs a{qkv, ld, cos_t, sin_t, q_out, ldq, k, v, (int8_t*)k_exp, (int8_t*)v_exp,
              LzPages{table, (int)width, (int)pages, lz_log2(page_size)}, row_start, kv_len,
              (int)rows, (int)positions, (int)B, (int)H, (int)KV, turn};
  const uint32_t grid = (uint32_t)lz_cdiv(threads, 256);
  hipStream_t s = lz_stream(stream);
#define RUN(T, HD, E8)                                                   \
  do {                                                                   \
    if (turn) kv_write_kernel<T, HD, E8, true><<<grid, 256, 0, s>>>(a);  \
    else kv_write_kernel<T, HD, E8, false><<<grid, 256, 0, s>>>(a);      \
  } while (0)
  LZ_CACHE_CASES(dtype, cache_dtype, hd, RUN);
#undef RUN
  return lz_check_launch(what);
}

LZ_EXPORT int lz_kv_write(const void* qkv, int64_t ld, int dtype, int64_t rows, const void* cos_t, const void* sin_t,
                          int64_t positions, void* q_out, int64_t ldq, void* k, void* v, void* k_exp, void* v_exp,
                          int cache_dtype, int64_t pages, int64_t page_size, const int32_t* table, int64_t width,
                          const int32_t* row_start, const int32_t* kv_len, int64_t B, int64_t H, int64_t KV, int64_t hd,
                          void* stream) {
  return write("lz_kv_write", qkv, ld, dtype, rows, cos_t, sin_t, positions, q_out, ldq, k, v, k_exp, v_exp, cache_dtype,
               pages, page_size, table, width, row_start, kv_len, nullptr, B, H, KV, hd, stream);
}

LZ_EXPORT int lz_kv_write_at(const void* qkv, int64_t ld, int dtype, int64_t rows, const void* cos_t, const void* sin_t,
                             int64_t positions, void* q_out, int64_t ldq, void* k, void* v, void* k_exp, void* v_exp,
                             int cache_dtype, int64_t pages, int64_t page_size, const int32_t* table, int64_t width,
                             const int32_t* row_start, const int32_t* kv_len, const int32_t* row_position, int64_t B,
                             int64_t H, int64_t KV, int64_t hd, void* stream) {
  LZ_REQUIRE(rows == 0 || row_position, "lz_kv_write_at: no positions");
  return write("lz_kv_write_at", qkv, ld, dtype, rows, cos_t, sin_t, positions, q_out, ldq, k, v, k_exp, v_exp, cache_dtype,
               pages, page_size, table, width, row_start, kv_len, row_position, B, H, KV, hd, stream);
}

LZ_EXPORT int lz_kv_keep(void* k, void* v, void* k_exp, void* v_exp, int cache_dtype, int64_t layers, int64_t pages,
                         int64_t page_size, int64_t KV, int64_t hd, const int64_t* slots, int64_t rows,
                         const int32_t* row_start, int64_t B, const int32_t* kept, int64_t ldk, int64_t nodes,
                         const int32_t* counts, void* stream) {
  LZ_REQUIRE(cache_dtype == LZ_BF16 || cache_dtype == LZ_F16 || cache_dtype == LZ_F32 || cache_dtype == LZ_E4M3,
             "lz_kv_keep: bad dtype %d", cache_dtype);
  LZ_REQUIRE(hd == 32 || hd == 64 || hd == 128, "lz_kv_keep: head dim %lld (32, 64 or 128)", (long long)hd);
  LZ_REQUIRE(lz_page_size_ok(page_size), "lz_kv_keep: page size %lld (a power of two, 16 to 1024)", (long long)page_size);
  LZ_REQUIRE(layers > 0 && layers <= 65536 && pages > 0 && pages <= INT32_MAX && KV > 0 && KV <= 65536 && B > 0 &&
                 B <= 65535 && rows >= 0 && rows <= INT32_MAX && nodes >= 0 && nodes <= INT32_MAX,
             "lz_kv_keep: bad shape");
  LZ_REQUIRE(k && v && lz_aligned16(k) && lz_aligned16(v), "lz_kv_keep: pages must be 16-byte aligned");
  LZ_REQUIRE(cache_dtype != LZ_E4M3 || (k_exp && v_exp), "lz_kv_keep: an e4m3 cache needs its exponents");
  if (rows == 0 || nodes == 0) return LZ_OK;
  LZ_REQUIRE(slots && row_start && kept && counts && ldk >= nodes, "lz_kv_keep: bad arguments");
  const bool e8 = cache_dtype == LZ_E4M3;
  const int64_t chunks = hd * (e8 ? 1 : lz_esize(cache_dtype)) / 16, threads = layers * 2 * KV * chunks;
  LZ_REQUIRE(threads <= (int64_t)UINT32_MAX - 255, "lz_kv_keep: too many heads");
  KeepArgs a{k, v, (int8_t*)k_exp, (int8_t*)v_exp, slots, row_start, kept, counts, ldk, pages * page_size,
             (int)rows, (int)layers, (int)KV, lz_log2(page_size), (int)nodes};
  const dim3 grid((uint32_t)lz_cdiv(threads, 256), (uint32_t)B);
  if (e8) kv_keep_kernel<true><<<grid, 256, 0, lz_stream(stream)>>>(a, (int)chunks);
  else kv_keep_kernel<false><<<grid, 256, 0, lz_stream(stream)>>>(a, (int)chunks);
  return lz_check_launch("lz_kv_keep");
}


LZ_EXPORT int lz_kv_read(const void* k, const void* v, const void* k_exp, const void* v_exp, int cache_dtype,
                         int64_t pages, int64_t page_size, const int32_t* table, int64_t width, const int32_t* start,
                         int64_t B, int64_t KV, int64_t hd, void* k_out, void* v_out, int dtype, int64_t rows,
                         void* stream) {
  if (int rc = lz_check_pages("lz_kv_read", k, v, k_exp, v_exp, cache_dtype, dtype, pages, page_size, table, width, B, KV,
                           hd))
    return rc;
  LZ_REQUIRE(rows >= 0 && rows <= INT32_MAX, "lz_kv_read: bad shape");
  LZ_REQUIRE(rows == 0 || (start && k_out && v_out && lz_aligned16(k_out) && lz_aligned16(v_out)),
             "lz_kv_read: outputs must be 16-byte aligned");
  if (rows == 0) return LZ_OK;
  const int64_t threads = rows * KV * (hd * lz_esize(dtype) / 16);
  LZ_REQUIRE(threads <= (int64_t)UINT32_MAX - 255, "lz_kv_read: too many rows");
  ReadArgs a{k, v, (const int8_t*)k_exp, (const int8_t*)v_exp,
             LzPages{table, (int)width, (int)pages, lz_log2(page_size)}, start, k_out, v_out, (int)rows, (int)B, (int)KV};
  const uint32_t grid = (uint32_t)lz_cdiv(threads, 256);
#define RUN(T, HD, E8) kv_read_kernel<T, HD, E8><<<grid, 256, 0, lz_stream(stream)>>>(a)
  LZ_CACHE_CASES(dtype, cache_dtype, hd, RUN);
#undef RUN
  return lz_check_launch("lz_kv_read");
}

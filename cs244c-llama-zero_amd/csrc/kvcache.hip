// Writing a paged key/value cache and reading it back.
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
};

// One thread per (row, head, 16 bytes of its lower half and the same of its
// upper half): a head is HD / 2 / N neighbouring lanes.
template <typename T, int HD, bool k8>
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
  const int pos = base + row;
  const bool there = pos >= 0 && pos < a.positions;
  if (head < a.H + a.KV) {
    if (there) {
      const T* cp = static_cast<const T*>(a.cos) + (int64_t)pos * HD + i;
      const T* sp = static_cast<const T*>(a.sin) + (int64_t)pos * HD + i;
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

LZ_EXPORT int lz_kv_write(const void* qkv, int64_t ld, int dtype, int64_t rows, const void* cos_t, const void* sin_t,
                          int64_t positions, void* q_out, int64_t ldq, void* k, void* v, void* k_exp, void* v_exp,
                          int cache_dtype, int64_t pages, int64_t page_size, const int32_t* table, int64_t width,
                          const int32_t* row_start, const int32_t* kv_len, int64_t B, int64_t H, int64_t KV, int64_t hd,
                          void* stream) {
  if (int rc = lz_check_pages("lz_kv_write", k, v, k_exp, v_exp, cache_dtype, dtype, pages, page_size, table, width, B, KV,
                           hd))
    return rc;
  const int esz = lz_esize(dtype);
  LZ_REQUIRE(rows >= 0 && rows <= INT32_MAX && H > 0 && H <= 65536 && positions > 0 && positions <= INT32_MAX,
             "lz_kv_write: bad shape");
  LZ_REQUIRE(ld >= (H + 2 * KV) * hd && ldq >= H * hd, "lz_kv_write: row strides shorter than the rows");
  LZ_REQUIRE(rows == 0 || (qkv && q_out && cos_t && sin_t && row_start && kv_len && lz_aligned16(qkv) &&
                           lz_aligned16(q_out) && lz_aligned16(cos_t) && lz_aligned16(sin_t) && ld * esz % 16 == 0 &&
                           ldq * esz % 16 == 0),
             "lz_kv_write: rows and tables must be 16-byte aligned");
  if (rows == 0) return LZ_OK;
  const int64_t threads = rows * (H + 2 * KV) * (hd * esz / 32);
  LZ_REQUIRE(threads <= (int64_t)UINT32_MAX - 255, "lz_kv_write: too many rows");
  WriteArgs a{qkv, ld, cos_t, sin_t, q_out, ldq, k, v, (int8_t*)k_exp, (int8_t*)v_exp,
              LzPages{table, (int)width, (int)pages, lz_log2(page_size)}, row_start, kv_len,
              (int)rows, (int)positions, (int)B, (int)H, (int)KV};
  const uint32_t grid = (uint32_t)lz_cdiv(threads, 256);
#define RUN(T, HD, E8) kv_write_kernel<T, HD, E8><<<grid, 256, 0, lz_stream(stream)>>>(a)
  LZ_CACHE_CASES(dtype, cache_dtype, hd, RUN);
#undef RUN
  return lz_check_launch("lz_kv_write");
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

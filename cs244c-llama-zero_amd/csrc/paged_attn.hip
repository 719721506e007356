// Attention of new tokens over a paged key/value cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  j <= kv_len - new + i
//
// for the i-th of a sequence's `new` last tokens, whose keys and values are in
// the cache already.  One wave per (row, head): its lanes take a key each for
// the scores and a few columns each for the sum.
#include <algorithm>

#include "kvcache.h"

namespace {

struct PagedArgs {
  const void* q;
  int64_t ldq;
  const void* k;
  const void* v;
  const int8_t* k_exp;
  const int8_t* v_exp;
  LzPages pg;
  const int32_t* row_start;
  const int32_t* kv_len;
  void* o;
  int64_t ldo;
  float scale;
  int rows, B, H, KV;
};

template <typename T, bool k8>
__device__ __forceinline__ float cache_elem(const void* p, int64_t i, float unit) {
  if constexpr (k8) return __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t*>(p)[i], 0) * unit;
  else return Elem<T>::load(static_cast<const T*>(p), i);
}

template <typename T, int HD, bool k8>
__global__ void __launch_bounds__(64) paged_attn_row_kernel(PagedArgs a) {
  const int row = blockIdx.x / a.H, h = blockIdx.x % a.H, lane = threadIdx.x;
  const int g = h / (a.H / a.KV);
  const int b = lz_seq_of_row(a.row_start, a.B, a.rows, row);
  if (b < 0) return;
  const int n_keys = min(a.kv_len[b] - a.row_start[b + 1] + row + 1, a.pg.width << a.pg.log_size);
  const T* q = static_cast<const T*>(a.q) + row * a.ldq + (int64_t)h * HD;
  constexpr int C = HD / 32;  // columns of lane l % 32: keys of the two halves of the wave meet at the end
  float acc[C] = {}, m = -INFINITY, l = 0.f;
  for (int j0 = 0; j0 < n_keys; j0 += 64) {
    const int j = j0 + lane;
    const int page = j < n_keys ? a.pg.page_of(b, j) : -1;
    const int64_t tok = (((int64_t)page * a.KV + g) << a.pg.log_size) + (j & ((1 << a.pg.log_size) - 1));
    float s = -INFINITY;
    if (page >= 0) {
      const float unit = k8 ? lz_pow2(a.k_exp[tok]) : 1.f;
      s = 0.f;
      for (int d = 0; d < HD; ++d) s = fmaf(Elem<T>::load(q, d), cache_elem<T, k8>(a.k, tok * HD + d, unit), s);
      s *= a.scale;
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float alpha = m_new == m ? 1.f : expf(m - m_new);
    const float p = page >= 0 ? expf(s - m_new) : 0.f;
    l = l * alpha + wave_sum(p);
    m = m_new;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] *= alpha;
    for (int t = 0; t < 64; t += 2) {
      const int from = t + (lane >> 5);
      const float pt = __shfl(p, from, 64);
      const int pgt = __shfl(page, from, 64);
      const int jt = j0 + from;
      if (pgt < 0) continue;
      const int64_t tt = (((int64_t)pgt * a.KV + g) << a.pg.log_size) + (jt & ((1 << a.pg.log_size) - 1));
      const float unit = k8 ? lz_pow2(a.v_exp[tt]) : 1.f;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = fmaf(pt, cache_elem<T, k8>(a.v, tt * HD + c * 32 + (lane & 31), unit), acc[c]);
    }
  }
  T* o = static_cast<T*>(a.o) + row * a.ldo + (int64_t)h * HD;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float x = acc[c] + __shfl_xor(acc[c], 32, 64);
    if (lane < 32) Elem<T>::store(o, c * 32 + lane, l == 0.f ? 0.f : x / l);
  }
}

}  // namespace

LZ_EXPORT int64_t lz_paged_attn_workspace(int, int, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) {
  return 0;
}

LZ_EXPORT int lz_paged_attn(const void* q, int64_t ldq, int dtype, int64_t rows, const void* k, const void* v,
                            const void* k_exp, const void* v_exp, int cache_dtype, int64_t pages, int64_t page_size,
                            const int32_t* table, int64_t width, const int32_t* row_start, const int32_t* kv_len,
                            int64_t B, int64_t H, int64_t KV, int64_t hd, int64_t max_new, int64_t max_len, float scale,
                            void* o, int64_t ldo, void* workspace, int64_t ws_bytes, void* stream) {
  if (int rc = lz_check_pages("lz_paged_attn", k, v, k_exp, v_exp, cache_dtype, dtype, pages, page_size, table, width, B,
                              KV, hd))
    return rc;
  const int esz = lz_esize(dtype);
  LZ_REQUIRE(H > 0 && H % KV == 0 && H <= 65536 && rows >= 0 && rows * H <= INT32_MAX / 64 && max_new >= 0 && max_len >= 0,
             "lz_paged_attn: bad shape");
  LZ_REQUIRE(ldq >= H * hd && ldo >= H * hd, "lz_paged_attn: row strides shorter than the rows");
  LZ_REQUIRE(rows == 0 || (q && o && row_start && kv_len && lz_aligned16(q) && lz_aligned16(o) && ldq * esz % 16 == 0 &&
                           ldo * esz % 16 == 0),
             "lz_paged_attn: rows must be 16-byte aligned");
  if (rows == 0) return LZ_OK;
  PagedArgs a{q, ldq, k, v, (const int8_t*)k_exp, (const int8_t*)v_exp,
              LzPages{table, (int)width, (int)pages, lz_log2(page_size)}, row_start, kv_len, o, ldo, scale,
              (int)rows, (int)B, (int)H, (int)KV};
  const uint32_t grid = (uint32_t)(rows * H);
#define RUN(T, HD, E8) paged_attn_row_kernel<T, HD, E8><<<grid, 64, 0, lz_stream(stream)>>>(a)
  LZ_CACHE_CASES(dtype, cache_dtype, hd, RUN);
#undef RUN
  return lz_check_launch("lz_paged_attn");
}

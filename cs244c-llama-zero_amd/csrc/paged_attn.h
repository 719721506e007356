// What the kernels of attention over a paged cache share.
#pragma once
#include "attn_tiles.h"
#include "kvcache.h"

// Packed rows: the `new` tokens of a sequence times the G = H / KV query heads
// of one kv head are one list of new * G rows, row m = token m / G, head m % G
// of the group, so that one pass over a kv head's keys and values serves all
// of them.  A block of rows goes over the keys in up to nsplit parts of
// `chunk` keys (a multiple of 64); parts of one block meet in the workspace.
struct LzPagedArgs {
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
  float* part;  // [rows * H][nsplit][hd], then [rows * H][nsplit][2]: maximum and sum
  float scale;
  int rows, B, H, KV, nqb, nsplit, chunk;
  int most;  // packed rows of a sequence that the grid is for; those behind them are left
};

// paged_tile.hip: 16-bit rows in blocks of kPagedTileRows; `groups`
// (1 or 2) of its waves share a block's keys.  LZ_OK or a status.
constexpr int kPagedTileRows = 128;
int lz_paged_tile(const LzPagedArgs& a, int dtype, bool e4m3, int64_t hd, int groups, uint32_t blocks, hipStream_t stream);

namespace {

typedef LzPagedArgs PagedArgs;

// A workgroup's place.  With kv heads for the eight XCDs the blocks of one
// (sequence, kv head) pair go to one of them, so that the keys and values its
// row blocks share are fetched into one L2.  With fewer heads that would leave a
// long sequence to some of the XCDs: its blocks go round all of them (4 x up to
// 188 new tokens over up to 8979 in fp32, 2 heads of 32: 66 us, on two XCDs
// 115; where the pairs are many it can lose: single tokens of 4 x up to 5720, 18/6
// heads of 64, 13.2 and 12.2).
struct PagedPlace {
  int b, g, qb, split;
  __device__ __forceinline__ PagedPlace(const PagedArgs& a, uint32_t bid) {
    const uint32_t pairs = (uint32_t)(a.B * a.KV);
    const uint32_t rest = bid / pairs, pair = (bid + (a.KV % 8 ? rest : 0)) % pairs;
    b = (int)(pair / (uint32_t)a.KV);
    g = (int)(pair % (uint32_t)a.KV);
    split = (int)(rest / (uint32_t)a.nqb);
    qb = a.nqb - 1 - (int)(rest % (uint32_t)a.nqb);  // the blocks with the most keys first
  }
};

// Rows m0 .. m0 + BM - 1 of a pair's packed rows and the keys that they see:
// row m's are 0 .. sees(m) - 1.
struct PagedRows {
  int m0, count;  // count: rows of the pair that are computed
  int row0, base, G, cap;
  __host__ __device__ __forceinline__ PagedRows(const PagedArgs& a, int b, int m0_)
      : PagedRows(a, a.row_start[b], a.row_start[b + 1], a.kv_len[b], m0_) {}
  // of a sequence whose rows are lo .. hi - 1, len tokens long
  __host__ __device__ __forceinline__ PagedRows(const PagedArgs& a, int lo, int hi, int len, int m0_) {
    m0 = m0_;
    G = a.H / a.KV;
    base = (int)((uint32_t)len - (uint32_t)hi + 1u);  // keys that row r of q sees: base + r
    row0 = min(max(lo, 0), a.rows);  // both ends inside the call before the product
    count = min((min(max(hi, row0), a.rows) - row0) * G, a.most);
    cap = a.pg.width << a.pg.log_size;
  }
  __host__ __device__ __forceinline__ int row(int m) const { return row0 + m / G; }
  __host__ __device__ __forceinline__ int sees(int m) const { return min(max((int)((uint32_t)base + (uint32_t)row(m)), 0), cap); }
  // the keys that the block's rows see together, and the parts they make
  __host__ __device__ __forceinline__ int keys(int bm) const { return sees(min(m0 + bm, count) - 1); }
  static __host__ __device__ __forceinline__ int parts(const PagedArgs& a, int keys) {
    return min(max((int)(((uint32_t)keys + (uint32_t)a.chunk - 1) / (uint32_t)a.chunk), 1), a.nsplit);
  }
};

// Whether a row that sees `sees` keys sees one of k_lo .. k_hi - 1 (of pages
// that there are).  A maximum of -inf says that it does not or that all its
// scores are -inf: the former's output is zeros, the latter's NaN (0 / 0).  The
// latter's maximum is kept as kAllInf, beside which any finite score takes all
// the weight.
constexpr float kAllInf = -3.402823466e38f;
__host__ __device__ __forceinline__ bool sees_any(const PagedArgs& a, int b, int k_lo, int k_hi, int sees) {
  for (int key = k_lo; key < min(k_hi, sees); key = ((key >> a.pg.log_size) + 1) << a.pg.log_size)  // a page at a time
    if (a.pg.page_of(b, key) >= 0) return true;
  return false;
}

// A row's reference m for its weights 2^(s - m) (log2 units) is its running
// maximum, but moves only when that is more than kSlack above it: weights up to
// 2^8 are as exact in 16 and 32 bits as those up to 1, and the sums are
// multiplied down once or twice in a pass and not at every new maximum (2 x up
// to 1024 new tokens over up to 8192, 32/8 heads of 128, one wave group a block:
// 208 and 218 us).
constexpr float kSlack = 8.f;

// Two fp32 weights of the second product as N packed terms of the 16-bit format
// F, largest first.  Rounded to F once they would cost as much as the output's
// own rounding (1.1 to 1.4 times the error against float64); so:
//   paged_wave_kernel, bf16: three terms of eight significant bits, cut and not
//     rounded, so that each remainder is exact and the three add up to the
//     weight.  It is bound by memory: 16 x up to 4096 tokens, 32/8 heads of 128,
//     31.0 us, with one rounded term 30.5; 8 x up to 15 new over 4096 46, 38.
//   paged_tile_kernel, bf16: the cut weight and the rounded rest, off by 2^-16 of
//     the weight at most.  It is bound by the matrix cores: 2 x up to 1024 new
//     over up to 8192, 32/8 heads of 128, 199 us, with one term 155, three 244.
//   fp16: the cut weight and the rounded rest, off by 2^-22 at most.  The weights
//     are formed 2^7 times as large (kLift, in log2 units; so is their sum): up to
//     2^15, and what the smallest subnormal cuts off is 2^-32 of the reference.
template <typename F>
constexpr float kLift = F::kDtype == LZ_F16 ? 7.f : 0.f;
template <typename F, int N>
__device__ __forceinline__ void weight_terms(uint32_t (&w)[N], float a, float b) {
  if constexpr (F::kDtype == LZ_F16) {
    static_assert(N == 2);
    const auto cut = __builtin_amdgcn_cvt_pkrtz(a, b);
    w[0] = __builtin_bit_cast(uint32_t, cut);
    w[1] = F::pack2(a - (float)cut[0], b - (float)cut[1]);
  } else {
#pragma unroll
    for (int t = 0; t < N; ++t) {
      if (t == 1 && N == 2) {
        w[t] = F::pack2(a, b);
        break;
      }
      const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
      w[t] = __builtin_amdgcn_perm(y, x, 0x07060302u);
      a -= __uint_as_float(x & 0xffff0000u);
      b -= __uint_as_float(y & 0xffff0000u);
    }
  }
}
// Four pairs: the operand words of N MFMAs.
template <typename F, int N, typename Pair>
__device__ __forceinline__ void weight_words(uint4 (&w)[N], const Pair& pair) {
  uint32_t y[4][N];
#pragma unroll
  for (int e = 0; e < 4; ++e) weight_terms<F, N>(y[e], pair(2 * e), pair(2 * e + 1));
#pragma unroll
  for (int t = 0; t < N; ++t) w[t] = make_uint4(y[0][t], y[1][t], y[2][t], y[3][t]);
}

// Two e4m3 values of a word, times 2^e (exact in bf16, and in fp16 for what
// lz_kv_write stores of fp16 rows), as two values of the 16-bit format F.
template <typename F, bool kHi>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, float unit) {
  if constexpr (F::kDtype == LZ_F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, unit, kHi));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, unit, kHi));
}

template <int BYTES>
__device__ __forceinline__ void load_words(uint32_t* w, const void* p) {
  if constexpr (BYTES == 2) {
    w[0] = *static_cast<const uint16_t*>(p);
  } else if constexpr (BYTES == 4) {
    w[0] = *static_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 8) {
    const uint2 x = *static_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 x = static_cast<const uint4*>(p)[i];
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  }
}

// Whether a word of two 16-bit values of the format F, or an fp32 word, holds
// an infinity or NaN.
template <typename F>
__device__ __forceinline__ bool nonfinite16(uint32_t w) {
  constexpr uint32_t kExp = F::kDtype == LZ_F16 ? 0x7c00u : 0x7f80u;
  return (w & kExp) == kExp || ((w >> 16) & kExp) == kExp;
}
__device__ __forceinline__ bool nonfinite32(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u; }

}  // namespace

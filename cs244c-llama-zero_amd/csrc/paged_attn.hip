// Attention of new tokens over a paged key/value cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  j <= kv_len - new + i
//
// for the i-th of a sequence's `new` last tokens, whose keys and values are in
// the cache already; or, for a tree of drafted tokens, j < base and those j after
// them whose bits are set in row i's mask.  One pass over the keys with a running maximum and sum:
// per tile, S^T = K . Q^T, so that a lane owns one row's column and the
// probabilities are the B operand of O^T += V^T . P^T as they stand.
//
// paged_wave_kernel: few rows (a decoded token's heads, short chunks) and
// fp32.  Bound by the one read of K and V, so nothing is staged: a wave loads
// its own 32-key tiles (16 in fp32) straight into the operand registers, the
// next tile's while this one is computed, and the four waves of a workgroup
// take every fourth tile and meet in LDS once.  The contraction order of both
// products is free, so each lane loads 16 adjacent bytes wherever rows allow:
// of K it takes the pieces (4 j + lane / 16) of its key's row; of V it takes
// HD / 16 adjacent columns of eight keys and swaps rows and columns of that
// 8 x (HD / 16) block in registers (v_perm).
#include <algorithm>
#include <cmath>
#include <limits>

#include "paged_attn.h"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <typename T>
struct FmtOf;
template <>
struct FmtOf<uint16_t> {
  typedef FmtBF16 F;
};
template <>
struct FmtOf<_Float16> {
  typedef FmtF16 F;
};
template <>
struct FmtOf<float> {
  typedef FmtBF16 F;  // not used
};

template <typename F>
__device__ __forceinline__ f32x4_t mfma32(const uint4& a, const uint4& b, const f32x4_t& c) {
  if constexpr (F::kDtype == LZ_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

template <typename T, int HD, bool k8, int NQ>
struct Wave {
  static constexpr bool kWide = sizeof(T) == 4;  // fp32 rows
  typedef typename FmtOf<T>::F F;
  static constexpr int kEsz = k8 ? 1 : sizeof(T);      // bytes of a cached element
  static constexpr int NT = kWide ? 1 : 2;             // 16-key tiles at a time
  static constexpr int KT = 16 * NT;
  static constexpr int CE = HD / 4 < 16 / kEsz ? HD / 4 : 16 / kEsz;  // elements of a K piece
  static constexpr int NL = HD / 4 / CE, KW = CE * kEsz / 4;          // pieces of a lane, words of a piece
  static constexpr int VE = HD / 16, VB = VE * kEsz, VW = (VB + 3) / 4;  // columns, bytes and words of a lane's V
  static constexpr int NS = kWide ? HD / 4 : HD / 32;  // contraction steps of a score
  static constexpr int kTerms = F::kDtype == LZ_F16 ? 2 : 3;  // of a weight (16-bit rows)

  uint32_t k[NT][NL][KW];
  uint32_t v[NT][4][VW];
  uint32_t kx[NT], vx[NT];  // exponents of keys 4 g .. 4 g + 3

  __device__ __forceinline__ void load_k(const PagedArgs& a, const int64_t (&tok)[NT], int c16, int g4) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (tok[t] < 0) continue;  // uniform; the scores are masked
      const char* p = static_cast<const char*>(a.k) + ((tok[t] + c16) * HD + g4 * CE) * kEsz;
#pragma unroll
      for (int j = 0; j < NL; ++j) load_words<CE * kEsz>(k[t][j], p + j * 4 * CE * kEsz);
      if constexpr (k8) kx[t] = *reinterpret_cast<const uint32_t*>(a.k_exp + tok[t] + 4 * g4);
    }
  }
  __device__ __forceinline__ void load_v(const PagedArgs& a, const int64_t (&tok)[NT], int c16, int g4) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (tok[t] < 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < VW; ++w) v[t][i][w] = 0;
        if constexpr (k8) vx[t] = 0;
        continue;
      }
      const char* p = static_cast<const char*>(a.v) + ((tok[t] + 4 * g4) * HD + c16 * VE) * kEsz;
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<VB>(v[t][i], p + i * HD * kEsz);
      if constexpr (k8) vx[t] = *reinterpret_cast<const uint32_t*>(a.v_exp + tok[t] + 4 * g4);
    }
  }

  static __device__ __forceinline__ float unit(uint32_t x, int i) { return lz_pow2((int8_t)(x >> (8 * i))); }

  struct Query {
    uint4 h[kWide ? 1 : NS];
    float f[kWide ? NS : 1];
    __device__ __forceinline__ void load(const T* row, int g4) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        if constexpr (kWide) f[s] = row[((s / CE) * 4 + g4) * CE + s % CE];
        else h[s] = *reinterpret_cast<const uint4*>(row + ((8 * s / CE) * 4 + g4) * CE + 8 * s % CE);
      }
    }
  };

  // scores of the tile's keys 16 t + 4 g + i, unscaled but for e4m3's exponents
  __device__ __forceinline__ void scores(f32x4_t (&s)[NT], const Query& q) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        if constexpr (kWide) {
          float x;
          if constexpr (k8) x = e4m3_at(k[t][st / CE], st % CE);
          else x = __uint_as_float(k[t][st / CE][st % CE]);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, q.f[st], s[t], 0, 0, 0);
        } else {
          uint4 x;
          if constexpr (k8) {
            const uint32_t* w = k[t][8 * st / CE] + (8 * st % CE) / 4;
            x = make_uint4(e4m3_pair<F, false>(w[0], 1.f), e4m3_pair<F, true>(w[0], 1.f), e4m3_pair<F, false>(w[1], 1.f),
                           e4m3_pair<F, true>(w[1], 1.f));
          } else {
            x = make_uint4(k[t][st][0], k[t][st][1], k[t][st][2], k[t][st][3]);
          }
          s[t] = mfma32<F>(x, q.h[st], s[t]);
        }
      }
      if constexpr (k8)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] *= unit(kx[t], i);
    }
  }

  static __device__ __forceinline__ float e4m3_at(const uint32_t* w, int i) {
    switch (i & 3) {
      case 0: return __builtin_amdgcn_cvt_f32_fp8((int)w[i >> 2], 0);
      case 1: return __builtin_amdgcn_cvt_f32_fp8((int)w[i >> 2], 1);
      case 2: return __builtin_amdgcn_cvt_f32_fp8((int)w[i >> 2], 2);
      default: return __builtin_amdgcn_cvt_f32_fp8((int)w[i >> 2], 3);
    }
  }

  // The tile's V as operand words: 16-bit pairs of columns, or floats.
  struct Value {
    static constexpr int N = kWide ? VE : VE / 2;
    uint32_t w[NT][4][N];
  };
  __device__ __forceinline__ void widen(Value& x) const {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < Value::N; ++n) {
          if constexpr (!k8) x.w[t][i][n] = v[t][i][n];
          else if constexpr (kWide) x.w[t][i][n] = __float_as_uint(e4m3_at(v[t][i], n) * unit(vx[t], i));
          else x.w[t][i][n] = n & 1 ? e4m3_pair<F, true>(v[t][i][n >> 1], unit(vx[t], i)) : e4m3_pair<F, false>(v[t][i][n >> 1], unit(vx[t], i));
        }
  }

  // O^T += V^T . P^T.  acc[j]: columns (4 g + i) * VE + j of the lane's row.
  static __device__ __forceinline__ void pv(f32x4_t (&acc)[NQ][VE], const Value& x, const f32x4_t (&p)[NQ][NT]) {
    if constexpr (kWide) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < VE; ++j)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              acc[n][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.w[t][i][j]), p[n][t][i], acc[n][j], 0, 0, 0);
    } else {
      uint4 pb[NQ][kTerms];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
        weight_words<F>(pb[n], [&](int e) { return p[n][e >> 2][e & 3]; });
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = __builtin_amdgcn_perm(x.w[e >> 1][2 * (e & 1) + 1][j >> 1], x.w[e >> 1][2 * (e & 1)][j >> 1], sel);
        const uint4 v = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int t = kTerms - 1; t >= 0; --t) acc[n][j] = mfma32<F>(v, pb[n][t], acc[n][j]);  // the smallest first
      }
    }
  }

  // One value of V, as fp32.
  static __device__ __forceinline__ float v_elem(const PagedArgs& a, int64_t tok, int d) {
    if constexpr (k8) return __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t*>(a.v)[tok * HD + d], 0) * lz_pow2(a.v_exp[tok]);
    else return Elem<T>::load(static_cast<const T*>(a.v), tok * HD + d);
  }
};

template <typename T>
__device__ __forceinline__ float exp_of(float d) {
  if constexpr (sizeof(T) == 4) return exp_accurate(d);
  else return __builtin_amdgcn_exp2f(d);
}

// The maximum over the four lanes that hold a row's scores.
__device__ __forceinline__ float max_of_row(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_of_row(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

template <typename T, int HD>
__device__ __forceinline__ void store_row4(const PagedArgs& a, int row, int head, int d, const float4& x) {
  T* o = static_cast<T*>(a.o) + (int64_t)row * a.ldo + head * HD + d;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(o) = x;
  } else {
    typedef typename FmtOf<T>::F F;
    *reinterpret_cast<uint2*>(o) = make_uint2(F::pack2(x.x, x.y), F::pack2(x.z, x.w));
  }
}

// Rows: PagedRows, or (fp32) TreeRows, whose tiles from the first key that not all rows
// see on take each row's bits of its mask.
template <typename T, int HD, bool k8, int NQ, typename Rows>
__global__ void __launch_bounds__(256, 2) paged_wave_kernel(PagedArgs a) {
  constexpr bool kTree = std::is_same<Rows, TreeRows>::value;
  typedef Wave<T, HD, k8, NQ> W;
  constexpr int BM = 16 * NQ, KT = W::KT, NT = W::NT, VE = W::VE;
  constexpr int RS = HD + 4;  // floats of a parked row
  __shared__ __attribute__((aligned(16))) float park[4 * BM * RS];
  __shared__ float ml[4][BM][2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g4 = lane >> 4;
  const PagedPlace at(a, blockIdx.x);
  const int k_lo = at.split * a.chunk;
  // This wave's 16-key tiles: number x is at key k_lo + (x / NT * 4 + wave) *
  // KT + 16 * (x % NT).  Their pages are looked up 64 at a time, one a lane, the
  // first beside the sequence's length.
  auto key_of = [&](int x) { return k_lo + ((x / NT) * 4 + wave) * KT + 16 * (x % NT); };
  const int first_ids = a.pg.page_of(at.b, key_of(lane));

  const Rows rw(a, at.b, at.qb * BM);
  if (rw.m0 >= rw.count) return;
  const int n_keys = rw.keys(BM), n_parts = PagedRows::parts(a, n_keys);
  if (at.split >= n_parts) return;
  const int k_hi = at.split + 1 == n_parts ? n_keys : k_lo + a.chunk;

  typename W::Query q[NQ];
  int sees[NQ];
  const uint32_t* mask[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int m = min(rw.m0 + 16 * n + c16, rw.count - 1);  // rows past the last repeat it and are not stored
    sees[n] = rw.sees(m);
    if constexpr (kTree) mask[n] = a.mask + (int64_t)rw.row(m) * a.words;
    q[n].load(static_cast<const T*>(a.q) + (int64_t)rw.row(m) * a.ldq + (at.g * rw.G + m % rw.G) * HD, g4);
  }
  const int all_see = rw.all(rw.m0);  // keys that every row of the block sees

  f32x4_t acc[NQ][VE];
  float mx[NQ], sum[NQ];
  const float unit = sizeof(T) == 4 ? a.scale : a.scale * kLog2e;
  constexpr float lift = sizeof(T) == 4 ? 0.f : kLift<typename W::F>;

  int ids, ids_from;
  const int size_mask = (1 << a.pg.log_size) - 1;
  auto tokens = [&](int64_t (&tok)[NT], int tile) {
    const int x = tile * NT;
    if (x - ids_from >= 64) {
      ids_from = x;
      const int key = key_of(x + lane);
      ids = key < k_hi ? a.pg.page_of(at.b, key) : -1;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int id = __builtin_amdgcn_readlane(ids, x + t - ids_from);
      tok[t] = id < 0 ? -1 : (((int64_t)id * a.KV + at.g) << a.pg.log_size) + (key_of(x + t) & size_mask);
    }
  };

  W w;
  int64_t tok[NT], next[NT];
  const int n_tiles = max(0, (k_hi - k_lo - wave * KT + 4 * KT - 1) / (4 * KT));
  // An infinity of V that all rows see multiplies a weight's terms one by one: a
  // zero among them would make it NaN.  Where a sum is not finite the pass is
  // made again with such values out of the product, as in tiles with holes; the
  // others get the same bits.
  for (bool odd_pass = false;; odd_pass = true) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      mx[n] = -INFINITY;
      sum[n] = 0.f;
#pragma unroll
      for (int j = 0; j < VE; ++j) acc[n][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    ids = key_of(lane) < k_hi ? first_ids : -1;
    ids_from = 0;
    if (n_tiles > 0) {
      tokens(tok, 0);
      w.load_k(a, tok, c16, g4);
      w.load_v(a, tok, c16, g4);
    }
    for (int tile = 0; tile < n_tiles; ++tile) {
      const int key0 = key_of(tile * NT);
      const bool more = tile + 1 < n_tiles;
      f32x4_t s[NQ][NT];
#pragma unroll
      for (int n = 0; n < NQ; ++n) w.scores(s[n], q[n]);
      if (more) {
        tokens(next, tile + 1);
        w.load_k(a, next, c16, g4);
      }
      bool holes = odd_pass || key0 + KT > all_see;
#pragma unroll
      for (int t = 0; t < NT; ++t) holes |= tok[t] < 0;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        if (holes) {
          uint32_t bits = 0;
          if constexpr (kTree) bits = tree_bits(mask[n], a.words, key0 - all_see) >> (4 * g4);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (tok[t] < 0 || key0 + 16 * t + 4 * g4 + i >= sees[n] || (kTree && !((bits >> (16 * t + i)) & 1)))
                s[n][t][i] = -INFINITY;
        }
        float top = s[n][0][0];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][t][i]);
        top = max_of_row(top) * unit;
        const bool moved = top > mx[n] + (sizeof(T) == 4 ? 0.f : kSlack);
        if (__ballot(moved)) {
          const float m_new = moved ? top : mx[n];
          const float alpha = moved ? exp_of<T>(mx[n] - m_new) : 1.f;
          mx[n] = m_new;
          sum[n] *= alpha;
#pragma unroll
          for (int j = 0; j < VE; ++j) acc[n][j] *= alpha;
        }
        const float m0 = mx[n] == -INFINITY ? 0.f : mx[n];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = exp_of<T>(fmaf(s[n][t][i], unit, lift - m0));
            s[n][t][i] = p;
            sum[n] += p;
          }
      }
      typename W::Value x;
      w.widen(x);
      bool odd = false;
      if (holes) {
        // slots past the sequence hold anything: out, before they meet a zero
        // weight.  An infinity or NaN that only some of the rows see is taken
        // out too and added to those rows below.
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool there = key0 + 16 * t + 4 * g4 + i < n_keys;
#pragma unroll
            for (int e = 0; e < W::Value::N; ++e) {
              uint32_t& y = x.w[t][i][e];
              if (!there) y = 0;
              if constexpr (W::kWide) {
                if (nonfinite32(y)) {
                  y = 0;
                  odd = true;
                }
              } else if (nonfinite16<typename W::F>(y)) {
                if (nonfinite16<typename W::F>(y & 0xffffu)) y &= 0xffff0000u;
                if (nonfinite16<typename W::F>(y & 0xffff0000u)) y &= 0xffffu;
                odd = true;
              }
            }
          }
        odd = __ballot(odd) != 0;
      }
      if (more) w.load_v(a, next, c16, g4);
      W::pv(acc, x, s);
      if (odd) {
#pragma unroll 1
        for (int kk = 0; kk < KT; ++kk) {
          const int64_t tk = tok[kk / 16] + kk % 16;
          if (tok[kk / 16] < 0 || key0 + kk >= n_keys) continue;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float p = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i) p = kk / 16 == t && kk % 4 == i ? s[n][t][i] : p;
            p = __shfl(p, c16 + 16 * (kk % 16 / 4), 64);
            bool seen = key0 + kk < sees[n];
            if constexpr (kTree) seen = seen && (tree_bits(mask[n], a.words, key0 + kk - all_see) & 1);
            if (seen) {
#pragma unroll
              for (int j = 0; j < VE; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float y = W::v_elem(a, tk, (4 * g4 + i) * VE + j);
                  if (!(fabsf(y) < INFINITY)) acc[n][j][i] = fmaf(p, y, acc[n][j][i]);
                }
            }
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) tok[t] = next[t];
    }
    if (W::kWide || odd_pass) break;
    float zero = 0.f;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int j = 0; j < VE; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) zero = fmaf(acc[n][j][i], 0.f, zero);
    if (__ballot(zero != 0.f) == 0) break;  // NaN
  }

  // the four waves' parts, joined in a fixed order
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    sum[n] = sum_of_row(sum[n]);
    float* p = park + (wave * BM + 16 * n + c16) * RS;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) p[(4 * g4 + i) * VE + j] = acc[n][j][i];
    if (g4 == 0) {
      ml[wave][16 * n + c16][0] = mx[n];
      ml[wave][16 * n + c16][1] = sum[n];
    }
  }
  __syncthreads();
  for (int e = tid; e < BM * (HD / 4); e += 256) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4, m = rw.m0 + r;
    if (m >= rw.count) break;
    float top = ml[0][r][0];
#pragma unroll
    for (int i = 1; i < 4; ++i) top = fmaxf(top, ml[i][r][0]);
    float l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ml[i][r][0] == -INFINITY ? 0.f : exp_of<T>(ml[i][r][0] - top);
      const float4 z = *reinterpret_cast<const float4*>(park + (i * BM + r) * RS + d);
      if (f == 0.f && ml[i][r][1] == 0.f) continue;  // a wave that saw nothing
      l = fmaf(f, ml[i][r][1], l);
      y.x = fmaf(f, z.x, y.x);
      y.y = fmaf(f, z.y, y.y);
      y.z = fmaf(f, z.z, y.z);
      y.w = fmaf(f, z.w, y.w);
    }
    const int row = rw.row(m), head = at.g * rw.G + m % rw.G;
    if (top == -INFINITY && sees_any(a, at.b, k_lo, k_hi, rw, row, m)) top = kAllInf;
    if (n_parts == 1) {
      const float inv = top == -INFINITY ? 0.f : 1.f / l;
      store_row4<T, HD>(a, row, head, d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
    } else {
      const int64_t at_row = ((int64_t)row * a.H + head) * a.nsplit + at.split;
      *reinterpret_cast<float4*>(a.part + at_row * HD + d) = y;
      if (d == 0) {
        float* s2 = a.part + (int64_t)a.rows * a.H * a.nsplit * HD + at_row * 2;
        s2[0] = top;
        s2[1] = l;
      }
    }
  }
}

// The parts of rows that were split, joined: `per` groups of HD / 4 lanes for
// one (row, head), each with every per-th part, all loads of a thread
// independent; the groups meet in LDS in a fixed order.
template <typename T, int HD, typename Rows>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedArgs a, int bm, int per, int likely) {
  constexpr int kLanes = HD / 4;
  __shared__ float4 ys[256];
  __shared__ float ms[256], ls[256];
  const int tid = threadIdx.x, d = tid % kLanes * 4, grp = tid / kLanes % per, rows = 256 / (kLanes * per);
  const uint32_t rh = blockIdx.x * (uint32_t)rows + (uint32_t)(tid / (kLanes * per));
  const int row = (int)(rh / (uint32_t)a.H), head = (int)(rh % (uint32_t)a.H);
  const float* part = a.part + (int64_t)rh * a.nsplit * HD + d;
  const float* s2 = a.part + (int64_t)a.rows * a.H * a.nsplit * HD + (int64_t)rh * a.nsplit * 2;
  // A thread's first parts are fetched beside what says how many there are
  // (parts that were not written hold anything and are not used); of trees, whose
  // shares may leave few of nsplit parts, the `likely` ones, with two groups for
  // up to 12 and four for more (4 x 64 nodes over 32768, 32/8 heads of 128: 7.6 us,
  // with eight groups 12.5, with all of 33 parts 18.6).
  constexpr int kAhead = 4;
  float4 z[kAhead];
  float2 zs[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int i = grp + k * per;
    if (row < a.rows && i < (std::is_same<Rows, TreeRows>::value ? likely : a.nsplit)) {
      z[k] = *reinterpret_cast<const float4*>(part + (int64_t)i * HD);
      zs[k] = *reinterpret_cast<const float2*>(s2 + 2 * i);
    }
  }
  int n_parts = 0;
  if (row < a.rows) {
    // the guess that serves single tokens, with all that it needs in one round
    int b = (int)((int64_t)row * a.B / a.rows), lo = a.row_start[b], hi = a.row_start[b + 1], len = a.kv_len[b];
    if (row < lo || row >= hi) {
      b = lz_seq_of_row(a.row_start, a.B, a.rows, row);
      if (b >= 0) {
        lo = a.row_start[b];
        hi = a.row_start[b + 1];
        len = a.kv_len[b];
      }
    }
    if (b >= 0) {
      Rows rw = [&] {
        if constexpr (std::is_same<Rows, TreeRows>::value) return TreeRows(a, b, lo, hi, len, 0);
        else return PagedRows(a, lo, hi, len, 0);
      }();
      const int m = (row - rw.row0) * rw.G + head % rw.G;
      rw.m0 = m / bm * bm;
      if (m < rw.count) n_parts = PagedRows::parts(a, rw.keys(bm));
      if constexpr (std::is_same<Rows, TreeRows>::value)
        if (a.shares && m < rw.count) n_parts = a.parts[(int64_t)b * a.nqb + m / bm];
    }
  }
  if (n_parts == 1) n_parts = 0;  // was written whole
  if constexpr (std::is_same<Rows, TreeRows>::value)
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = grp + k * per;
      if (i >= likely && i < n_parts) {
        z[k] = *reinterpret_cast<const float4*>(part + (int64_t)i * HD);
        zs[k] = *reinterpret_cast<const float2*>(s2 + 2 * i);
      }
    }
  float top = -INFINITY, l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& v, const float2& t) {
    if (t.x == -INFINITY) return;  // saw nothing
    const float m_new = fmaxf(top, t.x);
    const float f = m_new == top ? 1.f : exp_of<T>(top - m_new), e = m_new == t.x ? 1.f : exp_of<T>(t.x - m_new);
    top = m_new;
    l = fmaf(l, f, e * t.y);
    y.x = fmaf(y.x, f, e * v.x);
    y.y = fmaf(y.y, f, e * v.y);
    y.z = fmaf(y.z, f, e * v.z);
    y.w = fmaf(y.w, f, e * v.w);
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (grp + k * per < n_parts) add(z[k], zs[k]);
#pragma unroll 4
  for (int i = grp + kAhead * per; i < n_parts; i += per)
    add(*reinterpret_cast<const float4*>(part + (int64_t)i * HD), *reinterpret_cast<const float2*>(s2 + 2 * i));
  if (per > 1) {
    ys[tid] = y;
    ms[tid] = top;
    ls[tid] = l;
    __syncthreads();
    if (grp != 0) return;
    for (int i = 1; i < per; ++i) top = fmaxf(top, ms[tid + i * kLanes]);
    l = 0.f;
    y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < per; ++i) {
      const int at = tid + i * kLanes;
      if (ms[at] == -INFINITY) continue;
      const float e = ms[at] == top ? 1.f : exp_of<T>(ms[at] - top);
      const float4 z = ys[at];
      l = fmaf(e, ls[at], l);
      y.x = fmaf(e, z.x, y.x);
      y.y = fmaf(e, z.y, y.y);
      y.z = fmaf(e, z.z, y.z);
      y.w = fmaf(e, z.w, y.w);
    }
  }
  if (n_parts == 0) return;
  const float inv = top == -INFINITY ? 0.f : 1.f / l;
  store_row4<T, HD>(a, row, head, d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
}

struct Plan {
  int bm;  // rows of a block: 16 or 32 (paged_wave_kernel) or kPagedTileRows
  int groups;  // of the tile kernel's waves
  int nqb, nsplit, chunk;
  int shares = 0, least = 0;  // tree_kernel
  int likely = 0;             // parts of most of its rows
  int waves = 4;              // tree_kernel, blocks of 32 rows
};

// Blocks of bm packed rows that have rows: not every sequence has max_new of them.
int64_t blocks_of(int64_t bm, int64_t packed, int64_t rows, int64_t B, int64_t KV, int64_t G) {
  return KV * std::min(B * lz_cdiv(packed, bm), std::min(B, rows) + rows * G / bm);
}

// Row blocks and parts.  Tiles of 128 rows where a sequence has 64 packed rows
// or more and the work is not little: at most 1.5 blocks of 32 rows a CU which
// go over at most 512 keys a CU, where the tile kernel's longer start and steps
// are the time (12/4 heads of 64: 3 prompts of up to 182 tokens 8.1 us, 9.6 in
// tiles; 4 of up to 400 16.3, 15.4 in tiles; 16 of up to 256 16 and 12).
// paged_wave_kernel: whole sequences where there is a block for every CU (32
// ragged sequences of up to 2048, 16/8 heads of 128: 34 us, in parts of 512
// keys 37), but four parts where some CUs would have one more than others and a
// third of the CUs' time would go by (36 of them: 42 us, whole 52; 58: 53 and
// 52; all 2048 long: 60 and 71 of 36, 93 and 84 of 58); fewer blocks than CUs:
// four workgroups a CU, so that lengths even out (16 of up to 4096, 32/8 heads:
// 27 us in eight parts, 33 in four), but two where that makes more than 16 parts
// to join (4 x 32768 in e4m3: 43 us in 16, 48 in 32), and parts of 512 keys at
// least, four of each wave's tiles (8 of up to 4096: 20 us, 23 in parts of 256;
// in e4m3 16.0, 19.2 and, in parts of 1024, 16.9), while every CU has one
// (1 x 8192: 13 us in 32, 19 in 8); short sequences whole, where the join costs
// more than their keys (1 x 512 over heads of 64: 6.7 us, 8.8 in parts; of 128:
// 8.8 and 9.3).  The tile kernel: one workgroup a CU, of two wave groups where
// that is all (1 x 512 new tokens over 4096: 64 us in two parts, 83 whole, 96
// whole with one group; in four parts, with one group, 65), and for up to a third
// more blocks where their keys are uneven, so that those of a second turn are
// short (a prompt of 2600, 16/8 heads: 58 us, 68 with one group; 3 chunks of 800
// over 4096 alike: 151 and 135); three parts of one group, two workgroups a CU,
// where a block each would leave a third of the CUs idle for long (1 x 600 over
// 8192, 32/8 heads: 125 us, whole 145; 1 x 1100 over 2200, 16/8 heads: 47 and 48;
// 1 x 700 over 3000, 32/8 heads, with blocks for two thirds: 76 and 62).
Plan make_plan(int dtype, int cache_dtype, int64_t rows, int64_t B, int64_t H, int64_t KV, int64_t hd, int64_t max_new,
               int64_t max_len) {
  Plan p;
  const int64_t G = H / KV, packed = std::max<int64_t>(1, std::min(max_new, rows)) * G, cus = lz_num_cus();
  const int64_t len = std::max<int64_t>(1, max_len), small = KV * lz_cdiv(rows * G, 32);
  const bool little = 2 * small <= 3 * cus && small * std::min<int64_t>(len, 1 << 20) <= 512 * cus;
  p.bm = packed <= 16 ? 16 : packed < 64 || little || dtype == LZ_F32 ? 32 : kPagedTileRows;
  p.nqb = (int)lz_cdiv(packed, p.bm);
  const int64_t blocks = blocks_of(p.bm, packed, rows, B, KV, G);
  const int64_t one = std::max<int64_t>(1, cus / blocks);
  int64_t chunk = lz_cdiv(len, one);
  if (p.bm != kPagedTileRows) {
    if (blocks < cus) {
      const int64_t even = lz_cdiv(len, std::min(4 * cus / blocks, std::max<int64_t>(16, 2 * cus / blocks)));
      chunk = std::max(even, std::min<int64_t>(512, chunk));
    } else if (3 * lz_cdiv(blocks, cus) * cus > 4 * blocks) {
      chunk = std::max<int64_t>(512, lz_cdiv(len, 4));
    }
    if (dtype != LZ_F32 && len <= (hd > 64 ? 512 : 768)) chunk = len;
  } else if (one == 1 && 3 * blocks <= 2 * cus && len >= 4096) {
    chunk = lz_cdiv(len, 3);
  }
  p.chunk = (int)std::max<int64_t>(256, lz_cdiv(chunk, 64) * 64);
  p.nsplit = (int)lz_cdiv(len, p.chunk);
  const bool uneven = len >= 1024 && (2 * max_new >= len || 10 * rows < 9 * B * std::min(max_new, rows));
  p.groups = blocks * p.nsplit <= cus || (uneven && 10 * blocks <= 13 * cus) ? 2 : 1;
  return p;
}

// Row blocks and shares of trees.  fp32: paged_wave_kernel, as above.  Else
// tree_kernel.  Up to a block a CU: a block's keys whole, by eight waves, up to a
// length that grows with the blocks, since shares cost their arithmetic and the
// join (16 bits, 32/8 heads of 128: 1 x 16 nodes over 2048 19 us whole, in shares
// 16, over 3000 26 and 17; 16 x 10 over 2048 21 and 27; 3 x 100 over 4096 33 and 48; 8 x
// 24 over 6000 55 and 43; 12/4 heads of 64 in e4m3: 1 x 16 over 1024 10.4 and 12.7);
// half as long where each block converts e4m3 heads of 128 by itself (2 x 40 over
// 2048: 28 and 23; 16 x 10 over 1024 24 and 36).  More blocks: shares where they are some sequences of uneven
// lengths (32 x 8 over up to 4096, e4m3: 60 us, whole 70) or a second turn would be
// nearly empty (2 x 160 over 8192: 74 us, whole 79, in e4m3 83 and 108; 4 x 140 over
// 6000: 63 and 61, 70 and 82).  Shares: two workgroups a CU, of 512 keys at least
// (1 x 16 over 8192 19 us, of 256: 22).
// Eight waves also for two blocks a CU of heads of 32 and 64, whose tiles leave
// room for a second workgroup (4 x 120 over 3000, 32/8 heads of 64: 23 us, four
// waves 26; of 128, 64 x 8 over 1024: 39 and 37), and not for texts of a tile or two a
// wave (1 x 8 over 128: 5.5 and 5.1).
// Blocks of 64 rows where a share is long and there are some for every eighth CU,
// and for e4m3 heads of 128, whose converted tiles two waves share (8 rows of 32
// sequences over up to 4096, 32/8 heads: 60 us, in blocks of 32 rows, whose bytes
// on the way spill, 72; 4 x 120 over 3000, 16/8 heads: 40 and 54; but 1 x 8 over
// 2500 22 and 20).
Plan make_tree_plan(int dtype, int cache_dtype, int64_t rows, int64_t B, int64_t H, int64_t KV, int64_t hd, int64_t max_new,
                    int64_t max_len) {
  Plan p = make_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len);
  p.likely = p.nsplit;
  if (dtype == LZ_F32) return p;
  const int64_t G = H / KV, packed = std::max<int64_t>(1, std::min(max_new, rows)) * G, cus = lz_num_cus();
  const int64_t len = std::max<int64_t>(1, max_len), blocks = blocks_of(32, packed, rows, B, KV, G);
  const bool converted = cache_dtype == LZ_E4M3 && hd == 128;
  const int64_t whole = (1536 + 16 * blocks) / (converted ? 2 : 1);
  const bool shared = blocks < cus ? len > whole : (len > 2048 && B >= 8) || (len > 4096 && 4 * blocks <= 5 * cus);
  const bool many = 8 * blocks_of(64, packed, rows, B, KV, G) >= cus;
  p.bm = shared && (len >= 4096 ? (packed > 32 && many) || converted : len > 2048 && many && converted) ? 64 : 32;
  p.groups = 1;
  p.nqb = (int)lz_cdiv(packed, p.bm);
  p.nsplit = 1;
  p.waves = !shared && len > 256 && blocks <= (hd == 128 ? 1 : 2) * cus ? 8 : 4;
  if (shared) {
    p.least = 512;
    p.shares = (int)std::max<int64_t>(1, 2 * cus / KV);
    p.nsplit = (int)std::min<int64_t>(lz_cdiv(len, p.least) + 1, 33);
    p.likely = (int)std::min<int64_t>(KV * p.shares / blocks_of(p.bm, packed, rows, B, KV, G) + 2, p.nsplit);
  }
  return p;
}

}  // namespace

static bool plannable(int64_t rows, int64_t B, int64_t H, int64_t KV, int64_t max_len) {
  return rows > 0 && B > 0 && H > 0 && KV > 0 && H % KV == 0 && max_len >= 0 && max_len <= INT32_MAX - 1024;
}

// Workspace of the parts and, for trees, of their counts.
static int64_t part_bytes(const Plan& p, int64_t rows, int64_t B, int64_t H, int64_t hd) {
  return p.nsplit > 1 ? rows * H * p.nsplit * (hd + 2) * 4 + (p.shares ? B * p.nqb * 4 : 0) : 0;
}

LZ_EXPORT int64_t lz_paged_attn_plan(int dtype, int cache_dtype, int64_t rows, int64_t B, int64_t H, int64_t KV,
                                     int64_t hd, int64_t max_new, int64_t max_len) {
  if (!plannable(rows, B, H, KV, max_len)) return 0;
  const Plan p = make_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len);
  return p.bm | (p.bm == kPagedTileRows ? p.groups : 1) << 8 | (int64_t)p.nsplit << 16;
}

LZ_EXPORT int64_t lz_paged_attn_workspace(int dtype, int cache_dtype, int64_t rows, int64_t B, int64_t H, int64_t KV,
                                          int64_t hd, int64_t max_new, int64_t max_len) {
  if (!plannable(rows, B, H, KV, max_len)) return 0;
  const Plan p = make_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len);
  return p.nsplit > 1 ? rows * H * p.nsplit * (hd + 2) * 4 : 0;
}

LZ_EXPORT int64_t lz_tree_attn_plan(int dtype, int cache_dtype, int64_t rows, int64_t B, int64_t H, int64_t KV, int64_t hd,
                                    int64_t max_new, int64_t max_len) {
  if (!plannable(rows, B, H, KV, max_len)) return 0;
  const Plan p = make_tree_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len);
  return p.bm | (int64_t)(p.shares ? 1 : 0) << 8 | (int64_t)(p.waves == 8 ? 1 : 0) << 9 | (int64_t)p.nsplit << 16;
}

LZ_EXPORT int64_t lz_tree_attn_workspace(int dtype, int cache_dtype, int64_t rows, int64_t B, int64_t H, int64_t KV,
                                         int64_t hd, int64_t max_new, int64_t max_len) {
  if (!plannable(rows, B, H, KV, max_len)) return 0;
  const Plan p = make_tree_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len);
  return part_bytes(p, rows, B, H, hd);
}

template <typename Rows>
static void run_waves(const PagedArgs& a, const Plan& p, int dtype, int cache_dtype, int64_t hd, uint32_t blocks,
                      hipStream_t s) {
#define RUN(T, HD, E8)                                                                                                   \
  do {                                                                                                                   \
    if constexpr (std::is_same<Rows, PagedRows>::value || std::is_same<T, float>::value) {                               \
      if (p.bm == 16) paged_wave_kernel<T, HD, E8, 1, Rows><<<blocks, 256, 0, s>>>(a);                                   \
      else paged_wave_kernel<T, HD, E8, 2, Rows><<<blocks, 256, 0, s>>>(a);                                              \
    }                                                                                                                    \
  } while (0)
  LZ_CACHE_CASES(dtype, cache_dtype, hd, RUN);
#undef RUN
}
template <typename Rows>
static void run_join(const PagedArgs& a, int dtype, int64_t hd, uint32_t blocks, int per, int likely, hipStream_t s) {
#define RUN(T, HD, E8) paged_join_kernel<T, HD, Rows><<<blocks, 256, 0, s>>>(a, a.bm, per, likely)
  LZ_CACHE_CASES(dtype, 0, hd, RUN);
#undef RUN
}

static int attend(const char* what, const void* q, int64_t ldq, int dtype, int64_t rows, const void* k, const void* v,
                  const void* k_exp, const void* v_exp, int cache_dtype, int64_t pages, int64_t page_size,
                  const int32_t* table, int64_t width, const int32_t* row_start, const int32_t* kv_len, int64_t B,
                  int64_t H, int64_t KV, int64_t hd, int64_t max_new, int64_t max_len, float scale, void* o, int64_t ldo,
                  void* workspace, int64_t ws_bytes, void* stream, const int32_t* base, const uint32_t* mask,
                  int64_t words) {
  if (int rc = lz_check_pages(what, k, v, k_exp, v_exp, cache_dtype, dtype, pages, page_size, table, width, B,
                              KV, hd))
    return rc;
  const int esz = lz_esize(dtype);
  LZ_REQUIRE(H > 0 && H % KV == 0 && H <= 65536 && rows >= 0 && rows * H <= INT32_MAX / 64 && max_new >= 0 &&
                 max_len >= 0 && max_len <= INT32_MAX - 1024,
             "%s: bad shape", what);
  // (-inf, a masked score, times 0 or a subnormal that is flushed would be NaN)
  LZ_REQUIRE(scale >= std::numeric_limits<float>::min() && scale * kLog2e < INFINITY, "%s: scale %g", what, (double)scale);
  LZ_REQUIRE(ldq >= H * hd && ldo >= H * hd, "%s: row strides shorter than the rows", what);
  LZ_REQUIRE(rows == 0 || (q && o && row_start && kv_len && lz_aligned16(q) && lz_aligned16(o) && ldq * esz % 16 == 0 &&
                           ldo * esz % 16 == 0),
             "%s: rows must be 16-byte aligned", what);
  if (rows == 0) return LZ_OK;
  const Plan p = mask ? make_tree_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len)
                      : make_plan(dtype, cache_dtype, rows, B, H, KV, hd, max_new, max_len);
  const int64_t need = part_bytes(p, rows, B, H, hd);
  LZ_REQUIRE(need == 0 || (workspace && lz_aligned16(workspace) && ws_bytes >= need),
             "%s: workspace of %lld bytes, %lld needed", what, (long long)ws_bytes, (long long)need);
  const int64_t blocks = p.shares ? KV * p.shares : B * KV * p.nqb * p.nsplit;
  const int64_t per = p.shares ? (p.likely <= 4 ? 1 : p.likely <= 12 ? 2 : 4) : p.nsplit <= 4 ? 1 : p.nsplit <= 16 ? 4 : 8;
  const int64_t joins = lz_cdiv(rows * H * (hd / 4) * per, 256);
  LZ_REQUIRE(p.shares == 0 || B * p.nqb < INT32_MAX / (lz_cdiv(width * page_size, 128) + 1), "%s: too many rows and pages", what);
  LZ_REQUIRE(blocks <= INT32_MAX / 256 && joins <= INT32_MAX / 256, "%s: too many rows", what);
  PagedArgs a{q, ldq, k, v, (const int8_t*)k_exp, (const int8_t*)v_exp,
              LzPages{table, (int)width, (int)pages, lz_log2(page_size)}, row_start, kv_len, o, ldo, (float*)workspace,
              scale, (int)rows, (int)B, (int)H, (int)KV, p.nqb, p.nsplit, p.chunk,
              (int)(std::min(max_new, rows) * (H / KV)), base, mask, (int)words, p.bm, p.shares, p.least,
              p.shares ? (int32_t*)((float*)workspace + rows * H * p.nsplit * (hd + 2)) : nullptr, p.waves};
  hipStream_t s = lz_stream(stream);
  const bool e8 = cache_dtype == LZ_E4M3;
  if (mask && dtype != LZ_F32) {
    if (int rc = lz_tree_tiles(a, dtype, e8, hd, (uint32_t)blocks, s)) return rc;
  } else if (p.bm == kPagedTileRows) {
    if (int rc = lz_paged_tile(a, dtype, e8, hd, p.groups, (uint32_t)blocks, s)) return rc;
  } else if (mask) {
    run_waves<TreeRows>(a, p, dtype, cache_dtype, hd, (uint32_t)blocks, s);
  } else {
    run_waves<PagedRows>(a, p, dtype, cache_dtype, hd, (uint32_t)blocks, s);
  }
  if (p.nsplit > 1) {
    if (mask) run_join<TreeRows>(a, dtype, hd, (uint32_t)joins, (int)per, p.likely, s);
    else run_join<PagedRows>(a, dtype, hd, (uint32_t)joins, (int)per, p.likely, s);
  }
  return lz_check_launch(what);
}

LZ_EXPORT int lz_paged_attn(const void* q, int64_t ldq, int dtype, int64_t rows, const void* k, const void* v,
                            const void* k_exp, const void* v_exp, int cache_dtype, int64_t pages, int64_t page_size,
                            const int32_t* table, int64_t width, const int32_t* row_start, const int32_t* kv_len,
                            int64_t B, int64_t H, int64_t KV, int64_t hd, int64_t max_new, int64_t max_len, float scale,
                            void* o, int64_t ldo, void* workspace, int64_t ws_bytes, void* stream) {
  return attend("lz_paged_attn", q, ldq, dtype, rows, k, v, k_exp, v_exp, cache_dtype, pages, page_size, table, width,
                row_start, kv_len, B, H, KV, hd, max_new, max_len, scale, o, ldo, workspace, ws_bytes, stream, nullptr,
                nullptr, 0);
}

LZ_EXPORT int lz_tree_attn(const void* q, int64_t ldq, int dtype, int64_t rows, const void* k, const void* v,
                           const void* k_exp, const void* v_exp, int cache_dtype, int64_t pages, int64_t page_size,
                           const int32_t* table, int64_t width, const int32_t* row_start, const int32_t* kv_len,
                           const int32_t* base, const int32_t* mask, int64_t words, int64_t B, int64_t H, int64_t KV,
                           int64_t hd, int64_t max_new, int64_t max_len, float scale, void* o, int64_t ldo,
                           void* workspace, int64_t ws_bytes, void* stream) {
  LZ_REQUIRE(words > 0 && words <= (1 << 20), "lz_tree_attn: %lld mask words a row", (long long)words);
  LZ_REQUIRE(rows == 0 || (base && mask), "lz_tree_attn: no mask");
  return attend("lz_tree_attn", q, ldq, dtype, rows, k, v, k_exp, v_exp, cache_dtype, pages, page_size, table, width,
                row_start, kv_len, B, H, KV, hd, max_new, max_len, scale, o, ldo, workspace, ws_bytes, stream, base,
                (const uint32_t*)mask, words);
}

// Attention over a paged cache for chunks of new tokens: the part that is
// bound by the matrix cores.
//
// A workgroup owns 128 packed rows (32 for each of four waves) of one kv head
// and goes over the keys 64 at a time, K and V in swizzled LDS tiles of two
// stages; S^T = K . Q^T, so a lane owns a row and the probabilities are the B
// operand of O^T += V^T . P^T as they stand, V^T read transposed from LDS.
// Packing the heads of a group into the rows lets one tile of K and V serve
// all of them, and only the steps that cross a wave's diagonal carry masks.
// 16-bit caches go straight from their pages into LDS (a load of 4 to 16 rows
// lies in one page); e4m3 ones pass through registers, where the next step's
// bytes wait while this one is computed, and become 16-bit values once for
// all four waves.
#include "paged_attn.h"

namespace {

template <typename F, int HD, bool k8>
struct Tiles {
  static constexpr int kTile = 64 * HD * 2;
  static constexpr int kRowsPerLoad = 1024 / (HD * 2), kChunks = HD / 8, kPer = 64 / kRowsPerLoad / 4;
  // e4m3: 16-byte pieces of a tile and of a thread
  static constexpr int kPieces = 64 * HD / 16, kMine = (kPieces + 255) / 256;

  char* ks;  // two K tiles, then two V tiles
  int lane, wave, tid;
  int ids;       // page of the 16-key tile ids_from + lane
  int ids_from;
  uint4 kr[kMine], vr[kMine];
  int kx[kMine], vx[kMine];

  __device__ __forceinline__ char* k_tile(int it) const { return ks + (it & 1) * kTile; }
  __device__ __forceinline__ char* v_tile(int it) const { return ks + (2 + (it & 1)) * kTile; }

  // The pages of steps it .. it + 15 (64 keys each).
  __device__ __forceinline__ void look_up(const PagedArgs& a, int b, int it, int n_keys) {
    ids_from = 4 * it;
    const int key = 64 * it + 16 * lane;
    ids = key < n_keys ? a.pg.page_of(b, key) : -1;
  }
  // bit t: the 16-key tile t of step it has a page (or holds no key at all)
  __device__ __forceinline__ uint32_t present(int it, int n_keys) const {
    const uint64_t ok = __ballot(ids >= 0 || 16 * (ids_from + lane) >= n_keys);
    return (uint32_t)(ok >> (4 * it - ids_from)) & 15u;
  }
  __device__ __forceinline__ int64_t token(const PagedArgs& a, int g, int it, int r) const {
    const int id = max(__builtin_amdgcn_readlane(ids, 4 * it + r / 16 - ids_from), 0);  // no page: any, zeroed later
    return (((int64_t)id * a.KV + g) << a.pg.log_size) + ((64 * it + r) & ((1 << a.pg.log_size) - 1));
  }

  __device__ __forceinline__ void issue(const PagedArgs& a, int g, int it) {
    if constexpr (!k8) {
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        char* dst = side ? v_tile(it) : k_tile(it);
        const char* src = static_cast<const char*>(side ? a.v : a.k);
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int blk = wave * kPer + q, r = blk * kRowsPerLoad + lane / kChunks;
          const int c = (lane % kChunks) ^ tswz<HD>(r);
          lz_dma16_first(lz_buffer_rsrc(src + token(a, g, it, blk * kRowsPerLoad) * HD * 2),
                         (uint32_t)((lane / kChunks) * HD * 2 + c * 16), 0, dst + blk * 1024);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int p = tid + 256 * j, r = p / (HD / 16), c = p % (HD / 16);
        if (kPieces % 256 && p >= kPieces) continue;
        const int id = max(__shfl(ids, 4 * it + r / 16 - ids_from, 64), 0);
        const int64_t tok = (((int64_t)id * a.KV + g) << a.pg.log_size) + ((64 * it + r) & ((1 << a.pg.log_size) - 1));
        kr[j] = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.k) + tok * HD + 16 * c);
        vr[j] = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.v) + tok * HD + 16 * c);
        kx[j] = a.k_exp[tok];
        vx[j] = a.v_exp[tok];
      }
    }
  }

  static __device__ __forceinline__ void put(char* tile, int r, int c, const uint4& x, int e) {
    const float unit = lz_pow2(e);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint4*>(tile + toff<HD>(r, 2 * c + h)) =
          make_uint4(e4m3_pair<F, false>(w[2 * h], unit), e4m3_pair<F, true>(w[2 * h], unit),
                     e4m3_pair<F, false>(w[2 * h + 1], unit), e4m3_pair<F, true>(w[2 * h + 1], unit));
  }
  // e4m3: the bytes of step it into its tiles
  __device__ __forceinline__ void put(int it) const {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int p = tid + 256 * j, r = p / (HD / 16), c = p % (HD / 16);
      if (kPieces % 256 && p >= kPieces) continue;
      put(k_tile(it), r, c, kr[j], kx[j]);
      put(v_tile(it), r, c, vr[j], vx[j]);
    }
  }
  // zeros into the V rows of step it that hold no token: their weights are
  // zero, what lies there may not be finite
  __device__ __forceinline__ void clear(int it, int n_keys, uint32_t here) const {
    for (int p = tid; p < 64 * kChunks; p += 256) {
      const int r = p / kChunks;
      if (64 * it + r >= n_keys || !((here >> (r / 16)) & 1))
        *reinterpret_cast<uint4*>(v_tile(it) + toff<HD>(r, p % kChunks)) = make_uint4(0, 0, 0, 0);
    }
  }
};

template <typename F, int HD>
__device__ __forceinline__ void step_scores(f32x16_t (&s)[2], const TileOffsets<HD>& to, const char* kt,
                                            const bf16x8_t (&qf)[HD / 16]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
    for (int t = 0; t < 2; ++t) s[t] = mfma16<F>(to.frag(kt, t, kk), qf[kk], s[t]);
}

// The fragment without its infinities and NaN.
template <typename F>
__device__ __forceinline__ bf16x8_t finite_part(const bf16x8_t& x) {
  uint4 w = __builtin_bit_cast(uint4, x);
  uint32_t* y = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (nonfinite16<F>(y[i] & 0xffffu)) y[i] &= 0xffff0000u;
    if (nonfinite16<F>(y[i] & 0xffff0000u)) y[i] &= 0xffffu;
  }
  return __builtin_bit_cast(bf16x8_t, w);
}

// One step's softmax and its part of the sum.  s: scores of keys 32 t + 8 (r /
// 4) + 4 half + r % 4 in register [t][r]; MASK: keys at or past `lim` (of this
// lane's row, from the step's first key) and 16-key tiles without their bit in
// `here` are not seen.
template <typename F, int HD, bool MASK>
__device__ __forceinline__ void step_sum(f32x16_t (&s)[2], f32x16_t (&o)[HD / 32], float& m, float& l,
                                         const TileOffsets<HD>& to, const char* vt, float unit, int lim, uint32_t here,
                                         bool odd, int half) {
  float mx = -INFINITY;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (MASK) {
        const int key = 32 * t + 8 * (r >> 2) + 4 * half + (r & 3);
        if (key >= lim || !((here >> (2 * t + (r >> 3))) & 1)) s[t][r] = -INFINITY;
      }
      mx = fmaxf(mx, s[t][r]);
    }
  mx = max_halves(mx) * unit;
  if (__ballot(mx > m)) {  // some row's maximum moved
    const float m_new = fmaxf(m, mx);
    const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
    l *= alpha;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
    m = m_new;
  }
  const float nm = m == -INFINITY ? 0.f : -m;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[t][r], unit, nm));
      s[t][r] = p;
      l += p;  // this lane's keys; the halves meet at the end
    }
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const bf16x8_t pb = pack8<F>(s[ks >> 1], 8 * (ks & 1));
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      bf16x8_t f = to.frag_t(vt, ks, i);
      if constexpr (MASK)
        if (odd) f = finite_part<F>(f);
      o[i] = mfma16<F>(f, pb, o[i]);
    }
  }
}

// Whether V rows lo .. hi - 1 of the tile hold an infinity or NaN.
template <typename F, int HD>
__device__ __forceinline__ bool rows_odd(const char* vt, int lo, int hi, int lane) {
  constexpr int kChunks = HD / 8, kRows = 64 / kChunks;
  bool odd = false;
  for (int r0 = lo; r0 < hi; r0 += kRows) {
    const int r = r0 + lane / kChunks;
    if (r < hi) {
      const uint4 x = *reinterpret_cast<const uint4*>(vt + r * HD * 2 + (lane % kChunks) * 16);
      odd |= nonfinite16<F>(x.x) || nonfinite16<F>(x.y) || nonfinite16<F>(x.z) || nonfinite16<F>(x.w);
    }
  }
  return __ballot(odd) != 0;
}

// What finite_part took out, added to the rows that see it.
template <typename F, int HD>
__device__ __forceinline__ void add_odd(f32x16_t (&o)[HD / 32], const f32x16_t (&s)[2], const char* vt, int lim,
                                        int lane) {
  const int half = lane >> 5, l32 = lane & 31;
#pragma unroll 1
  for (int key = 0; key < 64; ++key) {
    float p = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) p = key >> 5 == t && 4 * ((key & 31) >> 3) + (key & 3) == r ? s[t][r] : p;
    p = __shfl(p, l32 + 32 * ((key >> 2) & 1), 64);
    if (key < lim) {
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
          const float y = F::to_f(*reinterpret_cast<const uint16_t*>(vt + toff<HD>(key, d >> 3) + (d & 7) * 2));
          if (!(fabsf(y) < INFINITY)) o[i][r] = fmaf(p, y, o[i][r]);
        }
    }
  }
}

template <typename F, int HD, bool k8>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 2 : 3, HD == 128 ? 2 : 3)))
paged_tile_kernel(PagedArgs a) {
  typedef Tiles<F, HD, k8> T;
  constexpr int BM = kPagedTileRows;
  __shared__ __attribute__((aligned(1024))) char smem[4 * T::kTile];

  const PagedPlace at(a, blockIdx.x);
  const PagedRows rw(a, at.b, at.qb * BM);
  if (rw.m0 >= rw.count) return;
  const int n_keys = rw.keys(BM), n_parts = PagedRows::parts(a, n_keys);
  if (at.split >= n_parts) return;
  const int k_lo = at.split * a.chunk, k_hi = at.split + 1 == n_parts ? n_keys : k_lo + a.chunk;

  T tl;
  tl.ks = smem;
  tl.tid = threadIdx.x;
  tl.lane = tl.tid & 63;
  tl.wave = __builtin_amdgcn_readfirstlane(tl.tid >> 6);
  const int lane = tl.lane, half = lane >> 5, l32 = lane & 31;
  TileOffsets<HD> to;
  to.init(lane);

  // this wave's rows: the first sees `all` keys, the last `most`
  const int m_first = rw.m0 + 32 * tl.wave, m_last = min(m_first + 32, rw.count) - 1;
  const bool idle = m_first >= rw.count;
  const int all = idle ? 0 : rw.sees(m_first), most = idle ? 0 : rw.sees(m_last);
  const int m = min(m_first + l32, rw.count - 1);  // rows past the last repeat it and are not stored
  const int row = rw.row(m), head = at.g * rw.G + m % rw.G, sees = rw.sees(m);

  bf16x8_t qf[HD / 16];
  const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.ldq + head * HD + 8 * half;
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk) qf[kk] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4*>(qp + kk * 16));
  f32x16_t o[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float mx = -INFINITY, l = 0.f;
  const float unit = a.scale * kLog2e;

  int it = k_lo / 64;
  const int end = (k_hi + 63) / 64, free_end = min(all / 64, end), wave_end = min((most + 63) / 64, end);
  tl.look_up(a, at.b, it, n_keys);
  if (it < end) {
    tl.issue(a, at.g, it);
    if constexpr (k8) tl.put(it);
  }

  // Opens step it: its tiles are there and every wave is done with the other
  // stage, into which the next step's go.
  auto open_step = [&]() {
    dma_barrier();
    const uint32_t here = tl.present(it, n_keys);
    if (64 * it + 64 > n_keys || here != 15u) {  // the same for all waves
      tl.clear(it, n_keys, here);
      __syncthreads();
    }
    if (it + 1 < end) tl.issue(a, at.g, it + 1);
    return here;
  };
  auto close_step = [&]() {
    if constexpr (k8)
      if (it + 1 < end) tl.put(it + 1);
  };

  while (it < end) {
    // fifteen steps: the pages looked up serve one more, which they issue
    const int stop = min(it + 15, end);
    const bool clean = __ballot(tl.ids >= 0 || 16 * (tl.ids_from + lane) >= n_keys) == ~0ull;
    const int free_stop = clean ? min(stop, free_end) : it;
    for (; it < free_stop; ++it) {
      open_step();
      f32x16_t s[2];
      step_scores<F, HD>(s, to, tl.k_tile(it), qf);
      step_sum<F, HD, false>(s, o, mx, l, to, tl.v_tile(it), unit, 0, 15u, false, half);
      close_step();
    }
    for (; it < stop; ++it) {
      const uint32_t here = open_step();
      if (it < wave_end) {
        f32x16_t s[2];
        step_scores<F, HD>(s, to, tl.k_tile(it), qf);
        const bool odd = rows_odd<F, HD>(tl.v_tile(it), max(all - 64 * it, 0), min(64, n_keys - 64 * it), lane);
        step_sum<F, HD, true>(s, o, mx, l, to, tl.v_tile(it), unit, sees - 64 * it, here, odd, half);
        if (odd) add_odd<F, HD>(o, s, tl.v_tile(it), sees - 64 * it, lane);
      }
      close_step();
    }
    if (it < end) tl.look_up(a, at.b, it, n_keys);
  }

  l = sum_halves(l);
  if (m_first + l32 >= rw.count) return;
  if (n_parts == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* op = static_cast<uint16_t*>(a.o) + (int64_t)row * a.ldo + head * HD;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        store_bf16x4<F>(op + 32 * i + 8 * q4 + 4 * half, o[i][4 * q4] * inv, o[i][4 * q4 + 1] * inv,
                        o[i][4 * q4 + 2] * inv, o[i][4 * q4 + 3] * inv);
  } else {
    const int64_t at_row = ((int64_t)row * a.H + head) * a.nsplit + at.split;
    float* part = a.part + at_row * HD;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<float4*>(part + 32 * i + 8 * q4 + 4 * half) =
            make_float4(o[i][4 * q4], o[i][4 * q4 + 1], o[i][4 * q4 + 2], o[i][4 * q4 + 3]);
    if (half == 0) {
      float* s2 = a.part + (int64_t)a.rows * a.H * a.nsplit * HD + at_row * 2;
      s2[0] = mx;
      s2[1] = l;
    }
  }
}

}  // namespace

int lz_paged_tile(const LzPagedArgs& a, int dtype, bool e4m3, int64_t hd, uint32_t blocks, hipStream_t stream) {
#define RUN(F, HD)                                                                      \
  do {                                                                                  \
    if (e4m3) paged_tile_kernel<F, HD, true><<<blocks, 256, 0, stream>>>(a);            \
    else paged_tile_kernel<F, HD, false><<<blocks, 256, 0, stream>>>(a);                \
  } while (0)
  if (dtype == LZ_F16) {
    if (hd == 32) RUN(FmtF16, 32);
    else if (hd == 64) RUN(FmtF16, 64);
    else RUN(FmtF16, 128);
  } else {
    if (hd == 32) RUN(FmtBF16, 32);
    else if (hd == 64) RUN(FmtBF16, 64);
    else RUN(FmtBF16, 128);
  }
#undef RUN
  return lz_check_launch("lz_paged_attn");
}

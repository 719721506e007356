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
#include <type_traits>

#include "paged_attn.h"

namespace {

template <typename F, int HD, bool k8>
struct Tiles {
  static constexpr int kTile = 64 * HD * 2;
  static constexpr int kRowsPerLoad = 1024 / (HD * 2), kChunks = HD / 8, kPer = 64 / kRowsPerLoad / 4;
  // e4m3: 16-byte pieces of a tile and of a thread
  static constexpr int kPieces = 64 * HD / 16, kMine = (kPieces + 255) / 256;

  char* ks;  // this key group's two K tiles, then its two V tiles
  int lane, wave, tid;  // wave, tid: in the group of four waves
  int ids;       // page of the 16-key tile ids_from + lane
  int ids_from;
  uint4 kr[kMine], vr[kMine];
  int kx[kMine], vx[kMine];

  int stage;  // of the step that is computed
  __device__ __forceinline__ char* k_tile(int ahead = 0) const { return ks + (stage ^ ahead) * kTile; }
  __device__ __forceinline__ char* v_tile(int ahead = 0) const { return ks + (2 + (stage ^ ahead)) * kTile; }

  // The pages of steps it .. it + 15 (64 keys each).
  __device__ __forceinline__ void look_up(const PagedArgs& a, int b, int it, int n_keys) {
    ids_from = 4 * it;
    const int key = 64 * it + 16 * lane;
    ids = key < n_keys ? a.pg.page_of(b, key) : -1;
  }
  // bit t: the 16-key tile t from step it on has a page (or holds no key at all)
  __device__ __forceinline__ uint32_t present(int it, int n_keys) const {
    const uint64_t ok = __ballot(ids >= 0 || 16 * (ids_from + lane) >= n_keys);
    return (uint32_t)(ok >> (4 * it - ids_from));
  }
  // Step it's rows into the stage `ahead` of this one.  Each wave copies 16,
  // which lie in one page.
  __device__ __forceinline__ void issue(const PagedArgs& a, int g, int it, int ahead) {
    if constexpr (!k8) {
      const int id = max(__builtin_amdgcn_readlane(ids, 4 * it + wave - ids_from), 0);  // no page: any, zeroed later
      const int64_t tok =
          (((int64_t)id * a.KV + g) << a.pg.log_size) + ((64 * it + 16 * wave) & ((1 << a.pg.log_size) - 1));
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        char* dst = (side ? v_tile(ahead) : k_tile(ahead)) + wave * kPer * 1024;
        const lz_v4i rsrc = lz_buffer_rsrc(static_cast<const char*>(side ? a.v : a.k) + tok * HD * 2);
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int c = (lane % kChunks) ^ tswz<HD>(q * kRowsPerLoad + lane / kChunks);  // of the row in its 16
          const uint32_t off = (uint32_t)(q * 1024 + (lane / kChunks) * HD * 2 + c * 16);
          if (q == 0) lz_dma16_first(rsrc, off, 0, dst);
          else lz_dma16(rsrc, off, 0, dst + q * 1024);
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
  // e4m3: the bytes that issue() fetched into their tiles
  __device__ __forceinline__ void put(int ahead) const {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int p = tid + 256 * j, r = p / (HD / 16), c = p % (HD / 16);
      if (kPieces % 256 && p >= kPieces) continue;
      put(k_tile(ahead), r, c, kr[j], kx[j]);
      put(v_tile(ahead), r, c, vr[j], vx[j]);
    }
  }
  // zeros into the V rows of step it that hold no token: their weights are
  // zero, what lies there may not be finite
  __device__ __forceinline__ void clear(int it, int n_keys, uint32_t here) const {
    for (int p = tid; p < 64 * kChunks; p += 256) {
      const int r = p / kChunks;
      if (64 * it + r >= n_keys || !((here >> (r / 16)) & 1))
        *reinterpret_cast<uint4*>(v_tile() + toff<HD>(r, p % kChunks)) = make_uint4(0, 0, 0, 0);
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

// O^T += V^T . P^T of one step, each weight as two terms (weight_terms); vf: the
// fragments of V^T for its first 16 keys, read ahead as the others are here.
// ODD: infinities and NaN left out.
template <typename F, int HD, bool ODD>
__device__ __forceinline__ void step_sum(f32x16_t (&o)[HD / 32], const f32x16_t (&s)[2], bf16x8_t (&vf)[2][HD / 32],
                                         const TileOffsets<HD>& to, const char* vt) {
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    if (ks + 1 < 4)
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) vf[(ks + 1) & 1][i] = to.frag_t(vt, ks + 1, i);
    uint4 pb[2];
    weight_words<F>(pb, [&](int e) { return s[ks >> 1][8 * (ks & 1) + e]; });
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
        o[i] = mfma16<F>(ODD ? finite_part<F>(vf[ks & 1][i]) : vf[ks & 1][i], __builtin_bit_cast(bf16x8_t, pb[t]), o[i]);
  }
}

// One step's softmax and its part of the sum.  s: scores of keys 32 t + 8 (r /
// 4) + 4 half + r % 4 in register [t][r]; MASK: keys at or past `lim` (of this
// lane's row, from the step's first key) and 16-key tiles without their bit in
// `here` are not seen.  ODD: see step_sum().
template <typename F, int HD, bool MASK, bool ODD>
__device__ __forceinline__ void step_softmax(f32x16_t (&s)[2], f32x16_t (&o)[HD / 32], float& m, float& l,
                                             const TileOffsets<HD>& to, const char* vt, float unit, int lim,
                                             uint32_t here, int half) {
  bf16x8_t vf[2][HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) vf[0][i] = to.frag_t(vt, 0, i);
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
  const bool moved = mx > m + kSlack;
  if (__ballot(moved)) {
    const float m_new = moved ? mx : m;
    const float alpha = moved ? __builtin_amdgcn_exp2f(m - m_new) : 1.f;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
    m = m_new;
  }
  const float nm = kLift<F> - (m == -INFINITY ? 0.f : m);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[t][r], unit, nm));
      s[t][r] = p;
      l += p;  // this lane's keys; the halves meet at the end
    }
  step_sum<F, HD, ODD>(o, s, vf, to, vt);
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

// The w-th row block of a kv head in the order of the keys that blocks go over,
// most first: the long ones start at once and the short ones fill the gaps
// (eight prompts of up to 2048 tokens, 16 heads of 128, fp16: 121 us dealt in
// turn, 102 sequence after sequence, 87 so).  Lane b of a wave counts sequence
// b's blocks; a bisection finds the step count of the w-th one.
struct ByLength {
  int b, m0;  // sequence and first row; b < 0: there are fewer blocks

  static __device__ __forceinline__ int sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);  // row_ror 8, 4, 2, 1
    x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false);
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(h[0] + h[1], h[0] + h[1], false, false);
    return __builtin_amdgcn_readfirstlane((int)(q[0] + q[1]));
  }

  __device__ __forceinline__ ByLength(const PagedArgs& a, int w, int lane) {
    constexpr int BM = kPagedTileRows;
    if (a.B > 64) {  // sequence after sequence
      b = w / a.nqb;
      const PagedRows rw(a, b, 0);
      m0 = ((rw.count + BM - 1) / BM - 1 - w % a.nqb) * BM;
      if (m0 < 0) b = -1;
      return;
    }
    int count = 0, base = 0, nq = 0;
    const int G = a.H / a.KV, cap = a.pg.width << a.pg.log_size;
    if (lane < a.B) {
      const PagedRows rw(a, lane, 0);
      count = rw.count;
      base = (int)((uint32_t)rw.base + (uint32_t)rw.row0);  // keys that the sequence's first row sees
      nq = (count + BM - 1) / BM;
    }
    // this lane's first block with more than 64 s keys, nq: none; -1: all blocks
    auto first = [&](int s) {
      const uint32_t t = 64u * (uint32_t)s + 1u;
      if (s < 0) return 0;
      const int d = (int)(t - (uint32_t)base);  // token of its first row that sees t keys
      if (t > (uint32_t)cap || nq == 0 || d > (count - 1) / G) return nq;
      return max(d, 0) * G / BM;
    };
    b = -1;
    m0 = 0;
    if (w >= sum(nq)) return;
    int lo = -1, hi = cap / 64 + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (w < sum(nq - first(mid))) lo = mid;
      else hi = mid;
    }
    const int f0 = first(lo), f1 = first(hi), r = w - sum(nq - f1);
    int before = f1 - f0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(before, o, 64);
      if (lane >= o) before += y;
    }
    before -= f1 - f0;
    const uint64_t here = __ballot(before <= r && r < before + f1 - f0);
    if (here == 0) return;
    b = __builtin_ctzll(here);
    m0 = __builtin_amdgcn_readlane(f0 + r - before, b) * BM;
  }
};

// NG: groups of four waves that share the rows and take every NG-th step of
// the keys, each with tiles of its own; they meet in LDS at the end.
template <typename F, int HD, bool k8, int NG>
__global__ void __launch_bounds__(256 * NG) __attribute__((amdgpu_waves_per_eu(HD == 128 || NG == 2 ? 2 : 3, HD == 128 || NG == 2 ? 2 : 3)))
paged_tile_kernel(PagedArgs a) {
  typedef Tiles<F, HD, k8> T;
  constexpr int BM = kPagedTileRows;
  __shared__ __attribute__((aligned(1024))) char smem[NG * 4 * T::kTile];
  __shared__ float stats[NG == 2 ? 4 : 1][64][2];

  // kv heads go to the XCDs in turn, so that a head's keys and values are
  // fetched into few L2s
  const uint32_t rest = blockIdx.x / (uint32_t)a.KV;
  const ByLength block(a, (int)(rest / (uint32_t)a.nsplit), threadIdx.x & 63);
  if (block.b < 0) return;
  const struct {
    int b, g, split;
  } at = {block.b, (int)(blockIdx.x % (uint32_t)a.KV), (int)(rest % (uint32_t)a.nsplit)};
  const PagedRows rw(a, at.b, block.m0);
  const int n_keys = rw.keys(BM), n_parts = PagedRows::parts(a, n_keys);
  if (at.split >= n_parts) return;
  const int k_lo = at.split * a.chunk, k_hi = at.split + 1 == n_parts ? n_keys : k_lo + a.chunk;

  const int grp = NG == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  T tl;
  tl.ks = smem + grp * 4 * T::kTile;
  tl.tid = threadIdx.x & 255;
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
  float mx, l;
  const float unit = a.scale * kLog2e;
  const int end = (k_hi + 63) / 64, free_end = min(all / 64, end), wave_end = min((most + 63) / 64, end);

  // One pass over the keys, in rounds of NG steps; `rt` is a round's first
  // step.  Returns whether a sum is not finite: an infinity or NaN of V may
  // have met the zero weight of a row that does not see it.  Then the pass is
  // made again with ODD, which multiplies the finite part and adds the rest
  // where it is seen; the other rows get the same bits as ever.
  auto pass = [&](auto odd_pass) {
    constexpr bool ODD = decltype(odd_pass)::value;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    mx = -INFINITY;
    l = 0.f;
    int rt = k_lo / 64;
    tl.stage = 0;
    tl.look_up(a, at.b, rt, n_keys);
    if (rt + grp < end) {
      tl.issue(a, at.g, rt + grp, 0);
      if constexpr (k8) tl.put(0);
    }
    // Opens a round: its tiles are there and every wave is done with the other
    // stage, into which the next round's go.
    auto open_round = [&](auto full) {
      dma_barrier();
      uint32_t here = ~0u;
      if constexpr (!decltype(full)::value) {
        here = tl.present(rt, n_keys);
        constexpr uint32_t kAll = NG == 2 ? 0xffu : 0xfu;
        if (64 * (rt + NG) > n_keys || (here & kAll) != kAll) {  // the same for all waves
          tl.clear(rt + grp, n_keys, here >> (4 * grp));
          __syncthreads();
        }
      }
      if (rt + grp + NG < end) tl.issue(a, at.g, rt + grp + NG, 1);
      return here >> (4 * grp);
    };
    auto close_round = [&]() {
      if constexpr (k8)
        if (rt + grp + NG < end) tl.put(1);
      tl.stage ^= 1;
      rt += NG;
    };
    while (rt < end) {
      // the pages looked up serve one more round than is computed, which it issues
      const int stop = min(rt + 16 - NG, end);
      const bool clean = __ballot(tl.ids >= 0 || 16 * (tl.ids_from + lane) >= n_keys) == ~0ull;
      // rounds that lie before every row's diagonal and whose tiles are full
      const int free_stop = clean && !ODD ? min(stop, min(free_end - grp, n_keys / 64 - NG + 1)) : rt;
      while (rt < free_stop) {
        open_round(std::true_type{});
        f32x16_t s[2];
        step_scores<F, HD>(s, to, tl.k_tile(), qf);
        step_softmax<F, HD, false, false>(s, o, mx, l, to, tl.v_tile(), unit, 0, 15u, half);
        close_round();
      }
      while (rt < stop) {
        const uint32_t here = open_round(std::false_type{});
        const int it = rt + grp;
        if (it < wave_end) {
          f32x16_t s[2];
          step_scores<F, HD>(s, to, tl.k_tile(), qf);
          step_softmax<F, HD, true, ODD>(s, o, mx, l, to, tl.v_tile(), unit, sees - 64 * it, here, half);
          if constexpr (ODD) add_odd<F, HD>(o, s, tl.v_tile(), sees - 64 * it, lane);
        }
        close_round();
      }
      if (rt < end) tl.look_up(a, at.b, rt, n_keys);
    }
    float zero = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) zero = fmaf(o[i][r], 0.f, zero);
    return zero != 0.f;  // NaN
  };
  if (__syncthreads_or(pass(std::false_type{}))) pass(std::true_type{});

  l = sum_halves(l);
  if constexpr (NG == 2) {
    // the second group's sums into LDS, the first adds them to its own
    __syncthreads();
    float* park = reinterpret_cast<float*>(smem) + tl.wave * (HD / 2) * 64 + lane;
    if (grp == 1) {
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) park[(16 * i + r) * 64] = o[i][r];
      stats[tl.wave][lane][0] = mx;
      stats[tl.wave][lane][1] = l;
    }
    __syncthreads();
    if (grp == 1) return;
    const float m2 = stats[tl.wave][lane][0], l2 = stats[tl.wave][lane][1];
    const float top = fmaxf(mx, m2);
    const float f = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top), f2 = m2 == top ? 1.f : __builtin_amdgcn_exp2f(m2 - top);
    mx = top;
    l = fmaf(l, f, l2 * f2);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = fmaf(o[i][r], f, park[(16 * i + r) * 64] * f2);
  }
  if (m_first + l32 >= rw.count) return;
  if (mx == -INFINITY && sees_any(a, at.b, k_lo, k_hi, sees)) mx = kAllInf;
  if (n_parts == 1) {
    const float inv = mx == -INFINITY ? 0.f : 1.f / l;
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

int lz_paged_tile(const LzPagedArgs& a, int dtype, bool e4m3, int64_t hd, int groups, uint32_t blocks, hipStream_t stream) {
#define RUN(F, HD)                                                                      \
  do {                                                                                  \
    if (groups == 2) {                                                                  \
      if (e4m3) paged_tile_kernel<F, HD, true, 2><<<blocks, 512, 0, stream>>>(a);       \
      else paged_tile_kernel<F, HD, false, 2><<<blocks, 512, 0, stream>>>(a);           \
    } else if (e4m3) {                                                                  \
      paged_tile_kernel<F, HD, true, 1><<<blocks, 256, 0, stream>>>(a);                 \
    } else {                                                                            \
      paged_tile_kernel<F, HD, false, 1><<<blocks, 256, 0, stream>>>(a);                \
    }                                                                                   \
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

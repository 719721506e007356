// Attention of trees of drafted tokens over a paged cache, 16-bit rows.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  j < base, or bit j - base of
//   row i's mask is set
//
// A tree has some tens of packed rows over a text of any length, and all of its
// rows go over all of the text, so that the read of K and V bounds it up to 32
// rows or so, and the matrix and vector units together from there on.
//
// A workgroup takes blocks of 32 RG packed rows of a kv head and a stretch of
// their keys (Share).  S^T = K . Q^T, so a lane owns a row and its weights are the
// B operand of O^T += V^T . P^T as they stand; K and V lie in swizzled LDS rows
// (direct-to-LDS loads; e4m3 through registers), V^T is read transposed.  Only the
// tiles behind the text carry masks.
//
// RG = 1: each of the W waves (4, 8) takes every W-th tile of 32 keys, which is its
//   own: the next K is on its way as soon as this one's scores are formed, the next
//   V after this one's sum, and no wave waits for another until the end.  What is
//   on its way bounds it: a CU with four waves reads 43 GB/s, so that eight are
//   faster where a CU has one block (16 x 12 nodes over up to 2048, 16/8 heads of
//   128: 20.7 us, with four 25.5).
// RG = 2: the waves share stages of 64 keys, the next of which is on its way while
//   this one is computed; two waves for each 32 rows, a half of the keys each.
//   It reads K and V half as often where there are more rows, and its parts
//   come together at a barrier a stage (16 nodes of 8 sequences over up to 16384,
//   32/8 heads of 128, e4m3: 63 us, with RG 1 84; 16 nodes of one over 8192, 16
//   bits: 23 and 19).
//   A third form, of 128 rows, won 5 to 15 % over texts of 32768 and lost up to
//   half elsewhere; 64 rows in one wave's registers lost everywhere.
#include <type_traits>

#include "paged_attn.h"

namespace {

// Waits until at most N of this wave's vector loads are under way, and keeps
// reads of LDS behind it.
template <int N>
__device__ __forceinline__ void loads_left() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// What the wave has read from LDS is in registers: its rows may be overwritten.
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A block's tiles: a wave's own (RG 1) or the workgroup's.
template <typename F, int HD, bool k8, int RG, int W>
struct TreeTiles {
  static constexpr bool kOwn = RG == 1;
  static constexpr int kKeys = kOwn ? 32 : 64;      // of a tile
  static constexpr int kTile = kKeys * HD * 2;      // bytes of K or V
  static constexpr int kSmem = W * 2 * 32 * HD * 2; // the waves' K and V, or two stages of K and V
  static constexpr int kRowsPerLoad = 1024 / (HD * 2), kChunks = HD / 8, kPer = 16 / kRowsPerLoad;
  static constexpr int kLoads = 2 * kPer;  // RG 1: of a K or V tile
  static constexpr int kIds = kKeys / 16, kBatch = 64 / kIds;  // pages of a tile, tiles whose pages are held
  // e4m3: 16-byte pieces of a tile, and of a thread
  static constexpr int kPieces = kKeys * HD / 16, kMine = (kPieces + (kOwn ? 63 : 255)) / (kOwn ? 64 : 256);

  char* lds;  // RG 1: the wave's K and V; else the first stage's
  int lane, wave, k_lo, k_hi;
  int ids, later;  // page of 16 keys number `lane` from tile ids_from on, and 64 on
  int ids_from;
  uint4 raw[2][k8 ? kMine : 1];
  int ex[2][k8 ? kMine : 1];

  __device__ __forceinline__ char* tile(int side, int t) const { return lds + (kOwn ? side : 2 * (t & 1) + side) * kTile; }
  __device__ __forceinline__ int key_of(int t) const { return k_lo + (kOwn ? (W * t + wave) * 32 : 64 * t); }
  __device__ __forceinline__ int key_of_id(int t0) const { return key_of(t0 + lane / kIds) + 16 * (lane % kIds); }
  __device__ __forceinline__ int look_up(const PagedArgs& a, int b, int t0) const {
    const int key = key_of_id(t0);
    return key < k_hi ? a.pg.page_of(b, key) : -1;
  }
  __device__ __forceinline__ void begin(const PagedArgs& a, int b) {
    ids = look_up(a, b, 0);
    later = look_up(a, b, kBatch);
    ids_from = 0;
  }
  __device__ __forceinline__ void reach(const PagedArgs& a, int b, int t) {
    if (t - ids_from < kBatch) return;
    ids_from += kBatch;
    ids = later;
    later = look_up(a, b, ids_from + kBatch);
  }
  // Sixteen keys of a side of tile t on their way into LDS.
  __device__ __forceinline__ void fetch16(const PagedArgs& a, int g, int t, int side, int h) {
    const int id = max(__builtin_amdgcn_readlane(ids, kIds * (t - ids_from) + h), 0);  // no page: any, not used
    const int64_t tok =
        (((int64_t)id * a.KV + g) << a.pg.log_size) + ((key_of(t) + 16 * h) & ((1 << a.pg.log_size) - 1));
    const lz_v4i rsrc = lz_buffer_rsrc(static_cast<const char*>(side ? a.v : a.k) + tok * HD * 2);
    char* dst = tile(side, t) + h * 16 * HD * 2;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int c = (lane % kChunks) ^ tswz<HD>(q * kRowsPerLoad + lane / kChunks);  // of the row in its 16
      const uint32_t off = (uint32_t)(q * 1024 + (lane / kChunks) * HD * 2 + c * 16);
      if (q == 0) lz_dma16_first(rsrc, off, 0, dst);
      else lz_dma16(rsrc, off, 0, dst + q * 1024);
    }
  }
  // A side of tile t on its way: into LDS, or into registers.
  __device__ __forceinline__ void fetch(const PagedArgs& a, int g, int t, int side) {
    if constexpr (!k8) {
      if constexpr (kOwn) {
        fetch16(a, g, t, side, 0);
        fetch16(a, g, t, side, 1);
      } else {
        fetch16(a, g, t, side, wave);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int p = (kOwn ? lane : 64 * wave + lane) + (kOwn ? 64 : 256) * j, r = p / (HD / 16), c = p % (HD / 16);
        if (kPieces < 256 && !kOwn && p >= kPieces) continue;
        const int id = max(__shfl(ids, kIds * (t - ids_from) + r / 16, 64), 0);
        const int64_t tok = (((int64_t)id * a.KV + g) << a.pg.log_size) + ((key_of(t) + r) & ((1 << a.pg.log_size) - 1));
        raw[side][j] = *reinterpret_cast<const uint4*>(static_cast<const char*>(side ? a.v : a.k) + tok * HD + 16 * c);
        ex[side][j] = (side ? a.v_exp : a.k_exp)[tok];
      }
    }
  }
  // e4m3: what fetch() brought, into tile t as 16-bit values
  __device__ __forceinline__ void put(int t, int side) const {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int p = (kOwn ? lane : 64 * wave + lane) + (kOwn ? 64 : 256) * j, r = p / (HD / 16), c = p % (HD / 16);
      if (kPieces < 256 && !kOwn && p >= kPieces) continue;
      const float unit = lz_pow2(ex[side][j]);
      const uint32_t w[4] = {raw[side][j].x, raw[side][j].y, raw[side][j].z, raw[side][j].w};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint4*>(tile(side, t) + toff<HD>(r, 2 * c + h)) =
            make_uint4(e4m3_pair<F, false>(w[2 * h], unit), e4m3_pair<F, true>(w[2 * h], unit),
                       e4m3_pair<F, false>(w[2 * h + 1], unit), e4m3_pair<F, true>(w[2 * h + 1], unit));
    }
  }
  // zeros into the rows of V that hold no token: their weights are zero, what
  // lies there may not be finite
  __device__ __forceinline__ void clear(int t, int n_keys, uint32_t here) const {
    for (int p = kOwn ? lane : 64 * wave + lane; p < kKeys * kChunks; p += kOwn ? 64 : 256) {
      const int r = p / kChunks;
      if (key_of(t) + r >= n_keys || !((here >> (r / 16)) & 1))
        *reinterpret_cast<uint4*>(tile(1, t) + toff<HD>(r, p % kChunks)) = make_uint4(0, 0, 0, 0);
    }
  }
};

// Sums, and maxima, of the lanes up to this one.
template <typename Op>
__device__ __forceinline__ int scan(int x, int none, const Op& op) {
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x112, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x114, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x118, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x143, 0xc, 0xf, false));
  return x;
}

// A workgroup's share of a kv head's work, dealt out on the device: the plan
// knows bounds of the lengths alone, and blocks cut by those leave CUs without
// work where sequences are shorter or have fewer rows than others.  The row
// blocks of all sequences, one after another, each with its units of 128 keys,
// are one list, of which each of a.shares workgroups takes as much as the others:
// a stretch of up to several blocks, the first and last of them in part.  With
// a whole wave (up to 64 sequences are held in its lanes, more are looked through
// again for each block).
struct Share {
  int at, end;  // units of the list, of which `per` a workgroup
  int per;
  int up_to, nq, units;  // lane l: of sequence l: units of the list up to its last, row blocks, units of a block

  static __device__ __forceinline__ int2 size(const PagedArgs& a, int b) {
    if (b >= a.B) return make_int2(0, 0);
    const PagedRows rw(a, a.row_start[b], a.row_start[b + 1], a.kv_len[b], 0);
    const int nq = (rw.count + a.bm - 1) / a.bm;  // rows that see nothing are written too
    return make_int2(nq, nq ? max((min(max(a.kv_len[b], 0), rw.cap) + 127) >> 7, 1) : 0);
  }

  __device__ __forceinline__ Share(const PagedArgs& a, int w, int lane) {
    if (a.shares == 0) {  // a block each
      at = w;
      end = w + 1;
      return;
    }
    auto add = [](int x, int y) { return x + y; };
    auto larger = [](int x, int y) { return max(x, y); };
    int all = 0, most = 0;
    for (int b0 = (a.B - 1) & ~63; b0 >= 0; b0 -= 64) {  // the first 64 last: they stay
      const int2 s = size(a, b0 + lane);
      nq = s.x;
      units = s.y;
      up_to = scan(nq * units, 0, add);
      all += __builtin_amdgcn_readlane(up_to, 63);
      most = max(most, __builtin_amdgcn_readlane(scan(units, 0, larger), 63));
    }
    per = max(max((all + a.shares - 1) / a.shares, (most + a.nsplit - 2) / (a.nsplit - 1)), a.least >> 7);
    at = lz_stretch(w, per, all);
    end = lz_stretch(w + 1, per, all);
  }

  struct Block {
    int b, qb, from, units, part, parts;  // units from .. from + units - 1 of the block, its part-th of `parts`
  };
  // The block at the head of what is left, which is taken off.
  __device__ __forceinline__ Block next(const PagedArgs& a, int w, int lane) {
    if (a.shares == 0) {
      ++at;
      return Block{w / a.nqb, w % a.nqb, 0, INT32_MAX / 256, 0, 1};
    }
    int before = 0, b0 = 0, u = up_to, n = units, blocks = nq;
    uint64_t here;
    while ((here = __ballot(at < before + u)) == 0) {  // at < end <= all: there is one
      before += __builtin_amdgcn_readlane(u, 63);
      b0 += 64;
      const int2 s = size(a, b0 + lane);
      blocks = s.x;
      n = s.y;
      u = scan(blocks * n, 0, [](int x, int y) { return x + y; });
    }
    const int l = __builtin_ctzll(here);
    const int size = __builtin_amdgcn_readlane(n, l);
    const int first = before + __builtin_amdgcn_readlane(u, l) - __builtin_amdgcn_readlane(blocks, l) * size;
    Block k;
    k.b = b0 + l;
    k.qb = (at - first) / size;
    const int start = first + k.qb * size;
    k.from = at - start;
    k.units = min(size - k.from, end - at);
    k.part = w - start / per;
    k.parts = (start + size - 1) / per - start / per + 1;
    at += k.units;
    return k;
  }
};

template <typename F, int HD, bool k8, int RG, int W>
__global__ void __launch_bounds__(64 * W, 2) tree_kernel(PagedArgs a) {
  typedef TreeTiles<F, HD, k8, RG, W> T;
  constexpr int BM = 32 * RG, KG = W / RG;
  __shared__ __attribute__((aligned(1024))) char smem[T::kSmem];
  __shared__ float ml[W][32][2];
  T tl;
  const int tid = threadIdx.x;
  tl.lane = tid & 63;
  tl.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  tl.lds = smem + (T::kOwn ? tl.wave * 2 * T::kTile : 0);
  const int lane = tl.lane, half = lane >> 5, l32 = lane & 31;
  const int rg = tl.wave % RG, t32 = RG == 2 ? tl.wave / RG : 0;  // this wave's rows, and first half of a tile
  TileOffsets<HD> to;
  to.init(lane);
  const float unit = a.scale * kLog2e;

  // kv heads go to the XCDs in turn
  const int g = (int)(blockIdx.x % (uint32_t)a.KV), w = (int)(blockIdx.x / (uint32_t)a.KV);
  auto block = [&](const Share::Block& k) {
    const TreeRows rw(a, k.b, k.qb * BM);
    if (rw.m0 >= rw.count) return;  // the same for all waves
    const int n_keys = rw.len;
    tl.k_lo = k.from * 128;
    tl.k_hi = min(tl.k_lo + k.units * 128, n_keys);
    const bool idle = rw.m0 + 32 * rg >= rw.count;
    const int m = min(rw.m0 + 32 * rg + l32, rw.count - 1);  // rows past the last repeat it and are not stored
    const int row = rw.row(m);
    const uint32_t* mask = a.mask + (int64_t)row * a.words;
    tl.begin(a, k.b);
    bf16x8_t qf[HD / 16];
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)row * a.ldq + (g * rw.G + m % rw.G) * HD + 8 * half;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) qf[kk] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4*>(qp + kk * 16));
    f32x16_t o[HD / 32];
    float mx, l;
    const int span = tl.k_hi - tl.key_of(0), n_tiles = span > 0 ? (T::kOwn ? (span + 32 * W - 1) / (32 * W) : (span + 63) / 64) : 0;
    // tiles that every row sees whole
    const int free_span = min(rw.ctx, tl.k_hi) - tl.key_of(0);
    const int free_tiles = free_span >= T::kKeys ? (T::kOwn ? (free_span - 32) / (32 * W) + 1 : free_span / 64) : 0;
    uint64_t there = 0;
    bool odd = false;

    auto step = [&](int t, auto free_tile) {
      constexpr bool FREE = decltype(free_tile)::value;
      // its sixteens that have a page
      const uint32_t here = FREE ? 15u : (uint32_t)(there >> (T::kIds * (t % T::kBatch))) & ((1u << T::kIds) - 1u);
      const bool more = t + 1 < n_tiles;
      const int key0 = tl.key_of(t);
      if constexpr (T::kOwn) {
        if constexpr (!k8) loads_left<T::kLoads>();  // V may be under way
      } else {
        dma_barrier();  // the tile is there, and every wave is done with the last one
        if constexpr (!FREE)
          if (key0 + 64 > n_keys || here != (1u << T::kIds) - 1u) {  // the same for all waves
            tl.clear(t, n_keys, here);
            __syncthreads();
          }
        if (more) {
          tl.reach(a, k.b, t + 1);
          tl.fetch(a, g, t + 1, 0);
          tl.fetch(a, g, t + 1, 1);
        }
      }
      if (T::kOwn || !idle) {
        f32x16_t s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) s = mfma16<F>(to.frag(tl.tile(0, t), t32, kk), qf[kk], s);
        if constexpr (T::kOwn)
          if (more) {
            if constexpr (!k8) {
              reads_done();
              tl.reach(a, k.b, t + 1);
              tl.fetch(a, g, t + 1, 0);
            } else {
              tl.put(t + 1, 0);
              if (t + 2 < n_tiles) {
                tl.reach(a, k.b, t + 2);
                tl.fetch(a, g, t + 2, 0);
              }
            }
          }
        uint32_t mine = 0;
        if constexpr (!FREE) {
          const int first = key0 + 32 * t32, left = tl.k_hi - first, there2 = here >> (2 * t32);
          mine = tree_bits(mask, a.words, first - rw.ctx);
          if (left < 32) mine &= left > 0 ? (1u << left) - 1u : 0u;
          mine &= ((there2 & 1) ? 0xffffu : 0u) | ((there2 & 2) ? 0xffff0000u : 0u);
        }
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (!FREE)
            if (!((mine >> (4 * half) >> (8 * (e >> 2) + (e & 3))) & 1)) s[e] = -INFINITY;
          top = fmaxf(top, s[e]);
        }
        top = max_halves(top) * unit;
        const bool moved = top > mx + kSlack;
        if (__ballot(moved)) {
          const float m_new = moved ? top : mx;
          const float alpha = moved ? __builtin_amdgcn_exp2f(mx - m_new) : 1.f;
          l *= alpha;
#pragma unroll
          for (int i = 0; i < HD / 32; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
          mx = m_new;
        }
        const float nm = kLift<F> - (mx == -INFINITY ? 0.f : mx);
        if constexpr (T::kOwn) {
          if constexpr (!k8) {
            if (more) loads_left<T::kLoads>();
            else loads_left<0>();
          }
          if constexpr (!FREE)
            if (key0 + 32 > n_keys || here != 3u) tl.clear(t, n_keys, here);
        }
        // Sixteen keys at a time: the next ones' weights are formed while the matrix
        // cores work.
        auto weigh = [&](uint4 (&pb)[2], int ks) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[8 * ks + e], unit, nm));
            s[8 * ks + e] = x;
            l += x;  // this lane's keys; the halves meet at the end
          }
          weight_words<F>(pb, [&](int e) { return s[8 * ks + e]; });
        };
        uint4 pb[2][2];
        weigh(pb[0], 0);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          bf16x8_t vf[HD / 32];
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            vf[i] = to.frag_t(tl.tile(1, t), 2 * t32 + ks, i);
            if constexpr (!FREE)
              if (odd) vf[i] = finite_part<F>(vf[i]);
          }
          if (ks == 0) weigh(pb[1], 1);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) o[i] = mfma16<F>(vf[i], __builtin_bit_cast(bf16x8_t, pb[ks][x]), o[i]);
        }
        if constexpr (!FREE)
          if (odd) {
            // what finite_part took out, added to the rows that see it
#pragma unroll 1
            for (int x = 0; x < 32; ++x) {
              float p = 0.f;
#pragma unroll
              for (int e = 0; e < 16; ++e) p = 4 * (x >> 3) + (x & 3) == e ? s[e] : p;
              p = __shfl(p, l32 + 32 * ((x >> 2) & 1), 64);
              if ((mine >> x) & 1) {
                const int r = 32 * t32 + x;
#pragma unroll
                for (int i = 0; i < HD / 32; ++i)
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    const int d = 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
                    const float y =
                        F::to_f(*reinterpret_cast<const uint16_t*>(tl.tile(1, t) + toff<HD>(r, d >> 3) + (d & 7) * 2));
                    if (!(fabsf(y) < INFINITY)) o[i][e] = fmaf(p, y, o[i][e]);
                    __builtin_amdgcn_sched_barrier(0);  // one at a time: 64 reads in flight would cost the registers
                  }
              }
            }
          }
      }
      if (more) {
        if constexpr (!T::kOwn) {
          if constexpr (k8) {
            tl.put(t + 1, 0);
            tl.put(t + 1, 1);
          }
        } else if constexpr (!k8) {
          reads_done();
          tl.fetch(a, g, t + 1, 1);
        } else {
          tl.put(t + 1, 1);
          if (t + 2 < n_tiles) tl.fetch(a, g, t + 2, 1);
        }
      }
    };

    // A pass over the tiles.  Where a sum is not finite an infinity or NaN of V may
    // have met the zero weight of a row that does not see it, or a zero among a
    // weight's terms: then the pass is made again, with the finite part multiplied
    // and the rest added where it is seen.
    for (;;) {
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
      mx = -INFINITY;
      l = 0.f;
      if (n_tiles == 0) break;
      if (odd) tl.begin(a, k.b);
      tl.fetch(a, g, 0, 0);
      tl.fetch(a, g, 0, 1);
      if constexpr (k8) {
        tl.put(0, 0);
        tl.put(0, 1);
        if (T::kOwn && n_tiles > 1) {
          tl.fetch(a, g, 1, 0);
          tl.fetch(a, g, 1, 1);
        }
      }
      // pages that are missing are found a batch of tiles at a time
#pragma clang loop unroll(disable)
      for (int t = 0; t < n_tiles;) {
        const int stop = min(n_tiles, t + T::kBatch);
        there = __ballot(tl.ids >= 0);
        const bool whole = !odd && (there | __ballot(tl.key_of_id(t) >= tl.k_hi)) == ~0ull;
        const int free_stop = whole ? min(stop, free_tiles) : t;
#pragma clang loop unroll(disable)
        for (; t < free_stop; ++t) step(t, std::true_type{});
#pragma clang loop unroll(disable)
        for (; t < stop; ++t) step(t, std::false_type{});
      }
      float zero = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) zero = fmaf(o[i][e], 0.f, zero);
      const bool nan = zero != 0.f;
      if (odd || (T::kOwn ? __ballot(nan) == 0 : __syncthreads_or(nan) == 0)) break;
      odd = true;
    }

    // the waves' sums, those of the same rows joined in a fixed order
    l = sum_halves(l);
    if constexpr (!T::kOwn) __syncthreads();  // the last tile has been read
    char* mine = smem + tl.wave * 64 * HD * 2;
    float4* park = reinterpret_cast<float4*>(mine);  // [HD / 4][32], rows swapped about against bank conflicts
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d4 = 8 * i + 2 * q + half;
        park[d4 * 32 + (l32 ^ (d4 & 31))] = make_float4(o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]);
      }
    if (half == 0) {
      ml[tl.wave][l32][0] = mx;
      ml[tl.wave][l32][1] = l;
    }
    __syncthreads();
    for (int e = tid; e < BM * (HD / 4); e += 64 * W) {
      const int x = e / (HD / 4) % 32, y_rg = e / (HD / 4) / 32, d4 = e % (HD / 4), mm = rw.m0 + 32 * y_rg + x;
      if (mm >= rw.count) break;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < KG; ++i) top = fmaxf(top, ml[y_rg + RG * i][x][0]);
      float sum = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < KG; ++i) {
        const int from = y_rg + RG * i;
        // a wave that saw nothing holds zeros; one whose scores are NaN has no
        // maximum either, and its sums are NaN
        const float f = ml[from][x][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[from][x][0] - top);
        const float4 z = reinterpret_cast<const float4*>(smem + from * 64 * HD * 2)[d4 * 32 + (x ^ (d4 & 31))];
        sum = fmaf(f, ml[from][x][1], sum);
        y.x = fmaf(f, z.x, y.x);
        y.y = fmaf(f, z.y, y.y);
        y.z = fmaf(f, z.z, y.z);
        y.w = fmaf(f, z.w, y.w);
      }
      const int to_row = rw.row(mm), head = g * rw.G + mm % rw.G;
      if (top == -INFINITY && sees_any(a, k.b, tl.k_lo, tl.k_hi, rw, to_row)) top = kAllInf;
      if (k.parts == 1) {
        const float inv = top == -INFINITY ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + (int64_t)to_row * a.ldo + head * HD + 4 * d4) =
            make_uint2(F::pack2(y.x * inv, y.y * inv), F::pack2(y.z * inv, y.w * inv));
      } else {
        const int64_t at_row = ((int64_t)to_row * a.H + head) * a.nsplit + k.part;
        *reinterpret_cast<float4*>(a.part + at_row * HD + 4 * d4) = y;
        if (d4 == 0) {
          float* s2 = a.part + (int64_t)a.rows * a.H * a.nsplit * HD + at_row * 2;
          s2[0] = top;
          s2[1] = sum;
        }
      }
    }
  };
  Share share(a, w, lane);
  while (share.at < share.end) {
    const Share::Block k = share.next(a, w, lane);
    if (g == 0 && k.part == 0 && tid == 0 && a.parts) a.parts[(int64_t)k.b * a.nqb + k.qb] = k.parts;
    block(k);
    if (share.at < share.end) __syncthreads();  // the sums have been read
  }
}

template <typename F, int HD, bool k8>
void run(const LzPagedArgs& a, uint32_t blocks, hipStream_t s) {
  if (a.bm != 32) tree_kernel<F, HD, k8, 2, 4><<<blocks, 256, 0, s>>>(a);
  else if (a.waves == 8) tree_kernel<F, HD, k8, 1, 8><<<blocks, 512, 0, s>>>(a);
  else tree_kernel<F, HD, k8, 1, 4><<<blocks, 256, 0, s>>>(a);
}

}  // namespace

int lz_tree_tiles(const LzPagedArgs& a, int dtype, bool e4m3, int64_t hd, uint32_t blocks, hipStream_t s) {
#define RUN(HD)                                          \
  do {                                                   \
    if (dtype == LZ_F16) {                               \
      if (e4m3) run<FmtF16, HD, true>(a, blocks, s);     \
      else run<FmtF16, HD, false>(a, blocks, s);         \
    } else {                                             \
      if (e4m3) run<FmtBF16, HD, true>(a, blocks, s);    \
      else run<FmtBF16, HD, false>(a, blocks, s);        \
    }                                                    \
  } while (0)
  if (hd == 32) RUN(32);
  else if (hd == 64) RUN(64);
  else RUN(128);
#undef RUN
  return lz_check_launch("lz_tree_attn");
}

// Verification of drafted tokens against the model's logits, from given random
// numbers.
//
// Row i of a sequence holds the logits of what follows its node i; with the
// temperature T, p = softmax(x / T), or all of it on the arg-max where T <= 0.
//
//   without draft probabilities (a tree): t_i = the first token whose sum of p up
//     to it is over u_i; from the root on, the walk goes to the first child that
//     holds t_i, and ends with t_i where there is none.
//   with them (a chain): node j, drawn from q_j, is kept while u_j q_j(x_j) <
//     p_{j-1}(x_j); the token after the last kept one is chosen with u_0 from
//     max(p - q, 0) of the node that was not kept, or from p after the last.
//
// A choice falls on another token where an error in the sums crosses a token's
// border: in fp32 (2^-24) that is one row in a few hundred of a flat vocabulary of
// 128000, so weights and sums are formed in fp64, to 2^-39 or better.  A weight is
// 2^((x - m) log2(e) / T): its exponent in 32nds is rounded by adding 1.5 * 2^52,
// 2^(k/32) comes from a table (32 doubles fill LDS's 64 banks once, so any lanes
// read it without a conflict) and 2^(f/32), |f| <= 1/2, from the Taylor series to
// the fourth power (1.3e-12; in a loop by itself 1.9 T weights a second, where the
// series of 2^f to the tenth power makes 1.4).  That arithmetic bounds stats_kernel
// (16 trees of up to 32 nodes, 304 rows of 128256 in bf16: 33 us for 78 MB of
// logits; 8.3 to choose, 4.7 to walk).
//
// Every logit is read once: stats_kernel leaves each piece's largest logit and
// its sum of weights, a wave for each piece and no meeting of waves.  What remains
// works on pieces: a wave joins a row's sums, finds the piece that the choice falls
// into and goes over that one alone.  All rows of a tree choose at the same time,
// a wave each, and one wave walks through the choices in LDS.
#include <cfloat>
#include <type_traits>

#include "draft.h"
#include "kvcache.h"

namespace {

constexpr int kVec = 512;  // logits that a wave loads at a time, eight a lane

struct Piece {
  double sum;  // of 2^((x - top) log2(e) / T); NaN where no choice can be made
  float top;
  int arg;  // the first token with it
};

struct VerifyArgs {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  const void* uniform;
  const int32_t* row_start;
  const float* heat;  // [B]; null: heat_s
  const int32_t* parents;  // [B or 1][nodes], null: a chain
  const float* probs;
  int64_t ldp, ldq;
  Piece* pieces;  // [rows][n_pieces]
  double* rest;   // [B][n_pieces]
  int32_t* stop;  // [B]: the last kept node
  int32_t* choice;  // [rows]: what pick_kernel chose; null: walk_kernel chooses
  int32_t* counts;
  int32_t* kept;   // [B][nodes]
  int64_t* chosen;  // [B][nodes]
  float heat_s;
  int u_double, rows, B, V, nodes, n_pieces, piece, tree_nodes;
};

typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(2)));  // of rows that start anywhere

// 2^(k / 32)
__constant__ const double kRoots[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};

// A workgroup's table of them, in LDS, and 2^(t / 32).  With t = n + f the result
// is 2^(n >> 5) 2^((n & 31) / 32) 2^(f / 32): the exponent is added to the table's
// value, from which the part that n & 31 adds too is taken beforehand.
struct Exp {
  const int2* roots;

  // With the whole workgroup, before any use.
  __device__ __forceinline__ explicit Exp(int2* lds) : roots(lds) {
    const int k = threadIdx.x;
    if (k < 32) lds[k] = make_int2(__double2loint(kRoots[k]), __double2hiint(kRoots[k]) - (k << 15));
    __syncthreads();
  }
  // t <= 0 as two factors; below -32000 as -32000 (no sum of weights up to 1 holds
  // those), NaN too.
  __device__ __forceinline__ void parts(double t, double& series, double& power) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    t = fmax(t, -32000.0);
    const double z = t + kRound, f = t - (z - kRound);
    const int n = __double2loint(z);
    double p = 9.172562701824643e-09;  // (ln 2 / 32)^k / k!
    p = fma(p, f, 1.6938509724371819e-06);
    p = fma(p, f, 0.00023459619820224677);
    p = fma(p, f, 0.02166084939249829);
    series = fma(p, f, 1.0);
    const int2 r = roots[n & 31];
    power = __hiloint2double((int)(((uint32_t)n << 15) + (uint32_t)r.y), r.x);
  }
  __device__ __forceinline__ double operator()(double t) const {
    double series, power;
    parts(t, series, power);
    return series * power;
  }
  __device__ __forceinline__ void add_to(double& sum, double t) const {
    double series, power;
    parts(t, series, power);
    sum = fma(series, power, sum);
  }
};

// 32 log2(e) / T, or 0 where the arg-max is chosen.
__device__ __forceinline__ double per_heat(const VerifyArgs& a, int b) {
  const float t = a.heat ? a.heat[b] : a.heat_s;
  return t > 0.f ? 46.16624130844683 / (double)fminf(t, FLT_MAX) : 0.0;  // (an infinite T, too, takes from all alike)
}

// A row's number: below 0, and NaN, as 0; from 1 on as the double under it.
__device__ __forceinline__ double uniform_of(const VerifyArgs& a, int row) {
  const double u = a.u_double ? static_cast<const double*>(a.uniform)[row] : (double)static_cast<const float*>(a.uniform)[row];
  return fmin(fmax(u, 0.0), 0x1.fffffffffffffp-1);
}

// Eight logits of a row from v on; -inf past the vocabulary.
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* row, int v, int V) {
  if (v + 8 <= V) {
    T raw[8];
#pragma unroll
    for (int w = 0; w < (int)sizeof(T) / 2; ++w)
      reinterpret_cast<Words4*>(raw)[w] = reinterpret_cast<const Words4*>(row + v)[w];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::load(raw, e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = v + e < V ? Elem<T>::load(row, v + e) : -INFINITY;
  }
}

// A token's weight beside the largest logit `top` (finite).  Where it is no double
// above 0 (under 2^-1075), as a mask of the type's lowest value makes it, there is
// none: a number of 0 would choose it.
__device__ __forceinline__ double weight(const Exp& exp, float x, float top, double c) {
  const double t = ((double)x - (double)top) * c;  // -inf too
  return t < -34400.0 ? 0.0 : exp(t);
}

// Sums over the wave of the lanes up to this one, with DPP (row_shr 1, 2, 4, 8,
// row_bcast 15, 31): a tenth of the time of six shuffles through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ double shifted(double x) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROWS, 0xf, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ double sum_up_to(double x) {
  x += shifted<0x111, 0xf>(x);
  x += shifted<0x112, 0xf>(x);
  x += shifted<0x114, 0xf>(x);
  x += shifted<0x118, 0xf>(x);
  x += shifted<0x142, 0xa>(x);
  x += shifted<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double of_lane(double x, int lane) {  // a uniform lane
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane),
                          __builtin_amdgcn_readlane(__double2loint(x), lane));
}
__device__ __forceinline__ double sum_of_wave(double x) { return of_lane(sum_up_to(x), 63); }
template <int CTRL, int ROWS, typename Op>
__device__ __forceinline__ int fold(int x, int none, const Op& op) {
  return op(x, __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false));
}
template <typename Op>
__device__ __forceinline__ int of_wave(int x, int none, const Op& op) {
  x = fold<0x111, 0xf>(x, none, op);
  x = fold<0x112, 0xf>(x, none, op);
  x = fold<0x114, 0xf>(x, none, op);
  x = fold<0x118, 0xf>(x, none, op);
  x = fold<0x142, 0xa>(x, none, op);
  x = fold<0x143, 0xc>(x, none, op);
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int least_of_wave(int x) {
  return of_wave(x, INT32_MAX, [](int a, int b) { return min(a, b); });
}
// The largest of the lanes' floats (none of them NaN).
__device__ __forceinline__ float largest_of_wave(float x) {
  return __int_as_float(of_wave(__float_as_int(x), __float_as_int(-INFINITY),
                                [](int a, int b) { return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b))); }));
}

// A row's rows of the call, bounded: lo .. lo + n - 1.
struct Nodes {
  int lo, n;
  __device__ __forceinline__ Nodes(const VerifyArgs& a, int b) {
    lo = min(max(a.row_start[b], 0), a.rows);
    n = min(min(max(a.row_start[b + 1], lo), a.rows) - lo, a.nodes);
  }
};

// NV vectors of a piece, a wave each.
template <typename T, int NV>
__global__ void __launch_bounds__(256) stats_kernel(VerifyArgs a) {
  __shared__ int2 roots[32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t per_row = (uint32_t)(a.n_pieces + 3) / 4;
  const int row = (int)(blockIdx.x / per_row), p = (int)(blockIdx.x % per_row) * 4 + wave;
  const T* x_row = static_cast<const T*>(a.logits) + row * a.ld;
  float x[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) load8(x[k], x_row, (p * NV + k) * kVec + lane * 8, a.V);
  const Exp exp(roots);
  if (p >= a.n_pieces) return;
  const int b = a.heat ? lz_seq_of_row(a.row_start, a.B, a.rows, row) : 0;
  const double c = b < 0 ? 0.0 : per_heat(a, b);

  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, x[k][e]);
      nan |= x[k][e] != x[k][e];
    }
  top = largest_of_wave(top);
  nan = __ballot(nan) != 0;
  int arg = 0;
  double sum = 0.0;
  if (c == 0.0) {
    arg = INT32_MAX;
#pragma unroll
    for (int k = NV - 1; k >= 0; --k)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[k][e] == top) arg = (p * NV + k) * kVec + lane * 8 + e;
    arg = least_of_wave(arg);
  } else if (top > -INFINITY && top < INFINITY) {
    // (tokens that may not be chosen add 2^-1000 beside a sum of 1 or more)
    // (the largest's is 1: equal logits' sums are whole numbers)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) exp.add_to(sum, ((double)x[k][e] - (double)top) * c);
    sum = sum_of_wave(sum);
  }
  if (lane == 0) {
    Piece s;
    s.sum = nan || top == INFINITY ? __builtin_nan("") : sum;
    s.top = nan ? __builtin_nanf("") : top;
    s.arg = arg;
    a.pieces[(int64_t)row * a.n_pieces + p] = s;
  }
}

// A row's largest logit (NaN where there is one among them), the first token
// that has it (where the arg-max is chosen) and the sum of its weights, with a
// whole wave.
struct Row {
  const Piece* pieces;
  double c, sum;
  double mine;  // lane's piece of the first 64
  float top;
  int arg;

  __device__ __forceinline__ Row(const VerifyArgs& a, const Exp& exp, int row, double c_, int lane)
      : pieces(a.pieces + (int64_t)row * a.n_pieces), c(c_), sum(0.0), mine(0.0), top(-INFINITY), arg(INT32_MAX) {
    bool nan = false;
    for (int p = lane; p < a.n_pieces; p += 64) {
      const Piece s = pieces[p];
      nan |= s.top != s.top;
      if (s.top > top) {
        top = s.top;
        arg = s.arg;
      }
    }
    const float all = largest_of_wave(top);
    if (c == 0.0) arg = least_of_wave(top == all ? arg : INT32_MAX);
    top = __ballot(nan) ? __builtin_nanf("") : all;
    if (c != 0.0 && fine()) {
      double x = 0.0;
      for (int p = lane; p < a.n_pieces; p += 64) {
        const double y = of_piece(exp, p);
        if (p < 64) mine = y;
        x += y;
      }
      sum = sum_of_wave(x);
    }
  }
  // a piece's sum beside the row's largest logit
  __device__ __forceinline__ double of_piece(const Exp& exp, int p) const {
    const Piece s = pieces[p];
    return s.sum * weight(exp, s.top, top, c);
  }
  // whether a token can be chosen
  __device__ __forceinline__ bool fine() const {
    return c == 0.0 ? top > -INFINITY : top > -INFINITY && top < INFINITY;  // not for NaN
  }
};

// The first token whose sum up to it is over u times the sum of all, and the
// last one with a weight where rounding leaves none; -1 where all are zero.
// of_piece(p): a piece's sum; of_tokens(v, w): eight tokens' weights.
template <int NV, typename OfPiece, typename OfTokens>
__device__ __forceinline__ int pick(const VerifyArgs& a, double u, int lane, const OfPiece& of_piece, const OfTokens& of_tokens) {
  auto piece_sum = [&](int p0) { return p0 + lane < a.n_pieces ? of_piece(p0 + lane) : 0.0; };
  const double x0 = piece_sum(0), up0 = sum_up_to(x0);
  double all = of_lane(up0, 63);
  for (int p0 = 64; p0 < a.n_pieces; p0 += 64) all += sum_of_wave(piece_sum(p0));
  if (!(all > 0.0)) return -1;
  double target = u * all, run = 0.0;
  int piece = -1, last = 0;
  for (int p0 = 0; p0 < a.n_pieces; p0 += 64) {
    const double x = p0 ? piece_sum(p0) : x0, up_to = p0 ? sum_up_to(x) : up0;
    const uint64_t over = __ballot(x > 0.0 && run + up_to > target), some = __ballot(x > 0.0);
    if (over) {
      const int l = __builtin_ctzll(over);
      piece = p0 + l;
      run += of_lane(up_to, l) - of_lane(x, l);
      break;
    }
    if (some) last = p0 + 63 - __builtin_clzll(some);
    run += of_lane(up_to, 63);
  }
  if (piece < 0) {  // u is just under 1
    piece = last;
    target = INFINITY;
  }
  // a lane's tokens are adjacent: one sum over the lanes finds the one that holds it
  double w[NV][8], x = 0.0;
  const int v0 = piece * a.piece + lane * 8 * NV;
  int mine = -1;  // this lane's last token with a weight
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    of_tokens(v0 + 8 * k, w[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x += w[k][e];
      mine = w[k][e] > 0.0 ? v0 + 8 * k + e : mine;
    }
  }
  const double up_to = sum_up_to(x);
  const uint64_t over = __ballot(x > 0.0 && run + up_to > target), some = __ballot(x > 0.0);
  double at = run + (up_to - x);
  int token = mine;
  bool done = false;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      at += w[k][e];
      if (!done && w[k][e] > 0.0 && at > target) {
        token = v0 + 8 * k + e;
        done = true;
      }
    }
  if (over) return __builtin_amdgcn_readlane(token, __builtin_ctzll(over));
  return some ? __builtin_amdgcn_readlane(mine, 63 - __builtin_clzll(some)) : -1;
}

template <typename T, int NV>
__device__ __forceinline__ int pick_row(const VerifyArgs& a, const Exp& exp, const Row& r, int row, double u, int lane) {
  if (!r.fine()) return -1;
  if (r.c == 0.0) return r.arg;
  const T* x_row = static_cast<const T*>(a.logits) + row * a.ld;
  return pick<NV>(a, u, lane, [&](int p) { return p < 64 ? r.mine : r.of_piece(exp, p); },
                  [&](int v, double (&w)[8]) {
                    float x[8];
                    load8(x, x_row, v, a.V);
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = weight(exp, x[e], r.top, r.c);
                  });
}

// Every row's choice, a wave each.
template <typename T, int NV>
__global__ void __launch_bounds__(256) pick_kernel(VerifyArgs a) {
  __shared__ int2 roots[32];
  const Exp exp(roots);
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int b = a.heat ? lz_seq_of_row(a.row_start, a.B, a.rows, row) : 0;
  if (b < 0) return;
  const int t = pick_row<T, NV>(a, exp, Row(a, exp, row, per_heat(a, b), lane), row, uniform_of(a, row), lane);
  if (lane == 0) a.choice[row] = t;
}

// Without draft probabilities: one workgroup a sequence, which chooses for a few
// rows itself.
template <typename T, int NV>
__global__ void __launch_bounds__(1024) walk_kernel(VerifyArgs a) {
  __shared__ int2 roots[32];
  __shared__ int choice[kMostNodes], token[kMostNodes], parent[kMostNodes], path[kMostNodes];
  __shared__ int n_path;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Exp exp(roots);
  const Nodes s(a, b);
  const double c = per_heat(a, b);
  for (int i = tid; i < s.n; i += blockDim.x) {
    const int64_t t = a.tokens[s.lo + i];
    token[i] = t >= 0 && t < a.V ? (int)t : -2;
    parent[i] = a.parents && i < a.tree_nodes ? a.parents[b * a.ldp + i] : -1;
    if (a.choice) choice[i] = a.choice[s.lo + i];
  }
  for (int i = wave; i < s.n && !a.choice; i += 16) {
    const int t = pick_row<T, NV>(a, exp, Row(a, exp, s.lo + i, c, lane), s.lo + i, uniform_of(a, s.lo + i), lane);
    if (lane == 0) choice[i] = t;
  }
  __syncthreads();
  if (wave == 0) {
    int node = 0, count = 0;
    while (node < s.n) {
      if (lane == 0) path[count] = node;
      ++count;
      const int want = choice[node];
      int next = s.n;
      if (want < 0) break;
      if (!a.parents) {
        if (node + 1 < s.n && token[node + 1] == want) next = node + 1;
      } else {
        for (int i0 = node + 1; i0 < s.n; i0 += 64) {
          const int i = i0 + lane;
          const uint64_t ok = __ballot(i < s.n && parent[i] == node && token[i] == want);
          if (ok) {
            next = i0 + __builtin_ctzll(ok);
            break;
          }
        }
      }
      node = next;
    }
    if (lane == 0) n_path = count;
  }
  __syncthreads();
  const int count = n_path;
  if (tid == 0) a.counts[b] = count;
  for (int j = tid; j < a.nodes; j += blockDim.x) {
    a.kept[(int64_t)b * a.nodes + j] = j < count ? path[j] : -1;
    a.chosen[(int64_t)b * a.nodes + j] = j < count ? choice[path[j]] : -1;
  }
}

// With them: each workgroup of a sequence finds where its chain ends, four rows
// at a time, and sums what is left of p beside q over four pieces of that row.
template <typename T>
__global__ void __launch_bounds__(256) rest_kernel(VerifyArgs a) {
  __shared__ int2 roots[32];
  __shared__ int kept[4];
  const Exp exp(roots);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t groups = (uint32_t)(a.n_pieces + 3) / 4;
  const int b = (int)(blockIdx.x / groups), p = (int)(blockIdx.x % groups) * 4 + wave;
  const Nodes s(a, b);
  if (s.n == 0) return;
  const double c = per_heat(a, b);
  int stop = 0;
  for (bool more = true; more;) {
    const int node = stop + wave + 1;  // is it kept?
    bool ok = false;
    if (node < s.n) {
      const int64_t t = a.tokens[s.lo + node];
      const int row = s.lo + node - 1;
      const Row r(a, exp, row, c, lane);
      if (t >= 0 && t < a.V && r.fine()) {
        const float x = Elem<T>::load(static_cast<const T*>(a.logits) + row * a.ld, t);
        if (c == 0.0) ok = t == r.arg;
        else ok = uniform_of(a, s.lo + node) * (double)a.probs[(s.lo + node) * a.ldq + t] < weight(exp, x, r.top, c) / r.sum;
      }
    }
    if (lane == 0) kept[wave] = ok;
    __syncthreads();
    int run = 0;
    while (run < 4 && kept[run]) ++run;
    __syncthreads();
    stop += run;
    more = run == 4;
  }
  if (threadIdx.x == 0 && p == 0) a.stop[b] = stop;
  if (p >= a.n_pieces || c == 0.0) return;
  const int row = s.lo + stop;
  const Row r(a, exp, row, c, lane);
  double rest = 0.0;
  if (stop + 1 < s.n && r.fine()) {
    const T* x_row = static_cast<const T*>(a.logits) + row * a.ld;
    const float* q_row = a.probs + (row + 1) * a.ldq;
    const double per = 1.0 / r.sum;
    for (int v = p * a.piece + lane * 8; v < min((p + 1) * a.piece, a.V); v += kVec) {
      float x[8], q[8];
      load8(x, x_row, v, a.V);
      load8(q, q_row, v, a.V);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e < a.V) rest += fmax(weight(exp, x[e], r.top, c) * per - (double)q[e], 0.0);
    }
    rest = sum_of_wave(rest);
  }
  if (lane == 0) a.rest[(int64_t)b * a.n_pieces + p] = rest;
}

// The token after a chain's last kept one, a wave for each sequence.
template <typename T, int NV>
__global__ void __launch_bounds__(64) end_kernel(VerifyArgs a) {
  __shared__ int2 roots[32];
  const Exp exp(roots);
  const int b = blockIdx.x, lane = threadIdx.x;
  const Nodes s(a, b);
  int count = 0, last = -1;
  if (s.n > 0) {
    const int stop = a.stop[b], row = s.lo + stop;
    const double c = per_heat(a, b), u = uniform_of(a, s.lo);
    count = stop + 1;
    const Row r(a, exp, row, c, lane);
    if (c != 0.0 && r.fine() && stop + 1 < s.n) {
      const T* x_row = static_cast<const T*>(a.logits) + row * a.ld;
      const float* q_row = a.probs + (row + 1) * a.ldq;
      const double* rest = a.rest + (int64_t)b * a.n_pieces;
      const double per = 1.0 / r.sum;
      last = pick<NV>(a, u, lane, [&](int p) { return rest[p]; },
                  [&](int v, double (&w)[8]) {
                    float x[8], q[8];
                    load8(x, x_row, v, a.V);
                    load8(q, q_row, v, a.V);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                      w[e] = v + e < a.V ? fmax(weight(exp, x[e], r.top, c) * per - (double)q[e], 0.0) : 0.0;
                  });
    }
    if (last < 0) last = pick_row<T, NV>(a, exp, r, row, u, lane);  // nothing of q was not kept, or p is q
  }
  if (lane == 0) a.counts[b] = count;
  for (int j = lane; j < a.nodes; j += 64) {
    a.kept[(int64_t)b * a.nodes + j] = j < count ? j : -1;
    a.chosen[(int64_t)b * a.nodes + j] = j + 1 < count ? a.tokens[s.lo + j + 1] : j + 1 == count ? last : -1;
  }
}

// Pieces of 512 logits, of 2048 where those of 512 are more than a wave's lanes
// and more than two for every wave that the CUs hold: large calls then join fewer
// (32 chains of up to 8 over 128256 in fp32, drawn: 38.5 us, in short ones 45),
// small ones have more waves (4 of up to 5: 21.8 and 19.2, sampled 13.3 and 11.8).
int vectors(int64_t V, int64_t rows) { return V > 64 * kVec && rows * lz_cdiv(V, kVec) > 16384 ? 4 : 1; }

}  // namespace

LZ_EXPORT int64_t lz_verify_workspace(int64_t rows, int64_t B, int64_t V, int drawn) {
  if (rows <= 0 || B <= 0 || V <= 0 || V > (1 << 28)) return 0;
  const int64_t pieces = lz_cdiv(V, kVec * vectors(V, rows));
  return rows * pieces * (int64_t)sizeof(Piece) + (drawn ? B * pieces * 8 + B * 4 : rows * 4);
}

LZ_EXPORT int lz_verify_draft(const void* logits, int64_t ld, int dtype, int64_t rows, int64_t V, const int64_t* tokens,
                              const void* uniform, int u_double, const int32_t* row_start, int64_t B, int64_t nodes,
                              const float* temperature, float temperature_s, const int32_t* parents, int64_t ldp,
                              int64_t tree_nodes, const float* probs, int64_t ldq, int32_t* counts, int32_t* kept,
                              int64_t* chosen, void* workspace, int64_t ws_bytes, void* stream) {
  LZ_REQUIRE(dtype == LZ_BF16 || dtype == LZ_F16 || dtype == LZ_F32, "lz_verify_draft: bad dtype %d", dtype);
  LZ_REQUIRE(rows >= 0 && rows <= INT32_MAX - 4 && V > 0 && V <= (1 << 28) && B > 0 && B <= INT32_MAX / 256,
             "lz_verify_draft: bad shape");
  LZ_REQUIRE(nodes > 0 && nodes <= kMostNodes, "lz_verify_draft: %lld nodes a sequence (1 to %d)", (long long)nodes, kMostNodes);
  LZ_REQUIRE(!(parents && probs), "lz_verify_draft: draft probabilities are for chains");
  LZ_REQUIRE(!parents || (tree_nodes > 0 && tree_nodes <= INT32_MAX && (ldp == 0 || ldp >= tree_nodes)),
             "lz_verify_draft: trees of %lld nodes", (long long)tree_nodes);
  LZ_REQUIRE(row_start && counts && kept && chosen, "lz_verify_draft: bad arguments");
  LZ_REQUIRE(rows == 0 || (logits && tokens && uniform && (rows == 1 || (ld >= V && (!probs || ldq >= V)))),
             "lz_verify_draft: bad rows");
  const int nv = vectors(V, rows);
  const int64_t pieces = lz_cdiv(V, kVec * nv), need = lz_verify_workspace(rows, B, V, probs != nullptr);
  LZ_REQUIRE(need == 0 || (workspace && lz_aligned16(workspace) && ws_bytes >= need),
             "lz_verify_draft: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  const int64_t stats = rows * lz_cdiv(pieces, 4), rests = B * lz_cdiv(pieces, 4);
  LZ_REQUIRE(stats <= INT32_MAX / 256 && rests <= INT32_MAX / 256, "lz_verify_draft: too many rows");
  Piece* at = static_cast<Piece*>(workspace);
  double* rest = reinterpret_cast<double*>(at + rows * pieces);
  // 4 x 5 rows of 32000, sampled: 9.0 us with the choices in the walk, 11.9 apart;
  // 64 x 14 22.7 and 24.8, 16 x 32 21.9 and 20.2, 1 x 60 19.0 and 12.0; 64 x 8 of
  // 128256 38 and 41, 16 x 16 33.5 and 32.4, 16 x 32 52 and 42
  const bool apart = !probs && rows > 0 && nodes > 16;
  VerifyArgs a{logits, ld, tokens, uniform, row_start, temperature, parents, probs, ldp, ldq, at, rest,
               reinterpret_cast<int32_t*>(rest + B * pieces), apart ? reinterpret_cast<int32_t*>(rest) : nullptr, counts, kept,
               chosen, temperature_s, u_double,
               (int)rows, (int)B, (int)V, (int)nodes, (int)pieces, kVec * nv, (int)tree_nodes};
  hipStream_t s = lz_stream(stream);
#define RUN_PIECES(T, NV)                                                   \
  do {                                                                      \
    if (stats > 0) stats_kernel<T, NV><<<(uint32_t)stats, 256, 0, s>>>(a);  \
    if (probs) {                                                            \
      rest_kernel<T><<<(uint32_t)rests, 256, 0, s>>>(a);                    \
      end_kernel<T, NV><<<(uint32_t)B, 64, 0, s>>>(a);                      \
    } else {                                                                \
      if (apart) pick_kernel<T, NV><<<(uint32_t)lz_cdiv(rows, 4), 256, 0, s>>>(a); \
      walk_kernel<T, NV><<<(uint32_t)B, apart ? 256 : 1024, 0, s>>>(a);     \
    }                                                                       \
  } while (0)
#define RUN(T)                      \
  do {                              \
    if (nv == 4) RUN_PIECES(T, 4);  \
    else RUN_PIECES(T, 1);          \
  } while (0)
  if (dtype == LZ_BF16) RUN(uint16_t);
  else if (dtype == LZ_F16) RUN(_Float16);
  else RUN(float);
#undef RUN
#undef RUN_PIECES
  return lz_check_launch("lz_verify_draft");
}

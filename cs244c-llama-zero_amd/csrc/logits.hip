// Adjusting a row of logits before a token is chosen: penalties for tokens of
// the row's text, a bias and a mask of allowed tokens.
//
//   x = logit;  token t is in the text: x = x > 0 ? x / r : x * r
//   x -= f * (times t occurs after the prompt) + p * (1 if it does)
//   x += bias;  t is not allowed: x = -inf
//
// in fp32, whatever the logits' type.  One workgroup owns a slice of a row's
// vocabulary: it counts the text's tokens that fall into the slice in LDS
// (integer adds, so their order does not matter) and goes over the slice once.
// Ids outside the vocabulary count for nothing.
#include "lz_common.h"

namespace {

struct LogitsArgs {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;  // [B][ldt]
  int64_t ldt;
  const int32_t* lengths;  // tokens of a row that count; NULL: n_tokens
  const int32_t* prompts;  // of them, those of the prompt; NULL: none
  const float* rep;        // one for each row, or NULL: the scalar
  const float* pres;
  const float* freq;
  float rep_s, pres_s, freq_s;
  const float* bias;
  int64_t ldb;  // 0: one bias for all rows
  const void* mask;
  int64_t ldm;  // 0: one mask for all rows
  float* out;
  int64_t ldo;
  int B, V, n_tokens, mask_kind;  // mask_kind 0: none, 1: a byte a token, 2: a bit a token
};

typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(2)));  // of any rows

// NV * 2048 tokens of the vocabulary a workgroup: eight adjacent ones a thread
// and vector, whose logits are in flight while the text is counted.  Rows start
// at any element: loads and stores of 16 bytes need no alignment here (36 rows
// of 53151 in fp16 with a bias each: 6.7 us, 13.6 one element at a time).
template <typename T, int NV>
__global__ void __launch_bounds__(256) process_logits_kernel(LogitsArgs a) {
  constexpr int kSlice = NV * 2048;
  __shared__ __attribute__((aligned(16))) uint32_t cnt[kSlice];  // 2 * (times in the answer) + (1 if in the text)
  const int slices = (a.V + kSlice - 1) / kSlice;
  const int b = blockIdx.x / slices, lo = (blockIdx.x % slices) * kSlice;
  const int n = min(kSlice, a.V - lo);
  const int tid = threadIdx.x;
  const T* x_row = static_cast<const T*>(a.logits) + b * a.ld + lo;
  const float* b_row = a.bias ? a.bias + b * a.ldb + lo : nullptr;

  float x[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + tid) * 8;
    if (i + 8 <= n) {
      T raw[8];
#pragma unroll
      for (int w = 0; w < (int)sizeof(T) / 2; ++w)
        reinterpret_cast<Words4*>(raw)[w] = reinterpret_cast<const Words4*>(x_row + i)[w];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = Elem<T>::load(raw, e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] = i + e < n ? Elem<T>::load(x_row, i + e) : 0.f;
    }
  }

  const int len = a.tokens ? (a.lengths ? min(max(a.lengths[b], 0), a.n_tokens) : a.n_tokens) : 0;
  const int prompt = a.prompts ? a.prompts[b] : 0;
  if (len > 0) {  // the same for the whole workgroup
    for (int i = tid; i < kSlice / 4; i += 256) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int64_t* text = a.tokens + b * a.ldt;
#pragma unroll 4
    for (int i = tid; i < len; i += 256) {
      const uint64_t t = (uint64_t)(text[i] - lo);
      if (t < (uint64_t)n) {
        atomicOr(&cnt[t], 1u);
        if (i >= prompt) atomicAdd(&cnt[t], 2u);
      }
    }
    __syncthreads();
  }
  const float r = a.rep ? a.rep[b] : a.rep_s, p = a.pres ? a.pres[b] : a.pres_s, f = a.freq ? a.freq[b] : a.freq_s;

#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = (k * 256 + tid) * 8;
    if (i >= n) break;
    if (len > 0) {
      uint32_t c[8];
      *reinterpret_cast<uint4*>(c) = reinterpret_cast<const uint4*>(cnt + i)[0];
      *reinterpret_cast<uint4*>(c + 4) = reinterpret_cast<const uint4*>(cnt + i)[1];
      if (c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (c[e] & 1) x[k][e] = x[k][e] > 0.f ? x[k][e] / r : x[k][e] * r;
          if (c[e] >> 1) x[k][e] = x[k][e] - f * (float)(c[e] >> 1) - p;
        }
      }
    }
    float y[8] = {};
    if (b_row) {
      if (i + 8 <= n) {
        reinterpret_cast<Words4*>(y)[0] = reinterpret_cast<const Words4*>(b_row + i)[0];
        reinterpret_cast<Words4*>(y)[1] = reinterpret_cast<const Words4*>(b_row + i)[1];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < n) y[e] = b_row[i + e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[k][e] += y[e];
    }
    uint32_t allowed = 0xffu;
    if (a.mask_kind == 2) {  // i and lo are multiples of eight: the bits are in one word
      allowed = static_cast<const uint32_t*>(a.mask)[b * a.ldm + ((lo + i) >> 5)] >> (i & 31);
    } else if (a.mask_kind == 1) {
      const uint8_t* m = static_cast<const uint8_t*>(a.mask) + b * a.ldm + lo + i;
      uint8_t w[8] = {};
      if (i + 8 <= n) __builtin_memcpy(w, m, 8);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < n) w[e] = m[e];
      allowed = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) allowed |= (w[e] != 0) << e;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (allowed >> e) & 1 ? x[k][e] : -INFINITY;
    float* o = a.out + b * a.ldo + lo + i;
    if (i + 8 <= n) {
      reinterpret_cast<Words4*>(o)[0] = reinterpret_cast<const Words4*>(y)[0];
      reinterpret_cast<Words4*>(o)[1] = reinterpret_cast<const Words4*>(y)[1];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < n) o[e] = y[e];
    }
  }
}

}  // namespace

LZ_EXPORT int lz_process_logits(const void* logits, int64_t ld, int dtype, int64_t B, int64_t V, const int64_t* tokens,
                                int64_t ldt, int64_t n_tokens, const int32_t* lengths, const int32_t* prompts,
                                const float* rep, float rep_s, const float* pres, float pres_s, const float* freq,
                                float freq_s, const float* bias, int64_t ldb, const void* mask, int mask_kind,
                                int64_t ldm, float* out, int64_t ldo, void* stream) {
  LZ_REQUIRE(dtype == LZ_BF16 || dtype == LZ_F16 || dtype == LZ_F32, "lz_process_logits: bad dtype %d", dtype);
  LZ_REQUIRE(B >= 0 && V >= 0 && B <= INT32_MAX && V <= (1 << 28) && n_tokens >= 0 && n_tokens <= (1 << 30),
             "lz_process_logits: bad shape");
  LZ_REQUIRE(mask_kind >= 0 && mask_kind <= 2 && (mask_kind == 0) == (mask == nullptr),
             "lz_process_logits: mask kind %d", mask_kind);
  if (B == 0 || V == 0) return LZ_OK;
  LZ_REQUIRE(logits && out && ldo >= V && (B == 1 || ld >= V) && (tokens || n_tokens == 0), "lz_process_logits: bad arguments");
  // small slices where the rows are few and a slice's chain of loads is the
  // time; large ones where each reads a long text again
  const bool small = B * lz_cdiv(V, 8192) < 2 * lz_num_cus();
  const int64_t slices = lz_cdiv(V, small ? 2048 : 8192);
  LZ_REQUIRE(B * slices <= INT32_MAX / 256, "lz_process_logits: too many rows");
  LogitsArgs a{logits, ld, n_tokens ? tokens : nullptr, ldt, lengths, prompts, rep, pres, freq, rep_s, pres_s, freq_s,
               bias, ldb, mask, ldm, out, ldo, (int)B, (int)V, (int)n_tokens, mask_kind};
  const uint32_t grid = (uint32_t)(B * slices);
  hipStream_t s = lz_stream(stream);
#define RUN(T)                                                                           \
  do {                                                                                   \
    if (small) process_logits_kernel<T, 1><<<grid, 256, 0, s>>>(a);                      \
    else process_logits_kernel<T, 4><<<grid, 256, 0, s>>>(a);                            \
  } while (0)
  if (dtype == LZ_BF16) RUN(uint16_t);
  else if (dtype == LZ_F16) RUN(_Float16);
  else RUN(float);
#undef RUN
  return lz_check_launch("lz_process_logits");
}

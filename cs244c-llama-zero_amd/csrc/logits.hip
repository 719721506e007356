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

constexpr int kSlice = 4096;

template <typename T>
__global__ void __launch_bounds__(256) process_logits_kernel(LogitsArgs a) {
  __shared__ uint32_t cnt[kSlice];  // 2 * (times in the answer) + (1 if in the text)
  const int slices = (a.V + kSlice - 1) / kSlice;
  const int b = blockIdx.x / slices, lo = (blockIdx.x % slices) * kSlice;
  const int n = min(kSlice, a.V - lo);
  const int len = a.tokens ? (a.lengths ? min(max(a.lengths[b], 0), a.n_tokens) : a.n_tokens) : 0;
  const int prompt = a.prompts ? a.prompts[b] : 0;
  for (int i = threadIdx.x; i < n; i += 256) cnt[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < len; i += 256) {
    const int64_t t = a.tokens[b * a.ldt + i] - lo;
    if (t >= 0 && t < n) {
      atomicOr(&cnt[t], 1u);
      if (i >= prompt) atomicAdd(&cnt[t], 2u);
    }
  }
  __syncthreads();
  const float r = a.rep ? a.rep[b] : a.rep_s, p = a.pres ? a.pres[b] : a.pres_s, f = a.freq ? a.freq[b] : a.freq_s;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int v = lo + i;
    float x = Elem<T>::load(static_cast<const T*>(a.logits) + b * a.ld, v);
    const uint32_t c = cnt[i];
    if (c & 1) x = x > 0.f ? x / r : x * r;
    if (c >> 1) x = x - f * (float)(c >> 1) - p;
    if (a.bias) x += a.bias[b * a.ldb + v];
    bool ok = true;
    if (a.mask_kind == 1) ok = static_cast<const uint8_t*>(a.mask)[b * a.ldm + v] != 0;
    else if (a.mask_kind == 2) ok = (static_cast<const uint32_t*>(a.mask)[b * a.ldm + (v >> 5)] >> (v & 31)) & 1;
    a.out[b * a.ldo + v] = ok ? x : -INFINITY;
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
  const int64_t slices = lz_cdiv(V, kSlice);
  LZ_REQUIRE(B * slices <= INT32_MAX / 256, "lz_process_logits: too many rows");
  LogitsArgs a{logits, ld, n_tokens ? tokens : nullptr, ldt, lengths, prompts, rep, pres, freq, rep_s, pres_s, freq_s,
               bias, ldb, mask, ldm, out, ldo, (int)B, (int)V, (int)n_tokens, mask_kind};
  const uint32_t grid = (uint32_t)(B * slices);
  hipStream_t s = lz_stream(stream);
  if (dtype == LZ_BF16) process_logits_kernel<uint16_t><<<grid, 256, 0, s>>>(a);
  else if (dtype == LZ_F16) process_logits_kernel<_Float16><<<grid, 256, 0, s>>>(a);
  else process_logits_kernel<float><<<grid, 256, 0, s>>>(a);
  return lz_check_launch("lz_process_logits");
}

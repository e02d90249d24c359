// oxs_logprobs.hip — token log probabilities, entropy, ranks and alternatives
// of whole rows of logits, beside the sampler that draws from them.
//
// With z the (softcapped, scaled) logits of a row's present tokens and m the
// largest, one pass keeps m, s = sum e^(z - m) and t = sum (z - m) e^(z - m):
//   lse = m + ln s,  log p_i = (z_i - m) - ln s,  H = ln s - t / s.
// H's two terms are both >= 0, so nothing cancels.
//
// One workgroup per row; the alternatives are found one after the other, each
// by a pass for the largest key below the last.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/oxide_sampler.h"

namespace oxs_lp {

constexpr int kThreads = 256;
constexpr uint32_t kNoToken = 0xffffffffu;
// e^-200 is 0 in 32 bits: a difference below this (or NaN, of two infinities) adds nothing
constexpr float kFloor = -200.0f;

struct Params {
  oxs_logprobs b;
};

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// The logit of token i, -inf when it is not present.
template <int DT>
__device__ __forceinline__ float present_logit(const oxs_logprobs& b, uint32_t row, uint32_t i) {
  if (i >= b.vocab) return neg_inf();
  const size_t at = (size_t)row * (size_t)b.logits_ld + i;
  float l;
  if constexpr (DT == OXS_DTYPE_F32) l = ((const float*)b.logits)[at];
  else l = __uint_as_float((uint32_t)((const uint16_t*)b.logits)[at] << 16);
  if (l != l) return neg_inf();
  if (b.allowed_mask) {
    const uint32_t w = b.allowed_mask[(size_t)row * (size_t)b.mask_ld + (i >> 5)];
    if (!((w >> (i & 31u)) & 1u)) return neg_inf();
  }
  return l;
}

// Orders tokens: a larger logit first, then the lower id (+0.0 for both zeros).
__device__ __forceinline__ uint64_t key_of(float l, uint32_t i) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((uint64_t)o << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return ~(uint32_t)k; }

__device__ __forceinline__ float softcap(float l, float cap) { return cap > 0.0f ? cap * tanhf(l / cap) : l; }

template <int DT>
__global__ __launch_bounds__(kThreads) void row_kernel(Params p) {
  const oxs_logprobs& b = p.b;
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  __shared__ float s_m[kThreads], s_s[kThreads], s_t[kThreads];
  __shared__ uint64_t s_key[kThreads];
  __shared__ float s_tok[OXS_LOGPROBS_MAX_TOKENS];
  __shared__ uint32_t s_rank[OXS_LOGPROBS_MAX_TOKENS];
  float inv = 1.0f;
  if (b.temperatures) {
    const float t = b.temperatures[row];
    if (t > 1e-6f) inv = 1.0f / t;
  }
  for (uint32_t j = tid; j < b.tokens_per_row; j += kThreads) {
    s_tok[j] = present_logit<DT>(b, row, b.tokens[(size_t)row * (size_t)b.tokens_ld + j]);
    s_rank[j] = 0;
  }
  __syncthreads();
  // z relative to the largest so far, before the temperature
  float m = neg_inf(), s = 0.0f, t = 0.0f;
  for (uint32_t i = tid; i < b.vocab; i += kThreads) {
    const float l = present_logit<DT>(b, row, i);
    if (l == neg_inf()) continue;
    const float y = softcap(l, b.logit_softcap);
    if (y > m) {
      const float d = fmaxf((m - y) * inv, kFloor);
      const float f = expf(d);
      t = f * (t + d * s);
      s = f * s;
      m = y;
    }
    const float q = fmaxf((y - m) * inv, kFloor), e = expf(q);
    s += e;
    t += q * e;
    for (uint32_t j = 0; j < b.tokens_per_row; ++j) {
      const uint32_t id = b.tokens[(size_t)row * (size_t)b.tokens_ld + j];
      if (l > s_tok[j] || (l == s_tok[j] && i < id)) atomicAdd(&s_rank[j], 1u);
    }
  }
  s_m[tid] = m;
  s_s[tid] = s;
  s_t[tid] = t;
  __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) {
    if (tid < (uint32_t)o) {
      const float ma = s_m[tid], mb = s_m[tid + o], mm = fmaxf(ma, mb);
      if (mm != neg_inf()) {
        const float da = fmaxf((ma - mm) * inv, kFloor), db = fmaxf((mb - mm) * inv, kFloor);
        const float fa = expf(da), fb = expf(db);
        const float ta = fa * (s_t[tid] + da * s_s[tid]), tb = fb * (s_t[tid + o] + db * s_s[tid + o]);
        s_s[tid] = fa * s_s[tid] + fb * s_s[tid + o];
        s_t[tid] = ta + tb;
        s_m[tid] = mm;
      }
    }
    __syncthreads();
  }
  m = s_m[0];
  s = s_s[0];
  t = s_t[0];
  const bool empty = m == neg_inf(), over = m == __builtin_inff();
  const float ln_s = empty ? 0.0f : logf(s);
  const auto logprob = [&](float l) {  // of a raw logit
    if (l == neg_inf()) return neg_inf();
    const float y = softcap(l, b.logit_softcap);
    if (over) return y == m ? __builtin_nanf("") : neg_inf();
    return (y - m) * inv - ln_s;
  };
  if (tid == 0) {
    if (b.out_logsumexp) b.out_logsumexp[row] = empty || over ? m : m * inv + ln_s;
    if (b.out_entropy) b.out_entropy[row] = empty ? 0.0f : over ? __builtin_nanf("") : ln_s - t / s;
    if (b.out_status) b.out_status[row] = empty ? OXS_ROW_EMPTY : OXS_ROW_OK;
  }
  for (uint32_t j = tid; j < b.tokens_per_row; j += kThreads) {
    const size_t at = (size_t)row * b.tokens_per_row + j;
    if (b.out_logprobs) b.out_logprobs[at] = logprob(s_tok[j]);
    if (b.out_ranks) b.out_ranks[at] = s_tok[j] == neg_inf() ? 0u : s_rank[j] + 1u;
  }
  uint64_t last = ~0ull;
  for (uint32_t n = 0; n < b.top_n; ++n) {
    uint64_t best = 0;
    for (uint32_t i = tid; i < b.vocab; i += kThreads) {
      const float l = present_logit<DT>(b, row, i);
      if (l == neg_inf()) continue;
      const uint64_t k = key_of(l, i);
      if (k < last && k > best) best = k;
    }
    s_key[tid] = best;
    __syncthreads();
    for (int o = kThreads / 2; o > 0; o >>= 1) {
      if (tid < (uint32_t)o && s_key[tid + o] > s_key[tid]) s_key[tid] = s_key[tid + o];
      __syncthreads();
    }
    best = s_key[0];
    __syncthreads();
    if (tid == 0) {
      const size_t at = (size_t)row * b.top_n + n;
      if (b.out_top_ids) b.out_top_ids[at] = best ? key_id(best) : kNoToken;
      if (b.out_top_logprobs) b.out_top_logprobs[at] = best ? logprob(key_value(best)) : neg_inf();
    }
    last = best;
  }
}

}  // namespace oxs_lp

static bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1u)) == 0; }

extern "C" size_t oxs_logprobs_workspace_bytes(void) { return 16; }

extern "C" int oxs_token_logprobs(const oxs_logprobs* lp, void* stream) {
  if (!lp) return OXS_ERR_INVALID_ARGUMENT;
  const oxs_logprobs& b = *lp;
  if (b.vocab == 0) return OXS_ERR_SHAPE_MISMATCH;
  if (b.rows == 0) return OXS_OK;
  if (b.rows > (1u << 23) || b.vocab > (1u << 30) || b.tokens_per_row > OXS_LOGPROBS_MAX_TOKENS ||
      b.top_n > OXS_LOGPROBS_MAX_TOP)
    return OXS_ERR_LIMITS;
  if (b.logits_dtype != OXS_DTYPE_F32 && b.logits_dtype != OXS_DTYPE_BF16) return OXS_ERR_INVALID_ARGUMENT;
  if (!b.logits || (b.tokens_per_row && !b.tokens) || !b.workspace) return OXS_ERR_INVALID_ARGUMENT;
  if (b.rows > 1 && (b.logits_ld < (int64_t)b.vocab || (b.tokens_per_row && b.tokens_ld < (int64_t)b.tokens_per_row)))
    return OXS_ERR_INVALID_ARGUMENT;
  if (b.allowed_mask && b.mask_ld != 0 && b.mask_ld < (int64_t)((b.vocab + 31u) / 32u)) return OXS_ERR_INVALID_ARGUMENT;
  if (!aligned(b.logits, b.logits_dtype == OXS_DTYPE_F32 ? 4 : 2) || !aligned(b.workspace, 16) ||
      !aligned(b.tokens, 4) || !aligned(b.allowed_mask, 4) || !aligned(b.temperatures, 4) ||
      !aligned(b.out_logprobs, 4) || !aligned(b.out_ranks, 4) || !aligned(b.out_logsumexp, 4) ||
      !aligned(b.out_entropy, 4) || !aligned(b.out_top_ids, 4) || !aligned(b.out_top_logprobs, 4) ||
      !aligned(b.out_status, 4))
    return OXS_ERR_INVALID_ARGUMENT;
  if (b.workspace_bytes < oxs_logprobs_workspace_bytes()) return OXS_ERR_INVALID_ARGUMENT;
  oxs_lp::Params p{b};
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(b.rows), dim3(oxs_lp::kThreads), 0, (hipStream_t)stream, p);
  };
  if (b.logits_dtype == OXS_DTYPE_F32) go(oxs_lp::row_kernel<OXS_DTYPE_F32>);
  else go(oxs_lp::row_kernel<OXS_DTYPE_BF16>);
  return hipGetLastError() == hipSuccess ? OXS_OK : OXS_ERR_HIP;
}

// oxs_logprobs.hip — token log probabilities, entropy, ranks and alternatives
// of whole rows of logits, beside the sampler that draws from them.
//
// With z the (softcapped, scaled) logits of a row's present tokens and m the
// largest, one pass keeps m, s = sum e^(z - m) and t = sum (z - m) e^(z - m):
//   lse = m + ln s,  log p_i = (z_i - m) - ln s,  H = ln s - t / s.
// H's two terms are both >= 0, so nothing cancels. Differences to m are taken
// before the scaling, so large logits lose nothing either.
//
// rows_kernel: a workgroup reads a part of a row in tiles that stay in
// registers, the next tile's loads on their way while one is worked on; each
// thread keeps its own m, s and t, so the row is read once whatever is asked
// of it. merge_kernel: a wavefront joins the parts of a row where it was split
// over workgroups (few rows). Alternatives: the N-th largest of the 256
// threads' maxima is a bound that at least N logits reach, so only the few
// threads with a logit above it hold candidates; ranks are counted tile by
// tile against the given tokens' logits.
//
// What bounds it: long rows the read (512 rows of 262144 float32 83 us,
// 6.4 TB/s, where a kernel that only reads takes 77), bf16 the vector unit
// beside it (an exponential and six more operations per logit, twice the
// logits per byte: 2048 rows of 128256 93 us, 5.7 TB/s), decode batches the
// start, the selection and the join (64 rows of 128256 float32, 20
// alternatives: 18.8 us, of which the read alone takes 6.5 and the join 4),
// one row two launches (32000 logits 9.1 us, 8.6 from a graph). A join in the
// same launch, by the last workgroup of a row to finish, was no faster (16 rows
// 10.6 us for 4.6 and 2.3; 64 rows equal).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/oxide_sampler.h"

namespace oxs_lp {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
// 2^-256 is 0 in 32 bits: a difference below this (or NaN, of two infinities) adds nothing
constexpr float kFloor = -256.0f;
constexpr uint32_t kMaxSplits = 64;      // parts of a row
constexpr uint32_t kMaxParts = 4096;     // rows * (parts + 1) of a call that splits its rows, at most
constexpr uint32_t kMergeKeys = 10 * 64; // parts * top_n of a split row
constexpr uint32_t kRoom = OXS_LOGPROBS_MAX_TOP + 512;  // candidates of a wavefront: those kept, and 64 lanes' next 8

struct Params {
  oxs_logprobs b;
  uint32_t splits;  // workgroups per row
  uint32_t tiles;   // tiles per workgroup
  // a split row's parts, in the workspace: [row * splits + part]
  float4* stats;    // m (raw logit), s, t
  uint64_t* keys;   // [top_n] the part's largest keys, in order, 0 past the last
  // [row][splits + 1][tokens_per_row]: tokens of each part in front of the given tokens, then the tokens' logits
  uint32_t* counts;
};

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// Orders tokens: a larger logit first, then the lower id (+0.0 for both zeros).
__device__ __forceinline__ uint32_t order_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(float l, uint32_t i) { return ((uint64_t)order_of(l) << 32) | (uint32_t)~i; }
__device__ __forceinline__ float key_value(uint64_t k) { return order_value((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return ~(uint32_t)k; }

constexpr uint32_t kOrderNegInf = 0x007fffffu;  // order_of(-inf)
constexpr uint32_t kOrderZero = 0x80000000u;    // order_of(0)

// The largest float below every l with order_of(l) >= o (the zeros are one value).
__device__ __forceinline__ float just_below(uint32_t o) {
  return o <= kOrderNegInf ? neg_inf() : order_value(o == kOrderZero ? o - 2u : o - 1u);
}

// ---------------------------------------------------------------- wavefront reductions (result in every lane)

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t other, uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)other, (int)x, CTRL, ROWS, 0xf, false);
}
template <class F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t x, uint32_t identity, F f) {
  x = f(x, dpp<0x111, 0xf>(identity, x));  // lanes 1, 2, 4, 8 below in the row of 16
  x = f(x, dpp<0x112, 0xf>(identity, x));
  x = f(x, dpp<0x114, 0xf>(identity, x));
  x = f(x, dpp<0x118, 0xf>(identity, x));
  x = f(x, dpp<0x142, 0xa>(identity, x));  // the row before, into rows 1 and 3
  x = f(x, dpp<0x143, 0xc>(identity, x));  // lane 31, into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
  return wave_reduce(x, 0u, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ float wave_sum(float x) {
  return __uint_as_float(wave_reduce(__float_as_uint(x), 0u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(wave_reduce(__float_as_uint(x), __float_as_uint(neg_inf()), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}

// Lanes of `who` below this one.
__device__ __forceinline__ uint32_t mbcnt(uint64_t who) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u));
}

// Orders a wavefront's accesses to LDS across its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 1 / cap, finite for the smallest caps too (0 times it is 0)
__device__ __forceinline__ float inverse_cap(float cap) { return fminf(1.0f / cap, 3.402823466e38f); }

// cap tanh(l / cap), to about 3 units in the last place: (1 - e) / (1 + e) with
// e = e^(-2|x|), which cancels near 0, and the series up to x^9 below 1/4
// (the next term is 0.009 x^10 <= 2^-26 of the value there).
__device__ __forceinline__ float softcap_of(float l, float cap, float inv_cap) {
  const float x = l * inv_cap, a = fabsf(x);
  const float e = exp2_fast(a * (-2.0f * kLog2e));
  const float far = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
  const float w = a * a;
  float p = __builtin_fmaf(w, 62.0f / 2835.0f, -17.0f / 315.0f);
  p = __builtin_fmaf(w, p, 2.0f / 15.0f);
  p = __builtin_fmaf(w, p, -1.0f / 3.0f);
  const float near = __builtin_fmaf(a * w, p, a);
  return cap * __builtin_copysignf(a < 0.25f ? near : far, x);
}

// 1 / T of a row, as the decode step takes it: greedy rows stay as they are.
__device__ __forceinline__ float inverse_temperature(const oxs_logprobs& b, uint32_t row) {
  if (!b.temperatures) return 1.0f;
  const float t = b.temperatures[row];
  return t > 1e-6f ? 1.0f / t : 1.0f;
}

// 1 / T to the base 2; above 0 for an infinite T too, so that a difference to -inf stays infinite
__device__ __forceinline__ float binary_scale(float inv) { return fmaxf(inv * kLog2e, 1.2e-38f); }

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

// What a row's outputs follow from.
struct Row {
  float m, s, t;  // the largest raw logit; s and t relative to its z
  float cap, inv_cap, inv;
  float y_m, ln_s;
  bool empty, over;
  __device__ __forceinline__ Row(const oxs_logprobs& b, float inv_, float m_, float s_, float t_)
      : m(m_), s(s_), t(t_), cap(b.logit_softcap), inv(inv_) {
    inv_cap = inverse_cap(cap);
    empty = m == neg_inf();
    y_m = y_of(m);
    over = y_m == __builtin_inff();
    ln_s = empty ? 0.0f : logf(s);
  }
  __device__ __forceinline__ float y_of(float l) const { return cap > 0.0f ? softcap_of(l, cap, inv_cap) : l; }
  __device__ __forceinline__ float logprob(float l) const {  // of a raw logit
    if (l == neg_inf()) return l;
    const float y = y_of(l);
    if (over) return y == y_m ? __builtin_nanf("") : neg_inf();
    return (y - y_m) * inv - ln_s;
  }
  __device__ __forceinline__ void write(const oxs_logprobs& b, uint32_t row) const {
    if (b.out_logsumexp) b.out_logsumexp[row] = empty ? m : over ? y_m : y_m * inv + ln_s;
    if (b.out_entropy) b.out_entropy[row] = empty ? 0.0f : over ? __builtin_nanf("") : ln_s - kLn2 * (t / s);
    if (b.out_status) b.out_status[row] = empty ? OXS_ROW_EMPTY : OXS_ROW_OK;
  }
  // given token j, with logit l and `before` tokens in front of it
  __device__ __forceinline__ void write_token(const oxs_logprobs& b, uint32_t row, uint32_t j, float l,
                                              uint32_t before) const {
    const size_t at = (size_t)row * b.tokens_per_row + j;
    if (b.out_logprobs) b.out_logprobs[at] = logprob(l);
    if (b.out_ranks) b.out_ranks[at] = l == neg_inf() ? 0u : before + 1u;
  }
  __device__ __forceinline__ void write_top(const oxs_logprobs& b, uint32_t row, uint32_t n, uint64_t k) const {
    const size_t at = (size_t)row * b.top_n + n;
    if (b.out_top_ids) b.out_top_ids[at] = k ? key_id(k) : kNoToken;
    if (b.out_top_logprobs) b.out_top_logprobs[at] = k ? logprob(key_value(k)) : neg_inf();
  }
};

// The n largest of a wavefront's `count` <= kRoom keys in `keys` (LDS), in order, in its first places: n rounds of
// taking the largest. Rare: many equal logits, or rows that rise towards their end.
__device__ __forceinline__ uint32_t keep_largest(uint64_t* keys, uint32_t count, uint32_t n) {
  const uint32_t lane = threadIdx.x & 63u;
  constexpr int kPer = (kRoom + 63) / 64;
  uint64_t mine[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) mine[i] = lane + 64u * i < count ? keys[lane + 64u * i] : 0;
  wave_sync();
  const uint32_t kept = min(n, count);
  for (uint32_t r = 0; r < kept; ++r) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = mine[i] > best ? mine[i] : best;
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o);
      best = other > best ? other : best;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (mine[i] == best) mine[i] = 0;
    if (lane == 0) keys[r] = best;
  }
  wave_sync();
  return kept;
}

// How many of the `all` keys of a list in LDS, with kAhead - 1 zeros or more behind them, are above a key. Eight at a
// time, so that their reads overlap.
constexpr uint32_t kAhead = 8;
__device__ __forceinline__ uint32_t keys_above(const uint64_t* list, uint32_t all, uint64_t key) {
  uint32_t n = 0;
  for (uint32_t i = 0; i < all; i += kAhead) {
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) n += list[i + j] > key ? 1u : 0u;
  }
  return n;
}

// ---------------------------------------------------------------- the pass over the logits

// The parameters as they lie in memory, for what is needed after the pass only: read where they are used, they take
// no scalar registers during it.
__device__ __forceinline__ const Params& late_params() {
  uint64_t q = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(q));
  return *(const Params*)(const __attribute__((address_space(4))) Params*)q;
}

// A number of which the compiler knows nothing, so that what is computed from it in a rare branch is not kept in
// registers all the time.
__device__ __forceinline__ int32_t apart(int32_t x) {
  asm("" : "+v"(x));
  return x;
}

// The largest of N floats by their bits, as whole numbers: those of one sign are in the order of their magnitudes, so
// it is the largest signed number if that has no sign bit, else the smallest unsigned one. One instruction per value
// (half of one for pairs of bf16), where a maximum of floats takes one and a half, as it has to make signalling NaNs
// quiet first. NaN if a positive NaN, or nothing but negative ones, is among them.
template <int N>
__device__ __forceinline__ float largest_of(const float* v) {
  int32_t hi = (int32_t)__float_as_uint(v[0]);
  uint32_t lo = __float_as_uint(v[0]);
#pragma unroll
  for (int e = 1; e < N; ++e) {
    hi = max(hi, (int32_t)__float_as_uint(v[e]));
    lo = min(lo, __float_as_uint(v[e]));
  }
  return __uint_as_float(hi >= 0 ? (uint32_t)hi : lo);
}
template <int N>
__device__ __forceinline__ float largest_of_pairs(const u32x4* raw) {
  const uint32_t first = raw[0][0];
  i16x2 hi = __builtin_bit_cast(i16x2, first);
  u16x2 lo = __builtin_bit_cast(u16x2, first);
#pragma unroll
  for (int i = 1; i < 4 * N; ++i) {
    const uint32_t x = raw[i / 4][i % 4];  // (a bit cast of the element itself takes element 0)
    hi = __builtin_elementwise_max(hi, __builtin_bit_cast(i16x2, x));
    lo = __builtin_elementwise_min(lo, __builtin_bit_cast(u16x2, x));
  }
  const int32_t h = max((int32_t)hi[0], (int32_t)hi[1]);
  return __uint_as_float((h >= 0 ? (uint32_t)h : (uint32_t)min(lo[0], lo[1])) << 16);
}

// A thread's sums s = sum 2^q, t = sum q 2^q with q = (y - ref) c for its logits' y. ref follows the largest logit
// only when that is 2^kSlack away: the sums stay far from overflow, and most steps need no rescaling.
// q is y c - (ref c rounded) in one operation. What that rounding leaves out (rest) is the same for all terms, so it
// comes off the sums when ref changes.
constexpr float kSlack = 16.0f;
constexpr float kHuge = 1e31f;  // y c cannot overflow below this, as c <= 10^6 log2 e
struct Sums {
  float ref = -__builtin_inff(), rc = 0.0f, s = 0.0f, t = 0.0f;
  __device__ __forceinline__ float rest(float c) const {
    return fabsf(ref) < kHuge ? __builtin_fmaf(ref, c, -rc) : 0.0f;
  }
  __device__ __forceinline__ void shift(float by) {  // q + by in the place of q
    const float f = exp2_fast(by);
    t = f * __builtin_fmaf(by, s, t);
    s = f * s;
  }
  // makes s and t relative to `to` >= ref itself, or (settled = false) to what the next terms are relative to
  __device__ __forceinline__ void rebase(float to, float c, bool settled = false) {
    shift(-rest(c));
    shift(fmaxf((ref - to) * c, kFloor));  // (NaN, of two -inf: kFloor)
    ref = to;
    rc = ref * c;
    if (settled) return;
    shift(rest(c));
  }
  __device__ __forceinline__ bool behind(float top, float c) const { return (top - ref) * c > kSlack; }
  __device__ __forceinline__ bool huge() const { return fabsf(ref) >= kHuge && ref > neg_inf(); }
  // N more logits, of which none is 2^kSlack above ref
  template <int N, class Y>
  __device__ __forceinline__ void add(const float* v, float c, Y y) {
    // two sums of their own first: a row's terms then pass N / 2 + V / (kThreads N) additions, not V / kThreads
    float s0, s1, t0, t1;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float q0 = fmaxf(__builtin_fmaf(y(v[e]), c, -rc), kFloor);
      const float q1 = fmaxf(__builtin_fmaf(y(v[e + 1]), c, -rc), kFloor);
      const float p0 = exp2_fast(q0), p1 = exp2_fast(q1);
      s0 = e ? s0 + p0 : p0;
      s1 = e ? s1 + p1 : p1;
      t0 = e ? __builtin_fmaf(q0, p0, t0) : q0 * p0;
      t1 = e ? __builtin_fmaf(q1, p1, t1) : q1 * p1;
    }
    s += s0 + s1;
    t += t0 + t1;
  }
};

// G consecutive logits in one 16-byte load; a thread holds E of a tile as E / G groups that lie kThreads * G apart.
// Rows that do not begin on 16 bytes are cut at the boundaries all the same, and the tile in which a row begins or
// ends between two boundaries is loaded logit by logit.
template <int DT>
constexpr int group_size() { return DT == OXS_DTYPE_F32 ? 4 : 8; }

template <int DT, int E, bool MASK, bool CAP, bool TOP>
__global__ __launch_bounds__(kThreads, 4) void rows_kernel(Params p) {
  constexpr int G = group_size<DT>(), NG = E / G;
  constexpr uint32_t kSize = DT == OXS_DTYPE_F32 ? 4 : 2;
  constexpr uint32_t kTile = kThreads * E;
  const oxs_logprobs& b = p.b;
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t row = blockIdx.x / p.splits, part = blockIdx.x - row * p.splits;
  const uint32_t V = b.vocab, T = b.tokens_per_row, N = TOP ? b.top_n : 0u;
  constexpr uint32_t kStage = 512 / E;  // threads whose logits are looked at together
  __shared__ uint64_t s_keys[TOP ? kWaves : 1][TOP ? kRoom : 1];
  __shared__ __align__(16) float s_stage[TOP ? kWaves : 1][TOP ? 512 : 4];
  __shared__ uint32_t s_stage_id[TOP ? kWaves : 1][TOP ? kStage : 1];
  __shared__ uint32_t s_order[2][TOP ? kThreads : 1];
  __shared__ __align__(16) uint64_t s_list[TOP ? kThreads + kAhead : 1];
  __shared__ float s_m[kWaves], s_s[kWaves], s_t[kWaves];
  __shared__ uint32_t s_count[kWaves];
  __shared__ uint32_t s_before[kWaves][OXS_LOGPROBS_MAX_TOKENS];

  const char* base = (const char*)b.logits + (size_t)row * (size_t)b.logits_ld * kSize;
  // logits between the boundary before the row and its first one
  const uint32_t skip = ((uint32_t)(uintptr_t)base & 15u) / kSize;
  const uint32_t* mask = MASK ? b.allowed_mask + (size_t)row * (size_t)b.mask_ld : nullptr;
  const float inv = inverse_temperature(b, row), c = binary_scale(inv);
  const float cap = b.logit_softcap, inv_cap = CAP ? inverse_cap(cap) : 0.0f;
  const auto y_of = [&](float l) {
    if constexpr (CAP) return l == neg_inf() ? l : softcap_of(l, cap, inv_cap);
    else return l;
  };

  // lane j's given token; its logit (and mask word) are used after the first tile's
  uint32_t want = kNoToken, want_bits = 0, want_word = 0;
  if (lane < T) want = b.tokens[(size_t)row * (size_t)b.tokens_ld + lane];
  // a logit of an earlier token is in front from want_l on, of a later one above it
  float want_l = neg_inf(), want_below = neg_inf();
  uint32_t before = 0;  // tokens of this wavefront in front of lane j's

  Sums sums;
  float m = neg_inf();      // the thread's largest logit
  float floor = neg_inf();  // every alternative of the row is above it,
  float bound = neg_inf();  // and those of this wavefront's tokens to come above this
  uint32_t count = 0, round = 0;  // candidates of this wavefront; times the floor was raised
  uint64_t* keys = s_keys[TOP ? wave : 0];
  float* stage = s_stage[TOP ? wave : 0];
  uint32_t* stage_id = s_stage_id[TOP ? wave : 0];

  const uint32_t first = part * p.tiles;
  const uint32_t total = (V + skip + kTile - 1u) / kTile;
  const uint32_t last = min(first + p.tiles, total);
  // a tile's logits, as they lie in memory; -inf outside the row
  const auto fetch = [&](uint32_t tile, u32x4 (&to)[NG]) {
    const int32_t at = (int32_t)(tile * kTile + tid * G - skip);
    const int64_t begin = (int64_t)tile * kTile - (int64_t)skip;
    if (begin >= 0 && begin + kTile <= (int64_t)V) {
#pragma unroll
      for (int g = 0; g < NG; ++g)
        to[g] = __builtin_nontemporal_load((const u32x4*)(base + (uint32_t)(at + g * kThreads * G) * kSize));
    } else {  // the row begins or ends in the tile: logit by logit
      const int32_t mine = apart(at);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int32_t i = mine + (e / G) * kThreads * G + e % G;
        const uint32_t j = (uint32_t)min(max(i, 0), (int32_t)V - 1);
        if constexpr (DT == OXS_DTYPE_F32) {
          const uint32_t x = *(const uint32_t*)(base + j * kSize);
          to[e / G][e % G] = i == (int32_t)j ? x : 0xff800000u;
        } else {
          uint32_t x = *(const uint16_t*)(base + j * kSize);
          x = i == (int32_t)j ? x : 0xff80u;
          if (e & 1) to[e / G][(e % G) >> 1] |= x << 16;
          else to[e / G][(e % G) >> 1] = x;
        }
        if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // (the addresses of all at once would not fit)
      }
    }
  };
  // A wavefront's part of a group is 64 G tokens, whose mask is kWords words: all words of a tile come in one load
  // (two for rows that do not begin on 16 bytes), lane g kWords + i holding the bits of group g from token 32 i on,
  // and the lanes pass them on. Bits of tokens outside the row may be anything: those are -inf already.
  constexpr uint32_t kWords = 2 * G;
  uint32_t words[2] = {};
  const auto fetch_mask = [&](uint32_t tile) {
    if constexpr (MASK) {
      const int32_t end = (int32_t)((V + 31u) / 32u) - 1;
      const int32_t w = (int32_t)(tile * (kTile / 32u) + lane / kWords * (kThreads * G / 32u) + wave * kWords +
                                  lane % kWords - (skip ? 1u : 0u));
      words[0] = mask[min(max(w, 0), end)];
      if (skip) words[1] = mask[min(w + 1, end)];
    }
  };
  u32x4 raw[NG];
  fetch_mask(first);
  fetch(first, raw);
  if (want < V) {
    if constexpr (DT == OXS_DTYPE_F32) want_bits = *(const uint32_t*)(base + want * kSize);
    else want_bits = (uint32_t)*(const uint16_t*)(base + want * kSize) << 16;
    if constexpr (MASK) want_word = mask[want >> 5];
  }
  const auto want_set = [&]() {
    const float l = __uint_as_float(want_bits);
    const bool in = want < V && l == l && (!MASK || ((want_word >> (want & 31u)) & 1u));
    want_l = in ? l : neg_inf();
    want_below = just_below(order_of(want_l));
  };
  if (last <= first) want_set();  // a part past the row's end
  for (uint32_t tile = first; tile < last; ++tile) {
    // element e of group g is token at + g * kThreads * G + e (negative before the row: none)
    const int32_t at = (int32_t)(tile * kTile + tid * G - skip);  // V <= 2^30
    const int64_t begin = (int64_t)tile * kTile - (int64_t)skip;  // of the tile
    float v[E];
    uint32_t keep = 0;  // bit e: the mask allows element e
    if constexpr (MASK) {
      const uint32_t bits = __builtin_amdgcn_alignbit(words[1], words[0], 32u - skip);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t from = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(g * kWords + lane * G / 32u) * 4, (int)bits);
        keep |= ((from >> (lane * G % 32u)) & ((1u << G) - 1u)) << (g * G);
      }
    }
    u32x4 next[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) next[g] = raw[g];
    if (tile + 1u < last) {
      fetch_mask(tile + 1u);
      fetch(tile + 1u, next);
    }
    const Sums before_tile = sums;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (DT == OXS_DTYPE_F32) v[e] = __uint_as_float(raw[e / G][e % G]);
      else v[e] = __uint_as_float((e & 1) ? raw[e / G][(e % G) >> 1] & 0xffff0000u : raw[e / G][(e % G) >> 1] << 16);
      if constexpr (MASK) {
        const uint32_t in = (uint32_t)((int32_t)(keep << (31 - e)) >> 31);
        v[e] = __uint_as_float((__float_as_uint(v[e]) & in) | (~in & 0xff800000u));
      }
    }
    float top;  // the thread's largest of the tile
    if constexpr (DT == OXS_DTYPE_BF16 && !MASK) top = largest_of_pairs<NG>(raw);
    else top = largest_of<E>(v);
    const bool odd = top != top;
    // (Once per tile: once per eight logits of it took 116 us where this takes 106, 2048 rows of 128256 bf16 with 20
    // alternatives.)
    if (__ballot(sums.behind(y_of(top), c))) sums.rebase(fmaxf(sums.ref, y_of(top)), c);
    sums.add<E>(v, c, y_of);
    const bool slow = __ballot(odd || sums.huge()) != 0;
    if (__builtin_expect(slow, 0)) {
      // NaNs among the logits may have hidden the largest, and a huge one (a mask of the type's lowest value, say)
      // makes y c overflow: the tile again, from memory, logit by logit and with the difference first.
      sums = before_tile;
      top = neg_inf();
#pragma unroll 1
      for (int e = 0; e < E; ++e)
        top = fmaxf(top, present_logit<DT>(b, row, (uint32_t)(at + (e / G) * kThreads * G + e % G)));
      sums.rebase(fmaxf(sums.ref, y_of(top)), c, true);
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const float y = y_of(present_logit<DT>(b, row, (uint32_t)(at + (e / G) * kThreads * G + e % G)));
        const float q = fmaxf((y - sums.ref) * c, kFloor), f = exp2_fast(q);
        sums.s += f;
        sums.t = __builtin_fmaf(q, f, sums.t);
      }
      sums.shift(sums.rest(c));
    }
    m = fmaxf(m, top);
    if (tile == first) want_set();

    if constexpr (TOP) {
      // Raise the floor at the 1st, 4th, 16th, ... tile that more tiles follow than came before, and the last: at least
      // N logits so far are no less than the N-th largest of the 256 threads' maxima, so the rest cannot be
      // alternatives. (At the 4th of 5 too: 256 rows of 151936 bf16 27.0 us for 25.9 with 5 alternatives, 32.3 for
      // 31.0 with 32; 700 rows of 50257, 20 alternatives, 34.4 for 36.0.)
      const uint32_t n = tile - first + 1u;
      if (((n & (n - 1u)) == 0u && (n & 0x55555555u) && last - tile > n) || tile + 1u == last) {
        uint32_t* so = s_order[round & 1u];  // (a wavefront is at most one round ahead)
        ++round;
        so[tid] = order_of(m);
        __syncthreads();
        uint32_t o[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o[w] = so[w * 64 + lane];
        uint32_t lo = o[0], hi = o[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
          lo = min(lo, o[w]);
          hi = max(hi, o[w]);
        }
        lo = wave_reduce(lo, 0xffffffffu, [](uint32_t x, uint32_t y) { return min(x, y); });
        hi = wave_reduce(hi, 0u, [](uint32_t x, uint32_t y) { return max(x, y); }) + 1u;
        // at least N maxima are >= lo, fewer are >= hi
        for (int i = 0; i < 32 && hi - lo > 1u; ++i) {
          const uint32_t mid = lo + (hi - lo) / 2u;
          uint32_t k = 0;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) k += (uint32_t)__popcll(__ballot(o[w] >= mid));
          if (k >= N) lo = mid;
          else hi = mid;
          if (k >= N && k <= N + 4u) break;
        }
        floor = fmaxf(floor, just_below(lo));
        bound = fmaxf(bound, floor);
      }
      // The logits of the threads that have one above the bound go through LDS, kStage threads at a time, and every
      // lane then looks at a few of them.
      uint64_t rest = __ballot(top > bound);
      float above = bound;
      while (rest) {
        uint32_t lanes = min(kStage, (kRoom - count) / E);  // that fit whatever they hold
        if (lanes < min((uint32_t)__popcll(rest), 4u)) {
          count = keep_largest(keys, count, N);
          lanes = kStage;
          if (count == N) {  // a lower id may still come in this tile, of the same logit
            const float nth = key_value(keys[N - 1u]);
            above = fmaxf(above, just_below(order_of(nth)));
            bound = fmaxf(bound, nth);
          }
        }
        const uint32_t to = mbcnt(rest);
        const bool mine = ((rest >> lane) & 1u) && to < lanes;
        if (mine) {
#pragma unroll
          for (int e = 0; e < E; e += 4)
            *(float4*)&stage[to * E + e] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          stage_id[to] = (uint32_t)at;
        }
        const uint64_t sent = __ballot(mine);
        rest &= ~sent;
        const uint32_t n = (uint32_t)__popcll(sent) * E;
        wave_sync();
        for (uint32_t i0 = 0; i0 < n; i0 += 64u) {
          const uint32_t i = i0 + lane, e = i % E;
          const float x = i < n ? stage[i] : neg_inf();
          const uint64_t who = __ballot(x > above);
          if (!who) continue;
          if (x > above)
            keys[count + mbcnt(who)] = key_of(x, stage_id[i / E] + (e / G) * (kThreads * G) + e % G);
          count += (uint32_t)__popcll(who);
        }
        wave_sync();
      }
    }

    // Tokens in front of the given ones. (Counted through the scalar unit: a compare per logit on the vector unit,
    // where adding up the lanes' counts would take another, and a sum over the lanes per tile.)
    for (uint32_t j = 0; j < T; ++j) {
      const float l = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(want_l), (int)j));
      if (l == neg_inf()) continue;
      const float below =
          __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(want_below), (int)j));
      // None of the wavefront's logits is in front, in most tiles for a likely token (700 rows of 50257, 16 tokens: the
      // likeliest 92 -> 70 us, drawn ones 91 -> 84, any 90 -> 92).
      if (!__ballot(top > below)) continue;
      const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)want, (int)j);
      uint32_t k = 0;
      if (begin + kTile <= (int64_t)id || begin > (int64_t)id) {
        const float than = begin > (int64_t)id ? l : below;
        // Eight comparisons first, then their counts: none waits for the one before it.
#pragma unroll
        for (int e0 = 0; e0 < E; e0 += 8) {
          uint64_t in[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) in[e] = __ballot(v[e0 + e] > than);
          asm("" : "+s"(in[0]), "+s"(in[1]), "+s"(in[2]), "+s"(in[3]), "+s"(in[4]), "+s"(in[5]), "+s"(in[6]),
                   "+s"(in[7]));
#pragma unroll
          for (int e = 0; e < 8; ++e) k += (uint32_t)__popcll(in[e]);
        }
      } else {
        const int32_t to = (int32_t)id - apart(at);  // element e is before the token if its offset is below
#pragma unroll
        for (int e = 0; e < E; ++e)
          k += (uint32_t)__popcll(__ballot(v[e] > ((e / G) * kThreads * G + e % G < to ? below : l)));
      }
      if (lane == j) before += k;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) raw[g] = next[g];
  }

  // the workgroup's sums, relative to its largest logit
  const Params& late = late_params();
  const float wm = wave_max(m);
  if (lane < T) s_before[wave][lane] = before;
  sums.rebase(fmaxf(y_of(wm), sums.ref), c, true);
  {
    const float ws = wave_sum(sums.s), wt = wave_sum(sums.t);
    if (lane == 0) {
      s_m[wave] = wm;
      s_s[wave] = ws;
      s_t[wave] = wt;
    }
  }
  if constexpr (TOP) {
    // drop what the last floor leaves out (all are above the only one), and keep at most 64 candidates per wavefront
    if (round > 1u) {
      uint32_t kept = 0;
      for (uint32_t i0 = 0; i0 < count; i0 += 64u) {
        const uint64_t k = i0 + lane < count ? keys[i0 + lane] : 0;
        const bool in = k && key_value(k) > floor;
        const uint64_t who = __ballot(in);
        wave_sync();
        if (in) keys[kept + mbcnt(who)] = k;
        kept += (uint32_t)__popcll(who);
      }
      wave_sync();
      count = kept;
    }
    if (count > 64u) count = keep_largest(keys, count, N);
    if (lane == 0) s_count[wave] = count;
  }
  __syncthreads();
  float bm = s_m[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) bm = fmaxf(bm, s_m[w]);
  float bs = 0.0f, bt = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float d = fmaxf((y_of(s_m[w]) - y_of(bm)) * c, kFloor), f = exp2_fast(d);
    bs += f * s_s[w];
    bt += f * __builtin_fmaf(d, s_s[w], s_t[w]);
  }
  uint32_t all = 0;
  if constexpr (TOP) {  // one list of the workgroup's candidates
    uint32_t before_me = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < (int)wave) before_me += s_count[w];
      all += s_count[w];
    }
    if (lane < count) s_list[before_me + lane] = keys[lane];
    if (tid < kAhead) s_list[all + tid] = 0;
    __syncthreads();
  }
  before = 0;  // tokens of this part in front of given token tid
  if (tid < T) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) before += s_before[w][tid];
  }
  uint64_t mine = 0;
  uint32_t place = kNoToken;
  if (TOP && tid < all) {
    mine = s_list[tid];
    place = keys_above(s_list, all, mine);
  }
  if (late.splits > 1u) {
    const size_t at = (size_t)row * late.splits + part;
    if (tid == 0) late.stats[at] = make_float4(bm, bs, bt, 0.0f);
    uint32_t* counts = late.counts + (size_t)row * (late.splits + 1u) * T;
    if (tid < T) counts[part * T + tid] = before;
    if (tid < T && part == 0u) counts[late.splits * T + tid] = __float_as_uint(want_l);
    if (TOP && place < N) late.keys[at * N + place] = mine;
    if (TOP && tid >= all && tid < N) late.keys[at * N + tid] = 0;
    return;
  }
  const Row r(late.b, inv, bm, bs, bt);
  if (tid == 0) r.write(late.b, row);
  if (tid < T) r.write_token(late.b, row, tid, want_l, before);  // (T <= 64: the first wavefront)
  if (TOP && place < N) r.write_top(late.b, row, place, mine);
  if (TOP && tid >= all && tid < N) r.write_top(late.b, row, tid, 0);
}

// One wavefront joins the parts of a row. The alternatives are the keys no less than a bound that is found by halving
// a range of keys until N to N + 4 of them are above it. All that it reads is on its way before the first is waited for
// (the counts of the ninth token on aside).
template <bool CAP, bool TOP, int PER>
__global__ __launch_bounds__(64) void merge_kernel(Params p) {
  const oxs_logprobs& b = p.b;
  const uint32_t row = blockIdx.x, lane = threadIdx.x;
  const uint32_t S = p.splits, T = b.tokens_per_row, N = TOP ? b.top_n : 0u;
  __shared__ __align__(16) uint64_t s_best[64 + kAhead];
  const size_t at = (size_t)row * S;
  const uint32_t part = min(lane, S - 1u);
  float4 st = p.stats[at + part];
  uint64_t k[PER], floor = ~0ull;
  if constexpr (TOP) {
    const uint32_t last = S * N - 1u;
#pragma unroll
    for (int i = 0; i < PER; ++i) k[i] = p.keys[at * N + min(lane + 64u * i, last)];
    // the ceil(N / S)-th key of each part: N keys at least are no less than the smallest of them
    floor = p.keys[(at + part) * N + (N + S - 1u) / S - 1u];
#pragma unroll
    for (int i = 0; i < PER; ++i) k[i] = lane + 64u * i <= last ? k[i] : 0;
  }
  const uint32_t* counts = p.counts + (size_t)row * (S + 1u) * T;
  const auto count_of = [&](uint32_t j) { return counts[part * T + min(j, max(T, 1u) - 1u)]; };
  uint32_t some[kAhead];
#pragma unroll
  for (uint32_t j = 0; j < kAhead; ++j) some[j] = count_of(j);
  const float want_l = __uint_as_float(counts[S * T + min(lane, max(T, 1u) - 1u)]);
  if (lane >= S) st = make_float4(neg_inf(), 0.0f, 0.0f, 0.0f);
  const float inv = inverse_temperature(b, row), c = binary_scale(inv), cap = b.logit_softcap,
              inv_cap = CAP ? inverse_cap(cap) : 0.0f;
  const auto y_of = [&](float l) {
    if constexpr (CAP) return l == neg_inf() ? l : softcap_of(l, cap, inv_cap);
    else return l;
  };
  const float m = wave_max(st.x);
  const float d = fmaxf((y_of(st.x) - y_of(m)) * c, kFloor), f = exp2_fast(d);
  const Row r(b, inv, m, wave_sum(f * st.y), wave_sum(f * __builtin_fmaf(d, st.y, st.z)));
  if (lane == 0) r.write(b, row);
  uint32_t before = 0;
  for (uint32_t j0 = 0; j0 < T; j0 += kAhead) {
    if (j0) {
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) some[j] = count_of(j0 + j);
    }
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) {
      const uint32_t n = wave_sum(lane < S ? some[j] : 0u);
      if (lane == j0 + j) before = n;
    }
  }
  if (lane < T) r.write_token(b, row, lane, want_l, before);
  if constexpr (TOP) {
    uint32_t best = (uint32_t)(k[0] >> 32);
#pragma unroll
    for (int i = 1; i < PER; ++i) best = max(best, (uint32_t)(k[i] >> 32));
    best = wave_reduce(best, 0u, [](uint32_t x, uint32_t y) { return max(x, y); });
    const uint32_t low = wave_reduce((uint32_t)(floor >> 32), ~0u, [](uint32_t x, uint32_t y) { return min(x, y); });
    // keys >= lo are enough (or all there are); fewer than N are >= hi
    uint64_t lo = low ? (uint64_t)low << 32 : 1u, hi = (uint64_t)(best + 1u) << 32;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += (uint32_t)__popcll(__ballot(k[i] >= lo));
    for (int step = 0; step < 64 && n > N + 4u; ++step) {
      const uint64_t mid = lo + (hi - lo) / 2u;
      uint32_t above = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) above += (uint32_t)__popcll(__ballot(k[i] >= mid));
      if (above >= N) {
        lo = mid;
        n = above;
      } else {
        hi = mid;
      }
    }
    uint32_t all = 0;  // n of them: at most N + 4 <= 64, as keys differ
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = k[i] >= lo;
      const uint64_t who = __ballot(in);
      const uint32_t to = all + mbcnt(who);
      if (in && to < 64u) s_best[to] = k[i];
      all += (uint32_t)__popcll(who);
    }
    all = min(all, 64u);
    if (lane < kAhead) s_best[all + lane] = 0;
    wave_sync();
    uint32_t place = kNoToken;
    uint64_t mine = 0;
    if (lane < all) {
      mine = s_best[lane];
      place = keys_above(s_best, all, mine);
    }
    if (place < N) r.write_top(b, row, place, mine);
    if (lane >= all && lane < N) r.write_top(b, row, lane, 0);
  }
}

template <int DT, bool CAP>
static void launch(Params& p, hipStream_t st) {
  const oxs_logprobs& b = p.b;
  // Tiles of 8192 logits (32 per thread), or of 2048 where those would leave CUs without a workgroup and the join does
  // not have more to do for it than the rows less. 8192 and 2048, float32, us: no alternatives, 1 row of 32000 7.5 and
  // 5.4, 24 rows of 50257 8.5 and 6.9, 15 of 128256 8.0 and 7.7; 5 alternatives 1 row of 32000 10.5 and 9.0, 24 rows
  // 12.0 and 10.7, 60 rows 11.9 and 12.6; 1 row of 128256 with 10 10.7 and 10.2, with 20 11.7 and 12.6.
  const auto tiles_of = [&](uint32_t tile) { return (b.vocab + 7u + tile - 1u) / tile; };
  const uint32_t large = tiles_of(kThreads * 32), fine = tiles_of(kThreads * 8);
  const uint64_t groups = (uint64_t)b.rows * large;
  const bool small =
      b.top_n ? groups < 150u && fine <= kMaxSplits && fine * b.top_n <= kMergeKeys : groups < 256u;
  const uint32_t tiles = small ? fine : large;
  // A row is split where its parts fill CUs that whole rows leave idle, by more than the join costs: up to
  // more rows the longer they are. Split and whole, float32, 8 alternatives, us: 4000 logits 110 rows 10.1 and
  // 8.8; 32000 logits 60 rows 12.7 and 19.7, 250 rows 19.1 and 17.9; 128256 logits 250 rows 34.8 and 39.2,
  // 450 rows 52.9 and 47.1; 262144 logits 250 rows 57.3 and 65.8. About 1024 parts in all (2048: 64 rows of
  // 128256 with 20 alternatives 25.8 for 21.4).
  uint32_t splits = 1;
  if (large > 1u && b.rows < min(512u, 64u + 20u * large)) {
    splits = min(min(tiles, kMaxSplits), (1024u + b.rows - 1u) / b.rows);
    if (b.top_n) splits = min(splits, kMergeKeys / b.top_n);
  }
  p.tiles = (tiles + splits - 1u) / splits;
  p.splits = (tiles + p.tiles - 1u) / p.tiles;
  const dim3 grid(b.rows * p.splits);
  const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, p); };
  const auto by_top = [&](auto e, auto mask) {
    constexpr int kE = decltype(e)::value;
    constexpr bool kMask = decltype(mask)::value;
    if (b.top_n) go(rows_kernel<DT, kE, kMask, CAP, true>);
    else go(rows_kernel<DT, kE, kMask, CAP, false>);
  };
  const auto by_mask = [&](auto e) {
    if (b.allowed_mask) by_top(e, std::true_type{});
    else by_top(e, std::false_type{});
  };
  if (small) by_mask(std::integral_constant<int, 8>{});
  else by_mask(std::integral_constant<int, 32>{});
  if (p.splits == 1u) return;
  const auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(b.rows), dim3(64), 0, st, p); };
  if (b.top_n == 0u) join(merge_kernel<CAP, false, 1>);
  // (ten keys per lane where five would do cost 0.3 us)
  else if (p.splits * b.top_n <= 5u * 64u) join(merge_kernel<CAP, true, 5>);
  else join(merge_kernel<CAP, true, 10>);
}

}  // namespace oxs_lp

static bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1u)) == 0; }

// stats, keys and counts of kMaxParts parts
extern "C" size_t oxs_logprobs_workspace_bytes(void) {
  return (size_t)oxs_lp::kMaxParts * (16u + 8u * OXS_LOGPROBS_MAX_TOP + 4u * OXS_LOGPROBS_MAX_TOKENS);
}

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
  oxs_lp::Params p{};
  p.b = b;
  if (b.logit_softcap == __builtin_inff()) p.b.logit_softcap = 0.0f;  // what cap tanh(l / cap) tends to
  p.stats = (float4*)b.workspace;
  p.keys = (uint64_t*)(p.stats + oxs_lp::kMaxParts);
  p.counts = (uint32_t*)(p.keys + (size_t)oxs_lp::kMaxParts * OXS_LOGPROBS_MAX_TOP);
  const bool cap = p.b.logit_softcap > 0.0f;
  const hipStream_t st = (hipStream_t)stream;
  if (b.logits_dtype == OXS_DTYPE_F32) {
    if (cap) oxs_lp::launch<OXS_DTYPE_F32, true>(p, st);
    else oxs_lp::launch<OXS_DTYPE_F32, false>(p, st);
  } else {
    if (cap) oxs_lp::launch<OXS_DTYPE_BF16, true>(p, st);
    else oxs_lp::launch<OXS_DTYPE_BF16, false>(p, st);
  }
  return hipGetLastError() == hipSuccess ? OXS_OK : OXS_ERR_HIP;
}

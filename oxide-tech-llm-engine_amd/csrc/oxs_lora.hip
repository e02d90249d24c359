// oxs_lora.hip — low-rank adapters of many requests beside the projection
// that they share: y_b += B_a (s_a A_a x_b) for the adapter a of each row b.
//
// shrink_kernel: v_b = s_a A_a x_b into the workspace, a wavefront per row and
// one or four ranks. expand_kernel: y_b += B_a v_b on the matrix cores, 32
// rows (few: 8) in order of adapter x 64 or 128 outputs per wavefront, for each
// adapter among the rows in turn. single_kernel: both in one launch where there
// is little to do, each workgroup with the whole of v for its outputs.
//
// What bounds it: large batches the read and write of y (1024 rows of 128256
// float32 in 8 runs, rank 32: 236 us, 1.13 GB, 4.8 TB/s, a copy's rate; 64 rows,
// 16 adapters of rank 16: 25 us, 4.6 TB/s). f16 weights their conversion and
// the matrix instructions (256 rows of 151936, 4 adapters of rank 64, bf16 x and
// y: 67 us for 210 MB; 43 at a copy's rate). Rows with an adapter each the chain
// of loads (24 rows of 50257, float32 of rank 8: 17.3 us for 42 MB); one row the
// launch (32000 outputs, 4096 inputs: 5.5 us, 4.5 from a graph).
//
// Left out, measured: the first product on the matrix cores for rows that share
// an adapter (1024 rows 48 to 90 us, 24 here) or four rows per wavefront (44);
// row tiles of 64 (prompts 276 us for 230, f16 98 for 76); v through LDS (one row
// 7.0 us for 5.3); three or four pairs of operands on their way (registers
// spill: prompts 375 us for 232); row tiles side by side (prompts 259 us for 231)
// or in chunks of 32 to 256 ranges of outputs (within 5% either way); tiles of 2
// to 4 rows, or the second product row by row on the vector unit, where every
// row has an adapter of its own (14 us for 19 in the case above, but 42 for 13
// where 32 rows share one, which the host cannot tell).
//
// The matrix cores take bf16. A float is the sum of three bf16 (each the
// nearest to what is left of it: 2^-9 of it remains after one, 2^-18 after
// two, nothing of its 24 bits after three), a half of two, so the products of
// the parts in 32-bit sums give the product of the floats; of f32 weights'
// nine products the three below 2^-26 of the whole are left out.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/oxide_sampler.h"

namespace oxs_lora {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kRows = 32;        // rows of a matrix tile
constexpr uint32_t kGroup = 128;      // outputs of a group in the table
constexpr uint32_t kBlock = 16;       // ranks of a block: the depth of a matrix instruction
constexpr uint32_t kPlanes = 3;       // bf16 parts of a value of v
constexpr uint32_t kValueBytes = kPlanes * kBlock * 2;  // a row's values of a rank block: [part][16]

// Table, per slot:
//   a  [ranks, a multiple of 16][k, rounded up to 8], zero past the adapter's
//   b  [group of 128 outputs][rank block][half of the block][4][32] pieces of 8 ranks of one output, as a lane of a
//      matrix instruction takes them: piece (t, n) belongs to output 4 n + t of the group. The half of a block that
//      holds no rank is never read.
__host__ __device__ __forceinline__ uint32_t rank_blocks(uint32_t rank) { return (rank + kBlock - 1u) / kBlock; }
__host__ __device__ __forceinline__ uint32_t groups_of(uint32_t m) { return (m + kGroup - 1u) / kGroup; }
__host__ __device__ __forceinline__ uint32_t padded_k(uint32_t k) { return (k + 7u) & ~7u; }
__host__ __device__ __forceinline__ size_t a_elements(const oxs_lora_table& t) {
  return (size_t)rank_blocks(t.max_rank) * kBlock * padded_k(t.k);
}
__host__ __device__ __forceinline__ size_t b_elements(const oxs_lora_table& t) {
  return (size_t)groups_of(t.m) * rank_blocks(t.max_rank) * kBlock * kGroup;
}

template <int DT>
using Element = std::conditional_t<DT == OXS_DTYPE_F32, uint32_t, uint16_t>;

template <int DT>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (DT == OXS_DTYPE_F32) return __uint_as_float(bits);
  else if constexpr (DT == OXS_DTYPE_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else return __uint_as_float(bits << 16);
}

// Eight values from 16-byte aligned memory (two 16-byte loads for f32).
template <int DT>
struct Eight {
  u32x4 q[DT == OXS_DTYPE_F32 ? 2 : 1];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (DT == OXS_DTYPE_F32) return __uint_as_float(q[i / 4][i % 4]);
    else if constexpr (DT == OXS_DTYPE_F16) return widen<DT>((q[0][i / 2] >> (16 * (i % 2))) & 0xffffu);
    else return __uint_as_float(i % 2 ? q[0][i / 2] & 0xffff0000u : q[0][i / 2] << 16);
  }
};

// Two floats as the nearest bf16 pair, and that pair widened again.
__device__ __forceinline__ uint32_t narrow2(float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x, y}, bf16x2));
}
__device__ __forceinline__ float low(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// ---------------------------------------------------------------- the table

template <int DT>
__global__ __launch_bounds__(kThreads) void load_kernel(oxs_lora_table t, uint32_t slot, const Element<DT>* a,
                                                        int64_t a_ld, const Element<DT>* b, int64_t b_ld, uint32_t rank,
                                                        float scale) {
  const uint32_t blocks = rank_blocks(rank), kp = padded_k(t.k), all_blocks = rank_blocks(t.max_rank);
  const size_t na = (size_t)blocks * kBlock * kp, nb = (size_t)groups_of(t.m) * blocks * kBlock * kGroup;
  const size_t step = (size_t)gridDim.x * kThreads;
  Element<DT>* ta = (Element<DT>*)t.a + (size_t)slot * a_elements(t);
  Element<DT>* tb = (Element<DT>*)t.b + (size_t)slot * b_elements(t);
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < na + nb; i += step) {
    if (i < na) {
      const uint32_t r = (uint32_t)(i / kp), c = (uint32_t)(i % kp);
      ta[i] = r < rank && c < t.k ? a[(size_t)r * (size_t)a_ld + c] : 0;
    } else {
      const size_t j = i - na;
      // j counts [group][block][half][t][n][8 ranks] of the blocks that the adapter has
      const uint32_t e = (uint32_t)(j & 7u), n = (uint32_t)(j >> 3) & 31u, tt = (uint32_t)(j >> 8) & 3u;
      const uint32_t half = (uint32_t)(j >> 10) & 1u;
      const size_t gb = j >> 11;
      const uint32_t block = (uint32_t)(gb % blocks);
      const size_t group = gb / blocks;
      const uint32_t r = block * kBlock + half * 8u + e;
      const size_t out = group * kGroup + 4u * n + tt;
      tb[(group * all_blocks + block) * (kBlock * kGroup) + (j & 2047u)] =
          r < rank && out < t.m ? b[out * (size_t)b_ld + r] : 0;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    t.ranks[slot] = rank;
    t.scales[slot] = scale;
  }
}

// ---------------------------------------------------------------- v_b = s_a A_a x_b

__device__ __forceinline__ uint32_t rank_of(const oxs_lora_table& t, uint32_t a) {
  return a < t.max_adapters ? min(t.ranks[a], t.max_rank) : 0u;
}

// The parts of one value, for the matrix cores; an infinity or NaN has one part.
__device__ __forceinline__ void store_value(void* workspace, uint32_t row, uint32_t all_blocks, uint32_t r, float v) {
  uint16_t* to = (uint16_t*)workspace + ((size_t)row * all_blocks + r / kBlock) * (kValueBytes / 2) + r % kBlock;
  const uint32_t p0 = narrow2(v, 0.0f) & 0xffffu;
  const bool finite = fabsf(low(p0)) < __builtin_inff();
  const float v1 = finite ? v - low(p0) : 0.0f;
  const uint32_t p1 = narrow2(v1, 0.0f) & 0xffffu;
  const uint32_t p2 = narrow2(v1 - low(p1), 0.0f) & 0xffffu;
  to[0] = (uint16_t)p0;
  to[kBlock] = (uint16_t)p1;
  to[2 * kBlock] = (uint16_t)p2;
}

template <int DT>
__device__ __forceinline__ Eight<DT> load_eight(const Element<DT>* p) {
  Eight<DT> e;
  e.q[0] = *(const u32x4*)p;
  if constexpr (DT == OXS_DTYPE_F32) e.q[1] = *(const u32x4*)(p + 4);
  return e;
}

// The same from memory aligned to its elements only.
template <int DT>
__device__ __forceinline__ Eight<DT> load_unaligned(const Element<DT>* p) {
  Eight<DT> e;
  __builtin_memcpy(&e, p, sizeof(e));
  return e;
}

// Where a row stands when the rows of its window are ordered by adapter, and what the second kernel has to know of it.
struct Place {
  uint32_t row, slot, rank, unused;
};
constexpr uint32_t kWindow = 1024;  // rows that are ordered among each other

__device__ __forceinline__ void place_row(const oxs_lora_batch& b, uint32_t row, uint32_t a,
                                          uint32_t rank, Place* places) {
  __shared__ uint32_t s_count[kWaves];
  const uint32_t start = row - row % kWindow, n = min(b.batch - start, kWindow);
  uint32_t other[kWindow / kThreads];  // (all loads before the first is waited for)
#pragma unroll
  for (uint32_t i = 0; i < kWindow / kThreads; ++i)
    other[i] = b.adapters[start + min(threadIdx.x + i * kThreads, n - 1u)];
  uint32_t before = 0;
#pragma unroll
  for (uint32_t i = 0; i < kWindow / kThreads; ++i) {
    const uint32_t j = threadIdx.x + i * kThreads;
    before += j < n && (other[i] < a || (other[i] == a && start + j < row)) ? 1u : 0u;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
  if ((threadIdx.x & 63u) == 0u) s_count[threadIdx.x >> 6] = before;
  __syncthreads();
  if (threadIdx.x == 0) places[start + s_count[0] + s_count[1] + s_count[2] + s_count[3]] = Place{row, a, rank, 0u};
}

// The sum over a wavefront's lanes, in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float plus_dpp(float x) {
  const int from = __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, ROWS, 0xf, false);
  return x + __uint_as_float((uint32_t)from);
}
__device__ __forceinline__ float wave_sum(float x) {
  x = plus_dpp<0x111, 0xf>(x);  // lanes 1, 2, 4, 8 below in the row of 16
  x = plus_dpp<0x112, 0xf>(x);
  x = plus_dpp<0x114, 0xf>(x);
  x = plus_dpp<0x118, 0xf>(x);
  x = plus_dpp<0x142, 0xa>(x);  // the row before, into rows 1 and 3
  x = plus_dpp<0x143, 0xc>(x);  // lane 31, into rows 2 and 3
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}

// The products of x with PER rows of A over one wavefront, whose lanes take eight values at a time. The loads of kAhead
// times 512 values are on their way together; lanes past the end load what others do, for nothing: a load behind a
// branch would be waited for on its own (64 rows of 4096 values, 16 ranks: 6.8 us so, 4.7 here). Twice and four times
// kAhead: 7.7 and 13.8 us for 7.3 (256 rows of 2048, f16 of rank 64), as fewer wavefronts fit.
template <int WT, int XT, int PER>
struct Dots {
  static constexpr uint32_t kAhead = PER == 1 ? 4 : WT == OXS_DTYPE_F32 ? 1 : 2, kStride = 512;
  const Element<XT>* x;
  uint32_t k, eights, lane;
  Eight<XT> xv[kAhead];
  float x_over;  // the values past the last eight, one in a lane
  __device__ __forceinline__ uint32_t at(uint32_t i) const { return i < eights ? i : 0u; }
  __device__ __forceinline__ void load_x(uint32_t i0) {
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) xv[j] = load_unaligned<XT>(x + at(i0 + lane * 8u + j * kStride));
  }
  // The first x, before the row's adapter is known.
  __device__ __forceinline__ Dots(const Element<XT>* x_, uint32_t k_, uint32_t lane_)
      : x(x_), k(k_), eights(k_ & ~7u), lane(lane_) {
    if (eights) load_x(0);
    const uint32_t over = eights + lane;
    x_over = lane < 8u && over < k ? widen<XT>(x[over]) : 0.0f;
  }
  // Leaves x as it was found, for the next rows.
  __device__ __forceinline__ float sum(const Element<WT>* w, bool again) {  // in lane p: row p's
    const uint32_t kp = padded_k(k);
    float s[PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) s[p] = 0.0f;
    for (uint32_t i0 = 0; i0 < eights;) {
      Eight<WT> wv[kAhead][PER];
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j)
#pragma unroll
        for (int p = 0; p < PER; ++p)
          wv[j][p] = load_eight<WT>(w + (size_t)p * kp + at(i0 + lane * 8u + j * kStride));
#pragma unroll
      for (uint32_t j = 0; j < kAhead; ++j) {
        const bool in = i0 + lane * 8u + j * kStride < eights;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = in ? xv[j][e] : 0.0f;
#pragma unroll
          for (int p = 0; p < PER; ++p) s[p] = __builtin_fmaf(wv[j][p][e], v, s[p]);
        }
      }
      i0 += kAhead * kStride;
      load_x(again && i0 >= eights ? 0u : i0);
    }
    if (eights < k && lane < 8u) {  // (the table's rows are padded to whole eights)
#pragma unroll
      for (int p = 0; p < PER; ++p)
        s[p] = __builtin_fmaf(widen<WT>(w[(size_t)p * kp + eights + lane]), x_over, s[p]);
    }
    float v = 0.0f;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const float all = wave_sum(s[p]);
      if (lane == (uint32_t)p) v = all;
    }
    return v;
  }
};

// One wavefront per (row, PER ranks). The last workgroup of a row finds the row's place instead.
template <int WT, int XT, int PER>
__global__ __launch_bounds__(kThreads) void shrink_kernel(oxs_lora_table t, oxs_lora_batch b, Place* places) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t row = blockIdx.x, r0 = (blockIdx.y * kWaves + wave) * PER;
  const uint32_t a = b.adapters[row];
  if (blockIdx.y + 1u == gridDim.y) {
    place_row(b, row, a, rank_of(t, a), places);
    return;
  }
  Dots<WT, XT, PER> dots((const Element<XT>*)b.x + (size_t)row * (size_t)b.x_ld, t.k, lane);
  const uint32_t rank = rank_of(t, a), all_blocks = rank_blocks(t.max_rank);
  // With a rank per wavefront the weights are not waited for until the adapter's rank is known: a slot has room for
  // max_rank whatever it holds.
  if (PER == 1 ? a >= t.max_adapters : r0 >= rank_blocks(rank) * kBlock) return;
  const float scale = t.scales[a];
  const float v = dots.sum((const Element<WT>*)t.a + (size_t)a * a_elements(t) + (size_t)r0 * padded_k(t.k), false);
  // ranks past the adapter's, up to the block's end, are zero
  if (lane < PER && r0 + lane < rank_blocks(rank) * kBlock)
    store_value(b.workspace, row, all_blocks, r0 + lane, r0 + lane < rank ? v * scale : 0.0f);
}

// ---------------------------------------------------------------- y_b += B_a v_b

// Row i of the 32 x 32 output held in register r of a lane in half g.
__device__ __forceinline__ uint32_t out_row(uint32_t r, uint32_t g) { return 8u * (r >> 2) + 4u * g + (r & 3u); }

// The bf16 parts of eight weights.
template <int WT>
struct Parts {
  static constexpr int N = WT == OXS_DTYPE_F32 ? 3 : WT == OXS_DTYPE_F16 ? 2 : 1;
  bf16x8 p[N];
  __device__ __forceinline__ Parts(const Eight<WT>& w) {
    if constexpr (WT == OXS_DTYPE_BF16) {
      p[0] = __builtin_bit_cast(bf16x8, w.q[0]);
    } else {
      u32x4 q[N];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = w[2 * i], y = w[2 * i + 1];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          q[n][i] = narrow2(x, y);
          x -= low(q[n][i]);
          y -= high(q[n][i]);
        }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) p[n] = __builtin_bit_cast(bf16x8, q[n]);
    }
  }
};

// The adapters among a tile's rows, and the rank blocks of each, one after the other.
struct Cursor {
  uint32_t rest;  // rows whose adapter has not begun
  uint32_t same;  // rows of the present one; 0 past the last
  uint32_t slot, block, rank;
  __device__ __forceinline__ void adapter(uint32_t ids, uint32_t ranks) {
    const uint32_t at = rest ? (uint32_t)__builtin_ctz(rest) : 0u;
    const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)at);
    const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)ranks, (int)at);
    same = (uint32_t)__ballot(ids == a) & rest;
    rest &= ~same;
    block = 0;
    if (same) {  // past the last the addresses stay where they were
      slot = a;
      rank = r;
    }
  }
  __device__ __forceinline__ void next(uint32_t ids, uint32_t ranks) {
    if (same && (block + 1u) * kBlock < rank) ++block;
    else adapter(ids, ranks);
  }
};

// One wavefront: `rows` <= 32 rows (in order of adapter; at most 8 with RR = 4, where only the first four registers of
// a tile hold any) x 32 TT outputs (lane n: outputs TT n .. TT n + TT - 1); a workgroup: the same rows and kWaves
// ranges of outputs side by side. The rows are the first operand, the outputs the second, so a register holds one
// row's 32 TT outputs side by side over 32 lanes. With RR = 16 every product goes onto the same sums, the values of
// the rows of other adapters being 0 (128 selections per adapter and rank block less: f16 93 -> 77 us, as above);
// with RR = 4 it is computed for all of the rows and taken for the adapter's own.
// The operands of the next PF (adapter, rank block) pairs are on their way while one is worked on. With 16-bit y and
// weights one leaves registers for a third wavefront per SIMD: 2048 rows of 32000, one adapter, 56 us for 64; with
// float32 y it does not (256 rows of 128256, 8 adapters of rank 64, 100 us for 95).
template <int WT, int YT, int TT, int PF, int RR>
__global__ __launch_bounds__(kThreads, RR == 4 || (PF == 1 && WT != OXS_DTYPE_F32) ? 3 : 2) void expand_kernel(
    oxs_lora_table t, oxs_lora_batch b, const Place* places, uint32_t rows, uint32_t col_groups, uint32_t vec) {
  const uint32_t lane = threadIdx.x & 63u, n = lane & 31u, g = lane >> 5;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t row_tile = blockIdx.x / col_groups;
  const uint32_t col = (blockIdx.x - row_tile * col_groups) * kWaves + wave;
  Place my = {0u, OXS_LORA_NONE, 0u, 0u};
  if (n < rows && row_tile * rows + n < b.batch) my = places[row_tile * rows + n];
  const uint32_t live = (uint32_t)__ballot(my.rank != 0u);
  if (live == 0u || col * 32u * TT >= t.m) return;
  const uint32_t all_blocks = rank_blocks(t.max_rank);
  constexpr uint32_t kPieces = kBlock * kGroup;  // elements of a group's rank block
  constexpr uint32_t kPerGroup = kGroup / (32u * TT);
  // outputs 32 TT col + TT n + tt: piece (q, n') of its group with 4 n' + q = output % 128
  const uint32_t out0 = col * 32u * TT + TT * n;
  const uint32_t in_group = (col % kPerGroup) * 32u * TT + TT * n;
  const Element<WT>* wb = (const Element<WT>*)t.b + (size_t)(col / kPerGroup) * all_blocks * kPieces +
                          (g * 4u + in_group % 4u) * 256u + (in_group / 4u) * 8u;
  const uint16_t* vb = (const uint16_t*)b.workspace + (size_t)my.row * all_blocks * (kValueBytes / 2) + g * 8u;

  Cursor ahead;
  Eight<WT> w[PF][TT];
  Eight<OXS_DTYPE_BF16> v[PF][kPlanes];
  uint32_t same[PF];
  const auto fetch = [&](int i) {
    const Element<WT>* p = wb + (size_t)ahead.slot * b_elements(t) + (size_t)ahead.block * kPieces;
    const bool in = g == 0u || ahead.block * kBlock + 8u < ahead.rank;  // this half holds a rank
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      w[i][tt] = Eight<WT>{};
      if (in) w[i][tt] = load_eight<WT>(p + tt * 256u);
    }
#pragma unroll
    for (int q = 0; q < (int)kPlanes; ++q)
      v[i][q] = load_eight<OXS_DTYPE_BF16>(vb + ahead.block * (kValueBytes / 2) + q * kBlock);
    same[i] = ahead.same;
    ahead.next(my.slot, my.rank);
  };
  const auto begin = [&]() {
    ahead.rest = live;
    ahead.slot = ahead.rank = 0;
    ahead.adapter(my.slot, my.rank);
#pragma unroll
    for (int i = 0; i < PF; ++i) fetch(i);
  };
  begin();
  const bool one = same[0] == live;  // adapter for all rows

  // y, where a row has an adapter
  const uint32_t mine = live >> (4u * g);  // bit 8 (r / 4) + r % 4: register r's row
  using YE = Element<YT>;
  struct alignas(TT * sizeof(YE)) Vec {
    YE e[TT];
  };
  const auto y_at = [&](int r) {
    const uint32_t row = (uint32_t)__shfl((int)my.row, (int)out_row(r, g));
    return (YE*)b.y + (size_t)row * (size_t)b.y_ld + out0;
  };
  // (1024 rows of 128256 float32, 8 adapters: 238 us where y is aligned)
  const bool inside = (uint64_t)(col + 1u) * 32u * TT <= t.m, whole = vec != 0u && inside;
  Vec old[RR];
  const auto load_old = [&]() {
    if (whole) {
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const YE* p = y_at(r);
        if ((mine >> (8 * (r / 4) + r % 4)) & 1u) old[r] = *(const Vec*)p;
      }
    } else if (inside) {  // aligned to its elements only: in one access all the same (as above: 252 us, one by one 392)
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const YE* p = y_at(r);
        if ((mine >> (8 * (r / 4) + r % 4)) & 1u) __builtin_memcpy(&old[r], p, sizeof(Vec));
      }
    } else {
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        const YE* p = y_at(r);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
          if (((mine >> (8 * (r / 4) + r % 4)) & 1u) && out0 + tt < t.m) old[r].e[tt] = p[tt];
      }
    }
  };
  load_old();

  typedef float Acc __attribute__((ext_vector_type(RR)));
  Acc acc[TT];
  // The products of all adapters. TAKE: computed for all rows and taken for the adapter's own; otherwise onto the sums,
  // with values of 0 for the other rows.
  const auto products = [&](auto take) {
    constexpr bool TAKE = decltype(take)::value;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[tt] = Acc{};
    do {
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const uint32_t s = same[i];
        if (s) {
          bf16x8 vp[kPlanes];
#pragma unroll
          for (int q = 0; q < (int)kPlanes; ++q) {
            u32x4 x = v[i][q].q[0];
            if constexpr (!TAKE) {
#pragma unroll
              for (int j = 0; j < 4; ++j) x[j] = (s >> n) & 1u ? x[j] : 0u;
            }
            vp[q] = __builtin_bit_cast(bf16x8, x);
          }
          const uint32_t bits = s >> (4u * g);
#pragma unroll
          for (int tt = 0; tt < TT; ++tt) {
            const Parts<WT> wp(w[i][tt]);
            f32x16 d = {};
            if constexpr (!TAKE) {
#pragma unroll
              for (int r = 0; r < RR; ++r) d[r] = acc[tt][r];
            }
#pragma unroll
            for (int sum = 2; sum >= 0; --sum)  // the small products first
#pragma unroll
              for (int q = 0; q < Parts<WT>::N; ++q)
                if (q <= sum) d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vp[sum - q], wp.p[q], d, 0, 0, 0);
            if constexpr (TAKE) {
#pragma unroll
              for (int r = 0; r < RR; ++r) acc[tt][r] += (bits >> (8 * (r / 4) + r % 4)) & 1u ? d[r] : 0.0f;
            } else {
#pragma unroll
              for (int r = 0; r < RR; ++r) acc[tt][r] = d[r];
            }
          }
        }
        fetch(i);
      }
    } while (same[0]);
  };
  if constexpr (RR == 4) {
    products(std::true_type{});
  } else {
    products(std::false_type{});
    if (!one) {
      // 0 times an infinite weight is NaN in the other rows: once more, then, row by row
      float bad = 0.0f;
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int r = 0; r < RR; ++r) bad = __builtin_fmaf(acc[tt][r], 0.0f, bad);
      if (__ballot(bad != bad)) {
        begin();
        products(std::true_type{});
        load_old();  // (as it is: kept through the second pass, it would not fit in registers)
      }
    }
  }

  const auto sum = [&](int r) {
    Vec z;
    if constexpr (YT == OXS_DTYPE_BF16 && TT % 2 == 0) {
#pragma unroll
      for (int tt = 0; tt < TT; tt += 2) {
        const uint32_t pair =
            narrow2(widen<YT>(old[r].e[tt]) + acc[tt][r], widen<YT>(old[r].e[tt + 1]) + acc[tt + 1][r]);
        z.e[tt] = (YE)pair;
        z.e[tt + 1] = (YE)(pair >> 16);
      }
    } else {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) z.e[tt] = __float_as_uint(widen<YT>(old[r].e[tt]) + acc[tt][r]);
    }
    return z;
  };
  if (whole) {
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      YE* p = y_at(r);
      if ((mine >> (8 * (r / 4) + r % 4)) & 1u) *(Vec*)p = sum(r);
    }
  } else if (inside) {
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      YE* p = y_at(r);
      const Vec z = sum(r);
      if ((mine >> (8 * (r / 4) + r % 4)) & 1u) __builtin_memcpy(p, &z, sizeof(Vec));
    }
  } else {
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      YE* p = y_at(r);
      const Vec z = sum(r);
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
        if (((mine >> (8 * (r / 4) + r % 4)) & 1u) && out0 + tt < t.m) p[tt] = z.e[tt];
    }
  }
}

// ---------------------------------------------------------------- few rows: both products in one launch

// One workgroup: a row and kWaves * 128 outputs. It computes all of the row's v for itself, with B's first weights and
// y on their way meanwhile; lane (n, g) of a wavefront then has half g of the ranks of a block for outputs 4 n to
// 4 n + 3.
template <int WT, int XT, int YT>
__global__ __launch_bounds__(kThreads) void single_kernel(oxs_lora_table t, oxs_lora_batch b) {
  const uint32_t lane = threadIdx.x & 63u, n = lane & 31u, g = lane >> 5;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t row = blockIdx.y, col = blockIdx.x * kWaves + wave;
  __shared__ float s_v[OXS_LORA_MAX_RANK];
  const uint32_t a = b.adapters[row];
  Dots<WT, XT, 4> dots((const Element<XT>*)b.x + (size_t)row * (size_t)b.x_ld, t.k, lane);
  const uint32_t rank = rank_of(t, a), blocks = rank_blocks(rank);
  if (rank == 0u) return;
  const float scale = t.scales[a];
  const bool mine = (uint64_t)col * kGroup < t.m;  // this wavefront has outputs
  const Element<WT>* w = (const Element<WT>*)t.b + (size_t)a * b_elements(t) +
                         (size_t)(mine ? col : 0u) * rank_blocks(t.max_rank) * (kBlock * kGroup) + n * 8u;
  Eight<WT> wv[4];
  // A half that holds no rank takes the other's weights, to be multiplied by values of 0.
  const auto fetch = [&](uint32_t block) {
    const Element<WT>* p = w + (size_t)block * (kBlock * kGroup) + (block * kBlock + 8u * g < rank ? g * 1024u : 0u);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) wv[tt] = load_eight<WT>(p + tt * 256u);
  };
  fetch(0);
  using YE = Element<YT>;
  const uint32_t out = col * kGroup + 4u * n;
  YE* y = (YE*)b.y + (size_t)row * (size_t)b.y_ld;
  struct Vec {
    YE e[4];
  } old;
  const bool inside = (uint64_t)(col + 1u) * kGroup <= t.m;
  if (inside) {
    __builtin_memcpy(&old, y + out, sizeof(Vec));
  } else {
#pragma unroll
    for (uint32_t tt = 0; tt < 4; ++tt) old.e[tt] = y[min((uint64_t)out + tt, (uint64_t)t.m - 1u)];
  }
  const Element<WT>* wa = (const Element<WT>*)t.a + (size_t)a * a_elements(t) + (size_t)(wave * 4u) * padded_k(t.k);
  for (uint32_t block = 0; block < blocks; ++block) {
    const float v = dots.sum(wa + (size_t)block * kBlock * padded_k(t.k), block + 1u < blocks);
    const uint32_t r = block * kBlock + wave * 4u + lane;
    if (lane < 4u) s_v[r] = r < rank ? v * scale : 0.0f;
  }
  __syncthreads();
  if (!mine) return;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t block = 0; block < blocks; ++block) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s_v[block * kBlock + g * 8u + j];
    const Eight<WT> now[4] = {wv[0], wv[1], wv[2], wv[3]};
    fetch(min(block + 1u, blocks - 1u));
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[tt] = __builtin_fmaf(now[tt][j], v[j], acc[tt]);
  }
  Vec z;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    const float sum = widen<YT>(old.e[tt]) + (acc[tt] + __shfl_xor(acc[tt], 32));
    if constexpr (YT == OXS_DTYPE_BF16) z.e[tt] = (YE)narrow2(sum, 0.0f);
    else z.e[tt] = __float_as_uint(sum);
  }
  if (g) return;
  if (inside) {
    __builtin_memcpy(y + out, &z, sizeof(Vec));
  } else {
#pragma unroll
    for (uint32_t tt = 0; tt < 4; ++tt)
      if ((uint64_t)out + tt < t.m) y[out + tt] = z.e[tt];
  }
}

static bool known(int32_t dt, bool half) {
  return dt == OXS_DTYPE_F32 || dt == OXS_DTYPE_BF16 || (half && dt == OXS_DTYPE_F16);
}
static uint32_t size_of(int32_t dt) { return dt == OXS_DTYPE_F32 ? 4u : 2u; }
static bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1u)) == 0; }
static bool sizes_ok(const oxs_lora_table* t) {
  return t && t->m && t->k && t->max_adapters && t->max_rank && t->max_rank <= OXS_LORA_MAX_RANK &&
         t->m <= (1u << 30) && t->k <= (1u << 30) && t->max_adapters <= 65536u && known(t->dtype, true);
}
static bool table_ok(const oxs_lora_table* t) {
  return sizes_ok(t) && t->a && t->b && t->ranks && t->scales && aligned(t->a, 16) && aligned(t->b, 16) &&
         aligned(t->ranks, 4) && aligned(t->scales, 4);
}
static int launched() { return hipGetLastError() == hipSuccess ? OXS_OK : OXS_ERR_HIP; }

template <int V>
using Int = std::integral_constant<int, V>;
template <class F>
static void by_weights(int32_t dt, F f) {
  if (dt == OXS_DTYPE_F32) f(Int<OXS_DTYPE_F32>{});
  else if (dt == OXS_DTYPE_BF16) f(Int<OXS_DTYPE_BF16>{});
  else f(Int<OXS_DTYPE_F16>{});
}
template <class F>
static void by_values(int32_t dt, F f) {
  if (dt == OXS_DTYPE_F32) f(Int<OXS_DTYPE_F32>{});
  else f(Int<OXS_DTYPE_BF16>{});
}

}  // namespace oxs_lora

extern "C" int oxs_lora_table_bytes(const oxs_lora_table* table, size_t* a_bytes, size_t* b_bytes) {
  using namespace oxs_lora;
  if (!sizes_ok(table) || !a_bytes || !b_bytes) return OXS_ERR_INVALID_ARGUMENT;
  const size_t per = (size_t)table->max_adapters * size_of(table->dtype);
  *a_bytes = per * a_elements(*table);
  *b_bytes = per * b_elements(*table);
  return OXS_OK;
}

extern "C" int oxs_lora_load(const oxs_lora_table* table, uint32_t slot, const void* a, int64_t a_ld, const void* b,
                             int64_t b_ld, uint32_t rank, float scale, void* stream) {
  using namespace oxs_lora;
  if (!table_ok(table) || slot >= table->max_adapters || rank > table->max_rank) return OXS_ERR_INVALID_ARGUMENT;
  if (rank) {
    const uint32_t es = size_of(table->dtype);
    if (!a || !b || !aligned(a, es) || !aligned(b, es)) return OXS_ERR_INVALID_ARGUMENT;
    if ((rank > 1 && a_ld < (int64_t)table->k) || (table->m > 1 && b_ld < (int64_t)rank))
      return OXS_ERR_INVALID_ARGUMENT;
  }
  by_weights(table->dtype, [&](auto wt) {
    using E = Element<decltype(wt)::value>;
    hipLaunchKernelGGL(load_kernel<decltype(wt)::value>, dim3(1024), dim3(kThreads), 0, (hipStream_t)stream, *table,
                       slot, (const E*)a, a_ld, (const E*)b, b_ld, rank, scale);
  });
  return launched();
}

extern "C" size_t oxs_lora_workspace_bytes(const oxs_lora_table* table, uint32_t batch) {
  using namespace oxs_lora;
  if (!sizes_ok(table) || batch > 65536u) return 0;
  return (size_t)(batch ? batch : 1u) * (rank_blocks(table->max_rank) * kValueBytes + sizeof(Place));
}

extern "C" int oxs_lora_add(const oxs_lora_table* table, const oxs_lora_batch* batch, void* stream) {
  using namespace oxs_lora;
  if (!table_ok(table) || !batch) return OXS_ERR_INVALID_ARGUMENT;
  const oxs_lora_table& t = *table;
  const oxs_lora_batch& b = *batch;
  if (b.batch == 0) return OXS_OK;
  if (b.batch > 65536u) return OXS_ERR_LIMITS;
  if (!known(b.x_dtype, false) || !known(b.y_dtype, false)) return OXS_ERR_INVALID_ARGUMENT;
  if (!b.x || !b.y || !b.adapters || !b.workspace) return OXS_ERR_INVALID_ARGUMENT;
  if (b.batch > 1 && (b.x_ld < (int64_t)t.k || b.y_ld < (int64_t)t.m)) return OXS_ERR_INVALID_ARGUMENT;
  if (!aligned(b.x, size_of(b.x_dtype)) || !aligned(b.y, size_of(b.y_dtype)) || !aligned(b.adapters, 4) ||
      !aligned(b.workspace, 16) || b.workspace_bytes < oxs_lora_workspace_bytes(table, b.batch))
    return OXS_ERR_INVALID_ARGUMENT;
  if ((uint64_t)b.batch * t.m > (1ull << 31)) return OXS_ERR_LIMITS;
  const hipStream_t st = (hipStream_t)stream;
  const uint32_t blocks = rank_blocks(t.max_rank);
  Place* places = (Place*)((char*)b.workspace + (size_t)b.batch * blocks * kValueBytes);
  const auto even = [&](const void* p, int64_t ld, uint32_t es, uint32_t to) {
    return aligned(p, to) && (b.batch == 1 || ((uint64_t)ld * es) % to == 0);
  };
  // Both products in one launch while no workgroup has much of A to read, all together have not, and they are few. One
  // launch and two, us, replayed from a graph, rank 16 in bf16: one row of 32000 outputs, 896 inputs 3.3 and 5.9, 4096
  // 4.5 and 6.2, 8192 6.0 and 7.0, 4096 of rank 64 10.6 and 7.5; 128256 outputs, 4096 inputs, 1 row 4.8 and 7.0, 2 rows
  // 6.8 and 7.7, 4 rows 10.7 and 8.8; 512 inputs, 64 rows of 8000 6.0 and 6.8, 200 rows 14.7 and 8.8.
  const uint32_t singles = (t.m + kWaves * kGroup - 1u) / (kWaves * kGroup);
  const uint64_t a_bytes = (uint64_t)blocks * kBlock * padded_k(t.k) * size_of(t.dtype);
  const uint64_t groups = (uint64_t)b.batch * singles;
  if (groups <= 1024u && a_bytes <= (256u << 10) && groups * a_bytes <= (80u << 20)) {
    by_weights(t.dtype, [&](auto wt) {
      by_values(b.x_dtype, [&](auto xt) {
        by_values(b.y_dtype, [&](auto yt) {
          hipLaunchKernelGGL((single_kernel<decltype(wt)::value, decltype(xt)::value, decltype(yt)::value>),
                             dim3(singles, b.batch), dim3(kThreads), 0, st, t, b);
        });
      });
    });
    return launched();
  }
  by_weights(t.dtype, [&](auto wt) {
    constexpr int WT = decltype(wt)::value;
    by_values(b.x_dtype, [&](auto xt) {
      constexpr int XT = decltype(xt)::value;
      // A wavefront per 4 ranks reads x a quarter as often, one per rank has less to wait for: 128 rows of 4096 inputs,
      // rank 16, 8.7 and 8.5 us (both products, 2000 outputs), 192 rows 9.0 and 9.7, 1024 rows of rank 32 29 and 44.
      if ((uint64_t)b.batch * blocks >= 160u)
        hipLaunchKernelGGL((shrink_kernel<WT, XT, 4>), dim3(b.batch, blocks + 1u), dim3(kThreads), 0, st, t, b, places);
      else
        hipLaunchKernelGGL((shrink_kernel<WT, XT, 1>), dim3(b.batch, blocks * 4u + 1u), dim3(kThreads), 0, st, t, b,
                           places);
    });
    by_values(b.y_dtype, [&](auto yt) {
      constexpr int YT = decltype(yt)::value;
      const auto groups = [&](uint32_t outputs) { return (t.m + outputs * kWaves - 1u) / (outputs * kWaves); };
      const auto go = [&](auto kernel, auto width, uint32_t rows) {
        constexpr uint32_t TT = decltype(width)::value;
        const uint32_t vec = even(b.y, b.y_ld, size_of(YT), TT * size_of(YT)) ? 1u : 0u;
        const uint32_t row_tiles = (b.batch + rows - 1u) / rows;
        uint32_t col_groups = groups(32u * TT);
        // a multiple of 8: the workgroups of a range of outputs are all on one XCD, whose L2 then holds its weights
        // (prompts as above 228 -> 223 us)
        if (row_tiles > 1u) col_groups = (col_groups + 7u) / 8u * 8u;
        hipLaunchKernelGGL(kernel, dim3(row_tiles * col_groups), dim3(kThreads), 0, st, t, b, places, rows, col_groups,
                           vec);
      };
      // Tiles of 8 rows where those of 32 would be too few workgroups for the card: then each waits less, for fewer
      // adapters. Tiles of 32 and of 8 rows, us, rank 16 in bf16: 126 workgroups (64 rows of 32000 outputs, 64
      // adapters) 28.6 and 18.3; 198 (48 rows of 50257, 1 and 32) 15.9 and 15.3, 34.9 and 28.0; 251 (32 rows of 128256,
      // 1 and 32) 11.7 and 14.1, 31.4 and 31.0; 502 (64 rows, 1 and 16) 16.6 and 20.1, 25.5 and 26.0. f16, rank 32,
      // bf16 outputs: 251 (1 and 32) 10.2 and 13.3, 86 and 53; 502 (1 and 16) 13.7 and 21.3, 33.8 and 32.6.
      const uint32_t few = WT == OXS_DTYPE_F16 ? 256u : 200u;
      // Outputs per lane in tiles of 8 rows: f32 weights fill the registers at 4 (24 rows of 50257 outputs with an
      // adapter each: 18.5 us with 2, 22.0 with 4), the others' loads are wider for it (64 rows of 32000, 8 adapters:
      // 11.9 with 2, 9.5 with 4).
      constexpr int kFew = WT == OXS_DTYPE_F32 ? 2 : 4;
      if ((uint64_t)((b.batch + kRows - 1u) / kRows) * groups(128u) <= few)
        go(expand_kernel<WT, YT, kFew, 2, 4>, Int<kFew>{}, 8u);
      else
        go(expand_kernel<WT, YT, 4, YT == OXS_DTYPE_BF16 ? 1 : 2, 16>, Int<4>{}, kRows);
    });
  });
  return launched();
}

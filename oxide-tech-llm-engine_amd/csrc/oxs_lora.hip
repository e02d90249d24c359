// oxs_lora.hip — low-rank adapters of many requests beside the projection
// that they share: y_b += B_a (s_a A_a x_b) for the adapter a of each row b.
//
// Two launches: v_b = s_a A_a x_b into the workspace, then y_b += B_a v_b. A
// wavefront sums one value of v; a thread owns one value of y.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/oxide_sampler.h"

namespace oxs_lora {

constexpr int kThreads = 256;

template <int DT>
__device__ __forceinline__ float load(const void* p, size_t i) {
  if constexpr (DT == OXS_DTYPE_F32) return ((const float*)p)[i];
  else if constexpr (DT == OXS_DTYPE_F16) return (float)((const _Float16*)p)[i];
  else return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

// a value rounded to bf16, to the nearest, ties to even; NaN stays NaN
__device__ __forceinline__ uint16_t to_bf16(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void load_kernel(oxs_lora_table t, uint32_t slot, const void* a, int64_t a_ld,
                                                        const void* b, int64_t b_ld, uint32_t rank, float scale) {
  using E = std::conditional_t<DT == OXS_DTYPE_F32, uint32_t, uint16_t>;
  const size_t na = (size_t)rank * t.k, nb = (size_t)rank * t.m;
  const size_t step = (size_t)gridDim.x * kThreads;
  E* ta = (E*)t.a + (size_t)slot * t.max_rank * t.k;
  E* tb = (E*)t.b + (size_t)slot * t.max_rank * t.m;
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < na + nb; i += step) {
    if (i < na) ta[i] = ((const E*)a)[(i / t.k) * (size_t)a_ld + i % t.k];
    else {
      const size_t j = i - na;
      tb[(j / rank) * t.max_rank + j % rank] = ((const E*)b)[(j / rank) * (size_t)b_ld + j % rank];
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    t.ranks[slot] = rank;
    t.scales[slot] = scale;
  }
}

template <int WT, int XT>
__global__ __launch_bounds__(kThreads) void shrink_kernel(oxs_lora_table t, oxs_lora_batch b) {
  const uint32_t row = blockIdx.x, r = blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
  const uint32_t a = b.adapters[row];
  if (a >= t.max_adapters || r >= min(t.ranks[a], t.max_rank)) return;
  const size_t w0 = ((size_t)a * t.max_rank + r) * t.k, x0 = (size_t)row * (size_t)b.x_ld;
  float s = 0.0f;
  for (uint32_t i = lane; i < t.k; i += 64) s = __builtin_fmaf(load<WT>(t.a, w0 + i), load<XT>(b.x, x0 + i), s);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) ((float*)b.workspace)[(size_t)row * t.max_rank + r] = s * t.scales[a];
}

template <int WT, int YT>
__global__ __launch_bounds__(kThreads) void expand_kernel(oxs_lora_table t, oxs_lora_batch b) {
  const uint32_t blocks = (t.m + kThreads - 1) / kThreads;
  const uint32_t row = blockIdx.x / blocks, i = (blockIdx.x % blocks) * kThreads + threadIdx.x;
  const uint32_t a = b.adapters[row];
  if (a >= t.max_adapters || i >= t.m) return;
  const uint32_t rank = min(t.ranks[a], t.max_rank);
  if (rank == 0) return;
  const float* v = (const float*)b.workspace + (size_t)row * t.max_rank;
  const size_t w0 = ((size_t)a * t.m + i) * t.max_rank, at = (size_t)row * (size_t)b.y_ld + i;
  float s = 0.0f;
  for (uint32_t r = 0; r < rank; ++r) s = __builtin_fmaf(load<WT>(t.b, w0 + r), v[r], s);
  const float y = load<YT>(b.y, at) + s;
  if constexpr (YT == OXS_DTYPE_F32) ((float*)b.y)[at] = y;
  else ((uint16_t*)b.y)[at] = to_bf16(y);
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
  const size_t per = (size_t)table->max_adapters * table->max_rank * size_of(table->dtype);
  *a_bytes = per * table->k;
  *b_bytes = per * table->m;
  return OXS_OK;
}

extern "C" int oxs_lora_load(const oxs_lora_table* table, uint32_t slot, const void* a, int64_t a_ld, const void* b,
                             int64_t b_ld, uint32_t rank, float scale, void* stream) {
  using namespace oxs_lora;
  if (!table_ok(table) || slot >= table->max_adapters || rank > table->max_rank) return OXS_ERR_INVALID_ARGUMENT;
  if (rank) {
    const uint32_t es = size_of(table->dtype);
    if (!a || !b || !aligned(a, es) || !aligned(b, es)) return OXS_ERR_INVALID_ARGUMENT;
    if ((rank > 1 && a_ld < (int64_t)table->k) || (table->m > 1 && b_ld < (int64_t)rank)) return OXS_ERR_INVALID_ARGUMENT;
  }
  by_weights(table->dtype, [&](auto wt) {
    hipLaunchKernelGGL(load_kernel<decltype(wt)::value>, dim3(1024), dim3(kThreads), 0, (hipStream_t)stream, *table,
                       slot, a, a_ld, b, b_ld, rank, scale);
  });
  return launched();
}

extern "C" size_t oxs_lora_workspace_bytes(const oxs_lora_table* table, uint32_t batch) {
  using namespace oxs_lora;
  if (!sizes_ok(table) || batch > 65536u) return 0;
  return (size_t)(batch ? batch : 1u) * table->max_rank * 4u;
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
  const uint64_t grid = (uint64_t)((t.m + kThreads - 1) / kThreads) * b.batch;
  if (grid >= (1u << 24)) return OXS_ERR_LIMITS;
  by_weights(t.dtype, [&](auto wt) {
    constexpr int WT = decltype(wt)::value;
    by_values(b.x_dtype, [&](auto xt) {
      hipLaunchKernelGGL((shrink_kernel<WT, decltype(xt)::value>), dim3(b.batch, (t.max_rank + 3) / 4), dim3(kThreads),
                         0, (hipStream_t)stream, t, b);
    });
    by_values(b.y_dtype, [&](auto yt) {
      hipLaunchKernelGGL((expand_kernel<WT, decltype(yt)::value>), dim3((uint32_t)grid), dim3(kThreads), 0,
                         (hipStream_t)stream, t, b);
    });
  });
  return launched();
}

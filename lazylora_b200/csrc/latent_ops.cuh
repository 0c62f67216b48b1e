// Shared pieces of the latent-attention kernels (latent_cache.cu, latent_paged.cu,
// latent_expand.cu): the 16-bit types, the status word and the packed sequences' tile lookup.
#pragma once
#include <algorithm>

#include "host_common.cuh"
#include "ops.cuh"

namespace ll {

// The status word of the latent-attention launches on the current device (zero-initialised;
// ll_latent_status reads and clears it). nullptr when the CUDA call failed.
DevStatus* latent_status();

template <class T>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static constexpr uint32_t fmt = 1;     // kind::f16 operand format code
  static constexpr CUtensorMapDataType tma = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  LL_DEV static float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  LL_DEV static __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
  LL_DEV static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <>
struct Num<__half> {
  static constexpr uint32_t fmt = 0;
  static constexpr CUtensorMapDataType tma = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  LL_DEV static float to_f(__half v) { return __half2float(v); }
  LL_DEV static __half from_f(float v) { return __float2half_rn(v); }
  LL_DEV static uint32_t pack(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// Rows of sequence b in a packed tensor of `total` rows: [lo, hi), clamped into the tensor so that
// no value of cu can lead outside it.
LL_DEV void seq_range(const int32_t* cu, int b, int total, int& lo, int& hi) {
  lo = min(max(cu[b], 0), total);
  hi = min(max(cu[b + 1], lo), total);
}

// The tile-th tile of `rows` rows over all sequences, counted from the last one, for a whole warp:
// true and (b, first row within the sequence) when there is one. Lanes scan 32 sequences at a time.
// Counting from the end starts each sequence's causal tiles with the longest, so the short ones
// fill the launch's tail.
LL_DEV bool find_tile_from_end(const int32_t* cu, int B, int total, int rows, int tile, int& b, int& row0) {
  const int lane = threadIdx.x & 31;
  for (int hi_b = B; hi_b > 0; hi_b -= 32) {
    const int bb = hi_b - 1 - lane;
    int n = 0;
    if (bb >= 0) {
      int lo, hi;
      seq_range(cu, bb, total, lo, hi);
      n = (hi - lo + rows - 1) / rows;
    }
    int sum = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += v;
    }
    const int all = __shfl_sync(0xffffffffu, sum, 31);
    if (tile < all) {
      const uint32_t hit = __ballot_sync(0xffffffffu, tile < sum);
      const int src = __ffs(hit) - 1;
      b = hi_b - 1 - src;
      const int end = __shfl_sync(0xffffffffu, sum, src), cnt = __shfl_sync(0xffffffffu, n, src);
      row0 = (cnt - 1 - (tile - (end - cnt))) * rows;
      return true;
    }
    tile -= all;
  }
  return false;
}

}  // namespace ll

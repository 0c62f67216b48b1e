// The absorbed form of latent attention over a paged cache (see the header for the interface): all
// rows of a sequence's queries read the same cache rows, which are keys (all d_c + d_r values) and
// values (the first d_c) at once.
//   s_j = scale q . row_j,  m = max_j s_j,  p_j = exp(s_j - m),  l = sum_j p_j,
//   out = (sum_j p_j row_j[:d_c]) / l,  lse = m + log l.
// First form: one block per (sequence, 16 query rows), each warp two rows, a lane per key of a
// 32-key tile, running maximum and sum; CUDA cores throughout.
#include "latent_ops.cuh"

namespace ll {

struct PagedArgs {
  const void* q;
  const void* cache;
  const int32_t* bt;
  const int32_t* lens;
  void* out;
  float* lse;
  int64_t q_b, q_t, q_h, page_stride, row_stride, bt_stride;
  int pages, page_size, max_pages, Tq, H, d_c, d_r;
  float scale;
  DevStatus* st;
};

template <class T>
__global__ void __launch_bounds__(256) k_paged_simple(const PagedArgs a) {
  extern __shared__ float sm[];
  const int D = a.d_c + a.d_r, ld = D + 1;
  float* qs = sm;                 // [16][D]
  float* ks = sm + 16 * D;        // [32][ld]
  const int b = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32, rows = a.Tq * a.H;
  const int len = min(max(a.lens[b], 0), a.max_pages * a.page_size);
  for (int i = threadIdx.x; i < 16 * D; i += 256) {
    const int r = blockIdx.x * 16 + i / D;
    qs[i] = r < rows ? Num<T>::to_f(static_cast<const T*>(a.q)[b * a.q_b + (r / a.H) * a.q_t + (r % a.H) * a.q_h + i % D]) : 0.f;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0}, o[2][16] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * D; i += 256) {
      const int j = j0 + i / D;
      float v = 0.f;
      if (j < len) {
        const int pg = a.bt[b * a.bt_stride + j / a.page_size];
        if (pg >= 0 && pg < a.pages)
          v = Num<T>::to_f(static_cast<const T*>(a.cache)[pg * a.page_stride + (j % a.page_size) * a.row_stride + i % D]);
        else report(a.st, LL_ERR_RANGE, 73, b);
      }
      ks[(i / D) * ld + i % D] = v;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int r = blockIdx.x * 16 + warp * 2 + u;
      const int lim = len - a.Tq + r / a.H + 1;
      float s = 0.f;
      for (int d = 0; d < D; d++) s = fmaf(qs[(warp * 2 + u) * D + d], ks[lane * ld + d], s);
      s = j0 + lane < lim ? s * a.scale : -INFINITY;
      float mx = s;
      for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, off));
      mx = fmaxf(mx, m[u]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      const float p = __expf(s - ref), f = __expf(m[u] - ref);
      float ps = p;
      for (int off = 16; off; off >>= 1) ps += __shfl_xor_sync(~0u, ps, off);
      l[u] = l[u] * f + ps;
      m[u] = mx;
      for (int i = 0; i < 16; i++) o[u][i] *= f;
      for (int j = 0; j < 32; j++) {
        const float pj = __shfl_sync(~0u, p, j);
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (i * 32 < a.d_c) o[u][i] = fmaf(pj, ks[j * ld + i * 32 + lane], o[u][i]);
      }
    }
  }
  for (int u = 0; u < 2; u++) {
    const int r = blockIdx.x * 16 + warp * 2 + u;
    if (r >= rows) continue;
    const int64_t row = (int64_t)b * rows + r;
    for (int i = 0; i * 32 < a.d_c; i++)
      static_cast<T*>(a.out)[row * a.d_c + i * 32 + lane] = Num<T>::from_f(l[u] > 0.f ? o[u][i] / l[u] : 0.f);
    if (lane == 0) a.lse[row] = l[u] > 0.f ? m[u] + logf(l[u]) : -INFINITY;
  }
}

}  // namespace ll

using namespace ll;

extern "C" {

size_t ll_paged_latent_workspace_bytes(int B, int Tq, int H, int d_c) { return B > 0 && Tq > 0 && H > 0 && d_c > 0 ? 256 : 0; }

int ll_paged_latent_attention(const void* q, int64_t q_stride_b, int64_t q_stride_t, int64_t q_stride_h,
                              const void* cache, int64_t page_stride, int64_t row_stride, int pages, int page_size,
                              const int32_t* block_table, int64_t table_stride, int max_pages, const int32_t* seq_lens,
                              int B, int Tq, int H, int d_c, int d_r, float scale, int dtype, void* out, float* lse,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || Tq <= 0 || H <= 0 || d_c <= 0 || d_c % 128 || d_c > 512 || (d_r != 0 && d_r != 64) ||
      (dtype != 1 && dtype != 2) || pages <= 0 || page_size <= 0 || page_size % 8 || max_pages <= 0)
    return LL_ERR_ARG;
  if (B == 0) return LL_OK;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  PagedArgs a{q, cache, block_table, seq_lens, out, lse, q_stride_b, q_stride_t, q_stride_h, page_stride, row_stride,
              table_stride, pages, page_size, max_pages, Tq, H, d_c, d_r, scale, latent_status()};
  const int D = d_c + d_r, smem = (16 * D + 32 * (D + 1)) * 4;
  auto kern = dtype == 1 ? k_paged_simple<__nv_bfloat16> : k_paged_simple<__half>;
  LL_TRY(set_smem_attr(reinterpret_cast<const void*>(kern), smem));
  kern<<<dim3((Tq * H + 15) / 16, B), 256, smem, s>>>(a);
  return check_launch("k_paged_simple");
}

}  // extern "C"

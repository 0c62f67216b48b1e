// The expanded form of latent attention on packed sequences, forward and backward (see the header
// for the interface). Per head, with k = (k_nope | k_pe):
//   s_ij = scale q_i . k_j (visible j),  p = softmax(s),  o_i = sum_j p_ij v_j,
//   dv_j = sum_i p_ij g_i,  dp_ij = g_i . v_j,  ds_ij = p_ij (dp_ij - g_i . o_i) scale,
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i;  dk_pe sums dk's rotary part over the heads.
// First form: one block per (32 rows, head), each warp four rows, a lane per row of the other side;
// CUDA cores throughout. The backward pass runs one kernel over query rows (dq) and one over key
// rows (dk, dv), so that every sum has a fixed order.
#include "latent_ops.cuh"

namespace ll {

struct ExpandArgs {
  ll_latent_packed p;
  const void* g;
  int64_t g_t, g_h;
  const void* o;
  const float* lse_in;
  void* out;
  float* lse;
  void *dq, *dk, *dkpe, *dv;
  float* dkpe_ws;          // [H][Tk][d_r]
};

template <class T>
LL_DEV float k_at(const ll_latent_packed& p, int64_t row, int h, int d) {
  return Num<T>::to_f(d < p.d_n ? static_cast<const T*>(p.k_nope)[row * p.k_stride_t + h * p.k_stride_h + d]
                                : static_cast<const T*>(p.k_pe)[row * p.kpe_stride_t + d - p.d_n]);
}
template <class T>
LL_DEV float q_at(const ll_latent_packed& p, int64_t row, int h, int d) {
  return Num<T>::to_f(static_cast<const T*>(p.q)[row * p.q_stride_t + h * p.q_stride_h + d]);
}
template <class T>
LL_DEV float v_at(const ll_latent_packed& p, int64_t row, int h, int d) {
  return Num<T>::to_f(static_cast<const T*>(p.v)[row * p.v_stride_t + h * p.v_stride_h + d]);
}
template <class T>
LL_DEV float g_at(const ExpandArgs& a, int64_t row, int h, int d) {
  return Num<T>::to_f(static_cast<const T*>(a.g)[row * a.g_t + h * a.g_h + d]);
}

constexpr int kDk = 192, kDv = 128;

// MODE 0: forward; 1: dq; 2: dk and dv (rows are keys, the other side queries).
template <class T, int MODE>
__global__ void __launch_bounds__(256) k_expand_simple(const ExpandArgs a) {
  extern __shared__ float sm[];
  const ll_latent_packed& p = a.p;
  float* rk = sm;                        // own rows [32][192]: q, or k
  float* rv = rk + 32 * kDk;             // own rows [32][128]: g, or v
  float* ck = rv + 32 * kDv;             // other side [32][193]: k, or q
  float* cv = ck + 32 * (kDk + 1);       // other side [32][129]: v, or g
  float* cl = cv + 32 * (kDv + 1);       // lse and delta of the other side (MODE 2)
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, h = blockIdx.y;
  const int DK = p.d_n + p.d_r, DV = p.d_v;
  int b, r0;
  if (!find_tile_from_end(MODE == 2 ? p.cu_k : p.cu_q, p.B, MODE == 2 ? p.Tk : p.Tq, 32, blockIdx.x, b, r0)) return;
  int q_lo, q_hi, k_lo, k_hi;
  seq_range(p.cu_q, b, p.Tq, q_lo, q_hi);
  seq_range(p.cu_k, b, p.Tk, k_lo, k_hi);
  const int nq = q_hi - q_lo, nk = k_hi - k_lo, shift = nk - nq;
  const int n_row = MODE == 2 ? nk : nq, n_col = MODE == 2 ? nq : nk;
  const int64_t row_base = MODE == 2 ? k_lo : q_lo, col_base = MODE == 2 ? q_lo : k_lo;
  for (int i = threadIdx.x; i < 32 * DK; i += 256) {
    const int r = r0 + i / DK, d = i % DK;
    rk[(i / DK) * kDk + d] = r < n_row ? (MODE == 2 ? k_at<T>(p, row_base + r, h, d) : q_at<T>(p, row_base + r, h, d)) : 0.f;
  }
  if (MODE != 0)
    for (int i = threadIdx.x; i < 32 * DV; i += 256) {
      const int r = r0 + i / DV, d = i % DV;
      rv[(i / DV) * kDv + d] = r < n_row ? (MODE == 2 ? v_at<T>(p, row_base + r, h, d) : g_at<T>(a, row_base + r, h, d)) : 0.f;
    }
  __syncthreads();
  float m[4], l[4] = {}, x[4][6] = {}, y[4][4] = {}, rl[4], rd[4];
  for (int u = 0; u < 4; u++) {
    m[u] = -INFINITY;
    if (MODE == 1) {
      const int r = r0 + warp * 4 + u;
      float d = 0.f;
      if (r < n_row)
        for (int i = lane; i < DV; i += 32)
          d += rv[(warp * 4 + u) * kDv + i] * Num<T>::to_f(static_cast<const T*>(a.o)[((row_base + r) * p.H + h) * DV + i]);
      for (int off = 16; off; off >>= 1) d += __shfl_xor_sync(~0u, d, off);
      rd[u] = d;
      rl[u] = r < n_row ? a.lse_in[(int64_t)h * p.Tq + row_base + r] : 0.f;
    }
  }
  for (int c0 = 0; c0 < n_col; c0 += 32) {
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * DK; i += 256) {
      const int c = c0 + i / DK, d = i % DK;
      ck[(i / DK) * (kDk + 1) + d] = c < n_col ? (MODE == 2 ? q_at<T>(p, col_base + c, h, d) : k_at<T>(p, col_base + c, h, d)) : 0.f;
    }
    for (int i = threadIdx.x; i < 32 * DV; i += 256) {
      const int c = c0 + i / DV, d = i % DV;
      cv[(i / DV) * (kDv + 1) + d] = c < n_col ? (MODE == 2 ? g_at<T>(a, col_base + c, h, d) : v_at<T>(p, col_base + c, h, d)) : 0.f;
    }
    __syncthreads();
    if (MODE == 2) {
      if (threadIdx.x < 32) {
        const int c = c0 + lane;
        float d = 0.f;
        if (c < n_col)
          for (int i = 0; i < DV; i++)
            d += cv[lane * (kDv + 1) + i] * Num<T>::to_f(static_cast<const T*>(a.o)[((col_base + c) * p.H + h) * DV + i]);
        cl[lane] = c < n_col ? a.lse_in[(int64_t)h * p.Tq + col_base + c] : 0.f;
        cl[32 + lane] = d;
      }
      __syncthreads();
    }
    for (int u = 0; u < 4; u++) {
      const int r = r0 + warp * 4 + u, c = c0 + lane;
      const int qi = MODE == 2 ? c : r, ki = MODE == 2 ? r : c;
      const bool seen = qi < nq && ki < nk && (!p.causal || ki <= qi + shift);
      float s = 0.f, dp = 0.f;
      for (int d = 0; d < DK; d++) s = fmaf(rk[(warp * 4 + u) * kDk + d], ck[lane * (kDk + 1) + d], s);
      s = seen ? s * p.scale : -INFINITY;
      if (MODE == 0) {
        float mx = s;
        for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, off));
        mx = fmaxf(mx, m[u]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float pr = __expf(s - ref), f = __expf(m[u] - ref);
        float ps = pr;
        for (int off = 16; off; off >>= 1) ps += __shfl_xor_sync(~0u, ps, off);
        l[u] = l[u] * f + ps;
        m[u] = mx;
        for (int i = 0; i < 4; i++) y[u][i] *= f;
        for (int j = 0; j < 32; j++) {
          const float pj = __shfl_sync(~0u, pr, j);
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (i * 32 < DV) y[u][i] = fmaf(pj, cv[j * (kDv + 1) + i * 32 + lane], y[u][i]);
        }
      } else {
        for (int d = 0; d < DV; d++) dp = fmaf(rv[(warp * 4 + u) * kDv + d], cv[lane * (kDv + 1) + d], dp);
        const float lse = MODE == 1 ? rl[u] : cl[lane], delta = MODE == 1 ? rd[u] : cl[32 + lane];
        const float pr = seen ? __expf(s - lse) : 0.f;
        const float ds = seen ? pr * (dp - delta) * p.scale : 0.f;
        for (int j = 0; j < 32; j++) {
          const float dj = __shfl_sync(~0u, ds, j), pj = __shfl_sync(~0u, pr, j);
#pragma unroll
          for (int i = 0; i < 6; i++)
            if (i * 32 < DK) x[u][i] = fmaf(dj, ck[j * (kDk + 1) + i * 32 + lane], x[u][i]);
          if (MODE == 2)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (i * 32 < DV) y[u][i] = fmaf(pj, cv[j * (kDv + 1) + i * 32 + lane], y[u][i]);
        }
      }
    }
  }
  for (int u = 0; u < 4; u++) {
    const int r = r0 + warp * 4 + u;
    if (r >= n_row) continue;
    const int64_t row = row_base + r;
    if (MODE == 0) {
      for (int i = 0; i * 32 < DV; i++)
        static_cast<T*>(a.out)[(row * p.H + h) * DV + i * 32 + lane] = Num<T>::from_f(l[u] > 0.f ? y[u][i] / l[u] : 0.f);
      if (lane == 0) a.lse[(int64_t)h * p.Tq + row] = l[u] > 0.f ? m[u] + logf(l[u]) : -INFINITY;
    } else if (MODE == 1) {
      for (int i = 0; i * 32 < DK; i++) static_cast<T*>(a.dq)[(row * p.H + h) * DK + i * 32 + lane] = Num<T>::from_f(x[u][i]);
    } else {
      for (int i = 0; i * 32 < DV; i++) static_cast<T*>(a.dv)[(row * p.H + h) * DV + i * 32 + lane] = Num<T>::from_f(y[u][i]);
      for (int i = 0; i * 32 < DK; i++) {
        const int d = i * 32 + lane;
        if (d < p.d_n) static_cast<T*>(a.dk)[(row * p.H + h) * p.d_n + d] = Num<T>::from_f(x[u][i]);
        else a.dkpe_ws[((int64_t)h * p.Tk + row) * p.d_r + d - p.d_n] = x[u][i];
      }
    }
  }
}

// dk_pe[row][d] = sum over heads, heads in order.
template <class T>
__global__ void k_sum_heads(const float* __restrict__ ws, int H, int64_t n, T* __restrict__ out) {
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int h = 0; h < H; h++) s += ws[h * n + i];
  out[i] = Num<T>::from_f(s);
}

static int check_packed(const ll_latent_packed* p) {
  if (!p || p->B < 0 || p->Tq < 0 || p->Tk < 0 || p->H <= 0 || (p->d_n != 64 && p->d_n != 128) ||
      (p->d_v != 64 && p->d_v != 128) || (p->d_r != 0 && p->d_r != 64) || (p->dtype != 1 && p->dtype != 2))
    return LL_ERR_ARG;
  return LL_OK;
}

template <class T, int MODE>
static int launch_simple(const ExpandArgs& a, cudaStream_t s) {
  const int smem = (32 * kDk + 32 * kDv + 32 * (kDk + 1) + 32 * (kDv + 1) + 64) * 4;
  LL_TRY(set_smem_attr(reinterpret_cast<const void*>(k_expand_simple<T, MODE>), smem));
  const int tiles = (MODE == 2 ? a.p.Tk : a.p.Tq) / 32 + a.p.B;
  k_expand_simple<T, MODE><<<dim3(tiles, a.p.H), 256, smem, s>>>(a);
  return check_launch("k_expand_simple");
}

}  // namespace ll

using namespace ll;

extern "C" {

int ll_latent_forward(const ll_latent_packed* p, void* out, float* lse, void* stream) {
  LL_TRY(check_packed(p));
  if (p->B == 0 || p->Tq == 0) return LL_OK;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  ExpandArgs a{};
  a.p = *p;
  a.out = out;
  a.lse = lse;
  return p->dtype == 1 ? launch_simple<__nv_bfloat16, 0>(a, s) : launch_simple<__half, 0>(a, s);
}

size_t ll_latent_backward_workspace_bytes(const ll_latent_packed* p) {
  if (check_packed(p) != LL_OK) return 0;
  return (size_t)p->H * p->Tk * p->d_r * 4 + 256;
}

int ll_latent_backward(const ll_latent_packed* p, const void* g, int64_t g_stride_t, int64_t g_stride_h,
                       const void* out, const float* lse, void* dq, void* dk_nope, void* dk_pe, void* dv,
                       void* workspace, size_t workspace_bytes, void* stream) {
  LL_TRY(check_packed(p));
  if (p->B == 0) return LL_OK;
  if (workspace_bytes < ll_latent_backward_workspace_bytes(p)) return LL_ERR_WORKSPACE;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  ExpandArgs a{};
  a.p = *p;
  a.g = g;
  a.g_t = g_stride_t;
  a.g_h = g_stride_h;
  a.o = out;
  a.lse_in = lse;
  a.dq = dq;
  a.dk = dk_nope;
  a.dkpe = dk_pe;
  a.dv = dv;
  a.dkpe_ws = static_cast<float*>(workspace);
  const int64_t n = (int64_t)p->Tk * p->d_r;
  if (p->dtype == 1) {
    LL_TRY((launch_simple<__nv_bfloat16, 1>(a, s)));
    LL_TRY((launch_simple<__nv_bfloat16, 2>(a, s)));
    if (n) k_sum_heads<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a.dkpe_ws, p->H, n, static_cast<__nv_bfloat16*>(dk_pe));
  } else {
    LL_TRY((launch_simple<__half, 1>(a, s)));
    LL_TRY((launch_simple<__half, 2>(a, s)));
    if (n) k_sum_heads<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a.dkpe_ws, p->H, n, static_cast<__half*>(dk_pe));
  }
  return check_launch("k_sum_heads");
}

}  // extern "C"

// The paged latent cache's append and the rotary position rotation.
//
// A rotation turns each pair (a, b) of a vector's d_r rotary values by its token's angle:
//   (a', b') = (a cos - b sin, a sin + b cos),
// in fp32, rounded once to the 16-bit type; the gradient turns back (sin negated). Pairs are
// (2i, 2i + 1) or (i, i + d_r / 2). Cosines and sines come from a table row per position: computing
// them per call would cost more than reading 256 bytes that a token's heads share.
//
// Bound by bytes at prompt sizes and by launch latency at a decode step. One block takes a token;
// an item is 32 bytes in and 32 bytes out (two 16-byte accesses): 16 rotary values of one head (both
// halves of eight pairs) or 16 latent values, so a token's d_r / 16 (H + 1) + d_c / 16 items share the
// position's table row through L1. Offsets are 64-bit: a cache passes 2^32 bytes.
#include "latent_ops.cuh"

namespace ll {

__device__ DevStatus g_la_status;

DevStatus* latent_status() {
  static thread_local int dev_of = -1;
  static thread_local DevStatus* at = nullptr;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  if (dev != dev_of) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_la_status) != cudaSuccess) return nullptr;
    at = static_cast<DevStatus*>(p);
    dev_of = dev;
  }
  return at;
}

struct AppendArgs {
  const void* kv;
  const int64_t* slots;
  const int64_t* positions;
  const float* table;
  void* cache;
  const void* q;
  void* qo;
  int64_t kv_stride, page_stride, row_stride, q_t, q_h, qo_t, qo_h;
  int64_t n_slots;
  int table_rows, d_c, d_r, H, page_size, interleaved;
  float sign;        // -1 turns back
  DevStatus* st;
};

// Sixteen rotary values of one vector: pairs 8 i .. 8 i + 7.
template <class T>
LL_DEV void rotate16(const T* src, T* dst, const float* cs, int d_r, int i, bool interleaved, float sign) {
  const int h = d_r / 2;
  const int o0 = interleaved ? 16 * i : 8 * i, o1 = interleaved ? 16 * i + 8 : h + 8 * i;
  uint4 raw[2] = {*reinterpret_cast<const uint4*>(src + o0), *reinterpret_cast<const uint4*>(src + o1)};
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const float4 cv = *reinterpret_cast<const float4*>(cs + 8 * i + 4 * j);
    const float4 sv = *reinterpret_cast<const float4*>(cs + h + 8 * i + 4 * j);
    c[4 * j] = cv.x; c[4 * j + 1] = cv.y; c[4 * j + 2] = cv.z; c[4 * j + 3] = cv.w;
    s[4 * j] = sign * sv.x; s[4 * j + 1] = sign * sv.y; s[4 * j + 2] = sign * sv.z; s[4 * j + 3] = sign * sv.w;
  }
  const T* in = reinterpret_cast<const T*>(raw);
  float a[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    a[j] = Num<T>::to_f(in[interleaved ? 2 * j : j]);
    b[j] = Num<T>::to_f(in[interleaved ? 2 * j + 1 : 8 + j]);
  }
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float u = a[j] * c[j] - b[j] * s[j], v = a[j] * s[j] + b[j] * c[j];
    a[j] = u;
    b[j] = v;
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    w[j] = interleaved ? Num<T>::pack(a[j], b[j]) : Num<T>::pack(a[2 * j], a[2 * j + 1]);
    w[4 + j] = interleaved ? Num<T>::pack(a[4 + j], b[4 + j]) : Num<T>::pack(b[2 * j], b[2 * j + 1]);
  }
  *reinterpret_cast<uint4*>(dst + o0) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(dst + o1) = make_uint4(w[4], w[5], w[6], w[7]);
}

template <class T>
__global__ void __launch_bounds__(512) k_latent_append(const AppendArgs a) {
  const int64_t t = blockIdx.x;
  const int64_t pos = a.positions[t];
  const bool pos_ok = pos >= 0 && pos < a.table_rows;
  if (!pos_ok && threadIdx.x == 0) report(a.st, LL_ERR_RANGE, 71, (int)t);
  const float* cs = a.table + (pos_ok ? pos : 0) * a.d_r;
  const int per = a.d_r / 16, n_rot = per * a.H;
  T* row = nullptr;
  if (a.kv) {
    const int64_t slot = a.slots[t];
    if (slot >= a.n_slots && threadIdx.x == 0) report(a.st, LL_ERR_RANGE, 72, (int)t);
    if (slot >= 0 && slot < a.n_slots && pos_ok)
      row = static_cast<T*>(a.cache) + (slot / a.page_size) * a.page_stride + (slot % a.page_size) * a.row_stride;
  }
  const int items = n_rot + (a.kv ? per + a.d_c / 16 : 0);
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    if (i < n_rot) {
      const int h = i / per;
      if (pos_ok)
        rotate16<T>(static_cast<const T*>(a.q) + t * a.q_t + h * a.q_h, static_cast<T*>(a.qo) + t * a.qo_t + h * a.qo_h,
                    cs, a.d_r, i % per, a.interleaved != 0, a.sign);
    } else if (row) {
      const T* src = static_cast<const T*>(a.kv) + t * a.kv_stride;
      const int j = i - n_rot;
      if (j < per) {
        rotate16<T>(src + a.d_c, row + a.d_c, cs, a.d_r, j, a.interleaved != 0, a.sign);
      } else {
        const int o = (j - per) * 16;
        const uint4 x = *reinterpret_cast<const uint4*>(src + o), y = *reinterpret_cast<const uint4*>(src + o + 8);
        *reinterpret_cast<uint4*>(row + o) = x;
        *reinterpret_cast<uint4*>(row + o + 8) = y;
      }
    }
  }
}

static bool bad(const void* p, int64_t s0, int64_t s1 = 0) {
  return !p || (reinterpret_cast<uintptr_t>(p) & 15) || s0 % 8 || s1 % 8;
}

static int launch_append(const AppendArgs& a, int T, int dtype, cudaStream_t s) {
  const int items = a.d_r / 16 * a.H + (a.kv ? a.d_r / 16 + a.d_c / 16 : 0);
  const int threads = std::min(512, (items + 31) / 32 * 32);
  if (dtype == 1) k_latent_append<__nv_bfloat16><<<T, threads, 0, s>>>(a);
  else k_latent_append<__half><<<T, threads, 0, s>>>(a);
  return check_launch("k_latent_append");
}

}  // namespace ll

using namespace ll;

extern "C" {

int ll_latent_status(void* stream) {
  LL_STREAM(stream);
  DevStatus* st = latent_status();
  if (!st) return LL_ERR_CUDA;
  const int rc = read_status(st, s);
  if (rc != LL_OK) LL_TRY(reset_status(st, s));
  return rc;
}

int ll_latent_append(const void* kv, int64_t kv_stride, const int64_t* slots, const int64_t* positions,
                     const float* table, int table_rows, int T, int d_c, int d_r, int dtype, int interleaved,
                     void* cache, int64_t page_stride, int64_t row_stride, int pages, int page_size, const void* q_pe,
                     int64_t q_stride_t, int64_t q_stride_h, int H, void* q_out, int64_t qo_stride_t,
                     int64_t qo_stride_h, void* stream) {
  if (T < 0 || d_c <= 0 || d_c % 16 || d_r < 0 || d_r % 16 || (dtype != 1 && dtype != 2) || H < 0) return LL_ERR_ARG;
  if (pages <= 0 || page_size <= 0 || table_rows <= 0 || (page_size > 1 && row_stride < d_c + d_r) ||
      (pages > 1 && page_stride < d_c + d_r))
    return LL_ERR_ARG;
  if (!q_pe) H = 0;
  if (T == 0) return LL_OK;
  if (bad(kv, kv_stride) || bad(cache, page_stride, row_stride) || !slots || !positions || bad(table, 0)) return LL_ERR_ARG;
  if (H && (bad(q_pe, q_stride_t, q_stride_h) || bad(q_out, qo_stride_t, qo_stride_h))) return LL_ERR_ARG;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  AppendArgs a{kv, slots, positions, table, cache, q_pe, q_out, kv_stride, page_stride, row_stride, q_stride_t,
               q_stride_h, qo_stride_t, qo_stride_h, (int64_t)pages * page_size, table_rows, d_c, d_r, H, page_size,
               interleaved, 1.f, latent_status()};
  if (!a.st) return LL_ERR_CUDA;
  return launch_append(a, T, dtype, s);
}

int ll_latent_rotate(const void* x, int64_t x_stride_t, int64_t x_stride_h, const int64_t* positions,
                     const float* table, int table_rows, int T, int H, int d_r, int dtype, int interleaved,
                     int inverse, void* out, int64_t o_stride_t, int64_t o_stride_h, void* stream) {
  if (T < 0 || H < 0 || d_r <= 0 || d_r % 16 || (dtype != 1 && dtype != 2) || table_rows <= 0) return LL_ERR_ARG;
  if (T == 0 || H == 0) return LL_OK;
  if (bad(x, x_stride_t, x_stride_h) || bad(out, o_stride_t, o_stride_h) || !positions || bad(table, 0)) return LL_ERR_ARG;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  AppendArgs a{};
  a.positions = positions;
  a.table = table;
  a.table_rows = table_rows;
  a.q = x;
  a.q_t = x_stride_t;
  a.q_h = x_stride_h;
  a.qo = out;
  a.qo_t = o_stride_t;
  a.qo_h = o_stride_h;
  a.d_r = d_r;
  a.H = H;
  a.interleaved = interleaved;
  a.sign = inverse ? -1.f : 1.f;
  a.st = latent_status();
  if (!a.st) return LL_ERR_CUDA;
  return launch_append(a, T, dtype, s);
}

}  // extern "C"

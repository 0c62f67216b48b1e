// The paged latent cache's append and the rotary position rotation.
//
// A rotation turns each pair (a, b) of a vector's d_r rotary values by its token's angle:
//   (a', b') = (a cos - b sin, a sin + b cos),
// in fp32, rounded once to the 16-bit type; the gradient turns back (sin negated). Pairs are
// (2i, 2i + 1) or (i, i + d_r / 2). Cosines and sines come from a table row per position: computing
// them per call would cost more than reading 256 bytes that a token's heads share.
//
// Bound by bytes at prompt sizes and by launch latency at a decode step. One block takes a token; an item
// is 16 contiguous bytes in and out: 8 rotary values (pairs side by side), 8 + 8 of two halves (two such
// pieces), or 8 latent values to copy. A thread requests its first two items before the token's position
// and its table row (which the heads share through L1) have arrived: three dependent loads become two.
// Offsets are 64-bit: a cache passes 2^32 bytes.
// Measured: 9001 tokens with 64 heads (171 MB) 38 us, 4.5 TB/s, 69 % of the copy rate (four items ahead: 56 us, 320
// threads: 46 us); a decode step of 40 tokens 2.9 us. At 64 heads a token has 584 items and a block takes 512
// at a time, so the last 72 (the latent row) are requested only after the first ones' stores.
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
  int table_rows, d_c, d_r, H, page_size;
  uint32_t per_inv;  // ceil(2^32 / items of a rotary vector): i / items is the high word of i * per_inv (0: one item)
  float sign;        // -1 turns back
  DevStatus* st;
};

// An item's values: one piece of eight (IL: four pairs side by side), or the two pieces that hold the
// halves of eight pairs.
template <bool IL>
struct Piece {
  uint4 v[IL ? 1 : 2];
};

template <class T, bool IL>
LL_DEV Piece<IL> load_piece(const T* src, int d_r, int i) {
  Piece<IL> p;
  p.v[0] = *reinterpret_cast<const uint4*>(src + 8 * i);
  if constexpr (!IL) p.v[1] = *reinterpret_cast<const uint4*>(src + d_r / 2 + 8 * i);
  return p;
}

// Turns item i of a vector by the angles whose cosines, then sines, are at cs.
template <class T, bool IL>
LL_DEV void turn_piece(const Piece<IL>& p, T* dst, const float* cs, int d_r, int i, float sign) {
  constexpr int N = IL ? 4 : 8;
  const T* in = reinterpret_cast<const T*>(p.v);
  float a[N], b[N];
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 c = *reinterpret_cast<const float4*>(cs + N * i + j);
    const float4 s = *reinterpret_cast<const float4*>(cs + d_r / 2 + N * i + j);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sign * s.x, sign * s.y, sign * s.z, sign * s.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float x = Num<T>::to_f(in[IL ? 2 * (j + k) : j + k]), y = Num<T>::to_f(in[IL ? 2 * (j + k) + 1 : 8 + j + k]);
      a[j + k] = x * cc[k] - y * ss[k];
      b[j + k] = x * ss[k] + y * cc[k];
    }
  }
  if constexpr (IL) {
    *reinterpret_cast<uint4*>(dst + 8 * i) =
        make_uint4(Num<T>::pack(a[0], b[0]), Num<T>::pack(a[1], b[1]), Num<T>::pack(a[2], b[2]), Num<T>::pack(a[3], b[3]));
  } else {
    *reinterpret_cast<uint4*>(dst + 8 * i) =
        make_uint4(Num<T>::pack(a[0], a[1]), Num<T>::pack(a[2], a[3]), Num<T>::pack(a[4], a[5]), Num<T>::pack(a[6], a[7]));
    *reinterpret_cast<uint4*>(dst + d_r / 2 + 8 * i) =
        make_uint4(Num<T>::pack(b[0], b[1]), Num<T>::pack(b[2], b[3]), Num<T>::pack(b[4], b[5]), Num<T>::pack(b[6], b[7]));
  }
}

constexpr int kAppendThreads = 256, kAppendBatch = 2;

template <class T, bool IL>
__global__ void __launch_bounds__(kAppendThreads) k_latent_append(const AppendArgs a) {
  const int64_t t = blockIdx.x;
  const int per = a.d_r / (IL ? 8 : 16), n_rot = per * a.H, n_new = n_rot + (a.kv ? per : 0);
  const int items = n_new + (a.kv ? a.d_c / 8 : 0);
  const T* q = static_cast<const T*>(a.q) + t * a.q_t;
  const T* kv = static_cast<const T*>(a.kv) + t * a.kv_stride;
  T* qo = static_cast<T*>(a.qo) + t * a.qo_t;
  int64_t pos = 0;
  const float* cs = nullptr;
  T* row = nullptr;
  bool known = false;
  for (int i0 = threadIdx.x; i0 < items; i0 += kAppendThreads * kAppendBatch) {
    Piece<IL> p[kAppendBatch];
#pragma unroll
    for (int u = 0; u < kAppendBatch; u++) {
      const int i = i0 + u * kAppendThreads;
      const int h = a.per_inv ? __umulhi(i, a.per_inv) : i;
      if (i < n_rot) p[u] = load_piece<T, IL>(q + h * a.q_h, a.d_r, i - h * per);
      else if (i < n_new) p[u] = load_piece<T, IL>(kv + a.d_c, a.d_r, i - n_rot);
      else if (i < items) p[u].v[0] = *reinterpret_cast<const uint4*>(kv + 8 * (i - n_new));
    }
    if (!known) {
      known = true;
      pos = a.positions[t];
      const int64_t slot = a.kv ? a.slots[t] : -1;
      const bool pos_ok = pos >= 0 && pos < a.table_rows;
      if (threadIdx.x == 0) {
        if (!pos_ok) report(a.st, LL_ERR_RANGE, 71, (int)t);
        if (slot >= a.n_slots) report(a.st, LL_ERR_RANGE, 72, (int)t);
      }
      if (!pos_ok) return;
      cs = a.table + pos * a.d_r;
      if (slot >= 0 && slot < a.n_slots)
        row = static_cast<T*>(a.cache) + (slot / a.page_size) * a.page_stride + (slot % a.page_size) * a.row_stride;
    }
#pragma unroll
    for (int u = 0; u < kAppendBatch; u++) {
      const int i = i0 + u * kAppendThreads;
      if (i < n_rot) {
        const int h = a.per_inv ? __umulhi(i, a.per_inv) : i;
        turn_piece<T, IL>(p[u], qo + h * a.qo_h, cs, a.d_r, i - h * per, a.sign);
      } else if (row) {
        if (i < n_new) turn_piece<T, IL>(p[u], row + a.d_c, cs, a.d_r, i - n_rot, a.sign);
        else if (i < items) *reinterpret_cast<uint4*>(row + 8 * (i - n_new)) = p[u].v[0];
      }
    }
  }
}

static bool bad(const void* p, int64_t s0, int64_t s1 = 0) {
  return !p || (reinterpret_cast<uintptr_t>(p) & 15) || s0 % 8 || s1 % 8;
}

static int launch_append(AppendArgs& a, int T, int dtype, int interleaved, cudaStream_t s) {
  if (a.d_r) a.per_inv = (uint32_t)((0xffffffffull + a.d_r / (interleaved ? 8 : 16)) / (a.d_r / (interleaved ? 8 : 16)));
  auto* fn = dtype == 1 ? (interleaved ? k_latent_append<__nv_bfloat16, true> : k_latent_append<__nv_bfloat16, false>)
                        : (interleaved ? k_latent_append<__half, true> : k_latent_append<__half, false>);
  fn<<<T, kAppendThreads, 0, s>>>(a);
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
               0, 1.f, latent_status()};
  if (!a.st) return LL_ERR_CUDA;
  return launch_append(a, T, dtype, interleaved, s);
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
  a.sign = inverse ? -1.f : 1.f;
  a.st = latent_status();
  if (!a.st) return LL_ERR_CUDA;
  return launch_append(a, T, dtype, interleaved, s);
}

}  // extern "C"

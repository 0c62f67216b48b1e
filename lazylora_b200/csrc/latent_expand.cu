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

// ------------------------------------------------------------------------------- forward
// One CTA takes 256 query rows of one sequence and head as two tiles of 128 that alternate: while one
// tile's softmax runs, the tensor cores do the other's products.
//   S_t [128][128 keys] = Q_t K^T       (M = 128, N = 128, K = d_n + d_r)
//   O_t [128][d_v]     += P_t V         (P_t from tensor memory, 64 columns of O an instruction)
// Issue order per key tile i: S_0(i), O_1(i - 1), S_1(i), O_0(i). Per 256 x 128 scores at 192 / 128 that
// is 2560 cycles of products against 2048 of exponentials (16 a cycle): the tensor cores bound it.
// Tensor memory: S_0 | S_1 | O_0 | O_1, 128 columns each; P_t overwrites the first half of S_t.
//
// Shared memory holds Q (96 KB at 192) and a ring of eight 16 KB chunks (128 rows x 64 columns): a key
// tile takes three, a value tile two, in the order they are used and released.
//
// Softmax: a thread owns a row. As the row's reference only has to be within 2^8 of its running maximum,
// O_t is rescaled only when some row of the warp passes that. P is rounded to the 16-bit type (the tensor
// cores' operand, the output's own precision); sums in fp32 of the unrounded values.
constexpr int kExThreads = 384;        // warps 0-3, 4-7: softmax of tile 0, 1; 8: TMA; 9: MMA; 10, 11: none
// Registers: launched with 168 a thread (64,512 a block); the third warpgroup gives 96 of its up, the two
// softmax warpgroups take 48 each: 216 * 256 + 72 * 128 = 64,512.
constexpr int kExRegsMore = 216, kExRegsLess = 72;
constexpr int kExRing = 8;
constexpr int kExChunk = 128 * 128;    // bytes
constexpr int kExOps = 16;             // barriers of the ring's operands
constexpr float kExSlack = 8.f;

struct ExTma {
  CUtensorMap q, kn, kp, v, g;
};

struct ExFwdArgs {
  const int32_t *cu_q, *cu_k;
  void* out;
  float* lse;
  int B, Tq, Tk, H, nn, nr, nv, causal;    // 64-column chunks of d_n, d_r, d_v
  float scale_log2;
  DevStatus* st;
};

// The ring's bookkeeping, in step on the TMA and the MMA side: operands take consecutive slots.
struct ExRing {
  uint32_t e = 0;      // operands so far
  int slot = 0;        // the next slot
  LL_DEV int take(int chunks) {
    const int s = slot;
    slot = (slot + chunks) % kExRing;
    e++;
    return s;
  }
};

LL_DEV void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// After tcgen05.wait::ld: no use of r is scheduled before this point.
LL_DEV void ld32_ready(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                 "+r"(r[i + 6]), "+r"(r[i + 7])::"memory");
}
LL_DEV void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Sets rows from .. 127 of `chunks` ring chunks, the first in slot `slot`, to zero (threads t of n).
LL_DEV void zero_rows(uint8_t* ring, int slot, int chunks, int from, int t, int n) {
  for (int i = t; i < (128 - from) * chunks * 8; i += n) {
    const int c = i / ((128 - from) * 8), j = i % ((128 - from) * 8);
    *reinterpret_cast<uint4*>(ring + ((slot + c) % kExRing) * kExChunk + from * 128 + j * 16) = make_uint4(0, 0, 0, 0);
  }
}

// Key tiles of 128 that the query tile of `rows` rows from `q0` on sees.
LL_DEV int key_tiles(int q0, int rows, int nq, int nk, bool causal) {
  if (q0 >= nq) return 0;
  const int last = min(q0 + rows, nq) - 1;                     // the tile's last query sees the most
  const int see = causal ? min(nk, last + nk - nq + 1) : nk;
  return see > 0 ? (see + 127) / 128 : 0;
}

template <class T>
__global__ void __launch_bounds__(kExThreads, 1) k_ex_fwd(const __grid_constant__ ExTma tm, const ExFwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nqk = a.nn + a.nr;
  uint8_t* s_q = base;                                   // [tile][chunk]
  uint8_t* ring = s_q + 2 * nqk * kExChunk;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + kExRing * kExChunk);
  uint64_t *full = bars, *rel = full + kExOps, *q_full = rel + kExOps, *s_full = q_full + 2, *p_ready = s_full + 2,
           *pv_done = p_ready + 2, *drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, head = blockIdx.y;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kExOps + 4; i++) mbar_init(&bars[i], 1);
    mbar_init(&p_ready[0], 4);
    mbar_init(&p_ready[1], 4);
    mbar_init(&pv_done[0], 1);
    mbar_init(&pv_done[1], 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm.q);
    tma_prefetch_desc(&tm.kn);
    tma_prefetch_desc(&tm.kp);
    tma_prefetch_desc(&tm.v);
  }
  __syncwarp();
  pdl_wait();
  int b, q0, q_lo, q_hi, k_lo, k_hi;
  const bool any = find_tile_from_end(a.cu_q, a.B, a.Tq, 256, blockIdx.x, b, q0);
  if (any) {
    seq_range(a.cu_q, b, a.Tq, q_lo, q_hi);
    seq_range(a.cu_k, b, a.Tk, k_lo, k_hi);
  } else {
    q_lo = q_hi = k_lo = k_hi = q0 = 0;
  }
  const int nq = q_hi - q_lo, nk = k_hi - k_lo;
  const int n0 = key_tiles(q0, 128, nq, nk, a.causal), n1 = key_tiles(q0 + 128, 128, nq, nk, a.causal), n = max(n0, n1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_next();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kExRegsLess));
   if (warp == 8) {
    // ------------------------------------------------------------------------------- TMA
    if (lane == 0 && n > 0) {
      ExRing rg;
      bool ok = true;
      int owner[kExRing];                      // operand that last took a slot
#pragma unroll
      for (int i = 0; i < kExRing; i++) owner[i] = -1;
      auto load = [&](bool key, int row) {
        const int chunks = key ? nqk : a.nv, e = rg.e;
        int need = -1;
#pragma unroll
        for (int i = 0; i < kExRing; i++)
          if ((i - rg.slot + kExRing) % kExRing < chunks) {
            need = max(need, owner[i]);
            owner[i] = e;
          }
        if (need >= 0 && !mbar_wait(&rel[need % kExOps], (need / kExOps) & 1, abort_flag, a.st, 101)) return false;
        const int s = rg.take(chunks);
        uint64_t* bar = &full[e % kExOps];
        mbar_arrive_expect_tx(bar, chunks * kExChunk);
        for (int c = 0; c < chunks; c++) {
          uint8_t* dst = ring + ((s + c) % kExRing) * kExChunk;
          if (!key) tma_load_3d(dst, &tm.v, bar, c * 64, head, row);
          else if (c < a.nn) tma_load_3d(dst, &tm.kn, bar, c * 64, head, row);
          else tma_load_2d(dst, &tm.kp, bar, (c - a.nn) * 64, row);
        }
        return true;
      };
      for (int t = 0; t < 2; t++) {
        if ((t ? n1 : n0) > 0) {
          mbar_arrive_expect_tx(&q_full[t], nqk * kExChunk);
          for (int c = 0; c < nqk; c++)
            tma_load_3d(s_q + (t * nqk + c) * kExChunk, &tm.q, &q_full[t], c * 64, head, q_lo + q0 + t * 128);
        }
        if (t == 0) ok = load(true, k_lo);
      }
      if (ok) ok = load(false, k_lo);
      for (int i = 1; i < n && ok; i++) ok = load(true, k_lo + i * 128) && load(false, k_lo + i * 128);
      volatile int keep = 0;                   // everything issued has landed, also after an abort
      for (uint32_t e = rg.e > kExRing ? rg.e - kExRing : 0; e < rg.e; e++)
        mbar_wait_sleep(&full[e % kExOps], (e / kExOps) & 1, &keep, a.st, 102, 64);
      if (n0 > 0) mbar_wait_sleep(&q_full[0], 0, &keep, a.st, 103, 64);
      if (n1 > 0) mbar_wait_sleep(&q_full[1], 0, &keep, a.st, 104, 64);
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------- MMA
    const bool lead = elect_one();
    const uint32_t id_s = idesc_16bit(Num<T>::fmt, 128, 128, false, false);
    const uint32_t id_o = idesc_16bit(Num<T>::fmt, 128, 64, false, true);
    const MmaDesc q_d(smem_u32(s_q), 16, 1024), k_d(smem_u32(ring), 16, 1024), v_d(smem_u32(ring), 1024, 1024);
    bool ok = true;
    ExRing rg;                                 // operands alternate: key tile i is 2 i, value tile 2 i + 1
    int k_slot = 0, v_slot = 0;
#pragma unroll 1
    for (int step = 0; step < 2 * n + 1 && ok; step++) {
      const int t = step & 1, i = step >> 1;
      if (i < n) {
        if (t == 0) {
          if (!(ok = mbar_wait(&full[rg.e % kExOps], (rg.e / kExOps) & 1, abort_flag, a.st, 105))) break;
          k_slot = rg.take(nqk);
        }
        if (i < (t ? n1 : n0)) {
          if (i == 0 && !(ok = mbar_wait(&q_full[t], 0, abort_flag, a.st, 106))) break;
          tc_fence_after();
          if (lead) {
#pragma unroll 1
            for (int c = 0; c < nqk; c++) {
              const uint32_t q_lo16 = q_d.lo + (t * nqk + c) * (kExChunk / 16);
              const uint32_t k_lo16 = k_d.lo + ((k_slot + c) % kExRing) * (kExChunk / 16);
#pragma unroll
              for (int kk = 0; kk < 4; kk++)
                mma_16bit(tmem + t * 128, q_lo16 + kk * 2, q_d.hi, k_lo16 + kk * 2, k_d.hi, id_s, c + kk);
            }
            mma_commit(&s_full[t]);
          }
        }
        if (t == 1) {
          // the key tile is done with; the value tile comes next in the ring
          if (lead) mma_commit(&rel[(rg.e - 1) % kExOps]);
          if (!(ok = mbar_wait(&full[rg.e % kExOps], (rg.e / kExOps) & 1, abort_flag, a.st, 107))) break;
          v_slot = rg.take(a.nv);
        }
      }
      const int u = 1 - t, j = i - u;          // the other tile's outputs: O_1(i - 1), O_0(i)
      if (j < 0) continue;
      if (j < (u ? n1 : n0)) {
        if (!(ok = mbar_wait(&p_ready[u], j & 1, abort_flag, a.st, 108))) break;
        tc_fence_after();
        if (lead) {
#pragma unroll 1
          for (int c = 0; c < a.nv; c++) {
            const uint32_t v_lo16 = v_d.lo + ((v_slot + c) % kExRing) * (kExChunk / 16);
#pragma unroll
            for (int kk = 0; kk < 8; kk++)
              mma_16bit_ts(tmem + 256 + u * 128 + c * 64, tmem + u * 128 + kk * 8, v_lo16 + kk * 128, v_d.hi, id_o, j + kk);
          }
          mma_commit(&pv_done[u]);
        }
      }
      if (u == 1 && lead) mma_commit(&rel[(2 * j + 1) % kExOps]);
    }
    if (lead) mma_commit(drain);
    volatile int keep = 0;
    mbar_wait_sleep(drain, 0, &keep, a.st, 109, 64);
    __syncwarp();
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kExRegsMore));
    // --------------------------------------------------------------------------- softmax
    const int t = warp / 4, tiles = t ? n1 : n0;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16, s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
    const int row = q0 + t * 128 + (warp % 4) * 32 + lane;        // of the sequence
    const int see = a.causal ? min(nk, row + nk - nq + 1) : nk;   // keys the row sees
    const int see_all = a.causal ? min(nk, q0 + t * 128 + nk - nq + 1) : nk;   // and the tile's first row
    float ref = -1e30f, l = 0.f;
    bool ok = true;
    ExRing rv;
    for (int i = 0; i < tiles; i++) {
      rv.slot = (rv.slot + nqk) % kExRing;
      const int v_slot = rv.take(a.nv);
      if (!(ok = mbar_wait(&s_full[t], i & 1, abort_flag, a.st, 110))) break;
      tc_fence_after();
      uint32_t x[128];
#pragma unroll
      for (int c = 0; c < 128; c += 32) ld32(s_at + c, x + c);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 128; c += 32) ld32_ready(x + c);
      if (i * 128 + 128 > see_all) {
        const int lim = see - i * 128;
#pragma unroll
        for (int c = 0; c < 128; c++)
          if (c >= lim) x[c] = 0xff800000u;    // minus infinity
      }
      float m[4];
#pragma unroll
      for (int c = 0; c < 4; c++) m[c] = __uint_as_float(x[c]);
#pragma unroll
      for (int c = 4; c < 128; c++) m[c % 4] = fmaxf(m[c % 4], __uint_as_float(x[c]));
      const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * a.scale_log2;
      if (__any_sync(0xffffffffu, top > ref + kExSlack)) {
        const float now = fmaxf(ref, top), f = ex2(ref - now);
        ref = now;
        l *= f;
        if (i > 0) {
          if (!(ok = mbar_wait(&pv_done[t], (i - 1) & 1, abort_flag, a.st, 111))) break;
          tc_fence_after();
          for (int c = 0; c < a.nv * 64; c += 32) {
            uint32_t o[32];
            ld32(o_at + c, o);
            tmem_ld_wait();
            ld32_ready(o);
#pragma unroll
            for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            st32(o_at + c, o);
          }
        }
      }
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 64) {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float u = ex2(fmaf(__uint_as_float(x[c0 + c]), a.scale_log2, -ref));
          const float v = ex2(fmaf(__uint_as_float(x[c0 + c + 1]), a.scale_log2, -ref));
          s[c % 4] += u;
          s[c % 4 + 1] += v;
          w[c / 2] = Num<T>::pack(u, v);
        }
        st32(s_at + c0 / 2, w);
      }
      l += (s[0] + s[1]) + (s[2] + s[3]);
      if (i * 128 + 128 > nk) {
        // the value rows past the sequence's end, which may hold anything, must not meet P's zeros
        const uint32_t e = 2 * i + 1;
        if (!(ok = mbar_wait(&full[e % kExOps], (e / kExOps) & 1, abort_flag, a.st, 112))) break;
        zero_rows(ring, v_slot, a.nv, nk - i * 128, threadIdx.x % 128, 128);
        fence_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
    }
    if (ok && tiles > 0) ok = mbar_wait(&pv_done[t], (tiles - 1) & 1, abort_flag, a.st, 113);
    tc_fence_after();
    const bool live = !(l <= 0.f);
    const float inv = live ? 1.f / l : 0.f;
    T* dst = static_cast<T*>(a.out) + ((int64_t)(q_lo + row) * a.H + head) * (a.nv * 64);
    for (int c = 0; c < a.nv * 64; c += 32) {
      uint32_t o[32];
      if (tiles > 0) {
        ld32(o_at + c, o);
        tmem_ld_wait();
        ld32_ready(o);
      } else {
#pragma unroll
        for (int k = 0; k < 32; k++) o[k] = 0;
      }
      if (row < nq) {
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          uint32_t w[4];
#pragma unroll
          for (int z = 0; z < 4; z++)
            w[z] = Num<T>::pack(live ? __uint_as_float(o[k + 2 * z]) * inv : 0.f, live ? __uint_as_float(o[k + 2 * z + 1]) * inv : 0.f);
          *reinterpret_cast<uint4*>(dst + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (row < nq) a.lse[(int64_t)head * a.Tq + q_lo + row] = live ? (ref + log2f(l)) * 0.693147180559945309f : -INFINITY;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
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

// A 16-byte aligned pointer with positive strides that are multiples of 16 bytes, as the tensor maps take.
static bool bad16(const void* p, int64_t s0, int64_t s1) {
  return !p || (reinterpret_cast<uintptr_t>(p) & 15) || s0 <= 0 || s1 <= 0 || s0 % 8 || s1 % 8;
}

// [tokens][heads][columns] in boxes of 128 tokens x 64 columns of one head.
static int rows_map(CUtensorMap* m, CUtensorMapDataType dt, const void* base, int T, int64_t st, int H, int64_t sh,
                    int cols, uint32_t rows = 128) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)H, (uint64_t)T}, strides[2] = {(uint64_t)sh * 2, (uint64_t)st * 2};
  const uint32_t box[3] = {64, 1, rows};
  return make_map_nd(m, dt, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

static int packed_maps(ExTma* tm, const ll_latent_packed* p, uint32_t q_rows = 128, uint32_t k_rows = 128) {
  const CUtensorMapDataType dt = p->dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int dq = p->d_n + p->d_r;
  // an operand without rows is never loaded; its map is any valid one
  if (p->Tq) LL_TRY(rows_map(&tm->q, dt, p->q, p->Tq, p->q_stride_t, p->H, p->q_stride_h, dq, q_rows));
  if (p->Tk) {
    LL_TRY(rows_map(&tm->kn, dt, p->k_nope, p->Tk, p->k_stride_t, p->H, p->k_stride_h, p->d_n, k_rows));
    LL_TRY(rows_map(&tm->v, dt, p->v, p->Tk, p->v_stride_t, p->H, p->v_stride_h, p->d_v, k_rows));
    if (p->d_r)
      LL_TRY(make_map_2d(&tm->kp, dt, p->k_pe, 64, (uint64_t)p->Tk, (uint64_t)p->kpe_stride_t * 2, 64, k_rows,
                         CU_TENSOR_MAP_SWIZZLE_128B));
    else tm->kp = tm->kn;
  }
  if (!p->Tq) tm->q = tm->kn;
  if (!p->Tk) tm->kn = tm->kp = tm->v = tm->q;
  tm->g = tm->q;
  return LL_OK;
}

static int check_packed(const ll_latent_packed* p) {
  if (!p || p->B < 0 || p->Tq < 0 || p->Tk < 0 || p->H <= 0 || (p->d_n != 64 && p->d_n != 128) ||
      (p->d_v != 64 && p->d_v != 128) || (p->d_r != 0 && p->d_r != 64) || (p->dtype != 1 && p->dtype != 2) ||
      !(p->scale > 0.f))
    return LL_ERR_ARG;
  if (p->B == 0 || (p->Tq == 0 && p->Tk == 0)) return LL_OK;
  if (!p->cu_q || !p->cu_k || (int64_t)(p->Tq / 128 + p->B) * p->H > INT32_MAX || (int64_t)(p->Tk / 128 + p->B) * p->H > INT32_MAX)
    return LL_ERR_ARG;
  if (p->Tq && bad16(p->q, p->q_stride_t, p->q_stride_h)) return LL_ERR_ARG;
  if (p->Tk && (bad16(p->k_nope, p->k_stride_t, p->k_stride_h) || bad16(p->v, p->v_stride_t, p->v_stride_h) ||
                (p->d_r && bad16(p->k_pe, p->kpe_stride_t, 8))))
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
  if (!out || !lse || (reinterpret_cast<uintptr_t>(out) & 15)) return LL_ERR_ARG;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  ExTma tm;
  LL_TRY(packed_maps(&tm, p));
  ExFwdArgs a{p->cu_q, p->cu_k, out, lse, p->B, p->Tq, p->Tk, p->H, p->d_n / 64, p->d_r / 64, p->d_v / 64, p->causal,
              p->scale * 1.4426950408889634f, latent_status()};
  if (!a.st) return LL_ERR_CUDA;
  const int smem = 1024 + (2 * (a.nn + a.nr) + kExRing) * kExChunk + (2 * kExOps + 9) * 8 + 16;
  auto run = [&](auto kern) {
    LL_TRY(set_smem_attr(reinterpret_cast<const void*>(kern), smem));
    return launch_pdl("k_ex_fwd", kern, dim3(p->Tq / 256 + p->B, p->H), dim3(kExThreads), smem, s, tm, a);
  };
  return p->dtype == 1 ? run(k_ex_fwd<__nv_bfloat16>) : run(k_ex_fwd<__half>);
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

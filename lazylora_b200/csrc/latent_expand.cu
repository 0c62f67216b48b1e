// The expanded form of latent attention on packed sequences, forward and backward (see the header
// for the interface). Per head, with k = (k_nope | k_pe):
//   s_ij = scale q_i . k_j (visible j),  p = softmax(s),  o_i = sum_j p_ij v_j,
//   dv_j = sum_i p_ij g_i,  dp_ij = g_i . v_j,  ds_ij = p_ij (dp_ij - g_i . o_i) scale,
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i;  dk_pe sums dk's rotary part over the heads.
// Tiles are dealt from the cumulative lengths on the device; nothing is read back. Lengths that do not cover the
// rows are cut to them, and recorded by a warp without other work in the last block (the lightest tile, or none).
#include "latent_ops.cuh"

namespace ll {

// ------------------------------------------------------------------------------- forward
// One CTA takes 256 query rows of one sequence and head as two tiles of 128 that alternate: while one
// tile's softmax runs, the tensor cores do the other's products. Measured: 8000 tokens at 32 heads (655
// GFLOP) 565 us, 1.16 PFLOP/s; in a loop that holds the power limit (1000 W, 1.7 GHz) 647 us, 70 % of
// what a large cuBLAS product sustains there.
//   S_t [128][128 keys] = Q_t K^T       (M = 128, N = 128, K = d_n + d_r)
//   O_t [128][d_v]     += P_t V         (P_t from tensor memory)
// Issue order per key tile i: O_0(i - 1), S_0(i), O_1(i - 1), S_1(i). Per 256 x 128 scores at 192 / 128 that
// is 2560 cycles of products against 2048 of exponentials (16 a cycle). Neither is full: at 8000 tokens and 32
// heads a step takes 4200 cycles at 1.7 GHz (the power limit), the tensor pipe is active in 58 % of them, the
// exponentials' pipe in 47 %, and 29 % of the issue slots are taken. What is left is a tile's own chain: from its
// scores to its P (4200 less its products' 1280 cycles) only the other tile's products (1280) run beside it.
// Tensor memory: S_0 | S_1 | O_0 | O_1, 128 columns each; P_t overwrites the first half of S_t.
//
// Shared memory holds Q (96 KB at 192) and a ring of eight 16 KB chunks (128 rows x 64 columns): a key
// tile takes three, a value tile two, in the order they are used and released.
//
// Softmax: a thread owns a row. As the row's reference only has to be within 2^8 of its running maximum,
// O_t is rescaled only when some row of the warp passes that. P is rounded to the 16-bit type (the tensor
// cores' operand, the output's own precision); sums in fp32 of the unrounded values.
constexpr int kExThreads = 384;        // warps 0-3, 4-7: softmax of tile 0, 1; 8: TMA; 9: MMA; 10: checks; 11: none
// Registers: launched with 168 a thread (64,512 a block); the third warpgroup gives some of its up to the two
// softmax warpgroups: 224 * 256 + 56 * 128 = 176 * 256 + 152 * 128 = 64,512. (The backward's loading and issuing
// warps spill below 152, 4 % of a packed step; its element-wise warps need no more than 176.)
constexpr int kExRegsMore = 224, kExRegsLess = 56, kExBwdMore = 176, kExBwdLess = 152;
constexpr int kExRing = 8;
constexpr int kExChunk = 128 * 128;    // bytes
constexpr int kExOps = 16;             // barriers of the ring's operands
constexpr float kExSlack = 8.f;
// A wait that runs out records itself and raises the block's abort flag, after which every wait returns at
// once. The loading warps then stop (all lanes together), the issuing warps too; the element-wise warps go
// through their loops without leaving them, so that no warp-wide instruction loses lanes; the results are
// void, as the status says.

// The order in which blocks take (tile, head): heads in groups, in a group the longest tiles of its heads
// first, so that the launch ends on a group's short tiles; the groups (about four tiles per SM) keep the keys
// and values in use few enough for L2. A head after the other, the last heads' long tiles ended 12 % after
// the average SM (8000 tokens, 32 heads: 609 us; groups of 2, 4, 8 tiles an SM: 636, 555, 565).
struct ExOrder {
  int tiles, heads, group;
};
LL_DEV void ex_deal(const ExOrder& o, int& tile, int& head) {
  const int per = o.group * o.tiles, g = blockIdx.x / per, r = blockIdx.x % per, n = min(o.group, o.heads - g * o.group);
  tile = r / n;
  head = g * o.group + r % n;
}

struct ExTma {
  CUtensorMap q, kn, kp, v, g;
};

struct ExFwdArgs {
  const int32_t *cu_q, *cu_k;
  void* out;
  float* lse;
  int B, Tq, Tk, H, nn, nr, nv, causal;    // 64-column chunks of d_n, d_r, d_v
  ExOrder order;
  float scale_log2;
  DevStatus* st;
};

// The ring's bookkeeping, in step wherever it is kept: operands take consecutive slots; a value tile, whose
// chunks one instruction reads at a fixed distance, does not go around the end (the last slot is skipped).
struct ExRing {
  uint32_t e = 0;      // operands so far
  int slot = 0;        // the next slot
  LL_DEV int take(int chunks, bool values) {
    const int s = values && slot + chunks > kExRing ? 0 : slot;
    slot = (s + chunks) % kExRing;
    e++;
    return s;
  }
};

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

// 64 columns of an accumulator (zeros where nothing was summed), times f, as 32 words of the 16-bit type.
template <class T>
LL_DEV void load_acc64(uint32_t at, bool any, float f, uint32_t* w) {
  if (any) {
    uint32_t o[64];
    ld32(at, o);
    ld32(at + 32, o + 32);
    tmem_ld_wait();
    ld32_ready(o);
    ld32_ready(o + 32);
#pragma unroll
    for (int k = 0; k < 32; k++) w[k] = Num<T>::pack(__uint_as_float(o[2 * k]) * f, __uint_as_float(o[2 * k + 1]) * f);
  } else {
#pragma unroll
    for (int k = 0; k < 32; k++) w[k] = 0;
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
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int tile, head;
  ex_deal(a.order, tile, head);

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
  const bool any = find_tile<true>(a.cu_q, a.B, a.Tq, 256, tile, b, q0);
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
      // Lane c brings chunk c: boxes that one thread issues follow each other about 350 cycles apart.
      if (n > 0) {
        ExRing rg;
        bool ok = true;
        int owner = -1;                          // lane s: the operand that last took slot s
        auto load = [&](bool key, int row) {
          const int chunks = key ? nqk : a.nv, e = rg.e, s0 = rg.take(chunks, !key);
          const bool mine = lane < kExRing && (lane - s0 + kExRing) % kExRing < chunks;
          const int need = __reduce_max_sync(0xffffffffu, mine ? owner : -1);
          if (mine) owner = e;
          if (need >= 0 && !warp_wait_sleep(&rel[need % kExOps], (need / kExOps) & 1, abort_flag, a.st, 101, 64)) {
            rg.e--;
            return false;
          }
          uint64_t* bar = &full[e % kExOps];
          if (lane == 0) mbar_arrive_expect_tx(bar, chunks * kExChunk);
          __syncwarp();
          uint8_t* dst = ring + ((s0 + lane) % kExRing) * kExChunk;
          if (key && lane < a.nn) tma_load_3d(dst, &tm.kn, bar, lane * 64, head, row);
          else if (key && lane < nqk) tma_load_2d(dst, &tm.kp, bar, (lane - a.nn) * 64, row);
          else if (!key && lane < a.nv) tma_load_3d(dst, &tm.v, bar, lane * 64, head, row);
          __syncwarp();
          return true;
        };
        for (int t = 0; t < 2; t++) {
          if ((t ? n1 : n0) > 0) {
            if (lane == 0) mbar_arrive_expect_tx(&q_full[t], nqk * kExChunk);
            __syncwarp();
            if (lane < nqk)
              tma_load_3d(s_q + (t * nqk + lane) * kExChunk, &tm.q, &q_full[t], lane * 64, head, q_lo + q0 + t * 128);
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
      const uint32_t id_o = idesc_16bit(Num<T>::fmt, 128, a.nv * 64, false, true);
      const MmaDesc q_d(smem_u32(s_q), 16, 1024), k_d(smem_u32(ring), 16, 1024), v_d(smem_u32(ring), kExChunk, 1024);
      bool ok = true;
      ExRing rg;                                 // operands alternate: key tile i is 2 i, value tile 2 i + 1
      int k_slot = 0, v_slot = 0;
      auto operand = [&]() { return mbar_wait(&full[rg.e % kExOps], (rg.e / kExOps) & 1, abort_flag, a.st, 105); };
      // O_t(i) and S_t(i + 1) in one go, so that nothing is waited for in between
#pragma unroll 1
      for (int step = 0; step < 2 * n + 2 && ok; step++) {
        const int t = step & 1, i = (step >> 1) - 1, tiles = t ? n1 : n0;
        if (t == 0) {
          // value tile i, key tile i + 1
          if (i >= 0) {
            if (!(ok = operand())) break;
            v_slot = rg.take(a.nv, true);
          }
          if (i + 1 < n) {
            if (!(ok = operand())) break;
            k_slot = rg.take(nqk, false);
          }
        }
        if (i < 0 && tiles > 0 && !(ok = mbar_wait(&q_full[t], 0, abort_flag, a.st, 106))) break;
        if (i >= 0 && i < tiles) {
          if (!(ok = mbar_wait(&p_ready[t], i & 1, abort_flag, a.st, 107))) break;
        }
        tc_fence_after();
        if (!lead) continue;
        if (i >= 0 && i < tiles) {
          const uint32_t v_lo16 = v_d.lo + v_slot * (kExChunk / 16);
#pragma unroll
          for (int kk = 0; kk < 8; kk++)
            mma_16bit_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, v_lo16 + kk * 128, v_d.hi, id_o, i + kk);
          if (i + 1 == tiles) mma_commit(&pv_done[t]);
        }
        if (i >= 0 && t == 1) mma_commit(&rel[(2 * i + 1) % kExOps]);
        if (i + 1 < tiles) {
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
      __syncwarp();
      if (lead) mma_commit(drain);
      volatile int keep = 0;
      mbar_wait_sleep(drain, 0, &keep, a.st, 109, 64);
      __syncwarp();
    } else if (warp == 10 && blockIdx.x == gridDim.x - 1) {
      check_cu(a.cu_q, a.B, a.Tq, a.st, 75);
      check_cu(a.cu_k, a.B, a.Tk, a.st, 76);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kExRegsMore));
    // --------------------------------------------------------------------------- softmax
    const int t = warp / 4, tiles = t ? n1 : n0;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + 256 + t * 128 + lanes;
    const int row = q0 + t * 128 + (warp % 4) * 32 + lane;        // of the sequence
    const int see = a.causal ? min(nk, row + nk - nq + 1) : nk;   // keys the row sees
    const int see_all = a.causal ? min(nk, q0 + t * 128 + nk - nq + 1) : nk;   // and the tile's first row
    float ref = -1e30f, l = 0.f;
    ExRing rv;
    for (int i = 0; i < tiles; i++) {
      rv.take(nqk, false);
      const int v_slot = rv.take(a.nv, true);
      mbar_wait(&s_full[t], i & 1, abort_flag, a.st, 110);
      tc_fence_after();
      // the last tile's scores over a key tile release it
      if (threadIdx.x % 128 == 0 && (t == 1 || i >= n1)) mbar_arrive(&rel[(2 * i) % kExOps]);
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
          // (S_t(i) has arrived, and O_t(i - 1) was issued before it: its sums are complete)
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
      if (i * 128 + 128 > nk) {
        // the value rows past the sequence's end, which may hold anything, must not meet P's zeros
        const uint32_t e = 2 * i + 1;
        mbar_wait(&full[e % kExOps], (e / kExOps) & 1, abort_flag, a.st, 112);
        zero_rows(ring, v_slot, a.nv, nk - i * 128, threadIdx.x % 128, 128);
        fence_async_smem();
      }
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 64) {
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          float2 u = fma2(make_float2(__uint_as_float(x[c0 + c]), __uint_as_float(x[c0 + c + 1])),
                          make_float2(a.scale_log2, a.scale_log2), make_float2(-ref, -ref));
          u.x = ex2(u.x);
          u.y = ex2(u.y);
          sum[c / 2 % 2] = add2(sum[c / 2 % 2], u);
          w[c / 2] = Num<T>::pack(u.x, u.y);
        }
        st32(s_at + c0 / 2, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    }
    if (tiles > 0) mbar_wait(&pv_done[t], 0, abort_flag, a.st, 113);
    tc_fence_after();
    // the tile's products are done: its first query chunk is free as a stage, 4 KB a warp
    const bool live = !(l <= 0.f);
    const float inv = live ? 1.f / l : 0.f;
    const int w_row = row - lane;
    uint8_t* stage = s_q + t * nqk * kExChunk + (warp % 4) * 4096;
    uint8_t* dst = static_cast<uint8_t*>(a.out) + ((int64_t)(q_lo + w_row) * a.H + head) * (a.nv * 128);
    const bool summed = tiles > 0;
    for (int c = 0; c < a.nv; c++) {
      uint32_t w[32];
      load_acc64<T>(o_at + c * 64, summed, inv, w);
      if (!live)
#pragma unroll
        for (int k = 0; k < 32; k++) w[k] = 0;
      store_rows(stage, w, lane, nq - w_row, dst + c * 128, (int64_t)a.H * (a.nv * 128));
    }
    if (row < nq) a.lse[(int64_t)head * a.Tq + q_lo + row] = live ? (ref + log2f(l)) * 0.693147180559945309f : -INFINITY;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------- backward
// Two kernels, one over query rows (dq) and one over key rows (dk, dv): each output row is summed by one
// CTA in a fixed order, at the price of computing S and dP twice (7 products for 5). Both keep the tensor
// cores one step ahead of the element-wise work, which turns S and dP into P and dS:
//   issue order  S(i + 1), dP(i + 1), then the sums over step i.
// P and dS reach the tensor cores through tensor memory, rounded to the 16-bit type (as the gradients
// themselves); scale is applied to the fp32 sums.
// fp16 holds dS = P (dP - delta) up to 65504 only, where the gradients, after the scale and the sums, may be far
// within the type. So in fp16 a row of dS is held times a power of two, 1 until one of its values passes the
// type; then the row's largest value comes to 2^14 .. 2^15, and the sums so far with it. Ordinary values are as
// without it; a step's check costs fp16 4 to 7 % (forward and backward of 4100 tokens at 64 heads 1645 -> 1707 us,
// of 7 documents 635 -> 680; a vote of all 256 threads and the largest value itself 1818 and 690). bf16 has
// fp32's range.
// Per step the products take 2048 (dq: 128 keys) and about 1400 cycles (dk, dv: 64 queries) against 1024 and
// 512 of exponentials; measured 3000 and 1900. 4100 tokens at 64 heads: 0.59 ms (dq) and 0.68 ms (dk, dv); 7
// documents of 150 to 1024 tokens: 0.20 and 0.23 ms, half of it the blocks' first loads (120 KB, 5000 cycles
// with the set-up) and stores (3000).
//
// Tensor memory, 512 columns each:
//   dq:     S 0 (128), dP 128 (128), dQ 256 (192), dS 448 (64)
//   dk, dv: S^T 0 (64), dP^T 64 (64), dV 128 (128), dK 256 (192), P^T 448 (32), dS^T 480 (32)
// Threads: warps 0-3 and 4-7 the element-wise work, each group half of a tile's columns; 8 TMA; 9 the
// products of S and dP; 11 the sums (a warp that has issued a batch gets on only as the tensor cores take it
// up, so one issuer alone would leave them idle for its waits); 10 (dk, dv) the queries' statistics, (dq) the
// lengths' check.
struct ExBwdArgs {
  const int32_t *cu_q, *cu_k;
  const void *g, *o;
  int64_t g_t, g_h;
  const float* lse;
  float* delta;            // [H][Tq]: written by the dq kernel, read by the other
  float* dkpe;             // [H][Tk][64 nr]
  void *dq, *dk, *dv;
  int B, Tq, Tk, H, nn, nr, nv, causal;
  ExOrder order;
  float scale, scale_log2;
  DevStatus* st;
};

// P and dS (without the scale) of two scores, in packed operations.
struct PAndDs {
  float2 p, ds;
};
LL_DEV PAndDs p_and_ds(uint32_t s0, uint32_t s1, uint32_t d0, uint32_t d1, float scale_log2, float2 neg_lse2,
                       float2 neg_delta) {
  float2 p = fma2(make_float2(__uint_as_float(s0), __uint_as_float(s1)), make_float2(scale_log2, scale_log2), neg_lse2);
  p.x = ex2(p.x);
  p.y = ex2(p.y);
  return {p, mul2(p, add2(make_float2(__uint_as_float(d0), __uint_as_float(d1)), neg_delta))};
}
// Rows from .. rows - 1 of `chunks` consecutive chunks of `rows` rows to zero, by 256 threads.
LL_DEV void zero_tail(uint8_t* at, int chunks, int rows, int from) {
  for (int i = threadIdx.x; i < (rows - from) * chunks * 8; i += 256) {
    const int c = i / ((rows - from) * 8), j = i % ((rows - from) * 8);
    *reinterpret_cast<uint4*>(at + (c * rows + from) * 128 + j * 16) = make_uint4(0, 0, 0, 0);
  }
}

// A row's factor for a step whose dS this thread holds N values of (d, their squares' sum sq): f, or less when a
// value passes fp16's range. Threads t and t + 128 share row t of the tile, so their two warps vote; the sum of
// squares, one packed operation for two values, stands for the largest value until it passes the limit. The
// row's sums so far, `cols` columns from `acc` on, are brought to the new factor once `summed` has waited for them
// (false: there are none). A row that holds an infinity keeps its factor: its gradient is not finite either.
template <int N, class Summed>
LL_DEV float ds_factor(const uint32_t* d, float sq, float f, float* s_top, uint32_t acc, int cols, Summed summed) {
  constexpr float kMost = 65504.f;
  const int t = threadIdx.x, pair = 2 + t / 32 % 4;
  if (!bar_any<64>(pair, !(sq * (f * f) <= kMost * kMost))) return f;
  float m = 0.f;
#pragma unroll
  for (int c = 0; c < N; c++) m = fmaxf(m, fabsf(__uint_as_float(d[c])));
  s_top[t] = m * f;
  named_bar_sync(pair, 64);
  const float top = fmaxf(s_top[t % 128], s_top[t % 128 + 128]);
  // 2^(14 - e) for top = 2^e .. 2^(e + 1)
  const float less = top > kMost && top < INFINITY ? __uint_as_float((268u - (__float_as_uint(top) >> 23)) << 23) : 1.f;
  if (summed()) {
    for (int c = t / 128 * 32; c < cols; c += 64) {
      uint32_t o[32];
      ld32(acc + c, o);
      tmem_ld_wait();
      ld32_ready(o);
#pragma unroll
      for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * less);
      st32(acc + c, o);
    }
    tmem_st_wait();
  }
  return f * less;
}
// N values of dS, times their row's factor, as words of the 16-bit type.
template <class T, int N>
LL_DEV void pack_ds(const uint32_t* d, float f, uint32_t* w) {
  if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) w[c / 2] = Num<T>::pack(__uint_as_float(d[c]) * f, __uint_as_float(d[c + 1]) * f);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 2) w[c / 2] = Num<T>::pack(__uint_as_float(d[c]), __uint_as_float(d[c + 1]));
  }
}

template <class T>
__global__ void __launch_bounds__(kExThreads, 1) k_ex_dq(const __grid_constant__ ExTma tm, const ExBwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nqk = a.nn + a.nr;
  uint8_t* s_q = base;
  uint8_t* s_g = s_q + nqk * kExChunk;
  uint8_t* s_k = s_g + a.nv * kExChunk;                   // two key tiles
  uint8_t* s_v = s_k + 2 * nqk * kExChunk;                // one value tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_v + a.nv * kExChunk);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_rel = bars + 3, *v_full = bars + 5, *v_rel = bars + 6,
           *sp_full = bars + 7, *sp_free = bars + 8, *ds_ready = bars + 9, *acc_done = bars + 10, *drain = bars + 11;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_delta = reinterpret_cast<float*>(tmem_slot + 4);      // [128], read before the steps; in them [256] of ds_factor
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int tile, head;
  ex_deal(a.order, tile, head);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 13; i++) mbar_init(&bars[i], i == 8 || i == 9 ? 8 : 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm.q);
    tma_prefetch_desc(&tm.g);
    tma_prefetch_desc(&tm.kn);
    tma_prefetch_desc(&tm.kp);
    tma_prefetch_desc(&tm.v);
  }
  __syncwarp();
  pdl_wait();
  int b, q0, q_lo = 0, q_hi = 0, k_lo = 0, k_hi = 0;
  if (find_tile<true>(a.cu_q, a.B, a.Tq, 128, tile, b, q0)) {
    seq_range(a.cu_q, b, a.Tq, q_lo, q_hi);
    seq_range(a.cu_k, b, a.Tk, k_lo, k_hi);
  } else {
    q0 = 0;
  }
  const int nq = q_hi - q_lo, nk = k_hi - k_lo, n = key_tiles(q0, 128, nq, nk, a.causal);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_next();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kExBwdLess));
    if (warp == 8 && n > 0) {
      // ----------------------------------------------------------------- TMA (lane c: chunk c)
      bool ok = true;
      if (lane == 0) mbar_arrive_expect_tx(q_full, (nqk + a.nv) * kExChunk);
      __syncwarp();
      if (lane < nqk) tma_load_3d(s_q + lane * kExChunk, &tm.q, q_full, lane * 64, head, q_lo + q0);
      else if (lane < nqk + a.nv)
        tma_load_3d(s_g + (lane - nqk) * kExChunk, &tm.g, q_full, (lane - nqk) * 64, head, q_lo + q0);
      int nk_loads = 0, nv_loads = 0;
      for (int i = 0; i < n && ok; i++) {
        const int row = k_lo + i * 128;
        if (!(ok = warp_wait_sleep(&k_rel[i & 1], ((i >> 1) & 1) ^ 1, abort_flag, a.st, 121, 64))) break;
        if (lane == 0) mbar_arrive_expect_tx(&k_full[i & 1], nqk * kExChunk);
        __syncwarp();
        uint8_t* dst = s_k + ((i & 1) * nqk + lane) * kExChunk;
        if (lane < a.nn) tma_load_3d(dst, &tm.kn, &k_full[i & 1], lane * 64, head, row);
        else if (lane < nqk) tma_load_2d(dst, &tm.kp, &k_full[i & 1], (lane - a.nn) * 64, row);
        nk_loads++;
        if (!(ok = warp_wait_sleep(v_rel, (i & 1) ^ 1, abort_flag, a.st, 122, 64))) break;
        if (lane == 0) mbar_arrive_expect_tx(v_full, a.nv * kExChunk);
        __syncwarp();
        if (lane < a.nv) tma_load_3d(s_v + lane * kExChunk, &tm.v, v_full, lane * 64, head, row);
        nv_loads++;
      }
      volatile int keep = 0;                   // everything issued has landed, also after an abort
      mbar_wait_sleep(q_full, 0, &keep, a.st, 123, 64);
      for (int i = max(0, nk_loads - 2); i < nk_loads; i++)
        mbar_wait_sleep(&k_full[i & 1], (i >> 1) & 1, &keep, a.st, 124, 64);
      if (nv_loads > 0) mbar_wait_sleep(v_full, (nv_loads - 1) & 1, &keep, a.st, 125, 64);
    }
    __syncwarp();
    if (warp == 9) {
      // ----------------------------------------------------------------------------- MMA
      const bool lead = elect_one();
      const uint32_t id_s = idesc_16bit(Num<T>::fmt, 128, 128, false, false);
      const MmaDesc q_d(smem_u32(s_q), 16, 1024), g_d(smem_u32(s_g), 16, 1024), k_d(smem_u32(s_k), 16, 1024),
          v_d(smem_u32(s_v), 16, 1024);
      const uint32_t k_tile = nqk * (kExChunk / 16);
      bool ok = n == 0 || mbar_wait(q_full, 0, abort_flag, a.st, 126);
#pragma unroll 1
      for (int j = 0; j < n && ok; j++) {
        if (j > 0 && !(ok = mbar_wait(sp_free, (j - 1) & 1, abort_flag, a.st, 127))) break;
        if (!(ok = mbar_wait(&k_full[j & 1], (j >> 1) & 1, abort_flag, a.st, 128))) break;
        tc_fence_after();
        if (lead) {
#pragma unroll 1
          for (int c = 0; c < nqk; c++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              mma_16bit(tmem, q_d.lo + c * (kExChunk / 16) + kk * 2, q_d.hi,
                        k_d.lo + (j & 1) * k_tile + c * (kExChunk / 16) + kk * 2, k_d.hi, id_s, c + kk);
        }
        if (!(ok = mbar_wait(v_full, j & 1, abort_flag, a.st, 129))) break;
        tc_fence_after();
        if (lead) {
#pragma unroll 1
          for (int c = 0; c < a.nv; c++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              mma_16bit(tmem + 128, g_d.lo + c * (kExChunk / 16) + kk * 2, g_d.hi, v_d.lo + c * (kExChunk / 16) + kk * 2,
                        v_d.hi, id_s, c + kk);
          mma_commit(sp_full);
          mma_commit(v_rel);
        }
      }
      __syncwarp();
      if (lead) mma_commit(&drain[0]);
      volatile int keep = 0;
      mbar_wait_sleep(&drain[0], 0, &keep, a.st, 131, 64);
      __syncwarp();
    } else if (warp == 11) {
      // ------------------------------------------------------------------------ MMA, sums
      const bool lead = elect_one();
      const uint32_t id_o = idesc_16bit(Num<T>::fmt, 128, nqk * 64, false, true);
      const MmaDesc kt_d(smem_u32(s_k), kExChunk, 1024);
      const uint32_t k_tile = nqk * (kExChunk / 16);
#pragma unroll 1
      for (int i = 0; i < n; i++) {
        if (!mbar_wait(ds_ready, i & 1, abort_flag, a.st, 130)) break;
        tc_fence_after();
        if (lead) {
#pragma unroll
          for (int kk = 0; kk < 8; kk++)
            mma_16bit_ts(tmem + 256, tmem + 448 + kk * 8, kt_d.lo + (i & 1) * k_tile + kk * 128, kt_d.hi, id_o, i + kk);
          mma_commit(&k_rel[i & 1]);
          mma_commit(acc_done);
        }
      }
      __syncwarp();
      if (lead) mma_commit(&drain[1]);
      volatile int keep = 0;
      mbar_wait_sleep(&drain[1], 0, &keep, a.st, 135, 64);
      __syncwarp();
    } else if (warp == 10 && blockIdx.x == gridDim.x - 1) {
      check_cu(a.cu_q, a.B, a.Tq, a.st, 77);
      check_cu(a.cu_k, a.B, a.Tk, a.st, 78);
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------------- element-wise
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kExBwdMore));
    const int cw = warp / 4;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    const int row = q0 + (warp % 4) * 32 + lane;
    const int see = a.causal ? min(nk, row + nk - nq + 1) : nk, see_all = a.causal ? min(nk, q0 + nk - nq + 1) : nk;
    {
      // delta of the tile's rows, sixteen lanes a row and sixteen rows a warp, all loads at once (of rows and
      // columns that exist, whatever is past them: a load under a condition waits for the one before)
      uint4 gv[8], ov[8];
      const int c = min(lane % 16, a.nv * 8 - 1), r0 = q0 + warp * 16 + lane / 16;
      const T* gp = static_cast<const T*>(a.g) + head * a.g_h + c * 8;
      const T* op = static_cast<const T*>(a.o) + (int64_t)head * (a.nv * 64) + c * 8;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int64_t r = q_lo + max(0, min(r0 + i * 2, nq - 1));
        gv[i] = *reinterpret_cast<const uint4*>(gp + r * a.g_t);
        ov[i] = *reinterpret_cast<const uint4*>(op + r * a.H * (a.nv * 64));
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const T *gx = reinterpret_cast<const T*>(&gv[i]), *ox = reinterpret_cast<const T*>(&ov[i]);
        float d = 0.f;
#pragma unroll
        for (int z = 0; z < 8; z++) d = fmaf(Num<T>::to_f(gx[z]), Num<T>::to_f(ox[z]), d);
        if (lane % 16 >= a.nv * 8) d = 0.f;
#pragma unroll
        for (int off = 8; off; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
        if (lane % 16 == 0) s_delta[warp * 16 + i * 2 + lane / 16] = d;
      }
    }
    named_bar_sync(1, 256);
    const float delta = s_delta[row - q0];
    float lse2 = 0.f;
    if (row < nq) {
      const int64_t at = (int64_t)head * a.Tq + q_lo + row;
      lse2 = a.lse[at] * 1.4426950408889634f;
      if (cw == 0) a.delta[at] = delta;
    }
    float f = 1.f;                             // dS's factor (fp16)
    for (int i = 0; i < n; i++) {
      mbar_wait(sp_full, i & 1, abort_flag, a.st, 132);
      tc_fence_after();
      uint32_t x[64], y[64];
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        ld32(tmem + lanes + cw * 64 + c, x + c);
        ld32(tmem + 128 + lanes + cw * 64 + c, y + c);
      }
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        ld32_ready(x + c);
        ld32_ready(y + c);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sp_free);
      if (i * 128 + 128 > nk) {                // key rows past the end must not meet dS's zeros
        zero_tail(s_k + (i & 1) * nqk * kExChunk, nqk, 128, nk - i * 128);
        fence_async_smem();
      }
      uint32_t w[32];
      if constexpr (Num<T>::narrow) {
        float2 sq = make_float2(0.f, 0.f);
        auto compute = [&](int lim) {
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float2 d = p_and_ds(x[c], x[c + 1], y[c], y[c + 1], a.scale_log2, make_float2(-lse2, -lse2),
                                make_float2(-delta, -delta)).ds;
            d = make_float2(c < lim ? d.x : 0.f, c + 1 < lim ? d.y : 0.f);
            sq = fma2(d, d, sq);
            x[c] = __float_as_uint(d.x);
            x[c + 1] = __float_as_uint(d.y);
          }
        };
        if (i * 128 + 128 <= see_all) compute(64);       // every row sees every key
        else compute(see - i * 128 - cw * 64);
        f = ds_factor<64>(x, row < nq ? sq.x + sq.y : 0.f, f, s_delta, tmem + 256 + lanes, nqk * 64, [&] {
          if (i > 0) mbar_wait(acc_done, (i - 1) & 1, abort_flag, a.st, 136);
          tc_fence_after();
          return i > 0;
        });
        pack_ds<T, 64>(x, f, w);
      } else if (i * 128 + 128 <= see_all) {   // every row sees every key
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 d = p_and_ds(x[c], x[c + 1], y[c], y[c + 1], a.scale_log2, make_float2(-lse2, -lse2),
                                    make_float2(-delta, -delta)).ds;
          w[c / 2] = Num<T>::pack(d.x, d.y);
        }
      } else {
        const int lim = see - i * 128 - cw * 64;
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 d = p_and_ds(x[c], x[c + 1], y[c], y[c + 1], a.scale_log2, make_float2(-lse2, -lse2),
                                    make_float2(-delta, -delta)).ds;
          w[c / 2] = Num<T>::pack(c < lim ? d.x : 0.f, c + 1 < lim ? d.y : 0.f);
        }
      }
      if (i > 0) mbar_wait(acc_done, (i - 1) & 1, abort_flag, a.st, 133);
      tc_fence_after();
      st32(tmem + 448 + lanes + cw * 32, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
    }
    if (n > 0) mbar_wait(acc_done, (n - 1) & 1, abort_flag, a.st, 134);
    tc_fence_after();
    // every product is done: the query tile (first group) and its gradient's (second) are free as stages
    const int w_row = row - lane;
    uint8_t* stage = (cw ? s_g : s_q) + (warp % 4) * 4096;
    uint8_t* dst = static_cast<uint8_t*>(a.dq) + ((int64_t)(q_lo + w_row) * a.H + head) * (nqk * 128);
    for (int c = cw; c < nqk; c += 2) {
      uint32_t w[32];
      load_acc64<T>(tmem + 256 + lanes + c * 64, n > 0, a.scale / f, w);
      store_rows(stage, w, lane, nq - w_row, dst + c * 128, (int64_t)a.H * (nqk * 128));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

constexpr int kExQ = 64;                 // query rows a step of the key-row kernel
constexpr int kExQStages = 3;
constexpr int kExQChunk = kExQ * 128;    // bytes

template <class T>
__global__ void __launch_bounds__(kExThreads, 1) k_ex_dkv(const __grid_constant__ ExTma tm, const ExBwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nqk = a.nn + a.nr, stage = (nqk + a.nv) * kExQChunk;
  uint8_t* s_k = base;
  uint8_t* s_v = s_k + nqk * kExChunk;
  uint8_t* s_qg = s_v + a.nv * kExChunk;                  // stages of Q and dO
  float4* s_stat = reinterpret_cast<float4*>(s_qg + kExQStages * stage);      // [stage][32]: -lse, -delta of two queries
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_stat + kExQStages * 32);
  uint64_t *kv_full = bars, *q_full = bars + 1, *q_rel = q_full + kExQStages, *st_full = q_rel + kExQStages,
           *sp_full = st_full + kExQStages, *sp_free = sp_full + 1, *ds_ready = sp_full + 2, *acc_done = sp_full + 3,
           *drain = sp_full + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_top = reinterpret_cast<float*>(tmem_slot + 4);        // [256] of ds_factor
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int tile, head;
  ex_deal(a.order, tile, head);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 3 * kExQStages + 7; i++) mbar_init(&bars[i], &bars[i] == sp_free || &bars[i] == ds_ready ? 8 : 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm.q);
    tma_prefetch_desc(&tm.g);
    tma_prefetch_desc(&tm.kn);
    tma_prefetch_desc(&tm.kp);
    tma_prefetch_desc(&tm.v);
  }
  __syncwarp();
  pdl_wait();
  int b, k0, q_lo = 0, q_hi = 0, k_lo = 0, k_hi = 0;
  if (find_tile<false>(a.cu_k, a.B, a.Tk, 128, tile, b, k0)) {
    seq_range(a.cu_q, b, a.Tq, q_lo, q_hi);
    seq_range(a.cu_k, b, a.Tk, k_lo, k_hi);
  } else {
    k0 = 0;
  }
  const int nq = q_hi - q_lo, nk = k_hi - k_lo, shift = nk - nq;
  // the queries from the first that sees key k0 on
  const int first = k0 >= nk ? nq : a.causal ? max(0, k0 - shift) / kExQ * kExQ : 0;
  const int n = first < nq ? (nq - first + kExQ - 1) / kExQ : 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_next();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kExBwdLess));
    if (warp == 8 && n > 0) {
      // ----------------------------------------------------------------- TMA (lane c: chunk c)
      if (lane == 0) mbar_arrive_expect_tx(kv_full, (nqk + a.nv) * kExChunk);
      __syncwarp();
      if (lane < a.nn) tma_load_3d(s_k + lane * kExChunk, &tm.kn, kv_full, lane * 64, head, k_lo + k0);
      else if (lane < nqk) tma_load_2d(s_k + lane * kExChunk, &tm.kp, kv_full, (lane - a.nn) * 64, k_lo + k0);
      else if (lane < nqk + a.nv)
        tma_load_3d(s_v + (lane - nqk) * kExChunk, &tm.v, kv_full, (lane - nqk) * 64, head, k_lo + k0);
      int i = 0;
      for (; i < n; i++) {
        const int s = i % kExQStages, row = q_lo + first + i * kExQ;
        if (!warp_wait_sleep(&q_rel[s], ((i / kExQStages) & 1) ^ 1, abort_flag, a.st, 141, 64)) break;
        if (lane == 0) mbar_arrive_expect_tx(&q_full[s], stage);
        __syncwarp();
        uint8_t* dst = s_qg + s * stage + lane * kExQChunk;
        if (lane < nqk) tma_load_3d(dst, &tm.q, &q_full[s], lane * 64, head, row);
        else if (lane < nqk + a.nv) tma_load_3d(dst, &tm.g, &q_full[s], (lane - nqk) * 64, head, row);
      }
      volatile int keep = 0;                   // everything issued has landed, also after an abort
      mbar_wait_sleep(kv_full, 0, &keep, a.st, 142, 64);
      for (int k = max(0, i - kExQStages); k < i; k++)
        mbar_wait_sleep(&q_full[k % kExQStages], (k / kExQStages) & 1, &keep, a.st, 143, 64);
    }
    __syncwarp();
    if (warp == 9) {
      // ----------------------------------------------------------------------------- MMA
      const bool lead = elect_one();
      const uint32_t id_s = idesc_16bit(Num<T>::fmt, 128, kExQ, false, false);
      const MmaDesc k_d(smem_u32(s_k), 16, 1024), v_d(smem_u32(s_v), 16, 1024), q_d(smem_u32(s_qg), 16, 1024);
      constexpr uint32_t QC = kExQChunk / 16;
      bool ok = n == 0 || mbar_wait(kv_full, 0, abort_flag, a.st, 144);
#pragma unroll 1
      for (int j = 0; j < n && ok; j++) {
        const int s = j % kExQStages;
        if (j > 0 && !(ok = mbar_wait(sp_free, (j - 1) & 1, abort_flag, a.st, 145))) break;
        if (!(ok = mbar_wait(&q_full[s], (j / kExQStages) & 1, abort_flag, a.st, 146))) break;
        tc_fence_after();
        if (lead) {
          const uint32_t at = q_d.lo + s * (stage / 16);
#pragma unroll 1
          for (int c = 0; c < nqk; c++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              mma_16bit(tmem, k_d.lo + c * (kExChunk / 16) + kk * 2, k_d.hi, at + c * QC + kk * 2, q_d.hi, id_s, c + kk);
#pragma unroll 1
          for (int c = 0; c < a.nv; c++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              mma_16bit(tmem + 64, v_d.lo + c * (kExChunk / 16) + kk * 2, v_d.hi, at + (nqk + c) * QC + kk * 2, q_d.hi,
                        id_s, c + kk);
          mma_commit(sp_full);
        }
      }
      __syncwarp();
      if (lead) mma_commit(&drain[0]);
      volatile int keep = 0;
      mbar_wait_sleep(&drain[0], 0, &keep, a.st, 148, 64);
      __syncwarp();
    } else if (warp == 11) {
      // ------------------------------------------------------------------------ MMA, sums
      const bool lead = elect_one();
      const uint32_t id_k = idesc_16bit(Num<T>::fmt, 128, nqk * 64, false, true);
      const uint32_t id_v = idesc_16bit(Num<T>::fmt, 128, a.nv * 64, false, true);
      const MmaDesc qt_d(smem_u32(s_qg), kExQChunk, 1024);
      constexpr uint32_t QC = kExQChunk / 16;
#pragma unroll 1
      for (int i = 0; i < n; i++) {
        if (!mbar_wait(ds_ready, i & 1, abort_flag, a.st, 147)) break;
        tc_fence_after();
        if (lead) {
          const uint32_t at = qt_d.lo + (i % kExQStages) * (stage / 16);
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
            mma_16bit_ts(tmem + 128, tmem + 448 + kk * 8, at + nqk * QC + kk * 128, qt_d.hi, id_v, i + kk);
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
            mma_16bit_ts(tmem + 256, tmem + 480 + kk * 8, at + kk * 128, qt_d.hi, id_k, i + kk);
          mma_commit(&q_rel[i % kExQStages]);
          mma_commit(acc_done);
        }
      }
      __syncwarp();
      if (lead) mma_commit(&drain[1]);
      volatile int keep = 0;
      mbar_wait_sleep(&drain[1], 0, &keep, a.st, 154, 64);
      __syncwarp();
    } else if (warp == 10) {
      // ------------------------------------------------- statistics of the steps' queries
      if (a.Tq == 0 && blockIdx.x == gridDim.x - 1) {      // (with queries, k_ex_dq has checked)
        check_cu(a.cu_q, a.B, 0, a.st, 77);
        check_cu(a.cu_k, a.B, a.Tk, a.st, 78);
        __syncwarp();
      }
      for (int i = 0; i < n; i++) {
        const int s = i % kExQStages;
        mbar_wait_sleep(&q_rel[s], ((i / kExQStages) & 1) ^ 1, abort_flag, a.st, 149, 64);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int z = 0; z < 2; z++) {
          const int q = first + i * kExQ + lane * 2 + z;
          if (q < nq) {
            const int64_t at = (int64_t)head * a.Tq + q_lo + q;
            v[z] = -a.lse[at] * 1.4426950408889634f;
            v[2 + z] = -a.delta[at];
          }
        }
        s_stat[s * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&st_full[s]);
      }
    }
  } else {
    // ---------------------------------------------------------------------- element-wise
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kExBwdMore));
    const int cw = warp / 4;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    const int row = k0 + (warp % 4) * 32 + lane;
    float f = 1.f;                             // dS's factor (fp16)
    for (int i = 0; i < n; i++) {
      const int s = i % kExQStages, qa = first + i * kExQ;
      mbar_wait(&st_full[s], (i / kExQStages) & 1, abort_flag, a.st, 150);
      mbar_wait(sp_full, i & 1, abort_flag, a.st, 151);
      tc_fence_after();
      uint32_t x[32], y[32];
      ld32(tmem + lanes + cw * 32, x);
      ld32(tmem + 64 + lanes + cw * 32, y);
      tmem_ld_wait();
      ld32_ready(x);
      ld32_ready(y);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sp_free);
      if (qa + kExQ > nq) {                    // query rows past the end must not meet zeros of P and dS
        zero_tail(s_qg + s * stage, nqk + a.nv, kExQ, nq - qa);
        fence_async_smem();
      }
      uint32_t pw[16], dw[16];
      const float4* stat = s_stat + s * 32 + cw * 16;
      if constexpr (Num<T>::narrow) {
        float2 sq = make_float2(0.f, 0.f);
        auto compute = [&](int from, int to) {           // the queries that see the row
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float4 sd = stat[c / 2];
            PAndDs r = p_and_ds(x[c], x[c + 1], y[c], y[c + 1], a.scale_log2, make_float2(sd.x, sd.y),
                                make_float2(sd.z, sd.w));
            const bool u = c >= from && c < to, v = c + 1 >= from && c + 1 < to;
            r.ds = make_float2(u ? r.ds.x : 0.f, v ? r.ds.y : 0.f);
            sq = fma2(r.ds, r.ds, sq);
            pw[c / 2] = Num<T>::pack(u ? r.p.x : 0.f, v ? r.p.y : 0.f);
            y[c] = __float_as_uint(r.ds.x);
            y[c + 1] = __float_as_uint(r.ds.y);
          }
        };
        if (qa + kExQ <= nq && (!a.causal || k0 + 127 <= qa + shift)) compute(0, 32);
        else compute((a.causal ? row - shift - qa : 0) - cw * 32, nq - qa - cw * 32);
        f = ds_factor<32>(y, row < nk ? sq.x + sq.y : 0.f, f, s_top, tmem + 256 + lanes, nqk * 64, [&] {
          if (i > 0) mbar_wait(acc_done, (i - 1) & 1, abort_flag, a.st, 155);
          tc_fence_after();
          return i > 0;
        });
        pack_ds<T, 32>(y, f, dw);
      } else if (qa + kExQ <= nq && (!a.causal || k0 + 127 <= qa + shift)) {     // every query sees every row
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float4 sd = stat[c / 2];
          const PAndDs r = p_and_ds(x[c], x[c + 1], y[c], y[c + 1], a.scale_log2, make_float2(sd.x, sd.y),
                                    make_float2(sd.z, sd.w));
          pw[c / 2] = Num<T>::pack(r.p.x, r.p.y);
          dw[c / 2] = Num<T>::pack(r.ds.x, r.ds.y);
        }
      } else {
        const int from = (a.causal ? row - shift - qa : 0) - cw * 32, to = nq - qa - cw * 32;   // queries that see the row
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float4 sd = stat[c / 2];
          const PAndDs r = p_and_ds(x[c], x[c + 1], y[c], y[c + 1], a.scale_log2, make_float2(sd.x, sd.y),
                                    make_float2(sd.z, sd.w));
          const bool u = c >= from && c < to, v = c + 1 >= from && c + 1 < to;
          pw[c / 2] = Num<T>::pack(u ? r.p.x : 0.f, v ? r.p.y : 0.f);
          dw[c / 2] = Num<T>::pack(u ? r.ds.x : 0.f, v ? r.ds.y : 0.f);
        }
      }
      if (i > 0) mbar_wait(acc_done, (i - 1) & 1, abort_flag, a.st, 152);
      tc_fence_after();
      tmem_st16(tmem + 448 + lanes + cw * 16, pw);
      tmem_st16(tmem + 480 + lanes + cw * 16, dw);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
    }
    if (n > 0) mbar_wait(acc_done, (n - 1) & 1, abort_flag, a.st, 153);
    tc_fence_after();
    // every product is done: the key tile (first group) and the value tile (second) are free as stages
    const int w_row = row - lane;
    uint8_t* stage = (cw ? s_v : s_k) + (warp % 4) * 4096;
    const int64_t at = (int64_t)(k_lo + w_row) * a.H + head;
    for (int c = cw; c < a.nv + a.nn; c += 2) {
      const bool v = c < a.nv;
      const int cc = v ? c : c - a.nv, chunks = v ? a.nv : a.nn;
      uint32_t w[32];
      load_acc64<T>(tmem + lanes + (v ? 128 : 256) + cc * 64, n > 0, v ? 1.f : a.scale / f, w);
      store_rows(stage, w, lane, nk - w_row, static_cast<uint8_t*>(v ? a.dv : a.dk) + at * (chunks * 128) + cc * 128,
                 (int64_t)a.H * (chunks * 128));
    }
    for (int c = cw * 32; c < a.nr * 64; c += 64) {
      uint32_t w[32];
      if (n > 0) {
        ld32(tmem + lanes + 256 + a.nn * 64 + c, w);
        tmem_ld_wait();
        ld32_ready(w);
      }
#pragma unroll
      for (int k = 0; k < 32; k++) w[k] = n > 0 ? __float_as_uint(__uint_as_float(w[k]) * (a.scale / f)) : 0u;
      store_rows(stage, w, lane, nk - w_row,
                 reinterpret_cast<uint8_t*>(a.dkpe + ((int64_t)head * a.Tk + k_lo + w_row) * (a.nr * 64) + c), a.nr * 256);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// dk_pe[row][d] = sum over the heads, in their order; four values a thread, eight heads' loads in flight.
template <class T>
__global__ void __launch_bounds__(256) k_ex_sum_heads(const float* __restrict__ ws, int H, int64_t n, T* __restrict__ out) {
  pdl_wait();
  const int64_t i = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) * 4;
  if (i >= n) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int h0 = 0; h0 < H; h0 += 8) {
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = *reinterpret_cast<const float4*>(ws + (int64_t)min(h0 + k, H - 1) * n + i);
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (h0 + k < H) { s.x += v[k].x; s.y += v[k].y; s.z += v[k].z; s.w += v[k].w; }
  }
  *reinterpret_cast<uint2*>(out + i) = make_uint2(Num<T>::pack(s.x, s.y), Num<T>::pack(s.z, s.w));
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

static int packed_maps(ExTma* tm, const ll_latent_packed* p, uint32_t q_rows = 128) {
  const CUtensorMapDataType dt = p->dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int dq = p->d_n + p->d_r;
  // an operand without rows is never loaded; its map is any valid one
  if (p->Tq) LL_TRY(rows_map(&tm->q, dt, p->q, p->Tq, p->q_stride_t, p->H, p->q_stride_h, dq, q_rows));
  if (p->Tk) {
    LL_TRY(rows_map(&tm->kn, dt, p->k_nope, p->Tk, p->k_stride_t, p->H, p->k_stride_h, p->d_n));
    LL_TRY(rows_map(&tm->v, dt, p->v, p->Tk, p->v_stride_t, p->H, p->v_stride_h, p->d_v));
    if (p->d_r)
      LL_TRY(make_map_2d(&tm->kp, dt, p->k_pe, 64, (uint64_t)p->Tk, (uint64_t)p->kpe_stride_t * 2, 64, 128,
                         CU_TENSOR_MAP_SWIZZLE_128B));
    else tm->kp = tm->kn;
  }
  if (!p->Tq) tm->q = tm->kn;
  if (!p->Tk) tm->kn = tm->kp = tm->v = tm->q;
  tm->g = tm->q;
  return LL_OK;
}

static ExOrder ex_order(int rows, int per_tile, const ll_latent_packed* p) {
  const int tiles = rows / per_tile + p->B;      // at least the sum of ceil(length / per_tile)
  const int sms = std::max(1, device_info().sms);
  return {tiles, p->H, std::min(p->H, std::max(1, (4 * sms + tiles - 1) / tiles))};
}

static int check_packed(const ll_latent_packed* p) {
  if (!p || p->B < 0 || p->Tq < 0 || p->Tk < 0 || p->H <= 0 || (p->d_n != 64 && p->d_n != 128) ||
      (p->d_v != 64 && p->d_v != 128) || (p->d_r != 0 && p->d_r != 64) || (p->dtype != 1 && p->dtype != 2) ||
      !(p->scale > 0.f))
    return LL_ERR_ARG;
  if (p->B == 0 || (p->Tq == 0 && p->Tk == 0)) return LL_OK;
  if (!p->cu_q || !p->cu_k || ((int64_t)std::max(p->Tq, p->Tk) / 128 + p->B) * p->H > INT32_MAX)
    return LL_ERR_ARG;
  if (p->Tq && bad16(p->q, p->q_stride_t, p->q_stride_h)) return LL_ERR_ARG;
  if (p->Tk && (bad16(p->k_nope, p->k_stride_t, p->k_stride_h) || bad16(p->v, p->v_stride_t, p->v_stride_h) ||
                (p->d_r && bad16(p->k_pe, p->kpe_stride_t, 8))))
    return LL_ERR_ARG;
  return LL_OK;
}

template <class T>
static int run_backward(const ll_latent_packed* p, const ExTma& tq, const ExTma& tk, ExBwdArgs& a, void* dk_pe,
                        cudaStream_t s) {
  const int nqk = a.nn + a.nr;
  if (p->Tq) {
    const int smem = 1024 + (3 * nqk + 2 * a.nv) * kExChunk + 13 * 8 + 16 + 1024;
    LL_TRY(set_smem_attr(reinterpret_cast<const void*>(k_ex_dq<T>), smem));
    a.order = ex_order(p->Tq, 128, p);
    LL_TRY(launch_pdl("k_ex_dq", k_ex_dq<T>, dim3(a.order.tiles * p->H), dim3(kExThreads), smem, s, tq, a));
  }
  if (p->Tk) {
    const int smem =
        1024 + (nqk + a.nv) * (kExChunk + kExQStages * kExQChunk) + kExQStages * 512 + (3 * kExQStages + 7) * 8 + 16 + 1024;
    LL_TRY(set_smem_attr(reinterpret_cast<const void*>(k_ex_dkv<T>), smem));
    a.order = ex_order(p->Tk, 128, p);
    LL_TRY(launch_pdl("k_ex_dkv", k_ex_dkv<T>, dim3(a.order.tiles * p->H), dim3(kExThreads), smem, s, tk, a));
    const int64_t n = (int64_t)p->Tk * p->d_r;
    if (n)
      LL_TRY(launch_pdl("k_ex_sum_heads", k_ex_sum_heads<T>, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s,
                        (const float*)a.dkpe, p->H, n, static_cast<T*>(dk_pe)));
  }
  return LL_OK;
}

static size_t backward_floats(const ll_latent_packed* p) {
  return ((size_t)p->H * p->Tk * p->d_r + 63) / 64 * 64 + (size_t)p->H * p->Tq;
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
              ex_order(p->Tq, 256, p), p->scale * 1.4426950408889634f, latent_status()};
  if (!a.st) return LL_ERR_CUDA;
  const int smem = 1024 + (2 * (a.nn + a.nr) + kExRing) * kExChunk + (2 * kExOps + 9) * 8 + 16;
  auto run = [&](auto kern) {
    LL_TRY(set_smem_attr(reinterpret_cast<const void*>(kern), smem));
    return launch_pdl("k_ex_fwd", kern, dim3(a.order.tiles * p->H), dim3(kExThreads), smem, s, tm, a);
  };
  return p->dtype == 1 ? run(k_ex_fwd<__nv_bfloat16>) : run(k_ex_fwd<__half>);
}

size_t ll_latent_backward_workspace_bytes(const ll_latent_packed* p) {
  if (!p || p->H <= 0 || p->Tk < 0 || p->Tq < 0 || p->d_r < 0) return 0;
  return backward_floats(p) * 4 + 256;
}

int ll_latent_backward(const ll_latent_packed* p, const void* g, int64_t g_stride_t, int64_t g_stride_h,
                       const void* out, const float* lse, void* dq, void* dk_nope, void* dk_pe, void* dv,
                       void* workspace, size_t workspace_bytes, void* stream) {
  LL_TRY(check_packed(p));
  if (p->B == 0 || (p->Tq == 0 && p->Tk == 0)) return LL_OK;
  auto bad = [](const void* x) { return !x || (reinterpret_cast<uintptr_t>(x) & 15); };
  if (p->Tq && (bad16(g, g_stride_t, g_stride_h) || bad(out) || !lse || bad(dq))) return LL_ERR_ARG;
  if (p->Tk && (bad(dk_nope) || bad(dv) || (p->d_r && bad(dk_pe)))) return LL_ERR_ARG;
  if (bad(workspace)) return LL_ERR_ARG;
  if (workspace_bytes < ll_latent_backward_workspace_bytes(p)) return LL_ERR_WORKSPACE;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  ExTma tq, tk;
  LL_TRY(packed_maps(&tq, p));
  LL_TRY(packed_maps(&tk, p, kExQ));
  if (p->Tq) {
    const CUtensorMapDataType dt = p->dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    LL_TRY(rows_map(&tq.g, dt, g, p->Tq, g_stride_t, p->H, g_stride_h, p->d_v));
    LL_TRY(rows_map(&tk.g, dt, g, p->Tq, g_stride_t, p->H, g_stride_h, p->d_v, kExQ));
  }
  ExBwdArgs a{};
  a.cu_q = p->cu_q;
  a.cu_k = p->cu_k;
  a.g = g;
  a.o = out;
  a.g_t = g_stride_t;
  a.g_h = g_stride_h;
  a.lse = lse;
  a.dkpe = static_cast<float*>(workspace);
  a.delta = a.dkpe + ((size_t)p->H * p->Tk * p->d_r + 63) / 64 * 64;
  a.dq = dq;
  a.dk = dk_nope;
  a.dv = dv;
  a.B = p->B;
  a.Tq = p->Tq;
  a.Tk = p->Tk;
  a.H = p->H;
  a.nn = p->d_n / 64;
  a.nr = p->d_r / 64;
  a.nv = p->d_v / 64;
  a.causal = p->causal;
  a.scale = p->scale;
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.st = latent_status();
  if (!a.st) return LL_ERR_CUDA;
  return p->dtype == 1 ? run_backward<__nv_bfloat16>(p, tq, tk, a, dk_pe, s) : run_backward<__half>(p, tq, tk, a, dk_pe, s);
}

}  // extern "C"

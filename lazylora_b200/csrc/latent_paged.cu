// The absorbed form of latent attention over a paged cache (see the header for the interface): all
// rows (t, h) of a sequence's queries read the same cache rows, which are keys (all d_c + d_r values)
// and values (the first d_c) at once.
//   s_j = scale q . row_j,  p_j = 2^(s_j log2 e - m),  l = sum_j p_j,
//   out = (sum_j p_j row_j[:d_c]) / l,  lse = (m + log2 l) ln 2  for any reference m.
//
// Bound by HBM up to about 128 query rows (1152 bytes a key against 2 * 1088 flops a key and row).
// Both products are therefore taken transposed, with the cache rows as the tall operand A and the
// query rows as N, so that the tensor cores' work follows the number of rows instead of a padded
// 128, and one copy of a key tile in shared memory serves both:
//   S^T [64 keys][NT rows]  = tile (K-major) . Q^T       M = 64,  K = d_c + d_r
//   O^T [d_c][NT rows]     += tile^T (MN-major) . P^T    M = 128 (d_c / 128 times), K = 64 keys
// with NT = 16 .. 64 rows a CTA (more rows: more CTAs that read the same tiles, through L2, at the
// same time). O^T takes d_c / 128 * NT columns of tensor memory, S^T two times 64.
//
// A key tile lies in shared memory as eight groups of eight rows, [group][64-column chunk][8 rows][128
// bytes] with the 128-byte swizzle: one TMA box per group, so any page size that is a multiple of 8
// works and no page boundary lies inside a box, and a uniform group stride for both operand forms.
//
// Softmax: a thread owns one key and a quarter of the rows, S^T's tensor-memory lanes being keys. The
// reference m of a row only has to be within 2^8 of its running maximum, so a tile first asks (one
// barrier with a vote) whether any score passes its reference by more than 8; only then are the maxima
// taken across the keys, and O^T and l rescaled. l stays a partial sum per thread until the end. P is
// rounded to the 16-bit type for the tensor cores (at most 2^-8 or 2^-11 relative, as the output's own
// rounding); l sums the unrounded values in fp32.
//
// The tiles of all sequences, one after another, are dealt to the CTAs in equal contiguous ranges
// (from the lengths on the device, so a captured graph may be replayed with other lengths). A CTA whose
// range covers a sequence writes its output; pieces of a sequence go to the workspace (O in fp32, m, l)
// and k_paged_combine joins them in order. Ten warps: 0-7 softmax, rescaling, outputs; 8 TMA; 9 MMA.
//
// Measured (B200, 512 + 64 values a row): 44 sequences of 1 to 6000 keys at 64 heads 50 us, 4 of 50 to 70
// thousand 67 us (4.1 TB/s, 63 % of the copy rate), 24 times 2 tokens of 1500 to 5000 keys at 128 heads 85 us
// (512 TFLOP/s), one of 700 keys at 32 heads 11 us with the join. In the steady state a tile takes 3700
// cycles of which its load takes 3500: with 64 query rows in shared memory (74 KB) only two 74 KB tiles fit,
// so while one is computed (1150 cycles S^T, 850 softmax, 600 O^T) one load is in flight, and it shares the
// shared-memory ports with the products' operands (a 64 x 64 x 16 product reads 4 KB of them, 32 cycles, as
// long as it takes). The steps are three quarters of the long case (25 tiles an SM, 49 us); the rest is
// the start, the first maxima, the fp32 pieces written and read again, and the join's launch. Prefetching
// tiles into L2 and issuing S^T of the next tile ahead both measured slower.
//
// Rows of the last tile past the sequence's end, which may hold anything, are set to zero in shared
// memory before the second product (0 * NaN would reach the sums) and masked by their index.
#include "latent_ops.cuh"

namespace ll {

constexpr int kPgSoft = 256;           // softmax threads: warps 0-7; warp 8: TMA, warp 9: MMA
constexpr int kPgThreads = kPgSoft + 64;
constexpr int kPgKeys = 64;
constexpr float kPgSlack = 8.f;        // log2 of how far a score may pass its row's reference
constexpr float kPgNone = -1e30f;      // reference of a row that has seen no key

struct PagedArgs {
  const int32_t* bt;
  const int32_t* lens;
  void* out;
  float* lse;
  float* part;        // [G * 2][RT][NT][d_c] unnormalised pieces
  float* part_ml;     // [G * 2][RT][2][NT] their references (log2) and sums
  int* starts;        // [B + 1] weight before each sequence; last: weight of a range
  int64_t bt_stride;
  int pages, page_size, max_pages, B, Tq, H, rows, RT, G, nc, nchunk;   // chunks of 64: of d_c, of d_c + d_r
  float scale_log2;
  DevStatus* st;
};

struct PagedTma {
  CUtensorMap q, kv;
};

// (the host checks that this is an int)
LL_DEV int paged_room(const PagedArgs& a) { return a.max_pages * a.page_size; }
// A sequence's keys. A length outside the block table, which block 0 records, is cut to it: nothing is read outside.
LL_DEV int paged_len(const PagedArgs& a, int b) { return min(max(a.lens[b], 0), paged_room(a)); }
// A sequence without keys still has one (masked) tile, which writes its zeros.
LL_DEV int paged_tiles(int len) { return max(1, (len - 1) / kPgKeys + 1); }
// What a sequence weighs in the deal: its tiles, and before them the time that starting and ending it
// costs (query load, first maxima, output), which measured about two tiles.
constexpr int kPgStart = 2;
LL_DEV int paged_weight(int len) { return paged_tiles(len) + kPgStart; }

// tcgen05.ld of 16 lanes x 8 (or 4) columns twice: threads 0-15 take columns taddr .., threads 16-31
// columns taddr + SPLIT .. of the same lanes.
template <int SPLIT>
LL_DEV void tmem_ld_16x2_8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8], %9;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr), "n"(SPLIT));
}
template <int SPLIT>
LL_DEV void tmem_ld_16x2_4(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x4.b32 {%0,%1,%2,%3}, [%4], %5;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr), "n"(SPLIT));
}
// A softmax thread's NQ values of S^T.
template <int NQ>
LL_DEV void load_scores(uint32_t taddr, float (&v)[NQ]) {
  uint32_t raw[NQ];
#pragma unroll
  for (int c = 0; c + 8 <= NQ; c += 8) tmem_ld_16x2_8<NQ>(taddr + c, raw + c);
  if constexpr (NQ % 8) tmem_ld_16x2_4<NQ>(taddr + NQ - 4, raw + NQ - 4);
  tmem_ld_wait();
#pragma unroll
  for (int c = 0; c < NQ; c += 4)
    asm volatile("" : "+r"(raw[c]), "+r"(raw[c + 1]), "+r"(raw[c + 2]), "+r"(raw[c + 3])::"memory");
#pragma unroll
  for (int c = 0; c < NQ; c++) v[c] = __uint_as_float(raw[c]);
}

// Folds N values a thread across the 16 lanes of its half warp, halving the values a lane carries at each
// step instead of repeating every value in every lane (30 shuffles for 32 values instead of 128). Returns
// the first of the fold_left(N) value indexes that this lane ends up with.
constexpr int fold_left(int n) {
  for (int i = 0; i < 4; i++) n = n % 2 == 0 ? n / 2 : n;
  return n;
}
template <int N, int OFF, class Op>
LL_DEV int fold16(float* v, int lane, Op op) {
  if constexpr (OFF == 0) {
    return 0;
  } else if constexpr (N % 2 == 0) {
    const bool up = lane & OFF;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + N / 2], OFF);
      v[i] = op(up ? v[i + N / 2] : v[i], got);
    }
    return (up ? N / 2 : 0) + fold16<N / 2, OFF / 2>(v, lane, op);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], OFF));
    return fold16<N, OFF / 2>(v, lane, op);
  }
}

// The pieces [j, j_end) of sequence b, one after another, that make up a CTA's range of tiles.
struct PagedWalk {
  int left, b, j, n, len;
  LL_DEV void init(const PagedArgs& a, int b0, int j0, int count) {
    left = count;
    b = b0;
    j = j0;
    if (left > 0) set(a);
  }
  LL_DEV void set(const PagedArgs& a) {
    len = paged_len(a, b);
    n = paged_tiles(len);
  }
  LL_DEV int end() const { return min(n, j + left); }
  LL_DEV void next(const PagedArgs& a) {
    left -= end() - j;
    b++;
    j = 0;
    if (left > 0) set(a);
  }
};

template <class T, int NT>
__global__ void __launch_bounds__(kPgThreads, 1) k_paged(const __grid_constant__ PagedTma tm, const PagedArgs a) {
  constexpr int NQ = NT / 4;             // query rows of a softmax thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int nchunk = a.nchunk, group_bytes = nchunk * 1024, tile_bytes = 8 * group_bytes;
  uint8_t* s_kv = base;                               // two tiles
  uint8_t* s_q = s_kv + 2 * tile_bytes;               // [chunk][NT rows][128 bytes]
  uint8_t* s_p = s_q + nchunk * NT * 128;             // [64 keys][128 bytes]: P^T, rows of NT values
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_p + kPgKeys * 128);
  uint64_t *kv_full = bars, *kv_empty = bars + 2, *s_full = bars + 6, *q_full = bars + 8, *q_empty = bars + 9,
           *p_ready = bars + 10, *o_done = bars + 11, *o_free = bars + 12, *drain = bars + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_start = reinterpret_cast<int*>(tmem_slot + 2);        // first sequence, first tile of it, tiles before, after
  float* s_red = reinterpret_cast<float*>(tmem_slot + 8);              // [4 warps][64]
  float* s_col = s_red + 256;                                          // [64] a factor per row
  float* s_ref = s_col + 64;                                           // [64] the rows' references
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = blockIdx.x / a.RT, rt = blockIdx.x % a.RT;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 14; i++) mbar_init(&bars[i], i == 10 || i == 12 ? kPgSoft / 32 : 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm.q);
    tma_prefetch_desc(&tm.kv);
  }
  pdl_wait();
  if (warp == 0) {
    // the range of this CTA: each lane sums a run of consecutive sequences
    const int run = (a.B + 31) / 32, b_lo = min(lane * run, a.B), b_hi = min(b_lo + run, a.B);
    int mine = 0;
#pragma unroll 4
    for (int b = b_lo; b < b_hi; b++) mine += paged_weight(paged_len(a, b));
    int sum = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += v;
    }
    const int total = __shfl_sync(0xffffffffu, sum, 31), per = (total + a.G - 1) / a.G;
    const int first = min((int64_t)g * per, (int64_t)total), last = min((int64_t)first + per, (int64_t)total);
    if (lane == 0) {
      s_start[2] = s_start[3] = total - kPgStart * a.B;      // tiles before `first`, before `last`
      if (blockIdx.x == 0) a.starts[a.B] = per;
    }
    __syncwarp();
    int at = sum - mine;
    if (blockIdx.x == 0 || (first < sum && last >= at))
      for (int b = b_lo; b < b_hi; b++) {
        const int n = paged_tiles(paged_len(a, b)), before = at - kPgStart * b, end = at + n + kPgStart;
        if (blockIdx.x == 0) {
          a.starts[b] = at;
          if (a.lens[b] < 0 || a.lens[b] > paged_room(a)) report(a.st, LL_ERR_RANGE, 74, b);
        }
        if (first >= at && first < end) {
          s_start[0] = b;
          s_start[1] = max(0, first - at - kPgStart);
          s_start[2] = before + s_start[1];
        }
        if (last >= at && last < end) s_start[3] = before + max(0, last - at - kPgStart);
        at = end;
      }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_next();
  const uint32_t tmem = *tmem_slot, tmem_s = tmem + 256;
  const int count = s_start[3] - s_start[2];
  PagedWalk w;
  w.init(a, s_start[0], s_start[1], count);

  if (warp == 8) {
    // ------------------------------------------------------------------------------- TMA
    // Lane i takes the tile's group i of eight keys: it looks its page up while the stage is still in
    // use, then issues its own box.
    bool ok = true;
    uint32_t n = 0, seg = 0, q_loads = 0;
    for (; w.left > 0 && ok; w.next(a), seg++) {
      const int j0 = w.j, j1 = w.end();
      for (int j = j0; j < j1; j++, n++) {
        const int st = n & 1, key = j * kPgKeys + lane * 8;
        const int groups = (min(kPgKeys, max(0, w.len - j * kPgKeys)) + 7) / 8;
        int page = a.pages;                       // outside the map: reads zeros
        if (lane < groups) {
          const int at = key / a.page_size, id = a.bt[w.b * a.bt_stride + at];
          if (id >= 0 && id < a.pages) page = id;
          else report(a.st, LL_ERR_RANGE, 73, w.b);
        }
        const int off = key % a.page_size;
        // the second product releases a stage by halves, so the first four groups go ahead
        if (!(ok = warp_wait(&kv_empty[st * 2], ((n >> 1) & 1) ^ 1, abort_flag, a.st, 81))) break;
        if (lane == 0) mbar_expect_tx(&kv_full[st], min(groups, 4) * group_bytes);
        __syncwarp();
        uint8_t* dst = s_kv + st * tile_bytes + lane * group_bytes;
        if (lane < min(groups, 4)) tma_load_4d(dst, &tm.kv, &kv_full[st], 0, off, 0, page);
        ok = warp_wait(&kv_empty[st * 2 + 1], ((n >> 1) & 1) ^ 1, abort_flag, a.st, 82);
        if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], ok ? max(groups - 4, 0) * group_bytes : 0);
        __syncwarp();
        if (!ok) { n++; break; }
        if (lane >= 4 && lane < groups) tma_load_4d(dst, &tm.kv, &kv_full[st], 0, off, 0, page);
        if (j == j0) {
          if (lane == 0) {
            ok = mbar_wait(q_empty, (seg & 1) ^ 1, abort_flag, a.st, 80);
            if (ok) mbar_arrive_expect_tx(q_full, nchunk * NT * 128);
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) { n++; break; }
          q_loads++;
          if (lane < nchunk) tma_load_3d(s_q + lane * NT * 128, &tm.q, q_full, lane * 64, rt * NT, w.b);
        }
      }
    }
    volatile int keep = 0;                        // what was issued has landed, also after an abort
    if (n >= 1) mbar_wait_sleep(&kv_full[(n - 1) & 1], ((n - 1) >> 1) & 1, &keep, a.st, 83, 64);
    if (n >= 2) mbar_wait_sleep(&kv_full[n & 1], ((n - 2) >> 1) & 1, &keep, a.st, 84, 64);
    if (q_loads >= 1) mbar_wait_sleep(q_full, (q_loads - 1) & 1, &keep, a.st, 85, 64);
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------- MMA
    // The whole warp runs the loop (so that descriptors stay in uniform registers), one elected lane issues.
    // Strictly S^T(n), then tile n's second product: issuing S^T(n + 1) in between would hold up the release
    // of the stage that tile n + 2 lands in, and the loads are what bounds the loop (measured 5 % slower).
    const bool lead = elect_one();
    const uint32_t id_s = idesc_16bit(Num<T>::fmt, 64, NT, false, false);
    const uint32_t id_o = idesc_16bit(Num<T>::fmt, 128, NT, true, true);
    const MmaDesc q_d(smem_u32(s_q), 16, 1024), p_d(smem_u32(s_p), 1024, 1024);
    const MmaDesc k_d(smem_u32(s_kv), 16, group_bytes), v_d(smem_u32(s_kv), 1024, group_bytes);
    const uint32_t tile16 = tile_bytes >> 4, group16 = group_bytes >> 4;
    const int mts = a.nc / 2;
    uint32_t n = 0, piece = 0;
    bool ok = true;
    for (; w.left > 0 && ok; w.next(a), piece++) {
      const int j0 = w.j, j1 = w.end();
#pragma unroll 1
      for (int j = j0; j < j1; j++, n++) {
        const bool first = j == j0;
        if (!(ok = warp_wait(&kv_full[n & 1], (n >> 1) & 1, abort_flag, a.st, 86))) break;
        if (first && !(ok = warp_wait(q_full, piece & 1, abort_flag, a.st, 87))) break;
        tc_fence_after();
        const uint32_t at = tmem_s + (n & 1) * 64, k0 = k_d.lo + (n & 1) * tile16, v0 = v_d.lo + (n & 1) * tile16;
        if (lead) {
          for (int c = 0; c < nchunk; c++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              mma_16bit(at, k0 + c * 64 + kk * 2, k_d.hi, q_d.lo + c * (NT * 8) + kk * 2, q_d.hi, id_s, c + kk);
          mma_commit(&s_full[n & 1]);
          if (j == j1 - 1) mma_commit(q_empty);
        }
        if (!(ok = warp_wait(p_ready, n & 1, abort_flag, a.st, 88))) break;
        if (first && piece > 0 && !(ok = warp_wait(o_free, (piece - 1) & 1, abort_flag, a.st, 89))) break;
        tc_fence_after();
        if (lead) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
#pragma unroll
            for (int kk = half * 2; kk < half * 2 + 2; kk++)
#pragma unroll
              for (int mt = 0; mt < 4; mt++)
                if (mt < mts)
                  mma_16bit(tmem + mt * NT, v0 + kk * 2 * group16 + mt * 128, v_d.hi, p_d.lo + kk * 128, p_d.hi, id_o,
                            first && kk == 0 ? 0 : 1);
            mma_commit(&kv_empty[(n & 1) * 2 + half]);
          }
          if (j == j1 - 1) mma_commit(o_done);
        }
      }
    }
    __syncwarp();
    if (lead) mma_commit(drain);
    volatile int keep = 0;
    mbar_wait_sleep(drain, 0, &keep, a.st, 90, 64);
    __syncwarp();
  } else {
    // ------------------------------------------------- softmax, rescaling and the outputs
    // A wait that ran out does not leave the loops: the other waits then return at once, every
    // barrier still meets all 256 threads, and the results are void (the status says so).
    const int quarter = warp % 4, side = warp / 4, key_in = quarter * 16 + lane % 16;
    const int r0 = (side * 2 + lane / 16) * NQ;          // the thread's first query row in the tile
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int t0 = (rt * NT + r0) / a.H, h0 = (rt * NT + r0) % a.H;
    uint8_t* p_row = s_p + (key_in / 8) * 1024 + (key_in % 8) * 128;
    uint32_t n = 0, piece = 0;
    for (; w.left > 0; w.next(a)) {
      const int j0 = w.j, j1 = w.end();
      float ref[NQ], l[NQ];
#pragma unroll
      for (int c = 0; c < NQ; c++) { ref[c] = kPgNone; l[c] = 0.f; }
      if (threadIdx.x < NT) s_ref[threadIdx.x] = kPgNone;
      for (int j = j0; j < j1; j++, n++) {
        mbar_wait(&s_full[n & 1], (n >> 1) & 1, abort_flag, a.st, 91);
        tc_fence_after();
        const uint32_t s_at = tmem_s + (n & 1) * 64 + side * 2 * NQ + lanes;
        const int k0 = j * kPgKeys, key = k0 + key_in;
        const bool inside = k0 + kPgKeys <= w.len - a.Tq + 1;       // every row sees every key
        // hides the keys past each row's last one (row (t, h) sees w.len - Tq + 1 + t of them)
        auto mask = [&](float (&x)[NQ]) {
          int h = h0, see = w.len - a.Tq + 1 + t0;
#pragma unroll
          for (int c = 0; c < NQ; c++) {
            if (key >= see) x[c] = -INFINITY;
            if (++h == a.H) { h = 0; see++; }
          }
        };
        float v[NQ];
        load_scores<NQ>(s_at, v);
#pragma unroll
        for (int c = 0; c < NQ; c++) v[c] = fmaf(v[c], a.scale_log2, -ref[c]);
        if (!inside) mask(v);
        float top = v[0];
#pragma unroll
        for (int c = 1; c < NQ; c++) top = fmaxf(top, v[c]);
        const bool slow = bar_any<kPgSoft>(1, top > kPgSlack);
        if (slow) {
          // new references: each row's maximum so far
          load_scores<NQ>(s_at, v);
#pragma unroll
          for (int c = 0; c < NQ; c++) v[c] *= a.scale_log2;
          if (!inside) mask(v);
          float x[NQ];
#pragma unroll
          for (int c = 0; c < NQ; c++) x[c] = v[c];
          const int c0 = r0 + fold16<NQ, 8>(x, lane, [](float p, float q) { return fmaxf(p, q); });
#pragma unroll
          for (int c = 0; c < fold_left(NQ); c++) s_red[quarter * 64 + c0 + c] = x[c];
          named_bar_sync(1, kPgSoft);
          if (threadIdx.x < NT) {
            const int r = threadIdx.x;
            const float was = s_ref[r];
            const float now = fmaxf(fmaxf(fmaxf(s_red[r], s_red[64 + r]), fmaxf(s_red[128 + r], s_red[192 + r])), was);
            s_ref[r] = now;
            s_col[r] = ex2(was - now);
          }
          named_bar_sync(1, kPgSoft);
#pragma unroll
          for (int c = 0; c < NQ; c++) {
            ref[c] = s_ref[r0 + c];
            v[c] -= ref[c];
            l[c] *= s_col[r0 + c];
          }
        }
#pragma unroll
        for (int c = 0; c < NQ; c++) {
          v[c] = ex2(v[c]);
          l[c] += v[c];
        }
        // (S^T(n) was issued after tile n - 1's second product: P and O are free)
        if (slow && j > j0) {
          tc_fence_after();
          for (int i = side; i < a.nc / 2 * (NT / 16); i += 2) {
            const int c = i % (NT / 16) * 16;
            const uint32_t at = tmem + i / (NT / 16) * NT + c + lanes;
            float o[16];
            tmem_ld16(at, o);
            tmem_ld_wait();
            uint32_t u[16];
#pragma unroll
            for (int k = 0; k < 16; k++) u[k] = __float_as_uint(o[k] * s_col[c + k]);
            tmem_st16(at, u);
          }
          tmem_st_wait();
        }
#pragma unroll
        for (int c = 0; c < NQ; c += 4) {
          const int chunk = (r0 + c) / 8, half = (r0 + c) / 4 % 2;
          *reinterpret_cast<uint2*>(p_row + ((chunk ^ (key_in % 8)) * 16) + half * 8) =
              make_uint2(Num<T>::pack(v[c], v[c + 1]), Num<T>::pack(v[c + 2], v[c + 3]));
        }
        const int valid = w.len - k0;
        if (valid < kPgKeys) {
          const int from = max(valid, 0), per_row = a.nc * 8;
          for (int i = threadIdx.x; i < (kPgKeys - from) * per_row; i += kPgSoft) {
            const int r = from + i / per_row, c = i % per_row;
            *reinterpret_cast<uint4*>(s_kv + (n & 1) * tile_bytes + (r / 8) * group_bytes + (c / 8) * 1024 + (r % 8) * 128 +
                                      (c % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
      }
      // the piece's sums over its keys, in a fixed order
      const int c0 = r0 + fold16<NQ, 8>(l, lane, [](float p, float q) { return p + q; });
#pragma unroll
      for (int c = 0; c < fold_left(NQ); c++) s_red[quarter * 64 + c0 + c] = l[c];
      named_bar_sync(1, kPgSoft);
      const bool whole = j0 == 0 && j1 == w.n;
      const int64_t slot = ((int64_t)g * 2 + (n == (uint32_t)(j1 - j0) ? 0 : 1)) * a.RT + rt;
      if (threadIdx.x < NT) {
        const int r = threadIdx.x, row = rt * NT + r;
        const float sum = (s_red[r] + s_red[64 + r]) + (s_red[128 + r] + s_red[192 + r]);
        const bool any = !(sum <= 0.f);
        s_col[r] = any ? 1.f / sum : 0.f;
        if (!whole) {
          a.part_ml[slot * 2 * NT + r] = s_ref[r];
          a.part_ml[slot * 2 * NT + NT + r] = sum;
        } else if (row < a.rows) {
          a.lse[(int64_t)w.b * a.rows + row] = any ? (s_ref[r] + log2f(sum)) * 0.693147180559945309f : -INFINITY;
        }
      }
      named_bar_sync(1, kPgSoft);
      mbar_wait(o_done, piece & 1, abort_flag, a.st, 93);
      piece++;
      tc_fence_after();
      const int d_c = a.nc * 64;
      for (int j = side; j < a.nc / 2 * (NT / 16); j += 2) {
          const int mt = j / (NT / 16), c = j % (NT / 16) * 16;
          float o[16];
          tmem_ld16(tmem + mt * NT + c + lanes, o);
          tmem_ld_wait();
          const int d = mt * 128 + quarter * 32 + lane;
          if (!whole) {
            float* dst = a.part + (slot * NT + c) * d_c + d;
#pragma unroll
            for (int i = 0; i < 16; i++) dst[(int64_t)i * d_c] = o[i];
          } else {
            // neighbouring lanes trade values, so that each writes two adjacent ones of one row
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float x = o[i] * s_col[c + i], y = o[i + 1] * s_col[c + i + 1];
              const float z = __shfl_xor_sync(0xffffffffu, lane & 1 ? x : y, 1);
              const int row = rt * NT + c + i + (lane & 1);
              const uint32_t two = lane & 1 ? Num<T>::pack(z, y) : Num<T>::pack(x, z);
              if (row < a.rows)
                *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + ((int64_t)w.b * a.rows + row) * d_c + (d & ~1)) = two;
            }
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// Joins a split sequence's pieces: out = sum_g 2^(m_g - M) O_g / sum_g 2^(m_g - M) l_g with the running
// maximum M. A block takes ROWS query rows, a thread four values of each; rows of whole sequences are left
// alone. Bound by its two dependent rounds of loads (the sequence's range, its pieces), so the second one
// has many in flight: with few pieces a sequence ROWS = 4 and two pieces at a time; with many (few long
// sequences) one row, whose pieces GRP = 4 groups of threads take in turn, four at a time, and join in
// order (37 pieces: 25 us with one group, 6 with four).
template <class T, int GRP, int ROWS>
__global__ void __launch_bounds__(128 * GRP) k_paged_combine(const PagedArgs a, int NT) {
  constexpr int PC = GRP > 1 ? 4 : 2;
  __shared__ float4 s_o[GRP][128];
  __shared__ float2 s_ml[GRP];
  const int blocks = (a.rows + ROWS - 1) / ROWS;             // a sequence's
  const int b = blockIdx.x / blocks, row0 = blockIdx.x % blocks * ROWS, rt = row0 / NT, r0 = row0 % NT;
  const int grp = threadIdx.x / 128, t = threadIdx.x % 128;
  pdl_wait();
  const int before = a.starts[b], per = a.starts[a.B];
  const int tile0 = before + kPgStart, last = tile0 + paged_tiles(paged_len(a, b)) - 1;
  const int g0 = tile0 / per, n = last / per - g0 + 1;
  if (n == 1) return;
  const int d_c = a.nc * 64, d = min(t * 4, d_c - 4);
  float M[ROWS], L[ROWS];
  float4 o[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; k++) {
    M[k] = kPgNone;
    L[k] = 0.f;
    o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  auto join = [&](int k, float m, float l, float4 x) {
    const float now = fmaxf(M[k], m), f = ex2(M[k] - now), w = ex2(m - now);
    M[k] = now;
    L[k] = L[k] * f + w * l;
    o[k].x = o[k].x * f + w * x.x;
    o[k].y = o[k].y * f + w * x.y;
    o[k].z = o[k].z * f + w * x.z;
    o[k].w = o[k].w * f + w * x.w;
  };
  for (int i0 = grp; i0 < n; i0 += PC * GRP) {
    float m[PC][ROWS], l[PC][ROWS];
    float4 x[PC][ROWS];
#pragma unroll
    for (int i = 0; i < PC; i++) {
      // a CTA's first piece is in its slot 0, its last (when another) in slot 1; a row tile has NT rows,
      // so rows past the sequence's last are there to be read
      const int g = g0 + min(i0 + i * GRP, n - 1);
      const int64_t sl = ((int64_t)g * 2 + (before > g * per ? 1 : 0)) * a.RT + rt;
#pragma unroll
      for (int k = 0; k < ROWS; k++) {
        m[i][k] = a.part_ml[sl * 2 * NT + r0 + k];
        l[i][k] = a.part_ml[sl * 2 * NT + NT + r0 + k];
        x[i][k] = *reinterpret_cast<const float4*>(a.part + (sl * NT + r0 + k) * d_c + d);
      }
    }
#pragma unroll
    for (int i = 0; i < PC; i++)
      if (i0 + i * GRP < n)
#pragma unroll
        for (int k = 0; k < ROWS; k++) join(k, m[i][k], l[i][k], x[i][k]);
  }
  if constexpr (GRP > 1) {
    s_o[grp][t] = o[0];
    if (t == 0) s_ml[grp] = make_float2(M[0], L[0]);
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int i = 1; i < GRP; i++) join(0, s_ml[i].x, s_ml[i].y, s_o[i][t]);
  }
#pragma unroll
  for (int k = 0; k < ROWS; k++) {
    if (row0 + k >= a.rows) break;
    const bool any = !(L[k] <= 0.f);
    const float inv = any ? 1.f / L[k] : 0.f;
    const int64_t at = (int64_t)b * a.rows + row0 + k;
    if (t * 4 < d_c)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * d_c + d) =
          make_uint2(Num<T>::pack(o[k].x * inv, o[k].y * inv), Num<T>::pack(o[k].z * inv, o[k].w * inv));
    if (t == 0) a.lse[at] = any ? (M[k] + log2f(L[k])) * 0.693147180559945309f : -INFINITY;
  }
}

// Row tiles of a sequence, their height (a multiple of 16, the tiles' rows nearly equal) and the
// number of ranges the key tiles are dealt into, so that about every SM has one CTA. The number is a whole
// one: 51 to 73 row tiles fill 102 to 146 of 148 SMs, but 75 (4801 query rows a sequence) to 100 are not split
// and fill 75 to 100 (75 tokens of 64 heads against 3000 keys: 97 us).
struct PagedPlan {
  int RT, NT, G;
  size_t part, ml;        // workspace floats
};
static PagedPlan paged_plan(int Tq, int H, int d_c) {
  PagedPlan p;
  const int rows = Tq * H, sms = device_info().sms > 0 ? device_info().sms : 148;
  p.RT = (rows + 63) / 64;
  p.NT = ((rows + p.RT - 1) / p.RT + 15) / 16 * 16;
  p.G = std::max(1, sms / p.RT);
  p.part = p.G > 1 ? (size_t)p.G * 2 * p.RT * p.NT * d_c : 0;
  p.ml = p.G > 1 ? (size_t)p.G * 2 * p.RT * 2 * p.NT : 0;
  return p;
}

template <class T, int NT>
static int launch_paged(const PagedTma& tm, const PagedArgs& a, int smem, cudaStream_t s) {
  LL_TRY(set_smem_attr(reinterpret_cast<const void*>(k_paged<T, NT>), smem));
  return launch_pdl("k_paged", k_paged<T, NT>, dim3(a.G * a.RT), dim3(kPgThreads), smem, s, tm, a);
}

template <class T>
static int run_paged(const PagedTma& tm, const PagedArgs& a, int NT, cudaStream_t s) {
  const int smem = 1024 + 2 * a.nchunk * 8192 + a.nchunk * NT * 128 + kPgKeys * 128 + 144 + 4 * 384;
  if (NT == 16) LL_TRY((launch_paged<T, 16>(tm, a, smem, s)));
  else if (NT == 32) LL_TRY((launch_paged<T, 32>(tm, a, smem, s)));
  else if (NT == 48) LL_TRY((launch_paged<T, 48>(tm, a, smem, s)));
  else LL_TRY((launch_paged<T, 64>(tm, a, smem, s)));
  if (a.G == 1) return LL_OK;
  // Four groups a row from about eight pieces a sequence on. Whole calls with four groups and with one, B
  // sequences of 3000 keys at 64 heads: B = 8 21 and 29 us, 16 30.1 and 30.5, 24 39 and 34.5, 48 69 and 50.
  // The host knows the mean alone: one sequence of 70 thousand keys among 23 of at most 500 is cut into some
  // 120 pieces and takes 107 us by this rule, 42 with four groups.
  if (a.G > 8 * a.B)
    return launch_pdl("k_paged_combine", k_paged_combine<T, 4, 1>, dim3((unsigned)a.B * a.rows), dim3(512), 0, s, a, NT);
  return launch_pdl("k_paged_combine", k_paged_combine<T, 1, 4>, dim3((unsigned)a.B * ((a.rows + 3) / 4)), dim3(128), 0,
                    s, a, NT);
}

}  // namespace ll

using namespace ll;

extern "C" {

size_t ll_paged_latent_workspace_bytes(int B, int Tq, int H, int d_c) {
  if (B <= 0 || Tq <= 0 || H <= 0 || d_c <= 0 || (int64_t)Tq * H > (1 << 24)) return 0;
  const PagedPlan p = paged_plan(Tq, H, d_c);
  return (p.part + p.ml) * 4 + ((size_t)B + 1) * 8 + 1024;
}

int ll_paged_latent_attention(const void* q, int64_t q_stride_b, int64_t q_stride_row, const void* cache,
                              int64_t page_stride, int64_t row_stride, int pages, int page_size,
                              const int32_t* block_table, int64_t table_stride, int max_pages, const int32_t* seq_lens,
                              int B, int Tq, int H, int d_c, int d_r, float scale, int dtype, void* out, float* lse,
                              void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || Tq <= 0 || H <= 0 || d_c <= 0 || d_c % 128 || d_c > 512 || (d_r != 0 && d_r != 64) ||
      (dtype != 1 && dtype != 2) || pages <= 0 || page_size <= 0 || page_size % 8 || max_pages <= 0 || !(scale > 0.f))
    return LL_ERR_ARG;
  if ((int64_t)Tq * H > (1 << 24) || (int64_t)B * Tq * H > INT32_MAX || (int64_t)max_pages * page_size > INT32_MAX - 64 ||
      (int64_t)B * ((int64_t)max_pages * page_size / kPgKeys + 1 + kPgStart) > INT32_MAX)
    return LL_ERR_ARG;
  if (B == 0) return LL_OK;
  const int D = d_c + d_r;
  if (!q || !cache || !block_table || !seq_lens || !out || !lse || !workspace) return LL_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(workspace)) & 15)
    return LL_ERR_ARG;
  if (q_stride_b % 8 || q_stride_row % 8 || q_stride_b <= 0 || q_stride_row <= 0 || page_stride % 8 || row_stride % 8 ||
      row_stride < D || (pages > 1 && page_stride < D) || page_stride <= 0 || table_stride < 0)
    return LL_ERR_ARG;
  if (workspace_bytes < ll_paged_latent_workspace_bytes(B, Tq, H, d_c)) return LL_ERR_WORKSPACE;
  LL_TRY(check_arch());
  LL_STREAM(stream);
  g_launch_count = 0;
  const PagedPlan p = paged_plan(Tq, H, d_c);
  PagedArgs a{};
  a.bt = block_table;
  a.lens = seq_lens;
  a.out = out;
  a.lse = lse;
  Carver cv(workspace);
  a.part = cv.take<float>(p.part);
  a.part_ml = cv.take<float>(p.ml);
  a.starts = cv.take<int>((size_t)B + 1);
  a.bt_stride = table_stride;
  a.pages = pages;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.B = B;
  a.Tq = Tq;
  a.H = H;
  a.rows = Tq * H;
  a.RT = p.RT;
  a.G = p.G;
  a.nc = d_c / 64;
  a.nchunk = D / 64;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.st = latent_status();
  if (!a.st) return LL_ERR_CUDA;
  PagedTma tm;
  const CUtensorMapDataType dt = dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t qd[3] = {(uint64_t)D, (uint64_t)a.rows, (uint64_t)B};
  const uint64_t qs[2] = {(uint64_t)q_stride_row * 2, (uint64_t)q_stride_b * 2};
  const uint32_t qb[3] = {64, (uint32_t)p.NT, 1};
  LL_TRY(make_map_nd(&tm.q, dt, q, 3, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B));
  const uint64_t kd[4] = {64, (uint64_t)page_size, (uint64_t)a.nchunk, (uint64_t)pages};
  const uint64_t ks[3] = {(uint64_t)row_stride * 2, 128, (uint64_t)page_stride * 2};
  const uint32_t kb[4] = {64, 8, (uint32_t)a.nchunk, 1};
  LL_TRY(make_map_nd(&tm.kv, dt, cache, 4, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B));
  return dtype == 1 ? run_paged<__nv_bfloat16>(tm, a, p.NT, s) : run_paged<__half>(tm, a, p.NT, s);
}

}  // extern "C"

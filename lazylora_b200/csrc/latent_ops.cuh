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
  static constexpr bool narrow = false;  // a range short of fp32's
  LL_DEV static float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  LL_DEV static uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <>
struct Num<__half> {
  static constexpr uint32_t fmt = 0;
  static constexpr bool narrow = true;
  LL_DEV static float to_f(__half v) { return __half2float(v); }
  LL_DEV static uint32_t pack(float lo, float hi) {
    const __half2 p = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// kind::f16 instruction descriptor: operands of format fmt (0 fp16, 1 bf16), fp32 accumulation.
LL_DEV uint32_t idesc_16bit(uint32_t fmt, uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
  return 1u << 4 | fmt << 7 | fmt << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 | (n >> 3) << 17 | (m >> 4) << 24;
}

// One lane of a converged warp.
LL_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// A bounded wait of a whole warp with one outcome: lanes that left a loop apart after a timeout would meet
// the others' warp-wide instructions no more.
LL_DEV bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, DevStatus* st, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, st, where));
}
LL_DEV bool warp_wait_sleep(uint64_t* bar, uint32_t parity, volatile int* abort_flag, DevStatus* st, int where,
                            uint32_t ns_max) {
  return __all_sync(0xffffffffu, mbar_wait_sleep(bar, parity, abort_flag, st, where, ns_max));
}

// Barrier `id` of N threads, with a vote: whether p holds for any of them.
template <int N>
LL_DEV bool bar_any(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)p), "r"(id), "n"(N)
      : "memory");
  return r != 0;
}

// More bytes for the current phase to wait for, without arriving.
LL_DEV void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// A shared-memory operand descriptor (128-byte swizzle) as its two words: steps along the operand are
// additions to lo, in units of 16 bytes (shared addresses stay below 2^18, so the field never carries).
struct MmaDesc {
  uint32_t lo, hi;
  LL_DEV MmaDesc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    const uint64_t d = umma_desc(addr, lbo, sbo, kSwizzle128B);
    lo = (uint32_t)d;
    hi = (uint32_t)(d >> 32);
  }
};

// D[tmem] (+)= A B, kind::f16, both operands in shared memory.
LL_DEV void mma_16bit(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                      uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in tensor memory.
LL_DEV void mma_16bit_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 32 consecutive columns; thread i gets lane (base lane + i). Valid after tcgen05.wait::ld.
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

// Writes 128 bytes of each of a warp's 32 rows (lane = row, w its 32 words) through 4 KB of shared memory, so
// that eight lanes write a row's 128 bytes at once: rows apart by a token's stride, written 16 bytes a row
// and instruction, took 4000 cycles a 128 x 128 tile. rows: how many of the 32 exist; stride in bytes.
LL_DEV void store_rows(uint8_t* stage, const uint32_t* w, int lane, int rows, uint8_t* dst, int64_t stride) {
#pragma unroll
  for (int c = 0; c < 8; c++)
    *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) * 16)) =
        make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int r = i * 4 + lane / 8, c = lane % 8;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) * 16));
    if (r < rows) *reinterpret_cast<uint4*>(dst + r * stride + c * 16) = v;
  }
  __syncwarp();
}
// Two fp32 operations an instruction.
LL_DEV float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
LL_DEV float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
LL_DEV float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}

// 2^x (ex2.approx: 2 ulp, results below the normal range to zero).
LL_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows of sequence b in a packed tensor of `total` rows: [lo, hi), clamped into the tensor so that
// no value of cu can lead outside it.
LL_DEV void seq_range(const int32_t* cu, int b, int total, int& lo, int& hi) {
  lo = min(max(cu[b], 0), total);
  hi = min(max(cu[b + 1], lo), total);
}

// Records cumulative lengths that do not start at 0, rise and end at the tensor's rows (a warp).
LL_DEV void check_cu(const int32_t* cu, int B, int total, DevStatus* st, int where) {
  for (int b = threadIdx.x & 31; b <= B; b += 32) {
    const int at = cu[b];
    if ((b == 0 && at != 0) || (b < B ? cu[b + 1] < at : at != total)) report(st, LL_ERR_RANGE, where, b);
  }
}

// The tile-th tile of `rows` rows over all sequences, counted from the first or (FROM_END) from the last
// one, for a whole warp: true and (b, first row within the sequence) when there is one. Lanes scan 32
// sequences at a time. The causal kernels count from the side on which a sequence's tiles are longest, so
// that the short ones fill the launch's tail.
template <bool FROM_END>
LL_DEV bool find_tile(const int32_t* cu, int B, int total, int rows, int tile, int& b, int& row0) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int bb = FROM_END ? B - 1 - b0 - lane : b0 + lane;
    int n = 0;
    if (bb >= 0 && bb < B) {
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
      const int src = __ffs(__ballot_sync(0xffffffffu, tile < sum)) - 1;
      const int end = __shfl_sync(0xffffffffu, sum, src), cnt = __shfl_sync(0xffffffffu, n, src);
      const int at = tile - (end - cnt);
      b = __shfl_sync(0xffffffffu, bb, src);
      row0 = (FROM_END ? cnt - 1 - at : at) * rows;
      return true;
    }
    tile -= all;
  }
  return false;
}

}  // namespace ll

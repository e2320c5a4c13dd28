// The 4-bit KV pool: its row layout, the store that quantises and scatters new
// k/v rows, and the load that reads rows back as plain values.
//
// Format. A head row of D features is cut into blocks of 16. A block keeps one
// e4m3 scale s = rne_e4m3(min(max|x| / 6, 448)) and sixteen e2m1 codes
// rne_e2m1(x / s), clipped to +-6: a value is code * s, 4.5 bits per feature.
// The pool holds finite values only: a NaN is stored as 0 and does not count
// for the maximum, an infinity is clipped to the block's largest value
// (6 * 448). code * s has at most 2 + 4 significant bits and an exponent in
// [-10, 11], so it is exact in fp16 and in bf16, and attention over the pool
// multiplies exactly what load returns.
//
// Exactness of the codes: x, max|x| and s are floats, and a border between two
// codes (or two scales) times s (times 6) has at most 7 significant bits, so a
// quotient on a border is exact and one that is not keeps its side when it is
// rounded to fp32. Codes are therefore those of the exact quotient, and any
// correct implementation agrees bit for bit.
//
// Row of one token slot (fp4_row_bytes, a multiple of 16):
//   [K codes D/2 | V codes D/2] for each kv head, then
//   [K scales D/16 | V scales D/16] for each kv head, then padding.
// Feature 2i of a row sits in the low nibble of byte i. All heads of a token
// are one run, a page is one run of page_size rows: one bulk copy brings K and
// V, codes and scales. A row that would be a multiple of 128 bytes gets 16 more
// (8 heads x 128: 1168 instead of 1152, +1.4% traffic): consumers read the
// same offset of several rows at once, and with a pitch of 128 k bytes these
// fall into the same shared-memory banks (8-way conflicts).
#pragma once

#include "common.cuh"
#include "slot.cuh"

namespace b2a {

constexpr int kFp4Block = 16;  // features per scale

__host__ __device__ inline uint32_t fp4_row_bytes(int Hkv, int D) {
  uint32_t r = (uint32_t)Hkv * (uint32_t)(D + D / 8);
  r = (r + 15u) & ~15u;
  if (r % 128u == 0) r += 16u;
  return r;
}
// Offsets inside a token row: codes of K (V follows after D/2), scales of K (V after D/16).
__host__ __device__ __forceinline__ uint32_t fp4_code_off(int h, int D) { return (uint32_t)(h * D); }
__host__ __device__ __forceinline__ uint32_t fp4_scale_off(int h, int Hkv, int D) {
  return (uint32_t)(Hkv * D + h * (D / 8));
}

// Eight codes (one word) -> four fp16 pairs, in order. Exact.
__device__ __forceinline__ void fp4_word_to_h2(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}

// Two e4m3 scales (low byte first) -> an fp16 pair. Exact.
__device__ __forceinline__ uint32_t fp4_scale2_to_h2(uint32_t two_bytes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two_bytes));
  return r;
}

__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// float -> e4m3 byte, to nearest even, clipped to 448 (x >= 0, not NaN).
__device__ __forceinline__ uint32_t f_to_e4m3(float x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return r & 0xffu;
}

// Two floats -> a byte of two e2m1 codes (lo in the low nibble), nearest even, clipped to +-6.
__device__ __forceinline__ uint32_t f2_to_e2m1(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0;\n\t.reg .b16 h;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %1, %2;\n\t"
      "mov.b16 h, {b0, 0};\n\t"
      "cvt.u32.u16 %0, h;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

struct Fp4KvArgs {
  const void* k;  // store: new rows
  const void* v;
  void* k_out;  // load: destinations [n, Hkv, D]
  void* v_out;
  int64_t k_stride, v_stride;  // elements between token rows (store)
  const int32_t* slots;
  uint8_t* pool;
  int64_t num_slots;
  int64_t n;  // token rows
  int Hkv;
  int nblk;  // blocks of a head row: D / 16
  uint32_t row_bytes;
  float k_scale, v_scale;  // powers of two: a stored value stands for code * s * scale
};

template <typename T>
__device__ __forceinline__ void fp4_read16(const T* p, bool vec, float (&x)[16]) {
  if (vec) {
    load_vec<T, 16>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = DT<T>::to_f(p[i]);
  }
}

// Threads take blocks of 16 features, neighbours neighbouring blocks, so reads and writes are
// contiguous over a token's heads. HBM bounds both kernels at large n: a thread takes kFp4Unroll
// blocks kFp4Threads apart, so that many independent slot -> row reads are in flight, and one
// 64-bit division per thread finds the first token. Store and load of 16,391 fp32 tokens of
// 8 x 128 take 71.5 us (a block and a division per thread: 77), the load of 120,001 bf16 ones
// 127 us, 5.0 TB/s (149).
constexpr int kFp4Threads = 256;
constexpr int kFp4Unroll = 4;

struct Fp4Where {
  int64_t t;        // token row of the call
  int64_t slot;     // pool slot, -1 outside the pool
  int kind, h, blk; // 0 k / 1 v, kv head, unit of the head row
  bool have;
};

// The units of this thread, npr of them in a head row; `slots` reads go out together. STORE: a
// slot of -1 is a row without one, skipped; any other slot outside the pool is recorded.
template <bool STORE>
__device__ __forceinline__ void fp4_where(const Fp4KvArgs& a, int npr, Fp4Where (&w)[kFp4Unroll]) {
  const uint32_t half = (uint32_t)(a.Hkv * npr), per_tok = 2u * half;
  const int64_t i0 = (int64_t)blockIdx.x * (kFp4Threads * kFp4Unroll);
  const int64_t t0 = i0 / per_tok;
  const uint32_t r0 = (uint32_t)(i0 - t0 * per_tok) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kFp4Unroll; ++u) {
    const uint32_t r = r0 + u * kFp4Threads, dt = r / per_tok;
    uint32_t e = r - dt * per_tok;
    w[u].t = t0 + dt;
    w[u].kind = e >= half;
    e -= w[u].kind ? half : 0u;
    w[u].h = (int)(e / (uint32_t)npr);
    w[u].blk = (int)(e - (uint32_t)w[u].h * npr);
    w[u].have = w[u].t < a.n;
    w[u].slot = w[u].have ? a.slots[w[u].t] : 0;
  }
#pragma unroll
  for (int u = 0; u < kFp4Unroll; ++u) {
    if (w[u].slot < 0 || w[u].slot >= a.num_slots) {
      if (!STORE || w[u].slot != kNoSlot) watchdog_set(kWdBadSlot);
      w[u].slot = -1;
    }
  }
}

// x / s to nearest for |x| <= 2^13 and an e4m3 s > 0 with y = 1 / s to nearest: Markstein's
// correction of x * y by its remainder ("Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990), three operations instead of a division per element. The
// remainder is exact unless x is so small that the code is zero either way. The remainder of a
// zero is +0 whatever its sign, which x gives back: the code keeps it.
__device__ __forceinline__ float fp4_quotient(float x, float s, float y) {
  const float q = x * y;
  return copysignf(fmaf(fmaf(-q, s, x), y, q), x);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kFp4Threads) fp4_store_kernel(const Fp4KvArgs a) {
  pdl_wait_then_release();
  Fp4Where w[kFp4Unroll];
  fp4_where<true>(a, a.nblk, w);
  const int D = a.nblk * kFp4Block;
#pragma unroll
  for (int u = 0; u < kFp4Unroll; ++u) {
    if (!w[u].have || w[u].slot < 0) continue;
    const T* src = reinterpret_cast<const T*>(w[u].kind ? a.v : a.k) + w[u].t * (w[u].kind ? a.v_stride : a.k_stride) +
                   (w[u].h * a.nblk + w[u].blk) * kFp4Block;
    float x[16];
    fp4_read16<T>(src, VEC, x);
    const float inv_g = 1.f / (w[u].kind ? a.v_scale : a.k_scale);  // exact: a power of two
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[j] = (x[j] != x[j]) ? 0.f : x[j] * inv_g;
      amax = fmaxf(amax, fabsf(x[j]));
    }
    const uint32_t sb = f_to_e4m3(fminf(__fdiv_rn(amax, 6.f), 448.f));
    const uint32_t sh = fp4_scale2_to_h2(sb);
    const float s = __half2float(__ushort_as_half((unsigned short)(sh & 0xffffu)));
    uint32_t c[2] = {0u, 0u};
    if (s > 0.f) {
      const float y = __fdiv_rn(1.f, s);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        // 8192 / 448 is past the largest border: clipping changes no code and keeps infinities out
        x[j] = fp4_quotient(fminf(fmaxf(x[j], -8192.f), 8192.f), s, y);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j >> 2] |= f2_to_e2m1(x[2 * j], x[2 * j + 1]) << (8 * (j & 3));
    }
    uint8_t* row = a.pool + (size_t)w[u].slot * a.row_bytes;
    *reinterpret_cast<uint2*>(row + fp4_code_off(w[u].h, D) + w[u].kind * (D / 2) + w[u].blk * 8) = make_uint2(c[0], c[1]);
    row[fp4_scale_off(w[u].h, a.Hkv, D) + w[u].kind * a.nblk + w[u].blk] = (uint8_t)sb;
  }
}

// 8 + 1 bytes of a block in, 32 or 64 out. Neighbouring lanes hold neighbouring blocks and
// exchange 16-byte chunks, so that every store of a pair fills whole 32-byte sectors.
template <typename T>
__global__ void __launch_bounds__(kFp4Threads) fp4_load_kernel(const Fp4KvArgs a) {
  pdl_wait_then_release();
  constexpr int NC = (int)sizeof(T);      // 16-byte chunks of a block
  const int D = a.nblk * kFp4Block;
  const bool odd = threadIdx.x & 1;
  Fp4Where w[kFp4Unroll];
  fp4_where<false>(a, a.nblk, w);
  uint2 c[kFp4Unroll];
  uint32_t sb[kFp4Unroll];
#pragma unroll
  for (int u = 0; u < kFp4Unroll; ++u) {
    c[u] = make_uint2(0u, 0u);  // a slot outside the pool reads as zeros
    sb[u] = 0;
    if (w[u].slot >= 0) {
      const uint8_t* row = a.pool + (size_t)w[u].slot * a.row_bytes;
      c[u] = *reinterpret_cast<const uint2*>(row + fp4_code_off(w[u].h, D) + w[u].kind * (D / 2) + w[u].blk * 8);
      sb[u] = row[fp4_scale_off(w[u].h, a.Hkv, D) + w[u].kind * a.nblk + w[u].blk];
    }
  }
#pragma unroll
  for (int u = 0; u < kFp4Unroll; ++u) {
    const float g = w[u].kind ? a.v_scale : a.k_scale;
    const uint32_t sh = fp4_scale2_to_h2(sb[u] | (sb[u] << 8));
    uint4 x[NC];
    {
      uint32_t r[8], lo[4], hi[4];
      fp4_word_to_h2(c[u].x, lo);
      fp4_word_to_h2(c[u].y, hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[j] = h2_mul(lo[j], sh);
        r[4 + j] = h2_mul(hi[j], sh);
      }
      constexpr int PC = 8 / (int)sizeof(T);  // pairs of a chunk
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        float f[2 * PC];
#pragma unroll
        for (int j = 0; j < PC; ++j) {
          const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&r[k * PC + j]));
          f[2 * j] = p.x * g;
          f[2 * j + 1] = p.y * g;
        }
        store_vec<T, 2 * PC>(reinterpret_cast<T*>(&x[k]), f);
      }
    }
    // a pair's blocks lie next to each other in one token row (an even number of blocks a head)
    T* pair = reinterpret_cast<T*>(w[u].kind ? a.v_out : a.k_out) +
              ((w[u].t * a.Hkv + w[u].h) * (int64_t)a.nblk + (w[u].blk & ~1)) * kFp4Block;
    uint4* dst = reinterpret_cast<uint4*>(pair);
#pragma unroll
    for (int k = 0; k < NC; k += 2) {
      const uint4 give = odd ? x[k] : x[k + 1];
      uint4 got;
      got.x = __shfl_xor_sync(0xffffffffu, give.x, 1);
      got.y = __shfl_xor_sync(0xffffffffu, give.y, 1);
      got.z = __shfl_xor_sync(0xffffffffu, give.z, 1);
      got.w = __shfl_xor_sync(0xffffffffu, give.w, 1);
      if (w[u].have) {
        dst[k + odd] = odd ? got : x[k];
        dst[NC + k + odd] = odd ? x[k + 1] : got;
      }
    }
  }
}

}  // namespace b2a

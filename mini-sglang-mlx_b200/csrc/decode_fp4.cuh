// Paged decode attention over the 4-bit KV pool (one query row per request).
//
//   out[b, h] = softmax(scale * q[b, h] . K^T) . V,   K, V = code * s of fp4_kv.cuh
//
// Same plan, workspace, in-launch merge and error handling as decode_kernel
// (decode.cuh): a persistent grid, each CTA an equal share of the batch's page
// stream, one producer warp that brings whole token rows with bulk copies.
//
// What bounds it. A cached value is 0.56 bytes, so at HBM rate an SM receives
// about 40 values per clock (1.13 bytes and 2 G multiply-adds per K/V pair):
// expanding and multiplying them has to cost less than a clock per 40 values.
// One warp takes one to four units of 16 tokens x one kv head at a time; a unit is
//   S^T [16 tokens x 8 head columns] = K [16 x D] . Q^T      (D/16 MMAs)
//   O^T [D x 8]                     += V^T [D x 16] . P^T    (D/16 MMAs)
// with mma.sync m16n8k16, fp16 in, fp32 accumulate. The codes become MMA
// operands in registers: two codes per conversion, one packed multiply by the
// block's scale, exact in fp16. The k order of a product is free, so a lane
// takes D/4 consecutive features of a K row (one 16-byte shared load at D =
// 128), and Q is laid out to match; for V a lane takes D/8 consecutive features
// of four tokens, and the codes of two tokens are interleaved in the word
// before they are expanded, so an operand register holds one feature of two
// tokens without any shuffle.
//
// What is left. 72 requests of 1k to 32k tokens (32 / 8 heads x 128, 1.35 GB) take 268 to 288
// us in different runs, 4.7 to 5.0 TB/s; the same stream without the arithmetic takes 220 us, the arithmetic on resident rows 240.
// The core (64 conversions, 64 packed multiplies, 16 MMAs a unit) runs at 86 clocks a unit of an
// SM's 99 at HBM rate: m16n8k16 MMAs and the packed multiplies share a pipe (2.07 and 0.51 clocks
// each, measured to add up), which binds it more than instruction issue does.
//
// q enters as fp16 with each head row scaled by a power of two so that its
// largest element lies in [2^14, 2^15): bf16 has 8 significant bits, so only
// elements 2^28 times smaller than the largest lose any. The factor goes back
// through the softmax scale. fp32 q and P are split into two fp16 parts (22
// bits). The lazy maximum of decode_mma.cuh (it moves when a score exceeds it by
// more than 8) is kept 7 below the score that set it: weights lie in [0, 2^15] with
// the largest at least 2^7, so a weight that fp16 holds as a subnormal is off by
// at most 2^-32 of the largest. Softmax statistics and accumulators are fp32. A row that has seen a
// key therefore sums to at least 2^7: a smaller sum comes from infinite scores, or from ones past
// 2^27 whose rounding alone exceeds the softmax's range, and the row becomes NaN (fp4_row_lost).
#pragma once

#include "decode.cuh"
#include "decode_mma.cuh"
#include "fp4_kv.cuh"

namespace b2a {

// units of 16 tokens a warp takes at a time
// (measured at 8 kv heads x 128, 72 requests of 1k to 32k tokens: 332, 330, 282 us for 1, 2, 4
// units; 16 warps of 2 units, which need a combine per segment: 303 us). Four units of
// head_dim 256 would leave room for one stage, and 16 warps have registers for one unit.
__host__ __device__ constexpr int fp4_units_of(int NCW, int D) { return NCW == 16 ? 1 : D == 256 ? 2 : 4; }

struct Fp4DecodeSmem {
  uint32_t bars, cbuf, abort_flag, last_flag, total;
};

__host__ __device__ inline Fp4DecodeSmem fp4_decode_smem(int NSTAGE, uint32_t stage_bytes, int NCW, int WPH, int G,
                                                         int D) {
  Fp4DecodeSmem L;
  uint32_t off = (uint32_t)NSTAGE * stage_bytes;
  off = (off + 15u) & ~15u;
  L.bars = off;
  off += (uint32_t)NSTAGE * 16u;
  L.cbuf = off;
  if (WPH > 1) off += (uint32_t)NCW * (uint32_t)G * (uint32_t)(D + 2) * 4u;
  off = (off + 15u) & ~15u;
  L.abort_flag = off;
  L.last_flag = off + 16;
  L.total = off + 32;  // last_flag: one word per pending request
  return L;
}

// D += A (16x16 fp16, row) . B (16x8 fp16, col), fp32 accumulate.
__device__ __forceinline__ void mma_16816_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&p);
}

__device__ __forceinline__ float2 h2_to_f2(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }

// Power of two that brings a row's largest magnitude into [2^14, 2^15), and its inverse.
// Zero, infinite and NaN rows keep a factor of one.
__device__ __forceinline__ void fp4_row_factor(float amax, float& f, float& inv) {
  int e = (int)((__float_as_uint(amax) >> 23) & 0xff) - 127;
  if (!(amax > 0.f) || e > 127) e = 14;
  e = e < -100 ? -100 : e;
  f = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
  inv = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
}

constexpr float kNaN = __builtin_nanf("");

// Whether a row's weights are lost, for the weight sum of a row that has seen a key: 2^7 less what
// rounding takes from scores the softmax can tell apart (NaN: shown already).
__device__ __forceinline__ bool fp4_row_lost(float sum) { return sum < 1.f; }

// Softmax scale of a head row's raw scores, kept above zero: at the smallest normal float every score
// (raw ones stay below 2^35) is nothing already, while zero times a masked -inf would be NaN.
__device__ __forceinline__ float fp4_score_scale(float inv, float qscale) {
  return fmaxf(inv * qscale, 0x1p-126f);
}

// Words of codes a lane reads from one K row (D/4 features) and one V row (D/8 features).
template <int N>
__device__ __forceinline__ void fp4_lds(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// N consecutive scale bytes, each as an fp16 pair of twice the same value.
template <int N>
__device__ __forceinline__ void fp4_scales(const uint8_t* p, uint32_t (&s)[N]) {
  if constexpr (N == 1) {
    const uint32_t b = *p;
    s[0] = fp4_scale2_to_h2(b | (b << 8));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t h = fp4_scale2_to_h2(*reinterpret_cast<const uint16_t*>(p + i));
      s[i] = __byte_perm(h, 0, 0x1010);
      s[i + 1] = __byte_perm(h, 0, 0x3232);
    }
  }
}

// NU units of one head, their softmax step taken together. row0: shared address of token 0's
// row; with PART only nt of the 16 NU tokens are real. qf[p]: part p of Q^T (features of this
// lane's quarter, head column g).
template <int D, int SPLIT, int NU, bool PART>
__device__ __forceinline__ void fp4_units(const uint8_t* row0, uint32_t pitch, uint32_t code_off, uint32_t scale_off,
                                          int nt, int lane, const float (&qs)[2],
                                          const uint32_t (&qf)[SPLIT][D / 16][2], float (&acc)[D / 16][4],
                                          float (&mref)[2], float (&lsum)[2]) {
  constexpr unsigned FULL = 0xffffffffu;
  constexpr int KS = D / 16;  // MMAs of a product
  const int g = lane >> 2, t = lane & 3;
  // ---- S^T: rows g and g + 8 of each unit, features [t D/4, (t+1) D/4)
  // raw scores, x[u][0]: (token g, column 2t) [1]: (g, 2t+1) [2]: (g+8, 2t) [3]: (g+8, 2t+1)
  float x[NU][4];
  const uint8_t* krow = row0 + (uint32_t)g * pitch + code_off + t * (D / 8);
  const uint8_t* srow = row0 + (uint32_t)g * pitch + scale_off + t * (D / 64);
#pragma unroll
  for (int u = 0; u < NU; ++u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[u][i] = 0.f;
    uint32_t wa[D / 32], wb[D / 32];
    fp4_lds<D / 32>(krow + (16u * u) * pitch, wa);
    fp4_lds<D / 32>(krow + (16u * u + 8u) * pitch, wb);
    uint32_t sca[D / 64], scb[D / 64];  // a block's scale, twice
    fp4_scales<D / 64>(srow + (16u * u) * pitch, sca);
    fp4_scales<D / 64>(srow + (16u * u + 8u) * pitch, scb);
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {  // eight features of both rows: two MMAs
      uint32_t xa[4], xb[4];
      fp4_word_to_h2(wa[w], xa);
      fp4_word_to_h2(wb[w], xb);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xa[j] = h2_mul(xa[j], sca[w >> 1]);
        xb[j] = h2_mul(xb[j], scb[w >> 1]);
      }
#pragma unroll
      for (int p = 0; p < SPLIT; ++p) {
        mma_16816_f16(x[u], xa[0], xb[0], xa[1], xb[1], qf[p][2 * w][0], qf[p][2 * w][1]);
        mma_16816_f16(x[u], xa[2], xb[2], xa[3], xb[3], qf[p][2 * w + 1][0], qf[p][2 * w + 1][1]);
      }
    }
    if constexpr (PART) {
      if (16 * u + g >= nt) x[u][0] = x[u][1] = kNegInf;
      if (16 * u + g + 8 >= nt) x[u][2] = x[u][3] = kNegInf;
    }
  }
  float cm[2] = {fmaxf(x[0][0], x[0][2]), fmaxf(x[0][1], x[0][3])};
#pragma unroll
  for (int u = 1; u < NU; ++u) {
    cm[0] = fmaxf(cm[0], fmaxf(x[u][0], x[u][2]));
    cm[1] = fmaxf(cm[1], fmaxf(x[u][1], x[u][3]));
  }
  cm[0] *= qs[0];  // qs > 0 keeps the order
  cm[1] *= qs[1];
  const bool grow = cm[0] > mref[0] + 15.f || cm[1] > mref[1] + 15.f;
  if (__any_sync(FULL, grow)) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float v = cm[n];
      v = fmaxf(v, __shfl_xor_sync(FULL, v, 4));
      v = fmaxf(v, __shfl_xor_sync(FULL, v, 8));
      v = fmaxf(v, __shfl_xor_sync(FULL, v, 16));
      if (v > mref[n] + 15.f) {  // the same decision on every lane of the column
        const float alpha = (mref[n] == kNegInf) ? 0.f : ex2_approx(mref[n] - (v - 7.f));
        mref[n] = v - 7.f;
        lsum[n] *= alpha;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          acc[mt][n] *= alpha;
          acc[mt][2 + n] *= alpha;
        }
      }
    }
  }
  uint32_t pb[NU][SPLIT][2];  // P^T as the B operand: tokens 0-7 and 8-15 of each unit
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = ex2_approx(fmaf(x[u][i], qs[i & 1], -mref[i & 1]));
      if (PART) p[i] = (x[u][i] == kNegInf) ? 0.f : p[i];  // a column without a token yet: -inf - -inf
    }
    lsum[0] += p[0] + p[2];
    lsum[1] += p[1] + p[3];
    const uint32_t h0 = pack_h2(p[0], p[1]), h1 = pack_h2(p[2], p[3]);
    pb[u][0][0] = movmatrix_trans(h0);
    pb[u][0][1] = movmatrix_trans(h1);
    if constexpr (SPLIT == 2) {
      const float2 f0 = h2_to_f2(h0), f1 = h2_to_f2(h1);
      pb[u][1][0] = movmatrix_trans(pack_h2(p[0] - f0.x, p[1] - f0.y));
      pb[u][1][1] = movmatrix_trans(pack_h2(p[2] - f1.x, p[3] - f1.y));
    }
  }
  // ---- O^T: features [g D/8, (g+1) D/8) of tokens 2t, 2t+1, 2t+8, 2t+9 of each unit
  constexpr int NW = D / 64;               // words of codes per token
  constexpr int NS = D > 128 ? 2 : 1;      // scales per token
  const uint8_t* vrow = row0 + (uint32_t)(2 * t) * pitch + code_off + D / 2 + g * (D / 16);
  const uint8_t* wrow = row0 + (uint32_t)(2 * t) * pitch + scale_off + D / 16 + (g * (D / 8)) / 16;
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    uint32_t lo[2][NW], hi[2][NW], sc[2][NS];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int ta = 16 * u + 8 * b;  // token pair (ta + 2t, ta + 2t + 1)
      uint32_t wa[NW], wb[NW];
      fp4_lds<NW>(vrow + (uint32_t)ta * pitch, wa);
      fp4_lds<NW>(vrow + (uint32_t)(ta + 1) * pitch, wb);
#pragma unroll
      for (int q = 0; q < NS; ++q) {
        uint32_t sa = wrow[(uint32_t)ta * pitch + q], sb = wrow[(uint32_t)(ta + 1) * pitch + q];
        if constexpr (PART) {
          // rows past the last token hold whatever the stage held before: a zero scale
          // keeps their products finite (their weights are zero)
          if (ta + 2 * t >= nt) sa = 0;
          if (ta + 2 * t + 1 >= nt) sb = 0;
        }
        sc[b][q] = fp4_scale2_to_h2(sa | (sb << 8));
      }
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        // bytes of (token a, token b) codes: even features, odd features
        lo[b][w] = (wa[w] & 0x0f0f0f0fu) | ((wb[w] << 4) & 0xf0f0f0f0u);
        hi[b][w] = ((wa[w] >> 4) & 0x0f0f0f0fu) | (wb[w] & 0xf0f0f0f0u);
      }
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      uint32_t l0[4], h0[4], l1[4], h1[4];
      fp4_word_to_h2(lo[0][w], l0);
      fp4_word_to_h2(hi[0][w], h0);
      fp4_word_to_h2(lo[1][w], l1);
      fp4_word_to_h2(hi[1][w], h1);
      const int q = w >> 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a0 = h2_mul(l0[j], sc[0][q]), a1 = h2_mul(h0[j], sc[0][q]);
        const uint32_t a2 = h2_mul(l1[j], sc[1][q]), a3 = h2_mul(h1[j], sc[1][q]);
#pragma unroll
        for (int pp = 0; pp < SPLIT; ++pp) mma_16816_f16(acc[4 * w + j], a0, a1, a2, a3, pb[u][pp][0], pb[u][pp][1]);
      }
    }
  }
}

template <typename T, int D, int NCW>
__global__ void __launch_bounds__((NCW + 4) * 32, 1) decode_fp4_kernel(const DecodeArgs a, const float v_scale) {
  // programmatic dependent launch exactly as decode_kernel: the plan and the page ids are
  // read before the wait, everything the previous kernel may have written after it
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int SPLIT = sizeof(T) == 4 ? 2 : 1;
  constexpr int NU = fp4_units_of(NCW, D), TW = 16 * NU;
  constexpr int KS = D / 16;
  constexpr unsigned FULL = 0xffffffffu;
  extern __shared__ __align__(128) uint8_t smem[];
  const int G = a.Hq / a.Hkv;
  const Fp4DecodeSmem L = fp4_decode_smem(a.NSTAGE, a.stage_bytes, NCW, a.WPH, G, D);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* empty = full + a.NSTAGE;
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L.abort_flag);
  volatile int* s_last = reinterpret_cast<volatile int*>(smem + L.last_flag);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.NSTAGE; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], NCW);
    }
    *s_abort = 0;
    fence_mbar_init();
  }
  __syncthreads();

  const int seg0 = a.cta_indptr[blockIdx.x];
  const int seg1 = a.cta_indptr[blockIdx.x + 1];
  const bool last_first = decode_last_first(a, seg0, seg1);
  const int P = 1 << a.page_log2;
  const int TS = a.TS;

  // Register split: NCW + 4 warps launch with 96 (NCW 16) or 168 (NCW 8) registers a thread;
  // the consumers take 112 (232) and the last warpgroup, of which one warp works, keeps 32
  // (40): 512 x 112 + 128 x 32 = 640 x 96, and 256 x 232 + 128 x 40 = 384 x 168.
  if (warp >= NCW) {
    if constexpr (NCW == 16) asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp > NCW) return;
    // ------------------------------------------------------------ producer
    const uint64_t pol = l2_evict_first_policy();
    const uint8_t* pool = reinterpret_cast<const uint8_t*>(a.k_pool);
    const size_t rowB = a.row_bytes;
    // a stage is a run inside one page (P >= TS), or whole pages (stages start on page boundaries)
    const bool one_run = P >= TS;
    const int nseg = seg1 - seg0;
    int seg = -1, tok = 0, ntok = 0, pbeg = 0;
    auto advance = [&]() -> bool {  // to the next stage
      tok += TS;
      while (tok >= ntok) {
        if (++seg >= nseg) return false;
        int b, slot;
        decode_get_seg(a, decode_seg_at(a, seg0, seg1, last_first, seg), b, pbeg, ntok, slot);
        if (!decode_seg_ok(a, b, slot)) ntok = 0;  // the consumers skip it too (and report it)
        tok = 0;
      }
      return true;
    };
    auto copies = [&](int nt) { return one_run ? 1 : (nt + P - 1) >> a.page_log2; };
    auto first_id = [&]() -> int {  // this lane's page id of the stage at (seg, tok)
      return lane < copies(min(TS, ntok - tok)) ? a.kv_indices[pbeg + (tok >> a.page_log2) + lane] : -2;
    };
    int ctr = 0, st = 0;
    uint32_t ph = 1;
    bool waited = false;
    bool have = advance();
    int id = have ? first_id() : -2;
    while (have) {
      const int nt = min(TS, ntok - tok);
      const int ncopies = copies(nt);
      const int32_t* ids = a.kv_indices + pbeg + (tok >> a.page_log2);
      const int in_page = one_run ? tok & (P - 1) : 0;
      const int my_id = id;
      // the next stage's segment and page ids are on their way while this stage waits and copies
      have = advance();
      id = have ? first_id() : -2;
      // bad page ids never reach the copy engine: the error is recorded, the stage's
      // copies are skipped and the consumers run on what the stage held
      bool good = true;
      for (int j = lane; j < ncopies; j += 32) {
        const int64_t page = j < 32 ? my_id : ids[j];
        const int rows = one_run ? nt : min(P, nt - j * P);
        good = good && page >= 0 && page * P + in_page + rows <= a.num_slots;
      }
      good = __all_sync(FULL, good);
      if (!__all_sync(FULL, mbar_wait(&empty[st], ph, kWdDecodeEmpty)) || !__all_sync(FULL, *s_abort == 0)) {
        *s_abort = 1;
        break;
      }
      uint8_t* dst = smem + (size_t)st * a.stage_bytes;
      if (lane == 0) {
        if (good) {
          mbar_arrive_expect_tx(&full[st], (uint32_t)nt * a.row_bytes);
        } else {
          watchdog_set(kWdBadSlot);
          mbar_arrive(&full[st]);
        }
      }
      __syncwarp();
      if (!waited) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows of the previous kernel
        waited = true;
      }
      if (good) {
        for (int j0 = 0; j0 < ncopies; j0 += 32) {
          // consecutive page ids are consecutive slots: one bulk copy per run of them
          const int j = j0 + lane;
          const int64_t page = j < ncopies ? (j0 == 0 ? my_id : ids[j]) : -2;
          const int64_t prev = __shfl_up_sync(FULL, page, 1);
          const bool head = j < ncopies && (lane == 0 || page != prev + 1);
          const uint32_t heads = __ballot_sync(FULL, head);
          if (head) {
            const uint32_t above = lane == 31 ? 0u : (heads >> (lane + 1)) << (lane + 1);
            const int end = j0 + (above ? __ffs((int)above) - 1 : min(32, ncopies - j0));
            const int rows = one_run ? nt : min(end * P, nt) - j * P;
            bulk_g2s(dst + (size_t)j * P * rowB, pool + (page * P + in_page) * rowB, (uint32_t)rows * a.row_bytes,
                     &full[st], pol);
          }
        }
      }
      __syncwarp();
      ++ctr;
      if (++st == a.NSTAGE) {
        st = 0;
        ph ^= 1u;
      }
    }
    // never leave while our own copies may still be landing
    const int first = ctr > a.NSTAGE ? ctr - a.NSTAGE : 0;
    for (int i = first; i < ctr; ++i) mbar_wait(&full[i % a.NSTAGE], (uint32_t)(i / a.NSTAGE) & 1u, kWdDecodeDrain);
    return;
  }

  // -------------------------------------------------------------- consumers
  if constexpr (NCW == 16) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
  const int h = warp / a.WPH;
  const int sub = warp - h * a.WPH;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t code_off = fp4_code_off(h, D), scale_off = fp4_scale_off(h, a.Hkv, D);
  float* cbuf = reinterpret_cast<float*>(smem + L.cbuf);
  const T* qbase = reinterpret_cast<const T*>(a.q);
  int st = 0;
  uint32_t ph = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // q, the workspace and out follow the previous kernel
  const int4* segs = reinterpret_cast<const int4*>(a.segs);
  int4 next = seg1 > seg0 ? segs[decode_seg_at(a, seg0, seg1, last_first, 0)] : make_int4(0, 0, 0, -1);
  int pend[2] = {0, 0}, npend = 0;  // requests whose partial rows this CTA has written, tickets not yet taken
  for (int i = 0; i < seg1 - seg0; ++i) {
    const int b = next.x, ntok = next.z, slot = next.w;
    if (i + 1 < seg1 - seg0) next = segs[decode_seg_at(a, seg0, seg1, last_first, i + 1)];
    const bool good = decode_seg_ok(a, b, slot);
    if (!good && threadIdx.x == 0) watchdog_set(kWdBadPlan);
    if (good) {
    // ---- Q^T: head column g, features [t D/4, (t+1) D/4); zero columns past the group
    uint32_t qf[SPLIT][KS][2];
    float qs[2];
    {
      float qv[D / 4];
      if (g < G) {
        load_vec<T, D / 4>(qbase + ((size_t)b * a.Hq + h * G + g) * D + t * (D / 4), qv);
      } else {
#pragma unroll
        for (int e = 0; e < D / 4; ++e) qv[e] = 0.f;
      }
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < D / 4; ++e) amax = fmaxf(amax, fabsf(qv[e]));
      amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 2));
      float f, inv;
      fp4_row_factor(amax, f, inv);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float e0 = qv[4 * k + 2 * j] * f, e1 = qv[4 * k + 2 * j + 1] * f;
          qf[0][k][j] = pack_h2(e0, e1);
          if constexpr (SPLIT == 2) {
            const float2 r = h2_to_f2(qf[0][k][j]);
            qf[1][k][j] = pack_h2(e0 - r.x, e1 - r.y);
          }
        }
      }
      inv = fp4_score_scale(inv, a.qscale);
      qs[0] = __shfl_sync(FULL, inv, 8 * t);      // column 2t
      qs[1] = __shfl_sync(FULL, inv, 8 * t + 4);  // column 2t + 1
    }
    // the next segment's query row and merge range come closer while this one is streamed
    if (i + 1 < seg1 - seg0 && next.x >= 0 && next.x < a.B) {
      if (g < G) {
        const T* qn = qbase + ((size_t)next.x * a.Hq + h * G + g) * D + t * (D / 4);
        asm volatile("prefetch.global.L1 [%0];" ::"l"(qn));
        if (next.w >= 0) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.merge_indptr + next.x));
      }
    }
    float acc[KS][4];
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
    float mref[2] = {kNegInf, kNegInf}, lsum[2] = {0.f, 0.f};
    for (int tok = 0; tok < ntok; tok += TS) {
      const int nt = min(TS, ntok - tok);
      bool ok = mbar_try_wait(&full[st], ph);
      if (!__all_sync(FULL, ok)) {
        ok = __all_sync(FULL, *s_abort == 0);
        if (ok) ok = __all_sync(FULL, mbar_wait(&full[st], ph, kWdDecodeFull));
        if (!ok) *s_abort = 1;
      }
      if (ok) {
        const uint8_t* rows = smem + (size_t)st * a.stage_bytes;
        for (int t0 = sub * TW; t0 < nt; t0 += a.WPH * TW) {
          const uint8_t* row0 = rows + (uint32_t)t0 * a.row_bytes;
          if (nt - t0 >= TW) {
            fp4_units<D, SPLIT, NU, false>(row0, a.row_bytes, code_off, scale_off, TW, lane, qs, qf, acc, mref, lsum);
          } else {
            // the rows that are left, unit by unit: little code beside the full step (a second
            // copy of it costs instruction-cache misses)
#pragma unroll 1
            for (int t1 = t0; t1 < nt; t1 += 16) {
              fp4_units<D, SPLIT, 1, true>(row0, a.row_bytes, code_off, scale_off, nt - t1, lane, qs, qf, acc, mref, lsum);
              row0 += 16u * a.row_bytes;
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == a.NSTAGE) {
        st = 0;
        ph ^= 1u;
      }
    }
    // ---- row sums over the 8 lanes of each head column
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      lsum[n] += __shfl_xor_sync(FULL, lsum[n], 4);
      lsum[n] += __shfl_xor_sync(FULL, lsum[n], 8);
      lsum[n] += __shfl_xor_sync(FULL, lsum[n], 16);
    }
    // lane (g, t) holds features [g D/8, (g+1) D/8) of head columns 2t, 2t + 1: feature
    // 2 mt of the run in acc[mt][n], 2 mt + 1 in acc[mt][2 + n]
    constexpr int EPL = D / 8;
    if (a.WPH > 1) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int c = 2 * t + n;
        if (c < G) {
          float* mine = cbuf + ((size_t)warp * G + c) * (D + 2);
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
            *reinterpret_cast<float2*>(mine + g * EPL + 2 * mt) = make_float2(acc[mt][n], acc[mt][2 + n]);
          if (g == 0) *reinterpret_cast<float2*>(mine + D) = make_float2(mref[n], lsum[n]);
        }
      }
      named_bar_sync(1, NCW * 32);
      if (sub == 0) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int c = 2 * t + n;
          if (c < G) {
            float M = kNegInf, Lsum = 0.f;
            for (int s2 = 0; s2 < a.WPH; ++s2) M = fmaxf(M, cbuf[((size_t)(warp + s2) * G + c) * (D + 2) + D]);
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) acc[mt][n] = acc[mt][2 + n] = 0.f;
            for (int s2 = 0; s2 < a.WPH; ++s2) {
              const float* o = cbuf + ((size_t)(warp + s2) * G + c) * (D + 2);
              const float w = (o[D] == kNegInf) ? 0.f : exp2f(o[D] - M);
              Lsum += o[D + 1] * w;
#pragma unroll
              for (int mt = 0; mt < KS; ++mt) {
                const float2 v = *reinterpret_cast<const float2*>(o + g * EPL + 2 * mt);
                acc[mt][n] = fmaf(w, v.x, acc[mt][n]);
                acc[mt][2 + n] = fmaf(w, v.y, acc[mt][2 + n]);
              }
            }
            mref[n] = M;
            lsum[n] = Lsum;
          }
        }
      }
    }
    if (sub == 0) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int c = 2 * t + n;
        if (c < G) {
          const size_t row = (size_t)h * G + c;
          float r[EPL];
          // the sums reach 2^57 (2^31 weights of 2^15 and values of 2688): a row is divided before it
          // is scaled, and a partial row of a scale above 2^64 gives up 2^48, and so does its lsum
          const float part = v_scale > 0x1p64f ? 0x1p-48f : 1.f;
          float f = slot < 0 ? (lsum[n] > 0.f ? 1.f / lsum[n] : 0.f) : part;
          if (ntok > 0 && fp4_row_lost(lsum[n])) f = kNaN;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt) {
            r[2 * mt] = acc[mt][n] * f * v_scale;
            r[2 * mt + 1] = acc[mt][2 + n] * f * v_scale;
          }
          if (slot < 0) {
            store_vec<T, EPL>(reinterpret_cast<T*>(a.out) + ((size_t)b * a.Hq + row) * D + g * EPL, r);
          } else {
            store_vec<float, EPL>(a.ws_acc + ((size_t)slot * a.Hq + row) * D + g * EPL, r);
            if (g == 0)
              *reinterpret_cast<float2*>(a.ws_ml + ((size_t)slot * a.Hq + row) * 2) = make_float2(mref[n], lsum[n] * part);
          }
        }
      }
      if (slot >= 0) __threadfence();  // publish the partial rows at GPU scope before the ticket
    }
    if (a.WPH > 1) named_bar_sync(1, NCW * 32);  // cbuf is free again
    if (slot >= 0) pend[npend++] = b;
    }
    // Tickets of the pending requests, and the merge of those that this CTA completes: at the end
    // of the CTA's work (a share cuts at most two requests), because they cost all warps a fence,
    // two barriers and an atomic round trip.
    if (npend == 2 || (npend > 0 && i + 1 == seg1 - seg0)) {
      named_bar_sync(1, NCW * 32);  // every warp has written and fenced its rows
      if (threadIdx.x < (unsigned)npend) {
        const int pb = threadIdx.x ? pend[1] : pend[0];
        const int p0 = a.merge_indptr[pb], p1 = a.merge_indptr[pb + 1];
        const int prev = atomicAdd(&a.tickets[p0], 1);
        const bool last = prev == p1 - p0 - 1;
        if (last) a.tickets[p0] = 0;  // every partial has arrived: re-arm for the next call
        s_last[threadIdx.x] = last ? 1 : 0;
      }
      named_bar_sync(1, NCW * 32);
#pragma unroll 1
      for (int k = 0; k < npend; ++k) {
        const int pb = k ? pend[1] : pend[0];
        if (s_last[k]) {
          __threadfence();
          decode_merge_request<T, D>(a, pb, a.merge_indptr[pb], a.merge_indptr[pb + 1], warp, lane);
        }
      }
      npend = 0;
    }
  }
}

}  // namespace b2a

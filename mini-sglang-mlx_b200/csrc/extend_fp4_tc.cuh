// Ragged causal extend attention over the 4-bit KV pool on tcgen05 tensor cores
// (bf16 queries, head_dim 128, GQA group 1, 2, 4 or 8, any page size).
//
//   O = softmax(scale * Q K^T, causal to the bottom right) V,   K, V of fp4_kv.cuh
//
// The tile, the MMA order, the softmax and the counted releases of P are those
// of extend_tc.cuh (two 128-row tiles of one request and kv head share each block
// of 128 keys; S and O in TMEM, one softmax thread per row, P written over S). What
// differs is where K and V come from. A warpgroup of 128 threads expands the block:
// thread i owns key i, reads its 64 + 64 code bytes and 16 scale bytes from the pool
// (any slot: page ids are looked up per key, so every page size works and nothing is
// staged), and writes the fp16 rows into the SWIZZLE_128B tiles the MMAs read. Loads
// for block j + 1 are issued as soon as block j's registers are free, the page id of
// block j + 2 with them, so the two dependent reads hide behind a block's time.
// code * s is exact in fp16 (fp4_kv.cuh), and so is q after a power of two per row
// (decode_fp4.cuh), undone in the row's softmax scale: the products are exact.
//
// Few rows on a long prefix leave most SMs idle, so the keys of a work item can be
// cut into n_split runs of blocks (grid z). Each run writes its unnormalised rows
// and (m, l) to a workspace; the CTA that takes the item's last ticket joins them, in
// run order. Nothing waits for another CTA.
//
// Register split: 512 threads launch with 128 registers (65,536 in all); the softmax
// warpgroups take 168 each, the expanding one 112, the issuer's 64: 512 x 128 again.
#pragma once

#include "decode_fp4.cuh"
#include "extend_tc.cuh"
#include "fp4_kv.cuh"

namespace b2a {

constexpr int kF4Threads = 512;

struct F4Args {
  const __nv_bfloat16* q;
  const uint8_t* pool;
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_last_page_len;
  const int32_t* work;
  __nv_bfloat16* out;
  float* ws_acc;     // [item][head][split][256 rows][128]
  float* ws_ml;      // [item][head][split][256 rows][2]
  int32_t* tickets;  // [item][head]
  int64_t num_slots;
  uint32_t row_bytes;
  int page_log2;
  int Hq, Hkv, G, g_log2;
  int n_split;
  int item0;  // index of this launch's first work item
  float qscale;  // scale * k_scale * log2(e)
  float v_scale;
};

struct F4Smem {
  static constexpr uint32_t Q0 = 0;
  static constexpr uint32_t K0 = Q0 + 2 * kTcTileBytes;
  static constexpr uint32_t V0 = K0 + 2 * kTcTileBytes;
  static constexpr uint32_t BARS = V0 + 2 * kTcTileBytes;
  // q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], mma_done, spare, p_full at 14
  static constexpr int NBARS = 22;
  static constexpr uint32_t TMEM_SLOT = BARS + NBARS * 8;
  static constexpr uint32_t ABORT = TMEM_SLOT + 8;
  static constexpr uint32_t PCNT = ABORT + 8;
  static constexpr uint32_t LAST = PCNT + 32;
  static constexpr uint32_t QFAC = LAST + 16;  // float [2][128]: softmax scale of each row
  static constexpr uint32_t TOTAL = QFAC + 1024;
  static constexpr uint32_t ALLOC = TOTAL + 1024;
};

// fp16 x fp16 -> fp32, M = 128, N = 128.
__host__ __device__ constexpr uint32_t f4_idesc(bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 64 code bytes and 8 scale bytes of one row -> 128 fp16 in row `row` of an SW128 tile.
__device__ __forceinline__ void f4_expand_row(uint8_t* tile, int row, const uint4 (&c)[4], uint2 sc) {
  const uint32_t base = (uint32_t)row * 128u;
  const uint32_t x = (uint32_t)(row & 7);
#pragma unroll
  for (int q = 0; q < 4; ++q) {  // 16 code bytes: two blocks of 16 features
    const uint32_t two = ((q < 2 ? sc.x : sc.y) >> ((q & 1) * 16)) & 0xffffu;
    const uint32_t s01 = fp4_scale2_to_h2(two);
    const uint32_t s0 = __byte_perm(s01, 0, 0x1010), s1 = __byte_perm(s01, 0, 0x3232);
    const uint32_t w[4] = {c[q].x, c[q].y, c[q].z, c[q].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t r[4];
      fp4_word_to_h2(w[i], r);
      const uint32_t s = i < 2 ? s0 : s1;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = h2_mul(r[e], s);
      const int chunk = 4 * q + i;  // 16-byte chunk (8 features) of the row
      *reinterpret_cast<uint4*>(tile + (chunk >> 3) * kTcHalfBytes + base + (((uint32_t)(chunk & 7) ^ x) << 4)) =
          make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}

__global__ void __launch_bounds__(kF4Threads, 1) extend_fp4_tc_kernel(const F4Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F4Smem::BARS);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;   // [2]
  uint64_t* k_empty = bars + 3;  // [2]
  uint64_t* v_full = bars + 5;   // [2]
  uint64_t* v_empty = bars + 7;  // [2]
  uint64_t* s_full = bars + 9;   // [2] per tile
  uint64_t* mma_done = bars + 13;
  uint64_t* p_full = bars + 14;  // [tile * 4 + half]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + F4Smem::TMEM_SLOT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + F4Smem::ABORT);
  uint32_t* pcnt = reinterpret_cast<uint32_t*>(smem + F4Smem::PCNT);
  volatile int* s_last = reinterpret_cast<volatile int*>(smem + F4Smem::LAST);
  float* qfac = reinterpret_cast<float*>(smem + F4Smem::QFAC);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.G;
  const int TT = kTcRows >> a.g_log2;  // tokens per tile
  const int item = a.item0 + blockIdx.y;
  const int4 w = reinterpret_cast<const int4*>(a.work)[item];
  const int nq = min(w.z, 2 * TT);
  if (w.z > nq && threadIdx.x == 0) watchdog_set(kWdTileTooLarge);
  if (nq <= 0) return;  // unused entry behind a device-built work list
  const int r = w.x, tb = w.y;
  const int nq_t[2] = {min(nq, TT), max(0, nq - TT)};
  const int h = blockIdx.x;
  const int P = 1 << a.page_log2;
  const int q0 = a.qo_indptr[r];
  const int Lq = a.qo_indptr[r + 1] - q0;
  const int pbeg = a.kv_indptr[r];
  const int npages = a.kv_indptr[r + 1] - pbeg;
  const int Lkv = npages > 0 ? ((npages - 1) << a.page_log2) + (a.kv_last_page_len ? a.kv_last_page_len[r] : P) : 0;
  const int prefix = Lkv - Lq;
  // blocks each tile needs, then this CTA's run of them: [b0, b0 + nb)
  int nb_t[2];
  for (int t = 0; t < 2; ++t) {
    const int kv_end = nq_t[t] > 0 ? max(0, min(Lkv, prefix + tb + t * TT + nq_t[t])) : 0;
    nb_t[t] = (kv_end + kTcKeys - 1) / kTcKeys;
  }
  const int nb_all = max(nb_t[0], nb_t[1]);
  const int b0 = (int)((int64_t)nb_all * blockIdx.z / a.n_split);
  const int b1 = (int)((int64_t)nb_all * (blockIdx.z + 1) / a.n_split);
  for (int t = 0; t < 2; ++t) nb_t[t] = max(0, min(nb_t[t], b1) - b0);
  const int nb = max(nb_t[0], nb_t[1]);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);  // one arrive per expanding warp
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      for (int c = 0; c < 2; ++c) mbar_init(&p_full[i * 4 + c], 4);  // one arrive per softmax warp
    }
    mbar_init(mma_done, 1);
    for (int i = 0; i < 8; ++i) pcnt[i] = 0;
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_qk = f4_idesc(false);
      constexpr uint32_t idesc_pv = f4_idesc(true);
      bool ok = tc_wait(q_full, 0, abort_flag);
      auto issue_s = [&](int t, int j) {
        const uint32_t sQ = smem_u32(smem + F4Smem::Q0 + t * kTcTileBytes);
        const uint32_t sK = smem_u32(smem + F4Smem::K0 + (j & 1) * kTcTileBytes);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint64_t ad = sw128_desc(sQ + (kk >> 2) * kTcHalfBytes + (kk & 3) * 32, 16, 1024);
          const uint64_t bd = sw128_desc(sK + (kk >> 2) * kTcHalfBytes + (kk & 3) * 32, 16, 1024);
          tc_mma_f16(tmem + t * 128, ad, bd, idesc_qk, kk > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[t]);
      };
      auto p_done = [&](int idx, int j) -> bool {
        uint32_t v;
        asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(&pcnt[idx])) : "memory");
        return v >= 4u * (uint32_t)(j + 1);
      };
      auto issue_pv = [&](int t, int j, int half) {
        const uint32_t sV = smem_u32(smem + F4Smem::V0 + (j & 1) * kTcTileBytes);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int kk = half * 4 + q;
          const uint64_t bd = sw128_desc(sV + kk * 2048, kTcHalfBytes, 1024);
          tc_mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, bd, idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
        }
      };
      if (ok && nb > 0) {
        ok = tc_wait(&k_full[0], 0, abort_flag);
        if (ok) {
          tc_fence_after();
          for (int t = 0; t < 2; ++t)
            if (nb_t[t] > 0) issue_s(t, 0);
          tc_commit(&k_empty[0]);
        }
      }
      for (int j = 0; j < nb && ok; ++j) {
        if (!tc_wait(&v_full[j & 1], (uint32_t)(j >> 1) & 1u, abort_flag)) {
          ok = false;
          break;
        }
        const bool more = j + 1 < nb;
        bool k_next = false;
        for (int t = 0; t < 2 && ok; ++t) {
          if (j < nb_t[t]) {
            if (p_done(t * 4 + 1, j)) {
              tc_fence_after();
              issue_pv(t, j, 0);
              issue_pv(t, j, 1);
            } else {
              for (int half = 0; half < 2 && ok; ++half) {
                if (!p_done(t * 4 + half, j) && !tc_wait(&p_full[t * 4 + half], (uint32_t)j & 1u, abort_flag)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                issue_pv(t, j, half);
              }
            }
            if (!ok) break;
          }
          if (more && j + 1 < nb_t[t]) {
            if (!k_next) {
              if (!tc_wait(&k_full[(j + 1) & 1], (uint32_t)((j + 1) >> 1) & 1u, abort_flag)) {
                ok = false;
                break;
              }
              tc_fence_after();
              k_next = true;
            }
            issue_s(t, j + 1);
          }
        }
        if (!ok) break;
        tc_commit(&v_empty[j & 1]);
        if (more) tc_commit(&k_empty[(j + 1) & 1]);
      }
      // every MMA issued above has completed once mma_done fires (also on the abort path)
      tc_commit(mma_done);
      mbar_wait(mma_done, 0, kWdExtendDrain);
    }
  } else if (warp >= 12) {
    // ---------------------------------------------------------------- expanding warpgroup
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    constexpr unsigned FULL = 0xffffffffu;
    const int row = threadIdx.x - 384;  // key of a block, and row of a query tile
    const uint32_t code_off = fp4_code_off(h, kTcD), scale_off = fp4_scale_off(h, a.Hkv, kTcD);
    // pool row of this thread's key of block j; NULL past the last key
    auto page_of = [&](int j) -> int {
      const int key = (b0 + j) * kTcKeys + row;
      return j < nb && key < Lkv ? a.kv_indices[pbeg + (key >> a.page_log2)] : -1;
    };
    auto row_of = [&](int j, int page) -> const uint8_t* {
      const int key = (b0 + j) * kTcKeys + row;
      if (j >= nb || key >= Lkv) return nullptr;
      const int64_t slot = (int64_t)page * P + (key & (P - 1));
      if (page < 0 || slot >= a.num_slots) {
        watchdog_set(kWdBadSlot);
        return nullptr;  // the key reads as zeros
      }
      return a.pool + (size_t)slot * a.row_bytes;
    };
    auto load4 = [&](const uint8_t* p, uint4 (&c)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = p ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
    };
    uint4 kc[4], vc[4];
    uint2 ks = make_uint2(0, 0), vs = make_uint2(0, 0);
    const uint8_t* src = row_of(0, page_of(0));
    load4(src ? src + code_off : nullptr, kc);
    load4(src ? src + code_off + 64 : nullptr, vc);
    if (src) {
      ks = *reinterpret_cast<const uint2*>(src + scale_off);
      vs = *reinterpret_cast<const uint2*>(src + scale_off + 8);
    }
    int page_next = page_of(1);
    // ---- Q: fp16 rows scaled by a power of two; rows past the tile are zero
#pragma unroll 1
    for (int t = 0; t < 2; ++t) {
      const int tok = row >> a.g_log2, g = row & (G - 1);
      uint8_t* tile = smem + F4Smem::Q0 + t * kTcTileBytes;
      float f = 1.f, inv = 1.f;
      const bool have = tok < nq_t[t];
      const uint4* qrow = reinterpret_cast<const uint4*>(a.q + ((size_t)(q0 + tb + t * TT + tok) * a.Hq + h * G + g) * kTcD);
      float amax = 0.f;
      if (have) {
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {
          const uint4 v = qrow[c];
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(u[e] << 16)), fabsf(__uint_as_float(u[e] & 0xffff0000u))));
        }
      }
      fp4_row_factor(amax, f, inv);
      qfac[t * 128 + row] = inv * a.qscale;
#pragma unroll 4
      for (int c = 0; c < 16; ++c) {
        uint4 v = have ? qrow[c] : make_uint4(0, 0, 0, 0);
        uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          u[e] = pack_h2(__uint_as_float(u[e] << 16) * f, __uint_as_float(u[e] & 0xffff0000u) * f);
        *reinterpret_cast<uint4*>(tile + (c >> 3) * kTcHalfBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
            make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
    fence_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    for (int j = 0; j < nb; ++j) {
      const int st = j & 1;
      const uint32_t ph = (uint32_t)(j >> 1) & 1u;
      if (!__all_sync(FULL, tc_wait(&k_empty[st], ph ^ 1u, abort_flag))) break;
      f4_expand_row(smem + F4Smem::K0 + st * kTcTileBytes, row, kc, ks);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[st]);
      // the next block's row: its page id was read a block ago
      src = row_of(j + 1, page_next);
      page_next = page_of(j + 2);
      load4(src ? src + code_off : nullptr, kc);
      ks = src ? *reinterpret_cast<const uint2*>(src + scale_off) : make_uint2(0, 0);
      if (!__all_sync(FULL, tc_wait(&v_empty[st], ph ^ 1u, abort_flag))) break;
      f4_expand_row(smem + F4Smem::V0 + st * kTcTileBytes, row, vc, vs);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
      load4(src ? src + code_off + 64 : nullptr, vc);
      vs = src ? *reinterpret_cast<const uint2*>(src + scale_off + 8) : make_uint2(0, 0);
    }
  } else {
    // ---------------------------------------------------------------- softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    constexpr unsigned FULL = 0xffffffffu;
    const int t = (warp - 4) >> 2;              // tile of this warpgroup
    const int row = (threadIdx.x - 128) & 127;  // TMEM lane = tile row
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off;
    const uint32_t tO = tmem + 256 + t * 128 + lane_off;
    const int tok = row >> a.g_log2;
    const int lim_abs = min(prefix + tb + t * TT + tok, Lkv - 1);  // last visible key of this row
    float m = kNegInf, l = 0.f;
    bool ok = true;
    const int my_nb = nb_t[t];
    float qscale = 0.f;
    if (my_nb > 0) {
      ok = __all_sync(FULL, tc_wait(q_full, 0, abort_flag));
      qscale = qfac[t * 128 + row];
    }
    for (int j = 0; j < my_nb && ok; ++j) {
      ok = __all_sync(FULL, tc_wait(&s_full[t], (uint32_t)j & 1u, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const int limit = lim_abs - (b0 + j) * kTcKeys;  // columns 0..limit are visible
      const bool full = limit >= kTcKeys - 1;
      // pass 1: raw row max over the visible columns
      float mxs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mxs[i] = kNegInf;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t ua[32], ub[32];
        tmem_ld32(tS + half * 64, ua);
        tmem_ld32(tS + half * 64 + 32, ub);
        tmem_wait_ld();
        if (!full) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (half * 64 + i > limit) ua[i] = __float_as_uint(kNegInf);
            if (half * 64 + 32 + i > limit) ub[i] = __float_as_uint(kNegInf);
          }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          mxs[(i >> 2) & 7] = max3f(mxs[(i >> 2) & 7], __uint_as_float(ua[i]), __uint_as_float(ua[i + 1]));
          mxs[(i >> 2) & 7] = max3f(mxs[(i >> 2) & 7], __uint_as_float(ua[i + 2]), __uint_as_float(ua[i + 3]));
          mxs[(i >> 2) & 7] = max3f(mxs[(i >> 2) & 7], __uint_as_float(ub[i]), __uint_as_float(ub[i + 1]));
          mxs[(i >> 2) & 7] = max3f(mxs[(i >> 2) & 7], __uint_as_float(ub[i + 2]), __uint_as_float(ub[i + 3]));
        }
      }
      const float mx = fmaxf(max3f(mxs[0], mxs[1], mxs[2]), fmaxf(max3f(mxs[3], mxs[4], mxs[5]), fmaxf(mxs[6], mxs[7])));
      // the reference m stays 7 below the score that set it (decode_fp4.cuh)
      const float m_blk = mx * qscale - 7.f;  // qscale > 0 keeps the order
      float alpha = 1.f;
      if (m == kNegInf) {
        m = m_blk;
      } else if (m_blk - m > 8.f) {
        alpha = ex2_approx(m - m_blk);
        m = m_blk;
      }
      // O_t is stable here: s_full for this block implies PV_t of the previous block finished
      if (j > 0 && __any_sync(FULL, alpha != 1.f)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t u[32];
          tmem_ld32(tO + c * 32, u);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * alpha);
          tmem_st32(tO + c * 32, u);
        }
      }
      // pass 2: p = 2^(s * scale - m), packed to fp16 pairs over the first 64 columns of S.
      // A row that has seen no key yet (m = -inf) has every column masked below.
      const float msub = m == kNegInf ? 0.f : m;
      const uint64_t sc2 = f2(qscale, qscale);
      const uint64_t nm2 = f2(-msub, -msub);
      uint64_t ps2[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
      uint32_t ua[32], ub[32];
      tmem_ld32(tS, ua);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t(&cur)[32] = (c & 1) ? ub : ua;
        uint32_t(&nxt)[32] = (c & 1) ? ua : ub;
        if (c < 3) tmem_ld32(tS + (c + 1) * 32, nxt);
        uint32_t pk[16];
        float xv[32];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          f2_split(f2_fma(f2(__uint_as_float(cur[2 * i]), __uint_as_float(cur[2 * i + 1])), sc2, nm2), xv[2 * i], xv[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 32; ++i) xv[i] = ex2_approx(xv[i]);
        if (!full) {
#pragma unroll
          for (int i = 0; i < 32; ++i) xv[i] = (c * 32 + i <= limit) ? xv[i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          ps2[i & 3] = f2_add(ps2[i & 3], f2(xv[2 * i], xv[2 * i + 1]));
          pk[i] = pack_h2(xv[2 * i], xv[2 * i + 1]);
        }
        // P columns [16c, 16c+16): every S column below 32(c+1) has been read
        tmem_st16(tS + c * 16, pk);
        if (c & 1) {
          // release this half of P to the PV MMA while the rest is computed
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&p_full[t * 4 + (c >> 1)]);
            asm volatile("red.release.cta.shared::cta.add.u32 [%0], 1;" ::"r"(smem_u32(&pcnt[t * 4 + (c >> 1)])) : "memory");
          }
        }
        if (c < 3) tmem_wait_ld();
      }
      const uint64_t s01 = f2_add(f2_add(ps2[0], ps2[1]), f2_add(ps2[2], ps2[3]));
      float lo, hi;
      f2_split(s01, lo, hi);
      l = l * alpha + (lo + hi);
    }
    // ---- epilogue: O_t / l -> bf16 rows, or the unnormalised rows of a split item
    const bool got = __all_sync(FULL, mbar_wait(mma_done, 0, kWdExtendBar));
    tc_fence_after();
    const int g = row & (G - 1);
    const size_t part = ((size_t)item * a.Hkv + h) * a.n_split;  // first split of this item and head
    if (a.n_split == 1) {
      if (ok && got && nq_t[t] > 0) {
        const float inv = l > 0.f ? a.v_scale / l : 0.f;
        __nv_bfloat16* dst = a.out + ((size_t)(q0 + tb + t * TT + tok) * a.Hq + h * G + g) * kTcD;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t u[32];
          if (my_nb > 0) {
            tmem_ld32(tO + c * 32, u);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = 0u;
          }
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(__uint_as_float(u[2 * i]) * inv, __uint_as_float(u[2 * i + 1]) * inv);
          if (tok < nq_t[t]) {
            uint4* d4 = reinterpret_cast<uint4*>(dst + c * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) d4[i] = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
          }
        }
      }
    } else {
      const size_t mine = (part + blockIdx.z) * 256 + t * 128 + row;
      if (my_nb > 0 && ok && got) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t u[32];
          tmem_ld32(tO + c * 32, u);
          tmem_wait_ld();
          if (tok < nq_t[t]) {
            uint4* d4 = reinterpret_cast<uint4*>(a.ws_acc + mine * kTcD + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) d4[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
          }
        }
      }
      if (tok < nq_t[t]) *reinterpret_cast<float2*>(a.ws_ml + mine * 2) = make_float2(l != l ? 0.f : (l > 0.f ? m : kNegInf), l);
      __threadfence();  // publish this row at GPU scope before the ticket
      named_bar_sync(1, 256);
      if (threadIdx.x == 128) {
        const int prev = atomicAdd(&a.tickets[(size_t)item * a.Hkv + h], 1);
        const bool last = prev == a.n_split - 1;
        if (last) a.tickets[(size_t)item * a.Hkv + h] = 0;  // re-armed for the next call
        *s_last = last ? 1 : 0;
      }
      named_bar_sync(1, 256);
      if (*s_last) {
        __threadfence();
        // one warp per row: its partials in run order, read through L2 (other SMs wrote them)
        for (int i = warp - 4; i < 256; i += 8) {
          const int tt = i >> 7, rr = i & 127, tk = rr >> a.g_log2;
          if (tk >= nq_t[tt]) continue;
          float M = kNegInf, Ls = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int s = 0; s < a.n_split; ++s) {
            const size_t pr = (part + s) * 256 + i;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.ws_ml + pr * 2));
            if (ml.x == kNegInf) continue;
            const float4 v = __ldcg(reinterpret_cast<const float4*>(a.ws_acc + pr * kTcD) + lane);
            const float Mn = fmaxf(M, ml.x);
            const float keep = M == kNegInf ? 0.f : exp2f(M - Mn), wgt = exp2f(ml.x - Mn);
            Ls = Ls * keep + ml.y * wgt;
            acc.x = acc.x * keep + v.x * wgt;
            acc.y = acc.y * keep + v.y * wgt;
            acc.z = acc.z * keep + v.z * wgt;
            acc.w = acc.w * keep + v.w * wgt;
            M = Mn;
          }
          const float inv = Ls > 0.f ? a.v_scale / Ls : (Ls != Ls ? Ls : 0.f);
          __nv_bfloat16* dst = a.out + ((size_t)(q0 + tb + tt * TT + tk) * a.Hq + h * G + (rr & (G - 1))) * kTcD;
          reinterpret_cast<uint2*>(dst)[lane] = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

}  // namespace b2a

namespace b2a {

inline bool extend_fp4_tc_supported(int Hq, int Hkv, int D, int dtype) { return extend_tc_supported(Hq, Hkv, D, dtype); }

// Runs of key blocks per work item: as many as fill the SMs once (one CTA per SM), while a
// run keeps at least two blocks of keys.
inline int extend_fp4_splits(int64_t ctas, int sms, int64_t max_kv) {
  const int64_t fill = ctas > 0 ? sms / ctas : 1;
  const int64_t runs = (max_kv + 2 * kTcKeys - 1) / (2 * kTcKeys);
  return (int)std::max<int64_t>(1, std::min<int64_t>({fill, runs, 64}));
}

}  // namespace b2a

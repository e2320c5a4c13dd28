// Ragged causal extend attention over the 4-bit KV pool on tcgen05 tensor cores
// (bf16 or fp32 queries, head_dim 64, 128 or 256, GQA group 1, 2, 4 or 8, any page size).
//
//   O = softmax(scale * Q K^T, causal to the bottom right) V,   K, V of fp4_kv.cuh
//
// A 128-row tile packs 128 / G query tokens x the G heads of a kv head (extend_tc.cuh). A CTA
// runs two streams (one at head_dim 256, whose accumulators fill TMEM), each with its own S, P
// and O in TMEM and its own softmax warpgroup, one thread per row:
//   wide    an item of more than one tile: stream t owns tile t, both read every key block
//   narrow  an item of one tile: both streams own it, stream t reads the key blocks of parity t,
//           and their (m, l, O) are joined at the end, so that one stream's MMAs have the
//           other's softmax to run under
// MMA order of a stream: the PV product of a block, then its next S, so one stream's MMAs run
// under the other's softmax. A commit covers every earlier MMA of its thread, so s_full of a
// stream's next block also says that its PV has finished.
//
// K and V come from a warpgroup that expands them: a thread owns a key (K and V of one row; at
// 64 keys a block, K or V of it; page ids are looked up per key, so any page size works). Its
// warp copies the raw rows of its keys to shared memory (cp.async), the thread takes its row
// into registers and writes fp16 rows into the SWIZZLE_128B tiles that the MMAs read. The next
// block's copies go out as soon as the registers hold this one.
// code * s is exact in fp16 (fp4_kv.cuh), and so is a bf16 q after a power of two per row
// (decode_fp4.cuh), undone in the row's softmax scale: the products are exact. fp32 q and P are
// split into two fp16 parts each (22 bits): S sums two products per step and PV two, over blocks
// of 64 keys so that both parts of P find room beside S.
//
// Few rows on long prefixes leave most SMs idle, so the keys of an item can be cut into runs of
// run_keys keys (grid z). Each run writes its unnormalised rows and (m, l) to a workspace;
// the CTA that takes the item's last ticket joins them, in run order. Nothing waits for another
// CTA. The rows of run z of an item lie at place z of the item's n_split, or, in a smaller
// workspace (PACKED), behind the runs of the items before it: every warp of a split item counts
// those (f4_runs of each), and an item that finds no place for two runs is not cut. A variant of
// its own: with the count in front 8 requests of 1 to 16 new tokens take 102.8 us instead of 100.5.
//
// What bounds it (clock stamps, 16 query / 8 kv heads x 128): a wide block takes about 4,300
// clocks, 2,650 of them without the softmax, 3,900 without the expansion; the MMAs alone are
// 2,048. The softmax chain of a tile is the longer pole, as in extend_tc.cuh, and every CTA adds
// about 14,000 clocks of set-up, Q conversion and epilogue. 32 requests of 64 to 512 new tokens
// on prefixes up to 4,608 run in 259 us (637 TFLOP/s of visible work). A narrow block takes about
// 2,800 clocks, 2,500 of the expanding warps' and the issuers' waits in turn: 8 requests of 1 to
// 16 new tokens on 6,000 to 16,000 cached ones run in 100 us.
//
// Register split: 512 threads launch with 128 registers (65,536 in all); the softmax warpgroups
// take 168 each, the expanding one 112, the issuer's 64: 512 x 128 again.
#pragma once

#include "decode_fp4.cuh"
#include "extend_tc.cuh"
#include "fp4_kv.cuh"

namespace b2a {

constexpr int kF4Threads = 512;
constexpr int kF4Rows = 256;  // most partial rows of a run in the workspace (two tiles)

struct F4Args {
  const void* q;
  const uint8_t* pool;
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* kv_last_page_len;
  const int32_t* work;
  void* out;
  float* ws_acc;     // [item][head][run][F4Cfg::ROWS][D], or packed: [runs of the items][head][run] ..
  float* ws_ml;      // [item][head][run][F4Cfg::ROWS][2], alike
  int32_t* tickets;  // [item][head]
  int64_t num_slots;
  uint32_t row_bytes;
  int page_log2;
  int T, B;  // rows of q, requests (bounds of the work list)
  int Hq, Hkv, G, g_log2;
  int n_split;   // most runs of an item (grid z)
  int run_keys;  // keys of a run
  int ws_runs;   // packed workspace: runs of a head that it holds (0: n_split places for every item)
  int item0;     // index of this launch's first work item
  float qscale;  // scale * k_scale * log2(e)
  float v_scale;
};

template <int D, bool F32>
struct F4Cfg {
  static constexpr int KB = (F32 || D == 256) ? 64 : 128;  // keys of a block
  static constexpr int NS = D == 256 ? 1 : 2;     // streams
  static constexpr int STAGES = (F32 && D == 256) ? 1 : 2;  // K and V tiles in flight
  static constexpr bool WIDE = !F32 && D <= 128;  // items of two tiles
  static constexpr int ROWS = WIDE ? 256 : 128;  // rows of an item
  static constexpr uint32_t QTILE = 128u * D * 2u;
  static constexpr uint32_t KTILE = (uint32_t)KB * D * 2u;
  static constexpr int QTILES = (WIDE || F32) ? 2 : 1;  // two tiles, or the two parts of one
  static constexpr uint32_t QHALF = 128u * 128u;        // bytes between 64-feature columns of a tile
  static constexpr uint32_t KHALF = (uint32_t)KB * 128u;
  static constexpr int O_COL = NS * 128;  // TMEM columns: S_t at 128 t, O_t behind them
  static constexpr int PLO_COL = 64;      // fp32: low part of P beside S (64 columns)
  static constexpr uint32_t K0 = QTILES * QTILE;
  static constexpr uint32_t V0 = K0 + STAGES * KTILE;
  // raw rows: code bytes of K and V (of one of them at 64 keys a block), then the scales
  static constexpr int CODE_BYTES = KB == 128 ? D : D / 2;
  static constexpr int SCALE_BYTES = CODE_BYTES / 8;
  static constexpr uint32_t RAW_PITCH = CODE_BYTES + 16;  // 16-byte reads of 8 rows hit 32 banks
  static constexpr uint32_t RAW = V0 + STAGES * KTILE;
  static constexpr uint32_t BARS = RAW + 128 * RAW_PITCH;
  // q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], mma_done at 13, p_full at 14
  static constexpr int NBARS = 22;
  static constexpr uint32_t TMEM_SLOT = BARS + NBARS * 8;
  static constexpr uint32_t ABORT = TMEM_SLOT + 8;
  static constexpr uint32_t PCNT = ABORT + 8;
  static constexpr uint32_t LAST = PCNT + 32;
  static constexpr uint32_t QFAC = LAST + 16;    // float [2][128]: softmax scale of each row
  static constexpr uint32_t ML = QFAC + 1024;    // float2 [128]: (m, l) of stream 1 (narrow)
  static constexpr uint32_t TOTAL = ML + 1024;
  static constexpr uint32_t ALLOC = TOTAL + 1024;
  static_assert(ALLOC <= 232448, "tiles must fit in shared memory");
  // after the last MMA: stream 1's fp32 rows pass through the Q tiles, output rows through K and V
  static_assert(NS == 1 || 128u * D * 4u <= K0, "stream 1's rows must fit in the Q tiles");
  static_assert(NS == 1 || (WIDE ? 2u : 1u) * 128u * D * (F32 ? 4u : 2u) <= 2u * STAGES * KTILE, "output rows must fit");
};

// Whole-warp wait on an mbarrier phase: one try first, the abort flag and the bounded wait of
// extend_tc.cuh only behind it (a wait whose phase is complete is on every role's critical path).
__device__ __forceinline__ bool f4_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// MMAs whose SWIZZLE_128B descriptors (sw128_desc) come as words: lo holds the address and the
// LBO, hi the rest, which does not change. ACC: add to D.
template <bool ACC>
__device__ __forceinline__ void f4_mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "n"(ACC ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void f4_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// fp16 x fp16 -> fp32, M = 128, N = n.
__host__ __device__ constexpr uint32_t f4_idesc(bool b_mn_major, int n) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Asynchronous copy of N (4, 8 or 16) bytes to shared memory; zeros when `have` is false.
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool have) {
  const int n = have ? N : 0;
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Codes (D/2 bytes) and scales (D/16 bytes, packed in words) of one row -> D fp16 in row `row`
// of a SWIZZLE_128B tile whose 64-feature columns lie `half` bytes apart.
template <int D>
__device__ __forceinline__ void f4_expand_row(uint8_t* tile, uint32_t half, int row, const uint4* c,
                                              const uint32_t* sc) {
  const uint32_t base = (uint32_t)row * 128u;
  const uint32_t x = (uint32_t)(row & 7);
#pragma unroll
  for (int q = 0; q < D / 32; ++q) {  // 16 code bytes: two blocks of 16 features
    const uint32_t s01 = fp4_scale2_to_h2((sc[q >> 1] >> ((q & 1) * 16)) & 0xffffu);
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
      *reinterpret_cast<uint4*>(tile + (chunk >> 3) * half + base + (((uint32_t)(chunk & 7) ^ x) << 4)) =
          make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}

// Runs that a work item's nb key blocks (of KB keys) are cut into.
template <int KB>
__device__ __forceinline__ int f4_runs(const F4Args& a, int nb) {
  const int run = max(1, a.run_keys / KB);
  return a.n_split > 1 ? max(1, min(a.n_split, (nb + run - 1) / run)) : 1;
}

// Runs of the cut items among [0, item), by a whole warp: the kernel's own arithmetic for each.
template <int KB>
__device__ int f4_runs_before(const F4Args& a, int item, int tokens, int lane) {
  int sum = 0;
  for (int i = lane; i < item; i += 32) {
    const int4 w = reinterpret_cast<const int4*>(a.work)[i];
    if (w.z <= 0 || w.x < 0 || w.x >= a.B || w.y < 0) continue;
    const int q0 = a.qo_indptr[w.x], nq = min(min(w.z, tokens), q0 < 0 ? 0 : a.T - q0 - w.y);
    if (nq <= 0) continue;
    const int npages = a.kv_indptr[w.x + 1] - a.kv_indptr[w.x];
    const int Lkv = npages > 0 ? ((npages - 1) << a.page_log2) +
                                     (a.kv_last_page_len ? a.kv_last_page_len[w.x] : 1 << a.page_log2) : 0;
    const int prefix = Lkv - (a.qo_indptr[w.x + 1] - q0);
    const int n = f4_runs<KB>(a, (max(0, min(Lkv, prefix + w.y + nq)) + KB - 1) / KB);
    sum += n > 1 ? n : 0;
  }
  return __reduce_add_sync(0xffffffffu, sum);
}

template <int D, bool F32, bool PACKED>
__global__ void __launch_bounds__(kF4Threads, 1) extend_fp4_tc_kernel(const F4Args a) {
  using C = F4Cfg<D, F32>;
  using T = std::conditional_t<F32, float, __nv_bfloat16>;
  constexpr int KB = C::KB;
  constexpr unsigned FULL = 0xffffffffu;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;   // [2]
  uint64_t* k_empty = bars + 3;  // [2]
  uint64_t* v_full = bars + 5;   // [2]
  uint64_t* v_empty = bars + 7;  // [2]
  uint64_t* s_full = bars + 9;   // [2] per stream
  uint64_t* mma_done = bars + 13;
  uint64_t* p_full = bars + 14;  // [stream * 4 + half]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::TMEM_SLOT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::ABORT);
  uint32_t* pcnt = reinterpret_cast<uint32_t*>(smem + C::PCNT);
  volatile int* s_last = reinterpret_cast<volatile int*>(smem + C::LAST);
  float* qfac = reinterpret_cast<float*>(smem + C::QFAC);
  float2* ml1 = reinterpret_cast<float2*>(smem + C::ML);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.G;
  const int TT = kTcRows >> a.g_log2;  // tokens per tile
  const int item = a.item0 + blockIdx.y;
  const int4 w = reinterpret_cast<const int4*>(a.work)[item];
  if (w.z <= 0) return;  // unused entry behind a device-built work list
  const int r = w.x, tb = w.y;
  if (r < 0 || r >= a.B || tb < 0) {
    if (threadIdx.x == 0) watchdog_set(kWdBadPlan);
    return;
  }
  const int q0 = a.qo_indptr[r];
  // the tile's tokens, inside the kernel's tile and the rows of q
  const int nq = min(min(w.z, C::WIDE ? 2 * TT : TT), q0 < 0 ? 0 : a.T - q0 - tb);
  if (nq < w.z && threadIdx.x == 0) watchdog_set(kWdTileTooLarge);
  if (nq <= 0) return;
  const bool wide = C::WIDE && nq > TT;
  const int nq_t[2] = {min(nq, TT), wide ? nq - TT : min(nq, TT)};  // tokens of each stream's tile
  const int h = blockIdx.x;
  const int P = 1 << a.page_log2;
  const int Lq = a.qo_indptr[r + 1] - q0;
  const int pbeg = a.kv_indptr[r];
  const int npages = a.kv_indptr[r + 1] - pbeg;
  const int Lkv = npages > 0 ? ((npages - 1) << a.page_log2) + (a.kv_last_page_len ? a.kv_last_page_len[r] : P) : 0;
  const int prefix = Lkv - Lq;
  // key blocks of the item, and this CTA's run of them: [b0, b0 + nb)
  const int nb_all = (max(0, min(Lkv, prefix + tb + nq)) + KB - 1) / KB;
  const int run = max(1, a.run_keys / KB);
  int runs = f4_runs<KB>(a, nb_all);
  size_t part = 0;  // first run of this item and head, in a packed workspace
  if constexpr (PACKED) {
    if (runs > 1) {
      const int off = min(a.ws_runs, f4_runs_before<KB>(a, item, C::WIDE ? 2 * TT : TT, lane));
      runs = min(runs, a.ws_runs - off);
      if (runs < 2) runs = 1;
      part = (size_t)off * a.Hkv + (size_t)h * runs;
    }
  }
  if ((int)blockIdx.z >= runs) return;
  const int b0 = blockIdx.z * run;
  const int nb = ((int)blockIdx.z == runs - 1 ? nb_all : b0 + run) - b0;
  // blocks of each stream: wide, those its own rows need; narrow, every other one
  int nb_t[2];
  if (wide) {
    const int end0 = max(0, min(Lkv, prefix + tb + TT));  // tile 0 is full
    nb_t[0] = max(0, min((end0 + KB - 1) / KB - b0, nb));
    nb_t[1] = nb;
  } else {
    nb_t[0] = C::NS == 2 ? (nb + 1) >> 1 : nb;
    nb_t[1] = C::NS == 2 ? nb >> 1 : 0;
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], KB / 32);  // one arrive per expanding warp
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], KB / 32);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      for (int c = 0; c < 2; ++c) mbar_init(&p_full[i * 4 + c], 4);  // one arrive per softmax warp
    }
    mbar_init(mma_done, wide ? 1 : C::NS);  // one arrive per issuer
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
    if (warp == 0 || (warp == 2 && C::NS == 2 && !wide)) {
      // ---------------------------------------------------------------- MMA issuer
      // The whole warp runs the loop and one elected lane issues, so addresses and descriptors
      // stay warp-uniform.
      // Narrow: a thread per stream. MMAs block their issuer while the tensor pipe is busy, so
      // with one thread the waits of one stream would hold up the other's MMAs. Wide: one thread
      // for both. Two fall into step on the blocks they share, and both softmax warpgroups then
      // compete for the exponential units while the tensor cores idle (317 against 281 us on
      // the ragged batch); one thread's fixed order keeps them half a block apart.
      const int mine_t = warp >> 1;
      constexpr uint32_t idesc_qk = f4_idesc(false, KB);
      constexpr uint32_t idesc_pv = f4_idesc(true, D);
      auto slot = [](int j) { return C::STAGES == 2 ? j & 1 : 0; };
      auto phase = [](int j) { return (uint32_t)(C::STAGES == 2 ? j >> 1 : j) & 1u; };
      auto k_ready = [&](int j) -> bool {
        if (!f4_wait(&k_full[slot(j)], phase(j), abort_flag)) return false;
        tc_fence_after();
        return true;
      };
      const bool leader = elect_one();
      constexpr uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);  // SBO, version, swizzle
      const uint32_t base = (smem_u32(smem) & 0x3FFFFu) >> 4;
      constexpr uint32_t lbo_k = (16u >> 4) << 16, lbo_v = (C::KHALF >> 4) << 16;
      auto issue_s = [&](int t, int j) {
        const uint32_t aq = base + ((wide ? t * C::QTILE : 0u) >> 4) + lbo_k;
        const uint32_t bk = base + ((C::K0 + slot(j) * C::KTILE) >> 4) + lbo_k;
        const uint32_t d = tmem + t * 128;
        if (leader) {
          f4_mma_ss<false>(d, aq, bk, desc_hi, idesc_qk);
#pragma unroll
          for (int kk = 1; kk < D / 16; ++kk)
            f4_mma_ss<true>(d, aq + (((kk >> 2) * C::QHALF + (kk & 3) * 32) >> 4),
                            bk + (((kk >> 2) * C::KHALF + (kk & 3) * 32) >> 4), desc_hi, idesc_qk);
          if constexpr (F32) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              f4_mma_ss<true>(d, aq + ((C::QTILE + (kk >> 2) * C::QHALF + (kk & 3) * 32) >> 4),
                              bk + (((kk >> 2) * C::KHALF + (kk & 3) * 32) >> 4), desc_hi, idesc_qk);
          }
          tc_commit(&s_full[t]);
        }
        __syncwarp();
      };
      // P of a half released by all 4 softmax warps: an acquire load of the release count
      // instead of an mbarrier wait (extend_tc.cuh)
      auto p_done = [&](int idx, int jl) -> bool {
        uint32_t v;
        asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(&pcnt[idx])) : "memory");
        return __all_sync(FULL, v >= 4u * (uint32_t)(jl + 1));
      };
      auto issue_pv = [&](int t, int j, int jl, int half) {
        const uint32_t bv = base + ((C::V0 + slot(j) * C::KTILE) >> 4) + lbo_v;
        const uint32_t d = tmem + C::O_COL + t * D, p = tmem + t * 128;
        if (leader) {
#pragma unroll
          for (int q = 0; q < KB / 32; ++q) {
            const int kk = half * (KB / 32) + q;
            f4_mma_ts(d, p + kk * 8, bv + kk * (2048 >> 4), desc_hi, idesc_pv, (jl > 0 || kk > 0) ? 1u : 0u);
            if constexpr (F32) f4_mma_ts(d, p + C::PLO_COL + kk * 8, bv + kk * (2048 >> 4), desc_hi, idesc_pv, 1u);
          }
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (leader) tc_commit(bar);
        __syncwarp();
      };
      // the PV product of a stream's block jl, once its P is there
      auto pv = [&](int t, int j, int jl) -> bool {
        if (p_done(t * 4 + 1, jl)) {
          tc_fence_after();
          issue_pv(t, j, jl, 0);
          issue_pv(t, j, jl, 1);
          return true;
        }
        for (int half = 0; half < 2; ++half) {
          if (!p_done(t * 4 + half, jl) && !f4_wait(&p_full[t * 4 + half], (uint32_t)jl & 1u, abort_flag)) return false;
          tc_fence_after();
          issue_pv(t, j, jl, half);
        }
        return true;
      };
      bool ok = f4_wait(q_full, 0, abort_flag);
      if (wide) {
        if (ok && nb > 0 && (ok = k_ready(0))) {
          for (int t = 0; t < 2; ++t)
            if (nb_t[t] > 0) issue_s(t, 0);
          commit(&k_empty[0]);
        }
        for (int j = 0; j < nb && ok; ++j) {
          ok = f4_wait(&v_full[slot(j)], phase(j), abort_flag);
          bool k_next = false;
          for (int t = 0; t < 2 && ok; ++t) {
            if (j < nb_t[t]) ok = pv(t, j, j);
            if (ok && j + 1 < nb_t[t]) {
              if (!k_next) ok = k_next = k_ready(j + 1);
              if (ok) issue_s(t, j + 1);
            }
          }
          if (!ok) break;
          commit(&v_empty[slot(j)]);
          if (k_next) commit(&k_empty[slot(j + 1)]);
        }
      } else {
        // this stream's blocks: t, t + 2, .. of two streams, or all
        const int t = mine_t, first = t, step = C::NS, mine = nb_t[t];
        if (ok && mine > 0 && (ok = k_ready(first))) {
          issue_s(t, first);
          commit(&k_empty[slot(first)]);
        }
        for (int jl = 0; jl < mine && ok; ++jl) {
          const int j = first + jl * step;
          ok = f4_wait(&v_full[slot(j)], phase(j), abort_flag) && pv(t, j, jl);
          if (!ok) break;
          commit(&v_empty[slot(j)]);
          if (jl + 1 < mine && (ok = k_ready(j + step))) {
            issue_s(t, j + step);
            commit(&k_empty[slot(j + step)]);
          }
        }
      }
      // every MMA issued above has completed once mma_done fires (also on the abort path)
      commit(mma_done);
      mbar_wait(mma_done, 0, kWdExtendDrain);
    }
  } else if (warp >= 12) {
    // ---------------------------------------------------------------- expanding warpgroup
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    const int th = threadIdx.x - 384;
    const int row = th & (KB - 1);  // key of a block
    const bool do_k = KB == 128 || th < 64;  // at 64 keys a block: K or V of this key
    const uint32_t code_off = fp4_code_off(h, D) + (do_k ? 0 : D / 2);
    const uint32_t scale_off = fp4_scale_off(h, a.Hkv, D) + (do_k ? 0 : D / 16);
    // page id and pool slot of this lane's key of block j: -1 past the last key or for a bad
    // page id, which is recorded and read as zeros
    auto page_of = [&](int j) -> int {
      const int key = (b0 + j) * KB + row;
      return j < nb && key < Lkv ? a.kv_indices[pbeg + (key >> a.page_log2)] : -1;
    };
    auto slot_of = [&](int j, int page) -> int {
      const int key = (b0 + j) * KB + row;
      if (j >= nb || key >= Lkv) return -1;
      const int64_t sl = (int64_t)page * P + (key & (P - 1));
      if (page < 0 || sl >= a.num_slots) {
        watchdog_set(kWdBadSlot);
        return -1;
      }
      return (int)sl;
    };
    // A warp copies the raw bytes of its own 32 keys: NCH lanes take the 16-byte chunks of one
    // row, so a copy touches 32 / NCH rows instead of 32 (a lane loading its own row costs the
    // load unit 32 lines per instruction: 342 against 281 us on the ragged batch of 32 requests).
    constexpr int NCH = C::CODE_BYTES / 16;
    uint8_t* raw = smem + C::RAW + (uint32_t)(th & ~31) * C::RAW_PITCH;
    auto fetch = [&](int sl) {
      const uint32_t dst = smem_u32(raw);
#pragma unroll
      for (int it = 0; it < NCH; ++it) {
        const int rr = it * (32 / NCH) + lane / NCH, ch = lane % NCH;
        const int s2 = __shfl_sync(FULL, sl, rr);
        cp_async<16>(dst + rr * C::RAW_PITCH + ch * 16, a.pool + (size_t)max(s2, 0) * a.row_bytes + code_off + ch * 16, s2 >= 0);
      }
      cp_async<C::SCALE_BYTES>(dst + lane * C::RAW_PITCH + C::CODE_BYTES,
                               a.pool + (size_t)max(sl, 0) * a.row_bytes + scale_off, sl >= 0);
    };
    // One block's codes and scales of this thread's key, out of the raw rows; the next block's
    // rows then travel while this one is expanded (their page ids were read a block ago).
    const uint8_t* mine = raw + lane * C::RAW_PITCH;
    uint4 code[NCH];
    uint32_t sc[C::SCALE_BYTES / 4];
    int page_next = page_of(1);
    auto take = [&](int j) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
#pragma unroll
      for (int i = 0; i < NCH; ++i) code[i] = reinterpret_cast<const uint4*>(mine)[i];
#pragma unroll
      for (int i = 0; i < C::SCALE_BYTES / 4; ++i) sc[i] = reinterpret_cast<const uint32_t*>(mine + C::CODE_BYTES)[i];
      __syncwarp();
      fetch(slot_of(j + 1, page_next));
      page_next = page_of(j + 2);
    };
    auto put = [&](int j, bool is_k, const uint4* c, const uint32_t* s2) -> bool {
      const int st = C::STAGES == 2 ? j & 1 : 0;
      const uint32_t ph = (uint32_t)(C::STAGES == 2 ? j >> 1 : j) & 1u;
      if (!f4_wait(is_k ? &k_empty[st] : &v_empty[st], ph ^ 1u, abort_flag)) return false;
      f4_expand_row<D>(smem + (is_k ? C::K0 : C::V0) + st * C::KTILE, C::KHALF, row, c, s2);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(is_k ? &k_full[st] : &v_full[st]);
      return true;
    };
    fetch(slot_of(0, page_of(0)));
    if constexpr (KB == 128) {
      // K one block ahead of V: a stream's next S needs its K right after the PV that frees V's
      // tile, and V only after the softmax behind that S
      constexpr int NV = D / 32, NVS = D / 64;
      bool ok = true;
      uint4 vc[NV];
      uint32_t vs[NVS];
      if (nb > 0) {
        take(0);
        ok = put(0, true, code, sc);
      }
      for (int j = 0; j < nb && ok; ++j) {
#pragma unroll
        for (int i = 0; i < NV; ++i) vc[i] = code[NV + i];
#pragma unroll
        for (int i = 0; i < NVS; ++i) vs[i] = sc[NVS + i];
        if (j + 1 < nb) {
          take(j + 1);
          ok = put(j + 1, true, code, sc);
        }
        if (ok) ok = put(j, false, vc, vs);
      }
    } else {
      for (int j = 0; j < nb; ++j) {
        take(j);
        if (!put(j, do_k, code, sc)) break;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // never leave while own copies may still be landing
  } else {
    // ---------------------------------------------------------------- softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int t = (warp - 4) >> 2;              // stream of this warpgroup
    const int row = (threadIdx.x - 128) & 127;  // TMEM lane = tile row
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off;
    const uint32_t tO = tmem + C::O_COL + t * D + lane_off;
    const int tile = wide ? t : 0;
    const int tok = row >> a.g_log2;
    const bool live = tok < nq_t[t];
    // a warp whose rows all lie past the tile only keeps the protocol going: its rows of P
    // and O hold anything and are not read
    const bool warp_live = (((warp & 3) * 32) >> a.g_log2) < nq_t[t];
    const int lim_abs = min(prefix + tb + tile * TT + tok, Lkv - 1);  // last visible key of this row
    // ---- Q: fp16 rows scaled by a power of two (two parts for fp32); rows past the tile are
    // zero. D / 8 lanes take a row; wide, a warpgroup converts its own tile, else both share one.
    {
      constexpr int LPR = D / 8, RI = 32 / LPR;  // lanes of a row, rows of a step
      const int rows = wide ? 32 : 16;
      const int r0 = wide ? (warp & 3) * 32 : (warp - 4) * 16;
      uint8_t* qt = smem + (wide ? t * C::QTILE : 0u);
      const int ch = lane % LPR;
      constexpr int GI = F32 || RI == 1 ? 8 : (C::WIDE && RI == 2 ? 16 : 16 / RI);  // steps whose loads go out together
      constexpr int EV = F32 ? 2 : 1;             // 16-byte words of a lane's eight elements
#pragma unroll 1
      for (int i0 = 0; i0 < rows; i0 += GI * RI) {
        uint4 raw[GI][EV];
#pragma unroll
        for (int i = 0; i < GI; ++i) {
          const int rw = r0 + i0 + i * RI + lane / LPR, tk = rw >> a.g_log2;
          const T* src = reinterpret_cast<const T*>(a.q) +
                         ((size_t)(q0 + tb + tile * TT + tk) * a.Hq + h * G + (rw & (G - 1))) * D + 8 * ch;
#pragma unroll
          for (int e = 0; e < EV; ++e)
            raw[i][e] = i0 + i * RI < rows && tk < nq_t[tile] ? reinterpret_cast<const uint4*>(src)[e] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < GI; ++i) {
        if (i0 + i * RI >= rows) break;  // the next warp's rows
        const int rw = r0 + i0 + i * RI + lane / LPR;
        float v[8], amax, f, inv;
        if constexpr (F32) {
          const uint4 x = raw[i][0], y = raw[i][EV - 1];
          const uint32_t w8[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          amax = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = __uint_as_float(w8[e]);
            amax = fmaxf(amax, fabsf(v[e]));
          }
#pragma unroll
          for (int o = LPR / 2; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, o));
        } else {
          const uint32_t w4[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
          // non-negative bf16 pairs order like their bits
          uint32_t mx = __vmaxu2(__vmaxu2(w4[0] & 0x7fff7fffu, w4[1] & 0x7fff7fffu),
                                 __vmaxu2(w4[2] & 0x7fff7fffu, w4[3] & 0x7fff7fffu));
#pragma unroll
          for (int o = LPR / 2; o >= 1; o >>= 1) mx = __vmaxu2(mx, __shfl_xor_sync(FULL, mx, o));
          amax = __uint_as_float(max(mx << 16, mx & 0xffff0000u));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(w4[e] << 16);
            v[2 * e + 1] = __uint_as_float(w4[e] & 0xffff0000u);
          }
        }
        fp4_row_factor(amax, f, inv);
        if (ch == 0) qfac[tile * 128 + rw] = fp4_score_scale(inv, a.qscale);
        uint32_t u[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = v[2 * e] * f, x1 = v[2 * e + 1] * f;
          u[e] = pack_h2(x0, x1);
          if constexpr (F32) {
            const float2 hi = h2_to_f2(u[e]);
            lo[e] = pack_h2(x0 - hi.x, x1 - hi.y);
          }
        }
        const uint32_t off = (ch >> 3) * C::QHALF + rw * 128 + (((ch & 7) ^ (rw & 7)) << 4);
        *reinterpret_cast<uint4*>(qt + off) = make_uint4(u[0], u[1], u[2], u[3]);
        if constexpr (F32) *reinterpret_cast<uint4*>(qt + C::QTILE + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    float m = kNegInf, l = 0.f;
    bool ok = true;
    const int my_nb = t < C::NS ? nb_t[t] : 0;
    float qscale = 0.f;
    if (my_nb > 0) {
      ok = f4_wait(q_full, 0, abort_flag);
      qscale = qfac[tile * 128 + row];
    }
    for (int jl = 0; jl < my_nb && ok; ++jl) {
      ok = f4_wait(&s_full[t], (uint32_t)jl & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const int j = (C::NS == 2 && !wide) ? 2 * jl + t : jl;
      if (!warp_live) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          for (int c = 0; c < 2; ++c) {
            mbar_arrive(&p_full[t * 4 + c]);
            asm volatile("red.release.cta.shared::cta.add.u32 [%0], 1;" ::"r"(smem_u32(&pcnt[t * 4 + c])) : "memory");
          }
        }
        continue;
      }
      const int limit = lim_abs - (b0 + j) * KB;  // columns 0..limit are visible
      const bool full = limit >= KB - 1;
      // pass 1: raw row max over the visible columns
      float mxs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mxs[i] = kNegInf;
#pragma unroll
      for (int half = 0; half < KB / 64; ++half) {
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
      // O_t is stable here: s_full for this block implies that the stream's last PV has finished
      if (jl > 0 && __any_sync(FULL, alpha != 1.f)) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t u[32];
          tmem_ld32(tO + c * 32, u);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * alpha);
          tmem_st32(tO + c * 32, u);
        }
      }
      // pass 2: p = 2^(s * scale - m), packed to fp16 pairs over the first columns of S.
      // A row that has seen no key yet (m = -inf) has every column masked below.
      const float msub = m == kNegInf ? 0.f : m;
      const uint64_t sc2 = f2(qscale, qscale);
      const uint64_t nm2 = f2(-msub, -msub);
      uint64_t ps2[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
      uint32_t ua[32], ub[32];
      tmem_ld32(tS, ua);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < KB / 32; ++c) {
        uint32_t(&cur)[32] = (c & 1) ? ub : ua;
        uint32_t(&nxt)[32] = (c & 1) ? ua : ub;
        if (c < KB / 32 - 1) tmem_ld32(tS + (c + 1) * 32, nxt);
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
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 hi = h2_to_f2(pk[i]);
            pk[i] = pack_h2(xv[2 * i] - hi.x, xv[2 * i + 1] - hi.y);
          }
          tmem_st16(tS + C::PLO_COL + c * 16, pk);
        }
        if (KB == 64 || (c & 1)) {
          // release this half of P to the PV MMA while the rest is computed
          const int half = KB == 64 ? c : c >> 1;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            // the arrive first, then the counted release (extend_tc.cuh)
            mbar_arrive(&p_full[t * 4 + half]);
            asm volatile("red.release.cta.shared::cta.add.u32 [%0], 1;" ::"r"(smem_u32(&pcnt[t * 4 + half])) : "memory");
          }
        }
        if (c < KB / 32 - 1) tmem_wait_ld();
      }
      const uint64_t s01 = f2_add(f2_add(ps2[0], ps2[1]), f2_add(ps2[2], ps2[3]));
      float lo, hi;
      f2_split(s01, lo, hi);
      l = l * alpha + (lo + hi);
    }
    // a row that has seen a key in these blocks has weights, or none that hold (decode_fp4.cuh)
    if (my_nb > 0 && live && lim_abs >= (b0 + (C::NS == 2 && !wide ? t : 0)) * KB && fp4_row_lost(l)) l = kNaN;
    // ---- epilogue
    const bool got = __all_sync(FULL, mbar_wait(mma_done, 0, kWdExtendBar));
    tc_fence_after();
    ok = ok && got;
    // narrow: stream 1's rows go through shared memory (the tiles are no longer read) to stream
    // 0, which joins them with its own. 16-byte chunks are permuted by row against conflicts.
    float4* exch = reinterpret_cast<float4*>(smem);
    constexpr int CH = D / 4;  // chunks of a row
    const bool join = C::NS == 2 && !wide;
    float w0 = 1.f, w1 = 0.f;  // factors of the own and of stream 1's row
    if (join) {
      if (t == 1) {
        const bool any = my_nb > 0 && warp_live && ok;
        if (any) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t u[32];
            tmem_ld32(tO + c * 32, u);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              exch[row * CH + ((c * 8 + i) ^ (row & (CH - 1) & 15))] =
                  make_float4(__uint_as_float(u[4 * i]), __uint_as_float(u[4 * i + 1]), __uint_as_float(u[4 * i + 2]),
                              __uint_as_float(u[4 * i + 3]));
          }
        }
        ml1[row] = make_float2(any ? m : kNegInf, any ? l : 0.f);
      }
      named_bar_sync(1, 256);
      if (t == 0) {
        const float2 o = ml1[row];
        if (o.x != kNegInf || o.y != o.y) {
          if (m == kNegInf && l == l) {
            w0 = 0.f;
            w1 = 1.f;
            m = o.x;
            l = o.y;
          } else {
            const float M = fmaxf(m, o.x);
            w0 = exp2f(m - M);
            w1 = exp2f(o.x - M);
            l = l * w0 + o.y * w1;
            m = M;
          }
        }
      }
    }
    // 32 columns of this row: own accumulator (none without blocks) and stream 1's
    auto columns = [&](int c, float (&v)[32]) {
      uint32_t u[32];
      if (my_nb > 0) {
        tmem_ld32(tO + c * 32, u);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) u[i] = 0u;
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
      if (join && nb_t[1] > 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 x = exch[row * CH + ((c * 8 + i) ^ (row & (CH - 1) & 15))];
          v[4 * i] = v[4 * i] * w0 + x.x * w1;
          v[4 * i + 1] = v[4 * i + 1] * w0 + x.y * w1;
          v[4 * i + 2] = v[4 * i + 2] * w0 + x.z * w1;
          v[4 * i + 3] = v[4 * i + 3] * w0 + x.w * w1;
        }
      }
    };
    const bool writer = t < C::NS && (t == 0 || wide);  // this warpgroup's rows are the item's
    if constexpr (!PACKED) part = ((size_t)item * a.Hkv + h) * a.n_split;
    T* out = reinterpret_cast<T*>(a.out);
    if (runs == 1) {
      if (writer && ok && warp_live) {
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // before the scale: no end of fp32 is near
        // a warp's 32 rows go through shared memory, 16-byte chunks permuted by row, so that a
        // store writes whole rows and not 16 bytes of each of 32
        constexpr int CPR = D * (int)sizeof(T) / 16;  // chunks of a row
        uint4* stage = reinterpret_cast<uint4*>(smem + (C::NS == 1 ? 0u : C::K0) + t * 128u * D * sizeof(T)) +
                       (warp & 3) * 32 * CPR;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          columns(c, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = v[i] * inv * a.v_scale;
          constexpr int CPC = 32 * (int)sizeof(T) / 16;  // chunks of 32 columns
#pragma unroll
          for (int i = 0; i < CPC; ++i) {
            uint4 x;
            if constexpr (F32) {
              x = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                             __float_as_uint(v[4 * i + 3]));
            } else {
              x = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                             pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
            }
            stage[lane * CPR + ((c * CPC + i) ^ (lane & 7))] = x;
          }
        }
        __syncwarp();
        const int row0 = (warp & 3) * 32;
#pragma unroll 4
        for (int i = lane; i < 32 * CPR; i += 32) {
          const int rr = i / CPR, ch = i % CPR, rw = row0 + rr, tk = rw >> a.g_log2;
          if (tk < nq_t[t])
            reinterpret_cast<uint4*>(out + ((size_t)(q0 + tb + tile * TT + tk) * a.Hq + h * G + (rw & (G - 1))) * D)[ch] =
                stage[rr * CPR + (ch ^ (rr & 7))];
        }
      }
    } else {
      const size_t mine = (part + blockIdx.z) * C::ROWS + tile * 128 + row;
      if (writer && ok && warp_live) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float v[32];
          columns(c, v);
          if (live) store_vec<float, 32>(a.ws_acc + mine * D + c * 32, v);
        }
      }
      if (writer && live)
        *reinterpret_cast<float2*>(a.ws_ml + mine * 2) = make_float2(l != l ? 0.f : (l > 0.f && ok ? m : kNegInf), l);
      __threadfence();  // publish this row at GPU scope before the ticket
      named_bar_sync(1, 256);
      if (threadIdx.x == 128) {
        const int prev = atomicAdd(&a.tickets[(size_t)item * a.Hkv + h], 1);
        const bool last = prev == runs - 1;
        if (last) a.tickets[(size_t)item * a.Hkv + h] = 0;  // re-armed for the next call
        *s_last = last ? 1 : 0;
      }
      named_bar_sync(1, 256);
      if (*s_last) {
        __threadfence();
        // one warp per row: its partials in run order, read through L2 (other SMs wrote them)
        constexpr int EPT = D / 32;
        for (int i = warp - 4; i < (wide ? 256 : 128); i += 8) {
          const int tt = i >> 7, rr = i & 127, tk = rr >> a.g_log2;
          if (tk >= nq_t[tt]) continue;
          float M = kNegInf, Ls = 0.f, acc[EPT];
#pragma unroll
          for (int e = 0; e < EPT; ++e) acc[e] = 0.f;
          for (int s0 = 0; s0 < runs; s0 += 4) {
            float2 ml[4], v[4][EPT / 2];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const size_t pr = (part + min(s0 + u, runs - 1)) * C::ROWS + i;
              ml[u] = __ldcg(reinterpret_cast<const float2*>(a.ws_ml + pr * 2));
              if (s0 + u >= runs) ml[u] = make_float2(kNegInf, 0.f);
              const float2* src = reinterpret_cast<const float2*>(a.ws_acc + pr * D + lane * EPT);
#pragma unroll
              for (int e = 0; e < EPT / 2; ++e) v[u][e] = __ldcg(src + e);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if (ml[u].x == kNegInf) continue;  // no visible key in this run: its row was not written
              const float Mn = fmaxf(M, ml[u].x);
              const float keep = M == kNegInf ? 0.f : exp2f(M - Mn), wgt = exp2f(ml[u].x - Mn);
              Ls = Ls * keep + ml[u].y * wgt;
#pragma unroll
              for (int e = 0; e < EPT / 2; ++e) {
                acc[2 * e] = acc[2 * e] * keep + v[u][e].x * wgt;
                acc[2 * e + 1] = acc[2 * e + 1] * keep + v[u][e].y * wgt;
              }
              M = Mn;
            }
          }
          const float inv = Ls > 0.f ? 1.f / Ls : (Ls != Ls ? Ls : 0.f);
#pragma unroll
          for (int e = 0; e < EPT; ++e) acc[e] = acc[e] * inv * a.v_scale;
          store_vec<T, EPT>(out + ((size_t)(q0 + tb + tt * TT + tk) * a.Hq + h * G + (rr & (G - 1))) * D + lane * EPT, acc);
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

// ------------------------------------------------------------ host side
// Partial rows of a run in the workspace.
inline int extend_fp4_rows(int D, bool f32) { return !f32 && D <= 128 ? 256 : 128; }

// Query tokens per work item.
inline int extend_fp4_tile_tokens(int G, int D, bool f32) { return (!f32 && D <= 128 ? 2 : 1) * (kTcRows / G); }

// Cuts the keys of few work items into runs so that the CTAs (items x heads x runs) fill the
// SMs once: the shortest run of whole 128-key blocks, at least four of them, whose count of CTAs
// fits. keys[i]: keys that item i's last token sees. Sets run_keys and the most runs of an item.
inline void extend_fp4_runs(const int32_t* keys, int n_work, int Hkv, int sms, int* run_keys, int* n_split) {
  *run_keys = 0;
  *n_split = 1;
  int64_t most = 0, total = 0;
  for (int i = 0; i < n_work; ++i) {
    const int64_t nb = std::max<int64_t>(1, ((int64_t)keys[i] + 127) / 128);
    most = std::max(most, nb);
    total += nb;
  }
  const int64_t slots = sms / std::max(1, Hkv);  // runs that fit at once
  if (n_work <= 0 || slots <= n_work || most <= 4) return;
  int64_t run = std::max<int64_t>({4, (total + slots - 1) / slots, (most + 63) / 64});
  for (; run < most; ++run) {
    int64_t n = 0;
    for (int i = 0; i < n_work; ++i) n += (std::max<int64_t>(1, ((int64_t)keys[i] + 127) / 128) + run - 1) / run;
    if (n <= slots) break;
  }
  if (run >= most) return;
  *run_keys = (int)(run * 128);
  *n_split = (int)((most + run - 1) / run);
}

}  // namespace b2a

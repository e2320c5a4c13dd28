// Index tables of a prefill batch, built on the device from the requests' lengths.
//
// Replaces the host build of BaseAttnBackend._prepare_prefill
// (python/minisgl_mlx/attention/base.py:70-84), the positions / out_loc lookup of
// scheduler/scheduler.py:155-158 and b2a_extend_plan. For request b with L = lens[b]
// tokens, of which the first cached[b] are in the pool already, E = L - cached[b]:
//   qo_indptr, kv_indptr   exclusive sums of E and of ceil(L / P)
//   positions[qo_b + i]    cached[b] + i              (i < E)
//   out_loc[qo_b + i]      page_table[rows[b], cached[b] + i]
//   kv_indices[kv_b + p]   page_table[rows[b], p P] / P
//   work                   {b, first token, tokens, 0} per tile of tile_q new tokens, by
//                          falling cost tokens * (keys its last token sees), equal costs
//                          in request order
//
// One launch. It moves a few bytes per token and page, so what bounds a usual batch is
// latency: launches, and the chain scan -> search -> table entry. Every CTA therefore
// scans all B requests itself (12 bytes each, from L2) into shared memory instead of
// waiting for another CTA or launch to do it, finds the requests of its slice of tokens,
// pages and tiles by binary search there, and walks on from the first. A tile's place in
// the sorted list is the number of tiles that go before it, counted directly: all keys
// are unique (cost, then order), so no two tiles claim one place and no order of
// execution matters.
#pragma once

#include "common.cuh"

namespace b2a {

constexpr int kEmThreads = 256;
constexpr int kEmMaxBatch = 8192;  // three int32 prefix arrays of a batch in shared memory
constexpr int kEmKeys = 2048;      // tile keys compared per round
constexpr int kEmMaxTile = 256;    // cost < 2^39, so (cost, order) fits 64 bits
constexpr int kEmMaxWork = 1 << 24;
constexpr int kEmVec = 4;          // tokens, pages or tiles a thread walks from one search

struct ExtendMetaArgs {
  const int32_t* page_table;
  int64_t stride, table_rows;
  const int32_t* rows;
  const int32_t* cached;
  const int32_t* lens;
  int B, page_log2, tile_q;
  int32_t* qo_indptr;
  int32_t* positions;
  int32_t* out_loc;
  int64_t q_capacity;
  int32_t* last_indices;
  int32_t* kv_indptr;
  int32_t* kv_indices;
  int64_t idx_capacity;
  int32_t* last_page_len;
  int32_t* work;  // int4
  int work_capacity;
  int32_t* counts;  // [2]: new tokens, tiles
};

__host__ __device__ inline size_t extend_meta_smem(int B) {
  return (size_t)kEmKeys * 8 + 3 * (size_t)(B + 1) * 4;
}

struct EmReq {
  int cached, ext, pages;
};

// Lengths of request b, forced into the table's range (flagged once, by CTA 0).
__device__ __forceinline__ EmReq em_request(const ExtendMetaArgs& a, int b) {
  int L = a.lens[b], c = a.cached[b];
  const bool bad = L < 0 || (int64_t)L > a.stride || c < 0 || c > L || a.rows[b] < 0 || a.rows[b] >= a.table_rows;
  if (bad) {
    if (blockIdx.x == 0) watchdog_set(kWdMetaOverflow);
    L = L < 0 ? 0 : (int)min((int64_t)L, a.stride);
    c = min(max(c, 0), L);
  }
  return {c, L - c, (int)(((int64_t)L + (1 << a.page_log2) - 1) >> a.page_log2)};
}

// Last b in [0, B) with pre[b] <= x (pre ascending, pre[0] = 0): the owner of element x
// when x < pre[B].
__device__ __forceinline__ int em_find(const int32_t* pre, int B, int x) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Key of tile i of request b: dearer tiles and, among equals, earlier tiles are larger.
__device__ __forceinline__ unsigned long long em_key(const ExtendMetaArgs& a, const int32_t* qo, int b, int k, int i,
                                                     int& tb, int& nq) {
  const int ext = qo[b + 1] - qo[b];
  tb = k * a.tile_q;
  nq = min(a.tile_q, ext - tb);
  const unsigned long long cost = (unsigned long long)nq * (unsigned long long)((long long)a.cached[b] + tb + nq);
  return (cost << 24) | (unsigned long long)(kEmMaxWork - 1 - i);
}

__global__ void __launch_bounds__(kEmThreads) extend_meta_kernel(const ExtendMetaArgs a) {
  constexpr unsigned FULL = 0xffffffffu;
  extern __shared__ __align__(16) uint8_t em_smem[];
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(em_smem);
  int32_t* qo = reinterpret_cast<int32_t*>(em_smem + (size_t)kEmKeys * 8);  // [B + 1]
  int32_t* kv = qo + a.B + 1;
  int32_t* tl = kv + a.B + 1;
  __shared__ long long wsum[3][kEmThreads / 32];
  __shared__ int rank_of;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.B;

  // ---- exclusive sums of new tokens, pages and tiles: thread t owns a run of requests
  {
    const int per = (B + kEmThreads - 1) / kEmThreads;
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    long long s[3] = {0, 0, 0};
    for (int b = b0; b < b1; ++b) {
      const EmReq r = em_request(a, b);
      const int tiles = (r.ext + a.tile_q - 1) / a.tile_q;
      qo[b + 1] = r.ext;
      kv[b + 1] = r.pages;
      tl[b + 1] = tiles;
      s[0] += r.ext;
      s[1] += r.pages;
      s[2] += tiles;
    }
    long long inc[3] = {s[0], s[1], s[2]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        const long long y = __shfl_up_sync(FULL, inc[c], o);
        if (lane >= o) inc[c] += y;
      }
    }
    if (lane == 31) {
#pragma unroll
      for (int c = 0; c < 3; ++c) wsum[c][warp] = inc[c];
    }
    __syncthreads();
    long long base[3];
    bool fits = true;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      base[c] = inc[c] - s[c];
      long long all = 0;
      for (int w = 0; w < kEmThreads / 32; ++w) {
        if (w == warp) base[c] += all;
        all += wsum[c][w];
      }
      fits = fits && all <= (c == 2 ? (long long)kEmMaxWork : 0x7fffffffll);
    }
    if (!fits) {  // the same on every thread: the tables stay as they were
      if (blockIdx.x == 0 && tid == 0) watchdog_set(kWdMetaOverflow);
      return;
    }
    for (int b = b0; b < b1; ++b) {
      base[0] += qo[b + 1];
      qo[b + 1] = (int)base[0];
      base[1] += kv[b + 1];
      kv[b + 1] = (int)base[1];
      base[2] += tl[b + 1];
      tl[b + 1] = (int)base[2];
    }
    if (tid == 0) qo[0] = kv[0] = tl[0] = 0;
  }
  __syncthreads();
  const int T = qo[B], NP = kv[B], NT = tl[B];
  const int P = 1 << a.page_log2;
  const int gthreads = gridDim.x * kEmThreads;
  const int gid = blockIdx.x * kEmThreads + tid;

  // ---- per-request outputs
  for (int b = gid; b <= B; b += gthreads) {
    a.qo_indptr[b] = qo[b];
    a.kv_indptr[b] = kv[b];
    if (b < B) {
      a.last_indices[b] = qo[b + 1] - 1;
      const int np = kv[b + 1] - kv[b];
      const int L = a.cached[b] + (qo[b + 1] - qo[b]);
      a.last_page_len[b] = np > 0 ? min(max(L - ((np - 1) << a.page_log2), 1), P) : 0;
    }
  }
  if (gid == 0) {
    a.counts[0] = T;
    a.counts[1] = NT > a.work_capacity ? 0 : NT;
    if (T > a.q_capacity || NP > a.idx_capacity || NT > a.work_capacity) watchdog_set(kWdMetaOverflow);
  }

  // ---- positions and slots of the new tokens
  const int Tc = (int)min((int64_t)T, a.q_capacity);
  for (int64_t i0 = (int64_t)gid * kEmVec; i0 < Tc; i0 += (int64_t)gthreads * kEmVec) {
    int b = em_find(qo, B, (int)i0);
    const int i1 = (int)min(i0 + kEmVec, (int64_t)Tc);
    for (int i = (int)i0; i < i1; ++i) {
      while (qo[b + 1] <= i) ++b;  // requests without new tokens
      const int64_t row = a.rows[b];
      const int pos = a.cached[b] + i - qo[b];
      a.positions[i] = pos;
      if (row >= 0 && row < a.table_rows && pos >= 0 && pos < a.stride) a.out_loc[i] = a.page_table[row * a.stride + pos];
    }
  }

  // ---- page ids of every request's tokens
  const int NPc = (int)min((int64_t)NP, a.idx_capacity);
  for (int64_t i0 = (int64_t)gid * kEmVec; i0 < NPc; i0 += (int64_t)gthreads * kEmVec) {
    int b = em_find(kv, B, (int)i0);
    const int i1 = (int)min(i0 + kEmVec, (int64_t)NPc);
    for (int i = (int)i0; i < i1; ++i) {
      while (kv[b + 1] <= i) ++b;  // requests without tokens
      const int64_t row = a.rows[b];
      const int64_t col = (int64_t)(i - kv[b]) << a.page_log2;
      if (row >= 0 && row < a.table_rows && col < a.stride) {
        const int32_t e = a.page_table[row * a.stride + col];
        if (e < 0 || (e & (P - 1))) watchdog_set(kWdBadSlot);
        a.kv_indices[i] = e >> a.page_log2;
      }
    }
  }

  // ---- work list: unused entries are empty tiles, used ones go to their rank
  for (int i = (NT > a.work_capacity ? 0 : NT) + gid; i < a.work_capacity; i += gthreads)
    reinterpret_cast<int4*>(a.work)[i] = make_int4(0, 0, 0, 0);
  if (NT > a.work_capacity) return;  // flagged above, the list stays empty
  const int per = (NT + gridDim.x - 1) / gridDim.x;
  const int o0 = min(blockIdx.x * per, NT), o1 = min(o0 + per, NT);
  for (int own = o0; own < o1; ++own) {
    const int b = em_find(tl, B, own);
    int tb, nq;
    const unsigned long long mine = em_key(a, qo, b, own - tl[b], own, tb, nq);
    if (tid == 0) rank_of = 0;
    int before = 0;
    for (int k0 = 0; k0 < NT; k0 += kEmKeys) {
      const int n = min(kEmKeys, NT - k0);
      if (own == o0 || NT > kEmKeys) {  // one round serves every own tile when all keys fit
        __syncthreads();
        const int run = (n + kEmThreads - 1) / kEmThreads;
        const int j0 = min(tid * run, n), j1 = min(j0 + run, n);
        if (j0 < j1) {
          int kb = em_find(tl, B, k0 + j0);
          for (int j = j0; j < j1; ++j) {
            while (tl[kb + 1] <= k0 + j) ++kb;
            int x, y;
            keys[j] = em_key(a, qo, kb, k0 + j - tl[kb], k0 + j, x, y);
          }
        }
      }
      __syncthreads();
      for (int j = tid; j < n; j += kEmThreads) before += keys[j] > mine;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) before += __shfl_xor_sync(FULL, before, o);
    if (lane == 0 && before) atomicAdd(&rank_of, before);
    __syncthreads();
    if (tid == 0) reinterpret_cast<int4*>(a.work)[rank_of] = make_int4(b, tb, nq, 0);
    __syncthreads();
  }
}

}  // namespace b2a

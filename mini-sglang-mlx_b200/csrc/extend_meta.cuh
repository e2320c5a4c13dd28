// Index tables of a prefill batch, built on the device from the requests' lengths.
//
// Replaces the host build of BaseAttnBackend._prepare_prefill
// (python/minisgl_mlx/attention/base.py:70-84), the positions / out_loc lookup of
// scheduler/scheduler.py:155-158 and b2a_extend_plan. For request b with L = lens[b]
// tokens, of which the first cached[b] are in the pool already, E = L - cached[b]:
//   qo_indptr, kv_indptr   exclusive sums of E and of ceil(L / P)
//   positions[qo_b + i]    cached[b] + i              (i < E)
//   out_loc[qo_b + i]      page_table[rows[b], cached[b] + i]; -1 (no slot: a store skips the row)
//                          behind the last token, for a row outside the table, and everywhere
//                          when the batch does not fit its buffers
//   kv_indices[kv_b + p]   page_table[rows[b], p P] / P
//   work                   {b, first token, tokens, 0} per tile of tile_q new tokens, by
//                          falling cost tokens * (keys its last token sees), equal costs
//                          in request order
//
// One launch. It moves a few bytes per token and page, so what bounds a usual batch is
// latency: the launch, and the chain lengths -> scan -> search -> table entry. Every CTA
// therefore scans all B requests itself (12 bytes each, from L2) into shared memory
// instead of waiting for another CTA or launch to do it, and finds the owners of its
// tokens, pages and tiles by binary search there, four at a time so that their searches
// and table reads overlap. A tile's place in the sorted list is the number of tiles that
// go before it, counted directly: all keys are unique (cost, then order), so no two tiles
// claim one place and no order of execution matters. A warp counts for up to eight tiles at
// once, reading every key from shared memory once.
#pragma once

#include "common.cuh"
#include "slot.cuh"

namespace b2a {

constexpr int kEmThreads = 256;
constexpr int kEmMaxBatch = 8192;  // five int32 arrays of a batch in shared memory
constexpr int kEmKeys = 2048;      // tile keys compared per round
constexpr int kEmOwn = 8;          // tiles a warp ranks at once
constexpr int kEmMaxTile = 256;    // cost < 2^39, so (cost, order) fits 64 bits
constexpr int kEmMaxWork = 1 << 24;

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
  return (size_t)kEmKeys * 8 + 5 * (size_t)(B + 1) * 4;
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

// Adds, for the first N of a warp's tiles, the keys of this round that go before them.
template <int N>
__device__ __forceinline__ void em_count(const unsigned long long* keys, int n, int lane,
                                         const unsigned long long (&mine)[kEmOwn], int (&before)[kEmOwn]) {
#pragma unroll 4
  for (int j = lane; j < n; j += 32) {
    const unsigned long long x = keys[j];
#pragma unroll
    for (int m = 0; m < N; ++m) before[m] += x > mine[m];
  }
}

__global__ void __launch_bounds__(kEmThreads) extend_meta_kernel(const ExtendMetaArgs a) {
  constexpr unsigned FULL = 0xffffffffu;
  constexpr int NWARP = kEmThreads / 32;
  extern __shared__ __align__(16) uint8_t em_smem[];
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(em_smem);
  const int B = a.B;
  int32_t* qo = reinterpret_cast<int32_t*>(em_smem + (size_t)kEmKeys * 8);  // [B + 1] each
  int32_t* kv = qo + B + 1;
  int32_t* tl = kv + B + 1;
  int32_t* cached = tl + B + 1;
  int32_t* rows = cached + B + 1;  // -1: outside the table
  __shared__ long long wsum[3][NWARP];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = 1 << a.page_log2;

  // ---- exclusive sums of new tokens, pages and tiles: thread t owns a run of requests
  {
    const int per = (B + kEmThreads - 1) / kEmThreads;
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    long long s[3] = {0, 0, 0};
    bool bad = false;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
      // lengths are forced into the table's range (and flagged)
      const int L0 = a.lens[b], c0 = a.cached[b], r0 = a.rows[b];
      const int L = L0 < 0 ? 0 : (int)min((int64_t)L0, a.stride);
      const int c = min(max(c0, 0), L);
      const bool row_ok = r0 >= 0 && r0 < a.table_rows;
      bad = bad || L != L0 || c != c0 || !row_ok;
      const int ext = L - c, pages = (int)(((int64_t)L + P - 1) >> a.page_log2);
      const int tiles = (ext + a.tile_q - 1) / a.tile_q;
      qo[b + 1] = ext;
      kv[b + 1] = pages;
      tl[b + 1] = tiles;
      cached[b] = c;
      rows[b] = row_ok ? r0 : -1;
      s[0] += ext;
      s[1] += pages;
      s[2] += tiles;
    }
    if (bad && blockIdx.x == 0) watchdog_set(kWdMetaOverflow);
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
    bool small = true;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      base[c] = inc[c] - s[c];
      long long all = 0;
#pragma unroll
      for (int w = 0; w < NWARP; ++w) {
        if (w == warp) base[c] += all;
        all += wsum[c][w];
      }
      small = small && all <= (c == 2 ? (long long)kEmMaxWork : 0x7fffffffll);
    }
    if (!small) {  // the same on every thread: the tables of a batch without tokens
      if (blockIdx.x == 0 && tid == 0) watchdog_set(kWdMetaOverflow);
      for (int i = blockIdx.x * kEmThreads + tid; i < a.work_capacity; i += gridDim.x * kEmThreads)
        reinterpret_cast<int4*>(a.work)[i] = make_int4(0, 0, 0, 0);
      for (int64_t i = (int64_t)blockIdx.x * kEmThreads + tid; i < a.q_capacity; i += (int64_t)gridDim.x * kEmThreads)
        a.out_loc[i] = kNoSlot;
      for (int b = blockIdx.x * kEmThreads + tid; b <= B; b += gridDim.x * kEmThreads) {
        a.qo_indptr[b] = a.kv_indptr[b] = 0;
        if (b < B) {
          a.last_indices[b] = -1;
          a.last_page_len[b] = 0;
        }
      }
      if (blockIdx.x == 0 && tid < 2) a.counts[tid] = 0;
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
  // a batch that does not fit its buffers gets an empty work list: nothing reads past them
  const bool fits = T <= a.q_capacity && NP <= a.idx_capacity && NT <= a.work_capacity;
  const int gthreads = gridDim.x * kEmThreads;
  const int gid = blockIdx.x * kEmThreads + tid;

  // ---- per-request outputs
  for (int b = gid; b <= B; b += gthreads) {
    a.qo_indptr[b] = qo[b];
    a.kv_indptr[b] = kv[b];
    if (b < B) {
      a.last_indices[b] = (int)min((int64_t)qo[b + 1], a.q_capacity) - 1;  // inside the buffer, fits or not
      const int np = kv[b + 1] - kv[b];
      a.last_page_len[b] = np > 0 ? cached[b] + (qo[b + 1] - qo[b]) - ((np - 1) << a.page_log2) : 0;
    }
  }
  if (gid == 0) {
    a.counts[0] = T;
    a.counts[1] = fits ? NT : 0;
    if (!fits) watchdog_set(kWdMetaOverflow);
  }

  // ---- positions and slots of the new tokens. Every entry of out_loc is written: a captured step
  // stores as many rows as the buffer has, and a slot left from another batch may be in use
  const int Tc = (int)min((int64_t)T, a.q_capacity);
  for (int64_t i0 = gid; i0 < Tc; i0 += 4ll * gthreads) {
    int pos[4], loc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + (int64_t)u * gthreads;
      pos[u] = 0;
      loc[u] = kNoSlot;
      if (i < Tc) {
        const int b = em_find(qo, B, (int)i);
        pos[u] = cached[b] + (int)i - qo[b];
        if (fits && rows[b] >= 0) {
          loc[u] = __ldg(a.page_table + (int64_t)rows[b] * a.stride + pos[u]);
          if (loc[u] < 0) watchdog_set(kWdBadSlot);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + (int64_t)u * gthreads;
      if (i < Tc) {
        a.positions[i] = pos[u];
        a.out_loc[i] = loc[u];
      }
    }
  }
  for (int64_t i = (int64_t)Tc + gid; i < a.q_capacity; i += gthreads) a.out_loc[i] = kNoSlot;

  // ---- page ids of every request's tokens
  const int NPc = (int)min((int64_t)NP, a.idx_capacity);
  for (int64_t i0 = gid; i0 < NPc; i0 += 4ll * gthreads) {
    int e[4];
    bool have[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + (int64_t)u * gthreads;
      e[u] = -1;  // a row outside the table: no page, attention reads zeros
      have[u] = false;
      if (i < NPc) {
        const int b = em_find(kv, B, (int)i);
        have[u] = rows[b] >= 0;
        if (have[u]) e[u] = __ldg(a.page_table + (int64_t)rows[b] * a.stride + ((int64_t)((int)i - kv[b]) << a.page_log2));
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + (int64_t)u * gthreads;
      if (have[u] && (e[u] < 0 || (e[u] & (P - 1)))) watchdog_set(kWdBadSlot);
      if (i < NPc) a.kv_indices[i] = e[u] >> a.page_log2;  // -1 stays -1
    }
  }

  // ---- work list: unused entries are empty tiles, used ones go to their rank
  for (int i = (fits ? NT : 0) + gid; i < a.work_capacity; i += gthreads)
    reinterpret_cast<int4*>(a.work)[i] = make_int4(0, 0, 0, 0);
  if (!fits) return;
  // key of tile i = tile k of request b: dearer tiles and, among equals, earlier ones are larger
  auto tile_of = [&](int b, int i, int& tb, int& nq) -> unsigned long long {
    tb = (i - tl[b]) * a.tile_q;
    nq = min(a.tile_q, qo[b + 1] - qo[b] - tb);
    const unsigned long long cost = (unsigned long long)nq * (unsigned long long)((long long)cached[b] + tb + nq);
    return (cost << 24) | (unsigned long long)(kEmMaxWork - 1 - i);
  };
  const int per = (NT + (int)gridDim.x - 1) / (int)gridDim.x;
  const int o0 = min((int)blockIdx.x * per, NT), o1 = min(o0 + per, NT);
  for (int c0 = o0; c0 < o1; c0 += NWARP * kEmOwn) {
    // this warp's tiles of the chunk: c0 + warp + 8 m
    unsigned long long mine[kEmOwn];
    int before[kEmOwn];
#pragma unroll
    for (int m = 0; m < kEmOwn; ++m) {
      const int i = c0 + warp + NWARP * m;
      int tb, nq;
      before[m] = 0;
      mine[m] = i < o1 ? tile_of(em_find(tl, B, i), i, tb, nq) : ~0ull;  // ~0: nothing goes before it
    }
    const int n_own = min(kEmOwn, (o1 - c0 - warp + NWARP - 1) / NWARP);
    for (int k0 = 0; k0 < NT; k0 += kEmKeys) {
      const int n = min(kEmKeys, NT - k0);
      if (c0 == o0 || NT > kEmKeys) {  // one round's keys serve every chunk when they all fit
        __syncthreads();
        const int run = (n + kEmThreads - 1) / kEmThreads;
        const int j0 = min(tid * run, n), j1 = min(j0 + run, n);
        if (j0 < j1) {
          int b = em_find(tl, B, k0 + j0);
          for (int j = j0; j < j1; ++j) {
            while (tl[b + 1] <= k0 + j) ++b;
            int tb, nq;
            keys[j] = tile_of(b, k0 + j, tb, nq);
          }
        }
        __syncthreads();
      }
      switch (n_own) {  // uniform over the warp
        case 1:
          em_count<1>(keys, n, lane, mine, before);
          break;
        case 2:
          em_count<2>(keys, n, lane, mine, before);
          break;
        case 3:
          em_count<3>(keys, n, lane, mine, before);
          break;
        case 4:
          em_count<4>(keys, n, lane, mine, before);
          break;
        default:
          if (n_own > 4) em_count<kEmOwn>(keys, n, lane, mine, before);
      }
    }
#pragma unroll
    for (int m = 0; m < kEmOwn; ++m) {
      const int rank = __reduce_add_sync(FULL, before[m]);
      const int i = c0 + warp + NWARP * m;
      if (lane == 0 && i < o1) {
        const int b = em_find(tl, B, i);
        int tb, nq;
        tile_of(b, i, tb, nq);
        reinterpret_cast<int4*>(a.work)[rank] = make_int4(b, tb, nq, 0);
      }
    }
  }
}

}  // namespace b2a

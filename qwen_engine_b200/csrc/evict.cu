// Eviction from the paged cache by gathered attention weight: a request's cache of `len` entries goes down to `keep`, for
// every layer and kv head by itself.  Of the entries, those at positions below `first` and those less than `recent` behind
// the latest position stay; of the others the heaviest, the lowest place among equals, until `keep` are left.  Entries that
// stay and lie before place `keep` do not move; those that lie behind it move, in their order, into the places of those that
// go, in theirs.  So a step that is one entry over its budget moves one entry and not the whole cache, every place that is
// read lies behind `keep` and every place that is written before it (no order between the moves matters), and attention,
// which does not look at the order of its keys, reads `keep` entries as one run of places.
//
// Selecting.  The entries' ranks are keys: an order-preserving integer of the weight, the largest integer for those that stay
// in any case.  They are formed once, into shared memory; the keep-th largest is found digit by digit (8 bits a pass) from
// histograms; a cluster of CTAs shares a head's entries where there are many, its histograms and counts meeting in
// distributed shared memory (two histograms in turn, so that a pass is one meeting).  The last pass's histogram also says how many
// entries of every CTA are at the threshold, of which the lowest places stay.  Everybody's place in the lists of movers and of
// free places then follows from ballots in the order of the entries, a warp a run of them.
//
// What bounds it: in bulk, the copies (16 bytes a lane, four entries of a warp on their way; 4 layers x 4 caches of 32 768 entries of 8 heads to 4 096: 470 MB in
// 85 us, 5.5 TB/s, behind 50 us of selecting); for a step's eviction of one entry, the chain of meetings (28 layers of 1 025 entries 13.4 us, 28 x 8 caches
// of 4 097 97 us; CTAs, shared memory and launches go by the places of slots and tables: the former with 2 048 places 14.8 us, with 40 960 27).
#include "common.cuh"
#include <math.h>

#define EV_MAX_CTAS 8
#define EV_PER_CTA 4096          // entries of a head from which one more CTA joins its cluster
#define EV_SHORT 6144            // entries of a CTA up to which it has 256 threads ...
#define EV_MEDIUM 24576          // ... and up to which it has 512
#define EV_MAX_SMEM (200 * 1024)
#define EV_MOVES_INSIDE 64       // moves of a head, at most, that the selecting kernel makes itself

struct EvArgs {
  const int* block_tables; int max_blocks; int num_pages;
  const int* slot_ids; const int* lens;
  const float* weights; const int* positions; float* weights_out; int* positions_out;
  long head_stride;              // capacity: entries between a (layer, slot, head)'s row and the next
  int slots, Hkv, R, capacity, keep, first, recent;
  char* cache; int planes, page, row_bytes;
  int* moves; int most;          // [layer, request, head]: 1 + 2 most ints: how many, the places they come from, the places they go to; most: min(keep, capacity - keep)
};

__device__ __forceinline__ unsigned ev_key(float w) {
  w = fmaxf(w, -INFINITY) + 0.f;                // NaN as the lowest, -0 as +0
  const unsigned u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ int ev_ld_remote(const int* local, int cta) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(v) : "r"(cluster_map_shared(local, cta)) : "memory");
  return v;
}

// The keys and values of the moves below n, a warp `batch` (32 at most) of them at a time (batches first, first + step, ..): a lane works out where one comes
// from and goes to, then the warp copies one after the other, V a lane, four on their way.
template <typename V>
__device__ __forceinline__ void ev_move(const EvArgs& A, int layer, int r, int h, const int* moves, int n, int first, int step, int batch) {
  const int* table = A.block_tables + (size_t)r * A.max_blocks;
  const size_t plane_bytes = (size_t)A.Hkv * A.page * A.row_bytes;
  char* base = A.cache + (size_t)layer * A.num_pages * A.planes * plane_bytes + (size_t)h * A.page * A.row_bytes;
  const int lane = threadIdx.x & 31, vecs = A.row_bytes / (int)sizeof(V), all = A.planes * vecs;
  auto place = [&](int at) -> char* {             // null where no page is held
    const int b = at / A.page, p = table[b];
    return p >= 0 && p < A.num_pages ? base + (size_t)p * A.planes * plane_bytes + (size_t)(at - b * A.page) * A.row_bytes : nullptr;
  };
  for (int i = first * batch; i < n; i += step * batch) {
    char *f = nullptr, *t = nullptr;
    if (lane < batch && i + lane < n) {
      f = place(__ldcg(moves + 1 + i + lane));
      t = place(__ldcg(moves + 1 + A.most + i + lane));
      if (f == nullptr || t == nullptr) f = t = nullptr;
    }
    const int m = min(batch, n - i);
    for (int v = lane; v - lane < all; v += 32) {
      const int pl = v / vecs;
      const size_t o = pl * plane_bytes + (size_t)(v - pl * vecs) * sizeof(V);
      const bool in = v < all;
      for (int e = 0; e < m; e += 4) {
        V x[4];
        char* dst[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const char* src = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(f), (e + k) & 31));
          dst[k] = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(t), (e + k) & 31));
          if (e + k >= m || !in) dst[k] = nullptr;
          if (dst[k]) x[k] = *reinterpret_cast<const V*>(src + o);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (dst[k]) *reinterpret_cast<V*>(dst[k] + o) = x[k];
      }
    }
  }
}

// held: the keys lie in shared memory (else they are formed again wherever they are looked at).  MOVES: 0 where another kernel moves the
// entries, else the bytes that a lane moves at a time.
template <int MOVES, int EV_THREADS>
__global__ void __launch_bounds__(EV_THREADS, 1024 / EV_THREADS)
evict_select_kernel(EvArgs A, int held) {
  constexpr int EV_WARPS = EV_THREADS / 32, AHEAD = EV_THREADS <= 512 ? 8 : 4;      // AHEAD: loads of a thread on their way
  extern __shared__ unsigned keys[];              // the CTA's keys, and behind them a bit for every entry that stays
  __shared__ int hist[2][256];
  __shared__ int s_max[EV_WARPS], s_ties[EV_WARPS], s_holes[EV_WARPS], s_movers[EV_WARPS], warp_tot[8];
  __shared__ int x[3];                          // read by the other CTAs of the cluster: latest position, free places, movers
  __shared__ int digit_s, above_s, equal_s;
  pdl_launch_dependents();
  pdl_wait();
  const int C = (int)cluster_num_ctas(), rank = (int)cluster_cta_rank();
  const int r = blockIdx.y / A.Hkv, h = blockIdx.y - r * A.Hkv, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = A.slot_ids[r];
  int* moves = A.moves + (((size_t)layer * A.R + r) * A.Hkv + h) * (size_t)(1 + 2 * A.most);
  if (slot < 0 || slot >= A.slots) {            // no such slot: nothing is read or written (the whole cluster)
    if (rank == 0 && tid == 0) moves[0] = 0;
    return;
  }
  const size_t row = (((size_t)layer * A.slots + slot) * A.Hkv + h) * (size_t)A.head_stride;
  const float* W = A.weights + row;
  const int* P = A.positions + row;
  float* Wo = A.weights_out + row;
  int* Po = A.positions_out + row;
  const int len = min(max(A.lens[r], 0), A.capacity), keep = A.keep;
  const int per = ((len + C - 1) / C + 31) / 32 * 32;
  const int e0 = min(len, rank * per), e1 = min(len, e0 + per);
  if (len <= keep) {                            // nothing goes (the whole cluster)
    if (rank == 0 && tid == 0) moves[0] = 0;
    if (Wo != W) for (int j = e0 + tid; j < e1; j += EV_THREADS) Wo[j] = W[j];
    if (Po != P) for (int j = e0 + tid; j < e1; j += EV_THREADS) Po[j] = P[j];
    return;
  }
  // the latest position
  int latest = -0x7fffffff;
  for (int j = e0 + tid; j < e1; j += AHEAD * EV_THREADS) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (j + i * EV_THREADS < e1) latest = max(latest, P[j + i * EV_THREADS]);
  }
  latest = __reduce_max_sync(0xffffffffu, latest);
  if (lane == 0) s_max[warp] = latest;
  if (tid < 256) { hist[0][tid] = 0; hist[1][tid] = 0; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < EV_WARPS; ++w) latest = max(latest, s_max[w]);
  if (C > 1) {
    if (tid == 0) x[0] = latest;
    cluster_sync_all();
#pragma unroll
    for (int o = 0; o < EV_MAX_CTAS; ++o) if (o < C) latest = max(latest, ev_ld_remote(&x[0], o));
  }
  const int recent_from = latest - A.recent;
  auto key_of = [&](int p, float w) { return p < A.first || p > recent_from ? 0xffffffffu : ev_key(w); };
  unsigned* const bits = keys + per;              // (held only)
  auto key_at = [&](int j) { return held ? keys[j - e0] : key_of(P[j], W[j]); };
  // the keep-th largest key; the first pass forms the keys
  unsigned thr = 0u;
  int left = keep, ties_before = 0;
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    int* const hs = hist[pass & 1];
    if (pass == 0) {
      for (int j = e0 + tid; j < e1; j += AHEAD * EV_THREADS) {
        int p[AHEAD];
        float w[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          if (j + i * EV_THREADS < e1) { p[i] = P[j + i * EV_THREADS]; w[i] = W[j + i * EV_THREADS]; }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          if (j + i * EV_THREADS < e1) {
            const unsigned key = key_of(p[i], w[i]);
            if (held) keys[j + i * EV_THREADS - e0] = key;
            atomicAdd(&hs[key >> 24], 1);
          }
      }
    } else {
      const unsigned mask = 0xffffffffu << (shift + 8);
      for (int j = e0 + tid; j < e1; j += EV_THREADS) {
        const unsigned key = key_at(j);
        if ((key & mask) == thr) atomicAdd(&hs[(key >> shift) & 255u], 1);
      }
    }
    if (C > 1) cluster_sync_all(); else __syncthreads();
    int c = 0, mine[EV_MAX_CTAS];
    if (tid < 256) {
#pragma unroll
      for (int o = 0; o < EV_MAX_CTAS; ++o) mine[o] = C == 1 ? (o == 0 ? hs[255 - tid] : 0) : (o < C ? ev_ld_remote(&hs[255 - tid], o) : 0);
#pragma unroll
      for (int o = 0; o < EV_MAX_CTAS; ++o) c += mine[o];
      hist[(pass & 1) ^ 1][tid] = 0;              // everybody has read it: they are past this pass's meeting
    }
    int run = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (tid < 256 && lane == 31) warp_tot[warp] = run;
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < warp; ++w) run += warp_tot[w];
      if (run >= left && run - c < left) {
        digit_s = 255 - tid;
        above_s = run - c;
        equal_s = c;
        int before = 0;                           // (last pass: entries at the threshold in the CTAs before this one)
#pragma unroll
        for (int o = 0; o < EV_MAX_CTAS; ++o) if (o < rank) before += mine[o];
        x[0] = before;                            // (the others have read their copies of it long ago)
      }
    }
    __syncthreads();
    thr |= (unsigned)digit_s << shift;
    left -= above_s;
    ties_before = x[0];
  }
  // `left` of the entries at the threshold stay, the lowest places.  A warp has a run of entries: its ties, then its free places and movers, then the lists.
  const int run_len = (per / 32 + EV_WARPS - 1) / EV_WARPS * 32;
  const int j0 = min(e1, e0 + warp * run_len), j1 = min(e1, j0 + run_len);
  const bool choose = equal_s != left;            // (else every entry at the threshold stays, which is the rule but for equal weights)
  if (choose) {
    int n = 0;
    for (int j = j0; j < j1; j += 32) n += __popc(__ballot_sync(0xffffffffu, j + lane < j1 && key_at(j + lane) == thr));
    if (lane == 0) s_ties[warp] = n;
    __syncthreads();
    for (int w = 0; w < warp; ++w) ties_before += s_ties[w];
  }
  const unsigned below = (1u << lane) - 1u;
  // what the 32 entries from j on do: which stay, with `ties` the ties before them
  auto stay = [&](int j, int& ties) {
    const bool in = j + lane < j1;
    const unsigned key = in ? key_at(j + lane) : 0u;
    if (!choose) return in && key >= thr;
    const unsigned same = __ballot_sync(0xffffffffu, in && key == thr);
    const bool s = in && (key > thr || (key == thr && ties + __popc(same & below) < left));
    ties += __popc(same);
    return s;
  };
  int holes = 0, movers = 0, ties = ties_before;
  for (int j = j0; j < j1; j += 32) {
    const unsigned sb = __ballot_sync(0xffffffffu, stay(j, ties));
    if (held && lane == 0) bits[(j - e0) >> 5] = sb;
    // of the 32 entries, those before place `keep`
    const unsigned head = j + 32 <= keep ? 0xffffffffu : (j >= keep ? 0u : (1u << (keep - j)) - 1u);
    const unsigned valid = j + 32 <= j1 ? 0xffffffffu : (1u << (j1 - j)) - 1u;
    holes += __popc(~sb & head & valid);
    movers += __popc(sb & ~head);
  }
  if (lane == 0) { s_holes[warp] = holes; s_movers[warp] = movers; }
  __syncthreads();
  holes = movers = 0;
  int all_movers = 0, cta_holes = 0;
#pragma unroll
  for (int w = 0; w < EV_WARPS; ++w) {
    if (w < warp) { holes += s_holes[w]; movers += s_movers[w]; }
    cta_holes += s_holes[w];
    all_movers += s_movers[w];
  }
  if (C > 1) {
    if (tid == 0) { x[1] = cta_holes; x[2] = all_movers; }
    cluster_sync_all();
    int hs[EV_MAX_CTAS], ms[EV_MAX_CTAS];
#pragma unroll
    for (int o = 0; o < EV_MAX_CTAS; ++o) { hs[o] = o < C ? ev_ld_remote(&x[1], o) : 0; ms[o] = o < C ? ev_ld_remote(&x[2], o) : 0; }
    all_movers = 0;
#pragma unroll
    for (int o = 0; o < EV_MAX_CTAS; ++o) {
      if (o < rank) { holes += hs[o]; movers += ms[o]; }
      all_movers += ms[o];
    }
  }
  if (rank == 0 && tid == 0) moves[0] = all_movers;
  // The kept entries that do not move, where the outputs are other tensors: on their way while the lists are written.
  if (held && Wo != W) {
    for (int j = e0 + tid; j < min(e1, keep); j += AHEAD * EV_THREADS) {
      float w[AHEAD];
      int p[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (j + i * EV_THREADS < min(e1, keep)) { w[i] = W[j + i * EV_THREADS]; p[i] = P[j + i * EV_THREADS]; }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int at = j + i * EV_THREADS;
        if (at < min(e1, keep) && ((bits[(at - e0) >> 5] >> ((at - e0) & 31)) & 1u)) {
          Wo[at] = w[i];
          if (Po != P) Po[at] = p[i];
        }
      }
    }
  }
  ties = ties_before;
  for (int j = j0; j < j1; j += 32) {
    const unsigned sb = held ? bits[(j - e0) >> 5] : __ballot_sync(0xffffffffu, stay(j, ties));
    const unsigned head = j + 32 <= keep ? 0xffffffffu : (j >= keep ? 0u : (1u << (keep - j)) - 1u);
    const unsigned valid = j + 32 <= j1 ? 0xffffffffu : (1u << (j1 - j)) - 1u;
    const unsigned hb = ~sb & head & valid, mb = sb & ~head;
    if ((hb >> lane) & 1u) moves[1 + A.most + holes + __popc(hb & below)] = j + lane;
    if ((mb >> lane) & 1u) moves[1 + movers + __popc(mb & below)] = j + lane;
    holes += __popc(hb);
    movers += __popc(mb);
    if (!(held && Wo != W) && ((sb & head) >> lane) & 1u) {
      if (Wo != W) Wo[j + lane] = W[j + lane];
      if (Po != P) Po[j + lane] = P[j + lane];
    }
  }
  __threadfence();
  cluster_sync_all();                           // both lists are whole, and nobody's shared memory is read any more
  for (int i = rank * EV_THREADS + tid; i < all_movers; i += C * EV_THREADS) {
    const int from = __ldcg(moves + 1 + i), to = __ldcg(moves + 1 + A.most + i);
    Wo[to] = W[from];
    Po[to] = P[from];
  }
  if (MOVES == 16) ev_move<uint4>(A, layer, r, h, moves, all_movers, warp * C + rank, C * EV_WARPS, 4);
  if (MOVES == 4) ev_move<uint32_t>(A, layer, r, h, moves, all_movers, warp * C + rank, C * EV_WARPS, 4);
  if (MOVES == 2) ev_move<uint16_t>(A, layer, r, h, moves, all_movers, warp * C + rank, C * EV_WARPS, 4);
}

template <typename V>
__global__ void __launch_bounds__(256)
evict_move_kernel(EvArgs A, int batch) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.y / A.Hkv, h = blockIdx.y - r * A.Hkv, layer = blockIdx.z;
  const int* moves = A.moves + (((size_t)layer * A.R + r) * A.Hkv + h) * (size_t)(1 + 2 * A.most);
  ev_move<V>(A, layer, r, h, moves, moves[0], blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8, batch);
}

template <int MOVES, int THREADS>
static cudaError_t ev_select_with(dim3 grid, size_t smem, cudaStream_t stream, const EvArgs& args, int held) {
  if (smem > 48 * 1024) {
    static unsigned long long configured = 0;
    const cudaError_t e = qe_once_a_device(configured, [] {
      return cudaFuncSetAttribute(evict_select_kernel<MOVES, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_MAX_SMEM);
    });
    if (e != cudaSuccess) return e;
  }
  return qe_launch_cluster(evict_select_kernel<MOVES, THREADS>, grid, dim3(THREADS), smem, stream, grid.x, args, held);
}
// Threads of a CTA: 256 for short runs of entries (four CTAs an SM take turns at their meetings), 512 or 1 024 for long ones.
template <int MOVES>
static cudaError_t ev_select(dim3 grid, size_t smem, cudaStream_t stream, const EvArgs& args, int held, long per) {
  if (per <= EV_SHORT) return ev_select_with<MOVES, 256>(grid, smem, stream, args, held);
  if (per <= EV_MEDIUM) return ev_select_with<MOVES, 512>(grid, smem, stream, args, held);
  return ev_select_with<MOVES, 1024>(grid, smem, stream, args, held);
}

extern "C" int qe_evict_tokens(void* cache, int layers, int num_pages, int planes, int Hkv, int page_size, int row_bytes,
                               const int* block_tables, int max_blocks, const int* slot_ids, const int* lens, int R,
                               const float* weights, const int* positions, float* weights_out, int* positions_out, int slots,
                               long head_stride, int capacity, int keep, int first, int recent, int* moves, cudaStream_t stream) {
  if (layers <= 0 || R <= 0 || Hkv <= 0) return 0;
  if (keep < 1 || first < 0 || recent < 0) QE_REFUSE("evict_tokens: a budget of %d with %d first and %d recent entries", keep, first, recent);
  if ((long)R * Hkv > 65535 || layers > 65535) QE_REFUSE("evict_tokens: %d requests of %d heads, %d layers are more than a launch takes", R, Hkv, layers);
  const int most = capacity > keep ? (capacity - keep < keep ? capacity - keep : keep) : 0;
  EvArgs args{block_tables, max_blocks, num_pages, slot_ids, lens, weights, positions, weights_out, positions_out, head_stride,
              slots, Hkv, R, capacity, keep, first, recent, (char*)cache, planes, page_size, row_bytes, moves, most};
  // CTAs a head: one, where the heads of all layers and requests are as many as the SMs (a cluster's meetings cost more than a longer run of
  // entries: 128 heads of 32 768 entries, 8 CTAs each 90 us), else up to EV_MAX_CTAS; and as many as hold the keys
  unsigned ctas = 1;
  const long heads = (long)R * Hkv * layers;
  while (ctas < EV_MAX_CTAS && ((heads * ctas < 148 && (long)ctas * EV_PER_CTA < capacity) || (long)capacity * 33 / 8 > (long)ctas * (EV_MAX_SMEM - 256))) ctas *= 2;
  const size_t per = ((capacity + ctas - 1) / ctas + 31) / 32 * 32;
  const int held = per * 4 + per / 8 <= EV_MAX_SMEM;
  const size_t smem = held ? per * 4 + per / 8 : 0;
  const dim3 select((unsigned)ctas, (unsigned)(R * Hkv), (unsigned)layers);
  // a few moves are made by the kernel that lists them: one launch less
  const int unit = row_bytes % 16 == 0 && ((uintptr_t)cache & 15) == 0 ? 16 : (row_bytes % 4 == 0 && ((uintptr_t)cache & 3) == 0 ? 4 : 2);
  const bool inside = most <= EV_MOVES_INSIDE;
  cudaError_t e;
  if (!inside) e = ev_select<0>(select, smem, stream, args, held, (long)per);
  else if (unit == 16) e = ev_select<16>(select, smem, stream, args, held, (long)per);
  else if (unit == 4) e = ev_select<4>(select, smem, stream, args, held, (long)per);
  else e = ev_select<2>(select, smem, stream, args, held, (long)per);
  if (e == cudaSuccess && !inside) {
    // moves of a warp at a time: 32, where that still gives every SM 16 warps, else 4
    const int batch = heads * most >= 148L * 16 * 32 ? 32 : 4;
    const unsigned blocks = (unsigned)((most + 8 * batch - 1) / (8 * batch) < 64 ? (most + 8 * batch - 1) / (8 * batch) : 64);
    const dim3 grid(blocks, (unsigned)(R * Hkv), (unsigned)layers);
    if (unit == 16) e = qe_launch(evict_move_kernel<uint4>, grid, dim3(256), 0, stream, args, batch);
    else if (unit == 4) e = qe_launch(evict_move_kernel<uint32_t>, grid, dim3(256), 0, stream, args, batch);
    else e = qe_launch(evict_move_kernel<uint16_t>, grid, dim3(256), 0, stream, args, batch);
  }
  if (e != cudaSuccess) { qe_set_error("evict_tokens: launch failed: %s", cudaGetErrorString(e)); (void)cudaGetLastError(); return 2; }
  QE_CHECK_LAUNCH("evict_tokens");
  return 0;
}

// Eviction from the paged cache by gathered attention weight: a request's cache of `len` entries goes down to `keep`, for
// every layer and kv head by itself.  Of the entries, those at positions below `first` and those less than `recent` behind
// the latest position stay; of the others the heaviest, the lowest place among equals, until `keep` are left.  Entries that
// stay and lie before place `keep` do not move; those that lie behind it move, in their order, into the places of those that
// go, in theirs.  So a step that is one entry over its budget moves one entry and not the whole cache, every place that is
// read lies behind `keep` and every place that is written before it (no order between the moves matters), and attention,
// which does not look at the order of its keys, reads `keep` entries as one run of places.
//
// Selecting.  The entries' ranks are keys: an order-preserving integer of the weight, the largest integer for those that stay
// in any case.  The keep-th largest key is found digit by digit (8 bits a pass) from histograms; a cluster of CTAs shares a
// head's entries where there are many, its histograms and counts meeting in distributed shared memory.  Then everybody's
// place in the lists of movers and of free places follows from counts in the order of the entries.
#include "common.cuh"
#include <math.h>

#define EV_THREADS 512
#define EV_WARPS (EV_THREADS / 32)
#define EV_MAX_CTAS 8
#define EV_PER_CTA 4096          // entries of a head from which one more CTA joins its cluster

struct EvArgs {
  const int* block_tables; int max_blocks; int num_pages;
  const int* slot_ids; const int* lens;
  const float* weights; const int* positions; float* weights_out; int* positions_out;
  long head_stride;              // capacity: entries between a (layer, slot, head)'s row and the next
  int slots, Hkv, R, capacity, keep, first, recent;
  int* moves;                    // [layer, request, head]: 1 + 2 keep ints: how many, the places they come from, the places they go to
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
__device__ __forceinline__ int ev_block_sum(int v, int* s) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
  for (int w = 0; w < EV_WARPS; ++w) t += s[w];
  return t;
}
// the sum over the threads before this one, and over all (`total`)
__device__ __forceinline__ int ev_block_before(bool flag, int* s, int& total) {
  const unsigned b = __ballot_sync(0xffffffffu, flag);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) s[warp] = __popc(b);
  __syncthreads();
  int before = __popc(b & ((1u << lane) - 1u));
  total = 0;
  for (int w = 0; w < EV_WARPS; ++w) {
    if (w < warp) before += s[w];
    total += s[w];
  }
  return before;
}

__global__ void __launch_bounds__(EV_THREADS)
evict_select_kernel(EvArgs A) {
  __shared__ int hist[256];
  __shared__ int s_red[EV_WARPS];
  __shared__ int x[4];                          // read by the other CTAs of the cluster
  __shared__ int digit_s, above_s, warp_tot[8];
  pdl_launch_dependents();
  pdl_wait();
  const int C = (int)cluster_num_ctas(), rank = (int)cluster_cta_rank();
  const int r = blockIdx.y / A.Hkv, h = blockIdx.y - r * A.Hkv, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = A.slot_ids[r];
  int* moves = A.moves + (((size_t)layer * A.R + r) * A.Hkv + h) * (size_t)(1 + 2 * A.keep);
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
  for (int j = e0 + tid; j < e1; j += EV_THREADS) latest = max(latest, P[j]);
  latest = __reduce_max_sync(0xffffffffu, latest);
  if (lane == 0) s_red[warp] = latest;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < EV_WARPS; ++w) latest = max(latest, s_red[w]);
    x[0] = latest;
  }
  cluster_sync_all();
  latest = ev_ld_remote(&x[0], 0);
  for (int o = 1; o < C; ++o) latest = max(latest, ev_ld_remote(&x[0], o));
  const int recent_from = latest - A.recent;
  auto key_of = [&](int j) {
    const int p = P[j];
    return p < A.first || p > recent_from ? 0xffffffffu : ev_key(W[j]);
  };
  // the keep-th largest key
  unsigned thr = 0u;
  int left = keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    const unsigned mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int j = e0 + tid; j < e1; j += EV_THREADS) {
      const unsigned key = key_of(j);
      if ((key & mask) == (thr & mask)) atomicAdd(&hist[(key >> shift) & 255u], 1);
    }
    cluster_sync_all();
    int c = 0;
    if (tid < 256)
      for (int o = 0; o < C; ++o) c += ev_ld_remote(&hist[255 - tid], o);
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
      if (run >= left && run - c < left) { digit_s = 255 - tid; above_s = run - c; }
    }
    __syncthreads();
    thr |= (unsigned)digit_s << shift;
    left -= above_s;
    cluster_sync_all();
  }
  // `left` of the entries at the threshold stay, the lowest places
  int ties = 0;
  for (int j = e0 + tid; j < e1; j += EV_THREADS) ties += key_of(j) == thr;
  ties = ev_block_sum(ties, s_red);
  if (tid == 0) x[1] = ties;
  cluster_sync_all();
  int ties_before = 0;
  for (int o = 0; o < rank; ++o) ties_before += ev_ld_remote(&x[1], o);
  // twice over the entries in their order: count movers and free places, then list them
  int holes = 0, movers = 0;                    // of the CTAs before this one (second time)
  for (int pass = 0; pass < 2; ++pass) {
    int t_run = ties_before, h_run = holes, m_run = movers;
    for (int b = e0; b < e1; b += EV_THREADS) {
      const int j = b + tid;
      const bool in = j < e1;
      const unsigned key = in ? key_of(j) : 0u;
      int tot;
      const int t_before = t_run + ev_block_before(in && key == thr, s_red, tot);
      t_run += tot;
      const bool stays = in && (key > thr || (key == thr && t_before < left));
      const bool hole = in && !stays && j < keep, mover = stays && j >= keep;
      const int h_at = h_run + ev_block_before(hole, s_red, tot);
      h_run += tot;
      const int m_at = m_run + ev_block_before(mover, s_red, tot);
      m_run += tot;
      if (pass == 1) {
        if (mover) moves[1 + m_at] = j;
        if (hole) moves[1 + keep + h_at] = j;
        if (stays && j < keep) {
          if (Wo != W) Wo[j] = W[j];
          if (Po != P) Po[j] = P[j];
        }
      }
    }
    if (pass == 0) {
      if (tid == 0) { x[2] = h_run; x[3] = m_run; }
      cluster_sync_all();
      for (int o = 0; o < rank; ++o) { holes += ev_ld_remote(&x[2], o); movers += ev_ld_remote(&x[3], o); }
      int all = 0;
      for (int o = 0; o < C; ++o) all += ev_ld_remote(&x[3], o);
      if (rank == 0 && tid == 0) moves[0] = all;
    }
  }
  __threadfence();
  cluster_sync_all();                           // both lists are whole
  const int n = *reinterpret_cast<volatile int*>(moves);
  for (int i = rank * EV_THREADS + tid; i < n; i += C * EV_THREADS) {
    const int from = __ldcg(moves + 1 + i), to = __ldcg(moves + 1 + keep + i);
    Wo[to] = W[from];
    Po[to] = P[from];
  }
}

// The listed entries' keys and values, a warp an entry; V is what one lane moves at a time.
template <typename V>
__global__ void __launch_bounds__(256)
evict_move_kernel(EvArgs A, char* cache, int planes, int page_size, int row_bytes) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.y / A.Hkv, h = blockIdx.y - r * A.Hkv, layer = blockIdx.z;
  const int* moves = A.moves + (((size_t)layer * A.R + r) * A.Hkv + h) * (size_t)(1 + 2 * A.keep);
  const int n = moves[0];
  const int* table = A.block_tables + (size_t)r * A.max_blocks;
  const size_t plane_bytes = (size_t)A.Hkv * page_size * row_bytes;
  char* base = cache + (size_t)layer * A.num_pages * planes * plane_bytes;
  const int lane = threadIdx.x & 31, vecs = row_bytes / (int)sizeof(V);
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const int from = moves[1 + i], to = moves[1 + A.keep + i];
    const int fb = from / page_size, tb = to / page_size;
    const int fp = table[fb], tp = table[tb];
    if (fp < 0 || tp < 0 || fp >= A.num_pages || tp >= A.num_pages) continue;     // no page held there
    const char* src = base + (size_t)fp * planes * plane_bytes + ((size_t)h * page_size + (from - fb * page_size)) * row_bytes;
    char* dst = base + (size_t)tp * planes * plane_bytes + ((size_t)h * page_size + (to - tb * page_size)) * row_bytes;
    for (int v = lane; v < planes * vecs; v += 32) {
      const int pl = v / vecs, o = v - pl * vecs;
      reinterpret_cast<V*>(dst + pl * plane_bytes)[o] = reinterpret_cast<const V*>(src + pl * plane_bytes)[o];
    }
  }
}

extern "C" int qe_evict_tokens(void* cache, int layers, int num_pages, int planes, int Hkv, int page_size, int row_bytes,
                               const int* block_tables, int max_blocks, const int* slot_ids, const int* lens, int R,
                               const float* weights, const int* positions, float* weights_out, int* positions_out, int slots,
                               long head_stride, int capacity, int keep, int first, int recent, int* moves, cudaStream_t stream) {
  if (layers <= 0 || R <= 0 || Hkv <= 0) return 0;
  if (keep < 1 || first < 0 || recent < 0) QE_REFUSE("evict_tokens: a budget of %d with %d first and %d recent entries", keep, first, recent);
  if ((long)R * Hkv > 65535 || layers > 65535) QE_REFUSE("evict_tokens: %d requests of %d heads, %d layers are more than a launch takes", R, Hkv, layers);
  EvArgs args{block_tables, max_blocks, num_pages, slot_ids, lens, weights, positions, weights_out, positions_out, head_stride,
              slots, Hkv, R, capacity, keep, first, recent, moves};
  unsigned ctas = 1;
  while (ctas < EV_MAX_CTAS && (long)ctas * EV_PER_CTA < capacity) ctas *= 2;
  qe_launch_cluster(evict_select_kernel, dim3(ctas, (unsigned)(R * Hkv), (unsigned)layers), dim3(EV_THREADS), 0, stream, ctas, args);
  QE_CHECK_LAUNCH("evict_tokens");
  const int most = capacity > keep ? (capacity - keep < keep ? capacity - keep : keep) : 0;
  if (most == 0) return 0;
  const unsigned blocks = (unsigned)((most + 7) / 8 < 64 ? (most + 7) / 8 : 64);
  const dim3 grid(blocks, (unsigned)(R * Hkv), (unsigned)layers);
  if (row_bytes % 16 == 0 && ((uintptr_t)cache & 15) == 0)
    qe_launch(evict_move_kernel<uint4>, grid, dim3(256), 0, stream, args, (char*)cache, planes, page_size, row_bytes);
  else if (row_bytes % 4 == 0 && ((uintptr_t)cache & 3) == 0)
    qe_launch(evict_move_kernel<uint32_t>, grid, dim3(256), 0, stream, args, (char*)cache, planes, page_size, row_bytes);
  else
    qe_launch(evict_move_kernel<uint16_t>, grid, dim3(256), 0, stream, args, (char*)cache, planes, page_size, row_bytes);
  QE_CHECK_LAUNCH("evict_tokens");
  return 0;
}

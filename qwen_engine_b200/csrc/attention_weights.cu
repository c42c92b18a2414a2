// Gathered attention weights: what every cached key has received from the queries so far,
//
//   out[slot_r, c, j] = (j < ctx_r ? weights[slot_r, c, j] : 0) + sum over the request's counted rows i and the heads h of kv head
//                       c's group of softmax_j(s_hij),      j < ctx_r + n_r,
//
// with the scores, masks and sinks of the attention that read the same keys.  This file: the kernels for every type, head
// size and number of rows, on the CUDA cores; the ones for bfloat16 are in files of their own.
//
// A weight needs its row's whole softmax before the first sum over a column, and the scores of a prompt (rows x keys) are
// too many to keep, so they are formed twice: one kernel goes along the rows and leaves maximum and sum of each (in parts,
// where rows are few and keys many), the other goes along the keys and adds up exp(s - m) / z down every column.  The
// second gives a tile of keys to one CTA for all its rows, so that a sum has one order and nothing is added atomically.
// Scores are formed by the same instructions both times: no weight exceeds 1.
//
// What bounds them: the products, two of the scores' size at about 20 TFLOP/s (float32, 1 500 tokens behind 500, 32 / 8 heads of 128: 1.6 ms); small
// steps, the latency of a tile (3 portions of up to 37 tokens: 27 us for three launches).
#include "attention_weights.cuh"

#define AW_KC 32               // channels at a time
#define AW_THREADS 256         // 16 x 16, a thread RM rows and KM keys: tiles of 16 RM rows and 16 KM keys

// Channels lie across: row d of an array holds channel d of the tile's rows (keys), four side by side; the fours are in the order aw_col says, so that neither
// the stores (eight threads a row, four channels each) nor the loads (fours of one channel) meet in a bank.
template <int RM, int KM>
struct AwTile {
  static constexpr int ROWS = 16 * RM, KEYS = 16 * KM;
  float q[AW_KC][ROWS + 4];
  float k[AW_KC][KEYS + 4];
};
template <int N> __device__ __forceinline__ int aw_col(int d, int four) { return 4 * (four ^ ((d >> 2) & (N >= 32 ? 7 : 3))); }
// which of a tile's rows (keys) a thread has: one, four side by side, or four of either half
template <int M> __device__ __forceinline__ int aw_own(int t, int i) { return M == 1 ? t : (M == 4 ? 4 * t + i : (i < 4 ? 4 * t + i : 64 + 4 * t + i - 4)); }
template <int M, int N> __device__ __forceinline__ void aw_take(const float (&row)[N], int d, int t, float (&v)[M]) {
  if constexpr (M == 1) {
    v[0] = row[aw_col<N - 4>(d, t >> 2) + (t & 3)];
  } else {
#pragma unroll
    for (int h = 0; h < M / 4; ++h) {
      const float4 x = *reinterpret_cast<const float4*>(row + aw_col<N - 4>(d, 16 * h + t));
      v[4 * h] = x.x; v[4 * h + 1] = x.y; v[4 * h + 2] = x.z; v[4 * h + 3] = x.w;
    }
  }
}

// four channels from d on of a row of D (null: zeros), in one piece where it lies on a multiple of its size
template <typename T>
__device__ __forceinline__ void aw_fetch(const T* p, int d, int D, float (&v)[4]) {
  if (p != nullptr && d + 4 <= D && ((reinterpret_cast<uintptr_t>(p + d) & (4 * sizeof(T) - 1)) == 0)) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + d));
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
      const uint2 raw = __ldg(reinterpret_cast<const uint2*>(p + d));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int x = 0; x < 4; ++x) v[x] = to_f32(e[x]);
    }
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = p != nullptr && d + x < D ? to_f32(p[d + x]) : 0.f;
  }
}

// s[i][j] of the thread's rows (of the tile from rho0 on) and keys (from key0 on) of head c; rows and keys that do not exist read as zeros.
template <typename T, int RM, int KM>
__device__ __forceinline__ void aw_products(const AwArgs& A, const AwReq& R, int r, int c, int rho0, int key0, AwTile<RM, KM>& sm, float (&s)[RM][KM]) {
  using Tile = AwTile<RM, KM>;
  constexpr int NQ = (Tile::ROWS + 31) / 32, NK = (Tile::KEYS + 31) / 32;      // rows and keys of which a thread fetches four channels
  const int G = A.Hq / A.Hkv, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < KM; ++j) s[i][j] = 0.f;
  const int at = tid >> 3, ch = (tid & 7) * 4;    // row (key) at + 32 i, channels ch .. of every AW_KC
  const T* qp[NQ];
  const T* kp[NK];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int rho = rho0 + at + 32 * i;
    qp[i] = nullptr;
    if (rho < R.n * G && at + 32 * i < Tile::ROWS) {
      const int t = rho / G, g = rho - t * G;
      qp[i] = reinterpret_cast<const T*>(A.q) + (size_t)(R.row0 + t) * A.q_stride + (size_t)(c * G + g) * A.D;
    }
  }
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int key = key0 + at + 32 * i;
    const int page = key < R.total && at + 32 * i < Tile::KEYS ? aw_page(A, r, key) : -1;
    kp[i] = page >= 0 ? reinterpret_cast<const T*>(A.pages) + (((size_t)page * A.planes * A.Hkv + c) * A.page + key - aw_block(A, key) * A.page) * A.D : nullptr;
  }
  float qv[NQ][4], kv[NK][4];
  auto fetch = [&](int d) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) aw_fetch(qp[i], d, A.D, qv[i]);
#pragma unroll
    for (int i = 0; i < NK; ++i) aw_fetch(kp[i], d, A.D, kv[i]);
  };
  fetch(ch);
  for (int d0 = 0; d0 < A.D; d0 += AW_KC) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NQ; ++i)
      if (at + 32 * i < Tile::ROWS)
#pragma unroll
        for (int x = 0; x < 4; ++x) sm.q[ch + x][aw_col<Tile::ROWS>(ch, (at >> 2) + 8 * i) + (at & 3)] = qv[i][x];
#pragma unroll
    for (int i = 0; i < NK; ++i)
      if (at + 32 * i < Tile::KEYS)
#pragma unroll
        for (int x = 0; x < 4; ++x) sm.k[ch + x][aw_col<Tile::KEYS>(ch, (at >> 2) + 8 * i) + (at & 3)] = kv[i][x];
    __syncthreads();
    if (d0 + AW_KC < A.D) fetch(d0 + AW_KC + ch);  // the next channels, while these are multiplied
#pragma unroll 8
    for (int d = 0; d < AW_KC; ++d) {
      float av[RM], bv[KM];
      aw_take(sm.q[d], d, ty, av);
      aw_take(sm.k[d], d, tx, bv);
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < KM; ++j) s[i][j] = fmaf(av[i], bv[j], s[i][j]);
    }
  }
}

template <typename T, int RM, int KM>
__global__ void __launch_bounds__(AW_THREADS, 2)
attention_weights_rows_kernel(AwArgs A, int few_rows) {
  using Tile = AwTile<RM, KM>;
  __shared__ Tile sm;
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.z, c = blockIdx.y, tile = blockIdx.x / A.parts, part = blockIdx.x - tile * A.parts;
  const AwReq R = aw_req(A, r);
  const int G = A.Hq / A.Hkv, rho0 = tile * Tile::ROWS, rows = R.counted * G;
  if (rho0 >= rows || (long)R.n * G <= few_rows) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  // the tile's keys, and this part's share of their tiles
  const int first = R.ctx + rho0 / G, last = R.ctx + (min(rho0 + Tile::ROWS, rows) - 1) / G;
  const int lo = A.window > 0 ? max(0, first - A.window + 1) / Tile::KEYS * Tile::KEYS : 0;
  const int tiles = (last - lo) / Tile::KEYS + 1, per = (tiles + A.parts - 1) / A.parts;
  float m[RM], z[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) { m[i] = -INFINITY; z[i] = 0.f; }
  for (int kt = part * per; kt < min(tiles, (part + 1) * per); ++kt) {
    const int key0 = lo + kt * Tile::KEYS;
    float s[RM][KM];
    aw_products<T, RM, KM>(A, R, r, c, rho0, key0, sm, s);
    unsigned held = 0u;
#pragma unroll
    for (int j = 0; j < KM; ++j) held |= (unsigned)(aw_page(A, r, key0 + aw_own<KM>(tx, j)) >= 0) << j;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int rho = rho0 + aw_own<RM>(ty, i), pos = rho < rows ? R.ctx + rho / G : -1;
      const float slope = A.slopes ? A.slopes[c * G + rho % G] : 0.f;
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < KM; ++j) {
        const int key = key0 + aw_own<KM>(tx, j);
        const bool seen = ((held >> j) & 1u) && key <= pos && (A.window <= 0 || key > pos - A.window);
        s[i][j] = seen ? aw_score(A, s[i][j], slope, pos - key) : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
      const float base = aw_base(mx);
      float sum = z[i] * exp2f(m[i] - base);
#pragma unroll
      for (int j = 0; j < KM; ++j) sum += exp2f(s[i][j] - base);
      m[i] = mx; z[i] = sum;
    }
  }
  // a row's 16 threads put their maxima and sums together
#pragma unroll
  for (int i = 0; i < RM; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m[i], o), oz = __shfl_xor_sync(0xffffffffu, z[i], o);
      const float nm = fmaxf(m[i], om), base = aw_base(nm);
      z[i] = z[i] * exp2f(m[i] - base) + oz * exp2f(om - base);
      m[i] = nm;
    }
    const int rho = rho0 + aw_own<RM>(ty, i);
    if (tx == 0 && rho < rows) {
      const int t = rho / G;
      float* st = A.stats + (((size_t)(R.row0 + t) * A.Hq + c * G + (rho - t * G)) * A.parts + part) * 2;
      st[0] = m[i]; st[1] = z[i];
    }
  }
}

template <typename T, int RM, int KM>
__global__ void __launch_bounds__(AW_THREADS, 2)
attention_weights_keys_kernel(AwArgs A, int few_rows, int parts, float* sums_out, long ld) {
  using Tile = AwTile<RM, KM>;
  __shared__ Tile sm;
  __shared__ float2 row[Tile::ROWS];
  __shared__ float sums[16][Tile::KEYS];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.z, c = blockIdx.y, part = blockIdx.x % parts, key0 = (int)(blockIdx.x / parts) * Tile::KEYS;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  const int G = A.Hq / A.Hkv;
  if (key0 >= R.total || slot < 0 || slot >= A.slots || (few_rows >= 0 && (long)R.n * G <= few_rows)) return;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  // the rows that see any of these keys
  const int t0 = max(0, key0 - R.ctx);
  const int t1 = A.window > 0 ? (int)min((long)R.counted, (long)key0 + Tile::KEYS - 1 + A.window - R.ctx) : R.counted;
  float acc[KM];
  unsigned held = 0u;
#pragma unroll
  for (int j = 0; j < KM; ++j) {
    acc[j] = 0.f;
    held |= (unsigned)(aw_page(A, r, key0 + aw_own<KM>(tx, j)) >= 0) << j;
  }
  // this part's share of their tiles
  const int row_tiles = t1 > t0 ? ((t1 - t0) * G + Tile::ROWS - 1) / Tile::ROWS : 0, per = (row_tiles + parts - 1) / parts;
  for (int rt = part * per; rt < min(row_tiles, (part + 1) * per); ++rt) {
    const int rho0 = t0 * G + rt * Tile::ROWS;
    if (tid < Tile::ROWS) {
      const int rho = rho0 + tid;
      float2 v = make_float2(0.f, 0.f);
      if (rho < t1 * G) {
        const int t = rho / G, head = c * G + (rho - t * G);
        v = aw_merge(A.stats + ((size_t)(R.row0 + t) * A.Hq + head) * A.parts * 2, A.parts, A.sinks ? A.sinks + head : nullptr);
      }
      row[tid] = v;
    }
    float s[RM][KM];
    aw_products<T, RM, KM>(A, R, r, c, rho0, key0, sm, s);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int own = aw_own<RM>(ty, i), rho = rho0 + own;
      const int pos = rho < t1 * G ? R.ctx + rho / G : -1;
      const float slope = A.slopes ? A.slopes[c * G + rho % G] : 0.f;
      const float2 mz = row[own];
#pragma unroll
      for (int j = 0; j < KM; ++j) {
        const int key = key0 + aw_own<KM>(tx, j);
        const bool seen = ((held >> j) & 1u) && key <= pos && (A.window <= 0 || key > pos - A.window);
        if (seen) acc[j] += exp2f(aw_score(A, s[i][j], slope, pos - key) - mz.x) * mz.y;
      }
    }
    __syncthreads();                              // `row` is written anew
  }
#pragma unroll
  for (int j = 0; j < KM; ++j) sums[ty][aw_own<KM>(tx, j)] = acc[j];
  __syncthreads();
  const int key = key0 + tid;
  if (tid < Tile::KEYS && key < R.total) {
    float total = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) total += sums[y][tid];
    if (sums_out) {
      sums_out[(((size_t)part * A.R + r) * A.Hkv + c) * ld + key] = total;
    } else {
      const size_t at = ((size_t)slot * A.Hkv + c) * A.capacity + key;
      A.out[at] = key < R.ctx ? A.weights[at] + total : total;
      if (A.positions && key >= R.ctx) A.positions[at] = A.step_positions[R.row0 + key - R.ctx];
    }
  }
}

__global__ void __launch_bounds__(256)
attention_weights_finish_kernel(AwArgs A, const float* __restrict__ sums, long ld, int parts, int few_rows) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.y, r = blockIdx.z, k = blockIdx.x * 256 + threadIdx.x;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  if ((few_rows >= 0 && (long)R.n * (A.Hq / A.Hkv) <= few_rows) || k >= R.total || slot < 0 || slot >= A.slots) return;
  float total = 0.f;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) total += sums[(((size_t)p * A.R + r) * A.Hkv + c) * ld + k];
  const size_t at = ((size_t)slot * A.Hkv + c) * A.capacity + k;
  A.out[at] = k < R.ctx ? A.weights[at] + total : total;
  if (A.positions && k >= R.ctx) A.positions[at] = A.step_positions[R.row0 + k - R.ctx];
}

cudaError_t aw_finish(const AwArgs& A, const float* sums, long ld, int parts, int few_rows, int max_total, cudaStream_t stream) {
  return qe_launch(attention_weights_finish_kernel, dim3((unsigned)((max_total + 255) / 256), (unsigned)A.Hkv, (unsigned)A.R), dim3(256), 0, stream, A, sums, ld, parts, few_rows);
}

template <typename T, int RM, int KM>
static cudaError_t aw_rows(const AwArgs& A, long rows, int few_rows, cudaStream_t stream) {
  const long tiles = (rows + 16 * RM - 1) / (16 * RM);
  if (tiles == 0) return cudaSuccess;
  return qe_launch(attention_weights_rows_kernel<T, RM, KM>, dim3((unsigned)(tiles * A.parts), (unsigned)A.Hkv, (unsigned)A.R), dim3(AW_THREADS), 0, stream, A, few_rows);
}
template <typename T, int RM, int KM>
static cudaError_t aw_keys(const AwArgs& A, int max_total, int few_rows, int parts, float* sums, cudaStream_t stream) {
  const cudaError_t e = qe_launch(attention_weights_keys_kernel<T, RM, KM>, dim3((unsigned)((max_total + 16 * KM - 1) / (16 * KM) * parts), (unsigned)A.Hkv, (unsigned)A.R),
                                  dim3(AW_THREADS), 0, stream, A, few_rows, parts, sums, (long)max_total);
  return e != cudaSuccess || sums == nullptr ? e : aw_finish(A, sums, max_total, parts, few_rows, max_total, stream);
}
// Tiles: 16 rows where no request has more (decoded tokens), else 64 rows x 128 keys (32 products a thread for 12 numbers from shared memory, two CTAs an
// SM; with 128 x 128 there is one, whose 8 warps do not cover each other), or 64 x 64 where those are fewer than two an SM.
template <typename T>
static cudaError_t aw_dispatch(const AwArgs& A, long rows, int max_total, int few_rows, int parts, float* sums, cudaStream_t stream) {
  const bool small = (rows + 63) / 64 * ((max_total + 127) / 128) * A.Hkv * A.R < 296;
  const cudaError_t e = rows <= 16 ? aw_rows<T, 1, 8>(A, rows, few_rows, stream) : (small ? aw_rows<T, 4, 4>(A, rows, few_rows, stream) : aw_rows<T, 4, 8>(A, rows, few_rows, stream));
  if (e != cudaSuccess) return e;
  if (rows <= 16) return aw_keys<T, 1, 8>(A, max_total, few_rows, parts, sums, stream);
  return small ? aw_keys<T, 4, 4>(A, max_total, few_rows, parts, sums, stream) : aw_keys<T, 4, 8>(A, max_total, few_rows, parts, sums, stream);
}

// parts, parts2: of the rows' keys (stats: [T Hq, parts, 2]), and of the keys' rows (sums: [parts2, R, Hkv, max_total] where there is more than one).
// few_rows: requests of at most so many rows (a query token x a query head of a kv head's group) are left to another kernel (-1: none).
extern "C" int qe_attention_weights(const void* q, long q_stride, int T, const void* pages, int num_pages, int planes,
                                    const int* block_tables, int max_blocks, const int* cu_q, const int* ctx_lens, const int* slot_ids,
                                    const int* counted, const int* step_positions, int* positions, const float* weights, float* out,
                                    int slots, long capacity, int R, int Hq, int Hkv, int D, int page, int window, float scale,
                                    float softcap, const float* slopes, const float* sinks, float* stats, int parts, int max_q, int max_total,
                                    int few_rows, int parts2, float* sums, int dtype, cudaStream_t stream) {
  if (R <= 0 || max_total <= 0) return 0;
  if (Hkv < 1 || Hq % Hkv || D < 1 || page < 1) QE_REFUSE("attention_weights: heads %d/%d, head_dim %d, pages of %d", Hq, Hkv, D, page);
  if (R > 65535 || Hkv > 65535) QE_REFUSE("attention_weights: %d requests, %d kv heads are more than a launch takes", R, Hkv);
  if (parts < 1 || parts2 < 1 || (parts2 > 1 && sums == nullptr)) QE_REFUSE("attention_weights: %d and %d parts", parts, parts2);
  AwArgs A{q, q_stride, T, pages, num_pages, planes, block_tables, max_blocks, cu_q, ctx_lens, slot_ids, counted, step_positions, positions,
           weights, out, slots, capacity, R, Hq, Hkv, D, page, aw_shift(page), window, scale, softcap, slopes, sinks, stats, parts};
  const long rows = (long)max_q * (Hq / Hkv);
  if ((rows + 15) / 16 * parts > 0x7fffffffL) QE_REFUSE("attention_weights: %d tokens are more than a launch takes", max_q);
  const cudaError_t e = dtype == QE_DTYPE_F32 ? aw_dispatch<float>(A, rows, max_total, few_rows, parts2, parts2 > 1 ? sums : nullptr, stream)
                                               : aw_dispatch<__nv_bfloat16>(A, rows, max_total, few_rows, parts2, parts2 > 1 ? sums : nullptr, stream);
  if (e != cudaSuccess) { qe_set_error("attention_weights: launch failed: %s", cudaGetErrorString(e)); (void)cudaGetLastError(); return 2; }
  return 0;
}

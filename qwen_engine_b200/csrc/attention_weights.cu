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
#include "attention_weights.cuh"

#define AW_TILE 64             // rows and keys of a tile
#define AW_KC 32               // channels at a time
#define AW_THREADS 256
#define AW_PITCH (AW_TILE + 4)

struct AwTile {
  float q[AW_KC][AW_PITCH];
  float k[AW_KC][AW_PITCH];
};

// s[i][j] of rows rho0 + 4 ty + i and keys key0 + 4 tx + j of head c; rows and keys that do not exist read as zeros.
template <typename T>
__device__ __forceinline__ void aw_products(const AwArgs& A, const AwReq& R, int r, int c, int rho0, int key0, AwTile& sm, float (&s)[4][4]) {
  const int G = A.Hq / A.Hkv, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
  // this thread fetches channels of row / key tid / 4
  const int who = tid >> 2, ch = (tid & 3) * 8;
  const T* qp = nullptr;
  const T* kp = nullptr;
  {
    const int rho = rho0 + who;
    if (rho < R.n * G) {
      const int t = rho / G, g = rho - t * G;
      qp = reinterpret_cast<const T*>(A.q) + (size_t)(R.row0 + t) * A.q_stride + (size_t)(c * G + g) * A.D;
    }
    const int key = key0 + who;
    const int page = key < R.total ? aw_page(A, r, key) : -1;
    if (page >= 0)
      kp = reinterpret_cast<const T*>(A.pages) + (((size_t)page * A.planes * A.Hkv + c) * A.page + key % A.page) * A.D;
  }
  for (int d0 = 0; d0 < A.D; d0 += AW_KC) {
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int d = d0 + ch + x;
      sm.q[ch + x][who] = qp && d < A.D ? to_f32(qp[d]) : 0.f;
      sm.k[ch + x][who] = kp && d < A.D ? to_f32(kp[d]) : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int d = 0; d < AW_KC; ++d) {
      const float4 a = *reinterpret_cast<const float4*>(&sm.q[d][4 * ty]);
      const float4 b = *reinterpret_cast<const float4*>(&sm.k[d][4 * tx]);
      const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(av[i], bv[j], s[i][j]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(AW_THREADS)
attention_weights_rows_kernel(AwArgs A, int few_rows) {
  __shared__ AwTile sm;
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.z, c = blockIdx.y, tile = blockIdx.x / A.parts, part = blockIdx.x - tile * A.parts;
  const AwReq R = aw_req(A, r);
  const int G = A.Hq / A.Hkv, rho0 = tile * AW_TILE, rows = R.counted * G;
  if (rho0 >= rows || (long)R.n * G <= few_rows) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  // the tile's keys, and this part's share of their tiles
  const int first = R.ctx + rho0 / G, last = R.ctx + (min(rho0 + AW_TILE, rows) - 1) / G;
  const int lo = A.window > 0 ? max(0, first - A.window + 1) / AW_TILE * AW_TILE : 0;
  const int tiles = (last - lo) / AW_TILE + 1, per = (tiles + A.parts - 1) / A.parts;
  float m[4], z[4], slope[4];
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rho = rho0 + 4 * ty + i;
    m[i] = -INFINITY; z[i] = 0.f;
    pos[i] = rho < rows ? R.ctx + rho / G : -1;
    slope[i] = A.slopes ? A.slopes[c * G + rho % G] : 0.f;
  }
  for (int kt = part * per; kt < min(tiles, (part + 1) * per); ++kt) {
    const int key0 = lo + kt * AW_TILE;
    float s[4][4];
    aw_products<T>(A, R, r, c, rho0, key0, sm, s);
    bool held[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) held[j] = aw_page(A, r, key0 + 4 * tx + j) >= 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + 4 * tx + j;
        const bool seen = held[j] && key <= pos[i] && (A.window <= 0 || key > pos[i] - A.window);
        s[i][j] = seen ? aw_score(A, s[i][j], slope[i], pos[i] - key) : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
      if (mx == -INFINITY) continue;
      float sum = z[i] * exp2f(m[i] - mx);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += exp2f(s[i][j] - mx);
      m[i] = mx; z[i] = sum;
    }
  }
  // a row's 16 threads put their maxima and sums together
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m[i], o), oz = __shfl_xor_sync(0xffffffffu, z[i], o);
      const float nm = fmaxf(m[i], om);
      if (nm != -INFINITY) z[i] = z[i] * exp2f(m[i] - nm) + oz * exp2f(om - nm);
      m[i] = nm;
    }
    const int rho = rho0 + 4 * ty + i;
    if (tx == 0 && rho < rows) {
      const int t = rho / G;
      float* st = A.stats + (((size_t)(R.row0 + t) * A.Hq + c * G + (rho - t * G)) * A.parts + part) * 2;
      st[0] = m[i]; st[1] = z[i];
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(AW_THREADS)
attention_weights_keys_kernel(AwArgs A, int few_rows) {
  __shared__ AwTile sm;
  __shared__ float2 row[AW_TILE];
  __shared__ float sums[16][AW_PITCH];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.z, c = blockIdx.y, key0 = blockIdx.x * AW_TILE;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  const int G = A.Hq / A.Hkv;
  if (key0 >= R.total || slot < 0 || slot >= A.slots || (few_rows >= 0 && (long)R.n * G <= few_rows)) return;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  // the rows that see any of these keys
  const int t0 = max(0, key0 - R.ctx);
  const int t1 = A.window > 0 ? (int)min((long)R.counted, (long)key0 + AW_TILE - 1 + A.window - R.ctx) : R.counted;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  bool held[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) held[j] = aw_page(A, r, key0 + 4 * tx + j) >= 0;
  for (int rho0 = t0 * G; rho0 < t1 * G; rho0 += AW_TILE) {
    if (tid < AW_TILE) {
      const int rho = rho0 + tid;
      float2 v = make_float2(0.f, 0.f);
      if (rho < t1 * G) {
        const int t = rho / G, head = c * G + (rho - t * G);
        v = aw_merge(A.stats + ((size_t)(R.row0 + t) * A.Hq + head) * A.parts * 2, A.parts, A.sinks ? A.sinks + head : nullptr);
      }
      row[tid] = v;
    }
    float s[4][4];
    aw_products<T>(A, R, r, c, rho0, key0, sm, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rho = rho0 + 4 * ty + i;
      const int pos = rho < t1 * G ? R.ctx + rho / G : -1;
      const float slope = A.slopes ? A.slopes[c * G + rho % G] : 0.f;
      const float2 mz = row[4 * ty + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + 4 * tx + j;
        const bool seen = held[j] && key <= pos && (A.window <= 0 || key > pos - A.window);
        if (seen) acc[j] += exp2f(aw_score(A, s[i][j], slope, pos - key) - mz.x) * mz.y;
      }
    }
    __syncthreads();                              // `row` is written anew
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) sums[ty][4 * tx + j] = acc[j];
  __syncthreads();
  const int key = key0 + tid;
  if (tid < AW_TILE && key < R.total) {
    float total = 0.f;
#pragma unroll
    for (int y = 0; y < 16; ++y) total += sums[y][tid];
    const size_t at = ((size_t)slot * A.Hkv + c) * A.capacity + key;
    A.out[at] = key < R.ctx ? A.weights[at] + total : total;
    if (A.positions && key >= R.ctx) A.positions[at] = A.step_positions[R.row0 + key - R.ctx];
  }
}

// few_rows: requests of at most so many rows (a query token x a query head of a kv head's group) are left to another kernel (-1: none).
extern "C" int qe_attention_weights(const void* q, long q_stride, int T, const void* pages, int num_pages, int planes,
                                    const int* block_tables, int max_blocks, const int* cu_q, const int* ctx_lens, const int* slot_ids,
                                    const int* counted, const int* step_positions, int* positions, const float* weights, float* out,
                                    int slots, long capacity, int R, int Hq, int Hkv, int D, int page, int window, float scale,
                                    float softcap, const float* slopes, const float* sinks, float* stats, int parts, int max_q, int max_total,
                                    int few_rows, int dtype, cudaStream_t stream) {
  if (R <= 0 || max_total <= 0) return 0;
  if (Hkv < 1 || Hq % Hkv || D < 1 || page < 1) QE_REFUSE("attention_weights: heads %d/%d, head_dim %d, pages of %d", Hq, Hkv, D, page);
  if (R > 65535 || Hkv > 65535) QE_REFUSE("attention_weights: %d requests, %d kv heads are more than a launch takes", R, Hkv);
  if (parts < 1) QE_REFUSE("attention_weights: %d parts", parts);
  AwArgs A{q, q_stride, T, pages, num_pages, planes, block_tables, max_blocks, cu_q, ctx_lens, slot_ids, counted, step_positions, positions,
           weights, out, slots, capacity, R, Hq, Hkv, D, page, aw_shift(page), window, scale, softcap, slopes, sinks, stats, parts};
  const long row_tiles = ((long)max_q * (Hq / Hkv) + AW_TILE - 1) / AW_TILE, key_tiles = ((long)max_total + AW_TILE - 1) / AW_TILE;
  if (row_tiles * parts > 0x7fffffffL) QE_REFUSE("attention_weights: %d rows are more than a launch takes", max_q);
  const dim3 grid_rows((unsigned)(row_tiles * parts), (unsigned)Hkv, (unsigned)R), grid_keys((unsigned)key_tiles, (unsigned)Hkv, (unsigned)R);
  if (dtype == QE_DTYPE_F32) {
    if (row_tiles > 0) qe_launch(attention_weights_rows_kernel<float>, grid_rows, dim3(AW_THREADS), 0, stream, A, few_rows);
    qe_launch(attention_weights_keys_kernel<float>, grid_keys, dim3(AW_THREADS), 0, stream, A, few_rows);
  } else {
    if (row_tiles > 0) qe_launch(attention_weights_rows_kernel<__nv_bfloat16>, grid_rows, dim3(AW_THREADS), 0, stream, A, few_rows);
    qe_launch(attention_weights_keys_kernel<__nv_bfloat16>, grid_keys, dim3(AW_THREADS), 0, stream, A, few_rows);
  }
  QE_CHECK_LAUNCH("attention_weights");
  return 0;
}

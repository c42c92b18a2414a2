// What the kernels that gather attention weights (attention_weights*.cu) share: their arguments and the score of a pair.
#pragma once
#include "common.cuh"
#include <math.h>

#define AW_LOG2E 1.4426950408889634f

// Rows of request r: its query tokens x the query heads of one kv head's group (row = token * G + head of the group).  The
// query at place t of the step's tokens of request r stands behind ctx_lens[r] + t cached tokens.
struct AwArgs {
  const void* q; long q_stride; int T;               // queries of the step: T rows, q_stride elements apart, Hq D wide
  const void* pages; int num_pages, planes;          // [num_pages, planes, Hkv, page, D]; plane 0 holds the keys
  const int* block_tables; int max_blocks;
  const int* cu_q; const int* ctx_lens; const int* slot_ids; const int* counted;     // counted: null, or rows of each request that count
  const int* step_positions; int* positions;         // positions: null, or where the new tokens' positions are noted
  const float* weights; float* out;                  // [slots, Hkv, capacity]
  int slots; long capacity;
  int R, Hq, Hkv, D, page, page_shift, window;      // page_shift: log2 of the page, -1 where it is no power of two
  float scale, softcap;
  const float* slopes; const float* sinks;
  float* stats; int parts;                           // [(token * Hq + head), parts, 2]: a part's maximum (of log2) and sum
};

// what request r brings: its first row, tokens, tokens that count, cached tokens, and places (all of them clamped to what exists)
struct AwReq { int row0, n, counted, ctx, total; };
__device__ __forceinline__ AwReq aw_req(const AwArgs& A, int r) {
  AwReq q;
  q.row0 = min(max(A.cu_q[r], 0), A.T);
  q.n = min(max(A.cu_q[r + 1] - q.row0, 0), A.T - q.row0);
  q.ctx = max(A.ctx_lens[r], 0);
  const long most = min((long)A.max_blocks * A.page, A.capacity);
  q.ctx = (int)min((long)q.ctx, most);
  q.n = (int)min((long)q.n, most - q.ctx);
  q.total = q.ctx + q.n;
  q.counted = A.counted ? min(max(A.counted[r], 0), q.n) : q.n;
  return q;
}

// log2(e) times the score of a pair whose raw product is x; dist = the query's place - the key's
__device__ __forceinline__ float aw_score(const AwArgs& A, float x, float slope, int dist) {
  x *= A.scale;
  if (A.softcap > 0.f) x = A.softcap * tanhf(x / A.softcap);
  if (A.slopes) x -= slope * (float)dist;
  return x * AW_LOG2E;
}

__device__ __forceinline__ int aw_block(const AwArgs& A, int key) { return A.page_shift >= 0 ? key >> A.page_shift : key / A.page; }
__host__ __forceinline__ int aw_shift(int page) {
  int s = 0;
  while ((1 << s) < page) ++s;
  return (1 << s) == page ? s : -1;
}
// 2^x by the instruction alone (results below 2^-126 are zero)
__device__ __forceinline__ float aw_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }

// a key's page, or -1: no place of the table, or a place that holds no page
__device__ __forceinline__ int aw_page(const AwArgs& A, int r, int key) {
  const int b = aw_block(A, key);
  if (b >= A.max_blocks) return -1;
  const int p = A.block_tables[(size_t)r * A.max_blocks + b];
  return p < A.num_pages ? p : -1;
}

// A row's maximum as exponents are taken relative to it: 0 where there is none (a row that sees nothing, or nothing but -inf and NaN), so that
// what is added up is 0, or NaN for a NaN.
__device__ __forceinline__ float aw_base(float m) { return m == -INFINITY ? 0.f : m; }

// A row's parts put together: the maximum, and the reciprocal of the softmax's denominator (0 for a row that sees nothing, NaN for one
// that sees a NaN).
__device__ __forceinline__ float2 aw_merge(const float* st, int parts, const float* sink) {
  float m = -INFINITY, z = 0.f;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, st[2 * p]);
  const float base = aw_base(m);
  for (int p = 0; p < parts; ++p) z += st[2 * p + 1] * exp2f(st[2 * p] - base);
  if (m == -INFINITY) return make_float2(0.f, z);       // (0 or NaN)
  if (sink) z += exp2f(*sink * AW_LOG2E - m);
  return make_float2(m, 1.f / z);
}

// Adds the parts of the keys' sums ([parts, R, Hkv, ld]) up, in their order, and writes the output of the requests of more than few_rows rows (attention_weights.cu).
cudaError_t aw_finish(const AwArgs& A, const float* sums, long ld, int parts, int few_rows, int max_total, cudaStream_t stream);

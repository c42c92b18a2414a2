// Verification of drafted tokens against the target's probabilities, with given uniform numbers.
//
// Request r has the logit rows starts[r] .. starts[r + 1] - 1 of the step: row i is followed by draft i, the last row by no
// draft.  With p the softmax of row i's logits (those at or above the top_k-th largest, divided by the temperature; one-hot
// at the lowest of the largest logits where the temperature is 0) and q the draft's probabilities, formed alike from the
// draft model's logits or one-hot at the draft where none are given, draft i stands if u_i q(d_i) < p(d_i).  Behind the
// drafts in front of the first that falls comes one more token, drawn with the number of the request's last row: from
// max(p - q, 0) of the row whose draft fell, or from p of the last row where all stand (the first index whose running sum
// exceeds u times the whole).  That makes the tokens' distribution the target's, whatever q is.
//
// Two kernels.  The first reads every logit once: a row is shared by a cluster of up to VF_MAX_CTAS CTAs, and each
// leaves its chunk's maximum and sum of exponentials.  The second has a cluster for every request: it puts the chunks' sums
// together, holds the drafts against them, and draws.
//
// The top_k-th largest logit.  Of a chunk's logits only the k largest can be among the row's k largest, and the k-th largest of
// the threads' maxima (of the maxima of either half of their logits, for a k of some hundreds) is a lower bound of the chunk's k-th largest: hardly
// more than k logits reach it.  (A thread without a logit above -inf counts with the lowest finite number, so the bound is one of the logits above
// -inf; where fewer than k of those are listed, they are all that the row has, and all are kept.)  The CTAs list theirs, and the k-th largest of the
// lists (each number compared with every other, or bit by bit) is the row's.  Where k is large, or the lists overflow (equal logits), the digits of an order-preserving integer are found one
// after the other from histograms that meet in distributed shared memory.
//
// Precision.  Whether a draft stands is one comparison of float32 exponentials with float64 sums: it goes the other way
// than exact arithmetic for about one u in 10^7.  Drawing is another matter: a running sum over V terms has V borders, and an
// error of 10^-8 in the sums moves a border across u for one draw in some hundreds.  So the second kernel forms exponentials
// (to 10^-12 of their value: a table of 2^(i / 32) and a polynomial of degree 4) and sums in float64, for the one or two rows of a
// request that it draws from.  It goes over them once: max(p - q, 0) needs the quotient of the rows' whole sums, but which
// terms are positive is decided well enough by the first kernel's (a term that this gets wrong is 10^-8 of p), so sums of e_p and
// e_q over the positive terms and over all are taken together and the quotient is applied to the sums.
//
// What bounds them: the first, memory (64 requests of 5 drafts over 151 936 logits: 428 MB in 79 us, 5.4 TB/s; with a top_k of 20 in every second
// request 105); the second, the float64 exponentials of its one or two rows and the chain around them (the same case 55 us; 1 request of 4
// drafts 16 us behind the first kernel's 6).
#include "common.cuh"
#include <math.h>
#include <float.h>

#define VF_MAX_CTAS 8      // CTAs of a cluster at most: chunks of a row
#define VF_MAX_DRAW 16     // ... of the cluster that draws for a request
#define VF_THREADS 512
#define VF_WARPS (VF_THREADS / 32)

struct __align__(16) VfPart { double z; float m; int arg; };     // of a chunk: sum of exp((x - m) / T), maximum, its lowest place

// order-preserving map float -> uint32 (larger float, larger key; NaN lowest, -0 as +0)
__device__ __forceinline__ unsigned vf_key(float f) {
  f = fmaxf(f, -INFINITY) + 0.f;
  const unsigned u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// elements e .. e + 3 of a row, -inf where there are none
__device__ __forceinline__ float4 vf_raw(const float* p, int e, int V) {
  float4 v;
  if (e >= 0 && e + 4 <= V && (reinterpret_cast<uintptr_t>(p + e) & 15) == 0) {
    v = __ldg(reinterpret_cast<const float4*>(p + e));
  } else {
    v.x = e >= 0 && e < V ? __ldg(p + e) : -INFINITY;
    v.y = e + 1 >= 0 && e + 1 < V ? __ldg(p + e + 1) : -INFINITY;
    v.z = e + 2 >= 0 && e + 2 < V ? __ldg(p + e + 2) : -INFINITY;
    v.w = e + 3 >= 0 && e + 3 < V ? __ldg(p + e + 3) : -INFINITY;
  }
  return v;
}
__device__ __forceinline__ float4 vf_clean(const float4& v) {
  return make_float4(fmaxf(v.x, -INFINITY), fmaxf(v.y, -INFINITY), fmaxf(v.z, -INFINITY), fmaxf(v.w, -INFINITY));
}

// A row as groups of four logits that lie on 16-byte boundaries: group g holds the elements 4 g - lead ..; the elements of a
// group that are not the row's read as -inf.  `get` reads NaN as -inf, too.
struct VfRow {
  const float* p;
  int lead, V, groups;
  __device__ __forceinline__ VfRow(const float* row, int V_) : p(row), V(V_) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    groups = (lead + V_ + 3) >> 2;
  }
  // as the memory holds them (nothing waits for the load until the values are used)
  __device__ __forceinline__ float4 raw(int g) const { return vf_raw(p, 4 * g - lead, V); }
  __device__ __forceinline__ float4 get(int g) const { return vf_clean(raw(g)); }
};

// log2(e) / T, finite and not zero whatever T > 0 (-inf times it is -inf)
__device__ __forceinline__ float vf_scale(float T) { return fmaxf(fminf(1.4426950408889634f / T, FLT_MAX), FLT_MIN); }

// The request that row n (of the target's rows, or of the drafts: less = 1) belongs to: the last r with starts[r] - r * less <= n, found by
// the whole CTA with one round of loads (every CTA of a cluster finds the same one, whatever the starts are).
__device__ __forceinline__ int vf_owner(const int* starts, int R, int n, int less, int* s) {
  if (threadIdx.x == 0) *s = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < R; r += VF_THREADS)
    if (starts[r] - r * less <= n && (r + 1 == R || starts[r + 1] - (r + 1) * less > n)) atomicMax(s, r);
  __syncthreads();
  return *s;
}

__device__ __forceinline__ float vf_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float vf_unkey(unsigned k) { return k == 0u ? -INFINITY : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ unsigned vf_ld_remote(const unsigned* local, int cta) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(cluster_map_shared(local, cta)) : "memory");
  return v;
}

#define VF_LIST 1024         // logits of a chunk that may reach the lower bound
#define VF_ALL 2048          // ... of a row's chunks together
#define VF_RANKED 512        // ... up to which each is compared with every other
#define VF_LIST_K 768        // top_k a chunk up to which the lists are tried (a bound from 2 x 512 maxima says little beyond)
#define VF_AHEAD 4           // groups of four logits that a thread asks for at a time

__device__ __forceinline__ float2 vf_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 vf_mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float vf_max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// A thread's running maximum and sum of exponentials take a group in.  A NaN (a logit that is one, or inf - inf) shows in the sum,
// which is then formed again, logit by logit.
__device__ __forceinline__ void vf_take(const float4& x, float c, float& m, float& s) {
  const float top = fmaxf(vf_max3(x.x, x.y, x.z), x.w);
  if (top > m) {
    s *= vf_ex2((m - top) * c);
    m = top;
  }
  const float2 nm = make_float2(-m, -m), cc = make_float2(c, c);
  const float2 a = vf_mul2(vf_add2(make_float2(x.x, x.y), nm), cc), b = vf_mul2(vf_add2(make_float2(x.z, x.w), nm), cc);
  float t = (vf_ex2(a.x) + vf_ex2(a.y)) + (vf_ex2(b.x) + vf_ex2(b.y));
  if (t != t) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    t = 0.f;
    for (int j = 0; j < 4; ++j) t += v[j] == m ? 1.f : (v[j] < m ? vf_ex2((v[j] - m) * c) : 0.f);
  }
  s += t;
}

__global__ void __launch_bounds__(VF_THREADS, 3)
verify_sums_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ starts,
                   const float* __restrict__ temperature, const int* __restrict__ top_k, VfPart* __restrict__ parts,
                   unsigned* __restrict__ thresholds, int N, int R, int V) {
  __shared__ unsigned hist[256], list[VF_LIST];
  __shared__ __align__(16) unsigned all[VF_ALL + 4];
  __shared__ unsigned digit_s, above_s, listed, bound, found, sizes[VF_MAX_CTAS];
  __shared__ unsigned warp_tot[VF_WARPS];
  __shared__ int warp_two[2][VF_WARPS];
  __shared__ double sz[VF_WARPS];
  __shared__ int owner;
  pdl_launch_dependents();
  pdl_wait();
  const int C = (int)cluster_num_ctas(), rank = (int)cluster_cta_rank(), y = blockIdx.x / C;
  const bool draft = y >= N;
  const int r = vf_owner(starts, R, draft ? y - N : y, draft ? 1 : 0, &owner);
  const float T = temperature[r];
  const bool greedy = !(T > 0.f);
  if (draft && greedy) return;                  // (the whole cluster: the row is not looked at)
  const VfRow row(draft ? draft_logits + (size_t)(y - N) * V : logits + (size_t)y * V, V);
  const int per = (row.groups + C - 1) / C;
  const int g0 = min(row.groups, rank * per), g1 = min(row.groups, g0 + per);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int k = top_k[r];
  const bool some = !greedy && k > 0 && k < V;  // the row keeps its k largest
  const float c = vf_scale(T);
  // the thread's groups: g0 + tid + i VF_THREADS, the first and the last of the row (which may reach beyond it) with care
  float m = -FLT_MAX, s = 0.f, half[2] = {-INFINITY, -INFINITY};      // half: the maxima of every second group, for the bound of a large top_k
  int at = 0x7fffffff;
  if (greedy) m = -INFINITY;
  for (int g = g0 + tid; g < g1; g += VF_AHEAD * VF_THREADS) {
    float4 x[VF_AHEAD];
    if (g >= 1 && g + (VF_AHEAD - 1) * VF_THREADS < g1 - 1) {
#pragma unroll
      for (int i = 0; i < VF_AHEAD; ++i) x[i] = __ldg(reinterpret_cast<const float4*>(row.p - row.lead) + g + i * VF_THREADS);
    } else {
#pragma unroll
      for (int i = 0; i < VF_AHEAD; ++i)
        x[i] = g + i * VF_THREADS < g1 ? row.get(g + i * VF_THREADS) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
#pragma unroll
    for (int i = 0; i < VF_AHEAD; ++i) {
      if (!greedy && !some) {
        vf_take(x[i], c, m, s);
      } else {
        const float top = fmaxf(vf_max3(x[i].x, x[i].y, x[i].z), x[i].w);
        if (greedy && top > m) {                // (groups come in rising order: the lowest place of the thread's maximum)
          const int e = 4 * (g + i * VF_THREADS) - row.lead;
          at = x[i].x == top ? e : (x[i].y == top ? e + 1 : (x[i].z == top ? e + 2 : e + 3));
        }
        m = fmaxf(m, top);
        half[i & 1] = fmaxf(half[i & 1], top);
      }
    }
  }
  // the chunk's maximum
  const unsigned mine = g0 + tid < g1 ? vf_key(m) : 0u;        // 0: this thread has no logit
  const unsigned wmax = __reduce_max_sync(0xffffffffu, mine);
  if (lane == 0) warp_tot[warp] = wmax;
  if (tid == 0) listed = 0u;
  __syncthreads();
  unsigned cmax = 0u;
#pragma unroll
  for (int w = 0; w < VF_WARPS; ++w) cmax = max(cmax, warp_tot[w]);
  if (greedy) {
    // the lowest place that holds it
    const int a = __reduce_min_sync(0xffffffffu, mine == cmax ? at : 0x7fffffff);
    __syncthreads();
    if (lane == 0) warp_tot[warp] = (unsigned)a;
    __syncthreads();
    if (tid == 0) {
      unsigned b = warp_tot[0];
      for (int w = 1; w < VF_WARPS; ++w) b = min(b, warp_tot[w]);
      parts[(size_t)y * C + rank] = VfPart{0.0, vf_unkey(cmax), (int)b};
    }
    return;                                     // (the whole cluster)
  }
  const float cm = fmaxf(vf_unkey(cmax), -FLT_MAX);
  // the sum, relative to the chunk's maximum
  double z = s > 0.f ? (double)(s * (m == cm ? 1.f : vf_ex2((m - cm) * c))) : 0.0;

  unsigned thr = 0u;
  if (some) {
    bool from_list = false;
    const int kc = (k + C - 1) / C;
    if (kc <= VF_LIST_K) {
      // The high half of the k / C-th largest of the threads' maxima, in every chunk: at least k logits, or all above -inf, reach the
      // least of those numbers, so it is a lower bound of the k-th largest of the logits above -inf.
      unsigned low = 0u;
      const unsigned h0 = vf_key(half[0]), h1 = g0 + tid + VF_THREADS < g1 ? vf_key(half[1]) : 0u;
      for (int bit = 31; bit >= 16; --bit) {
        const unsigned cand = low | (1u << bit);
        int n = kc <= VF_THREADS / 4 ? __syncthreads_count(mine >= cand) : __syncthreads_count(mine != 0u && h0 >= cand) + __syncthreads_count(h1 >= cand);
        if (n >= kc) low = cand;
      }
      if (tid == 0) bound = low;
      cluster_sync_all();
      for (int o = 0; o < C; ++o) low = min(low, vf_ld_remote(&bound, o));
      if (mine >= low)                          // (few threads look at their logits again)
        for (int g = g0 + tid; g < g1; g += VF_AHEAD * VF_THREADS) {
          float4 x4[VF_AHEAD];
#pragma unroll
          for (int i = 0; i < VF_AHEAD; ++i)
            if (g + i * VF_THREADS < g1) x4[i] = row.raw(g + i * VF_THREADS);
#pragma unroll
          for (int i = 0; i < VF_AHEAD; ++i) {
            if (g + i * VF_THREADS >= g1) break;
            const float4 v = vf_clean(x4[i]);
            const float x[4] = {v.x, v.y, v.z, v.w};
            const int e = 4 * (g + i * VF_THREADS) - row.lead;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (vf_key(x[j]) >= low && e + j >= 0 && e + j < V) {
                if (*reinterpret_cast<volatile unsigned*>(&listed) > VF_LIST) break;      // (it overflowed: nothing more is counted)
                const unsigned n = atomicAdd(&listed, 1u);
                if (n < VF_LIST) list[n] = vf_key(x[j]);
              }
          }
        }
      cluster_sync_all();
      if (tid < C) sizes[tid] = vf_ld_remote(&listed, tid);
      __syncthreads();
      unsigned total = 0u, most = 0u;
      for (int o = 0; o < C; ++o) { most = max(most, sizes[o]); total += sizes[o]; }
      from_list = most <= VF_LIST && total <= VF_ALL;
      if (from_list)
        for (unsigned i = tid; i < total; i += VF_THREADS) {
          unsigned at = i;
          int o = 0;
          while (at >= sizes[o]) at -= sizes[o++];
          all[i] = vf_ld_remote(&list[at], o);
        }
      if (from_list && tid < 4) all[total + tid] = 0u;         // (read four at a time below)
      cluster_sync_all();                       // the lists have been read
      if (from_list) {
        if (total < (unsigned)k) {
          thr = 0u;                             // all that is above -inf is listed, and stays
        } else if (total <= VF_RANKED) {
          // the k-th largest: the one with fewer than k above it and at least k with its equals
          if (tid < total) {
            const unsigned key = all[tid];
            int above = 0, equal = 0;
            for (unsigned j = 0; j < total; j += 4) {
              const uint4 o = *reinterpret_cast<const uint4*>(all + j);
              above += (o.x > key) + (o.y > key) + (o.z > key) + (o.w > key);
              equal += (o.x == key) + (o.y == key) + (o.z == key) + (o.w == key);
            }
            if (above < k && above + equal >= k) found = key;
          }
          __syncthreads();
          thr = found;
        } else {
          // bit by bit
          unsigned keys[VF_ALL / VF_THREADS];
#pragma unroll
          for (int i = 0; i < VF_ALL / VF_THREADS; ++i) keys[i] = (unsigned)(i * VF_THREADS + tid) < total ? all[i * VF_THREADS + tid] : 0u;
          for (int bit = 31; bit >= 0; --bit) {
            const unsigned cand = thr | (1u << bit);
            int n = 0;
#pragma unroll
            for (int i = 0; i < VF_ALL / VF_THREADS; ++i) n += keys[i] >= cand;
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0) warp_two[bit & 1][warp] = n;         // (two in turn: one meeting a bit)
            __syncthreads();
            n = 0;
#pragma unroll
            for (int w = 0; w < VF_WARPS; ++w) n += warp_two[bit & 1][w];
            if (n >= k) thr = cand;
          }
        }
        for (unsigned i = tid; i < listed; i += VF_THREADS)      // (the chunk's kept logits are in its list)
          if (list[i] >= thr) {
            const float x = vf_unkey(list[i]);
            z += x == cm ? 1.0 : (double)vf_ex2((x - cm) * c);
          }
      }
    }
    if (!from_list) {
      unsigned left = (unsigned)k;              // the threshold is the left-th largest among the keys with the digits found so far
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += VF_THREADS) hist[i] = 0u;
        __syncthreads();
        const unsigned mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        for (int g = g0 + tid; g < g1; g += VF_THREADS) {
          const float4 v = row.get(g);
          const float x[4] = {v.x, v.y, v.z, v.w};
          const int e = 4 * g - row.lead;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned key = vf_key(x[j]);
            if (e + j >= 0 && e + j < V && (key & mask) == (thr & mask)) atomicAdd(&hist[(key >> shift) & 255u], 1u);
          }
        }
        cluster_sync_all();
        // every CTA adds the histograms up; thread t has the digit 255 - t
        unsigned n = 0u;
        if (tid < 256) {
          for (int o = 0; o < C; ++o) n += vf_ld_remote(&hist[255 - tid], o);
        }
        unsigned run = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned up = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += up;
        }
        if (lane == 31) warp_tot[warp] = run;
        __syncthreads();
        if (tid < 256) {
          for (int w = 0; w < warp; ++w) run += warp_tot[w];
          if (run >= left && run - n < left) { digit_s = 255u - tid; above_s = run - n; }
        }
        __syncthreads();
        thr |= digit_s << shift;
        left -= above_s;
        cluster_sync_all();                     // the others' histograms have been read
      }
      if (mine >= thr)
        for (int g = g0 + tid; g < g1; g += VF_THREADS) {
          const float4 v = row.get(g);
          const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (vf_key(x[j]) >= thr) z += x[j] == cm ? 1.0 : (double)vf_ex2((x[j] - cm) * c);
        }
    }
  }
  if (rank == 0 && tid == 0) thresholds[y] = thr;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  if (lane == 0) sz[warp] = z;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < VF_WARPS; ++w) z += sz[w];
    parts[(size_t)y * C + rank] = VfPart{z, cm, 0};
  }
}

// ---- the drafts against the sums, and the token behind them ------------------------------------------------------------------

struct VfStat { float m; double z; };
// a row's chunks put together; a whole chunk at a time is on its way
__device__ __forceinline__ VfStat vf_stat(const VfPart* parts, size_t y, int chunks, float c) {
  VfStat s{-FLT_MAX, 0.0};
  float m[VF_MAX_CTAS];
  double z[VF_MAX_CTAS];
#pragma unroll
  for (int o = 0; o < VF_MAX_CTAS; ++o) {
    const bool in = o < chunks;
    m[o] = in ? __ldg(&parts[y * chunks + o].m) : -FLT_MAX;
    z[o] = in ? __ldg(&parts[y * chunks + o].z) : 0.0;
  }
#pragma unroll
  for (int o = 0; o < VF_MAX_CTAS; ++o) s.m = fmaxf(s.m, m[o]);
#pragma unroll
  for (int o = 0; o < VF_MAX_CTAS; ++o) s.z += z[o] * (m[o] == s.m ? 1.0 : (double)vf_ex2((m[o] - s.m) * c));
  return s;
}
// the lowest place of a row's largest logit, -1 where none is above -inf
__device__ __forceinline__ int vf_argmax(const VfPart* parts, size_t y, int chunks) {
  float m = -INFINITY;
  int at = 0x7fffffff;
  for (int o = 0; o < chunks; ++o) {
    const VfPart p = parts[y * chunks + o];
    if (p.m > m) { m = p.m; at = p.arg; }
  }
  return at == 0x7fffffff ? -1 : at;
}
// exp((x - m) / T) in float64, x <= m finite: with y = 32 log2(e) (x - m) / T = 32 i + j + f, 2^i 2^(j / 32) (1 + f' + f'^2 / 2 + f'^3 / 6 + f'^4 / 24),
// f' = f ln 2 / 32.  The first term left out is below (ln 2 / 64)^5 / 120 = 1.3 10^-12.  k = 32 log2(e) / T; `pow` holds 2^(j / 32).
// y below -28 000 counts as that (10^-263, which no sum notices).  The bound on y is one on its high word: nothing
// is selected in float64.  About 30 instructions, 7.5 cycles a warp on an SM, of which the float64 unit works 5.
__device__ __forceinline__ double vf_exp(float x, double m, double k, const double* pow) {
  double y = ((double)x - m) * k;                      // (not x k - m k, whose rounding would show where m is large)
  y = __hiloint2double((int)min((unsigned)__double2hiint(y), 0xC0DB5800u), __double2loint(y));
  const double shift = 6755399441055744.0;      // 1.5 2^52: the sum's low word is y rounded to an integer
  const double t = y + shift;
  const int n = __double2loint(t);
  const double f = y - (t - shift);
  constexpr double L = 0.021660849392498290;    // ln 2 / 32
  const double q = fma(fma(fma(f, L * L * L * L / 24.0, L * L * L / 6.0), f, L * L / 2.0), f, L);
  const double e = pow[n & 31];
  const double v = fma(e * f, q, e);
  return __hiloint2double(__double2hiint(v) + ((n >> 5) << 20), __double2loint(v));
}
// A logit as the exponentials take it: where the row's maximum is +inf, 0 for those that are and -inf for the others.
__device__ __forceinline__ float vf_level(float x, bool infinite) { return infinite ? (x == INFINITY ? 0.f : -INFINITY) : x; }
#define VF_NOTHING 1e-200     // a weight up to which a place has none

__device__ __forceinline__ double vf_ld_remote(const double* local, int cta) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(v) : "r"(cluster_map_shared(local, cta)) : "memory");
  return v;
}

__global__ void __launch_bounds__(VF_THREADS, 2)
verify_draw_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ draft_tokens,
                   const int* __restrict__ starts, const float* __restrict__ temperature, const float* __restrict__ uniform,
                   const VfPart* __restrict__ parts, const unsigned* __restrict__ thresholds, int* __restrict__ tokens,
                   int* __restrict__ counts, int chunks, int N, int R, int V) {
  __shared__ double s_all_p[VF_WARPS], s_all_q[VF_WARPS], s_pos_p[VF_WARPS], s_pos_q[VF_WARPS];
  __shared__ double x_tot[4], x_all[4 * VF_MAX_DRAW], pow2[32];
  __shared__ int first_s, hit_s[VF_WARPS], any_s[VF_WARPS];
  if (threadIdx.x < 32) pow2[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
  pdl_launch_dependents();
  pdl_wait();
  const int C = (int)cluster_num_ctas(), rank = (int)cluster_cta_rank(), r = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = N - R;
  const int lo = min(max(starts[r], 0), N), hi = min(max(starts[r + 1], lo), N);
  const int n = hi - lo - 1, d0 = lo - r;       // drafts, the first one's index
  if (n < 0 || d0 < 0 || d0 + n > D) {          // row starts that make no sense: no rows, no tokens
    if (rank == 0 && tid == 0) counts[r] = 0;
    return;
  }
  const float T = temperature[r];
  const bool greedy = !(T > 0.f);
  const float c = vf_scale(T);
  if (tid == 0) first_s = n;
  __syncthreads();
  for (int i = tid; i < n; i += VF_THREADS) {
    const int d = draft_tokens[d0 + i];
    bool stands = false;
    if (d >= 0 && d < V) {
      if (greedy) {
        stands = vf_argmax(parts, lo + i, chunks) == d;
      } else {
        const VfStat sp = vf_stat(parts, lo + i, chunks, c);
        const float x = fmaxf(logits[(size_t)(lo + i) * V + d], -INFINITY);                 // (NaN as -inf)
        const double p = vf_key(x) >= thresholds[lo + i] ? (x == sp.m ? 1.0 : (double)vf_ex2((x - sp.m) * c)) : 0.0;
        double q = 1.0, zq = 1.0;
        if (draft_logits) {
          const VfStat sq = vf_stat(parts, N + d0 + i, chunks, c);
          const float xd = fmaxf(draft_logits[(size_t)(d0 + i) * V + d], -INFINITY);
          q = vf_key(xd) >= thresholds[N + d0 + i] ? (xd == sq.m ? 1.0 : (double)vf_ex2((xd - sq.m) * c)) : 0.0;
          zq = sq.z;
        }
        stands = (double)uniform[lo + i] * q * sp.z < p * zq;     // (false where a row has no finite logit)
      }
    }
    if (!stands) atomicMin(&first_s, i);
  }
  __syncthreads();
  const int a = first_s;                        // drafts that stand
  if (rank == 0) {
    for (int i = tid; i <= n; i += VF_THREADS)
      if (i != a) tokens[lo + i] = i < a ? draft_tokens[d0 + i] : -1;
    if (tid == 0) counts[r] = a + 1;
  }
  if (greedy) {
    if (rank == 0 && tid == 0) tokens[lo + a] = max(vf_argmax(parts, lo + a, chunks), 0);
    return;
  }
  const VfRow P(logits + (size_t)(lo + a) * V, V);
  const unsigned thr_p = thresholds[lo + a];
  const bool fell = a < n;
  const float* q_row = fell && draft_logits ? draft_logits + (size_t)(d0 + a) * V : nullptr;
  const unsigned thr_q = q_row ? thresholds[N + d0 + a] : 0u;
  const VfStat sp_a = vf_stat(parts, lo + a, chunks, c), sq_a = q_row ? vf_stat(parts, N + d0 + a, chunks, c) : VfStat{0.f, 1.0};
  const float mp = sp_a.m, mq = sq_a.m;
  const int gone = fell && !q_row ? draft_tokens[d0 + a] : -1;
  const int per = (P.groups + C - 1) / C;
  const int g0 = min(P.groups, rank * per), g1 = min(P.groups, g0 + per);
  const int wper = (per + VF_WARPS - 1) / VF_WARPS;
  const int w0 = min(g1, g0 + warp * wper), w1 = min(g1, w0 + wper);      // the warp's groups: ranges in the order of the row
  const double kk = 46.166241308446828 / (double)T;      // 32 log2(e) / T
  const bool inf_p = mp == INFINITY, inf_q = mq == INFINITY;
  const float top_p = inf_p ? 0.f : mp, top_q = inf_q ? 0.f : mq;
  const double mp64 = (double)top_p, mq64 = (double)top_q;
  // the least logit that is kept: -inf is not, whatever the top_k
  const float least_p = inf_p ? 0.f : fmaxf(vf_unkey(thr_p), -FLT_MAX), least_q = inf_q ? 0.f : fmaxf(vf_unkey(thr_q), -FLT_MAX);
  auto level = [&](const float4& v, bool infinite) {
    const float4 x = vf_clean(v);
    return infinite ? make_float4(vf_level(x.x, true), vf_level(x.y, true), vf_level(x.z, true), vf_level(x.w, true)) : x;
  };
  const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  const double rho0 = q_row ? sp_a.z / sq_a.z : 0.0;        // Z_p / Z_q as the first kernel has it
  double t_all_p = 0.0, t_all_q = 0.0, t_pos_p = 0.0, t_pos_q = 0.0;
  // the next two groups are on their way while one's exponentials are formed
  float4 np[2], nq[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int g = w0 + lane + 32 * i;
    np[i] = nq[i] = none;
    if (g < w1) {
      np[i] = P.raw(g);
      if (q_row) nq[i] = vf_raw(q_row, 4 * g - P.lead, V);
    }
  }
  for (int g = w0 + lane; g < w1; g += 32) {
    const float4 xp = level(np[0], inf_p), xq = level(nq[0], inf_q);
    np[0] = np[1]; nq[0] = nq[1];
    if (g + 64 < w1) {
      np[1] = P.raw(g + 64);
      if (q_row) nq[1] = vf_raw(q_row, 4 * (g + 64) - P.lead, V);
    }
    const float hi_p = fmaxf(fmaxf(xp.x, xp.y), fmaxf(xp.z, xp.w)), hi_q = fmaxf(fmaxf(xq.x, xq.y), fmaxf(xq.z, xq.w));
    if (hi_p < least_p && !(q_row && hi_q >= least_q)) continue;         // (with a top-k most groups)
    const float x[4] = {xp.x, xp.y, xp.z, xp.w}, y[4] = {xq.x, xq.y, xq.z, xq.w};
    double p[4], q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = vf_exp(x[j], mp64, kk, pow2);
    if (q_row) {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = vf_exp(y[j], mq64, kk, pow2);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in_p = x[j] >= least_p, in_q = q_row && y[j] >= least_q;
      if (in_p) t_all_p += p[j];
      if (in_q) t_all_q += q[j];
      if (in_p && 4 * g - P.lead + j != gone && (!in_q || p[j] > rho0 * q[j])) {
        t_pos_p += p[j];
        if (in_q) t_pos_q += q[j];
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    t_all_p += __shfl_xor_sync(0xffffffffu, t_all_p, o);
    t_pos_p += __shfl_xor_sync(0xffffffffu, t_pos_p, o);
    if (q_row) {
      t_all_q += __shfl_xor_sync(0xffffffffu, t_all_q, o);
      t_pos_q += __shfl_xor_sync(0xffffffffu, t_pos_q, o);
    }
  }
  if (lane == 0) { s_all_p[warp] = t_all_p; s_all_q[warp] = t_all_q; s_pos_p[warp] = t_pos_p; s_pos_q[warp] = t_pos_q; }
  __syncthreads();
  if (tid < 4) {
    const double* src = tid == 0 ? s_all_p : (tid == 1 ? s_all_q : (tid == 2 ? s_pos_p : s_pos_q));
    double t = 0.0;
    for (int w = 0; w < VF_WARPS; ++w) t += src[w];
    x_tot[tid] = t;
  }
  cluster_sync_all();
  if (tid < 4 * C) x_all[tid] = vf_ld_remote(&x_tot[tid & 3], tid >> 2);
  __syncthreads();
  double all_p = 0.0, all_q = 0.0, pos_p = 0.0, pos_q = 0.0;
  for (int o = 0; o < C; ++o) { all_p += x_all[4 * o]; all_q += x_all[4 * o + 1]; pos_p += x_all[4 * o + 2]; pos_q += x_all[4 * o + 3]; }
  // weights: max(e_p - rho e_q, 0), or e_p but for the draft that fell; e_p where nothing is left of them, or all drafts stand
  const double rho = q_row && all_q > 0.0 ? all_p / all_q : 0.0;
  const bool plain = !fell || !(pos_p - rho * pos_q > VF_NOTHING);
  double total = 0.0, before = 0.0, mine = 0.0;
  for (int o = 0; o < C; ++o) {
    const double t = plain ? x_all[4 * o] : fmax(x_all[4 * o + 2] - rho * x_all[4 * o + 3], 0.0);
    if (o < rank) before += t;
    if (o == rank) mine = t;
    total += t;
  }
  cluster_sync_all();                           // the others' sums have been read
  auto weights = [&](int g, double (&w)[4]) {
    const float4 xp = level(P.raw(g), inf_p), xq = q_row && !plain ? level(vf_raw(q_row, 4 * g - P.lead, V), inf_q) : none;
    const float x[4] = {xp.x, xp.y, xp.z, xp.w}, y[4] = {xq.x, xq.y, xq.z, xq.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = x[j] >= least_p ? vf_exp(x[j], mp64, kk, pow2) : 0.0;
      if (plain) continue;
      if (y[j] >= least_q && q_row) w[j] = fmax(w[j] - rho * vf_exp(y[j], mq64, kk, pow2), 0.0);
      if (4 * g - P.lead + j == gone) w[j] = 0.0;
    }
  };
  auto warp_sum = [&](int w) { return plain ? s_all_p[w] : fmax(s_pos_p[w] - rho * s_pos_q[w], 0.0); };
  const double target = (double)fminf(fmaxf(uniform[hi - 1], 0.f), 0.99999994f) * total;
  // the CTA, and in it the warp, whose range holds the first running sum above the target
  const double after_all = before + mine;
  if (!(total > VF_NOTHING)) {
    if (rank == 0 && tid == 0) tokens[lo + a] = 0;          // no logit is finite
    return;
  }
  if (!(before <= target && target < after_all)) return;
  double run = before;
  int w = 0;
  for (; w < VF_WARPS; ++w) {
    if (run + warp_sum(w) > target) break;
    run += warp_sum(w);
  }
  if (w == VF_WARPS) {                          // (rounding: the last warp that has any weight)
    for (w = VF_WARPS - 1; w > 0 && !(warp_sum(w) > VF_NOTHING); --w) {}
    run -= warp_sum(w);
  }
  // that warp's range again, 32 groups for each warp of the CTA at a time: which of them, then which of its logits
  const int f0 = min(g1, g0 + w * wper), f1 = min(g1, f0 + wper);
  int last = -1;                                // the last place with any weight: the answer, should rounding leave no other
  for (int gb = f0; gb < f1; gb += 32 * VF_WARPS) {
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    const int g = gb + 32 * warp + lane;
    if (g < f1) weights(g, v);
    const double s = (v[0] + v[1]) + (v[2] + v[3]);
    double inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    __syncthreads();                            // (the warps' sums of the first time, or of the round before, have been read)
    if (lane == 31) s_all_q[warp] = inc;
    __syncthreads();
    double mine_from = run;
    for (int i = 0; i < warp; ++i) mine_from += s_all_q[i];
    const unsigned some = __ballot_sync(0xffffffffu, s > VF_NOTHING);
    const unsigned over = __ballot_sync(0xffffffffu, s > VF_NOTHING && mine_from + inc > target);
    const int who = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : -1);
    int at = -1;
    if (who >= 0 && lane == who) {
      double b = mine_from + (inc - s);
      for (int j = 0; j < 4; ++j) {
        if (v[j] > VF_NOTHING) at = 4 * g - P.lead + j;
        b += v[j];
        if (over && v[j] > VF_NOTHING && b > target) break;
      }
    }
    if (who >= 0) at = __shfl_sync(0xffffffffu, at, who);
    if (lane == 0) { hit_s[warp] = over ? at : -1; any_s[warp] = at; }
    __syncthreads();
    int hit = -1;
    for (int i = VF_WARPS - 1; i >= 0; --i) if (hit_s[i] >= 0) hit = hit_s[i];          // the first warp's
    for (int i = 0; i < VF_WARPS; ++i) if (any_s[i] >= 0) last = any_s[i];
    if (hit >= 0) { last = hit; break; }
    for (int i = 0; i < VF_WARPS; ++i) run += s_all_q[i];
  }
  if (tid == 0 && last >= 0) tokens[lo + a] = last;
}

extern "C" int qe_verify_drafts(const float* logits, const int* draft_tokens, const float* draft_logits, const int* starts,
                                const float* temperature, const int* top_k, const float* uniform, int* tokens, int* counts,
                                void* parts, unsigned* thresholds, int N, int R, int V, cudaStream_t stream) {
  if (R <= 0 || N <= 0) return 0;
  if (V <= 0) QE_REFUSE("verify_drafts: empty vocabulary");
  if (N < R) QE_REFUSE("verify_drafts: %d rows for %d requests", N, R);
  const long rows = (long)N + (draft_logits ? N - R : 0);
  if (rows > 0x7fffffffL / VF_MAX_DRAW) QE_REFUSE("verify_drafts: %ld rows are more than a launch takes", rows);
  // CTAs a row: three rounds of the CTAs that the SMs hold at once, so that a CTA reads a long run of a row where there are many rows;
  // a request to draw for: a CTA an SM.  (Always eight: 64 requests of five drafts, 151 936 logits, 228 us for the first kernel.)
  unsigned ctas = 1, draw = 1;
  while (ctas < VF_MAX_CTAS && rows * ctas < 1332 && V / (2 * ctas) >= 2048) ctas *= 2;
  while (draw < VF_MAX_DRAW && (long)R * draw < 148 && V / (2 * draw) >= 2048) draw *= 2;
  if (draw > 8) {
    static unsigned long long configured = 0;
    const cudaError_t e = qe_once_a_device(configured, [] { return cudaFuncSetAttribute(verify_draw_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
    if (e != cudaSuccess) QE_REFUSE("verify_drafts: clusters of %u CTAs: %s", draw, cudaGetErrorString(e));
  }
  qe_launch_cluster(verify_sums_kernel, dim3((unsigned)(rows * ctas)), dim3(VF_THREADS), 0, stream, ctas, logits, draft_logits,
                    starts, temperature, top_k, (VfPart*)parts, thresholds, N, R, V);
  QE_CHECK_LAUNCH("verify_drafts");
  qe_launch_cluster(verify_draw_kernel, dim3((unsigned)R * draw), dim3(VF_THREADS), 0, stream, draw, logits, draft_logits,
                    draft_tokens, starts, temperature, uniform, (const VfPart*)parts, thresholds, tokens, counts, (int)ctas, N, R, V);
  QE_CHECK_LAUNCH("verify_drafts");
  return 0;
}

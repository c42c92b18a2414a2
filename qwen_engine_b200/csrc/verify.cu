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
// Two kernels.  The first reads every logit once: a row is shared by a cluster of VF_CTAS CTAs, and each leaves its chunk's
// maximum and sum of exponentials; rows with a top-k first find the top_k-th largest logit together (by the digits of an
// order-preserving integer, the histograms meeting in distributed shared memory).  The second has a cluster for every
// request: it puts the chunks' sums together, holds the drafts against them, and draws.
//
// Precision.  Whether a draft stands is one comparison of float32 exponentials with float64 sums: it goes the other way
// than exact arithmetic for about one u in 10^7.  Drawing is another matter: a running sum over V terms has V borders, and an
// error of 10^-8 in the sums moves a border across u for one draw in a thousand.  So the second kernel forms exponentials
// and sums in float64, for the one or two rows of a request that it draws from.
#include "common.cuh"
#include <math.h>
#include <float.h>

#define VF_CTAS 8          // CTAs of a cluster: chunks of a row
#define VF_THREADS 512
#define VF_WARPS (VF_THREADS / 32)

struct __align__(16) VfPart { double z; float m; int arg; };     // of a chunk: sum of exp((x - m) / T), maximum, its lowest place

// order-preserving map float -> uint32 (larger float, larger key; NaN lowest, -0 as +0)
__device__ __forceinline__ unsigned vf_key(float f) {
  f = fmaxf(f, -INFINITY) + 0.f;
  const unsigned u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A row as groups of four logits that lie on 16-byte boundaries: group g holds the elements 4 g - lead ..; the elements of a
// group that are not the row's read as -inf.  NaN reads as -inf.
struct VfRow {
  const float* p;
  int lead, V, groups;
  __device__ __forceinline__ VfRow(const float* row, int V_) : p(row), V(V_) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    groups = (lead + V_ + 3) >> 2;
  }
  __device__ __forceinline__ float4 get(int g) const {
    const int e = 4 * g - lead;
    float4 v;
    if (e >= 0 && e + 4 <= V) {
      v = __ldg(reinterpret_cast<const float4*>(p + e));
    } else {
      v.x = e >= 0 && e < V ? __ldg(p + e) : -INFINITY;
      v.y = e + 1 >= 0 && e + 1 < V ? __ldg(p + e + 1) : -INFINITY;
      v.z = e + 2 >= 0 && e + 2 < V ? __ldg(p + e + 2) : -INFINITY;
      v.w = e + 3 >= 0 && e + 3 < V ? __ldg(p + e + 3) : -INFINITY;
    }
    v.x = fmaxf(v.x, -INFINITY); v.y = fmaxf(v.y, -INFINITY);
    v.z = fmaxf(v.z, -INFINITY); v.w = fmaxf(v.w, -INFINITY);
    return v;
  }
};

// the request that row n (of the target's rows, or of the drafts) belongs to: the last r with starts[r] - r * less <= n
__device__ __forceinline__ int vf_owner(const int* starts, int R, int n, int less) {
  int lo = 0, hi = R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] - mid * less <= n) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(VF_THREADS)
verify_sums_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ starts,
                   const float* __restrict__ temperature, const int* __restrict__ top_k, VfPart* __restrict__ parts,
                   unsigned* __restrict__ thresholds, int N, int R, int V) {
  __shared__ unsigned hist[256];
  __shared__ unsigned digit_s, above_s;
  __shared__ unsigned warp_tot[8];
  __shared__ double sz[VF_WARPS];
  __shared__ float sm[VF_WARPS];
  __shared__ int si[VF_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int rank = (int)cluster_cta_rank(), y = blockIdx.y;
  const bool draft = y >= N;
  const int r = vf_owner(starts, R, draft ? y - N : y, draft ? 1 : 0);
  const float T = temperature[r];
  const bool greedy = !(T > 0.f);
  if (draft && greedy) return;                  // (the whole cluster: the row is not looked at)
  const VfRow row(draft ? draft_logits + (size_t)(y - N) * V : logits + (size_t)y * V, V);
  const int per = (row.groups + VF_CTAS - 1) / VF_CTAS;
  const int g0 = min(row.groups, rank * per), g1 = min(row.groups, g0 + per);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  unsigned thr = 0u;
  const int k = top_k[r];
  if (!greedy && k > 0 && k < V) {
    unsigned left = (unsigned)k;                // the threshold is the left-th largest among the keys with the digits found so far
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
      unsigned c = 0u;
      if (tid < 256) {
        for (int o = 0; o < VF_CTAS; ++o) c += (unsigned)__float_as_int(cluster_ld_f32(cluster_map_shared(&hist[255 - tid], o)));
      }
      unsigned run = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      if (tid < 256 && lane == 31) warp_tot[warp] = run;
      __syncthreads();
      if (tid < 256) {
        for (int w = 0; w < warp; ++w) run += warp_tot[w];
        if (run >= left && run - c < left) { digit_s = 255u - tid; above_s = run - c; }
      }
      __syncthreads();
      thr |= digit_s << shift;
      left -= above_s;
      cluster_sync_all();                       // the others' histograms have been read
    }
    if (rank == 0 && tid == 0) thresholds[y] = thr;
  } else if (rank == 0 && tid == 0) {
    thresholds[y] = 0u;
  }

  // the chunk's maximum and sum: every thread keeps its own running maximum
  float m = -FLT_MAX, bv = -INFINITY;
  double z = 0.0;
  int bi = 0x7fffffff;
  const float c = fminf(1.4426950408889634f / T, FLT_MAX);
  for (int g = g0 + tid; g < g1; g += VF_THREADS) {
    const float4 v = row.get(g);
    const float x[4] = {v.x, v.y, v.z, v.w};
    const int e = 4 * g - row.lead;
    if (greedy) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > bv) { bv = x[j]; bi = e + j; }         // (a thread's elements come in rising order)
      continue;
    }
    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if (top > m) {
      z *= (double)exp2f((m - top) * c);
      m = top;
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (thr == 0u || vf_key(x[j]) >= thr) s += x[j] == m ? 1.f : exp2f((x[j] - m) * c);
    z += (double)s;
  }
  if (greedy) m = bv;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const double oz = __shfl_xor_sync(0xffffffffu, z, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    const float nm = fmaxf(m, om);
    if (!greedy) z = z * (m == nm ? 1.0 : (double)exp2f((m - nm) * c)) + oz * (om == nm ? 1.0 : (double)exp2f((om - nm) * c));
    if (om > m || (om == m && oi < bi)) bi = oi;
    m = nm;
  }
  if (lane == 0) { sz[warp] = z; sm[warp] = m; si[warp] = bi; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < VF_WARPS; ++w) {
      const float nm = fmaxf(m, sm[w]);
      if (!greedy) z = z * (m == nm ? 1.0 : (double)exp2f((m - nm) * c)) + sz[w] * (sm[w] == nm ? 1.0 : (double)exp2f((sm[w] - nm) * c));
      if (sm[w] > m || (sm[w] == m && si[w] < bi)) bi = si[w];
      m = nm;
    }
    parts[(size_t)y * VF_CTAS + rank] = VfPart{z, m, bi};
  }
}

// ---- the drafts against the sums, and the token behind them ------------------------------------------------------------------

struct VfStat { float m; double z; };
__device__ __forceinline__ VfStat vf_stat(const VfPart* parts, size_t y, float c) {
  VfStat s{-FLT_MAX, 0.0};
  for (int o = 0; o < VF_CTAS; ++o) s.m = fmaxf(s.m, __ldg(&parts[y * VF_CTAS + o].m));
  for (int o = 0; o < VF_CTAS; ++o) {
    const float m = __ldg(&parts[y * VF_CTAS + o].m);
    s.z += __ldg(&parts[y * VF_CTAS + o].z) * (m == s.m ? 1.0 : (double)exp2f((m - s.m) * c));
  }
  return s;
}
__device__ __forceinline__ int vf_argmax(const VfPart* parts, size_t y) {
  float m = -INFINITY;
  int at = 0x7fffffff;
  for (int o = 0; o < VF_CTAS; ++o) {
    const VfPart p = parts[y * VF_CTAS + o];
    if (p.m > m) { m = p.m; at = p.arg; }
  }
  return at == 0x7fffffff ? 0 : at;
}
__device__ __forceinline__ double vf_exp(float x, float m, double inv_t) { return x == m ? 1.0 : exp(((double)x - (double)m) * inv_t); }

__device__ __forceinline__ double vf_block_sum(double v, double* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < VF_WARPS; ++w) t += s[w];
  return t;
}
__device__ __forceinline__ double vf_ld_remote(const double* local, int cta) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(v) : "r"(cluster_map_shared(local, cta)) : "memory");
  return v;
}

__global__ void __launch_bounds__(VF_THREADS)
verify_draw_kernel(const float* __restrict__ logits, const float* __restrict__ draft_logits, const int* __restrict__ draft_tokens,
                   const int* __restrict__ starts, const float* __restrict__ temperature, const float* __restrict__ uniform,
                   const VfPart* __restrict__ parts, const unsigned* __restrict__ thresholds, int* __restrict__ tokens,
                   int* __restrict__ counts, int N, int R, int V) {
  __shared__ double s_sum[VF_WARPS];
  __shared__ double x_a, x_b;
  __shared__ int first_s;
  pdl_launch_dependents();
  pdl_wait();
  const int rank = (int)cluster_cta_rank(), r = blockIdx.y;
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
  const float c = fminf(1.4426950408889634f / T, FLT_MAX);
  if (tid == 0) first_s = n;
  __syncthreads();
  for (int i = tid; i < n; i += VF_THREADS) {
    const int d = draft_tokens[d0 + i];
    bool stands = false;
    if (d >= 0 && d < V) {
      if (greedy) {
        stands = vf_argmax(parts, lo + i) == d;
      } else {
        const VfStat sp = vf_stat(parts, lo + i, c);
        const float x = logits[(size_t)(lo + i) * V + d];
        const double p = vf_key(x) >= thresholds[lo + i] ? (x == sp.m ? 1.0 : (double)exp2f((x - sp.m) * c)) : 0.0;
        double q = 1.0, zq = 1.0;
        if (draft_logits) {
          const VfStat sq = vf_stat(parts, N + d0 + i, c);
          const float xd = draft_logits[(size_t)(d0 + i) * V + d];
          q = vf_key(xd) >= thresholds[N + d0 + i] ? (xd == sq.m ? 1.0 : (double)exp2f((xd - sq.m) * c)) : 0.0;
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
    if (rank == 0 && tid == 0) tokens[lo + a] = vf_argmax(parts, lo + a);
    return;
  }
  const VfRow P(logits + (size_t)(lo + a) * V, V);
  const unsigned thr_p = thresholds[lo + a];
  const float mp = vf_stat(parts, lo + a, c).m;
  const double inv_t = 1.0 / (double)T;
  const bool fell = a < n;
  const float* q_row = fell && draft_logits ? draft_logits + (size_t)(d0 + a) * V : nullptr;
  const unsigned thr_q = q_row ? thresholds[N + d0 + a] : 0u;
  const float mq = q_row ? vf_stat(parts, N + d0 + a, c).m : 0.f;
  const int gone = fell && !q_row ? draft_tokens[d0 + a] : -1;
  const int per = (P.groups + VF_CTAS - 1) / VF_CTAS;
  const int g0 = min(P.groups, rank * per), g1 = min(P.groups, g0 + per);
  const int wper = (per + VF_WARPS - 1) / VF_WARPS;
  const int w0 = min(g1, g0 + warp * wper), w1 = min(g1, w0 + wper);      // the warp's groups: ranges in the order of the row
  auto q_get = [&](int e) {
    return e >= 0 && e < V ? fmaxf(__ldg(q_row + e), -INFINITY) : -INFINITY;
  };
  double rho = 0.0;                             // Z_p / Z_q
  if (q_row) {
    double zp = 0.0, zq = 0.0;
    for (int g = w0 + lane; g < w1; g += 32) {
      const float4 v = P.get(g);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float xq = q_get(4 * g - P.lead + j);
        if (vf_key(x[j]) >= thr_p) zp += vf_exp(x[j], mp, inv_t);
        if (vf_key(xq) >= thr_q) zq += vf_exp(xq, mq, inv_t);
      }
    }
    zp = vf_block_sum(zp, s_sum);
    zq = vf_block_sum(zq, s_sum);
    if (tid == 0) { x_a = zp; x_b = zq; }
    cluster_sync_all();
    zp = zq = 0.0;
    for (int o = 0; o < VF_CTAS; ++o) { zp += vf_ld_remote(&x_a, o); zq += vf_ld_remote(&x_b, o); }
    cluster_sync_all();
    rho = zp / zq;
  }
  // weights: e_p - rho e_q where positive; e_p but for the draft that fell; e_p
  bool plain = false;
  auto weights = [&](int g, double (&w)[4]) {
    const float4 v = P.get(g);
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 4 * g - P.lead + j;
      w[j] = vf_key(x[j]) >= thr_p ? vf_exp(x[j], mp, inv_t) : 0.0;
      if (plain) continue;
      if (q_row) {
        const float xq = q_get(e);
        if (vf_key(xq) >= thr_q) w[j] = fmax(w[j] - rho * vf_exp(xq, mq, inv_t), 0.0);
      } else if (e == gone) {
        w[j] = 0.0;
      }
    }
  };
  double total = 0.0, before = 0.0, mine = 0.0;
  for (int pass = 0; pass < 2; ++pass) {        // a second time where nothing is left of p - q: then from p
    double s = 0.0;
    for (int g = w0 + lane; g < w1; g += 32) {
      double w[4];
      weights(g, w);
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
    mine = vf_block_sum(s, s_sum);
    if (tid == 0) x_a = mine;
    cluster_sync_all();
    total = before = 0.0;
    for (int o = 0; o < VF_CTAS; ++o) {
      const double t = vf_ld_remote(&x_a, o);
      if (o < rank) before += t;
      total += t;
    }
    cluster_sync_all();
    if (total > 0.0 || plain) break;
    plain = true;
  }
  const double target = (double)fminf(fmaxf(uniform[hi - 1], 0.f), 0.99999994f) * total;
  // the CTA, and in it the warp, whose range holds the first running sum above the target (the last CTA that has any weight, should rounding leave none)
  double after_all = before + mine;
  if (!(total > 0.0)) {
    if (rank == 0 && tid == 0) tokens[lo + a] = 0;          // no logit is finite
    return;
  }
  if (!(before <= target && target < after_all)) return;
  double run = before;
  int w = 0;
  for (; w < VF_WARPS; ++w) {
    if (run + s_sum[w] > target) break;
    run += s_sum[w];
  }
  if (w == VF_WARPS) {                          // (rounding: the last warp that has any weight)
    for (w = VF_WARPS - 1; w > 0 && !(s_sum[w] > 0.0); --w) {}
    run -= s_sum[w];
  }
  if (warp != w) return;
  int last = -1;                                // the last place with any weight: the answer, should rounding leave no other
  for (int gb = w0; gb < w1; gb += 32) {
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    const int g = gb + lane;
    if (g < w1) weights(g, v);
    const double s = (v[0] + v[1]) + (v[2] + v[3]);
    double inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const unsigned some = __ballot_sync(0xffffffffu, s > 0.0);
    const unsigned over = __ballot_sync(0xffffffffu, s > 0.0 && run + inc > target);
    const int who = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : -1);
    if (who >= 0) {
      int at = -1;
      if (lane == who) {
        double b = run + (inc - s);
        for (int j = 0; j < 4; ++j) {
          if (v[j] > 0.0) at = 4 * g - P.lead + j;
          b += v[j];
          if (over && v[j] > 0.0 && b > target) break;
        }
      }
      last = __shfl_sync(0xffffffffu, at, who);
    }
    if (over) break;
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0 && last >= 0) tokens[lo + a] = last;
}

extern "C" int qe_verify_drafts(const float* logits, const int* draft_tokens, const float* draft_logits, const int* starts,
                                const float* temperature, const int* top_k, const float* uniform, int* tokens, int* counts,
                                void* parts, unsigned* thresholds, int N, int R, int V, cudaStream_t stream) {
  if (R <= 0 || N <= 0) return 0;
  if (V <= 0) QE_REFUSE("verify_drafts: empty vocabulary");
  if (N < R) QE_REFUSE("verify_drafts: %d rows for %d requests", N, R);
  const long rows = (long)N + (draft_logits ? N - R : 0);
  if (rows > 65535 || R > 65535) QE_REFUSE("verify_drafts: %ld rows are more than a launch takes (65535)", rows);
  qe_launch_cluster(verify_sums_kernel, dim3(VF_CTAS, (unsigned)rows), dim3(VF_THREADS), 0, stream, VF_CTAS, logits, draft_logits,
                    starts, temperature, top_k, (VfPart*)parts, thresholds, N, R, V);
  QE_CHECK_LAUNCH("verify_drafts");
  qe_launch_cluster(verify_draw_kernel, dim3(VF_CTAS, (unsigned)R), dim3(VF_THREADS), 0, stream, VF_CTAS, logits, draft_logits,
                    draft_tokens, starts, temperature, uniform, (const VfPart*)parts, thresholds, tokens, counts, N, R, V);
  QE_CHECK_LAUNCH("verify_drafts");
  return 0;
}

// Gathered attention weights of a few rows (decoded tokens, a verification step's drafts) in bfloat16: at most 32 rows of a
// request meet each kv head (query tokens x the query heads of its group).  What it computes: attention_weights.cu.
//
// The keys are the work: a key's row is 2 D bytes, and all it takes part in are 2 D products per row.  So every key is read
// once, straight from its page into the registers of the warp that multiplies it (32 keys of 64 channels while the ones before are multiplied,
// no shared memory between), and the scores are kept until the rows' sums are known: 4 bytes a row and key.
//
// A warp multiplies 32 keys at a time with mma.sync m16n8k16, queries as A, keys as B.  A sum over channels does not care for
// their order, so a lane's share of B is what it can load in one piece: for the l-th 32 channels lane 4 n + x loads channels 8 x
// .. 8 x + 7 of key n, the B fragments of two products, and the queries' fragments are laid out in shared memory to match.
// Nor does the order of the keys matter: column n of product t is key 8 (n / 2) + 2 t + n % 2, which leaves every lane eight
// consecutive keys of a row.
//
// Two forms.  Where a request's scores fit the shared memory of a cluster (parts of its keys, a CTA each), the CTAs keep them
// there, exchange their rows' maxima and sums through distributed shared memory, and finish their keys: one launch, nothing
// but keys and weights through memory.  Else the scores go to scratch memory and a second kernel adds them up.  Scratch memory goes by the widths of slots
// and tables (a captured call is replayed with other lengths) as long as that is little; beyond, the requests' scores lie one behind the other, and what
// finds no room is formed twice (32 x 5 rows, 8 000 to 1 800 keys held in 131 072 places, 242 us with 0.27 GB of scratch memory for 205 with 2.7).
//
// What bounds them: the keys, from memory (4 requests of 131 071 keys, 32 / 8 heads of 128: 1.07 GB in 205 us, 5.2 TB/s, and 23 us for the second kernel);
// with more rows a key the scores' way through L2 and their instructions (32 x 5 rows behind up to 8 200 keys 77 us); with few keys the launch
// (1 request of 1 024 keys, 16 / 8 heads: 6.4 us in a cluster).
#include "attention_weights.cuh"

#define AF_THREADS 256
#define AF_WARPS (AF_THREADS / 32)
#define AF_GROUP 32              // keys of a warp at a time
#define AF_MAX_CTAS 8            // CTAs of a cluster

__device__ __forceinline__ void af_mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// 16 bytes of a key: read once, so not kept in L1, and the first to leave L2 (where the scores stay)
__device__ __forceinline__ uint64_t af_first_out() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint4 af_ld_key(const void* p, uint64_t policy) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy));
  return v;
}

// The scores of the CTA's keys [key0, key1) (key0 a multiple of 32) against the request's rows, in units of log2(e), -inf where
// a row may not see a key: S[row * ld + key - key0] (null: nowhere); and the rows' maxima and sums over those keys into row_max / row_sum (of all MT x 16 rows).
// MT: tiles of 16 rows; PLAIN: scores are neither bent nor biased.  A warp goes through its keys 64 channels at a time, the next 64 (of the same
// 32 keys or of its next ones) on their way while these are multiplied.
template <int MT, bool PLAIN>
__device__ __forceinline__ void af_scores(const AwArgs& A, const AwReq& R, int r, int c, int key0, int key1, float* S, size_t ld,
                                          uint4* frags, float (*warp_ml)[MT * 16][2], float* row_max, float* row_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = lane >> 2, x = lane & 3;
  const int G = A.Hq / A.Hkv, rows = R.counted * G;
  const int chunks = (A.D + 63) / 64, steps = chunks * 4;
  const uint64_t policy = af_first_out();
  const bool one_page = A.page % 8 == 0;          // a lane's eight keys lie in one page
  const size_t page_elems = (size_t)A.planes * A.Hkv * A.page * A.D;
  // the four keys whose channels this lane loads, of the 32 from j on: 8 (n / 2) + n % 2 + 0, 2, 4, 6; null where there is none
  auto keys = [&](int j, const __nv_bfloat16* (&kp)[4]) {
    const int mine = j + 8 * (n >> 1) + (n & 1);
    const __nv_bfloat16* base = reinterpret_cast<const __nv_bfloat16*>(A.pages) + 8 * x;
    if (one_page) {
      const int page = mine < key1 ? aw_page(A, r, mine) : -1;
      const __nv_bfloat16* p = base + (size_t)max(page, 0) * page_elems + ((size_t)c * A.page + (mine - aw_block(A, mine) * A.page)) * A.D;
#pragma unroll
      for (int t = 0; t < 4; ++t) kp[t] = page >= 0 && mine + 2 * t < key1 ? p + 2 * t * A.D : nullptr;
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int key = mine + 2 * t, page = key < key1 ? aw_page(A, r, key) : -1;
        kp[t] = page >= 0 ? base + (size_t)page * page_elems + ((size_t)c * A.page + (key - aw_block(A, key) * A.page)) * A.D : nullptr;
      }
    }
  };
  auto fetch = [&](const __nv_bfloat16* const (&kp)[4], int ch, uint4 (&k)[4][2]) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        const int d = 64 * ch + 32 * l;
        k[t][l] = kp[t] != nullptr && d + 8 * x < A.D ? af_ld_key(kp[t] + d, policy) : make_uint4(0u, 0u, 0u, 0u);
      }
  };
  const int step = AF_WARPS * AF_GROUP;
  int j0 = key0 + warp * AF_GROUP;
  const __nv_bfloat16 *kp[4], *kn[4];
  uint4 cur[4][2], nxt[4][2];
  if (j0 < key1) {
    keys(j0, kp);
    fetch(kp, 0, cur);
  }
  // the queries as A fragments, in the order of the lanes' channels; rows and channels that do not exist are zero
  for (int i = tid; i < MT * steps * 32; i += AF_THREADS) {
    const int l = i & 31, st = (i >> 5) % steps, mt = i / (32 * steps);
    const int d = 32 * (st >> 1) + 8 * (l & 3) + 4 * (st & 1);
    uint32_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int rho = mt * 16 + (l >> 2) + 8 * (k & 1), ch = d + 2 * (k >> 1);
      uint32_t w = 0u;
      if (rho < rows && ch < A.D) {
        const int t = rho / G;
        const unsigned short* q = reinterpret_cast<const unsigned short*>(A.q) + (size_t)(R.row0 + t) * A.q_stride + (size_t)(c * G + rho - t * G) * A.D + ch;
        w = (uint32_t)q[0] | ((uint32_t)q[1] << 16);
      }
      v[k] = w;
    }
    frags[i] = make_uint4(v[0], v[1], v[2], v[3]);
  }
  __syncthreads();
  float m[MT][2], z[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) { m[mt][h] = -INFINITY; z[mt][h] = 0.f; }
  const float sc = A.scale * AW_LOG2E;
  const int last_pos = R.ctx + max(R.counted, 1) - 1;
  for (; j0 < key1; j0 += step) {
    float s[MT][4][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < 4; ++t) s[mt][t][0] = s[mt][t][1] = s[mt][t][2] = s[mt][t][3] = 0.f;
    const bool more = j0 + step < key1;
    // which of the warp's 32 keys lie in a page
    unsigned b[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) b[t] = __ballot_sync(0xffffffffu, kp[t] != nullptr);
    if (more) keys(j0 + step, kn);
    for (int ch = 0; ch < chunks; ++ch) {
      if (ch + 1 < chunks) fetch(kp, ch + 1, nxt);
      else if (more) fetch(kn, 0, nxt);
#pragma unroll
      for (int l = 0; l < 2; ++l)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint4* f = frags + ((size_t)mt * steps + 4 * ch + 2 * l) * 32 + lane;
          const uint4 a0 = f[0], a1 = f[32];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            af_mma(s[mt][t], a0, cur[t][l].x, cur[t][l].y);
            af_mma(s[mt][t], a1, cur[t][l].z, cur[t][l].w);
          }
        }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int l = 0; l < 2; ++l) cur[t][l] = nxt[t][l];
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) kp[t] = kn[t];
    // every row sees all 32 keys
    const bool all = j0 + AF_GROUP <= R.ctx + 1 && (A.window <= 0 || j0 > last_pos - A.window) && (b[0] & b[1] & b[2] & b[3]) == 0xffffffffu;
    unsigned held = 0u;                             // of the lane's eight keys of a row, j0 + 8 x ..
    if (!all) {
#pragma unroll
      for (int e = 0; e < 8; ++e) held |= ((b[e >> 1] >> (4 * (2 * x + (e & 1)))) & 1u) << e;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (mt * 16 + 8 * h >= rows) continue;      // (the warp's)
        const int rho = mt * 16 + 8 * h + n;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s[mt][e >> 1][2 * h + (e & 1)];
        if (PLAIN) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= sc;
        } else {
          const int p = R.ctx + rho / G;
          const float slope = A.slopes ? A.slopes[c * G + rho % G] : 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = aw_score(A, v[e], slope, p - (j0 + 8 * x + e));
        }
        if (!all) {
          const int p = rho < rows ? R.ctx + rho / G : -1;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = j0 + 8 * x + e;
            if (!(((held >> e) & 1u) && key <= p && (A.window <= 0 || key > p - A.window))) v[e] = -INFINITY;
          }
        }
        if (rho < rows && S != nullptr) {
          float4* dst = reinterpret_cast<float4*>(S + rho * ld + (j0 - key0) + 8 * x);
          dst[0] = make_float4(v[0], v[1], v[2], v[3]);
          dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
        const float mx = fmaxf(fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]))), m[mt][h]);
        const float nb = mx == -INFINITY ? 0.f : -mx;
        float sum = z[mt][h] * aw_ex2(m[mt][h] + nb);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += aw_ex2(v[e] + nb);
        z[mt][h] = sum;
        m[mt][h] = mx;
      }
  }
  // the four lanes of a row, then the warps
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m[mt][h], o), oz = __shfl_xor_sync(0xffffffffu, z[mt][h], o);
        const float nm = fmaxf(m[mt][h], om), base = aw_base(nm);
        z[mt][h] = z[mt][h] * aw_ex2(m[mt][h] - base) + oz * aw_ex2(om - base);
        m[mt][h] = nm;
      }
      if (x == 0) { warp_ml[warp][mt * 16 + 8 * h + n][0] = m[mt][h]; warp_ml[warp][mt * 16 + 8 * h + n][1] = z[mt][h]; }
    }
  __syncthreads();
  if (tid < MT * 16) {
    float mm = -INFINITY, zz = 0.f;
#pragma unroll
    for (int w = 0; w < AF_WARPS; ++w) mm = fmaxf(mm, warp_ml[w][tid][0]);
    const float base = aw_base(mm);
#pragma unroll
    for (int w = 0; w < AF_WARPS; ++w) zz += warp_ml[w][tid][1] * aw_ex2(warp_ml[w][tid][0] - base);
    row_max[tid] = mm;
    row_sum[tid] = zz;
  }
  __syncthreads();
}

// the keys that any row sees begin here (a multiple of 32)
__device__ __forceinline__ int af_first(const AwArgs& A, const AwReq& R) {
  return A.window > 0 ? max(0, R.ctx - A.window + 1) / AF_GROUP * AF_GROUP : 0;
}
__device__ __forceinline__ bool af_mine(const AwArgs& A, const AwReq& R, int max_rows) {     // (requests with more rows are another kernel's)
  return (long)R.n * (A.Hq / A.Hkv) <= max_rows;
}

// ---- a request's scores in the shared memory of a cluster ----------------------------------------------------------------------

template <int MT, bool PLAIN>
__global__ void __launch_bounds__(AF_THREADS, 2)
attention_weights_cluster_kernel(AwArgs A, int max_rows, int part_keys) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ float warp_ml[AF_WARPS][MT * 16][2];
  __shared__ float row_max[MT * 16], row_sum[MT * 16];
  __shared__ float2 row[MT * 16];
  pdl_launch_dependents();
  pdl_wait();
  const int C = (int)cluster_num_ctas(), rank = (int)cluster_cta_rank(), c = blockIdx.y, r = blockIdx.z, tid = threadIdx.x;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  if (!af_mine(A, R, max_rows) || slot < 0 || slot >= A.slots || R.total == 0) return;      // (the whole cluster)
  const int G = A.Hq / A.Hkv, rows = R.counted * G;
  const int first = af_first(A, R);
  const int per = ((R.total - first + C - 1) / C + AF_GROUP - 1) / AF_GROUP * AF_GROUP;
  const int key0 = min(first + rank * per, R.total), key1 = min(key0 + per, R.total);
  const int steps = (A.D + 63) / 64 * 4;
  uint4* frags = reinterpret_cast<uint4*>(raw);
  float* S = reinterpret_cast<float*>(frags + MT * steps * 32);
  const size_t ld = part_keys + 4;                // (off 32 banks, so that the rows' stores do not meet)
  af_scores<MT, PLAIN>(A, R, r, c, key0, key1, S, ld, frags, warp_ml, row_max, row_sum);
  cluster_sync_all();
  if (tid < MT * 16) {
    float m = -INFINITY, z = 0.f;
    for (int o = 0; o < C; ++o) m = fmaxf(m, cluster_ld_f32(cluster_map_shared(&row_max[tid], o)));
    float2 v = make_float2(0.f, 0.f);
    if (tid < rows) {
      const float base = aw_base(m);
      for (int o = 0; o < C; ++o) {
        const float om = cluster_ld_f32(cluster_map_shared(&row_max[tid], o));
        z += cluster_ld_f32(cluster_map_shared(&row_sum[tid], o)) * exp2f(om - base);
      }
      if (A.sinks) z += exp2f(A.sinks[c * G + tid % G] * AW_LOG2E - base);
      v = m == -INFINITY ? make_float2(0.f, z == z ? 0.f : z) : make_float2(m, 1.f / z);
    }
    row[tid] = v;
  }
  cluster_sync_all();                             // (the others' statistics have been read)
  const size_t base = ((size_t)slot * A.Hkv + c) * A.capacity;
  auto finish = [&](int key, float t) {
    A.out[base + key] = key < R.ctx ? A.weights[base + key] + t : t;
    if (A.positions && key >= R.ctx) A.positions[base + key] = A.step_positions[R.row0 + key - R.ctx];
  };
  if (key1 - key0 <= AF_THREADS) {                // a key a thread
    const int key = key0 + tid;
    if (key < key1) {
      float t = 0.f;
#pragma unroll 4
      for (int rho = 0; rho < rows; ++rho) t = fmaf(aw_ex2(S[rho * ld + tid] - row[rho].x), row[rho].y, t);
      finish(key, t);
    }
  } else {                                        // four
    for (int key = key0 + 4 * tid; key < key1; key += 4 * AF_THREADS) {
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int rho = 0; rho < rows; ++rho) {
        const float4 s = *reinterpret_cast<const float4*>(S + rho * ld + (key - key0));
        const float2 mz = row[rho];
        t[0] = fmaf(aw_ex2(s.x - mz.x), mz.y, t[0]); t[1] = fmaf(aw_ex2(s.y - mz.x), mz.y, t[1]);
        t[2] = fmaf(aw_ex2(s.z - mz.x), mz.y, t[2]); t[3] = fmaf(aw_ex2(s.w - mz.x), mz.y, t[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key + e < key1) finish(key + e, t[e]);
    }
  }
  if (A.out != A.weights)                         // keys that lie before every row's window
    for (int key = rank * AF_THREADS + tid; key < first; key += C * AF_THREADS) A.out[base + key] = A.weights[base + key];
}

// ---- the scores through scratch memory -------------------------------------------------------------------------------------------

// Where a request's scores lie: element (head, row, key - af_first) at base + (head * rows + row) * ld + key - af_first, base < 0 where they are not kept.
struct AfPlace { long base, ld; int rows; };

// ld > 0: [request, kv head, max_rows, ld].  ld == 0: the requests' scores one behind the other, as many floats as each has, as far as `room` reaches: memory by
// what is held and not by the widths of slots and tables; a request that finds no room is formed again by attention_weights_again_kernel.
__device__ __forceinline__ AfPlace af_place(const AwArgs& A, const AwReq& R, int r, int max_rows, long ld, long room, long* sums) {
  if (ld > 0) return AfPlace{(long)r * A.Hkv * max_rows * ld, ld, max_rows};
  const int G = A.Hq / A.Hkv, tid = threadIdx.x;
  auto width = [&](const AwReq& Q) { return (long)((Q.total - af_first(A, Q) + AF_GROUP - 1) / AF_GROUP * AF_GROUP); };
  long before = 0;
  for (int i = tid; i < r; i += AF_THREADS) {
    const AwReq Q = aw_req(A, i);
    if (af_mine(A, Q, max_rows)) before += width(Q) * (Q.counted * G);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((tid & 31) == 0) sums[tid >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < AF_WARPS; ++w) before += sums[w];
  before *= A.Hkv;
  const long own = width(R) * (R.counted * G);
  return AfPlace{before + own * A.Hkv <= room ? before : -1, width(R), R.counted * G};
}

// stats: [request, kv head, max_rows, parts, 2]
__device__ __forceinline__ float* af_stats(const AwArgs& A, int r, int c, int max_rows, int row) {
  return A.stats + (((size_t)r * A.Hkv + c) * max_rows + row) * A.parts * 2;
}

// the keys of a part: at least least_keys, a multiple of 32, so that a short request has fewer parts
__device__ __forceinline__ int2 af_part(const AwArgs& A, const AwReq& R, int part, int least_keys) {
  const int first = af_first(A, R);
  const int per = (max((R.total - first + A.parts - 1) / A.parts, least_keys) + AF_GROUP - 1) / AF_GROUP * AF_GROUP;
  const int key0 = min(first + part * per, R.total);
  return make_int2(key0, min(key0 + per, R.total));
}

template <int MT, bool PLAIN>
__global__ void __launch_bounds__(AF_THREADS, 2)
attention_weights_scores_kernel(AwArgs A, int max_rows, int least_keys, float* scores, long ld, long room) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ float warp_ml[AF_WARPS][MT * 16][2];
  __shared__ float row_max[MT * 16], row_sum[MT * 16];
  __shared__ long sums[AF_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int part = blockIdx.x, c = blockIdx.y, r = blockIdx.z, tid = threadIdx.x;
  const AwReq R = aw_req(A, r);
  if (!af_mine(A, R, max_rows)) return;
  const int G = A.Hq / A.Hkv, rows = R.counted * G;
  const int2 keys = af_part(A, R, part, least_keys);
  const int key0 = keys.x, key1 = keys.y;
  float* st = af_stats(A, r, c, max_rows, min(tid, max_rows - 1)) + part * 2;      // of row tid
  if (key0 == key1) {
    if (tid < rows) { st[0] = -INFINITY; st[1] = 0.f; }
    return;
  }
  const AfPlace place = af_place(A, R, r, max_rows, ld, room, sums);
  float* S = place.base < 0 ? nullptr : scores + place.base + (long)c * place.rows * place.ld + (key0 - af_first(A, R));
  af_scores<MT, PLAIN>(A, R, r, c, key0, key1, S, place.ld, reinterpret_cast<uint4*>(raw), warp_ml, row_max, row_sum);
  if (tid < rows) {
    st[0] = row_max[tid];
    st[1] = row_sum[tid];
  }
}

__global__ void __launch_bounds__(AF_THREADS)
attention_weights_sum_kernel(AwArgs A, int max_rows, const float* __restrict__ scores, long ld, long room) {
  __shared__ float2 row[32];
  __shared__ long sums[AF_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.y, r = blockIdx.z, tid = threadIdx.x;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  if (!af_mine(A, R, max_rows) || slot < 0 || slot >= A.slots || (int)blockIdx.x * AF_THREADS * 4 >= R.total) return;
  const int G = A.Hq / A.Hkv, rows = R.counted * G, first = af_first(A, R);
  if (tid < rows) row[tid] = aw_merge(af_stats(A, r, c, max_rows, tid), A.parts, A.sinks ? A.sinks + c * G + tid % G : nullptr);
  const AfPlace place = af_place(A, R, r, max_rows, ld, room, sums);
  __syncthreads();
  const int k0 = (blockIdx.x * AF_THREADS + tid) * 4;
  if (k0 >= R.total || (place.base < 0 && k0 >= first)) return;
  const float* S = scores + place.base + (long)c * place.rows * place.ld + (k0 - first);
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  if (k0 >= first) {                              // (first is a multiple of 32, rows of the scratch memory are whole runs of 32 keys)
#pragma unroll 4
    for (int rho = 0; rho < rows; ++rho) {
      const float4 s = __ldcs(reinterpret_cast<const float4*>(S + rho * place.ld));
      const float2 mz = row[rho];
      t[0] = fmaf(aw_ex2(s.x - mz.x), mz.y, t[0]); t[1] = fmaf(aw_ex2(s.y - mz.x), mz.y, t[1]);
      t[2] = fmaf(aw_ex2(s.z - mz.x), mz.y, t[2]); t[3] = fmaf(aw_ex2(s.w - mz.x), mz.y, t[3]);
    }
  }
  const size_t base = ((size_t)slot * A.Hkv + c) * A.capacity;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int key = k0 + e;
    if (key >= R.total) break;
    A.out[base + key] = key < R.ctx ? A.weights[base + key] + t[e] : t[e];
    if (A.positions && key >= R.ctx) A.positions[base + key] = A.step_positions[R.row0 + key - R.ctx];
  }
}

// The keys of requests whose scores found no room: their scores once more, AF_AGAIN keys of a part at a time into shared memory, and the sums.
#define AF_AGAIN 512
template <int MT, bool PLAIN>
__global__ void __launch_bounds__(AF_THREADS, 2)
attention_weights_again_kernel(AwArgs A, int max_rows, int least_keys, long room) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ float warp_ml[AF_WARPS][MT * 16][2];
  __shared__ float row_max[MT * 16], row_sum[MT * 16];
  __shared__ float2 row[MT * 16];
  __shared__ long sums[AF_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.y, r = blockIdx.z, tid = threadIdx.x;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  if (!af_mine(A, R, max_rows) || slot < 0 || slot >= A.slots) return;
  const int2 keys = af_part(A, R, blockIdx.x, least_keys);
  if (keys.x == keys.y || af_place(A, R, r, max_rows, 0, room, sums).base >= 0) return;      // (the whole CTA)
  const int G = A.Hq / A.Hkv, rows = R.counted * G;
  if (tid < rows) row[tid] = aw_merge(af_stats(A, r, c, max_rows, tid), A.parts, A.sinks ? A.sinks + c * G + tid % G : nullptr);
  uint4* frags = reinterpret_cast<uint4*>(raw);
  float* S = reinterpret_cast<float*>(frags + MT * ((A.D + 63) / 64 * 4) * 32);
  const size_t base = ((size_t)slot * A.Hkv + c) * A.capacity;
  for (int key0 = keys.x; key0 < keys.y; key0 += AF_AGAIN) {
    const int key1 = min(key0 + AF_AGAIN, keys.y);
    af_scores<MT, PLAIN>(A, R, r, c, key0, key1, S, AF_AGAIN + 4, frags, warp_ml, row_max, row_sum);
    for (int key = key0 + tid; key < key1; key += AF_THREADS) {
      float t = 0.f;
#pragma unroll 4
      for (int rho = 0; rho < rows; ++rho) t = fmaf(aw_ex2(S[rho * (AF_AGAIN + 4) + (key - key0)] - row[rho].x), row[rho].y, t);
      A.out[base + key] = key < R.ctx ? A.weights[base + key] + t : t;
      if (A.positions && key >= R.ctx) A.positions[base + key] = A.step_positions[R.row0 + key - R.ctx];
    }
    __syncthreads();                              // S and the queries' fragments are written anew
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------

static size_t af_frag_bytes(int mt, int D) { return (size_t)mt * ((D + 63) / 64) * 4 * 512; }

// Shared memory of a CTA of the cluster form for parts of `part_keys` keys; 0 where the kernels do not take the sizes.
extern "C" long qe_attention_weights_few_smem(int max_rows, int D, int part_keys) {
  if (max_rows < 1 || max_rows > 32 || D < 8 || D % 8 || D > 1024) return 0;
  const int mt = max_rows > 16 ? 2 : 1;
  return (long)af_frag_bytes(mt, D) + (long)max_rows * (part_keys + 4) * 4;
}

template <int MT, bool PLAIN>
static cudaError_t af_launch(const AwArgs& A, int max_rows, int ctas, int part_keys, size_t smem, float* scores, long ld, long room, int max_total, cudaStream_t stream) {
  if (ctas > 0) {
    if (smem > 48 * 1024) {
      static unsigned long long configured = 0;
      const cudaError_t e = qe_once_a_device(configured, [] {
        return cudaFuncSetAttribute(attention_weights_cluster_kernel<MT, PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
      });
      if (e != cudaSuccess) return e;
    }
    return qe_launch_cluster(attention_weights_cluster_kernel<MT, PLAIN>, dim3((unsigned)ctas, (unsigned)A.Hkv, (unsigned)A.R), dim3(AF_THREADS), smem, stream,
                             (unsigned)ctas, A, max_rows, part_keys);
  }
  const size_t frag = af_frag_bytes(MT, A.D);
  if (frag > 48 * 1024) {
    static unsigned long long configured = 0;
    const cudaError_t e = qe_once_a_device(configured, [] {
      return cudaFuncSetAttribute(attention_weights_scores_kernel<MT, PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    });
    if (e != cudaSuccess) return e;
  }
  cudaError_t e = qe_launch(attention_weights_scores_kernel<MT, PLAIN>, dim3((unsigned)A.parts, (unsigned)A.Hkv, (unsigned)A.R), dim3(AF_THREADS), frag, stream,
                            A, max_rows, part_keys, scores, ld, room);
  if (e != cudaSuccess) return e;
  e = qe_launch(attention_weights_sum_kernel, dim3((unsigned)((max_total + AF_THREADS * 4 - 1) / (AF_THREADS * 4)), (unsigned)A.Hkv, (unsigned)A.R),
                dim3(AF_THREADS), 0, stream, A, max_rows, (const float*)scores, ld, room);
  if (e != cudaSuccess || ld > 0) return e;
  const size_t again = frag + (size_t)max_rows * (AF_AGAIN + 4) * 4;
  if (again > 48 * 1024) {
    static unsigned long long configured = 0;
    e = qe_once_a_device(configured, [] {
      return cudaFuncSetAttribute(attention_weights_again_kernel<MT, PLAIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 180 * 1024);
    });
    if (e != cudaSuccess) return e;
  }
  return qe_launch(attention_weights_again_kernel<MT, PLAIN>, dim3((unsigned)A.parts, (unsigned)A.Hkv, (unsigned)A.R), dim3(AF_THREADS), again, stream,
                   A, max_rows, part_keys, room);
}

// The requests of at most `max_rows` rows (a query token x a query head of a kv head's group), 32 at most.  ctas > 0: clusters of so many
// CTAs (1, 2, 4, 8) hold the scores, part_keys keys a CTA at most (a multiple of 32; span <= ctas part_keys); 0: parts of at least part_keys, and `scores`, scratch
// memory of `room` floats, does: [R, Hkv, max_rows, ld] with ld a multiple of 32 and at least span, or, with ld == 0, whatever there is (af_place).
// stats: [R, Hkv, max_rows, parts, 2].  span: the most keys that a request's rows
// see between them, from a multiple of 32 on (max_total without a window).
extern "C" int qe_attention_weights_few(const void* q, long q_stride, int T, const void* pages, int num_pages, int planes,
                                        const int* block_tables, int max_blocks, const int* cu_q, const int* ctx_lens, const int* slot_ids,
                                        const int* counted, const int* step_positions, int* positions, const float* weights, float* out,
                                        int slots, long capacity, int R, int Hq, int Hkv, int D, int page, int window, float scale,
                                        float softcap, const float* slopes, const float* sinks, float* stats, int parts, int max_rows,
                                        int max_total, int span, int ctas, int part_keys, float* scores, long ld, long room, cudaStream_t stream) {
  if (R <= 0 || max_total <= 0) return 0;
  if (Hkv < 1 || Hq % Hkv || page < 1) QE_REFUSE("attention_weights: heads %d/%d, pages of %d", Hq, Hkv, page);
  if (R > 65535 || Hkv > 65535) QE_REFUSE("attention_weights: %d requests, %d kv heads are more than a launch takes", R, Hkv);
  const long smem = qe_attention_weights_few_smem(max_rows, D, part_keys);
  if (smem == 0 || ((uintptr_t)pages & 15)) QE_REFUSE("attention_weights: %d rows of %d channels are not for the kernel of few rows", max_rows, D);
  if (ctas > 0 && (ctas > AF_MAX_CTAS || (ctas & (ctas - 1)) || part_keys % AF_GROUP || (long)ctas * part_keys < span || smem > 220 * 1024))
    QE_REFUSE("attention_weights: %d CTAs of %d keys for %d", ctas, part_keys, span);
  if (ctas == 0 && (scores == nullptr || stats == nullptr || parts < 1 || ld % AF_GROUP || (ld != 0 && (ld < span || room / ld / max_rows / Hkv < R))))
    QE_REFUSE("attention_weights: scratch memory for %d keys is needed", span);
  AwArgs A{q, q_stride, T, pages, num_pages, planes, block_tables, max_blocks, cu_q, ctx_lens, slot_ids, counted, step_positions, positions,
           weights, out, slots, capacity, R, Hq, Hkv, D, page, aw_shift(page), window, scale, softcap, slopes, sinks, stats, parts};
  const bool plain = softcap <= 0.f && slopes == nullptr;
  cudaError_t e;
  if (max_rows > 16) e = plain ? af_launch<2, true>(A, max_rows, ctas, part_keys, smem, scores, ld, room, max_total, stream) : af_launch<2, false>(A, max_rows, ctas, part_keys, smem, scores, ld, room, max_total, stream);
  else e = plain ? af_launch<1, true>(A, max_rows, ctas, part_keys, smem, scores, ld, room, max_total, stream) : af_launch<1, false>(A, max_rows, ctas, part_keys, smem, scores, ld, room, max_total, stream);
  if (e != cudaSuccess) { qe_set_error("attention_weights: launch failed: %s", cudaGetErrorString(e)); (void)cudaGetLastError(); return 2; }
  QE_CHECK_LAUNCH("attention_weights");
  return 0;
}

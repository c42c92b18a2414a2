// Gathered attention weights of prompt portions in bfloat16, on the fifth-generation tensor cores.  What they are:
// attention_weights.cu.  As there, the scores are formed twice, once along the rows (maximum and sum of each) and once along
// the keys (the sums down the columns).
//
// Both passes are one kernel: a CTA keeps up to four tiles of 128 rows of one operand in shared memory (A: the queries' rows in the first pass,
// keys in the second) and streams tiles of 128 rows of the other (B) past them, 128 x 128 products S = A B^T by
// tcgen05.mma into one of four accumulators of tensor memory.  A thread owns a row of A (= a lane of tensor memory): its
// running maximum and sum over the columns in the first pass, its sum in the second; nothing is exchanged between threads but at
// the end.  Four tiles of A a tile of B keep the reads from L2 at 8 KB a product.  Ten warps: two groups of four read accumulators
// (products alternate between them), one fetches tiles with TMA, one issues the products.
//
// A unit is a (request, kv head, group of A tiles) and a part of the B tiles; parts are merged by a small kernel behind each
// pass, in their order, so sums do not depend on which CTA was first.  Between the passes it leaves every row's -maximum
// and 1 / sum in the order of the second pass's columns.
//
// What bounds it: a product of 128 x 128 x 128 takes the tensor cores 512 cycles and its 16 384 exponentials the
// special-function unit 1 024.
//
// Every wait is bounded: one that runs out records a code, raises the CTA's abort flag, and the CTA leaves without writing.
#include "attention_weights.cuh"
#include "tcgen05.cuh"

#define AT2_TILE 128
#define AT2_THREADS 320
#define AT2_BLOCK_BYTES (AT2_TILE * 128)         // 64 channels of a tile: 128-byte swizzled rows
#define AT2_BLOCKS 12                            // such blocks in shared memory
#define AT2_MAX_RING 4
#define AT2_COLS 512

static __device__ int g_awtc_status = 0;

struct __align__(1024) AwTcSmem {
  unsigned char tiles[AT2_BLOCKS][AT2_BLOCK_BYTES];
  uint64_t a_full, b_full[AT2_MAX_RING], b_empty[AT2_MAX_RING], s_full[4], s_empty[4];
  uint32_t tmem_base;
  int abort_flag, missing;
  float2 meet[AT2_TILE];
};

struct AwTc {
  int few_rows;                // requests of at most so many rows are another kernel's
  int tpt;                     // tokens of a tile of queries
  int kb, na, ring;            // 64-channel blocks of a tile, A tiles of a unit at most (1, 2, 4), B tiles in flight
  int box, parts;              // keys of a TMA box; parts of a unit's B tiles
  int tiles;                   // rows of `negm` and `inv` for a kv head: tiles of queries of all requests
  float* negm; float* inv;     // [Hkv, tiles, 128]: first pass's result, for the second
  float* sums; long sums_ld;   // [parts, R, Hkv, sums_ld]: second pass's parts (null: it writes the output)
};

__device__ __forceinline__ float at2_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float2 at2_fma(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 at2_add(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float at2_max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// waits for the loads from tensor memory; the registers are operands, so that nothing that reads them is moved in front of it
__device__ __forceinline__ void at2_wait_ld(uint32_t (&u)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
               :: "memory");
}

// where request r's tiles of queries begin among all requests' (a tile never holds two requests' rows)
__device__ __forceinline__ int at2_tile0(const AwReq& R, int r, int tpt) { return R.row0 / tpt + r; }

// one thread's share of the first pass: its row's running maximum and sum, and the keys it may see
struct At2Row { float m, z, slope; int lo, hi, pos; };

// 32 scores of the row, columns c0 .. c0 + 31 of the key tile that starts at key `base`
template <bool GENERAL>
__device__ __forceinline__ void at2_row_chunk(const AwArgs& A, const AwReq& R, int r, const uint32_t (&u)[32], int base, int c0, At2Row& st, bool missing) {
  const int k0 = base + c0;
  const bool in = k0 >= st.lo && k0 + 32 <= st.hi && !missing, out = k0 >= st.hi || k0 + 32 <= st.lo;
  if (__all_sync(0xffffffffu, out)) return;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
  if (GENERAL) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = aw_score(A, v[i], st.slope, st.pos - (k0 + i));
  }
  const float sc = GENERAL ? 1.f : A.scale * AW_LOG2E;
  if (!__all_sync(0xffffffffu, in)) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int key = k0 + i;
      v[i] = key >= st.lo && key < st.hi ? v[i] : -INFINITY;
    }
    if (missing) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = aw_page(A, r, k0 + i) >= 0 ? v[i] : -INFINITY;
    }
  }
  float ma = at2_max3(v[0], v[1], v[2]), mb = at2_max3(v[3], v[4], v[5]);
#pragma unroll
  for (int i = 6; i < 30; i += 4) { ma = at2_max3(ma, v[i], v[i + 1]); mb = at2_max3(mb, v[i + 2], v[i + 3]); }
  const float mx = fmaxf(st.m, at2_max3(ma, mb, fmaxf(v[30], v[31])) * sc);      // (the scale is positive)
  const float nb = mx == -INFINITY ? 0.f : -mx;
  const float2 sc2 = make_float2(sc, sc), nb2 = make_float2(nb, nb);
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float2 x = at2_fma(make_float2(v[i], v[i + 1]), sc2, nb2), y = at2_fma(make_float2(v[i + 2], v[i + 3]), sc2, nb2);
    s0 = at2_add(s0, make_float2(at2_ex2(x.x), at2_ex2(x.y)));
    s1 = at2_add(s1, make_float2(at2_ex2(y.x), at2_ex2(y.y)));
  }
  st.z = st.z * at2_ex2(st.m + nb) + ((s0.x + s0.y) + (s1.x + s1.y));
  st.m = mx;
}

// The second pass's: 32 columns (rows of queries) of the thread's key; lo, hi: the columns that see it; nm, iv: the columns' -maximum and 1 / sum.
template <bool GENERAL>
__device__ __forceinline__ void at2_key_chunk(const AwArgs& A, const uint32_t (&u)[32], int c0, int lo, int hi, const float* nm, const float* iv,
                                              int c, int G, int dist0, float2& acc) {
  const bool in = c0 >= lo && c0 + 32 <= hi, out = c0 >= hi || c0 + 32 <= lo;
  if (__all_sync(0xffffffffu, out)) return;
  const bool whole = __all_sync(0xffffffffu, in);
  const float sc = GENERAL ? 1.f : A.scale * AW_LOG2E;
  const float2 sc2 = make_float2(sc, sc);
  float2 a0 = make_float2(0.f, 0.f), a1 = a0;
  int t = 0, g = 0;
  if (GENERAL) { t = c0 / G; g = c0 - t * G; }
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = __uint_as_float(u[i + e]);
      if (GENERAL) {
        v[e] = aw_score(A, v[e], A.slopes ? A.slopes[c * G + g] : 0.f, dist0 + t);
        if (++g == G) { g = 0; ++t; }
      }
      if (!whole) v[e] = c0 + i + e >= lo && c0 + i + e < hi ? v[e] : -INFINITY;
    }
    const float4 m4 = __ldg(reinterpret_cast<const float4*>(nm + c0 + i)), i4 = __ldg(reinterpret_cast<const float4*>(iv + c0 + i));
    const float2 x = at2_fma(make_float2(v[0], v[1]), sc2, make_float2(m4.x, m4.y)), y = at2_fma(make_float2(v[2], v[3]), sc2, make_float2(m4.z, m4.w));
    a0 = at2_fma(make_float2(at2_ex2(x.x), at2_ex2(x.y)), make_float2(i4.x, i4.y), a0);
    a1 = at2_fma(make_float2(at2_ex2(y.x), at2_ex2(y.y)), make_float2(i4.z, i4.w), a1);
  }
  acc = at2_add(acc, at2_add(a0, a1));
}

template <int PASS, bool GENERAL>
__global__ void __launch_bounds__(AT2_THREADS, 1)
attention_weights_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, AwArgs A, AwTc C) {
  extern __shared__ unsigned char raw[];
  AwTcSmem& sm = *reinterpret_cast<AwTcSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = blockIdx.y, r = blockIdx.z, part = blockIdx.x % C.parts, G = A.Hq / A.Hkv, tpt = C.tpt;
  pdl_launch_dependents();
  pdl_wait();                                     // (lengths and counts are an earlier kernel's)
  const AwReq R = aw_req(A, r);
  if ((long)R.n * G <= C.few_rows) return;
  const int slot = A.slot_ids[r];
  // the unit's A tiles a0 .. a0 + n_a - 1, and its part b0 .. b1 - 1 of the B tiles that meet them
  int a0, n_a, b0, b1;
  {
    const int groups = gridDim.x / C.parts, order = blockIdx.x / C.parts;
    const int group = PASS == 1 ? groups - 1 - order : order;                     // (the longest units first)
    a0 = group * C.na;
    if (PASS == 1) {
      const int nq = (R.counted + tpt - 1) / tpt;
      if (a0 >= nq) return;
      n_a = min(C.na, nq - a0);
      const int first = R.ctx + a0 * tpt, last = R.ctx + min((a0 + n_a) * tpt, R.counted) - 1;
      b0 = A.window > 0 ? max(0, first - A.window + 1) / AT2_TILE : 0;
      b1 = last / AT2_TILE + 1;
    } else {
      const int nk = (R.total + AT2_TILE - 1) / AT2_TILE;
      if (a0 >= nk || slot < 0 || slot >= A.slots) return;
      n_a = min(C.na, nk - a0);
      const int t0 = max(0, a0 * AT2_TILE - R.ctx);
      const int t1 = A.window > 0 ? (int)min((long)R.counted, (long)(a0 + n_a) * AT2_TILE - 1 + A.window - R.ctx) : R.counted;
      b0 = t0 / tpt;
      b1 = t1 > t0 ? (t1 + tpt - 1) / tpt : b0;
    }
    const int per = max(2, (b1 - b0 + C.parts - 1) / C.parts);
    b0 = min(b1, b0 + part * per);
    b1 = min(b1, b0 + per);
  }
  const int n_seq = n_a == 3 ? 4 : n_a, steps = b1 - b0;     // products of a step, numbered as if there were 1, 2 or 4
  const bool work = steps > 0;
  const int tile_blocks = C.kb, n_ring = C.ring;
  auto a_tile = [&](int a) { return sm.tiles[a * tile_blocks]; };
  auto b_tile = [&](int s) { return sm.tiles[(C.na + s) * tile_blocks]; };
  volatile int* abort_flag = &sm.abort_flag;
  if (tid == 0) {
    mbar_init(&sm.a_full, 1);
    for (int s = 0; s < AT2_MAX_RING; ++s) { mbar_init(&sm.b_full[s], 1); mbar_init(&sm.b_empty[s], 1); }
    for (int s = 0; s < 4; ++s) { mbar_init(&sm.s_full[s], 1); mbar_init(&sm.s_empty[s], AT2_TILE); }
    sm.abort_flag = 0;
    sm.missing = 0;
    mbar_init_fence();
  }
  if (work && warp == 9) tc_alloc(&sm.tmem_base, AT2_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = work ? sm.tmem_base : 0u;
  if (PASS == 1 && work) {
    // does a key of the part lie in no page?
    const int k1 = min(b1 * AT2_TILE, R.total), f = b0 * AT2_TILE / A.page, l = (k1 - 1) / A.page;
    for (int b = f + tid; b <= l; b += AT2_THREADS)
      if (aw_page(A, r, b * A.page) < 0) sm.missing = 1;
    __syncthreads();
  }

  if (warp == 8) {
    // ================= fetching ============================================================================
    if (work) {
      auto fetch_q = [&](unsigned char* dst, int tile, uint64_t* bar) {
        if (lane < C.kb) tma_load_3d(dst + lane * AT2_BLOCK_BYTES, &map_q, bar, lane * 64, c * G, R.row0 + tile * tpt);
      };
      auto fetch_k = [&](unsigned char* dst, int tile, uint64_t* bar) {
        const int boxes = AT2_TILE / C.box;
        for (int i = lane; i < boxes * C.kb; i += 32) {
          const int b = i / C.kb, k = i - b * C.kb, key = tile * AT2_TILE + b * C.box;
          int page = aw_page(A, r, key);
          if (page < 0) page = A.num_pages;       // outside the tensor: zeros
          tma_load_5d(dst + k * AT2_BLOCK_BYTES + b * C.box * 128, &map_k, bar, k * 64, key % A.page, c, 0, page);
        }
      };
      const uint32_t q_bytes = (uint32_t)C.kb * (uint32_t)(tpt * G) * 128u, k_bytes = (uint32_t)C.kb * AT2_BLOCK_BYTES;
      const uint32_t a_bytes = PASS == 1 ? q_bytes : k_bytes, b_bytes = PASS == 1 ? k_bytes : q_bytes;
      if (lane == 0) mbar_expect_tx(&sm.a_full, a_bytes * n_a);
      __syncwarp();
      int issued = 0;
      bool ok = true;
      for (int s = 0; s < steps; ++s) {
        const int st = s % n_ring;
        if (s >= n_ring) ok = mbar_wait(&sm.b_empty[st], ((s / n_ring) - 1) & 1, abort_flag, 1, &g_awtc_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&sm.b_full[st], b_bytes);
        __syncwarp();
        if (PASS == 1) fetch_k(b_tile(st), b0 + s, &sm.b_full[st]); else fetch_q(b_tile(st), b0 + s, &sm.b_full[st]);
        ++issued;
        if (s == 0)
          for (int a = 0; a < n_a; ++a) {
            if (PASS == 1) fetch_q(a_tile(a), a0 + a, &sm.a_full); else fetch_k(a_tile(a), a0 + a, &sm.a_full);
          }
      }
      if (*abort_flag && lane == 0) {
        // giving up: the copies in flight land before the CTA leaves (bounded)
        for (uint32_t i = 0; i < TC_WAIT_LIMIT; ++i) if (mbar_try_wait(&sm.a_full, 0)) break;
        for (int s = max(0, issued - n_ring); s < issued; ++s)
          for (uint32_t i = 0; i < TC_WAIT_LIMIT; ++i) if (mbar_try_wait(&sm.b_full[s % n_ring], (s / n_ring) & 1)) break;
      }
    }
  } else if (warp == 9) {
    // ================= products: one thread ==================================================================
    if (work && lane == 0) {
      constexpr uint32_t idesc = make_idesc(AT2_TILE, AT2_TILE);
      const int ks = (A.D + 15) / 16;
      bool ok = mbar_wait(&sm.a_full, 0, abort_flag, 2, &g_awtc_status);
      for (int s = 0; ok && s < steps; ++s) {
        const int st = s % n_ring;
        ok = mbar_wait(&sm.b_full[st], (s / n_ring) & 1, abort_flag, 3, &g_awtc_status);
        for (int a = 0; ok && a < n_a; ++a) {
          const int i = s * n_seq + a, acc = i & 3;
          if (i >= 4) ok = mbar_wait(&sm.s_empty[acc], ((i >> 2) - 1) & 1, abort_flag, 4, &g_awtc_status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = make_smem_desc(smem_u32(a_tile(a))), db = make_smem_desc(smem_u32(b_tile(st)));
          for (int k = 0; k < ks; ++k) {
            const uint64_t off = (uint64_t)(k >> 2) * (AT2_BLOCK_BYTES >> 4) + 2 * (k & 3);
            tc_mma_bf16(tmem + acc * AT2_TILE, da + off, db + off, idesc, k != 0);
          }
          tc_commit(&sm.s_full[acc]);
        }
        if (ok) tc_commit(&sm.b_empty[st]);
      }
    }
  } else {
    // ================= the two groups that read accumulators ====================================================
    const int w = warp >> 2, rr = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    At2Row row[2];
    float2 sum[2];
    int key[2];
    const bool missing = PASS == 1 && sm.missing != 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int a = n_seq == 4 ? w + 2 * x : (n_seq == 2 ? w : 0);
      sum[x] = make_float2(0.f, 0.f);
      if (PASS == 1) {
        const int t = (a0 + a) * tpt + rr / G;
        const bool valid = rr < tpt * G && t < R.counted && a < n_a;
        row[x].m = -INFINITY; row[x].z = 0.f;
        row[x].pos = R.ctx + t;
        row[x].hi = valid ? row[x].pos + 1 : 0;
        row[x].lo = A.window > 0 ? max(0, row[x].pos - A.window + 1) : 0;
        row[x].slope = GENERAL && A.slopes && valid ? A.slopes[c * G + rr % G] : 0.f;
      } else {
        key[x] = (a0 + a) * AT2_TILE + rr;
      }
    }
    bool ok = true;
    for (int i = w; i < steps * n_seq; i += 2) {
      const int s = i / n_seq, a = i - s * n_seq, acc = i & 3;
      if (a >= n_a) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(&sm.s_full[acc], (i >> 2) & 1, abort_flag, 5, &g_awtc_status));
      if (!ok) break;
      tc_fence_after();
      const uint32_t col = lanes + acc * AT2_TILE;
      const int tile = b0 + s;
      const bool second = n_seq == 4 && a >= 2;
      // the second pass: the columns [lo, hi) see this thread's key
      int lo = 0, hi = 0, dist0 = 0;
      const float *nm = nullptr, *iv = nullptr;
      if (PASS == 2) {
        const int k = second ? key[1] : key[0], tok0 = tile * tpt;
        lo = max(0, k - R.ctx - tok0) * G;
        hi = max(0, min(tpt, R.counted - tok0)) * G;
        if (A.window > 0) hi = (int)max(0L, min((long)hi, ((long)k + A.window - R.ctx - tok0) * G));
        if (k >= R.total) hi = 0;
        dist0 = R.ctx + tok0 - k;
        const size_t at = ((size_t)c * C.tiles + at2_tile0(R, r, tpt) + tile) * AT2_TILE;
        nm = C.negm + at; iv = C.inv + at;
      }
      uint32_t u[2][32];
      tc_ld_32x32b_x32(col, u[0]);
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        at2_wait_ld(u[ch & 1]);
        if (ch < 3) tc_ld_32x32b_x32(col + 32 * (ch + 1), u[(ch + 1) & 1]);
        else { tc_fence_before(); mbar_arrive(&sm.s_empty[acc]); }
        if (PASS == 1) {
          if (second) at2_row_chunk<GENERAL>(A, R, r, u[ch & 1], tile * AT2_TILE, 32 * ch, row[1], missing);
          else at2_row_chunk<GENERAL>(A, R, r, u[ch & 1], tile * AT2_TILE, 32 * ch, row[0], missing);
        } else {
          if (second) at2_key_chunk<GENERAL>(A, u[ch & 1], 32 * ch, lo, hi, nm, iv, c, G, dist0, sum[1]);
          else at2_key_chunk<GENERAL>(A, u[ch & 1], 32 * ch, lo, hi, nm, iv, c, G, dist0, sum[0]);
        }
      }
    }
    // one A tile: both groups have seen some of its columns
    if (n_seq == 1) {
      if (w == 1) sm.meet[rr] = PASS == 1 ? make_float2(row[0].m, row[0].z) : make_float2(sum[0].x + sum[0].y, 0.f);
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      if (w == 0) {
        const float2 o = sm.meet[rr];
        if (PASS == 1) {
          const float m = fmaxf(row[0].m, o.x);
          if (m != -INFINITY) row[0].z = row[0].z * exp2f(row[0].m - m) + o.y * exp2f(o.x - m);
          row[0].m = m;
        } else {
          sum[0].x += o.x;
        }
      }
    }
    if (ok && !*abort_flag) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int a = n_seq == 4 ? w + 2 * x : (n_seq == 2 ? w : 0);
        if (a >= n_a || (x == 1 && n_seq != 4) || (n_seq == 1 && w == 1)) continue;
        if (PASS == 1) {
          const int t = (a0 + a) * tpt + rr / G;
          if (rr < tpt * G && t < R.counted) {
            float* st = A.stats + (((size_t)(R.row0 + t) * A.Hq + c * G + rr % G) * C.parts + part) * 2;
            st[0] = row[x].m; st[1] = row[x].z;
          }
        } else if (key[x] < R.total) {
          const int k = key[x];
          const float total = aw_page(A, r, k) >= 0 ? sum[x].x + sum[x].y : 0.f;
          if (C.sums) {
            C.sums[(((size_t)part * A.R + r) * A.Hkv + c) * C.sums_ld + k] = total;
          } else {
            const size_t at = ((size_t)slot * A.Hkv + c) * A.capacity + k;
            A.out[at] = k < R.ctx ? A.weights[at] + total : total;
            if (A.positions && k >= R.ctx) A.positions[at] = A.step_positions[R.row0 + k - R.ctx];
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (work && warp == 9) {
    tc_fence_after();
    tc_dealloc(tmem, AT2_COLS);
  }
}

// Every row's parts put together, in the order of the second pass's columns; columns without a row get weight 0.
__global__ void __launch_bounds__(AT2_TILE)
attention_weights_merge_kernel(AwArgs A, AwTc C) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.y, r = blockIdx.z, tile = blockIdx.x, rr = threadIdx.x, G = A.Hq / A.Hkv;
  const AwReq R = aw_req(A, r);
  if ((long)R.n * G <= C.few_rows || tile * C.tpt >= R.counted) return;
  const int t = tile * C.tpt + rr / G;
  float2 v = make_float2(INFINITY, 0.f);
  if (rr < C.tpt * G && t < R.counted) {
    const int head = c * G + rr % G;
    v = aw_merge(A.stats + ((size_t)(R.row0 + t) * A.Hq + head) * C.parts * 2, C.parts, A.sinks ? A.sinks + head : nullptr);
  }
  const size_t at = ((size_t)c * C.tiles + at2_tile0(R, r, C.tpt) + tile) * AT2_TILE + rr;
  C.negm[at] = -v.x;
  C.inv[at] = v.y;
}

__global__ void __launch_bounds__(256)
attention_weights_finish_kernel(AwArgs A, AwTc C) {
  pdl_launch_dependents();
  pdl_wait();
  const int c = blockIdx.y, r = blockIdx.z, k = blockIdx.x * 256 + threadIdx.x;
  const AwReq R = aw_req(A, r);
  const int slot = A.slot_ids[r];
  if ((long)R.n * (A.Hq / A.Hkv) <= C.few_rows || k >= R.total || slot < 0 || slot >= A.slots) return;
  float total = 0.f;
  for (int p = 0; p < C.parts; ++p) total += C.sums[(((size_t)p * A.R + r) * A.Hkv + c) * C.sums_ld + k];
  const size_t at = ((size_t)slot * A.Hkv + c) * A.capacity + k;
  A.out[at] = k < R.ctx ? A.weights[at] + total : total;
  if (A.positions && k >= R.ctx) A.positions[at] = A.step_positions[R.row0 + k - R.ctx];
}

extern "C" int qe_attention_weights_tc_status() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_awtc_status, sizeof(int));
  return v;
}
extern "C" void qe_attention_weights_tc_clear_status() {
  int v = 0;
  cudaMemcpyToSymbol(g_awtc_status, &v, sizeof(int));
}

// Whether the kernels take the sizes: channels in steps of 8 up to 256, at most 128 query heads a kv head, pages of a multiple of 8 keys.
extern "C" int qe_attention_weights_tc_supported(int Hq, int Hkv, int D, int page) {
  return Hkv >= 1 && Hq % Hkv == 0 && Hq / Hkv <= AT2_TILE && D >= 8 && D % 8 == 0 && D <= 256 && page >= 8 && page % 8 == 0;
}
// A tiles a unit
extern "C" int qe_attention_weights_tc_group(int D) { return D <= 128 ? 4 : (D <= 192 ? 2 : 1); }

template <int PASS, bool GENERAL>
static cudaError_t at2_launch(dim3 grid, cudaStream_t stream, const CUtensorMap& q, const CUtensorMap& k, const AwArgs& A, const AwTc& C) {
  const size_t smem = sizeof(AwTcSmem) + 1024;
  static_assert(tc_room_for_all(sizeof(AwTcSmem) + 1024, AT2_COLS), "tensor memory for every CTA that finds room on an SM");
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attention_weights_tc_kernel<PASS, GENERAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  return qe_launch(attention_weights_tc_kernel<PASS, GENERAL>, grid, dim3(AT2_THREADS), smem, stream, q, k, A, C);
}

// The requests of more than few_rows rows.  stats: [T Hq, parts1, 2] floats; merged: [2, Hkv, T / (128 / G) + R, 128]; sums:
// [parts2, R, Hkv, max_total] where parts2 > 1.  max_q, max_total: the most tokens of a request and the most places it may hold.
extern "C" int qe_attention_weights_tc(const void* q, long q_stride, int T, const void* pages, int num_pages, int planes,
                                       const int* block_tables, int max_blocks, const int* cu_q, const int* ctx_lens, const int* slot_ids,
                                       const int* counted, const int* step_positions, int* positions, const float* weights, float* out,
                                       int slots, long capacity, int R, int Hq, int Hkv, int D, int page, int window, float scale,
                                       float softcap, const float* slopes, const float* sinks, float* stats, int parts1, int parts2, float* merged,
                                       float* sums, int max_q, int max_total, int few_rows, cudaStream_t stream) {
  if (R <= 0 || max_total <= 0 || max_q <= 0) return 0;
  if (!qe_attention_weights_tc_supported(Hq, Hkv, D, page)) QE_REFUSE("attention_weights: heads %d/%d, head_dim %d, pages of %d are not for the tensor cores", Hq, Hkv, D, page);
  if ((((uintptr_t)q | (uintptr_t)pages) & 15) || q_stride % 8) QE_REFUSE("attention_weights: operands must be 16-byte aligned");
  if (((uintptr_t)merged & 15) || merged == nullptr || stats == nullptr || parts1 < 1 || parts2 < 1 || (parts2 > 1 && sums == nullptr))
    QE_REFUSE("attention_weights: scratch memory is needed");
  if (R > 65535 || Hkv > 65535) QE_REFUSE("attention_weights: %d requests, %d kv heads are more than a launch takes", R, Hkv);
  const int G = Hq / Hkv;
  AwTc C{};
  C.few_rows = few_rows;
  C.tpt = AT2_TILE / G;
  C.kb = (D + 63) / 64;
  C.na = qe_attention_weights_tc_group(D);
  C.ring = (AT2_BLOCKS - C.na * C.kb) / C.kb;
  if (C.ring > AT2_MAX_RING) C.ring = AT2_MAX_RING;
  C.box = 8;
  while (C.box < AT2_TILE && page % (2 * C.box) == 0) C.box *= 2;
  C.tiles = T / C.tpt + R;
  C.negm = merged;
  C.inv = merged + (size_t)Hkv * C.tiles * AT2_TILE;
  C.sums = parts2 > 1 ? sums : nullptr;
  C.sums_ld = max_total;
  AwArgs A{q, q_stride, T, pages, num_pages, planes, block_tables, max_blocks, cu_q, ctx_lens, slot_ids, counted, step_positions, positions,
           weights, out, slots, capacity, R, Hq, Hkv, D, page, window, scale, softcap, slopes, sinks, stats, parts1};
  CUtensorMap map_q, map_k;
  {
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)T};
    const uint64_t strides[2] = {(uint64_t)D * 2, (uint64_t)q_stride * 2};
    const uint32_t box[3] = {64, (uint32_t)G, (uint32_t)C.tpt};
    if (!qe_tensor_map_bf16(q, 3, dims, strides, box, &map_q)) return 1;
  }
  {
    const uint64_t P = (uint64_t)page;
    const uint64_t dims[5] = {(uint64_t)D, P, (uint64_t)Hkv, (uint64_t)planes, (uint64_t)num_pages};
    const uint64_t strides[4] = {(uint64_t)D * 2, P * D * 2, (uint64_t)Hkv * P * D * 2, (uint64_t)planes * Hkv * P * D * 2};
    const uint32_t box[5] = {64, (uint32_t)C.box, 1, 1, 1};
    if (!qe_tensor_map_bf16(pages, 5, dims, strides, box, &map_k)) return 1;
  }
  const int q_tiles = (max_q + C.tpt - 1) / C.tpt, k_tiles = (max_total + AT2_TILE - 1) / AT2_TILE;
  const dim3 grid1((unsigned)((q_tiles + C.na - 1) / C.na * parts1), (unsigned)Hkv, (unsigned)R), grid2((unsigned)((k_tiles + C.na - 1) / C.na * parts2), (unsigned)Hkv, (unsigned)R);
  const bool general = softcap > 0.f || slopes != nullptr;
  C.parts = parts1;
  cudaError_t e = general ? at2_launch<1, true>(grid1, stream, map_q, map_k, A, C) : at2_launch<1, false>(grid1, stream, map_q, map_k, A, C);
  if (e == cudaSuccess) e = qe_launch(attention_weights_merge_kernel, dim3((unsigned)q_tiles, (unsigned)Hkv, (unsigned)R), dim3(AT2_TILE), 0, stream, A, C);
  C.parts = parts2;
  if (e == cudaSuccess) e = general ? at2_launch<2, true>(grid2, stream, map_q, map_k, A, C) : at2_launch<2, false>(grid2, stream, map_q, map_k, A, C);
  if (e == cudaSuccess && C.sums)
    e = qe_launch(attention_weights_finish_kernel, dim3((unsigned)((max_total + 255) / 256), (unsigned)Hkv, (unsigned)R), dim3(256), 0, stream, A, C);
  if (e != cudaSuccess) { qe_set_error("attention_weights: launch failed: %s", cudaGetErrorString(e)); (void)cudaGetLastError(); return 2; }
  QE_CHECK_LAUNCH("attention_weights");
  return 0;
}

// Gathered attention weights of prompt portions in bfloat16, on the fifth-generation tensor cores.  What they are:
// attention_weights.cu.  As there, the scores are formed twice, once along the rows (maximum and sum of each) and once along
// the keys (the sums down the columns).
//
// Both passes are one kernel: a CTA keeps up to four tiles of 128 rows of one operand in shared memory (A: the queries' rows in the first pass,
// keys in the second) and streams tiles of 128 rows of the other (B) past them, 128 x 128 products S = A B^T by
// tcgen05.mma into one of four accumulators of tensor memory.  A thread owns a row of A (= a lane of tensor memory): its
// running maximum and sum over the columns in the first pass, its sum in the second; nothing is exchanged between threads but at
// the end.  Four tiles of A a tile of B keep the reads from L2 at 8 KB a product.  Eighteen warps: four groups of four read one accumulator
// each, one warp fetches tiles with TMA, one issues the products.
//
// A unit is a (request, kv head, group of A tiles) and a part of the B tiles; parts are merged by a small kernel behind each
// pass, in their order, so sums do not depend on which CTA was first.  Between the passes it leaves -log2 of every row's whole
// sum, exponentials and maximum together, in the order of the second pass's columns: a weight is then one exponential.  That number is rounded
// to float32, so a weight is off by up to 2^-24 ln 2 times its size relative to itself, as it is by the rounding of its score.
//
// What bounds it: a product of 128 x 128 x 128 takes the tensor cores 512 cycles at best (both operands from shared memory, 8 KB every 64 cycles, are
// all that it delivers; measured, with the readers beside it, about 950), its 16 384 exponentials the special-function unit 1 024.  No unit is
// saturated (4 096 tokens: special functions 65 % of an SM's cycles, tensor cores 36 and 40 %, issue slots 45 and 41 %; the passes 105 and 131 us on
// cold caches): a group of readers has one accumulator, which the next product gets when its last columns have been read, and waits for it.  An eighth of the exponentials is a polynomial (at2_poly2), two at a time on the float32
// units: none 256, an eighth 249, a quarter 259, three eighths 271 us for a prompt of 4 096 tokens with 32 / 8 heads (one CTA walking several
// units 269: some are empty, and they are dealt out beforehand; 128 x 256 products in two accumulators 258).  With all heads' longest units first and
// a unit an SM instead of four: 217.
//
// Every wait is bounded: one that runs out records a code, raises the CTA's abort flag, and the CTA leaves without writing.
#include "attention_weights.cuh"
#include "tcgen05.cuh"

#define AT2_TILE 128
#define AT2_GROUPS 4                              // groups of four warps that read accumulators, one each
#define AT2_READERS (128 * AT2_GROUPS)
#define AT2_THREADS (AT2_READERS + 64)
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
  float2 meet[AT2_GROUPS][AT2_TILE];
  float4 negl[4 * AT2_GROUPS][2][32];            // second pass: a tile's columns' values for each warp, two tiles in turn
};

struct AwTc {
  int few_rows;                // requests of at most so many rows are another kernel's
  int tpt;                     // tokens of a tile of queries
  int kb, na, ring;            // 64-channel blocks of a tile, A tiles of a unit at most (1, 2, 4), B tiles in flight
  int box, parts;              // keys of a TMA box; parts of a unit's B tiles
  int tiles;                   // rows of `negl` for a kv head: tiles of queries of all requests
  float* negl;                 // [Hkv, tiles, 128]: first pass's result, for the second
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
__device__ __forceinline__ float2 at2_mul(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float at2_max_nan(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ float at2_max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// waits for the loads from tensor memory; the registers are operands, so that nothing that reads them is moved in front of it
__device__ __forceinline__ void at2_wait_ld(uint32_t (&u)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
               :: "memory");
}

// where request r's tiles of queries begin among all requests' (a tile never holds two requests' rows)
__device__ __forceinline__ int at2_tile0(const AwReq& R, int r, int tpt) { return R.row0 / tpt + r; }

// 2^x of two x <= 0 (or a little above) without the special-function unit: x = n + f, |f| <= 1/2, 2^f by a polynomial of degree 5 that is 1 at 0 and
// whose largest relative error on the interval is least (fitted by weighted least squares; 1.6 10^-7 with its float32 coefficients), times 2^n.
// NaN stays NaN: a weight must not depend on which columns come here.
__device__ __forceinline__ float2 at2_poly2(float2 x) {
  x.x = at2_max_nan(x.x, -127.f); x.y = at2_max_nan(x.y, -127.f);         // (2^-127 counts as 0)
  const float magic = 12582912.f;                              // 1.5 2^23: the sum's low bits are x rounded to an integer
  const float2 t = at2_add(x, make_float2(magic, magic)), n = at2_add(t, make_float2(-magic, -magic));
  const float2 f = at2_fma(n, make_float2(-1.f, -1.f), x);
  float2 p = make_float2(0.001326472731307149f, 0.001326472731307149f);
  p = at2_fma(p, f, make_float2(0.009671512991189957f, 0.009671512991189957f));
  p = at2_fma(p, f, make_float2(0.05550733581185341f, 0.05550733581185341f));
  p = at2_fma(p, f, make_float2(0.24022242426872253f, 0.24022242426872253f));
  p = at2_fma(p, f, make_float2(0.6931470036506653f, 0.6931470036506653f));
  p = at2_fma(p, f, make_float2(1.f, 1.f));
  // 2^n as a factor, which a NaN survives
  return at2_mul(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}
// whether the pair of columns 2 j, 2 j + 1 of a chunk goes there
__device__ constexpr bool at2_on_poly(int j) { return (j & 7) == 1; }
__device__ __forceinline__ float2 at2_exp2(float2 x, bool poly) { return poly ? at2_poly2(x) : make_float2(at2_ex2(x.x), at2_ex2(x.y)); }

// one thread's share of the first pass: its row's running maximum and sum, and the keys it may see
struct At2Row { float m, z, slope; int lo, hi, pos; };

// 32 scores of the row, columns c0 .. c0 + 31 of the key tile that starts at key `base`
template <bool GENERAL>
__device__ __forceinline__ void at2_row_chunk(const AwArgs& A, int r, uint32_t (&u)[32], int base, int c0, At2Row& st, bool missing) {
  const int k0 = base + c0;
  const bool in = k0 >= st.lo && k0 + 32 <= st.hi && !missing, out = k0 >= st.hi || k0 + 32 <= st.lo;
  if (__all_sync(0xffffffffu, out)) return;
  if (GENERAL) {
#pragma unroll
    for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(aw_score(A, __uint_as_float(u[i]), st.slope, st.pos - (k0 + i)));
  }
  const float sc = GENERAL ? 1.f : A.scale * AW_LOG2E;
  if (!__all_sync(0xffffffffu, in)) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int key = k0 + i;
      if (!(key >= st.lo && key < st.hi) || (missing && aw_page(A, r, key) < 0)) u[i] = 0xff800000u;      // -inf
    }
  }
  float ma = at2_max3(__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]));
  float mb = at2_max3(__uint_as_float(u[3]), __uint_as_float(u[4]), __uint_as_float(u[5]));
#pragma unroll
  for (int i = 6; i < 30; i += 4) {
    ma = at2_max3(ma, __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
    mb = at2_max3(mb, __uint_as_float(u[i + 2]), __uint_as_float(u[i + 3]));
  }
  const float mx = fmaxf(st.m, at2_max3(ma, mb, fmaxf(__uint_as_float(u[30]), __uint_as_float(u[31]))) * sc);      // (the scale is positive)
  const float nb = mx == -INFINITY ? 0.f : -mx;
  const float2 sc2 = make_float2(sc, sc), nb2 = make_float2(nb, nb);
  float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float2 x = at2_fma(make_float2(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])), sc2, nb2);
    const float2 e = at2_exp2(x, at2_on_poly(j));
    if (j & 1) s1 = at2_add(s1, e); else s0 = at2_add(s0, e);
  }
  st.z = st.z * at2_ex2(st.m + nb) + ((s0.x + s0.y) + (s1.x + s1.y));
  st.m = mx;
}

// The second pass's: 32 columns (rows of queries) of the thread's key; lo, hi: the columns that see it; nl: the columns' values (shared memory).
template <bool GENERAL>
__device__ __forceinline__ void at2_key_chunk(const AwArgs& A, uint32_t (&u)[32], int c0, int lo, int hi, const float* nl, int c, int G,
                                              int dist0, float2& acc) {
  const bool in = c0 >= lo && c0 + 32 <= hi, out = c0 >= hi || c0 + 32 <= lo;
  if (__all_sync(0xffffffffu, out)) return;
  const float sc = GENERAL ? 1.f : A.scale * AW_LOG2E;
  if (GENERAL) {
    int t = c0 / G, g = c0 - t * G;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      u[i] = __float_as_uint(aw_score(A, __uint_as_float(u[i]), A.slopes ? A.slopes[c * G + g] : 0.f, dist0 + t));
      if (++g == G) { g = 0; ++t; }
    }
  }
  if (!__all_sync(0xffffffffu, in)) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c0 + i < lo || c0 + i >= hi) u[i] = 0xff800000u;      // -inf
  }
  const float2 sc2 = make_float2(sc, sc);
  float2 a0 = make_float2(0.f, 0.f), a1 = a0;
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    const float4 l4 = *(reinterpret_cast<const float4*>(nl + c0) + (j >> 1));
    const float2 x = at2_fma(make_float2(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])), sc2, make_float2(l4.x, l4.y));
    const float2 y = at2_fma(make_float2(__uint_as_float(u[2 * j + 2]), __uint_as_float(u[2 * j + 3])), sc2, make_float2(l4.z, l4.w));
    a0 = at2_add(a0, at2_exp2(x, at2_on_poly(j)));
    a1 = at2_add(a1, at2_exp2(y, at2_on_poly(j + 1)));
  }
  acc = at2_add(acc, at2_add(a0, a1));
}

template <int PASS, bool GENERAL>
__global__ void __launch_bounds__(AT2_THREADS, 1)
attention_weights_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, AwArgs A, AwTc C) {
  extern __shared__ unsigned char raw[];
  AwTcSmem& sm = *reinterpret_cast<AwTcSmem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = blockIdx.x / C.parts % A.Hkv, r = blockIdx.z, part = blockIdx.x % C.parts, G = A.Hq / A.Hkv, tpt = C.tpt;
  pdl_launch_dependents();
  pdl_wait();                                     // (lengths and counts are an earlier kernel's)
  const AwReq R = aw_req(A, r);
  if ((long)R.n * G <= C.few_rows) return;
  const int slot = A.slot_ids[r];
  // the unit's A tiles a0 .. a0 + n_a - 1, and its part b0 .. b1 - 1 of the B tiles that meet them
  int a0, n_a, b0, b1;
  {
    // the longest units first, all heads' before the next: CTAs start in this order, and what starts last is short
    const int groups = gridDim.x / (C.parts * A.Hkv), order = blockIdx.x / (C.parts * A.Hkv);
    const int group = PASS == 1 ? groups - 1 - order : order;
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
  if (work && warp == 4 * AT2_GROUPS + 1) tc_alloc(&sm.tmem_base, AT2_COLS);
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

  if (warp == 4 * AT2_GROUPS) {
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
  } else if (warp == 4 * AT2_GROUPS + 1) {
    // ================= products ================================================================================
    // The whole warp walks the loop and one lane is elected for each instruction (tcgen05.cuh says why); with the descriptors worked
    // out beside the loop.  (One lane in a branch, descriptors worked out in the loop: 180 cycles an instruction, and the readers waited.)
    if (work) {
      constexpr uint32_t idesc = make_idesc(AT2_TILE, AT2_TILE);
      const int ks = (A.D + 15) / 16;
      const uint64_t d0 = make_smem_desc(smem_u32(sm.tiles[0]));
      const uint32_t tile_step = (uint32_t)tile_blocks * (AT2_BLOCK_BYTES >> 4);
      bool ok = __all_sync(0xffffffffu, mbar_wait(&sm.a_full, 0, abort_flag, 2, &g_awtc_status));
      int st = 0, i = 0;
      uint32_t b_par = 0;
      for (int s = 0; ok && s < steps; ++s, i += n_seq) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.b_full[st], b_par, abort_flag, 3, &g_awtc_status));
        const uint64_t db = d0 + (uint32_t)(C.na + st) * tile_step;
        uint64_t da = d0;
        for (int a = 0; ok && a < n_a; ++a, da += tile_step) {
          const int acc = (i + a) & 3, use = (i + a) >> 2;
          if (use > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm.s_empty[acc], (use - 1) & 1, abort_flag, 4, &g_awtc_status));
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + acc * AT2_TILE;
          if (ks == 8) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t off = (uint32_t)(k >> 2) * (AT2_BLOCK_BYTES >> 4) + 2 * (k & 3);
              tc_mma_bf16_elect(d, da + off, db + off, idesc, k != 0);
            }
          } else {
            for (int k = 0; k < ks; ++k) {
              const uint32_t off = (uint32_t)(k >> 2) * (AT2_BLOCK_BYTES >> 4) + 2 * (k & 3);
              tc_mma_bf16_elect(d, da + off, db + off, idesc, k != 0);
            }
          }
          tc_commit_elect(&sm.s_full[acc]);
        }
        if (ok) tc_commit_elect(&sm.b_empty[st]);
        if (++st == n_ring) { st = 0; b_par ^= 1; }
      }
    }
  } else {
    // ================= the groups that read accumulators ========================================================
    // group w reads accumulator w: products w, w + 4, .. of tile w % n_seq; groups with one tile share its columns
    const int w = warp >> 2, rr = (warp & 3) * 32 + lane, a = w % n_seq, share = AT2_GROUPS / n_seq;
    const uint32_t col = tmem + ((uint32_t)((warp & 3) * 32) << 16) + w * AT2_TILE;
    const bool mine = a < n_a;
    At2Row row;
    float2 sum = make_float2(0.f, 0.f);
    int key = 0;
    const bool missing = PASS == 1 && sm.missing != 0;
    if (PASS == 1) {
      const int t = (a0 + a) * tpt + rr / G;
      const bool valid = rr < tpt * G && t < R.counted && mine;
      row.m = -INFINITY; row.z = 0.f;
      row.pos = R.ctx + t;
      row.hi = valid ? row.pos + 1 : 0;
      row.lo = A.window > 0 ? max(0, row.pos - A.window + 1) : 0;
      row.slope = GENERAL && A.slopes && valid ? A.slopes[c * G + rr % G] : 0.f;
    } else {
      key = (a0 + a) * AT2_TILE + rr;
    }
    bool ok = true;
    // the second pass: the columns' values of the next tile are on their way while this one's are used, from every warp's own copy
    const float4* nl_row = PASS == 2 ? reinterpret_cast<const float4*>(C.negl + ((size_t)c * C.tiles + at2_tile0(R, r, tpt) + b0) * AT2_TILE) + lane : nullptr;
    float4 nl_next = make_float4(0.f, 0.f, 0.f, 0.f);
    if (PASS == 2 && mine && w / n_seq < steps) nl_next = __ldg(nl_row + (size_t)(w / n_seq) * 32);
    if (mine)
      for (int s = w / n_seq, use = 0; s < steps; s += share, ++use) {
        if (PASS == 2) {
          sm.negl[warp][use & 1][lane] = nl_next;
          if (s + share < steps) nl_next = __ldg(nl_row + (size_t)(s + share) * 32);
          __syncwarp();
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.s_full[w], use & 1, abort_flag, 5, &g_awtc_status));
        if (!ok) break;
        tc_fence_after();
        const int tile = b0 + s;
        // the second pass: the columns [lo, hi) see this thread's key
        int lo = 0, hi = 0, dist0 = 0;
        if (PASS == 2) {
          const int tok0 = tile * tpt;
          lo = max(0, key - R.ctx - tok0) * G;
          hi = max(0, min(tpt, R.counted - tok0)) * G;
          if (A.window > 0) hi = (int)max(0L, min((long)hi, ((long)key + A.window - R.ctx - tok0) * G));
          if (key >= R.total) hi = 0;
          dist0 = R.ctx + tok0 - key;
        }
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t u[32];
          tc_ld_32x32b_x32(col + 32 * ch, u);
          at2_wait_ld(u);
          if (ch == 3) { tc_fence_before(); mbar_arrive(&sm.s_empty[w]); }
          if (PASS == 1) at2_row_chunk<GENERAL>(A, r, u, tile * AT2_TILE, 32 * ch, row, missing);
          else at2_key_chunk<GENERAL>(A, u, 32 * ch, lo, hi, reinterpret_cast<const float*>(sm.negl[warp][use & 1]), c, G, dist0, sum);
        }
      }
    float total = sum.x + sum.y;
    if (n_seq < 4) {
      // the groups that share a tile put their columns together, in the groups' order
      sm.meet[w][rr] = PASS == 1 ? make_float2(row.m, row.z) : make_float2(total, 0.f);
      asm volatile("bar.sync 1, %0;\n" :: "n"(AT2_READERS) : "memory");
      if (w < n_seq)
        for (int o = w + n_seq; o < AT2_GROUPS; o += n_seq) {
          const float2 v = sm.meet[o][rr];
          if (PASS == 1) {
            const float m = fmaxf(row.m, v.x), base = aw_base(m);
            row.z = row.z * exp2f(row.m - base) + v.y * exp2f(v.x - base);
            row.m = m;
          } else {
            total += v.x;
          }
        }
    }
    if (ok && !*abort_flag && w < n_seq && mine) {
      if (PASS == 1) {
        const int t = (a0 + a) * tpt + rr / G;
        if (rr < tpt * G && t < R.counted) {
          float* st = A.stats + (((size_t)(R.row0 + t) * A.Hq + c * G + rr % G) * C.parts + part) * 2;
          st[0] = row.m; st[1] = row.z;
        }
      } else if (key < R.total) {
        if (aw_page(A, r, key) < 0) total = 0.f;
        if (C.sums) {
          C.sums[(((size_t)part * A.R + r) * A.Hkv + c) * C.sums_ld + key] = total;
        } else {
          const size_t at = ((size_t)slot * A.Hkv + c) * A.capacity + key;
          A.out[at] = key < R.ctx ? A.weights[at] + total : total;
          if (A.positions && key >= R.ctx) A.positions[at] = A.step_positions[R.row0 + key - R.ctx];
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (work && warp == 4 * AT2_GROUPS + 1) {
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
  float v = -INFINITY;                              // (a weight of 0)
  if (rr < C.tpt * G && t < R.counted) {
    const int head = c * G + rr % G;
    const float2 mz = aw_merge(A.stats + ((size_t)(R.row0 + t) * A.Hq + head) * C.parts * 2, C.parts, A.sinks ? A.sinks + head : nullptr);
    if (mz.y != 0.f) v = log2f(mz.y) - mz.x;        // (a row that sees nothing gives nothing, one that sees a NaN gives NaN)
  }
  C.negl[((size_t)c * C.tiles + at2_tile0(R, r, C.tpt) + tile) * AT2_TILE + rr] = v;
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
  static unsigned long long configured = 0;
  const cudaError_t e = qe_once_a_device(configured, [&] {
    return cudaFuncSetAttribute(attention_weights_tc_kernel<PASS, GENERAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  });
  if (e != cudaSuccess) return e;
  return qe_launch(attention_weights_tc_kernel<PASS, GENERAL>, grid, dim3(AT2_THREADS), smem, stream, q, k, A, C);
}

// The requests of more than few_rows rows.  stats: [T Hq, parts1, 2] floats; merged: [Hkv, T / (128 / G) + R, 128]; sums:
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
  C.negl = merged;
  C.sums = parts2 > 1 ? sums : nullptr;
  C.sums_ld = max_total;
  AwArgs A{q, q_stride, T, pages, num_pages, planes, block_tables, max_blocks, cu_q, ctx_lens, slot_ids, counted, step_positions, positions,
           weights, out, slots, capacity, R, Hq, Hkv, D, page, aw_shift(page), window, scale, softcap, slopes, sinks, stats, parts1};
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
  const dim3 grid1((unsigned)((q_tiles + C.na - 1) / C.na * parts1 * Hkv), 1, (unsigned)R), grid2((unsigned)((k_tiles + C.na - 1) / C.na * parts2 * Hkv), 1, (unsigned)R);
  const bool general = softcap > 0.f || slopes != nullptr;
  C.parts = parts1;
  cudaError_t e = general ? at2_launch<1, true>(grid1, stream, map_q, map_k, A, C) : at2_launch<1, false>(grid1, stream, map_q, map_k, A, C);
  if (e == cudaSuccess) e = qe_launch(attention_weights_merge_kernel, dim3((unsigned)q_tiles, (unsigned)Hkv, (unsigned)R), dim3(AT2_TILE), 0, stream, A, C);
  C.parts = parts2;
  if (e == cudaSuccess) e = general ? at2_launch<2, true>(grid2, stream, map_q, map_k, A, C) : at2_launch<2, false>(grid2, stream, map_q, map_k, A, C);
  if (e == cudaSuccess && C.sums)
    e = aw_finish(A, C.sums, C.sums_ld, parts2, few_rows, max_total, stream);
  if (e != cudaSuccess) { qe_set_error("attention_weights: launch failed: %s", cudaGetErrorString(e)); (void)cudaGetLastError(); return 2; }
  QE_CHECK_LAUNCH("attention_weights");
  return 0;
}

// Attention of prompt portions over a 4-bit cache on the 5th-generation tensor cores, head sizes 64 and 128.  The pages that the
// portions see are expanded once, to float16 (attention_kv4.cu: kv4_pages_kernel), and this kernel reads those.
//
// Float16 and not bfloat16: a value s c + m has up to twelve bits, of which bfloat16 keeps eight; the rounded keys alone moved the
// outputs by 2.4 times their own rounding (2,048 tokens of 28 heads over 4: 3.8e-3 against 64 bits, 1.7e-3 now).  Its range is
// made enough by powers of two: keys, and values, of a (request, kv head) are divided by the one that brings the largest of them to 2^13..2^14
// (found on the device), a query row by its own that brings its largest to 1..2.  A value keeps eleven bits, or what lies over 2^-38 of
// that largest (float16's last step, 2^-24).  The factors meet again in the exponent's factor and behind the last division.
//
// The arrangement is near that of the framework's two-tile prompt kernel: a CTA owns two consecutive tiles of TOK = 128 / G tokens times
// the G heads of a group (rows r = token * G + head) and fetches every tile of 128 keys once for both.  Warp 0 fetches Q and
// the keys (two stages), warp 11 the values (one), a thread of warp 1 and one of warp 10 issue the MMAs of a tile each (S_A, S_B, O_A, O_B
// fill the 512 columns of tensor memory), warps 2..5 and 6..9 are the softmax of a tile, one thread per row; a row's
// probabilities go to shared memory as operand A of P V.  Its own are:
//  * the conversion of Q in place;
//  * turns: the tiles' exponentials alternate, so that one tile's run while the other's scores are fetched and its products
//    made (2,048 tokens of 28 heads over 4, the whole call: 60 us, 62 without; 384 after 8,191: 102, 109);
//  * two multiply-adds, or sums, an instruction (61 against 65 us);
//  * PARTS: where a step has few pairs of tiles and each sees many keys (a portion late in a long prompt), the key tiles of a pair
//    are cut into parts for a CTA each, which leave (reference, sum, accumulator) in the scratch for a kernel that joins them.
//    384 tokens after 8,191 beside 15 decoding requests, 28 heads over 4: 44 pairs on 148 SMs.
// Bound by a warp's chain: of the 4,100 cycles that a pair of key tiles takes, 2 x 1,480 are exponentials (2 x 1,024 the unit's own
// time), the products 2,048; before the first and after the last tile a CTA takes 5,400 and 6,000.
// Every wait is bounded: on expiry the kernel records a code in `status` and winds down.
#include <cuda_fp16.h>

#include <cfloat>

#include "tc_common.cuh"

#ifndef CO_HEAD_DIM
#define CO_HEAD_DIM 128
#endif

namespace {
typedef __nv_bfloat16 bf16;
constexpr int HD = CO_HEAD_DIM;
constexpr bool SUPPORTED = HD == 64 || HD == 128;
constexpr int BN = 128;                          // key positions per tile
constexpr int KCH = SUPPORTED ? HD / 64 : 1;     // 64-column chunks of the head dimension
constexpr int CHUNK_BYTES = 128 * 128;           // 128 rows of 128 bytes
constexpr int TILE_BYTES = KCH * CHUNK_BYTES;    // a tile of Q, K or V
constexpr int P_BYTES = 2 * CHUNK_BYTES;         // 128 rows x 128 float16
constexpr int K_STAGES = 2;
constexpr int SMEM_BYTES = 2 * TILE_BYTES + K_STAGES * TILE_BYTES + TILE_BYTES + 2 * P_BYTES + 1024 /* alignment slack */ + 256 /* barriers */;
static_assert(SMEM_BYTES <= 227 * 1024, "two query tiles, the stages and the probabilities fit shared memory");
constexpr unsigned FLOAT16 = ~((1u << 7) | (1u << 10));      // of an instruction descriptor: both operands float16, not bfloat16
// Probabilities are 2^LIFT times over their reference, which the maximum passes by 2^8 at most (2^15 at most enter the products): what
// float16 drops then lies under 2^-32 of a reference that the sum holds, where without it 131,072 keys of just under 2^-25 would be 0.4 % of the
// sum and nothing of the products.
constexpr float LIFT = 7.f;
constexpr int PART_FLOATS = 256 * (HD + 2);      // what a CTA of a part leaves: 256 rows, then their references and sums

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));   // ex2(-inf) = +0
  return y;
}
__device__ __forceinline__ unsigned pack_half(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&v);
}

// Shared memory by its own address: through a pointer, whose alignment by hand hides where it points, these become generic accesses.
__device__ __forceinline__ uint4 ld_shared(unsigned at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Two at a time: a b + c, a + b.
__device__ __forceinline__ unsigned long long pair_f32(unsigned lo, unsigned hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float2 of_pair(unsigned long long v) {
  unsigned lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
  return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}

struct Shape {
  int G, TOK, nkv, page_size, cache_rows, window, rows_per_box, n_req, pairs, parts, table_ld;
  float scale_log2;
};

constexpr int THREADS = 384;
__global__ void __launch_bounds__(THREADS, 1)
kv4_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  bf16* __restrict__ out, long out_stride, const int* __restrict__ block_tables, const int* __restrict__ cu_q,
                  const int* __restrict__ kv_lens, const float2* __restrict__ factors, Shape sh, float* __restrict__ scratch,
                  int* __restrict__ status) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* q_s = tiles;                                   // [tile][KCH][128 rows][128 B]
  unsigned char* k_s = q_s + 2 * TILE_BYTES;                    // [K_STAGES][KCH][128 rows][128 B]
  unsigned char* v_s = k_s + K_STAGES * TILE_BYTES;             // [KCH][128 rows][128 B]
  unsigned char* p_s = v_s + TILE_BYTES;                        // [tile][2][128 rows][128 B]
  unsigned long long* bars = (unsigned long long*)(p_s + 2 * P_BYTES);
  unsigned long long* q_full = bars;                // 1
  unsigned long long* q_ready = bars + 1;           // [tile] Q is float16 (one arrival per softmax warp)
  unsigned long long* k_full = q_ready + 2;         // [K_STAGES]
  unsigned long long* k_empty = k_full + K_STAGES;  // [K_STAGES] both tiles' Q K^T have read the stage
  unsigned long long* v_full = k_empty + K_STAGES;  // 1
  unsigned long long* v_empty = v_full + 1;         // 1: both tiles' P V have read the stage
  unsigned long long* s_full = v_empty + 1;         // [tile] MMA -> softmax: S is complete
  unsigned long long* s_free = s_full + 2;          // [tile] softmax -> MMA: S is in registers (one arrival per warp)
  unsigned long long* p_full = s_free + 2;          // [tile] softmax -> MMA: P written, O rescaled (one arrival per warp)
  unsigned long long* pv_done = p_full + 2;         // [tile] MMA -> softmax: O += P V is complete
  unsigned long long* turn = pv_done + 2;           // [tile][quarter] the other tile's warp is through with its exponentials
  unsigned* tmem_slot = (unsigned*)(turn + 8);
  static_assert((5 + 2 * K_STAGES + 16) * 8 + 4 <= 256, "barriers fit their slot");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1); mbar_init(v_full, 1); mbar_init(v_empty, 2);
    for (int s = 0; s < K_STAGES; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 2); }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_ready[t], 4); mbar_init(&s_full[t], 1); mbar_init(&s_free[t], 4); mbar_init(&p_full[t], 4); mbar_init(&pv_done[t], 1);
      for (int x = 0; x < 4; ++x) mbar_init(&turn[4 * t + x], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_base = *tmem_slot;
  co_pdl_launch_dependents();
  co_pdl_wait();

  // Late rows see the most keys: their pairs of tiles are started first, for all (request, kv head) before any earlier pair.
  const unsigned unit = blockIdx.x / (unsigned)sh.parts, request = unit / (unsigned)sh.nkv, late = request / (unsigned)sh.n_req;
  const int part = (int)(blockIdx.x - unit * sh.parts), kvh = (int)(unit - request * sh.nkv), b = (int)(request - late * sh.n_req);
  const int pair = sh.pairs - 1 - (int)late, G = sh.G, TOK = sh.TOK, RT = TOK * G;
  const int tok0 = cu_q[b], q_len = cu_q[b + 1] - tok0, kv_len = kv_lens[b];
  const int rows = q_len * G;
  const bool active_a = 2 * pair * RT < rows, active_b = (2 * pair + 1) * RT < rows;
  const int base_pos = kv_len - q_len;
  const int first_a = 2 * pair * RT, first_b = first_a + RT;
  const int token_a = 2 * pair * TOK, token_b = token_a + TOK;
  const int key_first = sh.window > 0 ? max(0, base_pos + token_a - sh.window + 1) : 0, tile_first = key_first / BN;
  const int pos_hi_a = base_pos + min(q_len, token_a + TOK) - 1, pos_hi_b = base_pos + min(q_len, token_b + TOK) - 1;      // (a request shorter than its rows: negative ones see nothing)
  const int all_a = active_a && pos_hi_a >= 0 ? pos_hi_a / BN - tile_first + 1 : 0;  // key tiles of tile A, of tile B
  const int all_b = active_b && pos_hi_b >= 0 ? pos_hi_b / BN - tile_first + 1 : 0;
  const int all = all_a > all_b ? all_a : all_b;
  const int j0 = (int)((long long)all * part / sh.parts), j1 = (int)((long long)all * (part + 1) / sh.parts);      // of this part
  const int n_a = max(0, min(all_a, j1) - j0), n_b = max(0, min(all_b, j1) - j0), n_tiles = n_b > n_a ? n_b : n_a;

  if (warp == 0 || warp == 11) {
    // Warp 0 fetches Q and the keys, warp 11 the values.
    if (n_tiles > 0) {
      if (warp == 0 && lane == 0) {
        mbar_expect_tx(q_full, (unsigned)(KCH * RT * 128 * (active_b ? 2 : 1)));
        for (int t = 0; t < (active_b ? 2 : 1); ++t)
          for (int c = 0; c < KCH; ++c)
            tma_load_3d(q_s + t * TILE_BYTES + c * CHUNK_BYTES, &map_q, c * 64, kvh * G, tok0 + (2 * pair + t) * TOK, q_full);
      }
      const int* table = block_tables + (size_t)b * sh.table_ld;
      const int boxes = BN / sh.rows_per_box;       // lane i < boxes fetches box i of every tile
      // The first row of this lane's box of key tile j in the expanded pages.  A page that is not there: a box beyond them,
      // fetched as zeros.
      auto box_row = [&](int j) {
        if (lane >= boxes || j >= n_tiles) return 0;
        const int pos = (tile_first + j0 + j) * BN + lane * sh.rows_per_box, blk = pos / sh.page_size;
        const int page = blk < sh.table_ld ? table[blk] : -1;
        return page >= 0 ? (page * sh.nkv + kvh) * sh.page_size + (pos - blk * sh.page_size) : sh.cache_rows;
      };
      auto fetch = [&](const CUtensorMap* map, unsigned char* dst, int row, unsigned long long* full) {
        if (lane == 0) mbar_expect_tx(full, (unsigned)TILE_BYTES);
        __syncwarp();
        if (lane < boxes)
          for (int c = 0; c < KCH; ++c) tma_load_2d(dst + c * CHUNK_BYTES + lane * sh.rows_per_box * 128, map, c * 64, row, full);
      };
      auto wait_for = [&](unsigned long long* bar, unsigned parity) {
        int ok = 1;
        if (lane == 0 && !mbar_wait(bar, parity)) { atomicExch(status, 31); ok = 0; }
        return __shfl_sync(0xffffffffu, ok, 0) != 0;
      };
      const bool keys = warp == 0;
      const int stages = keys ? K_STAGES : 1;
      int row = box_row(0);
      for (int i = 0; i < n_tiles; ++i) {
        const int row_next = box_row(i + 1), stage = i % stages;
        if (i >= stages && !wait_for(keys ? &k_empty[stage] : v_empty, (unsigned)(i / stages - 1) & 1)) break;
        if (keys) fetch(&map_k, k_s + (size_t)stage * TILE_BYTES, row, &k_full[stage]);
        else fetch(&map_v, v_s, row, v_full);
        row = row_next;
      }
    }
  } else if (warp == 1 || warp == 10) {
    // The MMAs of tile A, of tile B: neither waits for the other's softmax.
    if (lane == 0 && n_tiles > 0) {
      const int t = warp == 1 ? 0 : 1, mine = t ? n_b : n_a;
      constexpr unsigned idesc_qk = umma_idesc(128, BN) & FLOAT16;
      constexpr unsigned idesc_pv = umma_idesc_b_mn(128, HD) & FLOAT16;
      auto issue_qk = [&](int j) {        // S = Q K(j)^T; K(j) has landed and S is free
        const unsigned char* k_src = k_s + (size_t)(j % K_STAGES) * TILE_BYTES;
#pragma unroll
        for (int c = 0; c < KCH; ++c) {
          const unsigned long long dq = umma_desc(q_s + t * TILE_BYTES + c * CHUNK_BYTES), dk = umma_desc(k_src + c * CHUNK_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem_base + 128 * t, dq + 2 * k, dk + 2 * k, idesc_qk, (c | k) != 0);
        }
        umma_commit(&s_full[t]);
      };
      auto issue_pv = [&](int j) {        // O += P V(j); P and V(j) have been waited for
        const unsigned long long dv = umma_desc_offsets(v_s, CHUNK_BYTES, 1024);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk) {   // 16 positions: 32 bytes along a row of P (64 per chunk), 16 rows of V further
          const unsigned long long dp = umma_desc(p_s + t * P_BYTES + (kk >> 2) * CHUNK_BYTES) + 2 * (kk & 3);
          umma_bf16(tmem_base + 256 + 128 * t, dp, dv + (unsigned long long)(kk * 128), idesc_pv, (j | kk) != 0);
        }
        umma_commit(&pv_done[t]);
      };
      // Both issuers go through every stage, so that each of its barriers' phases has two arrivals, also where one has no more tiles.
      bool ok = mine == 0 || mbar_wait(&q_ready[t], 0);
      if (!ok) atomicExch(status, 32);
      if (ok && !mbar_wait(&k_full[0], 0)) { atomicExch(status, 33); ok = false; }
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (mine > 0) issue_qk(0);
        umma_commit(&k_empty[0]);
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        // The next scores first: they wait only for the softmax threads to hold S(j) in registers.
        if (j + 1 < n_tiles) {
          if (!mbar_wait(&k_full[(j + 1) % K_STAGES], (unsigned)((j + 1) / K_STAGES) & 1)) { atomicExch(status, 33); ok = false; break; }
          if (j + 1 < mine) {
            if (!mbar_wait(&s_free[t], (unsigned)j & 1)) { atomicExch(status, 34); ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            issue_qk(j + 1);
          }
          umma_commit(&k_empty[(j + 1) % K_STAGES]);
        }
        if (j < mine && !mbar_wait(&p_full[t], (unsigned)j & 1)) { atomicExch(status, 35); ok = false; break; }
        if (!mbar_wait(v_full, (unsigned)j & 1)) { atomicExch(status, 36); ok = false; break; }
        if (j < mine) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          issue_pv(j);
        }
        umma_commit(v_empty);
      }
    }
  } else {
    // Softmax warps: 2..5 for tile A, 6..9 for tile B; TMEM lane quarter = warp % 4; one thread per row.
    const int t = warp >= 6 ? 1 : 0;
    const int quarter = warp & 3;
    const int my_tiles = t ? n_b : n_a;
    const bool active = t ? active_b : active_a;
    const int row = quarter * 32 + lane;
    const int row_first = t ? first_b : first_a;
    const bool valid = active && row < RT && row_first + row < rows;
    float m = -INFINITY, l = 0.f, row_scale = 0.f;
    bool ok = true;
    const unsigned lane_addr = tmem_base + ((unsigned)(quarter * 32) << 16);
    const unsigned col_s = 128 * t, col_o = 256 + 128 * t;
    if (n_tiles > 0 && active) {
      // The row of Q to float16, its largest element brought to 1..2; the rows beyond the tile's whole tokens, which were not
      // fetched, to zeros, so that their scores are 0 and their threads walk the same path as the others.  Pieces in an order of
      // the row's own, so that the lanes do not meet in the same banks.
      if (!mbar_wait(q_full, 0)) { if (lane == 0) atomicExch(status, 37); ok = false; }
      const unsigned q_row = smem_u32(q_s + t * TILE_BYTES + row * 128);
      uint4 v[KCH][8];
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < KCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[c][i] = ld_shared(q_row + c * CHUNK_BYTES + ((i ^ (row & 7)) << 4));
          const unsigned w[4] = {v[c][i].x, v[c][i].y, v[c][i].z, v[c][i].w};
#pragma unroll
          for (int x = 0; x < 4; ++x) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[x] << 16)), fabsf(__uint_as_float(w[x] & 0xffff0000u))));
        }
      const int e = min(max((int)(__float_as_uint(most) >> 23), 1), 253);          // 2^(e - 127) <= most
      const float down = __uint_as_float((unsigned)(254 - e) << 23);
      // A normal number: a factor of zero (a row of zeros over small keys), or one that is not finite, would turn the masked scores' -inf, or a
      // score of zero, into not-a-number.  Scores that meet either bound are zero to working precision, or beyond float32.  The powers of
      // two first, whose product is exact where the factor is normal.
      row_scale = fminf(fmaxf(factors[b * sh.nkv + kvh].x * __uint_as_float((unsigned)e << 23) * sh.scale_log2, FLT_MIN), FLT_MAX);
#pragma unroll
      for (int c = 0; c < KCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          unsigned w[4] = {v[c][i].x, v[c][i].y, v[c][i].z, v[c][i].w};
#pragma unroll
          for (int x = 0; x < 4; ++x)
            w[x] = row < RT ? pack_half(__uint_as_float(w[x] << 16) * down, __uint_as_float(w[x] & 0xffff0000u) * down) : 0u;
          st_shared(q_row + c * CHUNK_BYTES + ((i ^ (row & 7)) << 4), w[0], w[1], w[2], w[3]);
        }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[t]);
    }
    if (my_tiles > 0) {
      const unsigned p_row = smem_u32(p_s + t * P_BYTES + row * 128);
      // Rows that are not kept see everything, so that they take no part in the choice of the path below.
      const int pos = base_pos + (row_first + row) / G;
      const int hi = valid ? pos : 0x7fffffff;
      const int lo = valid && sh.window > 0 ? max(0, pos - sh.window + 1) : 0;
      for (int j = 0; j < my_tiles && ok; ++j) {
        if (!mbar_wait(&s_full[t], (unsigned)j & 1)) { if (lane == 0) atomicExch(status, 37); ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        unsigned sr[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nowait(lane_addr + col_s + 32 * i, sr[i]);
        tmem_wait_ld();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[t]);
        const int key0 = (tile_first + j0 + j) * BN;
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const int hi_col = hi - key0, lo_col = lo - key0;        // columns lo_col..hi_col are seen
        if (!__all_sync(0xffffffffu, hi_col >= BN - 1 && lo_col <= 0)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (i * 32 + c > hi_col) sr[i][c] = __float_as_uint(-INFINITY);
          if (sh.window > 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (i * 32 + c < lo_col) sr[i][c] = __float_as_uint(-INFINITY);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 32; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], __uint_as_float(sr[i][c]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        // The reference m follows the running maximum lazily (p stays below 2^(8 + LIFT), inside float16's range), and the warp
        // decides together, because rescaling O is a warp-wide access to tensor memory.
        const float m_row = fmaxf(m, mx * row_scale);            // scale > 0 keeps the order
        const bool move = m == -INFINITY ? m_row != -INFINITY : m_row - m > 8.0f;
        const bool moved = __any_sync(0xffffffffu, move);
        const float m_new = moved ? m_row : m;
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float corr = ex2_approx(m - m_use);
        if (j > 0) {
          // P V(j - 1) has read the P tile that is about to be overwritten, and O is whole again
          if (!mbar_wait(&pv_done[t], (unsigned)(j - 1) & 1)) { if (lane == 0) atomicExch(status, 38); ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (moved) {
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
              unsigned o[32];
              tmem_ld32(lane_addr + col_o + c0, o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
              tmem_st32(lane_addr + col_o + c0, o);
            }
            tmem_wait_st();
          }
        }
        // The tiles' warps of an SM's quarter take turns at the exponentials, A(j) B(j) A(j + 1) ..: together they would wait together, too.
        const int before = t ? j : j - 1;            // the other tile's step whose exponentials come before these
        if (before >= 0 && before < (t ? n_a : n_b) && !mbar_wait(&turn[4 * t + quarter], (unsigned)before & 1)) {
          if (lane == 0) atomicExch(status, 38);
          ok = false;
          break;
        }
        // Exponentials, 32 columns at a time, each group packed and stored at once: row `row` of chunk i / 2 of the P tile,
        // 16-byte piece c at c ^ (row % 8).
        const unsigned scale_bits = __float_as_uint(row_scale), use_bits = __float_as_uint(LIFT - m_use);
        const unsigned long long scale2 = pair_f32(scale_bits, scale_bits), use2 = pair_f32(use_bits, use_bits);
        unsigned long long sum2[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unsigned pr[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 x = of_pair(fma2(pair_f32(sr[i][2 * c], sr[i][2 * c + 1]), scale2, use2));
            const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
            sum2[c & 3] = add2(sum2[c & 3], pair_f32(__float_as_uint(p0), __float_as_uint(p1)));
            pr[c] = pack_half(p0, p1);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
            st_shared(p_row + (i >> 1) * CHUNK_BYTES + ((((i & 1) * 4 + c) ^ (row & 7)) << 4), pr[4 * c], pr[4 * c + 1], pr[4 * c + 2], pr[4 * c + 3]);
        }
        if (lane == 0) mbar_arrive(&turn[4 * (1 - t) + quarter]);
        const float2 all = of_pair(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])));
        l = l * corr + (all.x + all.y);
        m = m_new;
        fence_proxy_async();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (ok) {
        if (!mbar_wait(&pv_done[t], (unsigned)(my_tiles - 1) & 1)) { if (lane == 0) atomicExch(status, 39); ok = false; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
    }
    if (active && ok) {
      // Rows leave by way of the tile's probabilities' place, 64 columns at a time: written by a thread a row each, every store to memory
      // would meet 32 rows (9,500 cycles a CTA instead of 6,000).
      // The sum first, then the values' factor (for parts: behind the join), so that neither passes the range of float32 before the answer does.
      const float v_factor = sh.parts > 1 ? 1.f : factors[b * sh.nkv + kvh].y;
      const float inv = sh.parts > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      if (sh.parts > 1 && valid)
        *reinterpret_cast<float2*>(scratch + (size_t)blockIdx.x * PART_FLOATS + 256 * HD + (t * 128 + row) * 2) = make_float2(m, l);
      const int token = (row_first + row) / G;
      const long long place = !valid ? -1
                              : sh.parts > 1 ? (long long)blockIdx.x * PART_FLOATS + (t * 128 + row) * HD
                                             : (long long)(tok0 + token) * out_stride + (kvh * G + row_first + row - token * G) * HD;
      const unsigned stage = smem_u32(p_s + t * P_BYTES);
#pragma unroll 1
      for (int c0 = 0; c0 < HD; c0 += 64) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unsigned o[32];
          if (my_tiles > 0) {
            tmem_ld32(lane_addr + col_o + c0 + 32 * h, o);     // warp-collective
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = 0;
          }
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * inv * v_factor);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            st_shared(stage + row * 256 + (((h * 8 + c) ^ (row & 7)) << 4), o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        }
        __syncwarp();
        const int piece = lane & 15;
        uint4 v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = quarter * 32 + 2 * i + (lane >> 4);
          v[i] = ld_shared(stage + r * 256 + ((piece ^ (r & 7)) << 4));
        }
        if (sh.parts > 1) {
          float* to = scratch + c0 + piece * 4;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const long long at = __shfl_sync(0xffffffffu, place, 2 * i + (lane >> 4));
            if (at >= 0) *reinterpret_cast<uint4*>(to + at) = v[i];
          }
        } else {
          bf16* to = out + c0 + piece * 4;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const long long at = __shfl_sync(0xffffffffu, place, 2 * i + (lane >> 4));
            const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(v[i].x), __uint_as_float(v[i].y));
            const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(v[i].z), __uint_as_float(v[i].w));
            if (at >= 0) *reinterpret_cast<uint2*>(to + at) = make_uint2(*reinterpret_cast<const unsigned*>(&x), *reinterpret_cast<const unsigned*>(&y));
          }
        }
        __syncwarp();
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(512) : "memory");
  }
}

// Joins the parts of every row, a warp per row, parts in ascending order.  Bound by what the parts left (3 parts of 10,752 rows: 17 MB).
__global__ void __launch_bounds__(256)
kv4_prompt_join_kernel(const float* __restrict__ scratch, bf16* __restrict__ out, long out_stride, const int* __restrict__ cu_q,
                       const float2* __restrict__ factors, Shape sh) {
  constexpr int C = SUPPORTED ? HD / 32 : 2;         // neighbouring columns per lane: 2 or 4
  co_pdl_launch_dependents();
  const int rr = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, kvh = blockIdx.y, b = blockIdx.z, G = sh.G, RT = sh.TOK * G;
  co_pdl_wait();
  const int tok0 = cu_q[b], rows = (cu_q[b + 1] - tok0) * G;
  if (rr >= rows) return;
  const int pair = rr / (2 * RT), in = rr - pair * 2 * RT, row = in < RT ? in : 128 + in - RT;
  const int unit = (sh.pairs - 1 - pair) * sh.nkv * sh.n_req + b * sh.nkv + kvh;
  const float* base = scratch + (size_t)unit * sh.parts * PART_FLOATS;
  float M = -INFINITY, den = 0.f, acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  // The reference may still move: what has been added up is scaled when it does.
#pragma unroll 4
  for (int p = 0; p < sh.parts; ++p) {
    const float* src = base + (size_t)p * PART_FLOATS;
    const float2 ml = *reinterpret_cast<const float2*>(src + 256 * HD + row * 2);
    float x[C];
    if constexpr (C == 4) {
      const float4 v = *reinterpret_cast<const float4*>(src + row * HD + lane * 4);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(src + row * HD + lane * 2);
      x[0] = v.x; x[1] = v.y;
    }
    const float N = fmaxf(M, ml.x), f = M == -INFINITY ? 0.f : exp2f(M - N), g = ml.x == -INFINITY ? 0.f : exp2f(ml.x - N);
    M = N;
    den = den * f + ml.y * g;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = acc[c] * f + x[c] * g;
  }
  const float inv = den == 0.f ? 0.f : 1.f / den, v_factor = factors[b * sh.nkv + kvh].y;
  bf16* dst = out + (size_t)(tok0 + rr / G) * out_stride + (size_t)(kvh * G + rr % G) * HD + lane * C;
  unsigned w[C / 2];
#pragma unroll
  for (int c = 0; c < C / 2; ++c) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(acc[2 * c] * inv * v_factor, acc[2 * c + 1] * inv * v_factor);
    w[c] = *reinterpret_cast<const unsigned*>(&v);
  }
  if constexpr (C == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<unsigned*>(dst) = w[0];
}

int pairs_of(int nh, int nkv, int max_rows) {
  const int G = nh / nkv, RT = 128 / G * G;
  return (max_rows + 2 * RT - 1) / (2 * RT);
}
}  // namespace

// Whether the kernel takes this head grouping and page size at the compiled head size.
CO_EXPORT int coheryn_kv4_prompt_takes(int nh, int nkv, int page_size) {
  return SUPPORTED && nkv > 0 && nh % nkv == 0 && nh / nkv <= 128 && page_size >= 16 && (BN % page_size == 0 || page_size % BN == 0);
}

// Into how many parts the key tiles of a pair of row tiles are cut: as many as fill the SMs, of eight tiles at least.  tokens: of the n requests.
CO_EXPORT int coheryn_kv4_prompt_parts(int nh, int nkv, int n, int tokens, int max_rows, int max_kv_len, int window) {
  const int G = nh / nkv, RT = 128 / G * G;
  const long most = ((long)tokens * G + 2 * RT - 1) / (2 * RT) + n - 1, grid = (long)pairs_of(nh, nkv, max_rows) * n;
  const long units = nkv * (grid < most ? grid : most);
  const long keys = window > 0 && window + max_rows / G < max_kv_len ? window + max_rows / G : max_kv_len;
  long parts = 148 / (units < 1 ? 1 : units);
  if (parts > (keys + BN - 1) / BN / 8) parts = (keys + BN - 1) / BN / 8;
  return parts < 1 ? 1 : parts > 32 ? 32 : (int)parts;
}
CO_EXPORT long coheryn_kv4_prompt_scratch_floats(int nh, int nkv, int n, int max_rows, int parts) {
  return parts > 1 ? (long)pairs_of(nh, nkv, max_rows) * n * nkv * parts * PART_FLOATS : 0;
}

// q: [total_tokens, >= nh * HD] bfloat16 rows of stride q_stride; k, v: float16 pages [num_pages, nkv, page_size, HD], and the factors [n, nkv, 2]
// that multiply them back (device); requests 0..n-1 all go through this kernel.
CO_EXPORT int coheryn_kv4_prompt(const void* q, long q_stride, int total_tokens, void* out, long out_stride, const void* k, const void* v, int num_pages,
                                 const int* block_tables, int table_ld, const int* cu_q, const int* kv_lens, int n, int nh, int nkv, int page_size,
                                 int window, float scale, int max_rows, const float* factors, int parts, float* scratch, long scratch_floats,
                                 int* status, cudaStream_t stream) {
  if (!coheryn_kv4_prompt_takes(nh, nkv, page_size)) CO_FAIL("kv4_prompt: head size %d, %d heads over %d, pages of %d", HD, nh, nkv, page_size);
  if (n <= 0 || max_rows <= 0) return 0;
  if (!(scale > 0.f)) CO_FAIL("kv4_prompt: the scale must be positive");
  const long cache_rows = (long)num_pages * nkv * page_size;
  const long ctas = (long)pairs_of(nh, nkv, max_rows) * n * nkv * parts;
  if (cache_rows >= (1L << 31) || ctas >= (1L << 31) || n > 65535 || nkv > 65535) CO_FAIL("kv4_prompt: %ld rows of pages, %ld CTAs", cache_rows, ctas);
  if ((uintptr_t)factors & 7) CO_FAIL("kv4_prompt: the factors must be 8-byte aligned");
  if (parts < 1 || scratch_floats < coheryn_kv4_prompt_scratch_floats(nh, nkv, n, max_rows, parts) || ((uintptr_t)scratch & 15))
    CO_FAIL("kv4_prompt: %d parts in a scratch of %ld floats", parts, scratch_floats);
  const int G = nh / nkv, TOK = 128 / G;
  const Shape sh{G, TOK, nkv, page_size, (int)cache_rows, window, page_size >= BN ? BN : page_size, n, pairs_of(nh, nkv, max_rows), parts, table_ld,
                 scale * 1.4426950408889634f};
  CUtensorMap mq, mk, mv;
  {
    cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)nh, (cuuint64_t)total_tokens};
    cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)TOK};
    if (!make_map_nd(&mq, q, 3, dims, strides, box)) CO_FAIL("kv4_prompt: the query tensor map was refused");
  }
  for (auto x : {&mk, &mv}) {
    cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)cache_rows};
    cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)sh.rows_per_box};
    if (!make_map_nd(x, x == &mk ? k : v, 2, dims, strides, box)) CO_FAIL("kv4_prompt: the tensor map of the pages was refused");
  }
  cudaError_t e = cudaFuncSetAttribute(kv4_prompt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
  if (e != cudaSuccess) CO_FAIL("kv4_prompt: %d bytes of shared memory: %s", SMEM_BYTES, cudaGetErrorString(e));
  co_launch(kv4_prompt_kernel, dim3((unsigned)ctas), dim3(THREADS), (size_t)SMEM_BYTES, stream, mq, mk, mv, (bf16*)out, out_stride, block_tables, cu_q, kv_lens,
            (const float2*)factors, sh, scratch, status);
  CO_CHECK_LAUNCH("kv4_prompt");
  if (parts > 1) {
    co_launch(kv4_prompt_join_kernel, dim3((unsigned)((max_rows + 7) / 8), (unsigned)nkv, (unsigned)n), dim3(256), 0, stream, (const float*)scratch,
              (bf16*)out, out_stride, cu_q, (const float2*)factors, sh);
    CO_CHECK_LAUNCH("kv4_prompt_join");
  }
  return 0;
}

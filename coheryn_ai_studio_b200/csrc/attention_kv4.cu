// Keys and values held in 4 bits, and the attention over their pages; compiled for one head size (CO_HEAD_DIM, a
// multiple of 32 up to 256).
//
// A row's channels are taken in groups of 32.  A group of values x has, in bfloat16,
//   minimum m = min(x),   scale s = (max(x) - min(x)) / 15   (float32 arithmetic, then rounded),
// and per channel a code c = clamp(rint((x - m) / s), 0, 15); it stands for s c + m, at most s / 2 (and the rounding of
// s and m) from x.  A group that is constant has s = 0.  A group that holds a value that is not finite has s and m not
// a number.  5 bits a value with the pairs: 3.2 times as many positions as bfloat16 in the same memory.
//
// A page keeps, per kv head, page_size / 16 tiles of 16 positions; a tile is TB = 10 HD bytes, codes first, pairs behind.
// Both tiles lie as the fragments of mma.sync.m16n8k16 want them, so that a lane's codes and pairs come by loads of 8
// and 16 bytes that no two lanes contend for and no code has to change its lane (lane = 4 g + t):
//  * keys: rows of HD / 2 bytes; word t NG + u of a row (NG = HD / 32) holds channels 32 u + 8 t + 0..7, lowest bits
//    first; then 16 rows of NG pairs (s low half, m high half).
//  * values: for group u, lane (g, t), p = 0, 1 a word: low half row 4 t + 2 p, high half row 4 t + 2 p + 1, each
//    channels 32 u + 4 g + 0..3; then for (u, t) the scales of rows 4 t..4 t + 3 and their minima.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "tc_common.cuh"

#ifndef CO_HEAD_DIM
#define CO_HEAD_DIM 128
#endif

namespace {
typedef __nv_bfloat16 bf16;
constexpr int HD = CO_HEAD_DIM;
constexpr int NG = HD / 32;           // groups of a row
constexpr int TB = 10 * HD;           // bytes of a tile
constexpr int CODES = 8 * HD;         // of which codes
static_assert(HD % 32 == 0 && HD >= 32 && HD <= 256, "head size must be a multiple of 32 in 32..256");

constexpr int BAD_INDEX = 41;         // status: a slot, a position or a block-table entry lies outside its table

__device__ __forceinline__ float lo_bf16(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf16(unsigned w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ unsigned bits(__nv_bfloat162 v) { return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ unsigned bits(__half2 v) { return *reinterpret_cast<unsigned*>(&v); }
__device__ __forceinline__ __half2 half_pair(unsigned w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ unsigned pack(float a, float b) { return bits(__floats2bfloat162_rn(a, b)); }
__device__ __forceinline__ unsigned pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&v);
}

// The start of the tile that holds row `row` of a page.
__device__ __forceinline__ size_t tile_at(long long page, int nkv, int kvh, int page_size, int row) {
  return (((size_t)page * nkv + kvh) * (page_size >> 4) + (row >> 4)) * TB;
}

// ------------------------------------------------------------------------------------
// Rotation and write.  Queries are rotated into their own rows; keys are rotated and rounded to the compute type, as a cache in
// that type would hold them, and then quantised, values quantised as they are.  Every product and sum of the rotation is rounded
// by itself (no fused multiply-add): the codes are then the same function of the inputs wherever it is computed.
// Quotients are estimated by one reciprocal; only an estimate that lies within 2^-14 of a border between two codes is divided
// out, so that the code is that of the division.
//
// A thread has 4 neighbouring channels of each half of a head, which turn together: every element is read once, and the
// angles that a thread reads lie together with its neighbours' (8 neighbouring channels per thread, their partners read a
// second time and angles 64 bytes apart from lane to lane, took 23 us instead of 17 for 2,048 tokens of 28 + 8 heads of 128 and
// their pages read back: the loads' wavefronts bound it).  The eight threads of a group agree on its minimum and maximum by three shuffles.  Heads
// that turn another number of channels, or whose halves are not whole groups, go to the kernel after it.  Bound by
// the latency of its few loads and of the shuffles (half of the issue slots; 19 MB read and 17 MB written there), at decoding by one launch.
// ------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<bf16>(const bf16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = lo_bf16(w[i]); x[2 * i + 1] = hi_bf16(w[i]); }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<bf16>(bf16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack(x[0], x[1]), pack(x[2], x[3]), pack(x[4], x[5]), pack(x[6], x[7]));
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&x)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
}
template <>
__device__ __forceinline__ void load4<bf16>(const bf16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = lo_bf16(v.x); x[1] = hi_bf16(v.x); x[2] = lo_bf16(v.y); x[3] = hi_bf16(v.y);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <>
__device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
template <>
__device__ __forceinline__ void store4<bf16>(bf16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack(a, b), pack(c, d));
}
// N values rounded to the compute type.
template <int N>
__device__ __forceinline__ void rounded(float (&)[N], const float*) {}
template <int N>
__device__ __forceinline__ void rounded(float (&x)[N], const bf16*) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const unsigned w = pack(x[i], x[i + 1]);
    x[i] = lo_bf16(w);
    x[i + 1] = hi_bf16(w);
  }
}
// The pair (scale low half, minimum high half) of a group and the codes of this thread's N values of it, the first lowest.  The group's
// threads are neighbours, THREADS of them, and come here together.
template <int THREADS, int N>
__device__ __forceinline__ uint2 quantised(const float (&x)[N]) {
  float lo = x[0], hi = x[0];
  bool finite = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite = finite && fabsf(x[i]) < INFINITY;
  }
  const unsigned group = ((1u << THREADS) - 1) << (threadIdx.x & 31 & ~(THREADS - 1));
#pragma unroll
  for (int o = 1; o < THREADS; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(group, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(group, hi, o));
  }
  finite = __all_sync(group, finite);
  bf16 s16 = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), m16 = __float2bfloat16_rn(lo);
  float s = __bfloat162float(s16), m = __bfloat162float(m16);
  if (!(finite && fabsf(s) < INFINITY && fabsf(m) < INFINITY)) {
    s16 = m16 = __ushort_as_bfloat16(0x7fff);
    s = 0.f;
  }
  unsigned codes = 0;
  if (s > 0.f) {
    const float inverse = 1.f / s;
    const bool usual = inverse < 1e37f;                 // (a subnormal scale has no reciprocal)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = __fsub_rn(x[i], m);
      float c = d * inverse;
      if (!usual || fabsf(c - floorf(c) - 0.5f) < 6.1e-5f) c = __fdiv_rn(d, s);
      codes |= (unsigned)fminf(fmaxf(rintf(c), 0.f), 15.f) << (4 * i);
    }
  }
  return make_uint2((unsigned)__bfloat16_as_ushort(s16) | (unsigned)__bfloat16_as_ushort(m16) << 16, codes);
}
// Where the codes of channels 32 u + 4 i + 0..3 of row r lie in a key and in a value tile, in 16 bits; and the pairs.
__device__ __forceinline__ unsigned short* key_codes(unsigned char* tile, int r, int u, int i) {
  return reinterpret_cast<unsigned short*>(tile) + 2 * (r * (4 * NG) + (i >> 1) * NG + u) + (i & 1);
}
__device__ __forceinline__ unsigned short* value_codes(unsigned char* tile, int r, int u, int i) {
  return reinterpret_cast<unsigned short*>(tile) + 2 * (((u * 8 + i) * 4 + (r >> 2)) * 2 + ((r >> 1) & 1)) + (r & 1);
}
__device__ __forceinline__ void put_pair(unsigned char* tile, bool values, int r, int u, unsigned pair) {
  if (values) {
    unsigned short* at = reinterpret_cast<unsigned short*>(tile + CODES) + (u * 4 + (r >> 2)) * 8 + (r & 3);
    at[0] = (unsigned short)pair;
    at[4] = (unsigned short)(pair >> 16);
  } else {
    reinterpret_cast<unsigned*>(tile + CODES)[r * NG + u] = pair;
  }
}

// Rotations of whole heads (TURN) and no rotation, heads whose halves are whole groups.
template <typename T, bool TURN>
__global__ void __launch_bounds__(256, 8)
kv4_write_halves_kernel(const T* __restrict__ qkv, long ld, const int* __restrict__ positions, const float2* __restrict__ cos_sin, int n_cos,
                        const int* __restrict__ slots, unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache, int num_pages,
                        T* __restrict__ q_out, int nh, int nkv, int page_size, int first_head, int* __restrict__ status) {
  constexpr int TPH = HD / 8, AT_ONCE = 256 / TPH, HALF = HD / 2;      // threads of a head, heads of a block
  co_pdl_launch_dependents();
  const int place = threadIdx.x / TPH, piece = threadIdx.x % TPH, head = first_head + blockIdx.y * AT_ONCE + place;
  if (place >= AT_ONCE || head >= nh + 2 * nkv) return;
  const int token = blockIdx.x, c0 = piece * 4;
  co_pdl_wait();
  const T* src = qkv + (size_t)token * ld + (size_t)head * HD + c0;
  float x[2][4];
  load4(src, x[0]);
  load4(src + HALF, x[1]);
  const bool values = head >= nh + nkv;
  const int slot = head >= nh ? slots[token] : 0;
  if (TURN && !values) {
    const int pos = positions[token];
    if (pos < 0 || pos >= n_cos) {
      if (status) *status = BAD_INDEX;
    } else {
      const float4* turn = reinterpret_cast<const float4*>(cos_sin + (size_t)pos * HALF + c0);
      const float4 a = turn[0], b = turn[1];
      const float cs[4] = {a.x, a.z, b.x, b.z}, sn[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float l = __fsub_rn(__fmul_rn(x[0][i], cs[i]), __fmul_rn(x[1][i], sn[i]));
        x[1][i] = __fadd_rn(__fmul_rn(x[1][i], cs[i]), __fmul_rn(x[0][i], sn[i]));
        x[0][i] = l;
      }
    }
  }
  if (head < nh) {
    T* dst = q_out + (size_t)token * nh * HD + (size_t)head * HD + c0;
    store4(dst, x[0][0], x[0][1], x[0][2], x[0][3]);
    store4(dst + HALF, x[1][0], x[1][1], x[1][2], x[1][3]);
    return;
  }
  if (slot < 0) return;                                 // a row that is not kept
  const int page = slot / page_size, row = slot - page * page_size, r = row & 15;
  if (page >= num_pages) {
    if (status) *status = BAD_INDEX;
    return;
  }
  unsigned char* tile = (values ? v_cache : k_cache) + tile_at(page, nkv, head - nh - (values ? nkv : 0), page_size, row);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int u = (h * HALF + c0) / 32, i = piece & 7;
    rounded(x[h], (const T*)nullptr);
    const uint2 q = quantised<8>(x[h]);
    *(values ? value_codes(tile, r, u, i) : key_codes(tile, r, u, i)) = (unsigned short)q.y;
    if (i == 0) put_pair(tile, values, r, u, q.x);
  }
}

// Any even number of turned channels, any head: a thread has 8 neighbouring channels.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_write_kernel(const T* __restrict__ qkv, long ld, const int* __restrict__ positions, const float2* __restrict__ cos_sin, int n_cos,
                 const int* __restrict__ slots, unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache, int num_pages,
                 T* __restrict__ q_out, int nh, int nkv, int rot, int page_size, int first_head, int* __restrict__ status) {
  constexpr int TPH = HD / 8, AT_ONCE = 256 / TPH;
  co_pdl_launch_dependents();
  const int place = threadIdx.x / TPH, piece = threadIdx.x % TPH, head = first_head + blockIdx.y * AT_ONCE + place;
  if (place >= AT_ONCE || head >= nh + 2 * nkv) return;
  const int token = blockIdx.x, c0 = piece * 8, half = rot >> 1;
  co_pdl_wait();
  const T* src = qkv + (size_t)token * ld + (size_t)head * HD;
  float x[8];
  load8(src + c0, x);
  const bool values = head >= nh + nkv;
  if (c0 < rot && !values) {
    const int pos = positions[token];
    if (pos < 0 || pos >= n_cos) {
      if (status) *status = BAD_INDEX;
    } else {
      const float2* angles = cos_sin + (size_t)pos * half;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + i;
        if (c >= rot) continue;
        const bool upper = c >= half;
        const float2 a = angles[upper ? c - half : c];
        x[i] = __fadd_rn(__fmul_rn(x[i], a.x), __fmul_rn(co_to_float<T>(src[upper ? c - half : c + half]), upper ? a.y : -a.y));
      }
    }
  }
  if (head < nh) {
    store8(q_out + (size_t)token * nh * HD + (size_t)head * HD + c0, x);
    return;
  }
  const int slot = slots[token];
  if (slot < 0) return;
  const int page = slot / page_size, row = slot - page * page_size, r = row & 15, u = piece >> 2, t = piece & 3;
  if (page >= num_pages) {
    if (status) *status = BAD_INDEX;
    return;
  }
  unsigned char* tile = (values ? v_cache : k_cache) + tile_at(page, nkv, head - nh - (values ? nkv : 0), page_size, row);
  rounded(x, (const T*)nullptr);
  const uint2 q = quantised<4>(x);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *(values ? value_codes(tile, r, u, 2 * t + i) : key_codes(tile, r, u, 2 * t + i)) = (unsigned short)(q.y >> (16 * i));
  if (t == 0) put_pair(tile, values, r, u, q.x);
}

// ------------------------------------------------------------------------------------
// Pages as values: [entry, kv head, page_size, HD] in float32, bfloat16, or scaled float16 (for attention_kv4_prompt.cu).  One block per (page, kv head).
// With `lens` the entries are rows of a block table (request = blockIdx.z): rows at or behind the request's length, or in front of the
// window of its first new token, are zeros (whatever they hold, it meets probabilities of zero), entries that lie wholly there are left out, and
// `out_table` gets the entry's place among the output pages, or -1.
// Bound by the bytes written (16 of 21 bits a value).
// ------------------------------------------------------------------------------------
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store4<__half>(__half* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_f16(a, b), pack_f16(c, d));
}
// The rows [lo, hi) of entry j of request b's block table that its new tokens see (hi = 0: the entry is not needed).
struct Seen { int lo, hi; };
__device__ __forceinline__ Seen rows_seen(const int* cu_q, const int* lens, int b, int j, int page_size, int window) {
  const int len = lens[b], first_new = len - (cu_q[b + 1] - cu_q[b]);
  const int first_key = window > 0 ? max(0, first_new - window + 1) : 0;
  const int lo = max(0, first_key - j * page_size), hi = min(page_size, len - j * page_size);
  return hi > lo ? Seen{lo, hi} : Seen{0, 0};
}

// The largest magnitude among the keys, and among the values, that a request's new tokens see of a kv head, from the pairs alone (a group's
// values lie between m and m + 15 s): `parts` partial answers per list (request, kv head), so that a list's factors, and with them its
// rows' rounding, do not depend on what others hold.  A fifth of the pages' bytes; bound by a warp's chain of reads, an entry after
// the other, so as many warps as an SM holds (384 tokens after 8,191 beside 15 requests, the whole call: 99 us, 102 with 8 warps a block).
constexpr int RANGE_BLOCKS = 128, RANGE_WARPS = 32;
int range_parts(long long lists) { return lists < RANGE_BLOCKS ? (int)(RANGE_BLOCKS / (lists < 1 ? 1 : lists)) : 1; }
__global__ void __launch_bounds__(32 * RANGE_WARPS)
kv4_range_kernel(const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache, int num_pages, int nkv, int page_size,
                 const int* __restrict__ table, int table_ld, int width, const int* __restrict__ cu_q, const int* __restrict__ lens, int window,
                 int parts, float2* __restrict__ partial) {
  __shared__ float2 most[RANGE_WARPS];
  co_pdl_launch_dependents();
  co_pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_page = page_size >> 4;
  const int list = blockIdx.x / parts, part = blockIdx.x - list * parts, b = list / nkv, kvh = list - b * nkv;
  float k_most = 0.f, v_most = 0.f;
  // A warp takes an entry at a time.
  for (int j = part * RANGE_WARPS + warp; j < width; j += parts * RANGE_WARPS) {
    const int page = table[(size_t)b * table_ld + j];                                   // (asked for at once with the lengths)
    const Seen rows = rows_seen(cu_q, lens, b, j, page_size, window);
    if (rows.hi == 0 || page < 0 || page >= num_pages) continue;
    for (int tile = rows.lo >> 4; tile < per_page && tile * 16 < rows.hi; ++tile) {
      const size_t at = tile_at(page, nkv, kvh, page_size, tile * 16) + CODES;
      for (int i = lane; i < 16 * NG; i += 32) {         // keys: row i / NG
        const unsigned w = reinterpret_cast<const unsigned*>(k_cache + at)[i];
        const float m = hi_bf16(w);
        const int r = tile * 16 + i / NG;
        if (r >= rows.lo && r < rows.hi) k_most = fmaxf(k_most, fmaxf(fabsf(m), fabsf(fmaf(15.f, lo_bf16(w), m))));
      }
      for (int i = lane; i < 4 * NG; i += 32) {          // values: rows 4 (i % 4)..
        const uint4 w = reinterpret_cast<const uint4*>(v_cache + at)[i];
        const float sc[4] = {lo_bf16(w.x), hi_bf16(w.x), lo_bf16(w.y), hi_bf16(w.y)}, mn[4] = {lo_bf16(w.z), hi_bf16(w.z), lo_bf16(w.w), hi_bf16(w.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = tile * 16 + (i & 3) * 4 + e;
          if (r >= rows.lo && r < rows.hi) v_most = fmaxf(v_most, fmaxf(fabsf(mn[e]), fabsf(fmaf(15.f, sc[e], mn[e]))));
        }
      }
    }
  }
  k_most = co_warp_max(k_most);
  v_most = co_warp_max(v_most);
  if (lane == 0) most[warp] = make_float2(k_most, v_most);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < RANGE_WARPS; ++w) { k_most = fmaxf(k_most, most[w].x); v_most = fmaxf(v_most, most[w].y); }
    partial[blockIdx.x] = make_float2(k_most, v_most);
  }
}
// The power of two that brings a largest magnitude to 2^13..2^14, and its inverse; both are normal numbers for every finite one (magnitudes
// under 2^-113 are brought up by 2^126).  A group whose m + 15 s passes the largest float32 stands for an infinity there, here as well.
__device__ __forceinline__ float2 to_float16_range(float most) {
  const int e = min(max((int)(__float_as_uint(most) >> 23), 14), 254);
  return make_float2(__uint_as_float((unsigned)(267 - e) << 23), __uint_as_float((unsigned)(e - 13) << 23));
}

template <typename T>
__global__ void __launch_bounds__(128)
kv4_pages_kernel(const unsigned char* __restrict__ k_cache, const unsigned char* __restrict__ v_cache, int num_pages, int nkv, int page_size,
                 const int* __restrict__ table, int table_ld, int width, int slots, const int* __restrict__ cu_q, const int* __restrict__ lens, int window,
                 T* __restrict__ k_out, T* __restrict__ v_out, int* __restrict__ out_table, const float2* __restrict__ range, int range_parts,
                 float2* __restrict__ factors, int* __restrict__ status) {
  constexpr bool HALF = sizeof(T) == 2 && !std::is_same<T, bf16>::value;
  __shared__ float2 most[4];
  co_pdl_launch_dependents();
  co_pdl_wait();
  const int j = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  // The loads that depend on nothing first: a block lives for little more than its chain of them.
  const int page = table[(size_t)b * table_ld + j];
  Seen seen = lens ? rows_seen(cu_q, lens, b, j, page_size, window) : Seen{0, page_size};
  // A request's entries that are seen lie side by side: the first of them takes the first of its `slots` pages.
  const int slot = lens && window > 0 ? j - max(0, lens[b] - (cu_q[b + 1] - cu_q[b]) - window + 1) / page_size : j;
  const long long entry = (long long)b * slots + slot;
  int* place = out_table ? out_table + (size_t)b * width + j : nullptr;
  float k_by = 1.f, v_by = 1.f;
  if constexpr (HALF) {             // float16: times the powers of two that the largest values ask for
    static_assert(RANGE_BLOCKS <= 128, "a thread per partial answer of a list");
    const int list = b * nkv + kvh;
    const float2 x = (int)threadIdx.x < range_parts ? range[(size_t)list * range_parts + threadIdx.x] : make_float2(0.f, 0.f);
    const float kx = co_warp_max(x.x), vx = co_warp_max(x.y);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = make_float2(kx, vx);
    __syncthreads();
    const float2 k2 = to_float16_range(fmaxf(fmaxf(most[0].x, most[1].x), fmaxf(most[2].x, most[3].x)));
    const float2 v2 = to_float16_range(fmaxf(fmaxf(most[0].y, most[1].y), fmaxf(most[2].y, most[3].y)));
    k_by = k2.x;
    v_by = v2.x;
    if (j == 0 && threadIdx.x == 0) factors[list] = make_float2(k2.y, v2.y);
  }
  if (seen.hi == 0 || slot >= slots) {       // (more than there is room for: lengths that are not those the call was sized by)
    if (place && kvh == 0 && threadIdx.x == 0) *place = -1;
    if (seen.hi && status && threadIdx.x == 0) *status = BAD_INDEX;
    return;
  }
  const bool known = page >= 0 && page < num_pages;
  if (!known) seen.hi = 0;
  if (kvh == 0 && threadIdx.x == 0) {
    if (place) *place = known ? (int)entry : -1;
    if (status && (!known || (lens && lens[b] > width * page_size))) *status = BAD_INDEX;      // (or the table ends before the request)
  }
  T* ko = k_out + ((size_t)entry * nkv + kvh) * page_size * HD;
  T* vo = v_out + ((size_t)entry * nkv + kvh) * page_size * HD;
  for (int tile = 0; tile < page_size >> 4; ++tile) {
    const unsigned char* kt = k_cache + tile_at(known ? page : 0, nkv, kvh, page_size, tile * 16);
    const unsigned char* vt = v_cache + tile_at(known ? page : 0, nkv, kvh, page_size, tile * 16);
    for (int i = threadIdx.x; i < 16 * 4 * NG; i += 128) {
      const int r = i / (4 * NG), w = i % (4 * NG), u = w >> 2, t = w & 3;    // u, t: consecutive threads, consecutive channels
      float x[8];
      const bool keep = tile * 16 + r >= seen.lo && tile * 16 + r < seen.hi;
      const unsigned word = reinterpret_cast<const unsigned*>(kt)[r * (4 * NG) + t * NG + u];
      const unsigned sm = reinterpret_cast<const unsigned*>(kt + CODES)[r * NG + u];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float y = fmaf(lo_bf16(sm), (float)((word >> (4 * c)) & 15), hi_bf16(sm));
        x[c] = keep ? (HALF ? y * k_by : y) : 0.f;
      }
      store8(ko + (size_t)(tile * 16 + r) * HD + u * 32 + t * 8, x);
    }
    for (int i = threadIdx.x; i < 32 * NG; i += 128) {
      const int t = i / (8 * NG), w = i % (8 * NG), u = w >> 3, g = w & 7;
      const uint2 words = reinterpret_cast<const uint2*>(vt)[u * 32 + g * 4 + t];
      const uint4 sm = reinterpret_cast<const uint4*>(vt + CODES)[u * 4 + t];
      const float sc[4] = {lo_bf16(sm.x), hi_bf16(sm.x), lo_bf16(sm.y), hi_bf16(sm.y)};
      const float mn[4] = {lo_bf16(sm.z), hi_bf16(sm.z), lo_bf16(sm.w), hi_bf16(sm.w)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = tile * 16 + 4 * t + e;
        const unsigned h = (e < 2 ? words.x : words.y) >> (16 * (e & 1));
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float y = fmaf(sc[e], (float)((h >> (4 * c)) & 15), mn[e]);
          x[c] = r >= seen.lo && r < seen.hi ? (HALF ? y * v_by : y) : 0.f;
        }
        store4(vo + (size_t)r * HD + u * 32 + g * 4, x[0], x[1], x[2], x[3]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------
// How the keys of a step are cut.  The visible positions of a request (from the 16 that hold the first one on) are
// counted in units of UNIT positions, of which every list (request, kv head, tile of query rows) has the same number.  All
// units of the step, list after list, are cut into equal shares, one per CTA, from the lengths on the device: a long
// context beside short ones keeps no CTA waiting, and a captured launch serves every length.  A share may end inside a
// list and go on with the next; what a CTA has of a list that it does not hold whole goes to the scratch, at place
// 2 * CTA for the list that its share begins in and 2 * CTA + 1 for the one that it begins inside the share.  Whoever has a
// list's first unit notes its number of parts and the place of the first for the kernel that joins them.
// A list costs its CTAs about EXTRA units more than its positions (its queries, the first tiles' way, the warps' meeting), and counts as
// longer by so much, in front of its first unit: else the shares that hold many short lists finish last (64 requests of 40 heads over 8
// and every length up to 16,384: 135 us, 149 without, in short runs, after which the power limit holds both to 149; of 28 over 4, up to 8,000: 47.5, 69).  Not where there is a CTA for every unit, nor
// where every list is one unit.
// ------------------------------------------------------------------------------------
constexpr int UNIT = 128, EXTRA = 2;

struct Cut {                       // of one request
  int tok0, q_len, kv_len;
  int lo16, units;                 // first tile of 16 positions; units from there on, at least one if there are rows
  int span;                        // units and what a list costs besides
  int row_tiles;                   // 0: the request is not for this kernel
};
__device__ __forceinline__ Cut cut_of(const int* cu_q, const int* kv_lens, int b, int G, int rows_per_tile, int max_rows, int window, int extra) {
  Cut c;
  c.tok0 = cu_q[b];
  c.q_len = cu_q[b + 1] - c.tok0;
  c.kv_len = kv_lens[b];
  const int rows = c.q_len * G;
  const int first = window > 0 ? max(0, c.kv_len - c.q_len - window + 1) : 0;
  c.lo16 = first >> 4;
  c.row_tiles = rows > 0 && rows <= max_rows ? (rows + rows_per_tile - 1) / rows_per_tile : 0;
  c.units = c.row_tiles ? max(1, (c.kv_len - c.lo16 * 16 + UNIT - 1) / UNIT) : 0;
  c.span = c.row_tiles ? c.units + extra : 0;
  return c;
}
// The length of all lists together, and in `extra` what every one counts beside its units.  One warp; all lanes get the answer.
__device__ __forceinline__ int all_units(const int* cu_q, const int* kv_lens, int B, int nkv, int G, int rows_per_tile, int max_rows, int window,
                                         int& extra) {
  int units = 0, lists = 0;
  for (int b = threadIdx.x & 31; b < B; b += 32) {
    const Cut c = cut_of(cu_q, kv_lens, b, G, rows_per_tile, max_rows, window, 0);
    units += c.units * c.row_tiles * nkv;
    lists += c.row_tiles * nkv;
  }
  units = __reduce_add_sync(0xffffffffu, units);
  lists = __reduce_add_sync(0xffffffffu, lists);
  extra = units <= (int)gridDim.x || units == lists ? 0 : EXTRA;      // (lists of one unit each are not cut)
  return units + extra * lists;
}
// The shares: share i of `shares` is units [share_start(i), share_start(i + 1)).
__device__ __forceinline__ int share_start(int i, int shares, int total) { return (int)((long long)total * i / shares); }
// The share that holds unit x.
__device__ __forceinline__ int share_of(int x, int shares, int total) { return (int)((((long long)x + 1) * shares - 1) / total); }

struct Place {                     // a unit's request, and the request's first unit
  int b, first;
  Cut cut;
};
// One warp; all lanes get the answer.
__device__ __forceinline__ Place find_unit(const int* cu_q, const int* kv_lens, int B, int nkv, int G, int rows_per_tile, int max_rows,
                                           int window, int extra, int unit, int b_from, int first) {
  const int lane = threadIdx.x & 31;
  Place p;
  p.b = -1;
  int before = first;
  for (int b0 = b_from; b0 < B && p.b < 0; b0 += 32) {
    const int b = b0 + lane;
    Cut c = {0, 0, 0, 0, 0, 0, 0};
    if (b < B) c = cut_of(cu_q, kv_lens, b, G, rows_per_tile, max_rows, window, extra);
    const int mine = c.span * c.row_tiles * nkv;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const int start = before + sum - mine;
    const unsigned hit = __ballot_sync(0xffffffffu, unit >= start && unit < start + mine);
    if (hit) {
      const int src = __ffs(hit) - 1;
      p.b = b0 + src;
      p.first = __shfl_sync(0xffffffffu, start, src);
      p.cut.tok0 = __shfl_sync(0xffffffffu, c.tok0, src);
      p.cut.q_len = __shfl_sync(0xffffffffu, c.q_len, src);
      p.cut.kv_len = __shfl_sync(0xffffffffu, c.kv_len, src);
      p.cut.lo16 = __shfl_sync(0xffffffffu, c.lo16, src);
      p.cut.units = __shfl_sync(0xffffffffu, c.units, src);
      p.cut.row_tiles = __shfl_sync(0xffffffffu, c.row_tiles, src);
      p.cut.span = p.cut.units + extra;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return p;
}

// The merge of partial results (maximum, sum, accumulator) in ascending order; a maximum of -inf carries nothing.
__device__ __forceinline__ float factor(float m, float M) { return m == -INFINITY ? 0.f : exp2f(m - M); }

// ------------------------------------------------------------------------------------
// Attention in float32 arithmetic: any compute type, any alignment, any rows.  A CTA per (token, kv head, part of the visible tiles)
// walks its tiles with its warps side by side; a lane has two halves of one key row for the scores and four channels of a group for
// the sums.  HC heads of the group at a time share a tile's codes.  Bound by the latency of a warp's chain; so many warps, as many
// heads at a time as fit the registers (28 tokens of 14 heads over 2, 256 positions: 12.1 us by 8 heads, 14.2 by 4; 12 tokens of 32
// over 8, 300 positions: 19.6 by 8, of which half idle, 14.7 by 4), and parts (joined by a kernel after it) while there are
// fewer CTAs than the GPU holds.
// ------------------------------------------------------------------------------------
constexpr int SW = HD > 128 ? 8 : 16;        // warps
constexpr int VU = (HD / 4 + 31) / 32;       // units of four channels per lane

template <typename T, int HC>
__global__ void __launch_bounds__(32 * SW)
kv4_simple_kernel(const T* __restrict__ q, long q_ld, T* __restrict__ out, long out_ld, const unsigned char* __restrict__ k_cache,
                  const unsigned char* __restrict__ v_cache, int num_pages, const int* __restrict__ table, int table_ld, int n_req,
                  const int* __restrict__ token_req, const int* __restrict__ positions, int nh, int nkv, int page_size, int window,
                  float scale_log2, float* __restrict__ scratch, int* __restrict__ status) {
  __shared__ __align__(16) float qs[HC][HD];
  __shared__ float sp[SW][HC][16];
  __shared__ float merge[SW / 2][HC][HD + 2];
  co_pdl_launch_dependents();
  co_pdl_wait();
  const int token = blockIdx.x, kvh = blockIdx.y, part = blockIdx.z, parts = gridDim.z, G = nh / nkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int pos = positions[token];
  const int req = token_req[token];
  if (req < 0 || req >= n_req) {
    if (tid == 0 && status) *status = BAD_INDEX;
    pos = -1;                          // sees nothing
  }
  const int* pages = table + (size_t)(pos < 0 ? 0 : req) * table_ld;
  const int lo = window > 0 ? max(0, pos - window + 1) : 0, first = lo >> 4, tiles = pos < 0 ? 0 : (pos >> 4) - first + 1;
  const int tile_first = first + (int)((long long)tiles * part / parts), tile_end = first + (int)((long long)tiles * (part + 1) / parts);
  for (int h0 = 0; h0 < G; h0 += HC) {
    const int n = min(HC, G - h0);
    __syncthreads();
    for (int i = tid; i < HC * HD; i += 32 * SW) {
      const int h = i / HD;
      qs[h][i % HD] = h < n ? co_to_float<T>(q[(size_t)token * q_ld + (size_t)(kvh * G + h0 + h) * HD + i % HD]) : 0.f;
    }
    __syncthreads();
    float m[HC], l[HC], acc[HC][VU][4];
#pragma unroll
    for (int h = 0; h < HC; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
#pragma unroll
      for (int v = 0; v < VU; ++v)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[h][v][c] = 0.f;
    }
    for (int tile = tile_first + warp; tile < tile_end; tile += SW) {
      const int blk = tile * 16 / page_size;
      const int page = blk < table_ld ? pages[blk] : -1;
      if (page < 0 || page >= num_pages) {
        if (lane == 0 && status) *status = BAD_INDEX;
        continue;
      }
      const size_t at = tile_at(page, nkv, kvh, page_size, tile * 16 - blk * page_size);
      const unsigned char *kt = k_cache + at, *vt = v_cache + at;
      // Scores: lane = (row, half); words t = 2 half, 2 half + 1 of every group.
      const int r = lane >> 1, half = lane & 1;
      float s[HC];
#pragma unroll
      for (int h = 0; h < HC; ++h) s[h] = 0.f;
#pragma unroll
      for (int u = 0; u < NG; ++u) {
        const unsigned sm = reinterpret_cast<const unsigned*>(kt + CODES)[r * NG + u];
        const float sc = lo_bf16(sm), mn = hi_bf16(sm);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int t = 2 * half + w;
          const unsigned word = reinterpret_cast<const unsigned*>(kt)[r * (4 * NG) + t * NG + u];
          float x[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) x[c] = fmaf(sc, (float)((word >> (4 * c)) & 15), mn);
#pragma unroll
          for (int h = 0; h < HC; ++h) {
            const float4 a = *reinterpret_cast<const float4*>(&qs[h][u * 32 + t * 8]), b = *reinterpret_cast<const float4*>(&qs[h][u * 32 + t * 8 + 4]);
            s[h] = fmaf(a.x, x[0], fmaf(a.y, x[1], fmaf(a.z, x[2], fmaf(a.w, x[3], s[h]))));
            s[h] = fmaf(b.x, x[4], fmaf(b.y, x[5], fmaf(b.z, x[6], fmaf(b.w, x[7], s[h]))));
          }
        }
      }
      const int p = tile * 16 + r;
      const bool seen = p >= lo && p <= pos;
#pragma unroll
      for (int h = 0; h < HC; ++h) {
        s[h] += __shfl_xor_sync(0xffffffffu, s[h], 1);
        s[h] = seen ? s[h] * scale_log2 : -INFINITY;
        const float M = fmaxf(m[h], co_warp_max(s[h]));
        const float f = factor(m[h], M);
        const float e = s[h] == -INFINITY ? 0.f : exp2f(s[h] - M);
        m[h] = M;
        l[h] = l[h] * f + (half == 0 ? e : 0.f);
        if (half == 0) sp[warp][h][r] = e;
#pragma unroll
        for (int v = 0; v < VU; ++v)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[h][v][c] *= f;
      }
      __syncwarp();
      // Sums: a lane has four channels of VU groups.
#pragma unroll
      for (int v = 0; v < VU; ++v) {
        const int unit = v * 32 + lane, u = unit >> 3, g = unit & 7;
        if (unit >= HD / 4) break;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint2 words = reinterpret_cast<const uint2*>(vt)[u * 32 + g * 4 + t];
          const uint4 sm = reinterpret_cast<const uint4*>(vt + CODES)[u * 4 + t];
          const float sc[4] = {lo_bf16(sm.x), hi_bf16(sm.x), lo_bf16(sm.y), hi_bf16(sm.y)};
          const float mn[4] = {lo_bf16(sm.z), hi_bf16(sm.z), lo_bf16(sm.w), hi_bf16(sm.w)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = 4 * t + e;
            if (tile * 16 + row < lo || tile * 16 + row > pos) continue;
            const unsigned hw = (e < 2 ? words.x : words.y) >> (16 * (e & 1));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float x = fmaf(sc[e], (float)((hw >> (4 * c)) & 15), mn[e]);
#pragma unroll
              for (int h = 0; h < HC; ++h) acc[h][v][c] = fmaf(sp[warp][h][row], x, acc[h][v][c]);
            }
          }
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < HC; ++h) l[h] = co_warp_sum(l[h]);
    // The warps meet: the upper half of them leaves its sums, the lower half adds its own in the same order for every row.
    auto leave = [&](float (*dst)[HD + 2]) {
#pragma unroll
      for (int h = 0; h < HC; ++h) {
        if (lane == 0) { dst[h][HD] = m[h]; dst[h][HD + 1] = l[h]; }
#pragma unroll
        for (int v = 0; v < VU; ++v) {
          const int unit = v * 32 + lane;
          if (unit < HD / 4)
#pragma unroll
            for (int c = 0; c < 4; ++c) dst[h][unit * 4 + c] = acc[h][v][c];
        }
      }
    };
    if (warp >= SW / 2) leave(merge[warp - SW / 2]);
    __syncthreads();
    if (warp < SW / 2) {
      float (*other)[HD + 2] = merge[warp];
#pragma unroll
      for (int h = 0; h < HC; ++h) {
        const float M = fmaxf(m[h], other[h][HD]), f = factor(m[h], M), g = factor(other[h][HD], M);
        m[h] = M;
        l[h] = l[h] * f + other[h][HD + 1] * g;
#pragma unroll
        for (int v = 0; v < VU; ++v) {
          const int unit = v * 32 + lane;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (unit < HD / 4) acc[h][v][c] = acc[h][v][c] * f + other[h][unit * 4 + c] * g;
        }
      }
      __syncwarp();
      leave(other);
    }
    __syncthreads();
    for (int i = tid; i < n * HD; i += 32 * SW) {
      const int h = i / HD, c = i % HD, head = kvh * G + h0 + h;
      float M = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
      for (int w = 0; w < SW / 2; ++w) M = fmaxf(M, merge[w][h][HD]);
#pragma unroll
      for (int w = 0; w < SW / 2; ++w) {
        const float f = factor(merge[w][h][HD], M);
        den += f * merge[w][h][HD + 1];
        num += f * merge[w][h][c];
      }
      if (parts == 1) {
        out[(size_t)token * out_ld + (size_t)head * HD + c] = co_from_float<T>(den == 0.f ? 0.f : num / den);
      } else {
        float* dst = scratch + (((size_t)token * nh + head) * parts + part) * (HD + 2);
        dst[c] = num;
        if (c == 0) { dst[HD] = M; dst[HD + 1] = den; }
      }
    }
  }
}

// Joins the parts of a row: a warp per (token, head), in ascending order of the parts.
template <typename T>
__global__ void __launch_bounds__(128)
kv4_simple_join_kernel(const float* __restrict__ scratch, int parts, T* __restrict__ out, long out_ld, int nh, int rows) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  co_pdl_launch_dependents();
  if (row >= rows) return;
  co_pdl_wait();
  const float* src = scratch + (size_t)row * parts * (HD + 2);
  float M = -INFINITY, den = 0.f, acc[HD / 32];
  for (int p = lane; p < parts; p += 32) M = fmaxf(M, src[p * (HD + 2) + HD]);
  M = co_warp_max(M);
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) acc[i] = 0.f;
  for (int p = 0; p < parts; ++p) {
    const float f = factor(src[p * (HD + 2) + HD], M);
    den += f * src[p * (HD + 2) + HD + 1];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] += f * src[p * (HD + 2) + i * 32 + lane];
  }
  T* dst = out + (size_t)(row / nh) * out_ld + (size_t)(row % nh) * HD;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) dst[i * 32 + lane] = co_from_float<T>(den == 0.f ? 0.f : acc[i] / den);
}

// ------------------------------------------------------------------------------------
// Attention of few query rows per kv head (decoding, short runs) on mma.sync.m16n8k16: one CTA per share of the units, four warps,
// each with pairs of tiles of its own (pair i of a list's share goes to warp i mod 4) in a ring of its own that it fills with
// cp.async, so that warps never wait for one another before the end (bulk copies of whole tiles by one lane took more
// instructions: their operands go through uniform registers).  Decoding is
// bound by the cache's bytes, and with 5 bits a value nearly as much by the instructions that turn codes into operands,
// those of the half-rate integer pipe first; hence:
//  * positions are the M side of both products and the 8 NT query rows (token, head of the group) the N side, so a group
//    of up to 8 heads wastes no product;
//  * keys: the bits of code c, masked out of a half word, are the float16 c 2^-24 (a subnormal, which the tensor cores take
//    as it is) or 16 c 2^-24, so two codes cost one logical operation and eight one shift; the queries of the
//    odd channels are divided by 16.  The group's scale multiplies float32 sums, and the minima's share, sum over the groups
//    of m sum(q), is one product more over the groups in the place of the channels, with sum(q) as three bfloat16 terms.
//    No key is rounded.  Queries enter as float16 times the power of two that brings the row's largest to 2^14..2^15:
//    exact, but for elements under 2^-24 of it;
//  * values: s c + m in float16 with one rounding (1024 + c - 1024 is exact, then one fused multiply-add on pairs).  A pair of tiles has its
//    scales and minima turned to float16 in their place when it has landed (32 pieces of 16 bytes at head size 128, one a lane), times a
//    power of two that follows the largest of them, so that a value keeps eleven bits, or what lies over 2^-34 of the largest.  In
//    bfloat16 the values' rounding alone made 2.25e-3 against 64 bits; 1.7e-3 now, of which the outputs' own is 1.65e-3.  The scale
//    put on the probability instead takes fewer instructions but rounds p s, whose error meets s c and not s c + m;
//  * probabilities leave the first product's registers for the second's by movmatrix (transposed), not through memory, in float16 and
//    2^LIFT times over their reference: one term (as two bfloat16 terms, which the values' type asked for before, they took twice the
//    products and movmatrix: 64 x up to 16,384 151 us, 143 now; 2 x up to 131,072 43.4, 40.6);
//  * the reference that scores are counted from moves (and the accumulators are scaled) only when a score exceeds it by more
//    than 2^SLACK.
//  * the values' product of a pair and the scores of the next stand in one run of code without a branch, so that a warp
//    has work of both kinds to issue.
// The rows' sums stay per lane and meet once at the end, as do the warps.
// ------------------------------------------------------------------------------------
constexpr int WARPS = 4;
constexpr int K_STAGES = 2, V_STAGES = 3;      // pairs of key tiles and of value tiles in a warp's ring: values are used one pair later
constexpr int PAIR = 2 * TB;
constexpr int RING = (K_STAGES + V_STAGES) * PAIR;
constexpr float NOTHING = -3.0e38f;      // a reference that no score has met
constexpr float SLACK = 8.f;
constexpr float LIFT = 7.f;              // probabilities are 2^LIFT times over their reference: 2^15 at most, and 2^-32 of it is float16's least

template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// A tile, by a warp: 16 bytes per lane and round; zeros when `bytes` is 0 (16: the copy).
__device__ __forceinline__ void copy_tile(unsigned dst, const unsigned char* src, int lane, int bytes) {
  constexpr int WHOLE = TB / 512, REST = TB % 512 / 16;
#pragma unroll
  for (int i = 0; i < WHOLE; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 512 * i), "l"(src + 512 * i), "r"(bytes) : "memory");
  if (REST && lane < REST)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 512 * WHOLE), "l"(src + 512 * WHOLE), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from nothing: an accumulator that starts at zero without a register set to it.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ unsigned transposed(unsigned v) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));   // ex2(-inf) = +0
  return y;
}
// (word & mask) | constant as one instruction: written out, since the two constants would otherwise make two of it.
__device__ __forceinline__ unsigned masked(unsigned word, unsigned mask, unsigned constant) {
  unsigned r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(word), "r"(mask), "r"(constant));
  return r;
}
// Codes j and j + 4 of a word as the float16 pair 1024 + c, and as the float16 pair c 2^-24 (j even) or 16 c 2^-24 (j odd).
__device__ __forceinline__ unsigned codes1024(unsigned word, int j) { return masked(word >> (4 * j), 0x000f000fu, 0x64006400u); }
__device__ __forceinline__ unsigned codes16(unsigned word, int j) { return (j < 2 ? word : word >> 8) & (j & 1 ? 0x00f000f0u : 0x000f000fu); }
template <int N>
__device__ __forceinline__ void load_words(const unsigned* p, unsigned (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 v = reinterpret_cast<const uint2*>(p)[i];
      w[2 * i] = v.x; w[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p[i];
  }
}
constexpr int MLD = HD + 4;              // a row of the warps' meeting: HD channels, reference, sum
template <int NT>
constexpr size_t items_smem() {           // rings, or the warps' meeting and what a cluster's CTAs leave one another
  const size_t ring = (size_t)WARPS * RING, merge = (size_t)(WARPS + 1) * 8 * NT * MLD * sizeof(float);
  return ring > merge ? ring : merge;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared memory `p` in CTA `rank` of the cluster, and floats from there.
__device__ __forceinline__ unsigned in_cluster(const void* p, unsigned rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(unsigned at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(unsigned at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

// The query rows of a tile as the products' N side: lane (g, t) has row g of every eight, channels 32 u + 8 t + 0..7.
constexpr int MG = (NG + 3) / 4;         // products for the minima
template <int NT>
struct Queries {
  unsigned f[NT][NG][4];
  unsigned sums[NT][MG][2];              // sum(q) 2^-24 of row g, group 4 i + t, in three terms
  float cs[NT][2];                       // what the scores of rows 2 t, 2 t + 1 are multiplied by
};
template <int NT>
struct Sums {
  float o[NG][2][NT][4];                 // channels 32 u + 4 g + 2 h, + 1 (first index of four: rows 2 t, 2 t + 1)
  float m[NT][2], l[NT][2];              // reference and sum of rows 2 t, 2 t + 1
};

template <int NT>
__device__ __forceinline__ void load_queries(Queries<NT>& qr, const bf16* __restrict__ q, long q_ld, int tok0, int G, int kvh, int row0, int rows,
                                             float scale_log2) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g, row = row0 + r;
    const bf16* src = q + (size_t)(tok0 + row / G) * q_ld + (size_t)(kvh * G + row % G) * HD;
    uint4 v[NG];
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      v[u] = make_uint4(0, 0, 0, 0);
      if (r < rows) v[u] = *reinterpret_cast<const uint4*>(src + u * 32 + t * 8);
      const unsigned w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(lo_bf16(w[i])), fabsf(hi_bf16(w[i]))));
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^(14 - e) with 2^e <= most < 2^(e + 1), and 2^24 times its inverse
    const int e = min(max((int)(__float_as_uint(most) >> 23), 15), 240);
    const float by = __uint_as_float((unsigned)(268 - e) << 23), back = __uint_as_float((unsigned)(e - 14) << 23) * 16777216.f;
    qr.cs[nt][0] = scale_log2 * __shfl_sync(0xffffffffu, back, 8 * t);
    qr.cs[nt][1] = scale_log2 * __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
    for (int i = 0; i < MG; ++i) qr.sums[nt][i][0] = qr.sums[nt][i][1] = 0;
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const unsigned w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      float x[8], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __half2float(__float2half_rn(lo_bf16(w[i]) * by));
        x[2 * i + 1] = __half2float(__float2half_rn(hi_bf16(w[i]) * by * 0.0625f));
        sum += fmaf(16.f, x[2 * i + 1], x[2 * i]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) qr.f[nt][u][j] = pack_f16(x[j], x[j + 4]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == (u & 3)) {
        sum *= 1.f / 16777216.f;
        const float a = __bfloat162float(__float2bfloat16_rn(sum)), b = __bfloat162float(__float2bfloat16_rn(sum - a));
        qr.sums[nt][u >> 2][0] = pack(a, b);
        qr.sums[nt][u >> 2][1] = pack(sum - a - b, 0.f);
      }
    }
  }
}

// The scores of a tile's 16 positions, up to the rows' factors: s[nt] has positions r0, r0 and r0 + 2, r0 + 2 of rows 2 t, 2 t + 1,
// r0 = 4 (g / 2) + g % 2.
template <int NT>
__device__ __forceinline__ void tile_scores(float (&s)[NT][4], const Queries<NT>& qr, const unsigned char* kt) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, r0 = 4 * (g >> 1) + (g & 1);
  unsigned ka[NG], kb[NG], pa[NG], pb[NG];
  load_words<NG>(reinterpret_cast<const unsigned*>(kt) + r0 * (4 * NG) + t * NG, ka);
  load_words<NG>(reinterpret_cast<const unsigned*>(kt) + (r0 + 2) * (4 * NG) + t * NG, kb);
  const unsigned* pairs = reinterpret_cast<const unsigned*>(kt + CODES);
  load_words<NG>(pairs + r0 * NG, pa);
  load_words<NG>(pairs + (r0 + 2) * NG, pb);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
  for (int x = 0; x < MG; ++x) {
    const int u = min(4 * x + t, NG - 1);
    const unsigned wa = pairs[r0 * NG + u], wb = pairs[(r0 + 2) * NG + u];
    const unsigned ma = __byte_perm(wa, wa, 0x3232), mb = __byte_perm(wb, wb, 0x3232);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma_bf16(s[nt], ma, mb, ma, mb, qr.sums[nt][x][0], qr.sums[nt][x][1]);
  }
#pragma unroll
  for (int u = 0; u < NG; ++u) {
    unsigned a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { a[j] = codes16(ka[u], j); b[j] = codes16(kb[u], j); }
    const float sa = lo_bf16(pa[u]), sb = lo_bf16(pb[u]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float d[4];
      mma_f16_first(d, a[0], b[0], a[1], b[1], qr.f[nt][u][0], qr.f[nt][u][1]);
      mma_f16(d, a[2], b[2], a[3], b[3], qr.f[nt][u][2], qr.f[nt][u][3]);
      s[nt][0] = fmaf(sa, d[0], s[nt][0]);
      s[nt][1] = fmaf(sa, d[1], s[nt][1]);
      s[nt][2] = fmaf(sb, d[2], s[nt][2]);
      s[nt][3] = fmaf(sb, d[3], s[nt][3]);
    }
  }
}

// Adds a tile's values, weighted: pf[nt] holds the probabilities of the 16 positions for row g of every eight.  The tile's pairs are float16 (see `to_half`).
template <int NT>
__device__ __forceinline__ void tile_values(Sums<NT>& sm, const unsigned (&pf)[NT][2], const unsigned char* vt) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  const __half2 k1024 = __floats2half2_rn(1024.f, 1024.f);
#pragma unroll
  for (int u = 0; u < NG; ++u) {
    const uint2 w = reinterpret_cast<const uint2*>(vt)[u * 32 + lane];
    const uint4 pairs = reinterpret_cast<const uint4*>(vt + CODES)[u * 4 + t];
    const __half2 s01 = half_pair(pairs.x), s23 = half_pair(pairs.y), m01 = half_pair(pairs.z), m23 = half_pair(pairs.w);
    unsigned a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = bits(__hfma2(__hsub2(half_pair(codes1024(w.x, j)), k1024), s01, m01));
      b[j] = bits(__hfma2(__hsub2(half_pair(codes1024(w.y, j)), k1024), s23, m23));
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mma_f16(sm.o[u][0][nt], a[0], a[1], b[0], b[1], pf[nt][0], pf[nt][1]);
      mma_f16(sm.o[u][1][nt], a[2], a[3], b[2], b[3], pf[nt][0], pf[nt][1]);
    }
  }
}

// CLUSTER: the CTAs of a cluster cut one list among themselves and join it through their shared memory, without a second kernel.
template <int NT, int PER_SM, bool CLUSTER>
__global__ void __launch_bounds__(32 * WARPS, PER_SM)
kv4_items_kernel(const bf16* __restrict__ q, long q_ld, bf16* __restrict__ out, long out_ld, const unsigned char* __restrict__ k_cache,
                 const unsigned char* __restrict__ v_cache, int num_pages, const int* __restrict__ block_tables, int table_ld,
                 const int* __restrict__ cu_q, const int* __restrict__ kv_lens, int B, int nh, int nkv, int page_size, int window,
                 float scale_log2, int max_rows, int csize, float* __restrict__ scratch, int* __restrict__ status) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int COLS = 8 * NT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int r0 = 4 * (g >> 1) + (g & 1);        // see tile_scores
  co_pdl_wait();
  co_pdl_launch_dependents();
  const int G = nh / nkv;
  int total = 0, shares = 0, unit = 0, unit_end = 0, extra = 0;
  Place at;
  const int most_tiles = (max_rows + COLS - 1) / COLS, own_list = CLUSTER ? (int)blockIdx.x / csize : 0, rank = CLUSTER ? (int)blockIdx.x % csize : 0;
  if constexpr (CLUSTER) {
    at.b = own_list / (nkv * most_tiles);
    at.cut = cut_of(cu_q, kv_lens, at.b, G, COLS, max_rows, window, 0);
    if (own_list % most_tiles >= at.cut.row_tiles) return;      // the whole cluster
  } else {
    total = all_units(cu_q, kv_lens, B, nkv, G, COLS, max_rows, window, extra);
    shares = min((int)gridDim.x, total);
    if ((int)blockIdx.x >= shares) return;
    unit = share_start(blockIdx.x, shares, total);
    unit_end = share_start(blockIdx.x + 1, shares, total);
    at = find_unit(cu_q, kv_lens, B, nkv, G, COLS, max_rows, window, extra, unit, 0, 0);
  }
  unsigned char* ring = smem + (size_t)warp * RING;       // keys, then values
  const unsigned ring_lane = smem_u32(ring) + lane * 16;
  const unsigned char *k_lane = k_cache + lane * 16, *v_lane = v_cache + lane * 16;

  for (bool first_list = true; at.b >= 0; first_list = false) {
    const Cut c = at.cut;
    int row_tile, kvh, u_first, u_end, s_first = 0, s_end = 0;
    if constexpr (CLUSTER) {
      row_tile = own_list % most_tiles;
      kvh = own_list / most_tiles % nkv;
      u_first = share_start(rank, csize, c.units);
      u_end = share_start(rank + 1, csize, c.units);
    } else {
      const int list = (unit - at.first) / c.span;
      s_first = unit - at.first - list * c.span;
      s_end = min(c.span, s_first + unit_end - unit);
      u_first = max(0, s_first - extra);
      u_end = max(0, s_end - extra);
      row_tile = list % c.row_tiles;
      kvh = list / c.row_tiles;
    }
    const int row0 = row_tile * COLS, rows = min(COLS, c.q_len * G - row0);      // query rows of this tile
    const int* table = block_tables + (size_t)at.b * table_ld;
    const int tile_end = min(c.lo16 + u_end * (UNIT / 16), (c.kv_len + 15) >> 4);
    const int tile0 = c.lo16 + u_first * (UNIT / 16) + 2 * warp;
    const int n_pairs = tile_end > tile0 ? (tile_end - tile0 + 2 * WARPS - 1) / (2 * WARPS) : 0;    // of this warp
    const int base_pos = c.kv_len - c.q_len;

    // Where the warp's tiles lie in a cache, 16 pairs at a time, a tile per lane; `valid`: the lanes whose tile exists.
    long long place = 0;
    unsigned valid = 0;
    auto fetch_places = [&](int i0) {
      const int tile = tile0 + (i0 + (lane >> 1)) * 2 * WARPS + (lane & 1), per_page = page_size >> 4;
      bool ok = tile < tile_end;
      place = 0;
      if (ok) {
        const int blk = tile / per_page, page = blk < table_ld ? table[blk] : -1;
        ok = page >= 0 && page < num_pages;
        if (ok) place = (((long long)page * nkv + kvh) * per_page + (tile - blk * per_page)) * TB;
        else if (status) *status = BAD_INDEX;
      }
      valid = __ballot_sync(0xffffffffu, ok);
    };
    unsigned known = 0;              // two bits per pair, the latest lowest: the tile is there (zeros otherwise)
    auto issue = [&](int i, int v_stage) {        // one group per call, with or without copies
      known <<= 2;
      if (i < n_pairs) {
        if ((i & 15) == 0) fetch_places(i);
        const unsigned there = (valid >> (2 * (i & 15))) & 3u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const long long from = __shfl_sync(0xffffffffu, place, 2 * (i & 15) + h);
          const int bytes = (there >> h) & 1u ? 16 : 0;
          copy_tile(ring_lane + (i & 1) * PAIR + h * TB, k_lane + from, lane, bytes);
          copy_tile(ring_lane + (K_STAGES + v_stage) * PAIR + h * TB, v_lane + from, lane, bytes);
        }
        known |= there;
      }
      cp_async_commit();
    };
    issue(0, 0);
    issue(1, 1);

    Queries<NT> qr;
    load_queries<NT>(qr, q, q_ld, c.tok0, G, kvh, row0, rows, scale_log2);
    Sums<NT> sm;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sm.m[nt][0] = sm.m[nt][1] = NOTHING;
      sm.l[nt][0] = sm.l[nt][1] = 0.f;
#pragma unroll
      for (int u = 0; u < NG; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) sm.o[u][h][nt][i] = 0.f;
    }
    // Positions [all_lo, all_hi] are visible to every row of the tile.
    const int all_hi = base_pos + row0 / G, last = base_pos + (row0 + rows - 1) / G;
    const int all_lo = window > 0 ? max(0, last - window + 1) : 0;

    float s[2][NT][4];
    unsigned pf[2][NT][2];
    // The values' power of two: 2^(137 - v_exp) brings what was the largest magnitude when it was chosen to 2^10..2^11; up to v_limit it stays.
    int v_exp = 137;
    unsigned v_limit = 0;
    // The pairs of a pair of value tiles from bfloat16 to float16 in their place, times that power of two (exact, but for what lies under
    // 2^-34 of the largest).  Positions outside what any query sees may hold anything (a stale row, a page's end): their pairs become
    // zero, so that nothing which is not finite meets a probability of zero.
    auto to_half = [&](unsigned char* values, bool whole, int key0, unsigned there) {
      constexpr int PIECES = 8 * NG, ROUNDS = (PIECES + 31) / 32;         // of four rows' scales and minima each
      uint4 w[ROUNDS];
      float most = 0.f;
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int x = r * 32 + lane, h = x / (4 * NG), p = x - h * (4 * NG);
        w[r] = make_uint4(0, 0, 0, 0);
        if (PIECES % 32 == 0 || x < PIECES) w[r] = reinterpret_cast<const uint4*>(values + h * TB + CODES)[p];
        if (!whole) {
          const int first = key0 + 16 * h + 4 * (p & 3);
          const int lo = window > 0 ? all_hi - window + 1 : 0;
          auto seen = [&](int pos) { return ((there >> h) & 1u) && pos <= last && pos >= lo; };
          const unsigned k01 = (seen(first) ? 0xffffu : 0u) | (seen(first + 1) ? 0xffff0000u : 0u);
          const unsigned k23 = (seen(first + 2) ? 0xffffu : 0u) | (seen(first + 3) ? 0xffff0000u : 0u);
          w[r].x &= k01; w[r].y &= k23; w[r].z &= k01; w[r].w &= k23;
        }
        const float sc = fmaxf(fmaxf(lo_bf16(w[r].x), hi_bf16(w[r].x)), fmaxf(lo_bf16(w[r].y), hi_bf16(w[r].y)));
        const float mn = fmaxf(fmaxf(fabsf(lo_bf16(w[r].z)), fabsf(hi_bf16(w[r].z))), fmaxf(fabsf(lo_bf16(w[r].w)), fabsf(hi_bf16(w[r].w))));
        most = fmaxf(most, fmaxf(mn, 16.f * sc));          // a value is at most twice that
      }
      const unsigned all_most = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
      if (all_most > v_limit) {
        const int e = min(max((int)(all_most >> 23), 18), 254), by = 127 + v_exp - e;
        const float f = by > 0 ? __uint_as_float((unsigned)by << 23) : 0.f;
        v_exp = e;
        v_limit = (unsigned)min(e + 4, 254) << 23;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < NG; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) sm.o[u][h][nt][i] *= f;
      }
      const float by = __uint_as_float((unsigned)(264 - v_exp) << 23);
      auto half = [&](unsigned v) { return pack_f16(lo_bf16(v) * by, hi_bf16(v) * by); };
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int x = r * 32 + lane, h = x / (4 * NG), p = x - h * (4 * NG);
        if (PIECES % 32 == 0 || x < PIECES)
          reinterpret_cast<uint4*>(values + h * TB + CODES)[p] = make_uint4(half(w[r].x), half(w[r].y), half(w[r].z), half(w[r].w));
      }
      __syncwarp();
    };
    // From the scores s of pair i, whose values are at `values`, to its probabilities pf.
    auto probabilities = [&](int i, unsigned char* values) {
      const int key0 = (tile0 + i * 2 * WARPS) * 16;
      const unsigned there = (known >> 2) & 3u;        // of pair i: pair i + 1 was issued last
      const bool whole = there == 3u && key0 >= all_lo && key0 + 31 <= all_hi;
      float y[2][NT][4];            // exponents: scores (times log2 e) from the row's reference
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) y[h][nt][x] = fmaf(s[h][nt][x], qr.cs[nt][x & 1], -sm.m[nt][x & 1]);
      if (!whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = nt * 8 + 2 * t + (x & 1), hi = r < rows ? base_pos + (row0 + r) / G : -1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int pos = key0 + 16 * h + r0 + (x & 2);
              if (!((there >> h) & 1u) || pos > hi || (window > 0 && pos <= hi - window)) y[h][nt][x] = -INFINITY;
            }
          }
      }
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) grew = grew || fmaxf(y[0][nt][x], y[1][nt][x]) > SLACK + LIFT;
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float M = sm.m[nt][e];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int x = e; x < 4; x += 2) M = y[h][nt][x] == -INFINITY ? M : fmaxf(M, fmaf(s[h][nt][x], qr.cs[nt][e], -LIFT));
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
            const float f = ex2(sm.m[nt][e] - M);
            sm.m[nt][e] = M;
            sm.l[nt][e] *= f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int x = e; x < 4; x += 2) y[h][nt][x] = y[h][nt][x] == -INFINITY ? -INFINITY : fmaf(s[h][nt][x], qr.cs[nt][e], -M);
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h) { sm.o[u][h][nt][e] *= f; sm.o[u][h][nt][2 + e] *= f; }
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            y[h][nt][x] = ex2(y[h][nt][x]);
            sm.l[nt][x & 1] += y[h][nt][x];
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) pf[h][nt][x] = transposed(pack_f16(y[h][nt][2 * x], y[h][nt][2 * x + 1]));
        }
      to_half(values, whole, key0, there);
    };

    unsigned char* values = ring + K_STAGES * PAIR;            // of pair i
    if (n_pairs > 0) {
      cp_async_wait<1>();
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) tile_scores<NT>(s[h], qr, ring + h * TB);
      probabilities(0, values);
    }
    int v_stage = 0;
#pragma unroll 1
    for (int i = 0; i < n_pairs; ++i) {
      unsigned char* now = values;
      if (i + 1 < n_pairs) {
        // Keys of pair i + 2 go where pair i's were, values where pair i - 1's were.
        issue(i + 2, v_stage == 0 ? V_STAGES - 1 : v_stage - 1);
        v_stage = v_stage == V_STAGES - 1 ? 0 : v_stage + 1;
        values = ring + (K_STAGES + v_stage) * PAIR;
        cp_async_wait<1>();
        __syncwarp();                // pair i + 1 landed for all lanes
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tile_values<NT>(sm, pf[h], now + h * TB);
          tile_scores<NT>(s[h], qr, ring + ((i + 1) & 1) * PAIR + h * TB);
        }
        probabilities(i + 1, values);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) tile_values<NT>(sm, pf[h], now + h * TB);
      }
      __syncwarp();                  // all lanes are done with pair i
    }

    cp_async_wait<0>();
    __syncthreads();                 // the rings become the warps' meeting
    float* merge = reinterpret_cast<float*>(smem);
    const float v_back = __uint_as_float((unsigned)(v_exp - 17) << 23), lift_back = 1.f / 128.f;         // 2^(v_exp - 137 - LIFT), 2^-LIFT
    static_assert(LIFT == 7.f, "the exponents of the factors back");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = sm.l[nt][e];
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        float* dst = merge + (size_t)(warp * COLS + nt * 8 + 2 * t + e) * MLD;
        if (g == 0) { dst[HD] = sm.m[nt][e]; dst[HD + 1] = sum * lift_back; }
#pragma unroll
        for (int u = 0; u < NG; ++u)
          *reinterpret_cast<float4*>(dst + u * 32 + g * 4) =
              make_float4(sm.o[u][0][nt][e] * v_back, sm.o[u][0][nt][2 + e] * v_back, sm.o[u][1][nt][e] * v_back, sm.o[u][1][nt][2 + e] * v_back);
      }
    __syncthreads();
    const int slot = 2 * blockIdx.x + (first_list ? 0 : 1);
    float* acc_out = scratch + (size_t)slot * COLS * HD;
    float2* ml_out = reinterpret_cast<float2*>(scratch + (size_t)2 * gridDim.x * COLS * HD) + (size_t)slot * COLS;
    float* left = merge + (size_t)WARPS * COLS * MLD;          // for the cluster: a row's channels, reference and sum
    if (!CLUSTER && tid == 0 && s_first == 0) {
      int2* heads = reinterpret_cast<int2*>(scratch + (size_t)2 * gridDim.x * COLS * (HD + 2));
      heads[((size_t)at.b * nkv + kvh) * most_tiles + row_tile] =
          make_int2(share_of(unit + c.span - 1, shares, total) - (int)blockIdx.x + 1, slot);
    }
    const bool whole_list = !CLUSTER && s_first == 0 && s_end == c.span;
    for (int x = tid; x < rows * (HD / 4); x += 32 * WARPS) {
      const int r = x / (HD / 4), ch = x % (HD / 4) * 4;
      float M = NOTHING, den = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, merge[(size_t)(w * COLS + r) * MLD + HD]);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* src = merge + (size_t)(w * COLS + r) * MLD;
        const float f = exp2f(src[HD] - M);
        const float4 v = *reinterpret_cast<const float4*>(src + ch);
        den += f * src[HD + 1];
        acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      }
      if (whole_list) {
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const int row = row0 + r;
        bf16* dst = out + (size_t)(c.tok0 + row / G) * out_ld + (size_t)(kvh * G + row % G) * HD + ch;
        store4<bf16>(dst, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      } else if (CLUSTER) {
        *reinterpret_cast<float4*>(left + r * MLD + ch) = acc;
        if (ch == 0) *reinterpret_cast<float2*>(left + r * MLD + HD) = make_float2(M, den);
      } else {
        *reinterpret_cast<float4*>(acc_out + (size_t)r * HD + ch) = acc;
        if (ch == 0) ml_out[r] = make_float2(M, den);
      }
    }
    if constexpr (CLUSTER) {
      cluster_barrier();
      // The rows' pieces of four channels, shared among the CTAs; parts in ascending order.
      for (int x = rank * 32 * WARPS + tid; x < rows * (HD / 4); x += csize * 32 * WARPS) {
        const int r = x / (HD / 4), ch = x % (HD / 4) * 4;
        float M = NOTHING, den = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int p = 0; p < csize; ++p) M = fmaxf(M, ld_cluster2(in_cluster(left + r * MLD + HD, p)).x);
#pragma unroll 8
        for (int p = 0; p < csize; ++p) {
          const float2 ml = ld_cluster2(in_cluster(left + r * MLD + HD, p));
          const float4 v = ld_cluster4(in_cluster(left + r * MLD + ch, p));
          const float f = exp2f(ml.x - M);
          den += f * ml.y;
          acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const int row = row0 + r;
        store4<bf16>(out + (size_t)(c.tok0 + row / G) * out_ld + (size_t)(kvh * G + row % G) * HD + ch, acc.x * inv, acc.y * inv, acc.z * inv,
                     acc.w * inv);
      }
      cluster_barrier();               // nobody leaves while its part may still be read
      return;
    }
    unit += s_end - s_first;
    if (unit >= unit_end) return;
    __syncthreads();                 // the meeting becomes the rings again
    if (unit - at.first >= c.span * c.row_tiles * nkv)
      at = find_unit(cu_q, kv_lens, B, nkv, G, COLS, max_rows, window, extra, unit, at.b + 1, unit);
  }
}

// Joins the parts of the lists' rows.  A warp takes every `step`-th eight of a row's parts, four channels per lane.  WIDE: one CTA
// per row, its warps side by side over the parts, their sums added in order at the end; else one CTA per list and a warp per
// row.  Bound by its chain of dependent reads (the list's note, then references and accumulators at once); with many
// lists, of few parts each, by the number of CTAs.  So WIDE where the lists have more parts than a warp reads at once (both kernels, us: 14
// parts each, 224 rows, 16.0 wide, 17.1 by list; 9 parts, 512 rows, 29.9, 34.1; 7 parts, 448 rows, 23.0, 22.4; 2 parts, 1,792 rows, 29.0, 22.7).
constexpr int CW = 8;
template <bool WIDE>
__global__ void __launch_bounds__(32 * CW)
kv4_join_kernel(const float* __restrict__ scratch, int ctas, bf16* __restrict__ out, long out_ld, const int* __restrict__ cu_q, int nh, int nkv,
                int cols, int max_rows) {
  constexpr int V = (HD + 127) / 128;
  __shared__ float part[WIDE ? CW : 1][HD];
  __shared__ float part_den[CW];
  const int kvh = blockIdx.y, b = blockIdx.z, G = nh / nkv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Safe ahead of the wait: the kernel before starts this one only after its own wait for whatever made the lengths.
  const int tok0 = cu_q[b], rows = (cu_q[b + 1] - tok0) * G;
  const int row_tile = WIDE ? (int)blockIdx.x / cols : (int)blockIdx.x;
  if (rows > max_rows || (WIDE ? (int)blockIdx.x : row_tile * cols) >= rows) return;
  const size_t per_part = (size_t)cols * HD;
  const float2* all_ml = reinterpret_cast<const float2*>(scratch + (size_t)2 * ctas * per_part);
  const int2* heads = reinterpret_cast<const int2*>(scratch + (size_t)2 * ctas * cols * (HD + 2));
  co_pdl_wait();
  const int2 head = heads[((size_t)b * nkv + kvh) * ((max_rows + cols - 1) / cols) + row_tile];
  const int parts = head.x;
  if (parts == 1) return;
  // Part 0 is at head.y = 2 cta or 2 cta + 1, part p at 2 (cta + p).
  auto place = [&](int p) { return p == 0 ? head.y : (head.y & ~1) + 2 * p; };
  const int col_end = WIDE ? (int)blockIdx.x % cols + 1 : min(cols, rows - row_tile * cols);
  for (int col = WIDE ? (int)blockIdx.x % cols : warp; col < col_end; col += CW) {
    auto ml_of = [&](int p) { return all_ml[(size_t)place(p) * cols + col]; };
    float4 acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = NOTHING, den = 0.f;
    for (int p = lane; p < parts; p += 32) M = fmaxf(M, ml_of(p).x);
    bool known = false;               // M: after the first accumulators are on their way
    for (int p0 = WIDE ? warp * 8 : 0; p0 < parts; p0 += WIDE ? CW * 8 : 8) {
      const float2 ml = lane < 8 && p0 + lane < parts ? ml_of(p0 + lane) : make_float2(NOTHING, 0.f);
      float4 in[8][V];
#pragma unroll
      for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int ch = v * 128 + lane * 4;
          in[p][v] = p0 + p < parts && ch < HD ? *reinterpret_cast<const float4*>(scratch + place(p0 + p) * per_part + (size_t)col * HD + ch)
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      if (!known) M = co_warp_max(M);
      known = true;
      const float f = exp2f(ml.x - M);
      den += f * ml.y;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float fp = __shfl_sync(0xffffffffu, f, p);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          acc[v].x += fp * in[p][v].x; acc[v].y += fp * in[p][v].y; acc[v].z += fp * in[p][v].z; acc[v].w += fp * in[p][v].w;
        }
      }
    }
    den = co_warp_sum(den);
    if (WIDE) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int ch = v * 128 + lane * 4;
        if (ch < HD) *reinterpret_cast<float4*>(&part[warp][ch]) = acc[v];
      }
      if (lane == 0) part_den[warp] = den;
      __syncthreads();
      if (warp >= V) return;
      const int used = min(CW, (parts + 7) / 8), ch = threadIdx.x * 4;
      acc[0] = make_float4(0.f, 0.f, 0.f, 0.f);
      den = 0.f;
      for (int w = 0; w < used && ch < HD; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&part[w][ch]);
        acc[0].x += x.x; acc[0].y += x.y; acc[0].z += x.z; acc[0].w += x.w;
        den += part_den[w];
      }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const int row = row_tile * cols + col;
    bf16* dst = out + (size_t)(tok0 + row / G) * out_ld + (size_t)(kvh * G + row % G) * HD;
#pragma unroll
    for (int v = 0; v < (WIDE ? 1 : V); ++v) {
      const int ch = (WIDE ? warp : v) * 128 + lane * 4;
      if (ch < HD) store4<bf16>(dst + ch, acc[v].x * inv, acc[v].y * inv, acc[v].z * inv, acc[v].w * inv);
    }
  }
}

int tiles_of(int max_rows) { return max_rows <= 8 || HD > 128 ? 1 : 2; }
// CTAs that are resident per SM, by their registers.
constexpr int MOST = HD <= 128 ? 4 : 2, FEWER = HD <= 128 ? 3 : 2;

// How a step's units get their CTAs.
//  * A cluster per list, while every cluster is resident at once and a CTA gets four units at most: one kernel, and no chain of reads through
//    memory after it.  Against equal shares, heads 32 over 8, one token each (us): 1 x 900 positions 6.2 (7.9), 4 x 1,900 9.0 (11.3),
//    8 x 1,900 11.9 (16.5), 24 x 900 13.3 (18.3); four tokens each of heads 28 over 4, 4 x 1,900 12.1 (24.0).  A list has its CTAs to itself, so
//    one long list beside short ones may lose: 8 requests of 100 positions but one of 1,900, 10.0 (9.2).
//    Clusters as large as are resident, and no larger than gives every CTA a unit (1 x 200: 5.8 with two CTAs, 6.7 with four).  A cluster lies
//    in one GPC, whose last SMs it may not fill: 64 clusters of 4 run at once at two CTAs per SM, 72 do not (11.9 against 19.3 us at
//    1,900 positions), 104 do at three per SM, 112 do not.  Sixteen pay for four lists and more than eight units (1,900: 6.8 against 7.5),
//    no more (8 lists: 8.1 against 7.6).  More than two units per CTA only where the equal shares would give an SM several too
//    (8 lists of 3,900: 9.3 against 9.1; 32 lists: 11.5 against 15.4).
//  * Equal shares otherwise, one per resident CTA.  Three CTAs per SM, whose 168 registers let a warp work ahead, beat four of 128 (2 x 131,072,
//    28 heads over 4: 45.4 against 48.5; 64 x 8,192: 78 against 85), but where four give every unit a CTA at once (24 x 700: 12.6 against 14.6).
struct Split {
  int csize;       // CTAs of the cluster that has a list to itself; 0: all units in equal shares, joined by a kernel after it
  int per_sm;      // resident CTAs per SM, for which the kernel is built
  int ctas;
};
Split split_of(int B, int nkv, int max_rows, int max_kv_len) {
  const int nt = tiles_of(max_rows);
  const long long lists = (long long)B * nkv * ((max_rows + 8 * nt - 1) / (8 * nt));
  const int units = max(1, (int)((max_kv_len + UNIT - 1LL) / UNIT));         // of a list, at most
  if (units > 1) {
    int c = 0, per_sm = 2;
    if (HD <= 128 && lists <= 4 && units > 8) c = 16;
    for (int x : {8, 4, 2})
      if (c == 0 && lists * x <= 256) c = x;
    for (int x : {8, 4, 2})
      if (FEWER == 3 && nt == 1 && c < 8 && x > c && lists * x <= 416) { c = x; per_sm = 3; break; }
    if (c) {
      while (c > 2 && units <= c / 2) c /= 2;
      if (units <= 4 * c && (units <= 2 * c || lists * units > 148 * 2)) return {c, per_sm, (int)(lists * c)};
    }
  }
  const long long all = lists * units;
  const int per_sm = nt == 2 ? 2 : all > 148 * FEWER && all <= 148 * MOST ? MOST : FEWER;
  return {0, per_sm, (int)(all < 148 * per_sm ? all : 148 * per_sm)};
}

template <int NT, int PER_SM, bool CLUSTER>
int launch_items(const void* q, long q_ld, void* out, long out_ld, const void* k_cache, const void* v_cache, int num_pages, const int* table,
                 int table_ld, const int* cu_q, const int* kv_lens, int B, int nh, int nkv, int page_size, int window, float scale_log2,
                 int max_rows, int ctas, int csize, float* scratch, int* status, cudaStream_t stream) {
  constexpr size_t SMEM = items_smem<NT>();
  auto kernel = kv4_items_kernel<NT, PER_SM, CLUSTER>;
  cudaError_t e = SMEM > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM) : cudaSuccess;
  if (e == cudaSuccess && csize > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) CO_FAIL("kv4_attention: %zu bytes of shared memory, clusters of %d: %s", SMEM, csize, cudaGetErrorString(e));
  e = co_launch_cluster(csize, kernel, dim3((unsigned)ctas), dim3(32 * WARPS), SMEM, stream, (const bf16*)q, q_ld, (bf16*)out, out_ld,
                        (const unsigned char*)k_cache, (const unsigned char*)v_cache, num_pages, table, table_ld, cu_q, kv_lens, B, nh, nkv,
                        page_size, window, scale_log2, max_rows, csize, scratch, status);
  if (e != cudaSuccess) {
    cudaGetLastError();
    CO_FAIL("kv4_items: launch failed: %s", cudaGetErrorString(e));
  }
  CO_CHECK_LAUNCH("kv4_items");
  return 0;
}
}  // namespace

CO_EXPORT int coheryn_kv4_head_dim() { return HD; }

static int check_pages(const char* what, int nkv, int page_size, int num_pages) {
  if (nkv < 1 || page_size < 16 || page_size % 16) CO_FAIL("%s: %d kv heads, pages of %d positions (a multiple of 16)", what, nkv, page_size);
  if (num_pages < 1 || (long long)num_pages * page_size > 0x7fffffffLL)
    CO_FAIL("%s: %d pages of %d positions do not fit 32-bit slots", what, num_pages, page_size);
  return 0;
}

CO_EXPORT int coheryn_kv4_write(const void* qkv, long ld, int dtype, const int* positions, const float* cos_sin, int n_cos, const int* slots,
                                void* k_cache, void* v_cache, int num_pages, void* q_out, int T, int nh, int nkv, int rot, int page_size,
                                int* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (check_pages("kv4_write", nkv, page_size, num_pages)) return 1;
  if (rot < 0 || rot > HD || (rot & 1)) CO_FAIL("kv4_write: %d rotated channels of %d", rot, HD);
  if (nh < 0) CO_FAIL("kv4_write: %d heads", nh);
  const int align = dtype == CO_F32 ? 4 : 8;
  if (((uintptr_t)qkv & 15) || ld % align || ((uintptr_t)q_out & 15) || ((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) ||
      ((uintptr_t)cos_sin & 15))
    CO_FAIL("kv4_write: operands must be 16-byte aligned");
  const int first = rot ? 0 : nh;        // without a rotation there is nothing to do for the queries
  const int at_once = 256 / (HD / 8), rounds = (nh + 2 * nkv - first + at_once - 1) / at_once;
  if (rounds > 65535) CO_FAIL("kv4_write: %d heads", nh + 2 * nkv);
  const dim3 grid((unsigned)T, (unsigned)rounds);
  auto with = [&](auto* x) {
    typedef decltype(x) P;
    typedef std::remove_pointer_t<P> E;
    if (HD % 64 == 0 && (rot == HD || rot == 0))
      co_launch(rot ? kv4_write_halves_kernel<E, true> : kv4_write_halves_kernel<E, false>, grid, dim3(256), 0, stream, (P)qkv, ld, positions,
                (const float2*)cos_sin, n_cos, slots, (unsigned char*)k_cache, (unsigned char*)v_cache, num_pages, (P)q_out, nh, nkv, page_size, first,
                status);
    else
      co_launch(kv4_write_kernel<E>, grid, dim3(256), 0, stream, (P)qkv, ld, positions, (const float2*)cos_sin, n_cos, slots, (unsigned char*)k_cache,
                (unsigned char*)v_cache, num_pages, (P)q_out, nh, nkv, rot, page_size, first, status);
  };
  if (dtype == CO_F32) with((float*)nullptr);
  else with((bf16*)nullptr);
  CO_CHECK_LAUNCH("kv4_write");
  return 0;
}

constexpr int PAGES_F16 = 2;      // beside the dtype codes

static int launch_pages(const void* k_cache, const void* v_cache, int num_pages, int nkv, int page_size, const int* table, int table_ld,
                        int width, int slots, int n, const int* cu_q, const int* lens, int window, void* k_out, void* v_out, int dtype, int* out_table,
                        const float2* range, int parts, float2* factors, int* status, cudaStream_t stream) {
  if (nkv > 65535 || n > 65535) CO_FAIL("kv4_pages: %d requests, %d kv heads", n, nkv);
  const dim3 grid((unsigned)width, (unsigned)nkv, (unsigned)n);
  auto with = [&](auto* x) {
    typedef decltype(x) P;
    co_launch(kv4_pages_kernel<std::remove_pointer_t<P>>, grid, dim3(128), 0, stream, (const unsigned char*)k_cache, (const unsigned char*)v_cache,
              num_pages, nkv, page_size, table, table_ld, width, slots, cu_q, lens, window, (P)k_out, (P)v_out, out_table, range, parts, factors, status);
  };
  if (dtype == CO_F32) with((float*)nullptr);
  else if (dtype == PAGES_F16) with((__half*)nullptr);
  else with((bf16*)nullptr);
  CO_CHECK_LAUNCH("kv4_pages");
  return 0;
}

// pages [n] -> k_out, v_out [n, nkv, page_size, HD].
CO_EXPORT int coheryn_kv4_pages(const void* k_cache, const void* v_cache, int num_pages, int nkv, int page_size, const int* pages, int n,
                                void* k_out, void* v_out, int dtype, int* status, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (check_pages("kv4_pages", nkv, page_size, num_pages)) return 1;
  if (((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) || ((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15))
    CO_FAIL("kv4_pages: operands must be 16-byte aligned");
  return launch_pages(k_cache, v_cache, num_pages, nkv, page_size, pages, n, n, n, 1, nullptr, nullptr, 0, k_out, v_out, dtype, nullptr, nullptr, 0,
                      nullptr, status, stream);
}

// Into how many parts the float32 kernel cuts a row's tiles: one tile per warp at least, and no more CTAs than are resident.
CO_EXPORT int coheryn_kv4_simple_parts(int T, int nkv, int max_kv_len, int window) {
  if (max_kv_len <= 0 || T <= 0 || nkv <= 0) return 1;
  const int keys = window > 0 && window < max_kv_len ? window : max_kv_len;
  const long long by_size = ((long long)keys + 16 * SW - 1) / (16 * SW), by_slots = 148LL * 2 / ((long long)T * nkv);
  const long long parts = by_size < by_slots ? by_size : by_slots;
  return parts < 1 ? 1 : (int)parts;
}
CO_EXPORT long coheryn_kv4_simple_scratch_floats(int T, int nh, int parts) { return parts > 1 ? (long)T * nh * parts * (HD + 2) : 0; }

CO_EXPORT int coheryn_kv4_attention_simple(const void* q, long q_ld, void* out, long out_ld, int dtype, const void* k_cache, const void* v_cache,
                                           int num_pages, const int* table, int table_ld, int n_req, const int* token_req, const int* positions, int T,
                                           int nh, int nkv, int page_size, int window, float scale, int parts, float* scratch,
                                           long scratch_floats, int* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  if (check_pages("kv4_attention", nkv, page_size, num_pages)) return 1;
  if (nh < 1 || nh % nkv || nkv > 65535) CO_FAIL("kv4_attention: %d heads do not group over %d kv heads", nh, nkv);
  if (((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15)) CO_FAIL("kv4_attention: caches must be 16-byte aligned");
  if (parts < 1 || parts > 65535 || scratch_floats < coheryn_kv4_simple_scratch_floats(T, nh, parts))
    CO_FAIL("kv4_attention: %d parts in a scratch of %ld floats", parts, scratch_floats);
  const float scale_log2 = scale * 1.4426950408889634f;
  auto with = [&](auto* x) {
    typedef decltype(x) P;
    typedef std::remove_pointer_t<P> E;
    co_launch(nh / nkv <= 4 ? kv4_simple_kernel<E, 4> : kv4_simple_kernel<E, 8>, dim3((unsigned)T, (unsigned)nkv, (unsigned)parts), dim3(32 * SW), 0,
              stream, (P)q, q_ld, (P)out, out_ld, (const unsigned char*)k_cache, (const unsigned char*)v_cache, num_pages, table, table_ld, n_req, token_req,
              positions, nh, nkv, page_size, window, scale_log2, scratch, status);
    co_count_launch();
    if (parts > 1)
      co_launch(kv4_simple_join_kernel<E>, dim3((unsigned)(((long long)T * nh + 3) / 4)), dim3(128), 0, stream, (const float*)scratch, parts, (P)out,
                out_ld, nh, T * nh);
  };
  if (dtype == CO_F32) with((float*)nullptr);
  else with((bf16*)nullptr);
  CO_CHECK_LAUNCH("kv4_attention_simple");
  return 0;
}

// Floats of scratch that coheryn_kv4_attention needs; max_rows: the largest q_len * heads / kv_heads among the requests
// that it takes, max_kv_len: the most positions that one's rows see, from a multiple of 16 on.
CO_EXPORT long coheryn_kv4_scratch_floats(int B, int nkv, int max_rows, int max_kv_len) {
  const Split split = split_of(B, nkv, max_rows, max_kv_len);
  if (split.csize) return 0;
  const int cols = 8 * tiles_of(max_rows);
  return 2L * split.ctas * cols * (HD + 2) + 2L * B * nkv * ((max_rows + cols - 1) / cols);
}

// Attention of the requests with at most `max_rows` query rows per kv head, in bfloat16: q [T, nh * HD] of stride q_ld, out likewise;
// request b's rows are tokens cu_q[b] .. cu_q[b + 1], at the last positions of its kv_lens[b].  Other requests' rows are left.
CO_EXPORT int coheryn_kv4_attention(const void* q, long q_ld, void* out, long out_ld, const void* k_cache, const void* v_cache, int num_pages,
                                    const int* table, int table_ld, const int* cu_q, const int* kv_lens, int B, int nh, int nkv, int page_size,
                                    int window, float scale, int max_rows, int max_kv_len, float* scratch, long scratch_floats, int* status,
                                    cudaStream_t stream) {
  if (B <= 0 || max_rows <= 0) return 0;
  if (check_pages("kv4_attention", nkv, page_size, num_pages)) return 1;
  if (nh < 1 || nh % nkv || nkv > 65535) CO_FAIL("kv4_attention: %d heads do not group over %d kv heads", nh, nkv);
  if ((q_ld & 7) || (out_ld & 3) || ((uintptr_t)q & 15) || ((uintptr_t)out & 7) || ((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15))
    CO_FAIL("kv4_attention: q and the caches must be 16-byte aligned, out 8-byte");
  if (max_kv_len < 0 || B > 65535) CO_FAIL("kv4_attention: %d requests of at most %d positions", B, max_kv_len);
  if ((long long)B * nkv * ((max_rows + 7) / 8) * (max_kv_len / UNIT + 1LL + EXTRA) > 0x7fffffffLL)
    CO_FAIL("kv4_attention: %d requests of %d positions and %d kv heads", B, max_kv_len, nkv);
  const Split split = split_of(B, nkv, max_rows, max_kv_len);
  const int nt = tiles_of(max_rows), ctas = split.ctas, csize = split.csize;
  if (scratch_floats < coheryn_kv4_scratch_floats(B, nkv, max_rows, max_kv_len) || ((uintptr_t)scratch & 15))
    CO_FAIL("kv4_attention: the scratch is too small or not 16-byte aligned");
  constexpr int NT = HD <= 128 ? 2 : 1;
  auto launch = nt == 2 ? (csize ? launch_items<NT, 2, true> : launch_items<NT, 2, false>)
                : csize ? (split.per_sm == 2 ? launch_items<1, 2, true> : launch_items<1, FEWER, true>)
                : split.per_sm == MOST ? launch_items<1, MOST, false> : launch_items<1, FEWER, false>;
  const int rc = launch(q, q_ld, out, out_ld, k_cache, v_cache, num_pages, table, table_ld, cu_q, kv_lens, B, nh, nkv, page_size, window,
                        scale * 1.4426950408889634f, max_rows, ctas, csize ? csize : 1, scratch, status, stream);
  if (rc || csize || max_kv_len <= UNIT) return rc;    // joined already, or no list is longer than one unit
  const int cols = 8 * nt;
  const bool wide = ctas > 8LL * B * nkv * ((max_rows + cols - 1) / cols);
  co_launch(wide ? kv4_join_kernel<true> : kv4_join_kernel<false>, dim3((unsigned)(wide ? max_rows : (max_rows + cols - 1) / cols), (unsigned)nkv, (unsigned)B),
            dim3(32 * CW), 0, stream, (const float*)scratch, ctas, (bf16*)out, out_ld, cu_q, nh, nkv, cols, max_rows);
  CO_CHECK_LAUNCH("kv4_join");
  return 0;
}

// Floats that the factors of coheryn_kv4_expand take: two per list (request, kv head), then the partial answers that they are formed from.
CO_EXPORT long coheryn_kv4_factor_floats(int n, int nkv) {
  const long lists = (long)n * nkv;
  return 2 * lists + 2 * lists * range_parts(lists);
}

// The pages of requests b = 0..n-1 of a block table, dense: of request b's entries those that its new tokens see, `slots` at most,
// become pages b * slots.. of k_out and v_out [n * slots, nkv, page_size, HD], and out_table [n, width] says which (-1: not needed).  Rows at or
// behind a request's length, or in front of what its first new token sees, are zeros.  In bfloat16, or, with `factors` (float32
// [coheryn_kv4_factor_floats(n, nkv)]; place 2 (b nkv + kv head) gets what that list's keys have to be multiplied by, the next what its values do), in
// scaled float16.
CO_EXPORT int coheryn_kv4_expand(const void* k_cache, const void* v_cache, int num_pages, int nkv, int page_size, const int* table, int table_ld,
                                 int width, int slots, int n, const int* cu_q, const int* kv_lens, int window, void* k_out, void* v_out, int* out_table,
                                 float* factors, int* status, cudaStream_t stream) {
  if (n <= 0 || width <= 0) return 0;
  if (check_pages("kv4_expand", nkv, page_size, num_pages)) return 1;
  if (((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) || ((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15) || ((uintptr_t)factors & 7))
    CO_FAIL("kv4_expand: operands must be 16-byte aligned");
  if (width > table_ld || slots < 1) CO_FAIL("kv4_expand: %d entries of rows of %d, %d pages", width, table_ld, slots);
  const long long lists = (long long)n * nkv;
  const int parts = range_parts(lists);
  float2* range = factors ? reinterpret_cast<float2*>(factors) + lists : nullptr;
  if (factors) {
    if (lists * parts > 0x7fffffffLL) CO_FAIL("kv4_expand: %d requests of %d kv heads", n, nkv);
    co_launch(kv4_range_kernel, dim3((unsigned)(lists * parts)), dim3(32 * RANGE_WARPS), 0, stream, (const unsigned char*)k_cache, (const unsigned char*)v_cache,
              num_pages, nkv, page_size, table, table_ld, width, cu_q, kv_lens, window, parts, range);
    CO_CHECK_LAUNCH("kv4_range");
  }
  return launch_pages(k_cache, v_cache, num_pages, nkv, page_size, table, table_ld, width, slots, n, cu_q, kv_lens, window, k_out, v_out,
                      factors ? PAGES_F16 : CO_BF16, out_table, (const float2*)range, parts, reinterpret_cast<float2*>(factors), status, stream);
}

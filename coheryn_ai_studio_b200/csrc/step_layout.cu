// A step's index arrays from its requests' lengths and page lists.
//
// Request b holds starts[b] positions and brings q_lens[b] tokens; its pages are
// pages[page_cu[b] .. page_cu[b + 1]), for the table's entries from first[b] (0 without `first`) on:
//   cu_q[b + 1]     = q_lens[0] + .. + q_lens[b],          kv_lens[b] = starts[b] + q_lens[b]
//   token i of b:     position p = starts[b] + i, request b, slot = page(p / page_size) * page_size + p % page_size
//   table[b][j]     = pages[page_cu[b] + j - first[b]] from first[b] on, -1 behind the list; entries before
//                     first[b] stay, and with `first` so does what lies behind the list.
// Rows of positions, token_req and slots behind the last token are left as they are, and a slot whose page
// is missing or negative is -1.
//
// The step's arrays are a few hundred KB at most, so the call is bound by one launch; the table is the large one
// (256 requests of 32,768 positions: 2 MB).  Blocks are of two kinds: those of the first kind take TOKENS_PER_BLOCK tokens
// each and need the prefix sums, which every one of them forms for itself in shared memory (one pass over q_lens: at
// 256 requests a load and ten shuffles; a kernel of its own for the sums would cost a launch); those of the second
// kind write rows of the table and need none.
//
// An ordinary launch without an early start of its successor: kernels of a step look at its lengths and tables ahead of
// their own wait.
#include "common.cuh"

namespace {
constexpr int THREADS = 256;
constexpr int TOKENS_PER_BLOCK = 1024;
constexpr int TABLE_PER_BLOCK = 2048;   // table entries of one row
constexpr int MAX_REQUESTS = 12000;     // prefix sums in 48 KB of shared memory

constexpr int BAD_LENGTH = 51;          // status codes
constexpr int BAD_PAGES = 52;

struct Lists {
  const int* pages;
  const int* page_cu;
  const int* first;
  int n_pages;
};
// The list of request b: its first table entry, its place in `pages` and its length (0 when the offsets do not fit).
__device__ __forceinline__ bool list_of(const Lists& l, int b, int& first, int& from, int& n) {
  first = l.first ? l.first[b] : 0;
  from = l.page_cu[b];
  const int to = l.page_cu[b + 1];
  const bool ok = first >= 0 && from >= 0 && to >= from && to <= l.n_pages;
  n = ok ? to - from : 0;
  if (!ok) { first = first < 0 ? 0 : first; from = 0; }
  return ok;
}

__global__ void __launch_bounds__(THREADS)
step_layout_kernel(const int* __restrict__ starts, const int* __restrict__ q_lens, Lists lists, int B, int T, int page_size,
                   int* __restrict__ cu_q, int* __restrict__ kv_lens, int* __restrict__ positions, int* __restrict__ token_req,
                   int* __restrict__ table, int W, int* __restrict__ slots, int* __restrict__ status, int token_blocks, int chunks) {
  extern __shared__ int cu[];             // [B + 1], blocks of tokens
  __shared__ int warp_sums[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int bad = 0;
  if ((int)blockIdx.x >= token_blocks) {
    // Rows of the table, `chunks` blocks each: the row's list is looked up once.
    const int x = blockIdx.x - token_blocks, b = x / chunks, j0 = (x - b * chunks) * TABLE_PER_BLOCK;
    int first, from, n;
    list_of(lists, b, first, from, n);
    int* row = table + (long long)b * W;
    const int end = min(lists.first ? min(W, first + n) : W, j0 + TABLE_PER_BLOCK);
#pragma unroll 4
    for (int j = max(j0, first) + tid; j < end; j += THREADS) row[j] = j - first < n ? lists.pages[from + j - first] : -1;
    return;
  }
  // Prefix sums of the lengths: THREADS at a time, a warp scan and the warps' totals before it.
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += THREADS) {
    const int b = b0 + tid;
    int q = b < B ? q_lens[b] : 0;
    if (q < 0) { q = 0; bad = BAD_LENGTH; }
    int sum = q;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    int base = before, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) base += warp_sums[w];
      all += warp_sums[w];
    }
    if (b < B) cu[b + 1] = base + sum;
    before += all;
    __syncthreads();
  }
  if (tid == 0) cu[0] = 0;
  __syncthreads();
  if (blockIdx.x == 0) {
    if (cu_q)
      for (int b = tid; b <= B; b += THREADS) cu_q[b] = cu[b];
    for (int b = tid; b < B; b += THREADS) {
      const int s = starts[b], q = cu[b + 1] - cu[b];
      if (kv_lens) kv_lens[b] = s + q;
      int first, from, n;
      const bool ok = list_of(lists, b, first, from, n);
      if (s < 0 || (long long)s + q > 0x7fffffffLL || cu[b + 1] < cu[b]) bad = BAD_LENGTH;      // (the last: offsets beyond 32 bits)
      else if (!ok || (n && (long long)first + n > W)) bad = BAD_PAGES;
    }
    if (tid == 0 && (slots || positions || token_req) && cu[B] > T) bad = BAD_LENGTH;
  }
  const int tokens = min(cu[B], T);
  const int t0 = blockIdx.x * TOKENS_PER_BLOCK;
  for (int t = t0 + tid; t < min(tokens, t0 + TOKENS_PER_BLOCK); t += THREADS) {
    int lo = 0, hi = B;                    // cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    const int s = starts[lo], pos = s + (t - cu[lo]);
    if (positions) positions[t] = pos;
    if (token_req) token_req[t] = lo;
    if (slots) {
      int first, from, n, page = -1;
      list_of(lists, lo, first, from, n);
      const int j = pos < 0 ? -1 : pos / page_size;
      // Entries before `first` are not written by this call, so they may be read here.
      if (j >= first && j - first < n) page = lists.pages[from + j - first];
      else if (j >= 0 && j < first && j < W) page = table[(long long)lo * W + j];
      const long long slot = page < 0 ? -1 : (long long)page * page_size + (pos - j * page_size);
      if (slot < 0 || slot > 0x7fffffffLL) bad = pos < 0 ? BAD_LENGTH : BAD_PAGES;
      slots[t] = slot > 0x7fffffffLL ? -1 : (int)slot;
    }
  }
  if (bad && status) *status = bad;
}
}  // namespace

// cu_q [B + 1], kv_lens [B], positions [T], token_req [T] and slots [T] may be null; table [B, W] is written.
CO_EXPORT int coheryn_step_layout(const int* starts, const int* q_lens, const int* page_cu, const int* pages, int n_pages,
                                  const int* first, int B, int T, int page_size, int* cu_q, int* kv_lens, int* positions,
                                  int* token_req, int* table, int W, int* slots, int* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (B >= MAX_REQUESTS) CO_FAIL("step_layout: at most %d requests, not %d", MAX_REQUESTS - 1, B);
  if (page_size < 1 || W < 1 || T < 0 || n_pages < 0) CO_FAIL("step_layout: page size %d, table width %d, %d tokens", page_size, W, T);
  const Lists lists{pages, page_cu, first, n_pages};
  const int token_blocks = T > TOKENS_PER_BLOCK ? (T + TOKENS_PER_BLOCK - 1) / TOKENS_PER_BLOCK : 1;
  const int chunks = (W - 1) / TABLE_PER_BLOCK + 1;
  const long long table_blocks = (long long)B * chunks;
  if (token_blocks + table_blocks > 0x7fffffffLL) CO_FAIL("step_layout: a table of %d x %d entries", B, W);
  step_layout_kernel<<<dim3((unsigned)(token_blocks + table_blocks)), dim3(THREADS), sizeof(int) * (size_t)(B + 1), stream>>>(
      starts, q_lens, lists, B, T, page_size, cu_q, kv_lens, positions, token_req, table, W, slots, status, token_blocks, chunks);
  CO_CHECK_LAUNCH("step_layout");
  return 0;
}

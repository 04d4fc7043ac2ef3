// Which pages of a long context a token's attention reads.
//
// Scores: s[t, g, j] = max over the heads h of key head g's group of q[t, h] . means[page(t, j), g], for the full pages j before
// the token's own (j < position / page_size), -inf behind them and for pages the table does not hold.  Sums in 32-bit.
//
// Choice: per (token, key head) the first `first` pages, the last `recent` ones up to the token's own, and of the pages between
// the best-scored, `top` in all; of equal scores the lower page, what is not a number behind every number.  Ascending, -1 behind
// the last.
#include "mma_tiles.cuh"
#include "page_batch.cuh"
#include "umma_attention.cuh"

using namespace dinfer;
using dinfer_mma::cp_async16;
using dinfer_mma::cp_async_commit;
using dinfer_mma::cp_async_wait;
using dinfer_mma::mma_bf16;

namespace {

constexpr int WARPS = 8;

// Any sizes and types: a warp per (token, key head, page).
template <typename T>
__global__ void __launch_bounds__(WARPS * 32)
page_scores_kernel(const T* __restrict__ q, int64_t ldq, const T* __restrict__ means, int num_pages, const int* __restrict__ table,
                   int width, const int* __restrict__ cu, int num_reqs, const int* __restrict__ positions,
                   float* __restrict__ out, int64_t ldt, int64_t ldg, int H, int Hkv, int D, int page_size, int pages) {
  pdl_enter();
  const int t = blockIdx.x, g = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = request_of(cu, num_reqs, t);
  if (r < 0) return;
  const int group = H / Hkv, full = positions[t] / page_size;
  float* row = out + (int64_t)t * ldt + (int64_t)g * ldg;
  for (int j = blockIdx.z * WARPS + warp; j < pages; j += gridDim.z * WARPS) {
    float best = -INFINITY;
    const int page = j < full ? table[(int64_t)r * width + j] : -1;
    if (page >= 0 && page < num_pages) {
      const T* m = means + ((int64_t)page * Hkv + g) * D;
      for (int h = 0; h < group; ++h) {
        const T* x = q + (int64_t)t * ldq + (int64_t)(g * group + h) * D;
        float s = 0.f;
        for (int e = lane; e < D; e += 32) s = fmaf(to_f32<T>(x[e]), to_f32<T>(m[e]), s);
        s = warp_sum(s);
        best = h == 0 || s > best || s != s ? s : best;
        if (s != s) break;
      }
    }
    if (lane == 0) row[j] = best;
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {        // NaN where one of the two is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Bfloat16, head sizes 64 and 128, groups of up to 16 heads: a warp holds the means of 32 pages of a (request, key head) as the
// A operand of mma.sync and runs the tokens of its tile past them, eight columns (tokens x heads, the group filled up to a power of two
// with its last head) at a time.  Both operands go from memory straight into registers: the order of the elements of a sum is free, so a lane
// takes 16 bytes of its rows at the same places, two steps of 16 elements at once.  The maximum over the heads is taken in the columns.
constexpr int TILE_TOKENS = 64;

template <int D, int GP>             // GP: the group, filled up to a power of two
__global__ void __launch_bounds__(WARPS * 32)
page_scores_mma_kernel(const __nv_bfloat16* __restrict__ q, int64_t ldq, const __nv_bfloat16* __restrict__ means, int num_pages,
                       const int* __restrict__ table, int width, const int* __restrict__ cu, int num_reqs,
                       const int* __restrict__ positions, float* __restrict__ out, int64_t ldt, int64_t ldg, int group, int Hkv,
                       int page_size, int pages) {
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  const int g = blockIdx.y, j0 = (blockIdx.z * WARPS + warp) * 32;
  if (j0 >= pages) return;
  const int3 tile = token_tile(cu, num_reqs, TILE_TOKENS, blockIdx.x);
  if (tile.x < 0) return;
  constexpr int NT8 = GP > 8 ? GP / 8 : 1;                 // products of eight columns a step
  constexpr int STEP = GP > 8 ? 1 : 8 / GP;                // tokens of a step
  // rows gr + {0, 8, 16, 24}: pages j0 + ...; a page that is not held scores -inf
  unsigned held = 0;
  uint4 a[4][D / 32];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int j = j0 + gr + 8 * u;
    const int page = j < pages ? table[(int64_t)tile.x * width + j] : -1;
    const bool ok = page >= 0 && page < num_pages;
    const __nv_bfloat16* row = means + ((int64_t)(ok ? page : 0) * Hkv + g) * D + tq * 8;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) a[u][k] = ok ? *reinterpret_cast<const uint4*>(row + k * 32) : make_uint4(0, 0, 0, 0);
    held |= (ok ? 1u : 0u) << u;
  }
  auto load_q = [&](int i, uint4 (&b)[NT8][D / 32]) {
    const int t = tile.y + min(i + gr / GP, tile.z - 1);
#pragma unroll
    for (int n = 0; n < NT8; ++n) {
      const int h = min(GP > 8 ? n * 8 + gr : gr % GP, group - 1);
      const __nv_bfloat16* row = q + (int64_t)t * ldq + (int64_t)(g * group + h) * D + tq * 8;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) b[n][k] = *reinterpret_cast<const uint4*>(row + k * 32);
    }
  };
  uint4 b[NT8][D / 32];
  load_q(0, b);
  for (int i = 0; i < tile.z; i += STEP) {
    float c[2][4];
#pragma unroll
    for (int n = 0; n < NT8; ++n) {
      float d[2][4] = {};
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma_bf16(d[m], a[2 * m][k].x, a[2 * m + 1][k].x, a[2 * m][k].y, a[2 * m + 1][k].y, b[n][k].x, b[n][k].y);
          mma_bf16(d[m], a[2 * m][k].z, a[2 * m + 1][k].z, a[2 * m][k].w, a[2 * m + 1][k].w, b[n][k].z, b[n][k].w);
        }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[m][e] = n == 0 ? d[m][e] : max_nan(c[m][e], d[m][e]);
    }
    if (i + STEP < tile.z) load_q(i + STEP, b);
    // columns 2tq and 2tq + 1 -> tokens
    constexpr int MINE = GP == 1 ? 2 : 1;                  // tokens a lane writes
#pragma unroll
    for (int w = 0; w < MINE; ++w) {
      const int at = i + (GP >= 8 ? 0 : 2 * tq / GP) + w;
      const int t = tile.y + min(at, tile.z - 1);
      const int full = min(positions[t] / page_size, pages);
      const bool writes = at < tile.z && (GP >= 8 ? tq == 0 : 2 * tq % GP == 0);
      float* row = out + (int64_t)t * ldt + (int64_t)g * ldg + j0;
#pragma unroll
      for (int v = 0; v < 4; ++v) {                        // rows gr + 8 v
        float x = c[v / 2][2 * (v & 1) + w];
        if (GP > 1) {
          x = max_nan(x, c[v / 2][2 * (v & 1) + 1]);
          if (GP >= 4) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, 1));
          if (GP >= 8) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, 2));
        }
        const int j = gr + 8 * v;
        if (writes && j0 + j < pages) row[j] = (held >> v & 1) && j0 + j < full ? x : -INFINITY;
      }
    }
  }
}

// Bfloat16, head sizes 64 and 128, many tokens: 128 pages of a (request, key head) are the rows of a tcgen05.mma, up to 128 (token, head)
// pairs its columns (the group filled up to a power of two, GP, with its last head), D its depth; S comes out in tensor memory with a page
// to a lane, so that a thread takes the maximum over a token's heads among its own registers and a warp writes 32 pages of a
// token side by side.  A block keeps its pages and walks runs of tokens: while the products of a run are made, the next run's rows
// of q are on their way and the results of the run before are written.  Two blocks share an SM.  The waits for the products are
// bounded.  Bound by what it writes (4 bytes a token, key head and page) and by the rows of q from L2: 4096 tokens
// of 32 heads of 128 over 8 against 512 pages (102 MB, 16 GFLOP) take 40 us, 39 % of a copy's rate (the kernel above 114): the steps
// of a run (products, tensor memory, maxima, stores) and its barrier, tensor pipe 19 %.  256 pages a block with three buffers of rows, one
// block an SM, took 45 us.
constexpr int U_ROWS = 128, U_COLS = 128, U_NT = 256;
// From so many tokens on, and so many a request.  us, the kernel above and this one, 32 heads of 128 over 8, pages of 64: 64 tokens behind 28000 18.9
// and 6.2, 1024 tokens 26.8 and 13.4, 64 tokens behind 8000 beside 4 single ones 16.4 and 5.8, beside 62 20.6 and 15.1, 64 single ones 9.9 and
// 21.5 (a run holds tokens of one request).
constexpr int MANY_TOKENS = 16, MANY_TOKENS_A_REQUEST = 2;

template <int D, int GP>
__global__ void __launch_bounds__(U_NT, 2)
page_scores_umma_kernel(const __nv_bfloat16* __restrict__ q, int64_t ldq, const __nv_bfloat16* __restrict__ means, int num_pages,
                        const int* __restrict__ table, int width, const int* __restrict__ cu, int num_reqs,
                        const int* __restrict__ positions, float* __restrict__ out, int64_t ldt, int64_t ldg, int group, int Hkv,
                        int page_size, int pages, int tiles, int per_block, int* status) {
  using namespace dinfer_umma;
  constexpr int TOKENS = U_COLS / GP, NH = D / 64, C = D / 8;
  constexpr uint32_t A_HALF = U_ROWS * 128, B_HALF = U_COLS * 128;
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t s_done[2];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_full[3][TOKENS];                                // of the run before, this one and the next
  __shared__ volatile int s_abort;
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y, j0 = blockIdx.z * U_ROWS;
  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  unsigned char* sA = smem_dyn + (base - smem_u32(smem_dyn));      // [NH][128 pages][128 B], TMA's 128-byte swizzle
  unsigned char* sB = sA + NH * A_HALF;                            // [2][NH][128 columns][128 B]
  int y = blockIdx.x * per_block;
  const int end = min(tiles, y + per_block);
  int3 tile = y < end ? token_tile(cu, num_reqs, TOKENS, y) : make_int3(-1, 0, 0);
  if (tile.x < 0) return;                                          // (the whole block alike)
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&s_done[0]), 1);
    mbar_init(smem_u32(&s_done[1]), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(2 * U_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  // this thread's page: lane quarter warp % 4 of tensor memory, half of the columns warp / 4
  const int j = j0 + (warp & 3) * 32 + lane;
  bool held = false;
  auto load_pages = [&](int request) {
    const int* row_table = table + (int64_t)request * width;
    for (int i = threadIdx.x; i < U_ROWS * C; i += U_NT) {
      const int row = i / C, c = i % C;
      const int page = j0 + row < pages ? row_table[j0 + row] : -1;
      const bool ok = page >= 0 && page < num_pages;
      cp_async16(sA + (c >> 3) * A_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4), means + ((int64_t)(ok ? page : 0) * Hkv + g) * D + c * 8, ok);
    }
    const int page = j < pages ? row_table[j] : -1;
    held = page >= 0 && page < num_pages;
  };
  // this thread's copies of a run: the same 16 bytes of the same head of every STEP-th token (so many columns further on the swizzle is the same)
  constexpr int COLS = U_NT / C, STEP = COLS / GP;
  static_assert(COLS % 8 == 0 && COLS % GP == 0, "a thread's columns have one head and one swizzle");
  const int col0 = threadIdx.x / C, c0 = threadIdx.x % C;
  const uint32_t dst0 = (c0 >> 3) * B_HALF + col0 * 128 + (((c0 & 7) ^ (col0 & 7)) << 4);
  const __nv_bfloat16* src0 = q + (int64_t)(g * group + min(col0 % GP, group - 1)) * D + c0 * 8;
  auto load_tokens = [&](const int3& run, int b, int i0) {           // run number i0
    unsigned char* dst = sB + b * NH * B_HALF + dst0;
    const __nv_bfloat16* src = src0 + (int64_t)(run.y + col0 / GP) * ldq;
#pragma unroll
    for (int k = 0; k < U_COLS / COLS; ++k) {
      const bool ok = col0 / GP + k * STEP < run.z;
      cp_async16(dst + k * COLS * 128, ok ? src : q, ok);
      src += (int64_t)STEP * ldq;
    }
    cp_async_commit();
    if (threadIdx.x < TOKENS) s_full[i0 % 3][threadIdx.x] = threadIdx.x < run.z ? positions[run.y + threadIdx.x] / page_size : 0;
  };
  auto write = [&](const int3& run, int i) {                        // the results of products i
    const int b = i & 1;
    if (!mbar_wait(smem_u32(&s_done[b]), (i >> 1) & 1)) { s_abort = 1; atomicExch(status, 67); return; }
    tc_fence_after();
    const uint32_t addr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + b * U_COLS;
    constexpr int PER = 32 / GP;                                    // tokens of 32 columns
    const int* full = s_full[i % 3];
    const int mine = held ? j : 0x7fffffff;
#pragma unroll
    for (int u = 0; u < U_COLS / 64; ++u) {
      const int col = (warp >> 2) * (U_COLS / 2) + u * 32, first = col / GP;
      if (first >= run.z) break;                                    // (a warp alike)
      float v[32];
      tmem_ld32(addr + col, v);
      tmem_ld_wait();
      float* row = out + (int64_t)(run.y + first) * ldt + (int64_t)g * ldg + j;
      const int n = j < pages ? run.z - first : 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        float x = v[k * GP];
#pragma unroll
        for (int h = 1; h < GP; ++h) x = max_nan(x, v[k * GP + h]);
        if (k < n) *row = mine < full[first + k] ? x : -INFINITY;
        row += ldt;
      }
    }
  };
  int ends = cu[tile.x + 1];                                       // of the request
  load_pages(tile.x);
  load_tokens(tile, 0, 0);
  int3 before = make_int3(-1, 0, 0);                                // the run whose results are to be written
  for (int i = 0;; ++i) {
    const int b = i & 1;
    cp_async_wait<0>();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();                                               // the run is here; tensor memory b has been read
    if (s_abort) break;
    if (threadIdx.x == 0) {
      tc_fence_after();
      constexpr uint32_t idesc = idesc_bf16(U_ROWS, U_COLS, 0);
      const uint64_t da = desc_k_major(smem_u32(sA)), db = desc_k_major(smem_u32(sB) + b * NH * B_HALF);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        tc_mma(tmem + b * U_COLS, da + (uint64_t)(((k / 4) * A_HALF + (k % 4) * 32) >> 4),
               db + (uint64_t)(((k / 4) * B_HALF + (k % 4) * 32) >> 4), idesc, k > 0 ? 1u : 0u);
      tc_commit(smem_u32(&s_done[b]));
    }
    ++y;
    const bool same = y < end && tile.y + TOKENS < ends;
    int3 next = make_int3(tile.x, tile.y + TOKENS, min(TOKENS, ends - tile.y - TOKENS));
    if (!same) next = y < end ? token_tile(cu, num_reqs, TOKENS, y) : make_int3(-1, 0, 0);
    // the other buffer is free once the products before have been made
    if (before.x >= 0 && !mbar_wait(smem_u32(&s_done[b ^ 1]), ((i - 1) >> 1) & 1)) { s_abort = 1; atomicExch(status, 67); }
    if (same) load_tokens(next, b ^ 1, i + 1);
    if (before.x >= 0) write(before, i - 1);
    if (!same) {
      write(tile, i);
      if (next.x < 0) break;
      __syncthreads();                                             // (everyone has written: the lists of full pages are free)
      load_pages(next.x);
      load_tokens(next, b ^ 1, i + 1);
      ends = cu[next.x + 1];
      before.x = -1;
    } else {
      before = tile;
    }
    tile = next;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    if (s_abort)
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * U_COLS) : "memory");
  }
}

template <int D, int GP>
int run_scores_umma(const __nv_bfloat16* q, int64_t ldq, const __nv_bfloat16* means, int num_pages, const int* table, int width, const int* cu,
                    int num_reqs, const int* positions, float* out, int64_t ldt, int64_t ldg, int T, int group, int Hkv, int page_size,
                    int pages, int sms, int* status, cudaStream_t stream) {
  auto kernel = page_scores_umma_kernel<D, GP>;
  constexpr int smem = (D / 64) * (U_ROWS + 2 * U_COLS) * 128 + 1024, tokens = U_COLS / GP;
  static thread_local int set_for = -1;                            // the attribute belongs to the device
  int dev = 0;
  cudaGetDevice(&dev);
  if (set_for != dev) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return cuda_status("page_scores: shared memory");
    set_for = dev;
  }
  const int tiles = T / tokens + (num_reqs < T ? num_reqs : T), z = (pages + U_ROWS - 1) / U_ROWS;
  // a block's pages are loaded once for all its runs of tokens: as few blocks as fill the SMs twice over
  const int64_t fill = 2 * (int64_t)sms / ((int64_t)Hkv * z);
  const int blocks = fill < 1 ? 1 : (int)fill, per_block = (tiles + blocks - 1) / blocks;
  launch_pdl(kernel, dim3((tiles + per_block - 1) / per_block, Hkv, z), dim3(U_NT), smem, stream, q, ldq, means, num_pages, table, width, cu,
             num_reqs, positions, out, ldt, ldg, group, Hkv, page_size, pages, tiles, per_block, status);
  return cuda_status("page_scores (many tokens)");
}

// Scores as whole numbers of the same order, the lowest for what is not a number; none is 0.
__device__ __forceinline__ unsigned order_of(float s) {
  const int b = __float_as_int(s + 0.f);                      // -0 counts as 0
  const unsigned k = (unsigned)(b ^ ((b >> 31) | (int)0x80000000));
  return s == s ? k : 1u;
}

// Any sizes: a warp per (token, key head), the best of the rest again and again.
__global__ void __launch_bounds__(WARPS * 32)
choose_pages_kernel(const float* __restrict__ scores, int64_t ldt, int64_t ldg, const int* __restrict__ positions, int page_size,
                    int first, int recent, int top, int pages, int* __restrict__ out, int64_t rows, int Hkv) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int t = (int)(row / Hkv), g = (int)(row % Hkv);
  const int pos = positions[t];
  const int own = pos < 0 ? -1 : min(pos / page_size, pages - 1);
  const int lo = min(first, own + 1), hi = max(own + 1 - recent, lo);   // candidates are [lo, hi)
  const int picks = min(top - lo - (own + 1 - hi), hi - lo);
  const float* s = scores + (int64_t)t * ldt + (int64_t)g * ldg;
  int* dst = out + row * top;
  // the picks, best first: (order, lower page) below the one before
  unsigned long long last = ~0ull;
  unsigned long long bound = 0;
  for (int i = 0; i < picks; ++i) {
    unsigned long long best = 0;
    for (int j = lo + lane; j < hi; j += 32) {
      const unsigned long long key = ((unsigned long long)order_of(s[j]) << 32) | (0xffffffffu - (unsigned)j);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    last = bound = best;
  }
  // ascending: the first pages, the candidates at or above the last pick, the recent pages
  int at = 0;
  for (int j = lane; j < lo; j += 32) dst[j] = j;
  at = lo;
  if (picks > 0)
    for (int j0 = lo; j0 < hi; j0 += 32) {
      const int j = j0 + lane;
      const bool in = j < hi && (((unsigned long long)order_of(s[j]) << 32) | (0xffffffffu - (unsigned)j)) >= bound;
      const unsigned mask = __ballot_sync(0xffffffffu, in);
      if (in) dst[at + __popc(mask & ((1u << lane) - 1))] = j;
      at += __popc(mask);
    }
  for (int j = hi + lane; j <= own; j += 32) dst[at + j - hi] = j;
  at += own + 1 - hi;
  for (int i = at + lane; i < top; i += 32) dst[i] = -1;
}

// Up to 2048 pages: a warp per (token, key head), the candidates' orders in registers (page lo + 32 i + lane; 0: none), read once.
// First a bound that few more candidates reach than there are picks, to the upper bits: up to 32 picks by the lanes' own maxima (as
// many lanes as picks reach it), else counted over all.  The candidates that reach it go to a list in shared memory, ascending, and are
// ranked against one another; a pick's place among the picks is its place in the list.  Where too many reach the bound (equal
// scores) the order of the last pick is found bit by bit, and of the candidates of that order the lowest are taken.
// Bound by instructions: 4096 tokens of 8 key heads choosing 16 of up to 512 pages (41 MB) take 29 us, 22 % of a copy's rate (27 M warp
// instructions, issue slots 77 % busy); 8 single tokens 3.2.  A lane's pages side by side instead, for wider loads and no ballots, took 62.
constexpr int SHORT_LIST = 64;

template <int NPL>
__global__ void __launch_bounds__(WARPS * 32)
choose_registers_kernel(const float* __restrict__ scores, int64_t ldt, int64_t ldg, const int* __restrict__ positions, int page_size,
                        int first, int recent, int top, int pages, int* __restrict__ out, int rows, int Hkv) {
  __shared__ __align__(16) uint2 s_list[WARPS][SHORT_LIST + 2];   // (order, page)
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * WARPS + warp;
  if (row >= rows) return;
  const int t = row / Hkv, g = row - t * Hkv;
  const int pos = positions[t];
  const int own = pos < 0 ? -1 : min(pos / page_size, pages - 1);
  const int lo = min(first, own + 1), hi = max(own + 1 - recent, lo);   // candidates are [lo, hi)
  const int picks = min(top - lo - (own + 1 - hi), hi - lo);
  int* dst = out + (int64_t)row * top;
  const unsigned below = (1u << lane) - 1;
  int at = lo;
  for (int j = lane; j < lo; j += 32) dst[j] = j;
  if (picks == hi - lo) {
    for (int j = lo + lane; j < hi; j += 32) dst[j] = j;
    at = hi;
  } else if (picks > 0) {
    const float* s = scores + (int64_t)t * ldt + (int64_t)g * ldg + lo + lane;
    const int n_mine = hi - lo - lane;                       // this lane's candidates are 32 i < n_mine
    unsigned key[NPL], best = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) key[i] = __float_as_uint(32 * i < n_mine ? s[32 * i] : 0.f);
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      key[i] = 32 * i < n_mine ? order_of(__uint_as_float(key[i])) : 0u;
      best = max(best, key[i]);
    }
    unsigned bound = 0;
    if (picks <= 32) {
#pragma unroll
      for (int bit = 31; bit >= 18; --bit) {
        const unsigned tried = bound | (1u << bit);
        if (__popc(__ballot_sync(0xffffffffu, best >= tried)) >= picks) bound = tried;
      }
    } else {
#pragma unroll 1
      for (int bit = 31; bit >= 16; --bit) {
        const unsigned tried = bound | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) n += key[i] >= tried;
        if ((int)__reduce_add_sync(0xffffffffu, (unsigned)n) >= picks) bound = tried;
      }
    }
    bound = max(bound, 1u);
    int n = 0;
    uint2* list = s_list[warp];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const bool mine = key[i] >= bound;
      const unsigned in = __ballot_sync(0xffffffffu, mine);
      const int k = n + __popc(in & below);
      if (mine && k < SHORT_LIST) list[k] = make_uint2(key[i], (unsigned)(lo + 32 * i + lane));
      n += __popc(in);
    }
    if (n <= SHORT_LIST) {
      if (lane == 0) list[n] = make_uint2(0u, 0u);
      __syncwarp();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int me = lane + 32 * half;
        if (32 * half >= n) break;
        const uint2 a = me < n ? list[me] : make_uint2(0u, 0u);
        int above = 0;                                       // larger ones, and equal ones lower down
        for (int i = 0; i < n; i += 2) {
          const uint4 v = *reinterpret_cast<const uint4*>(list + i);
          above += (v.x > a.x - (i < me)) + (v.z > a.x - (i + 1 < me));
        }
        const bool in = me < n && above < picks;
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (in) dst[at + __popc(mask & below)] = (int)a.y;
        at += __popc(mask);
      }
    } else {
      unsigned last = 0;                                     // the largest order that at least `picks` candidates reach
#pragma unroll 1
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned tried = last | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) c += key[i] >= tried;
        if ((int)__reduce_add_sync(0xffffffffu, (unsigned)c) >= picks) last = tried;
      }
      int above = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) above += key[i] > last;
      int equal = picks - (int)__reduce_add_sync(0xffffffffu, (unsigned)above);
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const unsigned same = __ballot_sync(0xffffffffu, key[i] == last);
        const bool in = key[i] > last || (key[i] == last && __popc(same & below) < equal);
        equal = max(0, equal - __popc(same));
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        if (in) dst[at + __popc(mask & below)] = lo + 32 * i + lane;
        at += __popc(mask);
      }
    }
  }
  // behind the picks the recent pages
  for (int j = hi + lane; j <= own; j += 32) dst[at + j - hi] = j;
  at += own + 1 - hi;
  for (int i = at + lane; i < top; i += 32) dst[i] = -1;
}

// More pages, up to 16384: a block per (token, key head).  Up to 32 picks as above: the bound from the maxima of the block's threads, the
// candidates that reach it into a list (in no order: a rank among equals, and a place among the picks, go by the page), which one
// warp ranks.  512 tokens of 8 key heads over 2200 pages take 38 us (126 by the kernel for any sizes), over 8100 119 (561), over 16200 333
// (1072); one token 5.4 (35), 7 (160), 8.6 (376).
// Otherwise, or where too many reach the bound, the order of the last pick bit by bit over the block.
template <int NPL>
__global__ void __launch_bounds__(WARPS * 32)
choose_block_kernel(const float* __restrict__ scores, int64_t ldt, int64_t ldg, const int* __restrict__ positions, int page_size,
                    int first, int recent, int top, int pages, int* __restrict__ out, int Hkv) {
  __shared__ int s_count[2][WARPS];
  __shared__ unsigned s_best[WARPS * 32], s_bound;
  __shared__ uint2 s_list[SHORT_LIST];
  __shared__ int s_n;
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int t = (int)(row / Hkv), g = (int)(row % Hkv);
  const int pos = positions[t];
  const int own = pos < 0 ? -1 : min(pos / page_size, pages - 1);
  const int lo = min(first, own + 1), hi = max(own + 1 - recent, lo);
  const int picks = min(top - lo - (own + 1 - hi), hi - lo);
  int* dst = out + row * top;
  const float* s = scores + (int64_t)t * ldt + (int64_t)g * ldg;
  int turn = 0;
  auto total = [&](int n, int* before) {                     // of the block; before: of the warps below
    n = (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
    if (lane == 0) s_count[turn][warp] = n;
    __syncthreads();
    int sum = 0, below = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w == warp) below = sum;
      sum += s_count[turn][w];
    }
    if (before) *before = below;
    turn ^= 1;                                               // (the next sum's writes meet nobody still reading this one's)
    return sum;
  };
  for (int j = threadIdx.x; j < lo; j += WARPS * 32) dst[j] = j;
  int at = lo;
  if (picks == hi - lo) {
    for (int j = lo + threadIdx.x; j < hi; j += WARPS * 32) dst[j] = j;
    at = hi;
  } else if (picks > 0) {
    unsigned key[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int j = lo + i * WARPS * 32 + threadIdx.x;
      key[i] = j < hi ? order_of(s[j]) : 0u;
    }
    bool listed = false;
    if (picks <= 32) {
      unsigned best = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) best = max(best, key[i]);
      s_best[threadIdx.x] = best;
      if (threadIdx.x == 0) s_n = 0;
      __syncthreads();
      if (warp == 0) {
        unsigned b[WARPS], bound = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) b[w] = s_best[w * 32 + lane];
#pragma unroll 1
        for (int bit = 31; bit >= 16; --bit) {
          const unsigned tried = bound | (1u << bit);
          int n = 0;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) n += b[w] >= tried;
          if ((int)__reduce_add_sync(0xffffffffu, (unsigned)n) >= picks) bound = tried;
        }
        if (lane == 0) s_bound = max(bound, 1u);
      }
      __syncthreads();
      const unsigned bound = s_bound;
      if (best >= bound)
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (key[i] >= bound) {
            const int k = atomicAdd(&s_n, 1);
            if (k < SHORT_LIST) s_list[k] = make_uint2(key[i], (unsigned)(lo + i * WARPS * 32 + (int)threadIdx.x));
          }
      __syncthreads();
      const int n = s_n;
      listed = n <= SHORT_LIST;
      if (listed && warp == 0) {
        bool in[2];
        uint2 a[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int me = lane + 32 * half;
          a[half] = me < n ? s_list[me] : make_uint2(0u, 0u);
          int above = 0;                                     // larger ones, and equal ones of a lower page
          for (int i = 0; i < n; ++i) {
            const uint2 v = s_list[i];
            above += v.x > a[half].x || (v.x == a[half].x && v.y < a[half].y);
          }
          in[half] = me < n && above < picks;
        }
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (lane + 32 * half < n) s_list[lane + 32 * half].x = in[half];
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (in[half]) {
            int lower = 0;                                   // picks of a lower page
            for (int i = 0; i < n; ++i) {
              const uint2 v = s_list[i];
              lower += v.x && v.y < a[half].y;
            }
            dst[at + lower] = (int)a[half].y;
          }
      }
      if (listed) at += picks;
    }
    if (!listed) {
      unsigned last = 0;
#pragma unroll 1
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned tried = last | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) n += key[i] >= tried;
        if (total(n, nullptr) >= picks) last = tried;
      }
      int above = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) above += key[i] > last;
      int equal = picks - total(above, nullptr);
#pragma unroll 1
      for (int i0 = 0; i0 < NPL; ++i0) {
        unsigned k = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) k = i == i0 ? key[i] : k;
        int below;
        const unsigned same = __ballot_sync(0xffffffffu, k == last);
        const int sames = total(lane == 0 ? __popc(same) : 0, &below);
        const bool in = k > last || (k == last && below + __popc(same & ((1u << lane) - 1)) < equal);
        equal = max(0, equal - sames);
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        const int ins = total(lane == 0 ? __popc(mask) : 0, &below);
        if (in) dst[at + below + __popc(mask & ((1u << lane) - 1))] = lo + i0 * WARPS * 32 + threadIdx.x;
        at += ins;
      }
    }
  }
  for (int j = hi + threadIdx.x; j <= own; j += WARPS * 32) dst[at + j - hi] = j;
  at += own + 1 - hi;
  for (int i = at + threadIdx.x; i < top; i += WARPS * 32) dst[i] = -1;
}

}  // namespace

// out[t * ldt + g * ldg + j] for j < pages; rows behind the last request's tokens are left as they are.
// (The arguments of the calls lie in one struct, 8 bytes a field: a caller packs them and hands over one address.)
struct PageScoresArgs {
  const void* q;
  int64_t ldq;
  const void* means;
  int64_t num_pages;
  const int* table;
  int64_t width;
  const int* cu_seqlens;
  int64_t num_reqs;
  const int* positions;
  float* out;
  int64_t ldt, ldg, T, H, Hkv, D, page_size, pages, dtype, sms;
  int* status;                   // of the kernels with bounded waits
  cudaStream_t stream;
};

DINFER_API int dinfer_page_scores(const PageScoresArgs* a) {
  const void *q = a->q, *means = a->means;
  const int64_t ldq = a->ldq, ldt = a->ldt, ldg = a->ldg, most = 0x7fffffff;
  const int *table = a->table, *cu_seqlens = a->cu_seqlens, *positions = a->positions;
  float* out = a->out;
  cudaStream_t stream = a->stream;
  if (a->T > most || a->num_pages > most || a->width > most || a->num_reqs >= most || a->H > most || a->Hkv > most || a->D > most || a->page_size > most || a->pages > most)
    return refuse(DINFER_BAD_ARGUMENT, "page_scores: a size beyond 32 bits");
  const int num_pages = (int)a->num_pages, width = (int)a->width, num_reqs = (int)a->num_reqs, T = (int)a->T, H = (int)a->H, Hkv = (int)a->Hkv,
            D = (int)a->D, page_size = (int)a->page_size, pages = (int)a->pages, dtype = (int)a->dtype;
  if (T < 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || page_size <= 0 || num_reqs <= 0 || pages < 0 || pages > width)
    return refuse(DINFER_BAD_ARGUMENT, "page_scores: sizes T=%d H=%d Hkv=%d D=%d page=%d pages=%d of %d", T, H, Hkv, D,
                  page_size, pages, width);
  if (T == 0 || pages == 0) return DINFER_OK;
  if (Hkv > 65535) return refuse(DINFER_BAD_ARGUMENT, "page_scores: %d key heads", Hkv);
  const int group = H / Hkv;
  const int64_t z = ((int64_t)pages + WARPS * 32 - 1) / (WARPS * 32);
  if (dtype == DINFER_BF16 && (D == 64 || D == 128) && group <= 16 && ldq % 8 == 0 && ((uintptr_t)q | (uintptr_t)means) % 16 == 0 && z <= 65535) {
    if (a->status && T >= MANY_TOKENS && T >= MANY_TOKENS_A_REQUEST * (int64_t)num_reqs && ((int64_t)pages + U_ROWS - 1) / U_ROWS <= 65535) {
      const __nv_bfloat16 *qb = (const __nv_bfloat16*)q, *mb = (const __nv_bfloat16*)means;
      const int sms = (int)a->sms;
#define DINFER_SCORES(GP)                                                                                                              \
  return D == 64 ? run_scores_umma<64, GP>(qb, ldq, mb, num_pages, table, width, cu_seqlens, num_reqs, positions, out, ldt, ldg, T, group, \
                                           Hkv, page_size, pages, sms, a->status, stream)                                              \
                 : run_scores_umma<128, GP>(qb, ldq, mb, num_pages, table, width, cu_seqlens, num_reqs, positions, out, ldt, ldg, T, group, \
                                            Hkv, page_size, pages, sms, a->status, stream)
      if (group == 1) DINFER_SCORES(1);
      if (group == 2) DINFER_SCORES(2);
      if (group <= 4) DINFER_SCORES(4);
      if (group <= 8) DINFER_SCORES(8);
      DINFER_SCORES(16);
#undef DINFER_SCORES
    }
    const int64_t tiles = (int64_t)T / TILE_TOKENS + (num_reqs < T ? num_reqs : T);     // of every way the tokens may be dealt out
    const dim3 grid((unsigned)tiles, Hkv, (unsigned)z);
#define DINFER_SCORES(GP)                                                                                                       \
  launch_pdl(D == 64 ? page_scores_mma_kernel<64, GP> : page_scores_mma_kernel<128, GP>, grid, dim3(WARPS * 32), 0, stream,   \
             (const __nv_bfloat16*)q, ldq, (const __nv_bfloat16*)means, num_pages, table, width, cu_seqlens, num_reqs,       \
             positions, out, ldt, ldg, group, Hkv, page_size, pages)
    if (group == 1) DINFER_SCORES(1);
    else if (group == 2) DINFER_SCORES(2);
    else if (group <= 4) DINFER_SCORES(4);
    else if (group <= 8) DINFER_SCORES(8);
    else DINFER_SCORES(16);
#undef DINFER_SCORES
    return cuda_status("page_scores");
  }
  DINFER_DISPATCH_DTYPE(dtype, E, {
    launch_pdl(page_scores_kernel<E>, dim3(T, Hkv, min((pages + WARPS - 1) / WARPS, 64)), dim3(WARPS * 32), 0, stream, (const E*)q,
               ldq, (const E*)means, num_pages, table, width, cu_seqlens, num_reqs, positions, out, ldt, ldg, H, Hkv, D,
               page_size, pages);
    return cuda_status("page_scores");
  });
}

// scores [t * ldt + g * ldg + j], j < pages; out int32 [T, Hkv, top].  recent >= 1 (a token's own page is always read).
struct ChoosePagesArgs {
  const float* scores;
  int64_t ldt, ldg;
  const int* positions;
  int64_t page_size, first, recent, top, pages;
  int* out;
  int64_t T, Hkv;
  cudaStream_t stream;
};

DINFER_API int dinfer_choose_pages(const ChoosePagesArgs* a) {
  const float* scores = a->scores;
  const int64_t ldt = a->ldt, ldg = a->ldg, most = 0x3fffffff;
  const int* positions = a->positions;
  int* out = a->out;
  cudaStream_t stream = a->stream;
  if (a->page_size > most || a->first > most || a->recent > most || a->top > most || a->pages > most || a->T > most || a->Hkv > most)
    return refuse(DINFER_BAD_ARGUMENT, "choose_pages: a size beyond 30 bits");
  const int page_size = (int)a->page_size, first = (int)a->first, recent = (int)a->recent, top = (int)a->top, pages = (int)a->pages,
            T = (int)a->T, Hkv = (int)a->Hkv;
  if (T < 0 || Hkv <= 0 || page_size <= 0 || pages <= 0 || first < 0 || recent < 1 || top < first + recent)
    return refuse(DINFER_BAD_ARGUMENT, "choose_pages: sizes T=%d Hkv=%d page=%d pages=%d, %d first and %d recent of %d", T, Hkv,
                  page_size, pages, first, recent, top);
  if (T == 0) return DINFER_OK;
  const int64_t rows = (int64_t)T * Hkv;
  if (pages > 2048 && pages <= 16384 && rows <= 0x7fffffff) {
    auto kernel = pages <= 4096 ? choose_block_kernel<16> : pages <= 8192 ? choose_block_kernel<32> : choose_block_kernel<64>;
    launch_pdl(kernel, dim3((unsigned)rows), dim3(WARPS * 32), 0, stream, scores, ldt, ldg, positions, page_size, first, recent, top,
               pages, out, Hkv);
    return cuda_status("choose_pages");
  }
  if (pages <= 2048 && rows <= 0x7fffffff - WARPS) {
    auto kernel = pages <= 128 ? choose_registers_kernel<4> : pages <= 256 ? choose_registers_kernel<8>
                  : pages <= 512 ? choose_registers_kernel<16> : pages <= 1024 ? choose_registers_kernel<32>
                  : choose_registers_kernel<64>;
    launch_pdl(kernel, dim3((unsigned)((rows + WARPS - 1) / WARPS)), dim3(WARPS * 32), 0, stream, scores, ldt, ldg, positions,
               page_size, first, recent, top, pages, out, (int)rows, Hkv);
    return cuda_status("choose_pages");
  }
  launch_pdl(choose_pages_kernel, dim3((unsigned)((rows + WARPS - 1) / WARPS)), dim3(WARPS * 32), 0, stream, scores, ldt, ldg,
             positions, page_size, first, recent, top, pages, out, rows, Hkv);
  return cuda_status("choose_pages");
}

DINFER_DEFINE_LAST_ERROR()

// Which pages of a long context a token's attention reads.
//
// Scores: s[t, g, j] = max over the heads h of key head g's group of q[t, h] . means[page(t, j), g], for the full pages j before
// the token's own (j < position / page_size), -inf behind them and for pages the table does not hold.  Sums in 32-bit.
//
// Choice: per (token, key head) the first `first` pages, the last `recent` ones up to the token's own, and of the pages between
// the best-scored, `top` in all; of equal scores the lower page, what is not a number behind every number.  Ascending, -1 behind
// the last.
#include "common.cuh"

using namespace dinfer;

namespace {

// last r with cu_seqlens[r] <= t (requests without tokens are passed over), -1 behind the last request's tokens
__device__ __forceinline__ int request_of(const int* cu, int num_reqs, int t) {
  if (t >= cu[num_reqs] || t < cu[0]) return -1;
  int lo = 0, hi = num_reqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

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

// Scores as whole numbers of the same order; 0 for what is not a number, 1 for -inf.
__device__ __forceinline__ unsigned order_of(float s) {
  if (s != s) return 0u;
  const unsigned b = __float_as_uint(s + 0.f);                // -0 counts as 0
  return (b & 0x80000000u ? ~b : b | 0x80000000u) - 0x007fffffu + 1u;
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

}  // namespace

// out[t * ldt + g * ldg + j] for j < pages; rows behind the last request's tokens are left as they are.
DINFER_API int dinfer_page_scores(const void* q, int64_t ldq, const void* means, int num_pages, const int* table, int width,
                                  const int* cu_seqlens, int num_reqs, const int* positions, float* out, int64_t ldt, int64_t ldg,
                                  int T, int H, int Hkv, int D, int page_size, int pages, int dtype, cudaStream_t stream) {
  if (T < 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || page_size <= 0 || num_reqs <= 0 || pages < 0 || pages > width)
    return refuse(DINFER_BAD_ARGUMENT, "page_scores: sizes T=%d H=%d Hkv=%d D=%d page=%d pages=%d of %d", T, H, Hkv, D,
                  page_size, pages, width);
  if (T == 0 || pages == 0) return DINFER_OK;
  if (Hkv > 65535) return refuse(DINFER_BAD_ARGUMENT, "page_scores: %d key heads", Hkv);
  DINFER_DISPATCH_DTYPE(dtype, E, {
    launch_pdl(page_scores_kernel<E>, dim3(T, Hkv, min((pages + WARPS - 1) / WARPS, 64)), dim3(WARPS * 32), 0, stream, (const E*)q,
               ldq, (const E*)means, num_pages, table, width, cu_seqlens, num_reqs, positions, out, ldt, ldg, H, Hkv, D,
               page_size, pages);
    return cuda_status("page_scores");
  });
}

// scores [t * ldt + g * ldg + j], j < pages; out int32 [T, Hkv, top].  recent >= 1 (a token's own page is always read).
DINFER_API int dinfer_choose_pages(const float* scores, int64_t ldt, int64_t ldg, const int* positions, int page_size, int first,
                                   int recent, int top, int pages, int* out, int T, int Hkv, cudaStream_t stream) {
  if (T < 0 || Hkv <= 0 || page_size <= 0 || pages <= 0 || first < 0 || recent < 1 || top < first + recent)
    return refuse(DINFER_BAD_ARGUMENT, "choose_pages: sizes T=%d Hkv=%d page=%d pages=%d, %d first and %d recent of %d", T, Hkv,
                  page_size, pages, first, recent, top);
  if (T == 0) return DINFER_OK;
  const int64_t rows = (int64_t)T * Hkv;
  launch_pdl(choose_pages_kernel, dim3((unsigned)((rows + WARPS - 1) / WARPS)), dim3(WARPS * 32), 0, stream, scores, ldt, ldg,
             positions, page_size, first, recent, top, pages, out, rows, Hkv);
  return cuda_status("choose_pages");
}

DINFER_DEFINE_LAST_ERROR()

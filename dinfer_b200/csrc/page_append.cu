// After the q/k/v projection of attention over chosen pages: a token's heads normed and turned, q into rows of its own, k and v
// into the token's slot of the paged cache, and for every page that becomes full the mean of its keys:
//
//     q, k: x / sqrt(mean(x^2) + eps) * w, then the first `rot` elements turned by the token's row of the angle table
//           (pairs (i, i + rot/2), or (2i, 2i + 1) with `interleaved`);  v: as it is
//     means[page, g] = (1 / page_size) sum over the page's offsets o of the cached key (rounded as it is cached)
//
// The projection's rows are only read, so the call may be repeated.  A page is full when its last offset is written; the token
// that writes it makes the mean.  The page's other keys are taken from this step's rows where this step brings them (made again:
// no block waits for another's store) and from the cache where an earlier step did, so that a mean does not depend on how a
// prompt was cut into portions.  32-bit arithmetic, one rounding to the storage type at the end.
//
// Layouts: qkv [T, (H + 2 Hkv) D], cache [pages, 2, Hkv, page_size, D], means [pages, Hkv, D]; slot = page * page_size + offset,
// -1 for a row that is not kept (padding).
#include "common.cuh"

using namespace dinfer;

namespace {

constexpr int WARPS = 8;
constexpr int MAX_D = 512;

struct Append {
  int64_t ld, ldq;
  const int* positions;
  float eps;
  const float* cos_sin;
  int table_rows, rot, interleaved;
  const int* slots;
  int num_pages, page_size, H, Hkv, D;
};

// One head's row by one warp, any size: normed and turned into xs (32-bit, [D]).
template <typename TA, typename TW>
__device__ void finish_row(const TA* x, const TW* w, const float* cs, const Append& p, float* xs, int lane) {
  float ss = 0.f;
  for (int e = lane; e < p.D; e += 32) {
    const float v = to_f32<TA>(x[e]);
    xs[e] = v;
    ss += v * v;
  }
  if (w) {
    const float rinv = rsqrtf(warp_sum(ss) / (float)p.D + p.eps);
    for (int e = lane; e < p.D; e += 32) xs[e] = xs[e] * rinv * to_f32<TW>(w[e]);
  }
  __syncwarp();
  const int half = p.rot >> 1;
  for (int i = lane; i < half; i += 32) {                     // a pair belongs to one lane
    const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + half;
    const float u = xs[a], v = xs[b], c = cs[i], s = cs[half + i];
    xs[a] = u * c - v * s;
    xs[b] = v * c + u * s;
  }
  __syncwarp();
}

// The token's row of the angle table.  The caller's table reaches its positions; one it does not reach reads row 0.
__device__ __forceinline__ const float* angles(const Append& p, int t) {
  if (p.rot == 0) return nullptr;
  const int pos = p.positions[t];
  return p.cos_sin + (int64_t)(pos >= 0 && pos < p.table_rows ? pos : 0) * p.rot;
}

template <typename TA, typename TW>
__global__ void __launch_bounds__(WARPS * 32)
append_kernel(const TA* __restrict__ qkv, TA* __restrict__ q_out, const TW* __restrict__ q_weight,
              const TW* __restrict__ k_weight, TA* cache, TA* __restrict__ means, const Append p) {
  __shared__ float sm[WARPS][MAX_D];
  pdl_enter();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = p.slots[t];
  const bool kept = slot >= 0 && slot / p.page_size < p.num_pages;
  const int page = kept ? slot / p.page_size : 0, off = kept ? slot % p.page_size : 0;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * p.D;
  float* xs = sm[warp];
  const float* cs = angles(p, t);
  const TA* row = qkv + (int64_t)t * p.ld;
  for (int head = warp; head < p.H + 2 * p.Hkv; head += WARPS) {
    const TA* x = row + (int64_t)head * p.D;
    if (head >= p.H + p.Hkv) {
      if (kept) {
        TA* dst = cache + ((int64_t)page * 2 + 1) * plane + ((int64_t)(head - p.H - p.Hkv) * p.page_size + off) * p.D;
        for (int e = lane; e < p.D; e += 32) dst[e] = x[e];
      }
      continue;
    }
    if (head >= p.H && !kept) continue;
    finish_row<TA, TW>(x, head < p.H ? q_weight : k_weight, cs, p, xs, lane);
    TA* dst = head < p.H ? q_out + (int64_t)t * p.ldq + (int64_t)head * p.D
                         : cache + (int64_t)page * 2 * plane + ((int64_t)(head - p.H) * p.page_size + off) * p.D;
    for (int e = lane; e < p.D; e += 32) dst[e] = from_f32<TA>(xs[e]);
    __syncwarp();
  }
  if (!kept || off != p.page_size - 1) return;
  // the page is full: its mean, a warp per key head
  for (int g = warp; g < p.Hkv; g += WARPS) {
    float sum[MAX_D / 32] = {};
    for (int o = 0; o < p.page_size; ++o) {
      const int back = p.page_size - 1 - o, u = t - back;
      if (u >= 0 && p.slots[u] == slot - back) {               // brought by this step
        finish_row<TA, TW>(qkv + (int64_t)u * p.ld + (int64_t)(p.H + g) * p.D, k_weight, angles(p, u), p, xs, lane);
#pragma unroll
        for (int i = 0; i < MAX_D / 32; ++i)
          if (lane + 32 * i < p.D) sum[i] += to_f32<TA>(from_f32<TA>(xs[lane + 32 * i]));
        __syncwarp();
      } else {
        const TA* k = cache + (int64_t)page * 2 * plane + ((int64_t)g * p.page_size + o) * p.D;
#pragma unroll
        for (int i = 0; i < MAX_D / 32; ++i)
          if (lane + 32 * i < p.D) sum[i] += to_f32<TA>(k[lane + 32 * i]);
      }
    }
    TA* dst = means + ((int64_t)page * p.Hkv + g) * p.D;
#pragma unroll
    for (int i = 0; i < MAX_D / 32; ++i)
      if (lane + 32 * i < p.D) dst[lane + 32 * i] = from_f32<TA>(sum[i] / (float)p.page_size);
  }
}

template <typename TA, typename TW>
int run(const void* qkv, void* q_out, const void* qw, const void* kw, void* cache, void* means, const Append& p, int T,
        cudaStream_t stream) {
  launch_pdl(append_kernel<TA, TW>, dim3(T), dim3(WARPS * 32), 0, stream, (const TA*)qkv, (TA*)q_out, (const TW*)qw,
             (const TW*)kw, (TA*)cache, (TA*)means, p);
  return cuda_status("page_append");
}

}  // namespace

// w_dtype: element type of the norm weights (both given or neither).  cos_sin: f32 [table_rows, rot], rot 0: no rotation.
DINFER_API int dinfer_page_append(const void* qkv, int64_t ld, const int* positions, const void* q_weight,
                                  const void* k_weight, float eps, const float* cos_sin, int table_rows, int rot,
                                  int interleaved, void* q_out, int64_t ldq, void* cache, void* means, const int* slots,
                                  int num_pages, int page_size, int T, int H, int Hkv, int D, int dtype, int w_dtype,
                                  cudaStream_t stream) {
  if (T < 0 || H <= 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || num_pages < 0)
    return refuse(DINFER_BAD_ARGUMENT, "page_append: sizes T=%d H=%d Hkv=%d D=%d page=%d", T, H, Hkv, D, page_size);
  if (D > MAX_D) return refuse(DINFER_BAD_ARGUMENT, "page_append: head size %d is above %d", D, MAX_D);
  if (rot < 0 || rot > D || rot % 2 || (rot > 0 && (!cos_sin || table_rows <= 0)))
    return refuse(DINFER_BAD_ARGUMENT, "page_append: %d turned elements of %d, %d angle rows", rot, D, table_rows);
  if (T == 0) return DINFER_OK;
  const Append p{ld, ldq, positions, eps, cos_sin, table_rows, rot, interleaved, slots, num_pages, page_size, H, Hkv, D};
  DINFER_DISPATCH_DTYPE(dtype, TA, {
    DINFER_DISPATCH_DTYPE(w_dtype, TW, { return (run<TA, TW>(qkv, q_out, q_weight, k_weight, cache, means, p, T, stream)); });
  });
}

DINFER_DEFINE_LAST_ERROR()

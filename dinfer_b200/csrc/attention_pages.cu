// Attention over chosen pages of the paged cache: token t at position p, head h of key head g's group, reads the keys of the
// pages chosen[t, g, :] (-1: none) up to its own position,
//
//     out[t, h] = sum_i softmax_i(scale q[t, h] . k_i) v_i      over  { i <= p : i / page_size in chosen[t, g] }
//
// A page named twice counts twice; a number outside the request's table, or a page the table does not hold, is no page; a token
// that sees no key gets zeros; rows behind the last request's tokens are left as they are.  Scores, weights and sums in 32-bit.
// What a token does not see is never multiplied, so that it may hold anything.
#include "common.cuh"

using namespace dinfer;

namespace {

__device__ __forceinline__ int request_of(const int* cu, int num_reqs, int t) {
  if (t >= cu[num_reqs] || t < cu[0]) return -1;
  int lo = 0, hi = num_reqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

struct Pages {
  int64_t ldq, ldo;
  int num_pages;
  const int* table;
  int width;
  const int* cu;
  int num_reqs;
  const int* positions;
  const int* chosen;
  int top, T, H, Hkv, D, page_size;
  float scale;
};

constexpr int WARPS = 4;
constexpr int KEYS = 4;

// Any sizes: a warp per (token, head), the lanes split the elements, four keys at a time.
template <typename T, int C>   // C >= ceil(D / 32)
__global__ void __launch_bounds__(WARPS * 32)
attention_pages_kernel(const T* __restrict__ q, T* __restrict__ out, const T* __restrict__ cache, const Pages p) {
  pdl_enter();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y * WARPS + warp;
  if (h >= p.H) return;
  const int r = request_of(p.cu, p.num_reqs, t);
  if (r < 0) return;
  const int* table = p.table + (int64_t)r * p.width;
  const int g = h / (p.H / p.Hkv), pos = p.positions[t];
  const int* chosen = p.chosen + ((int64_t)t * p.Hkv + g) * p.top;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * p.D;
  float qv[C], acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = lane + 32 * c;
    qv[c] = e < p.D ? to_f32<T>(q[(int64_t)t * p.ldq + (int64_t)h * p.D + e]) * p.scale : 0.f;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < p.top; ++i) {
    const int j = chosen[i];
    if (j < 0 || j >= p.width) continue;
    const int page = table[j];
    if (page < 0 || page >= p.num_pages) continue;
    const int64_t keys = min((int64_t)p.page_size, pos - (int64_t)j * p.page_size + 1);
    const T* kp = cache + (int64_t)page * 2 * plane + (int64_t)g * p.page_size * p.D;
    for (int o = 0; o < keys; o += KEYS) {
      float s[KEYS];
#pragma unroll
      for (int u = 0; u < KEYS; ++u) {
        s[u] = 0.f;
        if (o + u < keys)
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (lane + 32 * c < p.D) s[u] = fmaf(qv[c], to_f32<T>(kp[(int64_t)(o + u) * p.D + lane + 32 * c]), s[u]);
      }
      float n = m;
#pragma unroll
      for (int u = 0; u < KEYS; ++u) {
        s[u] = o + u < keys ? warp_sum(s[u]) : -INFINITY;
        n = fmaxf(n, s[u]);
      }
      const float base = n == -INFINITY ? 0.f : n;
      const float alpha = expf(m - base);
      l *= alpha;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] *= alpha;
#pragma unroll
      for (int u = 0; u < KEYS; ++u) {
        if (o + u >= keys) break;
        const float w = expf(s[u] - base);
        l += w;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (lane + 32 * c < p.D) acc[c] = fmaf(w, to_f32<T>(kp[plane + (int64_t)(o + u) * p.D + lane + 32 * c]), acc[c]);
      }
      m = n;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = lane + 32 * c;
    if (e < p.D) out[(int64_t)t * p.ldo + (int64_t)h * p.D + e] = from_f32<T>(acc[c] * inv);
  }
}

template <typename T>
int run(const void* q, void* out, const void* cache, const Pages& p, cudaStream_t stream) {
  const dim3 grid(p.T, (p.H + WARPS - 1) / WARPS), block(WARPS * 32);
  if (p.D <= 64) launch_pdl(attention_pages_kernel<T, 2>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  else if (p.D <= 128) launch_pdl(attention_pages_kernel<T, 4>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  else launch_pdl(attention_pages_kernel<T, 16>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  return cuda_status("attention_pages");
}

}  // namespace

// chosen int32 [T, Hkv, top]; cache [num_pages, 2, Hkv, page_size, D].
DINFER_API int dinfer_attention_pages(const void* q, int64_t ldq, void* out, int64_t ldo, const void* cache, int num_pages,
                                      const int* table, int width, const int* cu_seqlens, int num_reqs, const int* positions,
                                      const int* chosen, int top, int T, int H, int Hkv, int D, int page_size, float scale,
                                      int dtype, cudaStream_t stream) {
  if (T < 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 512 || page_size <= 0 || num_reqs <= 0 || top <= 0 || width < 0)
    return refuse(DINFER_BAD_ARGUMENT, "attention_pages: sizes T=%d H=%d Hkv=%d D=%d page=%d top=%d", T, H, Hkv, D, page_size, top);
  if ((H + WARPS - 1) / WARPS > 65535) return refuse(DINFER_BAD_ARGUMENT, "attention_pages: %d heads", H);
  if (T == 0) return DINFER_OK;
  const Pages p{ldq, ldo, num_pages, table, width, cu_seqlens, num_reqs, positions, chosen, top, T, H, Hkv, D, page_size, scale};
  DINFER_DISPATCH_DTYPE(dtype, E, { return run<E>(q, out, cache, p, stream); });
}

DINFER_DEFINE_LAST_ERROR()

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

// ---- head sizes 64 and 128, rows on 16-byte boundaries: a lane owns eight consecutive elements of a head (16 lanes a head of
// 128, 8 a head of 64), the warp takes the token's next heads in turn and has asked for all of them before it works on the first.
// A rotation partner rot/2 further on is another lane's (one exchange an element), a neighbour the lane's own.  Half of the
// blocks, the first to start, only make means: a block whose token does not fill a page leaves at once, so that the long ones do not
// start last.
// Bound by memory (rows in, rows out).  4096 tokens of 32 + 8 + 8 heads of 128: @APPEND@
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 x = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
#pragma unroll
  for (int j = 0; j < 4; ++j) { const float2 f = __bfloat1622float2(h[j]); v[2 * j] = f.x; v[2 * j + 1] = f.y; }
}
template <typename T> struct alignas(16) Vec8 { T v[8]; };
template <typename T> __device__ __forceinline__ void widen8(const Vec8<T>& x, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(x.v[j]);
}
template <typename T> __device__ __forceinline__ Vec8<T> narrow8(const float (&v)[8]) {
  Vec8<T> x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x.v[j] = from_f32<T>(v[j]);
  return x;
}

// What a lane holds of the rotation of its eight elements: value * c + partner * s (the sign of the pair's first element in s).
struct Turn { float c[8], s[8]; };

// `l` the lane's place among the head's lanes.
__device__ __forceinline__ void load_turn(const float* cs, int rot, int interleaved, int l, Turn& t) {
  const int half = rot >> 1;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = l * 8 + j;
    const bool in = e < rot;
    const int i = interleaved ? e >> 1 : (e < half ? e : e - half);
    const bool first = interleaved ? !(e & 1) : e < half;
    t.c[j] = in ? cs[i] : 1.f;
    const float s = in ? cs[half + i] : 0.f;
    t.s[j] = first ? -s : s;
  }
}

// v: the lane's elements (32-bit); w: its norm weights; LANES: lanes of a head
template <int LANES>
__device__ __forceinline__ void finish8(float (&v)[8], bool norm, const float (&w)[8], float eps, const Turn& t, int rot, int interleaved) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float rinv = rsqrtf(ss / (float)(LANES * 8) + eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * rinv * w[j];
  }
  if (rot == 0) return;
  const int lane = threadIdx.x & 31, l = lane % LANES;
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float a = v[j], b = v[j + 1];
      if (l * 8 + j >= rot) break;
      v[j] = fmaf(b, t.s[j], a * t.c[j]);
      v[j + 1] = fmaf(a, t.s[j + 1], b * t.c[j + 1]);
    }
  } else {
    const int hop = rot / 16;                                // lanes to the partner
    const int from = l < hop ? lane + hop : l < 2 * hop ? lane - hop : lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float other = __shfl_sync(0xffffffffu, v[j], from);
      if (l < 2 * hop) v[j] = fmaf(other, t.s[j], v[j] * t.c[j]);
    }
  }
}

constexpr int MAX_PAGE = 128;        // tokens of a page

template <typename TA, typename TW, int D>
__global__ void __launch_bounds__(WARPS * 32)
append_lanes_kernel(const TA* __restrict__ qkv, TA* __restrict__ q_out, const TW* __restrict__ q_weight,
                    const TW* __restrict__ k_weight, TA* cache, TA* __restrict__ means, const Append p) {
  constexpr int LANES = D / 8, PER = 32 / LANES, AHEAD = 3;     // lanes of a head, heads of a warp at once, turns asked for ahead
  pdl_enter();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES, side = lane / LANES;
  const int slot = p.slots[t];
  const bool kept = slot >= 0 && slot / p.page_size < p.num_pages;
  const int page = kept ? slot / p.page_size : 0, off = kept ? slot % p.page_size : 0;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * D;
  const bool norm = q_weight != nullptr;
  Turn turn;
  if (blockIdx.y == 0) {
    if (!kept || off != p.page_size - 1) return;
    // the page becomes full: a warp per key head, its groups of lanes take the offsets in turn
    unsigned brought[MAX_PAGE / 32];                         // offsets whose key this step brings, by distance to the last
#pragma unroll
    for (int i = 0; i < MAX_PAGE / 32; ++i) {
      const int back = i * 32 + lane;
      brought[i] = __ballot_sync(0xffffffffu, back < p.page_size && t - back >= 0 && p.slots[max(t - back, 0)] == slot - back);
    }
    float w[8];
    if (norm) load8<TW>(k_weight + l * 8, w);
    for (int g = warp; g < p.Hkv; g += WARPS) {
      float sum[8] = {};
      const TA* cached = cache + (int64_t)page * 2 * plane + (int64_t)g * p.page_size * D + l * 8;
#pragma unroll 2
      for (int o0 = 0; o0 < p.page_size; o0 += PER) {
        const int o = o0 + side, back = p.page_size - 1 - o;
        const bool in = o < p.page_size;
        unsigned word = brought[0];
#pragma unroll
        for (int i = 1; i < MAX_PAGE / 32; ++i) word = back >> 5 == i ? brought[i] : word;
        const bool now = in && (word >> (back & 31) & 1);
        const int u = now ? t - back : t;
        const TA* src = !in || now ? qkv + (int64_t)u * p.ld + (int64_t)(p.H + g) * D + l * 8 : cached + (int64_t)o * D;
        float v[8];
        load8<TA>(src, v);
        if (__any_sync(0xffffffffu, now)) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = v[j];
          if (p.rot) load_turn(angles(p, u), p.rot, p.interleaved, l, turn);
          finish8<LANES>(x, norm, w, p.eps, turn, p.rot, p.interleaved);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = now ? to_f32<TA>(from_f32<TA>(x[j])) : v[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += in ? v[j] : 0.f;
      }
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] /= (float)p.page_size;
      if (side == 0) *reinterpret_cast<Vec8<TA>*>(means + ((int64_t)page * p.Hkv + g) * D + l * 8) = narrow8<TA>(sum);
    }
    return;
  }
  const int heads = p.H + 2 * p.Hkv;
  const TA* row = qkv + (int64_t)t * p.ld + l * 8;
  float wq[8], wk[8];
  if (norm) { load8<TW>(q_weight + l * 8, wq); load8<TW>(k_weight + l * 8, wk); }
  if (p.rot) load_turn(angles(p, t), p.rot, p.interleaved, l, turn);
  for (int h0 = warp * PER; h0 < heads; h0 += WARPS * PER * AHEAD) {
    Vec8<TA> in[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int head = h0 + u * WARPS * PER + side;
      if (head < heads) in[u] = *reinterpret_cast<const Vec8<TA>*>(row + (int64_t)head * D);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (h0 + u * WARPS * PER >= heads) break;              // (the whole warp alike)
      const int head = h0 + u * WARPS * PER + side;
      float v[8];
      widen8<TA>(in[u], v);
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = head < p.H ? wq[j] : wk[j];
      finish8<LANES>(v, norm, w, p.eps, turn, p.rot, p.interleaved);
      if (head < p.H) {
        *reinterpret_cast<Vec8<TA>*>(q_out + (int64_t)t * p.ldq + (int64_t)head * D + l * 8) = narrow8<TA>(v);
      } else if (head < heads && kept) {
        const bool key = head < p.H + p.Hkv;
        const int g = key ? head - p.H : head - p.H - p.Hkv;
        TA* dst = cache + ((int64_t)page * 2 + (key ? 0 : 1)) * plane + ((int64_t)g * p.page_size + off) * D + l * 8;
        *reinterpret_cast<Vec8<TA>*>(dst) = key ? narrow8<TA>(v) : in[u];
      }
    }
  }
}

template <typename TA, typename TW>
int run(const void* qkv, void* q_out, const void* qw, const void* kw, void* cache, void* means, const Append& p, int T,
        cudaStream_t stream) {
  const bool aligned = ((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)qw | (uintptr_t)kw | (uintptr_t)cache | (uintptr_t)means) % 16 == 0 &&
                       p.ld % 8 == 0 && p.ldq % 8 == 0;
  if (aligned && (p.D == 64 || p.D == 128) && p.page_size <= MAX_PAGE && (p.interleaved || p.rot % 16 == 0)) {
    auto kernel = p.D == 64 ? append_lanes_kernel<TA, TW, 64> : append_lanes_kernel<TA, TW, 128>;
    launch_pdl(kernel, dim3(T, 2), dim3(WARPS * 32), 0, stream, (const TA*)qkv, (TA*)q_out, (const TW*)qw, (const TW*)kw,
               (TA*)cache, (TA*)means, p);
    return cuda_status("page_append");
  }
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

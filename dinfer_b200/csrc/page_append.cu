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
              const TW* __restrict__ k_weight, TA* __restrict__ cache, const Append p) {
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
}

// The means of the pages whose last offset the step wrote, from the cache, behind the launch that wrote it: a block per token, a warp per
// key head.
template <typename TA>
__global__ void __launch_bounds__(WARPS * 32) any_means_kernel(const TA* __restrict__ cache, TA* __restrict__ means, const Append p) {
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = p.slots[blockIdx.x], page = slot / p.page_size;
  if (slot < 0 || page >= p.num_pages || slot % p.page_size != p.page_size - 1) return;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * p.D;
  for (int g = warp; g < p.Hkv; g += WARPS)
    for (int e = lane; e < p.D; e += 32) {
      const TA* k = cache + (int64_t)page * 2 * plane + (int64_t)g * p.page_size * p.D + e;
      float sum = 0.f;
#pragma unroll 8
      for (int o = 0; o < p.page_size; ++o) sum += to_f32<TA>(k[(int64_t)o * p.D]);
      means[((int64_t)page * p.Hkv + g) * p.D + e] = from_f32<TA>(sum / (float)p.page_size);
    }
}

// ---- head sizes 64 and 128, rows on 16-byte boundaries, a rotation over a multiple of 8 elements.  A lane owns eight elements of a head
// (16 lanes a head of 128, 8 a head of 64) as two runs of four, chosen so that the pairs it turns are its own: of the turned part of a
// neox head elements 4 l + {0..3} and their partners rot/2 further on, elsewhere eight in a row.  A warp asks for several heads
// before it works on the first.  Bound by memory: the rows once in and once
// out.  4096 tokens of 32 + 8 + 8 heads of 128 (103 MB) take 25 us, 63 % of a copy's rate: the norms' and rotations' instructions and
// the tail of the means stand beside the loads (a warp per head took 59).
template <typename T> struct alignas(4 * sizeof(T)) Vec4 { alignas(4 * sizeof(T)) T v[4]; };
template <typename T> struct Lane8 { Vec4<T> a, b; };
template <typename T> __device__ __forceinline__ Lane8<T> load_lane(const T* row, int a, int b) {
  return {*reinterpret_cast<const Vec4<T>*>(row + a), *reinterpret_cast<const Vec4<T>*>(row + b)};
}
template <typename T> __device__ __forceinline__ void store_lane(T* row, int a, int b, const Lane8<T>& x) {
  *reinterpret_cast<Vec4<T>*>(row + a) = x.a;
  *reinterpret_cast<Vec4<T>*>(row + b) = x.b;
}
template <typename T> __device__ __forceinline__ void widen(const Lane8<T>& x, float (&v)[8]);
template <> __device__ __forceinline__ void widen<float>(const Lane8<float>& x, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[j] = x.a.v[j]; v[4 + j] = x.b.v[j]; }
}
template <> __device__ __forceinline__ void widen<__nv_bfloat16>(const Lane8<__nv_bfloat16>& x, float (&v)[8]) {
  const unsigned *a = reinterpret_cast<const unsigned*>(x.a.v), *b = reinterpret_cast<const unsigned*>(x.b.v);
#pragma unroll
  for (int j = 0; j < 2; ++j) {                                // a bfloat16 is the upper half of the number it stands for
    v[2 * j] = __uint_as_float(a[j] << 16); v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
    v[4 + 2 * j] = __uint_as_float(b[j] << 16); v[5 + 2 * j] = __uint_as_float(b[j] & 0xffff0000u);
  }
}
template <typename T> __device__ __forceinline__ Lane8<T> narrow(const float (&v)[8]);
template <> __device__ __forceinline__ Lane8<float> narrow<float>(const float (&v)[8]) {
  return {{v[0], v[1], v[2], v[3]}, {v[4], v[5], v[6], v[7]}};
}
template <> __device__ __forceinline__ Lane8<__nv_bfloat16> narrow<__nv_bfloat16>(const float (&v)[8]) {
  Lane8<__nv_bfloat16> x;                                      // two at a time
  __nv_bfloat162 *a = reinterpret_cast<__nv_bfloat162*>(x.a.v), *b = reinterpret_cast<__nv_bfloat162*>(x.b.v);
  a[0] = __floats2bfloat162_rn(v[0], v[1]); a[1] = __floats2bfloat162_rn(v[2], v[3]);
  b[0] = __floats2bfloat162_rn(v[4], v[5]); b[1] = __floats2bfloat162_rn(v[6], v[7]);
  return x;
}

// Where lane l of a head's lanes finds its elements, and the four angles of its pairs.
struct Place { int a, b; bool turns, neox; };
__device__ __forceinline__ Place place_of(const Append& p, int l) {
  const bool turns = l * 8 < p.rot, neox = turns && !p.interleaved;
  return {neox ? 4 * l : 8 * l, neox ? 4 * l + (p.rot >> 1) : 8 * l + 4, turns, neox};
}
__device__ __forceinline__ void load_turn(const float* cs, const Place& at, int rot, int l, float4& c, float4& s) {
  if (!at.turns) return;                                       // (angles 4 l .. 4 l + 3 in either layout)
  c = *reinterpret_cast<const float4*>(cs + 4 * l);
  s = *reinterpret_cast<const float4*>(cs + (rot >> 1) + 4 * l);
}

template <int LANES>
__device__ __forceinline__ void finish(float (&v)[8], bool norm, const float (&w)[8], float eps, const Place& at, const float4& c, const float4& s) {
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
  if (!at.turns) return;
  auto turn = [](float& x, float& y, float co, float si) {
    const float a = x, b = y;
    x = fmaf(a, co, -b * si);
    y = fmaf(b, co, a * si);
  };
  if (at.neox) {
    turn(v[0], v[4], c.x, s.x); turn(v[1], v[5], c.y, s.y); turn(v[2], v[6], c.z, s.z); turn(v[3], v[7], c.w, s.w);
  } else {
    turn(v[0], v[1], c.x, s.x); turn(v[2], v[3], c.y, s.y); turn(v[4], v[5], c.z, s.z); turn(v[6], v[7], c.w, s.w);
  }
}

constexpr int MAX_PAGE = 128;        // tokens of a page
constexpr int FEW_TOKENS = 512, FEW_SPAN = 8;

// Of `span` tokens from t0 on (32 at most), those whose slot is a page's last.
__device__ __forceinline__ unsigned page_ends(const Append& p, int t0, int T, int span, int& slot) {
  const int t = t0 + (threadIdx.x & 31);
  slot = t < T && t < t0 + span ? p.slots[t] : -1;
  return __ballot_sync(0xffffffffu, slot >= 0 && slot % p.page_size == p.page_size - 1 && slot / p.page_size < p.num_pages);
}

// The means of key head g of the pages that a span of tokens from t0 on fills, by a block: its warps' groups of lanes take the offsets
// in turn and come together in an order that depends on nothing but the page size.  ROWS: keys that this step brings are made again from
// its rows; else all come from the cache (behind the launch that wrote them).
template <typename TA, typename TW, int D, bool ROWS>
__device__ __forceinline__ void make_means(const TA* qkv, const TW* k_weight, const TA* cache, TA* means, int t0, int g, int T, const Append& p) {
  constexpr int LANES = D / 8, PER = 32 / LANES, AHEAD = 4;
  __shared__ float s_sum[WARPS][D];
  __shared__ int s_token[ROWS ? MAX_PAGE : 1];               // the step's token that brings an offset's key, or -1
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES, side = lane / LANES;
  int slots, all_slots[ROWS ? FEW_TOKENS / (WARPS * 32) : 1];
  if (ROWS)
#pragma unroll
    for (int i = 0; i < FEW_TOKENS / (WARPS * 32); ++i) {
      const int u = threadIdx.x + i * WARPS * 32;
      all_slots[i] = u < T ? p.slots[u] : -1;
    }
  unsigned ends = page_ends(p, t0, T, ROWS ? FEW_SPAN : 32, slots);
  if (!ends) return;
  const Place at = place_of(p, l);
  const bool norm = k_weight != nullptr;
  for (; ends; ends &= ends - 1) {
    const int slot = __shfl_sync(0xffffffffu, slots, __ffs(ends) - 1), page = slot / p.page_size;
    const TA* cached = cache + ((int64_t)page * 2 * p.Hkv + g) * p.page_size * D;
    float sum[8] = {};
    if (ROWS) {                                              // (whatever order the batch has its tokens in)
      if (threadIdx.x < MAX_PAGE) s_token[threadIdx.x] = -1;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < FEW_TOKENS / (WARPS * 32); ++i) {
        const unsigned o = (unsigned)all_slots[i] - (unsigned)page * p.page_size;
        if (all_slots[i] >= 0 && o < (unsigned)p.page_size) s_token[o] = threadIdx.x + i * WARPS * 32;
      }
      __syncthreads();
    }
    for (int o0 = warp * PER; o0 < p.page_size; o0 += WARPS * PER * AHEAD) {
      Lane8<TA> in[AHEAD];
      int from[AHEAD];                                       // token of this step, or -1
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) from[u] = ROWS ? s_token[min(o0 + u * WARPS * PER + side, p.page_size - 1)] : -1;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int o = min(o0 + u * WARPS * PER + side, p.page_size - 1);
        in[u] = load_lane<TA>(from[u] >= 0 ? qkv + (int64_t)from[u] * p.ld + (int64_t)(p.H + g) * D : cached + o * D, at.a, at.b);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int o = o0 + u * WARPS * PER + side;
        float v[8];
        widen<TA>(in[u], v);
        if (ROWS && __any_sync(0xffffffffu, from[u] >= 0)) {
          float w[8], x[8];
          if (norm) widen<TW>(load_lane<TW>(k_weight, at.a, at.b), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = v[j];
          float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
          if (p.rot) load_turn(angles(p, max(from[u], 0)), at, p.rot, l, c, s);
          finish<LANES>(x, norm, w, p.eps, at, c, s);
          float y[8];
          widen<TA>(narrow<TA>(x), y);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = from[u] >= 0 ? y[j] : v[j];
        }
        if (o < p.page_size)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += v[j];
      }
    }
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
    if (side == 0) {
      *reinterpret_cast<float4*>(&s_sum[warp][at.a]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
      *reinterpret_cast<float4*>(&s_sum[warp][at.b]) = make_float4(sum[4], sum[5], sum[6], sum[7]);
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float all = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) all += s_sum[w][threadIdx.x];
      means[((int64_t)page * p.Hkv + g) * D + threadIdx.x] = from_f32<TA>(all / (float)p.page_size);
    }
    __syncthreads();
  }
}

template <typename TA, int D>
__global__ void __launch_bounds__(WARPS * 32)
page_means_kernel(const TA* __restrict__ cache, TA* __restrict__ means, int T, const Append p) {
  pdl_enter();
  make_means<TA, TA, D, false>(nullptr, nullptr, cache, means, blockIdx.x * 32, blockIdx.y, T, p);
}

// WPT: warps that share a token's heads.  MEANS: the first `mean_blocks` blocks make the means, from this step's rows and the cache.
template <typename TA, typename TW, int D, int WPT, bool MEANS>
__global__ void __launch_bounds__(WARPS * 32, MEANS ? 2 : 4)
append_lanes_kernel(const TA* __restrict__ qkv, TA* __restrict__ q_out, const TW* __restrict__ q_weight,
                    const TW* __restrict__ k_weight, TA* cache, TA* __restrict__ means, int T, int mean_blocks, const Append p) {
  // lanes of a head, heads of a warp at once, heads asked for ahead
  constexpr int LANES = D / 8, PER = 32 / LANES, AHEAD = 3;
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES, side = lane / LANES;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * D;
  const bool norm = q_weight != nullptr;
  const Place at = place_of(p, l);
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (MEANS && (int)blockIdx.x < mean_blocks) {
    make_means<TA, TW, D, true>(qkv, k_weight, cache, means, blockIdx.x / p.Hkv * FEW_SPAN, blockIdx.x % p.Hkv, T, p);
    return;
  }
  const int t = ((int)blockIdx.x - mean_blocks) * (WARPS / WPT) + warp / WPT;
  if (t >= T) return;
  // everything that waits for nothing goes out first: slot, position, the first heads, the weights; then the angles
  const int slot = p.slots[t], pos = p.rot ? p.positions[t] : 0;
  const int heads = p.H + 2 * p.Hkv;
  const int first = warp % WPT * PER + side;
  constexpr int STEP = WPT * PER;                              // heads from one of a lane's to the next
  const TA* src = qkv + (int64_t)t * p.ld + first * D;
  Lane8<TA> in[AHEAD];
  auto load = [&](int h0) {
    if (h0 - side + (AHEAD - 1) * STEP + PER <= heads) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) in[u] = load_lane<TA>(src + u * STEP * D, at.a, at.b);
    } else {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)                          // (no branch between the loads)
        in[u] = load_lane<TA>(src + (min(h0 + u * STEP, heads - 1) - h0) * D, at.a, at.b);
    }
    src += AHEAD * STEP * D;
  };
  load(first);
  float w[8];
  if (norm) widen<TW>(load_lane<TW>(first < p.H ? q_weight : k_weight, at.a, at.b), w);
  if (p.rot) load_turn(p.cos_sin + (int64_t)(pos >= 0 && pos < p.table_rows ? pos : 0) * p.rot, at, p.rot, l, c, s);
  const int page = slot / p.page_size, off = slot - page * p.page_size;
  const bool kept = slot >= 0 && page < p.num_pages;
  TA* q_row = q_out + (int64_t)t * p.ldq;
  TA* c_row = cache + (kept ? (int64_t)page * 2 * plane + (int64_t)off * D : 0);
  const int head_step = p.page_size * D;                       // (the values follow the keys as key heads Hkv on)
  bool keys = first >= p.H;                                    // whose weights w holds
  for (int h0 = first; h0 - side < heads; h0 += STEP * AHEAD) {
    if (h0 != first) load(h0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int head = h0 + u * STEP;
      if (head - side >= heads) break;                         // (the whole warp alike)
      if (head - side < p.H + p.Hkv) {                         // values are left as they are
        if (norm && !keys && head >= p.H) {
          keys = true;
          widen<TW>(load_lane<TW>(k_weight, at.a, at.b), w);
        }
        __syncwarp();
        float v[8];
        widen<TA>(in[u], v);
        finish<LANES>(v, norm, w, p.eps, at, c, s);
        if (head < p.H + p.Hkv) in[u] = narrow<TA>(v);
      }
      if (head < p.H) store_lane<TA>(q_row + head * D, at.a, at.b, in[u]);
      else if (head < heads && kept) store_lane<TA>(c_row + (int64_t)(head - p.H) * head_step, at.a, at.b, in[u]);
    }
  }
}

template <typename TA, typename TW>
int run(const void* qkv, void* q_out, const void* qw, const void* kw, void* cache, void* means, const Append& p, int T,
        cudaStream_t stream) {
  const bool aligned = ((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)qw | (uintptr_t)kw | (uintptr_t)cache | (uintptr_t)means | (uintptr_t)p.cos_sin) % 16 == 0 &&
                       p.ld % 8 == 0 && p.ldq % 8 == 0;
  if (aligned && (p.D == 64 || p.D == 128) && p.page_size <= MAX_PAGE && p.rot % 8 == 0 && p.Hkv <= 65535) {
    // few tokens: a block each, so that a token's heads are all under way at once, the means in the same launch; many: a warp's start
    // (slot, angles, weights) is paid for half of a token's heads, the means in a launch of their own.  us, the first way and the second, 32 + 8
    // + 8 heads of 128: 1 token 2.9 and 6.6, 256 tokens 5.0 and 8.2, 512 tokens 7.5 and 8.7, 1024 tokens 12.9 and 11.8, 2048 tokens
    // 24 and 13; 64 single ones 3.3 and 8.2
    const bool few = T <= FEW_TOKENS;
    auto kernel = few ? (p.D == 64 ? append_lanes_kernel<TA, TW, 64, 8, true> : append_lanes_kernel<TA, TW, 128, 8, true>)
                      : (p.D == 64 ? append_lanes_kernel<TA, TW, 64, 2, false> : append_lanes_kernel<TA, TW, 128, 2, false>);
    const int mean_blocks = few ? (T + FEW_SPAN - 1) / FEW_SPAN * p.Hkv : 0, per = few ? 1 : WARPS / 2;
    launch_pdl(kernel, dim3(mean_blocks + (T + per - 1) / per), dim3(WARPS * 32), 0, stream, (const TA*)qkv, (TA*)q_out, (const TW*)qw,
               (const TW*)kw, (TA*)cache, (TA*)means, T, mean_blocks, p);
    if (!few)
      launch_pdl(p.D == 64 ? page_means_kernel<TA, 64> : page_means_kernel<TA, 128>, dim3((T + 31) / 32, p.Hkv), dim3(WARPS * 32), 0, stream,
                 (const TA*)cache, (TA*)means, T, p);
    return cuda_status("page_append");
  }
  launch_pdl(append_kernel<TA, TW>, dim3(T), dim3(WARPS * 32), 0, stream, (const TA*)qkv, (TA*)q_out, (const TW*)qw,
             (const TW*)kw, (TA*)cache, p);
  launch_pdl(any_means_kernel<TA>, dim3(T), dim3(WARPS * 32), 0, stream, (const TA*)cache, (TA*)means, p);
  return cuda_status("page_append");
}

}  // namespace

// What the call takes, 8 bytes a field (a caller packs them and hands over one address).  w_dtype: element type of the norm weights (both
// given or neither); cos_sin: f32 [table_rows, rot], rot 0: no rotation.
struct PageAppendArgs {
  const void* qkv;
  int64_t ld;
  const int* positions;
  const void *q_weight, *k_weight;
  double eps;
  const float* cos_sin;
  int64_t table_rows, rot, interleaved;
  void* q_out;
  int64_t ldq;
  void *cache, *means;
  const int* slots;
  int64_t num_pages, page_size, T, H, Hkv, D, dtype, w_dtype;
  cudaStream_t stream;
};

DINFER_API int dinfer_page_append(const PageAppendArgs* args) {
  const PageAppendArgs& a = *args;
  const int64_t most = 0x7fffffff;
  if (a.T < 0 || a.H <= 0 || a.Hkv <= 0 || a.D <= 0 || a.page_size <= 0 || a.num_pages < 0 || a.T > most / 16 || a.H > 65535 || a.Hkv > 65535 ||
      a.page_size > most || a.num_pages * a.page_size > most || a.table_rows > most)
    return refuse(DINFER_BAD_ARGUMENT, "page_append: sizes T=%lld H=%lld Hkv=%lld D=%lld, %lld pages of %lld", (long long)a.T, (long long)a.H,
                  (long long)a.Hkv, (long long)a.D, (long long)a.num_pages, (long long)a.page_size);
  if (a.D > MAX_D) return refuse(DINFER_BAD_ARGUMENT, "page_append: head size %lld is above %d", (long long)a.D, MAX_D);
  if (a.rot < 0 || a.rot > a.D || a.rot % 2 || (a.rot > 0 && (!a.cos_sin || a.table_rows <= 0)))
    return refuse(DINFER_BAD_ARGUMENT, "page_append: %lld turned elements of %lld, %lld angle rows", (long long)a.rot, (long long)a.D, (long long)a.table_rows);
  if (a.T == 0) return DINFER_OK;
  const Append p{a.ld, a.ldq, a.positions, (float)a.eps, a.cos_sin, (int)a.table_rows, (int)a.rot, (int)a.interleaved, a.slots,
                 (int)a.num_pages, (int)a.page_size, (int)a.H, (int)a.Hkv, (int)a.D};
  DINFER_DISPATCH_DTYPE(a.dtype, TA, {
    DINFER_DISPATCH_DTYPE(a.w_dtype, TW, {
      return (run<TA, TW>(a.qkv, a.q_out, a.q_weight, a.k_weight, a.cache, a.means, p, (int)a.T, a.stream));
    });
  });
}

DINFER_DEFINE_LAST_ERROR()

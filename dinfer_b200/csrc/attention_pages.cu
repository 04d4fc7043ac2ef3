// Attention over chosen pages of the paged cache: token t at position p, head h of key head g's group, reads the keys of the
// pages chosen[t, g, :] (-1: none) up to its own position,
//
//     out[t, h] = sum_i softmax_i(scale q[t, h] . k_i) v_i      over  { i <= p : i / page_size in chosen[t, g] }
//
// A page named twice counts twice; a number outside the request's table, or a page the table does not hold, is no page; a token
// that sees no key gets zeros, one all of whose scores are -inf what is not a number (0 / 0); rows behind the last request's tokens
// are left as they are.  Scores, weights and sums in 32-bit.
// What a token does not see is never multiplied, so that it may hold anything.
#include <cooperative_groups.h>
#include <float.h>

#include "mma_tiles.cuh"
#include "page_batch.cuh"

using namespace dinfer;
using namespace dinfer_mma;

namespace {

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
constexpr int KEYS = 4, ANY_WARPS = 8;

// Any sizes: a block per (token, head); its warps take runs of four keys in turn, the lanes split the elements, and the warps come
// together in shared memory.  Bound by the rows' way from memory, which every head of a group goes alone; one token of 16 heads of 96,
// 16 pages of 64, 36 us (a warp per head, key by key: 555); 32 single ones 107 (1046).
template <typename T, int C>   // C >= ceil(D / 32)
__global__ void __launch_bounds__(ANY_WARPS * 32)
attention_pages_kernel(const T* __restrict__ q, T* __restrict__ out, const T* __restrict__ cache, const Pages p) {
  __shared__ float s_acc[ANY_WARPS][C * 32], s_m[ANY_WARPS], s_l[ANY_WARPS];
  pdl_enter();
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = request_of(p.cu, p.num_reqs, t);
  if (r < 0) return;                                       // (the whole block alike)
  const int* table = p.table + (int64_t)r * p.width;
  const int g = h / (p.H / p.Hkv), pos = p.positions[t];
  const int* chosen = p.chosen + ((int64_t)t * p.Hkv + g) * p.top;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * p.D;
  float qv[C], acc[C];
  int at[C];                                               // the lane's elements; behind the last one the last one, against a zero
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = lane + 32 * c;
    at[c] = min(e, p.D - 1);
    qv[c] = e < p.D ? to_f32<T>(q[(int64_t)t * p.ldq + (int64_t)h * p.D + e]) * p.scale : 0.f;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const unsigned runs = (p.page_size + KEYS - 1) / KEYS;
  bool none = true;                                        // whether the token sees no key at all
  for (int i = 0; i < p.top; ++i) {
    const int j = chosen[i];
    if (j < 0 || j >= p.width) continue;
    const int page = table[j];
    if (page < 0 || page >= p.num_pages) continue;
    const int keys = (int)min((int64_t)p.page_size, pos - (int64_t)j * p.page_size + 1);
    none &= keys <= 0;
    const T* kp = cache + (int64_t)page * 2 * plane + (int64_t)g * p.page_size * p.D;
    // (the runs of all pages go round the warps, whatever a page holds of them)
    for (int o = (int)((warp - i * runs) % ANY_WARPS) * KEYS; o < keys; o += ANY_WARPS * KEYS) {
      T k[KEYS][C], v[KEYS][C];
#pragma unroll
      for (int u = 0; u < KEYS; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) k[u][c] = kp[(int64_t)min(o + u, keys - 1) * p.D + at[c]];
#pragma unroll
      for (int u = 0; u < KEYS; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) v[u][c] = kp[plane + (int64_t)min(o + u, keys - 1) * p.D + at[c]];
      float s[KEYS], n = m;
#pragma unroll
      for (int u = 0; u < KEYS; ++u) {
        s[u] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (lane + 32 * c < p.D) s[u] = fmaf(qv[c], to_f32<T>(k[u][c]), s[u]);
        s[u] = warp_sum(s[u]);
        if (o + u < keys) n = fmaxf(n, s[u]);
      }
      const float base = n == -INFINITY ? 0.f : n, alpha = expf(m - base);
      l *= alpha;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] *= alpha;
#pragma unroll
      for (int u = 0; u < KEYS; ++u)
        if (o + u < keys) {
          const float w = expf(s[u] - base);
          l += w;
#pragma unroll
          for (int c = 0; c < C; ++c) acc[c] = fmaf(w, to_f32<T>(v[u][c]), acc[c]);
        }
      m = n;
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) s_acc[warp][lane + 32 * c] = acc[c];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  float top = s_m[0], sum = 0.f;
#pragma unroll
  for (int w = 1; w < ANY_WARPS; ++w) top = fmaxf(top, s_m[w]);
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int w = 0; w < ANY_WARPS; ++w) sum = fmaf(s_l[w], expf(s_m[w] - base), sum);
  const float inv = 1.f / sum;                             // (scores of -inf alone: 0 / 0)
  for (int e = threadIdx.x; e < p.D; e += ANY_WARPS * 32) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < ANY_WARPS; ++w) o = fmaf(s_acc[w][e], expf(s_m[w] - base), o);
    out[(int64_t)t * p.ldo + (int64_t)h * p.D + e] = from_f32<T>(none ? 0.f : o * inv);
  }
}

template <typename T>
int run(const void* q, void* out, const void* cache, const Pages& p, cudaStream_t stream) {
  const dim3 grid(p.T, p.H), block(ANY_WARPS * 32);
  if (p.D <= 64) launch_pdl(attention_pages_kernel<T, 2>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  else if (p.D <= 128) launch_pdl(attention_pages_kernel<T, 4>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  else if (p.D <= 256) launch_pdl(attention_pages_kernel<T, 8>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  else launch_pdl(attention_pages_kernel<T, 16>, grid, block, 0, stream, (const T*)q, (T*)out, (const T*)cache, p);
  return cuda_status("attention_pages");
}

// ------------------------------------------------------------------------------------------------
// 32-bit, head sizes 64 and 128, groups of up to 8 heads: a token and key head to a block, or to a cluster of up to eight that share its
// keys.  The warps take runs of eight keys in turn, straight from memory: a lane holds D / 32 elements of every row, sixteen rows on
// their way at once.  A run's 8 x G scores are summed over the lanes by exchanging halves (a lane ends with the sums it owns: 31 exchanges
// for 32 sums instead of 160), the softmax's statistics live with the owner, and the weights go round lane by lane.  The warps, then the
// blocks of the cluster, come together in shared memory.  Bound by the rows' way from memory: 64 single tokens of 8 key heads, 16
// pages of 64 keys of 128 (537 MB) take 88 us, 93 % of a copy's rate; a single one 9.5 us, 300 neighbouring ones 230 us (2.5 GB,
// from L2).  A block that walked the pages of four neighbouring tokens together, each page read once into shared memory for all, took
// 77, 93 and 338 us there: the products with what lies in shared memory bound it.
constexpr int L_KEYS = 8;

template <int D, int G>
__global__ void __launch_bounds__(WARPS * 32, 2)
pages_float_kernel(const float* __restrict__ q, float* __restrict__ out, const float* __restrict__ cache, const Pages p, int splits) {
  constexpr int E = D / 32, N = L_KEYS * G, OWN = N > 32 ? N / 32 : 1, STEPS = N >= 32 ? 5 : N == 16 ? 4 : 3;
  struct alignas(E * 4) Vec { float v[E]; };
  __shared__ float s_acc[WARPS][G][D + 2];
  __shared__ float c_o[G][D], c_ml[G][2];
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = blockIdx.y;
  const int t = blockIdx.x / splits, split = blockIdx.x - t * splits, group = p.H / p.Hkv, P = p.page_size;
  const int r = request_of(p.cu, p.num_reqs, t);
  if (r < 0) return;                                       // (the whole cluster alike)
  const int* table = p.table + (int64_t)r * p.width;
  const int* chosen = p.chosen + ((int64_t)t * p.Hkv + g) * p.top;
  const int64_t plane = (int64_t)p.Hkv * P * D;
  const int pos = p.positions[t];
  Vec x[G];
#pragma unroll
  for (int h = 0; h < G; ++h)
    x[h] = *reinterpret_cast<const Vec*>(q + (int64_t)t * p.ldq + (int64_t)(g * group + min(h, group - 1)) * D + lane * E);
  float acc[G][E], m[OWN], l[OWN];
#pragma unroll
  for (int h = 0; h < G; ++h)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[h][e] = 0.f;
#pragma unroll
  for (int o = 0; o < OWN; ++o) { m[o] = -INFINITY; l[o] = 0.f; }
  // Sum (key i, head h) is number h * 8 + i; what halving by lane bits 16, 8, ... leaves with a lane: its upper STEPS bits, and the OWN last
  // ones side by side.
  const int own = N >= 32 ? lane * OWN : lane >> (5 - STEPS);
  const int key = own % L_KEYS;                            // of the lane's first sum; the heads of all of them are one
  const int runs = P / L_KEYS;
  bool saw = false;                                        // a key
  for (int u = split * WARPS + warp; u < p.top * runs; u += splits * WARPS) {
    const int j = chosen[u / runs], part = u % runs * L_KEYS;
    if (j < 0 || j >= p.width || (int64_t)j * P + part > pos) continue;
    const int page = table[j];
    if (page < 0 || page >= p.num_pages) continue;
    const int n = min(L_KEYS, pos - j * P - part + 1);     // keys that the token sees
    saw = true;
    const float* rows = cache + (int64_t)page * 2 * plane + ((int64_t)g * P + part) * D + lane * E;
    Vec k[L_KEYS], v[L_KEYS];
#pragma unroll
    for (int i = 0; i < L_KEYS; ++i) k[i] = *reinterpret_cast<const Vec*>(rows + min(i, n - 1) * D);
#pragma unroll
    for (int i = 0; i < L_KEYS; ++i) v[i] = *reinterpret_cast<const Vec*>(rows + plane + min(i, n - 1) * D);
    float s[N];
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
      for (int i = 0; i < L_KEYS; ++i) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) d = fmaf(x[h].v[e], k[i].v[e], d);
        s[h * L_KEYS + i] = d;
      }
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
      const int bit = 16 >> step, half = N >> (step + 1);
      const bool upper = lane & bit;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < half) {
          const float give = upper ? s[i] : s[i + half], keep = upper ? s[i + half] : s[i];
          s[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
        }
    }
#pragma unroll
    for (int bit = 16 >> STEPS; bit > 0; bit >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], bit);
    // softmax of the lane's sums; the eight keys of a head lie in neighbouring lanes
    float top = -INFINITY;
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      s[o] = key + o < n ? s[o] * p.scale : -INFINITY;
      top = fmaxf(top, s[o]);
    }
#pragma unroll
    for (int bit = N >= 32 ? 4 / OWN : (1 << (5 - STEPS)) * 4; bit >= (N >= 32 ? 1 : 1 << (5 - STEPS)); bit >>= 1)
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, bit));
    top = fmaxf(top, m[0]);
    const float base = top == -INFINITY ? 0.f : top, alpha = expf(m[0] - base);
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      s[o] = key + o < n ? expf(s[o] - base) : 0.f;
      l[o] = fmaf(l[o], alpha, s[o]);
    }
    m[0] = top;
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const float a = __shfl_sync(0xffffffffu, alpha, N >= 32 ? h * L_KEYS / OWN : (h * L_KEYS) << (5 - STEPS));
#pragma unroll
      for (int e = 0; e < E; ++e) acc[h][e] *= a;
    }
#pragma unroll
    for (int i = 0; i < L_KEYS; ++i)
      if (i < n) {                                         // (a warp alike; what is not seen is not multiplied)
#pragma unroll
        for (int h = 0; h < G; ++h) {
          const int at = h * L_KEYS + i;
          const float w = __shfl_sync(0xffffffffu, s[N >= 32 ? at % OWN : 0], N >= 32 ? at / OWN : at << (5 - STEPS));
#pragma unroll
          for (int e = 0; e < E; ++e) acc[h][e] = fmaf(w, v[i].v[e], acc[h][e]);
        }
      }
  }
  // a head's sum over its owners: eight keys, lanes that hold the same sum (fewer than 32 sums) counted once
  float sum = l[0];
#pragma unroll
  for (int o = 1; o < OWN; ++o) sum += l[o];
#pragma unroll
  for (int bit = N >= 32 ? 4 / OWN : (1 << (5 - STEPS)) * 4; bit >= (N >= 32 ? 1 : 1 << (5 - STEPS)); bit >>= 1)
    sum += __shfl_xor_sync(0xffffffffu, sum, bit);
#pragma unroll
  for (int h = 0; h < G; ++h) {
    const int src = N >= 32 ? h * L_KEYS / OWN : (h * L_KEYS) << (5 - STEPS);
    const float m_w = __shfl_sync(0xffffffffu, m[0], src), l_h = __shfl_sync(0xffffffffu, sum, src);
    // (-inf is the maximum of a warp that saw no key; of one all of whose scores are -inf it is the lowest number: where no score is
    // larger the result is 0 / 0)
    const float m_h = saw ? fmaxf(m_w, -FLT_MAX) : m_w;
#pragma unroll
    for (int e = 0; e < E; ++e) s_acc[warp][h][lane * E + e] = acc[h][e];
    if (lane == 0) { s_acc[warp][h][D] = m_h; s_acc[warp][h][D + 1] = l_h; }
  }
  __syncthreads();
  float* orow = out + (int64_t)t * p.ldo + (int64_t)g * group * D;
  for (int idx = threadIdx.x; idx < group * D; idx += WARPS * 32) {
    const int h = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_acc[w][h][D]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = expf(s_acc[w][h][D] - base);
      L = fmaf(s_acc[w][h][D + 1], f, L);
      o = fmaf(s_acc[w][h][d], f, o);
    }
    if (splits == 1) orow[idx] = M == -INFINITY ? 0.f : o / L;
    else {
      c_o[h][d] = o;
      if (d == 0) { c_ml[h][0] = M; c_ml[h][1] = L; }
    }
  }
  if (splits == 1) return;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int share = (group * D + splits - 1) / splits;
  for (int idx = split * share + threadIdx.x; idx < min(group * D, (split + 1) * share); idx += WARPS * 32) {
    const int h = idx / D;
    float M = -INFINITY;
    for (int r2 = 0; r2 < splits; ++r2) M = fmaxf(M, cluster.map_shared_rank(&c_ml[0][0], r2)[h * 2]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, o = 0.f;
    for (int r2 = 0; r2 < splits; ++r2) {
      const float* ml = cluster.map_shared_rank(&c_ml[0][0], r2) + h * 2;
      const float f = expf(ml[0] - base);
      L = fmaf(ml[1], f, L);
      o = fmaf(cluster.map_shared_rank(&c_o[0][0], r2)[idx], f, o);
    }
    orow[idx] = M == -INFINITY ? 0.f : o / L;
  }
  cluster.sync();                                          // nobody leaves while another reads its memory
}

template <int D, int G>
int run_float(const void* q, void* out, const void* cache, const Pages& p, int sms, cudaStream_t stream) {
  // blocks that share a token's keys: as far as all run at the same time (two an SM), each with a run of keys a warp at least
  int splits = 1;
  while (splits < 8 && (int64_t)p.T * p.Hkv * splits * 2 <= 2 * sms && (int64_t)splits * 2 * WARPS * L_KEYS <= (int64_t)p.top * p.page_size) splits *= 2;
  launch_pdl_cluster(pages_float_kernel<D, G>, dim3((unsigned)(p.T * splits), p.Hkv), dim3(WARPS * 32), dim3(splits), 0, stream,
                     (const float*)q, (float*)out, (const float*)cache, p, splits);
  return cuda_status("attention_pages (32-bit)");
}

// Whether the 32-bit kernel takes the call.
bool float_rows(const void* q, const void* out, const void* cache, const Pages& p) {
  return (p.D == 64 || p.D == 128) && p.page_size % L_KEYS == 0 && p.H / p.Hkv <= 8 && p.ldq % 4 == 0 && p.ldo % 4 == 0 &&
         (((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache) & 15) == 0 && p.Hkv <= 65535 &&
         (int64_t)p.top * (p.page_size / L_KEYS) < 0x7fffff00;
}

// ------------------------------------------------------------------------------------------------
// Bfloat16, head sizes 64 and 128, pages of 16 to 128 tokens, groups of up to 16 heads: few tokens (decode steps).
// A CTA owns a (token, key head) and, with splits, a share of its keys.  Tiles of 64 keys (a piece of a page or several pages) ride a
// ring of cp.async stages; a warp takes 16 of a tile's keys as the rows of S^T = K Q^T (the group's heads are the columns, so
// nothing of the product is spent on padding beyond 8 heads) and of O^T += V^T P^T, with a softmax of its own.  The four warps
// meet in shared memory at the end, the CTAs of a (token, key head), a cluster, through distributed shared memory.
// Bound by memory: 64 requests' tokens, 8 key heads of 128, 16 pages of 64 keys (266 MB) take 53 us, 75 % of a copy's rate (4 stages, or more CTAs a
// token than fit at once: 62 to 86); a chat's token 7, most of it the chain of starts (a warp per head and key by key: 548).
constexpr int NT = 128, BN = 64, MAX_TOP = 1024;

template <int D> __device__ __forceinline__ int swz(int row, int chunk) { return row * D + ((chunk ^ (row & 7)) << 3); }

template <int D, int NH8, int STAGES>
__global__ void __launch_bounds__(NT)
pages_token_kernel(const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ cache,
                   const Pages p, int splits) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __nv_bfloat16* sK = reinterpret_cast<__nv_bfloat16*>(smem_raw);          // [STAGES][BN][D]
  __nv_bfloat16* sV = sK + STAGES * BN * D;                                // [STAGES][BN][D]
  int2* s_page = reinterpret_cast<int2*>(sV + STAGES * BN * D);            // [top]: (page, keys the token sees of it)
  __shared__ int s_count;
  constexpr int NHEADS = NH8 * 8;
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  const int t = blockIdx.x / splits, split = blockIdx.x % splits, g = blockIdx.y;
  const int r = request_of(p.cu, p.num_reqs, t);
  if (r < 0) return;                                       // (the whole cluster alike)
  const int group = p.H / p.Hkv, P = p.page_size;
  if (warp == 0) {
    const int pos = p.positions[t];
    const int* chosen = p.chosen + ((int64_t)t * p.Hkv + g) * p.top;
    int n = 0;
    for (int i0 = 0; i0 < p.top; i0 += 32) {
      const int j = i0 + lane < p.top ? chosen[i0 + lane] : -1;
      int page = -1;
      if (j >= 0 && j < p.width && (int64_t)j * P <= pos) page = p.table[(int64_t)r * p.width + j];
      const bool ok = page >= 0 && page < p.num_pages;
      const unsigned mask = __ballot_sync(0xffffffffu, ok);
      if (ok) s_page[n + __popc(mask & ((1u << lane) - 1))] = make_int2(page, min(P, pos - j * P + 1));
      n += __popc(mask);
    }
    if (lane == 0) s_count = n;
  }
  // Q^T as the B operand: head nt*8 + gr, elements ks*16 + {2tq, 2tq+1} and + 8
  unsigned qb[D / 16][NH8][2];
#pragma unroll
  for (int nt = 0; nt < NH8; ++nt) {
    const int head = nt * 8 + gr;
    const __nv_bfloat16* row = q + (int64_t)t * p.ldq + (int64_t)(g * group + head) * D + 2 * tq;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qb[ks][nt][0] = head < group ? *reinterpret_cast<const unsigned*>(row + ks * 16) : 0u;
      qb[ks][nt][1] = head < group ? *reinterpret_cast<const unsigned*>(row + ks * 16 + 8) : 0u;
    }
  }
  __syncthreads();
  const int n_pages = s_count;
  const int p_log2 = 31 - __clz(P);
  int tile = 0, tile_end = ((n_pages << p_log2) + BN - 1) / BN;
  {
    const int per = (tile_end + splits - 1) / splits;
    tile = split * per;
    tile_end = min(tile_end, tile + per);
  }
  const int n_tiles = max(0, tile_end - tile);
  const int64_t plane = (int64_t)p.Hkv * P * D;
  auto load_tile = [&](int i) {
    constexpr int C = D / 8, ROWS = NT / C;                // a warp's copies cover whole rows
    const int chunk = threadIdx.x % C;
    __nv_bfloat16 *k = sK + (i % STAGES) * BN * D, *v = sV + (i % STAGES) * BN * D;
#pragma unroll
    for (int r0 = 0; r0 < BN; r0 += ROWS) {
      const int row = r0 + threadIdx.x / C;
      const int key = (tile + i) * BN + row;               // in the list's order
      const int e = key >> p_log2, o = key & (P - 1);
      const int2 entry = e < n_pages ? s_page[e] : make_int2(0, 0);
      const bool ok = o < entry.y;
      const __nv_bfloat16* src = cache + (ok ? (int64_t)entry.x * 2 * plane + ((int64_t)g * P + o) * D + chunk * 8 : 0);
      cp_async16(k + swz<D>(row, chunk), src, ok);
      cp_async16(v + swz<D>(row, chunk), ok ? src + plane : src, ok);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < n_tiles) load_tile(i);
    cp_async_commit();
  }
  float ot[D / 16][NH8][4];
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int nt = 0; nt < NH8; ++nt) ot[i][nt][0] = ot[i][nt][1] = ot[i][nt][2] = ot[i][nt][3] = 0.f;
  float m_run[NH8][2], l_run[NH8][2];                      // heads nt*8 + 2tq + {0, 1}
#pragma unroll
  for (int nt = 0; nt < NH8; ++nt) { m_run[nt][0] = m_run[nt][1] = -INFINITY; l_run[nt][0] = l_run[nt][1] = 0.f; }
  const float scale_log2 = p.scale * 1.4426950408889634f;
  const int key_off = warp * 16;

  for (int i = 0; i < n_tiles; ++i) {
    cp_async_wait<STAGES - 2>();
    __syncthreads();                                       // tile i is here, and everyone is done with tile i - 1
    if (i + STAGES - 1 < n_tiles) load_tile(i + STAGES - 1);
    cp_async_commit();
    const __nv_bfloat16 *kt = sK + (i % STAGES) * BN * D, *vt = sV + (i % STAGES) * BN * D;
    // the warp's 16 keys lie in one page (pages hold a multiple of 16 keys)
    const int key = (tile + i) * BN + key_off, e = key >> p_log2, o = key & (P - 1);
    const int seen = e < n_pages ? s_page[e].y - o : 0;
    if (seen <= 0) continue;
    const bool vis0 = gr < seen, vis1 = gr + 8 < seen;
    float st[NH8][4], st2[NH8][4];                         // two accumulators: half the dependent chain
#pragma unroll
    for (int nt = 0; nt < NH8; ++nt) {
      st[nt][0] = st[nt][1] = st[nt][2] = st[nt][3] = 0.f;
      st2[nt][0] = st2[nt][1] = st2[nt][2] = st2[nt][3] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ks += 2) {
      unsigned a[4], b[4];
      ldmatrix_x4(a, kt + swz<D>(key_off + (lane & 15), ks * 2 + (lane >> 4)));
      ldmatrix_x4(b, kt + swz<D>(key_off + (lane & 15), (ks + 1) * 2 + (lane >> 4)));
#pragma unroll
      for (int nt = 0; nt < NH8; ++nt) {
        mma_bf16(st[nt], a[0], a[1], a[2], a[3], qb[ks][nt][0], qb[ks][nt][1]);
        mma_bf16(st2[nt], b[0], b[1], b[2], b[3], qb[ks + 1][nt][0], qb[ks + 1][nt][1]);
      }
    }
    bool rescale = false;
    float alpha[NH8][2];
    unsigned pb[NH8][2];
#pragma unroll
    for (int nt = 0; nt < NH8; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float s0 = vis0 ? (st[nt][c] + st2[nt][c]) * scale_log2 : -INFINITY;
        const float s1 = vis1 ? (st[nt][c + 2] + st2[nt][c + 2]) * scale_log2 : -INFINITY;
        float mx = fmaxf(s0, s1);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m_new = fmaxf(m_run[nt][c], mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        alpha[nt][c] = fast_exp2(m_run[nt][c] - m_use);
        rescale |= m_new != m_run[nt][c];
        const float p0 = fast_exp2(s0 - m_use), p1 = fast_exp2(s1 - m_use);
        l_run[nt][c] = l_run[nt][c] * alpha[nt][c] + p0 + p1;
        m_run[nt][c] = m_new;
        st[nt][c] = p0;
        st[nt][c + 2] = p1;
      }
      // the weights are rounded to bfloat16, which the second product takes (half a step, 2^-8 of each; their sum is of the weights before):
      // against 64 bits a result is off by 1.2 to 1.4 times what rounding it alone costs
      pb[nt][0] = movmatrix_trans(pack_bf16(st[nt][0], st[nt][1]));
      pb[nt][1] = movmatrix_trans(pack_bf16(st[nt][2], st[nt][3]));
    }
    if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int nt = 0; nt < NH8; ++nt) {
          ot[d][nt][0] *= alpha[nt][0]; ot[d][nt][1] *= alpha[nt][1];
          ot[d][nt][2] *= alpha[nt][0]; ot[d][nt][3] *= alpha[nt][1];
        }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      unsigned a[4];
      ldmatrix_x4_trans(a, vt + swz<D>(key_off + (lane & 7) + ((lane >> 4) << 3), d * 2 + ((lane >> 3) & 1)));
#pragma unroll
      for (int nt = 0; nt < NH8; ++nt) mma_bf16(ot[d][nt], a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- the four warps come together: sums relative to the CTA's maximum, in shared memory
  float* w_o = reinterpret_cast<float*>(smem_raw);         // [4][NHEADS][D]
  float* w_m = w_o + 4 * NHEADS * D;                       // [4][NHEADS]
  float* w_l = w_m + 4 * NHEADS;
  float* c_o = w_l + 4 * NHEADS;                           // [NHEADS][D]
  float* c_ml = c_o + NHEADS * D;                          // [NHEADS][2]
#pragma unroll
  for (int nt = 0; nt < NH8; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = l_run[nt][c];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int head = nt * 8 + 2 * tq + c;
      if (gr == 0) { w_m[warp * NHEADS + head] = m_run[nt][c]; w_l[warp * NHEADS + head] = l; }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        w_o[(warp * NHEADS + head) * D + d * 16 + gr] = ot[d][nt][c];
        w_o[(warp * NHEADS + head) * D + d * 16 + gr + 8] = ot[d][nt][c + 2];
      }
    }
  }
  __syncthreads();
  const int64_t orow = (int64_t)t * p.ldo + (int64_t)g * group * D;     // (a page of the list holds a key that the token sees)
  for (int idx = threadIdx.x; idx < group * D; idx += NT) {
    const int head = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, w_m[w * NHEADS + head]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = fast_exp2(w_m[w * NHEADS + head] - base);
      L += w_l[w * NHEADS + head] * f;
      acc += w_o[(w * NHEADS + head) * D + d] * f;
    }
    if (splits == 1) {
      out[orow + idx] = __float2bfloat16_rn(n_pages == 0 ? 0.f : acc / L);
    } else {
      c_o[idx] = acc;
      if (d == 0) { c_ml[head * 2] = M; c_ml[head * 2 + 1] = L; }
    }
  }
  if (splits == 1) return;

  // ---- the CTAs of the cluster come together: each writes its share of the outputs
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int share = (group * D + splits - 1) / splits;
  for (int idx = split * share + threadIdx.x; idx < min(group * D, (split + 1) * share); idx += NT) {
    const int head = idx / D;
    float M = -INFINITY;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, cluster.map_shared_rank(c_ml, s)[head * 2]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float* ml = cluster.map_shared_rank(c_ml, s) + head * 2;
      const float f = fast_exp2(ml[0] - base);
      L += ml[1] * f;
      acc += cluster.map_shared_rank(c_o, s)[idx] * f;
    }
    out[orow + idx] = __float2bfloat16_rn(n_pages == 0 ? 0.f : acc / L);
  }
  cluster.sync();                                          // nobody leaves while another reads its memory
}

template <int D, int NH8>
int run_token(const void* q, void* out, const void* cache, const Pages& p, int splits, cudaStream_t stream) {
  constexpr int STAGES = 3;
  const size_t tiles = (size_t)STAGES * 2 * BN * D * 2 + (size_t)p.top * sizeof(int2);
  const size_t fold = (size_t)(4 * (NH8 * 8) * (D + 2) + NH8 * 8 * (D + 2)) * 4;
  const size_t smem = tiles > fold ? tiles : fold;
  auto kernel = pages_token_kernel<D, NH8, STAGES>;
  static thread_local int set_for = -1;                    // the attribute belongs to the device
  int dev = 0;
  cudaGetDevice(&dev);
  if (set_for != dev) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, STAGES * 2 * BN * D * 2 + MAX_TOP * 8);
    if (e != cudaSuccess) return cuda_status("attention_pages: shared memory");
    set_for = dev;
  }
  launch_pdl_cluster(kernel, dim3((unsigned)(p.T * splits), p.Hkv), dim3(NT), dim3(splits), smem, stream, (const __nv_bfloat16*)q,
                     (__nv_bfloat16*)out, (const __nv_bfloat16*)cache, p, splits);
  return cuda_status("attention_pages (tokens)");
}

// Whether the tensor-core kernels take the call: rows that 16-byte loads and pair stores address, sizes they are made for.
bool tensor_cores(const void* q, const void* out, const void* cache, const Pages& p) {
  const int group = p.H / p.Hkv;
  return (p.D == 64 || p.D == 128) && p.page_size >= 16 && p.page_size <= 128 && !(p.page_size & (p.page_size - 1)) && group <= 16 &&
         p.top <= MAX_TOP && p.ldq % 8 == 0 && p.ldo % 2 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)cache % 16 == 0 &&
         (uintptr_t)out % 4 == 0 && p.Hkv <= 65535;
}
}  // namespace

// What the call takes, 8 bytes a field (a caller packs them and hands over one address).  chosen int32 [T, Hkv,
// top]; cache [num_pages, 2, Hkv, page_size, D]; sms: the device's multiprocessors.
struct AttentionPagesArgs {
  const void* q;
  int64_t ldq;
  void* out;
  int64_t ldo;
  const void* cache;
  int64_t num_pages;
  const int* table;
  int64_t width;
  const int* cu_seqlens;
  int64_t num_reqs;
  const int *positions, *chosen;
  int64_t top, T, H, Hkv, D, page_size;
  double scale;
  int64_t sms, dtype;
  cudaStream_t stream;
};

DINFER_API int dinfer_attention_pages(const AttentionPagesArgs* a) {
  const int64_t most = 0x7fffffff;
  if (a->num_pages > most || a->width > most || a->num_reqs >= most || a->top > most || a->T > most / 8 || a->H > most || a->Hkv > most || a->D > most || a->page_size > most)
    return refuse(DINFER_BAD_ARGUMENT, "attention_pages: a size beyond 32 bits");
  const void *q = a->q, *cache = a->cache;
  void* out = a->out;
  const int64_t ldq = a->ldq, ldo = a->ldo;
  const int *table = a->table, *cu_seqlens = a->cu_seqlens, *positions = a->positions, *chosen = a->chosen;
  const int num_pages = (int)a->num_pages, width = (int)a->width, num_reqs = (int)a->num_reqs, top = (int)a->top, T = (int)a->T, H = (int)a->H,
            Hkv = (int)a->Hkv, D = (int)a->D, page_size = (int)a->page_size;
  const float scale = (float)a->scale;
  cudaStream_t stream = a->stream;
  const int sms = (int)a->sms, dtype = (int)a->dtype;
  if (T < 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 512 || page_size <= 0 || num_reqs <= 0 || top <= 0 || width < 0)
    return refuse(DINFER_BAD_ARGUMENT, "attention_pages: sizes T=%d H=%d Hkv=%d D=%d page=%d top=%d", T, H, Hkv, D, page_size, top);
  if (H > 65535) return refuse(DINFER_BAD_ARGUMENT, "attention_pages: %d heads", H);
  if (T == 0) return DINFER_OK;
  const Pages p{ldq, ldo, num_pages, table, width, cu_seqlens, num_reqs, positions, chosen, top, T, H, Hkv, D, page_size, scale};
  if (dtype == DINFER_BF16 && tensor_cores(q, out, cache, p)) {
    // CTAs that share a token's keys: as far as all run at the same time (two an SM), each with a tile of its own at least
    int splits = 1;
    while (splits < 8 && (int64_t)T * Hkv * splits * 2 <= 2 * sms && splits * 2 * BN <= (int64_t)top * page_size) splits *= 2;
    if (D == 128) return H / Hkv <= 8 ? run_token<128, 1>(q, out, cache, p, splits, stream) : run_token<128, 2>(q, out, cache, p, splits, stream);
    return H / Hkv <= 8 ? run_token<64, 1>(q, out, cache, p, splits, stream) : run_token<64, 2>(q, out, cache, p, splits, stream);
  }
  if (dtype == DINFER_F32 && float_rows(q, out, cache, p)) {
    const int group = H / Hkv;
#define DINFER_FLOAT(G) return D == 64 ? run_float<64, G>(q, out, cache, p, sms, stream) : run_float<128, G>(q, out, cache, p, sms, stream)
    if (group == 1) DINFER_FLOAT(1);
    if (group == 2) DINFER_FLOAT(2);
    if (group <= 4) DINFER_FLOAT(4);
    DINFER_FLOAT(8);
#undef DINFER_FLOAT
  }
  DINFER_DISPATCH_DTYPE(dtype, E, { return run<E>(q, out, cache, p, stream); });
}

DINFER_DEFINE_LAST_ERROR()

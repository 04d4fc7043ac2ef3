// Attention over chosen pages of the paged cache: token t at position p, head h of key head g's group, reads the keys of the
// pages chosen[t, g, :] (-1: none) up to its own position,
//
//     out[t, h] = sum_i softmax_i(scale q[t, h] . k_i) v_i      over  { i <= p : i / page_size in chosen[t, g] }
//
// A page named twice counts twice; a number outside the request's table, or a page the table does not hold, is no page; a token
// that sees no key gets zeros; rows behind the last request's tokens are left as they are.  Scores, weights and sums in 32-bit.
// What a token does not see is never multiplied, so that it may hold anything.
#include <cooperative_groups.h>

#include "mma_tiles.cuh"

using namespace dinfer;
using namespace dinfer_mma;

namespace {

// The request of token t: the first whose tokens end behind it (every lane of a full warp asks; requests without tokens are passed
// over), -1 where there is none.
__device__ __forceinline__ int request_of(const int* cu, int num_reqs, int t) {
  int ended = 0;
  for (int i0 = 0; i0 < num_reqs; i0 += 32) {
    const int i = i0 + (threadIdx.x & 31);
    ended += __popc(__ballot_sync(0xffffffffu, i < num_reqs && cu[i + 1] <= t));
  }
  return ended < num_reqs && t >= cu[0] ? ended : -1;
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


// ------------------------------------------------------------------------------------------------
// Bfloat16, head sizes 64 and 128, pages of 16 to 128 tokens, groups of up to 16 heads: few tokens (decode steps).
// A CTA owns a (token, key head) and, with splits, a share of its keys.  Tiles of 64 keys (a piece of a page or several pages) ride a
// ring of cp.async stages; a warp takes 16 of a tile's keys as the rows of S^T = K Q^T (the group's heads are the columns, so
// nothing of the product is spent on padding beyond 8 heads) and of O^T += V^T P^T, with a softmax of its own.  The four warps
// meet in shared memory at the end, the CTAs of a (token, key head), a cluster, through distributed shared memory.
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
      // the weights are rounded to bfloat16 for the second product (2^-9 of each; their sum is taken before)
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
  const int64_t orow = (int64_t)t * p.ldo + (int64_t)g * group * D;
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
      out[orow + idx] = __float2bfloat16_rn(L == 0.f ? 0.f : acc / L);
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
    out[orow + idx] = __float2bfloat16_rn(L == 0.f ? 0.f : acc / L);
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

// ------------------------------------------------------------------------------------------------
// The same sizes, many tokens (portions of prompts).  Token by token every page would be read once for each token that chose it; here
// the work is turned round: for every (request, key head, page) the tokens that chose it are listed, and a tile of up to 128 rows
// (tokens of the list x the group's heads) meets the page's keys once, on the tensor cores.  What a tile makes for a (token, page)
// pair is a partial result: the sum of weights times values relative to the pair's own maximum, that maximum and the sum of weights,
// in 32 bits; a last kernel joins the partial results of each token in the order of its list.  Lists are filled with atomic
// counters, so a token's place in a tile varies from run to run, but no row of a tile depends on the others, and results do not vary.
//
// The partial results are the traffic that bounds it (top x D x 4 bytes a token and head, written and read once).  The step is therefore
// cut into slabs, key heads x runs of tokens, one after the other, whose partial results take SLAB_BYTES at most.
#ifndef SLAB_MB
#define SLAB_MB 128
#endif
constexpr int64_t SLAB_BYTES = (int64_t)SLAB_MB << 20;
constexpr int ROWS = 128;
constexpr int64_t MAX_COUNTERS = 1 << 24;   // lists of all slabs (requests x table width x key heads x runs of tokens): 64 MB of counters

struct Slabs {
  int heads, tokens, chunks, count;     // key heads and tokens of a slab, runs of tokens, slabs (key-head part slowest)
  int keys;                             // counters of a slab: heads x requests x table width, to a multiple of 32
  int tile_tokens;                      // tokens of a tile
  int64_t list, tiles;                  // room of a slab: list entries, tiles
  int *counts, *cursors, *base;         // cursors [count][2]: list entries and tiles given out
  int2 *place;                          // of every choice: its list (-1: no page, -2: behind the last request) and its place there
  int2 *entries;                        // of a list: token with the keys it sees of the page in the upper 8 bits, and its pair
  int4* desc;                           // a tile: page, first entry, tokens, key head in the slab
  float *part, *ml;                     // [heads][tokens][top][group][D], and (maximum in log2 units, sum of weights)
  int64_t bytes, zeroed;                // the workspace; what must be zero at the start (from counts on)
};

Slabs slabs_of(const Pages& p, unsigned char* at) {
  Slabs s;
  const int group = p.H / p.Hkv;
  const int64_t per_token = (int64_t)group * p.top * p.D * 4;             // of one key head
  s.tokens = p.T;
  s.chunks = 1;
  while (s.tokens * per_token > SLAB_BYTES && s.tokens > ROWS) {
    ++s.chunks;
    s.tokens = ((p.T + s.chunks - 1) / s.chunks + 31) / 32 * 32;
  }
  s.chunks = (p.T + s.tokens - 1) / s.tokens;
  s.heads = (int)(SLAB_BYTES / (s.tokens * per_token));
  s.heads = s.heads < 1 ? 1 : s.heads > p.Hkv ? p.Hkv : s.heads;
  const int parts = (p.Hkv + s.heads - 1) / s.heads;
  s.heads = (p.Hkv + parts - 1) / parts;
  s.count = parts * s.chunks;
  const int64_t keys = ((int64_t)s.heads * p.num_reqs * p.width + 31) / 32 * 32;
  s.keys = (int)(keys > INT32_MAX / 2 ? INT32_MAX / 2 : keys);
  s.tile_tokens = ROWS / group;
  s.list = (int64_t)s.heads * s.tokens * p.top;
  s.tiles = s.list / s.tile_tokens + (s.list < keys ? s.list : keys) + 1;
  unsigned char* start = at;
  auto take = [&](int64_t bytes) { unsigned char* x = at; at += (bytes + 255) / 256 * 256; return x; };
  s.counts = (int*)take((int64_t)s.count * s.keys * 4);
  s.cursors = (int*)take((int64_t)s.count * 2 * 4);
  s.zeroed = at - start;
  s.base = (int*)take((int64_t)s.count * s.keys * 4);
  s.place = (int2*)take((int64_t)p.T * p.Hkv * p.top * 8);
  s.entries = (int2*)take((int64_t)s.count * s.list * 8);
  s.desc = (int4*)take((int64_t)s.count * s.tiles * 16);
  s.part = (float*)take(s.list * group * p.D * 4);
  s.ml = (float*)take(s.list * group * 8);
  s.bytes = at - start;
  return s;
}

__device__ __forceinline__ int slab_of(const Slabs& s, int t, int g) { return g / s.heads * s.chunks + t / s.tokens; }

__global__ void __launch_bounds__(256) pages_clear_kernel(int4* at, int64_t n) {
  pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) at[i] = make_int4(0, 0, 0, 0);
}

// How often each (request, page) of a slab was chosen, and the place of every choice in its list.  A warp takes 32 tokens of a key head;
// those whose next choice is the same page count together (neighbours choose much the same pages).
__global__ void __launch_bounds__(128)
pages_count_kernel(const Pages p, const Slabs s) {
  pdl_enter();
  const int lane = threadIdx.x & 31, t = blockIdx.x * 32 + lane, g = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (g >= p.Hkv) return;
  int r = -1;
  if (t < p.T && t >= p.cu[0] && t < p.cu[p.num_reqs]) {     // the first request whose tokens end behind it
    int lo = 0, hi = p.num_reqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.cu[mid + 1] > t) hi = mid; else lo = mid + 1;
    }
    r = lo;
  }
  const int pos = r < 0 ? -1 : p.positions[t];
  const int64_t at = ((int64_t)t * p.Hkv + g) * p.top;
  const int slab = slab_of(s, min(t, p.T - 1), g), row = (g % s.heads * p.num_reqs + r) * p.width;
#pragma unroll 4
  for (int i = 0; i < p.top; ++i) {
    const int j = r >= 0 ? p.chosen[at + i] : -1;
    int key = r < 0 ? -2 : -1;
    if (j >= 0 && j < p.width && (int64_t)j * p.page_size <= pos) {
      const int page = p.table[(int64_t)r * p.width + j];
      if (page >= 0 && page < p.num_pages) key = row + j;
    }
    // (the 32 tokens may lie in two slabs: those count apart)
    const unsigned long long id = key >= 0 ? (unsigned long long)slab << 32 | (unsigned)key : ~0ull;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    int first = 0;
    const int leader = __ffs(same) - 1;
    if (key >= 0 && lane == leader) first = atomicAdd(s.counts + (int64_t)slab * s.keys + key, __popc(same));
    first = __shfl_sync(0xffffffffu, first, leader);
    if (t < p.T) s.place[at + i] = make_int2(key, first + __popc(same & ((1u << lane) - 1)));
  }
}

// A list and tiles for every (request, page) that was chosen: a warp adds up its 32 and takes room once.
__global__ void __launch_bounds__(256)
pages_lists_kernel(const Pages p, const Slabs s) {
  pdl_enter();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int lane = threadIdx.x & 31;
  const bool in = i < (int64_t)s.count * s.keys;
  const int slab = in ? (int)(i / s.keys) : 0, key = in ? (int)(i % s.keys) : 0;     // (the same slab in a whole warp)
  const int c = in ? s.counts[i] : 0, tiles = (c + s.tile_tokens - 1) / s.tile_tokens;
  int c_sum = c, t_sum = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, c_sum, o), b = __shfl_up_sync(0xffffffffu, t_sum, o);
    if (lane >= o) { c_sum += a; t_sum += b; }
  }
  int c_at = 0, t_at = 0;
  if (lane == 31 && c_sum > 0) {
    c_at = atomicAdd(s.cursors + slab * 2, c_sum);
    t_at = atomicAdd(s.cursors + slab * 2 + 1, t_sum);
  }
  c_at = __shfl_sync(0xffffffffu, c_at, 31) + c_sum - c;
  t_at = __shfl_sync(0xffffffffu, t_at, 31) + t_sum - tiles;
  if (!in || c == 0) return;
  s.base[i] = c_at;
  const int request_page = key % (p.num_reqs * p.width), gl = key / (p.num_reqs * p.width);
  const int page = p.table[request_page];
  for (int k = 0; k < tiles; ++k)
    s.desc[(int64_t)slab * s.tiles + t_at + k] = make_int4(page, c_at + k * s.tile_tokens, min(s.tile_tokens, c - k * s.tile_tokens), gl);
}

__global__ void __launch_bounds__(128)
pages_fill_kernel(const Pages p, const Slabs s) {
  pdl_enter();
  const int64_t at = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int per = p.Hkv * p.top;
  if (at >= (int64_t)p.T * per) return;
  const int2 place = s.place[at];
  if (place.x < 0) return;
  const int t = (int)(at / per), i = (int)(at - (int64_t)t * per), g = i / p.top, slab = slab_of(s, t, g);
  const int seen = min(p.page_size, p.positions[t] - p.chosen[at] * p.page_size + 1);
  const int pair = (g % s.heads * s.tokens + t % s.tokens) * p.top + i - g * p.top;
  s.entries[(int64_t)slab * s.list + s.base[(int64_t)slab * s.keys + place.x] + place.y] = make_int2(t | seen << 24, pair);
}

// 0 where a packed bfloat16 is not a number or infinite
__device__ __forceinline__ unsigned finite2(unsigned x) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu;
  return x;
}
__device__ __forceinline__ bool odd2(unsigned x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; }

// Tiles of 128 rows, a warp owns 16.  A block takes tile after tile: while it works on one, the next one's keys and values are on their way
// into the other half of its shared memory, and once the scores are made, the next one's rows of Q into the registers that held
// this one's.  Q goes from memory straight into fragments: the order of the elements of a product's sum is free, so a lane takes 16 bytes of its
// rows and of the keys' at the same places, two steps of 16 elements at once.
constexpr int PORTION_NT = ROWS * 2;

template <int D, int P>
__global__ void __launch_bounds__(PORTION_NT, 2)
pages_portion_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ cache, const Pages p, const Slabs s, int slab) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  // [2] x keys [P][D], 16-byte pieces exchanged by (key & 1) * 4, and values [P][D], by key & 7
  __nv_bfloat16* smem = reinterpret_cast<__nv_bfloat16*>(smem_raw);
  pdl_enter();
  const int tiles = s.cursors[slab * 2 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  const int g0 = slab / s.chunks * s.heads, group = p.H / p.Hkv;
  const int64_t plane = (int64_t)p.Hkv * P * D;
  const int4* desc = s.desc + (int64_t)slab * s.tiles;
  const int2* entries = s.entries + (int64_t)slab * s.list;
  float *s_part = s.part, *s_ml = s.ml;
  constexpr int C = D / 8;
  auto load_tile = [&](const int4& d, int stage) {
    const __nv_bfloat16* keys = cache + (int64_t)d.x * 2 * plane + (int64_t)(g0 + d.w) * P * D;
    __nv_bfloat16* k = smem + stage * 2 * P * D;
    const int chunk = threadIdx.x % C;
#pragma unroll
    for (int row = threadIdx.x / C; row < P; row += PORTION_NT / C) {
      cp_async16(k + row * D + ((chunk ^ ((row & 1) << 2)) << 3), keys + row * D + chunk * 8, true);
      cp_async16(k + P * D + row * D + ((chunk ^ (row & 7)) << 3), keys + plane + row * D + chunk * 8, true);
    }
  };
  // this lane's two rows of every tile: a token of its list and a head of the group
  int row_token[2], row_head[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = warp * 16 + gr + 8 * u;
    row_token[u] = row / group;
    row_head[u] = row - row_token[u] * group;
  }
  int2 entry[2];                                            // (of a tile; x < 0: no row)
  auto load_entries = [&](const int4& d) {
#pragma unroll
    for (int u = 0; u < 2; ++u) entry[u] = row_token[u] < d.z ? entries[d.y + row_token[u]] : make_int2(-1, 0);
  };
  uint4 qa[D / 32][2];
  int part[2], seen[2];                                     // (pair, head) of the partial results, -1: no row; keys that the row sees
  auto load_rows = [&](const int4& d) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool in = row_token[u] < d.z;
      const int t = entry[u].x & 0xffffff;
      part[u] = in ? entry[u].y * group + row_head[u] : -1;
      seen[u] = in ? (unsigned)entry[u].x >> 24 : P;
      const __nv_bfloat16* row = q + (in ? (int64_t)t * p.ldq + (int64_t)((g0 + d.w) * group + row_head[u]) * D + tq * 8 : 0);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) qa[k][u] = *reinterpret_cast<const uint4*>(row + k * 32);
    }
  };
  int tile = blockIdx.x;
  int4 d = tile < tiles ? desc[tile] : make_int4(0, 0, 0, 0), d_next = d;
  if (tile < tiles) {
    load_tile(d, 0);
    load_entries(d);
    load_rows(d);
    if (tile + (int)gridDim.x < tiles) d_next = desc[tile + gridDim.x];
  }
  cp_async_commit();
  const float scale_log2 = p.scale * 1.4426950408889634f;
  for (int stage = 0; tile < tiles; stage ^= 1) {
    const int next = tile + gridDim.x;
    cp_async_wait<0>();
    __syncthreads();                                        // the tile is here, and everyone is done with the one before
    if (next < tiles) {
      load_tile(d_next, stage ^ 1);
      load_entries(d_next);
    }
    cp_async_commit();
    const __nv_bfloat16 *sK = smem + stage * 2 * P * D, *sV = sK + P * D;
    const int mine[2] = {part[0], part[1]}, sees[2] = {seen[0], seen[1]};
    const bool active = warp * 16 < d.z * group;
    unsigned pa[P / 16][4];
    if (active) {
      float st[P / 8][4];
#pragma unroll
      for (int n = 0; n < P / 8; ++n) st[n][0] = st[n][1] = st[n][2] = st[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
#pragma unroll
        for (int n = 0; n < P / 8; ++n) {
          const int row = n * 8 + gr;
          const uint4 b = *reinterpret_cast<const uint4*>(sK + row * D + (((k * 4 + tq) ^ ((row & 1) << 2)) << 3));
          mma_bf16(st[n], qa[k][0].x, qa[k][1].x, qa[k][0].y, qa[k][1].y, b.x, b.y);
          mma_bf16(st[n], qa[k][0].z, qa[k][1].z, qa[k][0].w, qa[k][1].w, b.z, b.w);
        }
      float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < P / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          st[n][c] = n * 8 + 2 * tq + (c & 1) < sees[c >> 1] ? st[n][c] * scale_log2 : -INFINITY;
          mx[c >> 1] = fmaxf(mx[c >> 1], st[n][c]);
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
        mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
      }
      const float base[2] = {mx[0] == -INFINITY ? 0.f : mx[0], mx[1] == -INFINITY ? 0.f : mx[1]};
#pragma unroll
      for (int n = 0; n < P / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          st[n][c] = fast_exp2(st[n][c] - base[c >> 1]);
          l[c >> 1] += st[n][c];
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
      }
      // the weights are rounded to bfloat16 for the second product (2^-9 of each; their sum is taken before)
#pragma unroll
      for (int k = 0; k < P / 16; ++k) {
        pa[k][0] = pack_bf16(st[2 * k][0], st[2 * k][1]);
        pa[k][1] = pack_bf16(st[2 * k][2], st[2 * k][3]);
        pa[k][2] = pack_bf16(st[2 * k + 1][0], st[2 * k + 1][1]);
        pa[k][3] = pack_bf16(st[2 * k + 1][2], st[2 * k + 1][3]);
      }
      if (tq == 0)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (mine[u] >= 0) *reinterpret_cast<float2*>(s_ml + (int64_t)mine[u] * 2) = make_float2(mx[u], l[u]);
    }
    if (next < tiles) load_rows(d_next);
    // A value that is not a finite number, in a page that some row sees in part: a weight of zero would carry it into rows that do not
    // see it.  Those products are then made without such values, and rows that see them get them one by one.
    bool odd = false;
    if (active && __any_sync(0xffffffffu, sees[0] < P || sees[1] < P)) {
      for (int i = lane; i < P * C; i += 32) {
        const uint4 v = *reinterpret_cast<const uint4*>(sV + i * 8);
        odd |= odd2(v.x) || odd2(v.y) || odd2(v.z) || odd2(v.w);
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (active) {
#pragma unroll 2
      for (int db = 0; db < D / 16; ++db) {
        float o[2][4] = {};
#pragma unroll
        for (int k = 0; k < P / 16; ++k) {
          unsigned b[4];
          const int row = k * 16 + (lane & 15);
          ldmatrix_x4_trans(b, sV + row * D + (((db * 2 + (lane >> 4)) ^ (row & 7)) << 3));
          if (odd)
#pragma unroll
            for (int x = 0; x < 4; ++x) b[x] = finite2(b[x]);
          mma_bf16(o[0], pa[k][0], pa[k][1], pa[k][2], pa[k][3], b[0], b[1]);
          mma_bf16(o[1], pa[k][0], pa[k][1], pa[k][2], pa[k][3], b[2], b[3]);
        }
        if (odd) {
#pragma unroll
          for (int k = 0; k < P / 16; ++k)
            for (int x = 0; x < 16; ++x) {
              const int key = k * 16 + x, from = (lane & ~3) | ((x & 7) >> 1);
              const unsigned w0 = __shfl_sync(0xffffffffu, x < 8 ? pa[k][0] : pa[k][2], from);
              const unsigned w1 = __shfl_sync(0xffffffffu, x < 8 ? pa[k][1] : pa[k][3], from);
              const float w[2] = {__uint_as_float(x & 1 ? w0 & 0xffff0000u : w0 << 16), __uint_as_float(x & 1 ? w1 & 0xffff0000u : w1 << 16)};
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const int col = db * 16 + n * 8 + 2 * tq + (c & 1);
                  const float v = __bfloat162float(sV[key * D + (((col >> 3) ^ (key & 7)) << 3) + (col & 7)]);
                  if (!isfinite(v) && key < sees[c >> 1]) o[n][c] += w[c >> 1] * v;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (mine[u] >= 0) {
            float* dst = s_part + (int64_t)mine[u] * D + db * 16 + 2 * tq;
            *reinterpret_cast<float2*>(dst) = make_float2(o[0][2 * u], o[0][2 * u + 1]);
            *reinterpret_cast<float2*>(dst + 8) = make_float2(o[1][2 * u], o[1][2 * u + 1]);
          }
      }
    }
    tile = next;
    d = d_next;
    if (tile + (int)gridDim.x < tiles) d_next = desc[tile + gridDim.x];
  }
  cp_async_wait<0>();
}

// A warp per (token, head) of a slab: the partial results of the token's pages, in the order of its list.
template <int D>
__global__ void __launch_bounds__(256)
pages_join_kernel(__nv_bfloat16* __restrict__ out, const Pages p, const Slabs s, int slab) {
  pdl_enter();
  constexpr int E = D / 32, AHEAD = 8;                      // elements a lane; partial results asked for at once
  struct alignas(E * 4) Vec { float v[E]; };
  const int lane = threadIdx.x & 31, group = p.H / p.Hkv;
  const int g0 = slab / s.chunks * s.heads, t0 = slab % s.chunks * s.tokens;
  const int heads = min(s.heads, p.Hkv - g0) * group;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int tl = w / heads, hl = w - tl * heads, t = t0 + tl;
  if (tl >= s.tokens || t >= p.T) return;
  const int gl = hl / group, h = hl - gl * group;
  const int2* place = s.place + ((int64_t)t * p.Hkv + g0 + gl) * p.top;
  const int pair0 = (gl * s.tokens + tl) * p.top;
  const float2* ml = reinterpret_cast<const float2*>(s.ml) + h;
  const float* part = s.part + (int64_t)h * D + lane * E;
  float M = -INFINITY, L = 0.f, acc[E] = {};
  for (int i0 = 0; i0 < p.top; i0 += 32) {
    const int mine = i0 + lane < p.top ? place[i0 + lane].x : -1;
    if (i0 == 0 && __shfl_sync(0xffffffffu, mine, 0) == -2) return;       // behind the last request
    const float2 x = mine >= 0 ? ml[(pair0 + i0 + lane) * group] : make_float2(-INFINITY, 0.f);
    const float m = fmaxf(M, warp_max(x.x)), base = m == -INFINITY ? 0.f : m;
    const float f = mine >= 0 ? fast_exp2(x.x - base) : 0.f, again = fast_exp2(M - base);
    M = m;
    L = fmaf(L, again, warp_sum(f * x.y));
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= again;
    // the pages there are, in the list's order, several asked for at once
    unsigned mask = __ballot_sync(0xffffffffu, mine >= 0);
    while (mask) {
      Vec v[AHEAD];
      float w_i[AHEAD];
      unsigned rest = mask;
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = rest ? __ffs(rest) - 1 : __ffs(mask) - 1;
        w_i[u] = __shfl_sync(0xffffffffu, f, i);
        v[u] = *reinterpret_cast<const Vec*>(part + (int64_t)(pair0 + i0 + i) * group * D);
        if (!rest) w_i[u] = -1.f;
        rest &= rest - 1;
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (w_i[u] >= 0.f || w_i[u] != w_i[u])
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(w_i[u], v[u].v[e], acc[e]);
      mask = rest;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  __nv_bfloat16* dst = out + (int64_t)t * p.ldo + (int64_t)(g0 + gl) * group * D + (int64_t)h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<unsigned*>(dst + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, int P>
int run_portions(const void* q, void* out, const void* cache, const Pages& p, const Slabs& s, int sms, cudaStream_t stream) {
  auto kernel = pages_portion_kernel<D, P>;
  constexpr int smem = 2 * 2 * P * D * 2;
  if (smem > 48 * 1024) {
    static thread_local int set_for = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (set_for != dev) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return cuda_status("attention_pages: shared memory");
      set_for = dev;
    }
  }
  launch_pdl(pages_clear_kernel, dim3((unsigned)((s.zeroed / 16 + 255) / 256)), dim3(256), 0, stream, (int4*)s.counts, s.zeroed / 16);
  launch_pdl(pages_count_kernel, dim3((p.T + 31) / 32, (p.Hkv + 3) / 4), dim3(128), 0, stream, p, s);
  launch_pdl(pages_lists_kernel, dim3((unsigned)(((int64_t)s.count * s.keys + 255) / 256)), dim3(256), 0, stream, p, s);
  launch_pdl(pages_fill_kernel, dim3((unsigned)(((int64_t)p.T * p.Hkv * p.top + 127) / 128)), dim3(128), 0, stream, p, s);
  const int64_t joined = ((int64_t)s.tokens * s.heads * (p.H / p.Hkv) + 7) / 8;
  for (int i = 0; i < s.count; ++i) {
    launch_pdl(kernel, dim3((unsigned)(s.tiles < 2 * sms ? s.tiles : 2 * sms)), dim3(PORTION_NT), smem, stream, (const __nv_bfloat16*)q, (const __nv_bfloat16*)cache, p, s, i);
    launch_pdl(pages_join_kernel<D>, dim3((unsigned)joined), dim3(256), 0, stream, (__nv_bfloat16*)out, p, s, i);
  }
  return cuda_status("attention_pages (portions)");
}

// Whether the tensor-core kernels take the call: rows that 16-byte loads and pair stores address, sizes they are made for.
bool tensor_cores(const void* q, const void* out, const void* cache, const Pages& p) {
  const int group = p.H / p.Hkv;
  return (p.D == 64 || p.D == 128) && p.page_size >= 16 && p.page_size <= 128 && !(p.page_size & (p.page_size - 1)) && group <= 16 &&
         p.top <= MAX_TOP && p.ldq % 8 == 0 && p.ldo % 2 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)cache % 16 == 0 &&
         (uintptr_t)out % 4 == 0 && p.Hkv <= 65535;
}
}  // namespace

// Bytes of workspace with which the call takes its portions' form (any smaller one: token by token).
DINFER_API int64_t dinfer_attention_pages_workspace(int num_reqs, int width, int top, int T, int H, int Hkv, int D) {
  if (T <= 0 || T >= 1 << 24 || H <= 0 || Hkv <= 0 || H % Hkv || H / Hkv > 16 || top <= 0 || width <= 0 || num_reqs <= 0 || D <= 0) return 0;
  Pages p{};
  p.width = width; p.num_reqs = num_reqs; p.top = top; p.T = T; p.H = H; p.Hkv = Hkv; p.D = D;
  if ((int64_t)Hkv * num_reqs * width > MAX_COUNTERS) return 0;
  const Slabs s = slabs_of(p, nullptr);
  return (int64_t)s.count * s.keys > MAX_COUNTERS ? 0 : s.bytes;
}

// chosen int32 [T, Hkv, top]; cache [num_pages, 2, Hkv, page_size, D].
DINFER_API int dinfer_attention_pages(const void* q, int64_t ldq, void* out, int64_t ldo, const void* cache, int num_pages,
                                      const int* table, int width, const int* cu_seqlens, int num_reqs, const int* positions,
                                      const int* chosen, int top, int T, int H, int Hkv, int D, int page_size, float scale,
                                      void* workspace, int64_t workspace_bytes, int sms, int dtype, cudaStream_t stream) {
  if (T < 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 512 || page_size <= 0 || num_reqs <= 0 || top <= 0 || width < 0)
    return refuse(DINFER_BAD_ARGUMENT, "attention_pages: sizes T=%d H=%d Hkv=%d D=%d page=%d top=%d", T, H, Hkv, D, page_size, top);
  if ((H + WARPS - 1) / WARPS > 65535) return refuse(DINFER_BAD_ARGUMENT, "attention_pages: %d heads", H);
  if (T == 0) return DINFER_OK;
  const Pages p{ldq, ldo, num_pages, table, width, cu_seqlens, num_reqs, positions, chosen, top, T, H, Hkv, D, page_size, scale};
  if (dtype == DINFER_BF16 && tensor_cores(q, out, cache, p)) {
    const int64_t need = workspace ? dinfer_attention_pages_workspace(num_reqs, width, top, T, H, Hkv, D) : 0;
    if (need > 0 && workspace_bytes >= need) {
      const Slabs s = slabs_of(p, (unsigned char*)workspace);
#define DINFER_PAGES(P_) case P_: return D == 128 ? run_portions<128, P_>(q, out, cache, p, s, sms, stream) : run_portions<64, P_>(q, out, cache, p, s, sms, stream)
      switch (page_size) { DINFER_PAGES(16); DINFER_PAGES(32); DINFER_PAGES(64); DINFER_PAGES(128); }
#undef DINFER_PAGES
    }
    // CTAs that share a token's keys: as far as all run at the same time (two an SM), each with a tile of its own at least
    int splits = 1;
    while (splits < 8 && (int64_t)T * Hkv * splits * 2 <= 2 * sms && splits * 2 * BN <= (int64_t)top * page_size) splits *= 2;
    if (D == 128) return H / Hkv <= 8 ? run_token<128, 1>(q, out, cache, p, splits, stream) : run_token<128, 2>(q, out, cache, p, splits, stream);
    return H / Hkv <= 8 ? run_token<64, 1>(q, out, cache, p, splits, stream) : run_token<64, 2>(q, out, cache, p, splits, stream);
  }
  DINFER_DISPATCH_DTYPE(dtype, E, { return run<E>(q, out, cache, p, stream); });
}

DINFER_DEFINE_LAST_ERROR()

// Attention over chosen pages for many tokens (portions of prompts) on the 5th-generation tensor cores (tcgen05 + TMEM + TMA):
// bfloat16, head sizes 64 and 128, groups of up to 128 heads, pages of 16 to 128 tokens.  Token t at position p, head h of key head g's
// group:
//     out[t, h] = sum_i softmax_i(scale q[t, h] . k_i) v_i      over  { i <= p : i / page_size in chosen[t, g] }
//
// Neighbouring tokens choose much the same pages.  The tokens of a request are cut into row tiles of 128 (token, head) rows, two to a
// block, and for every (pair of row tiles, key head) a first kernel collects the pages that any of its tokens chose, ascending, with one
// bit per token that says whether it did.  The block then walks that list as the attention over a whole context walks its keys:
//     S[128, 64]  = Q K^T          tcgen05.mma, Q and K K-major in shared memory, S in tensor memory (two buffers)
//     P = softmax step             one thread per row (= TMEM lane): tcgen05.ld, keys of pages that the row's token did not choose
//                                  (or that lie behind it) to -inf, exp2, P as bfloat16 over the columns of its S
//     O[128, D]  += P V            tcgen05.mma accumulating in tensor memory; O is rescaled in place only when a row's maximum grows
//                                  by more than 2^8
// A page is read once for the 256 rows, not once for each token that chose it.  A warp none of whose rows sees a tile passes it with zeros.
// 4096 tokens of 32 heads of 128 over 8, 16 pages of 64 each behind 28672, take 354 to 378 us by the clock under load (token by token 2700).  64
// neighbouring tokens choose some 85 pages among them, so that the products are five times what the tokens chose: 1.0 PFLOP/s, 59 % of a
// library product's rate.  Bound by Q K^T and its place in the chain of a key tile (1.1 us; without the softmax as long, with one product of eight
// in Q K^T a third less: every product reads 128 rows of Q for 64 keys from shared memory) and by the last of four rounds of blocks, half
// full.  A row tile that passed by the key tiles none of its tokens chose (a fifth) gained nothing, since both walk the same ring.
// Few tokens fill few SMs: then the blocks of a cluster share a pair's list, a run of its key tiles each, and fold their results
// through distributed shared memory behind two cluster barriers, each block writing out a share of the 256 rows.
//
// Warp roles (384 threads): warp 0 brings Q (once) and K, warp 11 V, page by page through a map over the cache, each on a ring of its own;
// warps 1 and 10 issue the products of the two row tiles; warps 2..9 are softmax and output, four per row tile.  Every mbarrier wait
// is bounded.
//
// A weight of zero times a value that is not a finite number is not zero: such a value in any of a block's pages makes an element of every
// row's result one that is not finite.  Where a row's result has one, the block's rows are made again at its end, key by key and
// only from keys that they see.  The same goes for a block one of whose tokens names a page twice (it then counts twice, which a bit
// cannot say).
#include <cuda.h>
#include <math.h>

#include "page_batch.cuh"
#include "split_umma.cuh"
#include "umma_attention.cuh"

using namespace dinfer;
using namespace dinfer_umma;
using dinfer_split::commit_if;
using dinfer_split::elect_lane;
using dinfer_split::mma_if;
using dinfer_split::mma_ts_if;
using dinfer_split::uniform;

namespace {

constexpr int BM = 128, BN = 64, STAGES = 4, NTHREADS = 384;    // BM rows of a row tile, two row tiles a block
constexpr int MMA_WARP_B = 10, V_WARP = 11;                     // the second MMA issuer, the V producer
constexpr int LIST_SLOTS = 1024;                                // entries of a list in shared memory (fewer where a row tile has more than 32 tokens)
constexpr int TWICE = 1 << 30;                                  // in a list's count: some token names a page twice

struct Params {
  const __nv_bfloat16* q; int64_t ldq;
  __nv_bfloat16* out; int64_t ldo;
  const __nv_bfloat16* cache; int num_pages;
  const int* table; int width;
  const int* cu; int B;
  const int* positions;
  const int* chosen; int top;
  int T, H, Hkv, group, page_size;
  float scale, scale_log2;
  int tile_tokens;                     // tokens of a row tile
  int words;                           // 32-bit words of its bits
  int unit, per_tile;                  // keys of a list entry (a page, or 64 of its keys), entries of a key tile
  int cap;                             // entries that a list has room for (a multiple of per_tile)
  int pairs;                           // pairs of row tiles that the grid counts
  int ksplit;                          // blocks of a cluster that share a pair's list (1, 2, 4 or 8)
  int* counts;                         // [pairs][Hkv]: entries, to a multiple of per_tile
  int2* entries;                       // [pairs][Hkv][cap]: first row of the entry's keys in key head 0's share of the cache (-1: none), first position
  unsigned* masks;                     // [pairs][Hkv][cap][2][words]
  int* status;
};

// The pair of row tiles `y` of the batch (every lane of a full warp asks): request, first token, tokens; request -1 beyond the last.
__device__ __forceinline__ int3 pair_of(const Params& p, int y) { return token_tile(p.cu, p.B, 2 * p.tile_tokens, y); }

// The list of a pair of row tiles and key head: bits of the pages of a window in shared memory, then the pages that have any, in order.
constexpr int LIST_NT = 256, WINDOW_WORDS = 8192;

__global__ void __launch_bounds__(LIST_NT) page_lists_kernel(const Params p) {
  __shared__ unsigned s_bits[WINDOW_WORDS];
  __shared__ int s_warp[LIST_NT / 32];
  pdl_enter();
  const int g = blockIdx.x, y = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int3 pair = pair_of(p, y);
  if (pair.x < 0) return;
  const int* table = p.table + (int64_t)pair.x * p.width;
  const int64_t at = ((int64_t)y * p.Hkv + g);
  int2* entries = p.entries + at * p.cap;
  unsigned* masks = p.masks + at * p.cap * 2 * p.words;
  const int per_page = p.page_size / p.unit, bits = 2 * p.words, window = WINDOW_WORDS / bits;
  int n = 0, twice = 0;                                         // entries so far; whether a token names a page twice
  int far = -1;                                                 // (a page behind the furthest token's own is seen by none)
  for (int tl = lane; tl < pair.z; tl += 32) far = max(far, p.positions[pair.y + tl]);
  far = __reduce_max_sync(0xffffffffu, far);
  const int last = far < 0 ? -1 : min(p.width - 1, far / p.page_size);
  for (int w0 = 0; w0 <= last; w0 += window) {
    const int pages = min(window, last + 1 - w0);
    for (int i = threadIdx.x; i < pages * bits; i += LIST_NT) s_bits[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < pair.z * p.top; i += LIST_NT) {
      const int tl = i / p.top, t = pair.y + tl, j = p.chosen[((int64_t)t * p.Hkv + g) * p.top + i - tl * p.top];
      if (j >= w0 && j < w0 + pages && (int64_t)j * p.page_size <= p.positions[t]) {
        const int w = tl / p.tile_tokens, bit = tl - w * p.tile_tokens;
        const unsigned mine = 1u << (bit & 31);
        if (atomicOr(&s_bits[(j - w0) * bits + w * p.words + (bit >> 5)], mine) & mine) twice = 1;
      }
    }
    __syncthreads();
    for (int j0 = 0; j0 < pages; j0 += LIST_NT) {
      const int j = j0 + threadIdx.x;
      bool in = false;
      int page = -1;
      if (j < pages) {
        for (int w = 0; w < bits; ++w) in |= s_bits[j * bits + w] != 0;
        if (in) page = table[w0 + j];
        in = in && page >= 0 && page < p.num_pages;
      }
      const unsigned ball = __ballot_sync(0xffffffffu, in);
      if (lane == 0) s_warp[warp] = __popc(ball);
      __syncthreads();
      int below = 0, all = 0;
#pragma unroll
      for (int w = 0; w < LIST_NT / 32; ++w) {
        below += w < warp ? s_warp[w] : 0;
        all += s_warp[w];
      }
      if (in) {
        const int e0 = n + (below + __popc(ball & ((1u << lane) - 1))) * per_page;
        for (int x = 0; x < per_page; ++x) {
          entries[e0 + x] = make_int2(page * 2 * p.Hkv * p.page_size + x * p.unit, (w0 + j) * p.page_size + x * p.unit);
          for (int w = 0; w < bits; ++w) masks[(int64_t)(e0 + x) * bits + w] = s_bits[j * bits + w];
        }
      }
      n += all * per_page;
      __syncthreads();
    }
  }
  const int full = (n + p.per_tile - 1) / p.per_tile * p.per_tile;
  for (int e = n + threadIdx.x; e < full; e += LIST_NT) {       // the last key tile is filled up with entries that nobody sees
    entries[e] = make_int2(-1, 0);
    for (int w = 0; w < bits; ++w) masks[(int64_t)e * bits + w] = 0;
  }
  twice = __syncthreads_or(twice);
  if (threadIdx.x == 0) p.counts[at] = full | (twice ? TWICE : 0);
}

// The rows of a block once more, a warp per row and key by key, from nothing but what the row's token sees.
template <int D>
__device__ __noinline__ void rows_again(const Params& p, int request, int first, int tokens, int g, int row0, int row1) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int* table = p.table + (int64_t)request * p.width;
  const int64_t plane = (int64_t)p.Hkv * p.page_size * D;
  for (int row = row0 + warp; row < row1; row += NTHREADS / 32) {  // of the pair's 256
    const int w = row / BM, r = row % BM, token = r / p.group;
    if (token >= p.tile_tokens || w * p.tile_tokens + token >= tokens) continue;
    const int t = first + w * p.tile_tokens + token, h = g * p.group + r % p.group, pos = p.positions[t];
    float qv[D / 32], acc[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      qv[c] = __bfloat162float(p.q[(int64_t)t * p.ldq + (int64_t)h * D + lane + 32 * c]) * p.scale;
      acc[c] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    bool any = false;
    for (int i = 0; i < p.top; ++i) {
      const int j = p.chosen[((int64_t)t * p.Hkv + g) * p.top + i];
      if (j < 0 || j >= p.width || (int64_t)j * p.page_size > pos) continue;
      const int page = table[j];
      if (page < 0 || page >= p.num_pages) continue;
      const __nv_bfloat16* kp = p.cache + (int64_t)page * 2 * plane + (int64_t)g * p.page_size * D;
      const int keys = min(p.page_size, pos - j * p.page_size + 1);
      any = true;
      for (int o = 0; o < keys; ++o) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) s = fmaf(qv[c], __bfloat162float(kp[o * D + lane + 32 * c]), s);
        s = warp_sum(s);
        const float n = fmaxf(m, s), base = n == -INFINITY ? 0.f : n, alpha = expf(m - base), w = expf(s - base);
        m = n;
        l = fmaf(l, alpha, w);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(acc[c], alpha, w * __bfloat162float(kp[plane + o * D + lane + 32 * c]));
      }
    }
    const float inv = any ? 1.f / l : 0.f;                      // (scores of -inf alone: 0 / 0)
#pragma unroll
    for (int c = 0; c < D / 32; ++c) p.out[(int64_t)t * p.ldo + (int64_t)h * D + lane + 32 * c] = __float2bfloat16_rn(acc[c] * inv);
  }
}

// Whether token t sees any key of the pages it chose.  (Not inlined: the registers of this rare way are not the kernel's.)
__device__ __noinline__ bool sees_a_key(const Params& p, int request, int t, int g) {
  const int *chosen = p.chosen + ((int64_t)t * p.Hkv + g) * p.top, *table = p.table + (int64_t)request * p.width;
  const int width = p.width, num_pages = p.num_pages, page_size = p.page_size, top = p.top, pos = p.positions[t];
  for (int i = 0; i < top; ++i) {
    const int j = chosen[i];
    if (j < 0 || j >= width || (int64_t)j * page_size > pos) continue;
    const int page = table[j];
    if (page >= 0 && page < num_pages) return true;
  }
  return false;
}

template <int D> constexpr size_t smem_bytes() {
  return (size_t)(2 * BM * D * 2 + 2 * STAGES * BN * D * 2) + 1024;
}

__device__ __forceinline__ uint64_t pair_f32(float lo, float hi) { return (uint64_t)__float_as_uint(hi) << 32 | __float_as_uint(lo); }

// NP: entries of a key tile
template <int D, int NP>
__global__ void __launch_bounds__(NTHREADS, 1)
attention_pages_umma_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, const Params p) {
  constexpr int NH = D / 64;                          // 64-wide halves of the head
  constexpr uint32_t Q_HALF = BM * 128, KV_HALF = BN * 128;
  constexpr uint32_t Q_BYTES = NH * Q_HALF, KV_BYTES = NH * KV_HALF;
  constexpr int TMEM_COLS = 512, O_COL = 256;         // S of (row tile w, buffer b) at (2w + b) * 64; O of A 256, of B 384
  extern __shared__ unsigned char smem_dyn[];
  __shared__ __align__(8) uint64_t q_full, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES],
      s_full[2][2], p_full[2][2], pv_done[2], o_full[2];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_odd;
  __shared__ int s_first[LIST_SLOTS];                  // the list's beginning: first positions and bits
  __shared__ unsigned s_bits[LIST_SLOTS * 2];
  __shared__ float x_max[2 * BM], x_sum[2 * BM];       // what the other blocks of a cluster found for the rows that this one writes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.ksplit > 1 ? (int)cluster_ctarank() : 0, hk = blockIdx.x / p.ksplit;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
    mbar_init(smem_u32(&q_full), 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&k_full[s]), 1); mbar_init(smem_u32(&k_empty[s]), 2);       // empty: both MMA issuers
      mbar_init(smem_u32(&v_full[s]), 1); mbar_init(smem_u32(&v_empty[s]), 2);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&s_full[w][0]), 1);
      mbar_init(smem_u32(&s_full[w][1]), 1);
      mbar_init(smem_u32(&p_full[w][0]), 4);               // an arrival a warp; one for each buffer, since a warp may be a tile ahead
      mbar_init(smem_u32(&p_full[w][1]), 4);
      mbar_init(smem_u32(&pv_done[w]), 1);
      mbar_init(smem_u32(&o_full[w]), 1);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_enter();
  const int3 pair = pair_of(p, blockIdx.y);
  if (pair.x < 0) return;                              // beyond the batch's pairs
  const int64_t at = (int64_t)blockIdx.y * p.Hkv + hk;
  // this block's run of the list's key tiles
  const int count = p.counts[at], all_tiles = (count & ~TWICE) / p.per_tile, per = (all_tiles + p.ksplit - 1) / p.ksplit;
  const int tile0 = min(rank * per, all_tiles), n_tiles = min(per, all_tiles - tile0);
  const int2* entries = p.entries + at * p.cap + tile0 * p.per_tile;
  const unsigned* masks = p.masks + (at * p.cap + tile0 * p.per_tile) * 2 * p.words;
  const bool b_on = pair.z > p.tile_tokens;            // the second row tile exists

  const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  const uint32_t sQ = base, sK = sQ + 2 * Q_BYTES, sV = sK + STAGES * KV_BYTES;
  if (NP > 1 && n_tiles > 0 && n_tiles <= STAGES) {
    // the last tile may have entries that are no page, whose slots hold what was there: zeros, if no tile came before on its stage
    // (what is not a finite number would have the block's rows made again, for nothing)
    const uint32_t at0 = (n_tiles - 1) * KV_BYTES;
    for (int i = threadIdx.x; i < (int)(2 * KV_BYTES / 16); i += NTHREADS) {
      const uint32_t off = i < (int)(KV_BYTES / 16) ? sK + at0 + i * 16 : sV + at0 + i * 16 - KV_BYTES;
      *reinterpret_cast<uint4*>(smem_dyn + (off - smem_u32(smem_dyn))) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before TMA writes the same bytes
    __syncthreads();
  }
  const int held = min(n_tiles * p.per_tile, LIST_SLOTS / p.words), bits = 2 * p.words;
  if (warp == 0) {                                                 // the producer of Q and K needs no more than the barriers it has set up
    if (lane == 0) s_odd = count & TWICE ? 1 : 0;
    asm volatile("bar.arrive 1, %0;" ::"n"(NTHREADS) : "memory");
  } else {
    if (warp == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      for (int i = threadIdx.x - 64; i < held; i += NTHREADS - 64) s_first[i] = entries[i].y;
      for (int i = threadIdx.x - 64; i < held * bits; i += NTHREADS - 64) s_bits[i] = masks[i];
    }
    tc_fence_before();
    asm volatile("bar.sync 1, %0;" ::"n"(NTHREADS) : "memory");
    tc_fence_after();
  }
  const uint32_t tmem = s_tmem_base;

  if (warp == 0 || warp == V_WARP) {
    // ---- TMA producers: warp 0 Q (once, lane 0) and the K tiles, another warp the V tiles; per tile one copy per entry and 64-wide
    // half, spread over the lanes.  The next tile's entries are asked for while the ring's stage is waited for.
    const int kv = warp == 0 ? 0 : 1;
    if (kv == 0 && lane == 0) {
      const uint32_t qb = smem_u32(&q_full);
      // (a box has tile_tokens x group rows, at most 128)
      const uint32_t rows = (uint32_t)(p.tile_tokens * p.group) * 128;
      mbar_expect_tx(qb, (b_on ? 2 : 1) * NH * rows);
      for (int w = 0; w < (b_on ? 2 : 1); ++w)
        for (int h = 0; h < NH; ++h)
          tma_load_3d(sQ + w * Q_BYTES + h * Q_HALF, &map_q, h * 64, hk * p.group, pair.y + w * p.tile_tokens, qb);
    }
    const int n_ops = p.per_tile * NH, x = lane / NH, h = lane % NH;       // copies of a tile, <= 8
    const bool mine = lane < n_ops;
    int row = mine && n_tiles > 0 ? entries[x].x : -1;
    for (int j = 0; j < n_tiles; ++j) {
      const int s = j % STAGES;
      const bool valid = row >= 0;
      const uint32_t bytes = __reduce_add_sync(0xffffffffu, valid ? (uint32_t)(p.unit * 128) : 0u);
      const int row_k = row + (kv * p.Hkv + hk) * p.page_size;
      const int next = mine && j + 1 < n_tiles ? entries[(j + 1) * p.per_tile + x].x : -1;
      bool ok = true;
      if (lane == 0) ok = mbar_wait(smem_u32(kv == 0 ? &k_empty[s] : &v_empty[s]), ((j / STAGES) & 1) ^ 1);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) { if (lane == 0) { s_abort = 1; atomicExch(p.status, 61); } break; }
      const uint32_t bar = smem_u32(kv == 0 ? &k_full[s] : &v_full[s]);
      if (lane == 0) {
        if (bytes == 0) mbar_arrive(bar); else mbar_expect_tx(bar, bytes);
      }
      __syncwarp();
      if (valid) tma_load_2d((kv == 0 ? sK : sV) + s * KV_BYTES + h * KV_HALF + x * p.unit * 128, &map_kv, h * 64, row_k, bar);
      row = next;
    }
  } else if (warp == 1 || warp == MMA_WARP_B) {
    // ---- MMA issue: a warp per row tile, one lane of which issues.  Each runs its tile's chain on its own, so neither waits for the
    // other's softmax; the K and V stages go back to the producers when both have committed (or, without a second row tile, plainly
    // arrived on) their empty barriers.
    const int w = uniform(warp == 1 ? 0 : 1);
    const bool on = w == 0 || b_on;
    const uint32_t lead = elect_lane(), tm = uniform(tmem);
    constexpr uint32_t idesc_qk = idesc_bf16(BM, BN, 0), idesc_pv = idesc_bf16(BM, D, 1);
    const uint64_t dq = desc_k_major(uniform(sQ + w * Q_BYTES)), dk = desc_k_major(uniform(sK)), dv = desc_mn_major(uniform(sV), KV_HALF);
    const uint32_t o_tmem = tm + O_COL + w * 128;
    auto issue_qk = [&](int t) {                                    // S_w[t % 2] = Q_w K(t)^T
      const uint64_t dks = dk + (uint64_t)((t % STAGES) * (KV_BYTES >> 4));
      const uint32_t s_tmem = tm + (2 * w + (t & 1)) * BN;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        mma_if(lead, s_tmem, dq + (uint64_t)(((k / 4) * Q_HALF + (k % 4) * 32) >> 4),
               dks + (uint64_t)(((k / 4) * KV_HALF + (k % 4) * 32) >> 4), idesc_qk, k > 0 ? 1u : 0u);
      commit_if(lead, smem_u32(&s_full[w][t & 1]));
    };
    auto issue_pv = [&](int s, int j) {                             // O_w += P_w V(j), P from the columns of S_w[j % 2]
      const uint32_t p_tmem = tm + (2 * w + (j & 1)) * BN;
      const uint64_t dvs = dv + (uint64_t)(s * (KV_BYTES >> 4));
#pragma unroll
      for (int k = 0; k < BN / 16; ++k)
        mma_ts_if(lead, o_tmem, p_tmem + k * 8, dvs + (uint64_t)((k * 16 * 128) >> 4), idesc_pv, (j > 0 || k > 0) ? 1u : 0u);
    };
    bool ok = true;
    auto fail = [&](int code) {
      if (lead) { s_abort = 1; atomicExch(p.status, code); }
      ok = false;
    };
    // (the lanes wait each for itself and go on together: what one saw, all saw)
    if (on && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&q_full), 0))) fail(62);
    auto take_k = [&](int t) {                                      // S of key tile t, or the stage handed back once it is full
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&k_full[t % STAGES]), (t / STAGES) & 1))) { fail(63); return; }
      if (on) {
        tc_fence_after();
        issue_qk(t);
        commit_if(lead, smem_u32(&k_empty[t % STAGES]));
      } else if (lead) {
        mbar_arrive(smem_u32(&k_empty[t % STAGES]));
      }
    };
    for (int t = 0; t < 2 && t < n_tiles && ok; ++t) take_k(t);
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int s = j % STAGES;
      if (on && !__all_sync(0xffffffffu, mbar_spin(smem_u32(&p_full[w][j & 1]), (j >> 1) & 1))) { fail(64); break; }
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&v_full[s]), (j / STAGES) & 1))) { fail(63); break; }
      if (on) {
        tc_fence_after();
        issue_pv(s, j);
        commit_if(lead, smem_u32(&pv_done[w]));                     // O_w is quiet until the next P V
        if (j + 1 == n_tiles) commit_if(lead, smem_u32(&o_full[w]));   // this row tile's last P V
        commit_if(lead, smem_u32(&v_empty[s]));
      } else if (lead) {
        mbar_arrive(smem_u32(&v_empty[s]));
      }
      if (j + 2 < n_tiles) take_k(j + 2);                           // into the buffer of S that tile j just left
    }
  } else {                                                          // ---- softmax and output: one thread per row
    const int w = (warp - 2) >> 2;                                  // row tile A (warps 2..5) or B (warps 6..9)
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int token = r / p.group;                                  // of the row tile
    const bool row_ok = token < p.tile_tokens && w * p.tile_tokens + token < pair.z;
    const int t = pair.y + w * p.tile_tokens + token;
    const int pos = row_ok ? p.positions[t] : -1;
    const int n_w = w == 0 || b_on ? n_tiles : 0;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + 2 * w * BN, o_addr = lane_addr + O_COL + w * 128;
    float m_run = -INFINITY, l_run = 0.f;                           // reference maximum (scaled, log2 units), running sum
    bool ok = true;
    const int my_word = w * p.words + (row_ok ? token >> 5 : 0), my_bit = token & 31;
    constexpr int UNIT = BN / NP;
    // the keys of each entry of a tile that this row sees, by its bit and by what is not behind it; made for the next tile
    // when a tile's weights have been handed over
    int seen[NP];
    auto look = [&](int j) {
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        const int e = j * NP + x;
        const unsigned word = e < held ? s_bits[e * bits + my_word] : masks[(int64_t)e * bits + my_word];
        const int first = e < held ? s_first[e] : entries[e].y;
        seen[x] = row_ok && (word >> my_bit & 1) ? max(0, min(UNIT, pos - first + 1)) : 0;
      }
    };
    // the weights are in tensor memory before a warp's lane says so
    auto hand_over = [&](int j) {
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&p_full[w][j & 1]));
    };
    if (n_w > 0) look(0);
    for (int j = 0; j < n_w; ++j) {
      if (!mbar_wait(smem_u32(&s_full[w][j & 1]), (j >> 1) & 1)) { s_abort = 1; atomicExch(p.status, 65); ok = false; break; }
      tc_fence_after();
      bool some = false, part = false;
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        some |= seen[x] > 0;
        part |= seen[x] > 0 && seen[x] < UNIT;
      }
      if (!__any_sync(0xffffffffu, some)) {                         // nothing here for the warp's rows: weights of zero
        uint32_t zero[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) zero[i] = 0;
        tmem_st16(s_addr + (j & 1) * BN, zero);
        tmem_st16(s_addr + (j & 1) * BN + 16, zero);
        hand_over(j);
        if (j + 1 < n_w) look(j + 1);
        continue;
      }
      float s0[64];
      tmem_ld32(s_addr + (j & 1) * BN, *reinterpret_cast<float(*)[32]>(s0));
      tmem_ld32(s_addr + (j & 1) * BN + 32, *reinterpret_cast<float(*)[32]>(s0 + 32));
      tmem_ld_wait();
      if (__any_sync(0xffffffffu, part)) {                          // (the token's own page)
#pragma unroll
        for (int i = 0; i < BN; ++i)
          if (i % UNIT >= seen[i / UNIT]) s0[i] = -INFINITY;
      }
      // maximum of the raw scores of the entries that the row sees (the scale is positive), as short chains
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        constexpr int CH = UNIT < 32 ? 4 : 8;
        float mq[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) mq[i] = s0[x * UNIT + i];
#pragma unroll
        for (int i = CH; i < UNIT; ++i) mq[i % CH] = fmaxf(mq[i % CH], s0[x * UNIT + i]);
#pragma unroll
        for (int i = CH / 2; i > 0; i >>= 1)
#pragma unroll
          for (int k = 0; k < i; ++k) mq[k] = fmaxf(mq[k], mq[k + i]);
        if (seen[x] > 0) mx = fmaxf(mx, mq[0]);
      }
      mx *= p.scale_log2;
      // raise the reference maximum only when it grows by more than 8 (in log2 units)
      const bool raise = mx > m_run + 8.f;
      if (j > 0 && __any_sync(0xffffffffu, raise)) {
        // O_w must be quiet: P V of tile j-1 complete (P V of tile j waits for our P, and S of tile j came behind P V of tile j-2)
        if (!mbar_wait(smem_u32(&pv_done[w]), (j - 1) & 1)) { s_abort = 1; atomicExch(p.status, 65); ok = false; break; }
        tc_fence_after();
        const float alpha = raise ? fast_exp2(m_run - mx) : 1.f;     // m_run = -inf gives 0
        l_run *= alpha;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= alpha;
          tmem_st32(o_addr + c * 32, o);
        }
        tmem_st_wait();
      }
      if (raise) m_run = mx;
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      // 2^(s * scale - m); of an entry that the row does not see 2^-inf = 0 (a score there that is not a finite number makes the row's
      // sums one that is not, and the block's rows are made again)
      uint32_t pw[BN / 2];                                          // P: 64 keys = 32 columns
      uint64_t sq[4] = {};                                          // eight partial sums: short dependency chains
      const uint64_t scale2 = pair_f32(p.scale_log2, p.scale_log2);
#pragma unroll
      for (int x = 0; x < NP; ++x) {
        const float neg = seen[x] > 0 ? neg_m : -INFINITY;
        const uint64_t neg2 = pair_f32(neg, neg);
#pragma unroll
        for (int i = x * UNIT; i < (x + 1) * UNIT; i += 2) {
          uint64_t e;
          asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e) : "l"(pair_f32(s0[i], s0[i + 1])), "l"(scale2), "l"(neg2));
          const float lo = fast_exp2(__uint_as_float((unsigned)e)), hi = fast_exp2(__uint_as_float((unsigned)(e >> 32)));
          asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sq[i / 2 & 3]) : "l"(pair_f32(lo, hi)));
          pw[i / 2] = pack_bf16(lo, hi);                            // (half a step, 2^-8 of each; their sum is of the weights before)
        }
      }
      asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sq[0]) : "l"(sq[1]));
      asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sq[2]) : "l"(sq[3]));
      asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sq[0]) : "l"(sq[2]));
      l_run += __uint_as_float((unsigned)sq[0]) + __uint_as_float((unsigned)(sq[0] >> 32));
      tmem_st32(s_addr + (j & 1) * BN, reinterpret_cast<const float(&)[32]>(pw));
      hand_over(j);
      if (j + 1 < n_w) look(j + 1);
    }
    if (ok) {                                                       // (without a tile Q's rows, which the output goes through, have to be there)
      if (!mbar_wait(smem_u32(n_w > 0 ? &o_full[w] : &q_full), 0)) { s_abort = 1; atomicExch(p.status, 66); ok = false; }
      tc_fence_after();
    }
    const bool rows_on = w == 0 || b_on;
    bool odd = false, none = false;                                 // to be made again; weights that add up to zero
    __nv_bfloat16* dst = row_ok ? p.out + (int64_t)t * p.ldo + (int64_t)(hk * p.group + r % p.group) * D : nullptr;
    // a warp's rows go through the shared memory of Q, which is free now, so that neighbouring lanes store neighbouring pieces
    unsigned char* stage = smem_dyn + (sQ - smem_u32(smem_dyn)) + w * Q_BYTES + quarter * 32 * D * 2;
    constexpr int ROW16 = D / 8;                                    // 16-byte pieces of a row; piece c of row i lies at c ^ (i & 7)
    auto keep = [&](float (&o)[32], int c, float l, float inv) {
      if (l == 0.f)                                                 // a row that sees nothing
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) odd |= row_ok && !isfinite(o[i]);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        uint4 v;
        v.x = pack_bf16(o[q4 * 8] * inv, o[q4 * 8 + 1] * inv); v.y = pack_bf16(o[q4 * 8 + 2] * inv, o[q4 * 8 + 3] * inv);
        v.z = pack_bf16(o[q4 * 8 + 4] * inv, o[q4 * 8 + 5] * inv); v.w = pack_bf16(o[q4 * 8 + 6] * inv, o[q4 * 8 + 7] * inv);
        *reinterpret_cast<uint4*>(stage + lane * D * 2 + (((c * 4 + q4) ^ (lane & 7)) << 4)) = v;
      }
    };
    auto write = [&]() {
      __syncwarp();
#pragma unroll 4
      for (int i0 = 0; i0 < 32; i0 += 32 / ROW16) {
        const int i = i0 + lane / ROW16, c = lane % ROW16;
        __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), i));
        if (to) reinterpret_cast<uint4*>(to)[c] = *reinterpret_cast<const uint4*>(stage + i * D * 2 + ((c ^ (i & 7)) << 4));
      }
    };
    if (p.ksplit == 1) {
      if (ok && rows_on) {
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        odd = row_ok && !(l_run == l_run);
        none = row_ok && l_run == 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (n_w > 0) {
            tmem_ld32(o_addr + c * 32, o);
            tmem_ld_wait();
          }
          keep(o, c, l_run, inv);
        }
        write();
      }
    } else {
      // The rows are dealt out in runs of 32 (one warp's): block `dest` writes the run out, the others send it their unnormalised O, their
      // reference maximum and their sum, into the stages, which are free once every block's products are complete (the first
      // barrier).  What a block receives: [sender][4-column group][row of the block's runs] float4.
      constexpr int C4 = D / 4;
      const int run = w * 4 + quarter, runs_per = 8 / p.ksplit, dest = run / runs_per, rows_r = runs_per * 32;
      const int rloc = (run % runs_per) * 32 + lane;
      const bool mine = ok && n_w > 0;                              // O_w of this block holds something
      cluster_sync_all();
      if (dest != rank) {
        const int slot = rank < dest ? rank : rank - 1;
        if (mine) {
          const uint32_t remote = map_to_rank(sK, (uint32_t)dest) + (uint32_t)((slot * C4 * rows_r + rloc) * 16);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(o_addr + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int q4 = 0; q4 < 8; ++q4)
              st_cluster_f32x4(remote + (uint32_t)((c * 8 + q4) * rows_r * 16), o[q4 * 4], o[q4 * 4 + 1], o[q4 * 4 + 2], o[q4 * 4 + 3]);
          }
        }
        st_cluster_f32(map_to_rank(smem_u32(&x_max[slot * rows_r + rloc]), (uint32_t)dest), mine ? m_run : -INFINITY);
        st_cluster_f32(map_to_rank(smem_u32(&x_sum[slot * rows_r + rloc]), (uint32_t)dest), mine ? l_run : 0.f);
      }
      cluster_sync_all();
      if (dest == rank && rows_on && ok) {
        float m_all = mine ? m_run : -INFINITY;
        for (int sl = 0; sl < p.ksplit - 1; ++sl) m_all = fmaxf(m_all, x_max[sl * rows_r + rloc]);
        const float base_m = m_all == -INFINITY ? 0.f : m_all;
        const float a_own = mine && l_run != 0.f ? fast_exp2(m_run - base_m) : 0.f;
        float l_all = mine ? l_run * a_own : 0.f;
        for (int sl = 0; sl < p.ksplit - 1; ++sl) {
          const float l_p = x_sum[sl * rows_r + rloc];
          if (l_p != 0.f) l_all += l_p * fast_exp2(x_max[sl * rows_r + rloc] - base_m);
        }
        const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
        odd = row_ok && !(l_all == l_all);
        none = row_ok && l_all == 0.f;
        const float4* recv = reinterpret_cast<const float4*>(smem_dyn + (sK - smem_u32(smem_dyn)));
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (mine) {                                               // the whole warp or none of it: tcgen05.ld is a warp's instruction
            tmem_ld32(o_addr + c * 32, o);
            tmem_ld_wait();
          }
          // (a block none of whose keys a row sees holds sums of zeros for it, or what is not a finite number; its part counts only
          // where that shows)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (mine) odd |= row_ok && !isfinite(o[i]);
            o[i] = a_own != 0.f ? o[i] * a_own : 0.f;
          }
          for (int sl = 0; sl < p.ksplit - 1; ++sl) {
            const float l_p = x_sum[sl * rows_r + rloc];
            if (l_p != 0.f) {
              const float a_p = fast_exp2(x_max[sl * rows_r + rloc] - base_m);
#pragma unroll
              for (int q4 = 0; q4 < 8; ++q4) {
                const float4 v = recv[(sl * C4 + c * 8 + q4) * rows_r + rloc];
                o[q4 * 4] = fmaf(a_p, v.x, o[q4 * 4]); o[q4 * 4 + 1] = fmaf(a_p, v.y, o[q4 * 4 + 1]);
                o[q4 * 4 + 2] = fmaf(a_p, v.z, o[q4 * 4 + 2]); o[q4 * 4 + 3] = fmaf(a_p, v.w, o[q4 * 4 + 3]);
              }
            }
          }
          keep(o, c, l_all, inv);
        }
        write();
      }
    }
    // (a row that sees keys, whose scores are all -inf: made again, it is not a number)
    if (none) odd |= sees_a_key(p, pair.x, t, hk);
    if (odd) s_odd = 1;
  }
  if (p.ksplit > 1 && (warp < 2 || warp >= MMA_WARP_B)) {           // the other warps pass the cluster's two barriers too
    cluster_sync_all();
    cluster_sync_all();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (s_abort) {                                                  // copies and products in flight come to their end first
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
  if (s_odd) rows_again<D>(p, pair.x, pair.y, pair.z, hk, rank * (2 * BM / p.ksplit), (rank + 1) * (2 * BM / p.ksplit));
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<EncodeTiledFn>(ok ? f : nullptr);
  }();
  return fn;
}

// Clusters of so many blocks that the device runs at a time (an SM holds one block, a cluster's SMs are neighbours), asked once a device.
template <int D, int NP>
int max_clusters(int ksplit) {
  static thread_local int asked_for = -1, found[4];
  int dev = 0;
  cudaGetDevice(&dev);
  if (asked_for != dev) {
    for (int i = 1; i < 4; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(64 << i); cfg.blockDim = dim3(NTHREADS); cfg.dynamicSmemBytes = smem_bytes<D>();
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1 << i; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr; cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&found[i], attention_pages_umma_kernel<D, NP>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        found[i] = 0;                                      // none: lists are not shared
      }
    }
    asked_for = dev;
  }
  return found[ksplit == 2 ? 1 : ksplit == 4 ? 2 : 3];
}

template <int D, int NP>
int launch(const CUtensorMap& mq, const CUtensorMap& mkv, Params& p, cudaStream_t stream) {
  static_assert((size_t)2 * STAGES * BN * D * 2 >= (size_t)7 * 32 * D * 4, "the stages hold what seven senders bring");
  auto k = attention_pages_umma_kernel<D, NP>;
  constexpr size_t sm = smem_bytes<D>();
  static thread_local int set_for = -1;                    // the attribute belongs to the device
  int dev = 0;
  cudaGetDevice(&dev);
  if (set_for != dev) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm) != cudaSuccess)
      return cuda_status("attention_pages_umma: shared memory");
    set_for = dev;
  }
  // blocks that share a list: as far as all clusters run at the same time, each with four key tiles of the longest list there may be
  p.ksplit = 1;
  for (int ks = 2; ks <= 8 && p.cap / p.per_tile >= ks * 4 && (int64_t)p.pairs * p.Hkv <= max_clusters<D, NP>(ks); ks *= 2) p.ksplit = ks;
  launch_pdl(page_lists_kernel, dim3(p.Hkv, p.pairs), dim3(LIST_NT), 0, stream, p);
  launch_pdl_cluster(k, dim3(p.Hkv * p.ksplit, p.pairs), dim3(NTHREADS), dim3(p.ksplit), sm, stream, mq, mkv, p);
  return cuda_status("attention_pages_umma");
}

int64_t room(Params& p, unsigned char* at) {
  p.tile_tokens = BM / p.group;
  p.words = (p.tile_tokens + 31) / 32;
  p.unit = p.page_size < BN ? p.page_size : BN;
  p.per_tile = BN / p.unit;
  // pairs of every way the tokens may be dealt out: a request's last one may be all but empty
  const int64_t tile = 2 * p.tile_tokens, pairs = (p.T + (tile - 1) * (p.B < p.T ? p.B : p.T)) / tile;
  p.pairs = (int)(pairs > INT32_MAX ? INT32_MAX : pairs);
  const int64_t most = (int64_t)2 * p.tile_tokens * p.top, pages = most < p.width ? most : p.width;
  p.cap = (int)((pages * (p.page_size / p.unit) + p.per_tile - 1) / p.per_tile * p.per_tile);
  unsigned char* start = at;
  auto take = [&](int64_t bytes) { unsigned char* x = at; at += (bytes + 255) / 256 * 256; return x; };
  const int64_t lists = pairs * p.Hkv;
  p.counts = (int*)take(lists * 4);
  p.entries = (int2*)take(lists * p.cap * 8);
  p.masks = (unsigned*)take(lists * p.cap * 2 * p.words * 4);
  return at - start;
}

constexpr int64_t MAX_ROOM = 1ll << 30;

}  // namespace

DINFER_DEFINE_LAST_ERROR()

static int64_t workspace_of(int num_reqs, int width, int top, int T, int H, int Hkv, int D, int page_size, Params& p) {
  if (T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || H / Hkv > BM || top <= 0 || width <= 0 || num_reqs <= 0 || (D != 64 && D != 128)) return 0;
  if (page_size < 16 || page_size > 128 || (page_size & (page_size - 1)) || (int64_t)width * page_size > INT32_MAX) return 0;
  if ((int64_t)2 * (BM / (H / Hkv)) * top > INT32_MAX) return 0;        // (a block's tokens' entries, which the lists are made from)
  p.width = width; p.B = num_reqs; p.top = top; p.T = T; p.H = H; p.Hkv = Hkv; p.group = H / Hkv; p.page_size = page_size;
  const int64_t bytes = room(p, nullptr);
  return p.pairs > 65535 || bytes > MAX_ROOM ? 0 : bytes;
}

// Bytes of workspace that the call wants; 0 where it does not take the sizes, or (sms > 0, the device's multiprocessors) where token by
// token is the shorter way.  Both are estimated, in microseconds.  Token by token every page is read for each token that chose it, at what L2 gives:
//     7 + T Hkv top page_size D 4 / 6.3e6
// or, where the tensor-core kernel for tokens does not take the call (groups above 16, more than 1024 chosen pages), for each head of each
// token, which the kernel for any sizes does at half that, and at 26 keys of a token and head in a microsecond:
//     7 + max(T H top page_size D 4 / 3e6, top page_size / 26)
// Here a block takes 1 a key tile of 64, 20 pass before and after, and n neighbouring tokens choose some top n^0.4 pages among them.
// The longest list (one request may bring all tokens but one each of the others) ends the step, or the lists of all do:
//     20 + max(tiles of the longest / ksplit, tiles of all / SMs)
// Measured at 32 heads of 128 over 8, 16 pages of 64 behind 8000 tokens (us, token by token and here): 32 tokens 26 and 26, 48 tokens 47
// and 31, 64 tokens 51 and 32, 256 tokens 173 and 38, 512 tokens 343 and 54, 64 tokens beside 16 single ones 70 and 77, 256 beside 16 190 and
// 78, 256 beside 64 224 and 102, 64 single ones 55 and 54; 32 heads of 64 over 4, 24 pages of 32: 32 tokens 12 and 23, 128 tokens 20 and 30.
// By the kernel for any sizes and here: 64 heads of 128 over 1, 16 pages of 64: 2 tokens 39 and 21, 24 tokens 231 and 25, 300 tokens 2698 and 44,
// 30 beside 30 single ones 548 and 31; 24 heads of 64 over 1, 8 pages of 16: 2 tokens 8 and 14, 24 tokens 14 and 17, 100 tokens 44 and
// 17; 8 heads of 128 over 2, 1100 pages of 16: 2 tokens 682 and 55, 24 tokens 925 and 90.
DINFER_API int64_t dinfer_attention_pages_umma_workspace(int num_reqs, int width, int top, int T, int H, int Hkv, int D, int page_size, int sms) {
  Params p{};
  const int64_t bytes = workspace_of(num_reqs, width, top, T, H, Hkv, D, page_size, p);
  if (bytes == 0 || sms <= 0) return bytes;
  const double tokens = T, keys = (double)(top < width ? top : width) * page_size, row = D * 4;
  const double by_token = 7.0 + (H / Hkv > 16 || top > 1024 ? fmax(tokens * H * keys * row / 3e6, keys / 26) : tokens * Hkv * keys * row / 6.3e6);
  auto tiles = [&](double n) { return fmin((double)width, top * pow(fmax(n, 1.0), 0.4)) * page_size / BN; };
  const double most = 2.0 * p.tile_tokens, longest = fmin(T - num_reqs + 1.0, most), mean = fmin((double)T / num_reqs, most);
  const double lists = fmax((double)T / most, (double)(num_reqs < T ? num_reqs : T)) * Hkv;
  int ks = 1;
  while (ks < 8 && lists * ks * 2 <= sms && tiles(longest) >= ks * 8) ks *= 2;
  return 20.0 + fmax(tiles(longest) / ks, lists * tiles(mean) / sms) < by_token ? bytes : 0;
}

// What the call takes, 8 bytes a field (a caller packs them and hands over one address).  As
// dinfer_attention_pages, for rows and bases on 16-byte boundaries and a positive scale.
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
  void* workspace;
  int64_t workspace_bytes;
  int* status;
  cudaStream_t stream;
};

DINFER_API int dinfer_attention_pages_umma(const AttentionPagesArgs* a) {
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
  void* workspace = a->workspace;
  const int64_t workspace_bytes = a->workspace_bytes;
  int* status = a->status;
  Params p{};
  const int64_t need = workspace_of(num_reqs, width, top, T, H, Hkv, D, page_size, p);
  if (need == 0) return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: sizes T=%d H=%d Hkv=%d D=%d page=%d top=%d width=%d", T, H, Hkv, D, page_size, top, width);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255) || !status)
    return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: a workspace of %lld bytes and a status word are required", (long long)need);
  if (!(scale > 0.f)) return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: the score scale must be positive, got %g", (double)scale);
  if ((ldq % 8) || (ldo % 8) || (((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache) & 15))
    return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: rows and bases must be 16-byte aligned");
  const int64_t cache_rows = (int64_t)num_pages * 2 * Hkv * page_size;
  if (num_pages <= 0 || cache_rows > INT32_MAX) return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: %d pages are too many rows for a tensor map's coordinate", num_pages);
  EncodeTiledFn fn = encode_fn();
  if (!fn) return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: cuTensorMapEncodeTiled is not available from this driver");
  p.q = (const __nv_bfloat16*)q; p.ldq = ldq; p.out = (__nv_bfloat16*)out; p.ldo = ldo; p.cache = (const __nv_bfloat16*)cache;
  p.num_pages = num_pages; p.table = table; p.width = width; p.cu = cu_seqlens; p.B = num_reqs; p.positions = positions;
  p.chosen = chosen; p.top = top; p.T = T; p.H = H; p.Hkv = Hkv; p.group = H / Hkv; p.page_size = page_size; p.scale = scale;
  p.scale_log2 = scale * 1.4426950408889634f; p.status = status;
  room(p, (unsigned char*)workspace);
  CUtensorMap mq, mkv;
  {
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)ldq * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)p.tile_tokens};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: tensor map of q failed with %d", (int)r);
  }
  {
    cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)cache_rows};
    cuuint64_t strides[1] = {(cuuint64_t)D * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)p.unit};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(&mkv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return refuse(DINFER_BAD_ARGUMENT, "attention_pages_umma: tensor map of the cache failed with %d", (int)r);
  }
  switch (p.per_tile) {
    case 1: return D == 64 ? launch<64, 1>(mq, mkv, p, stream) : launch<128, 1>(mq, mkv, p, stream);
    case 2: return D == 64 ? launch<64, 2>(mq, mkv, p, stream) : launch<128, 2>(mq, mkv, p, stream);
    default: return D == 64 ? launch<64, 4>(mq, mkv, p, stream) : launch<128, 4>(mq, mkv, p, stream);
  }
}

// Which request a token of the step belongs to, from the offsets of the requests' tokens (cu_seqlens [requests + 1]).
#pragma once
#include "common.cuh"

namespace dinfer {

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

// The token tile `y` of a batch whose requests are cut into runs of up to `tile` tokens: its request, first token and tokens (every
// lane of a full warp asks); request -1 beyond the last tile.
__device__ __forceinline__ int3 token_tile(const int* cu, int num_reqs, int tile, int y) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int i0 = 0; i0 < num_reqs; i0 += 32) {
    const int i = i0 + lane;
    const int begin = i < num_reqs ? cu[i] : 0, tokens = i < num_reqs ? cu[i + 1] - begin : 0;
    const int n = (tokens + tile - 1) / tile;
    int incl = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, y >= before + incl - n && y < before + incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int at = y - before - __shfl_sync(0xffffffffu, incl - n, src);
      const int b = __shfl_sync(0xffffffffu, begin, src), k = __shfl_sync(0xffffffffu, tokens, src);
      return make_int3(i0 + src, b + at * tile, min(tile, k - at * tile));
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return make_int3(-1, 0, 0);
}

}  // namespace dinfer

// Device route plan of many routes over several workgroups: the same stable
// counting sort and the same tile descriptors as k_route_plan (plan_dev.h), whose
// single workgroup ranks 64 routes in about 0.8 us whatever the rest of the chip
// does. Three launches: every block of 4096 routes counts its buckets; one block
// scans the counts over blocks and buckets and writes the descriptors; every
// block ranks its routes from its buckets' first positions on. 65536 routes of 32
// experts: 13 us (4.7 + 5.1 + 5.3 in a trace: the launches' own times), 54 us in
// one workgroup; 32768 of 64: 13 against 25.
#include "plan_dev.h"

namespace keep {

constexpr int PB_ROUTES = 4096;                    // of a block
constexpr int PB_WAVE = PB_ROUTES / PLAN_WAVES;    // of a wave: 256
constexpr int PB_PER = PB_WAVE / 64;

struct PlanBlocksArgs {
  const int32_t* rhs;
  int R, E, tile, blocks, max_tiles;
  int32_t *order, *inverse, *counts, *offsets, *te, *to, *tc, *n_tiles;
  int32_t* hist;  // [blocks][E + 1], then each bucket's first position [E + 1]
};

__device__ __forceinline__ int pb_bucket(const PlanBlocksArgs& a, int r) {
  const int e = a.rhs[r];
  return e < 0 || e >= a.E ? a.E : e;
}

__global__ __launch_bounds__(PLAN_THREADS) void k_plan_count(PlanBlocksArgs a) {
  __shared__ int cnt[PLAN_MAX_E + 1];
  const int EB = a.E + 1;
  for (int e = threadIdx.x; e < EB; e += PLAN_THREADS) cnt[e] = 0;
  __syncthreads();
  const int r0 = blockIdx.x * PB_ROUTES;
#pragma unroll
  for (int i = 0; i < PB_ROUTES / PLAN_THREADS; ++i) {
    const int r = r0 + i * PLAN_THREADS + (int)threadIdx.x;
    if (r < a.R) atomicAdd(&cnt[pb_bucket(a, r)], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < EB; e += PLAN_THREADS) a.hist[blockIdx.x * EB + e] = cnt[e];
}

__global__ __launch_bounds__(PLAN_THREADS) void k_plan_scan(PlanBlocksArgs a) {
  __shared__ int cnt[PLAN_MAX_E + 1], run[PLAN_MAX_E + 1], tbase[PLAN_MAX_E + 1], wtot[2][PLAN_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, E = a.E, EB = E + 1, tile = a.tile;
  // every block's first position within the bucket
  for (int e = tid; e < EB; e += PLAN_THREADS) {
    int acc = 0;
    for (int b = 0; b < a.blocks; b += 8) {
      int c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = b + i < a.blocks ? a.hist[(b + i) * EB + e] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (b + i < a.blocks) a.hist[(b + i) * EB + e] = acc;
        acc += c[i];
      }
    }
    cnt[e] = acc;
  }
  __syncthreads();
  // the buckets' first positions and first tiles: two neighbouring buckets a thread, scanned over the lanes and the waves
  const int b0 = 2 * tid, b1 = b0 + 1;
  const int c0 = b0 < EB ? cnt[b0] : 0, c1 = b1 < EB ? cnt[b1] : 0;
  const int t0 = b0 < E ? (c0 + tile - 1) / tile : 0, t1 = b1 < E ? (c1 + tile - 1) / tile : 0;
  int vc = c0 + c1, vt = t0 + t1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int oc = __shfl_up(vc, d, 64), ot = __shfl_up(vt, d, 64);
    if (lane >= d) {
      vc += oc;
      vt += ot;
    }
  }
  if (lane == 63) {
    wtot[0][wv] = vc;
    wtot[1][wv] = vt;
  }
  __syncthreads();
  int ec = vc - (c0 + c1), et = vt - (t0 + t1);
  for (int w = 0; w < wv; ++w) {
    ec += wtot[0][w];
    et += wtot[1][w];
  }
  if (b0 < EB) {
    run[b0] = ec;
    tbase[b0] = et;
  }
  if (b1 < EB) {
    run[b1] = ec + c0;
    tbase[b1] = et + t0;
  }
  if (b0 == E) a.n_tiles[0] = et;
  if (b1 == E) a.n_tiles[0] = et + t0;
  __syncthreads();
  for (int e = tid; e < EB; e += PLAN_THREADS) a.hist[a.blocks * EB + e] = run[e];
  for (int e = tid; e < E; e += PLAN_THREADS) {
    a.counts[e] = cnt[e];
    a.offsets[e] = run[e];
  }
  // a wave per expert in turn, a lane per tile; the invalid routes' tiles (expert -1) and empty ones follow
  for (int e = wv; e < E; e += PLAN_WAVES) {
    const int nt = (cnt[e] + tile - 1) / tile;
    for (int i = lane; i < nt; i += 64) {
      const int ti = tbase[e] + i;
      if (ti < a.max_tiles) {
        a.te[ti] = e;
        a.to[ti] = run[e] + i * tile;
        a.tc[ti] = min(tile, cnt[e] - i * tile);
      }
    }
  }
  const int nbad = (cnt[E] + tile - 1) / tile;
  for (int ti = tbase[E] + tid; ti < a.max_tiles; ti += PLAN_THREADS) {
    const int i = ti - tbase[E];
    const bool b = i < nbad;
    a.te[ti] = b ? -1 : 0;
    a.to[ti] = b ? run[E] + i * tile : 0;
    a.tc[ti] = b ? min(tile, cnt[E] - i * tile) : 0;
  }
}

__global__ __launch_bounds__(PLAN_THREADS) void k_plan_scatter(PlanBlocksArgs a) {
  __shared__ int wh[PLAN_WAVES][PLAN_MAX_E + 1];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, EB = a.E + 1;
  for (int i = tid; i < PLAN_WAVES * EB; i += PLAN_THREADS) wh[i / EB][i % EB] = 0;
  const int r0 = blockIdx.x * PB_ROUTES + wv * PB_WAVE;
  int ev[PB_PER];
#pragma unroll
  for (int i = 0; i < PB_PER; ++i) {
    const int r = r0 + i * 64 + lane;
    ev[i] = r < a.R ? pb_bucket(a, r) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PB_PER; ++i)
    if (ev[i] >= 0) atomicAdd(&wh[wv][ev[i]], 1);
  __syncthreads();
  // each wave's first position in every bucket
  for (int e = tid; e < EB; e += PLAN_THREADS) {
    int acc = a.hist[a.blocks * EB + e] + a.hist[blockIdx.x * EB + e];
    for (int w = 0; w < PLAN_WAVES; ++w) {
      const int c = wh[w][e];
      wh[w][e] = acc;
      acc += c;
    }
  }
  __syncthreads();
  // a route's rank among the lanes below it with its bucket; the last of those lanes moves the wave's position on (one
  // wave's LDS operations run in order)
  const int nbits = 32 - __builtin_clz((unsigned)a.E);
#pragma unroll
  for (int i = 0; i < PB_PER; ++i) {
    const int e = ev[i], r = r0 + i * 64 + lane;
    uint64_t peers = __ballot(e >= 0);
    for (int b = 0; b < nbits; ++b) {
      const bool bit = (e >> b) & 1;
      const uint64_t m = __ballot(bit);
      peers &= bit ? m : ~m;
    }
    if (e >= 0) {
      const int pos = wh[wv][e] + __popcll(peers & ((1ull << lane) - 1ull));
      if (lane == 63 || (peers >> (lane + 1)) == 0ull) wh[wv][e] = pos + 1;
      a.order[pos] = r;
      a.inverse[r] = pos;
    }
  }
}

}  // namespace keep

using namespace keep;

extern "C" int64_t keep_route_plan_blocks_workspace_bytes(int64_t R, int64_t E) {
  if (!dims_ok({R, E}) || R < 1 || E < 1 || E > PLAN_MAX_E) return 0;
  return ((R + PB_ROUTES - 1) / PB_ROUTES + 1) * (E + 1) * 4;
}

extern "C" int keep_route_plan_blocks(const int32_t* rhs, int64_t R, int64_t E, int64_t tile, int32_t* order,
                                      int32_t* inverse, int32_t* counts, int32_t* offsets, int32_t* tile_expert,
                                      int32_t* tile_offset, int32_t* tile_count, int64_t max_tiles, int32_t* n_tiles_out,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  KEEP_REQUIRE_DIMS(R, E, tile, max_tiles);
  KEEP_REQUIRE(R >= 1 && R <= 0x7fffffffLL - PB_ROUTES, "bad route count");
  KEEP_REQUIRE(E >= 1 && E <= PLAN_MAX_E, "E must be in 1..%d", PLAN_MAX_E);
  KEEP_REQUIRE(tile >= 1 && tile <= 4096, "tile must be in 1..4096");
  KEEP_REQUIRE(max_tiles >= (R + tile - 1) / tile + E, "max_tiles must be >= ceil(R/tile) + E");
  KEEP_REQUIRE(rhs && order && inverse && counts && offsets && tile_expert && tile_offset && tile_count && n_tiles_out &&
                   workspace,
               "null pointer argument");
  const int64_t need = keep_route_plan_blocks_workspace_bytes(R, E);
  KEEP_REQUIRE(need <= 0x7fffffffLL, "too many routes");
  KEEP_REQUIRE(workspace_bytes >= need && aligned(workspace, 4), "workspace needs %lld bytes, has %lld", (long long)need,
               (long long)workspace_bytes);
  const PlanBlocksArgs a{rhs, (int)R, (int)E, (int)tile, (int)((R + PB_ROUTES - 1) / PB_ROUTES), (int)max_tiles, order,
                         inverse, counts, offsets, tile_expert, tile_offset, tile_count, n_tiles_out, (int32_t*)workspace};
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(k_plan_count, dim3(a.blocks), dim3(PLAN_THREADS), 0, s, a);
  hipLaunchKernelGGL(k_plan_scan, dim3(1), dim3(PLAN_THREADS), 0, s, a);
  hipLaunchKernelGGL(k_plan_scatter, dim3(a.blocks), dim3(PLAN_THREADS), 0, s, a);
  return launch_status("keep_route_plan_blocks");
}

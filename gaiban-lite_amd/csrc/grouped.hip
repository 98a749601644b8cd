// Linears grouped by expert over bf16 or int8 weights [E, N, K]: slot i's activation row
// times its expert's weights, the slots sorted by expert in padded blocks (dsv4moe_align).
#include <algorithm>
#include <cmath>

#include "product_gemm.h"
#include "../../include/dsv4moe.h"

namespace dsv4 {

// Tiles of `tok` rows per expert with slots, estimated from the mean (the routes are on the
// device).
static double tiles_per_expert(const ProductParams& p, int tok) {
  const double used = p.slots < p.experts ? p.slots : p.experts;
  const double share = p.slots / used / tok;
  return share <= 0.85 ? 1.0 : share + 0.5;
}

// Weights that one tile reads, in whole lines, and more of them than the 256 MB cache in front
// of HBM would still hold when a call after the next reads them again.
static bool weights_once(const ProductParams& p, int tok) {
  const double used = p.slots < p.experts ? p.slots : p.experts;
  return tiles_per_expert(p, tok) == 1.0 && p.kbytes % 128 == 0 && used * p.n * p.kbytes > 96e6;
}

template <class Op, int TOK, int CH, int WM, int WN, bool SWIGLU>
static void launch_grouped_gemm(ProductParams p, hipStream_t stream) {
  p.tile_blocks = TOK / p.block_size;
  p.tiles_n = (p.n + CH - 1) / CH;
  const int64_t items = ((int64_t)p.blocks * p.tiles_n + kTileXcds - 1) / kTileXcds * kTileXcds;
  const dim3 grid((unsigned)(items < kGemmCus ? items : kGemmCus));
  if (weights_once(p, TOK))
    hipLaunchKernelGGL((product_gemm_kernel<Op, TOK, CH, WM, WN, true, SWIGLU, true>), grid, dim3(512), 0, stream, p);
  else
    hipLaunchKernelGGL((product_gemm_kernel<Op, TOK, CH, WM, WN, true, SWIGLU, false>), grid, dim3(512), 0, stream, p);
}

template <class Op, int TOK, int CH, int WM, int WN, int WK, int S, bool SWIGLU>
static void launch_grouped_tile(ProductParams p, hipStream_t stream) {
  p.tile_blocks = TOK / p.block_size;
  p.tiles_m = p.blocks;
  p.tiles_n = (p.n + CH - 1) / CH;
  const dim3 block(64 * WM * WN * WK);
  // a launch has fewer than 2^32 threads; workgroups that stay have no such limit
  if ((int64_t)p.blocks * p.tiles_n * block.x > 0xFFFFFFFFll)
    return launch_grouped_gemm<Op, 128, 256, 2, 4, SWIGLU>(p, stream);
  const dim3 grid((unsigned)(p.blocks * p.tiles_n));
  if (weights_once(p, TOK))
    hipLaunchKernelGGL((product_tile_kernel<Op, TOK, CH, WM, WN, WK, S, true, SWIGLU, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((product_tile_kernel<Op, TOK, CH, WM, WN, WK, S, true, SWIGLU, false>), grid, block, 0, stream, p);
}

// The kernel of a call.  Blocks of up to 32 slots: 64 x 128 tiles where there are two per CU (300
// tokens x 6 over 64 experts, N=1024, K=4096 114 us against 124 with 32 x 64; 60 x 2 over 8
// experts, N=K=4096, one per CU, 44.8 against 42.8), but 16 x 32 tiles with 512 bytes of K a
// stage for blocks of up to 16 (64 tokens x 6 over 256 experts, N=4096, K=2048 480 us, 7.0 TB/s,
// against 505 with 32 x 64 and 510 with 64 x 128), unless the rows are too short for them (K=1024
// 271 us against 237) or many experts have more than 16 slots and are read twice (500 x 6 over
// 256 experts, int8, N=K=4096 717 us against 646).
// Longer blocks: the least time by a model -- a start, then a CU's share of the tiles times (K
// blocks x time per block + end), or the experts' weights at 6.4 TB/s (the workgroups that stay:
// 5.9) where that is more, half of the second and later readings coming from the caches; the
// tiles per expert are estimated from the mean (the routes are on the device).  us, bf16, model /
// measured: 5000 tokens x 4 over 64 experts, N=K=1024: 128 x 256 62 / 58, 256 x 256 63 / 65, 128
// x 128 73 / 68, 64 x 128 77 / 80, 64 x 64 96 / 92; 200 x 2 over 8, N=2048, K=1024: 64 x 64 8.6 /
// 8.8, 64 x 128 11.3 / 10.7, 128 x 128 16 / 13; 700 x 4 over 64, N=1024, K=2048: 64 x 128 42 /
// 47, 128 x 256 46 / 65; 1500 x 6 over 64, N=2816, K=2048 256 x 256 170 / 184, 128 x 256 180 /
// 210, 128 x 128 186 / 238.
template <class Op, bool SWIGLU>
static void launch_grouped(const ProductParams& p, hipStream_t stream) {
  const double used = p.slots < p.experts ? p.slots : p.experts;
  auto tiles = [&](int tok, int ch) { return used * tiles_per_expert(p, tok) * ((p.n + ch - 1) / ch); };
  if (p.block_size <= 32) {
    if (tiles(64, 128) >= 2 * kGemmCus && (p.block_size > 16 || p.kbytes <= 2048 || p.slots > 10 * used))
      return launch_grouped_tile<Op, 64, 128, 2, 4, 1, 3, SWIGLU>(p, stream);
    if (p.block_size <= 16) return launch_grouped_tile<Op, 16, 32, 1, 1, 4, 2, SWIGLU>(p, stream);
    return launch_grouped_tile<Op, 32, 64, 1, 2, 2, 3, SWIGLU>(p, stream);
  }
  struct Tile {
    int tok, ch;
    double start, block, end, rate;
    void (*launch)(ProductParams, hipStream_t);
  };
  static const Tile kernels[] = {
      {128, 256, 5.0, 1.0, 3.0, 5.9e6, launch_grouped_gemm<Op, 128, 256, 2, 4, SWIGLU>},
      {256, 256, 5.0, 1.62, 3.0, 5.9e6, launch_grouped_gemm<Op, 256, 256, 4, 2, SWIGLU>},
      {128, 128, 5.0, 0.55, 2.5, 5.9e6, launch_grouped_gemm<Op, 128, 128, 4, 2, SWIGLU>},
      {64, 128, 4.0, 0.38, 1.2, 6.4e6, launch_grouped_tile<Op, 64, 128, 2, 4, 1, 3, SWIGLU>},
      {64, 64, 4.0, 0.25, 0.6, 6.4e6, launch_grouped_tile<Op, 64, 64, 4, 2, 1, 3, SWIGLU>},
  };
  const Tile* best = nullptr;
  double least = 0.0;
  for (const Tile& t : kernels) {
    const double rounds = std::ceil(tiles(t.tok, t.ch) / kGemmCus);
    const double read = used * p.n * p.kbytes / t.rate * (0.5 + 0.5 * tiles_per_expert(p, t.tok));
    const double time = std::max(read, t.start + rounds * (p.kblocks * t.block + t.end));
    if (best == nullptr || time < least) best = &t, least = time;
  }
  best->launch(p, stream);
}

}  // namespace dsv4

using namespace dsv4;

int dsv4_launch_grouped(const ProductParams& params, bool int8, bool swiglu, hipStream_t stream) {
  ProductParams p = params;
  if (int8 && swiglu) launch_grouped<ProductInt8, true>(p, stream);
  else if (int8) launch_grouped<ProductInt8, false>(p, stream);
  else if (swiglu) launch_grouped<ProductBf16, true>(p, stream);
  else launch_grouped<ProductBf16, false>(p, stream);
  DSV4_CHECK_LAUNCH("product_tile_kernel");
  return DSV4MOE_OK;
}

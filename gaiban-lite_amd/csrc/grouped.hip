// Linears grouped by expert over bf16 or int8 weights [E, N, K]: slot i's activation row
// times its expert's weights, the slots sorted by expert in padded blocks (dsv4moe_align).
#include "product_gemm.h"
#include "../../include/dsv4moe.h"

namespace dsv4 {

template <class Op, int TOK, int CH, int WM, int WN, int WK, int S, bool SWIGLU>
static void launch_grouped_tile(ProductParams p, hipStream_t stream) {
  p.tile_blocks = TOK / p.block_size;
  p.tiles_m = p.blocks;
  p.tiles_n = (p.n + CH - 1) / CH;
  const dim3 grid((unsigned)(p.blocks * p.tiles_n));
  hipLaunchKernelGGL((product_tile_kernel<Op, TOK, CH, WM, WN, WK, S, true, SWIGLU>), grid, dim3(64 * WM * WN * WK), 0, stream,
                     p);
}

template <class Op, int TOK, int CH, int WM, int WN, bool SWIGLU>
static void launch_grouped_gemm(ProductParams p, hipStream_t stream) {
  p.tile_blocks = TOK / p.block_size;
  p.tiles_n = (p.n + CH - 1) / CH;
  const int64_t items = ((int64_t)p.blocks * p.tiles_n + kTileXcds - 1) / kTileXcds * kTileXcds;
  const dim3 grid((unsigned)(items < kGemmCus ? items : kGemmCus));
  hipLaunchKernelGGL((product_gemm_kernel<Op, TOK, CH, WM, WN, true, SWIGLU>), grid, dim3(512), 0, stream, p);
}

template <class Op, bool SWIGLU>
static void launch_grouped(const ProductParams& p, hipStream_t stream) {
  const int per_expert = p.slots / p.experts;
  if (per_expert >= 64) return launch_grouped_gemm<Op, 256, 256, 4, 2, SWIGLU>(p, stream);
  if (p.block_size <= 16) launch_grouped_tile<Op, 16, 32, 1, 1, 4, 2, SWIGLU>(p, stream);
  else if (p.block_size <= 32) launch_grouped_tile<Op, 32, 128, 1, 4, 2, 3, SWIGLU>(p, stream);
  else launch_grouped_tile<Op, 64, 128, 2, 4, 1, 3, SWIGLU>(p, stream);
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

// W8A8 linear in 8-bit integers: out[M,N] = bf16( (Q[M,K] . Wq[N,K]^T) * s[m] * ws[n] ),
// activations quantised per token, weights int8 with one bf16 scale per output channel.
// The products are summed exactly in int32 (K <= 65536: below 2^31), so the tiles, their
// order and the K blocks do not show in the result.
#include "product_gemm.h"
#include "../../include/dsv4moe.h"

namespace dsv4 {

// ------------------------------------------------------------ quantiser
// Eight values of a row as fp32.
template <int X>
__device__ __forceinline__ void load8_as_float(const void* x, int64_t at, float (&f)[8]) {
  if constexpr (X == DSV4MOE_DTYPE_FP32) {
    const f32x4* src = reinterpret_cast<const f32x4*>(static_cast<const float*>(x) + at);
    const f32x4 a = src[0], b = src[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = a[e];
      f[4 + e] = b[e];
    }
  } else {
    const u32x4 v = load16(static_cast<const uint16_t*>(x) + at);
    if constexpr (X == DSV4MOE_DTYPE_BF16) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(v[e] << 16);
        f[2 * e + 1] = __uint_as_float(v[e] & 0xFFFF0000u);
      }
    } else {
      typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
      const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)h[e];
    }
  }
}

// The largest magnitude as bits: |v| orders like its bits, NaN above infinity above
// every finite value, so a row's NaN or infinity is not lost in the maximum.
__device__ __forceinline__ uint32_t max_magnitude(uint32_t amax, const float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(f[e]) & 0x7FFFFFFFu);
  return amax;
}
constexpr uint32_t kInfBits = 0x7F800000u;
// s = max(amax, 1e-12) / 127; NaN for a row with a NaN or an infinity, which makes
// its outputs NaN instead of hiding it
__device__ __forceinline__ float int8_row_scale(uint32_t amax) {
  if (amax >= kInfBits) return __uint_as_float(0x7FC00000u);
  return fmaxf(__uint_as_float(amax), 1e-12f) / 127.0f;
}
// eight codes rint(v / s) (IEEE quotient, half to even), or zeros where s is NaN
__device__ __forceinline__ u32x2 int8_codes(const float (&f)[8], float s) {
  u32x2 out = {0, 0};
  if (s == s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e >> 2] |= ((uint32_t)(int)__builtin_rintf(f[e] / s) & 0xFFu) << (8 * (e & 3));
  }
  return out;
}

// LANES lanes per row, HELD chunks of 8 values per lane held in registers (a longer row is
// read again for its codes).
template <int X, int LANES, int HELD>
__global__ __launch_bounds__(256) void act_quant_int8_kernel(const void* __restrict__ x, int64_t m, int k,
                                                             int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t part[4];
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (LANES == 64 && row >= m) return;  // LANES == 256: one row per workgroup
  const int lane = threadIdx.x % LANES;
  const int chunks = k / 8;
  const int64_t base = row * k;
  float f[HELD][8];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (lane + LANES * i < chunks) load8_as_float<X>(x, base + (int64_t)(lane + LANES * i) * 8, f[i]);
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (lane + LANES * i < chunks) amax = max_magnitude(amax, f[i]);
  for (int c = lane + LANES * HELD; c < chunks; c += LANES) {
    float g[8];
    load8_as_float<X>(x, base + (int64_t)c * 8, g);
    amax = max_magnitude(amax, g);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, off, 64));
  if constexpr (LANES == 256) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  const float s = int8_row_scale(amax);
  if (lane == 0) scale[row] = s;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (lane + LANES * i < chunks)
      *reinterpret_cast<u32x2*>(q + base + (int64_t)(lane + LANES * i) * 8) = int8_codes(f[i], s);
  for (int c = lane + LANES * HELD; c < chunks; c += LANES) {
    float g[8];
    load8_as_float<X>(x, base + (int64_t)c * 8, g);
    *reinterpret_cast<u32x2*>(q + base + (int64_t)c * 8) = int8_codes(g, s);
  }
}

template <int X>
static void launch_quant(const void* x, int64_t m, int k, int8_t* q, float* scale, hipStream_t stream) {
  if (m <= 1024)
    hipLaunchKernelGGL((act_quant_int8_kernel<X, 256, 4>), dim3((unsigned)m), dim3(256), 0, stream, x, m, k, q, scale);
  else
    hipLaunchKernelGGL((act_quant_int8_kernel<X, 64, 8>), dim3((unsigned)((m + 3) / 4)), dim3(256), 0, stream, x, m, k,
                       q, scale);
}

template <int TOK, int CH, int WM, int WN, int S>
static void launch_tile(ProductParams p, hipStream_t stream) {
  p.tiles_m = (int)((p.rows + TOK - 1) / TOK);
  p.tiles_n = (p.n + CH - 1) / CH;
  const int items = p.tiles_m * p.tiles_n;
  const dim3 grid((unsigned)((items + kTileXcds - 1) / kTileXcds * kTileXcds));
  hipLaunchKernelGGL((product_tile_kernel<ProductInt8, TOK, CH, WM, WN, S, false, false>), grid, dim3(64 * WM * WN), 0,
                     stream, p);
}

template <int TOK, int CH, int WM, int WN>
static void launch_gemm(ProductParams p, hipStream_t stream) {
  p.tiles_m = (int)((p.rows + TOK - 1) / TOK);
  p.tiles_n = (p.n + CH - 1) / CH;
  const int64_t items = ((int64_t)p.tiles_m * p.tiles_n + kTileXcds - 1) / kTileXcds * kTileXcds;
  const dim3 grid((unsigned)(items < kGemmCus ? items : kGemmCus));
  hipLaunchKernelGGL((product_gemm_kernel<ProductInt8, TOK, CH, WM, WN, false, false>), grid, dim3(512), 0, stream, p);
}

}  // namespace dsv4

using namespace dsv4;

int dsv4_launch_act_quant_int8(const void* x, int32_t x_dtype, int64_t m, int64_t k, int8_t* q, float* scale,
                               hipStream_t stream) {
  if (x_dtype == DSV4MOE_DTYPE_BF16) launch_quant<DSV4MOE_DTYPE_BF16>(x, m, (int)k, q, scale, stream);
  else if (x_dtype == DSV4MOE_DTYPE_FP16) launch_quant<DSV4MOE_DTYPE_FP16>(x, m, (int)k, q, scale, stream);
  else launch_quant<DSV4MOE_DTYPE_FP32>(x, m, (int)k, q, scale, stream);
  DSV4_CHECK_LAUNCH("act_quant_int8_kernel");
  return DSV4MOE_OK;
}

int dsv4_launch_int8_gemm(const int8_t* a, const float* a_scale, int64_t m, int64_t n, int64_t k, const int8_t* wq,
                          const uint16_t* ws, uint16_t* out, hipStream_t stream) {
  ProductParams p{};
  p.x = reinterpret_cast<const uint8_t*>(a);
  p.rows = m;
  p.w = reinterpret_cast<const uint8_t*>(wq);
  p.n = p.out_n = (int)n;
  p.kbytes = (int)k;
  p.kblocks = (int)((k + kBlockBytes - 1) / kBlockBytes);
  p.x_scale = a_scale;
  p.w_scale = ws;
  p.out = out;
  if (m <= 16) launch_tile<16, 64, 1, 4, 6>(p, stream);
  else if (m <= 64) launch_tile<64, 64, 2, 2, 4>(p, stream);
  else if ((m + 255) / 256 * ((n + 255) / 256) >= 192) launch_gemm<256, 256, 4, 2>(p, stream);
  else if ((m + 255) / 256 * ((n + 127) / 128) >= 192) launch_gemm<256, 128, 4, 2>(p, stream);
  else launch_tile<128, 128, 2, 2, 3>(p, stream);
  DSV4_CHECK_LAUNCH("product_tile_kernel");
  return DSV4MOE_OK;
}

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
// Eight codes rint(fl(v / s)), half to even, or zeros where s is NaN.  With inv = fl(1 / s)
// the product y = fl(v * inv) is off the quotient by at most 127 * (2^-24 + 2^-24 + 2^-48) <
// 1.6e-5, the IEEE quotient by 127 * 2^-24 < 0.8e-5, so where y lies more than 2^-15 =
// 3.05e-5 from a half they round to the same integer; the few other values take the
// division.  Adding 1.5 * 2^23 rounds y, half to even, and leaves the code in the low byte.
// Against the division for every value: 2000 rows of 4096 bf16 10.6 -> 9.1 us.
__device__ __forceinline__ u32x2 int8_codes(const float (&f)[8], float s, float inv) {
  constexpr float kMagic = 12582912.0f;
  u32x2 out = {0, 0};
  if (s != s) return out;
  uint32_t t[8];
  float off = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = f[e] * inv;
    const float r = y + kMagic;
    off = fmaxf(off, fabsf(y - (r - kMagic)));
    t[e] = __float_as_uint(r);
  }
  if (off > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (uint32_t)(int)__builtin_rintf(f[e] / s);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)  // the low bytes of four
    out[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[4 * h + 3], t[4 * h + 2], 0x0C0C0400u),
                                   __builtin_amdgcn_perm(t[4 * h + 1], t[4 * h], 0x0C0C0400u), 0x05040100u);
  return out;
}

// LANES lanes per row, HELD chunks of 8 values per lane held in registers (a longer row is
// read again for its codes).
template <int X, int LANES, int HELD>
__global__ __launch_bounds__(256) void act_quant_int8_kernel(const void* __restrict__ x, int64_t m, int k,
                                                             int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int kWavesPerRow = LANES / 64;
  __shared__ uint32_t part[4];
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const bool in = row < m;
  const int lane = threadIdx.x % LANES;
  const int chunks = in ? k / 8 : 0;
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
  if constexpr (kWavesPerRow > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWavesPerRow; ++w) amax = max(amax, part[wave / kWavesPerRow * kWavesPerRow + w]);
  }
  const float s = int8_row_scale(amax);
  const float inv = 1.0f / s;
  if (in && lane == 0) scale[row] = s;
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (lane + LANES * i < chunks)
      *reinterpret_cast<u32x2*>(q + base + (int64_t)(lane + LANES * i) * 8) = int8_codes(f[i], s, inv);
  for (int c = lane + LANES * HELD; c < chunks; c += LANES) {
    float g[8];
    load8_as_float<X>(x, base + (int64_t)c * 8, g);
    *reinterpret_cast<u32x2*>(q + base + (int64_t)c * 8) = int8_codes(g, s, inv);
  }
}

template <int X, int LANES, int HELD>
static void launch_quant_as(const void* x, int64_t m, int k, int8_t* q, float* scale, hipStream_t stream) {
  constexpr int kRows = 256 / LANES;
  constexpr int64_t kMost = (int64_t)kRows << 23;  // rows of a launch, which has fewer than 2^32 threads
  constexpr int kItem = X == DSV4MOE_DTYPE_FP32 ? 4 : 2;
  for (int64_t at = 0; at < m; at += kMost) {
    const int64_t rows = m - at < kMost ? m - at : kMost;
    hipLaunchKernelGGL((act_quant_int8_kernel<X, LANES, HELD>), dim3((unsigned)((rows + kRows - 1) / kRows)),
                       dim3(256), 0, stream, static_cast<const char*>(x) + at * k * kItem, rows, k, q + at * k,
                       scale + at);
  }
}

// A workgroup per row, or with many short rows a wavefront: M=32768 K=2048 38 against 46 us
// (5.3 TB/s), M=48 3.3 us against 5.9, M=2000 K=4096 8.4 against 10.2, M=8192 K=4096 22.1
// against 25.7 (4.6 TB/s).  Held rows: M=8192 K=16384 78 us (5.1 TB/s) against 87 read twice.
template <int X>
static void launch_quant(const void* x, int64_t m, int k, int8_t* q, float* scale, hipStream_t stream) {
  if (m > 1024 && k <= 2048) launch_quant_as<X, 64, 4>(x, m, k, q, scale, stream);
  else if (k <= 4096) launch_quant_as<X, 256, 2>(x, m, k, q, scale, stream);
  else if (k <= 8192) launch_quant_as<X, 256, 4>(x, m, k, q, scale, stream);
  else launch_quant_as<X, 256, 8>(x, m, k, q, scale, stream);
}

// ------------------------------------------------------------ few tokens
// Up to 16 tokens in one launch: every workgroup quantises all of them into LDS (while its
// first weights are under way) and then streams strips of 16 channels.  The K of a strip is
// dealt out in slices of 256 bytes to eight wavefronts; a wavefront copies its own slices, 16
// rows x 256 bytes at a time, into kFewStages stages of its own, so that nothing but the end
// of a strip needs a barrier: there the eight partial sums (exact, int32) are added.  A lane
// whose token does not exist reads another's codes, for a column that nothing stores.
// Weights from HBM, us, against the quantiser and a tile kernel: N=K=4096 M=1 8.0 / 13.8, M=8
// 10.8 / 14.3, N=16384 M=1 17.3 (3.9 TB/s) / 21.6, N=4096 K=2048 M=16 9.0 / 10.1.  Two copies
// of the weights in turn: N=16384 K=4096 15.1 -> 14.2 by strips that begin at parts of K of
// their own, N=131072 M=8 100 -> 91 (5.9 TB/s) by copies past the caches.
struct FewParams {
  const void* x;
  int m, n, k;
  const uint8_t* w;
  const uint16_t* ws;
  uint16_t* out;
};
constexpr int kFewWaves = 8;
constexpr int kFewSlice = 256;                      // K bytes of a wavefront per stage
constexpr int kFewRound = kFewWaves * kFewSlice;    // K bytes of a workgroup per stage
constexpr int kFewStages = 3;                       // (four measured the same)
constexpr int kFewCodes = 44 * 1024;                // all tokens' codes

static int64_t few_code_bytes(int64_t m, int64_t k) { return m * ((k + kFewRound - 1) / kFewRound * kFewRound); }

__device__ __forceinline__ void lds_wait_all() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#endif
}

template <int X, bool ONCE>
__global__ __launch_bounds__(512) void int8_few_kernel(FewParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t lds[kFewWaves * kFewStages * 16 * kFewSlice];
  __shared__ __attribute__((aligned(256))) uint8_t codes[kFewCodes];  // [m][rounds * kFewRound]
  __shared__ i32x4 sums[2][kFewWaves][64];
  __shared__ uint32_t amax_of[16][kFewWaves];
  __shared__ float scale_of[16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15;
  const int j = lane >> 4;
  const int strips = p.n >> 4;
  const int rounds = (p.k + kFewRound - 1) / kFewRound;
  const int code_row = rounds * kFewRound;

  // this wavefront's copies: 4 rows x 256 bytes each, part q of row r at q ^ r
  const uint32_t ring = __builtin_amdgcn_readfirstlane(lds_addr(lds + wave * kFewStages * 16 * kFewSlice));
  const int copy_row = lane >> 4;
  const __amdgpu_buffer_rsrc_t w_rsrc =
      __builtin_amdgcn_make_buffer_rsrc((void*)p.w, (short)0, (int)((int64_t)p.n * p.k), kTileRsrcFlags);
  const int mine = strips > (int)blockIdx.x ? (strips - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  const int steps = mine * rounds;  // over this workgroup's strips
  // the part of K of a step: a strip's first differs from its neighbours' (as first_block)
  auto round_of = [&](int step) { return (step + (blockIdx.x + step / rounds * gridDim.x) * 5) % rounds; };
  auto copy = [&](int step, int stage) {
    const int strip = blockIdx.x + step / rounds * gridDim.x;
    const int k0 = round_of(step) * kFewRound + wave * kFewSlice;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 4 + copy_row;
      const int at = k0 + lds_part<kFewSlice>(row, lane & 15) * 16;
      const uint32_t off = step < steps && at < p.k ? (uint32_t)((strip * 16 + row) * p.k + at) : kTileOob;
      copy_weights16<ONCE>(w_rsrc, ring + stage * 16 * kFewSlice + i * 1024, off, 0);
    }
  };
#pragma unroll
  for (int s = 0; s < kFewStages - 1; ++s) copy(s, s);

  // quantise: a row by 8, 4, 2 or 1 wavefronts, 8 values of a lane at a time
  const int per_row = p.m == 1 ? 8 : (p.m == 2 ? 4 : (p.m <= 4 ? 2 : 1));
  const int chunks = p.k / 8;
  const int c0 = wave % per_row * 64 + lane;
  for (int r = wave / per_row; r < p.m; r += kFewWaves / per_row) {
    uint32_t amax = 0;
#pragma unroll 4
    for (int c = c0; c < chunks; c += 64 * per_row) {
      float f[8];
      load8_as_float<X>(p.x, (int64_t)r * p.k + c * 8, f);
      amax = max_magnitude(amax, f);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, off, 64));
    if (lane == 0) amax_of[r][wave % per_row] = amax;
  }
  __syncthreads();
  for (int r = wave / per_row; r < p.m; r += kFewWaves / per_row) {
    uint32_t amax = 0;
    for (int w = 0; w < per_row; ++w) amax = max(amax, amax_of[r][w]);
    const float s = int8_row_scale(amax);
    const float inv = 1.0f / s;
    if (c0 == 0) scale_of[r] = s;
#pragma unroll 4
    for (int c = c0; c < code_row / 8; c += 64 * per_row) {
      u32x2 q = {0, 0};
      if (c < chunks) {
        float f[8];
        load8_as_float<X>(p.x, (int64_t)r * p.k + c * 8, f);
        q = int8_codes(f, s, inv);
      }
      // 16-byte parts of each 256 bytes in the order of the weights' rows
      const int at = (c >> 5) * kFewSlice + lds_part<kFewSlice>(r, c >> 1 & 15) * 16 + (c & 1) * 8;
      *reinterpret_cast<u32x2*>(codes + r * code_row + at) = q;
    }
  }
  __syncthreads();

  const int token = n16 % p.m;
  const uint8_t* my_codes = codes + token * code_row + wave * kFewSlice;
  i32x4 acc = {0, 0, 0, 0};
  int stage = 0, turn = 0;
  for (int step = 0; step < steps; ++step) {
    lds_dma_wait_keep<(kFewStages - 2) * 4>();
    const uint8_t* ws = lds + (wave * kFewStages + stage) * 16 * kFewSlice;
    const uint8_t* xs = my_codes + round_of(step) * kFewRound;
    u32x4 wf[4], xf[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      wf[d] = load16(ws + n16 * kFewSlice + lds_part<kFewSlice>(n16, 4 * d + j) * 16);
      xf[d] = load16(xs + lds_part<kFewSlice>(token, 4 * d + j) * 16);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) acc = ProductInt8::mfma(wf[d], xf[d], acc);
    // the fragments are in registers before their stage is filled again
    lds_wait_all();
    const int refill = stage == 0 ? kFewStages - 1 : stage - 1;
    copy(step + kFewStages - 1, refill);
    stage = stage + 1 == kFewStages ? 0 : stage + 1;
    if ((step + 1) % rounds != 0) continue;
    // the end of a strip (two sets of sums in turn: one barrier)
    sums[turn][wave][lane] = acc;
    acc = i32x4{0, 0, 0, 0};
    __syncthreads();
    if (wave == (step / rounds) % kFewWaves) {
      const int strip = blockIdx.x + step / rounds * gridDim.x;
      i32x4 total = sums[turn][0][lane];
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) total += sums[turn][w][lane];
      if (n16 < p.m) {
        const float xs16 = scale_of[n16];
        const u32x2 s = *reinterpret_cast<const u32x2*>(p.ws + strip * 16 + 4 * j);
        const float w4[4] = {__uint_as_float(s[0] << 16), __uint_as_float(s[0] & 0xFFFF0000u),
                             __uint_as_float(s[1] << 16), __uint_as_float(s[1] & 0xFFFF0000u)};
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)total[e] * xs16 * w4[e];
        *reinterpret_cast<u32x2*>(p.out + (int64_t)n16 * p.n + strip * 16 + 4 * j) =
            u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    }
    turn ^= 1;
  }
  lds_dma_wait_all();
}

template <int X>
static int launch_few(const FewParams& p, hipStream_t stream) {
  const int strips = p.n / 16;
  const dim3 grid((unsigned)(strips < kGemmCus ? strips : kGemmCus));
  // weights that the cache in front of HBM would not hold until the next call bypass it
  if (p.k % 128 == 0 && (int64_t)p.n * p.k > 96000000)
    hipLaunchKernelGGL((int8_few_kernel<X, true>), grid, dim3(512), 0, stream, p);
  else
    hipLaunchKernelGGL((int8_few_kernel<X, false>), grid, dim3(512), 0, stream, p);
  DSV4_CHECK_LAUNCH("int8_few_kernel");
  return DSV4MOE_OK;
}

template <int TOK, int CH, int WM, int WN, int WK, int S>
static void launch_tile(ProductParams p, hipStream_t stream) {
  p.tiles_m = (int)((p.rows + TOK - 1) / TOK);
  p.tiles_n = (p.n + CH - 1) / CH;
  const int items = p.tiles_m * p.tiles_n;
  const dim3 grid((unsigned)((items + kTileXcds - 1) / kTileXcds * kTileXcds));
  hipLaunchKernelGGL((product_tile_kernel<ProductInt8, TOK, CH, WM, WN, WK, S, false, false, false>), grid,
                     dim3(64 * WM * WN * WK), 0, stream, p);
}

template <int TOK, int CH, int WM, int WN>
static void launch_gemm(ProductParams p, hipStream_t stream) {
  p.tiles_m = (int)((p.rows + TOK - 1) / TOK);
  p.tiles_n = (p.n + CH - 1) / CH;
  const int64_t items = ((int64_t)p.tiles_m * p.tiles_n + kTileXcds - 1) / kTileXcds * kTileXcds;
  const dim3 grid((unsigned)(items < kGemmCus ? items : kGemmCus));
  hipLaunchKernelGGL((product_gemm_kernel<ProductInt8, TOK, CH, WM, WN, false, false, false>), grid, dim3(512), 0, stream, p);
}

// The tile with the least time by a model: a start, then its workgroups' share of tiles per
// CU times the K blocks, each block's time measured on a full card (us, 128 bytes of K):
// 32 x 64 0.175, 64 x 64 0.25, 128 x 128 0.47, 256 x 128 0.85, 256 x 256 1.62 (it takes 54
// against 59, 66, 128 and 179 us of a CU per 256 x 256 outputs and 32 blocks; the smaller
// ones are for grids that would leave CUs idle).  Measured with the quantiser, N=K=4096: M=64
// 13.0 / 16.5 / 19.2 / 27.7 / 43.3 us, M=300 22.8 / 19.5 / 20.6 / 29.5 / 44.9, M=2000
// 99.6 / 74.9 / 44.1 / 40.5 / 52.3.
static void launch_product(const ProductParams& p, hipStream_t stream) {
  struct Tile {
    int tok, ch;
    double start, block;
    void (*launch)(ProductParams, hipStream_t);
  };
  static const Tile tiles[] = {
      {32, 64, 3.4, 0.175, launch_tile<32, 64, 1, 2, 2, 3>}, {64, 64, 4.0, 0.25, launch_tile<64, 64, 2, 4, 1, 3>},
      {128, 128, 2.0, 0.47, launch_gemm<128, 128, 4, 2>},    {256, 128, 3.0, 0.85, launch_gemm<256, 128, 4, 2>},
      {256, 256, 3.0, 1.62, launch_gemm<256, 256, 4, 2>},
  };
  const Tile* best = nullptr;
  double least = 0.0;
  for (const Tile& t : tiles) {
    const int64_t items = (p.rows + t.tok - 1) / t.tok * ((p.n + t.ch - 1) / t.ch);
    const double time = t.start + (double)((items + kGemmCus - 1) / kGemmCus) * p.kblocks * t.block;
    if (best == nullptr || time < least) best = &t, least = time;
  }
  best->launch(p, stream);
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
  launch_product(p, stream);
  DSV4_CHECK_LAUNCH("product_tile_kernel");
  return DSV4MOE_OK;
}

// One launch, or the quantiser and the product.
int dsv4_launch_int8_linear(const void* x, int32_t x_dtype, int64_t m, int64_t n, int64_t k, const int8_t* wq,
                            const uint16_t* ws, int8_t* q, float* scale, uint16_t* out, hipStream_t stream) {
  if (m <= 16 && few_code_bytes(m, k) <= kFewCodes) {
    const FewParams p{x, (int)m, (int)n, (int)k, reinterpret_cast<const uint8_t*>(wq), ws, out};
    if (x_dtype == DSV4MOE_DTYPE_BF16) return launch_few<DSV4MOE_DTYPE_BF16>(p, stream);
    if (x_dtype == DSV4MOE_DTYPE_FP16) return launch_few<DSV4MOE_DTYPE_FP16>(p, stream);
    return launch_few<DSV4MOE_DTYPE_FP32>(p, stream);
  }
  const int rc = dsv4_launch_act_quant_int8(x, x_dtype, m, k, q, scale, stream);
  if (rc != DSV4MOE_OK) return rc;
  return dsv4_launch_int8_gemm(q, scale, m, n, k, wq, ws, out, stream);
}

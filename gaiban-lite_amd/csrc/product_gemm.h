// The product of product_tile.h for many rows: one workgroup of eight wavefronts per CU,
// two stages of 256 or 128 rows x CH channels in LDS.
#pragma once

#include <type_traits>

#include "product_tile.h"

namespace dsv4 {

constexpr int kGemmCus = 256;
constexpr int kGemmGroup = 4;  // dense: token tiles that walk the channel tiles together

// The tiles of a grouped call, built by every workgroup for itself from the blocks'
// experts: a tile is up to tile_blocks neighbouring blocks of one expert.  kChunk blocks
// at a time.
struct TileList {
  static constexpr int kPer = 4;
  static constexpr int kChunk = 512 * kPer;
  int expert[kChunk];  // of each block, -1: none
  uint16_t first[kChunk];
  int wave_last[8], wave_count[8];

  // Called by 512 threads; returns the number of tiles of blocks [base, base + kChunk).
  __device__ __forceinline__ int build(const ProductParams& p, int base, int active) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = threadIdx.x * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = base + b0 + i;
      const int e = b < active ? p.expert_ids[b] : -1;
      expert[b0 + i] = e >= 0 && e < p.experts ? e : -1;
    }
    __syncthreads();
    // the last run start at or before each block: a maximum over threads
    int before = b0 > 0 ? expert[b0 - 1] : -2, last = -1;
    bool start[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      start[i] = expert[b0 + i] != before;
      if (start[i]) last = b0 + i;
      before = expert[b0 + i];
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(last, off, 64);
      if (lane >= off) last = max(last, v);
    }
    if (lane == 63) wave_last[wave] = last;
    int run = __shfl_up(last, 1, 64);
    if (lane == 0) run = -1;
    __syncthreads();
    for (int w = 0; w < wave; ++w) run = max(run, wave_last[w]);
    // every tile_blocks-th block of a run begins a tile
    bool lead[kPer];
    int count = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (start[i]) run = b0 + i;
      lead[i] = expert[b0 + i] >= 0 && (b0 + i - run) % p.tile_blocks == 0;
      count += lead[i];
    }
    int sum = count;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(sum, off, 64);
      if (lane >= off) sum += v;
    }
    if (lane == 63) wave_count[wave] = sum;
    __syncthreads();
    int at = sum - count, total = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < wave) at += wave_count[w];
      total += wave_count[w];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lead[i]) first[at++] = (uint16_t)(b0 + i);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(total);
  }
  // blocks of the tile that begins at block b of the chunk
  __device__ __forceinline__ int blocks(int b, int tile_blocks) const {
    const int lane = threadIdx.x & 63;
    const int i = b + lane;
    const uint64_t other = __ballot(lane >= tile_blocks || i >= kChunk || expert[min(i, kChunk - 1)] != expert[b]);
    return __builtin_ctzll(other);  // tile_blocks <= 32: a bit is set
  }
};
struct NoTileList {};

// One workgroup per CU, eight wavefronts (WM x WN), two stages.  Wavefront (wm, wn) owns
// columns c * WM + wm and strips wn * TN .. as in product_tile_kernel.  Half the strips'
// fragments are held, a strip's registers being refilled behind its MFMAs with the strip
// half a block later; the rows' fragments of the next block are read during the second
// half.  So no MFMA waits for the reads of eight wavefronts at once, and what has been
// read of a block (its rows and first strips when it begins, the other strips in its
// middle) makes room for the copies of block kb + 2 at once: each lands one and a half
// blocks later.  The two barriers of a block stand behind a strip's MFMAs, so that the
// reads before them have landed.
//
// Grouped: the workgroups stay and walk the items (tile, channel tile) of their XCD's share
// in that order, so one XCD's L2 serves an expert's rows to all its channel tiles.  Columns
// without rows are not multiplied: COLS of the TM columns of a wavefront, chosen per tile.
template <class Op, int TOK, int CH, int WM, int WN, bool GROUPED, bool SWIGLU>
__global__ __launch_bounds__(512, 1) void product_gemm_kernel(ProductParams p) {
  constexpr int kWaves = WM * WN;
  constexpr int TM = TOK / 16 / WM;
  constexpr int TN = CH / 16 / WN;
  constexpr int H = TN / 2;
  constexpr int kStage = (TOK + CH) * kBlockBytes;
  static_assert(kWaves == 8 && TM * 16 * WM == TOK && TN * 16 * WN == CH && TN % 2 == 0, "eight wavefronts");
  static_assert(TM <= 2 * H, "two columns' fragments per strip of the second half");
  static_assert(TOK / 8 % kWaves == 0 && CH / 16 % kWaves == 0, "every wavefront issues the same copies");
  __shared__ __attribute__((aligned(16))) uint8_t ring[2 * kStage];
  __shared__ TileRows<TOK> rows;
  __shared__ std::conditional_t<GROUPED, TileList, NoTileList> list;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN;
  const int wn = wave % WN;
  const int n16 = lane & 15;
  const int j = lane >> 4;
  const int key = swz128(n16);
  const int last = p.kblocks - 1;
  const uint32_t tail = p.kbytes - last * kBlockBytes;  // bytes of the last block
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(&ring[0]));
  constexpr int kXCopies = TOK / 8 / kWaves;
  constexpr int kWCopies = CH / 8 / kWaves;
  constexpr int kCopies = kXCopies + kWCopies;
  constexpr int kEarly = kXCopies + kWCopies / 2;  // copies of the part of a block that is read first
  // the 16-byte part of a row that this lane copies: the same in all its copies, groups of
  // eight rows that are odd or even with the wavefront
  const uint32_t part = ((lane & 7) ^ (lane >> 3) ^ (wave & 1)) * 16;

  // the group of eight weight rows that copy i fills: first those of the wavefront columns'
  // strips below H, then the others
  auto w_group = [&](int i) {
    const int l = wave + kWaves * (i % (kWCopies / 2));
    return l / (2 * H) * 2 * TN + l % (2 * H) + (i < kWCopies / 2 ? 0 : 2 * H);
  };

  auto tile = [&](int tm, int tn, int expert, int first, int count, const uint8_t* xbase, uint32_t xbytes) {
    rows.template fill<GROUPED>(p, first, count);
    __syncthreads();
    const __amdgpu_buffer_rsrc_t x_rsrc =
        __builtin_amdgcn_make_buffer_rsrc((void*)xbase, (short)0, (int)xbytes, kTileRsrcFlags);
    const uint8_t* wbase = p.w + (int64_t)expert * p.n * p.kbytes;
    const __amdgpu_buffer_rsrc_t w_rsrc =
        __builtin_amdgcn_make_buffer_rsrc((void*)wbase, (short)0, (int)((int64_t)p.n * p.kbytes), kTileRsrcFlags);
    uint32_t x_off[kXCopies], w_off[kWCopies];
#pragma unroll
    for (int i = 0; i < kXCopies; ++i)
      x_off[i] = x_row_offset<GROUPED>(p, rows.id[(wave + kWaves * i) * 8 + (lane >> 3)]) + part;
#pragma unroll
    for (int i = 0; i < kWCopies; ++i)
      w_off[i] = w_row_offset<CH, TN, WN, SWIGLU>(p, tn, w_group(i) * 8 + (lane >> 3)) + part;
    // One copy of block kb into stage `u`; past the end of K: zeros.
    auto copy = [&](int kb, int u, int i) {
      const uint32_t limit = kb < last ? kBlockBytes : (kb == last ? tail : 0);
      const int soff = min(kb, last) * kBlockBytes;
      if (i < kXCopies)
        lds_copy16(x_rsrc, base + u * kStage + (wave + kWaves * i) * 1024, part < limit ? x_off[i] : kTileOob, soff);
      else
        lds_copy16(w_rsrc, base + u * kStage + TOK * kBlockBytes + w_group(i - kXCopies) * 1024,
                   part < limit ? w_off[i - kXCopies] : kTileOob, soff);
    };
    typename Op::Acc acc[TN][TM];
#pragma unroll
    for (int r = 0; r < TN; ++r)
#pragma unroll
      for (int c = 0; c < TM; ++c) acc[r][c] = Op::zero();

    struct Frag {
      u32x4 d[2];
    };
    auto read = [&](const uint8_t* from, int row) {
      const uint8_t* at = from + row * kBlockBytes;
      return Frag{{load16(at + ((j ^ key) * 16)), load16(at + (((4 + j) ^ key) * 16))}};
    };
    auto read_strip = [&](int u, int r) { return read(&ring[u * kStage + TOK * kBlockBytes], (wn * TN + r) * 16 + n16); };
    auto read_column = [&](int u, int c) { return read(&ring[u * kStage], (c * WM + wm) * 16 + n16); };

#pragma unroll
    for (int i = 0; i < kCopies; ++i) copy(0, 0, i);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) copy(1, 1, i);
    lds_dma_wait_keep<2 * kCopies - kEarly>();
    __syncthreads();

    auto loop = [&](auto cols_c) __attribute__((always_inline)) {
      constexpr int COLS = decltype(cols_c)::value;
      Frag wf[H], xa[COLS], xb[COLS];
      auto step = [&](int kb, auto u_c, const Frag(&cur)[COLS], Frag(&nxt)[COLS]) __attribute__((always_inline)) {
        constexpr int u = decltype(u_c)::value;
#pragma unroll
        for (int r = 0; r < TN; ++r) {
          // copies of block kb + 2 into what has been read of block kb: spread over the strips
          // behind the barrier
          const int first = r < H ? 0 : kEarly, count = r < H ? kEarly : kCopies - kEarly;
          const int slots = (H - 1) * 2 * COLS, at = (r % H - 1) * 2 * COLS;
#pragma unroll
          for (int m = 0; m < 2 * COLS; ++m) {
            const int d = m / COLS, c = m % COLS;
            acc[r][c] = Op::mfma(wf[r % H].d[d], cur[c].d[d], acc[r][c]);
            __builtin_amdgcn_sched_barrier(0);
            if (r % H > 0) {
#pragma unroll
              for (int i = 0; i < count; ++i)
                if (i * slots / count == at + m) copy(kb + 2, u, first + i);
            }
          }
          if (r % H == 0) {
            // Strip 0: the later part of block kb has landed, and every wavefront has its
            // rows and first strips of block kb in registers.  Strip H: the early part of
            // block kb + 1 has landed, the rest of block kb is in registers.
            lds_dma_wait_keep<kCopies>();
            __syncthreads();
          }
          wf[r % H] = r < H ? read_strip(u, r + H) : read_strip(u ^ 1, r - H);
          if (r >= H) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if ((r - H) * 2 + c < COLS) nxt[(r - H) * 2 + c] = read_column(u ^ 1, (r - H) * 2 + c);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
#pragma unroll
      for (int c = 0; c < COLS; ++c) xa[c] = read_column(0, c);
#pragma unroll
      for (int r = 0; r < H; ++r) wf[r] = read_strip(0, r);
      // an odd number of blocks: the last step multiplies zeros
      for (int kb = 0; kb < p.kblocks; kb += 2) {
        step(kb, std::integral_constant<int, 0>{}, xa, xb);
        step(kb + 1, std::integral_constant<int, 1>{}, xb, xa);
      }
    };
    if constexpr (GROUPED) {
      const int columns = (rows.rows() + 15) >> 4;
      const int mine = columns > wm ? (columns - wm + WM - 1) / WM : 0;
      if (TM == 4 && mine > 3) loop(std::integral_constant<int, TM>{});
      else if (TM >= 3 && mine > 2) loop(std::integral_constant<int, TM < 3 ? TM : 3>{});
      else if (mine > 1) loop(std::integral_constant<int, 2>{});
      else loop(std::integral_constant<int, 1>{});
    } else {
      loop(std::integral_constant<int, TM>{});
    }
    lds_dma_wait_all();
    __syncthreads();  // every wavefront has read its last fragments and its copies have landed
    store_tile<Op, TOK, TM, TN, WM, WN, GROUPED, SWIGLU>(p, acc, ring, rows, tm, tn, expert);
  };

  if constexpr (GROUPED) {
    const int active = min(p.blocks, *p.post_padded / p.block_size);  // none where the ids were out of range (-1)
    const int xcd = blockIdx.x % kTileXcds;
    for (int chunk = 0; chunk < active; chunk += TileList::kChunk) {
      __syncthreads();
      const int64_t items = (int64_t)list.build(p, chunk, active) * p.tiles_n;
      const int64_t end = items * (xcd + 1) / kTileXcds;
      for (int64_t it = items * xcd / kTileXcds + blockIdx.x / kTileXcds; it < end; it += gridDim.x / kTileXcds) {
        const int b = list.first[it / p.tiles_n];
        const int count = list.blocks(b, p.tile_blocks) * p.block_size;
        const int expert = __builtin_amdgcn_readfirstlane(list.expert[b]);
        tile(0, (int)(it % p.tiles_n), expert, (chunk + b) * p.block_size, count, p.x, (uint32_t)(p.rows * p.kbytes));
        __syncthreads();  // the output tile and the rows have been read
      }
    }
  } else {
    const int items = p.tiles_m * p.tiles_n;
    const int per_xcd = (items + kTileXcds - 1) / kTileXcds;
    const int item = (blockIdx.x % kTileXcds) * per_xcd + blockIdx.x / kTileXcds;
    if (item >= items) return;
    const int group = item / (kGemmGroup * p.tiles_n);
    const int gm = min(kGemmGroup, p.tiles_m - group * kGemmGroup);
    const int in_group = item - group * kGemmGroup * p.tiles_n;
    const int tm = group * kGemmGroup + in_group % gm;
    const int64_t row0 = (int64_t)tm * TOK;
    const int count = (int)(p.rows - row0 < TOK ? p.rows - row0 : TOK);
    tile(tm, in_group / gm, 0, 0, count, p.x + row0 * p.kbytes, (uint32_t)count * (uint32_t)p.kbytes);
  }
}

}  // namespace dsv4

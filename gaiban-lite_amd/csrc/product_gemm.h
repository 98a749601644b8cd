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
  static constexpr int kPer = 2;
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

// 16 bytes of LDS at a byte address and a constant offset.
__device__ __forceinline__ u32x4 lds_load16(uint32_t at, int off) {
  typedef __attribute__((address_space(3))) const u32x4* ptr;
  return *(ptr)(uintptr_t)(at + off);
}

// A value the compiler knows nothing of from here on.
__device__ __forceinline__ void opaque(uint32_t& v) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(v));
#endif
}

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
// The workgroups stay and walk their share of the tiles; the last two blocks of a tile
// copy the first two of the next, so that its first reads are under way during the stores.
// An XCD takes neighbouring items: grouped, all channel tiles of an expert's rows; dense,
// kGemmGroup row tiles walking the channel tiles together.  Columns without rows are not
// multiplied (grouped): COLS of the TM columns of a wavefront, chosen per tile.
//
// The MFMA bounds it, at the clock that its power leaves: int8 M=8192 N=16384 K=4096 414 to 451
// us (2.4-2.6 PTOP/s, MFMA busy 0.68 of the cycles); 8192 tokens x 6 over 256 bf16 experts, N=K=
// 4096, where the weights are streamed as well, 1786 us (0.66).  All tiles begin at
// K = 0: in first_block's order the rows that tiles share miss the L2 (447 -> 462 us).
template <class Op, int TOK, int CH, int WM, int WN, bool GROUPED, bool SWIGLU, bool ONCE>
__global__ __launch_bounds__(512, 1) void product_gemm_kernel(ProductParams p) {
  constexpr int kWaves = WM * WN;
  constexpr int TM = TOK / 16 / WM;
  constexpr int TN = CH / 16 / WN;
  constexpr int H = TN / 2;
  constexpr int kXStage = TOK * kBlockBytes, kWStage = CH * kBlockBytes;
  constexpr int kOutStrips = SWIGLU ? TN / 2 : TN;  // a wavefront's strips of output channels
  constexpr int kPass = kOutStrips < 4 ? kOutStrips : 4;  // strips that a wavefront stores together
  static_assert(kWaves == 8 && TM * 16 * WM == TOK && TN * 16 * WN == CH && TN % 2 == 0, "eight wavefronts");
  static_assert(TM <= 2 * H && TM <= 4, "two columns' fragments per strip of the second half");
  static_assert(TOK / 8 % kWaves == 0 && CH / 16 % kWaves == 0, "every wavefront issues the same copies");
  static_assert(kOutStrips % kPass == 0 && (kPass & (kPass - 1)) == 0, "whole passes of the stores");
  __shared__ __attribute__((aligned(128))) uint8_t ring[2 * (kXStage + kWStage)];  // rows, then weights
  __shared__ __attribute__((aligned(16))) uint8_t staged[kWaves][16 * kPass * 32];
  __shared__ TileRows<GROUPED ? TOK : 1> rows[3];  // in turn: one tile may still be stored when the next but one is listed
  __shared__ std::conditional_t<GROUPED, TileList, NoTileList> list;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN;
  const int wn = wave % WN;
  const int n16 = lane & 15;
  const int j = lane >> 4;
  const int last = p.kblocks - 1;
  const int steps = (p.kblocks + 1) & ~1;  // an odd number of blocks: one more of zeros
  const uint32_t tail = p.kbytes - last * kBlockBytes;  // bytes of the last block
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(&ring[0]));
  constexpr int kXCopies = TOK / 8 / kWaves;
  constexpr int kWCopies = CH / 8 / kWaves;
  constexpr int kCopies = kXCopies + kWCopies;
  constexpr int kEarly = kXCopies + kWCopies / 2;  // copies of the part of a block that is read first
  // the row of each group of eight and its 16-byte part that this lane copies: the same in
  // all its copies
  const int lane_row = lane >> 3;
  const uint32_t part = lds_part<128>(lane_row, lane & 7) * 16;
  // the group of eight weight rows that copy i fills: first those of the wavefront columns'
  // strips below H, then the others
  auto w_group = [&](int i) {
    const int l = wave + kWaves * (i % (kWCopies / 2));
    return l / (2 * H) * 2 * TN + l % (2 * H) + (i < kWCopies / 2 ? 0 : 2 * H);
  };

  // the first channel of a group of eight weight rows, from the tile's first
  auto w_row = [&](int group) {
    const int strip = group >> 1;
    if constexpr (SWIGLU) {
      const int r = strip % TN;
      return (strip / TN * (TN / 2) + r % (TN / 2)) * 16 + (group & 1) * 8 + (r < TN / 2 ? 0 : p.n >> 1);
    } else {
      return group * 8;
    }
  };

  // ---- the items of this workgroup
  struct Item {
    int tm, tn;    // dense: the row tile
    int expert;
    int first;     // grouped: its first sorted slot
    int count;     // rows, 0: no item
  };
  const int xcd = blockIdx.x % kTileXcds;
  int64_t at, end;
  int chunk = -1, active = 0;  // grouped: the first block of the listed chunk
  if constexpr (GROUPED) {
    active = min(p.blocks, *p.post_padded / p.block_size);  // none where the ids were out of range (-1)
    at = end = 0;
  } else {
    const int64_t items = (int64_t)p.tiles_m * p.tiles_n;
    end = items * (xcd + 1) / kTileXcds;
    at = items * xcd / kTileXcds + blockIdx.x / kTileXcds;
  }
  // by the whole workgroup
  auto next_item = [&]() {
    Item t{0, 0, 0, 0, 0};
    if constexpr (GROUPED) {
      while (at >= end) {
        chunk = chunk < 0 ? 0 : chunk + TileList::kChunk;
        if (chunk >= active) return t;
        __syncthreads();
        const int64_t items = (int64_t)list.build(p, chunk, active) * p.tiles_n;
        end = items * (xcd + 1) / kTileXcds;
        at = items * xcd / kTileXcds + blockIdx.x / kTileXcds;
      }
      const int b = list.first[at / p.tiles_n];
      t.tn = (int)(at % p.tiles_n);
      t.expert = __builtin_amdgcn_readfirstlane(list.expert[b]);
      t.first = __builtin_amdgcn_readfirstlane((chunk + b) * p.block_size);
      t.count = __builtin_amdgcn_readfirstlane(list.blocks(b, p.tile_blocks) * p.block_size);
    } else {
      if (at >= end) return t;
      const int group = (int)(at / (kGemmGroup * p.tiles_n));
      const int gm = min(kGemmGroup, p.tiles_m - group * kGemmGroup);
      const int in_group = (int)(at - (int64_t)group * kGemmGroup * p.tiles_n);
      t.tm = group * kGemmGroup + in_group % gm;
      t.tn = in_group / gm;
      t.count = (int)min((int64_t)TOK, p.rows - (int64_t)t.tm * TOK);
    }
    at += gridDim.x / kTileXcds;
    return t;
  };

  // ---- copies: of the tile that `aim` chose
  __amdgpu_buffer_rsrc_t x_rsrc, w_rsrc;
  // Offsets in VGPRs are few, the loop has none to spare: copies of weights, and of a dense
  // call's rows, differ from the first by whole rows.  (Rows past the last are past the
  // buffer's end; with SwiGLU gate rows past the last read up rows, for channels that
  // nothing stores.)
  constexpr int kXOffs = GROUPED ? kXCopies : 1;
  uint32_t x_off[kXOffs], w_off;
  auto aim = [&](const Item& t, int slot) {
    const uint8_t* xbase = p.x;
    uint32_t xbytes;
    if constexpr (GROUPED) {
      xbytes = t.count > 0 ? (uint32_t)(p.rows * p.kbytes) : 0;  // below 2^31 (host check)
#pragma unroll
      for (int i = 0; i < kXCopies; ++i)
        x_off[i] = x_row_offset<true>(p, t.count > 0 ? rows[slot].id[(wave + kWaves * i) * 8 + lane_row] : -1) + part;
    } else {
      xbase += (int64_t)t.tm * TOK * p.kbytes;
      xbytes = (uint32_t)t.count * (uint32_t)p.kbytes;
      x_off[0] = (uint32_t)(wave * 8 + lane_row) * (uint32_t)p.kbytes + part;
    }
    x_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)xbase, (short)0, (int)xbytes, kTileRsrcFlags);
    const uint8_t* wbase = p.w + (int64_t)t.expert * p.n * p.kbytes;
    const int wbytes = t.count > 0 ? (int)((int64_t)p.n * p.kbytes) : 0;
    w_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)wbase, (short)0, wbytes, kTileRsrcFlags);
    w_off = (uint32_t)(t.tn * (SWIGLU ? CH / 2 : CH) + w_row(w_group(0)) + lane_row) * (uint32_t)p.kbytes + part;
  };
  // One copy of block kb into stage `u`; past the end of K: zeros.
  auto copy = [&](int kb, int u, int i) __attribute__((always_inline)) {
    const uint32_t limit = kb < last ? kBlockBytes : (kb == last ? tail : 0);
    const int soff = min(kb, last) * kBlockBytes;
    // the sums stay in the loop: hoisted, each copy's would take a register of its own
    uint32_t off = i >= kXCopies ? w_off : x_off[GROUPED ? i : 0];
    opaque(off);
    off = part < limit ? off : kTileOob;
    if (i < kXCopies) {
      if constexpr (!GROUPED) off += kWaves * 8 * i * (uint32_t)p.kbytes;
      lds_copy16(x_rsrc, base + u * kXStage + (wave + kWaves * i) * 1024, off, soff);
    } else {
      off += (uint32_t)(w_row(w_group(i - kXCopies)) - w_row(w_group(0))) * (uint32_t)p.kbytes;
      copy_weights16<ONCE>(w_rsrc, base + 2 * kXStage + u * kWStage + w_group(i - kXCopies) * 1024, off, soff);
    }
  };

  struct Frag {
    u32x4 d[2];
  };
  // fragment addresses: strips, columns and stages are constants beside two lane addresses
  // each (part 4 + j lies at the other half of part j's row, 64 bytes off)
  uint32_t x_lds = base + (wm * 16 + n16) * kBlockBytes + lds_part<128>(n16, j) * 16;
  uint32_t w_lds = base + 2 * kXStage + (wn * TN * 16 + n16) * kBlockBytes + lds_part<128>(n16, j) * 16;
  uint32_t x_lds4 = x_lds ^ 64, w_lds4 = w_lds ^ 64;
  opaque(x_lds), opaque(x_lds4), opaque(w_lds), opaque(w_lds4);
  auto read_strip = [&](int u, int r) __attribute__((always_inline)) {
    const int off = u * kWStage + r * 16 * kBlockBytes;
    return Frag{{lds_load16(w_lds, off), lds_load16(w_lds4, off)}};
  };
  auto read_column = [&](int u, int c) __attribute__((always_inline)) {
    const int off = u * kXStage + c * WM * 16 * kBlockBytes;
    return Frag{{lds_load16(x_lds, off), lds_load16(x_lds4, off)}};
  };

  typename Op::Acc acc[TN][TM];
  Item now = next_item(), next{0, 0, 0, 0, 0};
  if (now.count == 0) return;
  int slot = 0;  // of `rows`: the current tile's
  if constexpr (GROUPED) {
    rows[0].template fill<GROUPED>(p, now.first, now.count);
    __syncthreads();
  }
  aim(now, 0);
#pragma unroll
  for (int i = 0; i < kCopies; ++i) copy(0, 0, i);
#pragma unroll
  for (int i = 0; i < kCopies; ++i) copy(1, 1, i);

  // all blocks of the current tile with COLS columns
  auto multiply = [&](auto cols_c) __attribute__((always_inline)) {
    constexpr int COLS = decltype(cols_c)::value;
    Frag wf[H], xa[COLS], xb[COLS];
    auto step = [&](int ahead, auto u_c, const Frag(&cur)[COLS], Frag(&nxt)[COLS]) __attribute__((always_inline)) {
      constexpr int u = decltype(u_c)::value;
#pragma unroll
      for (int r = 0; r < TN; ++r) {
        // copies of block `ahead`, two later, into what has been read of this one: spread
        // over the strips behind the barrier
        const int first = r < H ? 0 : kEarly, count = r < H ? kEarly : kCopies - kEarly;
        const int slots = (H - 1) * 2 * COLS, s0 = (r % H - 1) * 2 * COLS;
#pragma unroll
        for (int m = 0; m < 2 * COLS; ++m) {
          const int d = m / COLS, c = m % COLS;
          acc[r][c] = Op::mfma(wf[r % H].d[d], cur[c].d[d], acc[r][c]);
          __builtin_amdgcn_sched_barrier(0);
          if (r % H > 0) {
#pragma unroll
            for (int i = 0; i < count; ++i)
              if (i * slots / count == s0 + m) copy(ahead, u, first + i);
          }
        }
        if (r % H == 0) {
          // Strip 0: the later part of this block has landed, and every wavefront has its
          // rows and first strips of it in registers.  Strip H: the early part of the next
          // block has landed, the rest of this one is in registers.
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
    for (int kb = 0; kb < steps; kb += 2) {
      int ahead = kb + 2;
      if (ahead == steps) {  // from here on the next tile's blocks
        aim(next, slot == 2 ? 0 : slot + 1);
        ahead = 0;
      }
      step(ahead, std::integral_constant<int, 0>{}, xa, xb);
      step(ahead + 1, std::integral_constant<int, 1>{}, xb, xa);
    }
  };

  while (true) {
    next = next_item();
    if constexpr (GROUPED) {
      if (next.count > 0) rows[slot == 2 ? 0 : slot + 1].template fill<GROUPED>(p, next.first, next.count);
    }
#pragma unroll
    for (int r = 0; r < TN; ++r)
#pragma unroll
      for (int c = 0; c < TM; ++c) acc[r][c] = Op::zero();
    lds_dma_wait_keep<2 * kCopies - kEarly>();  // the early part of the first block has landed
    __syncthreads();
    int mine = TM;
    if constexpr (GROUPED) {
      const int columns = (rows[slot].rows() + 15) >> 4;
      mine = columns > wm ? (columns - wm + WM - 1) / WM : 0;
    }
    if (!GROUPED || mine > 3) multiply(std::integral_constant<int, TM>{});
    else if (mine > 2) multiply(std::integral_constant<int, TM < 3 ? TM : 3>{});
    else if (mine > 1) multiply(std::integral_constant<int, TM < 2 ? TM : 2>{});
    else multiply(std::integral_constant<int, 1>{});
    // vmcnt(0): registers reloaded for the stores.  A wavefront may branch past their use, and
    // the compiler then waits for them in the K loop, where its wait is one for the copies just
    // issued (bf16 SwiGLU, 8192 tokens x 6 over 256 experts 1870 -> 1786 us)
    if constexpr (GROUPED) __builtin_amdgcn_s_waitcnt(0x0F70);
    // store: a wavefront's tile, kPass strips of a column of 16 rows at a time
    {
      uint8_t* mine_lds = &staged[wave][0];
      constexpr int kParts = 2 * kPass;
      constexpr int kRowBytes = 16 * kParts;
      constexpr int kRowsPerStore = 64 / kParts;
      const int half = p.n >> 1;
      const int strip0 = (now.tn * WN + wn) * kOutStrips;
      int id[TM];
      float factor[TM];
#pragma unroll
      for (int c = 0; c < TM; ++c) {
        const int row = (c * WM + wm) * 16 + n16;
        if constexpr (GROUPED) id[c] = rows[slot].id[row];
        else id[c] = row < now.count ? row : -1;
        factor[c] = GROUPED ? 1.0f : 0.0f;
        if constexpr (GROUPED) factor[c] = rows[slot].factor[row];
      }
      float xscale[TM];
      if constexpr (Op::kInt8) {
#pragma unroll
        for (int c = 0; c < TM; ++c)
          xscale[c] = id[c] < 0 ? 0.0f
                                : p.x_scale[GROUPED ? (int64_t)((uint32_t)id[c] / (uint32_t)p.per_row)
                                                    : (int64_t)now.tm * TOK + id[c]];
      }
#pragma unroll
      for (int pass = 0; pass < kOutStrips / kPass; ++pass) {
        float wscale[SWIGLU ? 2 : 1][kPass][4];
        if constexpr (Op::kInt8) {
#pragma unroll
          for (int g = 0; g < (SWIGLU ? 2 : 1); ++g)
#pragma unroll
            for (int r = 0; r < kPass; ++r) {
              const int ch = min((strip0 + pass * kPass + r) * 16 + 4 * j, p.out_n - 4) + g * half;
              const u32x2 sc = *reinterpret_cast<const u32x2*>(p.w_scale + (int64_t)now.expert * p.n + ch);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                wscale[g][r][e] = __uint_as_float((e & 1) ? sc[e >> 1] & 0xFFFF0000u : sc[e >> 1] << 16);
            }
        }
#pragma unroll
        for (int c = 0; c < TM; ++c) {
          auto value = [&](int g, int r, int e) {
            const int strip = g * kOutStrips + pass * kPass + r;
            if constexpr (Op::kInt8) return (float)acc[strip][c][e] * xscale[c] * wscale[g][r][e];
            else return acc[strip][c][e];
          };
#pragma unroll
          for (int r = 0; r < kPass; ++r) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (SWIGLU) v[e] = swiglu_value(value(0, r, e), value(1, r, e), p.clamp);
              else v[e] = value(0, r, e);
              if constexpr (GROUPED) v[e] *= factor[c];
            }
            const int q = (2 * r + (j >> 1)) ^ (n16 & (kParts - 1));
            *reinterpret_cast<u32x2*>(mine_lds + n16 * kRowBytes + q * 16 + (j & 1) * 8) =
                u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
          }
#pragma unroll
          for (int i = 0; i < 16 / kRowsPerStore; ++i) {
            const int row = i * kRowsPerStore + lane / kParts, q = lane % kParts;
            const int ch = (strip0 + pass * kPass + (q >> 1)) * 16 + (q & 1) * 8;
            const u32x4 o = load16(mine_lds + row * kRowBytes + ((q ^ (row & (kParts - 1))) * 16));
            const int to = __shfl(id[c], row, 64);
            if (to < 0 || ch >= p.out_n) continue;
            const int64_t dst = GROUPED ? (int64_t)to : (int64_t)now.tm * TOK + to;
            *reinterpret_cast<u32x4*>(p.out + dst * p.out_n + ch) = o;
          }
        }
      }
    }
    if (next.count == 0) break;
    now = next;
    slot = slot == 2 ? 0 : slot + 1;
  }
  lds_dma_wait_all();
}

}  // namespace dsv4

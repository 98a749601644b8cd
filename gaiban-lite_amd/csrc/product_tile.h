// Products of activation rows with weight rows, out[i, n] = x[row(i), :] . W[n, :],
// shared by the int8 linear (int8_linear.hip) and the linears grouped by expert
// (grouped.hip).
//
// One operand layout serves both element types.  Rows are handled as bytes, in blocks
// of 128 bytes of K (64 bf16 or 128 int8 values).  16 bytes are one lane's operand of
// one MFMA in either type: 8 bf16 of v_mfma_f32_16x16x32_bf16 or 16 int8 of
// v_mfma_i32_16x16x64_i8, lane group j = lane / 16 holding K bytes 16 j .. + 15 of a
// 64-byte half block.  Weights are the MFMA's A operand (its rows are channels) and
// activations its B operand, so a lane's four accumulators are four neighbouring
// channels of one token.
#pragma once

#include "common.h"

namespace dsv4 {

typedef __attribute__((ext_vector_type(4))) int i32x4;

constexpr int kTileXcds = 8;
constexpr uint32_t kTileOob = 0x80000000u;  // beyond every buffer (each below 2^31 bytes): reads zeros
constexpr int kTileRsrcFlags = 0x00020000;
constexpr int kBlockBytes = 128;  // K bytes of a row per block

struct ProductBf16 {
  typedef f32x4 Acc;
  static constexpr bool kInt8 = false;
  __device__ static __forceinline__ Acc zero() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ static __forceinline__ Acc mfma(u32x4 w, u32x4 x, Acc c) {
    return mfma_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c);
  }
};
struct ProductInt8 {
  typedef i32x4 Acc;
  static constexpr bool kInt8 = true;
  __device__ static __forceinline__ Acc zero() { return i32x4{0, 0, 0, 0}; }
  __device__ static __forceinline__ Acc mfma(u32x4 w, u32x4 x, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w), __builtin_bit_cast(i32x4, x), c, 0, 0,
                                                 0);
  }
};

// Where 16-byte part `part` of a row of a block of BLOCK bytes (128 or a multiple of 256)
// lies in the row's bytes of LDS.  The LDS serves a ds_read_b128 in sets of 16 lanes (0-3,
// 12-15, 20-27 and 4-11, 16-19, 28-31 of each half of a wavefront: measured by moving one
// lane at a time onto another's banks); with part j of row r at j ^ (r & 7), for rows of
// whole 256 bytes j ^ (r & 15), lanes (row r, part j = lane / 16) of a set fall into all
// sixteen slots of the 256 bytes of banks: no conflict in the K loop (SQ_LDS_BANK_CONFLICT
// counts the stores, 1% of the busy cycles; swz128's order, made for other reads, has four
// conflicts a read here: int8 M=8192 N=16384 K=4096 476 -> 451 us without them).
template <int BLOCK>
__device__ __forceinline__ int lds_part(int row, int part) { return part ^ (row & (BLOCK == 128 ? 7 : 15)); }

// The K block a channel tile begins with (it wraps round to the ones before).  Workgroups that
// run in step and all begin at K = 0 ask for the same bytes of rows that lie a power of two
// apart, which fall on few of the memory's channels; begun anywhere, they spread.  (In order of
// tn it would not do: the channel seems to mix the rows' address bits with those of K, and some
// row lengths cancel.)  16 x 32 tiles over 256 experts, bf16: 300 tokens x 6, N=1024, K=4096
// 399 -> 310 us (5.4 -> 6.9 TB/s), 64 tokens, N=4096, K=2048 504 -> 487.
__device__ __forceinline__ int first_block(int tn, int kblocks) {
  return (int)(((uint32_t)tn * 0x9E3779B9u >> 16) % (uint32_t)kblocks);
}

struct ProductParams {
  const uint8_t* x;  // activation rows of `kbytes` bytes
  int64_t rows;      // their number
  const uint8_t* w;  // weight rows [n] of `kbytes` bytes, per expert
  int n;
  int kbytes;        // a multiple of 16
  int kblocks;       // ceil(kbytes / 128)
  int tiles_m, tiles_n;
  const float* x_scale;     // int8: [rows]
  const uint16_t* w_scale;  // int8: bf16 [experts][n]
  uint16_t* out;
  int out_n;         // channels of an output row: n, or n / 2 with SwiGLU
  // grouped: the slots sorted by expert in padded blocks
  const int32_t* sorted_ids;
  const int32_t* expert_ids;
  const int32_t* post_padded;
  int capacity;      // of sorted_ids
  int blocks;        // entries of expert_ids
  int block_size;
  int tile_blocks;   // blocks of one expert that a tile takes together
  int slots;         // tokens * topk
  int per_row;       // slots that one activation row serves (topk, or 1)
  int experts;
  const float* route_weights;  // [slots] or null
  float clamp;
};

// The tile of grouped work item block `b`: a run of up to tile_blocks blocks of one
// expert, taken by the run's first block (every tile_blocks-th block of its expert's);
// nslots = 0 for a block that has no work of its own.  Called by whole wavefronts.
struct GroupedTile {
  int expert;
  int first_slot;  // in sorted_ids
  int nslots;
};
__device__ __forceinline__ GroupedTile grouped_tile(const ProductParams& p, int b) {
  GroupedTile t{0, b * p.block_size, 0};
  const int lane = threadIdx.x & 63;
  const int active = min(p.blocks, *p.post_padded / p.block_size);  // none where the ids were out of range (-1)
  if (b >= active) return t;
  const int e = p.expert_ids[b];
  if (e < 0 || e >= p.experts) return t;
  if (p.tile_blocks > 1) {
    // blocks of this expert before b: lane i looks at b - 1 - i, 64 at a time
    int before = 0;
    for (int at = b - 1; at >= 0; at -= 64) {
      const int i = at - lane;
      const uint64_t other = __ballot(i < 0 || p.expert_ids[max(i, 0)] != e);
      if (other != 0) {
        before += __builtin_ctzll(other);
        break;
      }
      before += 64;
    }
    if (before % p.tile_blocks != 0) return t;
    const int i = b + lane;
    const uint64_t other = __ballot(lane >= p.tile_blocks || i >= active || p.expert_ids[min(i, active - 1)] != e);
    t.nslots = __builtin_ctzll(other) * p.block_size;  // tile_blocks < 64: a bit is set
  } else {
    t.nslots = p.block_size;
  }
  t.expert = e;
  return t;
}

// lds_copy16 of weights.  ONCE: by one workgroup alone, so the lines need not stay in the
// caches (nt).  One token over 256 experts (N=K=4096) 36.6 -> 33.8 us, 64 tokens (K=2048) 549
// -> 521, 1000 tokens 1553 -> 1460 (5.9 TB/s); weights that several tiles read lose by it (64
// experts, 512 rows each, 585 -> 650), and so do rows that are not whole 128-byte lines, whose
// ends two blocks share (K=1424 41 -> 46.5), and weights that the cache in front of HBM still
// holds from the call before (a dense call over 67 MB 15.9 -> 20.0).
template <bool ONCE>
__device__ __forceinline__ void copy_weights16(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, uint32_t voffset,
                                               uint32_t soffset) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voffset), "s"(rsrc),
                   "s"(__builtin_amdgcn_readfirstlane(soffset))
                 : "memory", "m0");
  else
    lds_copy16(rsrc, lds, voffset, soffset);
#endif
}

// silu(min(g, L)) * clamp(u, -L, L), or without limits where L = 0.  Comparisons, which a NaN
// fails: fminf would turn it into L, and a row whose scale is NaN into finite numbers.
__device__ __forceinline__ float swiglu_value(float g, float u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
  }
  return silu_rcp(g) * u;
}

// The rows of a tile, by the whole workgroup.
template <int TOK>
struct TileRows {
  int id[TOK];                    // output row, or -1
  float factor[TOK];              // its route weight
  int used[(TOK + 63) / 64];      // rows up to the last that has one, per 64

  // `count` rows from sorted slot `first` on (grouped) or the first `count` (dense)
  template <bool GROUPED>
  __device__ __forceinline__ void fill(const ProductParams& p, int first, int count) {
    for (int r = threadIdx.x; r < TOK; r += blockDim.x) {
      int i = -1;
      float f = 1.0f;
      if (r < count) {
        if constexpr (GROUPED) {
          if (first + r < p.capacity) i = p.sorted_ids[first + r];
          if ((uint32_t)i >= (uint32_t)p.slots) i = -1;
          if (i >= 0 && p.route_weights != nullptr) f = p.route_weights[i];
        } else {
          i = r;
        }
      }
      id[r] = i;
      factor[r] = f;
      const uint64_t have = __ballot(i >= 0);
      if ((r & 63) == 0) used[r >> 6] = have ? (r & ~63) + 64 - __builtin_clzll(have) : 0;
    }
  }
  // behind a barrier: rows up to the last that has an output
  __device__ __forceinline__ int rows() const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < (TOK + 63) / 64; ++i) n = max(n, used[i]);
    return __builtin_amdgcn_readfirstlane(n);
  }
};

// Byte offset in the activations of output row `id`, or out of range for -1.
template <bool GROUPED>
__device__ __forceinline__ uint32_t x_row_offset(const ProductParams& p, int id) {
  const uint32_t row = GROUPED ? (uint32_t)id / (uint32_t)p.per_row : (uint32_t)id;
  return id >= 0 ? row * (uint32_t)p.kbytes : kTileOob;
}

// Byte offset in the expert's weights of row `row` of channel tile tn (WN wavefront columns
// of TN strips), or out of range past the last channel.
template <int CH, int TN, int WN, bool SWIGLU>
__device__ __forceinline__ uint32_t w_row_offset(const ProductParams& p, int tn, int row) {
  int ch;
  bool in;
  if constexpr (SWIGLU) {
    const int strip = row >> 4, r = strip % TN;  // strip r of wavefront column strip / TN
    const int half = p.n >> 1;
    ch = ((tn * WN + strip / TN) * (TN / 2) + r % (TN / 2)) * 16 + (row & 15);
    in = ch < half;
    ch += r < TN / 2 ? 0 : half;
  } else {
    ch = tn * CH + row;
    in = ch < p.n;
  }
  return in ? (uint32_t)ch * (uint32_t)p.kbytes : kTileOob;
}

// The workgroup's finished tile to the output, through `lds` (TOK rows of all its output
// channels) so that whole rows are stored: 16-byte part q of row r is kept at
// q ^ (r mod parts).  Every wavefront has read its last fragments from `lds`; of WK wavefronts
// that shared a tile's K the first has the sums.
template <class Op, int TOK, int TM, int TN, int WM, int WN, int WK, bool GROUPED, bool SWIGLU>
__device__ __forceinline__ void store_tile(const ProductParams& p, const typename Op::Acc (&acc)[TN][TM],
                                           uint8_t* lds, const TileRows<TOK>& rows, int tm, int tn, int expert) {
  constexpr int kOutStrips = SWIGLU ? TN / 2 : TN;  // a wavefront's strips of output channels
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN % WM;
  const int wn = wave % WN;
  const int n16 = lane & 15;
  const int j = lane >> 4;
  const int half = p.n >> 1;
  constexpr int kParts = 2 * kOutStrips * WN;
  constexpr int kRowBytes = 16 * kParts;
  static_assert((kParts & (kParts - 1)) == 0, "parts of a row: a power of two");
  float wscale[TN][4];
  const int out_strip0 = (tn * WN + wn) * kOutStrips;
  if constexpr (Op::kInt8) {
#pragma unroll
    for (int r = 0; r < TN; ++r) {
      const int ch = (out_strip0 + (SWIGLU ? r % kOutStrips : r)) * 16 + 4 * j;
      const int at = min(ch, p.out_n - 4) + (SWIGLU && r >= kOutStrips ? half : 0);
      const u32x2 s = *reinterpret_cast<const u32x2*>(p.w_scale + (int64_t)expert * p.n + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) wscale[r][e] = __uint_as_float((e & 1) ? s[e >> 1] & 0xFFFF0000u : s[e >> 1] << 16);
    }
  }
#pragma unroll
  for (int c = 0; c < TM; ++c) {
    if (WK > 1 && wave >= WM * WN) break;
    const int row = (c * WM + wm) * 16 + n16;
    const int id = rows.id[row];
    const float factor = rows.factor[row];
    float xscale = 0.0f;
    if constexpr (Op::kInt8) {
      if (id >= 0) xscale = p.x_scale[GROUPED ? (int64_t)(id / p.per_row) : (int64_t)tm * TOK + id];
    }
    auto value = [&](int r, int e) {
      if constexpr (Op::kInt8)
        return (float)acc[r][c][e] * xscale * wscale[r][e];
      else
        return acc[r][c][e];
    };
#pragma unroll
    for (int r = 0; r < kOutStrips; ++r) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (SWIGLU)
          v[e] = swiglu_value(value(r, e), value(kOutStrips + r, e), p.clamp);
        else
          v[e] = value(r, e);
        if constexpr (GROUPED) v[e] *= factor;
      }
      const int part = (2 * (wn * kOutStrips + r) + (j >> 1)) ^ (row & (kParts - 1));
      *reinterpret_cast<u32x2*>(&lds[row * kRowBytes + part * 16 + (j & 1) * 8]) =
          u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TOK * kParts; i += 64 * WM * WN * WK) {
    const int row = i / kParts, q = i % kParts;
    const int ch = tn * (kParts * 8) + q * 8;
    const int id = rows.id[row];
    if (id < 0 || ch >= p.out_n) continue;
    const int64_t dst = GROUPED ? (int64_t)id : (int64_t)tm * TOK + id;
    *reinterpret_cast<u32x4*>(p.out + dst * p.out_n + ch) =
        load16(&lds[row * kRowBytes + ((q ^ (row & (kParts - 1))) * 16)]);
  }
}

// Few rows, where the weights' stream is the bound, and small dense calls: TOK rows x CH
// channels per workgroup, K in blocks of 128 * WK bytes through a ring of S stages in LDS.
// buffer_load ... lds copies a stage (16-byte parts as lds_part says); the copies of block
// kb + S - 1 are issued behind the barrier of block kb, when every wavefront has read block
// kb - 1 out of the stage they refill, so S - 2 blocks are in flight while one is computed.
// Wavefront (wk, wm, wn) takes the wk-th 128 bytes of every block for token columns
// c * WM + wm (16 rows each; interleaved, so that a partly filled tile loads the wavefronts
// alike) and strips wn * TN .. of the tile (16 channels each); the WK partial sums are added
// in that order.  With SwiGLU a wavefront's first TN / 2 strips are gate channels and the
// others the same up channels.
// The weights' stream bounds it: 256 bf16 experts, 64 tokens x 6, N=4096, K=2048 479 us (7.0
// TB/s) with 16 x 32 tiles of 512 bytes of K, 1000 tokens x 6, N=K=4096 1351 us (6.4 TB/s) with
// 64 x 128.  Wide pieces of few rows: copies of 128 bytes of each of 64 to 128 rows stop at 5.8
// TB/s however many are in flight.
template <class Op, int TOK, int CH, int WM, int WN, int WK, int S, bool GROUPED, bool SWIGLU, bool ONCE>
__global__ __launch_bounds__(64 * WM * WN * WK) void product_tile_kernel(ProductParams p) {
  constexpr int kWaves = WM * WN * WK;
  constexpr int TM = TOK / 16 / WM;
  constexpr int TN = CH / 16 / WN;
  constexpr int kBlock = 128 * WK;       // K bytes of a row per block
  constexpr int kLanes = 8 * WK;         // lanes that copy a row of a block
  constexpr int kRowsPerCopy = 64 / kLanes;
  constexpr int kStage = (TOK + CH) * kBlock;
  constexpr int kOutStrips = SWIGLU ? TN / 2 : TN;  // a wavefront's strips of output channels
  constexpr int kPartial = TN * TM * 1024;          // a wavefront's sums
  static_assert(WK == 1 || WK == 2 || WK == 4 || WK == 8, "whole rows per copy");
  static_assert(TM * 16 * WM == TOK && TN * 16 * WN == CH, "whole strips and columns per wavefront");
  static_assert(!SWIGLU || TN % 2 == 0, "gate and up strips in one wavefront");
  static_assert(CH / kRowsPerCopy % kWaves == 0, "every wavefront issues the same weight copies");
  static_assert(TOK * kOutStrips * 16 * WN * 2 <= S * kStage, "the output tile fits the ring");
  static_assert((WK - 1) * WM * WN * kPartial <= S * kStage, "the partial sums fit the ring");
  __shared__ __attribute__((aligned(256))) uint8_t ring[S * kStage];
  __shared__ TileRows<TOK> rows;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave / (WM * WN);
  const int wm = wave / WN % WM;
  const int wn = wave % WN;
  const int n16 = lane & 15;
  const int j = lane >> 4;

  int tm, tn, expert = 0, first = 0, valid;
  const uint8_t* xbase = p.x;
  uint32_t xbytes;
  if constexpr (GROUPED) {
    // neighbouring workgroups, which run on different XCDs, take neighbouring channel tiles:
    // few blocks still use every XCD
    tm = blockIdx.x / p.tiles_n;
    tn = blockIdx.x % p.tiles_n;
    const GroupedTile t = grouped_tile(p, tm);
    valid = __builtin_amdgcn_readfirstlane(t.nslots);
    if (valid == 0) return;
    expert = __builtin_amdgcn_readfirstlane(t.expert);
    first = t.first_slot;
    xbytes = (uint32_t)(p.rows * p.kbytes);  // below 2^31 (host check)
  } else {
    const int items = p.tiles_m * p.tiles_n;
    const int per_xcd = (items + kTileXcds - 1) / kTileXcds;
    const int item = (blockIdx.x % kTileXcds) * per_xcd + blockIdx.x / kTileXcds;
    if (item >= items) return;
    tm = item % p.tiles_m;
    tn = item / p.tiles_m;
    const int64_t row0 = (int64_t)tm * TOK;
    valid = (int)(p.rows - row0 < TOK ? p.rows - row0 : TOK);
    xbase += row0 * p.kbytes;
    xbytes = (uint32_t)valid * (uint32_t)p.kbytes;
  }

  const __amdgpu_buffer_rsrc_t x_rsrc =
      __builtin_amdgcn_make_buffer_rsrc((void*)xbase, (short)0, (int)xbytes, kTileRsrcFlags);
  const uint8_t* wbase = p.w + (int64_t)expert * p.n * p.kbytes;
  const __amdgpu_buffer_rsrc_t w_rsrc =
      __builtin_amdgcn_make_buffer_rsrc((void*)wbase, (short)0, (int)((int64_t)p.n * p.kbytes), kTileRsrcFlags);

  // copy q of a stage fills 1 KiB, its rows kRowsPerCopy q .. (tokens, then weights)
  constexpr int kXGroups = TOK / kRowsPerCopy;
  constexpr int kXCopies = (kXGroups + kWaves - 1) / kWaves;  // the last ones may repeat a group
  constexpr int kWCopies = CH / kRowsPerCopy / kWaves;
  constexpr int kCopies = kXCopies + kWCopies;
  uint32_t x_off[kXCopies], w_off[kWCopies], x_part[kXCopies], w_part[kWCopies];
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(&ring[0]));
  // Bytes past the end of K, and whole blocks past it (the ring runs on without a branch),
  // are read out of range: zeros.
  const int kblocks = (p.kbytes + kBlock - 1) / kBlock;
  const int last = kblocks - 1;
  const uint32_t tail = p.kbytes - last * kBlock;  // bytes of the last block
  const int k0 = ONCE ? first_block(tn, kblocks) : 0;
  auto place = [&](int kb) { return kb + k0 < kblocks ? kb + k0 : kb + k0 - kblocks; };
  auto limit = [&](int kb) { return kb > last ? 0 : (place(kb) < last ? (uint32_t)kBlock : tail); };
#pragma unroll
  for (int i = 0; i < kWCopies; ++i) {
    const int row = (wave + kWaves * i) * kRowsPerCopy + lane / kLanes;
    w_part[i] = lds_part<kBlock>(row, lane % kLanes) * 16;
    w_off[i] = w_row_offset<CH, TN, WN, SWIGLU>(p, tn, row) + w_part[i];
  }
  auto copy_w = [&](int kb, int stage) {
#pragma unroll
    for (int i = 0; i < kWCopies; ++i)
      copy_weights16<ONCE>(w_rsrc, base + stage * kStage + TOK * kBlock + (wave + kWaves * i) * 1024,
                 w_part[i] < limit(kb) ? w_off[i] : kTileOob, (kb > last ? 0 : place(kb) * kBlock));
  };
  auto copy_x = [&](int kb, int stage) {
#pragma unroll
    for (int i = 0; i < kXCopies; ++i)
      lds_copy16(x_rsrc, base + stage * kStage + (wave + kWaves * i) % kXGroups * 1024,
                 x_part[i] < limit(kb) ? x_off[i] : kTileOob, (kb > last ? 0 : place(kb) * kBlock));
  };
  // the first weights do not wait for the rows' ids
#pragma unroll
  for (int s = 0; s < S - 1; ++s) copy_w(s, s);
  rows.template fill<GROUPED>(p, first, valid);
  __syncthreads();
  valid = rows.rows();
#pragma unroll
  for (int i = 0; i < kXCopies; ++i) {
    const int row = (wave + kWaves * i) % kXGroups * kRowsPerCopy + lane / kLanes;
    x_part[i] = lds_part<kBlock>(row, lane % kLanes) * 16;
    x_off[i] = x_row_offset<GROUPED>(p, rows.id[row]) + x_part[i];
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) copy_x(s, s);

  typename Op::Acc acc[TN][TM];
#pragma unroll
  for (int r = 0; r < TN; ++r)
#pragma unroll
    for (int c = 0; c < TM; ++c) acc[r][c] = Op::zero();

  // the columns of this wavefront that hold rows
  const int columns = (valid + 15) >> 4;
  const int mine = columns > wm ? (columns - wm + WM - 1) / WM : 0;
  const int part0 = lds_part<kBlock>(n16, wk * 8 + j) * 16, part1 = lds_part<kBlock>(n16, wk * 8 + 4 + j) * 16;

  int stage = 0;
  for (int kb = 0; kb < kblocks; ++kb) {
    // this wavefront's copies of block kb have landed (the first S - 1 blocks' weights were
    // copied ahead of their rows)
    if (kb < S - 2) lds_dma_wait_keep<(S - 2) * kXCopies>();
    else lds_dma_wait_keep<(S - 2) * kCopies>();
    __syncthreads();  // ... and everyone's; block kb - 1 has been read by all
    const int refill = stage == 0 ? S - 1 : stage - 1;
    copy_x(kb + S - 1, refill);
    copy_w(kb + S - 1, refill);
    const uint8_t* xs = &ring[stage * kStage];
    const uint8_t* ws = xs + TOK * kBlock;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int part = d == 0 ? part0 : part1;
      u32x4 wf[TN];
#pragma unroll
      for (int r = 0; r < TN; ++r) wf[r] = load16(ws + ((wn * TN + r) * 16 + n16) * kBlock + part);
#pragma unroll
      for (int c = 0; c < TM; ++c) {
        if (c >= mine) continue;
        const u32x4 xf = load16(xs + ((c * WM + wm) * 16 + n16) * kBlock + part);
#pragma unroll
        for (int r = 0; r < TN; ++r) acc[r][c] = Op::mfma(wf[r], xf, acc[r][c]);
      }
    }
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  lds_dma_wait_all();
  __syncthreads();  // every wavefront has read its last fragments and its copies have landed

  if constexpr (WK > 1) {
    typedef typename Op::Acc Acc;
    Acc* partial = reinterpret_cast<Acc*>(ring);
    if (wk > 0) {
#pragma unroll
      for (int r = 0; r < TN; ++r)
#pragma unroll
        for (int c = 0; c < TM; ++c) partial[((wave - WM * WN) * TN * TM + r * TM + c) * 64 + lane] = acc[r][c];
    }
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int k = 0; k < WK - 1; ++k)
#pragma unroll
        for (int r = 0; r < TN; ++r)
#pragma unroll
          for (int c = 0; c < TM; ++c)
            acc[r][c] += partial[((k * WM * WN + wave) * TN * TM + r * TM + c) * 64 + lane];
    }
    __syncthreads();  // before the output tile takes their place
  }
  store_tile<Op, TOK, TM, TN, WM, WN, WK, GROUPED, SWIGLU>(p, acc, ring, rows, tm, tn, expert);
}

}  // namespace dsv4

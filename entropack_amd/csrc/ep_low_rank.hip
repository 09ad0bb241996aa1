// Low-rank adapters of many requests beside a shared product: out[t] = y[t] + scale[a] (x[t] down[a]^T) up[a]^T.
//
//   shrink   planes[p] = scale[a] x[order[p]] . down[a]^T      grouped_stream_kernel (ep_grouped.hpp), bound by reading x
//   expand   out[order[p]] = y[order[p]] + planes[p] . up[a]^T   low_rank_expand_kernel, bound by reading y and writing out
//   reduce   sum_p planes[p]^T q[order[p]]                     low_rank_reduce_kernel, low_rank_finish_kernel: the gradients of down (q = x, planes of the
//                                                              output's gradient) and of up (q = the output's gradient)
// The narrow rows in between ("planes") are kept as three bf16 parts that add up to the f32 value exactly, so that the second product runs on
// the bf16 matrix cores and loses nothing, also where y and the update cancel. (Two parts are off by up to 2^-16 of the value, which
// the output's rounding hides only where nothing cancels.) A rank's three parts meet the same element of the other operand.
#include "ep_grouped_tile.hpp"

namespace ep {

struct LowRankArgs {
  const uint16_t* planes;          // [entries][4 padded]: for every 16 ranks 16 values, 16 remainders, 16 last parts, 16 zeros
  const uint16_t* up;              // [groups][N][rank]
  const uint16_t* y;               // [rows][N], or null for zero
  uint16_t* out;
  const int32_t* order;
  const int32_t* offsets;
  int64_t ldu, up_group, ldy, ldo;
  int entries, groups, rank, padded, N, rows;
};

// 8 consecutive elements of a row of `up` from element e on; elements from `rank` on are zero. PIECES: rank, ldu and the
// address allow 16-byte loads.
template <bool PIECES>
__device__ __forceinline__ uint4 up_piece(const uint16_t* __restrict__ row, int e, int rank) {
  if constexpr (PIECES) {
    // No branch around the load: one per load would serialise them.
    const uint4 v = *reinterpret_cast<const uint4*>(row + (e < rank ? e : 0));
    const uint32_t keep = e < rank ? ~0u : 0u;
    return make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
  } else {
    uint32_t word[4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < rank) word[i >> 1] |= static_cast<uint32_t>(row[e + i]) << (16 * (i & 1));
    return make_uint4(word[0], word[1], word[2], word[3]);
  }
}

// Eight bf16 plus eight sums, each rounded once.
__device__ __forceinline__ uint4 add_to_pieces(uint4 in, const f32x4& first, const f32x4& second) {
  uint32_t word[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4& four = i < 2 ? first : second;
    const float low = __uint_as_float(word[i] << 16) + four[2 * (i & 1)];
    const float high = __uint_as_float(word[i] & 0xFFFF0000u) + four[2 * (i & 1) + 1];
    word[i] = bf16_bits_of(low) | bf16_bits_of(high) << 16;
  }
  return make_uint4(word[0], word[1], word[2], word[3]);
}

// Few rows per adapter: a block takes 16 rows of one adapter and 256 columns, a wave 64 of them. The matrix cores are given the rows
// of `up` as the left operand, ordered so that a lane ends up with two runs of 8 consecutive columns of its row (row m of tile j
// is column 32 (j / 2) + 8 (m / 4) + 4 (j % 2) + m % 4 of the 64). The inner dimension is [value | remainder] and [last part | zeros] of
// 16 ranks, all against the same `up`. There is no LDS and nothing to wait for but the loads: 61 rows of 48 adapters take 3.6 us.
template <bool PIECES, bool WIDE>
__global__ __launch_bounds__(256) void low_rank_expand_kernel(LowRankArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column_tiles = (a.N + 255) / 256;
  const RowTile tile = find_row_tile(a.offsets, a.groups, a.entries, static_cast<int>(blockIdx.x / column_tiles), 16);
  if (tile.group < 0) return;
  const int n0 = static_cast<int>(blockIdx.x % column_tiles) * 256 + wave * 64;
  if (n0 >= a.N) return;
  const int in_row = lane & 15, quarter = lane >> 4;
  const int at = in_row < tile.rows ? a.order[tile.first + in_row] : -1;
  const int64_t to = at < a.rows ? at : -1;
  const int n = n0 + 8 * quarter;
  uint4 in[2];                                               // y is requested before anything else
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    in[h] = make_uint4(0, 0, 0, 0);
    if (WIDE && a.y != nullptr && to >= 0 && n + 32 * h < a.N) in[h] = *reinterpret_cast<const uint4*>(a.y + to * a.ldy + n + 32 * h);
  }
  f32x4 acc[4] = {};
  if (tile.group < a.groups) {
    const uint16_t* planes = a.planes + (static_cast<int64_t>(tile.first) + (in_row < tile.rows ? in_row : tile.rows - 1)) * (4 * a.padded) + 8 * quarter;
    const uint16_t* up[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = n0 + 32 * (j >> 1) + 8 * (in_row >> 2) + 4 * (j & 1) + (in_row & 3);
      up[j] = a.up + tile.group * a.up_group + (row < a.N ? row : a.N - 1) * a.ldu;
    }
    for (int e0 = 0; e0 < a.padded; e0 += 16) {
      const bf16x8 fp = *reinterpret_cast<const bf16x8*>(planes + 4 * e0);
      const bf16x8 last = *reinterpret_cast<const bf16x8*>(planes + 4 * e0 + 32);
      bf16x8 fu[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) fu[j] = __builtin_bit_cast(bf16x8, up_piece<PIECES>(up[j], e0 + 8 * (quarter & 1), a.rank));
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fu[j], last, acc[j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fu[j], fp, acc[j], 0, 0, 0);
    }
  }
  if (to < 0) return;
  // Column n + 32 (j / 2) + 4 (j % 2) + i is in register i of tile j.
  uint16_t* out = a.out + to * a.ldo + n;
  if constexpr (WIDE) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (n + 32 * h >= a.N) continue;
      *reinterpret_cast<uint4*>(out + 32 * h) = add_to_pieces(in[h], acc[2 * h], acc[2 * h + 1]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const int column = 32 * (c >> 3) + (c & 7);
      if (n + column >= a.N) continue;
      const float v = a.y != nullptr ? __uint_as_float(static_cast<uint32_t>(a.y[to * a.ldy + n + column]) << 16) : 0.0f;
      out[column] = static_cast<uint16_t>(bf16_bits_of(v + acc[c >> 2][c & 3]));
    }
  }
}

// Many rows per adapter: bound by reading y and writing out. A block takes 64 rows of one adapter, 16 per wave, and 128 columns.
// Memory wants neighbouring lanes at neighbouring addresses (a load whose lanes are on sixteen rows, as the fragments of the kernel
// above are, occupies the address path four times as long). So `up` goes through LDS,
// STEP ranks at a time, fetched once for all 64 rows, and the planes are the left operand: lane l then holds, over the eight
// 16-column tiles (row m of tile j is column 8 m + j), 8 consecutive columns 8 (l % 16) .. of rows 4 (l / 16) + i: sixteen lanes
// read and write 256 consecutive bytes of a row. Small blocks, so that many are resident and the last round is short (256 columns per block
// took a fifth more, 512 columns 30 %). The narrow rows' fragments are asked for with `up`, before the barrier, so that both arrive
// together: 7993 rows of 4096, rank 32, 26.6 us, 31.8 with the fragments loaded where they are used (131 MB, 21 us at the rate of a large
// read and write; a part of y comes from the last-level cache where a call is repeated).
// STEP: the least of 16, 32 and 64 that the rank fits, 64 beyond.
constexpr int kTallColumns = 128;

template <bool PIECES, bool WIDE, int STEP>
__global__ __launch_bounds__(256) void low_rank_expand_tall_kernel(LowRankArgs a) {
  constexpr int kPieces = STEP / 8, kMoves = kTallColumns * kPieces / 256;
  constexpr int kPitch = STEP * 2 + 16;                      // bytes per column of `up`: an odd number of 16-byte pieces, all banks
  __shared__ __align__(16) uint8_t up_tile[kTallColumns * kPitch];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int column_tiles = (a.N + kTallColumns - 1) / kTallColumns;
  const RowTile tile = find_row_tile(a.offsets, a.groups, a.entries, static_cast<int>(blockIdx.x / column_tiles), 64);
  if (tile.group < 0) return;
  const int first_column = static_cast<int>(blockIdx.x % column_tiles) * kTallColumns;
  const int in_row = lane & 15, quarter = lane >> 4, n = first_column + 8 * in_row;
  const bool grouped = tile.group < a.groups;
  int64_t to[4];                                             // rows 16 wave + 4 quarter + i
  uint4 in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 16 * wave + 4 * quarter + i;
    const int at = row < tile.rows ? a.order[tile.first + row] : -1;
    to[i] = at < a.rows ? at : -1;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    in[i] = make_uint4(0, 0, 0, 0);
    if (WIDE && a.y != nullptr && to[i] >= 0 && n < a.N) in[i] = *reinterpret_cast<const uint4*>(a.y + to[i] * a.ldy + n);
  }
  f32x4 acc[8] = {};
  if (grouped) {
    const int plane_row = 16 * wave + in_row < tile.rows ? 16 * wave + in_row : tile.rows - 1;
    const uint16_t* planes = a.planes + (static_cast<int64_t>(tile.first) + plane_row) * (4 * a.padded) + 8 * quarter;
    const uint16_t* up = a.up + tile.group * a.up_group;
    for (int rank0 = 0; rank0 < a.padded; rank0 += STEP) {
      uint4 moved[kMoves];
#pragma unroll
      for (int m = 0; m < kMoves; ++m) {
        const int cell = tid + 256 * m, column = first_column + cell / kPieces;
        moved[m] = up_piece<PIECES>(up + (column < a.N ? column : a.N - 1) * a.ldu, rank0 + 8 * (cell % kPieces), a.rank);
      }
      // 16 ranks each: values and remainders (quarters 0, 1 and 2, 3), then last parts and zeros. Asked for with `up`; past the end the first again.
      const int ranks = a.padded - rank0 < STEP ? a.padded - rank0 : STEP;
      bf16x8 narrow[STEP / 16][2];
#pragma unroll
      for (int i = 0; i < STEP / 16; ++i) {
        const uint16_t* from = planes + 4 * (rank0 + (16 * i < ranks ? 16 * i : 0));
        narrow[i][0] = *reinterpret_cast<const bf16x8*>(from);
        narrow[i][1] = *reinterpret_cast<const bf16x8*>(from + 32);
      }
      if (rank0 > 0) __syncthreads();                        // the stretch before has been read
#pragma unroll
      for (int m = 0; m < kMoves; ++m) {
        const int cell = tid + 256 * m, column = cell / kPieces;                  // column 8 m + j lies at 16 j + m
        *reinterpret_cast<uint4*>(up_tile + ((column & 7) * 16 + (column >> 3)) * kPitch + 16 * (cell % kPieces)) = moved[m];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < STEP / 16; ++i) {
        if (16 * i >= ranks) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bf16x8 fu = *reinterpret_cast<const bf16x8*>(up_tile + (16 * j + in_row) * kPitch + 2 * (16 * i + 8 * (quarter & 1)));
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(narrow[i][1], fu, acc[j], 0, 0, 0);
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(narrow[i][0], fu, acc[j], 0, 0, 0);
        }
      }
    }
  }
  // Row 4 quarter + i, column n + j is in register i of tile j.
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (to[i] < 0) continue;
    uint16_t* out = a.out + to[i] * a.ldo + n;
    const f32x4 low = {acc[0][i], acc[1][i], acc[2][i], acc[3][i]}, high = {acc[4][i], acc[5][i], acc[6][i], acc[7][i]};
    if constexpr (WIDE) {
      if (n < a.N) *reinterpret_cast<uint4*>(out) = add_to_pieces(in[i], low, high);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (n + j >= a.N) continue;
        const float v = a.y != nullptr ? __uint_as_float(static_cast<uint32_t>(a.y[to[i] * a.ldy + n + j]) << 16) : 0.0f;
        out[j] = static_cast<uint16_t>(bf16_bits_of(v + (j < 4 ? low[j & 3] : high[j & 3])));
      }
    }
  }
}

// sum over a group's places of planes[p][e] q[order[p]][n] for all e < rank: out[g][e][n], or out[g][n][e] when
// transposed. The products are the weights' gradient of ep_grouped_tile.hpp with the planes as left operand, the three parts' sums folded
// into one where the tile is stored. They are bound by
// reading q, and the groups alone make too few tiles to fill the card, so the places of every group are divided into chunks, each
// chunk writes its f32 sums to a matrix of its own, and this kernel adds a group's chunks in their order and rounds once.
// A block takes 64 columns and 16 ranks of one group, a wave one of the ranks; bound by the latency of its loads: both gradients of 4
// adapters of rank 16, 4099 rows of 4096, 5.2 us (4 waves with four ranks each take twice as long). One launch sums both gradients, as one launch of tiles makes their parts:
// the blocks of the first before those of the second.
struct Finish {
  const float* parts;
  uint16_t* out;
  int width, transposed;
};

__global__ __launch_bounds__(1024) void low_rank_finish_kernel(Finish of_first, Finish of_second, int first_blocks, int chunk, int padded, int rank,
                                                               const int32_t* __restrict__ offsets) {
  __shared__ uint16_t turned[64][18];
  const bool second = static_cast<int>(blockIdx.x) >= first_blocks;
  const Finish f = second ? of_second : of_first;
  const int block = static_cast<int>(blockIdx.x) - (second ? first_blocks : 0), width = f.width;
  const int column_tiles = (width + 63) / 64, rank_tiles = padded / 16;
  const int at = block / column_tiles, n0 = block % column_tiles * 64;
  const int group = at / rank_tiles, e0 = at % rank_tiles * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // The chunks of the groups before this one, and this one's.
  int before = 0;
  for (int g = lane; g < group; g += 64) before += (offsets[g + 1] - offsets[g] + chunk - 1) / chunk;
  before = __builtin_amdgcn_readlane(wave_inclusive_sum(before), 63);
  const int chunks = (offsets[group + 1] - offsets[group] + chunk - 1) / chunk;
  const int64_t matrix = static_cast<int64_t>(padded) * width;
  const int n = n0 + lane, e = e0 + wave;
  float sum = 0.0f;
  if (n < width) {
    const float* from = f.parts + before * matrix + static_cast<int64_t>(e) * width + n;
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) sum += from[c * matrix];
  }
  const uint16_t bits = static_cast<uint16_t>(bf16_bits_of(sum));
  if (!f.transposed) {
    if (n < width && e < rank) f.out[(static_cast<int64_t>(group) * rank + e) * width + n] = bits;
    return;
  }
  turned[lane][wave] = bits;
  __syncthreads();
  const int column = n0 + (threadIdx.x >> 4), of = e0 + (threadIdx.x & 15);
  if (column < width && of < rank) f.out[(static_cast<int64_t>(group) * width + column) * rank + of] = turned[threadIdx.x >> 4][threadIdx.x & 15];
}

// The parts of both gradients, tiles of 128 x 128: the blocks of the first before those of the second. 4 adapters of rank 16, 4099 rows
// of 4096 on either side, 20 us (reading both sides takes 11). Ranks to 32 fit one tile of rows; rank 64 takes two, each of which reads the other
// operand: 2 adapters, 20000 rows of 8192, 222 us (reading both sides 106).
__global__ __launch_bounds__(kTileThreads, 2) void low_rank_reduce_kernel(TileArgs of_first, TileArgs of_second, int first_blocks) {
  __shared__ __align__(1024) uint8_t stage0[2 * kTile * 128];
  __shared__ __align__(1024) uint8_t stage1[2 * kTile * 128];
  __shared__ int32_t row_at[kTile];
  __shared__ float scale_at[kTile];
  const bool second = static_cast<int>(blockIdx.x) >= first_blocks;
  const TileArgs g = second ? of_second : of_first;
  BlockTile tile;
  if (!find_block_tile<kGradWeight>(g, static_cast<int>(blockIdx.x) - (second ? first_blocks : 0), kTile, tile)) return;
  compute_tile<false, kGradWeight, true, true, kTile, kTile, true>(g, tile, stage0, stage1, row_at, scale_at);
}

// Both transposes that the gradients need, [groups][rows][columns] to [groups][columns][out_rows] with zeros in rows .. out_rows: 64 x 64
// blocks by way of LDS, those of the first matrix before those of the second. Latency: four adapters of rank 16 and 4096 features
// 4.3 us in one launch (two of torch's, 6 us each).
struct Transpose {
  const uint16_t* in;
  uint16_t* out;
  int64_t ld, group;
  int rows, columns, out_rows;
  int row_tiles, column_tiles;     // of 64; rows counted to out_rows
};

__global__ __launch_bounds__(256) void low_rank_transpose_kernel(Transpose first, Transpose second, int first_blocks) {
  __shared__ uint16_t turned[64][66];
  const bool of_first = static_cast<int>(blockIdx.x) < first_blocks;
  const Transpose t = of_first ? first : second;
  const int block = static_cast<int>(blockIdx.x) - (of_first ? 0 : first_blocks);
  const int column0 = block % t.column_tiles * 64, row0 = block / t.column_tiles % t.row_tiles * 64;
  const int64_t group = block / t.column_tiles / t.row_tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column = column0 + lane;
  const uint16_t* in = t.in + group * t.group + (column < t.columns ? column : 0);
  uint16_t held[16];                             // all loads before the first is used; those outside read row or column 0
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = row0 + 4 * i + wave;
    held[i] = in[(row < t.rows ? row : 0) * t.ld];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = row0 + 4 * i + wave;
    turned[lane][4 * i + wave] = row < t.rows && column < t.columns ? held[i] : 0;
  }
  __syncthreads();
  uint16_t* out = t.out + group * t.columns * t.out_rows;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int turned_row = column0 + 4 * i + wave, at = row0 + lane;
    if (turned_row < t.columns && at < t.out_rows) out[static_cast<int64_t>(turned_row) * t.out_rows + at] = turned[4 * i + wave][lane];
  }
}

// Places per chunk: about 1024 tiles in all, both gradients', at least 128 places each (a chunk of fewer does not outlast its own prologue).
static int reduce_chunk(int64_t entries, int64_t rank, int64_t K, int64_t N) {
  const int64_t tiles = ((K + kTile - 1) / kTile + (N + kTile - 1) / kTile) * (((rank + 15) / 16 * 64 + kTile - 1) / kTile);
  const int64_t chunks = tiles >= 1024 ? 1 : 1024 / tiles;
  int64_t chunk = (entries + chunks - 1) / chunks;
  chunk = chunk < 128 ? 128 : (chunk + 63) / 64 * 64;
  return static_cast<int>(chunk < (1 << 30) ? chunk : 1 << 30);
}

static int padded_rank(int64_t rank) { return static_cast<int>((rank + 15) / 16 * 16); }
static int64_t whole_pieces(int64_t elements) { return (elements + 7) / 8 * 8; }
static size_t whole_lines(size_t bytes) { return (bytes + 255) / 256 * 256; }
static size_t planes_bytes(int64_t entries, int64_t rank) { return static_cast<size_t>(entries) * static_cast<size_t>(padded_rank(rank)) * 8; }

// The adapters and the rows they are for.
struct Grouping {
  const int32_t* order;
  const int32_t* offsets;
  int64_t entries;
  int groups;
};

// planes[p] = scale[a] x[order[p]] . down[a]^T; K a whole number of pieces.
static int shrink(const Grouping& g, const void* x, int64_t ldx, const void* down, int64_t ldd, int64_t down_group, const float* scale, void* planes, int64_t rank, int64_t K,
                  hipStream_t s) {
  GroupedArgs a = {};
  a.x = static_cast<const uint8_t*>(x), a.w = static_cast<const uint8_t*>(down), a.scale_x = scale, a.y = planes, a.row_of = g.order, a.offsets = g.offsets;
  a.ldx_bytes = ldx * 2, a.ldw_bytes = ldd * 2, a.group_bytes = down_group * 2, a.k_bytes = K * 2, a.ldy = 4 * padded_rank(rank);
  a.entries = static_cast<int>(g.entries), a.groups = g.groups, a.N = static_cast<int>(rank), a.x_rows = static_cast<int>(g.entries), a.out_kind = kOutBF16;
  // All of a rank up to 64 in one block, so that x is read once. 4099 rows of 4096: rank 16 9.0 us (8 waves 10.5; 500 rows 6.0 against
  // 5.4), rank 64 16.1 us (32 ranks per block 19.2); 7993 rows, rank 32, 18.5 us (16 rows per block 19.6,
  // 48 rows on 6 waves, which need one round of blocks instead of two, 19.8; reading x takes 10.6).
  if (rank > 32) return launch_stream_of<false, 2, 4, 4, true>(a, s);
  if (rank > 16) return launch_stream_of<false, 2, 2, 8, true>(a, s);
  return g.entries >= 2048 ? launch_stream_of<false, 1, 1, 4, true>(a, s) : launch_stream_of<false, 1, 1, 8, true>(a, s);
}

// out[order[p]] = y[order[p]] + planes[p] . up[a]^T, rows of no group as in y.
static int expand(const Grouping& g, const void* planes, const void* up, int64_t ldu, int64_t up_group, const void* y, int64_t ldy, void* out, int64_t ldo, int64_t rank,
                  int64_t N, hipStream_t s) {
  LowRankArgs a = {};
  a.planes = static_cast<const uint16_t*>(planes), a.up = static_cast<const uint16_t*>(up), a.y = static_cast<const uint16_t*>(y);
  a.out = static_cast<uint16_t*>(out), a.order = g.order, a.offsets = g.offsets;
  a.ldu = ldu, a.up_group = up_group, a.ldy = ldy, a.ldo = ldo;
  a.entries = static_cast<int>(g.entries), a.groups = g.groups, a.rank = static_cast<int>(rank), a.padded = padded_rank(rank), a.N = static_cast<int>(N);
  a.rows = static_cast<int>(g.entries);
  auto in_pieces = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool pieces = in_pieces(up, ldu) && up_group % 8 == 0 && rank % 8 == 0;
  const bool wide = in_pieces(out, ldo) && N % 8 == 0 && (y == nullptr || in_pieces(y, ldy));
  const bool tall = g.entries / g.groups >= 32;              // most blocks of 64 rows are then at least half full
  const int columns = tall ? kTallColumns : 256;
  const int64_t blocks = most_row_tiles(g.entries, g.groups, tall ? 64 : 16) * ((N + columns - 1) / columns);
  if (!launch_fits(blocks, 256)) return EP_HIP_EUNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
#define EP_EXPAND(PIECES, WIDE)                                                                                               \
  if (!tall) hipLaunchKernelGGL((low_rank_expand_kernel<PIECES, WIDE>), grid, dim3(256), 0, s, a);                             \
  else if (a.padded <= 16) hipLaunchKernelGGL((low_rank_expand_tall_kernel<PIECES, WIDE, 16>), grid, dim3(256), 0, s, a);      \
  else if (a.padded <= 32) hipLaunchKernelGGL((low_rank_expand_tall_kernel<PIECES, WIDE, 32>), grid, dim3(256), 0, s, a);      \
  else hipLaunchKernelGGL((low_rank_expand_tall_kernel<PIECES, WIDE, 64>), grid, dim3(256), 0, s, a)
  if (pieces && wide) {
    EP_EXPAND(true, true);
  } else if (pieces) {
    EP_EXPAND(true, false);
  } else if (wide) {
    EP_EXPAND(false, true);
  } else {
    EP_EXPAND(false, false);
  }
#undef EP_EXPAND
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

// The chunks' sums of a gradient of so many columns.
static size_t reduce_bytes(int64_t entries, int groups, int64_t rank, int chunk, int64_t width) {
  return static_cast<size_t>(most_chunks(entries, groups, chunk)) * static_cast<size_t>(padded_rank(rank)) * static_cast<size_t>(width) * 4;
}

// out[a][e][n] (transposed: out[a][n][e]) = sum over a's places of planes[p][e] q[order[p]][n]; rows of q readable to a whole number of pieces.
struct Reduction {
  const void* planes;
  const void* q;
  int64_t ldq, width;
  void* out;
  bool transposed;
  void* parts;
};

// One or two of them.
static int reduce(const Grouping& g, int64_t rank, int chunk, const Reduction* all, int count, hipStream_t s) {
  const int padded = padded_rank(rank);
  TileArgs tiles[2] = {};
  Finish sums[2] = {};
  int64_t blocks[2] = {}, finish[2] = {};
  for (int i = 0; i < count; ++i) {
    const Reduction& r = all[i];
    TileArgs& t = tiles[i];
    t.a = static_cast<const uint8_t*>(r.planes), t.b = static_cast<const uint8_t*>(r.q), t.y = r.parts, t.row_of = g.order, t.offsets = g.offsets;
    t.lda_bytes = padded * int64_t{8}, t.ldb_bytes = r.ldq * 2, t.ldy = r.width, t.group_y = padded * r.width;
    t.entries = static_cast<int>(g.entries), t.groups = g.groups, t.x_rows = static_cast<int>(g.entries), t.out_kind = kOutF32;
    t.rows = 4 * padded, t.columns = static_cast<int>(r.width), t.chunk = chunk;
    sums[i] = {static_cast<const float*>(r.parts), static_cast<uint16_t*>(r.out), static_cast<int>(r.width), r.transposed ? 1 : 0};
    blocks[i] = most_chunks(g.entries, g.groups, chunk) * ((t.rows + kTile - 1) / kTile) * ((r.width + kTile - 1) / kTile);
    finish[i] = static_cast<int64_t>(g.groups) * (padded / 16) * ((r.width + 63) / 64);
  }
  if (!launch_fits(blocks[0] + blocks[1], kTileThreads) || !launch_fits(finish[0] + finish[1], 1024)) return EP_HIP_EUNSUPPORTED;
  hipLaunchKernelGGL(low_rank_reduce_kernel, dim3(static_cast<unsigned>(blocks[0] + blocks[1])), dim3(kTileThreads), 0, s, tiles[0], tiles[1], static_cast<int>(blocks[0]));
  EP_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(low_rank_finish_kernel, dim3(static_cast<unsigned>(finish[0] + finish[1])), dim3(1024), 0, s, sums[0], sums[1], static_cast<int>(finish[0]), chunk, padded,
                     static_cast<int>(rank), g.offsets);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

// Which gradients a call gives.
enum : int { kWantX = 1, kWantDown = 2, kWantUp = 4, kWantAll = 7 };

// Where they keep what lies between their products, each part only where a gradient asked for reads it: the transpose of up and the
// planes of the output's gradient (of x and of down), the transpose of down (of x), the chunks' sums (of down, of up). The chunks' sums
// are f32 matrices, one per chunk, and a group with places has a chunk at least: up to twice the gradients' own size for a bank whose
// adapters all have rows. The chunks do not depend on what is asked for, so neither do the sums' values.
struct GradRoom {
  size_t up_turned, down_turned, planes, down_parts, up_parts, bytes;
  int chunk;
};

static GradRoom grad_room(int64_t entries, int groups, int64_t rank, int64_t K, int64_t N, int wanted) {
  GradRoom r = {};
  const size_t g = static_cast<size_t>(groups);
  size_t end = 0;
  auto take = [&](bool needed, size_t bytes) {
    const size_t at = end;
    if (needed) end += whole_lines(bytes);
    return at;
  };
  const bool back = (wanted & (kWantX | kWantDown)) != 0;
  r.chunk = reduce_chunk(entries, rank, K, N);
  r.up_turned = take(back, g * static_cast<size_t>(rank * whole_pieces(N)) * 2);                       // [groups][rank][whole pieces of N]
  r.down_turned = take((wanted & kWantX) != 0, g * static_cast<size_t>(K * whole_pieces(rank)) * 2);     // [groups][K][whole pieces of rank]
  r.planes = take(back, planes_bytes(entries, rank));
  r.down_parts = take((wanted & kWantDown) != 0, reduce_bytes(entries, groups, rank, r.chunk, K));
  r.up_parts = take((wanted & kWantUp) != 0, reduce_bytes(entries, groups, rank, r.chunk, N));
  r.bytes = end;
  return r;
}

static bool low_rank_valid(const Grouping& g, int64_t rank, int64_t K, int64_t N) {
  return g.order != nullptr && g.offsets != nullptr && g.entries > 0 && g.entries <= kMostEntries && g.groups > 0 && rank > 0 && rank <= 4096 && K > 0 && N > 0 &&
         K <= 0x3FFFFF00 / g.groups && N <= 0x3FFFFF00 / g.groups;
}

// The rows that one launch of the shrink takes, 16 per block of 256 threads: fewer than 2^28.
static bool rows_fit(int64_t entries, int groups) { return launch_fits(most_row_tiles(entries, groups, 16), 256); }

// Rows read in whole 16-byte pieces, the last one zero from `width` on.
static bool rows_in_pieces(const void* base, int64_t ld, int64_t width) {
  return base != nullptr && reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld % 8 == 0 && ld >= whole_pieces(width);
}

}  // namespace ep

extern "C" {

size_t ep_hip_low_rank_planes_bytes(int64_t entries, int64_t rank) { return entries <= 0 || rank <= 0 ? 0 : ep::planes_bytes(entries, rank); }

int ep_hip_low_rank_update(const void* x_dev, int64_t ldx, const void* down_dev, int64_t ldd, int64_t down_group, const void* up_dev, int64_t ldu, int64_t up_group,
                           const float* scale_dev, const void* y_dev, int64_t ldy, void* planes_dev, void* out_dev, int64_t ldo, const int32_t* order_dev,
                           const int32_t* offsets_dev, int64_t entries, int groups, int64_t rank, int64_t K, int64_t N, void* stream) {
  using namespace ep;
  const Grouping g = {order_dev, offsets_dev, entries, groups};
  if (!low_rank_valid(g, rank, K, N) || planes_dev == nullptr || reinterpret_cast<uintptr_t>(planes_dev) % 16 != 0) return EP_HIP_EINVAL;
  if (!rows_in_pieces(x_dev, ldx, K) || !rows_in_pieces(down_dev, ldd, K) || down_group % 8 != 0 || down_group < 0) return EP_HIP_EINVAL;
  if (up_dev == nullptr || out_dev == nullptr || ldu < rank || up_group < 0 || ldo < N || (y_dev != nullptr && ldy < N)) return EP_HIP_EINVAL;
  if (!rows_fit(entries, groups)) return EP_HIP_EUNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int status = shrink(g, x_dev, ldx, down_dev, ldd, down_group, scale_dev, planes_dev, rank, whole_pieces(K), s);
  return status != EP_HIP_OK ? status : expand(g, planes_dev, up_dev, ldu, up_group, y_dev, ldy, out_dev, ldo, rank, N, s);
}

size_t ep_hip_low_rank_grad_workspace(int64_t entries, int groups, int64_t rank, int64_t K, int64_t N) {
  if (entries <= 0 || groups <= 0 || rank <= 0 || K <= 0 || N <= 0) return 0;
  return ep::grad_room(entries, groups, rank, K, N, ep::kWantAll).bytes;
}

size_t ep_hip_low_rank_grad_workspace_for(int64_t entries, int groups, int64_t rank, int64_t K, int64_t N, int grad_x, int grad_down, int grad_up) {
  using namespace ep;
  if (entries <= 0 || groups <= 0 || rank <= 0 || K <= 0 || N <= 0) return 0;
  return grad_room(entries, groups, rank, K, N, (grad_x != 0 ? kWantX : 0) | (grad_down != 0 ? kWantDown : 0) | (grad_up != 0 ? kWantUp : 0)).bytes;
}

int ep_hip_low_rank_update_grad(const void* grad_dev, int64_t ldg, const void* x_dev, int64_t ldx, const void* down_dev, int64_t ldd, int64_t down_group,
                                const void* up_dev, int64_t ldu, int64_t up_group, const float* scale_dev, const void* planes_dev, void* grad_x_dev, int64_t ldgx,
                                void* grad_down_dev, void* grad_up_dev, const int32_t* order_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t rank,
                                int64_t K, int64_t N, void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace ep;
  const Grouping g = {order_dev, offsets_dev, entries, groups};
  if (!low_rank_valid(g, rank, K, N) || !rows_in_pieces(grad_dev, ldg, N)) return EP_HIP_EINVAL;
  if (grad_x_dev == nullptr && grad_down_dev == nullptr && grad_up_dev == nullptr) return EP_HIP_EINVAL;
  const bool back = grad_x_dev != nullptr || grad_down_dev != nullptr;         // the narrow rows' gradient is needed
  if (back && (up_dev == nullptr || ldu < rank || up_group < 0)) return EP_HIP_EINVAL;
  if (grad_x_dev != nullptr && (down_dev == nullptr || ldd < K || down_group < 0 || ldgx < K)) return EP_HIP_EINVAL;
  if (grad_down_dev != nullptr && !rows_in_pieces(x_dev, ldx, K)) return EP_HIP_EINVAL;
  if (grad_up_dev != nullptr && (planes_dev == nullptr || reinterpret_cast<uintptr_t>(planes_dev) % 16 != 0)) return EP_HIP_EINVAL;
  if (!rows_fit(entries, groups)) return EP_HIP_EUNSUPPORTED;
  const GradRoom room = grad_room(entries, groups, rank, K, N, (grad_x_dev != nullptr ? kWantX : 0) | (grad_down_dev != nullptr ? kWantDown : 0) | (grad_up_dev != nullptr ? kWantUp : 0));
  if (workspace_dev == nullptr || reinterpret_cast<uintptr_t>(workspace_dev) % 256 != 0 || workspace_bytes < room.bytes) return EP_HIP_EINVAL;
  uint8_t* const base = static_cast<uint8_t*>(workspace_dev);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (back) {
    // The gradient of the narrow rows is a shrink by up^T, that of x an expand by down^T.
    auto tiles = [](Transpose& t) { return t.column_tiles = (t.columns + 63) / 64, t.row_tiles = (t.out_rows + 63) / 64, static_cast<int64_t>(t.column_tiles) * t.row_tiles; };
    Transpose up = {static_cast<const uint16_t*>(up_dev), reinterpret_cast<uint16_t*>(base + room.up_turned), ldu, up_group, static_cast<int>(N), static_cast<int>(rank),
                    static_cast<int>(whole_pieces(N)), 0, 0};
    Transpose down = {static_cast<const uint16_t*>(down_dev), reinterpret_cast<uint16_t*>(base + room.down_turned), ldd, down_group, static_cast<int>(rank), static_cast<int>(K),
                      static_cast<int>(whole_pieces(rank)), 0, 0};
    const int64_t first = tiles(up) * groups, second = tiles(down) * (grad_x_dev != nullptr ? groups : 0);
    if (!launch_fits(first + second, 256)) return EP_HIP_EUNSUPPORTED;
    hipLaunchKernelGGL(low_rank_transpose_kernel, dim3(static_cast<unsigned>(first + second)), dim3(256), 0, s, up, down, static_cast<int>(first));
    EP_HIP_TRY(hipGetLastError());
    const int64_t turned = whole_pieces(N);
    if (const int status = shrink(g, grad_dev, ldg, base + room.up_turned, turned, rank * turned, scale_dev, base + room.planes, rank, turned, s)) return status;
    if (grad_x_dev != nullptr) {
      const int64_t ranks = whole_pieces(rank);
      if (const int status = expand(g, base + room.planes, base + room.down_turned, ranks, K * ranks, nullptr, 0, grad_x_dev, ldgx, rank, K, s)) return status;
    }
  }
  Reduction wanted[2];
  int count = 0;
  if (grad_down_dev != nullptr) wanted[count++] = {base + room.planes, x_dev, ldx, K, grad_down_dev, false, base + room.down_parts};
  if (grad_up_dev != nullptr) wanted[count++] = {planes_dev, grad_dev, ldg, N, grad_up_dev, true, base + room.up_parts};
  return count != 0 ? reduce(g, rank, room.chunk, wanted, count, s) : EP_HIP_OK;
}

}  // extern "C"

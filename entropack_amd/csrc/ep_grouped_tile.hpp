// The 128 x 128 block tile of the products on grouped rows: forward (bf16, int8), gradient of the rows, gradient of the weights.
//
// All three are sums over an inner index of a left and a right operand; they differ in which index of each operand lies
// contiguous in memory. A "row" operand (x, w in the forward, dy in the rows' gradient) has the inner index contiguous, which
// is the shape of a matrix-core fragment; its tile is 128 rows of 128 bytes. A "column" operand (w in the rows' gradient; dy
// and x in the weights') has its outer index contiguous; its tile is 64 inner rows of 256 bytes, and the fragments are taken
// from LDS with the transposing reads (ds_read_b64_tr_b16: 16 lanes read a 4 x 16 block of two-byte elements and each
// receives a column of four).
//
// Tiles go from memory straight into LDS (global_load_lds_dwordx4, 1 KiB per wave and instruction) in two stages; the K loop
// is written out for both so that the compiler waits for loads in flight only at the barrier that publishes a stage. LDS rows
// cannot be padded then, so the 16-byte pieces of a row are permuted, piece c of row r at place c ^ ((r >> 1) & 7) (row
// operand: sixteen rows read at one logical piece cover all banks) or c ^ ((r & 3) << 2) (column operand: the four inner rows
// of a transposing read cover all banks). Two blocks of four waves (64 x 64 each) share a CU, so that one block's barrier and
// epilogue hide behind the other's products.
//
// Ends: a lane whose piece lies past the operand's end loads a piece of zeros instead, so any inner length is exact, whatever
// lies in memory behind it; rows past the tile's last repeat it and are dropped when the tile is stored.
#pragma once

#include "ep_grouped.hpp"

namespace ep {

__device__ __align__(16) const uint32_t kZeroPiece[4] = {0, 0, 0, 0};

// Workgroups go to the eight XCDs round-robin in launch order, and each XCD has its own L2. The tiles of the output are taken in
// parts of `kPartRows` row tiles by `part_columns` column tiles, as many as an XCD holds blocks at a time (one on each of its 32
// CUs), and every XCD works through parts of its own: its blocks then share the operand tiles they stream.
constexpr int kPartRows = 8, kPartColumns = 4, kXcds = 8;

struct TileOrder {
  int column_tiles, part_columns, parts_across;
};

inline TileOrder tile_order(int64_t columns, int tile) {
  TileOrder o;
  o.column_tiles = static_cast<int>((columns + tile - 1) / tile);
  o.parts_across = (o.column_tiles + kPartColumns - 1) / kPartColumns;
  o.part_columns = (o.column_tiles + o.parts_across - 1) / o.parts_across;
  return o;
}

inline int64_t tile_blocks(const TileOrder& o, int64_t row_tiles) {
  const int64_t parts = (row_tiles + kPartRows - 1) / kPartRows * o.parts_across;
  return (parts + kXcds - 1) / kXcds * kXcds * kPartRows * o.part_columns;
}

// Row tile and column tile of this block; a column tile from column_tiles on has no work.
__device__ __forceinline__ void tile_of_block(const TileOrder& o, int& row_tile, int& column_tile) {
  const int block = static_cast<int>(blockIdx.x), xcd = block % kXcds, at = block / kXcds;
  const int size = kPartRows * o.part_columns;
  const int part = at / size * kXcds + xcd, within = at % size;
  row_tile = part / o.parts_across * kPartRows + within % kPartRows;
  column_tile = part % o.parts_across * o.part_columns + within / kPartRows;
}

struct TileArgs {
  const uint8_t* a;                // left operand
  const uint8_t* b;                // right operand
  const float* scale_x;            // int8 forward: per row of a, per row of every b
  const float* scale_w;
  const void* bias;                // forward: [groups][columns], in the output's type
  void* y;
  const int32_t* row_of;           // forward: place p reads row row_of[p] of a; weights' gradient: of b (null: row p)
  const int32_t* order;            // rows' gradient: place p is written to row order[p] of y (null: row p)
  const int32_t* offsets;
  int64_t lda_bytes, ldb_bytes, group_b_bytes, ldy, group_y;
  int entries, groups, x_rows, out_kind;
  int rows;                        // weights' gradient: rows of y (columns of a)
  int columns;                     // columns of y
  int inner;                       // forward, rows' gradient: the inner length in bytes of the row operand
  TileOrder tiles;                 // 256 x 256 tiles
};

enum : int { kForward = 0, kGradRows = 1, kGradWeight = 2 };

constexpr int kTile = 128, kTileStage = 2 * 128 * 128;      // a stage: 16 KiB of each operand

// Stores a wave's part of a tile, NI x NJ tiles of 32 x 32 whose first row is row `first_row` of the block's tile and whose first
// column is column `first_column` of y, 32 rows at a time through `slab`, LDS private to the wave (32 rows of 32 NJ floats, after
// scales and bias): from there rows are written 16 bytes at a time where they allow it, else element by element. Register r of lane l holds row
// 8 (r / 4) + 4 (l / 32) + r % 4 and column l % 32 of its 32 x 32 tile; in the slab, rows with bit 2 set keep their columns
// rotated by 32, so that the two halves of a register go to different banks.
// row_offset(row): where row `row` of the block's tile (less than `rows`) starts in y.
template <bool INT8, int MODE, int NI, int NJ, typename Acc, typename RowOffset>
__device__ __forceinline__ void store_wave_part(const TileArgs& g, Acc (&acc)[NI][NJ], float* slab, const float* scale_at, RowOffset row_offset, int group, int rows,
                                                int first_row, int first_column) {
  constexpr int kWidth = 32 * NJ;
  const int lane = threadIdx.x & 63;
  const int out_bytes = g.out_kind == kOutF32 ? 4 : 2;
  const int per_piece = 16 / out_bytes;
  const bool wide = reinterpret_cast<uintptr_t>(g.y) % 16 == 0 && g.ldy % per_piece == 0 && g.group_y % per_piece == 0 && g.columns % per_piece == 0;
  auto slab_at = [](int row, int column) { return row * kWidth + ((column + ((row & 4) << 3)) & (kWidth - 1)); };
  static_assert((kWidth & (kWidth - 1)) == 0, "columns are rotated within a row");
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row0 = first_row + 32 * i;
    if (row0 >= rows) continue;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int n = first_column + 32 * j + (lane & 31);
      const int n_in = n < g.columns ? n : g.columns - 1;
      const bool has_bias = MODE == kForward && g.bias != nullptr && group < g.groups;
      const float bv = has_bias ? load_bias(g.bias, g.out_kind, group * g.columns + n_in) : 0.0f;
      float sb = 1.0f;
      if constexpr (INT8) sb = group < g.groups ? g.scale_w[static_cast<int64_t>(group) * g.columns + n_in] : 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = 8 * (r / 4) + 4 * (lane >> 5) + (r % 4);
        float v;
        if constexpr (INT8) {
          // int32 -> f32, times the activation row's scale, times the weight row's, plus bias: each one rounded operation.
          v = __fmul_rn(__fmul_rn(static_cast<float>(acc[i][j][r]), scale_at[row0 + row]), sb);
          if (has_bias) v = __fadd_rn(v, bv);
          if (group == g.groups) v = 0.0f;
        } else {
          v = acc[i][j][r] + bv;
        }
        slab[slab_at(row, 32 * j + (lane & 31))] = v;
      }
    }
    if (!wide) {
#pragma unroll 1
      for (int at = lane; at < 32 * kWidth; at += 64) {
        const int row = at / kWidth, column = at % kWidth, n = first_column + column;
        if (row0 + row < rows && n < g.columns) store_out(g.y, g.out_kind, row_offset(row0 + row) + n, slab[slab_at(row, column)]);
      }
    } else if (g.out_kind == kOutF32) {
#pragma unroll
      for (int at = 0; at < 32 * (kWidth / 4); at += 64) {
        const int row = (at + lane) / (kWidth / 4), column = 4 * ((at + lane) % (kWidth / 4));
        const int n = first_column + column;
        if (row0 + row >= rows || n >= g.columns) continue;
        *reinterpret_cast<uint4*>(static_cast<float*>(g.y) + row_offset(row0 + row) + n) = *reinterpret_cast<const uint4*>(slab + slab_at(row, column));
      }
    } else {
#pragma unroll
      for (int at = 0; at < 32 * (kWidth / 8); at += 64) {
        const int row = (at + lane) / (kWidth / 8), column = 8 * ((at + lane) % (kWidth / 8));
        const int n = first_column + column;
        if (row0 + row >= rows || n >= g.columns) continue;
        const float* from = slab + slab_at(row, column);
        const float4 lo = *reinterpret_cast<const float4*>(from);
        const float4 hi = *reinterpret_cast<const float4*>(from + 4);
        uint4 packed;
        if (g.out_kind == kOutBF16) {
          packed = make_uint4(bf16_bits_of(lo.x) | bf16_bits_of(lo.y) << 16, bf16_bits_of(lo.z) | bf16_bits_of(lo.w) << 16,
                              bf16_bits_of(hi.x) | bf16_bits_of(hi.y) << 16, bf16_bits_of(hi.z) | bf16_bits_of(hi.w) << 16);
        } else {
          auto half_bits = [](float v) { return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v))); };
          packed = make_uint4(half_bits(lo.x) | half_bits(lo.y) << 16, half_bits(lo.z) | half_bits(lo.w) << 16, half_bits(hi.x) | half_bits(hi.y) << 16,
                              half_bits(hi.z) | half_bits(hi.w) << 16);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(g.y) + row_offset(row0 + row) + n) = packed;
      }
    }
  }
}

// TAIL = false: the inner length is a whole number of steps (256 x 256: of rounds of two; and, in the rows' gradient, the columns a whole number of tiles), so
// that no piece lies outside.
// GATHER: the weights' gradient with row_of (the other modes look at the pointer).
template <bool INT8, int MODE, bool TAIL, bool GATHER>
__global__ __launch_bounds__(256, 2) void grouped_tile_kernel(TileArgs g) {
  static_assert(!INT8 || MODE == kForward, "gradients are bf16");
  constexpr bool kColumnA = MODE == kGradWeight, kColumnB = MODE != kForward;
  __shared__ __align__(1024) uint8_t stage0[kTileStage];
  __shared__ __align__(1024) uint8_t stage1[kTileStage];
  __shared__ int32_t row_at[kTile];                         // rows' gradient: where each row of the tile is written
  __shared__ float scale_at[kTile];                         // int8: the scale of each row of the tile
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;
  const int column_tiles = (g.columns + kTile - 1) / kTile;
  const int n0 = static_cast<int>(blockIdx.x % column_tiles) * kTile;
  const int tile_at = static_cast<int>(blockIdx.x / column_tiles);

  int group, first, rows, m0 = 0, steps, inner;             // inner: bytes (row operand left) or inner rows (both columns)
  if constexpr (MODE == kGradWeight) {
    const int row_tiles = (g.rows + kTile - 1) / kTile;
    group = tile_at / row_tiles;
    m0 = tile_at % row_tiles * kTile;
    first = __builtin_amdgcn_readfirstlane(g.offsets[group]);
    inner = __builtin_amdgcn_readfirstlane(g.offsets[group + 1]) - first;
    rows = g.rows - m0 < kTile ? g.rows - m0 : kTile;
    steps = (inner + 63) / 64;
  } else {
    const RowTile tile = find_row_tile(g.offsets, g.groups, g.entries, tile_at, kTile);
    if (tile.group < 0) return;
    group = tile.group;
    first = tile.first;
    rows = tile.rows;
    inner = g.inner;
    steps = group < g.groups ? (inner + 127) / 128 : 0;     // rows of no group: zero
  }
  const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(kZeroPiece);

  auto source_of = [&](int place) {
    if (g.row_of == nullptr) return place;
    const int row = g.row_of[place];
    return row < g.x_rows ? row : g.x_rows - 1;
  };

  // What this lane loads. Row operand, load c: tile row 8 (wave + 4 c) + lane / 8, piece `piece_r`. Column operand, load c: inner row
  // 4 (wave + 4 c) + lane / 16, piece `piece_c`.
  const int piece_r = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);       // (row >> 1) & 7 is the same for all c
  const int piece_c = (lane & 15) ^ ((lane >> 4) << 2);
  const uint8_t* from_a[4];
  const uint8_t* from_b[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if constexpr (kColumnA) {
      from_a[c] = g.a + (first + 4 * (wave + 4 * c) + (lane >> 4)) * g.lda_bytes + (m0 + 8 * piece_c) * int64_t{2};
    } else {
      const int row = 8 * (wave + 4 * c) + (lane >> 3);
      const int place = first + (row < rows ? row : rows - 1);
      from_a[c] = g.a + (MODE == kForward ? source_of(place) : place) * g.lda_bytes + 16 * piece_r;
    }
    if constexpr (MODE == kForward) {
      const int n = n0 + 8 * (wave + 4 * c) + (lane >> 3);
      from_b[c] = g.b + (group < g.groups ? group : 0) * g.group_b_bytes + (n < g.columns ? n : g.columns - 1) * g.ldb_bytes + 16 * piece_r;
    } else if constexpr (MODE == kGradRows) {
      from_b[c] = g.b + (group < g.groups ? group : 0) * g.group_b_bytes + (4 * (wave + 4 * c) + (lane >> 4)) * g.ldb_bytes + (n0 + 8 * piece_c) * int64_t{2};
    } else {
      from_b[c] = g.b + (n0 + 8 * piece_c) * int64_t{2};
    }
  }
  const bool a_outside = kColumnA && m0 + 8 * piece_c >= g.rows;
  const bool b_outside = kColumnB && n0 + 8 * piece_c >= g.columns;
  // Weights' gradient: rows of b for one step, looked up a step before they are loaded.
  int row_b[4] = {};
  auto look_up = [&](int step) {
    if constexpr (MODE == kGradWeight) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = 64 * step + 4 * (wave + 4 * c) + (lane >> 4);
        const int place = first + (at < inner ? at : inner - 1);
        row_b[c] = GATHER ? g.row_of[place] : place;
      }
    }
  };
  auto to_lds = [&](const uint8_t* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  auto select = [&](bool inside, const uint8_t* from) {     // bitwise: a branch here would break the flow of the K loop
    const uint64_t mask = inside ? ~uint64_t{0} : 0;
    return reinterpret_cast<const uint8_t*>((reinterpret_cast<uint64_t>(from) & mask) | (reinterpret_cast<uint64_t>(zeros) & ~mask));
  };
  auto load_a = [&](uint8_t* stage, int step, int c) {
    const uint8_t* from;
    if constexpr (kColumnA) from = select(!a_outside & (64 * step + 4 * (wave + 4 * c) + (lane >> 4) < inner), from_a[c] + step * (64 * g.lda_bytes));
    else if constexpr (TAIL) from = select(128 * step + 16 * piece_r < inner, from_a[c] + step * int64_t{128});
    else from = from_a[c] + step * int64_t{128};
    to_lds(from, stage + 1024 * (wave + 4 * c));
  };
  auto load_b = [&](uint8_t* stage, int step, int c) {
    const uint8_t* from;
    if constexpr (MODE == kForward) {
      if constexpr (TAIL) from = select(128 * step + 16 * piece_r < inner, from_b[c] + step * int64_t{128});
      else from = from_b[c] + step * int64_t{128};
    } else if constexpr (MODE == kGradRows) {
      if constexpr (TAIL) from = select(!b_outside & (2 * (64 * step + 4 * (wave + 4 * c) + (lane >> 4)) < inner), from_b[c] + step * (64 * g.ldb_bytes));
      else from = from_b[c] + step * (64 * g.ldb_bytes);
    } else {
      from = select(!b_outside & (64 * step + 4 * (wave + 4 * c) + (lane >> 4) < inner), from_b[c] + (row_b[c] < g.x_rows ? row_b[c] : g.x_rows - 1) * g.ldb_bytes);
    }
    to_lds(from, stage + 16384 + 1024 * (wave + 4 * c));
  };

  using Acc = typename std::conditional<INT8, i32x16, f32x16>::type;
  using Frag = typename std::conditional<INT8, i32x4, bf16x8>::type;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  Acc acc[2][2] = {};
  Frag frag[2][4];                                          // two of a, two of b; a set is read while the other is multiplied
  // Row operand: row lane % 32 of a 32-row tile, piece 2 kk + lane / 32. Column operand: for inner rows 8 (lane / 32) .. + 8 of slice
  // kk the lane reads, twice, inner row 4 h + (lane % 16) / 4 and columns 16 ((lane / 16) % 2) + 4 (lane % 4) .. + 4 of the 32.
  const int turn = ((lane & 31) >> 1) & 7;
  const int quad = (lane & 15) >> 2;
  const uint32_t column_row = static_cast<uint32_t>((8 * (lane >> 5) + quad) * 256 + 8 * (lane & 1));
  const int column_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  auto read_one = [&](int set, const uint8_t* stage, int kk, int t) {
    const bool of_a = t < 2;
    const int tile = of_a ? 64 * wave_m + 32 * t : 64 * wave_n + 32 * (t - 2);
    const uint8_t* operand = stage + (of_a ? 0 : 16384);
    if ((of_a && kColumnA) || (!of_a && kColumnB)) {
      const uint32_t at = column_row + static_cast<uint32_t>(kk * 16 * 256) + 16 * static_cast<uint32_t>(((tile >> 3) + column_piece) ^ (quad << 2));
      const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(operand + at));
      const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(operand + at + 4 * 256));
      const s16x8 both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
      frag[set][t] = __builtin_bit_cast(Frag, both);
    } else {
      const uint32_t at = static_cast<uint32_t>((tile + (lane & 31)) * 128 + (((2 * kk + (lane >> 5)) ^ turn) * 16));
      frag[set][t] = *reinterpret_cast<const Frag*>(operand + at);
    }
  };
  auto multiply_one = [&](int set, int m) {
    const int i = m >> 1, j = m & 1;
    if constexpr (INT8) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(frag[set][i], frag[set][2 + j], acc[i][j], 0, 0, 0);
    else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[set][i], frag[set][2 + j], acc[i][j], 0, 0, 0);
  };

  if (MODE == kGradRows && tid < kTile) {
    const int place = first + (tid < rows ? tid : rows - 1);
    row_at[tid] = g.order != nullptr ? g.order[place] : place;
  }
  if (INT8 && tid < kTile) scale_at[tid] = g.scale_x[source_of(first + (tid < rows ? tid : rows - 1))];
  if (steps > 0) {
    auto clamp = [&](int step) { return step < steps ? step : steps - 1; };
    // One step on `here` while `there` is filled: the left operand's pieces of a tile are requested right after the barrier that
    // frees their stage, the right operand's during the first slice of the next step, so that every load has most of a step to
    // land. Past the last tile the loads repeat it, which nobody reads.
    auto k_step = [&](uint8_t* here, uint8_t* there, int step) {
      const int next = clamp(step + 1), second = clamp(step + 2);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        multiply_one(0, m);
        load_b(there, next, m);
        read_one(1, here, 1, m);
        __builtin_amdgcn_sched_barrier(0);
      }
      look_up(second);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        multiply_one(1, m);
        read_one(0, here, 2, m);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        multiply_one(0, m);
        read_one(1, here, 3, m);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);                   // vmcnt(0): this wave's part of `there` has landed
      __syncthreads();
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        multiply_one(1, m);
        load_a(here, second, m);
        read_one(0, there, 0, m);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    look_up(0);
#pragma unroll
    for (int c = 0; c < 4; ++c) load_a(stage0, 0, c);
#pragma unroll
    for (int c = 0; c < 4; ++c) load_b(stage0, 0, c);
    look_up(clamp(1));
#pragma unroll
    for (int c = 0; c < 4; ++c) load_a(stage1, clamp(1), c);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 4; ++t) read_one(0, stage0, 0, t);
    int step = 0;
    for (; step + 2 <= steps; step += 2) {                  // (a branch between the two steps would cost a wait for all loads)
      k_step(stage0, stage1, step);
      k_step(stage1, stage0, step + 1);
    }
    if (step < steps) k_step(stage0, stage1, step);
    __builtin_amdgcn_s_waitcnt(0x0F70);
  }
  __syncthreads();                                          // every load has landed and every fragment is read: the stages are free

  float* slab = reinterpret_cast<float*>(stage0) + wave * (32 * 64);
  auto row_offset = [&](int row) -> int64_t {
    if constexpr (MODE == kGradWeight) return group * g.group_y + (m0 + row) * g.ldy;
    else if constexpr (MODE == kGradRows) return row_at[row] * g.ldy;
    else return (static_cast<int64_t>(first) + row) * g.ldy;
  };
  store_wave_part<INT8, MODE>(g, acc, slab, scale_at, row_offset, group, rows, 64 * wave_m, n0 + 64 * wave_n);
}

// ---- 256 x 256 tiles: products of many tiles ------------------------------------------------------------------------------------
//
// Four waves share a 256 x 256 tile, 128 x 128 each, one wave per SIMD with its sums in 256 registers: sixteen matrix-core
// instructions per eight fragments, half the LDS reads of the 128 x 128 tile per operation. Stages, permutations and the order
// of a step are those of the 128 x 128 kernel: all loads of a tile are requested in the last slice of the step two before it,
// right after the barrier that frees their stage.
// A weight that comes from memory takes longer than the step that is left to it (eight experts of 4096 x 4096 do not stay in
// the last-level cache), so every step also touches the lines of the tile `kAhead` steps on, one 4-byte load per line into a
// scratch corner of LDS that nobody reads: they are in the L2 when their turn comes. The wait before the barrier leaves these
// loads in flight.
constexpr int kWideTile = 256, kWideStage = 2 * 256 * 128, kWideThreads = 256;

template <bool INT8, int MODE, bool TAIL, bool GATHER>
__global__ __launch_bounds__(kWideThreads, 1) void grouped_wide_kernel(TileArgs g) {
  static_assert(!INT8 || MODE == kForward, "gradients are bf16");
  constexpr bool kColumnA = MODE == kGradWeight, kColumnB = MODE != kForward;
  __shared__ __align__(1024) uint8_t stage0[kWideStage];
  __shared__ __align__(1024) uint8_t stage1[kWideStage];
  __shared__ int32_t row_at[kWideTile];
  __shared__ float scale_at[kWideTile];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;
  int tile_at, column_tile;
  tile_of_block(g.tiles, tile_at, column_tile);
  if (column_tile >= g.tiles.column_tiles) return;
  const int n0 = column_tile * kWideTile;

  int group, first, rows, m0 = 0, steps, inner;
  if constexpr (MODE == kGradWeight) {
    const int row_tiles = (g.rows + kWideTile - 1) / kWideTile;
    group = tile_at / row_tiles;
    if (group >= g.groups) return;
    m0 = tile_at % row_tiles * kWideTile;
    first = __builtin_amdgcn_readfirstlane(g.offsets[group]);
    inner = __builtin_amdgcn_readfirstlane(g.offsets[group + 1]) - first;
    rows = g.rows - m0 < kWideTile ? g.rows - m0 : kWideTile;
    steps = (inner + 63) / 64;
  } else {
    const RowTile tile = find_row_tile(g.offsets, g.groups, g.entries, tile_at, kWideTile);
    if (tile.group < 0) return;
    group = tile.group;
    first = tile.first;
    rows = tile.rows;
    inner = g.inner;
    steps = group < g.groups ? (inner + 127) / 128 : 0;
  }
  const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(kZeroPiece);
  auto source_of = [&](int place) {
    if (g.row_of == nullptr) return place;
    const int row = g.row_of[place];
    return row < g.x_rows ? row : g.x_rows - 1;
  };
  const int64_t weight_at = (group < g.groups ? group : 0) * g.group_b_bytes;
  auto select = [&](bool inside, const uint8_t* from) {     // bitwise: a branch here would break the flow of the K loop
    const uint64_t mask = inside ? ~uint64_t{0} : 0;
    return reinterpret_cast<const uint8_t*>((reinterpret_cast<uint64_t>(from) & mask) | (reinterpret_cast<uint64_t>(zeros) & ~mask));
  };
  // Row operand, load c < 8: tile row 8 (wave + 4 c) + lane / 8, piece `piece_r`. Column operand, load c: inner row 2 (wave + 4 c) +
  // lane / 32, piece `piece_c`. The addresses are kept and moved on in place: a register that a load in flight has as its address
  // is not written again before that load has landed (the compiler waits for all loads if it is).
  const int piece_r = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
  const int piece_c = (lane & 31) ^ (((2 * (wave & 1) + (lane >> 5)) & 3) << 2);
  const int inner_row = 2 * wave + (lane >> 5);             // of load 0; 8 more per load
  const bool a_inside = !kColumnA || m0 + 8 * piece_c < g.rows;
  const bool b_inside = !kColumnB || n0 + 8 * piece_c < g.columns;
  const uint8_t* from[16];                                  // 0..7: the left operand's loads, 8..15: the right one's
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    if constexpr (kColumnA) {
      from[c] = g.a + (first + inner_row + 8 * c) * g.lda_bytes + (m0 + 8 * piece_c) * int64_t{2};
    } else {
      const int row = 8 * (wave + 4 * c) + (lane >> 3);
      const int place = first + (row < rows ? row : rows - 1);
      from[c] = g.a + (MODE == kForward ? source_of(place) : place) * g.lda_bytes + 16 * piece_r;
    }
    if constexpr (MODE == kForward) {
      const int n = n0 + 8 * (wave + 4 * c) + (lane >> 3);
      from[8 + c] = g.b + weight_at + (n < g.columns ? n : g.columns - 1) * g.ldb_bytes + 16 * piece_r;
    } else if constexpr (MODE == kGradRows) {
      from[8 + c] = g.b + weight_at + (inner_row + 8 * c) * g.ldb_bytes + (n0 + 8 * piece_c) * int64_t{2};
    } else {
      from[8 + c] = nullptr;                                // looked up for every step
    }
  }
  const uint8_t* const b_columns = g.b + (n0 + 8 * piece_c) * int64_t{2};
  // Weights' gradient: the rows of b of one step. With row_of, the two rows of a load are the same for each half of the wave, so
  // their numbers come through scalar loads, which the counted waits below do not see, one step before they are used.
  int low_row[8], high_row[8];
  auto look_up = [&](int step) {
    if constexpr (MODE == kGradWeight && GATHER) {
      typedef const __attribute__((address_space(4))) int32_t* ScalarPointer;
      const ScalarPointer table = (ScalarPointer)(g.row_of);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int at = 64 * step + 2 * (wave + 4 * c);
        low_row[c] = table[first + (at < inner ? at : inner - 1)];
        high_row[c] = table[first + (at + 1 < inner ? at + 1 : inner - 1)];
      }
    }
  };
  // Moves load `load` to tile `step` from the tile before it (step 0: to where it starts). A piece outside the operand becomes zeros; past
  // the last tile the loads repeat it, which nobody reads.
  auto move_to = [&](int step, int load) {
    const bool of_a = load < 8;
    const int c = load & 7;
    if ((of_a && kColumnA) || (!of_a && MODE == kGradRows)) {
      const int64_t apart = of_a ? 64 * g.lda_bytes : 64 * g.ldb_bytes;
      const uint8_t* next = from[load] + (step > 0 && step < steps ? apart : 0);
      if (of_a) from[load] = select(a_inside & (64 * step + inner_row + 8 * c < inner), next);
      else if constexpr (TAIL) from[load] = select(b_inside & (2 * (64 * step + inner_row + 8 * c) < inner), next);
      else from[load] = next;
    } else if (!of_a && MODE == kGradWeight) {
      int row;
      if constexpr (GATHER) {
        row = (lane >> 5) != 0 ? high_row[c] : low_row[c];
        row = row < g.x_rows ? row : g.x_rows - 1;
      } else {
        row = first + 64 * step + inner_row + 8 * c;
      }
      from[load] = select(b_inside & (64 * step + inner_row + 8 * c < inner), b_columns + row * g.ldb_bytes);
    } else {
      const uint8_t* next = from[load] + (step > 0 && step < steps ? 128 : 0);
      if constexpr (TAIL) from[load] = select(128 * step + 16 * piece_r < inner, next);
      else from[load] = next;
    }
  };
  auto load_one = [&](uint8_t* stage, int load) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from[load],
                                     (__attribute__((address_space(3))) void*)(stage + (load < 8 ? 0 : 32768) + 1024 * (wave + 4 * (load & 7))), 16, 0, 0);
  };
  using Acc = typename std::conditional<INT8, i32x16, f32x16>::type;
  using Frag = typename std::conditional<INT8, i32x4, bf16x8>::type;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  Acc acc[4][4] = {};
  Frag frag[2][8];                                          // four of a, four of b
  const int turn = ((lane & 31) >> 1) & 7;
  const int quad = (lane & 15) >> 2;
  const uint32_t column_row = static_cast<uint32_t>((8 * (lane >> 5) + quad) * 512 + 8 * (lane & 1));
  const int column_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  auto read_one = [&](int set, const uint8_t* stage, int kk, int t) {
    const bool of_a = t < 4;
    const int tile = of_a ? 128 * wave_m + 32 * t : 128 * wave_n + 32 * (t - 4);
    const uint8_t* operand = stage + (of_a ? 0 : 32768);
    if ((of_a && kColumnA) || (!of_a && kColumnB)) {
      const uint32_t at = column_row + static_cast<uint32_t>(kk * 16 * 512) + 16 * static_cast<uint32_t>(((tile >> 3) + column_piece) ^ (quad << 2));
      const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(operand + at));
      const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(operand + at + 4 * 512));
      const s16x8 both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
      frag[set][t] = __builtin_bit_cast(Frag, both);
    } else {
      const uint32_t at = static_cast<uint32_t>((tile + (lane & 31)) * 128 + (((2 * kk + (lane >> 5)) ^ turn) * 16));
      frag[set][t] = *reinterpret_cast<const Frag*>(operand + at);
    }
  };
  auto multiply_one = [&](int set, int m) {
    const int i = m >> 2, j = m & 3;
    if constexpr (INT8) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(frag[set][i], frag[set][4 + j], acc[i][j], 0, 0, 0);
    else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[set][i], frag[set][4 + j], acc[i][j], 0, 0, 0);
  };

  if (MODE == kGradRows) {
    const int place = first + (tid < rows ? tid : rows - 1);
    row_at[tid] = g.order != nullptr ? g.order[place] : place;
  }
  if (INT8) scale_at[tid] = g.scale_x[source_of(first + (tid < rows ? tid : rows - 1))];
  if (steps > 0) {
    // One step on `here` while `there`, the next tile, lands.
    auto k_step = [&](uint8_t* here, uint8_t* there, int step) {
#pragma unroll
      for (int slice = 0; slice < 3; ++slice) {
#pragma unroll
        for (int m = 0; m < 16; ++m) {
          multiply_one(slice & 1, m);
          if (slice == 0 && m % 2 == 0) {
            move_to(step + 1, 8 + m / 2);
            load_one(there, 8 + m / 2);
          }
          if (m < 8) read_one((slice & 1) ^ 1, here, slice + 1, m);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      look_up(step + 2);
      // This wave's part of `there` has landed and its reads of `here` are complete.
      __builtin_amdgcn_s_waitcnt(0x0070);                   // vmcnt(0), lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int m = 0; m < 16; ++m) {
        multiply_one(1, m);
        if (m % 2 == 0) {
          move_to(step + 2, m / 2);
          load_one(here, m / 2);
        }
        if (m < 8) read_one(0, there, 0, m);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    look_up(0);
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      move_to(0, c);
      load_one(stage0, c);
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      move_to(1, c);
      load_one(stage1, c);
    }
    look_up(1);
    __builtin_amdgcn_s_waitcnt(0x0F78);                     // vmcnt(8): the first tile has landed
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int t = 0; t < 8; ++t) read_one(0, stage0, 0, t);
    // Whole rounds of two steps: a branch between them would cost a wait for all loads, a step of its own behind the loop moves of
    // all sums. An odd number of steps is followed by one of zeros (TAIL).
    for (int step = 0; step < steps; step += 2) {
      k_step(stage0, stage1, step);
      k_step(stage1, stage0, step + 1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);
  }
  __syncthreads();                                          // every load has landed and every fragment is read: the stages are free
  float* slab = reinterpret_cast<float*>(stage0) + wave * (32 * 128);
  auto row_offset = [&](int row) -> int64_t {
    if constexpr (MODE == kGradWeight) return group * g.group_y + (m0 + row) * g.ldy;
    else if constexpr (MODE == kGradRows) return row_at[row] * g.ldy;
    else return (static_cast<int64_t>(first) + row) * g.ldy;
  };
  store_wave_part<INT8, MODE>(g, acc, slab, scale_at, row_offset, group, rows, 128 * wave_m, n0 + 128 * wave_n);
}

}  // namespace ep

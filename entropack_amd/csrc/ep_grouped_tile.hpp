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
};

enum : int { kForward = 0, kGradRows = 1, kGradWeight = 2 };

constexpr int kTile = 128, kTileStage = 2 * 128 * 128;      // a stage: 16 KiB of each operand

// TAIL = false: the inner length is a whole number of steps (and, in the rows' gradient, the columns a whole number of tiles), so
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

  // The wave's 64 x 64 part, 32 rows at a time: through LDS private to the wave (as f32, after scales and bias) when rows can be
  // written 16 bytes at a time, else element by element. Register r of lane l holds row 8 (r / 4) + 4 (l / 32) + r % 4, column
  // l % 32 of its 32 x 32 tile; in the slab, rows with bit 2 set keep their columns rotated by 32, so that the two halves of a
  // register go to different banks.
  const int out_bytes = g.out_kind == kOutF32 ? 4 : 2;
  const int per_piece = 16 / out_bytes;
  const bool wide = reinterpret_cast<uintptr_t>(g.y) % 16 == 0 && g.ldy % per_piece == 0 && g.group_y % per_piece == 0 && g.columns % per_piece == 0;
  float* slab = reinterpret_cast<float*>(stage0) + wave * (32 * 64);
  auto slab_at = [](int row, int column) { return row * 64 + ((column + ((row & 4) << 3)) & 63); };
  auto row_offset = [&](int row) -> int64_t {               // row < rows
    if constexpr (MODE == kGradWeight) return group * g.group_y + (m0 + row) * g.ldy;
    else if constexpr (MODE == kGradRows) return row_at[row] * g.ldy;
    else return (static_cast<int64_t>(first) + row) * g.ldy;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row0 = 64 * wave_m + 32 * i;
    if (row0 >= rows) break;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + 64 * wave_n + 32 * j + (lane & 31);
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
        if (wide) slab[slab_at(row, 32 * j + (lane & 31))] = v;
        else if (row0 + row < rows && n < g.columns) store_out(g.y, g.out_kind, row_offset(row0 + row) + n, v);
      }
    }
    if (!wide) continue;
    if (g.out_kind == kOutF32) {
#pragma unroll
      for (int at = 0; at < 32 * 16; at += 64) {
        const int row = (at + lane) / 16, column = 4 * ((at + lane) % 16);
        const int n = n0 + 64 * wave_n + column;
        if (row0 + row >= rows || n >= g.columns) continue;
        *reinterpret_cast<uint4*>(static_cast<float*>(g.y) + row_offset(row0 + row) + n) = *reinterpret_cast<const uint4*>(slab + slab_at(row, column));
      }
    } else {
#pragma unroll
      for (int at = 0; at < 32 * 8; at += 64) {
        const int row = (at + lane) / 8, column = 8 * ((at + lane) % 8);
        const int n = n0 + 64 * wave_n + column;
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

}  // namespace ep

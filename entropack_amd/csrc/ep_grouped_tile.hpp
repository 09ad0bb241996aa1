// The block tiles of the products on grouped rows: forward (bf16, int8), gradient of the rows, gradient of the weights.
//
// All three are sums over an inner index of a left and a right operand; they differ in which index of each operand lies
// contiguous in memory. A "row" operand (x, w in the forward, dy in the rows' gradient) has the inner index contiguous, which
// is the shape of a matrix-core fragment; its tile is rows of 128 bytes. A "column" operand (w in the rows' gradient; dy and x
// in the weights') has its outer index contiguous; its tile is 64 inner rows, and the fragments are taken from LDS with the
// transposing reads (ds_read_b64_tr_b16: 16 lanes read a 4 x 16 block of two-byte elements and each receives a column of
// four).
//
// Four waves share a tile of TM x TN, TM / 2 x TN / 2 each. Tiles go from memory straight into LDS (global_load_lds_dwordx4, 1 KiB
// per wave and instruction) in two stages; the K loop is written out for both so that the compiler waits for loads in flight
// only at the barrier that publishes a stage. LDS rows cannot be padded then, so the 16-byte pieces of a row are permuted,
// piece c of row r at place c ^ ((r >> 1) & 7) (row operand: sixteen rows read at one logical piece cover all banks) or
// c ^ ((r & 3) << 2) (column operand: the four inner rows of a transposing read cover all banks).
//
// 256 x 256 (one block per CU, one wave per SIMD with its sums in 256 registers): sixteen matrix-core instructions per eight
// fragments, so that neither LDS nor the load path sets the pace; what does is the card's power limit. The loads of a step are
// spread over half of it: asked for all at once they fill the load path for longer than the matrix cores work, and the wave
// that issues them stalls. 128 x 128 (two blocks per CU): for groups of few rows.
//
// Ends: a lane whose piece lies past the operand's end loads a piece of zeros instead, so any inner length is exact, whatever
// lies in memory behind it; rows past the tile's last repeat it and are dropped when the tile is stored.
#pragma once

#include "ep_grouped.hpp"

namespace ep {

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
  int compute_units;               // blocks of 256 x 256 tiles that run at a time
  int chunk;                       // weights' gradient, 128 x 128: 0, or places per chunk: y is then f32 [chunk][rows][columns], one matrix
};                                 //   per chunk of a group's places (numbered like row tiles of `chunk` places)

enum : int { kForward = 0, kGradRows = 1, kGradWeight = 2 };

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
    order_in_wave();
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
        uint16_t* to = static_cast<uint16_t*>(g.y) + row_offset(row0 + row) + n;
        if constexpr (MODE == kGradWeight) {
          // Gradients of whole weights are read again much later, if at all from a cache: 580 -> 547 us for eight of 4096 x 4096.
          typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
          __builtin_nontemporal_store(u32x4{packed.x, packed.y, packed.z, packed.w}, reinterpret_cast<u32x4*>(to));
        } else {
          *reinterpret_cast<uint4*>(to) = packed;
        }
      }
    }
    order_in_wave();                                        // the slab is free again
  }
}

// What one block computes: rows [first_row, first_row + rows) of a group's rows (weights' gradient: of the weight) and columns n0 on.
struct BlockTile {
  int group;       // `groups`: rows of no group, which are written as zeros (weights' gradient: the matrix of y, a group's or a chunk's)
  int first;       // the place of the first row (weights' gradient: of the group)
  int rows;
  int m0;          // weights' gradient: first row
  int n0;
  int inner;       // forward, rows' gradient: bytes of the row operand; weights' gradient: places of the group
  int steps;
};

// A column operand's tile of 64 inner rows of 2 W bytes: load c of a wave takes inner row first_inner + per_load * c.
template <int W>
struct ColumnLoads {
  static constexpr int kRowsPerLoad = 512 / W;              // inner rows of 2 W bytes in 1 KiB
  static constexpr int kInnerPerLoad = 4 * kRowsPerLoad;    // four waves
  static constexpr int kPitch = 2 * W;
  __device__ static int first_inner(int wave, int lane) { return kRowsPerLoad * wave + lane / (W / 8); }
  __device__ static int piece(int wave, int lane) { return (lane % (W / 8)) ^ ((first_inner(wave, lane) & 3) << 2); }
};

// FOLD (weights' gradient to f32): the rows of y are the narrow rows' three parts, 64 rows for 16 ranks as they lie in the planes, and are added
// up here: y has a row per rank.
// TAIL = false: the inner length is a whole number of rounds of two steps (and, in the rows' gradient, the columns a whole number of
// tiles), so that no piece lies outside. GATHER: the weights' gradient with row_of (the other modes look at the pointer).
template <bool INT8, int MODE, bool TAIL, bool GATHER, int TM, int TN, bool FOLD = false, int STAGE>
__device__ __forceinline__ void compute_tile(const TileArgs& g, const BlockTile& tile, uint8_t (&stage0)[STAGE], uint8_t (&stage1)[STAGE], int32_t* row_at, float* scale_at) {
  static_assert(!INT8 || MODE == kForward, "gradients are bf16");
  static_assert(STAGE >= (TM + TN) * 128, "a stage holds both operands' tiles");
  constexpr bool kColumnA = MODE == kGradWeight, kColumnB = MODE != kForward;
  constexpr int NI = TM / 64, NJ = TN / 64;                 // 32 x 32 tiles of a wave
  constexpr int kLoadsA = TM / 32, kLoadsB = TN / 32;       // loads of a wave and step
  constexpr int kReads = NI + NJ, kMultiplies = NI * NJ, kStageB = TM * 128;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;
  const int group = tile.group, first = tile.first, rows = tile.rows, m0 = tile.m0, n0 = tile.n0, inner = tile.inner, steps = tile.steps;
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
  // Row operand, load c: tile row 8 (wave + 4 c) + lane / 8, piece `piece_r`. Column operand, load c: inner row inner_a (inner_b) +
  // kInnerPerLoad c, piece piece_a (piece_b). The addresses are kept and moved on in place: a register that a load in flight has as
  // its address is not written again before that load has landed (the compiler waits for all loads if it is).
  using ColumnsA = ColumnLoads<TM>;
  using ColumnsB = ColumnLoads<TN>;
  const int piece_r = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
  const int piece_a = ColumnsA::piece(wave, lane), inner_a = ColumnsA::first_inner(wave, lane);
  const int piece_b = ColumnsB::piece(wave, lane), inner_b = ColumnsB::first_inner(wave, lane);
  const bool a_inside = !kColumnA || m0 + 8 * piece_a < g.rows;
  const bool b_inside = !kColumnB || n0 + 8 * piece_b < g.columns;
  const uint8_t* from_a[kLoadsA];
  const uint8_t* from_b[kLoadsB];
#pragma unroll
  for (int c = 0; c < kLoadsA; ++c) {
    if constexpr (kColumnA) {
      from_a[c] = g.a + (first + inner_a + ColumnsA::kInnerPerLoad * c) * g.lda_bytes + (m0 + 8 * piece_a) * int64_t{2};
    } else {
      const int row = 8 * (wave + 4 * c) + (lane >> 3);
      const int place = first + (row < rows ? row : rows - 1);
      from_a[c] = g.a + (MODE == kForward ? source_of(place) : place) * g.lda_bytes + 16 * piece_r;
    }
  }
#pragma unroll
  for (int c = 0; c < kLoadsB; ++c) {
    if constexpr (MODE == kForward) {
      const int n = n0 + 8 * (wave + 4 * c) + (lane >> 3);
      from_b[c] = g.b + weight_at + (n < g.columns ? n : g.columns - 1) * g.ldb_bytes + 16 * piece_r;
    } else if constexpr (MODE == kGradRows) {
      from_b[c] = g.b + weight_at + (inner_b + ColumnsB::kInnerPerLoad * c) * g.ldb_bytes + (n0 + 8 * piece_b) * int64_t{2};
    } else {
      from_b[c] = nullptr;                                  // looked up for every step
    }
  }
  const uint8_t* const b_columns = g.b + (n0 + 8 * piece_b) * int64_t{2};
  // Weights' gradient with row_of: the row of b of every load, looked up a step before it is used (the barrier in between waits for all
  // loads anyway).
  int row_b[kLoadsB] = {};
  auto look_up = [&](int step) {
    if constexpr (MODE == kGradWeight && GATHER) {
#pragma unroll
      for (int c = 0; c < kLoadsB; ++c) {
        const int at = 64 * step + inner_b + ColumnsB::kInnerPerLoad * c;
        row_b[c] = g.row_of[first + (at < inner ? at : inner - 1)];
      }
    }
  };
  // Moves a load to tile `step` from the tile before it (step 0: to where it starts). A piece outside the operand becomes zeros; past
  // the last tile the loads repeat it or take zeros, which nobody reads.
  auto load_a = [&](uint8_t* stage, int step, int c) {
    if constexpr (kColumnA) {
      const uint8_t* next = from_a[c] + (step > 0 && step < steps ? 64 * g.lda_bytes : 0);
      from_a[c] = select(a_inside & (64 * step + inner_a + ColumnsA::kInnerPerLoad * c < inner), next);
    } else {
      const uint8_t* next = from_a[c] + (step > 0 && step < steps ? 128 : 0);
      if constexpr (TAIL) from_a[c] = select(128 * step + 16 * piece_r < inner, next);
      else from_a[c] = next;
    }
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from_a[c],
                                     (__attribute__((address_space(3))) void*)(stage + 1024 * (wave + 4 * c)), 16, 0, 0);
  };
  auto load_b = [&](uint8_t* stage, int step, int c) {
    if constexpr (MODE == kForward) {
      const uint8_t* next = from_b[c] + (step > 0 && step < steps ? 128 : 0);
      if constexpr (TAIL) from_b[c] = select(128 * step + 16 * piece_r < inner, next);
      else from_b[c] = next;
    } else if constexpr (MODE == kGradRows) {
      const uint8_t* next = from_b[c] + (step > 0 && step < steps ? 64 * g.ldb_bytes : 0);
      if constexpr (TAIL) from_b[c] = select(b_inside & (2 * (64 * step + inner_b + ColumnsB::kInnerPerLoad * c) < inner), next);
      else from_b[c] = next;
    } else {
      const int at = 64 * step + inner_b + ColumnsB::kInnerPerLoad * c;
      const int row = !GATHER ? first + at : (row_b[c] < g.x_rows ? row_b[c] : g.x_rows - 1);
      from_b[c] = select(b_inside & (at < inner), b_columns + row * g.ldb_bytes);
    }
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from_b[c],
                                     (__attribute__((address_space(3))) void*)(stage + kStageB + 1024 * (wave + 4 * c)), 16, 0, 0);
  };

  using Acc = typename std::conditional<INT8, i32x16, f32x16>::type;
  using Frag = typename std::conditional<INT8, i32x4, bf16x8>::type;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  Acc acc[NI][NJ] = {};
  Frag frag[2][kReads];                                     // NI of a, NJ of b; a set is read while the other is multiplied
  // Row operand: row lane % 32 of a 32-row tile, piece 2 kk + lane / 32. Column operand: for inner rows 8 (lane / 32) .. + 8 of slice
  // kk the lane reads, twice, inner row 4 h + (lane % 16) / 4 and columns 16 ((lane / 16) % 2) + 4 (lane % 4) .. + 4 of the 32.
  const int turn = ((lane & 31) >> 1) & 7;
  const int quad = (lane & 15) >> 2;
  const int column_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  auto read_one = [&](int set, const uint8_t* stage, int kk, int t) {
    const bool of_a = t < NI;
    const int at_tile = of_a ? (TM / 2) * wave_m + 32 * t : (TN / 2) * wave_n + 32 * (t - NI);
    const uint8_t* operand = stage + (of_a ? 0 : kStageB);
    if ((of_a && kColumnA) || (!of_a && kColumnB)) {
      const uint32_t pitch = of_a ? ColumnsA::kPitch : ColumnsB::kPitch;
      const uint32_t at = static_cast<uint32_t>(kk * 16 + 8 * (lane >> 5) + quad) * pitch + 8 * (lane & 1) + 16 * static_cast<uint32_t>(((at_tile >> 3) + column_piece) ^ (quad << 2));
      const s16x4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(operand + at));
      const s16x4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(operand + at + 4 * pitch));
      const s16x8 both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
      frag[set][t] = __builtin_bit_cast(Frag, both);
    } else {
      const uint32_t at = static_cast<uint32_t>((at_tile + (lane & 31)) * 128 + (((2 * kk + (lane >> 5)) ^ turn) * 16));
      frag[set][t] = *reinterpret_cast<const Frag*>(operand + at);
    }
  };
  auto multiply_one = [&](int set, int m) {
    const int i = m / NJ, j = m % NJ;
    if constexpr (INT8) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(frag[set][i], frag[set][NI + j], acc[i][j], 0, 0, 0);
    else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[set][i], frag[set][NI + j], acc[i][j], 0, 0, 0);
  };

  if (MODE == kGradRows && tid < TM) {
    const int place = first + (tid < rows ? tid : rows - 1);
    row_at[tid] = g.order != nullptr ? g.order[place] : place;
  }
  if (INT8 && tid < TM) scale_at[tid] = g.scale_x[source_of(first + (tid < rows ? tid : rows - 1))];
  if (steps > 0) {
    // One step on `here` while `there`, the next tile, lands: its left pieces were requested in the last slice of the step before,
    // right after the barrier that freed the stage, its right pieces are in the first slice of this one.
    constexpr int kApartA = kMultiplies / kLoadsA > 0 ? kMultiplies / kLoadsA : 1, kApartB = kMultiplies / kLoadsB > 0 ? kMultiplies / kLoadsB : 1;
    static_assert(kMultiplies >= kLoadsA && kMultiplies >= kLoadsB && kMultiplies >= kReads, "every load and read has a multiply in front of it");
    auto k_step = [&](uint8_t* here, uint8_t* there, int step) {
#pragma unroll
      for (int slice = 0; slice < 3; ++slice) {
#pragma unroll
        for (int m = 0; m < kMultiplies; ++m) {
          multiply_one(slice & 1, m);
          if (slice == 0 && m % kApartB == 0 && m / kApartB < kLoadsB) load_b(there, step + 1, m / kApartB);
          if (m < kReads) read_one((slice & 1) ^ 1, here, slice + 1, m);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (slice == 0) look_up(step + 2);
      }
      // This wave's part of `there` has landed and its reads of `here` are complete.
      __builtin_amdgcn_s_waitcnt(0x0070);                   // vmcnt(0), lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int m = 0; m < kMultiplies; ++m) {
        multiply_one(1, m);
        if (m % kApartA == 0 && m / kApartA < kLoadsA) load_a(here, step + 2, m / kApartA);
        if (m < kReads) read_one(0, there, 0, m);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    look_up(0);
#pragma unroll
    for (int c = 0; c < kLoadsA; ++c) load_a(stage0, 0, c);
#pragma unroll
    for (int c = 0; c < kLoadsB; ++c) load_b(stage0, 0, c);
#pragma unroll
    for (int c = 0; c < kLoadsA; ++c) load_a(stage1, 1, c);
    look_up(1);
    __builtin_amdgcn_s_waitcnt(0x0F70 | kLoadsA);           // vmcnt(kLoadsA): the first tile has landed
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int t = 0; t < kReads; ++t) read_one(0, stage0, 0, t);
    // Whole rounds of two steps: a branch between them would cost a wait for all loads, a step of its own behind the loop moves of
    // all sums. An odd number of steps is followed by one of zeros (TAIL).
    for (int step = 0; step < steps; step += 2) {
      k_step(stage0, stage1, step);
      k_step(stage1, stage0, step + 1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);
  }
  if constexpr (FOLD) {
    // A wave's 64 rows are one stretch of 16 ranks: values in registers 0 .. 7 of its first 32 x 32 tiles, remainders in 8 .. 15, last parts in
    // 0 .. 7 of the second, all three of a rank and column in one lane.
    static_assert(MODE == kGradWeight && TM == 128, "64 rows per wave");
    if (m0 + 64 * wave_m >= g.rows) return;
    float* const to = static_cast<float*>(g.y) + group * g.group_y + (m0 / 4 + 16 * wave_m) * g.ldy;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int n = n0 + (TN / 2) * wave_n + 32 * j + (lane & 31);
      if (n >= g.columns) continue;
#pragma unroll
      for (int r = 0; r < 8; ++r) to[(8 * (r / 4) + 4 * (lane >> 5) + r % 4) * g.ldy + n] = acc[0][j][r] + (acc[0][j][r + 8] + acc[1][j][r]);
    }
    return;
  }
  __syncthreads();                                          // every load has landed and every fragment is read: the stages are free
  static_assert(4 * 32 * (TN / 2) * 4 <= STAGE, "four slabs fit into a stage");
  float* slab = reinterpret_cast<float*>(stage0) + wave * (32 * (TN / 2));
  auto row_offset = [&](int row) -> int64_t {
    if constexpr (MODE == kGradWeight) return group * g.group_y + (m0 + row) * g.ldy;
    else if constexpr (MODE == kGradRows) return row_at[row] * g.ldy;
    else return (static_cast<int64_t>(first) + row) * g.ldy;
  };
  store_wave_part<INT8, MODE>(g, acc, slab, scale_at, row_offset, group, rows, (TM / 2) * wave_m, n0 + (TN / 2) * wave_n);
}

// The tile of `tile` x `tile` with number `at`, column tiles first; false past the last one.
template <int MODE>
__device__ __forceinline__ bool find_block_tile(const TileArgs& g, int64_t at, int tile, BlockTile& out) {
  const int column_tiles = (g.columns + tile - 1) / tile;
  const int row_tile = static_cast<int>(at / column_tiles);
  out.n0 = static_cast<int>(at % column_tiles) * tile;
  out.m0 = 0;
  if constexpr (MODE == kGradWeight) {
    const int row_tiles = (g.rows + tile - 1) / tile;
    out.m0 = row_tile % row_tiles * tile;
    if (g.chunk != 0) {
      const RowTile found = find_row_tile(g.offsets, g.groups, g.entries, row_tile / row_tiles, g.chunk);
      if (found.group < 0 || found.group == g.groups) return false;
      out.group = row_tile / row_tiles;                     // where the result goes
      out.first = found.first;
      out.inner = found.rows;
    } else {
      out.group = row_tile / row_tiles;
      if (out.group >= g.groups) return false;
      out.first = __builtin_amdgcn_readfirstlane(g.offsets[out.group]);
      out.inner = __builtin_amdgcn_readfirstlane(g.offsets[out.group + 1]) - out.first;
    }
    out.rows = g.rows - out.m0 < tile ? g.rows - out.m0 : tile;
    out.steps = (out.inner + 63) / 64;
  } else {
    const RowTile found = find_row_tile(g.offsets, g.groups, g.entries, row_tile, tile);
    if (found.group < 0) return false;
    out.group = found.group;
    out.first = found.first;
    out.rows = found.rows;
    out.inner = g.inner;
    out.steps = out.group < g.groups ? (out.inner + 127) / 128 : 0;      // rows of no group: zero
  }
  return true;
}

constexpr int kTile = 128, kWideTile = 256, kTileThreads = 256;

template <bool INT8, int MODE, bool TAIL, bool GATHER>
__global__ __launch_bounds__(kTileThreads, 2) void grouped_tile_kernel(TileArgs g) {
  __shared__ __align__(1024) uint8_t stage0[256 * 128];
  __shared__ __align__(1024) uint8_t stage1[256 * 128];
  __shared__ int32_t row_at[kTile];
  __shared__ float scale_at[kTile];
  BlockTile tile;
  if (!find_block_tile<MODE>(g, blockIdx.x, kTile, tile)) return;
  compute_tile<INT8, MODE, TAIL, GATHER, 128, 128>(g, tile, stage0, stage1, row_at, scale_at);
}

// 256 x 256 tiles, one per CU at a time. The tiles of the last, partial round are divided when that gives every part a CU of its own:
// into quarters of 128 x 128 (at most a quarter of the CUs' tiles are left) or halves of 256 x 128. A round of eight experts
// of 4096 x 4096 takes 105 us, the round of quarters a third of that.
template <bool INT8, int MODE, bool TAIL, bool GATHER>
__global__ __launch_bounds__(kTileThreads, 1) void grouped_wide_kernel(TileArgs g) {
  __shared__ __align__(1024) uint8_t stage0[512 * 128];
  __shared__ __align__(1024) uint8_t stage1[512 * 128];
  __shared__ int32_t row_at[kWideTile];
  __shared__ float scale_at[kWideTile];
  const int64_t column_tiles = (g.columns + kWideTile - 1) / kWideTile;
  const int64_t row_tiles = MODE == kGradWeight ? static_cast<int64_t>(g.groups) * ((g.rows + kWideTile - 1) / kWideTile)
                                                : count_row_tiles(g.offsets, g.groups, g.entries, kWideTile);
  const int64_t tiles = row_tiles * column_tiles, whole = tiles / g.compute_units * g.compute_units;
  const int left = static_cast<int>(tiles - whole);
  const int parts = 4 * left <= g.compute_units ? 4 : (2 * left <= g.compute_units ? 2 : 1);
  const int64_t block = blockIdx.x;
  const int64_t at = block < whole ? block : whole + (block - whole) / parts;
  const int part = block < whole ? -1 : static_cast<int>((block - whole) % parts);
  if (at >= tiles) return;
  BlockTile tile;
  if (!find_block_tile<MODE>(g, at, kWideTile, tile)) return;
  if (part < 0 || parts == 1) {
    compute_tile<INT8, MODE, TAIL, GATHER, 256, 256>(g, tile, stage0, stage1, row_at, scale_at);
    return;
  }
  const int right = part & 1, lower = part >> 1;
  tile.n0 += 128 * right;
  if (tile.n0 >= g.columns) return;
  if (parts == 2) {
    compute_tile<INT8, MODE, TAIL, GATHER, 256, 128>(g, tile, stage0, stage1, row_at, scale_at);
    return;
  }
  if (lower != 0) {
    if (tile.rows <= 128) return;
    tile.rows -= 128;
    if (MODE == kGradWeight) tile.m0 += 128;
    else tile.first += 128;
  }
  if (tile.rows > 128) tile.rows = 128;
  compute_tile<INT8, MODE, TAIL, GATHER, 128, 128>(g, tile, stage0, stage1, row_at, scale_at);
}

// Blocks of a launch: one per tile, and the parts of the last round.
inline int64_t wide_blocks(int64_t row_tiles, int64_t columns, int compute_units) {
  return row_tiles * ((columns + kWideTile - 1) / kWideTile) + 3 * (compute_units / 4) + compute_units / 2;
}

}  // namespace ep

// Products on grouped rows: what the kernels of experts (ep_grouped.hip) and of low-rank adapters (ep_low_rank.hip) share.
//
// Rows p = offsets[g] .. offsets[g + 1] - 1 of the grouped order meet the weight of group g; places from offsets[groups] on
// belong to no group. The sizes of the groups are known on the device only, so a launch covers the most row tiles there can
// be (every group may end inside a tile) and a block finds its tile by a scan over the offsets.
#pragma once

#include "ep_matrix.hpp"

namespace ep {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kMostEntries = int64_t{1} << 30;

// A launch has fewer than 2^32 work items.
inline bool launch_fits(int64_t blocks, int threads) { return blocks <= 0xFFFFFFFF / threads; }

// What a lane loads whose piece lies past an operand's end.
__device__ __align__(16) const uint32_t kZeroPiece[4] = {0, 0, 0, 0};

// 16 bytes of global memory. (An address chosen between an operand and the zeros has no address space of its own, and a load that
// might be one of LDS waits for every LDS access.)
__device__ __forceinline__ uint4 load_piece(const uint8_t* from) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 v = *(const __attribute__((address_space(1))) u32x4*)from;
  return make_uint4(v.x, v.y, v.z, v.w);
}

struct RowTile {
  int group;       // `groups` for a tile of rows without a group, -1 past the last tile
  int first;       // first place of the tile
  int rows;        // 1 .. tile_rows places
  int index;       // number of the tile within its group
};

// Sums of lanes 0 .. l, through the data-parallel lane moves (six dependent adds; the same scan through LDS takes ten times as long,
// and every block of a product begins with one).
__device__ __forceinline__ int wave_inclusive_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);     // from 1 lane below, within rows of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);     // 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);     // 4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);     // 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);     // lane 15 of a row to the next row: rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);     // lane 31 to rows 2 and 3
  return v;
}

// Tile number `tile` of tiles of `tile_rows` places, in the order of the groups, those of no group last. Called by whole
// waves; the result is the same in every lane.
__device__ __forceinline__ RowTile find_row_tile(const int32_t* __restrict__ offsets, int groups, int entries, int tile, int tile_rows) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int g0 = 0; g0 < groups; g0 += 64) {
    const int g = g0 + lane;
    int low = 0, high = 0;
    if (g < groups) {
      low = offsets[g];
      high = offsets[g + 1];
    }
    const int n = (high - low + tile_rows - 1) / tile_rows;
    const int inclusive = wave_inclusive_sum(n);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + inclusive > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int index = tile - before - __builtin_amdgcn_readlane(inclusive - n, at);
      const int first = __builtin_amdgcn_readlane(low, at) + index * tile_rows;
      const int left = __builtin_amdgcn_readlane(high, at) - first;
      return {g0 + at, first, left < tile_rows ? left : tile_rows, index};
    }
    before += __builtin_amdgcn_readlane(inclusive, 63);
  }
  const int kept = __builtin_amdgcn_readfirstlane(offsets[groups]);
  const int64_t first = kept + static_cast<int64_t>(tile - before) * tile_rows;
  if (first >= entries) return {-1, 0, 0, 0};
  const int64_t left = entries - first;
  return {groups, static_cast<int>(first), static_cast<int>(left < tile_rows ? left : tile_rows), tile - before};
}

// LDS accesses before it, of any lane of this wave, come before those after it.
__device__ __forceinline__ void order_in_wave() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// How many tiles there are, those of no group included.
__device__ __forceinline__ int64_t count_row_tiles(const int32_t* __restrict__ offsets, int groups, int entries, int tile_rows) {
  const int lane = threadIdx.x & 63;
  int mine = 0;
  for (int g = lane; g < groups; g += 64) mine += (offsets[g + 1] - offsets[g] + tile_rows - 1) / tile_rows;
  if (lane == 0) mine += (entries - offsets[groups] + tile_rows - 1) / tile_rows;
  return __builtin_amdgcn_readlane(wave_inclusive_sum(mine), 63);
}

// The most tiles of `tile_rows` places that `entries` places in `groups` groups (and the places of none) make.
inline int64_t most_row_tiles(int64_t entries, int groups, int tile_rows) {
  const int64_t parts = groups + 1 < entries ? groups + 1 : entries;          // every part may end with a tile of its own
  return entries / tile_rows + parts;
}

// The most chunks of `chunk` places that `entries` places in `groups` groups make (places of no group are in none).
inline int64_t most_chunks(int64_t entries, int groups, int chunk) { return entries / chunk + (groups < entries ? groups : entries); }

// What a product on grouped rows is told. Place p reads row row_of[p] of x, or row p where row_of is null.
struct GroupedArgs {
  const uint8_t* x;
  const uint8_t* w;
  const float* scale_x;            // int8 products: per row of x, per row of every weight
  const float* scale_w;
  const void* bias;                // [groups][N], in the output's type
  void* y;
  const int32_t* row_of;
  const int32_t* offsets;
  int64_t ldx_bytes, ldw_bytes, group_bytes, k_bytes, ldy;
  int entries, groups, N, x_rows, out_kind;
};

__device__ __forceinline__ int source_row(const GroupedArgs& a, int place) {
  if (a.row_of == nullptr) return place;
  const int row = a.row_of[place];
  return row < a.x_rows ? row : a.x_rows - 1;
}

// ---- few rows per group: the weight's stream bounds the product -------------------------------------------------------------
//
// A block takes 16 MT rows and 16 NT weight rows; its waves take every WAVES-th piece of 256 bytes of K, each by itself, and the
// sums meet in LDS. Memory wants neighbouring lanes at neighbouring addresses: a load takes 256 bytes of each of four rows. The
// fragments of the 16 x 16 matrix-core instructions want sixteen rows (lane l holds 16 bytes of row l % 16, at byte 16 (l / 16)
// of a 64-byte step): the piece goes through LDS private to the wave, while the next one is on its way in registers, so that
// there is no barrier in the loop. Loading the fragments straight from memory occupies the address path four times as long.
// PLANES: the sums are multiplied with scale_x[group] and stored as three bf16 parts, the rounded value, the rounded remainder and what
// then remains: 8 bits of significand each, so that the three add up to the f32 value exactly (above 2^-110, where the last part leaves
// the range of bf16). Row p of y holds 64 columns for every 16 of N: 16 values, 16 remainders, 16 last parts and 16 zeros, which is how the
// products that read it take them; columns from N to the next multiple of 16 are 0.
template <bool INT8, int MT, int NT, int WAVES, bool PLANES>
__global__ __launch_bounds__(64 * WAVES) void grouped_stream_kernel(GroupedArgs a) {
  using Acc = typename std::conditional<INT8, i32x4, f32x4>::type;
  using Frag = typename std::conditional<INT8, i32x4, bf16x8>::type;
  using Cell = typename std::conditional<INT8, int32_t, float>::type;
  constexpr int kRows = 16 * MT, kColumns = 16 * NT, kPitch = kColumns + 4;
  constexpr int kStagedPitch = 256 + 16;           // bytes of a staged row: an odd number of 16-byte pieces, all banks
  constexpr int kStagedBytes = 16 * (MT + NT) * kStagedPitch, kSumsBytes = kRows * kPitch * 4;       // of a wave
  __shared__ __align__(16) uint8_t room[WAVES * (kStagedBytes > kSumsBytes ? kStagedBytes : kSumsBytes)];
  Cell(*sums)[kRows][kPitch] = reinterpret_cast<Cell(*)[kRows][kPitch]>(room);                       // once every wave is done with its stage
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column_tiles = (a.N + kColumns - 1) / kColumns;
  const int n0 = static_cast<int>(blockIdx.x % column_tiles) * kColumns;
  const RowTile tile = find_row_tile(a.offsets, a.groups, a.entries, static_cast<int>(blockIdx.x / column_tiles), kRows);
  if (tile.group < 0) return;
  if (tile.group == a.groups) {
    if constexpr (!PLANES) {                       // rows of no group
      for (int cell = threadIdx.x; cell < kRows * kColumns; cell += 64 * WAVES) {
        const int row = cell / kColumns, n = n0 + cell % kColumns;
        if (row < tile.rows && n < a.N) store_out(a.y, a.out_kind, (static_cast<int64_t>(tile.first) + row) * a.ldy + n, 0.0f);
      }
    }
    return;
  }
  uint8_t* const staged = room + wave * kStagedBytes;
  auto staged_at = [&](int row, int byte) { return staged + row * kStagedPitch + byte; };
  const int in_row = lane & 15;
  const int load_row = lane >> 4, load_at = 16 * (lane & 15);         // row 4 i + load_row of load i, its bytes
  const uint8_t* from_x[4 * MT];
#pragma unroll
  for (int i = 0; i < 4 * MT; ++i) {
    const int row = 4 * i + load_row;
    from_x[i] = a.x + source_row(a, tile.first + (row < tile.rows ? row : tile.rows - 1)) * a.ldx_bytes + load_at;
  }
  const uint8_t* from_w[4 * NT];
#pragma unroll
  for (int i = 0; i < 4 * NT; ++i) {
    const int n = n0 + 4 * i + load_row;
    from_w[i] = a.w + tile.group * a.group_bytes + (n < a.N ? n : a.N - 1) * a.ldw_bytes + load_at;
  }
  const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(kZeroPiece);
  Acc acc[MT][NT] = {};
  uint4 held_x[4 * MT], held_w[4 * NT];
  auto fetch = [&](int64_t kb) {                   // both operands are zero past the row's end
    const bool inside = kb + load_at < a.k_bytes;
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) held_w[i] = load_piece(inside ? from_w[i] + kb : zeros);
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) held_x[i] = load_piece(inside ? from_x[i] + kb : zeros);
  };
  const int64_t stride = WAVES * 256;
  if (wave * 256 < a.k_bytes) fetch(wave * 256);
  for (int64_t kb = wave * 256; kb < a.k_bytes; kb += stride) {
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) *reinterpret_cast<uint4*>(staged_at(4 * i + load_row, load_at)) = held_x[i];
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) *reinterpret_cast<uint4*>(staged_at(16 * MT + 4 * i + load_row, load_at)) = held_w[i];
    if (kb + stride < a.k_bytes) fetch(kb + stride);
    order_in_wave();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      Frag fx[MT], fw[NT];
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[t] = *reinterpret_cast<const Frag*>(staged_at(16 * t + in_row, 64 * s + 16 * (lane >> 4)));
#pragma unroll
      for (int j = 0; j < NT; ++j) fw[j] = *reinterpret_cast<const Frag*>(staged_at(16 * (MT + j) + in_row, 64 * s + 16 * (lane >> 4)));
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if constexpr (INT8) acc[t][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx[t], fw[j], acc[t][j], 0, 0, 0);
          else acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[t], fw[j], acc[t][j], 0, 0, 0);
        }
    }
    order_in_wave();
  }
  __syncthreads();
  // Register i of lane l holds row 4 (l / 16) + i and column l % 16 of its 16 x 16 tile.
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave][16 * t + 4 * (lane >> 4) + i][16 * j + in_row] = acc[t][j][i];
  __syncthreads();
  for (int cell = threadIdx.x; cell < kRows * kColumns; cell += 64 * WAVES) {
    const int row = cell / kColumns, column = cell % kColumns, n = n0 + column;
    if (row >= tile.rows) continue;
    Cell sum = sums[0][row][column];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += sums[w][row][column];
    const int64_t place = static_cast<int64_t>(tile.first) + row;
    if constexpr (PLANES) {
      const int padded = (a.N + 15) & ~15;
      if (n >= padded) continue;
      float v = n < a.N ? static_cast<float>(sum) : 0.0f;
      if (a.scale_x != nullptr && n < a.N) v = __fmul_rn(v, a.scale_x[tile.group]);      // rounded before it is divided into parts
      uint16_t* out = static_cast<uint16_t*>(a.y) + place * a.ldy + 4 * (n & ~15) + (n & 15);
      const uint32_t high = bf16_bits_of(v);
      const float rest = (high & 0x7F80u) == 0x7F80u ? 0.0f : v - __uint_as_float(high << 16);      // an infinity has no remainder
      const uint32_t middle = bf16_bits_of(rest);
      out[0] = static_cast<uint16_t>(high);
      out[16] = static_cast<uint16_t>(middle);
      out[32] = static_cast<uint16_t>(bf16_bits_of(rest - __uint_as_float(middle << 16)));
      out[48] = 0;
    } else if (n < a.N) {
      const bool has_bias = a.bias != nullptr;
      const float b = has_bias ? load_bias(a.bias, a.out_kind, tile.group * a.N + n) : 0.0f;
      float v;
      if constexpr (INT8) {
        // int32 -> f32, times the activation row's scale, times the weight row's, plus bias: each one rounded operation.
        v = __fmul_rn(__fmul_rn(static_cast<float>(sum), a.scale_x[source_row(a, tile.first + row)]), a.scale_w[static_cast<int64_t>(tile.group) * a.N + n]);
        if (has_bias) v = __fadd_rn(v, b);
      } else {
        v = static_cast<float>(sum) + b;
      }
      store_out(a.y, a.out_kind, place * a.ldy + n, v);
    }
  }
}

template <bool INT8, int MT, int NT, int WAVES, bool PLANES>
static int launch_stream_of(const GroupedArgs& a, hipStream_t s) {
  const int64_t blocks = most_row_tiles(a.entries, a.groups, 16 * MT) * ((a.N + 16 * NT - 1) / (16 * NT));
  if (!launch_fits(blocks, 64 * WAVES)) return EP_HIP_EUNSUPPORTED;
  hipLaunchKernelGGL((grouped_stream_kernel<INT8, MT, NT, WAVES, PLANES>), dim3(static_cast<unsigned>(blocks)), dim3(64 * WAVES), 0, s, a);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

}  // namespace ep

// Low-rank adapters of many requests beside a shared product: out[t] = y[t] + scale[a] (x[t] down[a]^T) up[a]^T.
//
//   shrink   planes[p] = scale[a] x[order[p]] . down[a]^T      grouped_stream_kernel (ep_grouped.hpp), bound by reading x
//   expand   out[order[p]] = y[order[p]] + planes[p] . up[a]^T   low_rank_expand_kernel, bound by reading y and writing out
//   reduce   sum_p planes[p]^T q[order[p]]                     grouped_tile_kernel, low_rank_finish_kernel: the gradients of down (q = x, planes of the
//                                                              output's gradient) and of up (q = the output's gradient)
// The narrow rows in between ("planes") are kept as two bf16 parts, value and remainder, so that the second product loses
// nothing that the output's own rounding would show: each rounding is off by at most 2^-8 of what it
// rounds, so the two parts together by at most 2^-16 of the f32 value.
#include "ep_grouped_tile.hpp"

namespace ep {

struct LowRankArgs {
  const uint16_t* planes;          // [entries][2 padded]
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
__device__ __forceinline__ bf16x8 up_piece(const uint16_t* __restrict__ row, int e, int rank) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if constexpr (PIECES) {
    if (e < rank) v = *reinterpret_cast<const uint4*>(row + e);
  } else {
    uint32_t word[4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < rank) word[i >> 1] |= static_cast<uint32_t>(row[e + i]) << (16 * (i & 1));
    v = make_uint4(word[0], word[1], word[2], word[3]);
  }
  return __builtin_bit_cast(bf16x8, v);
}

// A block takes 16 MT rows of one adapter and 256 columns, a wave 64 of them. The matrix cores are given the rows of `up` as
// the left operand, ordered so that a lane ends up with 16 consecutive columns of its row (row m of tile j is column
// 16 (m / 4) + 4 j + m % 4 of the wave's 64): y is read and out written 16 bytes at a time, 128 consecutive bytes per row, with no pass
// through LDS. The inner dimension is [value | remainder], both against the same `up`.
template <int MT, bool PIECES, bool WIDE>
__global__ __launch_bounds__(256) void low_rank_expand_kernel(LowRankArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column_tiles = (a.N + 255) / 256;
  const RowTile tile = find_row_tile(a.offsets, a.groups, a.entries, static_cast<int>(blockIdx.x / column_tiles), 16 * MT);
  if (tile.group < 0) return;
  const int n0 = static_cast<int>(blockIdx.x % column_tiles) * 256 + wave * 64;
  if (n0 >= a.N) return;
  const int in_row = lane & 15, quarter = lane >> 4;
  f32x4 acc[MT][4] = {};
  if (tile.group < a.groups) {
    const uint16_t* up[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 16 * (in_row >> 2) + 4 * j + (in_row & 3);
      up[j] = a.up + tile.group * a.up_group + (n < a.N ? n : a.N - 1) * a.ldu;
    }
    const uint16_t* planes[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int row = 16 * t + in_row;
      planes[t] = a.planes + (static_cast<int64_t>(tile.first) + (row < tile.rows ? row : tile.rows - 1)) * (2 * a.padded) + 8 * quarter;
    }
    for (int e0 = 0; e0 < 2 * a.padded; e0 += 32) {
      bf16x8 fp[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) fp[t] = *reinterpret_cast<const bf16x8*>(planes[t] + e0);
      const int e = e0 + 8 * quarter, in_up = e < a.padded ? e : e - a.padded;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 fu = up_piece<PIECES>(up[j], in_up, a.rank);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fu, fp[t], acc[t][j], 0, 0, 0);
      }
    }
  }
  // Lane (row in_row, quarter): columns n0 + 16 quarter + 4 j + i in register i of tile j.
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int row = 16 * t + in_row;
    if (row >= tile.rows) continue;
    int to = a.order[tile.first + row];
    if (to >= a.rows) continue;
    const int n = n0 + 16 * quarter;
    const uint16_t* from = a.y != nullptr ? a.y + to * a.ldy + n : nullptr;
    uint16_t* out = a.out + to * a.ldo + n;
    if constexpr (WIDE) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (n + 8 * h >= a.N) continue;
        uint4 in = make_uint4(0, 0, 0, 0);
        if (from != nullptr) in = *reinterpret_cast<const uint4*>(from + 8 * h);
        uint32_t word[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4& four = acc[t][2 * h + (i >> 1)];
          const float low = __uint_as_float(word[i] << 16) + four[2 * (i & 1)];
          const float high = __uint_as_float(word[i] & 0xFFFF0000u) + four[2 * (i & 1) + 1];
          word[i] = bf16_bits_of(low) | bf16_bits_of(high) << 16;
        }
        *reinterpret_cast<uint4*>(out + 8 * h) = make_uint4(word[0], word[1], word[2], word[3]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        if (n + c >= a.N) continue;
        const float v = from != nullptr ? __uint_as_float(static_cast<uint32_t>(from[c]) << 16) : 0.0f;
        out[c] = static_cast<uint16_t>(bf16_bits_of(v + acc[t][c >> 2][c & 3]));
      }
    }
  }
}

// sum over a group's places of planes[p][e] q[order[p]][n] for all e < rank (value + remainder): out[g][e][n], or out[g][n][e] when
// transposed. The products are the weights' gradient of ep_grouped_tile.hpp with the planes as left operand. They are bound by
// reading q, and the groups alone make too few tiles to fill the card, so the places of every group are divided into chunks, each
// chunk writes its f32 sums to a matrix of its own, and this kernel adds a group's chunks in their order and rounds once.
// A block takes 64 columns of one group, 64 ranks at a time.
__global__ __launch_bounds__(256) void low_rank_finish_kernel(const float* __restrict__ parts, int chunk, int padded, int rank, const int32_t* __restrict__ offsets,
                                                              int width, uint16_t* __restrict__ out, int transposed) {
  __shared__ uint16_t turned[64][66];
  const int column_tiles = (width + 63) / 64;
  const int group = static_cast<int>(blockIdx.x / column_tiles), n0 = static_cast<int>(blockIdx.x % column_tiles) * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // The chunks of the groups before this one, and this one's.
  int before = 0;
  for (int g = lane; g < group; g += 64) before += (offsets[g + 1] - offsets[g] + chunk - 1) / chunk;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d);
  const int chunks = (offsets[group + 1] - offsets[group] + chunk - 1) / chunk;
  const int64_t matrix = static_cast<int64_t>(2 * padded) * width;
  const float* from = parts + before * matrix;
  const int n = n0 + lane;
  for (int e0 = 0; e0 < rank; e0 += 64) {
    const int ranks = rank - e0 < 64 ? rank - e0 : 64;
    for (int e = wave; e < ranks; e += 4) {
      float sum = 0.0f;
      if (n < width) {
        const float* high = from + static_cast<int64_t>(e0 + e) * width + n;
        const float* low = high + static_cast<int64_t>(padded) * width;
#pragma unroll 4
        for (int c = 0; c < chunks; ++c) sum += high[c * matrix] + low[c * matrix];
      }
      const uint16_t bits = static_cast<uint16_t>(bf16_bits_of(sum));
      if (transposed) turned[lane][e] = bits;
      else if (n < width) out[(static_cast<int64_t>(group) * rank + e0 + e) * width + n] = bits;
    }
    if (transposed) {
      __syncthreads();
      const int columns = width - n0 < 64 ? width - n0 : 64;
      for (int cell = threadIdx.x; cell < columns * ranks; cell += 256)
        out[(static_cast<int64_t>(group) * width + n0 + cell / ranks) * rank + e0 + cell % ranks] = turned[cell / ranks][cell % ranks];
      __syncthreads();
    }
  }
}

// Places per chunk: about 1024 tiles in all, at least 128 places each (a chunk of fewer does not outlast its own prologue).
static int reduce_chunk(int64_t entries, int64_t rank, int64_t width) {
  const int64_t tiles = ((width + kTile - 1) / kTile) * (((rank + 15) / 16 * 32 + kTile - 1) / kTile);
  const int64_t chunks = tiles >= 1024 ? 1 : 1024 / tiles;
  int64_t chunk = (entries + chunks - 1) / chunks;
  chunk = chunk < 128 ? 128 : (chunk + 63) / 64 * 64;
  return static_cast<int>(chunk < (1 << 30) ? chunk : 1 << 30);
}

static int64_t reduce_chunks(int64_t entries, int groups, int chunk) {       // the most there can be
  return entries / chunk + (groups < entries ? groups : entries);
}

static bool low_rank_valid(const int32_t* order, const int32_t* offsets, int64_t entries, int groups, int64_t rows, int64_t rank, int64_t width) {
  return order != nullptr && offsets != nullptr && entries > 0 && entries <= kMostEntries && groups > 0 && rows == entries && rank > 0 && rank <= 4096 && width > 0 &&
         width <= 0x3FFFFFFF / groups;
}

}  // namespace ep

extern "C" {

size_t ep_hip_low_rank_planes_bytes(int64_t entries, int64_t rank) {
  if (entries <= 0 || rank <= 0) return 0;
  return static_cast<size_t>(entries) * static_cast<size_t>((rank + 15) / 16 * 16) * 4;
}

int ep_hip_low_rank_shrink(const void* x_dev, int64_t ldx, const void* down_dev, int64_t ldd, int64_t down_group, const float* scale_dev, void* planes_dev,
                           const int32_t* order_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t rank, int64_t K, void* stream) {
  using namespace ep;
  if (x_dev == nullptr || down_dev == nullptr || planes_dev == nullptr || !low_rank_valid(order_dev, offsets_dev, entries, groups, entries, rank, K)) return EP_HIP_EINVAL;
  if (K % 8 != 0 || ldx % 8 != 0 || ldd % 8 != 0 || down_group % 8 != 0 || ldx < K || ldd < K || down_group < 0) return EP_HIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(x_dev) % 16 != 0 || reinterpret_cast<uintptr_t>(down_dev) % 16 != 0 || reinterpret_cast<uintptr_t>(planes_dev) % 16 != 0) return EP_HIP_EINVAL;
  GroupedArgs a = {};
  a.x = static_cast<const uint8_t*>(x_dev), a.w = static_cast<const uint8_t*>(down_dev), a.scale_x = scale_dev, a.y = planes_dev, a.row_of = order_dev, a.offsets = offsets_dev;
  a.ldx_bytes = ldx * 2, a.ldw_bytes = ldd * 2, a.group_bytes = down_group * 2, a.k_bytes = K * 2, a.ldy = (rank + 15) / 16 * 16 * 2;
  a.entries = static_cast<int>(entries), a.groups = groups, a.N = static_cast<int>(rank), a.x_rows = static_cast<int>(entries), a.out_kind = kOutBF16;
  return launch_stream_of<false, 1, 1, 4, true>(a, static_cast<hipStream_t>(stream));
}

int ep_hip_low_rank_expand(const void* planes_dev, const void* up_dev, int64_t ldu, int64_t up_group, const void* y_dev, int64_t ldy, void* out_dev, int64_t ldo,
                           const int32_t* order_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t rank, int64_t N, void* stream) {
  using namespace ep;
  if (planes_dev == nullptr || up_dev == nullptr || out_dev == nullptr || !low_rank_valid(order_dev, offsets_dev, entries, groups, entries, rank, N)) return EP_HIP_EINVAL;
  if (ldu < rank || up_group < 0 || ldo < N || (y_dev != nullptr && ldy < N) || reinterpret_cast<uintptr_t>(planes_dev) % 16 != 0) return EP_HIP_EINVAL;
  LowRankArgs a = {};
  a.planes = static_cast<const uint16_t*>(planes_dev), a.up = static_cast<const uint16_t*>(up_dev), a.y = static_cast<const uint16_t*>(y_dev);
  a.out = static_cast<uint16_t*>(out_dev), a.order = order_dev, a.offsets = offsets_dev;
  a.ldu = ldu, a.up_group = up_group, a.ldy = ldy, a.ldo = ldo;
  a.entries = static_cast<int>(entries), a.groups = groups, a.rank = static_cast<int>(rank), a.padded = static_cast<int>((rank + 15) / 16 * 16), a.N = static_cast<int>(N);
  a.rows = static_cast<int>(entries);
  auto in_pieces = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool pieces = in_pieces(up_dev, ldu) && up_group % 8 == 0 && rank % 8 == 0;
  const bool wide = in_pieces(out_dev, ldo) && N % 8 == 0 && (y_dev == nullptr || in_pieces(y_dev, ldy));
  const int64_t blocks = most_row_tiles(entries, groups, 16) * ((N + 255) / 256);
  if (blocks > 0x7FFFFFFF) return EP_HIP_EUNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (pieces && wide) hipLaunchKernelGGL((low_rank_expand_kernel<1, true, true>), grid, dim3(256), 0, s, a);
  else if (pieces) hipLaunchKernelGGL((low_rank_expand_kernel<1, true, false>), grid, dim3(256), 0, s, a);
  else if (wide) hipLaunchKernelGGL((low_rank_expand_kernel<1, false, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((low_rank_expand_kernel<1, false, false>), grid, dim3(256), 0, s, a);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

size_t ep_hip_low_rank_reduce_workspace(int64_t entries, int groups, int64_t rank, int64_t width) {
  using namespace ep;
  if (entries <= 0 || groups <= 0 || rank <= 0 || width <= 0) return 0;
  return static_cast<size_t>(reduce_chunks(entries, groups, reduce_chunk(entries, rank, width))) * static_cast<size_t>((rank + 15) / 16 * 32) * static_cast<size_t>(width) * 4;
}

int ep_hip_low_rank_reduce(const void* planes_dev, const void* q_dev, int64_t ldq, void* out_dev, int transposed, const int32_t* order_dev, const int32_t* offsets_dev,
                           int64_t entries, int groups, int64_t rank, int64_t width, void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace ep;
  if (planes_dev == nullptr || q_dev == nullptr || out_dev == nullptr || workspace_dev == nullptr) return EP_HIP_EINVAL;
  if (!low_rank_valid(order_dev, offsets_dev, entries, groups, entries, rank, width)) return EP_HIP_EINVAL;
  const int64_t readable = (width + 7) / 8 * 8;
  if (ldq < readable || ldq % 8 != 0 || reinterpret_cast<uintptr_t>(q_dev) % 16 != 0 || reinterpret_cast<uintptr_t>(planes_dev) % 16 != 0) return EP_HIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(workspace_dev) % 16 != 0 || workspace_bytes < ep_hip_low_rank_reduce_workspace(entries, groups, rank, width)) return EP_HIP_EINVAL;
  const int padded = static_cast<int>((rank + 15) / 16 * 16);
  TileArgs t = {};
  t.a = static_cast<const uint8_t*>(planes_dev), t.b = static_cast<const uint8_t*>(q_dev), t.y = workspace_dev, t.row_of = order_dev, t.offsets = offsets_dev;
  t.lda_bytes = padded * int64_t{4}, t.ldb_bytes = ldq * 2, t.ldy = width, t.group_y = 2 * padded * width;
  t.entries = static_cast<int>(entries), t.groups = groups, t.x_rows = static_cast<int>(entries), t.out_kind = kOutF32;
  t.rows = 2 * padded, t.columns = static_cast<int>(width), t.chunk = reduce_chunk(entries, rank, width);
  const int64_t blocks = reduce_chunks(entries, groups, t.chunk) * ((t.rows + kTile - 1) / kTile) * ((width + kTile - 1) / kTile);
  const int64_t finish = groups * ((width + 63) / 64);
  if (blocks > 0x7FFFFFFF || finish > 0x7FFFFFFF) return EP_HIP_EUNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL((grouped_tile_kernel<false, kGradWeight, true, true>), dim3(static_cast<unsigned>(blocks)), dim3(kTileThreads), 0, s, t);
  EP_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(low_rank_finish_kernel, dim3(static_cast<unsigned>(finish)), dim3(256), 0, s, static_cast<const float*>(workspace_dev), t.chunk, padded,
                     static_cast<int>(rank), offsets_dev, static_cast<int>(width), static_cast<uint16_t*>(out_dev), transposed);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

}  // extern "C"

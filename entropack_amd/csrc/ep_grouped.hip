// Products of grouped rows with the weight of their group (a mixture's experts), and their gradients.
//
//   y[p]  = x[rows[p]] . w[g]^T (+ bias[g])                 few rows per group: grouped_stream_kernel (ep_grouped.hpp), else tiles
//   dx[p] = dy[p] . w[g]                                    tiles: grouped_tile_kernel, grouped_wide_kernel (ep_grouped_tile.hpp)
//   dw[g] = sum_p dy[p]^T x[rows[p]]                        tiles
//   db[g] = sum_p dy[p]                                     grouped_column_sums_kernel
#include "ep_grouped_tile.hpp"

namespace ep {

// Sums of a group's rows, column by column: a block takes 128 columns of one group, a lane two of them, its sixteen waves every
// sixteenth row each, eight rows under way at a time. The partial sums are added in a fixed order. Bound by reading dy where
// the groups make enough blocks: 16384 rows of 4096, 8 groups, 21.8 us (134 MB, 6.2 TB/s); one group, 32 blocks, 121 us. Four waves
// with one column per lane and one row under way took 154 and 1142 us; 72 rows of 1408 in 64 groups take 3.8 us (2.5 with those).
constexpr int kSumWaves = 16, kSumColumns = 128, kSumTogether = 8;

__global__ __launch_bounds__(64 * kSumWaves) void grouped_column_sums_kernel(const uint16_t* __restrict__ dy, int64_t lddy, const int32_t* __restrict__ offsets, int N,
                                                                             void* __restrict__ out, int out_kind, int pairs) {
  __shared__ float sums[kSumWaves][kSumColumns];
  const int column_tiles = (N + kSumColumns - 1) / kSumColumns;
  const int group = static_cast<int>(blockIdx.x / column_tiles);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = static_cast<int>(blockIdx.x % column_tiles) * kSumColumns + 2 * lane;
  const int first = offsets[group], last = offsets[group + 1];
  const uint16_t* column = dy + (n < N ? n : 0);
  const bool second = n + 1 < N;
  float low = 0.0f, high = 0.0f;
  for (int p = first + wave; p < last; p += kSumWaves * kSumTogether) {
    uint32_t held[kSumTogether];                 // rows past the last read it again and count as zero
#pragma unroll
    for (int i = 0; i < kSumTogether; ++i) {
      const int row = p + i * kSumWaves;
      const uint16_t* at = column + (row < last ? row : last - 1) * lddy;
      held[i] = pairs ? *reinterpret_cast<const uint32_t*>(at) : at[0] | static_cast<uint32_t>(at[second ? 1 : 0]) << 16;
    }
#pragma unroll
    for (int i = 0; i < kSumTogether; ++i) {
      const bool counts = p + i * kSumWaves < last;
      low += counts ? __uint_as_float(held[i] << 16) : 0.0f;
      high += counts ? __uint_as_float(held[i] & 0xFFFF0000u) : 0.0f;
    }
  }
  sums[wave][2 * lane] = low;
  sums[wave][2 * lane + 1] = high;
  __syncthreads();
  const int mine = static_cast<int>(blockIdx.x % column_tiles) * kSumColumns + static_cast<int>(threadIdx.x);
  if (threadIdx.x < kSumColumns && mine < N) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kSumWaves; ++w) sum += sums[w][threadIdx.x];
    store_out(out, out_kind, static_cast<int64_t>(group) * N + mine, sum);
  }
}

// ---- checks that every entry point makes --------------------------------------------------------------------------------------

static bool groups_valid(const int32_t* offsets, int64_t entries, int groups, const int32_t* row_of, int64_t x_rows) {
  if (offsets == nullptr || entries <= 0 || groups <= 0 || entries > kMostEntries) return false;
  return row_of != nullptr ? x_rows >= 1 && x_rows <= 0x7FFFFFFF : x_rows >= entries && x_rows <= 0x7FFFFFFF;
}

static bool kind_valid(int kind) { return kind == kOutBF16 || kind == kOutF16 || kind == kOutF32; }

static bool sizes_valid(int64_t N, int64_t K, int groups) {
  return N > 0 && K > 0 && K <= 0x3FFFFF00 && N <= 0x3FFFFF00 / groups;
}

// `rows` of `element_bytes` x K, `ld` elements apart, read in whole pieces of 16 bytes.
static bool rows_in_pieces(const void* base, int64_t ld, int64_t K, int element_bytes) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld >= K && (ld * element_bytes) % 16 == 0 && (K * element_bytes) % 16 == 0;
}

static int current_compute_units(int& units) {
  int device = 0;
  EP_HIP_TRY(hipGetDevice(&device));
  EP_HIP_TRY(hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device));
  return EP_HIP_OK;
}

// `tile` rows and columns per block: the 128 x 128 kernel or the 256 x 256 one.
template <bool INT8, int MODE, bool GATHER = true>
static int launch_tile(TileArgs t, int64_t row_tiles, int tile, hipStream_t s) {
  const int64_t blocks = tile == kWideTile ? wide_blocks(row_tiles, t.columns, t.compute_units) : row_tiles * ((t.columns + kTile - 1) / kTile);
  if (!launch_fits(blocks, kTileThreads)) return EP_HIP_EUNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool whole = t.inner % 256 == 0 && (MODE == kForward || t.columns % tile == 0);
  constexpr bool kAlways = MODE == kGradWeight;             // a group's rows are of any number
  if (tile == kWideTile) {
    if (whole && !kAlways) hipLaunchKernelGGL((grouped_wide_kernel<INT8, MODE, kAlways, GATHER>), grid, dim3(kTileThreads), 0, s, t);
    else hipLaunchKernelGGL((grouped_wide_kernel<INT8, MODE, true, GATHER>), grid, dim3(kTileThreads), 0, s, t);
  } else {
    if (whole && !kAlways) hipLaunchKernelGGL((grouped_tile_kernel<INT8, MODE, kAlways, GATHER>), grid, dim3(kTileThreads), 0, s, t);
    else hipLaunchKernelGGL((grouped_tile_kernel<INT8, MODE, true, GATHER>), grid, dim3(kTileThreads), 0, s, t);
  }
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

// Rows and columns per block of a product of grouped rows (forward, rows' gradient). The 256 x 256 tiles read each operand half
// as often as the 128 x 128 ones, but want half the device's compute units busy, tiles at least half full, and an inner dimension of 2 KB that pays for
// the longer ends of a tile. us, 128 and 256: 8 groups of 4096 x 4096, 192 rows per group 80 and 81, 256 130 and 110, 1024 332
// and 283; 64 of 2048 x 1408, 96 rows 118 and 122, 128 rows 142 and 124, 512 rows 396 and 289. 8 groups, 1024 rows, inner 512
// and 4096 columns: 58 and 62; inner 4096 and 512 columns (64 tiles): 66 and 72.
static int product_tile(int64_t entries, int groups, int64_t columns, int64_t inner_bytes, int compute_units) {
  const bool wide = entries / groups >= kWideTile / 2 && entries * columns / (kWideTile * kWideTile) >= compute_units / 2 && inner_bytes >= 2048;
  return wide ? kWideTile : kTile;
}

// Of a weights' gradient, whose inner dimension is a group's rows. 8 groups of 4096 x 4096, 256 rows per group 136 and 159 us, 512
// 209 and 220, 1024 357 and 339, 2048 594 and 557; 64 of 2048 x 1408, 512 rows 295 and 322, 1024 539 and 519.
static int grad_weight_tile(int64_t entries, int groups) { return entries / groups >= 768 ? kWideTile : kTile; }

// Places per chunk of a weights' gradient, 0 for a group's places at once. A tile takes 0.62 us per 64 places, however few tiles there
// are: with fewer tiles than compute units and long groups the places are divided so that about 512 blocks run, at least 512
// places each, and the chunks' f32 sums are added by a second kernel. us, at once and in chunks: 2 weights of 128 x 128, 32768
// rows each, 316 and 18; of 512 x 512, 319 and 81; one of 2048 x 1024, 8192 rows, 85 and 61; 8 of 1024 x 512, 2048 rows, 37 and
// 37; 8 of 512 x 512, 1024 rows, 19 and 30.
static int grad_weight_chunk(int64_t entries, int groups, int64_t N, int64_t K) {
  const int64_t tiles = groups * ((N + kTile - 1) / kTile) * ((K + kTile - 1) / kTile);
  if (tiles >= 256 || entries / groups < 4096) return 0;
  const int64_t chunk = entries * tiles / groups / 512;       // entries / groups places in 512 / tiles chunks
  return static_cast<int>(chunk < 512 ? 512 : (chunk + 63) / 64 * 64);
}

// out[g] = the sum of g's chunks, in their order, rounded once: a thread per element.
__global__ __launch_bounds__(256) void grouped_sum_chunks_kernel(const float* __restrict__ parts, int chunk, const int32_t* __restrict__ offsets, int N, int K,
                                                                 void* __restrict__ out, int64_t ld, int64_t group_out, int out_kind, int blocks_per_group) {
  const int group = static_cast<int>(blockIdx.x) / blocks_per_group, lane = threadIdx.x & 63;
  int before = 0;
  for (int g0 = 0; g0 < group; g0 += 64) {
    const int g = g0 + lane;
    before += __builtin_amdgcn_readlane(wave_inclusive_sum(g < group ? (offsets[g + 1] - offsets[g] + chunk - 1) / chunk : 0), 63);
  }
  const int chunks = (offsets[group + 1] - offsets[group] + chunk - 1) / chunk;
  const int64_t size = static_cast<int64_t>(N) * K, at = static_cast<int64_t>(static_cast<int>(blockIdx.x) % blocks_per_group) * 256 + threadIdx.x;
  if (at >= size) return;
  const float* from = parts + before * size + at;
  float sum = 0.0f;
#pragma unroll 8
  for (int c = 0; c < chunks; ++c) sum += from[c * size];
  store_out(out, out_kind, group * group_out + at / K * ld + at % K, sum);
}

template <bool INT8>
static int launch_grouped(const GroupedArgs& a, hipStream_t s) {
  // Few rows per group: the weights' stream. About one row per group: blocks of 16 weight rows; one token, two of eight experts 4096 x
  // 4096, 13.2 us (67 MB, 10.8 us at 6.2 TB/s) and 14.6 in int8, which the host's call bounds; 18 tokens, four of 64 experts 1408 x 2048, 31
  // us with the weights partly in the last-level cache, 56 from memory (243 MB, 4.3 TB/s), 33 in int8. From five rows on
  // 32 rows by 32 weight rows (64 tokens, two of eight, 62 us; 256 tokens, four of 64, 75), from 24 on by 64 (128 tokens, two of
  // eight, 61 us against 73; 512 tokens, four of 64, 98 against 96). From 48 on the 128 x 128 tiles: 256 tokens, two of eight, 82 us
  // against 91; 1024 tokens, four of 64, 106 against 135.
  const int mean = a.entries / a.groups;
  if (mean < 5) return launch_stream_of<INT8, 1, 1, 4, false>(a, s);
  if (mean < 24) return launch_stream_of<INT8, 2, 2, 2, false>(a, s);
  if (mean < 48) return launch_stream_of<INT8, 2, 4, 2, false>(a, s);
  TileArgs t = {};
  t.a = a.x, t.b = a.w, t.scale_x = a.scale_x, t.scale_w = a.scale_w, t.bias = a.bias, t.y = a.y, t.row_of = a.row_of, t.offsets = a.offsets;
  t.lda_bytes = a.ldx_bytes, t.ldb_bytes = a.ldw_bytes, t.group_b_bytes = a.group_bytes, t.ldy = a.ldy;
  t.entries = a.entries, t.groups = a.groups, t.x_rows = a.x_rows, t.out_kind = a.out_kind;
  t.columns = a.N, t.inner = static_cast<int>(a.k_bytes);
  if (const int status = current_compute_units(t.compute_units)) return status;
  const int tile = product_tile(a.entries, a.groups, a.N, a.k_bytes, t.compute_units);
  return launch_tile<INT8, kForward>(t, most_row_tiles(a.entries, a.groups, tile), tile, s);
}

}  // namespace ep

extern "C" {

int ep_hip_grouped_gemm_bf16(const void* x_dev, int64_t ldx, int64_t x_rows, const void* w_dev, int64_t ldw, int64_t w_group, const void* bias_dev, void* y_dev,
                             int64_t ldy, int out_kind, const int32_t* rows_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t N,
                             int64_t K, void* stream) {
  using namespace ep;
  if (x_dev == nullptr || w_dev == nullptr || y_dev == nullptr || !groups_valid(offsets_dev, entries, groups, rows_dev, x_rows)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || ldy < N) return EP_HIP_EINVAL;
  if (!rows_in_pieces(x_dev, ldx, K, 2) || !rows_in_pieces(w_dev, ldw, K, 2) || w_group % 8 != 0 || w_group < 0) return EP_HIP_EINVAL;
  GroupedArgs a = {};
  a.x = static_cast<const uint8_t*>(x_dev), a.w = static_cast<const uint8_t*>(w_dev), a.bias = bias_dev, a.y = y_dev, a.row_of = rows_dev, a.offsets = offsets_dev;
  a.ldx_bytes = ldx * 2, a.ldw_bytes = ldw * 2, a.group_bytes = w_group * 2, a.k_bytes = K * 2, a.ldy = ldy;
  a.entries = static_cast<int>(entries), a.groups = groups, a.N = static_cast<int>(N), a.x_rows = static_cast<int>(x_rows), a.out_kind = out_kind;
  return launch_grouped<false>(a, static_cast<hipStream_t>(stream));
}

int ep_hip_grouped_gemm_i8(const int8_t* x_dev, int64_t ldx, int64_t x_rows, const int8_t* w_dev, int64_t ldw, int64_t w_group, const float* scale_x_dev,
                           const float* scale_w_dev, const void* bias_dev, void* y_dev, int64_t ldy, int out_kind, const int32_t* rows_dev,
                           const int32_t* offsets_dev, int64_t entries, int groups, int64_t N, int64_t K, void* stream) {
  using namespace ep;
  if (x_dev == nullptr || w_dev == nullptr || y_dev == nullptr || scale_x_dev == nullptr || scale_w_dev == nullptr) return EP_HIP_EINVAL;
  if (!groups_valid(offsets_dev, entries, groups, rows_dev, x_rows)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || ldy < N) return EP_HIP_EINVAL;
  if (!rows_in_pieces(x_dev, ldx, K, 1) || !rows_in_pieces(w_dev, ldw, K, 1) || w_group % 16 != 0 || w_group < 0) return EP_HIP_EINVAL;
  GroupedArgs a = {};
  a.x = reinterpret_cast<const uint8_t*>(x_dev), a.w = reinterpret_cast<const uint8_t*>(w_dev), a.scale_x = scale_x_dev, a.scale_w = scale_w_dev;
  a.bias = bias_dev, a.y = y_dev, a.row_of = rows_dev, a.offsets = offsets_dev;
  a.ldx_bytes = ldx, a.ldw_bytes = ldw, a.group_bytes = w_group, a.k_bytes = K, a.ldy = ldy;
  a.entries = static_cast<int>(entries), a.groups = groups, a.N = static_cast<int>(N), a.x_rows = static_cast<int>(x_rows), a.out_kind = out_kind;
  return launch_grouped<true>(a, static_cast<hipStream_t>(stream));
}

int ep_hip_grouped_grad_rows_bf16(const void* dy_dev, int64_t lddy, const void* w_dev, int64_t ldw, int64_t w_group, void* dx_dev, int64_t lddx, int out_kind,
                                  const int32_t* order_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t N, int64_t K, void* stream) {
  using namespace ep;
  if (dy_dev == nullptr || w_dev == nullptr || dx_dev == nullptr || !groups_valid(offsets_dev, entries, groups, order_dev, entries)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || lddx < K) return EP_HIP_EINVAL;
  if (!rows_in_pieces(dy_dev, lddy, (N + 7) / 8 * 8, 2) || !rows_in_pieces(w_dev, ldw, K, 2) || w_group % 8 != 0 || w_group < 0) return EP_HIP_EINVAL;
  TileArgs t = {};
  t.a = static_cast<const uint8_t*>(dy_dev), t.b = static_cast<const uint8_t*>(w_dev), t.y = dx_dev, t.order = order_dev, t.offsets = offsets_dev;
  t.lda_bytes = lddy * 2, t.ldb_bytes = ldw * 2, t.group_b_bytes = w_group * 2, t.ldy = lddx;
  t.entries = static_cast<int>(entries), t.groups = groups, t.x_rows = static_cast<int>(entries), t.out_kind = out_kind;
  t.columns = static_cast<int>(K), t.inner = static_cast<int>(N * 2);
  if (const int status = current_compute_units(t.compute_units)) return status;
  const int tile = product_tile(entries, groups, K, t.inner, t.compute_units);
  return launch_tile<false, kGradRows>(t, most_row_tiles(entries, groups, tile), tile, static_cast<hipStream_t>(stream));
}

size_t ep_hip_grouped_grad_weight_workspace(int64_t entries, int groups, int64_t N, int64_t K) {
  using namespace ep;
  if (entries <= 0 || groups <= 0 || !sizes_valid(N, K, groups)) return 0;
  const int chunk = grad_weight_chunk(entries, groups, N, K);
  return chunk == 0 ? 0 : static_cast<size_t>(most_chunks(entries, groups, chunk)) * static_cast<size_t>(N) * static_cast<size_t>(K) * 4;
}

int ep_hip_grouped_grad_weight_bf16(const void* dy_dev, int64_t lddy, const void* x_dev, int64_t ldx, int64_t x_rows, void* dw_dev, int64_t lddw, int64_t dw_group,
                                    int out_kind, const int32_t* rows_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t N,
                                    int64_t K, void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace ep;
  if (dy_dev == nullptr || x_dev == nullptr || dw_dev == nullptr || !groups_valid(offsets_dev, entries, groups, rows_dev, x_rows)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || lddw < K || dw_group < 0) return EP_HIP_EINVAL;
  if (!rows_in_pieces(dy_dev, lddy, N, 2) || !rows_in_pieces(x_dev, ldx, K, 2)) return EP_HIP_EINVAL;
  TileArgs t = {};
  t.a = static_cast<const uint8_t*>(dy_dev), t.b = static_cast<const uint8_t*>(x_dev), t.y = dw_dev, t.row_of = rows_dev, t.offsets = offsets_dev;
  t.lda_bytes = lddy * 2, t.ldb_bytes = ldx * 2, t.ldy = lddw, t.group_y = dw_group;
  t.entries = static_cast<int>(entries), t.groups = groups, t.x_rows = static_cast<int>(x_rows), t.out_kind = out_kind;
  t.rows = static_cast<int>(N), t.columns = static_cast<int>(K);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int chunk = grad_weight_chunk(entries, groups, N, K)) {
    if (workspace_dev == nullptr || reinterpret_cast<uintptr_t>(workspace_dev) % 16 != 0 || workspace_bytes < ep_hip_grouped_grad_weight_workspace(entries, groups, N, K))
      return EP_HIP_EINVAL;
    t.y = workspace_dev, t.ldy = K, t.group_y = N * K, t.out_kind = kOutF32, t.chunk = chunk;
    const int64_t row_tiles = most_chunks(entries, groups, chunk) * ((N + kTile - 1) / kTile), per_group = (N * K + 255) / 256;
    const int status = rows_dev != nullptr ? launch_tile<false, kGradWeight, true>(t, row_tiles, kTile, s) : launch_tile<false, kGradWeight, false>(t, row_tiles, kTile, s);
    if (status != EP_HIP_OK) return status;
    hipLaunchKernelGGL(grouped_sum_chunks_kernel, dim3(static_cast<unsigned>(groups * per_group)), dim3(256), 0, s, static_cast<const float*>(workspace_dev), chunk, offsets_dev,
                       static_cast<int>(N), static_cast<int>(K), dw_dev, lddw, dw_group, out_kind, static_cast<int>(per_group));
    EP_HIP_TRY(hipGetLastError());
    return EP_HIP_OK;
  }
  if (const int status = current_compute_units(t.compute_units)) return status;
  const int tile = grad_weight_tile(entries, groups);
  const int64_t row_tiles = static_cast<int64_t>(groups) * ((N + tile - 1) / tile);
  return rows_dev != nullptr ? launch_tile<false, kGradWeight, true>(t, row_tiles, tile, s) : launch_tile<false, kGradWeight, false>(t, row_tiles, tile, s);
}

int ep_hip_grouped_column_sums_bf16(const void* dy_dev, int64_t lddy, const int32_t* offsets_dev, int groups, int64_t N, void* out_dev, int out_kind, void* stream) {
  using namespace ep;
  if (dy_dev == nullptr || offsets_dev == nullptr || out_dev == nullptr || groups <= 0 || N <= 0 || N > 0x7FFFFFFF / groups || lddy < N || !kind_valid(out_kind))
    return EP_HIP_EINVAL;
  const int64_t blocks = groups * ((N + kSumColumns - 1) / kSumColumns);
  if (!launch_fits(blocks, 64 * kSumWaves)) return EP_HIP_EUNSUPPORTED;
  const bool pairs = reinterpret_cast<uintptr_t>(dy_dev) % 4 == 0 && lddy % 2 == 0 && N % 2 == 0;
  hipLaunchKernelGGL(grouped_column_sums_kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * kSumWaves), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(dy_dev), lddy, offsets_dev, static_cast<int>(N), out_dev, out_kind, pairs ? 1 : 0);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

}  // extern "C"

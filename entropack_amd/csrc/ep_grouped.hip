// Products of grouped rows with the weight of their group (a mixture's experts), and their gradients.
//
//   y[p]  = x[order[p] / k] . w[g]^T (+ bias[g])            grouped_stream_kernel (ep_grouped.hpp)
//   dx[p] = dy[p] . w[g]                                    grouped_simple_kernel
//   dw[g] = sum_p dy[p]^T x[order[p] / k]                   grouped_simple_kernel
//   db[g] = sum_p dy[p]                                     grouped_column_sums_kernel
#include "ep_grouped.hpp"

namespace ep {

// The two gradients in their simplest form: 64 x 64 tiles, four waves of 32 x 32, elements brought into the order of the
// matrix-core fragments one by one on their way to LDS.
// WEIGHT = false: rows = places of a group, columns = K, summed over N.   WEIGHT = true: rows = N, columns = K, summed over places.
template <bool WEIGHT>
__global__ __launch_bounds__(256) void grouped_simple_kernel(const uint16_t* __restrict__ dy, int64_t lddy, const uint16_t* __restrict__ other, int64_t ld_other,
                                                             int64_t other_group, void* __restrict__ out, int64_t ld_out, int64_t out_group, int out_kind,
                                                             const int32_t* __restrict__ order, const int32_t* __restrict__ offsets, int entries, int groups,
                                                             int per_row, int x_rows, int N, int K) {
  constexpr int kPitch = 32 + 8;
  __shared__ __align__(16) uint16_t tile_a[64 * kPitch];
  __shared__ __align__(16) uint16_t tile_b[64 * kPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column_tiles = (K + 63) / 64;
  const int k0 = static_cast<int>(blockIdx.x % column_tiles) * 64;
  const int at = static_cast<int>(blockIdx.x / column_tiles);
  int group, first, rows, m0 = 0, inner;
  if constexpr (WEIGHT) {
    const int row_tiles = (N + 63) / 64;
    group = at / row_tiles;
    m0 = at % row_tiles * 64;
    first = offsets[group];
    inner = offsets[group + 1] - first;
    rows = N - m0 < 64 ? N - m0 : 64;
  } else {
    const RowTile tile = find_row_tile(offsets, groups, entries, at, 64);
    if (tile.group < 0) return;
    group = tile.group;
    first = tile.first;
    rows = tile.rows;
    inner = group < groups ? N : 0;
  }
  auto source = [&](int place) {
    if (order == nullptr) return place;
    const int row = static_cast<int>(static_cast<uint32_t>(order[place]) / static_cast<uint32_t>(per_row));
    return row < x_rows ? row : x_rows - 1;
  };
  f32x16 acc = {};
  for (int i0 = 0; i0 < inner; i0 += 32) {
    __syncthreads();
    for (int cell = threadIdx.x; cell < 64 * 32; cell += 256) {
      // dy is read along its columns, `other` along K: neighbouring threads take neighbouring elements of memory.
      const int r = WEIGHT ? cell % 64 : cell / 32, i = WEIGHT ? cell / 64 : cell % 32;
      uint16_t v = 0;
      if (r < rows && i0 + i < inner) v = WEIGHT ? dy[(first + i0 + i) * lddy + m0 + r] : dy[(first + r) * lddy + i0 + i];
      tile_a[r * kPitch + i] = v;
      const int c = cell % 64, b = cell / 64;
      uint16_t u = 0;
      if (k0 + c < K && i0 + b < inner) u = WEIGHT ? other[source(first + i0 + b) * ld_other + k0 + c] : other[group * other_group + (i0 + b) * ld_other + k0 + c];
      tile_b[c * kPitch + b] = u;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bf16x8 fa = *reinterpret_cast<const bf16x8*>(tile_a + ((wave >> 1) * 32 + (lane & 31)) * kPitch + s * 16 + (lane >> 5) * 8);
      const bf16x8 fb = *reinterpret_cast<const bf16x8*>(tile_b + ((wave & 1) * 32 + (lane & 31)) * kPitch + s * 16 + (lane >> 5) * 8);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb, acc, 0, 0, 0);
    }
  }
  const int column = k0 + (wave & 1) * 32 + (lane & 31);
  if (column >= K) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = (wave >> 1) * 32 + 8 * (r / 4) + 4 * (lane >> 5) + (r % 4);
    if (row >= rows) continue;
    int64_t to;
    if constexpr (WEIGHT) to = group * out_group + (m0 + row) * ld_out + column;
    else to = static_cast<int64_t>(order != nullptr ? order[first + row] : first + row) * ld_out + column;
    store_out(out, out_kind, to, acc[r]);
  }
}

// Sums of a group's rows, column by column: a block takes 64 columns of one group, its four waves every fourth row.
__global__ __launch_bounds__(256) void grouped_column_sums_kernel(const uint16_t* __restrict__ dy, int64_t lddy, const int32_t* __restrict__ offsets, int N,
                                                                  void* __restrict__ out, int out_kind) {
  __shared__ float sums[4][64];
  const int column_tiles = (N + 63) / 64;
  const int group = static_cast<int>(blockIdx.x / column_tiles);
  const int n = static_cast<int>(blockIdx.x % column_tiles) * 64 + (threadIdx.x & 63);
  const int wave = threadIdx.x >> 6;
  const int first = offsets[group], last = offsets[group + 1];
  float sum = 0.0f;
  if (n < N) {
    for (int p = first + wave; p < last; p += 4) sum += __uint_as_float(static_cast<uint32_t>(dy[p * lddy + n]) << 16);
  }
  sums[wave][threadIdx.x & 63] = sum;
  __syncthreads();
  if (wave == 0 && n < N)
    store_out(out, out_kind, static_cast<int64_t>(group) * N + n, (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]));
}

// ---- checks that every entry point makes --------------------------------------------------------------------------------------

static bool groups_valid(const int32_t* offsets, int64_t entries, int groups, const int32_t* order, int per_row, int64_t x_rows) {
  if (offsets == nullptr || entries <= 0 || groups <= 0 || entries > kMostEntries) return false;
  if (order != nullptr) return per_row >= 1 && x_rows >= 1 && x_rows <= 0x7FFFFFFF;
  return x_rows >= entries;
}

static bool kind_valid(int kind) { return kind == kOutBF16 || kind == kOutF16 || kind == kOutF32; }

static bool sizes_valid(int64_t N, int64_t K, int groups) {
  return N > 0 && K > 0 && K <= 0x3FFFFFFF && N <= 0x7FFFFFFF / groups;
}

// `rows` of `element_bytes` x K, `ld` elements apart, read in whole pieces of 16 bytes.
static bool rows_in_pieces(const void* base, int64_t ld, int64_t K, int element_bytes) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && ld >= K && (ld * element_bytes) % 16 == 0 && (K * element_bytes) % 16 == 0;
}

template <bool INT8>
static int launch_grouped(const GroupedArgs& a, hipStream_t s) {
  return launch_stream_of<INT8, 1, 2, 4, false>(a, s);
}

}  // namespace ep

extern "C" {

int ep_hip_grouped_gemm_bf16(const void* x_dev, int64_t ldx, int64_t x_rows, const void* w_dev, int64_t ldw, int64_t w_group, const void* bias_dev, void* y_dev,
                             int64_t ldy, int out_kind, const int32_t* order_dev, int per_row, const int32_t* offsets_dev, int64_t entries, int groups, int64_t N,
                             int64_t K, void* stream) {
  using namespace ep;
  if (x_dev == nullptr || w_dev == nullptr || y_dev == nullptr || !groups_valid(offsets_dev, entries, groups, order_dev, per_row, x_rows)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || ldy < N) return EP_HIP_EINVAL;
  if (!rows_in_pieces(x_dev, ldx, K, 2) || !rows_in_pieces(w_dev, ldw, K, 2) || w_group % 8 != 0 || w_group < 0) return EP_HIP_EINVAL;
  GroupedArgs a = {};
  a.x = static_cast<const uint8_t*>(x_dev), a.w = static_cast<const uint8_t*>(w_dev), a.bias = bias_dev, a.y = y_dev, a.order = order_dev, a.offsets = offsets_dev;
  a.ldx_bytes = ldx * 2, a.ldw_bytes = ldw * 2, a.group_bytes = w_group * 2, a.k_bytes = K * 2, a.ldy = ldy;
  a.entries = static_cast<int>(entries), a.groups = groups, a.N = static_cast<int>(N), a.per_row = per_row, a.x_rows = static_cast<int>(x_rows), a.out_kind = out_kind;
  return launch_grouped<false>(a, static_cast<hipStream_t>(stream));
}

int ep_hip_grouped_gemm_i8(const int8_t* x_dev, int64_t ldx, int64_t x_rows, const int8_t* w_dev, int64_t ldw, int64_t w_group, const float* scale_x_dev,
                           const float* scale_w_dev, const void* bias_dev, void* y_dev, int64_t ldy, int out_kind, const int32_t* order_dev, int per_row,
                           const int32_t* offsets_dev, int64_t entries, int groups, int64_t N, int64_t K, void* stream) {
  using namespace ep;
  if (x_dev == nullptr || w_dev == nullptr || y_dev == nullptr || scale_x_dev == nullptr || scale_w_dev == nullptr) return EP_HIP_EINVAL;
  if (!groups_valid(offsets_dev, entries, groups, order_dev, per_row, x_rows)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || ldy < N) return EP_HIP_EINVAL;
  if (!rows_in_pieces(x_dev, ldx, K, 1) || !rows_in_pieces(w_dev, ldw, K, 1) || w_group % 16 != 0 || w_group < 0) return EP_HIP_EINVAL;
  GroupedArgs a = {};
  a.x = reinterpret_cast<const uint8_t*>(x_dev), a.w = reinterpret_cast<const uint8_t*>(w_dev), a.scale_x = scale_x_dev, a.scale_w = scale_w_dev;
  a.bias = bias_dev, a.y = y_dev, a.order = order_dev, a.offsets = offsets_dev;
  a.ldx_bytes = ldx, a.ldw_bytes = ldw, a.group_bytes = w_group, a.k_bytes = K, a.ldy = ldy;
  a.entries = static_cast<int>(entries), a.groups = groups, a.N = static_cast<int>(N), a.per_row = per_row, a.x_rows = static_cast<int>(x_rows), a.out_kind = out_kind;
  return launch_grouped<true>(a, static_cast<hipStream_t>(stream));
}

int ep_hip_grouped_grad_rows_bf16(const void* dy_dev, int64_t lddy, const void* w_dev, int64_t ldw, int64_t w_group, void* dx_dev, int64_t lddx, int out_kind,
                                  const int32_t* order_dev, const int32_t* offsets_dev, int64_t entries, int groups, int64_t N, int64_t K, void* stream) {
  using namespace ep;
  if (dy_dev == nullptr || w_dev == nullptr || dx_dev == nullptr || !groups_valid(offsets_dev, entries, groups, order_dev, 1, entries)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || lddx < K) return EP_HIP_EINVAL;
  if (!rows_in_pieces(dy_dev, lddy, (N + 7) / 8 * 8, 2) || !rows_in_pieces(w_dev, ldw, K, 2) || w_group % 8 != 0 || w_group < 0) return EP_HIP_EINVAL;
  const int64_t blocks = most_row_tiles(entries, groups, 64) * ((K + 63) / 64);
  if (blocks > 0x7FFFFFFF) return EP_HIP_EUNSUPPORTED;
  hipLaunchKernelGGL(grouped_simple_kernel<false>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(dy_dev), lddy, static_cast<const uint16_t*>(w_dev), ldw, w_group, dx_dev, lddx, int64_t{0}, out_kind, order_dev,
                     offsets_dev, static_cast<int>(entries), groups, 1, static_cast<int>(entries), static_cast<int>(N), static_cast<int>(K));
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

int ep_hip_grouped_grad_weight_bf16(const void* dy_dev, int64_t lddy, const void* x_dev, int64_t ldx, int64_t x_rows, void* dw_dev, int64_t lddw, int64_t dw_group,
                                    int out_kind, const int32_t* order_dev, int per_row, const int32_t* offsets_dev, int64_t entries, int groups, int64_t N,
                                    int64_t K, void* stream) {
  using namespace ep;
  if (dy_dev == nullptr || x_dev == nullptr || dw_dev == nullptr || !groups_valid(offsets_dev, entries, groups, order_dev, per_row, x_rows)) return EP_HIP_EINVAL;
  if (!sizes_valid(N, K, groups) || !kind_valid(out_kind) || lddw < K || dw_group < 0) return EP_HIP_EINVAL;
  if (!rows_in_pieces(dy_dev, lddy, N, 2) || !rows_in_pieces(x_dev, ldx, K, 2)) return EP_HIP_EINVAL;
  const int64_t blocks = static_cast<int64_t>(groups) * ((N + 63) / 64) * ((K + 63) / 64);
  if (blocks > 0x7FFFFFFF) return EP_HIP_EUNSUPPORTED;
  hipLaunchKernelGGL(grouped_simple_kernel<true>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(dy_dev), lddy, static_cast<const uint16_t*>(x_dev), ldx, int64_t{0}, dw_dev, lddw, dw_group, out_kind, order_dev,
                     offsets_dev, static_cast<int>(entries), groups, per_row, static_cast<int>(x_rows), static_cast<int>(N), static_cast<int>(K));
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

int ep_hip_grouped_column_sums_bf16(const void* dy_dev, int64_t lddy, const int32_t* offsets_dev, int groups, int64_t N, void* out_dev, int out_kind, void* stream) {
  using namespace ep;
  if (dy_dev == nullptr || offsets_dev == nullptr || out_dev == nullptr || groups <= 0 || N <= 0 || N > 0x7FFFFFFF / groups || lddy < N || !kind_valid(out_kind))
    return EP_HIP_EINVAL;
  const int64_t blocks = groups * ((N + 63) / 64);
  hipLaunchKernelGGL(grouped_column_sums_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(dy_dev), lddy, offsets_dev, static_cast<int>(N), out_dev, out_kind);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

}  // extern "C"

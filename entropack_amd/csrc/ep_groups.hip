// Entries grouped by an id, and the weighted return of grouped rows to their tokens.
//
//   group_*           a stable counting sort of small integers: order (entries sorted by id, "no group" last), offsets (first
//                     place of every group), place (the inverse of order), rows (order / per_row). Integer work only; the result does not depend
//                     on timing: a wave counts 64 consecutive entries at a time by comparing their ids with ballots, bit by
//                     bit, so that an entry's rank among equal ids is a population count.
//   combine_*         out[t] = sum_j w[t, j] y[place[t k + j]] and its gradients. Bound by the rows of y.
#include "ep_grouped.hpp"

namespace ep {

constexpr int kGroupThreads = 1024, kGroupWaves = kGroupThreads / 64;

// The group of entry i, `groups` for an id outside [0, groups).
template <typename Id>
__device__ __forceinline__ int group_of(const Id* __restrict__ ids, int64_t i, int groups) {
  const Id id = ids[i];
  return id >= 0 && id < static_cast<Id>(groups) ? static_cast<int>(id) : groups;
}

// The lanes of this wave that hold the same key (lanes outside `among` are left out).
__device__ __forceinline__ uint64_t lanes_with_my_key(int key, int key_bits, uint64_t among) {
  uint64_t same = among;
  for (int b = 0; b < key_bits; ++b) {
    const bool set = (key >> b) & 1;
    const uint64_t with = __builtin_amdgcn_ballot_w64(set);
    same &= set ? with : ~with;
  }
  return same;
}

// counts[key] (LDS, this wave's row, cleared before) += this wave's entries [first, last).
template <typename Id>
__device__ __forceinline__ void count_entries(const Id* __restrict__ ids, int64_t first, int64_t last, int groups, int key_bits, int* counts) {
  const int lane = threadIdx.x & 63;
  constexpr int kTogether = 4;                   // loads under way at a time; those past the end read the last id
  for (int64_t from = first; from < last; from += 64 * kTogether) {
    int key[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int64_t at = from + 64 * i + lane;
      key[i] = group_of(ids, at < last ? at : last - 1, groups);
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const bool live = from + 64 * i + lane < last;
      const uint64_t same = lanes_with_my_key(key[i], key_bits, __builtin_amdgcn_ballot_w64(live));
      if (live && __builtin_ctzll(same) == lane) counts[key[i]] += __builtin_popcountll(same);
      order_in_wave();
    }
  }
}

// What the sort writes.
struct GroupOut {
  int32_t* order;
  int32_t* offsets;
  int32_t* place;
  int32_t* rows;                   // may be absent
  int per_row;

  __device__ __forceinline__ void put(int64_t entry, int to) const {
    order[to] = static_cast<int32_t>(entry);
    place[entry] = to;
    if (rows != nullptr) rows[to] = static_cast<int32_t>(static_cast<uint32_t>(entry) / static_cast<uint32_t>(per_row));
  }
};

// Gives every entry its place; next[key] (LDS, this wave's row) is the place of the wave's next entry with that key.
template <typename Id>
__device__ __forceinline__ void place_entries(const Id* __restrict__ ids, int64_t first, int64_t last, int groups, int key_bits, int* next, const GroupOut& out) {
  const int lane = threadIdx.x & 63;
  for (int64_t at = first; at < last; at += 64) {
    const bool live = at + lane < last;
    const int key = live ? group_of(ids, at + lane, groups) : 0;
    const uint64_t same = lanes_with_my_key(key, key_bits, __builtin_amdgcn_ballot_w64(live));
    if (live) {
      const int base = next[key];
      out.put(at + lane, base + __builtin_popcountll(same & ((uint64_t{1} << lane) - 1)));
      order_in_wave();                           // the leader moves the row on once every lane of the wave has read it
      if (__builtin_ctzll(same) == lane) next[key] = base + __builtin_popcountll(same);
    }
    order_in_wave();
  }
}

// Counts of one block's entries [block * chunk, ..) per key: table[block][key].
template <typename Id>
__global__ __launch_bounds__(kGroupThreads) void group_count_kernel(const Id* __restrict__ ids, int64_t entries, int64_t chunk, int groups,
                                                                    int key_bits, int32_t* __restrict__ table) {
  extern __shared__ int group_smem[];
  const int keys = groups + 1;
  for (int i = threadIdx.x; i < kGroupWaves * keys; i += kGroupThreads) group_smem[i] = 0;
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  const int64_t begin = blockIdx.x * chunk, end = begin + chunk < entries ? begin + chunk : entries;
  const int64_t share = ((end - begin + kGroupWaves * 64 - 1) / (kGroupWaves * 64)) * 64;
  const int64_t first = begin + wave * share, last = first + share < end ? first + share : end;
  count_entries(ids, first, last, groups, key_bits, group_smem + wave * keys);
  __syncthreads();
  for (int key = threadIdx.x; key < keys; key += kGroupThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) sum += group_smem[w * keys + key];
    table[static_cast<int64_t>(blockIdx.x) * keys + key] = sum;
  }
}

// Places this block's entries. What the other blocks hold of each key comes from `table`; a single block needs none.
// LDS: per-wave rows [kGroupWaves][keys], then before[keys] (entries of a key in earlier blocks) and others[keys] (in all
// other blocks). PER > 0: a block has 64 PER kGroupWaves entries, whose ranks stay in registers from the count to the
// placing; PER == 0: any number, which are read and ranked again.
template <typename Id, int PER>
__global__ __launch_bounds__(kGroupThreads) void group_place_kernel(const Id* __restrict__ ids, int64_t entries, int64_t chunk, int groups,
                                                                    int key_bits, const int32_t* __restrict__ table, int blocks, GroupOut out) {
  extern __shared__ int group_smem[];
  __shared__ int wave_sums[kGroupWaves];
  const int keys = groups + 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* counts = group_smem + wave * keys;
  int* before = group_smem + kGroupWaves * keys;
  int* others = before + keys;
  const int64_t begin = blockIdx.x * chunk, end = begin + chunk < entries ? begin + chunk : entries;
  const int64_t share = PER > 0 ? PER * 64 : ((end - begin + kGroupWaves * 64 - 1) / (kGroupWaves * 64)) * 64;
  const int64_t first = begin + wave * share, last = first + share < end ? first + share : end;
  int mine_key[PER > 0 ? PER : 1], rank[PER > 0 ? PER : 1];
#pragma unroll
  for (int i = 0; i < PER; ++i) mine_key[i] = first + 64 * i + lane < last ? group_of(ids, first + 64 * i + lane, groups) : 0;
  for (int i = threadIdx.x; i < (kGroupWaves + 2) * keys; i += kGroupThreads) group_smem[i] = 0;
  __syncthreads();
  if constexpr (PER == 0) {
    count_entries(ids, first, last, groups, key_bits, counts);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool live = first + 64 * i + lane < last;
      const uint64_t same = lanes_with_my_key(mine_key[i], key_bits, __builtin_amdgcn_ballot_w64(live));
      const int seen = live ? counts[mine_key[i]] : 0;
      rank[i] = seen + __builtin_popcountll(same & ((uint64_t{1} << lane) - 1));
      order_in_wave();                           // the leader moves the row on once every lane of the wave has read it
      if (live && __builtin_ctzll(same) == lane) counts[mine_key[i]] = seen + __builtin_popcountll(same);
      order_in_wave();
    }
  }
  if (table != nullptr) {
    const int cells = blocks * keys;             // integer sums: their order does not matter
    for (int i = threadIdx.x; i < cells; i += kGroupThreads) {
      const int n = table[i], block = i / keys, key = i % keys;
      if (n != 0 && block != static_cast<int>(blockIdx.x)) {
        atomicAdd(&others[key], n);
        if (block < static_cast<int>(blockIdx.x)) atomicAdd(&before[key], n);
      }
    }
  }
  __syncthreads();
  // Exclusive scan of the totals over the keys: a thread per key (at most kGroupThreads of them).
  const int key = threadIdx.x;
  int mine = 0;
  if (key < keys) {
    mine = others[key];
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) mine += group_smem[w * keys + key];
  }
  const int inclusive = wave_inclusive_sum(mine);
  if (lane == 63) wave_sums[wave] = inclusive;
  __syncthreads();
  int start = inclusive - mine;
  for (int w = 0; w < wave; ++w) start += wave_sums[w];
  if (key < keys) {
    if (blockIdx.x == 0) out.offsets[key] = start;           // offsets[groups]: entries that have a group
    int at = start + before[key];
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      const int n = group_smem[w * keys + key];
      group_smem[w * keys + key] = at;
      at += n;
    }
  }
  __syncthreads();
  if constexpr (PER == 0) {
    place_entries(ids, first, last, groups, key_bits, counts, out);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (first + 64 * i + lane < last) out.put(first + 64 * i + lane, counts[mine_key[i]] + rank[i]);
    }
  }
}

// One block sorts up to kOneBlock entries; beyond, a kernel before it counts blocks of 4096, and more than kGroupBlocks of
// those give each block a longer share. In 16 and 256 groups, one block: 1000 entries 3.2 and 3.7 us, 4096 5.7 and 7.4 us,
// 8192 9.0 and 12.4 us; two kernels: 4096 9.1 and 11.6 us, 8192 9.3 and 12.1 us besides a second launch, 16384 10.1 and
// 13.0 us, 131072 11.0 and 16.8 us. Latency bounds all of these (131072 ids of 64 bits and what is written of them, 2.6 MB,
// are 0.4 us); every block counting the others' ids by itself in place of the first kernel took 12.0 us for 16384 entries.
constexpr int64_t kOneBlock = 8 * kGroupThreads;
constexpr int64_t kGroupChunk = 4 * kGroupThreads;
constexpr int kGroupBlocks = 256;
constexpr int kMostGroups = 896;                 // a thread per key in the scan, 64 KiB of LDS

static int64_t group_chunk(int64_t entries) {
  if (entries <= kOneBlock) return entries <= kGroupThreads ? kGroupThreads : entries <= kGroupChunk ? kGroupChunk : kOneBlock;
  const int64_t even = (entries + kGroupBlocks - 1) / kGroupBlocks;
  return even < kGroupChunk ? kGroupChunk : (even + 63) / 64 * 64;
}

template <typename Id>
static int launch_group(const Id* ids, int64_t entries, int groups, const GroupOut& out, int32_t* table, hipStream_t s) {
  const int64_t chunk = group_chunk(entries);
  const int blocks = static_cast<int>((entries + chunk - 1) / chunk);
  const int keys = groups + 1;
  const size_t room = (kGroupWaves + 2) * keys * sizeof(int);
  int key_bits = 0;
  while ((groups >> key_bits) != 0) ++key_bits;
  if (entries <= kOneBlock) {
    if (chunk == kGroupThreads) hipLaunchKernelGGL((group_place_kernel<Id, 1>), dim3(1), dim3(kGroupThreads), room, s, ids, entries, chunk, groups, key_bits, nullptr, 1, out);
    else if (chunk == kGroupChunk) hipLaunchKernelGGL((group_place_kernel<Id, 4>), dim3(1), dim3(kGroupThreads), room, s, ids, entries, chunk, groups, key_bits, nullptr, 1, out);
    else hipLaunchKernelGGL((group_place_kernel<Id, 8>), dim3(1), dim3(kGroupThreads), room, s, ids, entries, chunk, groups, key_bits, nullptr, 1, out);
    EP_HIP_TRY(hipGetLastError());
    return EP_HIP_OK;
  }
  hipLaunchKernelGGL(group_count_kernel<Id>, dim3(blocks), dim3(kGroupThreads), kGroupWaves * keys * sizeof(int), s, ids, entries, chunk, groups, key_bits, table);
  EP_HIP_TRY(hipGetLastError());
  if (chunk == kGroupChunk)
    hipLaunchKernelGGL((group_place_kernel<Id, 4>), dim3(blocks), dim3(kGroupThreads), room, s, ids, entries, chunk, groups, key_bits, table, blocks, out);
  else
    hipLaunchKernelGGL((group_place_kernel<Id, 0>), dim3(blocks), dim3(kGroupThreads), room, s, ids, entries, chunk, groups, key_bits, table, blocks, out);
  EP_HIP_TRY(hipGetLastError());
  return EP_HIP_OK;
}

// ---- the weighted return ------------------------------------------------------------------------------------------------------

// VEC consecutive elements as floats. VEC = 8 takes 16-byte (bf16) or two 16-byte (float) accesses, VEC = 1 any address.
template <typename T, int VEC>
__device__ __forceinline__ void load_floats(const T* __restrict__ from, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 2) v[0] = __uint_as_float(static_cast<uint32_t>(*from) << 16);
    else v[0] = *from;
  } else if constexpr (sizeof(T) == 2) {
    const uint4 in = *reinterpret_cast<const uint4*>(from);
    const uint32_t word[4] = {in.x, in.y, in.z, in.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(word[i] << 16);
      v[2 * i + 1] = __uint_as_float(word[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 in = *reinterpret_cast<const float4*>(from + 4 * h);
      v[4 * h] = in.x, v[4 * h + 1] = in.y, v[4 * h + 2] = in.z, v[4 * h + 3] = in.w;
    }
  }
}

template <int VEC>
__device__ __forceinline__ void store_bf16(uint16_t* __restrict__ to, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *to = static_cast<uint16_t>(bf16_bits_of(v[0]));
  } else {
    *reinterpret_cast<uint4*>(to) = make_uint4(bf16_bits_of(v[0]) | bf16_bits_of(v[1]) << 16, bf16_bits_of(v[2]) | bf16_bits_of(v[3]) << 16,
                                               bf16_bits_of(v[4]) | bf16_bits_of(v[5]) << 16, bf16_bits_of(v[6]) | bf16_bits_of(v[7]) << 16);
  }
}

// One thread per VEC columns of a token; the token's rows are added in the order of its entries, in f32, and rounded once. Bound by
// memory: 16222 rows of 4096 to 8111 tokens, 199 MB, 30.8 us, 6.5 TB/s with half the rows read from the last-level cache (the
// call repeated on the same rows); 128 rows of 2048 to 32 tokens 3.9 us.
// place == nullptr: the rows of y lie in the order of the entries (and all count). weight == nullptr: plain sums.
template <typename Row, int VEC>
__global__ __launch_bounds__(256) void combine_rows_kernel(const Row* __restrict__ y, int64_t ldy, const int32_t* __restrict__ place,
                                                           const int32_t* __restrict__ kept_rows, const void* __restrict__ weight, int weight_kind,
                                                           int per_row, int64_t tokens, int width, uint16_t* __restrict__ out, int64_t ldo) {
  const int pieces = (width + VEC - 1) / VEC;
  const int64_t at = blockIdx.x * int64_t{256} + threadIdx.x;
  if (at >= tokens * pieces) return;
  const int64_t token = at / pieces;
  const int column = static_cast<int>(at % pieces) * VEC;
  const int kept = place != nullptr ? *kept_rows : 0;
  float sum[VEC] = {};
#pragma unroll 4
  for (int j = 0; j < per_row; ++j) {
    const int64_t entry = token * per_row + j;
    int64_t row = entry;
    if (place != nullptr) {
      row = place[entry];
      if (row >= kept) continue;                 // an entry of no group
    }
    float v[VEC];
    load_floats<Row, VEC>(y + row * ldy + column, v);
    const float w = weight != nullptr ? load_bias(weight, weight_kind, static_cast<int>(entry)) : 1.0f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = __builtin_fmaf(w, v[i], sum[i]);
  }
  store_bf16<VEC>(out + token * ldo + column, sum);
}

// Gradients, one block per token: grad_y[place] = w grad (zero for entries of no group), grad_w = <grad, y[place]>. The
// gradient row is read once for kMostTogether entries; dot products are summed lane by lane, then across the block, in a
// fixed order. Either result may be absent. Bound by memory: 8111 tokens, 16222 rows of 4096, both results, 332 MB, 58 us, 5.7 TB/s, a third of the reads from the last-level cache.
constexpr int kMostTogether = 8;

template <int VEC>
__global__ __launch_bounds__(256) void combine_grad_kernel(const uint16_t* __restrict__ grad, int64_t ldg, const uint16_t* __restrict__ y, int64_t ldy,
                                                           const int32_t* __restrict__ place, const int32_t* __restrict__ kept_rows,
                                                           const void* __restrict__ weight, int weight_kind, int per_row, int width,
                                                           uint16_t* __restrict__ grad_y, int64_t ldgy, void* __restrict__ grad_w) {
  __shared__ float partial[4][kMostTogether];
  const int64_t token = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int kept = *kept_rows;
  for (int j0 = 0; j0 < per_row; j0 += kMostTogether) {
    const int n = per_row - j0 < kMostTogether ? per_row - j0 : kMostTogether;
    float dot[kMostTogether] = {};
    for (int column = threadIdx.x * VEC; column < width; column += 256 * VEC) {
      float g[VEC];
      load_floats<uint16_t, VEC>(grad + token * ldg + column, g);
#pragma unroll
      for (int j = 0; j < kMostTogether; ++j) {
        if (j >= n) continue;
        const int64_t entry = token * per_row + j0 + j;
        const int64_t row = place[entry];
        const bool counts = row < kept;
        const float w = !counts ? 0.0f : (weight != nullptr ? load_bias(weight, weight_kind, static_cast<int>(entry)) : 1.0f);
        if (grad_w != nullptr && counts) {
          float v[VEC];
          load_floats<uint16_t, VEC>(y + row * ldy + column, v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) dot[j] = __builtin_fmaf(g[i], v[i], dot[j]);
        }
        if (grad_y != nullptr) {
          float v[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[i] = counts ? w * g[i] : 0.0f;
          store_bf16<VEC>(grad_y + row * ldgy + column, v);
        }
      }
    }
    if (grad_w == nullptr) continue;
#pragma unroll
    for (int j = 0; j < kMostTogether; ++j) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) dot[j] += __shfl_xor(dot[j], d);
      if (lane == 0) partial[wave][j] = dot[j];
    }
    __syncthreads();
    if (threadIdx.x < static_cast<unsigned>(n)) {
      const int j = threadIdx.x;
      store_out(grad_w, weight_kind, token * per_row + j0 + j, (partial[0][j] + partial[1][j]) + (partial[2][j] + partial[3][j]));
    }
    __syncthreads();
  }
}

// Blocks of 256 threads in a launch (fewer than 2^32 work items): more tokens take several.
constexpr int64_t kMostBlocks = 0xFFFFFFFF / 256;

// The weights from entry `entry` on, which may be absent.
static const void* weights_from(const void* weight, int kind, int64_t entry) {
  return weight != nullptr ? static_cast<const uint8_t*>(weight) + entry * (kind == kOutF32 ? 4 : 2) : nullptr;
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace ep

extern "C" {

size_t ep_hip_group_rows_workspace(int64_t entries, int groups) {
  if (entries <= 0 || groups <= 0) return 0;
  const int64_t chunk = ep::group_chunk(entries), blocks = (entries + chunk - 1) / chunk;
  return entries > ep::kOneBlock ? static_cast<size_t>(blocks) * static_cast<size_t>(groups + 1) * 4 : 0;
}

int ep_hip_group_rows(const void* ids_dev, int id_bytes, int64_t entries, int groups, int per_row, int32_t* order_dev, int32_t* offsets_dev, int32_t* place_dev,
                      int32_t* rows_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace ep;
  if (ids_dev == nullptr || order_dev == nullptr || offsets_dev == nullptr || place_dev == nullptr) return EP_HIP_EINVAL;
  if (entries <= 0 || groups <= 0 || per_row <= 0 || (id_bytes != 4 && id_bytes != 8)) return EP_HIP_EINVAL;
  if (entries > kMostEntries || groups > kMostGroups) return EP_HIP_EUNSUPPORTED;
  const size_t wanted = ep_hip_group_rows_workspace(entries, groups);
  if (wanted != 0 && (workspace_dev == nullptr || workspace_bytes < wanted)) return EP_HIP_EINVAL;
  int32_t* table = static_cast<int32_t*>(workspace_dev);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const GroupOut out = {order_dev, offsets_dev, place_dev, rows_dev, per_row};
  if (id_bytes == 4) return launch_group(static_cast<const int32_t*>(ids_dev), entries, groups, out, table, s);
  return launch_group(static_cast<const int64_t*>(ids_dev), entries, groups, out, table, s);
}

int ep_hip_combine_rows(const void* y_dev, int y_kind, int64_t ldy, const int32_t* place_dev, const int32_t* kept_rows_dev, const void* weight_dev, int weight_kind,
                        int per_row, int64_t tokens, int64_t width, void* out_dev, int64_t ldo, void* stream) {
  using namespace ep;
  if (y_dev == nullptr || out_dev == nullptr || (place_dev != nullptr && kept_rows_dev == nullptr)) return EP_HIP_EINVAL;
  if (tokens <= 0 || per_row <= 0 || width <= 0 || width > 0x3FFFFFFF || ldy < width || ldo < width) return EP_HIP_EINVAL;
  if ((y_kind != kOutBF16 && y_kind != kOutF32) || (weight_dev != nullptr && weight_kind != kOutBF16 && weight_kind != kOutF32)) return EP_HIP_EINVAL;
  if (tokens > kMostEntries / per_row) return EP_HIP_EUNSUPPORTED;
  const bool wide = width % 8 == 0 && ldy % 8 == 0 && ldo % 8 == 0 && aligned16(y_dev) && aligned16(out_dev);
  const int64_t pieces = wide ? width / 8 : width, together = kMostBlocks * 256 / pieces;            // tokens per launch
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int w = static_cast<int>(width);
  for (int64_t from = 0; from < tokens; from += together) {
    const int64_t here = tokens - from < together ? tokens - from : together, entry = from * per_row;
    const dim3 grid(static_cast<unsigned>((here * pieces + 255) / 256));
    uint16_t* const out = static_cast<uint16_t*>(out_dev) + from * ldo;
    const int32_t* const place = place_dev != nullptr ? place_dev + entry : nullptr;
    const int64_t row = place_dev != nullptr ? 0 : entry;     // rows of y are found by their place, or lie in the order of the entries
    const void* const weight = weights_from(weight_dev, weight_kind, entry);
#define EP_COMBINE(ROW, VEC)                                                                                                                         \
  hipLaunchKernelGGL((combine_rows_kernel<ROW, VEC>), grid, dim3(256), 0, s, static_cast<const ROW*>(y_dev) + row * ldy, ldy, place, kept_rows_dev, weight, \
                     weight_kind, per_row, here, w, out, ldo)
    if (y_kind == kOutBF16) {
      if (wide) EP_COMBINE(uint16_t, 8);
      else EP_COMBINE(uint16_t, 1);
    } else {
      if (wide) EP_COMBINE(float, 8);
      else EP_COMBINE(float, 1);
    }
#undef EP_COMBINE
    EP_HIP_TRY(hipGetLastError());
  }
  return EP_HIP_OK;
}

int ep_hip_combine_rows_grad(const void* grad_dev, int64_t ldg, const void* y_dev, int64_t ldy, const int32_t* place_dev, const int32_t* kept_rows_dev,
                             const void* weight_dev, int weight_kind, int per_row, int64_t tokens, int64_t width, void* grad_y_dev, int64_t ldgy,
                             void* grad_weight_dev, void* stream) {
  using namespace ep;
  if (grad_dev == nullptr || place_dev == nullptr || kept_rows_dev == nullptr || (grad_y_dev == nullptr && grad_weight_dev == nullptr)) return EP_HIP_EINVAL;
  if (grad_weight_dev != nullptr && (y_dev == nullptr || ldy < width)) return EP_HIP_EINVAL;
  if (tokens <= 0 || per_row <= 0 || width <= 0 || width > 0x3FFFFFFF || ldg < width || (grad_y_dev != nullptr && ldgy < width)) return EP_HIP_EINVAL;
  if ((weight_dev != nullptr || grad_weight_dev != nullptr) && weight_kind != kOutBF16 && weight_kind != kOutF32) return EP_HIP_EINVAL;
  if (tokens > kMostEntries / per_row) return EP_HIP_EUNSUPPORTED;
  const bool wide = width % 8 == 0 && ldg % 8 == 0 && aligned16(grad_dev) && (grad_weight_dev == nullptr || (ldy % 8 == 0 && aligned16(y_dev))) &&
                    (grad_y_dev == nullptr || (ldgy % 8 == 0 && aligned16(grad_y_dev)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint16_t* y = static_cast<const uint16_t*>(y_dev);
  uint16_t* grad_y = static_cast<uint16_t*>(grad_y_dev);
  const int w = static_cast<int>(width);
  for (int64_t from = 0; from < tokens; from += kMostBlocks) {               // a block per token
    const dim3 grid(static_cast<unsigned>(tokens - from < kMostBlocks ? tokens - from : kMostBlocks));
    const int64_t entry = from * per_row;
    const uint16_t* const grad = static_cast<const uint16_t*>(grad_dev) + from * ldg;
    const void* const weight = weights_from(weight_dev, weight_kind, entry);
    void* const grad_weight = const_cast<void*>(weights_from(grad_weight_dev, weight_kind, entry));
    if (wide)
      hipLaunchKernelGGL(combine_grad_kernel<8>, grid, dim3(256), 0, s, grad, ldg, y, ldy, place_dev + entry, kept_rows_dev, weight, weight_kind, per_row, w, grad_y, ldgy, grad_weight);
    else
      hipLaunchKernelGGL(combine_grad_kernel<1>, grid, dim3(256), 0, s, grad, ldg, y, ldy, place_dev + entry, kept_rows_dev, weight, weight_kind, per_row, w, grad_y, ldgy, grad_weight);
    EP_HIP_TRY(hipGetLastError());
  }
  return EP_HIP_OK;
}

}  // extern "C"

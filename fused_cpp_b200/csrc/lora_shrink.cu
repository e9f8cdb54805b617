// Coefficients of low-rank adapters: t[row] = scaling[a] * (A[a] x[row]) with a = the row's adapter, for rows in any order.
//
// A batch has few rows per adapter and a long K (one row of 7168 values against 16 to 64 ranks): what is read is x once and every
// adapter in use once, and latency is what counts.  So the K range is split over the warps of a cluster, each warp keeps ranks x rows partial sums of
// mma.sync.m16n8k16 (ranks are its M, rows its N: one row costs no more than eight), and the warps' sums meet in shared memory, the CTAs' in
// distributed shared memory, in a fixed order.  Fragments come straight from global memory with 16-byte loads: the order of the K elements inside a
// group of 32 may be any as long as both operands use the same, so that lane (g, q) takes elements 8q .. 8q + 7 of its row for
// two MMAs.
//
// The launch runs beside the row quantiser in front of it, whose results it does not need: everything is read through L2 and the wait
// stands at the end.
//
// A tile of 128 rows is one list of units: the rows of an adapter, in groups of up to 32.  Every CTA of a tile makes the list for itself.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "lora.h"
#include "ptx.cuh"
#include "row_quant.cuh"

namespace fmoe {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTileRows = 128;
constexpr int kUnitRows = 32;
constexpr int kRowTiles = kUnitRows / 8;                   // N tiles of a unit
constexpr int kRankTiles = kLoraRankBlock / 16;            // M tiles of a unit
constexpr int kUnitValues = kLoraRankBlock * kUnitRows;
constexpr int kMaxCluster = 8;

struct ShrinkArgs {
  const uint16_t* x;
  int64_t rows;
  int k;
  LoraAdapters adapters;
  uint16_t* t;
  int planes;
  int cluster;  // CTAs that share a unit's K range
  int stride;   // clusters that share a tile's units
};

struct ShrinkShared {
  int id[kTileRows];
  int slot_adapter[kTileRows], slot_rows[kTileRows], slot_first[kTileRows];
  int unit_slot[kTileRows], unit_row[kTileRows];  // unit -> slot, first row of it in `order`
  int order[kTileRows];                           // rows of the tile, slot by slot
  int warp_count[4];
  int units;
  alignas(16) float total[kUnitValues];
  alignas(16) float part[kWarps][kUnitValues];  // stored in pairs
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight values of a row of x from element k on; k is a multiple of 8, what lies behind the row's end is zero.
template <bool kVector>
__device__ __forceinline__ uint4 load_x8(const uint16_t* row, int k, int columns) {
  if constexpr (kVector) {
    return k < columns ? __ldcg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t words[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t low = k + 2 * i < columns ? __ldcg(row + k + 2 * i) : 0;
      const uint32_t high = k + 2 * i + 1 < columns ? __ldcg(row + k + 2 * i + 1) : 0;
      words[i] = low | (high << 16);
    }
    return make_uint4(words[0], words[1], words[2], words[3]);
  }
}

// The tile's units, in an order that the ids alone decide.
__device__ __forceinline__ void list_units(ShrinkShared& s, const ShrinkArgs& args, int64_t row0) {
  const int i = threadIdx.x;
  int before = 0, total = 0, first = kTileRows;
  if (i < kTileRows) s.id[i] = row0 + i < args.rows ? load_adapter_id(args.adapters, row0 + i) : -1;
  __syncthreads();
  const int mine = i < kTileRows ? s.id[i] : -1;
  if (mine >= 0) {
    for (int j = 0; j < kTileRows; ++j) {
      if (s.id[j] != mine) continue;
      first = min(first, j);
      before += j < i;
      ++total;
    }
  }
  const bool owner = mine >= 0 && first == i;
  const unsigned owners = __ballot_sync(0xffffffffu, owner);
  if (i < kTileRows && (i & 31) == 0) s.warp_count[i >> 5] = __popc(owners);
  __syncthreads();
  int slot = __popc(owners & ((1u << (i & 31)) - 1));
  for (int w = 0; w < 4 && w < (i >> 5); ++w) slot += s.warp_count[w];
  const int slots = s.warp_count[0] + s.warp_count[1] + s.warp_count[2] + s.warp_count[3];
  if (owner) {
    s.slot_adapter[slot] = mine;
    s.slot_rows[slot] = total;
    s.unit_row[i] = slot;  // for a moment: the slot of the adapter's first row
  }
  __syncthreads();
  const int my_slot = mine >= 0 ? s.unit_row[first] : 0;
  __syncthreads();
  if (i < slots) {
    int row_first = 0, unit_first = 0;
    for (int j = 0; j < i; ++j) {
      row_first += s.slot_rows[j];
      unit_first += (s.slot_rows[j] + kUnitRows - 1) / kUnitRows;
    }
    s.slot_first[i] = row_first;
    const int units = (s.slot_rows[i] + kUnitRows - 1) / kUnitRows;
    for (int u = 0; u < units; ++u) {
      s.unit_slot[unit_first + u] = i;
      s.unit_row[unit_first + u] = row_first + u * kUnitRows;
    }
    if (i == slots - 1) s.units = unit_first + units;
  }
  if (slots == 0 && i == 0) s.units = 0;
  __syncthreads();
  if (mine >= 0) s.order[s.slot_first[my_slot] + before] = i;
  __syncthreads();
}

template <bool kVector>
__global__ void __launch_bounds__(kThreads)
lora_shrink_kernel(const ShrinkArgs args) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  ShrinkShared& s = *reinterpret_cast<ShrinkShared*>(smem_raw);
  ptx::launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank_of_cta = static_cast<int>(blockIdx.x) % args.cluster;
  const int group = static_cast<int>(blockIdx.x) / args.cluster;
  const int tile = group / args.stride;
  const int64_t row0 = static_cast<int64_t>(tile) * kTileRows;
  list_units(s, args, row0);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int k32 = (args.k + 31) / 32;
  const int worker = rank_of_cta * kWarps + warp, workers = args.cluster * kWarps;
  const int chunk_begin = static_cast<int>(static_cast<int64_t>(k32) * worker / workers);
  const int chunk_end = static_cast<int>(static_cast<int64_t>(k32) * (worker + 1) / workers);
  const int rank_padded = lora_rank_padded(args.adapters.rank);
  const int rank_blocks = (args.adapters.rank + kLoraRankBlock - 1) / kLoraRankBlock;
  const int work = s.units * rank_blocks;
  for (int item = group - tile * args.stride; item < work; item += args.stride) {
    const int unit = item / rank_blocks;
    const int rank0 = (item - unit * rank_blocks) * kLoraRankBlock;
    const int slot = s.unit_slot[unit];
    const int adapter = s.slot_adapter[slot];
    const int order0 = s.unit_row[unit];
    const int count = min(kUnitRows, s.slot_first[slot] + s.slot_rows[slot] - order0);
    const int ranks = min(kLoraRankBlock, args.adapters.rank - rank0);
    float acc[kRankTiles][kRowTiles][4];
#pragma unroll
    for (int m = 0; m < kRankTiles; ++m)
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[m][n][v] = 0.0f;
    const uint16_t* x_rows[kRowTiles];
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) {
      const int local = 8 * n + g;
      x_rows[n] = local < count ? args.x + (row0 + s.order[order0 + local]) * args.k : nullptr;
    }
    const uint16_t* a_base = args.adapters.a + (static_cast<int64_t>(adapter) * args.adapters.rank + rank0) * args.adapters.a_stride;
    for (int chunk = chunk_begin; chunk < chunk_end; ++chunk) {
      const int k = chunk * 32 + 8 * q;
      uint4 xv[kRowTiles];
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) xv[n] = x_rows[n] != nullptr ? load_x8<kVector>(x_rows[n], k, args.k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < kRankTiles; ++m) {
        if (16 * m >= ranks) break;
        const int r = 16 * m + g;
        uint4 low = make_uint4(0, 0, 0, 0), high = low;
        if (k < args.adapters.a_stride) {
          if (r < ranks) low = __ldcg(reinterpret_cast<const uint4*>(a_base + static_cast<int64_t>(r) * args.adapters.a_stride + k));
          if (r + 8 < ranks) high = __ldcg(reinterpret_cast<const uint4*>(a_base + static_cast<int64_t>(r + 8) * args.adapters.a_stride + k));
        }
        const uint32_t first[4] = {low.x, high.x, low.y, high.y};
        const uint32_t second[4] = {low.z, high.z, low.w, high.w};
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
          if (8 * n >= count) break;
          mma_bf16(acc[m][n], first, xv[n].x, xv[n].y);
          mma_bf16(acc[m][n], second, xv[n].z, xv[n].w);
        }
      }
    }
    // Partial sums [rank][row] of the warps, then of the CTAs.
#pragma unroll
    for (int m = 0; m < kRankTiles; ++m)
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) {
        float* to = &s.part[warp][(16 * m + g) * kUnitRows + 8 * n + 2 * q];
        *reinterpret_cast<float2*>(to) = make_float2(acc[m][n][0], acc[m][n][1]);
        *reinterpret_cast<float2*>(to + 8 * kUnitRows) = make_float2(acc[m][n][2], acc[m][n][3]);
      }
    __syncthreads();
    for (int e = threadIdx.x; e < kUnitValues; e += kThreads) {
      float sum = s.part[0][e];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) sum += s.part[w][e];
      s.total[e] = sum;
    }
    if (args.cluster > 1) {
      cluster.sync();
    } else {
      __syncthreads();
    }
    const float scale = __ldcg(args.adapters.scaling + adapter);
    const int ranks_stored = min(kLoraRankBlock, rank_padded - rank0);
    // Element e = (row, rank), ranks side by side as they lie in t; every cluster-th one is this CTA's.
    for (int e = threadIdx.x * args.cluster + rank_of_cta; e < kLoraRankBlock * count; e += kThreads * args.cluster) {
      const int row = e / kLoraRankBlock, r = e % kLoraRankBlock;
      if (r >= ranks_stored) continue;
      const int at = r * kUnitRows + row;
      float sum = 0.0f;
      for (int c = 0; c < args.cluster; ++c) sum += args.cluster > 1 ? cluster.map_shared_rank(s.total, c)[at] : s.total[at];
      float rest = r < ranks ? __fmul_rn(sum, scale) : 0.0f;
      uint16_t* to = args.t + (row0 + s.order[order0 + row]) * rank_padded + rank0 + r;
      for (int plane = 0; plane < args.planes; ++plane) {
        const uint16_t bits = __bfloat16_as_ushort(__float2bfloat16_rn(rest));
        *to = bits;
        rest = __fsub_rn(rest, bf16_bits_to_f32(bits));  // exact; what is left of an infinity (NaN) is not wanted
        if (!isfinite(rest)) rest = 0.0f;
        to += args.rows * rank_padded;
      }
    }
    if (args.cluster > 1) {
      cluster.sync();  // nobody still reads these sums
    } else {
      __syncthreads();
    }
  }
  ptx::grid_dependency_wait();  // this kernel's end stands for the end of the one in front too
}

// Rows of x as int8 with a scale each: scale = amax * (1/127) in 32 bits (1 for a row of zeros), q = clamp(rint(x / scale), -128, 127).
constexpr int kQuantThreads = 256;

template <bool kVector>
__global__ void __launch_bounds__(kQuantThreads)
lora_quantize_kernel(const uint16_t* __restrict__ x, int cols, int cols_padded, int8_t* __restrict__ q, float* __restrict__ scale_out, int* status) {
  ptx::launch_dependents();
  __shared__ float smem[32];
  if (blockIdx.x == 0 && threadIdx.x < kStatusWords) status[threadIdx.x] = 0;
  const int64_t row = blockIdx.x;
  const uint16_t* const src = x + row * cols;
  float local = 0.0f;
  if constexpr (kVector) {
    for (int v = threadIdx.x; v < cols >> 3; v += kQuantThreads) local = fmaxf(local, amax8(reinterpret_cast<const uint4*>(src)[v]));
  } else {
    for (int c = threadIdx.x; c < cols; c += kQuantThreads) local = fmaxf(local, fabsf(bf16_bits_to_f32(src[c])));
  }
  const float amax = block_max(local, smem);
  const float scale = amax > 0.0f ? __fmul_rn(amax, 1.0f / 127.0f) : 1.0f;
  if (threadIdx.x == 0) scale_out[row] = scale;
  const float inverse = __fdiv_rn(1.0f, scale);
  uint2* const dst = reinterpret_cast<uint2*>(q + row * cols_padded);  // cols_padded is a multiple of 16
  for (int v = threadIdx.x; v < cols_padded >> 3; v += kQuantThreads) {
    float values[8];
    unpack8(load_x8<kVector>(src, 8 * v, cols), values);
    dst[v] = make_uint2(quantize4_torchref_fast<false>(values, scale, inverse, -128.0f), quantize4_torchref_fast<false>(values + 4, scale, inverse, -128.0f));
  }
}

}  // namespace

cudaError_t launch_lora_quantize(const uint16_t* x, int64_t rows, int k, int k_padded, int8_t* q, float* scale, int* status, cudaStream_t stream) {
  const bool vector = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto kernel = vector ? lora_quantize_kernel<true> : lora_quantize_kernel<false>;
  kernel<<<static_cast<unsigned>(rows), kQuantThreads, 0, stream>>>(x, k, k_padded, q, scale, status);
  return cudaGetLastError();
}

cudaError_t launch_lora_shrink(const uint16_t* x, int64_t rows, int k, const LoraAdapters& adapters, uint16_t* t, int planes, cudaStream_t stream) {
  ShrinkArgs args = {x, rows, k, adapters, t, planes, 1, 1};
  const bool vector = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto kernel = vector ? lora_shrink_kernel<true> : lora_shrink_kernel<false>;
  static PerDeviceOnce configured[2];
  const int device = current_device_ordinal();
  if (configured[vector].needed(device)) {
    const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(ShrinkShared)));
    if (error != cudaSuccess) return error;
    configured[vector].mark(device);
  }
  const int64_t tiles = (rows + kTileRows - 1) / kTileRows;
  // The K range is split over more CTAs the fewer tiles there are to fill the chip with.
  const int k32 = (k + 31) / 32;
  args.cluster = 1;
  while (args.cluster < kMaxCluster && tiles * args.cluster < 16 && args.cluster * kWarps * 2 <= k32) args.cluster *= 2;
  const int rank_blocks = (adapters.rank + kLoraRankBlock - 1) / kLoraRankBlock;
  const int64_t most = static_cast<int64_t>(adapters.count < kTileRows ? (adapters.count + kTileRows / kUnitRows < kTileRows ? adapters.count + kTileRows / kUnitRows : kTileRows) : kTileRows) *
                       rank_blocks;
  int64_t stride = 4ll * threshold_sms / (tiles * args.cluster);
  if (stride < 4) stride = 4;
  if (stride > most) stride = most;
  args.stride = static_cast<int>(stride);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles * args.stride * args.cluster));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = sizeof(ShrinkShared);
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = static_cast<unsigned>(args.cluster);
  attributes[0].val.clusterDim.y = 1;
  attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, kernel, args);
}

}  // namespace fmoe

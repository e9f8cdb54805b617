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
  alignas(16) int id[kTileRows];
  int slot_adapter[kTileRows], slot_rows[kTileRows], slot_first[kTileRows];
  int unit_slot[kTileRows], unit_row[kTileRows];  // unit -> slot, first row of it in `order`
  int order[kTileRows];                           // rows of the tile, slot by slot
  int warp_count[4];
  int units;
  alignas(16) float total[kUnitValues];  // [rank][row of the unit]
  // Behind it the warps' partial sums, [warp][rank][row of the unit] with as many ranks as a block of the adapters has.
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
  const int lane = i & 31;
  const int tile_rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), args.rows - row0));
  int before = 0, total = 0, first = kTileRows;
  if (i < kTileRows) s.id[i] = i < tile_rows ? load_adapter_id(args.adapters, row0 + i) : -1;
  __syncthreads();
  const int mine = i < kTileRows ? s.id[i] : -1;
  if (mine >= 0) {
    for (int j = 0; j < tile_rows; j += 4) {
      const int4 others = *reinterpret_cast<const int4*>(&s.id[j]);
      const int four[4] = {others.x, others.y, others.z, others.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool same = four[k] == mine;
        if (same && first == kTileRows) first = j + k;
        before += same && j + k < i;
        total += same;
      }
    }
  }
  const bool owner = mine >= 0 && first == i;
  const unsigned owners = __ballot_sync(0xffffffffu, owner);
  if (i < kTileRows && lane == 0) s.warp_count[i >> 5] = __popc(owners);
  __syncthreads();
  int slot = __popc(owners & ((1u << lane) - 1));
  int slots = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < (i >> 5)) slot += s.warp_count[w];
    slots += s.warp_count[w];
  }
  if (owner) {
    s.slot_adapter[slot] = mine;
    s.slot_rows[slot] = total;
    s.unit_row[i] = slot;  // for a moment: the slot of the adapter's first row
  }
  __syncthreads();
  const int my_slot = mine >= 0 ? s.unit_row[first] : 0;
  // Rows (low half) and units (high half) of the slots in front of slot i.
  const int rows = i < slots ? s.slot_rows[i] : 0;
  const int packed = rows | ((rows + kUnitRows - 1) / kUnitRows) << 16;
  int scan = packed;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, scan, offset);
    if (lane >= offset) scan += other;
  }
  __syncthreads();  // unit_row and warp_count are read
  if (i < kTileRows && lane == 31) s.warp_count[i >> 5] = scan;
  __syncthreads();
  int front = scan - packed;
  for (int w = 0; w < 4 && w < (i >> 5); ++w) front += s.warp_count[w];
  if (i < slots) {
    const int row_first = front & 0xffff, unit_first = front >> 16;
    s.slot_first[i] = row_first;
    for (int u = 0; u < packed >> 16; ++u) {
      s.unit_slot[unit_first + u] = i;
      s.unit_row[unit_first + u] = row_first + u * kUnitRows;
    }
    if (i == slots - 1) s.units = unit_first + (packed >> 16);
  }
  if (slots == 0 && i == 0) s.units = 0;
  __syncthreads();
  if (mine >= 0) s.order[s.slot_first[my_slot] + before] = i;
  __syncthreads();
}

struct Unit {
  const uint16_t* x;    // first row of the tile
  const uint16_t* a;    // first rank of the block
  const int* order;     // rows of the unit in the tile
  int count, ranks;
  int chunk_begin, chunk_end;  // of 32 K elements, for this warp
};

// A warp's partial sums of a unit of up to 16 kRankTiles ranks and 8 kRowTiles rows, to part [rank][row].  kUnroll chunks are in flight together.
template <bool kVector, int kRankTiles, int kRowTiles, int kUnroll>
__device__ __forceinline__ void multiply_unit(const ShrinkArgs& args, const Unit& unit, float* part) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
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
    x_rows[n] = local < unit.count ? unit.x + static_cast<int64_t>(unit.order[local]) * args.k : nullptr;
  }
  const int a_stride = args.adapters.a_stride;
  for (int chunk0 = unit.chunk_begin; chunk0 < unit.chunk_end; chunk0 += kUnroll) {
    uint4 xv[kUnroll][kRowTiles], low[kUnroll][kRankTiles], high[kUnroll][kRankTiles];
#pragma unroll
    for (int c = 0; c < kUnroll; ++c) {
      const int k = (chunk0 + c) * 32 + 8 * q;
      const bool inside = chunk0 + c < unit.chunk_end;
#pragma unroll
      for (int n = 0; n < kRowTiles; ++n) xv[c][n] = inside && x_rows[n] != nullptr ? load_x8<kVector>(x_rows[n], k, args.k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < kRankTiles; ++m) {
        const int r = 16 * m + g;
        const uint16_t* const a = unit.a + static_cast<int64_t>(r) * a_stride + k;
        low[c][m] = inside && k < a_stride && r < unit.ranks ? __ldcg(reinterpret_cast<const uint4*>(a)) : make_uint4(0, 0, 0, 0);
        high[c][m] = inside && k < a_stride && r + 8 < unit.ranks ? __ldcg(reinterpret_cast<const uint4*>(a + 8 * a_stride)) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int c = 0; c < kUnroll; ++c) {
#pragma unroll
      for (int m = 0; m < kRankTiles; ++m) {
        const uint32_t first[4] = {low[c][m].x, high[c][m].x, low[c][m].y, high[c][m].y};
        const uint32_t second[4] = {low[c][m].z, high[c][m].z, low[c][m].w, high[c][m].w};
#pragma unroll
        for (int n = 0; n < kRowTiles; ++n) {
          mma_bf16(acc[m][n], first, xv[c][n].x, xv[c][n].y);
          mma_bf16(acc[m][n], second, xv[c][n].z, xv[c][n].w);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kRankTiles; ++m) {
    if (16 * m >= unit.ranks) break;  // `part` ends there
#pragma unroll
    for (int n = 0; n < kRowTiles; ++n) {
      float* to = part + (16 * m + g) * kUnitRows + 8 * n + 2 * q;
      *reinterpret_cast<float2*>(to) = make_float2(acc[m][n][0], acc[m][n][1]);
      *reinterpret_cast<float2*>(to + 8 * kUnitRows) = make_float2(acc[m][n][2], acc[m][n][3]);
    }
  }
}

template <bool kVector>
__global__ void __launch_bounds__(kThreads, 2)
lora_shrink_kernel(const __grid_constant__ ShrinkArgs args) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  ShrinkShared& s = *reinterpret_cast<ShrinkShared*>(smem_raw);
  float* const parts = reinterpret_cast<float*>(smem_raw + sizeof(ShrinkShared));
  ptx::launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank_of_cta = static_cast<int>(blockIdx.x) % args.cluster;
  const int group = static_cast<int>(blockIdx.x) / args.cluster;
  const int tile = group / args.stride;
  const int64_t row0 = static_cast<int64_t>(tile) * kTileRows;
  list_units(s, args, row0);

  const int warp = threadIdx.x >> 5;
  const int k32 = (args.k + 31) / 32;
  const int worker = rank_of_cta * kWarps + warp, workers = args.cluster * kWarps;
  Unit unit;
  unit.x = args.x + row0 * args.k;
  unit.chunk_begin = static_cast<int>(static_cast<int64_t>(k32) * worker / workers);
  unit.chunk_end = static_cast<int>(static_cast<int64_t>(k32) * (worker + 1) / workers);
  const int rank_padded = lora_rank_padded(args.adapters.rank);
  const int rank_blocks = (args.adapters.rank + kLoraRankBlock - 1) / kLoraRankBlock;
  const int part_values = min(kLoraRankBlock, rank_padded) * kUnitRows;
  float* const part = parts + warp * part_values;
  const int work = s.units * rank_blocks;
  for (int item = group - tile * args.stride; item < work; item += args.stride) {
    const int index = item / rank_blocks;
    const int rank0 = (item - index * rank_blocks) * kLoraRankBlock;
    const int slot = s.unit_slot[index];
    const int adapter = s.slot_adapter[slot];
    const int order0 = s.unit_row[index];
    unit.order = s.order + order0;
    unit.count = min(kUnitRows, s.slot_first[slot] + s.slot_rows[slot] - order0);
    unit.ranks = min(kLoraRankBlock, args.adapters.rank - rank0);
    unit.a = args.adapters.a + (static_cast<int64_t>(adapter) * args.adapters.rank + rank0) * args.adapters.a_stride;
    if (unit.count <= 8) {
      if (unit.ranks <= 16) {
        multiply_unit<kVector, 1, 1, 4>(args, unit, part);
      } else if (unit.ranks <= 32) {
        multiply_unit<kVector, 2, 1, 2>(args, unit, part);
      } else {
        multiply_unit<kVector, 4, 1, 2>(args, unit, part);
      }
    } else if (unit.ranks <= 16) {
      multiply_unit<kVector, 1, 4, 2>(args, unit, part);
    } else if (unit.ranks <= 32) {
      multiply_unit<kVector, 2, 4, 1>(args, unit, part);
    } else {
      multiply_unit<kVector, 4, 4, 1>(args, unit, part);
    }
    __syncthreads();
    const float scale = __ldcg(args.adapters.scaling + adapter);
    // The warps' sums, then the CTAs'.  (Rows that the unit does not have are left out: nobody wrote their sums.)
    const int ranks16 = (unit.ranks + 15) & ~15;
    const int rows8 = unit.count <= 8 ? 8 : kUnitRows;
    for (int e = threadIdx.x; e < ranks16 * rows8; e += kThreads) {
      const int at = e / rows8 * kUnitRows + e % rows8;
      float sum = parts[at];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) sum += parts[w * part_values + at];
      s.total[at] = sum;
    }
    if (args.cluster > 1) {
      cluster.sync();
    } else {
      __syncthreads();
    }
    // Element e = (row, rank), ranks side by side as they lie in t; every cluster-th one is this CTA's.
    for (int e = threadIdx.x * args.cluster + rank_of_cta; e < ranks16 * unit.count; e += kThreads * args.cluster) {
      const int row = e / ranks16, r = e % ranks16;
      const int at = r * kUnitRows + row;
      float sum = 0.0f;
      if (args.cluster > 1) {
        float values[kMaxCluster];
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) values[c] = c < args.cluster ? cluster.map_shared_rank(s.total, c)[at] : 0.0f;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) sum += values[c];
      } else {
        sum = s.total[at];
      }
      float rest = r < unit.ranks ? __fmul_rn(sum, scale) : 0.0f;
      uint16_t* to = args.t + (row0 + unit.order[row]) * rank_padded + rank0 + r;
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

// The adapters in use by 256 rows, each once, in the order of their first rows.
__device__ void list_adapters(const ShrinkArgs& args, int64_t tile, int* lists) {
  static_assert(kQuantThreads == kLoraListRows, "a thread for each row");
  __shared__ alignas(16) int ids[kLoraListRows];
  __shared__ int warp_count[kLoraListRows / 32];
  const int i = threadIdx.x;
  const int64_t row = tile * kLoraListRows + i;
  const int mine = row < args.rows ? load_adapter_id(args.adapters, row) : -1;
  ids[i] = mine;
  __syncthreads();
  bool first = mine >= 0;
  for (int j = 0; first && j < i; j += 4) {
    const int4 others = *reinterpret_cast<const int4*>(&ids[j]);
    first = !(others.x == mine || (others.y == mine && j + 1 < i) || (others.z == mine && j + 2 < i) || (others.w == mine && j + 3 < i));
  }
  const unsigned firsts = __ballot_sync(0xffffffffu, first);
  if ((i & 31) == 0) warp_count[i >> 5] = __popc(firsts);
  __syncthreads();
  int slot = __popc(firsts & ((1u << (i & 31)) - 1)), slots = 0;
  for (int w = 0; w < kLoraListRows / 32; ++w) {
    if (w < (i >> 5)) slot += warp_count[w];
    slots += warp_count[w];
  }
  int* const list = lists + tile * kLoraListInts;
  if (i == 0) list[0] = slots;
  if (first) list[1 + slot] = mine;
}

template <bool kVector>
__global__ void __launch_bounds__(kQuantThreads)
lora_quantize_kernel(const uint16_t* __restrict__ x, int cols, int cols_padded, int8_t* __restrict__ q, float* __restrict__ scale_out, int* status,
                     const __grid_constant__ ShrinkArgs args, int* lists) {
  ptx::launch_dependents();
  __shared__ float smem[32];
  if (blockIdx.x == 0 && threadIdx.x < kStatusWords) status[threadIdx.x] = 0;
  if (blockIdx.x >= args.rows) {
    list_adapters(args, static_cast<int64_t>(blockIdx.x) - args.rows, lists);
    return;
  }
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

cudaError_t launch_lora_quantize(const uint16_t* x, int64_t rows, int k, int k_padded, int8_t* q, float* scale, int* status,
                                 const LoraAdapters& adapters, int* lists, cudaStream_t stream) {
  ShrinkArgs args = {};
  args.rows = rows;
  args.adapters = adapters;
  const int64_t tiles = lists != nullptr ? (rows + kLoraListRows - 1) / kLoraListRows : 0;
  const bool vector = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto kernel = vector ? lora_quantize_kernel<true> : lora_quantize_kernel<false>;
  kernel<<<static_cast<unsigned>(rows + tiles), kQuantThreads, 0, stream>>>(x, k, k_padded, q, scale, status, args, lists);
  return cudaGetLastError();
}

cudaError_t launch_lora_shrink(const uint16_t* x, int64_t rows, int k, const LoraAdapters& adapters, uint16_t* t, int planes, cudaStream_t stream) {
  ShrinkArgs args = {x, rows, k, adapters, t, planes, 1, 1};
  const bool vector = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto kernel = vector ? lora_shrink_kernel<true> : lora_shrink_kernel<false>;
  static PerDeviceOnce configured[2];
  const int device = current_device_ordinal();
  constexpr size_t kMostBytes = sizeof(ShrinkShared) + sizeof(float) * kWarps * kUnitValues;
  if (configured[vector].needed(device)) {
    const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostBytes));
    if (error != cudaSuccess) return error;
    configured[vector].mark(device);
  }
  const int64_t tiles = (rows + kTileRows - 1) / kTileRows;
  // The K range is split over more CTAs the fewer tiles there are to fill the chip with.
  const int k32 = (k + 31) / 32;
  args.cluster = 1;
  while (args.cluster < kMaxCluster && tiles * args.cluster < 16 && args.cluster * kWarps * 2 <= k32) args.cluster *= 2;
  const int rank_blocks = (adapters.rank + kLoraRankBlock - 1) / kLoraRankBlock;
  // Units of a tile at most: its rows, and an adapter's groups of 32 rows.
  const int64_t tile_rows = rows < kTileRows ? rows : kTileRows;
  const int64_t most = (adapters.count + tile_rows / kUnitRows < tile_rows ? adapters.count + tile_rows / kUnitRows : tile_rows) * rank_blocks;
  int64_t stride = 4ll * threshold_sms / (tiles * args.cluster);
  if (stride < 4) stride = 4;
  if (stride > most) stride = most;
  args.stride = static_cast<int>(stride);
  const int ranks16 = lora_rank_padded(adapters.rank);
  const size_t smem_bytes = sizeof(ShrinkShared) + sizeof(float) * kWarps * kUnitRows * (ranks16 < kLoraRankBlock ? ranks16 : kLoraRankBlock);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles * args.stride * args.cluster));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem_bytes;
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

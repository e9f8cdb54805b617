// The products of the gated feed-forward block over few rows (gated_gemm.cu has them over many): y = h W2^T, h = act(x Wg^T, x Wu^T),
// d_gate_up = (dy W2) times the derivatives, dx = d_gate_up W13.
//
// Such a product streams its weights once and does almost nothing else: HBM bounds it if enough SMs ask for weights, latency if not.  As in
// dense_gemm.cu a cluster of `parts` CTAs owns a block of 128 weight rows (the lanes of tensor memory; tokens are the columns) and splits the K range, the parts'
// sums meet through distributed shared memory in the order of the parts, and a CTA finishes every parts-th share of the token rows.  The weights
// of every pipeline stage are fetched before the wait for the kernel in front.
//   * The gated projection's block is 64 gate rows and the 64 up rows of the same channels: a token's gate and up lie 64 floats apart in the exchanged sums.
//   * dy W2 and d_gate_up W13 sum over the rows of the weight: its tiles are staged as 64 x 64 blocks and read M-major (gated_gemm.cu).
#include <cuda.h>

#include <mutex>

#include "common.cuh"
#include "gated.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace fmoe {

namespace {

constexpr int kBlockM = 128;        // weight rows per CTA (TMEM lanes)
constexpr int kBlockK = 64;         // elements of K per pipeline stage: 128 bytes
constexpr int kBlockKBytes = 128;
constexpr int kUmmaK = 16;
constexpr int kThreads = 192;       // warp 0: TMA, warp 1: tensor memory and MMA, warps 2..5: epilogue
constexpr int kWeightBytes = kBlockM * kBlockKBytes;
constexpr int kMaxStages = 10;
constexpr int kMaxParts = 8;        // portable cluster size
constexpr int kMinPartBlocks = 2;   // K blocks of a part, at least

enum class Epilogue { kPlain, kGated, kGatedBack };

// kDeep: one CTA per SM with all of its shared memory; otherwise two CTAs fit an SM.
template <int kRowTile, bool kDeep>
struct Config {
  static constexpr int kTokenBytes = kRowTile * kBlockKBytes;
  static constexpr int kStageBytes = kWeightBytes + kTokenBytes;
  static constexpr int kBudget = kDeep ? 200 * 1024 : 100 * 1024;
  static constexpr int kStages = kBudget / kStageBytes < kMaxStages ? kBudget / kStageBytes : kMaxStages;
  static constexpr int kTmemColumns = kRowTile < 32 ? 32 : kRowTile;
  static constexpr size_t kSmemBytes = 1024 /*alignment slack*/ + static_cast<size_t>(kStages) * kStageBytes + 512 /*control block*/;
  static_assert(kStages * kStageBytes >= kRowTile * kBlockM * 4, "the accumulator exchange reuses the stages");
};

struct Control {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(Control) <= 512, "control block exceeds its shared-memory reservation");

struct Args {
  uint16_t* out;
  int64_t rows;
  int n;           // output channels
  int k_blocks;
  int row_tiles, parts;
  int keep;             // the forward pass stores the derivatives
  float4* derivatives;  // see derivative_block
  int activation;
  float limit;
  int* status;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float4 load_cluster_float4(uint32_t smem_address, int cta) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_address), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}

// Four neighbouring sums of all parts.
__device__ __forceinline__ void sum_parts(uint32_t smem_address, int parts, float (&sum)[4]) {
  float4 values[kMaxParts];
#pragma unroll
  for (int c = 0; c < kMaxParts; ++c) {
    values[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < parts) values[c] = load_cluster_float4(smem_address, c);
  }
  float4 s = values[0];
#pragma unroll
  for (int c = 1; c < kMaxParts; ++c) {
    s.x += values[c].x;
    s.y += values[c].y;
    s.z += values[c].z;
    s.w += values[c].w;
  }
  sum[0] = s.x;
  sum[1] = s.y;
  sum[2] = s.z;
  sum[3] = s.w;
}

__device__ __forceinline__ void store4(uint16_t* to, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
}

template <Epilogue kEpilogue, bool kWeightByK, int kRowTile, bool kDeep>
__global__ void __launch_bounds__(kThreads)
gated_small_kernel(const __grid_constant__ CUtensorMap weight_map, const __grid_constant__ CUtensorMap token_map, const __grid_constant__ Args args) {
  using Cfg = Config<kRowTile, kDeep>;
  constexpr int kChannels = kEpilogue == Epilogue::kGated ? kBlockM / 2 : kBlockM;  // output channels of a block
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Control* ctl = reinterpret_cast<Control*>(smem + static_cast<size_t>(Cfg::kStages) * Cfg::kStageBytes);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  int* status = args.status;
  const int parts = args.parts;
  const int part = static_cast<int>(blockIdx.x) % parts;  // = rank in the cluster
  const int unit = static_cast<int>(blockIdx.x) / parts;  // row tiles of a channel block side by side: they share its weights
  const int block = unit / args.row_tiles;
  const int64_t row0 = static_cast<int64_t>(unit - block * args.row_tiles) * kRowTile;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRowTile), args.rows - row0));
  const int n0 = block * kChannels;
  const int kb_begin = part * args.k_blocks / parts;
  const int count = (part + 1) * args.k_blocks / parts - kb_begin;  // K blocks of this CTA, at least one

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      ptx::mbar_init(&ctl->full[s], 1);
      ptx::mbar_init(&ctl->empty[s], 1);
    }
    ptx::mbar_init(&ctl->acc_full, 1);
    ctl->abort_flag = 0;
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(&ctl->tmem_base, Cfg::kTmemColumns);
    ptx::tmem_relinquish();
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  volatile int* abort_flag = &ctl->abort_flag;

  if (warp == 0) {
    // ---------------- TMA producer (the whole warp walks the loops, one elected lane issues) ----------------
    const bool issuer = ptx::elect_one();
    const int ahead = count < Cfg::kStages ? count : Cfg::kStages;
    auto load_weights = [&](int stage, int i) {
      uint8_t* const to = smem + static_cast<size_t>(stage) * Cfg::kStageBytes;
      const int k0 = (kb_begin + i) * kBlockK;
      if constexpr (kEpilogue == Epilogue::kGated) {
        ptx::tma_load_2d(to, &weight_map, &ctl->full[stage], k0, n0);
        ptx::tma_load_2d(to + kWeightBytes / 2, &weight_map, &ctl->full[stage], k0, args.n + n0);
      } else if constexpr (kWeightByK) {
        ptx::tma_load_2d(to, &weight_map, &ctl->full[stage], n0, k0);
        ptx::tma_load_2d(to + kWeightBytes / 2, &weight_map, &ctl->full[stage], n0 + 64, k0);
      } else {
        ptx::tma_load_2d(to, &weight_map, &ctl->full[stage], k0, n0);
      }
    };
    auto load_tokens = [&](int stage, int i) {
      ptx::tma_load_2d(smem + static_cast<size_t>(stage) * Cfg::kStageBytes + kWeightBytes, &token_map, &ctl->full[stage], (kb_begin + i) * kBlockK,
                       static_cast<int>(row0));
    };
    // Weights of the first stages: they do not depend on the kernel that may still be running.
    for (int i = 0; i < ahead; ++i) {
      if (issuer) {
        ptx::mbar_arrive_expect_tx(&ctl->full[i], Cfg::kStageBytes);
        load_weights(i, i);
      }
    }
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    for (int i = 0; i < ahead; ++i) {
      if (issuer) load_tokens(i, i);
    }
    int stage = ahead == Cfg::kStages ? 0 : ahead;
    uint32_t phase = ahead == Cfg::kStages ? 1u : 0u;
    for (int i = ahead; i < count; ++i) {
      ptx::mbar_wait(&ctl->empty[stage], phase ^ 1u, abort_flag, status, 61);
      if (issuer) {
        ptx::mbar_arrive_expect_tx(&ctl->full[stage], Cfg::kStageBytes);
        load_weights(stage, i);
        load_tokens(stage, i);
      }
      if (++stage == Cfg::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Drain: every load must have landed before the CTA may exit (the MMA warp has consumed them unless it gave up).
    for (int back = 0; back < ahead; ++back) {
      int s = stage - 1 - back;
      uint32_t p = phase;
      if (s < 0) {
        s += Cfg::kStages;
        p ^= 1u;
      }
      const unsigned long long start = ptx::global_timer_ns();
      while (!ptx::mbar_try_wait(&ctl->full[s], p)) {
        if (ptx::global_timer_ns() - start > ptx::kWaitLimitNs) break;
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const bool issuer = ptx::elect_one();
    const uint32_t idesc = ptx::make_instr_desc(false, kBlockM, (rows + 15) & ~15) | (kWeightByK ? 1u << 15 : 0u);
    // M-major weights: the two 64-row blocks lie half a tile apart, the next 16 K elements two groups of eight 128-byte rows on.
    constexpr uint64_t kLead = static_cast<uint64_t>((kWeightBytes / 2) >> 4) << 16;
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < count; ++i) {
      ptx::mbar_wait(&ctl->full[stage], phase, abort_flag, status, 62);
      ptx::tcgen05_fence_after();
      const uint32_t stage_addr = ptx::smem_u32(smem + static_cast<size_t>(stage) * Cfg::kStageBytes);
      if (issuer) {
#pragma unroll
        for (int ks = 0; ks < kBlockK / kUmmaK; ++ks) {
          const uint64_t weights = kWeightByK ? (ptx::make_smem_desc_sw128(stage_addr + ks * 2048) & ~(0x3fffull << 16)) | kLead
                                              : ptx::make_smem_desc_sw128(stage_addr + ks * kUmmaK * 2);
          ptx::umma_ss<false>(tmem_base, weights, ptx::make_smem_desc_sw128(stage_addr + kWeightBytes + ks * kUmmaK * 2), idesc, (i > 0 || ks > 0) ? 1u : 0u);
        }
        ptx::tcgen05_commit(&ctl->empty[stage]);
      }
      if (++stage == Cfg::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (issuer) ptx::tcgen05_commit(&ctl->acc_full);
  }

  // ---------------- epilogue (warps 2..5): sums to shared memory, then every CTA its share of the token rows ----------------
  float* exchange = reinterpret_cast<float*>(smem);  // [rows][128 weight rows], once the stages are done with
  if (warp >= 2) {
    const int quarter = warp & 3;  // the TMEM lanes a warp may read are fixed by warp id % 4
    const int channel = quarter * 32 + lane;
    ptx::grid_dependency_wait();  // what the kernel in front reads or writes is written below
    ptx::mbar_wait(&ctl->acc_full, 0, abort_flag, status, 63);
    ptx::tcgen05_fence_after();
    const uint32_t acc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    for (int c0 = 0; c0 < rows; c0 += 16) {
      uint32_t bits[16];
      ptx::tmem_ld_x8(acc + c0, bits);
      ptx::tmem_ld_x8(acc + c0 + 8, bits + 8);
      ptx::tmem_ld_wait();
      // (Rows of the last sixteen that do not exist have room in the stages too.)
#pragma unroll
      for (int j = 0; j < 16; ++j) exchange[(c0 + j) * kBlockM + channel] = __uint_as_float(bits[j]);
      __syncwarp();  // the next tensor-memory load wants the whole warp
    }
  }
  __syncwarp();
  cluster_sync();  // every part's sums lie in its shared memory
  if (warp >= 2) {
    const uint32_t base = ptx::smem_u32(exchange);
    const int share = (rows + parts - 1) / parts;
    const int own_end = min(rows, (part + 1) * share);
    if constexpr (kEpilogue == Epilogue::kGated) {
      // Half a warp finishes 64 channels of a row, four per lane.
      const int c4 = 4 * (lane & 15);
      const int n = n0 + c4;
      for (int row = part * share + 2 * (warp - 2) + (lane >> 4); row < own_end; row += 8) {
        float gate[4], up[4], h[4], by_gate[4], by_up[4];
        sum_parts(base + 4u * static_cast<uint32_t>(row * kBlockM + c4), parts, gate);
        sum_parts(base + 4u * static_cast<uint32_t>(row * kBlockM + kBlockM / 2 + c4), parts, up);
        if (n >= args.n) continue;
        with_activation<false>(args.activation, [&](auto act) {
#pragma unroll
          for (int j = 0; j < 4; ++j) gated_with_derivatives(act, gate[j], up[j], args.limit, &h[j], &by_gate[j], &by_up[j]);
        });
        store4(args.out + (row0 + row) * args.n + n, h);
        if (args.keep) {
          float4* const by = args.derivatives + derivative_block(row0 + row, n, args.n) + (n & 31) / 4 * 32 + ((row0 + row) & 31);
          by[0] = make_float4(by_gate[0], by_gate[1], by_gate[2], by_gate[3]);
          by[256] = make_float4(by_up[0], by_up[1], by_up[2], by_up[3]);
        }
      }
    } else {
      const int c4 = 4 * lane;
      const int n = n0 + c4;
      for (int row = part * share + (warp - 2); row < own_end; row += 4) {
        float4 by_gate = make_float4(0.0f, 0.0f, 0.0f, 0.0f), by_up = by_gate;
        if constexpr (kEpilogue == Epilogue::kGatedBack) {
          if (n < args.n) {
            const float4* const by = args.derivatives + derivative_block(row0 + row, n, args.n) + (n & 31) / 4 * 32 + ((row0 + row) & 31);
            by_gate = __ldcs(by);
            by_up = __ldcs(by + 256);
          }
        }
        float sum[4];
        sum_parts(base + 4u * static_cast<uint32_t>(row * kBlockM + c4), parts, sum);
        if (n >= args.n) continue;
        if constexpr (kEpilogue == Epilogue::kGatedBack) {
          uint16_t* const to = args.out + (row0 + row) * 2 * args.n + n;
          const float d_gate[4] = {sum[0] * by_gate.x, sum[1] * by_gate.y, sum[2] * by_gate.z, sum[3] * by_gate.w};
          const float d_up[4] = {sum[0] * by_up.x, sum[1] * by_up.y, sum[2] * by_up.z, sum[3] * by_up.w};
          store4(to, d_gate);
          store4(to + args.n, d_up);
        } else {
          store4(args.out + (row0 + row) * args.n + n, sum);
        }
      }
    }
  }
  __syncwarp();
  cluster_sync();  // no part leaves while another may still read its sums

  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem_base, Cfg::kTmemColumns);
  }
}

// How many clusters of 1 .. kMaxParts CTAs can be resident at once with one CTA per SM (asked once per device: a cluster
// lives inside a GPC, so this is less than SMs / cluster size).  Also sets the kernels' shared-memory attributes.
struct Residency {
  int clusters[kMaxParts + 1] = {};
};

template <Epilogue kEpilogue, bool kWeightByK, int kRowTile, bool kDeep>
cudaError_t configure() {
  auto kernel = gated_small_kernel<kEpilogue, kWeightByK, kRowTile, kDeep>;
  const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Config<kRowTile, kDeep>::kSmemBytes));
  return error != cudaSuccess ? error : cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

template <Epilogue kEpilogue, bool kWeightByK, int kRowTile>
cudaError_t residency(Residency* out) {
  static std::mutex guard;  // a thread that finds the flag set has to find the table too
  static PerDeviceOnce configured;
  static Residency known[kMaxDevices];
  const std::lock_guard<std::mutex> lock(guard);
  const int device = current_device_ordinal();
  if (!configured.needed(device)) {
    *out = known[device];
    return cudaSuccess;
  }
  cudaError_t error = configure<kEpilogue, kWeightByK, kRowTile, true>();
  if (error == cudaSuccess) error = configure<kEpilogue, kWeightByK, kRowTile, false>();
  for (int parts = 1; parts <= kMaxParts && error == cudaSuccess; ++parts) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(parts));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = Config<kRowTile, true>::kSmemBytes;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = static_cast<unsigned>(parts);
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    error = cudaOccupancyMaxActiveClusters(&out->clusters[parts], gated_small_kernel<kEpilogue, kWeightByK, kRowTile, true>, &config);
  }
  if (error != cudaSuccess) return error;
  if (device >= 0 && device < kMaxDevices) known[device] = *out;
  configured.mark(device);
  return cudaSuccess;
}

template <Epilogue kEpilogue, bool kWeightByK, int kRowTile, bool kDeep>
cudaError_t launch_kernel(const Args& args, int64_t blocks, const CUtensorMap* maps, cudaStream_t stream, bool chained) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(blocks * args.parts));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = Config<kRowTile, kDeep>::kSmemBytes;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = static_cast<unsigned>(args.parts);
  attributes[0].val.clusterDim.y = 1;
  attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = chained ? 2 : 1;
  return cudaLaunchKernelEx(&config, gated_small_kernel<kEpilogue, kWeightByK, kRowTile, kDeep>, maps[0], maps[1], args);
}

struct Operands {
  const uint16_t* weight;
  int64_t weight_rows, weight_columns;  // as they lie in memory
  const uint16_t* tokens;
  int64_t token_stride;
  int k;
};

template <Epilogue kEpilogue, bool kWeightByK, int kRowTile>
cudaError_t launch_tile(Args args, const Operands& o, cudaStream_t stream, bool chained) {
  CUtensorMap maps[2];
  constexpr uint32_t kWeightBox = kEpilogue == Epilogue::kGated || kWeightByK ? 64 : kBlockM;
  if (!make_sw128_map(&maps[0], o.weight, false, static_cast<uint64_t>(o.weight_rows), static_cast<uint64_t>(o.weight_columns), kWeightBox) ||
      !make_sw128_map(&maps[1], o.tokens, false, static_cast<uint64_t>(args.rows), static_cast<uint64_t>(o.k), kRowTile, static_cast<uint64_t>(o.token_stride))) {
    return cudaErrorInvalidValue;
  }
  Residency one_per_sm;
  const cudaError_t error = residency<kEpilogue, kWeightByK, kRowTile>(&one_per_sm);
  if (error != cudaSuccess) return error;
  constexpr int kChannels = kEpilogue == Epilogue::kGated ? kBlockM / 2 : kBlockM;
  args.k_blocks = (o.k + kBlockK - 1) / kBlockK;
  args.row_tiles = static_cast<int>((args.rows + kRowTile - 1) / kRowTile);
  const int64_t blocks = static_cast<int64_t>((args.n + kChannels - 1) / kChannels) * args.row_tiles;
  if (blocks > (1ll << 27)) return cudaErrorInvalidValue;
  // As many parts as leave all clusters resident at once, two CTAs per SM if need be, every part at least two K blocks (dense_gemm.cu): one row of 7168 x 2048,
  // 2 / 4 / 6 parts of the gated projection: 24.5 / 22.2 / 20.7 us for the block; 256 rows, 4 / 2 parts of the down projection: 44.9 / 38.2 us.
  args.parts = 1;
  for (int parts = kMaxParts; parts > 1; --parts) {
    if (blocks <= 2 * one_per_sm.clusters[parts] && parts * kMinPartBlocks <= args.k_blocks) {
      args.parts = parts;
      break;
    }
  }
  if (blocks <= one_per_sm.clusters[args.parts]) return launch_kernel<kEpilogue, kWeightByK, kRowTile, true>(args, blocks, maps, stream, chained);
  return launch_kernel<kEpilogue, kWeightByK, kRowTile, false>(args, blocks, maps, stream, chained);
}

template <Epilogue kEpilogue, bool kWeightByK>
cudaError_t launch(const Args& args, const Operands& operands, cudaStream_t stream, bool chained) {
  if (args.rows <= 16) return launch_tile<kEpilogue, kWeightByK, 16>(args, operands, stream, chained);
  if (args.rows <= 32) return launch_tile<kEpilogue, kWeightByK, 32>(args, operands, stream, chained);
  if (args.rows <= 64) return launch_tile<kEpilogue, kWeightByK, 64>(args, operands, stream, chained);
  return launch_tile<kEpilogue, kWeightByK, 128>(args, operands, stream, chained);
}

}  // namespace

cudaError_t launch_gated_projection_small(const uint16_t* x, int64_t x_stride, const uint16_t* w13, int64_t rows, int hidden, int inter, int activation,
                                          float limit, uint16_t* h, float* derivatives, int* status, cudaStream_t stream, bool chained) {
  Args args = {};
  args.out = h;
  args.rows = rows;
  args.n = inter;
  args.keep = derivatives != nullptr ? 1 : 0;
  args.derivatives = reinterpret_cast<float4*>(derivatives);
  args.activation = activation;
  args.limit = limit;
  args.status = status;
  return launch<Epilogue::kGated, false>(args, {w13, 2 * static_cast<int64_t>(inter), hidden, x, x_stride, hidden}, stream, chained);
}

cudaError_t launch_gated_backward_small(const uint16_t* dy, int64_t dy_stride, const uint16_t* w2, const float* derivatives, int64_t rows, int hidden,
                                        int inter, uint16_t* d_gate_up, int* status, cudaStream_t stream, bool chained) {
  Args args = {};
  args.out = d_gate_up;
  args.rows = rows;
  args.n = inter;
  args.derivatives = reinterpret_cast<float4*>(const_cast<float*>(derivatives));
  args.status = status;
  return launch<Epilogue::kGatedBack, true>(args, {w2, hidden, inter, dy, dy_stride, hidden}, stream, chained);
}

cudaError_t launch_dense_small(const uint16_t* tokens, int64_t rows, int k, const uint16_t* weight, int n, bool weight_by_k, uint16_t* out, int* status,
                               cudaStream_t stream, bool chained) {
  Args args = {};
  args.out = out;
  args.rows = rows;
  args.n = n;
  args.status = status;
  if (weight_by_k) return launch<Epilogue::kPlain, true>(args, {weight, k, n, tokens, k, k}, stream, chained);
  return launch<Epilogue::kPlain, false>(args, {weight, n, k, tokens, k, k}, stream, chained);
}

}  // namespace fmoe

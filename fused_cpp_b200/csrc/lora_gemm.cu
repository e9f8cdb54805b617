// Dense W8A8 linear with the low-rank adapters of many requests:
//   out[row, n] = (acc * row scale) * channel scale (+ bias[n]) + sum over r of t[row, r] B[a, n, r],   acc = Xq W^T, a = the row's adapter,
// with the coefficients t of lora_front.cu.  The kernel of dense_gemm.cu (128 output channels of a cluster of `parts` CTAs that split the K
// range; their int32 sums meet in distributed shared memory) with the adapters' product beside it, in a second accumulator of tensor memory:
//   * Rows of a tile may have any adapters in any order.  For each adapter in use by the rows, [t of its rows, zeros for the others] x B[a]^T
//     is one of bf16 MMAs: a K block of 128-byte rows, as the weights' are, holds 64 ranks of one adapter or two or four adapters of up to 32 or 16
//     ranks, B[a] comes by the same ring of stages, and four warps write the masked coefficients where the token tile would lie.  A row's sum has only its own adapter's products and exact
//     zeros in it (adapters are finite by contract), whatever its neighbours ask for.
//   * A CTA finishes the rows [part * R, part * R + R) of its tile (R = rows / parts): it multiplies the adapters of those rows alone, so that
//     nothing of that product is exchanged, and every adapter's channels are read by the CTAs whose rows use it.
//   * The list of adapters comes from the ids before the wait for the kernels in front; what is behind it is the t and the tokens.
#include <cuda.h>

#include <mutex>

#include "common.cuh"
#include "gated.cuh"
#include "kernels.h"
#include "lora.h"
#include "ptx.cuh"

namespace fmoe {

namespace {

constexpr int kBlockM = 128;        // output channels per CTA (TMEM lanes)
constexpr int kBlockKBytes = 128;   // bytes of K per pipeline stage = one 128-byte swizzle row
constexpr int kUmmaKBytes = 32;     // bytes of K per tcgen05.mma, of either kind
constexpr int kThreads = 192;       // warp 0: TMA, warp 1: tensor memory and MMA, warps 2..5: masked coefficients, then epilogue
constexpr int kWeightBytes = kBlockM * kBlockKBytes;
constexpr int kMaxStages = 10;
constexpr int kMaxParts = 8;
constexpr int kLeastTile = 16;
constexpr int kMinPartBlocks = 2;
constexpr int kTileRows = 128;
constexpr int kWriters = 4;         // warps that write masked coefficients

template <int kRowTile, bool kDeep, int kTerms>
struct LoraConfig {
  static constexpr int kLoadBytes = kWeightBytes + kRowTile * kBlockKBytes;
  static constexpr int kBudget = kDeep ? 200 * 1024 : 98 * 1024;
  // Rows of a stage's token tile.  The terms of fp32 results' coefficients lie one under the other in it where they fit, so that a tile of B serves them all.
  static constexpr int kHeldRows = kTerms > 1 && kRowTile < 16 * kTerms ? 16 * kTerms : kRowTile;
  static constexpr int kStageBytes = kWeightBytes + kHeldRows * kBlockKBytes;
  static constexpr int kStages = kBudget / kStageBytes < kMaxStages ? kBudget / kStageBytes : kMaxStages;
  static constexpr int kTmemColumns = 2 * kRowTile;  // the int32 and the fp32 accumulator
  static constexpr size_t kSmemBytes = 1024 /*alignment slack*/ + static_cast<size_t>(kStages) * kStageBytes + 4096 /*control block*/;
  // With two parts and more a CTA finishes at most half of the rows (in whole sixteens).
  static_assert(kStages * kStageBytes >= (kRowTile + (kRowTile > 16 ? kRowTile / 2 : 16)) * kBlockM * 4, "the accumulator exchange and the adapters' sums reuse the stages");
};

struct LoraControl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t vacant[kMaxStages];        // the producer found the stage empty and leaves its token tile to the coefficients
  uint64_t coefficients[kMaxStages];  // the masked coefficients of the stage are written
  uint64_t acc_full;
  uint64_t listed;  // the list of adapters is there
  uint32_t tmem_base;
  volatile int abort_flag;
  int slots;
  alignas(16) float row_scale[kTileRows];
  alignas(16) float channel_scale[kBlockM];
  alignas(16) float channel_bias[kBlockM];
  int slot[kTileRows];  // of the own rows: place of their adapter in the list, -1 = none
  int slot_adapter[kTileRows];
};
static_assert(sizeof(LoraControl) <= 4096, "control block exceeds its shared-memory reservation");

struct KernelArgs {
  LoraGemmArgs g;
  int row_tiles, k_blocks, parts, vector_store, rank_blocks;
  LoraBlock block;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ int4 load_cluster_int4(uint32_t smem_address, int cta) {
  uint32_t remote;
  int4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_address), "r"(cta));
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      :
      : "r"(ptx::smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ float finish(int acc, float row_scale, float channel_scale, float bias, float delta) {
  return __fadd_rn(__fadd_rn(dequantize(acc, row_scale, channel_scale, FMOE_NUMERICS_TORCHREF), bias), delta);
}

__device__ __forceinline__ void store_value(const LoraGemmArgs& g, int64_t index, float value) {
  if (g.out_bf16) {
    static_cast<uint16_t*>(g.out)[index] = __bfloat16_as_ushort(__float2bfloat16_rn(value));
  } else {
    static_cast<float*>(g.out)[index] = value;
  }
}

template <int kRowTile, bool kDeep, int kTerms>
__global__ void __launch_bounds__(kThreads)
lora_gemm_kernel(const __grid_constant__ CUtensorMap weight_map, const __grid_constant__ CUtensorMap token_map, const __grid_constant__ CUtensorMap b_map,
                 const __grid_constant__ KernelArgs args) {
  using Cfg = LoraConfig<kRowTile, kDeep, kTerms>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  LoraControl* ctl = reinterpret_cast<LoraControl*>(smem + static_cast<size_t>(Cfg::kStages) * Cfg::kStageBytes);
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  int* status = args.g.status;
  const int parts = args.parts;
  const int part = static_cast<int>(blockIdx.x) % parts;  // = rank in the cluster
  const int unit = static_cast<int>(blockIdx.x) / parts;  // row tiles of a channel block side by side: they share its weights
  const int block = unit / args.row_tiles;
  const int64_t row0 = static_cast<int64_t>(unit - block * args.row_tiles) * kRowTile;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRowTile), args.g.rows - row0));
  const int rows_per_part = (rows + parts - 1) / parts;
  const int own_first = min(part * rows_per_part, rows);  // the rows of the tile that this CTA finishes
  const int own = min(rows_per_part, rows - own_first);
  const int n = args.g.n;
  const int n0 = block * kBlockM;
  const int kb_begin = part * args.k_blocks / parts;
  const int count = (part + 1) * args.k_blocks / parts - kb_begin;  // K blocks of this CTA, at least one

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      ptx::mbar_init(&ctl->full[s], 1);
      ptx::mbar_init(&ctl->empty[s], 1);
      ptx::mbar_init(&ctl->vacant[s], 1);
      ptx::mbar_init(&ctl->coefficients[s], kWriters);
    }
    ptx::mbar_init(&ctl->acc_full, 1);
    ptx::mbar_init(&ctl->listed, 1);
    ctl->slots = 0;
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
  if (warp == 2) {
    // The adapters of the own rows, each once, in the order of their first rows.
    int slots = 0;
    for (int base = 0; base < own; base += 32) {
      const int i = base + lane;
      const int id = i < own ? load_adapter_id(args.g.adapters, row0 + own_first + i) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, id);
      int slot = -1;  // of an earlier row's
      if (id >= 0) {
        for (int j = 0; j < slots; ++j) slot = ctl->slot_adapter[j] == id ? j : slot;
      }
      const bool first = id >= 0 && slot < 0 && (same & ((1u << lane) - 1)) == 0;
      const unsigned firsts = __ballot_sync(0xffffffffu, first);
      if (first) ctl->slot_adapter[slots + __popc(firsts & ((1u << lane) - 1))] = id;
      // A row whose adapter appears first in these 32 has the slot of that first row.
      if (id >= 0 && slot < 0) slot = slots + __popc(firsts & ((1u << (__ffs(same) - 1)) - 1));
      if (i < own) ctl->slot[i] = slot;
      slots += __popc(firsts);
      __syncwarp();
    }
    if (lane == 0) {
      ctl->slots = slots;
      ptx::mbar_arrive(&ctl->listed);
    }
  } else if (warp == 0) {
    // Weights of the first Cfg::kStages: they depend neither on the ids nor on the kernels that may still be running.
    if (ptx::elect_one()) {
      for (int i = 0; i < (count < Cfg::kStages ? count : Cfg::kStages); ++i) {
        ptx::mbar_arrive_expect_tx(&ctl->full[i], Cfg::kLoadBytes);
        ptx::tma_load_2d(smem + static_cast<size_t>(i) * Cfg::kStageBytes, &weight_map, &ctl->full[i], (kb_begin + i) * kBlockKBytes, n0);
      }
    }
    __syncwarp();
  }
  ptx::mbar_wait(&ctl->listed, 0, abort_flag, status, 56);
  const int slots = __shfl_sync(0xffffffffu, ctl->slots, 0);
  // K blocks of the adapters' product: for every plane of every 64 ranks, the adapters one after the other, per_block in a block.
  const int per_block = args.block.adapters;
  const int slot_blocks = (slots + per_block - 1) / per_block;
  const uint32_t adapter_bytes = static_cast<uint32_t>(kBlockM) * args.block.ranks * 2;  // of one adapter's tile
  const int own16 = (own + 15) & ~15;
  const int together = kTerms * own16 <= Cfg::kHeldRows ? kTerms : 1;  // terms of the coefficients in a block
  const int rounds = kTerms / together;
  const int extra = slot_blocks * args.rank_blocks * rounds;
  const int all = count + extra;

  if (warp == 0) {
    // ---------------- TMA producer (the whole warp walks the loops, one elected lane issues) ----------------
    const bool issuer = ptx::elect_one();
    const int ahead = count < Cfg::kStages ? count : Cfg::kStages;
    ptx::grid_dependency_wait();
    for (int i = 0; i < ahead; ++i) {
      if (issuer) {
        ptx::tma_load_2d(smem + static_cast<size_t>(i) * Cfg::kStageBytes + kWeightBytes, &token_map, &ctl->full[i], (kb_begin + i) * kBlockKBytes,
                         static_cast<int>(row0));
      }
    }
    int stage = ahead == Cfg::kStages ? 0 : ahead;
    uint32_t phase = ahead == Cfg::kStages ? 1u : 0u;
    for (int i = ahead; i < all; ++i) {
      ptx::mbar_wait(&ctl->empty[stage], phase ^ 1u, abort_flag, status, 51);
      if (issuer) {
        uint8_t* stage_base = smem + static_cast<size_t>(stage) * Cfg::kStageBytes;
        if (i < count) {
          ptx::mbar_arrive_expect_tx(&ctl->full[stage], Cfg::kLoadBytes);
          ptx::tma_load_2d(stage_base, &weight_map, &ctl->full[stage], (kb_begin + i) * kBlockKBytes, n0);
          ptx::tma_load_2d(stage_base + kWeightBytes, &token_map, &ctl->full[stage], (kb_begin + i) * kBlockKBytes, static_cast<int>(row0));
        } else {
          const int u = i - count;
          const int rank_block = u / slot_blocks / rounds;
          const int slot = u % slot_blocks * per_block;
          const int here = min(per_block, slots - slot);
          ptx::mbar_arrive(&ctl->vacant[stage]);
          ptx::mbar_arrive_expect_tx(&ctl->full[stage], here * adapter_bytes);
          for (int g = 0; g < here; ++g) {
            tma_load_3d(stage_base + g * adapter_bytes, &b_map, &ctl->full[stage], rank_block * kLoraRankBlock, n0, ctl->slot_adapter[slot + g]);
          }
        }
      }
      if (++stage == Cfg::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Drain: every load must have landed before the CTA may exit (the MMA warp has consumed them unless it gave up).
    const int pending = all < Cfg::kStages ? all : Cfg::kStages;
    for (int back = 0; back < pending; ++back) {
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
    const uint32_t idesc = ptx::make_instr_desc(true, kBlockM, (rows + 15) & ~15);
    const uint32_t b_desc_hi = lora_desc_hi(args.block.ranks);
    const uint32_t idesc_extra = ptx::make_instr_desc(false, kBlockM, (own + 15) & ~15);
    int stage = 0;
    uint32_t phase = 0;
    uint32_t used = 0;  // Cfg::kStages, one bit each, whose coefficients barrier is in its odd phase
    for (int i = 0; i < all; ++i) {
      ptx::mbar_wait(&ctl->full[stage], phase, abort_flag, status, 52);
      if (i >= count) {
        ptx::mbar_wait(&ctl->coefficients[stage], (used >> stage) & 1u, abort_flag, status, 53);
        used ^= 1u << stage;
      }
      ptx::tcgen05_fence_after();
      const uint32_t stage_addr = ptx::smem_u32(smem + static_cast<size_t>(stage) * Cfg::kStageBytes);
      if (issuer) {
        if (i < count) {
#pragma unroll
          for (int ks = 0; ks < kBlockKBytes / kUmmaKBytes; ++ks) {
            ptx::umma_ss<true>(tmem_base, ptx::make_smem_desc_sw128(stage_addr + ks * kUmmaKBytes),
                               ptx::make_smem_desc_sw128(stage_addr + kWeightBytes + ks * kUmmaKBytes), idesc, (i > 0 || ks > 0) ? 1u : 0u);
          }
        } else {
          const int rank_block = (i - count) / slot_blocks / rounds;
          const int here = min(per_block, slots - (i - count) % slot_blocks * per_block);
          const int steps = (min(args.block.ranks, args.g.adapters.rank - rank_block * kLoraRankBlock) + 15) >> 4;  // of an adapter
          for (int g = 0; g < here; ++g) {
            const uint32_t b_lo = (((stage_addr + g * adapter_bytes) & 0x3ffffu) >> 4) | (1u << 16);
            for (int ks = 0; ks < steps; ++ks) {
              // (B is this MMA's A operand: channels are the lanes.)
              for (int plane = 0; plane < together; ++plane) {
                ptx::umma_ss<false>(tmem_base + kRowTile, static_cast<uint64_t>(b_desc_hi) << 32 | (b_lo + 2u * ks),
                                    ptx::make_smem_desc_sw128(stage_addr + kWeightBytes + plane * own16 * kBlockKBytes + (g * steps + ks) * kUmmaKBytes), idesc_extra,
                                    (i > count || g > 0 || ks > 0 || plane > 0) ? 1u : 0u);
              }
            }
          }
        }
        ptx::tcgen05_commit(&ctl->empty[stage]);
      }
      if (++stage == Cfg::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (issuer) ptx::tcgen05_commit(&ctl->acc_full);
  } else if (extra > 0) {
    // ---------------- masked coefficients (warps 2..5) ----------------
    // A thread holds up to eight 16-byte pieces of the own rows' coefficients (all terms of them, or one after the other), and for each adapter in turn writes those of its rows and zeros
    // for the others.  (Loaded again for every adapter, by one warp: 201 rows of 1536 -> 24576 with four adapters of rank 64 97.6 us.)
    ptx::grid_dependency_wait();
    const int thread = static_cast<int>(threadIdx.x) - 64;
    const int rank_padded = lora_rank_padded(args.g.adapters.rank);
    const uint16_t* const t_rows = args.g.t + (row0 + own_first) * rank_padded;
    constexpr int kPieces = Cfg::kHeldRows * 8 / 128;  // of a thread
    const int share = args.block.ranks / 8;       // 16-byte pieces of an adapter in a row of 128 bytes: 2, 4 or 8
    int stage = count % Cfg::kStages;
    uint32_t used = 0;  // Cfg::kStages, one bit each, whose vacant barrier is in its odd phase
    for (int outer = 0; outer < args.rank_blocks * rounds; ++outer) {
      const int rank0 = outer / rounds * kLoraRankBlock;
      const int plane0 = outer % rounds;  // together == 1, or the first of all
      const int pieces = 2 * ((min(args.block.ranks, args.g.adapters.rank - rank0) + 15) >> 4);  // of 16 bytes with ranks, in an adapter's share of a row
      const uint16_t* const from = t_rows + rank0;
      uint4 value[kPieces];
      int block[kPieces];  // the row's adapter is in this block, at this piece (or in none)
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int e = thread + 128 * p;
        const int plane = kTerms > 1 ? (e / 8 >= own16) + (e / 8 >= 2 * own16) : 0, row = e / 8 - plane * own16, piece = e % 8;
        value[p] = make_uint4(0, 0, 0, 0);
        block[p] = -1;
        const int slot = plane < together && row < own ? ctl->slot[row] : -1;  // (a row from 3 * own16 on is none of its own)
        if (slot >= 0 && slot % per_block == piece / share) {
          block[p] = slot / per_block;
          if (piece % share < pieces) value[p] = __ldcg(reinterpret_cast<const uint4*>(from + ((plane0 + plane) * args.g.rows + row) * rank_padded) + piece % share);
        }
      }
      for (int b = 0; b < slot_blocks; ++b) {
        // (Not the empty barrier itself: these warps do not see its earlier phases, and would take one for another.)
        ptx::mbar_wait(&ctl->vacant[stage], (used >> stage) & 1u, abort_flag, status, 54);
        used ^= 1u << stage;
        uint8_t* const to = smem + static_cast<size_t>(stage) * Cfg::kStageBytes + kWeightBytes;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          const int e = thread + 128 * p;
          const int row = e / 8, piece = e % 8;
          // The 128-byte swizzle that the operand tiles have: the 16-byte piece's number is xor-ed with the row's in its group of eight.
          if (row < together * own16) *reinterpret_cast<uint4*>(to + row * kBlockKBytes + ((piece ^ (row & 7)) << 4)) = block[p] == b ? value[p] : make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&ctl->coefficients[stage]);
        if (++stage == Cfg::kStages) stage = 0;
      }
    }
  }

  // ---------------- epilogue (warps 2..5): one thread per channel ----------------
  const int quarter = warp & 3;  // the TMEM lanes a warp may read are fixed by warp id % 4
  const int channel = quarter * 32 + lane;
  const bool channel_ok = n0 + channel < n;
  const bool epilogue = warp >= 2;
  float channel_scale = 1.0f, bias = 0.0f;
  int* exchange = reinterpret_cast<int*>(smem);                          // [rows][128 channels], once the Cfg::kStages are done with
  float* deltas = reinterpret_cast<float*>(smem) + kRowTile * kBlockM;  // [own rows][128 channels]: the adapters' sums
  const uint32_t acc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  if (epilogue) {
    const int thread = static_cast<int>(threadIdx.x) - 64;
    // Before the wait, hence through L2: a scale or bias that an earlier call read at this address may still lie in L1.
    if (channel_ok) {
      channel_scale = __ldcg(args.g.w_scale + n0 + channel);
      if (args.g.bias != nullptr) bias = __ldcg(args.g.bias + n0 + channel);
    }
    ctl->channel_scale[channel] = channel_scale;
    ctl->channel_bias[channel] = bias;
    ptx::grid_dependency_wait();  // the row scales come from the quantiser
    if (thread < rows) ctl->row_scale[thread] = __ldcg(args.g.a_scale + row0 + thread);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    ptx::mbar_wait(&ctl->acc_full, 0, abort_flag, status, 55);
    ptx::tcgen05_fence_after();
    for (int c0 = 0; c0 < rows; c0 += 16) {
      uint32_t bits[16], delta[16];
      ptx::tmem_ld_x8(acc + c0, bits);
      ptx::tmem_ld_x8(acc + c0 + 8, bits + 8);
      if (parts == 1 && extra > 0) {
        ptx::tmem_ld_x8(acc + kRowTile + c0, delta);
        ptx::tmem_ld_x8(acc + kRowTile + c0 + 8, delta + 8);
      }
      ptx::tmem_ld_wait();
      if (parts > 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j) exchange[(c0 + j) * kBlockM + channel] = static_cast<int>(bits[j]);
      } else if (channel_ok) {
        const int count16 = min(16, rows - c0);
        const int64_t index = (row0 + c0) * n + n0 + channel;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (j >= count16) break;
          const float value = finish(static_cast<int>(bits[j]), ctl->row_scale[c0 + j], channel_scale, bias, extra > 0 ? __uint_as_float(delta[j]) : 0.0f);
          store_value(args.g, index + static_cast<int64_t>(j) * n, value);
        }
      }
      __syncwarp();  // the next tensor-memory load wants the whole warp
    }
    if (parts > 1 && extra > 0) {
      for (int c0 = 0; c0 < own; c0 += 16) {
        uint32_t bits[16];
        ptx::tmem_ld_x8(acc + kRowTile + c0, bits);
        ptx::tmem_ld_x8(acc + kRowTile + c0 + 8, bits + 8);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) deltas[(c0 + j) * kBlockM + channel] = __uint_as_float(bits[j]);
        __syncwarp();
      }
    }
  }
  if (parts > 1) {
    __syncwarp();
    cluster_sync();  // every part's accumulators lie in its shared memory
    if (epilogue) {
      // A warp finishes a row at a time, four channels per lane: 16-byte loads, all parts' in flight together.
      const int c4 = 4 * lane;
      const uint32_t mine = ptx::smem_u32(exchange) + 4u * static_cast<uint32_t>(c4);
      const int columns = n - (n0 + c4);  // channels of this lane that exist, if below four
      const float4 scales = *reinterpret_cast<const float4*>(ctl->channel_scale + c4);
      const float4 biases = *reinterpret_cast<const float4*>(ctl->channel_bias + c4);
      constexpr int kBatch = 2;  // rows of a warp whose loads are in flight together
      for (int first = warp - 2; first < own; first += 4 * kBatch) {
        int4 values[kBatch][kMaxParts];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int row = first + 4 * b;
#pragma unroll
          for (int c = 0; c < kMaxParts; ++c) {
            values[b][c] = make_int4(0, 0, 0, 0);
            if (c < parts && row < own) values[b][c] = load_cluster_int4(mine + static_cast<uint32_t>(own_first + row) * (kBlockM * 4), c);
          }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int row = first + 4 * b;
          if (row >= own || columns <= 0) continue;
          int4 sum = values[b][0];
#pragma unroll
          for (int c = 1; c < kMaxParts; ++c) {
            sum.x += values[b][c].x;
            sum.y += values[b][c].y;
            sum.z += values[b][c].z;
            sum.w += values[b][c].w;
          }
          float4 delta = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (extra > 0) delta = *reinterpret_cast<const float4*>(deltas + row * kBlockM + c4);
          const float row_scale = ctl->row_scale[own_first + row];
          const float out[4] = {finish(sum.x, row_scale, scales.x, biases.x, delta.x), finish(sum.y, row_scale, scales.y, biases.y, delta.y),
                                finish(sum.z, row_scale, scales.z, biases.z, delta.z), finish(sum.w, row_scale, scales.w, biases.w, delta.w)};
          const int64_t index = (row0 + own_first + row) * n + n0 + c4;
          if (args.vector_store && args.g.out_bf16) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(args.g.out) + index) = make_uint2(pack_bf16(out[0], out[1]), pack_bf16(out[2], out[3]));
          } else if (args.vector_store) {
            *reinterpret_cast<float4*>(static_cast<float*>(args.g.out) + index) = make_float4(out[0], out[1], out[2], out[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (j >= columns) break;
              store_value(args.g, index + j, out[j]);
            }
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no part leaves while another may still read its accumulators
  }

  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem_base, Cfg::kTmemColumns);
  }
}

// How many clusters of 1 .. kMaxParts CTAs can be resident at once with one CTA per SM (asked once per device).
struct Residency {
  int clusters[kMaxParts + 1] = {};
};

template <int kRowTile, bool kDeep, int kTerms>
cudaError_t configure() {
  auto kernel = lora_gemm_kernel<kRowTile, kDeep, kTerms>;
  const cudaError_t error =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(LoraConfig<kRowTile, kDeep, kTerms>::kSmemBytes));
  return error != cudaSuccess ? error : cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

template <int kRowTile, int kTerms>
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
  cudaError_t error = configure<kRowTile, true, kTerms>();
  if (error == cudaSuccess) error = configure<kRowTile, false, kTerms>();
  for (int parts = 1; parts <= kMaxParts && error == cudaSuccess; ++parts) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(parts));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = LoraConfig<kRowTile, true, kTerms>::kSmemBytes;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = static_cast<unsigned>(parts);
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    error = cudaOccupancyMaxActiveClusters(&out->clusters[parts], lora_gemm_kernel<kRowTile, true, kTerms>, &config);
  }
  if (error != cudaSuccess) return error;
  if (device >= 0 && device < kMaxDevices) known[device] = *out;
  configured.mark(device);
  return cudaSuccess;
}

template <int kRowTile, bool kDeep, int kTerms>
cudaError_t launch_kernel(const KernelArgs& args, int64_t blocks, const CUtensorMap* maps, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(blocks * args.parts));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = LoraConfig<kRowTile, kDeep, kTerms>::kSmemBytes;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = static_cast<unsigned>(args.parts);
  attributes[0].val.clusterDim.y = 1;
  attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, lora_gemm_kernel<kRowTile, kDeep, kTerms>, maps[0], maps[1], maps[2], args);
}

// How a call is cut: as many parts as leave all clusters resident at once, two CTAs per SM if need be, every part at least two K blocks (dense_gemm.cu).
struct Cut {
  int64_t blocks;
  int row_tiles, parts;
  bool deep;  // one CTA per SM
};

template <int kRowTile, int kTerms>
cudaError_t cut_rows(const KernelArgs& args, Cut* out) {
  Residency one_per_sm;
  const cudaError_t error = residency<kRowTile, kTerms>(&one_per_sm);
  if (error != cudaSuccess) return error;
  out->row_tiles = static_cast<int>((args.g.rows + kRowTile - 1) / kRowTile);
  out->blocks = static_cast<int64_t>((args.g.n + kBlockM - 1) / kBlockM) * out->row_tiles;
  if (out->blocks > (1ll << 27)) return cudaErrorInvalidValue;
  out->parts = 1;
  for (int parts = kMaxParts; parts > 1; --parts) {
    if (out->blocks <= 2 * one_per_sm.clusters[parts] && parts * kMinPartBlocks <= args.k_blocks) {
      out->parts = parts;
      break;
    }
  }
  out->deep = out->blocks <= one_per_sm.clusters[out->parts];
  return cudaSuccess;
}

template <int kRowTile, int kTerms>
cudaError_t launch_tile(KernelArgs args, const Cut& cut, cudaStream_t stream) {
  const LoraGemmArgs& g = args.g;
  const uint64_t k = static_cast<uint64_t>(g.k_padded);
  CUtensorMap maps[3];
  if (!make_sw128_map(&maps[0], g.weight, true, g.n, k, kBlockM) || !make_sw128_map(&maps[1], g.xq, true, g.rows, k, kRowTile) ||
      !make_adapter_map(&maps[2], g.adapters.b, g.adapters.rank, g.n, g.adapters.count, g.adapters.b_stride, args.block.ranks, kBlockM)) {
    return cudaErrorInvalidValue;
  }
  args.row_tiles = cut.row_tiles;
  args.parts = cut.parts;
  return cut.deep ? launch_kernel<kRowTile, true, kTerms>(args, cut.blocks, maps, stream) : launch_kernel<kRowTile, false, kTerms>(args, cut.blocks, maps, stream);
}

// Tiles of kRowTile rows, or of half as many where the chip has room for them: a CTA then has fewer adapters to go through.
template <int kRowTile, int kTerms>
cudaError_t launch_rows(const KernelArgs& args, const Cut& cut, cudaStream_t stream) {
  if constexpr (kRowTile > kLeastTile) {
    Cut half;
    const cudaError_t error = cut_rows<kRowTile / 2, kTerms>(args, &half);
    if (error != cudaSuccess) return error;
    if (half.deep && half.parts >= cut.parts) return launch_rows<kRowTile / 2, kTerms>(args, half, stream);
  }
  return launch_tile<kRowTile, kTerms>(args, cut, stream);
}

template <int kRowTile, int kTerms>
cudaError_t launch_up_to(const KernelArgs& args, cudaStream_t stream) {
  Cut cut;
  const cudaError_t error = cut_rows<kRowTile, kTerms>(args, &cut);
  return error != cudaSuccess ? error : launch_rows<kRowTile, kTerms>(args, cut, stream);
}

template <int kTerms>
cudaError_t launch_terms(const KernelArgs& args, cudaStream_t stream) {
  if (args.g.rows <= 16) return launch_up_to<16, kTerms>(args, stream);
  if (args.g.rows <= 32) return launch_up_to<32, kTerms>(args, stream);
  if (args.g.rows <= 64) return launch_up_to<64, kTerms>(args, stream);
  return launch_up_to<128, kTerms>(args, stream);
}

}  // namespace

cudaError_t launch_lora_gemm(const LoraGemmArgs& g, cudaStream_t stream) {
  KernelArgs args = {};
  args.g = g;
  args.k_blocks = (g.k_padded + kBlockKBytes - 1) / kBlockKBytes;
  args.rank_blocks = (g.adapters.rank + kLoraRankBlock - 1) / kLoraRankBlock;
  args.block = lora_block(g.adapters.rank);
  args.vector_store = dense_vector_store(g.out, g.n, g.out_bf16 != 0) ? 1 : 0;
  return g.planes > 1 ? launch_terms<kLoraPlanes>(args, stream) : launch_terms<1>(args, stream);
}

}  // namespace fmoe

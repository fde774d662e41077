// D = A * B on the 5th-generation tensor cores with the end of a fully connected layer in the same kernel: bias,
// activation, residual and a copy of the pre-activation on the way forward, the slope of the preceding activation on the
// way back.  A is M x K, B is N x K, either of them K-major (rows of K) or MN-major (rows of M or N), so that the layer, its
// input gradient and its weight gradient read the caller's tensors as they lie, slices of wider ones among them.
//
// pair_gemm_kernel: tiles of 256 x 256 (or 256 x 128) on clusters of two CTAs, persistent, for products that have a tile
// for most of the SM pairs.  solo_gemm_kernel: tiles of 128 x up to 128, whose steps a cluster of up to eight CTAs shares,
// for all others; a few rows of tokens become the columns of the tile, so that the weights fill its 128 rows.
//
// fp32: the tensor cores' fp32 accumulator drops the bits below its last place instead of rounding them, an error that
// grows with the number of additions and has one sign (k = 515 in three TF32 products a term: 3.9e-6 of the result, ten times
// that of fp32 multiply-adds).  So operands are cut into three bf16 parts (8 bits each, 24 in all; the three smallest of
// the nine products, below 2^-24, are left out), and a chain ends after every 64 terms: the epilogue warps add what
// the accumulator holds to sums of their own, rounded to nearest, while the other accumulator takes the next 64.
#include "fused_gemm.cuh"

#include "activation.cuh"
#include "tc_gemm.cuh"
#include "umma.cuh"

#include <algorithm>
#include <cstring>
#include <mutex>

namespace pdnn {
namespace {

using namespace umma;

// Reduction elements of a stage: a 128-byte row of 16-bit elements; of an fp32 operand's parts, three times as many bytes, half
// of that, for stages enough ahead (1024x1024x1024, 64 / 32 elements: 26.5 / 25.0 us; pairs are as fast either way, bound by their
// products, of which one of 256x128x16 is issued every 107 cycles).
constexpr int step_k(bool split) { return split ? 32 : 64; }
constexpr int kChainSteps = 2;     // fp32: stages whose products the accumulator takes before it is emptied
constexpr int kMostStages = 12;
constexpr int kSlotBytes = 4096;   // 32 rows of 128 bytes, swizzled as TMA does
constexpr int kSmemBudget = 232448;
// fp32 rows that go to fused_rows.cu, by the side on which the weights' rows lie
constexpr int few_rows(bool k_rows) { return k_rows ? 16 : 24; }
constexpr int kProducts = 6;       // products of parts that make an fp32 product

struct alignas(64) FusedArgs {
  CUtensorMap a_map, b_map, out_map, aux_map, pre_map;
  Finish f;
  unsigned* error_record;
  uint64_t wait_limit_ns;
  int tiles_m, tiles_n, group_m;     // tiles; rows of tiles that are walked together
  int kblocks, part_k;               // steps along K (of each product of parts); distance between two parts along K
  int a_mn, b_mn, stages;
  unsigned a_lbo, a_sbo, a_layout, a_kadv, b_lbo, b_sbo, b_layout, b_kadv, idesc;
  int out_tma, aux_tma, pre_tma;
  int beside;                        // the kernel needs nothing of the one ahead of it: it waits for that one at its end only
  // solo_gemm_kernel
  int bn, splits, blocks_per_split, swapped, tmem_cols;
  int out_vec, aux_vec, pre_vec, bias_vec;  // whole packets at a time
};

__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
               : "memory");
}
// (the barrier of the pair's first CTA counts the bytes)
__device__ __forceinline__ void load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar & kPeerBitMask), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1)
               : "memory");
}

// A wait of the whole warp: all lanes learn the same, so that none is left behind at a warp barrier when one gives up.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, const FusedArgs& a, unsigned where) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, a.error_record, a.wait_limit_ns, where));
}

__device__ __forceinline__ void wait_for_predecessor(const FusedArgs& a) {
  if (!a.beside) grid_dependency_wait();
}

// Which parts the i-th product of a step takes, the smallest products first (16-bit operands have one part and one product).
template <bool SPLIT>
__device__ __forceinline__ constexpr int part_of_a(int i) {
  return !SPLIT || i == 1 || i == 3 || i == 5 ? 0 : i == 0 ? 2 : 1;  // 2 0, 0 2, 1 1, 0 1, 1 0, 0 0
}
template <bool SPLIT>
__device__ __forceinline__ constexpr int part_of_b(int i) {
  return !SPLIT || i == 0 || i == 4 || i == 5 ? 0 : i == 1 ? 2 : 1;
}

// Where element byte `b` of row `r` of a slot is.
__device__ __forceinline__ uint32_t slot_at(int r, int b) { return (uint32_t)(r * 128 + ((((b >> 4) ^ (r & 7)) << 4) | (b & 15))); }

// A 16-byte chunk of a slot as floats, and back.
template <typename OutT>
__device__ __forceinline__ void unpack(uint4 q, float* v) {
  Vec16<OutT> p;
  p.raw = q;
#pragma unroll
  for (int i = 0; i < Vec16<OutT>::N; ++i) v[i] = to_f32(p.get(i));
}
template <typename OutT>
__device__ __forceinline__ uint4 pack(const float* v) {
  if constexpr (sizeof(OutT) == 4) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else if constexpr (std::is_same<OutT, __half>::value) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A slot's 32 rows from or to memory that TMA cannot reach (off a 16-byte boundary), neighbouring lanes on neighbouring
// elements.
template <typename OutT>
__device__ __forceinline__ void slot_from_memory(uint8_t* slot, const OutT* from, long long pitch, int rows, int cols, int lane) {
  constexpr int CB = 128 / (int)sizeof(OutT);
#pragma unroll 4
  for (int r = 0; r < 32; ++r)
#pragma unroll
    for (int c = lane; c < CB; c += 32)
      if (r < rows && c < cols) *reinterpret_cast<OutT*>(slot + slot_at(r, c * (int)sizeof(OutT))) = from[(long long)r * pitch + c];
}
template <typename OutT>
__device__ __forceinline__ void slot_to_memory(const uint8_t* slot, OutT* to, long long pitch, int rows, int cols, int lane) {
  constexpr int CB = 128 / (int)sizeof(OutT);
#pragma unroll 4
  for (int r = 0; r < 32; ++r)
#pragma unroll
    for (int c = lane; c < CB; c += 32)
      if (r < rows && c < cols) to[(long long)r * pitch + c] = *reinterpret_cast<const OutT*>(slot + slot_at(r, c * (int)sizeof(OutT)));
}

// ------------------------------------------------------------------------------------------------
// Clusters of two CTAs.  A tile is 256 rows x BN columns: each CTA loads its own 128 rows of A and half of the columns of B
// to a stage, rank 0 issues the MMAs of 256 x BN x 16 that read both shared memories, and each CTA finds its 128 rows of the
// accumulator in its own tensor memory, in one of two buffers, so that the end of a tile overlaps the MMAs of the
// next.  Warp 0 loads, warp 1 issues, warps 2 to 9 make the ends: 32 rows and half of the columns each, 128 bytes of a row at a time
// through a slot of shared memory that TMA fills (residual or slope argument) and empties.
// Bound by the tensor cores with shared memory close behind (64 bytes a cycle of operands and 64 of fills).
// ------------------------------------------------------------------------------------------------
constexpr int kPairThreads = 320, kEndWarps = 8;

template <typename OutT, int BN, bool SPLIT>
__global__ void __launch_bounds__(kPairThreads, 1) pair_gemm_kernel(const __grid_constant__ FusedArgs args) {
  extern __shared__ uint8_t smem_raw[];
  const FusedArgs& a = args;
  constexpr int kParts = SPLIT ? 3 : 1;  // of an operand in a stage
  constexpr int kStepK = step_k(SPLIT), kMmas = kStepK / 16;
  constexpr uint32_t kABytes = 128u * kStepK * 2u, kBBytes = (uint32_t)(BN / 2) * kStepK * 2u, kStage = kParts * (kABytes + kBBytes);
  constexpr uint32_t kBox = kStepK * 128u;  // 64 columns of an MN-major operand
  constexpr int CB = 128 / (int)sizeof(OutT), kCols = BN / 2, kBlocks = kCols / CB;  // columns of a block, of a warp; blocks of a warp
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = (int)(threadIdx.x & 31);
  const uint32_t rank = cluster_cta_rank();
  const bool leader = rank == 0;
  const int S = a.stages;
  const uint32_t slots_off = (uint32_t)S * kStage, bar_off = slots_off + 2u * kEndWarps * kSlotBytes;
  const uint32_t bars = base + bar_off;
  auto full_bar = [&](int s) { return bars + 8u * (uint32_t)s; };
  auto empty_bar = [&](int s) { return bars + 8u * (uint32_t)(kMostStages + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (uint32_t)(2 * kMostStages + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (uint32_t)(2 * kMostStages + 2 + b); };
  auto aux_bar = [&](int w, int b) { return bars + 8u * (uint32_t)(2 * kMostStages + 4 + 2 * w + b); };
  constexpr int kBars = 2 * kMostStages + 4 + 2 * kEndWarps;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + bar_off + 8 * kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + bar_off + 8 * kBars + 4);
  uint8_t* bias_strips = smem + bar_off + 8 * kBars + 16;  // 128 bytes a warp

  if ((int)threadIdx.x < kBars) {
    const int j = (int)threadIdx.x;
    mbar_init(bars + 8u * (uint32_t)j, j == 2 * kMostStages + 2 || j == 2 * kMostStages + 3 ? 2u * kEndWarps : 1u);
    if (j == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&a.a_map);
    prefetch_tensormap(&a.b_map);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 2u * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();  // the peer's barriers are initialised before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int total = a.tiles_m * a.tiles_n, first = (int)(blockIdx.x >> 1), step = (int)(gridDim.x >> 1);
  // a band of group_m rows of tiles is walked column by column, so that the tiles in flight share rows and columns
  auto tile_at = [&](int tile, int& m0, int& n0) {
    const int per = a.group_m * a.tiles_n, band = tile / per, rest = tile - band * per;
    const int high = min(a.group_m, a.tiles_m - band * a.group_m), nt = rest / high;
    m0 = (band * a.group_m + rest - nt * high) * 256 + (int)rank * 128;
    n0 = nt * BN;
  };

  if (warp == 0) {
    // ------------------------------- producer ------------------------------------------------
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    wait_for_predecessor(a);
#pragma unroll 1
    for (int tile = first; tile < total && ok; tile += step) {
      int m0, n0;
      tile_at(tile, m0, n0);
      n0 += (int)rank * (BN / 2);
#pragma unroll 1
      for (int kb = 0; kb < a.kblocks; ++kb) {
        if (!warp_wait(empty_bar(s), ph ^ 1u, abort_flag, a, 0x1100u + (unsigned)s)) {
          ok = false;
          break;
        }
        const uint32_t fb = full_bar(s);
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(fb, 2u * kStage);  // the bytes of both CTAs
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const uint32_t sa = base + (uint32_t)s * kStage + (uint32_t)part * kABytes;
            const uint32_t sb = base + (uint32_t)s * kStage + kParts * kABytes + (uint32_t)part * kBBytes;
            const int k = kb * kStepK + part * a.part_k;
            if (a.a_mn) {
              load_2d_pair(sa, &a.a_map, fb, m0, k);
              load_2d_pair(sa + kBox, &a.a_map, fb, m0 + 64, k);
            } else {
              load_2d_pair(sa, &a.a_map, fb, k, m0);
            }
            if (a.b_mn) {
              load_2d_pair(sb, &a.b_map, fb, n0, k);
              if (BN == 256) load_2d_pair(sb + kBox, &a.b_map, fb, n0 + 64, k);
            } else {
              load_2d_pair(sb, &a.b_map, fb, k, n0);
            }
          }
        }
        __syncwarp();
        if (++s == S) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer (rank 0) --------------------------------------
    wait_for_predecessor(a);
    grid_launch_dependents();  // the grid is a single wave, and its columns of tensor memory are taken
    if (leader) {
      const uint64_t a_desc0 = make_smem_desc(0, a.a_lbo, a.a_sbo, a.a_layout), b_desc0 = make_smem_desc(0, a.b_lbo, a.b_sbo, a.b_layout);
      const uint32_t a_kadv = a.a_kadv >> 4, b_kadv = a.b_kadv >> 4, idesc = a.idesc;
      const int chains = SPLIT ? (a.kblocks + kChainSteps - 1) / kChainSteps : 1;  // accumulator fills of a tile
      int s = 0;
      uint32_t ph = 0, buf = 0, aph = 0;
      bool ok = true;
#pragma unroll 1
      for (int tile = first; tile < total && ok; tile += step)
#pragma unroll 1
        for (int chain = 0; chain < chains && ok; ++chain) {
          if (!warp_wait(acc_empty_bar((int)buf), aph ^ 1u, abort_flag, a, 0x1200u + buf)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d = tmem_base + buf * (uint32_t)BN;
          const int steps = SPLIT ? min(kChainSteps, a.kblocks - chain * kChainSteps) : a.kblocks;
          uint32_t accumulate = 0u;
#pragma unroll 1
          for (int ks = 0; ks < steps; ++ks) {
            if (!warp_wait(full_bar(s), ph, abort_flag, a, 0x1300u + (unsigned)s)) {
              ok = false;
              break;
            }
            const uint32_t sa = (base + (uint32_t)s * kStage) & 0x3FFFFu;  // offset inside the CTA's shared memory
            const uint64_t da0 = a_desc0 + (uint64_t)(sa >> 4), db0 = b_desc0 + (uint64_t)((sa + kParts * kABytes) >> 4);
#pragma unroll
            for (int i = 0; i < (SPLIT ? kProducts : 1); ++i) {
              const uint64_t da = da0 + (uint64_t)(part_of_a<SPLIT>(i) * (kABytes >> 4)), db = db0 + (uint64_t)(part_of_b<SPLIT>(i) * (kBBytes >> 4));
#pragma unroll
              for (uint32_t k = 0; k < kMmas; ++k) {
                warp_mma_f16_pair(d, da + k * a_kadv, db + k * b_kadv, idesc, accumulate);
                accumulate = 1u;
              }
            }
            warp_commit_pair(empty_bar(s), cluster_map_shared(empty_bar(s), 1u));  // both CTAs may refill the stage
            if (++s == S) {
              s = 0;
              ph ^= 1u;
            }
          }
          if (!ok) break;
          warp_commit_pair(acc_full_bar((int)buf), cluster_map_shared(acc_full_bar((int)buf), 1u));
          if (++buf == 2u) {
            buf = 0;
            aph ^= 1u;
          }
        }
    }
  } else {
    // ------------------------------- ends (own 128 rows) --------------------------------------
    const int w = warp - 2, q = warp & 3, half = w >> 2;  // tensor memory lanes [32 q, 32 q + 32)
    uint8_t* slots = smem + slots_off + (size_t)w * 2 * kSlotBytes;
    const uint32_t slots_addr = base + slots_off + (uint32_t)w * 2u * kSlotBytes;
    OutT* strip = reinterpret_cast<OutT*>(bias_strips + w * 128);
    const Finish& f = a.f;
    const bool has_aux = f.aux != nullptr, has_pre = f.pre != nullptr;
    // Blocks take the two slots in turn; where the pre-activation is stored, too, it has the second one to itself.
    uint32_t blocks_done = 0, aux_phase = 0u, buf = 0, aph = 0;
    wait_for_predecessor(a);
    bool ok = true;
#pragma unroll 1
    for (int tile = first; tile < total && ok; tile += step) {
      int m0, n0;
      tile_at(tile, m0, n0);
      const int row0 = m0 + q * 32, col0 = n0 + half * kCols, rows_left = f.rows - row0;
      auto slot_of = [&](int block) { return has_pre ? 0 : (int)((blocks_done + (uint32_t)block) & 1u); };
      auto request_aux = [&](int block) {  // into its slot, whose last store has been read by now
        const int col = col0 + block * CB;
        if (!has_aux || col >= f.cols || rows_left <= 0) return;
        const int slot = slot_of(block);
        if (a.aux_tma) {
          if (lane == 0) {
            mbar_arrive_expect_tx(aux_bar(w, slot), kSlotBytes);
            load_2d(slots_addr + (uint32_t)slot * kSlotBytes, &a.aux_map, aux_bar(w, slot), col, row0);
          }
        } else {
          slot_from_memory<OutT>(slots + slot * kSlotBytes, static_cast<const OutT*>(f.aux) + (long long)row0 * f.aux_pitch + col,
                                 f.aux_pitch, rows_left, f.cols - col, lane);
        }
      };
      auto bias_at = [&](int block, float (&b)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = col0 + block * CB + lane + 32 * i;
          b[i] = f.bias != nullptr && 32 * i < CB && c < f.cols ? to_f32(static_cast<const OutT*>(f.bias)[c]) : 0.f;
        }
      };
      float bias[2];
      bias_at(0, bias);
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
      request_aux(0);
      float sums[SPLIT ? kCols : 1];
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) sums[i] = 0.f;
#pragma unroll 1
        for (int chain = 0; chain < a.kblocks; chain += kChainSteps) {
          if (!warp_wait(acc_full_bar((int)buf), aph, abort_flag, a, 0x1400u + buf)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t acc = tmem_base + ((uint32_t)(q * 32) << 16) + buf * (uint32_t)BN + (uint32_t)(half * kCols);
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t r[32];
            tmem_ld_32x32(acc + (uint32_t)c, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) sums[c + i] += __uint_as_float(r[i]);
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acc_empty_bar((int)buf) & kPeerBitMask);  // rank 0 collects both CTAs
          if (++buf == 2u) {
            buf = 0;
            aph ^= 1u;
          }
        }
        if (!ok) break;
      } else {
        if (!warp_wait(acc_full_bar((int)buf), aph, abort_flag, a, 0x1400u + buf)) break;
        tc_fence_after_sync();
      }
      const uint32_t acc = tmem_base + ((uint32_t)(q * 32) << 16) + buf * (uint32_t)BN + (uint32_t)(half * kCols);
#pragma unroll 1
      for (int block = 0; block < kBlocks; ++block) {
        const int col = col0 + block * CB, slot = slot_of(block);
        const bool inside = col < f.cols && rows_left > 0;
        if (f.bias != nullptr) {
          __syncwarp();
          strip[lane] = from_f32<OutT>(bias[0]);
          if (CB > 32) strip[lane + 32] = from_f32<OutT>(bias[1]);
          __syncwarp();
        }
        if (block + 1 < kBlocks) bias_at(block + 1, bias);
        uint8_t *my_row = slots + slot * kSlotBytes + lane * 128, *pre_row = slots + kSlotBytes + lane * 128;
        if (has_aux && inside) {
          if (a.aux_tma) {
            if (!warp_wait(aux_bar(w, slot), (aux_phase >> slot) & 1u, abort_flag, a, 0x1500u + (unsigned)slot)) {
              ok = false;
              break;
            }
            aux_phase ^= 1u << slot;
          } else {
            __syncwarp();
          }
        }
        // the slots of the next block: their stores have been read
        if (lane == 0 && !has_pre) bulk_wait_group_read<0>();
        __syncwarp();
        if (block + 1 < kBlocks && !has_pre) request_aux(block + 1);
        // Sixteen columns at a time, in a loop that is not unrolled: eight warps that are nowhere near one another in a long
        // stretch of code wait for instructions.  The next ones are on their way from tensor memory meanwhile.
        uint32_t next[SPLIT ? 1 : 16];
        if constexpr (!SPLIT) {
          tmem_ld_32x16(acc + (uint32_t)(block * CB), next);
          tmem_wait_ld();
        }
#pragma unroll 1
        for (int c = 0; c < CB; c += 16) {
          constexpr int N = Vec16<OutT>::N;
          float v[16];
          if constexpr (SPLIT) {
            const int from = (block * CB + c) / 16;
#pragma unroll
            for (int i = 0; i < 16; ++i) {  // (registers are not indexed at run time)
              v[i] = sums[i];
#pragma unroll
              for (int k = 1; k < kCols / 16; ++k) v[i] = from == k ? sums[k * 16 + i] : v[i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(next[i]);
            if (c + 16 < CB) {
              tmem_ld_32x16(acc + (uint32_t)(block * CB + c + 16), next);
            } else if (block + 1 == kBlocks) {  // the accumulator is free
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(acc_empty_bar((int)buf) & kPeerBitMask);
            }
          }
          if (f.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < 16; j += N) {
              float b[N];
              unpack<OutT>(*reinterpret_cast<const uint4*>(strip + c + j), b);
#pragma unroll
              for (int i = 0; i < N; ++i) v[j + i] += b[i];
            }
          }
          if (inside) {
            const int chunk = c / N;
            if (has_pre) {
#pragma unroll
              for (int j = 0; j < 16 / N; ++j)
                *reinterpret_cast<uint4*>(pre_row + (((chunk + j) ^ (lane & 7)) << 4)) = pack<OutT>(v + j * N);
            }
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
            if (has_aux) {
#pragma unroll
              for (int j = 0; j < 16 / N; ++j)
                unpack<OutT>(*reinterpret_cast<const uint4*>(my_row + (((chunk + j) ^ (lane & 7)) << 4)), x + j * N);
            }
            // (one body to a direction and activation, without branches inside: sixteen chains of latencies side by side)
            if (f.gradient) {
              with_activation(f.act, [&](auto act) {
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  const float2 s = slope_of<decltype(act)::value, OutT>(make_float2(x[i], x[i + 1]));
                  v[i] *= f.scale * s.x;
                  v[i + 1] *= f.scale * s.y;
                }
              });
            } else {
              with_activation(f.act, [&](auto act) {
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  const float2 o = value_of<decltype(act)::value, OutT>(make_float2(v[i], v[i + 1]));
                  v[i] = f.scale * o.x + x[i];
                  v[i + 1] = f.scale * o.y + x[i + 1];
                }
              });
            }
#pragma unroll
            for (int j = 0; j < 16 / N; ++j)
              *reinterpret_cast<uint4*>(my_row + (((chunk + j) ^ (lane & 7)) << 4)) = pack<OutT>(v + j * N);
          }
          if constexpr (!SPLIT) tmem_wait_ld();
        }
        if (inside) {
          fence_proxy_async_smem();
          __syncwarp();
          if (has_pre) {
            if (a.pre_tma) {
              if (lane == 0) store_2d(&a.pre_map, slots_addr + kSlotBytes, col, row0);
            } else {
              slot_to_memory<OutT>(slots + kSlotBytes, static_cast<OutT*>(f.pre) + (long long)row0 * f.pre_pitch + col, f.pre_pitch,
                                   rows_left, f.cols - col, lane);
            }
          }
          if (a.out_tma) {
            if (lane == 0) store_2d(&a.out_map, slots_addr + (uint32_t)slot * kSlotBytes, col, row0);
          } else {
            slot_to_memory<OutT>(slots + slot * kSlotBytes, static_cast<OutT*>(f.out) + (long long)row0 * f.out_pitch + col,
                                 f.out_pitch, rows_left, f.cols - col, lane);
          }
          if (lane == 0) bulk_commit_group();
          __syncwarp();
        }
        if (has_pre && block + 1 < kBlocks) {  // both slots are needed again
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          request_aux(block + 1);
        }
      }
      if (!ok) break;
      blocks_done += kBlocks;
      if constexpr (!SPLIT) {
        if (++buf == 2u) {
          buf = 0;
          aph ^= 1u;
        }
      }
    }
    if (lane == 0) bulk_wait_group_read<0>();
  }

  // ------------------------------- teardown ---------------------------------------------------
  if (a.beside) grid_dependency_wait();  // (who waits for this kernel has waited for both)
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {  // copies already issued may still be landing in shared memory
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
    __syncthreads();
  }
  cluster_sync_all();  // neither CTA leaves while the other may still use its shared and tensor memory
  if (warp == 1) tmem_dealloc_pair(tmem_base, 2u * BN);
}

// ------------------------------------------------------------------------------------------------
// One tile of 128 x bn to a cluster of `splits` CTAs, each of which takes a share of the steps along K.  Partial tiles go to
// shared memory, where each CTA of the cluster adds up its share of the tile's rows in the order of the ranks and finishes
// them, a packet to a thread.  swapped: the tile's rows are the columns of the result.  Two CTAs fit
// an SM, so that the end of one overlaps the loads of another.
// ------------------------------------------------------------------------------------------------
constexpr int kSoloThreads = 192, kSoloSmem = 110 * 1024, kSoloHead = 2048, kSplitCols = 64;

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// A packet of a row, `left` elements of which are inside it.
template <typename OutT>
__device__ __forceinline__ void load_packet(const OutT* p, bool vec, int left, float (&v)[Vec16<OutT>::N]) {
  constexpr int N = Vec16<OutT>::N;
  if (vec && left >= N) {
    unpack<OutT>(*reinterpret_cast<const uint4*>(p), v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? to_f32(p[i]) : 0.f;
  }
}
template <typename OutT>
__device__ __forceinline__ void store_packet(OutT* p, bool vec, int left, const float (&v)[Vec16<OutT>::N]) {
  constexpr int N = Vec16<OutT>::N;
  if (vec && left >= N) {
    *reinterpret_cast<uint4*>(p) = pack<OutT>(v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = from_f32<OutT>(v[i]);
  }
}

// The packets of a CTA's share of the result: item i is a packet of line i >> shift.
struct Share {
  int rows, rank, m0, n0, swapped, shift, items, cols;
  __device__ __forceinline__ Share(const FusedArgs& a, int splits, int rank_, int m0_, int n0_, int bn, int packet)
      : rows(128 / splits), rank(rank_), m0(m0_), n0(n0_), swapped(a.swapped), cols(a.f.cols) {
    shift = __ffs((swapped ? rows : bn) / packet) - 1;  // (a power of two)
    items = (swapped ? min(bn, a.f.rows - n0) : min(rows, a.f.rows - m0 - rank * rows)) << shift;
  }
  // Row and first column of the result, how many of its columns are inside, and the line and column of the partial tile.
  __device__ __forceinline__ void place(int i, int packet, long long& r, int& col, int& left, int& line, int& at) const {
    const int l = i >> shift, c = (i - (l << shift)) * packet;
    r = swapped ? n0 + l : m0 + rank * rows + l;
    col = swapped ? m0 + rank * rows + c : n0 + c;
    left = i < items ? cols - col : 0;
    line = swapped ? l : rank * rows + l;
    at = swapped ? rank * rows + c : c;
  }
};
// What is added to a thread's first packet, or its slope taken of, asked for before the ranks meet (whole packets only).
struct Extras {
  uint4 bias, aux;
  bool has_bias, has_aux;
};
template <typename OutT>
__device__ __forceinline__ Extras ask_for_extras(const FusedArgs& a, const Share& share) {
  constexpr int N = Vec16<OutT>::N;
  Extras e;
  e.bias = e.aux = make_uint4(0u, 0u, 0u, 0u);
  long long r;
  int col, left, l, c;
  share.place((int)threadIdx.x, N, r, col, left, l, c);
  e.has_bias = a.f.bias != nullptr && a.bias_vec && left >= N;
  e.has_aux = a.f.aux != nullptr && a.aux_vec && left >= N;
  if (e.has_bias) e.bias = *reinterpret_cast<const uint4*>(static_cast<const OutT*>(a.f.bias) + col);
  if (e.has_aux) e.aux = *reinterpret_cast<const uint4*>(static_cast<const OutT*>(a.f.aux) + r * a.f.aux_pitch + col);
  return e;
}

// Adds up the ranks' partial tiles in their order and finishes what comes of it, a packet to a thread, two packets at a
// time where few ranks leave registers for it.
template <typename OutT, int SPLITS>
__device__ __forceinline__ void finish_share(const FusedArgs& a, const Share& share, uint32_t partial, uint32_t line, const Extras& extras) {
  constexpr int N = Vec16<OutT>::N, U = SPLITS >= 4 ? 1 : 2;
  const Finish& f = a.f;
  for (int i0 = (int)threadIdx.x; i0 < share.items; i0 += U * kSoloThreads) {
    float z[U][N];
    float4 got[U][SPLITS][N / 4];
    long long r[U];
    int col[U], left[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int l, c;
      share.place(i0 + u * kSoloThreads, N, r[u], col[u], left[u], l, c);
      if (left[u] <= 0) continue;
      const uint32_t at = partial + (uint32_t)l * line + (uint32_t)c * 4u;
#pragma unroll
      for (int k = 0; k < SPLITS; ++k) {
        const uint32_t from = SPLITS == 1 ? at : cluster_map_shared(at, (uint32_t)k);
#pragma unroll
        for (int j = 0; j < N / 4; ++j) got[u][k][j] = SPLITS == 1 ? ld_shared_v4(from + 16u * j) : ld_cluster_v4(from + 16u * j);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (left[u] <= 0) continue;
      const bool first = u == 0 && i0 == (int)threadIdx.x;
      float x[N], b[N];
      if (first && extras.has_bias)
        unpack<OutT>(extras.bias, b);
      else if (f.bias != nullptr)
        load_packet<OutT>(static_cast<const OutT*>(f.bias) + col[u], a.bias_vec, left[u], b);
      if (first && extras.has_aux) {
        unpack<OutT>(extras.aux, x);
      } else if (f.aux != nullptr) {
        load_packet<OutT>(static_cast<const OutT*>(f.aux) + r[u] * f.aux_pitch + col[u], a.aux_vec, left[u], x);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < N / 4; ++j) {
        float4 s = got[u][0][j];
#pragma unroll
        for (int k = 1; k < SPLITS; ++k) {
          const float4 p = got[u][k][j];
          s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
        }
        z[u][4 * j] = s.x, z[u][4 * j + 1] = s.y, z[u][4 * j + 2] = s.z, z[u][4 * j + 3] = s.w;
      }
      if (f.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[u][j] += b[j];
      }
      if (f.pre != nullptr) store_packet<OutT>(static_cast<OutT*>(f.pre) + r[u] * f.pre_pitch + col[u], a.pre_vec, left[u], z[u]);
      if (f.gradient) {
        with_activation(f.act, [&](auto act) {
#pragma unroll
          for (int j = 0; j < N; j += 2) {
            const float2 s = slope_of<decltype(act)::value, OutT>(make_float2(x[j], x[j + 1]));
            z[u][j] *= f.scale * s.x;
            z[u][j + 1] *= f.scale * s.y;
          }
        });
      } else {
        with_activation(f.act, [&](auto act) {
#pragma unroll
          for (int j = 0; j < N; j += 2) {
            const float2 o = value_of<decltype(act)::value, OutT>(make_float2(z[u][j], z[u][j + 1]));
            z[u][j] = f.scale * o.x + x[j];
            z[u][j + 1] = f.scale * o.y + x[j + 1];
          }
        });
      }
      store_packet<OutT>(static_cast<OutT*>(f.out) + r[u] * f.out_pitch + col[u], a.out_vec, left[u], z[u]);
    }
  }
}

template <typename OutT, bool SPLIT>
__global__ void __launch_bounds__(kSoloThreads, 2) solo_gemm_kernel(const __grid_constant__ FusedArgs args) {
  extern __shared__ uint8_t smem_raw[];
  const FusedArgs& a = args;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = (int)(threadIdx.x & 31);
  const int splits = a.splits, rank = (int)blockIdx.x % splits, tile = (int)blockIdx.x / splits;
  const int S = a.stages, bn = SPLIT ? kSplitCols : a.bn;
  constexpr int kParts = SPLIT ? 3 : 1;  // of an operand in a stage
  constexpr int kStepK = step_k(SPLIT), kMmas = kStepK / 16;
  constexpr uint32_t kABytes = 128u * kStepK * 2u, kBox = kStepK * 128u;
  const uint32_t b_bytes = (uint32_t)(bn * kStepK) * 2u, stage_bytes = kParts * (kABytes + b_bytes), ring = base + 1024u;  // (the partial tile takes the ring's place)
  auto full_bar = [&](int s) { return base + 8u * (uint32_t)s; };
  auto empty_bar = [&](int s) { return base + 8u * (uint32_t)(kMostStages + s); };
  auto acc_full_bar = [&](int b) { return base + 8u * (uint32_t)(2 * kMostStages + b); };
  auto acc_empty_bar = [&](int b) { return base + 8u * (uint32_t)(2 * kMostStages + 2 + b); };
  constexpr int kBars = 2 * kMostStages + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 8 * kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 8 * kBars + 4);
  if ((int)threadIdx.x < kBars) {
    mbar_init(base + 8u * threadIdx.x, (int)threadIdx.x >= 2 * kMostStages + 2 ? 4u : 1u);
    if (threadIdx.x == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), (uint32_t)a.tmem_cols);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&a.a_map);
    prefetch_tensormap(&a.b_map);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int per = a.group_m * a.tiles_n, band = tile / per, rest = tile - band * per;
  const int high = min(a.group_m, a.tiles_m - band * a.group_m), nt = rest / high;
  const int m0 = (band * a.group_m + rest - nt * high) * 128, n0 = nt * bn;
  const int k0 = rank * a.blocks_per_split, k1 = min(k0 + a.blocks_per_split, a.kblocks);

  if (warp == 0) {
    // ------------------------------- producer ------------------------------------------------
    wait_for_predecessor(a);
    grid_launch_dependents();  // (the columns of tensor memory are taken)
    int s = 0;
    uint32_t ph = 0;
#pragma unroll 1
    for (int kb = k0; kb < k1; ++kb) {
      if (!warp_wait(empty_bar(s), ph ^ 1u, abort_flag, a, 0x2100u + (unsigned)s)) break;
      const uint32_t fb = full_bar(s);
      if (elect_one()) {
        mbar_arrive_expect_tx(fb, stage_bytes);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const uint32_t sa = ring + (uint32_t)s * stage_bytes + (uint32_t)part * kABytes;
          const uint32_t sb = ring + (uint32_t)s * stage_bytes + kParts * kABytes + (uint32_t)part * b_bytes;
          const int k = kb * kStepK + part * a.part_k;
          if (a.a_mn) {
            load_2d(sa, &a.a_map, fb, m0, k);
            load_2d(sa + kBox, &a.a_map, fb, m0 + 64, k);
          } else {
            load_2d(sa, &a.a_map, fb, k, m0);
          }
          if (a.b_mn) {
            load_2d(sb, &a.b_map, fb, n0, k);
            if (bn > 64) load_2d(sb + kBox, &a.b_map, fb, n0 + 64, k);
          } else {
            load_2d(sb, &a.b_map, fb, k, n0);
          }
        }
      }
      __syncwarp();
      if (++s == S) {
        s = 0;
        ph ^= 1u;
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer -----------------------------------------------
    const uint64_t a_desc0 = make_smem_desc(0, a.a_lbo, a.a_sbo, a.a_layout), b_desc0 = make_smem_desc(0, a.b_lbo, a.b_sbo, a.b_layout);
    const uint32_t a_kadv = a.a_kadv >> 4, b_kadv = a.b_kadv >> 4, idesc = a.idesc;
    int s = 0;
    uint32_t ph = 0, buf = 0, aph = 0, accumulate = 0u;
    wait_for_predecessor(a);
#pragma unroll 1
    for (int kb = k0; kb < k1; ++kb) {
      const int in_chain = (kb - k0) % kChainSteps;
      if (SPLIT && in_chain == 0) {
        if (!warp_wait(acc_empty_bar((int)buf), aph ^ 1u, abort_flag, a, 0x2200u + buf)) break;
        tc_fence_after_sync();
        accumulate = 0u;
      }
      const uint32_t d = tmem_base + (SPLIT ? buf * (uint32_t)kSplitCols : 0u);
      if (!warp_wait(full_bar(s), ph, abort_flag, a, 0x2300u + (unsigned)s)) break;
      const uint32_t sa = (ring + (uint32_t)s * stage_bytes) & 0x3FFFFu;
      const uint64_t da0 = a_desc0 + (uint64_t)(sa >> 4), db0 = b_desc0 + (uint64_t)((sa + kParts * kABytes) >> 4);
#pragma unroll
      for (int i = 0; i < (SPLIT ? kProducts : 1); ++i) {
        const uint64_t da = da0 + (uint64_t)(part_of_a<SPLIT>(i) * (kABytes >> 4)), db = db0 + (uint64_t)((uint32_t)part_of_b<SPLIT>(i) * (b_bytes >> 4));
#pragma unroll
        for (uint32_t k = 0; k < kMmas; ++k) {
          warp_mma_f16(d, da + k * a_kadv, db + k * b_kadv, idesc, accumulate);
          accumulate = 1u;
        }
      }
      warp_commit(empty_bar(s));
      if (++s == S) {
        s = 0;
        ph ^= 1u;
      }
      if (SPLIT && (in_chain == kChainSteps - 1 || kb + 1 == k1)) {
        warp_commit(acc_full_bar((int)buf));
        if (++buf == 2u) {
          buf = 0;
          aph ^= 1u;
        }
      }
    }
    if (!SPLIT) warp_commit(acc_full_bar(0));
  }
  // ------------------------------- partial tile -> shared memory ------------------------------
  // A line of 16 bytes more than it holds: [row][column], or [column][row] where rows are the result's columns.
  const uint32_t line = (uint32_t)(a.swapped ? 128 : bn) * 4u + 16u;
  wait_for_predecessor(a);
  const Share share(a, splits, rank, m0, n0, bn, Vec16<OutT>::N);
  const Extras extras = ask_for_extras<OutT>(a, share);
  if (warp >= 2) {
    const int q = warp & 3, row = q * 32 + lane;
    const uint32_t lanes = tmem_base + ((uint32_t)(q * 32) << 16);
    auto put = [&](int c0, const float* v) {  // 16 columns
      if (a.swapped) {
#pragma unroll
        for (int i = 0; i < 16; ++i) *reinterpret_cast<float*>(smem + 1024 + (size_t)(c0 + i) * line + row * 4) = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(smem + 1024 + (size_t)row * line + (c0 + i) * 4) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    };
    if constexpr (SPLIT) {
      float sums[kSplitCols];
#pragma unroll
      for (int i = 0; i < kSplitCols; ++i) sums[i] = 0.f;
      uint32_t buf = 0, aph = 0;
      bool ok = true;
#pragma unroll 1
      for (int kb = k0; kb < k1; kb += kChainSteps) {
        if (!warp_wait(acc_full_bar((int)buf), aph, abort_flag, a, 0x2400u + buf)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < kSplitCols; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32(lanes + buf * (uint32_t)kSplitCols + (uint32_t)c, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) sums[c + i] += __uint_as_float(r[i]);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty_bar((int)buf));
        if (++buf == 2u) {
          buf = 0;
          aph ^= 1u;
        }
      }
      // (the last accumulator is full: every copy into the ring has landed and every MMA has read it; so for all four warps)
      if (ok) {
#pragma unroll
        for (int c = 0; c < kSplitCols; c += 16) put(c, sums + c);
      }
    } else {
      if (warp_wait(acc_full_bar(0), 0u, abort_flag, a, 0x2400u)) {
        tc_fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < bn; c += 16) {
          uint32_t r[16];
          tmem_ld_32x16(lanes + (uint32_t)c, r);
          tmem_wait_ld();
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
          put(c, v);
        }
      }
    }
    tc_fence_before_sync();
  }
  __syncwarp();
  cluster_sync_all();
  // ------------------------------- the CTA's share of the result ------------------------------
  if (!*abort_flag) {
    switch (splits) {
      case 8: finish_share<OutT, 8>(a, share, base + 1024u, line, extras); break;
      case 4: finish_share<OutT, 4>(a, share, base + 1024u, line, extras); break;
      case 2: finish_share<OutT, 2>(a, share, base + 1024u, line, extras); break;
      default: finish_share<OutT, 1>(a, share, base + 1024u, line, extras);
    }
  } else {
    const uint64_t t0 = global_timer_ns();  // copies already issued may still be landing in shared memory
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  if (a.beside) grid_dependency_wait();
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while another may still read its partial tile
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, (uint32_t)a.tmem_cols);
  }
}

// ---- fp32 operands in three parts ---------------------------------------------------------------------
// x = p0 + p1 + p2 + (at most 2^-25 of x): each part the rest rounded to bf16, the rests themselves exact.  Both operands in one
// launch, eight elements of a row of the result to a thread: rows x cols of the source, zeros up to to_rows x to_cols.
struct SplitSide {
  const float* from;
  __nv_bfloat16* to;
  long long pitch, to_pitch, part_stride;
  int rows, cols, to_cols, packets;  // packets: the source is read 16 bytes at a time
  unsigned items, blocks;
};
struct SplitArgs {
  SplitSide side[2];
};
__global__ void __launch_bounds__(256) split_parts_kernel(const SplitArgs a) {
  overlap_wait();
  const bool second = blockIdx.x >= a.side[0].blocks;
  const SplitSide& s = a.side[second ? 1 : 0];
  const unsigned step = s.blocks * 256u, pieces = (unsigned)s.to_cols / 8u;
  for (unsigned i = (blockIdx.x - (second ? a.side[0].blocks : 0u)) * 256u + threadIdx.x; i < s.items; i += step) {
    const unsigned r = i / pieces;
    const int c = (int)(i - r * pieces) * 8;
    float v[8];
    const float* from = s.from + (long long)r * s.pitch + c;
    if (s.packets && (int)r < s.rows && c + 8 <= s.cols) {
      const float4 lo = *reinterpret_cast<const float4*>(from), hi = *reinterpret_cast<const float4*>(from + 4);
      v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (int)r < s.rows && c + j < s.cols ? from[j] : 0.f;
    }
    __nv_bfloat16* to = s.to + (long long)r * s.to_pitch + c;
#pragma unroll
    for (int part = 0; part < 3; ++part) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        if (part == 0) {  // (finite values beyond bf16's largest)
          if (__hisinf(p.x)) p.x = __float2bfloat16_rz(v[2 * j]);
          if (__hisinf(p.y)) p.y = __float2bfloat16_rz(v[2 * j + 1]);
        }
        v[2 * j] -= __low2float(p);
        v[2 * j + 1] -= __high2float(p);
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
      }
      *reinterpret_cast<uint4*>(to + part * s.part_stride) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
    else
      cudaGetLastError();
  });
  return fn;
}

// Boxes of row_bytes (128 or 64) x box_rows of a matrix of rows x cols elements, zeros outside it, swizzled.
bool matrix_map(CUtensorMap* map, int dtype, const void* p, long long pitch, long long rows, long long cols, int box_rows,
                int row_bytes = 128) {
  const EncodeFn fn = encoder();
  if (fn == nullptr) {
    fail(PDNN_ALLOCATION_PROBLEM, "cuTensorMapEncodeTiled is unavailable");
    return false;
  }
  const cuuint64_t es = dtype_size(dtype);
  if (rows == 1) pitch = (long long)((cols * es + 15) / 16 * 16 / es);  // (no row follows)
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * es};
  const cuuint32_t box[2] = {(cuuint32_t)(row_bytes / es), (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUtensorMapDataType dt = dtype == PDNN_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                               : dtype == PDNN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = fn(map, dt, 2, const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    fail(PDNN_INVALID_PARAMETER, "cuTensorMapEncodeTiled failed (%d): %lld x %lld, pitch %lld", (int)r, rows, cols, pitch);
  return r == CUDA_SUCCESS;
}

bool tma_ok(int dtype, const void* p, long long pitch, int rows) {
  const long long bytes = pitch * (long long)dtype_size(dtype);
  return aligned16(p) && (rows == 1 || (bytes % 16 == 0 && bytes < (1ll << 40)));
}
bool packets_ok(int dtype, const void* p, long long pitch) {
  return aligned16(p) && pitch * (long long)dtype_size(dtype) % 16 == 0;
}

// An operand as the kernels see it: `mn` rows or columns of the tile's side, MN-major or K-major.
struct Side {
  const void* p;
  long long pitch;
  int mn, mn_major;
};

struct Plan {
  bool pair;
  int bn, splits;
  bool swapped;
};

// Estimated times of the plans in us, their constants fitted to all plans' times of 128 products of 1 to 8192 rows (a step is 64 elements
// of K): over these the plan picked takes 1 % more than the best one (a fit to 24 products took 5 % more).
// A pair's step takes 0.39 us at 256 columns and 0.29 at 128 (an SM pulls its operands through L2 no faster), three quarters of that with
// few clusters in flight (but for fp32, whose products bound it: 2000x777x300 28.7 us, single CTAs 23.1), a tile no less than its end, 2.3
// and 2.2 us, all behind 8.3 and 5 us of launch, ramp and the last end.  A CTA alone takes 0.21 to 0.31 us a step by its columns, two
// thirds more where two share an SM (clusters of four and eight do before there is a CTA to every SM), behind 3.8 us, 0.022 a column for its
// end, 0.26 for each partial tile that it adds (0.75 where it ends on its own), and 0.0018 for every CTA's reads beside it.
Plan choose_plan(bool split, long long m, long long n, bool m_major, bool n_major, int kblocks, int sms) {
  const double products = split ? kProducts : 1;
  auto tiles = [](long long x, int t) { return (x + t - 1) / t; };
  Plan best{true, 128, 1, false};
  double least = 1e30;
  for (int bn : {256, 128}) {
    if (split && bn == 256) continue;
    const long long all = tiles(m, 256) * tiles(n, bn);
    const double waves = (double)tiles(all, sms / 2), busy = std::min(1.0, (double)all / (sms / 2));
    const double step = split ? 0.23 * products : (bn == 256 ? 0.39 : 0.29) * (0.77 + 0.23 * busy);
    const double t = waves * std::max(kblocks * step, bn == 256 ? 2.28 : 2.17) + (split ? 6.7 : bn == 256 ? 8.25 : 4.98);
    if (t < least) least = t, best = Plan{true, bn, 1, false};
  }
  for (int swapped = 0; swapped < 2; ++swapped)
    for (int bn : {16, 32, 64, 128}) {
      if (split && bn != kSplitCols) continue;
      if (bn < 64 && (swapped ? m_major : n_major)) continue;  // (an MN-major tile is whole boxes of 64 columns)
      const long long rows = swapped ? n : m, cols = swapped ? m : n;
      const long long all = tiles(rows, 128) * tiles(cols, bn);
      if (all > 8ll * sms) continue;
      for (int splits : {1, 2, 4, 8}) {
        const int steps = (kblocks + splits - 1) / splits;
        if (splits > 1 && steps * (splits - 1) >= kblocks) continue;  // a CTA without steps
        const long long ctas = all * splits;
        const double waves = (double)tiles(ctas, 2ll * sms), shared = ctas > sms - (splits == 8 ? 28 : splits == 4 ? 4 : 0) ? 1.65 : 1.0;
        const double step = (bn == 128 ? 0.31 : bn == 64 ? 0.21 : 0.24) * shared;
        const double t = 2.28 + 0.0018 * ctas + waves * (steps * step * products + 1.51 + 0.022 * bn * shared + (splits > 1 ? 0.26 * splits : 0.75));
        if (t < least) least = t, best = Plan{false, bn, splits, swapped != 0};
      }
    }
  return best;
}

int opt_in(const void* kernel, int bytes) {
  // once per kernel and device
  static std::mutex mu;
  struct Entry {
    const void* kernel;
    int dev;
  };
  static Entry known[256];
  static int count = 0;
  const int dev = current_device();
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < count; ++i)
    if (known[i].kernel == kernel && known[i].dev == dev) return PDNN_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused: cannot opt in to %d bytes of shared memory", bytes);
  }
  if (count < 256) known[count++] = Entry{kernel, dev};
  return PDNN_OK;
}

int launch_cluster(void (*kernel)(FusedArgs), const FusedArgs& args, unsigned grid, unsigned threads, size_t smem, unsigned cluster,
                   cudaStream_t s) {
  const int st = opt_in(reinterpret_cast<const void*>(kernel), kSmemBudget);
  if (st != PDNN_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused: launch failed: %s", cudaGetErrorString(e));
  }
  return check_launch("matmul_fused");
}

// dtype: of the operands (f16 or bf16); out_dtype: of the finish's tensors.
template <typename OutT, bool SPLIT>
int run_plan(const Plan& plan, int dtype, int out_dtype, Side x, Side y, int k, int part_k, const Finish& f, bool beside, cudaStream_t s) {
  const int sms = device_sm_count();
  FusedArgs a;
  std::memset(&a, 0, sizeof(a));
  if (plan.swapped) std::swap(x, y);
  const int bm = plan.pair ? 256 : 128;
  a.f = f;
  if (f.gradient && f.aux == nullptr) {  // the product alone
    a.f.gradient = 0;
    a.f.act = PDNN_ACT_NONE;
  }
  a.error_record = tc_error_record_address();
  if (a.error_record == nullptr) return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused: no error record");
  a.wait_limit_ns = kWaitLimitNs;
  a.beside = beside;
  a.tiles_m = (x.mn + bm - 1) / bm;
  a.tiles_n = (y.mn + plan.bn - 1) / plan.bn;
  a.group_m = std::min(a.tiles_m, 8);
  constexpr int kStepK = step_k(SPLIT);
  a.kblocks = (k + kStepK - 1) / kStepK;
  a.part_k = part_k;
  a.a_mn = x.mn_major;
  a.b_mn = y.mn_major;
  // MN-major: k-rows of 128 bytes, 64 columns after 64 columns; K-major: rows of one step, 128 bytes or 64, swizzled accordingly
  const unsigned row = kStepK * 2u;
  a.a_lbo = x.mn_major ? kStepK * 128u : 16u;
  a.b_lbo = y.mn_major ? kStepK * 128u : 16u;
  a.a_sbo = x.mn_major ? 1024u : 8u * row;
  a.b_sbo = y.mn_major ? 1024u : 8u * row;
  a.a_layout = x.mn_major || row == 128u ? 2u : 4u;
  a.b_layout = y.mn_major || row == 128u ? 2u : 4u;
  a.a_kadv = x.mn_major ? 2048u : 32u;
  a.b_kadv = y.mn_major ? 2048u : 32u;
  a.idesc = make_idesc(dtype == PDNN_BF16 ? 1 : 0, x.mn_major, y.mn_major, plan.bn, plan.pair ? 256 : 128);
  const long long depth = SPLIT ? 3ll * part_k : k;  // elements along K in memory
  const int b_cols = plan.pair ? plan.bn / 2 : plan.bn;
  auto operand_map = [&](CUtensorMap* map, const Side& side, int cols) {
    return side.mn_major ? matrix_map(map, dtype, side.p, side.pitch, depth, side.mn, kStepK)
                         : matrix_map(map, dtype, side.p, side.pitch, side.mn, depth, cols, (int)row);
  };
  if (!operand_map(&a.a_map, x, 128) || !operand_map(&a.b_map, y, b_cols)) return PDNN_INVALID_PARAMETER;
  if (plan.pair) {
    a.out_tma = tma_ok(out_dtype, f.out, f.out_pitch, f.rows);
    a.aux_tma = f.aux != nullptr && tma_ok(out_dtype, f.aux, f.aux_pitch, f.rows);
    a.pre_tma = f.pre != nullptr && tma_ok(out_dtype, f.pre, f.pre_pitch, f.rows);
    if ((a.out_tma && !matrix_map(&a.out_map, out_dtype, f.out, f.out_pitch, f.rows, f.cols, 32)) ||
        (a.aux_tma && !matrix_map(&a.aux_map, out_dtype, f.aux, f.aux_pitch, f.rows, f.cols, 32)) ||
        (a.pre_tma && !matrix_map(&a.pre_map, out_dtype, f.pre, f.pre_pitch, f.rows, f.cols, 32)))
      return PDNN_INVALID_PARAMETER;
    const int stage = (SPLIT ? 3 : 1) * (128 + plan.bn / 2) * kStepK * 2;
    const int fixed = 1024 + 2 * kEndWarps * kSlotBytes + 8 * (2 * kMostStages + 4 + 2 * kEndWarps) + 16 + kEndWarps * 128;
    a.stages = std::min(kMostStages, (kSmemBudget - fixed) / stage);
    const unsigned grid = (unsigned)std::min<long long>(2ll * a.tiles_m * a.tiles_n, sms / 2 * 2);
    void (*kernel)(FusedArgs) = nullptr;
    if constexpr (SPLIT)
      kernel = pair_gemm_kernel<OutT, 128, true>;
    else
      kernel = plan.bn == 256 ? pair_gemm_kernel<OutT, 256, false> : pair_gemm_kernel<OutT, 128, false>;
    tc_set_last_kernel("pair_gemm_kernel");
    return launch_cluster(kernel, a, grid, kPairThreads, (size_t)fixed + (size_t)a.stages * stage, 2, s);
  }
  a.bn = plan.bn;
  a.splits = plan.splits;
  a.blocks_per_split = ((k + 63) / 64 + plan.splits - 1) / plan.splits * (64 / kStepK);
  a.swapped = plan.swapped;
  const int columns = SPLIT ? 2 * kSplitCols : plan.bn;
  a.tmem_cols = std::max(32, columns);
  a.out_vec = packets_ok(out_dtype, f.out, f.out_pitch);
  a.aux_vec = packets_ok(out_dtype, f.aux, f.aux_pitch);
  a.pre_vec = packets_ok(out_dtype, f.pre, f.pre_pitch);
  a.bias_vec = packets_ok(out_dtype, f.bias, 0);
  const int stage = (SPLIT ? 3 : 1) * (128 + plan.bn) * kStepK * 2;
  // All of an SM's shared memory for stages where there is one CTA to an SM, with steps enough to use them (fewer where half of it holds
  // three stages alone), and clusters small enough to be placed all the same (us, half / all: 128x4096x4096 bf16, 64 columns, 32 steps, 13.9 /
  // 11.8; 256x2048x1000 f32 24.9 / 22.0; too few steps, 1024x1024x1024 bf16 7.7 / 8.3; clusters of eight, 130x8192x200 7.6 / 12.9).
  const long long ctas = (long long)a.tiles_m * a.tiles_n * plan.splits;
  const int half = (kSoloSmem - kSoloHead) / stage;
  const bool deep = a.blocks_per_split >= (half < 4 ? 16 : 24) && ctas <= (plan.splits <= 2 ? sms : plan.splits == 4 ? 128 : 0);
  a.stages = std::min(kMostStages, deep ? (kSmemBudget - kSoloHead) / stage : half);
  const size_t partial = plan.swapped ? (size_t)plan.bn * (128 * 4 + 16) : (size_t)128 * (plan.bn * 4 + 16);
  const size_t smem = kSoloHead + std::max((size_t)a.stages * stage, partial);
  tc_set_last_kernel("solo_gemm_kernel");
  void (*kernel)(FusedArgs) = solo_gemm_kernel<OutT, SPLIT>;
  return launch_cluster(kernel, a, (unsigned)(a.tiles_m * a.tiles_n * plan.splits), kSoloThreads, smem, (unsigned)plan.splits, s);
}

}  // namespace

bool fused_gemm_operand_ok(int dtype, const Matrix& m) { return dtype == PDNN_F32 || tma_ok(dtype, m.p, m.pitch, m.rows); }

int fused_gemm(int dtype, int ta, int tb, const Matrix& a, const Matrix& b, int k, const Finish& f, bool beside, cudaStream_t s) {
  const int sms = device_sm_count();
  Side x{a.p, a.pitch, f.rows, ta}, y{b.p, b.pitch, f.cols, !tb};
  const int kblocks = (k + 63) / 64;
  Plan plan = choose_plan(dtype == PDNN_F32, f.rows, f.cols, x.mn_major != 0, y.mn_major != 0, kblocks, sms);
  if (dtype == PDNN_F16) return run_plan<__half, false>(plan, dtype, dtype, x, y, k, 0, f, beside, s);
  if (dtype == PDNN_BF16) return run_plan<__nv_bfloat16, false>(plan, dtype, dtype, x, y, k, 0, f, beside, s);
  // fp32.  Few rows: cutting the weights into parts costs more than multiplying them (us, parts / rows, weights [n][k]: 4096x4096, 1 row 59 /
  // 15, 16 rows 60 / 48, 24 rows 61 / 85; 256x7296, 16 rows 13.8 / 13.4; [k][n]: 4096x4096, 24 rows 60 / 43, 32 rows 60 / 77).
  if (!ta && f.rows <= few_rows(tb != 0)) return fused_rows(tb != 0, a, b, k, f, s);
  // parts behind one another along K
  const int part_k = kblocks * 64;
  if (3ll * part_k > 0x7FFF0000ll) return fail(PDNN_INDEX_EXCEEDED, "matmul_fused: an fp32 sum of %d products is too long", k);  // (TMA counts in 32 bits)
  const Matrix* from[2] = {&a, &b};
  Side* side[2] = {&x, &y};
  size_t bytes[2], cols[2];
  for (int i = 0; i < 2; ++i) {
    cols[i] = side[i]->mn_major ? ((size_t)side[i]->mn + 7) / 8 * 8 : (size_t)part_k;
    bytes[i] = (side[i]->mn_major ? (size_t)part_k : (size_t)side[i]->mn) * cols[i] * 3 * 2;
    bytes[i] = (bytes[i] + 255) / 256 * 256;
  }
  char* scratch = nullptr;
  if (cudaMallocAsync(reinterpret_cast<void**>(&scratch), bytes[0] + bytes[1], s) != cudaSuccess) {
    cudaGetLastError();
    return fail(PDNN_ALLOCATION_PROBLEM, "matmul_fused: cannot allocate %zu bytes of scratch", bytes[0] + bytes[1]);
  }
  SplitArgs split;
  for (int i = 0; i < 2; ++i) {
    SplitSide& q = split.side[i];
    const size_t rows = side[i]->mn_major ? (size_t)part_k : (size_t)side[i]->mn, items = rows * (cols[i] / 8);
    if (items > 0x80000000u) {
      cudaFreeAsync(scratch, s);
      return fail(PDNN_INDEX_EXCEEDED, "matmul_fused: an fp32 operand of more than 2^34 elements");
    }
    q.from = static_cast<const float*>(from[i]->p);
    q.to = reinterpret_cast<__nv_bfloat16*>(scratch + (i == 0 ? 0 : bytes[0]));
    q.pitch = from[i]->pitch;
    q.to_pitch = side[i]->mn_major ? (long long)cols[i] : 3ll * part_k;
    q.part_stride = side[i]->mn_major ? (long long)part_k * (long long)cols[i] : part_k;
    q.rows = from[i]->rows;
    q.cols = from[i]->cols;
    q.to_cols = (int)cols[i];
    q.packets = packets_ok(PDNN_F32, from[i]->p, from[i]->pitch);
    q.items = (unsigned)items;
    q.blocks = grid_for(items, 256, sms);
    side[i]->p = q.to;
    side[i]->pitch = q.to_pitch;
  }
  launch_overlapped(split_parts_kernel, split.side[0].blocks + split.side[1].blocks, 256, s, split);
  int st = check_launch("matmul_fused: parts");
  if (st == PDNN_OK) st = run_plan<float, true>(plan, PDNN_BF16, PDNN_F32, x, y, k, part_k, f, false, s);
  cudaFreeAsync(scratch, s);
  return st;
}

}  // namespace pdnn

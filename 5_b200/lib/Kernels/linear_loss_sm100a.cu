// Softmax cross entropy of a linear layer over a vocabulary, without the matrix of its logits.
//
//   l = H W^T            (H: rows x width, W: vocab x width, float32 accumulation)
//   lse_r = log sum_v exp(l[r, v]),   loss_r = lse_r - l[r, target_r]
//   g[r, v] = dloss_r (exp(l[r, v] - lse_r) - [v == target_r]),   dH = g W,   dW = g^T H
//
// Forward: the product's tiles never leave the SM. A pair of CTAs computes a 256 x 256 tile of l as the
// dense kernel does (TMA ring, tcgen05.mma.cta_group::2, two accumulators in tensor memory); its epilogue,
// in which a lane holds a row, keeps the running maximum and the sum of exponentials of the row over the
// columns of the tile, and writes those two numbers per row and half tile instead of 256 logits. The tile
// that holds a row's target also writes that logit. A second kernel joins the partial pairs of each row.
//
// Gradient: the logits are computed again with the same kernel, whose epilogue now turns them into g,
// rounded to the operands' type, for one piece of the vocabulary at a time -- stored both as it stands and
// transposed, so that both products with it, dH += g W_piece and dW_piece = g^T H, read it along their
// inner dimension. Those products are the dense kernels' (lib/CAPI/Cuda.cpp enqueues them).
//
// Accuracy: the tensor cores cut what they add to a float32 accumulator instead of rounding it, so that its error grows
// with the number of additions. An accumulator therefore takes a run of 1024 of the width (64 additions), and the
// epilogue adds the runs in registers, with rounding. lse is off by 1.7e-7 of its size whatever the width, by 2.9e-6
// where all products have one sign; with one accumulator 6.4e-7 and 1.7e-5 at a width of 4096, 4.9e-6 and 1.6e-4 at
// 32768. (4096 x 32768 x 4096: 690 us, with one accumulator 680; runs of 512: 714 us, 1.0e-7 and 1.0e-6.) Both passes
// add alike, so that the gradient's logits are those of lse. A width of one run keeps to one accumulator and, in the
// epilogue, two alternating sets of 32 registers.
//
// g's stores: a lane holds a row, so lanes exchange words first, and what a warp writes at once covers whole
// sectors of both forms (1031 x 16411 x 1001: 49.5 us, when every lane stored its own values 57 us).
//
// Bound: the tensor pipe, 2 rows vocab width operations forward and 8 for forward and gradient (6 if the
// logits were kept). The exponentials, one per logit, run in the epilogue warps under the next tile's
// products: 65536 of them per tile and pair take 2048 cycles of the two SMs' special function units
// against 8 width cycles of products.
//
// Rounding g: dloss is often the same for all rows (one over their number), and rounding (p - 1) dloss would
// then be off by the same fraction in every row, which the sums over rows do not average out. The kernel
// therefore finds the largest |dloss| of the rows that count, uses dloss as a fraction of it, so that g is
// (p - 1) or p to the type's precision, and the products take the factor back in float32 before they are
// rounded. float16 also multiplies g by 2^14, because p may lie below the type's normal range.
// For dw, a sum over rows, one factor for all rows is right: next to the largest a row of a small dloss is small. A row
// of dh is that row's alone, and 2^-25 of the largest dloss may be more than all of it, in float16. Where dh goes
// through float32 sums, which it always does in float16, its g is therefore formed without dloss, and each row of the
// sums is multiplied by its own. (bfloat16 has float32's exponents.)
#include "gemm_epilogue.cuh"
#include "device_checks.cuh"
#include "gemm_launch.h"
#include "sm100_ptx.cuh"

#include <cfloat>

namespace hc {
namespace sm100 {

namespace loss {

constexpr int kTileM = 256;  // rows of H per pair, 128 per CTA
constexpr int kTileN = 256;  // rows of W per pair, 128 loaded by each CTA
constexpr int kCtaRows = 128;
constexpr int kBlockK = 128;  // of the width per ring stage: two 64-wide boxes per operand
constexpr int kUmmaK = 16;
constexpr int kStages = 3;
constexpr int kEpilogueWarps = 8;  // two per quarter of the tensor-memory lanes, half of the columns each
constexpr int kThreads = 64 + 32 * kEpilogueWarps;
constexpr int kTmemColumns = 512;  // two accumulators
constexpr int kColumnsPerWarp = kTileN / 2;
constexpr int kChunks = kColumnsPerWarp / 32;
// k blocks whose products are summed in an accumulator before the epilogue adds them to the logits ("a run").
constexpr int kRunBlocks = 8;
constexpr uint32_t kBoxBytes = kCtaRows * 64 * 2;
constexpr uint32_t kOperandBytes = 2 * kBoxBytes;
constexpr uint32_t kStageBytes = 2 * kOperandBytes;  // per CTA
constexpr uint32_t kBarrierBytes = 256;
constexpr uint32_t kSmemBytes = kStages * kStageBytes + kBarrierBytes + 1024;
static_assert(kSmemBytes <= 227 * 1024, "dynamic shared memory of one CTA");

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ long long target_of(const LinearLoss &p, long long row) {
  return p.targets_64 ? static_cast<const long long *>(p.targets)[row] : static_cast<const int *>(p.targets)[row];
}

// The power of two that g is multiplied by.
__device__ __forceinline__ float g_scale(int c_dtype) { return c_dtype == kCTypeF16 ? 16384.0f : 1.0f; }

__device__ __forceinline__ bool counts_row(const LinearLoss &p, long long target) {
  return target != p.ignore_index && target >= 0 && target < p.vocab_total;
}

// Walks the tiles down the rows of H within groups of `group_n` tile columns (see gemm_dense_pair_kernel).
__device__ __forceinline__ int2 tile_of(int tile, int tiles_m, int tiles_n, int group_n) {
  const int per_group = group_n * tiles_m;
  const int group = tile / per_group, first_n = group * group_n;
  const int width = min(group_n, tiles_n - first_n), inside = tile - group * per_group;
  return make_int2(inside / width, first_n + inside % width);
}

// ---------------------------------------------------------------- epilogues ---------

// Running maximum (times log2 e) and sum of exponentials of one row.
struct Running {
  float top;  // max l * log2(e), -inf before the first finite value
  float sum;  // sum exp2(l * log2(e) - top)
};

// 32 logits of this lane's row.
__device__ __forceinline__ void take_chunk(const uint32_t (&r)[32], Running &run) {
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < 32; ++j)
    top = fmaxf(top, __uint_as_float(r[j]));
  top = fmaxf(run.top, top * kLog2e);
  const float base = top == -INFINITY ? 0.0f : top;  // nothing finite yet: exp2(-inf - 0) = 0
  float sum = run.sum * exp2_fast(run.top - base);
  float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 32; ++j)
    part[j & 3] += exp2_fast(fmaf(__uint_as_float(r[j]), kLog2e, -base));
  run.top = top;
  run.sum = sum + ((part[0] + part[1]) + (part[2] + part[3]));
}

// The logit of a row's target, if it is among these 32.
__device__ __forceinline__ void take_target(const uint32_t (&r)[32], int offset, float *out) {
  if (static_cast<unsigned>(offset) < 32u) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      v = j == offset ? __uint_as_float(r[j]) : v;
    *out = v;
  }
}

// Between lanes that differ in `bit`: the lower one's b for the upper one's a.
__device__ __forceinline__ void swap_pieces(uint4 &a, uint4 &b, int lane, int bit) {
  const bool upper = (lane & bit) != 0;
  const uint4 give = upper ? a : b;
  const uint4 got = make_uint4(__shfl_xor_sync(0xffffffffu, give.x, bit), __shfl_xor_sync(0xffffffffu, give.y, bit),
                               __shfl_xor_sync(0xffffffffu, give.z, bit), __shfl_xor_sync(0xffffffffu, give.w, bit));
  if (upper)
    a = got;
  else
    b = got;
}

// kRuns: the width is more than one run.
template <bool kGrad, bool kRuns>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
linear_loss_kernel(const __grid_constant__ CUtensorMap tmap_h, const __grid_constant__ CUtensorMap tmap_w,
                   const LinearLoss p, uint32_t idesc, int tiles_m, int tiles_n, int group_n, int *status) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t bar_base = smem_base + kStages * kStageBytes;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (kStages + s); };
  auto tmem_full_bar = [&](uint32_t a) { return bar_base + 8u * (2 * kStages + a); };
  auto tmem_empty_bar = [&](uint32_t a) { return bar_base + 8u * (2 * kStages + 2 + a); };
  const uint32_t misc_off = (bar_base - smem_base) + 8u * (2 * kStages + 4);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_gen + misc_off);
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem_gen + misc_off + 4);

  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  const uint32_t cta_rank = cluster_cta_rank();  // 0: issues the MMAs, 1: partner

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (uint32_t a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar(a), 1);
      mbar_init(tmem_empty_bar(a), 2 * kEpilogueWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_descriptor(&tmap_h);
    tma_prefetch_descriptor(&tmap_w);
  }
  cluster_sync_all();  // both CTAs' barriers exist before either signals across the pair
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemColumns);
    tmem_relinquish_alloc_permit_pair();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  const int num_tiles = tiles_m * tiles_n;
  const int num_kb = (p.width + kBlockK - 1) / kBlockK;
  const int first_tile = static_cast<int>(blockIdx.x >> 1), tile_step = static_cast<int>(gridDim.x >> 1);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer ------
    if (lane == 0) {
      // The tile columns of a group are read again by every tile row: keep W, let H pass (as measured
      // for the dense kernel).
      const uint64_t pol_h = l2_policy_evict_normal(), pol_w = l2_policy_evict_last();
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
        const int2 at = tile_of(tile, tiles_m, tiles_n, group_n);
        const int m0 = at.x * kTileM + static_cast<int>(cta_rank) * kCtaRows;
        const int n0 = at.y * kTileN + static_cast<int>(cta_rank) * kCtaRows;
        // Rows past the end of H are not asked for where that can be helped: every SM's request for one goes to the
        // same place of the L2 (53 x 44544 x 768: 28.6 us, with boxes of 128 rows for both CTAs 70 us; 1 x 131072 x
        // 4096: 207 us and 1007 us). What is left in shared memory instead only reaches rows of l that nobody reads.
        const uint32_t h_bytes = 2u * static_cast<uint32_t>(p.h_box) * 128u;
        const uint32_t bytes = 2 * kOperandBytes + h_bytes + (at.x * kTileM + kCtaRows < p.rows ? h_bytes : 0u);
        if (!HC_CHECK(status, abort_flag, HC_CHECK_TILE_COORDINATES,
                      at.x >= 0 && at.x < tiles_m && at.y >= 0 && at.y < tiles_n))
          break;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag) ||
              !HC_CHECK(status, abort_flag, HC_CHECK_RING_STAGE, stage < static_cast<uint32_t>(kStages))) {
            ok = false;
            break;
          }
          const uint32_t h_dst = smem_base + stage * kStageBytes, w_dst = h_dst + kOperandBytes;
          const uint32_t leader_full = map_to_cta(full_bar(stage), 0);
          if (cta_rank == 0)
            mbar_arrive_expect_tx(full_bar(stage), bytes);
#pragma unroll
          for (int sub = 0; sub < kBlockK / 64; ++sub) {
            const int k0 = kb * kBlockK + sub * 64;  // (past the width: zeros)
            if (m0 < p.rows)
              tma_load_2d_pair_hint(h_dst + sub * kBoxBytes, &tmap_h, leader_full, k0, m0, pol_h);
            tma_load_2d_pair_hint(w_dst + sub * kBoxBytes, &tmap_w, leader_full, k0, n0, pol_w);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (CTA 0) -
    if (lane == 0 && cta_rank == 0) {
      uint32_t stage = 0, phase = 0, iter = 0;  // iter: accumulators filled
      bool ok = true;
      for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
        for (int kb = 0; ok && kb < num_kb; ++iter) {
          const uint32_t acc = iter & 1u;
          if (!mbar_wait(tmem_empty_bar(acc), ((iter >> 1) & 1u) ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          tcgen05_fence_after_sync();
          const int run_begin = kb, run_end = kRuns ? min(kb + kRunBlocks, num_kb) : num_kb;
          for (; kb < run_end; ++kb) {
            if (!mbar_wait(full_bar(stage), phase, abort_flag)) {
              ok = false;
              break;
            }
            tcgen05_fence_after_sync();
            const uint32_t h_addr = smem_base + stage * kStageBytes, w_addr = h_addr + kOperandBytes;
#pragma unroll
            for (int kk = 0; kk < kBlockK / kUmmaK; ++kk) {
              const uint64_t advance = static_cast<uint64_t>((kk % 4) * 2);  // 32 bytes inside the swizzle row
              umma_ss_pair<false>(tmem_base + acc * kTileN,
                                  make_smem_desc_sw128(h_addr + (kk / 4) * kBoxBytes, 16, 1024) + advance,
                                  make_smem_desc_sw128(w_addr + (kk / 4) * kBoxBytes, 16, 1024) + advance, idesc,
                                  (kb != run_begin || kk != 0) ? 1u : 0u);
            }
            umma_commit_pair(map_to_cta(empty_bar(stage), 0));
            umma_commit_pair(map_to_cta(empty_bar(stage), 1));
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) {
            umma_commit_pair(map_to_cta(tmem_full_bar(acc), 0));
            umma_commit_pair(map_to_cta(tmem_full_bar(acc), 1));
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue ----------
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    uint32_t iter = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
      const int2 at = tile_of(tile, tiles_m, tiles_n, group_n);
      const int row = at.x * kTileM + static_cast<int>(cta_rank) * kCtaRows + quarter * 32 + lane;
      const int col_base = at.y * kTileN + part * kColumnsPerWarp;
      const bool live = row < p.rows;
      if (!HC_CHECK(status, abort_flag, HC_CHECK_OUTPUT_RANGE,
                    row >= lane && row - lane < tiles_m * kTileM && col_base >= 0 && col_base < tiles_n * kTileN))  // (per warp)
        break;
      // What the row needs is fetched while its products are still running.
      long long target = -1;
      float scale = 0.0f, lse2 = 0.0f;
      bool nothing = true;  // of this row is in the gradient
      if (live) {
        target = target_of(p, row);
        if (kGrad) {
          // A row that does not count has no gradient, whatever its dloss and lse hold.
          const bool counts = counts_row(p, target);
          const float dloss = counts ? p.dloss[row] : 0.0f;
          nothing = dloss == 0.0f;
          scale = dloss / p.scales[0] * g_scale(p.c_dtype);
          lse2 = counts ? p.lse[row] * kLog2e : INFINITY;
        }
        target = target == p.ignore_index ? -1 : target - p.first_column;
      }
      // Whether g differs from what its transpose holds: not where dloss is the largest one, in all rows mostly.
      const bool plain = kGrad && p.g_plain != 0 && __any_sync(0xffffffffu, !nothing && scale != g_scale(p.c_dtype));
      const int target_col =
          target >= 0 && target < p.vocab ? static_cast<int>(target) - col_base : -1;  // within this warp's columns
      const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + part * kColumnsPerWarp;
      auto wait_for_sums = [&](uint32_t acc) {
        const bool ready = mbar_wait(tmem_full_bar(acc), (iter >> 1) & 1u, abort_flag);
        if (!__all_sync(0xffffffffu, ready))
          return false;
        tcgen05_fence_after_sync();
        return true;
      };
      auto release = [&](uint32_t acc) {  // the accumulator has been read: back to the MMA issuer
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0)
          mbar_arrive_cluster(map_to_cta(tmem_empty_bar(acc), 0));
      };
      Running run{-INFINITY, 0.0f};

      auto finish = [&](uint32_t (&r)[32], int chunk) {
        const int col0 = col_base + chunk * 32;
        if (col0 >= p.vocab)
          return;  // the same for the whole warp
        if constexpr (!kGrad) {
          take_target(r, live ? target_col - chunk * 32 : -1, p.target_logit + row);
          if (col0 + 32 > p.vocab) {  // columns past the vocabulary add nothing
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col0 + j >= p.vocab)
                r[j] = __float_as_uint(-INFINITY);
          }
          take_chunk(r, run);
        } else {
          // p - [v == target], then g, rounded to the operands' type; two neighbouring columns per word.
          uint32_t w[16];
          const int hit = target_col - chunk * 32;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float a = exp2_fast(fmaf(__uint_as_float(r[j]), kLog2e, -lse2));
            r[j] = __float_as_uint(j == hit ? a - 1.0f : a);
          }
          auto scaled_by = [&](float by) {
#pragma unroll
            for (int j = 0; j < 32; j += 2)
              w[j / 2] = pack_pair(__uint_as_float(r[j]) * by, __uint_as_float(r[j + 1]) * by, p.c_dtype);
            if (nothing) {  // exactly, also where the logits are not finite
#pragma unroll
              for (int j = 0; j < 16; ++j)
                w[j] = 0u;
            }
          };
          scaled_by(scale);
          // Transposed: two neighbouring lanes share their words, so that each writes two neighbouring rows of every
          // other column. (The pitch holds whole groups of 32 rows; what rows past the end get is not read.)
          const int row0 = row - lane;
          if (p.gt != nullptr && row0 < p.rows) {
            const int odd = lane & 1;
            uint16_t *gt = static_cast<uint16_t *>(p.gt) + static_cast<long long>(col0 + odd) * p.ldgt + (row - odd);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, w[j], 1);
              const uint32_t both = odd ? __byte_perm(other, w[j], 0x7632) : __byte_perm(w[j], other, 0x5410);
              if (col0 + 2 * j + odd < p.vocab)
                *reinterpret_cast<uint32_t *>(gt) = both;
              gt += 2 * p.ldgt;
            }
          }
          // As it stands: four lanes exchange their 16-byte pieces, so that together they write the 64 bytes of one row
          // after another (the pitch holds whole chunks of 32 columns).
          if (p.g != nullptr && row0 < p.rows) {
            if (plain)
              scaled_by(g_scale(p.c_dtype));
            uint4 piece[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              piece[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            swap_pieces(piece[0], piece[1], lane, 1);
            swap_pieces(piece[2], piece[3], lane, 1);
            swap_pieces(piece[0], piece[2], lane, 2);
            swap_pieces(piece[1], piece[3], lane, 2);
            const int quad = row - (lane & 3);
            uint16_t *g = static_cast<uint16_t *>(p.g) + static_cast<long long>(quad) * p.ldg + col0 + 8 * (lane & 3);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (quad + j < p.rows)
                *reinterpret_cast<uint4 *>(g + j * p.ldg) = piece[j];
          }
        }
      };

      if constexpr (!kRuns) {
        const uint32_t acc = iter & 1u;
        if (!wait_for_sums(acc))
          break;
        const uint32_t taddr = lanes + acc * kTileN;
        uint32_t ra[32], rb[32];
        tmem_load_32x32b_x32(taddr, ra);
#pragma unroll 1
        for (int chunk = 0; chunk < kChunks; chunk += 2) {
          tmem_load_wait_for(ra);
          tmem_load_32x32b_x32(taddr + (chunk + 1) * 32, rb);
          finish(ra, chunk);
          tmem_load_wait_for(rb);
          if (chunk + 2 < kChunks)
            tmem_load_32x32b_x32(taddr + (chunk + 2) * 32, ra);
          else
            release(acc);
          finish(rb, chunk + 1);
        }
        ++iter;
      } else {
        uint32_t l[kChunks][32];  // the runs' sums, added in their order
        for (int kb = 0; kb < num_kb; kb += kRunBlocks, ++iter) {
          const uint32_t acc = iter & 1u;
          ok = wait_for_sums(acc);
          if (!ok)
            break;
          const uint32_t taddr = lanes + acc * kTileN;
          if (kb == 0) {
#pragma unroll
            for (int chunk = 0; chunk < kChunks; ++chunk)
              tmem_load_32x32b_x32(taddr + chunk * 32, l[chunk]);
#pragma unroll
            for (int chunk = 0; chunk < kChunks; ++chunk)
              tmem_load_wait_for(l[chunk]);
          } else {
#pragma unroll
            for (int half = 0; half < 2 * kChunks; ++half) {
              uint32_t r[16];
              tmem_load_32x32b_x16(taddr + half * 16, r);
              tmem_load_wait_for(r);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                uint32_t &to = l[half / 2][half % 2 * 16 + j];
                to = __float_as_uint(__uint_as_float(to) + __uint_as_float(r[j]));
              }
            }
          }
          release(acc);
        }
        if (!ok)
          break;
#pragma unroll
        for (int chunk = 0; chunk < kChunks; ++chunk)
          finish(l[chunk], chunk);
      }
      if (!kGrad && live)
        p.partials[static_cast<long long>(at.y * 2 + part) * p.rows + row] = make_float2(run.top, run.sum);
    }
  }

  // Neither CTA leaves (or frees tensor memory) while its partner can still use it.
  tcgen05_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0) {
    if (threadIdx.x == 0)
      atomicCAS(status, 0, kStatusDeviceWaitTimeout);
    const long long start = clock64();
    while (clock64() - start < 2000000LL) {
    }
  }
  cluster_sync_all();
  tcgen05_fence_after_sync();
  if (warp == 1)
    tmem_dealloc_pair(tmem_base, kTmemColumns);
}

// Joins the partial pairs of each row: 32 rows per CTA, whose warps first share the parts (a lane each row), then
// the rows (a lane each warp's share). 4096 rows of 256 parts: 5 us.
constexpr int kJoinWarps = 32;

// A part's sum brought to the scale of `top`; a part without a value above -inf adds nothing.
__device__ __forceinline__ float joined(float2 v, float top) { return v.y == 0.0f ? 0.0f : v.y * exp2_fast(v.x - top); }

__global__ void __launch_bounds__(32 * kJoinWarps)
join_kernel(const LinearLoss p, int parts) {
  __shared__ float2 shared[kJoinWarps][33];
  constexpr int kAtOnce = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int row = static_cast<int>(blockIdx.x) * 32 + lane;
  float2 run = make_float2(-INFINITY, 0.0f);
  for (int k0 = warp; k0 < parts; k0 += kAtOnce * kJoinWarps) {
    float2 v[kAtOnce];
    float top = run.x;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int k = k0 + i * kJoinWarps;
      v[i] = make_float2(-INFINITY, 0.0f);
      if (k < parts && row < p.rows)
        v[i] = p.partials[static_cast<long long>(k) * p.rows + row];
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      top = fmaxf(top, v[i].x);
    float sum = joined(run, top);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      sum += joined(v[i], top);
    run = make_float2(top, sum);
  }
  shared[warp][lane] = run;
  __syncthreads();
  run = shared[lane][warp];
  row = static_cast<int>(blockIdx.x) * 32 + warp;
  float top = run.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = joined(run, top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane != 0 || row >= p.rows)
    return;
  const float lse = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);  // (a NaN stays one)
  const long long target = target_of(p, row);
  p.lse_out[row] = lse;
  p.loss_out[row] = target == p.ignore_index                   ? 0.0f
                    : (target < 0 || target >= p.vocab_total) ? NAN
                                                              : lse - p.target_logit[row];
}

// Before the gradient: the scales, by the grid's first CTA, and the rows of H with zeros in place of those that
// do not count, by the others. (Their g is zero, but the product g^T H would still make a NaN of a zero times
// an infinity or a NaN that such a row, padding say, may hold.)
template <typename Word>
__global__ void __launch_bounds__(256)
prepare_kernel(const LinearLoss p, float *scales, const uint16_t *src, long long lds, uint16_t *dst, long long ldd) {
  if (blockIdx.y == 0) {
    __shared__ float shared[8];
    if (blockIdx.x != 0)
      return;
    float top = 0.0f;
#pragma unroll 8
    for (int row = threadIdx.x; row < p.rows; row += 256) {
      const float d = fabsf(p.dloss[row]);
      if (d < INFINITY && counts_row(p, target_of(p, row)))
        top = fmaxf(top, d);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0)
      shared[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < 8; ++k)
        top = fmaxf(top, shared[k]);
      scales[0] = top > 0.0f ? top : 1.0f;
      scales[1] = scales[0] / g_scale(p.c_dtype);
    }
    return;
  }
  constexpr int kPer = sizeof(Word) / 2;
  const int words = (p.width + kPer - 1) / kPer;
  for (int row = blockIdx.y - 1; row < p.rows; row += gridDim.y - 1) {
    const bool counts = counts_row(p, target_of(p, row));
    for (int i = blockIdx.x * 256 + threadIdx.x; i < words; i += gridDim.x * 256) {
      const uint16_t *s = src + static_cast<long long>(row) * lds + i * kPer;
      uint16_t *d = dst + static_cast<long long>(row) * ldd + i * kPer;
      if (i * kPer + kPer <= p.width) {
        *reinterpret_cast<Word *>(d) = counts ? *reinterpret_cast<const Word *>(s) : Word{};
      } else {
        for (int e = 0; e < p.width - i * kPer; ++e)
          d[e] = counts ? s[e] : uint16_t{0};
      }
    }
  }
}

// A 16-bit matrix with aligned rows to one whose rows start anywhere: a thread writes eight elements from a 16-byte
// boundary of dst, which begin at any even byte of src, or what there is of them at the ends of a row.
__global__ void __launch_bounds__(256)
spread_kernel(const uint16_t *src, long long lds, uint16_t *dst, long long ldd, int rows, int cols) {
  const int pieces = (cols + 14) / 8;  // that can touch a row
  const long long total = static_cast<long long>(rows) * pieces;
  for (long long idx = blockIdx.x * 256LL + threadIdx.x; idx < total; idx += gridDim.x * 256LL) {
    const int row = total <= 0x7fffffffLL ? static_cast<int>(static_cast<unsigned>(idx) / static_cast<unsigned>(pieces))
                                          : static_cast<int>(idx / pieces);
    uint16_t *const d = dst + row * ldd;
    const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(d) & 15) / 2;  // elements before the row's first boundary
    const int col = static_cast<int>(idx - static_cast<long long>(row) * pieces) * 8 - lead;
    const uint16_t *const s = src + row * lds + col;
    if (col >= 0 && col + 8 <= cols) {
      uint4 v;
      if ((col & 1) == 0) {  // src's rows start on 16-byte boundaries
        const uint32_t *w = reinterpret_cast<const uint32_t *>(s);
        v = make_uint4(__ldg(w), __ldg(w + 1), __ldg(w + 2), __ldg(w + 3));
      } else {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(s + 1);
        const uint32_t first = __ldg(s), w0 = __ldg(w), w1 = __ldg(w + 1), w2 = __ldg(w + 2), last = __ldg(s + 7);
        v = make_uint4(first | (w0 << 16), (w0 >> 16) | (w1 << 16), (w1 >> 16) | (w2 << 16), (w2 >> 16) | (last << 16));
      }
      *reinterpret_cast<uint4 *>(d + col) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i >= 0 && col + i < cols)
          d[col + i] = s[i];
    }
  }
}

// dh = (float32 sums of g W) * dloss / g_scale, rounded to 16 bits, for a g formed without dloss.
template <typename Pair>
__global__ void __launch_bounds__(256)
narrow_kernel(const LinearLoss p, const float *src, long long lds, void *dst, long long ldd, int cols) {
  const float back = 1.0f / g_scale(p.c_dtype);  // (a power of two)
  for (int row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float *s = src + static_cast<long long>(row) * lds;
    uint16_t *d = static_cast<uint16_t *>(dst) + static_cast<long long>(row) * ldd;
    const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= cols)
      continue;
    const bool counts = counts_row(p, target_of(p, row));
    const float f = counts ? p.dloss[row] : 0.0f;
    const float4 v = *reinterpret_cast<const float4 *>(s + c);  // (lds is a multiple of 4)
    auto of = [&](float x) { return f == 0.0f ? 0.0f : x * back * f; };
    if (sizeof(Pair) == 8 && c + 4 <= cols) {
      *reinterpret_cast<uint2 *>(d + c) = make_uint2(pack_pair(of(v.x), of(v.y), p.c_dtype), pack_pair(of(v.z), of(v.w), p.c_dtype));
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < cols)
          d[c + i] = round_to_16(of(e[i]), p.c_dtype);
    }
  }
}

}  // namespace loss

int linear_loss_parts(int vocab) { return 2 * ((vocab + loss::kTileN - 1) / loss::kTileN); }

cudaError_t launch_linear_loss(const CUtensorMap &tmap_h, const CUtensorMap &tmap_w, const LinearLoss &p, bool grad,
                               int sm_count, int *status, cudaStream_t stream) {
  using namespace loss;
  static thread_local int configured_device = -1;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess)
    return err;
  if (configured_device != device) {
    for (const auto kernel : {linear_loss_kernel<false, false>, linear_loss_kernel<false, true>, linear_loss_kernel<true, false>,
                              linear_loss_kernel<true, true>}) {
      err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
      if (err != cudaSuccess)
        return err;
    }
    configured_device = device;
  }
  const int tiles_m = (p.rows + kTileM - 1) / kTileM, tiles_n = (p.vocab + kTileN - 1) / kTileN;
  const long long tiles = static_cast<long long>(tiles_m) * tiles_n;
  if (tiles <= 0 || tiles > 0x3fffffffLL)
    return cudaErrorInvalidValue;
  const long long clusters = tiles < sm_count / 2 ? tiles : sm_count / 2;
  const uint32_t idesc = make_idesc_f16(p.c_dtype == kCTypeBF16 ? 1u : 0u, false, false, kTileM, kTileN);
  const unsigned grid = static_cast<unsigned>(2 * clusters);
  const bool runs = p.width > kRunBlocks * kBlockK;
  const auto kernel = grad ? (runs ? linear_loss_kernel<true, true> : linear_loss_kernel<true, false>)
                           : (runs ? linear_loss_kernel<false, true> : linear_loss_kernel<false, false>);
  kernel<<<grid, kThreads, kSmemBytes, stream>>>(tmap_h, tmap_w, p, idesc, tiles_m, tiles_n, 8, status);
  return cudaGetLastError();
}

cudaError_t launch_linear_loss_join(const LinearLoss &p, cudaStream_t stream) {
  loss::join_kernel<<<(p.rows + 31) / 32, 32 * loss::kJoinWarps, 0, stream>>>(p, linear_loss_parts(p.vocab));
  return cudaGetLastError();
}

cudaError_t launch_linear_loss_prepare(const LinearLoss &p, float *scales, const void *h, long long ldh, void *copy,
                                       long long ldc, cudaStream_t stream) {
  const bool wide = (reinterpret_cast<uintptr_t>(h) & 15) == 0 && (ldh & 7) == 0;
  const int words = wide ? (p.width + 7) / 8 : p.width;
  const dim3 grid(copy == nullptr ? 1u : static_cast<unsigned>(words < 4096 ? (words + 255) / 256 : 16),
                  copy == nullptr ? 1u : static_cast<unsigned>(1 + (p.rows < 65534 ? p.rows : 65534)));
  const uint16_t *src = static_cast<const uint16_t *>(h);
  uint16_t *dst = static_cast<uint16_t *>(copy);
  if (wide)
    loss::prepare_kernel<uint4><<<grid, 256, 0, stream>>>(p, scales, src, ldh, dst, ldc);
  else
    loss::prepare_kernel<uint16_t><<<grid, 256, 0, stream>>>(p, scales, src, ldh, dst, ldc);
  return cudaGetLastError();
}

cudaError_t launch_spread(const void *src, long long lds, void *dst, long long ldd, int rows, int cols, int sm_count,
                          cudaStream_t stream) {
  if (rows == 0 || cols == 0)
    return cudaSuccess;
  const long long blocks = (static_cast<long long>(rows) * ((cols + 14) / 8) + 255) / 256, most = 16LL * sm_count;
  loss::spread_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(
      static_cast<const uint16_t *>(src), lds, static_cast<uint16_t *>(dst), ldd, rows, cols);
  return cudaGetLastError();
}

cudaError_t launch_linear_loss_narrow(const LinearLoss &p, const float *src, long long lds, void *dst, long long ldd, int cols,
                                      cudaStream_t stream) {
  if (p.rows == 0 || cols == 0)
    return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((cols + 1023) / 1024), static_cast<unsigned>(p.rows < 65535 ? p.rows : 65535));
  if ((ldd & 3) == 0 && (reinterpret_cast<uintptr_t>(dst) & 7) == 0)
    loss::narrow_kernel<uint2><<<grid, 256, 0, stream>>>(p, src, lds, dst, ldd, cols);
  else
    loss::narrow_kernel<uint16_t><<<grid, 256, 0, stream>>>(p, src, lds, dst, ldd, cols);
  return cudaGetLastError();
}

}  // namespace sm100
}  // namespace hc

// Products of a few rows with a matrix of 4-bit weights and group scales, for sm_100a.
//
//   C[i, j] = sum_groups s[j, g] sum_{k in group g} (q[j, k] - z[j, g]) A[i, k]
//
// q: 0..15, two to a byte (even k in the low half), rows of ceil(k / 2) bytes; s: one scale per row of q and
// group of 32, 64 or a multiple of 128 consecutive k, in A's type; z: one byte each, or 8 throughout. A: m <= 64 rows of
// float16 or bfloat16.
//
// Bound: HBM reads of q, half a byte per weight, as long as the work per weight hides under them: at the
// copy bandwidth an SM receives about 45 weights per cycle, so a warp may spend under three instructions
// per 32 of them. The weights therefore go to the tensor cores as integers: a nibble becomes a 16-bit float by
// being put under the exponent of 1024 (128 for bfloat16), one subtraction of 1024 + z -- exact -- serves two of
// them, and mma.sync (16 weights rows x 16 of k x 8 rows of A, float32 sums) does the rest. The group's
// scale multiplies the float32 sums of the group, so the only roundings are those of float32 sums and of the
// result: nothing is lost to a 16-bit product of scale and weight. (tcgen05 would want the weights expanded
// in shared memory and its sums drained from tensor memory at every group; with at most 8 columns in use
// the tensor work is a twentieth of the unpacking.)
//
// Layout of the work. A stage is 128 rows of q x 256 of k (16 KiB) and the m rows of A for them, brought by
// TMA into a ring of 128-byte-swizzled buffers (out-of-range rows, bytes and k read as zeros), so bytes in
// flight do not depend on registers. Eight warps take it: 4 of 32 rows x 2 of 128 k. In a 32-bit word of q
// sit 8 consecutive k; a lane reads the word its quad position names, and the four pairs (0,4) (1,5) (2,6)
// (3,7) that masks and shifts produce are used as the fragment's k pairs -- sums do not care in which order
// k runs, A's fragment is permuted alike.
//
// Rows of q that do not start on 16-byte boundaries (an odd k) cannot be addressed by a tensor map: a
// producer warp then copies each row's bytes with cp.async.bulk from the boundary below its start, and the
// consumers read at the row's own phase with a funnel shift.
//
// The (row block, stage of k) units are dealt out as one sequence, an equal share to every CTA, so that the GPU
// is evenly loaded whatever n and k are; a CTA whose share begins or ends inside a row block leaves float32
// sums, and the last of the CTAs that share a block adds them in their order (no CTA waits).
#pragma once

#include "gemm_epilogue.cuh"
#include "device_checks.cuh"
#include "gemm_launch.h"
#include "sm100_ptx.cuh"

namespace hc {
namespace sm100 {

namespace w4 {

constexpr int kRows = 128;        // rows of q per block
constexpr int kStageK = 256;      // of k per stage: 128 bytes of q
constexpr int kConsumers = 8;     // warps: 4 (rows) x 2 (k)
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kQuarterRows = 32;  // rows per consumer warp: two fragments of 16
constexpr uint32_t kQBytes = kRows * 128;
constexpr uint32_t kPhasePitch = 144;  // bytes per row of a stage copied at its own phase
constexpr uint32_t kQPhaseBytes = kRows * kPhasePitch;

// The ring: as many stages as fit with `kTiles` n-tiles of 8 rows of A.
template <int kTiles, bool kPhase>
struct Ring {
  static constexpr uint32_t kABoxBytes = 8 * kTiles * 128;      // 64 of k x padded m
  static constexpr uint32_t kABytes = (kStageK / 64) * kABoxBytes;
  static constexpr uint32_t kQStageBytes = kPhase ? (kQPhaseBytes + 1023) / 1024 * 1024 : kQBytes;
  static constexpr uint32_t kStageBytes = kQStageBytes + kABytes;
  // Two CTAs per SM for up to 16 rows of A, one beyond.
  static constexpr uint32_t kBudget = kTiles <= 2 ? 100 * 1024 : 192 * 1024;
  static constexpr int kStages = kBudget / kStageBytes < 8 ? static_cast<int>(kBudget / kStageBytes) : 8;
  // Behind the ring: barriers, then the place where the sums of the two k halves meet.
  static constexpr uint32_t kMeetBytes = kRows * 8 * kTiles * 4;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 256 + kMeetBytes + 1024;
  static_assert(kStages >= 2 && kSmemBytes <= (kTiles <= 2 ? 113 : 227) * 1024, "shared memory of a CTA");
};

template <bool kBf16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (x & mask) | magic
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(magic));
  return r;
}

// What a row's zero point subtracts from the expanded nibbles.
template <bool kBf16>
struct Zero {
  __nv_bfloat162 low;
  __device__ explicit Zero(int z) { low = __float2bfloat162_rn(128.0f + static_cast<float>(z)); }
  __device__ Zero() {}
};
template <>
struct Zero<false> {
  __half2 low, high;  // 1024 + z, and 64 + z for nibbles left four bits up
  __device__ explicit Zero(int z) {
    low = __float2half2_rn(1024.0f + static_cast<float>(z));
    high = __float2half2_rn(-64.0f - static_cast<float>(z));
  }
  __device__ Zero() {}
};

// Eight nibbles of a word as four pairs (0,4) (1,5) (2,6) (3,7) of exact 16-bit floats q - z.
__device__ __forceinline__ void expand(uint32_t w, const Zero<true> &z, uint32_t (&out)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), z.low);
    out[i] = *reinterpret_cast<const uint32_t *>(&d);
  }
}
__device__ __forceinline__ void expand(uint32_t w, const Zero<false> &z, uint32_t (&out)[4]) {
  const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = w >> (8 * i);
    const uint32_t v = and_or(x, 0x000f000fu, 0x64006400u);
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&v), z.low);
    out[2 * i] = *reinterpret_cast<const uint32_t *>(&d);
    const uint32_t u = and_or(x, 0x00f000f0u, 0x64006400u);  // 1024 + 16 q
    const __half2 e = __hfma2(*reinterpret_cast<const __half2 *>(&u), sixteenth, z.high);
    out[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&e);
  }
}

template <bool kBf16>
__device__ __forceinline__ float scale_value(uint16_t bits) {
  if constexpr (kBf16)
    return __uint_as_float(static_cast<uint32_t>(bits) << 16);
  else
    return __half2float(__ushort_as_half(bits));
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// Bulk copy, global -> shared; both addresses and the size multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}

// The units (row block, stage of k) of CTA `cta` are [first_unit(cta), first_unit(cta + 1)); owner_of is the
// CTA of a unit. There are at least as many units as CTAs.
__device__ __forceinline__ long long first_unit(long long cta, long long units, long long grid) { return cta * units / grid; }
__device__ __forceinline__ long long owner_of(long long unit, long long units, long long grid) {
  return ((unit + 1) * grid - 1) / units;
}

// Barriers of the consumer warps, and of the four of them that hold a block's sums.
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory"); }
__device__ __forceinline__ void half_sync() { asm volatile("bar.sync 2, %0;" ::"n"(16 * kConsumers) : "memory"); }

template <bool kBf16, int kTiles, bool kPhase, int kGroup>
__global__ void __launch_bounds__(kThreads, kTiles <= 2 ? 2 : 1)
gemm_w4_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_a, const W4 p,
               int *status) {
  using R = Ring<kTiles, kPhase>;
  constexpr int kGroupsPerStage = kStageK / kGroup;        // 2, 4 or 8
  constexpr int kGroupsPerHalf = kGroupsPerStage / 2;      // of a warp's 128 of k: 1, 2 or 4
  constexpr int kChunksPerGroup = kGroup / 32;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t bar_base = smem_base + R::kStages * R::kStageBytes;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (R::kStages + s); };
  volatile uint32_t *abort_flag =
      reinterpret_cast<volatile uint32_t *>(smem_gen + R::kStages * R::kStageBytes + 8u * 2 * R::kStages);
  volatile uint32_t *last_flag = abort_flag + 1;
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < R::kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), kConsumers);
    }
    *abort_flag = 0;
    mbar_fence_init();
    if (!kPhase)
      tma_prefetch_descriptor(&tmap_q);
    tma_prefetch_descriptor(&tmap_a);
  }
  __syncthreads();

  const long long grid = gridDim.x;
  const long long unit_begin = first_unit(blockIdx.x, p.units, grid), unit_end = first_unit(blockIdx.x + 1, p.units, grid);
  const int stages_k = p.stages_k;

  if (warp == kConsumers) {
    // ------------------------------------------------------------ producer ----------
    uint32_t stage = 0, phase = 0;
    long long block = unit_begin / stages_k;
    int ks = static_cast<int>(unit_begin - block * stages_k);
    for (long long unit = unit_begin; unit < unit_end; ++unit) {
      const bool free = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag);
      if (!__all_sync(0xffffffffu, free))
        break;
      const uint32_t q_dst = smem_base + stage * R::kStageBytes, a_dst = q_dst + R::kQStageBytes;
      if constexpr (!kPhase) {
        if (lane == 0) {
          mbar_arrive_expect_tx(full_bar(stage), R::kStageBytes);
          tma_load_2d(q_dst, &tmap_q, full_bar(stage), ks * 128, static_cast<int>(block) * kRows);
#pragma unroll
          for (int j = 0; j < kStageK / 64; ++j)
            tma_load_2d(a_dst + j * R::kABoxBytes, &tmap_a, full_bar(stage), ks * kStageK + j * 64, 0);
        }
      } else {
        // Each lane brings four rows: the 16-byte pieces from the boundary at or below the row's first
        // byte of this stage up to the last one that lies wholly inside q; what is left of q's very end
        // goes byte by byte.
        uint32_t bytes[kRows / 32], total = 0;
        const uint8_t *source[kRows / 32];
        const uint8_t *const q_end = p.q + (static_cast<long long>(p.n) - 1) * p.ldq + p.row_bytes;
#pragma unroll
        for (int i = 0; i < kRows / 32; ++i) {
          const long long row = block * kRows + i * 32 + lane;
          bytes[i] = 0;
          source[i] = nullptr;
          if (row < p.n) {
            const uint8_t *begin = p.q + row * p.ldq + ks * 128ll;
            const int wanted = min(128, p.row_bytes - ks * 128);  // at least 1
            const uint8_t *low = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(begin) & ~uintptr_t{15});
            const uint8_t *high = reinterpret_cast<const uint8_t *>(
                (reinterpret_cast<uintptr_t>(begin + wanted) + 15) & ~uintptr_t{15});
            const uint32_t dst = q_dst + static_cast<uint32_t>(i * 32 + lane) * kPhasePitch;
            if (high > q_end) {
              const uint8_t *whole = reinterpret_cast<const uint8_t *>(reinterpret_cast<uintptr_t>(q_end) & ~uintptr_t{15});
              if (whole < low)
                whole = low;
              for (const uint8_t *b = whole < begin ? begin : whole; b < begin + wanted; ++b)
                smem_gen[dst - smem_base + static_cast<uint32_t>(b - low)] = *b;
              fence_proxy_async_smem();
              high = whole;
            }
            source[i] = low;
            bytes[i] = static_cast<uint32_t>(high - low);
          }
          total += bytes[i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          total += __shfl_xor_sync(0xffffffffu, total, o);
        // The bytes stored above are ordered before the consumers' reads by lane 0's arrival.
        __syncwarp();
        if (lane == 0)
          mbar_arrive_expect_tx(full_bar(stage), total + R::kABytes);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kRows / 32; ++i)
          if (bytes[i] != 0)
            bulk_load(q_dst + static_cast<uint32_t>(i * 32 + lane) * kPhasePitch, source[i], bytes[i], full_bar(stage));
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < kStageK / 64; ++j)
            tma_load_2d(a_dst + j * R::kABoxBytes, &tmap_a, full_bar(stage), ks * kStageK + j * 64, 0);
        }
      }
      if (++stage == R::kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++ks == stages_k) {
        ks = 0;
        ++block;
      }
    }
  }

  // ---------------------------------------------------------------- consumers ----------
  const int row_warp = warp & 3, k_half = (warp >> 2) & 1;
  const int g = lane >> 2, q4 = lane & 3;  // fragment row (or row of A), position in the quad
  float *const meet = reinterpret_cast<float *>(smem_gen + R::kStages * R::kStageBytes + 256);
  uint32_t stage = 0, phase = 0;
  long long unit = unit_begin;
  bool ok = true;  // (a wait that ran out: the barriers below are still met)
  while (warp < kConsumers && unit < unit_end) {
    const long long block = unit / stages_k;
    const int ks_begin = static_cast<int>(unit - block * stages_k);
    const long long left = unit_end - unit;
    const int ks_end = left < stages_k - ks_begin ? ks_begin + static_cast<int>(left) : stages_k;
    float total[2][kTiles][4];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          total[f][t][e] = 0.0f;
    if (ok) {
      // This lane's four rows of q: two fragments, rows g and g + 8 of each.
      long long row[4];
      uint32_t row_at[4], row_shift[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int local = row_warp * kQuarterRows + i * 8 + g;
        row[i] = block * kRows + local;
        if (row[i] >= p.n)
          row[i] = p.n - 1;  // computed and not stored
        if constexpr (kPhase) {
          const uint32_t at = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(p.q) + (block * kRows + local) * p.ldq) & 15);
          row_at[i] = static_cast<uint32_t>(local) * kPhasePitch + (at & ~3u);
          row_shift[i] = 8 * (at & 3u);
        } else {
          row_at[i] = static_cast<uint32_t>(local) * 128;
          row_shift[i] = 0;
        }
      }
      // Scales and zero points of the warp's groups of a stage: group j of row i is held by quad position j.
      uint16_t next_scale[4];
      uint8_t next_zero[4];
      auto fetch = [&](int ks) {
        // (p.span: how many of the kernel's groups share a scale, for groups of several times 128.)
        const int group =
            min((ks * kGroupsPerStage + k_half * kGroupsPerHalf + (q4 % kGroupsPerHalf)) / p.span, p.groups - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          next_scale[i] = p.scales[row[i] * p.lds + group];
          next_zero[i] = p.zeros != nullptr ? p.zeros[row[i] * p.ldz + group] : uint8_t{8};
        }
      };
      fetch(ks_begin);
      for (int ks = ks_begin; ks < ks_end; ++ks) {
        uint32_t scale_bits[4], zero_bits[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          scale_bits[i] = next_scale[i];
          zero_bits[i] = next_zero[i];
        }
        if (ks + 1 < ks_end)
          fetch(ks + 1);
        const bool ready = mbar_wait(full_bar(stage), phase, abort_flag);
        if (!__all_sync(0xffffffffu, ready)) {
          ok = false;
          break;
        }
        const uint32_t q_addr = smem_base + stage * R::kStageBytes, a_addr = q_addr + R::kQStageBytes;
#pragma unroll
        for (int gi = 0; gi < kGroupsPerHalf; ++gi) {
          float scale[4];
          Zero<kBf16> zero[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t both = __shfl_sync(0xffffffffu, scale_bits[i] | (zero_bits[i] << 16), (lane & ~3) | gi);
            scale[i] = scale_value<kBf16>(static_cast<uint16_t>(both));
            zero[i] = Zero<kBf16>(static_cast<int>(both >> 16));
          }
          float sum[2][kTiles][4];
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sum[f][t][e] = 0.0f;
#pragma unroll
          for (int ci = 0; ci < kChunksPerGroup; ++ci) {
            const int chunk = k_half * 4 + gi * kChunksPerGroup + ci;  // 32 of k, 16 bytes of q
            // A: 8 consecutive k of one row per lane, paired as expand() pairs the weights.
            uint32_t b[kTiles][4];
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              const uint32_t box = a_addr + static_cast<uint32_t>(chunk >> 1) * R::kABoxBytes;
              const uint32_t piece = static_cast<uint32_t>((chunk & 1) * 4 + q4);
              const uint4 v = lds128(box + static_cast<uint32_t>(t * 8 + g) * 128 + ((piece ^ static_cast<uint32_t>(g)) << 4));
              b[t][0] = __byte_perm(v.x, v.z, 0x5410);
              b[t][1] = __byte_perm(v.x, v.z, 0x7632);
              b[t][2] = __byte_perm(v.y, v.w, 0x5410);
              b[t][3] = __byte_perm(v.y, v.w, 0x7632);
            }
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              uint32_t word[2], lo[4], hi[4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int i = 2 * f + h;
                if constexpr (kPhase) {
                  const uint32_t at = q_addr + row_at[i] + static_cast<uint32_t>(chunk * 16 + q4 * 4);
                  word[h] = __funnelshift_r(lds32(at), lds32(at + 4), row_shift[i]);
                } else {
                  word[h] = lds32(q_addr + row_at[i] + ((static_cast<uint32_t>(chunk) ^ static_cast<uint32_t>(g)) << 4) +
                                  static_cast<uint32_t>(q4 * 4));
                }
              }
              expand(word[0], zero[2 * f], lo);
              expand(word[1], zero[2 * f + 1], hi);
              const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
              for (int t = 0; t < kTiles; ++t) {
                mma<kBf16>(sum[f][t], a0, b[t][0], b[t][1]);
                mma<kBf16>(sum[f][t], a1, b[t][2], b[t][3]);
              }
            }
          }
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              total[f][t][0] = fmaf(scale[2 * f], sum[f][t][0], total[f][t][0]);
              total[f][t][1] = fmaf(scale[2 * f], sum[f][t][1], total[f][t][1]);
              total[f][t][2] = fmaf(scale[2 * f + 1], sum[f][t][2], total[f][t][2]);
              total[f][t][3] = fmaf(scale[2 * f + 1], sum[f][t][3], total[f][t][3]);
            }
        }
        __syncwarp();
        if (lane == 0)
          mbar_arrive(empty_bar(stage));
        if (++stage == R::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    unit += ks_end - ks_begin;

    // The two k halves meet in shared memory; lane (g, q4) of a fragment holds rows g and g + 8 and the
    // rows 2 q4, 2 q4 + 1 of A.
    auto place = [&](int f, int h, int t) {
      return (row_warp * kQuarterRows + f * 16 + h * 8 + g) * (8 * kTiles) + t * 8 + 2 * q4;
    };
    if (k_half == 1) {
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float2 *>(meet + place(f, h, t)) = make_float2(total[f][t][2 * h], total[f][t][2 * h + 1]);
    }
    consumers_sync();
    if (k_half == 0) {
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = *reinterpret_cast<const float2 *>(meet + place(f, h, t));
            total[f][t][2 * h] += v.x;
            total[f][t][2 * h + 1] += v.y;
          }
      bool store = true;
      if (ks_begin != 0 || ks_end != stages_k) {
        // Part of a block: leave the sums in this CTA's slot and count it in. The CTAs that share the
        // block are consecutive; the one that counts last adds all parts in their order.
        constexpr int kSlot = kRows * 8 * kTiles;
        const long long first = owner_of(block * stages_k, p.units, grid);
        const long long last = owner_of((block + 1) * stages_k - 1, p.units, grid);
        auto slot_of = [&](long long cta) {
          return p.partials + (2 * cta + (first_unit(cta, p.units, grid) / stages_k == block ? 0 : 1)) * kSlot;
        };
        float *mine = slot_of(blockIdx.x);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              __stcg(reinterpret_cast<float2 *>(mine + place(f, h, t)), make_float2(total[f][t][2 * h], total[f][t][2 * h + 1]));
        __threadfence();
        half_sync();
        if (threadIdx.x == 0) {
          const unsigned parts = static_cast<unsigned>(last - first + 1);
          const unsigned before = atomicAdd(p.counters + block, 1u);
          *last_flag = before + 1 == parts ? 1u : 0u;
          if (before + 1 == parts)
            p.counters[block] = 0u;  // as it was found
          __threadfence();
        }
        half_sync();
        store = *last_flag != 0;
        if (store) {
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                total[f][t][e] = 0.0f;
          for (long long cta = first; cta <= last; ++cta) {
            const float *part = slot_of(cta);
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
              for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float2 v = __ldcg(reinterpret_cast<const float2 *>(part + place(f, h, t)));
                  total[f][t][2 * h] += v.x;
                  total[f][t][2 * h + 1] += v.y;
                }
          }
        }
      }
      if (store) {
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const long long column = block * kRows + row_warp * kQuarterRows + f * 16 + (e >> 1) * 8 + g;
              const int i = t * 8 + 2 * q4 + (e & 1);
              if (i < p.m && column < p.n)
                store_c_element(p.c, static_cast<long long>(i) * p.ldc + column, total[f][t][e], p.c_dtype);
            }
      }
    }
    consumers_sync();  // `meet` is free again
  }
  __syncthreads();
  if (*abort_flag != 0) {
    if (threadIdx.x == 0)
      atomicCAS(status, 0, kStatusDeviceWaitTimeout);
    const long long start = clock64();
    while (clock64() - start < 2000000LL) {
    }
  }
}

template <bool kBf16, int kTiles, bool kPhase, int kGroup>
cudaError_t launch(const CUtensorMap &tmap_q, const CUtensorMap &tmap_a, const W4 &p, int *status, cudaStream_t stream) {
  using R = Ring<kTiles, kPhase>;
  static thread_local int configured_device = -1;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess)
    return err;
  if (configured_device != device) {
    err = cudaFuncSetAttribute(gemm_w4_kernel<kBf16, kTiles, kPhase, kGroup>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(R::kSmemBytes));
    if (err != cudaSuccess)
      return err;
    configured_device = device;
  }
  gemm_w4_kernel<kBf16, kTiles, kPhase, kGroup><<<p.grid, kThreads, R::kSmemBytes, stream>>>(tmap_q, tmap_a, p, status);
  return cudaGetLastError();
}

template <bool kBf16>
cudaError_t launch_w4(const CUtensorMap &tmap_q, const CUtensorMap &tmap_a, const W4 &p, int *status, cudaStream_t stream) {
  const int tiles = w4_tiles(p.m);
  const bool phase = p.phase != 0;
#define HC_W4(TILES, GROUP)                                                               \
  return phase ? launch<kBf16, TILES, true, GROUP>(tmap_q, tmap_a, p, status, stream)     \
               : launch<kBf16, TILES, false, GROUP>(tmap_q, tmap_a, p, status, stream)
#define HC_W4_GROUPS(TILES) \
  {                         \
    if (p.group == 32)      \
      HC_W4(TILES, 32);     \
    if (p.group == 64)      \
      HC_W4(TILES, 64);     \
    HC_W4(TILES, 128);      \
  }
  if (tiles == 1)
    HC_W4_GROUPS(1)
  if (tiles == 2)
    HC_W4_GROUPS(2)
  if (tiles == 4)
    HC_W4_GROUPS(4)
  HC_W4_GROUPS(8)
#undef HC_W4_GROUPS
#undef HC_W4
}

}  // namespace w4
}  // namespace sm100
}  // namespace hc

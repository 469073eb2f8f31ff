// Products of a few rows with a matrix of 4-bit weights and group scales, for sm_100a.
//
//   C[i, j] = sum_groups s[j, g] sum_{k in group g} (q[j, k] - z[j, g]) A[i, k]
//
// q: 0..15, two to a byte (even k in the low half), rows of ceil(k / 2) bytes; s: one scale per row of q and
// group of 32, 64 or a multiple of 128 consecutive k, in A's type; z: the low six bits of a byte each, or 8 throughout. A:
// m <= 64 rows of float16 or bfloat16.
//
// Bound: HBM reads of q, half a byte per weight. At the copy bandwidth an SM receives 45 weights per cycle, and
// turning them into 16-bit floats is integer work (masks and shifts, at half the issue rate): 5 to 7 such
// instructions per 8 weights leave little room for anything else.
//
// The weights enter the product as integers: a nibble becomes a float by being put under the exponent of 1024
// (128 for bfloat16), and one subtraction of 1024 + z, exact, serves two of them (Kim, Henry, Fahim, Hassan Awadalla,
// "Who Says Elephants Can't Run", 2022, describe it for weights of 8 and 4 bits). The group's scale
// multiplies the float32 sums of the group. So nothing is lost to a 16-bit product of scale and weight: the
// only roundings are those of float32 sums and of the result.
//
// q and A arrive by TMA in a ring of 128-byte-swizzled stages of 128 rows x 256 of k (out-of-range rows, bytes
// and k read as zeros), computed as C^T = W A^T. In a 32-bit word of q sit 8 consecutive k; masks and shifts
// pair them as (0,4) (1,5) (2,6) (3,7). Sums do not care in which order k runs, so A's pairs are formed alike.
//
// Up to 16 rows of A: mma.sync with 16 rows of q by 16 of k by 8 rows of A. The tensor work is small whatever
// the instruction, and a warp that expands weights into its own fragments and keeps its own sums hands nothing
// on: it only waits for stages. What is the same for several of them is done once: one more warp starts the loads
// and lays out scales and zero points ready to use, another forms A's pairs in shared memory. Four consumer warps
// of 32 rows make a CTA with these two, three CTAs share an SM. (1 x 16384 x 8192 in bfloat16: 24.7 us; with the
// scales fetched by every consumer a stage ahead 30.8, with one warp for loads, scales and pairs 26.8.)
//
// 17 to 64 rows: tcgen05.mma with M = 128 rows of q, N = 32 or 64. The expanded weights go to the tensor cores
// through tensor memory, not through shared memory (the expanded form is four times q's bytes, which shared
// memory would have to take and give back): a lane of an expanding warp owns a row of q, which is the lane its
// operand has to lie in. Two sets of four warps take one half of a stage's k each; a set has two operand
// buffers, so that a step's products run while the next is expanded. Four more warps collect: they read a
// group's sums, add them, times the group's scale, to the running ones, and write C or join parts while the next
// block is expanded already. The instructions are so small (N = 64 at most) that issuing them is what bounds
// the kernel: one thread takes about 70 cycles for each, so each set has an issuing warp of its own
// (64 x 18944 x 8192: 45.6 us with one, 39.1 with two, 37.9 with elect.sync in place of a lane's number). Here the
// weights are expanded in the order of k, so that A is read as it lies.
//
// Rows of q that do not all start on 16-byte boundaries (an odd k) have a pitch that no tensor map takes, but every
// sixteenth row lies at the same place between two boundaries: sixteen maps, of every sixteenth row from the
// boundary at or below its start, bring such rows, 8 rows of 144 bytes each. In shared memory the rows of a block
// then lie sorted by that place (position 8 r + i holds row 16 i + r), and the readers take words at a row's own
// phase with a funnel shift. (1 x 18944 x 8190: 33.0 us; when warps copied the rows with cp.async, 57.5 us.)
//
// A's boxes have no more rows than A (for the tensor cores, whole groups of eight). What the ring holds in the places
// of rows that are not there only reaches sums that nobody stores.
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
constexpr uint32_t kQBytes = kRows * 128;
constexpr int kPhases = w4_phases();
constexpr uint32_t kPhasePitch = 128 + 16;  // a row of a stage, with what precedes it to the boundary
constexpr uint32_t kQPhaseBytes = kRows * kPhasePitch;

// The row of a block at a position.
template <bool kPhase>
__device__ __forceinline__ int row_at_position(int position) {
  return kPhase ? (position & (kRows / kPhases - 1)) * kPhases + position / (kRows / kPhases) : position;
}

// The maps of q: one, or one for every phase.
template <bool kPhase>
struct QMaps {
  CUtensorMap map[kPhase ? kPhases : 1];
};

// (x & mask) | magic
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(magic));
  return r;
}

// What a row's zero point subtracts from the expanded nibbles. Six bits of it, for all numbers of rows of A alike: that
// is what 64 + z leaves in float16 four bits further up (set_pair), and all of it is exact in both types.
constexpr uint32_t kZeroBits = 0x3fu;
template <bool kBf16>
struct Zero {
  __nv_bfloat162 low;  // 128 + z
  __device__ void set(int z) { low = __float2bfloat162_rn(128.0f + static_cast<float>(z)); }
  // From the pair that StageScales stores.
  __device__ void set_pair(uint32_t pair) { low = *reinterpret_cast<const __nv_bfloat162 *>(&pair); }
};
template <>
struct Zero<false> {
  __half2 low, high;  // 1024 + z, and -(64 + z) for nibbles left four bits up
  __half2 mixed;      // -(1024 + z), -(64 + z)
  __device__ void set(int z) {
    low = __float2half2_rn(1024.0f + static_cast<float>(z));
    high = __float2half2_rn(-64.0f - static_cast<float>(z));
    mixed = __floats2half2_rn(-1024.0f - static_cast<float>(z), -64.0f - static_cast<float>(z));
  }
  __device__ void set_pair(uint32_t pair) {
    low = *reinterpret_cast<const __half2 *>(&pair);
    const uint32_t up = and_or(pair << 4, 0x03f003f0u, 0xd400d400u);
    high = *reinterpret_cast<const __half2 *>(&up);
  }
};

// Eight nibbles of a word as four pairs (0,4) (1,5) (2,6) (3,7) of exact 16-bit floats q - z.
__device__ __forceinline__ void expand(uint32_t w, const Zero<true> &z, uint32_t *out) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), z.low);
    out[i] = *reinterpret_cast<const uint32_t *>(&d);
  }
}
__device__ __forceinline__ void expand(uint32_t w, const Zero<false> &z, uint32_t *out) {
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

// The same in the order of k, pairs (0,1) (2,3) (4,5) (6,7), at two or three instructions more per word: a byte
// comes into both halves of a word, and of one of them the upper nibble counts (which bfloat16 has no bits for).
__device__ __forceinline__ void expand_in_order(uint32_t w, const Zero<true> &z, uint32_t *out) {
  const uint32_t upper = w >> 4;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t v = and_or(__byte_perm(w, upper, 0x0400u + 0x1111u * i), 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), z.low);
    out[i] = *reinterpret_cast<const uint32_t *>(&d);
  }
}
__device__ __forceinline__ void expand_in_order(uint32_t w, const Zero<false> &z, uint32_t *out) {
  const __half2 down = __floats2half2_rn(1.0f, 0.0625f);
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t v = and_or(__byte_perm(w, w, 0x1111u * i), 0x00f0000fu, 0x64006400u);  // 1024 + q, 1024 + 16 q
    const __half2 d = __hfma2(*reinterpret_cast<const __half2 *>(&v), down, z.mixed);
    out[i] = *reinterpret_cast<const uint32_t *>(&d);
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

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4 &v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Between a warp's reads of a stage and the arrival that gives the stage back. TMA refills it through the asynchronous
// proxy, and reads of the generic proxy are kept in front of that by a proxy fence only: without it the last words of a
// stage could be read from the next one (1 to 8 rows of float16: some thousand wrong sums in 3 x 300000 x 32768).
__device__ __forceinline__ void read_before_refill() {
  fence_proxy_async_smem();
  __syncwarp();
}

// 32 columns of this warp's lanes of tensor memory.
__device__ __forceinline__ void tmem_store_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
         "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
         "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
         "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// True in one lane of the (whole) warp, which the compiler knows to be one.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem]: 16-bit operands, the first from tensor memory (a lane per row, two of k
// per column).
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The units (row block, stage of k) of CTA `cta` are [first_unit(cta), first_unit(cta + 1)); owner_of is the CTA
// of a unit.
__device__ __forceinline__ int first_unit(const W4 &p, int cta) { return cta * p.share + min(cta, p.extra); }
__device__ __forceinline__ int owner_of(const W4 &p, int unit) {
  const int long_ones = p.extra * (p.share + 1);
  return unit < long_ones ? unit / (p.share + 1) : p.extra + (unit - long_ones) / p.share;
}

// Index checks of the checked build: a unit a CTA is about to load, and a block whose parts lie in first .. last.
__device__ __forceinline__ bool unit_ok(const W4 &p, uint32_t stage, int stages, int block, int ks, int *status,
                                        volatile uint32_t *abort_flag) {
  return HC_CHECK(status, abort_flag, HC_CHECK_RING_STAGE, stage < static_cast<uint32_t>(stages)) &&
         HC_CHECK(status, abort_flag, HC_CHECK_TILE_COORDINATES,
                  block >= 0 && static_cast<long long>(block) * kRows < p.n && ks >= 0 && ks < p.stages_k) &&
         HC_CHECK(status, abort_flag, HC_CHECK_TMA_COORDINATES, ks * 128 < p.row_bytes);
}
__device__ __forceinline__ bool parts_ok(const W4 &p, int cta, int first, int last, int block, int *status,
                                         volatile uint32_t *abort_flag) {
  return HC_CHECK(status, abort_flag, HC_CHECK_PARTIAL_SLOT,
                  first >= 0 && first <= cta && cta <= last && last < p.grid && block >= 0 &&
                      first_unit(p, first) < (block + 1) * p.stages_k && first_unit(p, last + 1) >= (block + 1) * p.stages_k);
}

// A CTA that did part of a row block leaves its sums in a slot of its own: its first if the block is the first
// it touches, else its second. Of the CTAs `first` .. that share a block only `first` may have begun before it.
__device__ __forceinline__ float *part_slot(const W4 &p, int cta, int first, int block, int slot_floats) {
  const int second = cta == first && first_unit(p, first) < block * p.stages_k ? 1 : 0;
  return p.partials + static_cast<size_t>(2 * cta + second) * slot_floats;
}

// After the slot is written: counts the part in and tells whether this CTA's is the last of the block's `parts`
// (which then adds all of them in their order). `sync` is a barrier of the threads that hold the sums, thread 0
// among them; its atomic operation releases what they wrote and acquires what the other CTAs' released.
template <typename Sync>
__device__ __forceinline__ bool count_part(const W4 &p, int block, int parts, volatile uint32_t *last_flag, Sync sync) {
  sync();
  if (threadIdx.x == 0) {
    unsigned before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + block) : "memory");
    const bool all = before + 1 == static_cast<unsigned>(parts);
    if (all)
      p.counters[block] = 0u;  // as it was found
    *last_flag = all ? 1u : 0u;
  }
  sync();
  const bool all = *last_flag != 0;
  sync();  // the flag may be written again
  return all;
}

// A stage of q; all lanes of a warp.
template <bool kPhase>
__device__ __forceinline__ void load_q(const QMaps<kPhase> &maps, uint32_t dst, uint32_t full, int block, int ks, int lane) {
  if constexpr (kPhase) {
    if (lane < kPhases)
      tma_load_2d(dst + static_cast<uint32_t>(lane) * (kRows / kPhases * kPhasePitch), &maps.map[lane], full, ks * 128,
                  block * (kRows / kPhases));
  } else {
    if (lane == 0)
      tma_load_2d(dst, &maps.map[0], full, ks * 128, block * kRows);
  }
}

// 32-bit words, or bytes packed into words, from an address aligned to all of them.
__device__ __forceinline__ void load_words(const void *src, uint32_t (&out)[1]) {
  out[0] = __ldg(static_cast<const uint32_t *>(src));
}
__device__ __forceinline__ void load_words(const void *src, uint32_t (&out)[2]) {
  const uint2 v = __ldg(static_cast<const uint2 *>(src));
  out[0] = v.x, out[1] = v.y;
}
__device__ __forceinline__ void load_words(const void *src, uint32_t (&out)[4]) {
  const uint4 v = __ldg(static_cast<const uint4 *>(src));
  out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
}
template <int kBytes>
__device__ __forceinline__ void load_bytes(const uint8_t *src, uint32_t (&out)[(kBytes + 3) / 4]) {
  if constexpr (kBytes == 2)
    out[0] = __ldg(reinterpret_cast<const uint16_t *>(src));
  else
    load_words(src, out);
}

// Eight consecutive 16-bit k of A in the order (0,4) (1,5) (2,6) (3,7).
__device__ __forceinline__ uint4 in_pairs(const uint4 &v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// The scales and zero points on their way from memory to the stages, four rows of q per lane of the warp that
// brings them: fetched as they lie in memory, kAhead stages early, and stored as pairs (the scale as a float,
// what the zero point subtracts as two 16-bit floats), [group of the stage][row].
template <bool kBf16, bool kPhase, int kGroup>
struct ScaleStream {
  static constexpr int kGroups = kStageK / kGroup;  // of a stage: 2, 4 or 8
  static constexpr int kAhead = 2;
  static constexpr int kZeroWords = (kGroups + 3) / 4;
  uint32_t scale[kAhead][kRows / 32][kGroups / 2], zero[kAhead][kRows / 32][kZeroWords];
  const uint16_t *scale_row[kRows / 32];
  const uint8_t *zero_row[kRows / 32];
  int left, ks;    // units still to be fetched; the stage of k of the next
  long long block;  // of the next

  __device__ __forceinline__ ScaleStream(const W4 &p, int unit_begin, int unit_end, int lane) {
    left = unit_end - unit_begin;
    block = unit_begin / p.stages_k;
    ks = unit_begin - static_cast<int>(block) * p.stages_k;
    point(p, lane);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      fetch(p, i, lane);
  }
  __device__ __forceinline__ void point(const W4 &p, int lane) {
#pragma unroll
    for (int i = 0; i < kRows / 32; ++i) {
      // Rows past the end take the last row's scales; their results are not stored.
      const long long at = block * kRows + row_at_position<kPhase>(i * 32 + lane), row = at < p.n ? at : p.n - 1;
      scale_row[i] = p.scales + row * p.lds;
      zero_row[i] = p.zeros + row * p.ldz;
    }
  }
  __device__ __forceinline__ void fetch(const W4 &p, int to, int lane) {
    if (--left < 0)
      return;
    const int first = ks * kGroups;
#pragma unroll
    for (int i = 0; i < kRows / 32; ++i) {
#pragma unroll
      for (int j = 0; j < kZeroWords; ++j)
        zero[to][i][j] = p.zeros == nullptr ? 0x08080808u : 0u;
      if (p.vector_scales) {  // whole groups of whole stages, on boundaries of as many
        load_words(scale_row[i] + first, scale[to][i]);
        if (p.zeros != nullptr)
          load_bytes<kGroups>(zero_row[i] + first, zero[to][i]);
      } else {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          // (p.span: how many of the kernel's groups share a scale, for groups of several times 128.)
          const int group = min(p.span == 1 ? first + j : (first + j) / p.span, p.groups - 1);
          const uint32_t v = scale_row[i][group];
          scale[to][i][j / 2] = j % 2 == 0 ? v : scale[to][i][j / 2] | v << 16;
          if (p.zeros != nullptr)
            zero[to][i][j / 4] |= static_cast<uint32_t>(zero_row[i][group]) << (8 * (j % 4));
        }
      }
    }
    if (++ks == p.stages_k) {
      ks = 0;
      ++block;
      if (left > 0)
        point(p, lane);
    }
  }
  // The oldest stage fetched goes to `at`, another is fetched.
  __device__ __forceinline__ void advance(const W4 &p, uint32_t at, int lane) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
#pragma unroll
      for (int i = 0; i < kRows / 32; ++i) {
        const uint32_t bits = j % 2 == 0 ? scale[0][i][j / 2] & 0xffffu : scale[0][i][j / 2] >> 16;
        const uint32_t pair = __byte_perm(zero[0][i][j / 4] & (kZeroBits * 0x01010101u), kBf16 ? 0x43434343u : 0x64646464u,
                                          0x4040u | (0x101u * (j % 4)));
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};"
                     :: "r"(at + static_cast<uint32_t>((j * kRows + i * 32 + lane) * 8)),
                        "r"(__float_as_uint(scale_value<kBf16>(static_cast<uint16_t>(bits)))), "r"(pair)
                     : "memory");
      }
#pragma unroll
    for (int i = 0; i < kRows / 32; ++i) {
#pragma unroll
      for (int j = 0; j < kGroups / 2; ++j)
        scale[0][i][j] = scale[1][i][j];
#pragma unroll
      for (int j = 0; j < kZeroWords; ++j)
        zero[0][i][j] = zero[1][i][j];
    }
    fetch(p, 1, lane);
  }
};

// A's pairs for mma.sync: rows of 512 bytes, of every other one the two halves of each 128 bytes change places
// too, so that the consumers' loads of a pair of rows fall into different banks.
__device__ __forceinline__ void arrange_plain_rows(uint32_t a_addr, int m, int lane) {
  for (int t = 0; t < m; t += 4) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      v[u] = lds128(a_addr + static_cast<uint32_t>(t + u) * 512 + static_cast<uint32_t>(lane) * 16);
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 4; ++u)
      sts128(a_addr + static_cast<uint32_t>(t + u) * 512 + ((static_cast<uint32_t>(lane) ^ ((t + u) & 1 ? 4u : 0u)) << 4),
             in_pairs(v[u]));
  }
  fence_proxy_async_smem();  // TMA writes here next
}

// ---------------------------------------------------------------- up to 16 rows of A ------------

namespace few {

constexpr int kConsumers = 4;  // warps, 32 rows of q each
constexpr int kLoadWarp = kConsumers, kHelperWarp = kConsumers + 1;
constexpr int kThreads = 32 * (kConsumers + 2);

// Two n-tiles of 8 rows of A at most. A stage also holds, for each of its groups and rows of q, the scale as a
// float and what the zero point subtracts, ready to use. Several CTAs share an SM; the ring is as long as
// that leaves room for.
template <int kTiles, bool kPhase, int kGroup>
struct Shape {
  static constexpr int kTokens = 8 * kTiles;
  static constexpr int kCtasPerSm = w4_few_ctas();
  static constexpr int kGroups = kStageK / kGroup;  // of a stage: 2, 4 or 8
  static constexpr uint32_t kABytes = kTokens * kStageK * 2;
  static constexpr uint32_t kQStageBytes = kPhase ? kQPhaseBytes : kQBytes;
  static constexpr uint32_t kScaleBytes = kGroups * kRows * 8;
  static constexpr uint32_t kStageBytes = kQStageBytes + kABytes + kScaleBytes;
  static constexpr uint32_t kBudget = (228 / kCtasPerSm - 1) * 1024 - 1024 - 128;
  static constexpr int kStages = kBudget / kStageBytes < 4 ? static_cast<int>(kBudget / kStageBytes) : 4;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 128 + 1024;
  static_assert(kStages >= 2 && kStageBytes % 1024 == 0, "ring");
};

// d = a b (+ d)
template <bool kBf16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  const float c0 = first ? 0.0f : d[0], c1 = first ? 0.0f : d[1], c2 = first ? 0.0f : d[2], c3 = first ? 0.0f : d[3];
  if constexpr (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory"); }

template <bool kBf16, int kTiles, bool kPhase, int kGroup>
__global__ void __launch_bounds__(kThreads, Shape<kTiles, kPhase, kGroup>::kCtasPerSm)
gemm_w4_few_kernel(const __grid_constant__ QMaps<kPhase> maps_q, const __grid_constant__ CUtensorMap tmap_a, const W4 p,
                   int *status) {
  using S = Shape<kTiles, kPhase, kGroup>;
  constexpr int kChunksPerGroup = kGroup / 32;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t bar_base = smem_base + S::kStages * S::kStageBytes;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (S::kStages + s); };
  auto ready_bar = [&](uint32_t s) { return bar_base + 8u * (2 * S::kStages + s); };  // arrived, and made ready
  volatile uint32_t *abort_flag =
      reinterpret_cast<volatile uint32_t *>(smem_gen + S::kStages * S::kStageBytes + 8u * 3 * S::kStages);
  volatile uint32_t *last_flag = abort_flag + 1;
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S::kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), kConsumers);
      mbar_init(ready_bar(s), 2);
    }
    *abort_flag = 0;
    mbar_fence_init();
    if (!kPhase)
      tma_prefetch_descriptor(&maps_q.map[0]);
    tma_prefetch_descriptor(&tmap_a);
  }
  __syncthreads();

  const int cta = static_cast<int>(blockIdx.x);
  const int unit_begin = first_unit(p, cta), unit_end = first_unit(p, cta + 1);
  const int stages_k = p.stages_k;

  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loads -------------
    // TMA loads, and the scales.
    ScaleStream<kBf16, kPhase, kGroup> scales(p, unit_begin, unit_end, lane);
    uint32_t stage = 0, phase = 0;
    int block = unit_begin / stages_k, ks = unit_begin - block * stages_k;
    for (int unit = unit_begin; unit < unit_end; ++unit) {
      const bool free = mbar_wait_asleep(empty_bar(stage), phase ^ 1u, abort_flag);
      if (!__all_sync(0xffffffffu, free) || !unit_ok(p, stage, S::kStages, block, ks, status, abort_flag))
        break;
      const uint32_t at = smem_base + stage * S::kStageBytes;
      if (lane == 0) {
        mbar_arrive_expect_tx(full_bar(stage), S::kQStageBytes + static_cast<uint32_t>(p.a_box) * (kStageK * 2));
        tma_load_2d(at + S::kQStageBytes, &tmap_a, full_bar(stage), ks * kStageK, 0);
      }
      __syncwarp();
      load_q<kPhase>(maps_q, at, full_bar(stage), block, ks, lane);
      scales.advance(p, at + S::kQStageBytes + S::kABytes, lane);
      __syncwarp();
      if (lane == 0)
        mbar_arrive(ready_bar(stage));
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++ks == stages_k) {
        ks = 0;
        ++block;
      }
    }
  } else if (warp == kHelperWarp) {
    // ------------------------------------------------------------ helper ------------
    // Forms A's pairs.
    uint32_t stage = 0, phase = 0;
    for (int unit = unit_begin; unit < unit_end; ++unit) {
      const uint32_t at = smem_base + stage * S::kStageBytes;
      const bool arrived = mbar_wait(full_bar(stage), phase, abort_flag);
      if (!__all_sync(0xffffffffu, arrived))
        break;
      arrange_plain_rows(at + S::kQStageBytes, p.m, lane);
      __syncwarp();
      if (lane == 0)
        mbar_arrive(ready_bar(stage));
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else {
    // ------------------------------------------------------------ consumers ---------
    const int g = lane >> 2, q4 = lane & 3;  // fragment row (or row of A), position in the quad
    // Row g of A, of which odd rows have the halves of 128 bytes exchanged.
    const uint32_t a_lane = S::kQStageBytes + static_cast<uint32_t>(g) * 512 + static_cast<uint32_t>(q4) * 16;
    const uint32_t a_swap = (g & 1) != 0 ? 64u : 0u;
    // This lane's four rows of q, two fragments, rows g and g + 8 of each: the word of the position, its phase.
    uint32_t row_at[4], row_shift[4];
    if constexpr (kPhase) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int position = warp * 32 + i * 8 + g;
        const uint32_t shift = static_cast<uint32_t>(
            (reinterpret_cast<uintptr_t>(p.q) + static_cast<long long>(row_at_position<kPhase>(position)) * p.ldq) & 15);
        row_at[i] = static_cast<uint32_t>(position) * kPhasePitch + (shift & ~3u) + static_cast<uint32_t>(q4) * 4;
        row_shift[i] = 8 * (shift & 3u);
      }
    }
    uint32_t stage = 0, phase = 0;
    int unit = unit_begin;
    while (unit < unit_end) {
      const int block = unit / stages_k, ks_begin = unit - block * stages_k;
      const int ks_end = min(stages_k, ks_begin + (unit_end - unit));
      float total[2][kTiles][4];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            total[f][t][e] = 0.0f;
      const uint32_t q_lane = static_cast<uint32_t>(warp * 32 + g) * 128 + (static_cast<uint32_t>(g) << 4) + static_cast<uint32_t>(q4) * 4;
      const uint32_t scale_lane = S::kQStageBytes + S::kABytes + static_cast<uint32_t>(warp * 32 + g) * 8;
      for (int ks = ks_begin; ks < ks_end; ++ks) {
        // (A wait that runs out raises the abort flag: what follows then computes on whatever the ring holds,
        // in bounds, and the launch is reported as failed.)
        mbar_wait(ready_bar(stage), phase, abort_flag);
        __syncwarp();
        const uint32_t q_addr = smem_base + stage * S::kStageBytes, a_even = q_addr + a_lane + a_swap, a_odd = q_addr + a_lane + 64 - a_swap;
#pragma unroll
        for (int gi = 0; gi < S::kGroups; ++gi) {
          float scale[4];
          Zero<kBf16> zero[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint2 v = lds64(q_addr + scale_lane + static_cast<uint32_t>(gi * kRows * 8 + i * 64));
            scale[i] = __uint_as_float(v.x);
            zero[i].set_pair(v.y);
          }
          float sum[2][kTiles][4];
#pragma unroll
          for (int ci = 0; ci < kChunksPerGroup; ++ci) {
            const int chunk = gi * kChunksPerGroup + ci;  // 32 of k, 16 bytes of q
            uint4 b[kTiles];  // 8 of k of one row of A, paired as expand() pairs the weights
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
              b[t] = lds128((chunk % 2 == 0 ? a_even : a_odd) + static_cast<uint32_t>((chunk / 2) * 128 + t * 4096));
            uint32_t word[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (kPhase) {
                const uint32_t at = q_addr + row_at[i] + static_cast<uint32_t>(chunk * 16);
                word[i] = __funnelshift_r(lds32(at), lds32(at + 4), row_shift[i]);
              } else {
                word[i] = lds32(((q_addr + q_lane) ^ static_cast<uint32_t>(chunk << 4)) + static_cast<uint32_t>(i) * 1024);
              }
            }
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              uint32_t lo[4], hi[4];
              expand(word[2 * f], zero[2 * f], lo);
              expand(word[2 * f + 1], zero[2 * f + 1], hi);
              const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
              for (int t = 0; t < kTiles; ++t) {
                mma<kBf16>(sum[f][t], a0, b[t].x, b[t].y, ci == 0);
                mma<kBf16>(sum[f][t], a1, b[t].z, b[t].w, false);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float &to = total[i / 2][t][2 * (i % 2) + e];
                to = fmaf(scale[i], sum[i / 2][t][2 * (i % 2) + e], to);
              }
        }
        read_before_refill();
        if (lane == 0)
          mbar_arrive(empty_bar(stage));
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      unit += ks_end - ks_begin;

      // Lane (g, q4) holds rows g and g + 8 of its fragments and the rows 2 q4, 2 q4 + 1 of A.
      auto place = [&](int i, int t) { return (warp * 32 + i * 8 + g) * S::kTokens + t * 8 + 2 * q4; };
      bool store = true;
      if (ks_begin != 0 || ks_end != stages_k) {
        constexpr int kSlot = kRows * S::kTokens;
        const int first = owner_of(p, block * stages_k), last = owner_of(p, (block + 1) * stages_k - 1);
        if (!parts_ok(p, cta, first, last, block, status, abort_flag))
          break;  // (the same for all consumers)
        float *mine = part_slot(p, cta, first, block, kSlot);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            __stcg(reinterpret_cast<float2 *>(mine + place(i, t)),
                   make_float2(total[i / 2][t][2 * (i % 2)], total[i / 2][t][2 * (i % 2) + 1]));
        store = count_part(p, block, last - first + 1, last_flag, [] { consumers_sync(); });
        if (store) {
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                total[f][t][e] = 0.0f;
          constexpr int kAhead = 4 / kTiles;  // parts whose loads are in flight together
          for (int part = first; part <= last; part += kAhead) {
            float2 v[kAhead][4][kTiles];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
              const float *from = part_slot(p, min(part + u, last), first, block, kSlot);
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                  v[u][i][t] = __ldcg(reinterpret_cast<const float2 *>(from + place(i, t)));
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                  if (part + u <= last) {
                    total[i / 2][t][2 * (i % 2)] += v[u][i][t].x;
                    total[i / 2][t][2 * (i % 2) + 1] += v[u][i][t].y;
                  }
          }
        }
      }
      if (store) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const long long column = static_cast<long long>(block) * kRows + row_at_position<kPhase>(warp * 32 + i * 8 + g);
              const int token = t * 8 + 2 * q4 + e;
              if (token < p.m && column < p.n)
                store_c_element(p.c, token * p.ldc + column, total[i / 2][t][2 * (i % 2) + e], p.c_dtype);
            }
      }
    }
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

}  // namespace few

// ---------------------------------------------------------------- 17 to 64 rows of A ------------

namespace many {

constexpr int kHalfK = 128;    // of a stage, for each of the two sets
constexpr int kCollectors = 4;  // warps, one per quarter of the tensor-memory lanes; the first ones of the CTA
constexpr int kExpanders = 8;   // warps: 2 sets x 4 quarters
constexpr int kProducerWarp = kCollectors + kExpanders, kMmaWarp = kProducerWarp + 1, kThreads = 32 * (kMmaWarp + 2);

// What follows from the rows of A a launch is made for (kTokens = 32 or 64, also N of the instruction), the group
// and q's alignment.
template <int kTokens, bool kPhase, int kGroup>
struct Shape {
  static constexpr int kGroupsPerHalf = kHalfK / kGroup;  // 1, 2 or 4
  // Of k between two hand-overs of a set. Every hand-over costs the issuing thread a wait and a commit, about as
  // much as four instructions of this size, so a half is handed over at once where tensor memory has room for
  // the sums of all its groups (with one issuing warp, 64 x 18944 x 8192 took 49 us so and 60 us in steps of 64).
  static constexpr int kStepK = kGroupsPerHalf * kTokens <= 128 ? kHalfK : kHalfK / 2;
  static constexpr int kSteps = kHalfK / kStepK;
  static constexpr int kAccs = kStepK / kGroup;  // groups of a step, each with sums of its own
  static constexpr int kSlots = kAccs * kTokens <= 64 ? 2 : 1;  // places for sums per set
  static constexpr uint32_t kOperandColumns = kStepK / 2;       // 32-bit columns of tensor memory per operand buffer
  static constexpr uint32_t kSumsAt = 4 * kOperandColumns;      // two operand buffers per set
  static constexpr uint32_t kUsedColumns = kSumsAt + 2 * kSlots * kAccs * kTokens;
  static constexpr uint32_t kTmemColumns = kUsedColumns <= 256 ? 256 : 512;
  static_assert(kUsedColumns <= 512, "tensor memory");
  static constexpr uint32_t kABoxBytes = kTokens * 128;    // 64 of k x kTokens rows of A
  static constexpr uint32_t kABytes = (kStageK / 64) * kABoxBytes;
  static constexpr uint32_t kQStageBytes = kPhase ? kQPhaseBytes : kQBytes;
  static constexpr uint32_t kStageBytes = kQStageBytes + kABytes;
  static constexpr int kStages = 192 * 1024 / kStageBytes < 6 ? static_cast<int>(192 * 1024 / kStageBytes) : 6;
  // Behind the ring: barriers, then a block's sums on their way to C.
  static constexpr uint32_t kTileBytes = kRows * kTokens * 4;
  static constexpr uint32_t kSmemBytes = kStages * kStageBytes + 256 + kTileBytes + 1024;
  static_assert(kStages >= 3 && kSmemBytes <= 227 * 1024, "shared memory of a CTA");
  static_assert(kStageBytes % 1024 == 0 && kQStageBytes % 1024 == 0, "swizzled boxes are 1 KiB aligned");
};

// Four columns of a row of C, as far as there are.
__device__ __forceinline__ void store_four(const W4 &p, int row, long long column, const float4 &v) {
  const long long at = row * p.ldc + column;
  if (column + 3 < p.n && p.c_vector != 0) {
    if (p.c_dtype == kCTypeF32)
      *reinterpret_cast<float4 *>(static_cast<float *>(p.c) + at) = v;
    else
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.c) + at) =
          make_uint2(pack_pair(v.x, v.y, p.c_dtype), pack_pair(v.z, v.w, p.c_dtype));
    return;
  }
  const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (column + i < p.n)
      store_c_element(p.c, at + i, e[i], p.c_dtype);
}

__device__ __forceinline__ void collectors_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kCollectors) : "memory"); }

template <bool kBf16, int kTokens, bool kPhase, int kGroup>
__global__ void __launch_bounds__(kThreads, 1)
gemm_w4_kernel(const __grid_constant__ QMaps<kPhase> maps_q, const __grid_constant__ CUtensorMap tmap_a, const W4 p,
               uint32_t idesc, int *status) {
  using S = Shape<kTokens, kPhase, kGroup>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t smem_base = (raw_addr + 1023u) & ~1023u;
  uint8_t *smem_gen = smem_raw + (smem_base - raw_addr);
  const uint32_t bar_base = smem_base + S::kStages * S::kStageBytes;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };                    // q and A have arrived
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (S::kStages + s); };    // both have been read
  auto operand_bar = [&](uint32_t set, uint32_t b) { return bar_base + 8u * (2 * S::kStages + 2 * set + b); };  // expanded
  // A step's products are done: its operand buffer is free, its sums are there.
  auto done_bar = [&](uint32_t set, uint32_t b) { return bar_base + 8u * (2 * S::kStages + 4 + 2 * set + b); };
  constexpr uint32_t kMiscOff = S::kStages * S::kStageBytes + 8u * (2 * S::kStages + 8);
  static_assert(8 * (2 * S::kStages + 8) + 12 <= 256, "barriers");
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem_gen + kMiscOff);
  volatile uint32_t *last_flag = abort_flag + 1;
  volatile uint32_t *tmem_slot = abort_flag + 2;
  const int warp = static_cast<int>(threadIdx.x >> 5), lane = static_cast<int>(threadIdx.x & 31);
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S::kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), kExpanders + kCollectors);  // q has been read, and A (the products are done)
    }
    for (uint32_t i = 0; i < 4; ++i) {
      mbar_init(operand_bar(i >> 1, i & 1), kExpanders / 2 + kCollectors);  // expanded, and its place for sums is free
      mbar_init(done_bar(i >> 1, i & 1), 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
    if (!kPhase)
      tma_prefetch_descriptor(&maps_q.map[0]);
    tma_prefetch_descriptor(&tmap_a);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), S::kTmemColumns);
    tmem_relinquish_alloc_permit();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  const int cta = static_cast<int>(blockIdx.x);
  const int unit_begin = first_unit(p, cta), unit_end = first_unit(p, cta + 1);
  const int stages_k = p.stages_k;

  if (warp == kProducerWarp) {
    // ------------------------------------------------------------ producer ----------
    uint32_t stage = 0, phase = 0;
    int block = unit_begin / stages_k, ks = unit_begin - block * stages_k;
    for (int unit = unit_begin; unit < unit_end; ++unit) {
      const bool free = mbar_wait_asleep(empty_bar(stage), phase ^ 1u, abort_flag);
      if (!__all_sync(0xffffffffu, free) || !unit_ok(p, stage, S::kStages, block, ks, status, abort_flag))
        break;
      const uint32_t q_dst = smem_base + stage * S::kStageBytes, a_dst = q_dst + S::kQStageBytes;
      if (lane == 0) {
        mbar_arrive_expect_tx(full_bar(stage), S::kQStageBytes + static_cast<uint32_t>(p.a_box) * (kStageK * 2));
#pragma unroll
        for (int j = 0; j < kStageK / 64; ++j)
          tma_load_2d(a_dst + j * S::kABoxBytes, &tmap_a, full_bar(stage), ks * kStageK + j * 64, 0);
      }
      __syncwarp();
      load_q<kPhase>(maps_q, q_dst, full_bar(stage), block, ks, lane);
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++ks == stages_k) {
        ks = 0;
        ++block;
      }
    }
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    const uint32_t set = static_cast<uint32_t>(warp - kMmaWarp);
    // ------------------------------------------------------------ MMA issuer --------
    // The whole warp walks along, so that the instructions' operands are known to be uniform; one lane issues.
    uint32_t stage = 0, step = 0;  // step: of a set, counted from the start
    bool ok = true;
    for (int unit = unit_begin; ok && unit < unit_end; ++unit) {
      const uint32_t a_addr = smem_base + stage * S::kStageBytes + S::kQStageBytes;
#pragma unroll
      for (uint32_t part = 0; part < S::kSteps; ++part, ++step) {
        const uint32_t buffer = step & 1u, slot = S::kSlots == 2 ? buffer : 0u;
        // (The expanding warps have waited for the stage, A included.)
        const bool ready = mbar_wait(operand_bar(set, buffer), (step >> 1) & 1u, abort_flag);
        ok = __all_sync(0xffffffffu, ready);
        if (!ok)
          break;
        tcgen05_fence_after_sync();
        const uint32_t sums = tmem_base + S::kSumsAt + (set * S::kSlots + slot) * (S::kAccs * kTokens);
        const uint32_t operand = tmem_base + (2 * set + buffer) * S::kOperandColumns;
        // 64 of k are one box of A.
        const uint64_t desc = make_smem_desc_sw128(a_addr + (set * kHalfK + part * S::kStepK) / 64 * S::kABoxBytes, 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (uint32_t kk = 0; kk < S::kStepK / 16; ++kk)
            umma_f16_ts(sums + (kk * 16 / kGroup) * kTokens, operand + kk * 8,
                        desc + (kk / 4) * (S::kABoxBytes >> 4) + (kk % 4) * 2, idesc, (kk * 16) % kGroup == 0 ? 0u : 1u);
          umma_commit(done_bar(set, buffer));
        }
        __syncwarp();
      }
      if (++stage == S::kStages)
        stage = 0;
    }
  } else if (warp >= kCollectors) {
    // ------------------------------------------------------------ expanding warps ---
    const uint32_t set = static_cast<uint32_t>(warp - kCollectors) >> 2;
    const int position = (warp & 3) * 32 + lane;  // in the block, and this lane's tensor-memory lane
    const int local = row_at_position<kPhase>(position);
    const uint32_t operands = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 2 * set * S::kOperandColumns;
    uint32_t stage = 0, phase = 0, step = 0;  // step: of this set, counted from the start
    bool ok = true;
    uint32_t row_at = static_cast<uint32_t>(position) * 128, row_shift = 0;
    if constexpr (kPhase) {
      const uint32_t at = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(p.q) + static_cast<long long>(local) * p.ldq) & 15);
      row_at = static_cast<uint32_t>(position) * kPhasePitch + set * 64 + (at & ~3u);
      row_shift = 8 * (at & 3u);
    }
    // Zero points of this stage and the next two, a byte per group. (Rows past the end take the last row's; what
    // becomes of them is not stored.)
    uint32_t raw[2] = {0x08080808u, 0x08080808u};
    auto fetch = [&](int unit, uint32_t &into) {
      if (p.zeros == nullptr || unit >= unit_end)
        return;
      const int at_block = unit / stages_k, at_ks = unit - at_block * stages_k;
      const long long row = min(static_cast<long long>(at_block) * kRows + local, static_cast<long long>(p.n) - 1);
      const uint8_t *const zeros = p.zeros + row * p.ldz;
      const int first = (at_ks * 2 + static_cast<int>(set)) * S::kGroupsPerHalf;
      into = 0u;
#pragma unroll
      for (int j = 0; j < S::kGroupsPerHalf; ++j)  // (p.span: how many of the kernel's groups share a scale)
        into |= static_cast<uint32_t>(zeros[min(p.span == 1 ? first + j : (first + j) / p.span, p.groups - 1)]) << (8 * j);
    };
    fetch(unit_begin, raw[0]);
    fetch(unit_begin + 1, raw[1]);
    for (int unit = unit_begin; ok && unit < unit_end; ++unit) {
      Zero<kBf16> zero[S::kGroupsPerHalf];
#pragma unroll
      for (int j = 0; j < S::kGroupsPerHalf; ++j)
        zero[j].set(static_cast<int>((raw[0] >> (8 * j)) & kZeroBits));
      raw[0] = raw[1];
      fetch(unit + 2, raw[1]);
      const bool ready = mbar_wait(full_bar(stage), phase, abort_flag);
      if (!__all_sync(0xffffffffu, ready))
        break;
      const uint32_t q_addr = smem_base + stage * S::kStageBytes + row_at;
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 64 of k at a time
        const uint32_t buffer = step & 1u;
        uint32_t w[8], r[32];
        if constexpr (kPhase) {
          uint32_t low = lds32(q_addr + half * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t high = lds32(q_addr + half * 32 + i * 4 + 4);
            w[i] = __funnelshift_r(low, high, row_shift);
            low = high;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t piece = set * 4 + static_cast<uint32_t>(2 * half + i);
            const uint4 v = lds128(q_addr + ((piece ^ (static_cast<uint32_t>(lane) & 7u)) << 4));
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          expand_in_order(w[i], zero[(half * 8 + i) * 8 / kGroup], r + 4 * i);
        if (half == 1) {
          read_before_refill();
          if (lane == 0)
            mbar_arrive(empty_bar(stage));  // this warp's rows of q have been read
        }
        if ((S::kSteps == 2 || half == 0) && step >= 2) {  // the step that had this buffer must be done
          const bool done = mbar_wait(done_bar(set, buffer), ((step >> 1) & 1u) ^ 1u, abort_flag);
          if (!__all_sync(0xffffffffu, done)) {
            ok = false;
            break;
          }
          tcgen05_fence_after_sync();
        }
        tmem_store_x32(operands + buffer * S::kOperandColumns + (S::kSteps == 1 ? half * 32 : 0), r);
        if (S::kSteps == 2 || half == 1) {
          tmem_store_wait();
          tcgen05_fence_before_sync();
          __syncwarp();
          if (lane == 0)
            mbar_arrive(operand_bar(set, buffer));
          ++step;
        }
      }
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else {
    // ------------------------------------------------------------ collecting warps --
    const int local = row_at_position<kPhase>(warp * 32 + lane);  // this lane's row of the block, i.e. column of C
    const uint32_t sums = tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + S::kSumsAt;
    constexpr int kGroups = kStageK / kGroup;  // of a stage: 2, 4 or 8
    uint32_t stage = 0, step = 0;
    bool ok = true;  // (a wait that ran out: the barriers below are still met)
    int unit = unit_begin;
    // Scales of this stage and the next two, two to a word. (A sector of them that is not in the cache yet takes
    // longer to arrive than a stage takes to expand. Rows past the end take the last row's.)
    uint32_t raw[2][kGroups / 2];
    auto fetch = [&](int at_unit, uint32_t (&into)[kGroups / 2]) {
      if (at_unit >= unit_end)
        return;
      const int at_block = at_unit / stages_k, first = (at_unit - at_block * stages_k) * kGroups;
      const long long row = min(static_cast<long long>(at_block) * kRows + local, static_cast<long long>(p.n) - 1);
      const uint16_t *const scales = p.scales + row * p.lds;
      if (p.vector_scales) {
        load_words(scales + first, into);
      } else {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          const uint32_t v = scales[min(p.span == 1 ? first + j : (first + j) / p.span, p.groups - 1)];
          into[j / 2] = j % 2 == 0 ? v : into[j / 2] | v << 16;
        }
      }
    };
    fetch(unit_begin, raw[0]);
    fetch(unit_begin + 1, raw[1]);
    if (lane == 0)
      for (uint32_t i = 0; i < 2 * S::kSlots; ++i)  // at first every place is free
        mbar_arrive(operand_bar(i & 1u, i >> 1));
    while (unit < unit_end) {
      const int block = unit / stages_k, ks_begin = unit - block * stages_k;
      const int ks_end = min(stages_k, ks_begin + (unit_end - unit));
      float total[kTokens];
#pragma unroll
      for (int t = 0; t < kTokens; ++t)
        total[t] = 0.0f;
      for (int ks = ks_begin; ok && ks < ks_end; ++ks) {
        uint32_t now[kGroups / 2];
#pragma unroll
        for (int j = 0; j < kGroups / 2; ++j) {
          now[j] = raw[0][j];
          raw[0][j] = raw[1][j];
        }
        fetch(unit + (ks - ks_begin) + 2, raw[1]);
#pragma unroll
        for (int part = 0; part < S::kSteps; ++part, ++step) {
          const uint32_t buffer = step & 1u, slot = S::kSlots == 2 ? buffer : 0u;
#pragma unroll
          for (uint32_t set = 0; set < 2; ++set) {
            const bool done = mbar_wait(done_bar(set, buffer), (step >> 1) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, done))
              ok = false;
            tcgen05_fence_after_sync();
#pragma unroll
            for (int j = 0; j < S::kAccs; ++j) {
              const int group = static_cast<int>(set) * (kGroups / 2) + part * S::kAccs + j;
              const float scale = scale_value<kBf16>(
                  static_cast<uint16_t>(group % 2 == 0 ? now[group / 2] & 0xffffu : now[group / 2] >> 16));
              const uint32_t at = sums + ((set * S::kSlots + slot) * S::kAccs + j) * kTokens;
#pragma unroll
              for (int t0 = 0; t0 < kTokens; t0 += 32) {
                uint32_t r[32];
                tmem_load_32x32b_x32(at + t0, r);
                tmem_load_wait_for(r);
#pragma unroll
                for (int t = 0; t < 32; ++t)
                  total[t0 + t] = fmaf(scale, __uint_as_float(r[t]), total[t0 + t]);
              }
            }
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0)  // the step that will fill this place next has it
              mbar_arrive(operand_bar(set, (step + S::kSlots) & 1u));
          }
        }
        if (lane == 0)
          mbar_arrive(empty_bar(stage));  // all products with this stage of A are done
        if (++stage == S::kStages)
          stage = 0;
      }
      unit += ks_end - ks_begin;

      // The sums, one token's 128 columns after another's: into shared memory where the block is all this CTA's,
      // else into its slot, from which the last of the CTAs that share it adds them up. Then warps take tokens and
      // lanes four columns each. (This code runs once per block, mostly from a cold instruction cache: it is
      // short, and all rows are kept, those past m being zeros.)
      constexpr int kSlot = kRows * kTokens;
      float *const tile = reinterpret_cast<float *>(smem_gen + S::kStages * S::kStageBytes + 256);
      const bool whole = ks_begin == 0 && ks_end == stages_k;
      int first = cta, last = cta;
      if (whole) {
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
          tile[t * kRows + local] = total[t];
        collectors_sync();
      } else {
        first = owner_of(p, block * stages_k);
        last = owner_of(p, (block + 1) * stages_k - 1);
        if (!parts_ok(p, cta, first, last, block, status, abort_flag))
          break;  // (the same for all collectors)
        float *const mine = part_slot(p, cta, first, block, kSlot) + local;
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
          __stcg(mine + t * kRows, total[t]);
        if (!count_part(p, block, last - first + 1, last_flag, [] { collectors_sync(); }))
          continue;
      }
      const long long column = static_cast<long long>(block) * kRows + 4 * lane;
      constexpr int kAtOnce = 4;  // tokens of a warp, and parts, whose loads are in flight together
#pragma unroll 1
      for (int t0 = warp; t0 < p.m; t0 += kCollectors * kAtOnce) {
        float4 sum[kAtOnce];
        if (whole) {
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u)
            sum[u] = *reinterpret_cast<const float4 *>(tile + min(t0 + u * kCollectors, kTokens - 1) * kRows + 4 * lane);
        } else {
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u)
            sum[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
          for (int part = first; part <= last; part += kAtOnce) {
            float4 v[kAtOnce][kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
              const float *const from = part_slot(p, min(part + i, last), first, block, kSlot) + 4 * lane;
#pragma unroll
              for (int u = 0; u < kAtOnce; ++u)
                v[i][u] = __ldcg(reinterpret_cast<const float4 *>(from + min(t0 + u * kCollectors, kTokens - 1) * kRows));
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
              if (part + i <= last)
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                  sum[u].x += v[i][u].x;
                  sum[u].y += v[i][u].y;
                  sum[u].z += v[i][u].z;
                  sum[u].w += v[i][u].w;
                }
          }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
          if (t0 + u * kCollectors < p.m)
            store_four(p, t0 + u * kCollectors, column, sum[u]);
      }
      if (whole)
        collectors_sync();  // `tile` is free again
    }
  }

  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  if (*abort_flag != 0) {
    if (threadIdx.x == 0)
      atomicCAS(status, 0, kStatusDeviceWaitTimeout);
    const long long start = clock64();
    while (clock64() - start < 2000000LL) {
    }
    __syncthreads();
  }
  if (warp == kMmaWarp)
    tmem_dealloc(tmem_base, S::kTmemColumns);
}

}  // namespace many

// ---------------------------------------------------------------- launch ------------------------

template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, uint32_t bytes, int *configured_device) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess && *configured_device != device) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (err == cudaSuccess)
      *configured_device = device;
  }
  return err;
}

template <bool kBf16, int kTokens, bool kPhase, int kGroup>
cudaError_t launch(const CUtensorMap *tmap_q, const CUtensorMap &tmap_a, const W4 &p, int *status, cudaStream_t stream) {
  static thread_local int configured_device = -1;
  QMaps<kPhase> maps;
  for (int i = 0; i < (kPhase ? kPhases : 1); ++i)
    maps.map[i] = tmap_q[i];
  if constexpr (kTokens <= 16) {
    using S = few::Shape<kTokens / 8, kPhase, kGroup>;
    auto kernel = few::gemm_w4_few_kernel<kBf16, kTokens / 8, kPhase, kGroup>;
    const cudaError_t err = allow_shared(kernel, S::kSmemBytes, &configured_device);
    if (err != cudaSuccess)
      return err;
    kernel<<<static_cast<unsigned>(p.grid), few::kThreads, S::kSmemBytes, stream>>>(maps, tmap_a, p, status);
  } else {
    using S = many::Shape<kTokens, kPhase, kGroup>;
    auto kernel = many::gemm_w4_kernel<kBf16, kTokens, kPhase, kGroup>;
    const cudaError_t err = allow_shared(kernel, S::kSmemBytes, &configured_device);
    if (err != cudaSuccess)
      return err;
    const uint32_t idesc = make_idesc_f16(kBf16 ? 1u : 0u, false, false, kRows, kTokens);
    kernel<<<static_cast<unsigned>(p.grid), many::kThreads, S::kSmemBytes, stream>>>(maps, tmap_a, p, idesc, status);
  }
  return cudaGetLastError();
}

template <bool kBf16>
cudaError_t launch_w4(const CUtensorMap *tmap_q, const CUtensorMap &tmap_a, const W4 &p, int *status, cudaStream_t stream) {
  const int tokens = w4_tokens(p.m);
  const bool phase = p.phase != 0;
#define HC_W4(TOKENS, GROUP)                                                               \
  return phase ? launch<kBf16, TOKENS, true, GROUP>(tmap_q, tmap_a, p, status, stream)     \
               : launch<kBf16, TOKENS, false, GROUP>(tmap_q, tmap_a, p, status, stream)
#define HC_W4_GROUPS(TOKENS) \
  {                          \
    if (p.group == 32)       \
      HC_W4(TOKENS, 32);     \
    if (p.group == 64)       \
      HC_W4(TOKENS, 64);     \
    HC_W4(TOKENS, 128);      \
  }
  if (tokens == 8)
    HC_W4_GROUPS(8)
  if (tokens == 16)
    HC_W4_GROUPS(16)
  if (tokens == 32)
    HC_W4_GROUPS(32)
  HC_W4_GROUPS(64)
#undef HC_W4_GROUPS
#undef HC_W4
}

}  // namespace w4
}  // namespace sm100
}  // namespace hc

// Expert products with 4-bit weights and group scales:
//   out[r, n] = sum_k x[r, k] * code[e, n, k] * scale[e, n, k / group],
// codes -8 .. 7, rows r of expert e, f32 accumulation.
//
// Weights as they lie in memory ("laid out"): codes + 8, two per byte, in the
// order in which a warp's MMA operands want them. Block (i, b) holds rows
// 16 i .. 16 i + 15 and columns 64 b .. 64 b + 63 as 32 lanes x 16 bytes: lane
// 4 g + q has rows g and g + 8 and, of each 32 columns, columns 8 q .. 8 q + 7.
// Word 2 j + s of its four is MMA step s of columns 32 j .. 32 j + 31; nibble
// (row half h, pair p) of its half-word c is column 8 q + 4 s + 2 p + c. So one
// 16-byte load gives four m16n8k16 A operands and one 16-byte load of x two B
// operands; the MMA's own column order is permuted on both sides alike.
// Scales lie as (E, N/16, K/group, 16), in f32, bf16 or f16. Rows and columns
// beyond N and K are codes 8 (value 0).
//
// Codes become 16-bit floats exactly (a mask, an exponent and a subtraction),
// a 64-column block (32 for groups of 32) is summed by the tensor cores in
// f32 and then multiplied by its f32 scale: no weight is rounded.
//
// int4_kernel, here: a few rows per expert, warp-level MMAs. int4_tile_kernel,
// int4_tile.cuh: more rows, tcgen05. Most rows, unless the caller wants exact
// weights: they become 16-bit tiles in a workspace (dequant_kernel, one
// rounding of code * scale to the activation type, which the MMA then takes as
// it takes 16-bit weights) for the 16-bit tcgen05 kernels.
#pragma once
#include "gemm_warp.cuh"
#include "norm.cuh"

namespace moe {
namespace int4 {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kBlockBytes = 512;    // 16 rows x 64 columns
constexpr int kMaxE = 256;
constexpr int kMaxStages = 6;
constexpr int kRanges = 8;          // K is summed as eight ranges of blocks, whatever the kernel's shape

struct Params {
  const uint8_t* data0;  // laid out codes; data1: the up projection (SwiGLU)
  const uint8_t* data1;
  const uint8_t* scale0;
  const uint8_t* scale1;
  const uint16_t* x;
  const int32_t* offsets;
  uint16_t* out;
  int32_t* status;
  int64_t ldo;
  int M, N, K, E;
  int n16, kb, groups;  // tiles of 16 rows, blocks of 64 columns, scale groups
  int group_shift;      // log2 of the group size
  int scale_dt, scale_shift;  // scale_shift: log2 of a scale's bytes
  int chunk;            // blocks in a stage
  int scale_slot;       // bytes of a tile's scales in a stage
  int f32_slot;         // bytes of a tile's f32 scales of a stage (behind the ring: their copy for 16-bit scales)
  int stage_bytes, stages;  // of one warp's ring
};

__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
  return r;
}

// The A operand of one MMA step from its word of eight codes u = code + 8,
// exactly: a nibble put into the mantissa of 2^m is the float 2^m + u, from which
// 2^m + 8 is subtracted (published for integer weights by Kim, Henry, Fahim and
// Awadalla, "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into
// Cloud Scale Production", 2022). m = 10 and 7 are the mantissas' lengths, so the
// mantissa's last bit counts 1; f16's longer one also takes the nibble 4 bits higher.
template <bool kF16>
__device__ __forceinline__ void codes_to_a(uint32_t w, uint32_t (&a)[4]) {
  if (kF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = i ? w >> 8 : w;
      const uint32_t lo = and_or(v, 0x000F000Fu, 0x64006400u);  // 1024 + u
      const uint32_t hi = and_or(v, 0x00F000F0u, 0x64006400u);  // 1024 + 16 u
      asm("sub.f16x2 %0, %1, %2;" : "=r"(a[2 * i]) : "r"(lo), "r"(0x64086408u));  // - 1032
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(a[2 * i + 1]) : "r"(hi), "r"(0x2C002C00u), "r"(0xD480D480u));  // / 16 - 72
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = and_or(i ? w >> (4 * i) : w, 0x000F000Fu, 0x43004300u);  // 128 + u
      asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(a[i]) : "r"(v), "r"(0x43084308u));  // - 136
    }
  }
}

// D = A B + D, with a zero D at first. Not volatile: the compiler may interleave
// the chains of several tiles and blocks.
template <bool kF16, bool kFirst>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const float c0 = kFirst ? 0.f : d[0], c1 = kFirst ? 0.f : d[1], c2 = kFirst ? 0.f : d[2], c3 = kFirst ? 0.f : d[3];
  if (kF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
}

struct Ctrl {
  uint64_t full[kWarps][kMaxStages];
  int abort;
  int experts;           // experts with rows
  int units;             // units of the launch (0 if the offsets are bad)
  int expert[kMaxE];     // their ids
  int first[kMaxE + 1];  // units before expert i
  int off[kMaxE + 1];
};
constexpr uint32_t kCtrlBytes = (sizeof(Ctrl) + 127) & ~uint32_t(127);

// Sums that wait in shared memory: kMt weight tiles x kNt token tiles of each warp.
template <int kMt, int kNt, bool kSplit>
struct Sums {
  static constexpr uint32_t kBytes = kWarps * kMt * kNt * 4 * 32 * 4;
  static constexpr uint32_t kBuffers = kSplit ? 2 : 1;  // read by other warps while the next unit's are made
  static constexpr uint32_t kFixed = kCtrlBytes + kBuffers * kBytes;
};

// Resident CTAs per SM that the kernel is built for.
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }

// Where a unit lies.
struct Unit {
  int e, row0, rows, tile0;  // expert, first row, rows (<= 8 kNt), first 16-row tile of the output
};

// A unit is kMt weight tiles (SwiGLU: half of them gate, half up rows) x one
// token tile of 8 kNt rows of one expert, over all of K. A CTA takes a
// contiguous run of units; consecutive units walk an expert's token tiles,
// then its weight tiles, so a CTA's warps find their rows of x in L1.
//
// Each warp streams weights for itself: its lane 0 brings `chunk` blocks of
// codes and their scales per stage of the warp's own ring by bulk copies, and
// nothing but the warp waits for them. kSplit false: a warp takes whole units,
// and no warp ever waits for another. kSplit true (few units: one or two
// decoded tokens): the eight warps share a unit, each one of the eight ranges
// that K's blocks are split into. The ranges' sums are joined in order,
// ((r0 + r1) + r2) + ..., in both forms, so a row's result depends neither on
// the form nor on the tile sizes nor on the other rows.
//
// Per 256 weights one MMA per token tile and 9 (f16) or 11 (bf16) instructions
// that make its operand. Bound by latency rather than by a pipe: 44 to 61% of
// the issue slots are used and 10 to 32% of HBM's peak, with 5 to 9 warps per
// scheduler that wait for x's loads, the operands' chain and, split, each other.
// 64 experts of 1408 x 2048 with groups of 128: one token (6 experts) 7 us, 16
// tokens 36 us, 93 tokens 59 us; f16 2048 x 1408 with 16 tokens 28 us (50 busy
// experts, 2.7 TB/s; an earlier build's copies alone took 21 us). The SwiGLU pair
// for a few rows keeps 80 registers a thread for three CTAs per SM and spills
// 136 to 228 bytes: gate and up of 1408 x 2048 for 98 rows of 49 experts 70 us.
template <int kMt, int kNt, bool kSplit, bool kSwiglu, bool kF16, bool kG32>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(kNt)) int4_kernel(const __grid_constant__ Params p) {
  constexpr int kOutMt = kSwiglu ? kMt / 2 : kMt;  // output tiles of a unit
  constexpr int kTok = 8 * kNt;
  using S = Sums<kMt, kNt, kSplit>;
  extern __shared__ __align__(128) uint8_t int4_smem[];
  Ctrl& c = *reinterpret_cast<Ctrl*>(int4_smem);
  float* sums = reinterpret_cast<float*>(int4_smem + kCtrlBytes);
  uint8_t* rings = int4_smem + kCtrlBytes + S::kBuffers * S::kBytes;
  volatile int* abort_flag = &c.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_trigger();
  if (tid < kWarps) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&c.full[tid][i], 1);
    if (tid == 0) c.abort = 0;
    fence_mbar_init();
  }
  pdl_wait();  // before the first global memory access
  for (int g = tid; g <= p.E; g += kThreads) c.off[g] = p.offsets[g];
  __syncthreads();
  const int tile_units = (p.n16 + kOutMt - 1) / kOutMt;
  if (warp == 0) {
    // the experts with rows and the units before each
    int n = 0, units = 0;
    bool bad = lane == 0 && (c.off[0] < 0 || c.off[p.E] > p.M);
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int rows = e < p.E ? c.off[e + 1] - c.off[e] : 0;
      bad |= rows < 0;
      const uint32_t has = __ballot_sync(0xffffffffu, rows > 0);
      const int u = rows > 0 ? (rows + kTok - 1) / kTok * tile_units : 0;
      int v = u;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
      }
      if (rows > 0) {
        const int i = n + __popc(has & ((1u << lane) - 1u));
        c.expert[i] = e;
        c.first[i] = units + v - u;
      }
      n += __popc(has);
      units += __shfl_sync(0xffffffffu, v, 31);
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      c.first[n] = units;
      c.experts = n;
      c.units = bad ? 0 : units;
      if (bad && p.status) atomicCAS(p.status, 0, MOE_ERR_BAD_OFFSETS);
    }
  }
  __syncthreads();
  const int u1 = static_cast<int>(static_cast<int64_t>(c.units) * (blockIdx.x + 1) / gridDim.x);
  constexpr int kStep = kSplit ? 1 : kWarps;
  const int u0 = static_cast<int>(static_cast<int64_t>(c.units) * blockIdx.x / gridDim.x) + (kSplit ? 0 : warp);
  if (u0 >= u1) return;  // the whole warp, or (kSplit) the whole CTA
  int at0 = 0;  // index of the first unit's expert
  {
    int hi = c.experts - 1;
    while (at0 < hi) {
      const int mid = (at0 + hi + 1) / 2;
      if (c.first[mid] <= u0) at0 = mid; else hi = mid - 1;
    }
  }
  // unit u, at or after the last one located with `at`
  auto locate = [&](int u, int& at) {
    while (u >= c.first[at + 1]) ++at;
    Unit r;
    r.e = c.expert[at];
    const int begin = c.off[r.e], rows = c.off[r.e + 1] - begin;
    int tile = u - c.first[at], tok = 0;
    if (rows > kTok) {
      const int tok_tiles = (rows + kTok - 1) / kTok;
      tok = tile % tok_tiles;
      tile /= tok_tiles;
    }
    r.row0 = begin + tok * kTok;
    r.rows = min(kTok, rows - tok * kTok);
    r.tile0 = tile * kOutMt;
    return r;
  };
  // this warp's blocks
  const int range = (p.kb + kRanges - 1) / kRanges;
  const int lo = kSplit ? min(p.kb, warp * range) : 0, hi = kSplit ? min(p.kb, lo + range) : p.kb;

  // ---------------------------------------------------------------- bulk copies (lane 0)
  uint8_t* ring = rings + warp * (p.stages * p.stage_bytes + kMt * p.f32_slot);
  float* f32_scales = reinterpret_cast<float*>(ring + p.stages * p.stage_bytes);
  int pu = u0, pb = lo, pat = at0;  // the next stage to bring: unit, first block
  uint32_t pstage = 0;
  int ptile = 0;            // first tile of the unit among all experts' ...
  int ptiles = 0;           // ... and its tiles
  auto place = [&]() {
    const Unit r = locate(pu, pat);
    ptile = r.e * p.n16 + r.tile0;
    ptiles = min(kOutMt, p.n16 - r.tile0);
  };
  place();
  if (lo == hi) pu = u1;  // K of fewer than eight blocks: nothing for this warp
  auto issue = [&]() {
    const int nb = min(p.chunk, hi - pb);
    if (lane == 0) {
      uint64_t* bar = &c.full[warp][pstage];
      uint8_t* stage = ring + pstage * p.stage_bytes;
      const int g0 = (pb * 64) >> p.group_shift;
      const int ng = min(((pb + nb) * 64 - 1) >> p.group_shift, p.groups - 1) - g0 + 1;
      const uint32_t data_bytes = nb * kBlockBytes, scale_bytes = static_cast<uint32_t>(ng * 16) << p.scale_shift;
      mbar_arrive_expect_tx(bar, (data_bytes + scale_bytes) * ptiles * (kSwiglu ? 2 : 1));
#pragma unroll
      for (int m = 0; m < kMt; ++m) {
        const bool up = kSwiglu && m >= kOutMt;
        const int t = up ? m - kOutMt : m;
        if (kOutMt > 1 && t >= ptiles) continue;
        bulk_load(stage + m * p.chunk * kBlockBytes,
                  (up ? p.data1 : p.data0) + (static_cast<int64_t>(ptile + t) * p.kb + pb) * kBlockBytes, data_bytes,
                  bar);
        bulk_load(stage + kMt * p.chunk * kBlockBytes + m * p.scale_slot,
                  (up ? p.scale1 : p.scale0) +
                      ((static_cast<int64_t>(ptile + t) * p.groups + g0) << (4 + p.scale_shift)),
                  scale_bytes, bar);
      }
    }
    if (++pstage == static_cast<uint32_t>(p.stages)) pstage = 0;
    pb += nb;
    if (pb == hi) {
      pb = lo;
      pu += kStep;
      if (pu < u1) place();
    }
  };
  for (int i = 0; i < p.stages && pu < u1; ++i) issue();

  // ---------------------------------------------------------------- products
  const int g = lane >> 2, q = lane & 3;
  const int full_blocks = p.K / 64;  // blocks without columns past K
  uint32_t stage = 0, phase = 0;
  int buf = 0, at = at0;
  bool ok = true;
  for (int u = u0; u < u1; u += kStep) {
    const Unit r = locate(u, at);
    // this lane's pieces of its tokens' rows (token 8 j + g; past the unit's
    // rows another of its rows, whose sums are not stored)
    const uint4* xp[kNt];
#pragma unroll
    for (int j = 0; j < kNt; ++j)
      xp[j] = reinterpret_cast<const uint4*>(
          p.x + static_cast<int64_t>(r.row0 + min(8 * j + g, r.rows - 1)) * p.K + 64 * lo + 8 * q);
    // Two sets of x values, loaded a block ahead, where the registers allow; else one.
    constexpr int kSets = kNt == 1 ? 2 : 1;
    uint4 xv[kSets][kNt][2];
    auto load_x = [&](uint4 (&v)[2], int j) {  // whole blocks; and on to the next
      v[0] = xp[j][0];
      v[1] = xp[j][4];
      xp[j] += 8;
    };
    float part[kMt][kNt][4];
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[m][j][e] = 0.f;
    // The sums of the ranges so far (kSplit false): in registers where they are few, else in shared memory.
    constexpr bool kTotRegs = kMt * kNt <= 2;
    float tot[kTotRegs ? kMt : 1][kTotRegs ? kNt : 1][4];
    float* mine = sums + buf * (S::kBytes / 4) + warp * kMt * kNt * 4 * 32 + lane;
    int boundary = range;  // the end of the range being summed
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (kTotRegs) tot[kTotRegs ? m : 0][kTotRegs ? j : 0][e] = 0.f;
          else mine[((m * kNt + j) * 4 + e) * 32] = 0.f;
        }
    const uint4* codes_at = nullptr;   // of the stage: this lane's codes of its first block ...
    const float* scales_at = nullptr;  // ... and the f32 scales of its first row
    int b0 = lo, g0 = 0;
    // block b of the stage, with the x values v; loads the set `to` of block b + 1 of kSets 1
    auto product = [&](int b, uint4 (&v)[kNt][2], bool more) {
      constexpr int kParts = kG32 ? 2 : 1;  // scaled sums per block
#pragma unroll
      for (int m = 0; m < kMt; ++m) {
        // tiles past N were not copied: their sums are not stored
        const uint4 codes = codes_at[(m * p.chunk + b - b0) * (kBlockBytes / 16)];
        const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
        float sc[kParts][2];
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          // (of a half block past the last group, what lies there: its sum is 0 and is left out)
          const float* at_group = scales_at + m * (p.f32_slot / 4) + (((64 * b + 32 * h) >> p.group_shift) - g0) * 16;
          sc[h][0] = at_group[0];
          sc[h][1] = at_group[8];
        }
        uint32_t a[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) codes_to_a<kF16>(word[i], a[i]);
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
          if (kNt > 1 && 8 * j >= r.rows) continue;
#pragma unroll
          for (int h = 0; h < kParts; ++h) {
            float d[4];
#pragma unroll
            for (int i = 4 / kParts * h; i < 4 / kParts * (h + 1); ++i) {
              const uint4& w = v[j][i / 2];
              const uint32_t x0 = i % 2 ? w.z : w.x, x1 = i % 2 ? w.w : w.y;
              if (i % (4 / kParts) == 0) mma<kF16, true>(d, a[i], x0, x1);
              else mma<kF16, false>(d, a[i], x0, x1);
            }
            if (kG32 && 64 * b + 32 * h >= p.K) continue;
            part[m][j][0] = fmaf(sc[h][0], d[0], part[m][j][0]);
            part[m][j][1] = fmaf(sc[h][0], d[1], part[m][j][1]);
            part[m][j][2] = fmaf(sc[h][1], d[2], part[m][j][2]);
            part[m][j][3] = fmaf(sc[h][1], d[3], part[m][j][3]);
          }
          if (kSets == 1 && m == kMt - 1 && more) load_x(v[j], j);
        }
      }
      if (!kSplit && b + 1 == boundary) {  // a range is done: add it to the sums so far
#pragma unroll
        for (int m = 0; m < kMt; ++m)
#pragma unroll
          for (int j = 0; j < kNt; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float& t = kTotRegs ? tot[kTotRegs ? m : 0][kTotRegs ? j : 0][e] : mine[((m * kNt + j) * 4 + e) * 32];
              t += part[m][j][e];
              part[m][j][e] = 0.f;
            }
        boundary += range;
      }
    };
    const int whole = min(hi, full_blocks);  // the blocks before K's last columns, if those are this warp's
    if (lo < whole) {
#pragma unroll
      for (int j = 0; j < kNt; ++j)
        if (8 * j < r.rows) load_x(xv[0][j], j);
    }
    while (b0 < hi) {
      const bool got = wait_parity_bounded(&c.full[warp][stage], phase, abort_flag, p.status);
      if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
      const int b1 = min(hi, b0 + p.chunk);
      const uint8_t* here = ring + stage * p.stage_bytes;
      codes_at = reinterpret_cast<const uint4*>(here) + lane;
      scales_at = reinterpret_cast<const float*>(here + kMt * p.chunk * kBlockBytes) + g;
      g0 = (b0 * 64) >> p.group_shift;
      if (p.scale_dt != MOE_DT_F32) {  // once per stage: the scales as f32, into the warp's own copy
        const int n = (min((b1 * 64 - 1) >> p.group_shift, p.groups - 1) - g0 + 1) * 16;
#pragma unroll
        for (int m = 0; m < kMt; ++m)
          for (int i = lane; i < n; i += 32)
            f32_scales[m * (p.f32_slot / 4) + i] =
                norm::load_one(here + kMt * p.chunk * kBlockBytes + m * p.scale_slot, p.scale_dt, i);
        scales_at = f32_scales + g;
        __syncwarp();
      }
      int b = b0;
      const int stop = min(b1, whole);
      if (kSets == 2) {
        // pairs of blocks, each set of x loaded while the other is used; a stage of odd length ends on a copy
#pragma unroll 1
        for (; b + 1 < stop; b += 2) {
          load_x(xv[1][0], 0);
          product(b, xv[0], false);
          if (b + 2 < whole) load_x(xv[0][0], 0);
          product(b + 1, xv[1 % kSets], false);
        }
        if (b < stop) {
          if (b + 1 < whole) load_x(xv[1 % kSets][0], 0);
          product(b, xv[0], false);
          xv[0][0][0] = xv[1 % kSets][0][0];
          xv[0][0][1] = xv[1 % kSets][0][1];
          ++b;
        }
      } else {
#pragma unroll 1
        for (; b < stop; ++b) product(b, xv[0], b + 1 < whole);
      }
      if (b < b1) {  // K's last columns
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
          xv[0][j][0] = norm::load16_if(xp[j], 64 * b + 8 * q < p.K);
          xv[0][j][1] = norm::load16_if(xp[j] + 4, 64 * b + 32 + 8 * q < p.K);
        }
        product(b, xv[0], false);
      }
      __syncwarp();  // the stage has been read: bring the one after the ring's others
      if (pu < u1) issue();
      if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; phase ^= 1u; }
      b0 = b1;
    }
    if (!kSplit) {
      if (!ok) break;
      // rows g, g + 8 of each tile, tokens 2 q, 2 q + 1 of each token tile
#pragma unroll
      for (int m = 0; m < kOutMt; ++m) {
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = 8 * j + 2 * q + (e & 1), ch = (r.tile0 + m) * 16 + g + ((e >> 1) << 3);
            if (tok >= r.rows || ch >= p.N) continue;
            auto total = [&](int t) {
              const float before = kTotRegs ? tot[kTotRegs ? t : 0][kTotRegs ? j : 0][e] : mine[((t * kNt + j) * 4 + e) * 32];
              return before + part[t][j][e];
            };
            float v = total(m);
            if (kSwiglu) v = v / (1.0f + __expf(-v)) * total(kMt - kOutMt + m);
            p.out[(r.row0 + tok) * p.ldo + ch] = static_cast<uint16_t>(gemm::pack2(v, 0.f, kF16) & 0xFFFFu);
          }
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < kMt; ++m)
#pragma unroll
        for (int j = 0; j < kNt; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) mine[((m * kNt + j) * 4 + e) * 32] = part[m][j][e];
      // all warps go on together or not at all
      ok = named_bar_and(1, kThreads, ok);
      if (!ok) break;
      const float* slab = sums + buf * (S::kBytes / 4);
      auto total = [&](int m, int n, int tok) {  // row n (0 .. 15) of tile m, token tok
        const int j = tok >> 3, e = ((n >> 3) << 1) | (tok & 1), l = ((n & 7) << 2) | ((tok & 7) >> 1);
        const float* v = slab + ((m * kNt + j) * 4 + e) * 32 + l;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          // an empty range adds nothing (its warp wrote zeros)
          t += v[w * kMt * kNt * 4 * 32];
        return t;
      };
      for (int i = tid; i < r.rows * kOutMt * 16; i += kThreads) {
        const int tok = i / (kOutMt * 16), n = i % (kOutMt * 16);
        const int ch = r.tile0 * 16 + n;
        if (ch >= p.N) continue;
        float v = total(n >> 4, n & 15, tok);
        if (kSwiglu) v = v / (1.0f + __expf(-v)) * total(kOutMt + (n >> 4), n & 15, tok);
        p.out[(r.row0 + tok) * p.ldo + ch] = static_cast<uint16_t>(gemm::pack2(v, 0.f, kF16) & 0xFFFFu);
      }
      buf ^= 1;
    }
  }
  if (!ok && lane == 0) {
    // let every copy in flight land before the CTA exits: the stages from here on
    const uint64_t t0 = globaltimer_ns();
    for (int i = 0; i < p.stages; ++i) {
      while (!mbar_try_wait(&c.full[warp][stage], phase) && globaltimer_ns() - t0 < 100000000ull) {
      }
      if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; phase ^= 1u; }
    }
  }
}

// ---------------------------------------------------------------- 16-bit weights for many rows
struct DequantParams {
  const uint8_t* data;   // of the first expert of the chunk
  const uint8_t* scale;
  const int32_t* offsets;  // of the first expert: experts without rows are skipped
  uint16_t* out;         // (experts, N, K)
  int N, K, n16, kb, groups, group_shift, scale_dt;
};

// A pair of exact 16-bit values times s in f32, each rounded once.
template <bool kF16>
__device__ __forceinline__ uint32_t scale_pair(uint32_t v, float s) {
  float lo, hi;
  if (kF16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    lo = f.x;
    hi = f.y;
  } else {
    lo = __uint_as_float(v << 16);
    hi = __uint_as_float(v & 0xFFFF0000u);
  }
  return gemm::pack2(lo * s, hi * s, kF16);
}

// One warp per 16 x 64 block: 16 bytes of codes per lane in, 4 x 16 bytes out
// (two rows, two runs of 8 columns), each value code * scale rounded once. The
// codes become floats as in the products (integer conversions run at a
// quarter of the rate).
template <bool kF16>
__global__ void __launch_bounds__(256) dequant_kernel(const DequantParams p) {
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int e = blockIdx.z;
  if (p.offsets[e + 1] <= p.offsets[e]) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x * 8 + warp, tile = blockIdx.y;  // a CTA walks along K
  if (b >= p.kb) return;
  const int64_t et = static_cast<int64_t>(e) * p.n16 + tile;
  const uint4 codes = *reinterpret_cast<const uint4*>(p.data + (et * p.kb + b) * kBlockBytes + lane * 16);
  const int g = lane >> 2, q = lane & 3;
  const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t a[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) codes_to_a<kF16>(word[i], a[i]);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int col = 64 * b + 32 * j + 8 * q;
    if (col >= p.K) continue;  // K is a multiple of 8
    const int64_t gi = (et * p.groups + (col >> p.group_shift)) * 16 + g;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = 16 * tile + 8 * h + g;
      if (n >= p.N) continue;
      const float s = norm::load_one(p.scale, p.scale_dt, gi + 8 * h);
      *reinterpret_cast<uint4*>(p.out + (static_cast<int64_t>(e) * p.N + n) * p.K + col) =
          make_uint4(scale_pair<kF16>(a[2 * j][h], s), scale_pair<kF16>(a[2 * j][2 + h], s),
                     scale_pair<kF16>(a[2 * j + 1][h], s), scale_pair<kF16>(a[2 * j + 1][2 + h], s));
    }
  }
}

// ---------------------------------------------------------------- quantiser
struct QuantParams {
  const void* w;  // (E, N, K)
  uint8_t* data;
  void* scale;
  int w_dt, scale_dt;
  int64_t E;
  int N, K, n16, kb, groups, group;
};

// The larger one, or NaN if either is (fmaxf gives the other).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One warp per 16-row tile and group of columns: the absolute maximum of each
// row's group (not finite if one of its weights is not: nor is the scale then),
// scale = max / 7 (1 for a group of zeros) rounded to the scales' type, code =
// round_half_even(w / scale) clamped to -8 .. 7, laid out. Groups of 32 write
// half a block per warp. 64 x 1408 x 2048 bf16 in 352 us (floor 72; each weight
// is read twice, one value per lane): it runs once per weight.
__global__ void __launch_bounds__(256) quantize_kernel(const QuantParams p) {
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + warp;
  if (unit >= p.E * p.n16 * p.groups) return;
  const int gi = static_cast<int>(unit % p.groups);
  const int64_t et = unit / p.groups;
  const int tile = static_cast<int>(et % p.n16);
  const int64_t e = et / p.n16;
  const int g = lane >> 2, q = lane & 3;
  const int col0 = gi * p.group;
  float scale[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = 16 * tile + 8 * h + g;
    float m = 0.f;
    if (n < p.N)
      for (int col = col0 + q; col < min(col0 + p.group, p.K); col += 4)
        m = max_nan(m, fabsf(norm::load_one(p.w, p.w_dt, (e * p.N + n) * p.K + col)));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float s = m == 0.f ? 1.0f : m / 7.0f;
    if (p.scale_dt == MOE_DT_BF16) s = __bfloat162float(__float2bfloat16_rn(s));
    else if (p.scale_dt == MOE_DT_F16) s = __half2float(__float2half_rn(s));
    if (s == 0.f) s = 1.0f;  // a maximum below the scale type's smallest value: codes 0
    scale[h] = s;
    if (q == 0) norm::store_one(p.scale, p.scale_dt, (et * p.groups + gi) * 16 + 8 * h + g, s);
  }
  // the 32-column halves of blocks in this group (the last group also writes K's padding)
  const int end = gi + 1 == p.groups ? p.kb * 64 : col0 + p.group;
  for (int col32 = col0; col32 < end; col32 += 32) {
    uint32_t word[2] = {0, 0};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = col32 + 8 * q + 4 * s + i, n = 16 * tile + 8 * h + g;  // i = 2 pair + odd
          int code = 0;
          if (n < p.N && col < p.K) {
            const float v = rintf(norm::load_one(p.w, p.w_dt, (e * p.N + n) * p.K + col) / scale[h]);
            code = static_cast<int>(fminf(7.f, fmaxf(-8.f, v)));
          }
          word[s] |= static_cast<uint32_t>(code + 8) << (16 * (i & 1) + 8 * (i >> 1) + 4 * h);
        }
    uint8_t* dst = p.data + (et * p.kb + col32 / 64) * kBlockBytes + lane * 16 + (col32 % 64) / 32 * 8;
    *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
  }
}

}  // namespace int4
}  // namespace moe

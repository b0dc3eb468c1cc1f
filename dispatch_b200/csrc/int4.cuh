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
// Few rows per expert: bound by the weights' bytes. See int4_kernel. Many
// rows: the weights become 16-bit tiles in a workspace (dequant_kernel, one
// rounding of code * scale to the activation type) for the tcgen05 kernels.
#pragma once
#include "gemm_warp.cuh"
#include "norm.cuh"

namespace moe {
namespace int4 {

constexpr int kWarps = 8;           // consumer warps, one 64-column block of a stage each
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kBlockBytes = 512;    // 16 rows x 64 columns
constexpr int kTileStage = kWarps * kBlockBytes;  // a 16-row tile's bytes in a stage
constexpr int kMaxE = 256;
constexpr int kMaxStages = 16;

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
  int f16, stages;
};

// The A operand of one MMA step from its word of eight codes.
template <bool kF16>
__device__ __forceinline__ void codes_to_a(uint32_t w, uint32_t (&a)[4]) {
  if (kF16) {
    // 1024 + u, and 1024 + 16 u for the nibble above it
    const __half2 c0 = __float2half2_rn(1032.f), inv = __float2half2_rn(0.0625f), c1 = __float2half2_rn(-72.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = w >> (8 * i);
      const uint32_t lo = (v & 0x000F000Fu) | 0x64006400u, hi = (v & 0x00F000F0u) | 0x64006400u;
      const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&lo), c0);
      const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&hi), inv, c1);
      a[2 * i] = *reinterpret_cast<const uint32_t*>(&l);
      a[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
    const __nv_bfloat162 c = __float2bfloat162_rn(136.f);  // 128 + u, less 136
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), c);
      a[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

struct Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  int abort;
  int experts;           // experts with rows
  int units;             // units of the launch (0 if the offsets are bad)
  int expert[kMaxE];     // their ids
  int first[kMaxE + 1];  // units before expert i
  int off[kMaxE + 1];
};
constexpr uint32_t kCtrlBytes = (sizeof(Ctrl) + 127) & ~uint32_t(127);

// A launch's shape: kMt 16-row weight tiles and kNt 8-row token tiles per unit.
template <int kMt, int kNt>
struct Shape {
  static constexpr uint32_t kDataStage = kMt * kTileStage;
  static constexpr uint32_t kRedBytes = kWarps * kMt * kNt * 4 * 32 * 4;
  static constexpr int kTok = 8 * kNt;
};

__host__ __device__ inline uint32_t scale_stage_bytes(int mt, int group_shift, int scale_shift) {
  return static_cast<uint32_t>(mt) * ((64 * kWarps) >> group_shift) * (16u << scale_shift);
}

template <int kMt, int kNt>
__host__ __device__ constexpr uint32_t fixed_smem() {
  return 128 + kCtrlBytes + 2 * Shape<kMt, kNt>::kRedBytes;
}

// Where a unit lies.
struct Unit {
  int e, row0, rows, tile0;  // expert, first row, rows (<= 8 kNt), first 16-row tile of the output
};

// A unit is kMt weight tiles (SwiGLU: half of them gate, half up rows) x one
// token tile of one expert, over all of K; consecutive units walk an expert's
// token tiles, then its weight tiles, so a CTA, which takes a contiguous run
// of units, streams contiguous weights and finds its rows of x in L1. Warp 8
// issues the bulk copies of 512-column stages (kMt tiles' blocks and their
// scales) into a ring that runs on across units; each of the other eight
// warps takes one 64-column block of a stage, so that one unit's columns are
// spread over the CTA and even a single token's few units keep the whole GPU
// loading. The warps' sums are joined in shared memory in a fixed order. A row's result
// does not depend on the unit's shape or on the other rows.
template <int kMt, int kNt, bool kSwiglu, bool kF16, bool kG32>
__global__ void __launch_bounds__(kThreads, 2) int4_kernel(const Params p) {
  using Sh = Shape<kMt, kNt>;
  constexpr int kOutTiles = kSwiglu ? kMt / 2 : kMt;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  Ctrl& c = *reinterpret_cast<Ctrl*>(base);
  float* red = reinterpret_cast<float*>(base + kCtrlBytes);
  uint8_t* ring = base + kCtrlBytes + 2 * Sh::kRedBytes;
  const uint32_t scale_stage = scale_stage_bytes(kMt, p.group_shift, p.scale_shift);
  const uint32_t stage_bytes = Sh::kDataStage + scale_stage;
  volatile int* abort_flag = &c.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], kWarps);
    }
    c.abort = 0;
    fence_mbar_init();
  }
  pdl_wait();  // before the first global memory access
  for (int g = tid; g <= p.E; g += kThreads) c.off[g] = p.offsets[g];
  __syncthreads();
  const int tile_units = (p.n16 + kOutTiles - 1) / kOutTiles;
  if (warp == 0) {
    // the experts with rows and the units before each
    int n = 0, units = 0;
    bool bad = lane == 0 && (c.off[0] < 0 || c.off[p.E] > p.M);
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int rows = e < p.E ? c.off[e + 1] - c.off[e] : 0;
      bad |= rows < 0;
      const uint32_t has = __ballot_sync(0xffffffffu, rows > 0);
      const int u = rows > 0 ? (rows + Sh::kTok - 1) / Sh::kTok * tile_units : 0;
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
  const int u0 = static_cast<int>(static_cast<int64_t>(c.units) * blockIdx.x / gridDim.x);
  const int u1 = static_cast<int>(static_cast<int64_t>(c.units) * (blockIdx.x + 1) / gridDim.x);
  if (u0 == u1) return;
  int at = 0;  // index of the unit's expert
  {
    int hi = c.experts - 1;
    while (at < hi) {
      const int mid = (at + hi + 1) / 2;
      if (c.first[mid] <= u0) at = mid; else hi = mid - 1;
    }
  }
  auto locate = [&](int u) {
    if (u >= c.first[at + 1]) ++at;
    Unit r;
    r.e = c.expert[at];
    const int begin = c.off[r.e], rows = c.off[r.e + 1] - begin;
    const int tok_tiles = (rows + Sh::kTok - 1) / Sh::kTok;
    const int local = u - c.first[at];
    const int tile = local / tok_tiles, tok = local - tile * tok_tiles;
    r.row0 = begin + tok * Sh::kTok;
    r.rows = min(Sh::kTok, rows - tok * Sh::kTok);
    r.tile0 = tile * kOutTiles;
    return r;
  };
  const int stages_per_unit = (p.kb + kWarps - 1) / kWarps;

  if (warp == kWarps) {
    // ------------------------------------------------------------ bulk copies
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      uint32_t issued_mask = 0, issued_parity = 0;
      bool ok = true;
      const uint32_t group_bytes = 16u << p.scale_shift;
      for (int u = u0; ok && u < u1; ++u) {
        const Unit r = locate(u);
        const int tiles = min(kOutTiles, p.n16 - r.tile0);
        for (int s = 0; s < stages_per_unit; ++s) {
          if (!wait_parity_bounded(&c.empty[stage], phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          const int b0 = s * kWarps, nb = min(kWarps, p.kb - b0);
          const int g0 = (b0 * 64) >> p.group_shift;
          const int ng = min((64 * kWarps) >> p.group_shift, p.groups - g0);
          const uint32_t per_tile = nb * kBlockBytes + ng * group_bytes;
          mbar_arrive_expect_tx(&c.full[stage], per_tile * tiles * (kSwiglu ? 2 : 1));
          uint8_t* dst = ring + stage * stage_bytes;
          for (int i = 0; i < (kSwiglu ? 2 : 1) * tiles; ++i) {
            const bool up = kSwiglu && i >= tiles;
            const int slot = up ? kOutTiles + i - tiles : i;
            const int64_t tile = static_cast<int64_t>(r.e) * p.n16 + r.tile0 + (up ? i - tiles : i);
            bulk_load(dst + slot * kTileStage, (up ? p.data1 : p.data0) + (tile * p.kb + b0) * kBlockBytes,
                      nb * kBlockBytes, &c.full[stage]);
            bulk_load(dst + Sh::kDataStage + slot * (scale_stage / kMt),
                      (up ? p.scale1 : p.scale0) + (tile * p.groups + g0) * group_bytes, ng * group_bytes,
                      &c.full[stage]);
          }
          issued_mask |= 1u << stage;
          issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        // let every copy in flight land before the CTA exits
        for (int i = 0; i < p.stages; ++i) {
          if (!(issued_mask & (1u << i))) continue;
          const uint32_t par = (issued_parity >> i) & 1u;
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&c.full[i], par) && globaltimer_ns() - t0 < 100000000ull) {
          }
        }
      }
    }
    return;
  }
  // -------------------------------------------------------------- MMA warps
  const int g = lane >> 2, q = lane & 3;
  uint32_t stage = 0, phase = 0;
  int buf = 0;
  bool ok = true;
  for (int u = u0; u < u1; ++u) {
    const Unit r = locate(u);
    const int tiles = min(kOutTiles, p.n16 - r.tile0);
    float acc[kMt][kNt][4];
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][j][e] = 0.f;
    for (int s = 0; ok && s < stages_per_unit; ++s) {
      const int b = s * kWarps + warp;
      // this lane's pieces of its tokens' rows (token 8 j + g): before the wait
      uint4 xv[kNt][2];
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          xv[j][h] = make_uint4(0, 0, 0, 0);
          const int col = 64 * b + 32 * h + 8 * q;
          if (8 * j + g < r.rows && col < p.K)
            xv[j][h] = *reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(r.row0 + 8 * j + g) * p.K + col);
        }
      const bool got = wait_parity_bounded(&c.full[stage], phase, abort_flag, p.status);
      if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
      if (b < p.kb) {
        const uint8_t* data = ring + stage * stage_bytes + warp * kBlockBytes + lane * 16;
        const uint8_t* scales = ring + stage * stage_bytes + Sh::kDataStage;
#pragma unroll
        for (int m = 0; m < kMt; ++m) {
          if (kSwiglu ? (m % kOutTiles) >= tiles : m >= tiles) continue;
          const uint4 codes = *reinterpret_cast<const uint4*>(data + m * kTileStage);
          const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
          constexpr int kParts = kG32 ? 2 : 1;  // scaled sums per block
          float sc[kParts][2];
#pragma unroll
          for (int h = 0; h < kParts; ++h) {
            const int gi = ((64 * warp + 32 * h) >> p.group_shift) * 16 + g;
            const uint8_t* at_tile = scales + m * (scale_stage / kMt);
            // the second half of K's last block may lie past the last group: nothing was copied for it
            const bool has = !kG32 || (64 * b + 32 * h) < p.K;
            sc[h][0] = has ? norm::load_one(at_tile, p.scale_dt, gi) : 0.f;
            sc[h][1] = has ? norm::load_one(at_tile, p.scale_dt, gi + 8) : 0.f;
          }
          uint32_t a[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) codes_to_a<kF16>(word[i], a[i]);
#pragma unroll
          for (int j = 0; j < kNt; ++j) {
            if (8 * j >= r.rows) continue;
#pragma unroll
            for (int h = 0; h < kParts; ++h) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int i = 4 / kParts * h; i < 4 / kParts * (h + 1); ++i) {
                const uint4& v = xv[j][i / 2];
                if (i % 2 == 0) gemm::mma_16816(d, a[i], v.x, v.y, kF16);
                else gemm::mma_16816(d, a[i], v.z, v.w, kF16);
              }
              acc[m][j][0] = fmaf(sc[h][0], d[0], acc[m][j][0]);
              acc[m][j][1] = fmaf(sc[h][0], d[1], acc[m][j][1]);
              acc[m][j][2] = fmaf(sc[h][1], d[2], acc[m][j][2]);
              acc[m][j][3] = fmaf(sc[h][1], d[3], acc[m][j][3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.empty[stage]);
      if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; phase ^= 1u; }
    }
    // ---- join the warps' sums: element (tile m, token tile j, e) of lane l
    float* slab = red + buf * (Sh::kRedBytes / 4);
#pragma unroll
    for (int m = 0; m < kMt; ++m)
#pragma unroll
      for (int j = 0; j < kNt; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) slab[(((warp * kMt + m) * kNt + j) * 4 + e) * 32 + lane] = acc[m][j][e];
    // all warps leave together or not at all
    ok = named_bar_and(1, 32 * kWarps, ok);
    if (!ok) break;
    auto total = [&](int m, int n, int tok) {  // row n (0 .. 15) of tile m, token tok
      const int j = tok >> 3, e = ((n >> 3) << 1) | (tok & 1), l = ((n & 7) << 2) | ((tok & 7) >> 1);
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += slab[(((w * kMt + m) * kNt + j) * 4 + e) * 32 + l];
      return t;
    };
    for (int i = tid; i < r.rows * kOutTiles * 16; i += 32 * kWarps) {
      const int tok = i / (kOutTiles * 16), n = i % (kOutTiles * 16);
      const int ch = r.tile0 * 16 + n;
      if (ch >= p.N) continue;
      float v = total(n >> 4, n & 15, tok);
      if (kSwiglu) {
        const float up = total(kOutTiles + (n >> 4), n & 15, tok);
        v = v / (1.0f + __expf(-v)) * up;
      }
      p.out[(r.row0 + tok) * p.ldo + ch] = static_cast<uint16_t>(gemm::pack2(v, 0.f, kF16) & 0xFFFFu);
    }
    buf ^= 1;
  }
}

// ---------------------------------------------------------------- 16-bit weights for many rows
struct DequantParams {
  const uint8_t* data;   // of the first expert of the chunk
  const uint8_t* scale;
  const int32_t* offsets;  // of the first expert: experts without rows are skipped
  uint16_t* out;         // (experts, N, K)
  int N, K, n16, kb, groups, group_shift, scale_dt, scale_shift, f16;
};

// One warp per 16 x 64 block: 16 bytes of codes per lane in, 4 x 16 bytes out
// (two rows, two runs of 8 columns), each value code * scale rounded once.
__global__ void __launch_bounds__(256) dequant_kernel(const DequantParams p) {
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int e = blockIdx.y;
  if (p.offsets[e + 1] <= p.offsets[e]) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t block = static_cast<int64_t>(blockIdx.x) * 8 + warp;
  if (block >= static_cast<int64_t>(p.n16) * p.kb) return;
  const int tile = static_cast<int>(block / p.kb), b = static_cast<int>(block % p.kb);
  const int64_t et = static_cast<int64_t>(e) * p.n16 + tile;
  const uint4 codes = *reinterpret_cast<const uint4*>(p.data + (et * p.kb + b) * kBlockBytes + lane * 16);
  const uint32_t word[4] = {codes.x, codes.y, codes.z, codes.w};
  const int g = lane >> 2, q = lane & 3;
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
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // columns 2 i, 2 i + 1: step i / 2, pair i % 2
        const uint32_t v = word[2 * j + i / 2] >> (8 * (i % 2) + 4 * h);
        const float lo = static_cast<float>(static_cast<int>(v & 15u) - 8);
        const float hi = static_cast<float>(static_cast<int>((v >> 16) & 15u) - 8);
        w[i] = gemm::pack2(lo * s, hi * s, p.f16);
      }
      *reinterpret_cast<uint4*>(p.out + (static_cast<int64_t>(e) * p.N + n) * p.K + col) =
          make_uint4(w[0], w[1], w[2], w[3]);
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

// One warp per 16-row tile and group of columns: the absolute maximum of each
// row's group, scale = max / 7 (1 for a group of zeros) rounded to the scales'
// type, code = round_half_even(w / scale) clamped to -8 .. 7, laid out. Groups
// of 32 write half a block per warp.
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
        m = fmaxf(m, fabsf(norm::load_one(p.w, p.w_dt, (e * p.N + n) * p.K + col)));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
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

// Expert products with 4-bit weights on the 5th-generation tensor cores, for
// more than a few rows per expert. Weights as laid out in int4.cuh.
//
// Tile: 128 weight rows (the MMA's M side; SwiGLU: 64 gate and the matching 64
// up rows) x up to 64 or 128 token rows of one expert (N), over all of K.
// Eight converter warps each stream one 16-row weight tile through a small
// ring of their own (bulk copies that only the warp waits for), make the codes
// 16-bit floats exactly, and write them as a K-major, 128-byte swizzled A
// operand; one warp brings the token rows by TMA, one issues the MMAs. The MMAs
// of one scale group accumulate in one of two TMEM buffers; the epilogue warps
// take each group's f32 sums from there and add them, times the row's scale,
// to sums in registers. So no weight is rounded, the scales act in f32, and a
// weight crosses HBM once, as 4 bits, per token tile.
//
// Bound by latency, not by a pipe: 64 experts of 1408 x 2048 and 48 rows take
// 74 us (1.6 TB/s), about 850 cycles per block of 64 columns; the time without
// the MMAs, the conversion, its stores or the fence is within 5% of it. What is
// left is the chain free stage -> converted -> MMAs -> free stage (38 to 45% of
// the issue slots used, HBM at 9 to 17% of its peak). The 128-row form's 576
// threads have 96 registers each and spill 200 to 364 bytes.
//
// Every wait is bounded; a role that gives up raises `abort`, the others
// follow, copies and MMAs in flight are waited for, and TMEM is freed.
#pragma once
#include "int4.cuh"

namespace moe {
namespace int4 {

constexpr int kTileRows = 128;
constexpr uint32_t kABytes = kTileRows * 128;  // 64 columns of A
constexpr int kTileStages = 8;                 // at most
constexpr int kCodeStages = 3;                 // of a converter's ring
constexpr int kAccCols = 64;                   // token columns of an epilogue thread
constexpr int kConvWarps = 8;

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// An MMA, and a commit, by the lanes with `lead`: the whole warp runs the
// issuing loop, so that descriptors and addresses stay in uniform registers.
__device__ __forceinline__ void mma_if(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}

// The kernel's two forms, by the most token rows of a tile (64 or 128).
template <int kTok>
struct TileShape {
  static constexpr int kEpi = kTok / 16;  // epilogue warps: 64 token columns per thread
  // 64-column blocks of a stage: the MMA warp's waits and commits are per
  // stage. With 64 rows a stage holds two (one block per stage, 512 tokens of
  // the 64-expert layer: 85 us, two: 74).
  static constexpr int kSub = kTok == 64 ? 2 : 1;
  // Scale groups that pass from the MMAs to the epilogue at a time: two sets
  // of this many buffers fill TMEM. One group at a time, the hand-over's latency
  // (~1000 cycles) sets the whole tile's pace.
  static constexpr int kSet = kTok == 64 ? 4 : 2;
  // Stages that a converter makes between two waits and fences (one: 94 us);
  // blocks of a stage of its ring.
  static constexpr int kBatch = 2;
  static constexpr int kCodeChunk = 4;
  static constexpr int kEpiWarp0 = 2 + kConvWarps;
  static constexpr int kThreads = 32 * (kEpiWarp0 + kEpi);
};

struct TileParams {
  CUtensorMap map_x;  // (M, K), box 64 x nt, 128-byte swizzle
  Params p;           // (its ring sizes are not used)
  int nt;             // token rows per tile: 64 or 128
  int tile_stages;
};

struct TileCtrl {
  uint64_t ready[kTileStages];  // token rows arrived and A written
  uint64_t empty[kTileStages];  // MMAs have read the stage
  uint64_t codes[kConvWarps][kCodeStages];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int experts, tiles;
  int expert[kMaxE];
  int first[kMaxE + 1];
  int off[kMaxE + 1];
};
constexpr uint32_t kTileCtrlBytes = (sizeof(TileCtrl) + 1023) & ~uint32_t(1023);
constexpr uint32_t kTileXchgBytes = 4 * 32 * 16 * 4;  // up values of 16 columns for up to four gate warps

__host__ __device__ constexpr uint32_t tile_fixed_smem() { return kTileCtrlBytes + kTileXchgBytes; }

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

template <bool kSwiglu, bool kF16, bool kG32, int kTok>
__global__ void __launch_bounds__(TileShape<kTok>::kThreads, 1)
    int4_tile_kernel(const __grid_constant__ TileParams tp) {
  using Sh = TileShape<kTok>;
  constexpr int kEpi = Sh::kEpi;
  constexpr int kOutTiles = kSwiglu ? 4 : 8;  // 16-row output tiles of a tile
  constexpr int kBatch = Sh::kBatch;
  const Params& p = tp.p;
  const int nt = tp.nt, S = tp.tile_stages;
  extern __shared__ __align__(1024) uint8_t tile_smem[];
  TileCtrl& c = *reinterpret_cast<TileCtrl*>(tile_smem);
  float* xchg = reinterpret_cast<float*>(tile_smem + kTileCtrlBytes);
  uint8_t* sA = tile_smem + tile_fixed_smem();
  constexpr int kSub = Sh::kSub;
  uint8_t* sB = sA + S * kSub * kABytes;
  uint8_t* sQ = sB + S * kSub * nt * 128;
  volatile int* abort_flag = &c.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(2 * Sh::kSet * nt)) tmem_cols <<= 1;

  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&c.ready[i], 1 + kConvWarps);
      mbar_init(&c.empty[i], 1);
    }
    for (int w = 0; w < kConvWarps; ++w)
      for (int i = 0; i < kCodeStages; ++i) mbar_init(&c.codes[w][i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.tfull[i], 1);
      mbar_init(&c.tempty[i], kEpi);
    }
    mbar_init(&c.drain, 1);
    c.abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tp.map_x);
  }
  if (warp == 1) {
    tmem_alloc(&c.tmem_base, tmem_cols);
    tmem_relinquish();
  }
  pdl_wait();  // before the first global memory access
  for (int g = tid; g <= p.E; g += Sh::kThreads) c.off[g] = p.offsets[g];
  __syncthreads();
  const int blocks = (p.n16 + kOutTiles - 1) / kOutTiles;  // of weight rows, per expert
  if (warp == 0) {
    // the experts with rows and the tiles before each
    int n = 0, tiles = 0;
    bool bad = lane == 0 && (c.off[0] < 0 || c.off[p.E] > p.M);
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int rows = e < p.E ? c.off[e + 1] - c.off[e] : 0;
      bad |= rows < 0;
      const uint32_t has = __ballot_sync(0xffffffffu, rows > 0);
      const int u = rows > 0 ? (rows + nt - 1) / nt * blocks : 0;
      int v = u;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
      }
      if (rows > 0) {
        const int i = n + __popc(has & ((1u << lane) - 1u));
        c.expert[i] = e;
        c.first[i] = tiles + v - u;
      }
      n += __popc(has);
      tiles += __shfl_sync(0xffffffffu, v, 31);
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      c.first[n] = tiles;
      c.experts = n;
      c.tiles = bad ? 0 : tiles;
      if (bad && p.status) atomicCAS(p.status, 0, MOE_ERR_BAD_OFFSETS);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = c.tmem_base;
  const int total = c.tiles;
  // tile t, at or after the last one located with `at`: token tiles of a
  // weight block are adjacent, so it is read again from L2
  auto locate = [&](int t, int& at) {
    while (t >= c.first[at + 1]) ++at;
    Unit r;
    r.e = c.expert[at];
    const int begin = c.off[r.e], rows = c.off[r.e + 1] - begin;
    int block = t - c.first[at], tok = 0;
    if (rows > nt) {
      const int tok_tiles = (rows + nt - 1) / nt;
      tok = block % tok_tiles;
      block /= tok_tiles;
    }
    r.row0 = begin + tok * nt;
    r.rows = min(nt, rows - tok * nt);
    r.tile0 = block * kOutTiles;
    return r;
  };
  const int steps_per_group = 1 << (p.group_shift - 4);  // MMAs of 16 columns
  int at = 0;

  if (warp == 0) {
    // ------------------------------------------------------------ token rows by TMA
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const Unit r = locate(t, at);
        for (int kb = 0; kb < p.kb; kb += kSub) {
          if (!wait_parity_bounded(&c.empty[stage], phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          const int n = min(kSub, p.kb - kb);
          mbar_arrive_expect_tx(&c.ready[stage], n * nt * 128);
          for (int i = 0; i < n; ++i)
            tma_load_2d(sB + (stage * kSub + i) * nt * 128, &tp.map_x, &c.ready[stage], (kb + i) * 64, r.row0);
          issued_mask |= 1u << stage;
          issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == static_cast<uint32_t>(S)) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        // let every copy in flight land before the CTA exits (a barrier that converters
        // no longer arrive on runs into the limit, long after its copy has landed)
        const uint64_t t0 = globaltimer_ns();
        for (int i = 0; i < S; ++i)
          while (((issued_mask >> i) & 1u) && !mbar_try_wait(&c.ready[i], (issued_parity >> i) & 1u) &&
                 globaltimer_ns() - t0 < 100000000ull) {
          }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // One thread's dependent instructions set the pace of the whole tile, so
    // the loop holds little: descriptors advance by addition, a stage has one
    // barrier, and groups of 64 columns or more end on stage boundaries.
    {
      const uint32_t lead = lane == 0;
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      const uint64_t a0 = sw128_kmajor_desc(smem_u32(sA)), b0 = sw128_kmajor_desc(smem_u32(sB));
      const uint32_t b_step = nt * 128 / 16;  // descriptors count 16 bytes
      const int blocks_per_group = kG32 ? 1 : 1 << (p.group_shift - 6);
      uint64_t ad = a0, bd = b0;
      bool ok = true, issued = false;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const Unit r = locate(t, at);
        // MMA width: the tile's rows rounded up to 16
        const uint32_t idesc = idesc_f16(kTileRows, min(nt, (r.rows + 15) & ~15), kF16);
        int left = 0;    // blocks left in the group
        int in_set = 0;  // groups in the set so far
        uint32_t d = 0;  // the group's buffer
        for (int kb = 0; kb < p.kb; kb += kSub) {
          if (!wait_parity_bounded(&c.ready[stage], phase, abort_flag, p.status)) { ok = false; break; }
          tc_fence_after();
          issued = true;
#pragma unroll
          for (int i = 0; i < kSub; ++i) {
            if (!ok || (kSub > 1 && kb + i >= p.kb)) continue;
            const uint64_t ai = ad + i * (kABytes / 16), bi = bd + i * b_step;
            const uint32_t more = left != 0;
            auto next_group = [&]() {
              if (in_set == 0) {  // a set's buffers have to be empty
                ok = wait_parity_bounded(&c.tempty[acc], acc_phase ^ 1u, abort_flag, p.status);
                tc_fence_after();
                d = tmem_base + acc * (Sh::kSet * nt);
              } else {
                d += nt;
              }
            };
            auto end_group = [&](bool last) {
              if (++in_set == Sh::kSet || last) {
                commit_if(lead, &c.tfull[acc]);
                acc ^= 1u;
                acc_phase ^= acc == 0 ? 1u : 0u;
                in_set = 0;
              }
            };
            if (!more) {
              left = min(blocks_per_group, p.kb - kb - i);
              next_group();
              if (!ok) continue;
            }
            mma_if(lead, d, ai, bi, idesc, more);
            mma_if(lead, d, ai + 2, bi + 2, idesc, 1u);
            if (kG32) {  // two groups in a block
              end_group(false);
              next_group();
              if (!ok) continue;
            }
            mma_if(lead, d, ai + 4, bi + 4, idesc, kG32 ? 0u : 1u);
            mma_if(lead, d, ai + 6, bi + 6, idesc, 1u);
            if (--left == 0) end_group(kb + i + 1 == p.kb);
          }
          if (!ok) break;
          commit_if(lead, &c.empty[stage]);
          ad += kSub * (kABytes / 16);
          bd += kSub * b_step;
          if (++stage == static_cast<uint32_t>(S)) { stage = 0; phase ^= 1u; ad = a0; bd = b0; }
        }
      }
      if (!ok && issued) {
        commit_if(lead, &c.drain);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&c.drain, 0) && globaltimer_ns() - t0 < 100000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp < Sh::kEpiWarp0) {
    // ------------------------------------------------------------ codes -> A
    const int w = warp - 2;  // 16-row tile of the 128 rows
    const bool up = kSwiglu && w >= kOutTiles;
    const uint8_t* data = up ? p.data1 : p.data0;
    const int mine = up ? w - kOutTiles : w;
    uint8_t* ring = sQ + w * kCodeStages * Sh::kCodeChunk * kBlockBytes;
    // the next stage to bring: tile, first block
    int pt = blockIdx.x, pb = 0, pat = 0;
    uint32_t pstage = 0;
    const uint8_t* psrc = nullptr;  // of the tile; null past N
    auto place = [&]() {
      const Unit r = locate(pt, pat);
      const int tile = r.tile0 + mine;
      psrc = tile < p.n16 ? data + (static_cast<int64_t>(r.e) * p.n16 + tile) * p.kb * kBlockBytes : nullptr;
    };
    if (pt < total) place();
    auto issue = [&]() {
      const int nb = min(Sh::kCodeChunk, p.kb - pb);
      if (lane == 0) {
        uint64_t* bar = &c.codes[w][pstage];
        mbar_arrive_expect_tx(bar, psrc ? nb * kBlockBytes : 0);
        if (psrc)
          bulk_load(ring + pstage * Sh::kCodeChunk * kBlockBytes, psrc + static_cast<int64_t>(pb) * kBlockBytes,
                    nb * kBlockBytes, bar);
      }
      if (++pstage == static_cast<uint32_t>(kCodeStages)) pstage = 0;
      pb += nb;
      if (pb == p.kb) {
        pb = 0;
        pt += gridDim.x;
        if (pt < total) place();
      }
    };
    for (int i = 0; i < kCodeStages && pt < total; ++i) issue();
    const int g = lane >> 2, q = lane & 3;
    // rows 16 w + g and + 8 (both g modulo 8), 16-byte chunks q and 4 + q of their 128 bytes
    const uint32_t row = smem_u32(sA) + (16 * w + g) * 128, chunk0 = (q ^ g) << 4, chunk1 = ((4 + q) ^ g) << 4;
    const uint32_t ring_at = smem_u32(ring) + lane * 16;
    constexpr int kBlocks = kBatch * kSub;
    uint32_t stage = 0, phase = 0, cstage = 0, cphase = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
      for (int b0 = 0; ok && b0 < p.kb; b0 += Sh::kCodeChunk) {
        bool got = wait_parity_bounded(&c.codes[w][cstage], cphase, abort_flag, p.status);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
        const uint32_t src = ring_at + cstage * Sh::kCodeChunk * kBlockBytes;
        const int nb = min(Sh::kCodeChunk, p.kb - b0);
        for (int b = 0; ok && b < nb; b += kBlocks) {
          const int n = min(kBlocks, nb - b);
          uint4 codes[kBlocks];
#pragma unroll
          for (int i = 0; i < kBlocks; ++i)
            if (i < n) codes[i] = lds128(src + (b + i) * kBlockBytes);
          // the batch's stages: the MMAs leave them in order, so its last is free after the others
          uint32_t at_stage[2], last_phase = phase;
          at_stage[0] = stage;
          if (++stage == static_cast<uint32_t>(S)) { stage = 0; phase ^= 1u; }
          at_stage[1] = at_stage[0];
          if (n > kSub) {
            at_stage[1] = stage;
            last_phase = phase;
            if (++stage == static_cast<uint32_t>(S)) { stage = 0; phase ^= 1u; }
          }
          got = wait_parity_bounded(&c.empty[at_stage[1]], last_phase ^ 1u, abort_flag, p.status);
          if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
#pragma unroll
          for (int i = 0; i < kBlocks; ++i) {
            if (i >= n) continue;
            uint32_t a[4][4];
            codes_to_a<kF16>(codes[i].x, a[0]);
            codes_to_a<kF16>(codes[i].y, a[1]);
            codes_to_a<kF16>(codes[i].z, a[2]);
            codes_to_a<kF16>(codes[i].w, a[3]);
            const uint32_t dst = row + (at_stage[i / kSub] * kSub + i % kSub) * kABytes;
            // word 2 j + s: columns 32 j + 8 q + 4 s .. + 3 of row g (a0, a2) and row g + 8 (a1, a3)
            sts128(dst + chunk0, a[0][0], a[0][2], a[1][0], a[1][2]);
            sts128(dst + chunk1, a[2][0], a[2][2], a[3][0], a[3][2]);
            sts128(dst + 1024 + chunk0, a[0][1], a[0][3], a[1][1], a[1][3]);
            sts128(dst + 1024 + chunk1, a[2][1], a[2][3], a[3][1], a[3][3]);
          }
          // one fence for the batch: it waits for the writes before it
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&c.ready[at_stage[0]]);
            if (n > kSub) mbar_arrive(&c.ready[at_stage[1]]);
          }
        }
        if (!ok) break;
        __syncwarp();  // the ring's stage has been read: bring the one after the others
        if (pt < total) issue();
        if (++cstage == static_cast<uint32_t>(kCodeStages)) { cstage = 0; cphase ^= 1u; }
      }
    }
    if (!ok && lane == 0) {
      // let every copy in flight land before the CTA exits: the stages from here on
      const uint64_t t0 = globaltimer_ns();
      for (int i = 0; i < kCodeStages; ++i) {
        while (!mbar_try_wait(&c.codes[w][cstage], cphase) && globaltimer_ns() - t0 < 100000000ull) {
        }
        if (++cstage == static_cast<uint32_t>(kCodeStages)) { cstage = 0; cphase ^= 1u; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    // Thread: weight row 32 quarter + lane of the tile, up to 64 token columns
    // (with eight warps, two warps per quarter take 64 columns each).
    const int ew = warp - Sh::kEpiWarp0, quarter = warp & 3;
    const int col0 = kEpi == 8 && ew >= 4 ? kAccCols : 0;
    const int row = 32 * quarter + lane;
    const bool up = kSwiglu && row >= 64;
    const int my_tile = (up ? row - 64 : row) >> 4;  // 16-row tile of the output block
    const uint8_t* scales = up ? p.scale1 : p.scale0;
    const int groups = (p.kb * 4 + steps_per_group - 1) >> (p.group_shift - 4);  // with one past K in the last block
    uint32_t acc = 0, acc_phase = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const Unit r = locate(t, at);
      const int cols = min(kAccCols, ((r.rows + 15) & ~15) - col0);  // may be <= 0
      const bool has = r.tile0 + my_tile < p.n16;
      const int64_t s0 = ((static_cast<int64_t>(r.e) * p.n16 + r.tile0 + my_tile) * p.groups) * 16 + (row & 15);
      auto scale_of = [&](int gi) {
        return has && gi < p.groups ? norm::load_one(scales, p.scale_dt, s0 + gi * 16) : 0.f;
      };
      norm::F2 sum[kAccCols / 2];
#pragma unroll
      for (int i = 0; i < kAccCols / 2; ++i) sum[i] = 0ull;
      constexpr int kSet = Sh::kSet;
      float sc[kSet];
#pragma unroll
      for (int i = 0; i < kSet; ++i) sc[i] = scale_of(i);
      bool ok = true;
      for (int g0 = 0; g0 < groups; g0 += kSet) {
        float nx[kSet];  // the next set's scales
#pragma unroll
        for (int i = 0; i < kSet; ++i) nx[i] = scale_of(g0 + kSet + i);
        const bool got = wait_parity_bounded(&c.tfull[acc], acc_phase, abort_flag, p.status);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
        tc_fence_after();
        const uint32_t tb = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * (kSet * nt) + col0;
#pragma unroll
        for (int c0 = 0; c0 < kAccCols; c0 += 16) {
          if (c0 >= cols) continue;
#pragma unroll
          for (int i = 0; i < kSet; i += 2) {  // two groups' loads in flight (one past the last is not used)
            uint32_t v[2][16];
            tmem_ld_x16(tb + i * nt + c0, v[0]);
            tmem_ld_x16(tb + (i + 1) * nt + c0, v[1]);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (g0 + i + h >= groups) continue;
              const norm::F2 s2 = norm::both(sc[i + h]);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                sum[c0 / 2 + k] = norm::fma2(
                    norm::pack(__uint_as_float(v[h][2 * k]), __uint_as_float(v[h][2 * k + 1])), s2, sum[c0 / 2 + k]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.tempty[acc]);
        acc ^= 1u;
        acc_phase ^= acc == 0 ? 1u : 0u;
#pragma unroll
        for (int i = 0; i < kSet; ++i) sc[i] = nx[i];
      }
      // the epilogue warps go on together or not at all
      ok = named_bar_and(1, 32 * kEpi, ok);
      if (!ok) break;
      const int ch = (r.tile0 + my_tile) * 16 + (row & 15);
      uint16_t* out = p.out + static_cast<int64_t>(r.row0 + col0) * p.ldo + ch;
      const int live = min(kAccCols, r.rows - col0);
#pragma unroll
      for (int c0 = 0; c0 < kAccCols; c0 += 16) {
        float v[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) norm::unpack(sum[c0 / 2 + k], v[2 * k], v[2 * k + 1]);
        if (kSwiglu) {
          // up warps (quarters 2, 3) hand 16 columns at a time to the gate warps; all epilogue
          // warps take part, whatever their columns
          float* xb = xchg + ((quarter & 1) + (col0 ? 2 : 0)) * 32 * 16 + lane;
          if (up) {
#pragma unroll
            for (int k = 0; k < 16; ++k) xb[k * 32] = v[k];
          }
          named_bar_sync(1, 32 * kEpi);
          if (!up) {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = v[k] / (1.0f + __expf(-v[k])) * xb[k * 32];
          }
          named_bar_sync(1, 32 * kEpi);
        }
        if (!up && ch < p.N) {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (c0 + k < live)
              out[(c0 + k) * p.ldo] = static_cast<uint16_t>(gemm::pack2(v[k], 0.f, kF16) & 0xFFFFu);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

}  // namespace int4
}  // namespace moe

// The norms before and after a block, fused with the block's gate, residual
// scale and residual add, and their gradients. Per row of H values:
//
//   r1  = rsqrt(mean(y^2) + eps)           z    = y r1 post        (z = y without post)
//   out = residual + a gate z              r2   = rsqrt(mean(out^2) + eps)
//   normed = out r2 next
//
// Without y, out is the residual itself and only normed is written: the norm
// at a block's entry. gate is absent, one value per channel, per row or per
// element; a is the residual scale.
//
// Gradients, with D = d_out and N = d_normed (either may be absent):
//   dfull = D + r2 (N next - out r2^2 mean(N next out))  = d_residual
//   dz    = a gate dfull                                  d_gate = a z dfull (summed over the broadcast)
//   d_y   = r1 (dz post - y r1^2 mean(dz post y))
//   d_post = sum_rows dz y r1                             d_next = sum_rows N out r2
// The backward kernel recomputes out, r1 and r2 from y and residual in f32
// instead of reading saved ones: the same bytes as reading out, and the
// gradient is that of the unrounded function.
//
// Both are bound by HBM. A row lives in the registers of one group of threads
// (8 values per thread and vector), so every array is read once and written
// once; all sums are f32, each output is rounded once.
#pragma once
#include "ptx.cuh"

namespace moe {
namespace norm {

constexpr int kMaxH = 16384;

struct Params {
  const void* y;         // null: no branch, out = residual
  const void* residual;
  const void* post;      // null: z = y
  const void* next;      // null: no second norm
  const void* gate;
  void* out;
  void* normed;
  const void* d_out;     // backward inputs, may be null
  const void* d_normed;
  void* d_y;             // backward outputs, may be null
  void* d_residual;
  void* d_gate;          // token and full modes
  float* part;           // backward: (slabs, 3, H) partial column sums: post, next, channel gate
  int64_t T;
  int64_t y_stride, res_stride, gate_stride, d_out_stride, d_normed_stride;  // elements between rows
  int H;
  int y_dt, res_dt, post_dt, next_dt, gate_dt, norm_dt;
  int gate_mode;
  int want_post, want_next, want_gate;
  float scale, eps;
};

// Eight values of a row as they lie in memory: 16 bytes (16-bit types) or 32.
struct Raw {
  uint4 a, b;
};

__device__ __forceinline__ Raw zero_raw() { return Raw{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}; }

// Values off .. off+7 of which the first n exist (the rest read as 0). kVec:
// 16-byte aligned and n is 0 or 8. Loads only, no conversion, so that several
// arrays' loads are in flight together.
template <bool kVec>
__device__ __forceinline__ Raw load_raw(const void* base, int dt, int64_t off, int n) {
  Raw r = zero_raw();
  if (kVec) {
    if (n > 0) {
      if (dt == MOE_DT_F32) {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + off);
        r.a = p[0];
        r.b = p[1];
      } else {
        r.a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + off);
      }
    }
  } else {
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < n) {
        if (dt == MOE_DT_F32) {
          w[i] = reinterpret_cast<const uint32_t*>(base)[off + i];
        } else {
          w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(base)[off + i]) << (16 * (i & 1));
        }
      }
    }
    r.a = make_uint4(w[0], w[1], w[2], w[3]);
    r.b = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return r;
}

__device__ __forceinline__ void to_f32(const Raw& r, int dt, float (&v)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dt == MOE_DT_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  } else if (dt == MOE_DT_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

__device__ __forceinline__ float load_one(const void* base, int dt, int64_t i) {
  if (dt == MOE_DT_F32) return reinterpret_cast<const float*>(base)[i];
  if (dt == MOE_DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
  return __half2float(reinterpret_cast<const __half*>(base)[i]);
}

__device__ __forceinline__ void store_one(void* base, int dt, int64_t i, float v) {
  if (dt == MOE_DT_F32) reinterpret_cast<float*>(base)[i] = v;
  else if (dt == MOE_DT_BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(base)[i] = __float2half_rn(v);
}

template <bool kVec>
__device__ __forceinline__ void store_f32(void* base, int dt, int64_t off, int n, const float (&v)[8]) {
  if (!kVec) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store_one(base, dt, off + i, v[i]);
    return;
  }
  if (n <= 0) return;
  if (dt == MOE_DT_F32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + off);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == MOE_DT_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + off) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A row's group: kTpr threads, kRpc groups per CTA.
template <int kTpr>
struct Group {
  static constexpr int kThreads = kTpr < 256 ? 256 : kTpr;
  static constexpr int kRpc = kThreads / kTpr;
  static constexpr int kWarps = kTpr / 32;
};

// Sum of one or two values over the group, in a fixed order. `slot` must
// differ from the slot of the previous call of the same group (two slots
// taken in turn: a warp may still read one while the next is written).
template <int kTpr>
__device__ __forceinline__ float2 group_sum(float2 v, float2 (*slots)[32], int slot, int group, int tx) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, d);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, d);
  }
  if (kTpr == 32) return v;
  if ((tx & 31) == 0) slots[slot][tx >> 5] = v;
  named_bar_sync(1 + group, kTpr);
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < Group<kTpr>::kWarps; ++w) {
    const float2 o = slots[slot][w];
    s.x += o.x;
    s.y += o.y;
  }
  return s;
}

__device__ __forceinline__ int valid_at(int H, int col) {
  const int n = H - col;
  return n < 0 ? 0 : n > 8 ? 8 : n;
}

// gate of 8 columns: raw for channel and full modes, one value for a row.
__device__ __forceinline__ void gate_f32(const Params& p, const Raw& raw, float row_gate, float (&g)[8]) {
  if (p.gate_mode == MOE_GATE_CHANNEL || p.gate_mode == MOE_GATE_FULL) {
    to_f32(raw, p.gate_dt, g);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = row_gate;
  }
}

template <bool kVec>
__device__ __forceinline__ Raw gate_raw(const Params& p, int64_t row, int col, int n) {
  if (p.gate_mode == MOE_GATE_CHANNEL) return load_raw<kVec>(p.gate, p.gate_dt, col, n);
  if (p.gate_mode == MOE_GATE_FULL) return load_raw<kVec>(p.gate, p.gate_dt, row * p.gate_stride + col, n);
  return zero_raw();
}

template <int kTpr, int kNv, bool kVec>
__global__ void __launch_bounds__(Group<kTpr>::kThreads) norm_forward_kernel(const Params p) {
  using G = Group<kTpr>;
  __shared__ float2 slots[G::kRpc][2][32];
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int group = threadIdx.x / kTpr, tx = threadIdx.x % kTpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * G::kRpc + group;
  if (row >= p.T) return;  // the whole group leaves
  Raw ry[kNv], rr[kNv], rg[kNv];
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
    const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
    ry[j] = p.y ? load_raw<kVec>(p.y, p.y_dt, row * p.y_stride + col, n) : zero_raw();
    rr[j] = load_raw<kVec>(p.residual, p.res_dt, row * p.res_stride + col, n);
    rg[j] = gate_raw<kVec>(p, row, col, n);
  }
  const float row_gate = p.gate_mode == MOE_GATE_TOKEN ? load_one(p.gate, p.gate_dt, row * p.gate_stride) : 1.f;
  float out[kNv][8];
  if (p.y) {
    float r1 = 1.f;
    if (p.post) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        float v[8];
        to_f32(ry[j], p.y_dt, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) s.x = fmaf(v[i], v[i], s.x);
      }
      s = group_sum<kTpr>(s, slots[group], 0, group, tx);
      r1 = rsqrtf(s.x / static_cast<float>(p.H) + p.eps);
    }
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      float v[8], g[8], w[8];
      to_f32(ry[j], p.y_dt, v);
      to_f32(rr[j], p.res_dt, out[j]);
      gate_f32(p, rg[j], row_gate, g);
      if (p.post) {
        to_f32(load_raw<kVec>(p.post, p.post_dt, col, n), p.post_dt, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r1 * w[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) out[j][i] = fmaf(p.scale * g[i], v[i], out[j][i]);
      // columns past the row hold 0 in v and out
      store_f32<kVec>(p.out, p.res_dt, row * p.H + col, n, out[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kNv; ++j) to_f32(rr[j], p.res_dt, out[j]);
  }
  if (!p.next) return;
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < kNv; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) s.x = fmaf(out[j][i], out[j][i], s.x);
  s = group_sum<kTpr>(s, slots[group], 1, group, tx);
  const float r2 = rsqrtf(s.x / static_cast<float>(p.H) + p.eps);
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
    const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
    float w[8];
    to_f32(load_raw<kVec>(p.next, p.next_dt, col, n), p.next_dt, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = out[j][i] * r2 * w[i];
    store_f32<kVec>(p.normed, p.norm_dt, row * p.H + col, n, w);
  }
}

// A group walks rows blockIdx.x * kRpc + group, + gridDim.x * kRpc, ...; its
// threads keep the column sums of their own columns in registers and write
// them once, as one slab of `part`, so the weights' gradients need no atomics
// and are the same bits in every run.
template <int kTpr, int kNv, bool kVec>
__global__ void __launch_bounds__(Group<kTpr>::kThreads) norm_backward_kernel(const Params p) {
  using G = Group<kTpr>;
  __shared__ float2 slots[G::kRpc][2][32];
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int group = threadIdx.x / kTpr, tx = threadIdx.x % kTpr;
  const float inv_h = 1.f / static_cast<float>(p.H);
  float acc_post[kNv][8], acc_next[kNv][8], acc_gate[kNv][8];
#pragma unroll
  for (int j = 0; j < kNv; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc_post[j][i] = acc_next[j][i] = acc_gate[j][i] = 0.f;
  int slot = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * G::kRpc + group; row < p.T;
       row += static_cast<int64_t>(gridDim.x) * G::kRpc) {
    Raw ry[kNv], rg[kNv], rd[kNv], rn[kNv];
    float out[kNv][8];
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      ry[j] = p.y ? load_raw<kVec>(p.y, p.y_dt, row * p.y_stride + col, n) : zero_raw();
      const Raw rr = load_raw<kVec>(p.residual, p.res_dt, row * p.res_stride + col, n);
      rd[j] = p.d_out ? load_raw<kVec>(p.d_out, p.res_dt, row * p.d_out_stride + col, n) : zero_raw();
      rn[j] = p.d_normed ? load_raw<kVec>(p.d_normed, p.norm_dt, row * p.d_normed_stride + col, n) : zero_raw();
      rg[j] = gate_raw<kVec>(p, row, col, n);
      to_f32(rr, p.res_dt, out[j]);
    }
    const float row_gate = p.gate_mode == MOE_GATE_TOKEN ? load_one(p.gate, p.gate_dt, row * p.gate_stride) : 1.f;
    // ---- recompute r1 and out
    float r1 = 1.f;
    if (p.y && p.post) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        float v[8];
        to_f32(ry[j], p.y_dt, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) s.x = fmaf(v[i], v[i], s.x);
      }
      s = group_sum<kTpr>(s, slots[group], slot, group, tx);
      slot ^= 1;
      r1 = rsqrtf(s.x * inv_h + p.eps);
    }
    float df[kNv][8];
#pragma unroll
    for (int j = 0; j < kNv; ++j) to_f32(rd[j], p.res_dt, df[j]);
    if (p.y && p.d_normed) {
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
        float v[8], g[8], w[8];
        to_f32(ry[j], p.y_dt, v);
        gate_f32(p, rg[j], row_gate, g);
        if (p.post) {
          to_f32(load_raw<kVec>(p.post, p.post_dt, col, n), p.post_dt, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = v[i] * r1 * w[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) out[j][i] = fmaf(p.scale * g[i], v[i], out[j][i]);
      }
    }
    // ---- through the second norm
    if (p.d_normed) {
      float2 s = make_float2(0.f, 0.f);
      float dn[kNv][8];
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
        float w[8];
        to_f32(rn[j], p.norm_dt, dn[j]);
        to_f32(load_raw<kVec>(p.next, p.next_dt, col, n), p.next_dt, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s.x = fmaf(out[j][i], out[j][i], s.x);
          s.y = fmaf(dn[j][i] * w[i], out[j][i], s.y);
        }
      }
      s = group_sum<kTpr>(s, slots[group], slot, group, tx);
      slot ^= 1;
      const float r2 = rsqrtf(s.x * inv_h + p.eps);
      const float c = s.y * inv_h * r2 * r2;
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
        float w[8];
        to_f32(load_raw<kVec>(p.next, p.next_dt, col, n), p.next_dt, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc_next[j][i] = fmaf(dn[j][i], out[j][i] * r2, acc_next[j][i]);
          df[j][i] = fmaf(r2, fmaf(dn[j][i], w[i], -out[j][i] * c), df[j][i]);
        }
      }
    }
    if (p.d_residual) {
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (j * kTpr + tx) * 8;
        store_f32<kVec>(p.d_residual, p.res_dt, row * p.H + col, valid_at(p.H, col), df[j]);
      }
    }
    if (!p.y) continue;
    // ---- through the gate and the first norm
    float2 s = make_float2(0.f, 0.f);
    float dzw[kNv][8];  // dz post (dz without post)
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      float v[8], g[8], w[8], dg[8];
      to_f32(ry[j], p.y_dt, v);
      gate_f32(p, rg[j], row_gate, g);
      if (p.post) {
        to_f32(load_raw<kVec>(p.post, p.post_dt, col, n), p.post_dt, w);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float dz = p.scale * g[i] * df[j][i];
        const float yhat = v[i] * r1;
        dg[i] = p.scale * yhat * w[i] * df[j][i];
        acc_post[j][i] = fmaf(dz, yhat, acc_post[j][i]);
        acc_gate[j][i] += dg[i];
        dzw[j][i] = dz * w[i];
        s.x = fmaf(dzw[j][i], v[i], s.x);
        s.y += dg[i];
      }
      if (p.gate_mode == MOE_GATE_FULL && p.d_gate)
        store_f32<kVec>(p.d_gate, p.gate_dt, row * p.H + col, n, dg);
    }
    float c = 0.f;
    if (p.post || (p.gate_mode == MOE_GATE_TOKEN && p.d_gate)) {
      s = group_sum<kTpr>(s, slots[group], slot, group, tx);
      slot ^= 1;
      if (p.post) c = s.x * inv_h * r1 * r1;
      if (p.gate_mode == MOE_GATE_TOKEN && p.d_gate && tx == 0) store_one(p.d_gate, p.gate_dt, row, s.y);
    }
    if (p.d_y) {
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        const int col = (j * kTpr + tx) * 8;
        float v[8];
        to_f32(ry[j], p.y_dt, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = r1 * fmaf(-v[i], c, dzw[j][i]);
        store_f32<kVec>(p.d_y, p.y_dt, row * p.H + col, valid_at(p.H, col), v);
      }
    }
  }
  if (!p.part) return;
  // join the CTA's groups in order, then one slab per CTA (also one without rows: zeros)
  __shared__ float join[G::kRpc > 1 ? G::kRpc : 1][G::kRpc > 1 ? kTpr * kNv * 8 : 1];
  float* part = p.part + static_cast<int64_t>(blockIdx.x) * 3 * p.H;
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    if (!(which == 0 ? p.want_post : which == 1 ? p.want_next : p.want_gate)) continue;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = which == 0 ? acc_post[j][i] : which == 1 ? acc_next[j][i] : acc_gate[j][i];
      if (G::kRpc > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) join[group][col + i] = v[i];
        __syncthreads();
        if (group == 0) {
          for (int o = 1; o < G::kRpc; ++o)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += join[o][col + i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (group == 0 && i < n) part[static_cast<int64_t>(which) * p.H + col + i] = v[i];
    }
  }
}

struct ReduceParams {
  const float* part;
  void* out[3];  // d_post, d_next, channel d_gate; null to skip
  int dt[3];
  int slabs, H;
};

// Column sums over the slabs: 32 columns per CTA, 8 slab lanes each, joined
// in a fixed order.
__global__ void __launch_bounds__(256) norm_reduce_kernel(const ReduceParams p) {
  __shared__ float sums[8][33];
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int which = blockIdx.y;
  if (!p.out[which]) return;
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < p.H) {
    const float* src = p.part + static_cast<int64_t>(which) * p.H + col;
    const int64_t step = static_cast<int64_t>(3) * p.H;
    int i = part;
    for (; i + 24 < p.slabs; i += 32) {  // four loads in flight
      const float a = src[i * step], b = src[(i + 8) * step], c = src[(i + 16) * step], d = src[(i + 24) * step];
      s += (a + b) + (c + d);
    }
    for (; i < p.slabs; i += 8) s += src[i * step];
  }
  sums[part][lane] = s;
  __syncthreads();
  if (part == 0 && col < p.H) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += sums[w][lane];
    store_one(p.out[which], p.dt[which], col, t);
  }
}

}  // namespace norm
}  // namespace moe

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
// HBM is the floor of both. Forward: 8192 x 2048 bf16 27 us (76% of the floor's
// rate), 1000 x 7168 f32 28 us (64%: two CTAs of 512 threads per SM, 3.4 waves of
// rows whose loads are waited for together). Backward: 63 us for 8192 x 2048 bf16,
// bound by the latency of a row's three sums on 16 warps per SM. A row lives in the registers of one group of threads
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

// The element types of a kernel: fixed (MOE_DT_*), or kAny: read from Params.
// A conversion whose type is only known at run time costs about five
// instructions per value instead of one (the backward of 8192 x 2048 bf16 ran
// 783 instructions per 8 values and thread, 134 us), so the usual combinations
// have kernels of their own.
constexpr int kAny = -1;
template <int kY, int kR, int kN, int kW>
struct Types {
  static constexpr bool kFixed = kY != kAny;
  static __device__ __forceinline__ int y(const Params& p) { return kFixed ? kY : p.y_dt; }
  static __device__ __forceinline__ int res(const Params& p) { return kFixed ? kR : p.res_dt; }
  static __device__ __forceinline__ int norm(const Params& p) { return kFixed ? kN : p.norm_dt; }
  static __device__ __forceinline__ int gate(const Params& p) { return kFixed ? kY : p.gate_dt; }
  static __device__ __forceinline__ int post(const Params& p) { return kFixed ? kW : p.post_dt; }
  static __device__ __forceinline__ int next(const Params& p) { return kFixed ? kW : p.next_dt; }
};
using AnyTypes = Types<kAny, kAny, kAny, kAny>;

// Eight values of a row as they lie in memory: 16 bytes (16-bit types) or 32.
struct Raw {
  uint4 a, b;
};

__device__ __forceinline__ Raw zero_raw() { return Raw{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}; }

// 16 bytes, or zeros. A predicated load instead of a branch, so that several
// arrays' loads are in flight together whatever their types.
__device__ __forceinline__ uint4 load16_if(const void* ptr, bool pred) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.u32 q, %5, 0;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
      "@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(ptr), "r"(pred ? 1u : 0u));
  return v;
}

// Values off .. off+7 of which the first n exist (the rest read as 0). kVec:
// 16-byte aligned and n is 0 or 8. Loads only, no conversion.
template <bool kVec>
__device__ __forceinline__ Raw load_raw(const void* base, int dt, int64_t off, int n) {
  Raw r = zero_raw();
  if (kVec) {
    const bool f32 = dt == MOE_DT_F32;
    const uint8_t* at = static_cast<const uint8_t*>(base) + (off << (f32 ? 2 : 1));
    r.a = load16_if(at, n > 0);
    r.b = load16_if(at + 16, n > 0 && f32);
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

// Two f32 values in one 64-bit register: the packed f32x2 instructions do the
// work of two scalar ones (each half rounded as the scalar one would).
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 both(float v) { return pack(v, v); }
__device__ __forceinline__ void unpack(F2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ float sum2(F2 v) {
  float lo, hi;
  unpack(v, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Eight values as four pairs.
__device__ __forceinline__ void to_pairs(const Raw& r, int dt, F2 (&v)[4]) {
  float f[8];
  to_f32(r, dt, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack(f[2 * i], f[2 * i + 1]);
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

__device__ __forceinline__ int valid_at(int H, int col) {
  const int n = H - col;
  return n < 0 ? 0 : n > 8 ? 8 : n;
}

template <bool kVec>
__device__ __forceinline__ void store_pairs(void* base, int dt, int64_t off, int n, const F2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack(v[i], f[2 * i], f[2 * i + 1]);
  store_f32<kVec>(base, dt, off, n, f);
}

// A row's group: kTpr threads, kRpc groups per CTA.
template <int kTpr>
struct Group {
  static constexpr int kThreads = kTpr < 256 ? 256 : kTpr;
  static constexpr int kRpc = kThreads / kTpr;
  static constexpr int kWarps = kTpr / 32;
};

__device__ __forceinline__ float group_add(float a, float b) { return a + b; }
__device__ __forceinline__ float2 group_add(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ float group_shfl(float v, int d) { return __shfl_xor_sync(0xffffffffu, v, d); }
__device__ __forceinline__ float2 group_shfl(float2 v, int d) {
  return make_float2(group_shfl(v.x, d), group_shfl(v.y, d));
}

// Sum of a value (float, or two in a float2) over the group, in a fixed order. `slot` must
// differ from the slot of the previous call of the same group (two slots
// taken in turn: a warp may still read one while the next is written).
template <int kTpr, typename V>
__device__ __forceinline__ V group_sum(V v, V (*slots)[kTpr / 32], int slot, int group, int tx) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = group_add(v, group_shfl(v, d));
  if (kTpr == 32) return v;
  if ((tx & 31) == 0) slots[slot][tx >> 5] = v;
  named_bar_sync(1 + group, kTpr);
  V s = slots[slot][0];
#pragma unroll
  for (int w = 1; w < kTpr / 32; ++w) s = group_add(s, slots[slot][w]);
  return s;
}

// gate of 8 columns: raw for channel and full modes, one value for a row.
template <class T>
__device__ __forceinline__ void gate_f32(const Params& p, const Raw& raw, float row_gate, float (&g)[8]) {
  if (p.gate_mode == MOE_GATE_CHANNEL || p.gate_mode == MOE_GATE_FULL) {
    to_f32(raw, T::gate(p), g);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = row_gate;
  }
}

template <class T, bool kVec>
__device__ __forceinline__ Raw gate_raw(const Params& p, int64_t row, int col, int n) {
  if (p.gate_mode == MOE_GATE_CHANNEL) return load_raw<kVec>(p.gate, T::gate(p), col, n);
  if (p.gate_mode == MOE_GATE_FULL) return load_raw<kVec>(p.gate, T::gate(p), row * p.gate_stride + col, n);
  return zero_raw();
}

template <class T, int kTpr, int kNv, bool kVec>
__global__ void __launch_bounds__(Group<kTpr>::kThreads, 1024 / Group<kTpr>::kThreads) norm_forward_kernel(const Params p) {
  using G = Group<kTpr>;
  __shared__ float slots[G::kRpc][2][kTpr / 32];
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int group = threadIdx.x / kTpr, tx = threadIdx.x % kTpr;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * G::kRpc + group;
  if (row >= p.T) return;  // the whole group leaves
  const float inv_h = 1.f / static_cast<float>(p.H);
  Raw ry[kNv], rr[kNv], rg[kNv];
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
    const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
    ry[j] = p.y ? load_raw<kVec>(p.y, T::y(p), row * p.y_stride + col, n) : zero_raw();
    rr[j] = load_raw<kVec>(p.residual, T::res(p), row * p.res_stride + col, n);
    rg[j] = gate_raw<T, kVec>(p, row, col, n);
  }
  const float row_gate = p.gate_mode == MOE_GATE_TOKEN ? load_one(p.gate, p.gate_dt, row * p.gate_stride) : 1.f;
  // the weights of one vector are small enough to load ahead of their sums
  Raw rp = zero_raw(), rn = zero_raw();
  if (kNv == 1) {
    const int col = tx * 8, n = valid_at(p.H, col);
    if (p.post) rp = load_raw<kVec>(p.post, T::post(p), col, n);
    if (p.next) rn = load_raw<kVec>(p.next, T::next(p), col, n);
  }
  float out[kNv][8];
  if (p.y) {
    float r1 = 1.f;
    if (p.post) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kNv; ++j) {
        float v[8];
        to_f32(ry[j], T::y(p), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(v[i], v[i], s);
      }
      r1 = rsqrtf(group_sum<kTpr>(s, slots[group], 0, group, tx) * inv_h + p.eps);
    }
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      float v[8], g[8], w[8];
      to_f32(ry[j], T::y(p), v);
      to_f32(rr[j], T::res(p), out[j]);
      gate_f32<T>(p, rg[j], row_gate, g);
      if (p.post) {
        to_f32(kNv == 1 ? rp : load_raw<kVec>(p.post, T::post(p), col, n), T::post(p), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r1 * w[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) out[j][i] = fmaf(p.scale * g[i], v[i], out[j][i]);
      // columns past the row hold 0 in v and out
      store_f32<kVec>(p.out, T::res(p), row * p.H + col, n, out[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kNv; ++j) to_f32(rr[j], T::res(p), out[j]);
  }
  if (!p.next) return;
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < kNv; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(out[j][i], out[j][i], s);
  const float r2 = rsqrtf(group_sum<kTpr>(s, slots[group], 1, group, tx) * inv_h + p.eps);
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
    const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
    float w[8];
    to_f32(kNv == 1 ? rn : load_raw<kVec>(p.next, T::next(p), col, n), T::next(p), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = out[j][i] * r2 * w[i];
    store_f32<kVec>(p.normed, T::norm(p), row * p.H + col, n, w);
  }
}

// ---------------------------------------------------------------- backward
// One row's values as the backward reads them: from registers filled by its
// own loads, or from a stage of shared memory (RingRow).
template <int kTpr, int kNv, bool kVec>
struct LoadedRow {
  const Params& p;
  int tx;
  Raw y_[kNv], res_[kNv], dout_[kNv], dn_[kNv], gate_[kNv];
  __device__ __forceinline__ LoadedRow(const Params& params, int64_t row, int t) : p(params), tx(t) {
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      y_[j] = p.y ? load_raw<kVec>(p.y, p.y_dt, row * p.y_stride + col, n) : zero_raw();
      res_[j] = load_raw<kVec>(p.residual, p.res_dt, row * p.res_stride + col, n);
      dout_[j] = p.d_out ? load_raw<kVec>(p.d_out, p.res_dt, row * p.d_out_stride + col, n) : zero_raw();
      dn_[j] = p.d_normed ? load_raw<kVec>(p.d_normed, p.norm_dt, row * p.d_normed_stride + col, n) : zero_raw();
      gate_[j] = gate_raw<AnyTypes, kVec>(p, row, col, n);
    }
  }
  __device__ __forceinline__ Raw column(const void* base, int dt, int j) const {
    const int col = (j * kTpr + tx) * 8;
    return load_raw<kVec>(base, dt, col, valid_at(p.H, col));
  }
  __device__ __forceinline__ Raw y(int j) const { return y_[j]; }
  __device__ __forceinline__ Raw res(int j) const { return res_[j]; }
  __device__ __forceinline__ Raw dout(int j) const { return dout_[j]; }
  __device__ __forceinline__ Raw dn(int j) const { return dn_[j]; }
  __device__ __forceinline__ Raw gate(int j) const { return gate_[j]; }
  __device__ __forceinline__ Raw post(int j) const { return column(p.post, p.post_dt, j); }
  __device__ __forceinline__ Raw next(int j) const { return column(p.next, p.next_dt, j); }
};

// Columns past the row hold zeros, in the stages as in the weights' copies.
template <class T, int kTpr>
struct RingRow {
  const Params& p;
  const uint8_t* stage;
  const uint8_t* cols;   // the weights' copies
  const int* off;        // of y, residual, d_out, d_normed, full gate in the stage
  const int* col_off;    // of post, next, channel gate
  int tx;
  __device__ __forceinline__ Raw read(const uint8_t* at, int dt, int j) const {
    const uint4* s = reinterpret_cast<const uint4*>(at + (j * kTpr + tx) * (dt == MOE_DT_F32 ? 32 : 16));
    Raw r = zero_raw();
    r.a = s[0];
    if (dt == MOE_DT_F32) r.b = s[1];
    return r;
  }
  __device__ __forceinline__ Raw y(int j) const { return read(stage + off[0], T::y(p), j); }
  __device__ __forceinline__ Raw res(int j) const { return read(stage + off[1], T::res(p), j); }
  __device__ __forceinline__ Raw dout(int j) const { return p.d_out ? read(stage + off[2], T::res(p), j) : zero_raw(); }
  __device__ __forceinline__ Raw dn(int j) const { return read(stage + off[3], T::norm(p), j); }
  __device__ __forceinline__ Raw gate(int j) const {
    if (p.gate_mode == MOE_GATE_CHANNEL) return read(cols + col_off[2], T::gate(p), j);
    return p.gate_mode == MOE_GATE_FULL ? read(stage + off[4], T::gate(p), j) : zero_raw();
  }
  __device__ __forceinline__ Raw post(int j) const { return read(cols + col_off[0], T::post(p), j); }
  __device__ __forceinline__ Raw next(int j) const { return read(cols + col_off[1], T::next(p), j); }
};

// The column sums of a thread's columns over its group's rows.
template <int kNv>
struct Sums {
  F2 post[kNv][4], next[kNv][4], gate[kNv][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kNv; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) post[j][i] = next[j][i] = gate[j][i] = 0ull;  // two zeros
  }
};

// The sums of a group: slots of one and of two values, taken in turn.
template <int kRpc, int kWarps>
struct SumSlots {
  float one[kRpc][2][kWarps];
  float2 two[kRpc][2][kWarps];
};

// Gradients of one row. `slot1`, `slot2` alternate over the rows' sums of each kind.
template <class T, int kTpr, int kNv, bool kVec, typename Row>
__device__ __forceinline__ void backward_row(const Params& p, const Row& in, int64_t row, float row_gate, float inv_h,
                                             float (*one)[kTpr / 32], float2 (*two)[kTpr / 32], int& slot1, int& slot2,
                                             int group, int tx, Sums<kNv>& acc) {
  auto gate_pairs = [&](int j, F2 (&g)[4]) {
    if (p.gate_mode == MOE_GATE_TOKEN) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = both(row_gate);
    } else {
      to_pairs(in.gate(j), T::gate(p), g);
    }
  };
  float r1 = 1.f;
  F2 y[kNv][4];
  if (p.y) {
#pragma unroll
    for (int j = 0; j < kNv; ++j) to_pairs(in.y(j), T::y(p), y[j]);
    if (p.post) {
      F2 s = 0ull;
#pragma unroll
      for (int j = 0; j < kNv; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fma2(y[j][i], y[j][i], s);
      const float t = group_sum<kTpr>(sum2(s), one, slot1, group, tx);
      slot1 ^= 1;
      r1 = rsqrtf(t * inv_h + p.eps);
    }
  }
  F2 df[kNv][4];
  // ---- out again, and through the second norm
  if (p.d_normed) {
    F2 sx = 0ull, sy = 0ull;
    F2 out[kNv][4];
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      F2 v[4], w[4];
      to_pairs(in.res(j), T::res(p), out[j]);
      if (p.y) {
        const F2 ar = both(p.scale * r1);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = mul2(y[j][i], ar);
        if (p.gate_mode != MOE_GATE_NONE) {
          gate_pairs(j, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], w[i]);
        }
        if (p.post) {
          to_pairs(in.post(j), T::post(p), w);
#pragma unroll
          for (int i = 0; i < 4; ++i) out[j][i] = fma2(v[i], w[i], out[j][i]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) out[j][i] = add2(out[j][i], v[i]);
        }
      }
      to_pairs(in.dn(j), T::norm(p), v);
      to_pairs(in.next(j), T::next(p), w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        df[j][i] = mul2(v[i], w[i]);
        sx = fma2(out[j][i], out[j][i], sx);
        sy = fma2(df[j][i], out[j][i], sy);
      }
    }
    const float2 s = group_sum<kTpr>(make_float2(sum2(sx), sum2(sy)), two, slot2, group, tx);
    slot2 ^= 1;
    const float r2 = rsqrtf(s.x * inv_h + p.eps);
    const F2 rr = both(r2), c = both(-s.y * inv_h * r2 * r2);
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      F2 v[4], d[4];
      to_pairs(in.dn(j), T::norm(p), v);
      to_pairs(in.dout(j), T::res(p), d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc.next[j][i] = fma2(v[i], mul2(out[j][i], rr), acc.next[j][i]);
        df[j][i] = fma2(rr, fma2(out[j][i], c, df[j][i]), d[i]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kNv; ++j) to_pairs(in.dout(j), T::res(p), df[j]);
  }
  if (p.d_residual) {
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8;
      store_pairs<kVec>(p.d_residual, T::res(p), row * p.H + col, valid_at(p.H, col), df[j]);
    }
  }
  if (!p.y) return;
  // ---- through the gate and the first norm; df becomes a dfull, then dz post
  F2 sx = 0ull, sy = 0ull;
  const F2 a = both(p.scale), rr = both(r1);
#pragma unroll
  for (int j = 0; j < kNv; ++j) {
    F2 w[4], yhat[4];
    if (p.post) {
      to_pairs(in.post(j), T::post(p), w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = both(1.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      df[j][i] = mul2(df[j][i], a);
      yhat[i] = mul2(y[j][i], rr);
    }
    if (p.gate_mode != MOE_GATE_NONE) {
      F2 g[4], dg[4];
      gate_pairs(j, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dg[i] = mul2(mul2(yhat[i], w[i]), df[j][i]);
        df[j][i] = mul2(df[j][i], g[i]);
      }
      if (p.gate_mode == MOE_GATE_CHANNEL) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc.gate[j][i] = add2(acc.gate[j][i], dg[i]);
      } else if (p.gate_mode == MOE_GATE_TOKEN) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sy = add2(sy, dg[i]);
      } else if (p.d_gate) {
        const int col = (j * kTpr + tx) * 8;
        store_pairs<kVec>(p.d_gate, T::gate(p), row * p.H + col, valid_at(p.H, col), dg);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc.post[j][i] = fma2(df[j][i], yhat[i], acc.post[j][i]);
      df[j][i] = mul2(df[j][i], w[i]);
      sx = fma2(df[j][i], y[j][i], sx);
    }
  }
  float c = 0.f;
  if (p.post || (p.gate_mode == MOE_GATE_TOKEN && p.d_gate)) {
    const float2 s = group_sum<kTpr>(make_float2(sum2(sx), sum2(sy)), two, slot2, group, tx);
    slot2 ^= 1;
    if (p.post) c = s.x * inv_h * r1 * r1;
    if (p.gate_mode == MOE_GATE_TOKEN && p.d_gate && tx == 0) store_one(p.d_gate, T::gate(p), row, s.y);
  }
  if (p.d_y) {
    const F2 nc = both(-c);
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) df[j][i] = mul2(rr, fma2(y[j][i], nc, df[j][i]));
      store_pairs<kVec>(p.d_y, T::y(p), row * p.H + col, valid_at(p.H, col), df[j]);
    }
  }
}

// Joins the CTA's groups in order and writes one slab of `part` (also for a
// CTA without rows: zeros), so the weights' gradients need no atomics and are
// the same bits in every run. All threads of the CTA call it.
template <int kTpr, int kNv, int kRpc>
__device__ __forceinline__ void write_sums(const Params& p, const Sums<kNv>& acc, int group, int tx,
                                           float* join) {
  float* part = p.part + static_cast<int64_t>(blockIdx.x) * 3 * p.H;
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    if (!(which == 0 ? p.want_post : which == 1 ? p.want_next : p.want_gate)) continue;
#pragma unroll
    for (int j = 0; j < kNv; ++j) {
      const int col = (j * kTpr + tx) * 8, n = valid_at(p.H, col);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        unpack(which == 0 ? acc.post[j][i] : which == 1 ? acc.next[j][i] : acc.gate[j][i], v[2 * i], v[2 * i + 1]);
      if (kRpc > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) join[(group * kTpr + tx) * 8 + i] = v[i];
        __syncthreads();
        if (group == 0) {
          for (int o = 1; o < kRpc; ++o)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += join[(o * kTpr + tx) * 8 + i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (group == 0 && i < n) part[static_cast<int64_t>(which) * p.H + col + i] = v[i];
    }
  }
}

// A group walks rows blockIdx.x * kRpc + group, + gridDim.x * kRpc, ...; its
// threads keep the column sums of their own columns in registers. This form
// loads each row when it comes to it: for rows of any alignment and mix of
// types, and rows too wide for the ring below.
template <int kTpr, int kNv, bool kVec>
__global__ void __launch_bounds__(Group<kTpr>::kThreads) norm_backward_kernel(const Params p) {
  using G = Group<kTpr>;
  using T = AnyTypes;
  __shared__ SumSlots<G::kRpc, kTpr / 32> slots;
  __shared__ float join[G::kRpc > 1 ? G::kThreads * 8 : 1];
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int group = threadIdx.x / kTpr, tx = threadIdx.x % kTpr;
  const float inv_h = 1.f / static_cast<float>(p.H);
  Sums<kNv> acc;
  acc.clear();
  int slot1 = 0, slot2 = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * G::kRpc + group; row < p.T;
       row += static_cast<int64_t>(gridDim.x) * G::kRpc) {
    const LoadedRow<kTpr, kNv, kVec> in(p, row, tx);
    const float row_gate = p.gate_mode == MOE_GATE_TOKEN ? load_one(p.gate, p.gate_dt, row * p.gate_stride) : 1.f;
    backward_row<T, kTpr, kNv, kVec>(p, in, row, row_gate, inv_h, slots.one[group], slots.two[group], slot1, slot2,
                                    group, tx, acc);
  }
  if (p.part) write_sums<kTpr, kNv, G::kRpc>(p, acc, group, tx, join);
}

// The ring form: one CTA of 512 threads per SM (128 registers a thread), whose
// groups share a copy of the weights in shared memory.
template <int kTpr>
struct RingGroup {
  static constexpr int kThreads = 512;
  static constexpr int kRpc = kThreads / kTpr;
};
constexpr int kRingStages = 3;

struct RingParams {
  Params p;
  int32_t* status;
  int off[5];       // y, residual, d_out, d_normed, full gate in a stage
  int row_bytes[5];  // 0: absent
  int stage_bytes;
  int stages;
  int col_off[3];    // post, next, channel gate, behind the stages
  int col_bytes[3];  // 0: absent
  int col_slot[3];   // bytes with the columns past the row
};

// The same walk with the rows' bytes brought by bulk copies, `stages` - 1 rows
// ahead: the arithmetic of a row (three sums over the group, each with its
// latency) then never waits for HBM, and the arrays are read from shared
// memory where they are used instead of living in registers.
template <class T, int kTpr, int kNv>
__global__ void __launch_bounds__(RingGroup<kTpr>::kThreads, 1)
    norm_backward_ring_kernel(const __grid_constant__ RingParams rp) {
  using G = RingGroup<kTpr>;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ SumSlots<G::kRpc, kTpr / 32> slots;
  __shared__ uint64_t full[G::kRpc][kRingStages];
  __shared__ int abort_word;
  const Params& p = rp.p;
  const int group = threadIdx.x / kTpr, tx = threadIdx.x % kTpr;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int g = 0; g < G::kRpc; ++g)
      for (int s = 0; s < rp.stages; ++s) mbar_init(&full[g][s], 1);
    abort_word = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();  // before the first global memory access
  volatile int* abort_flag = &abort_word;
  const float inv_h = 1.f / static_cast<float>(p.H);
  const int64_t step = static_cast<int64_t>(gridDim.x) * G::kRpc;
  uint8_t* mine = ring + group * rp.stages * rp.stage_bytes;
  if (p.H < kTpr * kNv * 8) {  // columns past the rows: zeros that no copy touches
    for (int s = 0; s < rp.stages; ++s)
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int end = (i < 4 ? rp.off[i + 1] : rp.stage_bytes);
        for (int b = rp.off[i] + rp.row_bytes[i] + tx * 16; b < end; b += kTpr * 16)
          *reinterpret_cast<uint4*>(mine + s * rp.stage_bytes + b) = make_uint4(0, 0, 0, 0);
      }
  }
  auto issue = [&](int64_t row, int s) {
    uint8_t* dst = mine + s * rp.stage_bytes;
    uint32_t bytes = 0;
#pragma unroll
    for (int i = 0; i < 5; ++i) bytes += rp.row_bytes[i];
    mbar_arrive_expect_tx(&full[group][s], bytes);
    auto copy = [&](int i, const void* base, int dt, int64_t stride) {
      if (rp.row_bytes[i])
        bulk_load(dst + rp.off[i], static_cast<const uint8_t*>(base) + (row * stride << (dt == MOE_DT_F32 ? 2 : 1)),
                  rp.row_bytes[i], &full[group][s]);
    };
    copy(0, p.y, T::y(p), p.y_stride);
    copy(1, p.residual, T::res(p), p.res_stride);
    copy(2, p.d_out, T::res(p), p.d_out_stride);
    copy(3, p.d_normed, T::norm(p), p.d_normed_stride);
    copy(4, p.gate, T::gate(p), p.gate_stride);
  };
  Sums<kNv> acc;
  acc.clear();
  int slot1 = 0, slot2 = 0;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * G::kRpc + group;
  if (tx == 0)
    for (int s = 0; s < rp.stages && row0 + s * step < p.T; ++s) issue(row0 + s * step, s);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint8_t* src = static_cast<const uint8_t*>(i == 0 ? p.post : i == 1 ? p.next : p.gate);
    for (int b = threadIdx.x * 16; b < rp.col_slot[i]; b += G::kThreads * 16)
      *reinterpret_cast<uint4*>(ring + rp.col_off[i] + b) =
          b < rp.col_bytes[i] ? *reinterpret_cast<const uint4*>(src + b) : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t row = row0; row < p.T; row += step) {
    const bool got = wait_parity_bounded(&full[group][stage], phase, abort_flag, rp.status);
    // the group goes on together or not at all; past this point its threads
    // have also finished the row before, whose stage can be filled again
    ok = kTpr == 32 ? __all_sync(0xffffffffu, got) : named_bar_and(1 + group, kTpr, got);
    if (!ok) break;
    const int64_t ahead = row + (rp.stages - 1) * step;
    if (rp.stages > 1 && tx == 0 && row != row0 && ahead < p.T) issue(ahead, stage == 0 ? rp.stages - 1 : stage - 1);
    const float row_gate = p.gate_mode == MOE_GATE_TOKEN ? load_one(p.gate, p.gate_dt, row * p.gate_stride) : 1.f;
    const RingRow<T, kTpr> in{p, mine + stage * rp.stage_bytes, ring, rp.off, rp.col_off, tx};
    backward_row<T, kTpr, kNv, true>(p, in, row, row_gate, inv_h, slots.one[group], slots.two[group], slot1, slot2,
                                    group, tx, acc);
    if (++stage == rp.stages) { stage = 0; phase ^= 1u; }
    if (rp.stages == 1 && row + step < p.T) {  // wide f32 rows: one at a time
      if (kTpr == 32) __syncwarp();
      else named_bar_sync(1 + group, kTpr);
      if (tx == 0) issue(row + step, 0);
    }
  }
  if (!ok && tx == 0) {
    // let every copy in flight land before the CTA exits
    const uint64_t t0 = globaltimer_ns();
    for (int i = 0; i < rp.stages; ++i) {
      while (!mbar_try_wait(&full[group][stage], phase) && globaltimer_ns() - t0 < 100000000ull) {
      }
      if (++stage == rp.stages) { stage = 0; phase ^= 1u; }
    }
  }
  // the stages are done with: their memory joins the groups' sums
  if (p.part) write_sums<kTpr, kNv, G::kRpc>(p, acc, group, tx, reinterpret_cast<float*>(ring));
}

struct ReduceParams {
  const float* part;
  void* out[3];  // d_post, d_next, channel d_gate; null to skip
  int dt[3];
  int slabs, H;
};

// Column sums over the slabs: 32 columns per CTA, 32 slab lanes of four loads
// in flight each, joined in a fixed order.
constexpr int kReduceThreads = 1024;

__global__ void __launch_bounds__(kReduceThreads) norm_reduce_kernel(const __grid_constant__ ReduceParams p) {
  constexpr int kLanes = kReduceThreads / 32;
  __shared__ float sums[kLanes][33];
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  const int which = blockIdx.y;
  void* out = which == 0 ? p.out[0] : which == 1 ? p.out[1] : p.out[2];
  if (!out) return;
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < p.H) {
    const float* src = p.part + static_cast<int64_t>(which) * p.H + col;
    const int64_t step = static_cast<int64_t>(3) * p.H;
    for (int i = part; i < p.slabs; i += 4 * kLanes) {
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = i + u * kLanes < p.slabs ? src[(i + u * kLanes) * step] : 0.f;
      s += (v[0] + v[1]) + (v[2] + v[3]);
    }
  }
  sums[part][lane] = s;
  __syncthreads();
  if (part == 0 && col < p.H) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kLanes; ++w) t += sums[w][lane];
    store_one(out, which == 0 ? p.dt[0] : which == 1 ? p.dt[1] : p.dt[2], col, t);
  }
}

}  // namespace norm
}  // namespace moe

// Tokens sorted by expert and back, with their gradients. With pos[f] the
// grouped row of flat slot f = t k + s (grouping.py; -1: the slot has no row):
//
//   permute            xs[pos[f]] = x[t]
//   unpermute          out[t]     = sum_s w[f] rows[pos[f]] (+ shared[t])
//                      (the combine; with w = 1 the gradient of permute)
//   combine backward   dy[pos[f]] = w[f] dout[t],   dw[f] = <dout[t], y[pos[f]]>
//
// HBM is the floor of all three: a token's row is read or written once and its
// k grouped rows once. A CTA takes one token and 8 columns per thread and step,
// so the k rows' loads or stores of a step are in flight together (16-bit rows;
// f32 rows one at a time). 4096 tokens, k 6, 2048 columns, bf16: permute 19 us,
// combine 28, its gradient 47, permute's 25, at 37 to 53% of HBM's peak; what
// is left is latency, of loads and of one token's work between barriers, and
// conversions whose types are only known at run time. Every output element has one writer; sums run
// over slots in order, in f32 and rounded once; dw's sum over H is f32 in a
// fixed order. Rows that no slot owns (at and after offsets[E]) are written as
// zeros by permute and combine backward, since they are gradients or inputs
// of a product over all rows.
#pragma once
#include "combine.cuh"
#include "norm.cuh"

namespace moe {
namespace permute {

constexpr int kMaxThreads = 256;
constexpr int kMaxK = combine::kMaxK;
constexpr int kSlots = 8;  // slots handled together in the combine backward

struct Params {
  const void* x;     // (T, H): x, dout, or the shared rows
  const void* rows;  // (T*k, H): the rows summed, or y (combine backward; unused without dw)
  void* out_rows;    // (T*k, H): xs, or dy
  void* out;         // (T, H)
  const int32_t* pos;
  const void* w;     // (T*k) in w_dt
  void* dw;
  const int32_t* n_rows;  // offsets + E: rows in use
  int32_t* status;
  int64_t T, H;
  int64_t x_stride, rows_stride;  // elements between rows
  int k;
  int x_dt, rows_dt, out_dt, w_dt;  // out_dt: out, or dy
};

// Grouped row of slot f, or -1; a corrupted position raises the status.
__device__ __forceinline__ int row_of(const Params& p, int64_t f) {
  const int r = p.pos[f];
  if (r < 0) return -1;
  if (r >= p.T * p.k) {
    if (p.status) atomicCAS(p.status, 0, MOE_ERR_BAD_OFFSETS);
    return -1;
  }
  return r;
}

// Zeros the rows that no slot owns: rows n_rows .. T*k-1, spread over the CTAs.
__device__ __forceinline__ void zero_tail(const Params& p, void* rows, int elem) {
  const int64_t all = p.T * p.k;
  int64_t used = *p.n_rows;
  used = used < 0 ? 0 : used;
  const int64_t vecs = p.H * elem / 16;
  for (int64_t r = used + blockIdx.x; r < all; r += gridDim.x) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(rows) + r * p.H * elem);
    for (int64_t v = threadIdx.x; v < vecs; v += blockDim.x) dst[v] = make_uint4(0, 0, 0, 0);
  }
}

// One CTA per token: 16-byte pieces of the row, read once, stored k times.
__global__ void __launch_bounds__(kMaxThreads) permute_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  __shared__ int row[kMaxK];
  const int64_t t = blockIdx.x;
  if (threadIdx.x < p.k) row[threadIdx.x] = row_of(p, t * p.k + threadIdx.x);
  const int elem = p.x_dt == MOE_DT_F32 ? 4 : 2;
  const int64_t vecs = p.H * elem / 16;
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.x) + t * p.x_stride * elem);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (threadIdx.x < vecs) v = src[threadIdx.x];
  __syncthreads();
  for (int64_t i = threadIdx.x; i < vecs; i += blockDim.x) {
    uint4 next = make_uint4(0, 0, 0, 0);
    if (i + blockDim.x < vecs) next = src[i + blockDim.x];
    for (int s = 0; s < p.k; ++s)
      if (row[s] >= 0) reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out_rows) + row[s] * p.H * elem)[i] = v;
    v = next;
  }
  zero_tail(p, p.out_rows, elem);
}

// One CTA per token: the slots' rows of 8 columns, summed in slot order.
// kWeighted: times w.
template <bool kWeighted>
__global__ void __launch_bounds__(kMaxThreads) unpermute_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  __shared__ int row[kMaxK];
  __shared__ float weight[kMaxK];
  const int64_t t = blockIdx.x;
  if (threadIdx.x < p.k) {
    row[threadIdx.x] = row_of(p, t * p.k + threadIdx.x);
    if (kWeighted) weight[threadIdx.x] = norm::load_one(p.w, p.w_dt, t * p.k + threadIdx.x);
  }
  __syncthreads();
  for (int64_t h = threadIdx.x * 8; h < p.H; h += blockDim.x * 8) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto add = [&](int s, const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = kWeighted ? fmaf(weight[s], v[i], acc[i]) : acc[i] + v[i];
    };
    if (p.rows_dt == MOE_DT_F32) {
      for (int s = 0; s < p.k; ++s) {
        if (row[s] < 0) continue;
        float v[8];
        combine::load8(p.rows, p.rows_dt, row[s] * p.rows_stride + h, v);
        add(s, v);
      }
    } else {
      for (int s0 = 0; s0 < p.k; s0 += kSlots) {
        uint4 raw[kSlots];
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          raw[j] = make_uint4(0, 0, 0, 0);
          if (s0 + j < p.k && row[s0 + j] >= 0) raw[j] = combine::load_raw16(p.rows, row[s0 + j] * p.rows_stride + h);
        }
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          if (s0 + j >= p.k) break;
          if (row[s0 + j] < 0) continue;
          float v[8];
          combine::unpack8(raw[j], p.rows_dt, v);
          add(s0 + j, v);
        }
      }
    }
    if (p.x) {
      float v[8];
      combine::load8(p.x, p.x_dt, t * p.x_stride + h, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += v[i];
    }
    combine::store8(p.out, p.out_dt, t * p.H + h, acc);
  }
}

// One CTA per token. kDw: also dw, from y's rows; without it only dout is read.
template <bool kDw>
__global__ void __launch_bounds__(kMaxThreads) combine_backward_kernel(const Params p) {
  pdl_trigger();
  pdl_wait();  // before the first global memory access
  __shared__ int row[kMaxK];
  __shared__ float weight[kMaxK];
  __shared__ float sums[kMaxThreads / 32][kMaxK];
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < p.k) {
    row[threadIdx.x] = row_of(p, t * p.k + threadIdx.x);
    weight[threadIdx.x] = norm::load_one(p.w, p.w_dt, t * p.k + threadIdx.x);
  }
  __syncthreads();
  for (int s0 = 0; s0 < p.k; s0 += kSlots) {
    float dot[kSlots];
#pragma unroll
    for (int j = 0; j < kSlots; ++j) dot[j] = 0.f;
    for (int64_t h = threadIdx.x * 8; h < p.H; h += blockDim.x * 8) {
      uint4 raw[kSlots];
      const bool y16 = kDw && p.rows_dt != MOE_DT_F32;
      if (y16) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          raw[j] = make_uint4(0, 0, 0, 0);
          if (s0 + j < p.k && row[s0 + j] >= 0) raw[j] = combine::load_raw16(p.rows, row[s0 + j] * p.rows_stride + h);
        }
      }
      float d[8];
      combine::load8(p.x, p.x_dt, t * p.x_stride + h, d);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (s0 + j >= p.k || row[s0 + j] < 0) continue;
        float v[8];
        if (kDw) {
          if (y16) combine::unpack8(raw[j], p.rows_dt, v);
          else combine::load8(p.rows, p.rows_dt, row[s0 + j] * p.rows_stride + h, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) dot[j] = fmaf(d[i], v[i], dot[j]);
        }
        if (p.out_rows) {
          const float ws = weight[s0 + j];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = ws * d[i];
          combine::store8(p.out_rows, p.out_dt, row[s0 + j] * p.H + h, v);
        }
      }
    }
    if (kDw) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
        if (lane == 0 && s0 + j < p.k) sums[warp][s0 + j] = dot[j];
      }
    }
  }
  if (kDw) {
    __syncthreads();
    if (threadIdx.x < p.k) {
      float s = 0.f;
      for (int w = 0; w < static_cast<int>(blockDim.x / 32); ++w) s += sums[w][threadIdx.x];
      norm::store_one(p.dw, p.w_dt, t * p.k + threadIdx.x, s);  // a slot without a row contributes nothing: 0
    }
  }
  if (p.out_rows) zero_tail(p, p.out_rows, p.out_dt == MOE_DT_F32 ? 4 : 2);
}

}  // namespace permute
}  // namespace moe

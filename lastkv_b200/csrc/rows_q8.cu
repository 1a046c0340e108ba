// Rows to int8 with fp32 group scales (sm_100a): the activations of the products with
// 4-bit weights (w4.cu).  A row's K columns are cut into groups of G = 32, 64 or 128
// (the last may be short); with y the row's fp32 values, a group keeps
//   s = max|y| / 127,   q = rne(y / s)   (all zero where s = 0)
// and stands for q * s.  Three sources of y, none of them rounded before q:
//   norm   h = x + residual (fp32; residual_out = bf16(h)),
//          y = h * rsqrt(mean(h^2) + eps) * weight
//   silu   y = g / (1 + exp(-g)) * u          for a [gate | up] row
//   plain  y = x
// A group that holds an infinity or a NaN gets that scale and zeros: its values are NaN.
//
// Group maxima compare the bit patterns of |y|, which order like the values and put
// NaN on top.  The quotient is y * (127 / max), one division per group; a group whose
// maximum is below 1e-30 divides by s instead, where the reciprocal would overflow.

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace lkv {

namespace {

constexpr int kVec = 8;  // columns per lane: one 16-byte load

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16_lo(w[i]);
    f[2 * i + 1] = bf16_hi(w[i]);
  }
}

// Group scale and quantised values of this lane's 8 columns; `lanes` = G / 8 neighbouring
// lanes share a group.  The whole warp calls it.  Returns the 8 int8 values, packed.
__device__ __forceinline__ uint2 quantise8(const float* y, int lanes, float* scale) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kVec; ++j) top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
  for (int o = lanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float amax = __uint_as_float(top);
  const float s = amax / 127.0f;
  *scale = s;
  int q[kVec];
  if (top >= 0x7f800000u || s == 0.f) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) q[j] = 0;
  } else if (amax >= 1e-30f) {
    const float inv = 127.0f / amax;
#pragma unroll
    for (int j = 0; j < kVec; ++j) q[j] = __float2int_rn(y[j] * inv);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) q[j] = max(-127, min(127, __float2int_rn(y[j] / s)));
  }
  uint2 r;
  r.x = (q[0] & 0xff) | (q[1] & 0xff) << 8 | (q[2] & 0xff) << 16 | (uint32_t)q[3] << 24;
  r.y = (q[4] & 0xff) | (q[5] & 0xff) << 8 | (q[6] & 0xff) << 16 | (uint32_t)q[7] << 24;
  return r;
}

struct NormQ8Params {
  const __nv_bfloat16* x;
  int64_t x_row;
  const __nv_bfloat16* residual;
  int64_t residual_row;
  __nv_bfloat16* residual_out;
  int64_t residual_out_row;
  const __nv_bfloat16* weight;
  int8_t* q;
  int64_t q_row;
  float* scale;
  int64_t scale_row;
  int hidden, group;
  float eps;
};

// One CTA per row, the row in registers (V vectors of 8 columns per thread): one pass
// over memory, one barrier for the sum of squares.
template <int V>
__global__ void __launch_bounds__(V <= 2 ? 1024 : 512) rmsnorm_q8_kernel(const NormQ8Params p) {
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  const int nvec = p.hidden / kVec;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint4* w4 = reinterpret_cast<const uint4*>(p.weight);
  uint4 wv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {  // the weight does not depend on the previous kernel
    const int c = threadIdx.x + i * blockDim.x;
    wv[i] = c < nvec ? w4[c] : zero;
  }
  pdl_wait();
  const uint4* x = reinterpret_cast<const uint4*>(p.x + row * p.x_row);
  const uint4* r = p.residual ? reinterpret_cast<const uint4*>(p.residual + row * p.residual_row) : nullptr;
  float h[V][kVec];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    unpack8(c < nvec ? x[c] : zero, h[i]);
    if (r && c < nvec) {
      float rv[kVec];
      unpack8(r[c], rv);
#pragma unroll
      for (int j = 0; j < kVec; ++j) h[i][j] += rv[j];
      reinterpret_cast<uint4*>(p.residual_out + row * p.residual_out_row)[c] =
          make_uint4(pack_bf16(h[i][0], h[i][1]), pack_bf16(h[i][2], h[i][3]), pack_bf16(h[i][4], h[i][5]),
                     pack_bf16(h[i][6], h[i][7]));
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) ss = fmaf(h[i][j], h[i][j], ss);
  }
  __shared__ float red[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  const float rs = 1.0f / sqrtf(ss / (float)p.hidden + p.eps);
  const int lanes = p.group / kVec;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    float w[kVec], y[kVec], s;
    unpack8(wv[i], w);
#pragma unroll
    for (int j = 0; j < kVec; ++j) y[j] = h[i][j] * rs * w[j];
    const uint2 q = quantise8(y, lanes, &s);
    if (c < nvec) {
      *reinterpret_cast<uint2*>(p.q + row * p.q_row + (int64_t)c * kVec) = q;
      if ((c & (lanes - 1)) == 0) p.scale[row * p.scale_row + c / lanes] = s;
    }
  }
}

// One warp per 256 columns of a row (whole groups), one 8-column vector per lane.
template <bool SILU>
__global__ void __launch_bounds__(256)
    rows_q8_kernel(const __nv_bfloat16* __restrict__ x, int64_t x_row, int8_t* __restrict__ q, int64_t q_row,
                   float* __restrict__ scale, int64_t scale_row, int64_t rows, int cols, int group) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, lanes = group / kVec, nvec = cols / kVec;
  const int chunks = (cols + 255) / 256;
  const int64_t total = rows * chunks;
  for (int64_t i = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5); i < total;
       i += (int64_t)gridDim.x * (blockDim.x >> 5)) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks) * 32 + lane;
    const uint4* src = reinterpret_cast<const uint4*>(x + row * x_row);
    float y[kVec], s;
    unpack8(c < nvec ? src[c] : make_uint4(0, 0, 0, 0), y);
    if (SILU) {
      float u[kVec];
      unpack8(c < nvec ? src[nvec + c] : make_uint4(0, 0, 0, 0), u);
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = y[j] / (1.0f + expf(-y[j])) * u[j];
    }
    const uint2 v = quantise8(y, lanes, &s);
    if (c < nvec) {
      *reinterpret_cast<uint2*>(q + row * q_row + (int64_t)c * kVec) = v;
      if ((c & (lanes - 1)) == 0) scale[row * scale_row + c / lanes] = s;
    }
  }
}

__global__ void __launch_bounds__(256)
    dequantize_q8_kernel(const int8_t* __restrict__ q, int64_t q_row, const float* __restrict__ scale,
                         int64_t scale_row, __nv_bfloat16* __restrict__ out, int64_t out_row, int64_t rows, int cols,
                         int group) {
  pdl_launch_dependents();
  pdl_wait();
  const int nvec = cols / kVec;
  const int64_t total = rows * nvec;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / nvec;
    const int c = (int)(i - row * nvec) * kVec;
    const uint2 v = *reinterpret_cast<const uint2*>(q + row * q_row + c);
    const float s = scale[row * scale_row + c / group];
    float f[kVec];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = (float)(int8_t)(v.x >> (8 * j)) * s;
      f[j + 4] = (float)(int8_t)(v.y >> (8 * j)) * s;
    }
    *reinterpret_cast<uint4*>(out + row * out_row + c) =
        make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
}

// `count` rows at p, `row` elements apart (a single row has no distance to speak of)
bool rows_ok(const void* p, int64_t count, int64_t row, int64_t cols, int elem, int align) {
  return p && (reinterpret_cast<uintptr_t>(p) % align) == 0 &&
         (count == 1 || (row >= cols && (row * elem) % align == 0));
}

bool q8_ok(const Q8RowsArgs& a) {
  return rows_ok(a.q, a.rows, a.q_row, a.cols, 1, 8) && rows_ok(a.scale, a.rows, a.scale_row, (a.cols + a.group - 1) / a.group, 4, 4);
}

int q8_shape(const Q8RowsArgs& a) {
  if (a.group != 32 && a.group != 64 && a.group != 128) return LKV_ERR_UNSUPPORTED;
  if (a.rows < 0 || a.rows > 0x7fffffff || a.cols <= 0 || a.cols % kVec) return LKV_ERR_INVALID_ARGUMENT;
  return LKV_OK;
}

// CTAs of 256 threads for `warps` warps of work: at most 16 waves of a full GPU, then strides.
int row_blocks(int64_t warps) { return (int)std::max<int64_t>(1, std::min<int64_t>((warps + 7) / 8, 148 * 8 * 16)); }

}  // namespace

int rmsnorm_q8(const void* x, int64_t x_row, const void* residual, int64_t residual_row, void* residual_out,
               int64_t residual_out_row, const void* weight, float eps, const Q8RowsArgs& a, cudaStream_t stream) {
  const int st = q8_shape(a);
  if (st != LKV_OK) return st;
  if (a.cols > 512 * 8 * kVec) return LKV_ERR_UNSUPPORTED;
  if (a.rows == 0) return LKV_OK;
  if (!rows_ok(x, a.rows, x_row, a.cols, 2, 16) || !rows_ok(weight, 1, a.cols, a.cols, 2, 16) || !q8_ok(a))
    return LKV_ERR_INVALID_ARGUMENT;
  if (residual && (!rows_ok(residual, a.rows, residual_row, a.cols, 2, 16) ||
                   !rows_ok(residual_out, a.rows, residual_out_row, a.cols, 2, 16)))
    return LKV_ERR_INVALID_ARGUMENT;
  NormQ8Params p{static_cast<const __nv_bfloat16*>(x),
                 x_row,
                 static_cast<const __nv_bfloat16*>(residual),
                 residual_row,
                 static_cast<__nv_bfloat16*>(residual_out),
                 residual_out_row,
                 static_cast<const __nv_bfloat16*>(weight),
                 a.q,
                 a.q_row,
                 a.scale,
                 a.scale_row,
                 a.cols,
                 a.group,
                 eps};
  const int nvec = a.cols / kVec;
  const int v = nvec <= 1024 ? 1 : nvec <= 2048 ? 2 : 8;
  const int threads = ((nvec + v - 1) / v + 31) / 32 * 32;
  void (*kernel)(const NormQ8Params) = v == 1   ? rmsnorm_q8_kernel<1>
                                       : v == 2 ? rmsnorm_q8_kernel<2>
                                                : rmsnorm_q8_kernel<8>;
  return launch_pdl(kernel, dim3((unsigned)a.rows), dim3(threads), 0, stream, p) == cudaSuccess ? LKV_OK
                                                                                                 : LKV_ERR_CUDA;
}

int rows_q8(const void* x, int64_t x_row, int silu, const Q8RowsArgs& a, cudaStream_t stream) {
  const int st = q8_shape(a);
  if (st != LKV_OK) return st;
  if (a.rows == 0) return LKV_OK;
  if (!rows_ok(x, a.rows, x_row, silu ? 2 * (int64_t)a.cols : a.cols, 2, 16) || !q8_ok(a)) return LKV_ERR_INVALID_ARGUMENT;
  const int blocks = row_blocks(a.rows * ((a.cols + 255) / 256));
  return launch_pdl(silu ? rows_q8_kernel<true> : rows_q8_kernel<false>, dim3(blocks), dim3(256), 0, stream,
                    static_cast<const __nv_bfloat16*>(x), x_row, a.q, a.q_row, a.scale, a.scale_row, a.rows, a.cols,
                    a.group) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

int dequantize_q8(const Q8RowsArgs& a, void* out, int64_t out_row, cudaStream_t stream) {
  const int st = q8_shape(a);
  if (st != LKV_OK) return st;
  if (a.rows == 0) return LKV_OK;
  if (!q8_ok(a) || !rows_ok(out, a.rows, out_row, a.cols, 2, 16)) return LKV_ERR_INVALID_ARGUMENT;
  const int blocks = row_blocks((a.rows * (a.cols / kVec) + 31) / 32);
  return launch_pdl(dequantize_q8_kernel, dim3(blocks), dim3(256), 0, stream, static_cast<const int8_t*>(a.q),
                    a.q_row, static_cast<const float*>(a.scale), a.scale_row, static_cast<__nv_bfloat16*>(out),
                    out_row, a.rows, a.cols, a.group) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

}  // namespace lkv

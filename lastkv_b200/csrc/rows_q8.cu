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
// The quotient is y * (127 / max), one division per group, rounded to the integer by the
// addition that puts it into the low byte of 1.5 * 2^23 + q (no conversion instruction, which
// runs at an eighth of the rate); a group whose maximum is below 1e-30 divides by s instead,
// where the reciprocal would overflow.

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

// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Group scale and quantised values of this lane's 8 columns; `lanes` = G / 8 neighbouring
// lanes share a group.  The whole warp calls it.  Returns the 8 int8 values, packed.
__device__ __forceinline__ uint2 quantise8(const float* y, int lanes, float* scale) {
  float amax = fabsf(y[0]);
#pragma unroll
  for (int j = 1; j < kVec; ++j) amax = max_nan(amax, fabsf(y[j]));
  for (int o = lanes >> 1; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float s = amax / 127.0f;
  *scale = s;
  if (!(amax < INFINITY) || s == 0.f) return make_uint2(0, 0);
  uint32_t q[kVec];
  if (amax >= 1e-30f) {
    const float inv = 127.0f / amax;
#pragma unroll
    for (int j = 0; j < kVec; ++j) q[j] = __float_as_uint(fmaf(y[j], inv, 12582912.0f));
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) q[j] = (uint32_t)max(-127, min(127, __float2int_rn(y[j] / s)));
  }
  return make_uint2(low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
}

// silu(g) * u for any gate.  Below -87, where 1 + exp(-g) is or nears infinity, silu(g) is
// g exp(g) to the last bit, and the product with a large u may still be an ordinary number: the
// exponential's halves go on either side of it.
__device__ __forceinline__ float silu_mul_far(float g, float u) {
  if (!(g < -87.f)) return g / (1.0f + expf(-g)) * u;
  const float half = expf(0.5f * g);
  return g * half * u * half;
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
  int64_t rows;
  int hidden, group;
  float eps;
};

// A CTA takes whole rows, a row in registers (V vectors of 8 columns per thread): one pass
// over memory, one barrier per row for the sum of squares.  The CTAs are persistent (at most
// 1536 threads per SM): the next row's loads are in flight while a row is reduced and stored.
// The weight is loaded once, beside the first row, and stays in registers.  (Rows of more than
// 16384 columns, V = 8, leave no registers for either.)  It is read after the dependency wait
// like the rows: it may be the previous kernel's output.
// Bound by the launch and one trip to memory for a few rows (with a residual, 1 x 4096 1.9 us), by
// HBM for long ones (2048 x 16384 43.2 us, 5.4 TB/s, 0.84 of the measured copy) and by issue slots
// in between: 2048 x 4096 16.1 us (3.6 TB/s, 0.56; two thirds of the cycles issue), 2048 x 8192
// 25.0, 512 x 32768 39.3 us.  A CTA per row instead of persistent ones: 20.1, 43.4 and 62.8 us for
// 2048 rows of 4096, 8192 and 16384.
template <int V, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_q8_kernel(const NormQ8Params p) {
  pdl_launch_dependents();
  const int nvec = p.hidden / kVec;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint4* w4 = reinterpret_cast<const uint4*>(p.weight);
  constexpr bool kAhead = V <= 2;
  uint4 wv[kAhead ? V : 1], xv[V], rv[V];
  pdl_wait();
  auto load = [&](int64_t row) {
    const uint4* x = reinterpret_cast<const uint4*>(p.x + row * p.x_row);
    const uint4* r = reinterpret_cast<const uint4*>(p.residual + row * p.residual_row);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      xv[i] = c < nvec ? x[c] : zero;
      rv[i] = p.residual && c < nvec ? r[c] : zero;
    }
  };
  __shared__ float red[2][32];  // two buffers: a row's barrier is the only one
  const int warps = blockDim.x >> 5, lanes = p.group / kVec;
  int buf = 0;
  if (kAhead) {
    load(blockIdx.x);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      wv[kAhead ? i : 0] = c < nvec ? w4[c] : zero;
    }
  }
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, buf ^= 1) {
    if (!kAhead) load(row);
    float h[V][kVec];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      float r[kVec];
      unpack8(xv[i], h[i]);
      unpack8(rv[i], r);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        h[i][j] += r[j];
        ss = fmaf(h[i][j], h[i][j], ss);
      }
      if (p.residual && c < nvec)
        reinterpret_cast<uint4*>(p.residual_out + row * p.residual_out_row)[c] =
            make_uint4(pack_bf16(h[i][0], h[i][1]), pack_bf16(h[i][2], h[i][3]), pack_bf16(h[i][4], h[i][5]),
                       pack_bf16(h[i][6], h[i][7]));
    }
    if (kAhead && row + gridDim.x < p.rows) load(row + gridDim.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (warps > 1) {
      if ((threadIdx.x & 31) == 0) red[buf][threadIdx.x >> 5] = ss;
      __syncthreads();
      ss = (threadIdx.x & 31) < warps ? red[buf][threadIdx.x & 31] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    const float rs = 1.0f / sqrtf(ss / (float)p.hidden + p.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      float w[kVec], y[kVec], s;
      unpack8(kAhead ? wv[kAhead ? i : 0] : c < nvec ? w4[c] : zero, w);
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = h[i][j] * rs * w[j];
      const uint2 q = quantise8(y, lanes, &s);
      if (c < nvec) {
        *reinterpret_cast<uint2*>(p.q + row * p.q_row + (int64_t)c * kVec) = q;
        if ((c & (lanes - 1)) == 0) p.scale[row * p.scale_row + c / lanes] = s;
      }
    }
  }
}

// One warp per 256 columns of a row (whole groups), one 8-column vector per lane.  One pass;
// SiLU 8 x 14336 1.7 us, 2048 x 14336 41 us (3.6 TB/s), plain 2048 x 4096 8.7 us (2.9 TB/s), 1000
// x 1544 in groups of 32 3.1 us.  Bound by its instructions (85 and 75 % of the cycles issue, 336 and
// 202 per 256 columns) more than by memory: an IEEE division in SiLU makes 46 us of the 41, an exact
// quotient by s in the rounding (two products and a rare division) 11.0 of the 8.7.  Four chunks' loads in flight per warp: SiLU 2048 rows 1 us less,
// 256 rows 8.4 against 6.7 us.
// __fdividef: the quotient's last bits are far below the int8 step.  Its denominator has to stay
// below 2^126; the test for gates past that costs 1.4 us of the 41.
template <bool SILU>
__global__ void __launch_bounds__(256)
    rows_q8_kernel(const __nv_bfloat16* __restrict__ x, int64_t x_row, int8_t* __restrict__ q, int64_t q_row,
                   float* __restrict__ scale, int64_t scale_row, int64_t rows, int cols, int group) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, lanes = group / kVec, nvec = cols / kVec;
  const uint32_t chunks = (cols + 255) / 256, total = (uint32_t)rows * chunks;
  const uint32_t stride = gridDim.x * (blockDim.x >> 5);
  for (uint32_t i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += stride) {
    const uint32_t row = i / chunks, c = (i - row * chunks) * 32 + lane;
    const uint4* src = reinterpret_cast<const uint4*>(x + (int64_t)row * x_row);
    const bool in = c < nvec;
    const uint4 zero = make_uint4(0, 0, 0, 0), g = in ? src[c] : zero, up = SILU && in ? src[nvec + c] : zero;
    float y[kVec], s;
    unpack8(g, y);
    if (SILU) {
      float u[kVec];
      unpack8(up, u);
      float least = y[0];
#pragma unroll
      for (int j = 1; j < kVec; ++j) least = fminf(least, y[j]);
      if (least < -87.f) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) y[j] = silu_mul_far(y[j], u[j]);
      } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) y[j] = __fdividef(y[j], 1.0f + expf(-y[j])) * u[j];
      }
    }
    const uint2 v = quantise8(y, lanes, &s);
    if (in) {
      *reinterpret_cast<uint2*>(q + row * q_row + (int64_t)c * kVec) = v;
      if ((c & (lanes - 1)) == 0) scale[row * scale_row + c / lanes] = s;
    }
  }
}

// One 8-column vector per thread: 2048 x 4096 6.6 us (3.8 TB/s; 70 % of the cycles issue), 1000 x
// 1544 2.7 us; four vectors in flight 8.5 and 4.1 us.
__global__ void __launch_bounds__(256)
    dequantize_q8_kernel(const int8_t* __restrict__ q, int64_t q_row, const float* __restrict__ scale,
                         int64_t scale_row, __nv_bfloat16* __restrict__ out, int64_t out_row, int64_t rows, int cols,
                         int group) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t nvec = cols / kVec, total = (uint32_t)rows * nvec, stride = gridDim.x * blockDim.x;
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    const uint32_t row = i / nvec, c = (i - row * nvec) * kVec;
    const uint2 v = *reinterpret_cast<const uint2*>(q + row * q_row + c);
    const float s = scale[row * scale_row + c / group];
    const uint32_t lo = v.x ^ 0x80808080u, hi = v.y ^ 0x80808080u;  // q + 128 as a byte
    float f[kVec];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // the byte under the exponent of 2^23 is 2^23 + q + 128
      f[j] = (__uint_as_float(__byte_perm(lo, 0x4b000000u, 0x7440 | j)) - 8388736.0f) * s;
      f[j + 4] = (__uint_as_float(__byte_perm(hi, 0x4b000000u, 0x7440 | j)) - 8388736.0f) * s;
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
  // work items are counted in 32 bits
  return a.rows * (a.cols / kVec) <= 0x7fffffff ? LKV_OK : LKV_ERR_UNSUPPORTED;
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
                 a.rows,
                 a.cols,
                 a.group,
                 eps};
  const int nvec = a.cols / kVec;
  const int v = nvec > 2048 ? 8 : nvec <= 1024 ? 1 : 2;
  const int threads = ((nvec + v - 1) / v + 31) / 32 * 32;
  void (*kernel)(const NormQ8Params) = v == 1   ? rmsnorm_q8_kernel<1, 1024>
                                       : v == 2 ? rmsnorm_q8_kernel<2, 1024>
                                                : rmsnorm_q8_kernel<8, 512>;
  const int64_t ctas = std::min<int64_t>(a.rows, 148 * std::max(1, 1536 / threads));
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(threads), 0, stream, p) == cudaSuccess ? LKV_OK
                                                                                                 : LKV_ERR_CUDA;
}

int rows_q8(const void* x, int64_t x_row, int silu, const Q8RowsArgs& a, cudaStream_t stream) {
  const int st = q8_shape(a);
  if (st != LKV_OK) return st;
  if (a.rows == 0) return LKV_OK;
  if (!rows_ok(x, a.rows, x_row, silu ? 2 * (int64_t)a.cols : a.cols, 2, 16) || !q8_ok(a)) return LKV_ERR_INVALID_ARGUMENT;
  const int64_t warps = a.rows * ((a.cols + 255) / 256);
  return launch_pdl(silu ? rows_q8_kernel<true> : rows_q8_kernel<false>, dim3(row_blocks(warps)), dim3(256), 0, stream,
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
  const int64_t warps = (a.rows * (a.cols / kVec) + 31) / 32;
  return launch_pdl(dequantize_q8_kernel, dim3(row_blocks(warps)), dim3(256), 0, stream,
                    static_cast<const int8_t*>(a.q), a.q_row, static_cast<const float*>(a.scale), a.scale_row,
                    static_cast<__nv_bfloat16*>(out), out_row, a.rows, a.cols, a.group) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

}  // namespace lkv

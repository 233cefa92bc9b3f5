// Bandwidth kernels of the 8-bit floating point path (the format: u15_fp8.cuh):
// RMSNorm with the residual's addition and quantised output, the row and
// weight quantisers, and the dequantiser.
#include "u15_fp8.cuh"
#include "u15_kernels.h"

namespace u15 {

namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float wsum(float v)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// largest of 16 lanes (a block of 128 columns at 8 columns a lane)
__device__ __forceinline__ float max16(float v)
{
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ void unpack8f(const uint4& u, float (&v)[8])
{
  const float2 a = unpack_bf2(u.x), b = unpack_bf2(u.y), c = unpack_bf2(u.z), d = unpack_bf2(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
__device__ __forceinline__ uint4 pack8f(const float (&v)[8])
{
  return make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]),
                    pack_bf2(v[6], v[7]));
}
__device__ __forceinline__ float amax8(const float (&v)[8])
{
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
  return m;
}
__device__ __forceinline__ int seg_expert_of(int row, const SegInfo& s)
{
  int e = s.expert[0];
#pragma unroll 1
  for (int i = 1; i < s.nseg; ++i)
    if (row >= s.off[i]) e = s.expert[i];
  return e;
}

// ---------------------------------------------------------------------
// s = bf16(x + delta); y = s / sqrt(mean(s^2) + eps) * w_e; q = e4m3(y).
// One CTA per row, NT threads with KW runs of 8 columns each, kept packed in
// registers between the sum of squares and the output (KW = 0: any width, the
// row read again). Sums in f32, and y is rounded once, to e4m3. x_out may be
// x or delta: every element is read and written by one thread.
// ---------------------------------------------------------------------
template <int NT, int KW>
__global__ void __launch_bounds__(NT)
    add_norm_fp8_kernel(const bf16* x, const bf16* delta, const bf16* __restrict__ w, bf16* x_out,
                        uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int dim, float eps,
                        SegInfo seg)
{
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.x;
  const long base = (long)row * dim;
  const bf16* wr = w + (long)seg_expert_of(row, seg) * dim;
  const int groups = fp8_groups(dim);
  __shared__ float red[NT / 32];

  // the row's run of 8 columns at c, the residual's sum rounded and stored
  auto load = [&](int c) -> uint4 {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (c < dim) {
      u = *reinterpret_cast<const uint4*>(x + base + c);
      if (delta != nullptr) {
        float a[8], b[8];
        unpack8f(u, a);
        unpack8f(*reinterpret_cast<const uint4*>(delta + base + c), b);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] += b[i];
        u = pack8f(a);
      }
      if (x_out != nullptr) *reinterpret_cast<uint4*>(x_out + base + c) = u;
    }
    return u;
  };
  auto squares = [&](const uint4& u, float acc) {
    float t[8];
    unpack8f(u, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __fmaf_rn(t[i], t[i], acc);
    return acc;
  };
  auto rstd = [&](float acc) {
    acc = wsum(acc);
    if (lane_id() == 0) red[warp_id()] = acc;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) t += red[i];
    return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(t, (float)dim) + eps));
  };
  // all lanes of a warp call this together: the block's largest is a shuffle
  auto out = [&](const uint4& u, int c, float inv) {
    float t[8], g[8];
    unpack8f(u, t);
    unpack8f(c < dim ? __ldg(reinterpret_cast<const uint4*>(wr + c)) : make_uint4(0, 0, 0, 0), g);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = c < dim ? t[i] * inv * g[i] : 0.0f;
    const uint32_t s = fp8_scale_byte(max16(amax8(t)));
    if (c < dim) {
      *reinterpret_cast<uint2*>(q + base + c) = fp8_codes8(t, fp8_inv_scale(s));
      if ((lane_id() & 15) == 0) scale[fp8_scale_at(row, c >> 7, groups)] = (uint8_t)s;
    }
  };

  if constexpr (KW > 0) {
    uint4 u[KW];
    float acc = 0.0f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      u[k] = load((k * NT + threadIdx.x) * 8);
      acc = squares(u[k], acc);
    }
    const float inv = rstd(acc);
#pragma unroll
    for (int k = 0; k < KW; ++k) out(u[k], (k * NT + threadIdx.x) * 8, inv);
  } else {
    float acc = 0.0f;
    for (int c0 = 0; c0 < dim; c0 += NT * 8) acc = squares(load(c0 + threadIdx.x * 8), acc);
    const float inv = rstd(acc);
    // the sum again: from x_out where it was stored (x or delta may be it)
    for (int c0 = 0; c0 < dim; c0 += NT * 8) {
      const int c = c0 + threadIdx.x * 8;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (c < dim) {
        if (x_out != nullptr)
          u = *reinterpret_cast<const uint4*>(x_out + base + c);
        else
          u = load(c);
      }
      out(u, c, inv);
    }
  }
}

// ---------------------------------------------------------------------
// q = e4m3 of each row in blocks of 128 columns. A warp takes 256 * U columns
// of one row: 8 columns a lane and step, 16 lanes a block.
// ---------------------------------------------------------------------
constexpr int kQU = 4;

__global__ void __launch_bounds__(256)
    quant_rows_fp8_kernel(const bf16* __restrict__ x, uint8_t* __restrict__ q,
                          uint8_t* __restrict__ scale, long tasks, int per_row, int cols)
{
  griddep_launch();
  griddep_wait();
  const long task = (long)blockIdx.x * 8 + warp_id();
  if (task >= tasks) return;
  const long row = task / per_row;
  const int c0 = (int)(task - row * per_row) * (256 * kQU) + (int)lane_id() * 8;
  const int groups = fp8_groups(cols);
  uint4 u[kQU];
#pragma unroll
  for (int k = 0; k < kQU; ++k) {
    u[k] = make_uint4(0, 0, 0, 0);
    if (c0 + k * 256 < cols)
      u[k] = *reinterpret_cast<const uint4*>(x + row * cols + c0 + k * 256);
  }
#pragma unroll
  for (int k = 0; k < kQU; ++k) {
    const int c = c0 + k * 256;
    float t[8];
    unpack8f(u[k], t);
    const uint32_t s = fp8_scale_byte(max16(amax8(t)));
    if (c < cols) {
      *reinterpret_cast<uint2*>(q + row * cols + c) = fp8_codes8(t, fp8_inv_scale(s));
      if ((lane_id() & 15) == 0) scale[fp8_scale_at(row, c >> 7, groups)] = (uint8_t)s;
    }
  }
}

// ---------------------------------------------------------------------
// Weights: one scale per 128 x 128 block, written for each of its rows. One
// CTA per block; 16 threads cover a row's 128 columns, 16 rows a step.
// ---------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    quant_weight_fp8_kernel(const bf16* __restrict__ w, uint8_t* __restrict__ q,
                            uint8_t* __restrict__ scale, int N, int K)
{
  const int b = blockIdx.x, e = blockIdx.z;
  const int r0 = blockIdx.y * 128, c = b * 128 + (threadIdx.x & 15) * 8;
  const int groups = fp8_groups(K);
  const bf16* we = w + (long)e * N * K;
  uint8_t* qe = q + (long)e * N * K;
  uint8_t* se = scale + (long)e * fp8_scale_bytes(N, K);
  __shared__ float red[8];
  uint4 u[8];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i * 16 + (threadIdx.x >> 4);
    u[i] = make_uint4(0, 0, 0, 0);
    if (r < N && c < K) u[i] = *reinterpret_cast<const uint4*>(we + (long)r * K + c);
    float t[8];
    unpack8f(u[i], t);
    m = fmaxf(m, amax8(t));
  }
  m = max16(m);
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
  if (lane_id() == 0) red[warp_id()] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, red[i]);
  const uint32_t s = fp8_scale_byte(m);
  const float inv = fp8_inv_scale(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i * 16 + (threadIdx.x >> 4);
    if (r >= N || c >= K) continue;
    float t[8];
    unpack8f(u[i], t);
    *reinterpret_cast<uint2*>(qe + (long)r * K + c) = fp8_codes8(t, inv);
  }
  if (threadIdx.x < 128 && r0 + (int)threadIdx.x < N)
    se[fp8_scale_at(r0 + threadIdx.x, b, groups)] = (uint8_t)s;
}

// y = bf16(q * 2^(s - 127)): 16 columns a thread
__global__ void __launch_bounds__(256)
    dequant_fp8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                       bf16* __restrict__ y, long total, int rows, int cols, long scale_stride)
{
  griddep_launch();
  griddep_wait();
  const int per_row = cols / 16, groups = fp8_groups(cols);
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const long row = i / per_row;
  const int c = (int)(i - row * per_row) * 16;
  const long e = row / rows, r = row - e * rows;
  const uint4 u = *reinterpret_cast<const uint4*>(q + row * cols + c);
  const float f = fp8_scale_value(scale[e * scale_stride + fp8_scale_at(r, c >> 7, groups)]);
  const uint32_t in[4] = {u.x, u.y, u.z, u.w};
  uint32_t o[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 a = fp8_pair(in[k]), b = fp8_pair(in[k] >> 16);
    o[2 * k] = pack_bf2(a.x * f, a.y * f);
    o[2 * k + 1] = pack_bf2(b.x * f, b.y * f);
  }
  uint4* d = reinterpret_cast<uint4*>(y + row * cols + c);
  d[0] = make_uint4(o[0], o[1], o[2], o[3]);
  d[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

}  // namespace

int launch_add_rms_norm_fp8(const void* x, const void* delta, const void* w, void* x_out,
                            uint8_t* q, uint8_t* scale, int rows, int dim, float eps,
                            const SegInfo& seg, cudaStream_t st)
{
  if (rows <= 0) return 0;
  const bf16 *xb = static_cast<const bf16*>(x), *db = static_cast<const bf16*>(delta),
             *wb = static_cast<const bf16*>(w);
  bf16* ob = static_cast<bf16*>(x_out);
  cudaError_t e;
  if (dim <= 4096)
    e = launch_pdl(add_norm_fp8_kernel<128, 4>, dim3(rows), dim3(128), st, xb, db, wb, ob, q,
                   scale, dim, eps, seg);
  else
    e = launch_pdl(add_norm_fp8_kernel<256, 0>, dim3(rows), dim3(256), st, xb, db, wb, ob, q,
                   scale, dim, eps, seg);
  return e == cudaSuccess ? 0 : 2;
}

int launch_quant_rows_fp8(const void* x, uint8_t* q, uint8_t* scale, int rows, int cols,
                          cudaStream_t st)
{
  if (rows <= 0) return 0;
  const int per_row = (cols + 256 * kQU - 1) / (256 * kQU);
  const long tasks = (long)rows * per_row;
  return launch_pdl(quant_rows_fp8_kernel, dim3((unsigned)((tasks + 7) / 8)), dim3(256), st,
                    static_cast<const bf16*>(x), q, scale, tasks, per_row, cols) == cudaSuccess
             ? 0
             : 2;
}

int launch_quant_weight_fp8(const void* w, uint8_t* q, uint8_t* scale, int n_experts, int N, int K,
                            cudaStream_t st)
{
  if (N <= 0 || n_experts <= 0) return 0;
  quant_weight_fp8_kernel<<<dim3(fp8_blocks(K), (N + 127) / 128, n_experts), 256, 0, st>>>(
      static_cast<const bf16*>(w), q, scale, N, K);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

int launch_dequant_fp8(const uint8_t* q, const uint8_t* scale, void* y, int n_experts, int rows,
                       int cols, cudaStream_t st)
{
  const long total = (long)n_experts * rows * (cols / 16);
  if (total <= 0) return 0;
  return launch_pdl(dequant_fp8_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), st, q,
                    scale, static_cast<bf16*>(y), total, rows, cols,
                    fp8_scale_bytes(rows, cols)) == cudaSuccess
             ? 0
             : 2;
}

}  // namespace u15

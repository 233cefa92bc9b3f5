// Bandwidth kernels of the 8-bit floating point path (the format: u15_fp8.cuh):
// RMSNorm with the residual's addition and quantised output, the row and
// weight quantisers, and the dequantiser.
#include "u15_fp8.cuh"
#include "u15_kernels.h"

#include <algorithm>

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
__device__ __forceinline__ void unpack8f(const uint4& u, float* v)
{
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8f(const float* v)
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
// NT threads take a row, KW runs of 16 columns each (eight lanes a block of
// 128), and walk the rows with the grid's stride; a row stays in registers
// between its sum of squares and its output. Sums in f32; s * w is exact
// (two bf16), the reciprocal root correctly rounded, so y carries two f32
// roundings ahead of its one to e4m3. x_out may be x or delta: every element
// is read and written by one thread.
// ---------------------------------------------------------------------

// 1 / sqrt(v), rounded once: r = 1 / s and s = sqrt(v) are rounded, and their
// exact residuals 1 - s r and v - s^2 (one fma each) give the next term of
// 1 / sqrt(s^2 + d) = 1 / s - d / (2 s^3)
__device__ __forceinline__ float rsqrt_exact(float v)
{
  const float s = __fsqrt_rn(v), r = __fdiv_rn(1.0f, s);
  const float e = __fmaf_rn(-s, r, 1.0f), d = __fmaf_rn(-s, s, v);
  return s == INFINITY ? 0.0f : __fmaf_rn(r, __fmaf_rn(-0.5f * d * r, r, e), r);
}

// threads of the norm resident on an SM
constexpr int kNormThreads = 1024;

// two f32 operations in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

template <int NT, int KW>
__global__ void __launch_bounds__(NT < 128 ? 128 : NT)
    add_norm_fp8_kernel(const bf16* x, const bf16* delta, const bf16* __restrict__ w, bf16* x_out,
                        uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int rows, int dim,
                        float eps, SegInfo seg)
{
  constexpr int kCta = NT < 128 ? 128 : NT, kRows = kCta / NT;   // rows a CTA takes at once
  griddep_launch();
  griddep_wait();
  const int lane_in = threadIdx.x % NT, groups = fp8_groups(dim);
  __shared__ float red[2][NT / 32];
  int par = 0;
  // every thread of the CTA runs the same number of rounds
  for (long r0 = (long)blockIdx.x * kRows; r0 < rows; r0 += (long)gridDim.x * kRows, par ^= 1) {
    const long row = r0 + threadIdx.x / NT;
    const bool live = row < rows;
    float2 t[KW][8];
    float2 acc2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int c = (k * NT + lane_in) * 16;
      float* v = &t[k][0].x;
      uint4 u[2] = {};
      if (live && c < dim) {
        const uint4* px = reinterpret_cast<const uint4*>(x + row * dim + c);
        u[0] = px[0];
        u[1] = px[1];
      }
      unpack8f(u[0], v);
      unpack8f(u[1], v + 8);
      if (delta != nullptr) {
        if (live && c < dim) {
          const uint4* pd = reinterpret_cast<const uint4*>(delta + row * dim + c);
          float b[16];
          unpack8f(pd[0], b);
          unpack8f(pd[1], b + 8);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] += b[i];
        }
        u[0] = pack8f(v);
        u[1] = pack8f(v + 8);
        unpack8f(u[0], v);
        unpack8f(u[1], v + 8);
      }
      if (x_out != nullptr && live && c < dim) {
        uint4* po = reinterpret_cast<uint4*>(x_out + row * dim + c);
        po[0] = u[0];
        po[1] = u[1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc2 = fma2(t[k][i], t[k][i], acc2);
    }
    float acc = wsum(acc2.x + acc2.y);
    if constexpr (NT > 32) {
      if (lane_id() == 0) red[par][warp_id()] = acc;
      __syncthreads();
      acc = 0.0f;
#pragma unroll
      for (int i = 0; i < NT / 32; ++i) acc += red[par][i];
    }
    const float inv = rsqrt_exact(__fdiv_rn(acc, (float)dim) + eps);
    const bf16* wr = w + (long)(live ? seg_expert_of((int)row, seg) : 0) * dim;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int c = (k * NT + lane_in) * 16;
      uint4 gw[2] = {};
      if (c < dim) {
        gw[0] = __ldg(reinterpret_cast<const uint4*>(wr + c));
        gw[1] = __ldg(reinterpret_cast<const uint4*>(wr + c) + 1);
      }
      float2 g[8];
      unpack8f(gw[0], &g[0].x);
      unpack8f(gw[1], &g[4].x);
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t[k][i] = mul2(mul2(t[k][i], g[i]), make_float2(inv, inv));
        m = fmaxf(m, fmaxf(fabsf(t[k][i].x), fabsf(t[k][i].y)));
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint32_t s = fp8_scale_byte(m);
      const float f = fp8_inv_scale(s, m);
      if (live && c < dim) {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 a = mul2(t[k][2 * i], make_float2(f, f)),
                       b = mul2(t[k][2 * i + 1], make_float2(f, f));
          h[i] = __byte_perm(fp8_codes2(a.x, a.y), fp8_codes2(b.x, b.y), 0x5410);
        }
        *reinterpret_cast<uint4*>(q + row * dim + c) = make_uint4(h[0], h[1], h[2], h[3]);
        if ((lane_id() & 7) == 0) scale[fp8_scale_at(row, c >> 7, groups)] = (uint8_t)s;
      }
    }
  }
}

// The same for rows too wide for registers: one CTA a row, which it reads twice.
__global__ void __launch_bounds__(512)
    add_norm_wide_fp8_kernel(const bf16* x, const bf16* delta, const bf16* __restrict__ w, bf16* x_out,
                             uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int dim, float eps,
                             SegInfo seg)
{
  griddep_launch();
  griddep_wait();
  const long row = blockIdx.x;
  const bf16* wr = w + (long)seg_expert_of((int)row, seg) * dim;
  const int groups = fp8_groups(dim);
  __shared__ float red[16];
  auto load = [&](int c) {
    uint4 u = *reinterpret_cast<const uint4*>(x + row * dim + c);
    if (delta == nullptr) return u;
    float a[8], b[8];
    unpack8f(u, a);
    unpack8f(*reinterpret_cast<const uint4*>(delta + row * dim + c), b);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] += b[i];
    return pack8f(a);
  };
  float acc = 0.0f;
  for (int c = threadIdx.x * 8; c < dim; c += 512 * 8) {
    const uint4 u = load(c);
    if (x_out != nullptr) *reinterpret_cast<uint4*>(x_out + row * dim + c) = u;
    float t[8];
    unpack8f(u, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __fmaf_rn(t[i], t[i], acc);
  }
  acc = wsum(acc);
  if (lane_id() == 0) red[warp_id()] = acc;
  __syncthreads();
  acc = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc += red[i];
  const float inv = rsqrt_exact(__fdiv_rn(acc, (float)dim) + eps);
  for (int c0 = 0; c0 < dim; c0 += 512 * 8) {
    const int c = c0 + threadIdx.x * 8;
    float t[8] = {}, g[8];
    if (c < dim) {
      // the sum from where it was stored: x or delta may be that place
      unpack8f(x_out != nullptr ? *reinterpret_cast<const uint4*>(x_out + row * dim + c) : load(c), t);
      unpack8f(__ldg(reinterpret_cast<const uint4*>(wr + c)), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = t[i] * g[i] * inv;
    }
    const float m = max16(amax8(t));
    const uint32_t s = fp8_scale_byte(m);
    if (c < dim) {
      *reinterpret_cast<uint2*>(q + row * dim + c) = fp8_codes8(t, fp8_inv_scale(s, m));
      if ((lane_id() & 15) == 0) scale[fp8_scale_at(row, c >> 7, groups)] = (uint8_t)s;
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
    const float m = max16(amax8(t));
    const uint32_t s = fp8_scale_byte(m);
    if (c < cols) {
      *reinterpret_cast<uint2*>(q + row * cols + c) = fp8_codes8(t, fp8_inv_scale(s, m));
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
  const float inv = fp8_inv_scale(s, m);
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

namespace {

template <int NT, int KW>
cudaError_t launch_norm(const bf16* x, const bf16* delta, const bf16* w, bf16* x_out, uint8_t* q,
                        uint8_t* scale, int rows, int dim, float eps, const SegInfo& seg,
                        int num_sms, cudaStream_t st)
{
  constexpr int kCta = NT < 128 ? 128 : NT, kRows = kCta / NT;
  const int grid = std::min((rows + kRows - 1) / kRows, num_sms * (kNormThreads / kCta));
  return launch_pdl(add_norm_fp8_kernel<NT, KW>, dim3(grid), dim3(kCta), st, x, delta, w, x_out, q,
                    scale, rows, dim, eps, seg);
}

}  // namespace

int launch_add_rms_norm_fp8(const void* x, const void* delta, const void* w, void* x_out,
                            uint8_t* q, uint8_t* scale, int rows, int dim, float eps,
                            const SegInfo& seg, int num_sms, cudaStream_t st)
{
  if (rows <= 0) return 0;
  const bf16 *xb = static_cast<const bf16*>(x), *db = static_cast<const bf16*>(delta),
             *wb = static_cast<const bf16*>(w);
  bf16* ob = static_cast<bf16*>(x_out);
  // the fewest threads that hold a row at up to 32 (wide rows: 48) columns each
  const auto k = dim <= 512     ? launch_norm<32, 1>
                 : dim <= 1024  ? launch_norm<32, 2>
                 : dim <= 2048  ? launch_norm<128, 1>
                 : dim <= 4096  ? launch_norm<128, 2>
                 : dim <= 8192  ? launch_norm<256, 2>
                 : dim <= 12288 ? launch_norm<256, 3>
                                : nullptr;
  const cudaError_t e =
      k != nullptr ? k(xb, db, wb, ob, q, scale, rows, dim, eps, seg, num_sms, st)
                   : launch_pdl(add_norm_wide_fp8_kernel, dim3(rows), dim3(512), st, xb, db, wb, ob,
                                q, scale, dim, eps, seg);
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

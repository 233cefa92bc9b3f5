// Bandwidth kernels of the 8-bit floating point path (the format: u15_fp8.cuh):
// RMSNorm with the residual's addition and quantised output, the row and
// weight quantisers, and the dequantiser.
#include "u15_fp8.cuh"
#include "u15_kernels.h"

#include <algorithm>
#include <atomic>

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
// (two bf16), the mean and the reciprocal root are off by about half a unit, so
// y carries little more than one f32 rounding ahead of its one to e4m3. x_out may
// be x or delta: a row is read whole before any of it is written.
// ---------------------------------------------------------------------

// 1 / sqrt(v) to within about half a unit: the hardware's approximation and one
// Newton step whose residual 1 - v r^2 is formed without rounding v r (an fma
// gives what the product lost)
__device__ __forceinline__ float rsqrt_newton(float v)
{
  const float r = rsqrtf(v);
  const float h = v * r, l = __fmaf_rn(v, r, -h);
  const float e = __fmaf_rn(-l, r, __fmaf_rn(-h, r, 1.0f));
  return v == INFINITY ? 0.0f : __fmaf_rn(0.5f * r, e, r);
}
// acc / dim the same way: inv_dim = 1 / dim as a rounded value and its rest. A sum
// past f32's range stays Inf (the rest, zero or negative for most widths, would
// make it NaN), and the row's finite values become 0.
__device__ __forceinline__ float mean_of(float acc, float2 inv_dim)
{
  return acc < INFINITY ? __fmaf_rn(acc, inv_dim.x, acc * inv_dim.y) : acc;
}

constexpr int kNormSmem = 200 * 1024;   // bytes of row stages on an SM

// max(m, |a|, |b|) in one instruction (NaN is dropped)
__device__ __forceinline__ float max_abs3(float m, float a, float b)
{
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}

// CTAs of a form on an SM: the registers that its row, gains and temporaries
// take (46 / 72 / 104 for 1 / 2 / 3 runs); the grid is no larger, since
// CTAs that wait for a place find the row stages empty (4096 x 4096: 7
// a SM 12.8 us, 12 14.7)
template <int NT, int KW>
constexpr int norm_ctas()
{
  return (KW == 1 ? 1280 : KW == 2 ? 896 : 512) / (NT < 128 ? 128 : NT);
}

template <int NT, int KW>
__global__ void __launch_bounds__(NT < 128 ? 128 : NT, norm_ctas<NT, KW>())
    add_norm_fp8_kernel(const bf16* x, const bf16* delta, const bf16* __restrict__ w, bf16* x_out,
                        uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int rows, int dim,
                        float2 inv_dim, float eps, SegInfo seg, unsigned* err)
{
  constexpr int kCta = NT < 128 ? 128 : NT, kRows = kCta / NT;   // rows a CTA takes at once
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ float red[2][NT / 32];
  griddep_launch();
  const uint32_t bar0 = smem_u32(bars), ring0 = smem_u32(ring);
  const int half = kRows * dim * 2, stage = delta != nullptr ? 2 * half : half;
  const int step = gridDim.x * kRows;
  auto fill = [&](int s, int r) {   // one thread: rows [r, r + kRows) into stage s
    const uint32_t n = (uint32_t)min(kRows, rows - r) * dim * 2;
    mbar_arrive_expect_tx(bar0 + 8 * s, delta != nullptr ? 2 * n : n);
    bulk_load(ring0 + s * stage, x + (long)r * dim, n, bar0 + 8 * s);
    if (delta != nullptr)
      bulk_load(ring0 + s * stage + half, delta + (long)r * dim, n, bar0 + 8 * s);
  };
  const int first = blockIdx.x * kRows;
  if (threadIdx.x == 0) {
    mbar_init(bar0, 1);
    mbar_init(bar0 + 8, 1);
    fence_barrier_init();
    griddep_wait();
    if (first < rows) fill(0, first);
    if (first + step < rows) fill(1, first + step);
  }
  __syncthreads();
  griddep_wait();
  // this thread's columns: k NT 16 + c0, and where their block's byte is
  const int sub = NT < 128 ? threadIdx.x / NT : 0, c0 = (threadIdx.x % NT) * 16;
  const int groups = fp8_groups(dim);
  bool col[KW];
  int sb_at[KW];
#pragma unroll
  for (int k = 0; k < KW; ++k) {
    const int c = k * NT * 16 + c0;
    col[k] = c < dim;
    sb_at[k] = (c >> 9) * kFp8SfTile + ((c >> 7) & 3);
  }
  uint32_t it = 0;
  int cur = -1;
  bool ok = true;
  uint4 gw[KW][2] = {};   // the gains of expert `cur`, read again only where it changes
  // every thread of the CTA runs the same number of rounds (rows + 2 step < 2^31)
  for (int r0 = first; r0 < rows; r0 += step, ++it) {
    const int st = it & 1, row = r0 + sub;
    const bool live = kRows == 1 || row < rows;
    const int e = live ? seg_expert_of(row, seg) : cur;
    if (e != cur) {
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const uint4* pw = reinterpret_cast<const uint4*>(w + (long)e * dim + k * NT * 16 + c0);
        if (col[k]) {
          gw[k][0] = __ldg(pw);
          gw[k][1] = __ldg(pw + 1);
        }
      }
      cur = e;
    }
    ok = mbar_wait(bar0 + 8 * st, (it >> 1) & 1, err, kDevWaitFull) && ok;
    const uint8_t* src = ring + st * stage + (sub * dim + c0) * 2;
    const long at = (long)row * dim + c0;
    float2 t[KW][8];
    float2 acc2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      float* v = &t[k][0].x;
      uint4 u[2] = {};
      const bool here = live && col[k];
      if (here) {
        u[0] = *reinterpret_cast<const uint4*>(src + k * NT * 32);
        u[1] = *reinterpret_cast<const uint4*>(src + k * NT * 32 + 16);
      }
      unpack8f(u[0], v);
      unpack8f(u[1], v + 8);
      if (delta != nullptr) {
        if (here) {
          float b[16];
          unpack8f(*reinterpret_cast<const uint4*>(src + k * NT * 32 + half), b);
          unpack8f(*reinterpret_cast<const uint4*>(src + k * NT * 32 + half + 16), b + 8);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] += b[i];
        }
        u[0] = pack8f(v);
        u[1] = pack8f(v + 8);
        unpack8f(u[0], v);
        unpack8f(u[1], v + 8);
      }
      if (x_out != nullptr && here) {
        uint4* po = reinterpret_cast<uint4*>(x_out + at + k * NT * 16);
        po[0] = u[0];
        po[1] = u[1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc2 = __ffma2_rn(t[k][i], t[k][i], acc2);
    }
    float acc = wsum(acc2.x + acc2.y);
    if (NT > 32 && lane_id() == 0) red[st][warp_id()] = acc;
    __syncthreads();   // every thread has its columns: the stage is free
    if (threadIdx.x == 0 && r0 + 2 * step < rows) fill(st, r0 + 2 * step);
    if constexpr (NT > 32) {
      acc = 0.0f;
#pragma unroll
      for (int i = 0; i < NT / 32; ++i) acc += red[st][i];
    }
    const float inv = rsqrt_newton(mean_of(acc, inv_dim) + eps);
    uint8_t* const srow = scale + fp8_scale_at(row, 0, groups);
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      float2 g[8];
      unpack8f(gw[k][0], &g[0].x);
      unpack8f(gw[k][1], &g[4].x);
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t[k][i] = __fmul2_rn(t[k][i], g[i]);
        m = max_abs3(m, t[k][i].x, t[k][i].y);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      // the largest |y| is the largest |s w| times 1 / root (rounding keeps
      // order), and the block's power of two goes into the same factor: y is
      // rounded as if it had been formed first
      m *= inv;
      const uint32_t s = fp8_scale_byte(m);
      float f = inv * fp8_inv_scale(s, m);
      if (f == INFINITY) {   // an all but zero block: two steps
        f = fp8_inv_scale(s, m);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[k][i] = __fmul2_rn(t[k][i], make_float2(inv, inv));
      }
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = __fmul2_rn(t[k][2 * i], make_float2(f, f)),
                     b = __fmul2_rn(t[k][2 * i + 1], make_float2(f, f));
        h[i] = __byte_perm(fp8_codes2(a.x, a.y), fp8_codes2(b.x, b.y), 0x5410);
      }
      if (live && col[k] && ok) {
        *reinterpret_cast<uint4*>(q + at + k * NT * 16) = make_uint4(h[0], h[1], h[2], h[3]);
        if ((lane_id() & 7) == 0) srow[sb_at[k]] = (uint8_t)s;
      }
    }
  }
}

// The same for rows too wide for registers: one CTA a row, which it reads twice
// (4096 x 16384 without / with a residual 52.6 / 82.6 us; bytes once: 30.8 / 71.8).
__global__ void __launch_bounds__(512)
    add_norm_wide_fp8_kernel(const bf16* x, const bf16* delta, const bf16* __restrict__ w,
                             bf16* x_out, uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                             int dim, float2 inv_dim, float eps, SegInfo seg)
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
  const float inv = rsqrt_newton(mean_of(acc, inv_dim) + eps);
  for (int c0 = 0; c0 < dim; c0 += 512 * 8) {
    const int c = c0 + threadIdx.x * 8;
    float t[8] = {}, g[8];
    if (c < dim) {
      // the sum from where it was stored: x or delta may be that place
      unpack8f(x_out != nullptr ? *reinterpret_cast<const uint4*>(x_out + row * dim + c) : load(c),
               t);
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

float2 inverse_of(int dim)
{
  const double inv = 1.0 / dim;
  return make_float2((float)inv, (float)(inv - (double)(float)inv));
}

template <int NT, int KW>
cudaError_t launch_norm(const bf16* x, const bf16* delta, const bf16* w, bf16* x_out, uint8_t* q,
                        uint8_t* scale, int rows, int dim, float eps, const SegInfo& seg,
                        unsigned* err, int num_sms, cudaStream_t st)
{
  static std::atomic<uint64_t> attr_set;
  constexpr int kCta = NT < 128 ? 128 : NT, kRows = kCta / NT;
  constexpr int kMost = 2 * 2 * kRows * NT * KW * 16 * 2;   // two stages of x and delta
  const auto k = add_norm_fp8_kernel<NT, KW>;
  if (!smem_attr_once(k, kMost, attr_set)) return cudaErrorInvalidValue;
  const int smem = 2 * kRows * dim * 2 * (delta != nullptr ? 2 : 1);
  const int per_sm = std::max(1, std::min(norm_ctas<NT, KW>(), kNormSmem / smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::min((rows + kRows - 1) / kRows, num_sms * per_sm));
  cfg.blockDim = dim3(kCta);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, x, delta, w, x_out, q, scale, rows, dim, inverse_of(dim), eps,
                            seg, err);
}

}  // namespace

int launch_add_rms_norm_fp8(const void* x, const void* delta, const void* w, void* x_out,
                            uint8_t* q, uint8_t* scale, int rows, int dim, float eps,
                            const SegInfo& seg, unsigned* err, int num_sms, cudaStream_t st)
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
      k != nullptr ? k(xb, db, wb, ob, q, scale, rows, dim, eps, seg, err, num_sms, st)
                   : launch_pdl(add_norm_wide_fp8_kernel, dim3(rows), dim3(512), st, xb, db, wb, ob,
                                q, scale, dim, inverse_of(dim), eps, seg);
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

// The routed projection in 8-bit floating point (the format: u15_fp8.cuh):
//
//   y[m][n] = epilogue( sum_b 2^(sx[m][b] + sw[n][b] - 254) sum_{k in b} xq[m][k] wq[n][k] )
//
// over the blocks b of 128 columns, wq and sw those of row m's expert. This
// form is the plain one: 16 rows x 128 columns a CTA, products and sums in f32
// on the FMA pipe, each block's sum scaled as it is added.
#include "u15_fp8.cuh"
#include "u15_kernels.h"

namespace u15 {

namespace {

using bf16 = __nv_bfloat16;
constexpr int kRows = 16;

template <int EPI>
__global__ void __launch_bounds__(256) gemm_fp8_plain_kernel(GemmFp8Args a, SegInfo seg)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  __shared__ float sx[kRows][132];
  __shared__ uint8_t sw[GU ? 2 : 1][128][132];
  const int s = blockIdx.z, e = seg.expert[s];
  const int m0 = blockIdx.y * kRows;
  const int lo = max(m0, seg.off[s]), hi = min(m0 + kRows, seg.off[s + 1]);
  if (lo >= hi) return;
  const int n0 = blockIdx.x * (GU ? 256 : 128);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int row = m0 + ty;
  const bool row_ok = row >= lo && row < hi;
  const int groups = fp8_groups(a.K), nb = fp8_blocks(a.K);
  const uint8_t* wq = a.wq + (long)e * a.N * a.K;
  const uint8_t* ws = a.sw + e * fp8_scale_bytes(a.N, a.K);
  float acc[2][8] = {};
  for (int b = 0; b < nb; ++b) {
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * 128; i += 256) {
      const int r = i >> 7, c = b * 128 + (i & 127);
      float v = 0.0f;
      if (m0 + r >= lo && m0 + r < hi && c < a.K)
        v = fp8_pair(a.xq[(long)(m0 + r) * a.K + c]).x;
      sx[r][i & 127] = v;
    }
    for (int i = threadIdx.x; i < (GU ? 2 : 1) * 128 * 128; i += 256) {
      const int h = i >> 14, r = (i >> 7) & 127, c = b * 128 + (i & 127);
      const int n = n0 + h * 128 + r;
      sw[h][r][i & 127] = n < a.N && c < a.K ? wq[(long)n * a.K + c] : 0;
    }
    __syncthreads();
    const float fx = row_ok ? fp8_scale_value(a.sx[fp8_scale_at(row, b, groups)]) : 0.0f;
    for (int h = 0; h < (GU ? 2 : 1); ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = n0 + h * 128 + j * 16 + tx;
        if (n >= a.N) continue;
        float t = 0.0f;
        for (int k = 0; k < 128; k += 2) {
          const float2 w2 =
              fp8_pair(*reinterpret_cast<const uint16_t*>(&sw[h][j * 16 + tx][k]));
          t = __fmaf_rn(sx[ty][k], w2.x, t);
          t = __fmaf_rn(sx[ty][k + 1], w2.y, t);
        }
        acc[h][j] += t * fx * fp8_scale_value(ws[fp8_scale_at(n, b, groups)]);
      }
  }
  if constexpr (GU) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float g = acc[0][j];
      acc[0][j] = __fdiv_rn(g, 1.0f + expf(-g)) * acc[1][j];
      m = fmaxf(m, fabsf(acc[0][j]));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t sb = fp8_scale_byte(m);
    const float inv = fp8_inv_scale(sb);
    if (!row_ok) return;
    const int nout = a.N / 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = blockIdx.x * 128 + j * 16 + tx;
      if constexpr (EPI == kEpiSwiglu) {
        static_cast<bf16*>(a.y)[(long)row * nout + c] = f2bf(acc[0][j]);
      } else {
        const float v = __fmaf_rn(acc[0][j], 0.0f, acc[0][j] * inv);
        static_cast<uint8_t*>(a.y)[(long)row * nout + c] =
            __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
      }
    }
    if (EPI == kEpiSwigluFp8 && tx == 0)
      a.sy[fp8_scale_at(row, blockIdx.x, fp8_groups(nout))] = (uint8_t)sb;
    return;
  }
  if (!row_ok) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int n = n0 + j * 16 + tx;
    if (n >= a.N) continue;
    float v = acc[0][j];
    const long at = (long)row * a.N + n;
    if (a.bias != nullptr) v += bf2f(static_cast<const bf16*>(a.bias)[(long)e * a.N + n]);
    if (EPI == kEpiResid) v += bf2f(static_cast<const bf16*>(a.resid)[at]);
    if (EPI == kEpiStoreF32)
      static_cast<float*>(a.y)[at] = v;
    else
      static_cast<bf16*>(a.y)[at] = f2bf(v);
  }
}

}  // namespace

int gemm_fp8(const GemmFp8Args& a, const SegInfo& seg, cudaStream_t st, std::string* err)
{
  if (a.M <= 0) return 0;
  const bool gu = a.epilogue == kEpiSwiglu || a.epilogue == kEpiSwigluFp8;
  const dim3 grid((a.N + (gu ? 255 : 127)) / (gu ? 256 : 128), (a.M + kRows - 1) / kRows, seg.nseg);
  switch (a.epilogue) {
    case kEpiStore: gemm_fp8_plain_kernel<kEpiStore><<<grid, 256, 0, st>>>(a, seg); break;
    case kEpiResid: gemm_fp8_plain_kernel<kEpiResid><<<grid, 256, 0, st>>>(a, seg); break;
    case kEpiSwiglu: gemm_fp8_plain_kernel<kEpiSwiglu><<<grid, 256, 0, st>>>(a, seg); break;
    case kEpiStoreF32: gemm_fp8_plain_kernel<kEpiStoreF32><<<grid, 256, 0, st>>>(a, seg); break;
    case kEpiSwigluFp8: gemm_fp8_plain_kernel<kEpiSwigluFp8><<<grid, 256, 0, st>>>(a, seg); break;
    default: return 2;
  }
  if (cudaGetLastError() == cudaSuccess) return 0;
  *err = "gemm_fp8: kernel launch failed";
  return 2;
}

}  // namespace u15

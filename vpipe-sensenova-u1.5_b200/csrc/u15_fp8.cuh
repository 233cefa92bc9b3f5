// 8-bit floating point (e4m3) with one power-of-two scale per block of 128
// columns: the scale rule, the packed scale layout and the conversions every
// fp8 kernel shares.
//
// A quantised tensor stands for q[r][c] * 2^(s[r][c / 128] - 127). The scale
// byte s is the smallest exponent whose 448-fold (e4m3's largest value)
// reaches the block's largest magnitude, so no finite value saturates. A
// power of two costs e4m3 nothing in relative precision (only the block's
// values below 2^-14 of the largest fall under its normal range), multiplies
// exactly, and is the form the tensor core applies by itself (UE8M0).
//
// Scales are packed in 512-byte tiles of 128 rows x 4 blocks, the image of
// the tensor core's scale columns (32 lanes x 4 columns x 4 bytes): one copy
// moves a tile to shared memory and one tcgen05.cp from there to TMEM.
#pragma once

#include <cuda_fp8.h>
#include <stdint.h>

#include "u15_common.cuh"

namespace u15 {

constexpr int kFp8Block = 128;       // columns (and weight rows) under one scale
constexpr int kFp8SfTile = 512;      // bytes of a packed tile: 128 rows x 4 blocks

__host__ __device__ __forceinline__ int fp8_blocks(int cols)
{
  return (int)(((long)cols + 127) / 128);
}
__host__ __device__ __forceinline__ int fp8_groups(int cols)
{
  return (int)(((long)cols + 511) / 512);
}
__host__ __device__ __forceinline__ long fp8_scale_bytes(long rows, int cols)
{
  return (rows + 127) / 128 * fp8_groups(cols) * kFp8SfTile;
}
// byte offset of (row r, block b) in the packed scales of a tensor with `groups`
__host__ __device__ __forceinline__ long fp8_scale_at(long r, int b, int groups)
{
  return ((r >> 7) * groups + (b >> 2)) * kFp8SfTile + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

// The scale byte of a block whose largest magnitude is amax: the smallest s
// with amax <= 448 * 2^(s - 127), from amax's exponent field and whether its
// mantissa is above 1.75 (448 = 1.75 * 2^8); 0 up to 448 * 2^-127 = 1.75 * 2^-119.
__device__ __forceinline__ uint32_t fp8_scale_byte(float amax)
{
  const uint32_t u = __float_as_uint(amax);
  const int s = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(s, 0);
}
// 2^(127 - s), a normal float for every s the rule gives (0 .. 248), by which
// a block's values are multiplied ahead of their rounding; 0 where the block
// holds an Inf (amax never counts a NaN): Inf * 0 is NaN, so a value that is
// not finite becomes the NaN code instead of saturating to 448, at no
// instruction per value
__device__ __forceinline__ float fp8_inv_scale(uint32_t s, float amax)
{
  return amax < INFINITY ? __uint_as_float((254u - s) << 23) : 0.0f;
}
// 2^(s - 127); s = 0 is 2^-127, a subnormal float
__device__ __forceinline__ float fp8_scale_value(uint32_t s)
{
  return s != 0 ? __uint_as_float(s << 23) : __uint_as_float(0x400000u);
}

// two f32 values as two e4m3 codes, lo in the low byte: rounded to nearest even
__device__ __forceinline__ uint32_t fp8_codes2(float lo, float hi)
{
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// e4m3 codes of v[0..8) * inv as 8 bytes, v[0] lowest
__device__ __forceinline__ uint2 fp8_codes8(const float (&v)[8], float inv)
{
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = fp8_codes2(v[2 * i] * inv, v[2 * i + 1] * inv);
  return make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
}
// the same for four values
__device__ __forceinline__ uint32_t fp8_codes4(const float (&v)[4], float inv)
{
  return __byte_perm(fp8_codes2(v[0] * inv, v[1] * inv), fp8_codes2(v[2] * inv, v[3] * inv), 0x5410);
}

// two e4m3 values as floats (exact)
__device__ __forceinline__ float2 fp8_pair(uint32_t lo16)
{
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(lo16 & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// ---------------------------------------------------------------------
// tcgen05 with block scales (kind::mxf8f6f4): D += 2^(sa - 127) 2^(sb - 127) A B^T.
// The instruction takes one UE8M0 byte a row and 32 columns of K from TMEM: a
// 32-bit column word holds four bytes, and the instruction descriptor names
// the byte to use. A word here is the packed tile's: the bytes of four
// 128-column blocks, so the four K = 32 steps of block b all name byte b % 4,
// and one copied tile serves 512 columns of K. Row m of an operand is lane
// m % 32, column m / 32 of its scale columns, in all four lane quadrants.
// ---------------------------------------------------------------------
// e4m3 x e4m3, K-major operands, UE8M0 scales: a/b format 0 (e4m3), N >> 3 at
// bit 17, scale type 1 (UE8M0) at bit 23, M >> 4 at bit 24
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N)
{
  return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}
// the byte of the scale words to use, for B at bit 4 and for A at bit 29
__device__ __forceinline__ uint32_t idesc_scale_byte(uint32_t id) { return (id << 4) | (id << 29); }

// One lane of a converged warp. The producers and issuers here run their
// loops with the whole warp and let this lane issue: addresses and
// descriptors then stay in uniform registers, which a loop inside
// `if (lane == 0)` has to move there for every instruction (an issuer of four
// MMAs a stage took ~105 cycles an MMA that way).
__device__ __forceinline__ bool elect_one()
{
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// The bounded waits for a whole warp: every lane gets the same answer, so the
// warp stays converged where a wait runs out.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, unsigned* err, unsigned code)
{
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}
__device__ __forceinline__ bool warp_wait_probe(uint32_t bar, uint32_t parity, unsigned* err,
                                                unsigned code)
{
  return __all_sync(0xffffffffu, mbar_wait_probe(bar, parity, err, code));
}
__device__ __forceinline__ bool warp_wait_cluster_probe(uint32_t bar, uint32_t parity, unsigned* err,
                                                        unsigned code)
{
  return __all_sync(0xffffffffu, mbar_wait_cluster_probe(bar, parity, err, code));
}

// a packed 512-byte tile in shared memory as 32 rows of 16 bytes: no swizzle,
// 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t smem_desc_sf(uint32_t smem_addr)
{
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(128 >> 4) << 32;   // SBO
  d |= (uint64_t)1 << 46;            // version
  return d;
}
// copy such a tile to 4 scale columns (every lane quadrant); MMAs issued
// after it by the same thread see it, MMAs before it are done with what it
// overwrites
__device__ __forceinline__ void sf_copy(uint32_t taddr, uint64_t desc)
{
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void sf_copy_pair(uint32_t taddr, uint64_t desc)
{
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate)
{
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_e4m3_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                              uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              uint32_t accumulate)
{
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 3-D tiled load into this CTA's shared memory (no multicast): coordinates
// (0, group, row block) of the packed scales
__device__ __forceinline__ void tma_load_sf(uint32_t smem_dst, const CUtensorMap* m, int group,
                                            int rowblk, uint32_t bar)
{
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(0), "r"(group), "r"(rowblk), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_sf_pair(uint32_t smem_dst, const CUtensorMap* m, int group,
                                                 int rowblk, uint32_t bar_cluster)
{
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(0), "r"(group), "r"(rowblk), "r"(bar_cluster)
      : "memory");
}

// untiled copy of `bytes` (a multiple of 16, both ends 16-byte aligned) to this
// CTA's shared memory, counted on its mbarrier
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes,
                                          uint32_t bar)
{
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// 32 bytes of one lane in one store: whole sectors, where two 16-byte stores
// send two half-filled ones (a lane owns a row here, so lanes do not share them)
__device__ __forceinline__ void store32b(void* p, const uint32_t (&v)[8])
{
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void load32b(const void* p, uint32_t (&v)[8])
{
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
                 "=r"(v[7])
               : "l"(p)
               : "memory");
}
// L2 prefetch of a tile (no shared memory, no completion to wait for)
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* m, int x, int y)
{
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(x), "r"(y)
               : "memory");
}
// 16 consecutive TMEM columns of this thread's lane
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Meet the cluster without ordering memory: for CTAs that have read their peers'
// shared memory (the loads' values are there) and may then exit. The releasing
// form waits for the results' global stores first.
__device__ __forceinline__ void cluster_sync_relaxed()
{
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// 16 bytes of this CTA's shared memory
__device__ __forceinline__ float4 ld_shared4(uint32_t addr)
{
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// 16 bytes of another CTA of the cluster's shared memory
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr)
{
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

}  // namespace u15

// The routed projection in 8-bit floating point (the format: u15_fp8.cuh):
//
//   y[m][n] = epilogue( sum_b 2^(sx[m][b] + sw[n][b] - 254) sum_{k in b} xq[m][k] wq[n][k] )
//
// over the blocks b of 128 columns, wq and sw those of row m's expert, on
// tcgen05.mma kind::mxf8f6f4, which multiplies in the block scales itself:
// products exact, sums f32 in TMEM, nothing to rescale on the way.
#include "u15_fp8.cuh"
#include "u15_kernels.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace u15 {

namespace {

using bf16 = __nv_bfloat16;

// ---------------------------------------------------------------------
// Many rows: a CTA pair (tcgen05 cta_group::2) computes 256 x 256 tiles.
//   warp 0     TMA producer (both CTAs): per stage two k-blocks of 128
//              columns, 128 rows of A and 128 of B a CTA, and the packed
//              scale tiles of their group: the two that the CTA's 128 rows of A
//              lie in, all 256 rows of B
//   warp 1     MMA issuer (leader): copies the stage's scales to TMEM, then
//              eight MMAs of K = 32, the block's scale byte in the descriptor
//   warps 2-9  epilogue, two a TMEM lane quadrant, half the columns each
// TMEM: two accumulators of 256 columns and the scales need more than 512
// columns, so the accumulators share 32: tile t + 1's MMAs wait until the
// epilogue has read those 32 columns of tile t (its first step, ~100 cycles),
// not the whole tile.
//
// SPLIT: fewer tiles than pairs. The k-blocks of a tile are split over the
// pairs of a cluster of 4, 6 or 8 CTAs, a cluster a tile; each CTA leaves its
// 128 x 256 partial sums in shared memory, over the ring, and finishes its share
// of the rows from every pair's (in pair order): 2100 rows x 512 x 4096 are 18
// tiles, 14.3 us on 18 pairs, 12.7 on 54.
// ---------------------------------------------------------------------
constexpr int kKps = 2;                        // k-blocks per stage
constexpr int kStg = 3;
constexpr int kTileBytes = 128 * 128;          // one operand, one k-block, one CTA
constexpr int kStageBytes = 2 * kKps * kTileBytes + 2048;   // operands, then the scales
constexpr int kTurn = 32 * 17;                 // floats a warp turns rows in (turned32)
constexpr int kSmemPair =
    kStg * kStageBytes + 1024 /*align*/ + 2048 /*amax*/ + 256 /*bars*/ + 8 * kTurn * 4;
constexpr int kThreadsPair = 320;
constexpr int kMaxPairs = 4;   // pairs a tile: clusters of 8 CTAs, the portable size
constexpr int kAccStep = 224;                  // accumulator 1 starts 32 columns early
constexpr int kSfCol = 480;                    // two sets of 8 + 8 scale columns

struct PairParams {
  int N;
  int n_units, n_nblk, n_kblk, n_full;
  int nseg;
  int seg_off[kMaxSeg + 1];
  int seg_expert[kMaxSeg];
  int unit_start[kMaxSeg + 1];
  int sf_blk_expert;   // scale row blocks of one expert
  int split;           // SPLIT: pairs a tile
  void* y;
  const bf16* resid;
  const bf16* bias;
  uint8_t* sy;
  unsigned* err;
};

struct PairTile {
  int m0, row_lo, row_hi, expert, nb, half;   // half: -1 full width
};

__device__ __forceinline__ PairTile pair_tile(const PairParams& p, int t)
{
  PairTile r;
  r.half = -1;
  if (t >= p.n_full) {
    const int h = t - p.n_full;
    t = p.n_full + (h >> 1);
    r.half = h & 1;
  }
  // units (256 rows of one segment, from its first row rounded down to 64) run
  // fastest: a round of the schedule reads few columns of B, and A stays in L2.
  // Rows from a multiple of 64 on begin at the first or third scale column of
  // their packed tile, so the four of a CTA's rows are taken from there on into
  // the next tile's columns. (Blocks of 256 rows of the whole pass would
  // need one scale tile, and a unit more where a segment straddles one.)
  const int unit = t % p.n_units;
  r.nb = t / p.n_units;
  int s = 0;
#pragma unroll 1
  for (int k = 1; k < p.nseg; ++k)
    if (unit >= p.unit_start[k]) s = k;
  r.m0 = (p.seg_off[s] & ~63) + (unit - p.unit_start[s]) * 256;
  r.row_lo = max(r.m0, p.seg_off[s]);
  r.row_hi = min(r.m0 + 256, p.seg_off[s + 1]);
  r.expert = p.seg_expert[s];
  return r;
}

// silu(g) * u. The division is off by two units at most: with an exact one as many of 50
// million quantised values (4096 rows x 24576 x 4096: 463, plain f32 sums 240) lie off the
// 64-bit rule's, as the sums' own error decides.
__device__ __forceinline__ float swiglu1(float g, float u)
{
  return __fdividef(g, 1.0f + expf(-g)) * u;
}

// 32 columns of one row, 32-byte aligned
__device__ __forceinline__ void store32(bf16* dst, const float (&v)[32])
{
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = pack_bf2(v[q * 16 + 2 * i], v[q * 16 + 2 * i + 1]);
    store32b(dst + q * 16, o);
  }
}
__device__ __forceinline__ void store32(float* dst, const float (&v)[32])
{
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(v[q * 8 + i]);
    store32b(dst + q * 8, o);
  }
}
__device__ __forceinline__ void add32(float (&v)[32], const bf16* src)
{
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t u[8];
    load32b(src + q * 16, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 a = unpack_bf2(u[i]);
      v[q * 16 + 2 * i] += a.x;
      v[q * 16 + 2 * i + 1] += a.y;
    }
  }
}
// Whether every row of [rows][cols] values of `size` bytes begins on 32 bytes.
__device__ __forceinline__ bool rows_lined(const void* p, long cols, int size)
{
  return (reinterpret_cast<uintptr_t>(p) & 31) == 0 && (cols * size & 31) == 0;
}
// 32 rows of 32 columns of a warp, a row a lane, where rows do not begin on 32 bytes or
// the columns end: turned in shared memory, so that 16 lanes store (and read the
// residual of) 16 neighbouring columns. With each lane at its own row an
// instruction touched 32 sectors for 64 bytes: 3282 rows x 2043 x 336 75 and 18.5 us.
template <int EPI, class T, class P>
__device__ __forceinline__ void turned32(const P& p, float* turn, const float (&v)[32], int row0,
                                         int row_lo, int row_hi, int expert, int col0, int ncols)
{
  const int lane = (int)lane_id(), r = lane >> 4, c = lane & 15;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int col = col0 + h * 16 + c;
    if (col0 + h * 16 >= ncols) break;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) turn[lane * 17 + j] = v[h * 16 + j];
    __syncwarp();
    const bool here = col < ncols;
    float b = 0.0f;
    if ((EPI == kEpiStore || EPI == kEpiStoreF32) && p.bias != nullptr && here)
      b = bf2f(p.bias[(long)expert * p.N + col]);
    // the residual's bits, all loads in flight together: places that are not the
    // segment's read one that is
    uint32_t a[16] = {};
    if constexpr (EPI == kEpiResid) {
      const unsigned short* src =
          reinterpret_cast<const unsigned short*>(p.resid) + min(col, ncols - 1);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        a[i] = src[(long)min(max(row0 + 2 * i + r, row_lo), row_hi - 1) * ncols];
    }
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = turn[(2 * i + r) * 17 + c];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = row0 + 2 * i + r;
      if (!here || row < row_lo || row >= row_hi) continue;
      if (EPI == kEpiResid)
        x[i] += __uint_as_float(a[i] << 16);
      else if (p.bias != nullptr)
        x[i] += b;
      T* const y = static_cast<T*>(p.y) + (long)row * ncols + col;
      if constexpr (sizeof(T) == 4)
        *y = x[i];
      else
        *y = f2bf(x[i]);
    }
  }
}

// four columns of a row, of which the first n exist; `whole`: all four, and
// rows are a multiple of four columns
__device__ __forceinline__ void store4(bf16* dst, const float (&v)[4], bool whole, int n)
{
  if (whole && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) dst[i] = f2bf(v[i]);
  }
}
__device__ __forceinline__ void store4(float* dst, const float (&v)[4], bool whole, int n)
{
  if (whole && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) dst[i] = v[i];
  }
}

// What is added to four columns of R rows, `step` rows apart from `row` on: their
// residual or the bias, as the bits of four bf16. All of a step's rows are read, and
// nothing waits for them, before the first is stored: y may be the residual, so no
// load passes a store, and row after row each load's wait showed (256 rows of 128
// columns: 7.4 us).
template <int EPI, int R, class P>
__device__ __forceinline__ void addend4(uint2 (&a)[R], const P& p, long row, int step, int n_rows,
                                        int expert, int col, int ncols)
{
  if constexpr (EPI == kEpiResid || EPI == kEpiStore || EPI == kEpiStoreF32) {
    const bf16* src = p.resid + row * ncols + col;
    long pitch = (long)step * ncols;
    if (EPI != kEpiResid) {
      if (p.bias == nullptr) return;
      src = p.bias + (long)expert * p.N + col;
      pitch = 0;
    }
    // four columns, aligned together
    if (col + 4 <= ncols && (ncols & 3) == 0 && (reinterpret_cast<uintptr_t>(src) & 7) == 0) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i < n_rows) a[i] = *reinterpret_cast<const uint2*>(src + i * pitch);
    } else {
      // places past the columns or the rows read the last there is
      const unsigned short* u = reinterpret_cast<const unsigned short*>(src);
      uint32_t x[R][4];
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[i][k] = u[min(i, n_rows - 1) * pitch + min(k, ncols - 1 - col)];
#pragma unroll
      for (int i = 0; i < R; ++i)
        a[i] = make_uint2(x[i][0] | x[i][1] << 16, x[i][2] | x[i][3] << 16);
    }
  }
}

// Four finished columns of a row, at column `col` of ncols, a warp a run of 128
// (with SwiGLU applied): the epilogue's other steps and the store. `blk`: the
// block of 128 outputs of a quantised row.
template <int EPI, class P>
__device__ __forceinline__ void finish4(float (&v)[4], uint2 a, const P& p, long row, int blk,
                                        int col, int ncols)
{
  if constexpr (EPI == kEpiSwigluFp8) {
    float m = 0.0f;   // never NaN: fmaxf drops them
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, fabsf(v[k]));
    m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
    const uint32_t sb = fp8_scale_byte(m);
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.y) + row * ncols + col) =
        fp8_codes4(v, fp8_inv_scale(sb, m));
    if (lane_id() == 0) p.sy[fp8_scale_at(row, blk, fp8_groups(ncols))] = (uint8_t)sb;
  } else {
    const long at = row * ncols + col;
    const bool whole = col + 4 <= ncols && (ncols & 3) == 0;
    if (EPI == kEpiResid || ((EPI == kEpiStore || EPI == kEpiStoreF32) && p.bias != nullptr)) {
      const float2 lo = unpack_bf2(a.x), hi = unpack_bf2(a.y);
      v[0] += lo.x;
      v[1] += lo.y;
      v[2] += hi.x;
      v[3] += hi.y;
    }
    if constexpr (EPI == kEpiStoreF32)
      store4(static_cast<float*>(p.y) + at, v, whole, ncols - col);
    else
      store4(static_cast<bf16*>(p.y) + at, v, whole, ncols - col);
  }
}

// Sends the residual of the rows first + k * step < end, `cols` columns from `col`
// on, towards L2, a row a thread: the epilogue reads them when the products are done.
template <class P>
__device__ __forceinline__ void prefetch_resid(const P& p, int first, int step, int end, int n_thr,
                                               int thr, int col, int cols)
{
  for (int j = first + thr * step; j < end; j += n_thr * step)
    for (int c = col; c < min(col + cols, p.N); c += 64)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.resid + (long)j * p.N + c));
}

template <int EPI, bool SPLIT>
__global__ void __launch_bounds__(kThreadsPair, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmA,
                         const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmBh,
                         const __grid_constant__ CUtensorMap tmSA,
                         const __grid_constant__ CUtensorMap tmSB,
                         const __grid_constant__ CUtensorMap tmSBh,
                         const __grid_constant__ PairParams p)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // [2 tiles][2 halves of the columns][128 rows]
  float* amax_sm = reinterpret_cast<float*>(smem + kStg * kStageBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStg * kStageBytes + 2048);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStg + 8);

  const uint32_t full0 = smem_u32(bars);        // leader: count 2 (one per CTA) + tx
  const uint32_t empty0 = full0 + 8 * kStg;     // each CTA: leader's multicast commit
  const uint32_t accf0 = empty0 + 8 * kStg;     // each CTA, per accumulator: the same
  const uint32_t accr = accf0 + 16;             // leader: 512 epilogue threads, a phase a tile
  const uint32_t drain = accr + 8;              // each CTA
  const uint32_t amax0 = drain + 8;             // each CTA, a lane quadrant: 64 threads

  const uint32_t w = warp_id();
  // rank: in the pair
  const uint32_t cta = cluster_ctarank(), rank = cta & 1, lead_cta = cta & ~1u;
  const bool leader = rank == 0;
  const uint16_t both = (uint16_t)(3u << lead_cta);   // the pair's CTAs, for commits
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStg; ++s) {
      mbar_init(full0 + 8 * s, 2);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(accf0, 1);
    mbar_init(accf0 + 8, 1);
    mbar_init(accr, 512);
    mbar_init(drain, 1);
    for (int i = 0; i < 4; ++i) mbar_init(amax0 + 8 * i, 64);
    fence_barrier_init();
  }
  if (w == 0) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  tc_fence_before();
  cluster_sync();   // barriers of both CTAs initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_launch();
  griddep_wait();

  const int n_tiles = p.n_full + 2 * (p.n_units * p.n_nblk - p.n_full);
  // tiles of this pair, and the k-blocks of them that it takes
  const int pair = SPLIT ? blockIdx.x / (2 * p.split) : blockIdx.x >> 1;
  const int n_pairs = SPLIT ? n_tiles : gridDim.x >> 1;
  const int n_st = (p.n_kblk + kKps - 1) / kKps, part = SPLIT ? (int)(cta >> 1) : 0;
  const int kb0 = SPLIT ? part * n_st / p.split * kKps : 0;
  const int kb1 = SPLIT ? min((part + 1) * n_st / p.split * kKps, p.n_kblk) : p.n_kblk;
  const uint32_t base = smem_u32(smem);

  if (w == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    uint32_t it = 0;
    bool ok = true;
    for (int t = pair; t < n_tiles && ok; t += n_pairs) {
      const PairTile ti = pair_tile(p, t);
      const bool half = ti.half >= 0;
      const int arow = ti.m0 + 128 * (int)rank;
      const int brow = ti.expert * p.N + ti.nb * 256 +
                       (half ? 128 * ti.half + 64 * (int)rank : 128 * (int)rank);
      const int sblk = ti.expert * p.sf_blk_expert + ti.nb * 2 + (half ? ti.half : 0);
      const uint32_t tx = kTileBytes + (half ? kTileBytes / 2 : kTileBytes);
      const uint32_t tx_sf = half ? 3 * kFp8SfTile : 4 * kFp8SfTile;
      const CUtensorMap *mb = half ? &tmBh : &tmB, *msb = half ? &tmSBh : &tmSB;
      for (int kb = kb0; kb < kb1; kb += kKps, ++it) {
        const uint32_t s = it % kStg, ph = (it / kStg) & 1;
        if (!warp_wait(empty0 + 8 * s, ph ^ 1, p.err, kDevWaitEmpty)) {
          ok = false;
          break;
        }
        const int nk = min(kKps, kb1 - kb);
        const uint32_t fb = mapa_shared(full0 + 8 * s, lead_cta);
        const uint32_t st = base + s * kStageBytes;
        // a scale tile serves four k-blocks: it comes with the first of them
        const bool sfs = kb == kb0 || (kb & 3) == 0;
        if (elect_one()) {
          mbar_arrive_expect_tx_cluster(fb, nk * tx + (sfs ? tx_sf : 0));
          if (sfs) {
            const uint32_t sf = st + 2 * kKps * kTileBytes;
            tma_load_sf_pair(sf, &tmSA, kb >> 2, arow >> 7, fb);
            tma_load_sf_pair(sf + 2 * kFp8SfTile, msb, kb >> 2, sblk, fb);
          }
#pragma unroll
          for (int hk = 0; hk < kKps; ++hk) {
            if (hk >= nk) break;
            const int kx = (kb + hk) * 128;
            tma_load_2d_pair(st + hk * kTileBytes, &tmA, kx, arow, fb);
            tma_load_2d_pair(st + (kKps + hk) * kTileBytes, mb, kx, brow, fb);
          }
        }
        __syncwarp();
      }
    }
    // unwinding (leader): the last fill of every stage, both CTAs' halves,
    // has landed once the leader's full barrier for it completes
    if (leader) {
      for (uint32_t s = 0; s < kStg; ++s) {
        if (it > s) {
          const uint32_t last = ((it - 1 - s) / kStg) * kStg + s;
          warp_wait(full0 + 8 * s, (last / kStg) & 1, p.err, kDevWaitDrain);
        }
      }
    }
  } else if (w == 1) {
    // ---------------- MMA issuer (leader only) ----------------
    if (leader) {
      uint32_t it = 0, sf_set = 0;
      int lt = 0;
      bool ok = true;
      for (int t = pair; t < n_tiles && ok; t += n_pairs, ++lt) {
        const bool half = t >= p.n_full;
        const uint32_t idesc = half ? idesc_e4m3(256, 128) : idesc_e4m3(256, 256);
        // the previous tile's shared columns have been read (and with them
        // all of the tile before it)
        if (lt > 0 && !warp_wait_cluster_probe(accr, (lt - 1) & 1, p.err, kDevWaitAccEmpty)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (lt & 1) * kAccStep;
        const uint32_t a_col = (pair_tile(p, t).m0 >> 5) & 3;   // of the unit's first row: 0 or 2
        for (int kb = kb0; kb < kb1; kb += kKps, ++it) {
          const uint32_t s = it % kStg, ph = (it / kStg) & 1;
          if (!warp_wait_probe(full0 + 8 * s, ph, p.err, kDevWaitFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int nk = min(kKps, kb1 - kb);
          const uint32_t st = base + s * kStageBytes;
          const bool sfs = kb == kb0 || (kb & 3) == 0;
          sf_set ^= sfs;
          const uint32_t sfa = tmem_base + kSfCol + sf_set * 16, sfb = sfa + 8;
          const uint64_t ad = smem_desc_sw128(st), bd = smem_desc_sw128(st + kKps * kTileBytes);
          if (elect_one()) {
            if (sfs) {
              const uint64_t sf = smem_desc_sf(st + 2 * kKps * kTileBytes);
              sf_copy_pair(sfa, sf);
              if (a_col) sf_copy_pair(sfa + 4, sf + (kFp8SfTile >> 4));
              sf_copy_pair(sfb, sf + 2 * (kFp8SfTile >> 4));
              if (!half) sf_copy_pair(sfb + 4, sf + 3 * (kFp8SfTile >> 4));
            }
#pragma unroll
            for (int hk = 0; hk < kKps; ++hk) {
              if (hk >= nk) break;
              const uint32_t id = idesc | idesc_scale_byte((kb + hk) & 3);
              // K = 32 steps are 32 bytes, 2 descriptor units, apart
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_e4m3_pair(d_tmem, ad + hk * (kTileBytes >> 4) + k * 2,
                              bd + hk * (kTileBytes >> 4) + k * 2, id, sfa + a_col, sfb,
                              ((kb - kb0 + hk) | k) != 0);
            }
            mma_commit_pair_mc(empty0 + 8 * s, both);
          }
          __syncwarp();
        }
        if (ok && elect_one()) mma_commit_pair_mc(accf0 + 8 * (lt & 1), both);
        __syncwarp();
      }
      if (elect_one()) mma_commit_pair_mc(drain, both);
      __syncwarp();
    }
    // both CTAs: every MMA that writes this CTA's TMEM has completed
    warp_wait(drain, 0, p.err, kDevWaitDrain);
  } else if constexpr (!SPLIT) {
    // ---------------- epilogue (warps 2..9, both CTAs) ----------------
    const int wq = (int)(w & 3), wh = (int)(w - 2) >> 2;   // lane quadrant, half of the columns
    const int r_in = wq * 32 + (int)lane_id();
    float* const turn = reinterpret_cast<float*>(bars) + 64 + ((int)w - 2) * kTurn;
    const uint32_t accr_leader = mapa_shared(accr, lead_cta);
    int lt = 0;
    for (int t = pair; t < n_tiles; t += n_pairs, ++lt) {
      const PairTile ti = pair_tile(p, t);
      const bool half = ti.half >= 0;
      const int acc = lt & 1;
      if (!warp_wait(accf0 + 8 * acc, (lt >> 1) & 1, p.err, kDevWaitAccFull)) break;
      tc_fence_after();
      const int row = ti.m0 + 128 * (int)rank + r_in;
      const bool row_ok = row >= ti.row_lo && row < ti.row_hi;
      const uint32_t tb = tmem_base + acc * kAccStep + ((uint32_t)(wq * 32) << 16);
      // the 32 columns the accumulators share are the last of accumulator 0
      // and the first of accumulator 1; their warps read them first
      const bool shared_here = wh == (acc ^ 1);
      bool released = t + n_pairs >= n_tiles;   // nobody waits for the last tile's
      auto release = [&] {
        if (released) return;
        released = true;
        tc_fence_before();
        mbar_arrive_cluster(accr_leader);
      };
      if (!shared_here) release();
      if constexpr (GU) {
        // columns [0, 128) are gate rows, [128, 256) the matching up rows;
        // this warp's 64 outputs in two runs of 32, the shared columns' first
        const int nout = p.N / 2;
        float h[2][32];
        int run[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          run[i] = wh * 2 + (acc == 0 && wh == 1 ? 1 - i : i);
          uint32_t g[32], u[32];
          tmem_ld32(tb + run[i] * 32, g);
          tmem_ld32(tb + 128 + run[i] * 32, u);
          tmem_ld_wait();
          release();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            h[i][j] = swiglu1(__uint_as_float(g[j]), __uint_as_float(u[j]));
        }
        if constexpr (EPI == kEpiSwiglu) {
          bf16* yrow = static_cast<bf16*>(p.y) + (long)row * nout + ti.nb * 128;
          const bool lined = rows_lined(p.y, nout, 2);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (!lined)
              turned32<EPI, bf16>(p, turn, h[i], row - (int)lane_id(), ti.row_lo, ti.row_hi,
                                  ti.expert, ti.nb * 128 + run[i] * 32, nout);
            else if (row_ok)
              store32(yrow + run[i] * 32, h[i]);
          }
        } else {
          // the row's largest of 128 outputs, over the quadrant's two warps
          float m = 0.0f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j) m = fmaxf(m, fabsf(h[i][j]));
          float* am = amax_sm + acc * 256;
          am[wh * 128 + r_in] = m;
          mbar_arrive(amax0 + 8 * wq);
          if (!warp_wait(amax0 + 8 * wq, lt & 1, p.err, kDevWaitAccFull)) break;
          m = fmaxf(m, am[(wh ^ 1) * 128 + r_in]);
          const uint32_t sb = fp8_scale_byte(m);
          const float inv = fp8_inv_scale(sb, m);
          if (row_ok) {
            uint8_t* yrow = static_cast<uint8_t*>(p.y) + (long)row * nout + ti.nb * 128;
            const bool whole_sectors = (reinterpret_cast<uintptr_t>(p.y) & 31) == 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint2 c[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = h[i][q * 8 + j];
                c[q] = fp8_codes8(v, inv);
              }
              const uint32_t o[8] = {c[0].x, c[0].y, c[1].x, c[1].y,
                                     c[2].x, c[2].y, c[3].x, c[3].y};
              if (whole_sectors) {
                store32b(yrow + run[i] * 32, o);
              } else {
                uint4* d = reinterpret_cast<uint4*>(yrow + run[i] * 32);
                d[0] = make_uint4(o[0], o[1], o[2], o[3]);
                d[1] = make_uint4(o[4], o[5], o[6], o[7]);
              }
            }
            if (wh == 0) p.sy[fp8_scale_at(row, ti.nb, fp8_groups(nout))] = (uint8_t)sb;
          }
        }
      } else {
        using Out = std::conditional_t<EPI == kEpiStoreF32, float, bf16>;
        const bool lined = rows_lined(p.y, p.N, sizeof(Out)) &&
                           (EPI == kEpiResid ? rows_lined(p.resid, p.N, 2)
                                             : p.bias == nullptr || rows_lined(p.bias, p.N, 2));
        const int n0 = ti.nb * 256 + (half ? 128 * ti.half : 0);
        const int nch = half ? 2 : 4;                 // chunks of 32 columns of this warp
        const int first = half ? wh * 2 : wh * 4;
        // a half-width tile uses columns [0, 128) of its accumulator: only
        // accumulator 1 shares any of them
        const int lead = acc == 0 && !half && wh == 1 ? 3 : 0;
        if (half && acc == 0) release();
#pragma unroll 1
        for (int i = 0; i < nch; ++i) {
          const int c = first + ((i + lead) & (nch - 1));
          uint32_t r[32];
          tmem_ld32(tb + c * 32, r);
          tmem_ld_wait();
          release();
          const int col0 = n0 + c * 32;
          if (col0 >= p.N) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (!lined || col0 + 32 > p.N) {
            turned32<EPI, Out>(p, turn, v, row - (int)lane_id(), ti.row_lo, ti.row_hi, ti.expert,
                               col0, p.N);
          } else if (row_ok) {
            if (EPI != kEpiResid && p.bias != nullptr)
              add32(v, p.bias + (long)ti.expert * p.N + col0);
            if constexpr (EPI == kEpiResid) add32(v, p.resid + (long)row * p.N + col0);
            store32(static_cast<Out*>(p.y) + (long)row * p.N + col0, v);
          }
        }
      }
    }
  }

  if constexpr (SPLIT) {
    // ---------------- partial sums, then whole rows ----------------
    // row r's 16-byte chunk c at r * 1024 + (c ^ (r & 7)) * 16: lanes that hold a row
    // each write, and a warp that takes a row reads, without bank conflicts
    const PairTile ti = pair_tile(p, pair);
    bool ok = true;
    if (w >= 2) {
      ok = warp_wait(accf0, 0, p.err, kDevWaitAccFull);
      tc_fence_after();
      const int wq = (int)(w & 3), wh = (int)(w - 2) >> 2, r_in = wq * 32 + (int)lane_id();
#pragma unroll 1
      for (int c = wh * 4; c < wh * 4 + 4; ++c) {
        uint32_t v[32];
        tmem_ld32(tmem_base + ((uint32_t)(wq * 32) << 16) + c * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4*>(smem + r_in * 1024 + (((c * 8 + i) ^ (r_in & 7)) << 4)) =
              make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
    }
    __syncthreads();
    cluster_sync();
    if (ok) {
      const int first = ti.m0 + 128 * (int)rank, step = (kThreadsPair / 32) * p.split;
      const int lo = max(ti.row_lo - first, 0), hi = min(ti.row_hi - first, 128);
      const int lane = (int)lane_id();
      // R rows a step of a warp from up to Q pairs, all their loads in flight
      auto finish = [&](auto r_, auto q_) {
        constexpr int R = decltype(r_)::value, Q = decltype(q_)::value;
        for (int j0 = lo + part + (int)w * p.split; j0 < hi; j0 += R * step) {
          uint2 a[2][R] = {};
          if constexpr (!GU) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              addend4<EPI>(a[h], p, first + j0, step, (hi - j0 + step - 1) / step, ti.expert,
                           ti.nb * 256 + h * 128 + lane * 4, p.N);
          }
          float4 v[Q][R][2] = {};
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            if (q >= p.split) break;
            const uint32_t from = mapa_shared(base, 2 * q + rank);
#pragma unroll
            for (int i = 0; i < R; ++i) {
              const int j = j0 + i * step;
              if (j >= hi) break;
#pragma unroll
              for (int h = 0; h < 2; ++h)
                v[q][i][h] = ld_cluster4(from + j * 1024 + (((lane + 32 * h) ^ (j & 7)) << 4));
            }
          }
#pragma unroll
          for (int i = 0; i < R; ++i) {
            if (j0 + i * step >= hi) break;
            float t[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float4 x = v[0][i][h];
#pragma unroll
              for (int q = 1; q < Q; ++q) {
                x.x += v[q][i][h].x;
                x.y += v[q][i][h].y;
                x.z += v[q][i][h].z;
                x.w += v[q][i][h].w;
              }
              t[h][0] = x.x;
              t[h][1] = x.y;
              t[h][2] = x.z;
              t[h][3] = x.w;
            }
            const long row = first + j0 + i * step;
            if constexpr (GU) {
#pragma unroll
              for (int k = 0; k < 4; ++k) t[0][k] = swiglu1(t[0][k], t[1][k]);
              finish4<EPI>(t[0], a[0][i], p, row, ti.nb, ti.nb * 128 + lane * 4, p.N / 2);
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h)
                finish4<EPI>(t[h], a[h][i], p, row, ti.nb, ti.nb * 256 + h * 128 + lane * 4, p.N);
            }
          }
        }
      };
      using std::integral_constant;
      if (p.split == 2)
        finish(integral_constant<int, 4>{}, integral_constant<int, 2>{});
      else
        finish(integral_constant<int, 2>{}, integral_constant<int, kMaxPairs>{});
    }
  }

  tc_fence_before();
  __syncthreads();
  // The peers' shared memory and TMEM stay alive until all are done with them:
  // every arrival on the leader's barriers and every commit has been waited for,
  // and partial sums are read, so nothing needs the results' stores to land first
  cluster_sync_relaxed();
  if (w == 0) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------
// Few rows: the weights are the bytes that count. A tile is 128 weight rows
// (SwiGLU: the 128 gate rows and the 128 up rows that go with them) by all the
// activation rows there are, MT at most, the weights as the MMA's M = 128 side, so a
// lane of the accumulator is an output column and its columns are the activation
// rows. A segment is a unit of its own (with its expert's weights) that finishes
// its rows of them; the rows of a pass begin at their first scale column.
// The k-blocks of a tile are split over the CTAs of a cluster; their partial
// sums meet in shared memory, each CTA adding (in rank order) and finishing
// its share of the rows. The runtime keeps one CTA with a TMEM allocation on
// an SM, so a CTA rings ~200 KB of weights, two k-blocks a stage (one k-block
// a stage: the issuer's ~200 cycles a stage showed).
//   warp 0     TMA producer
//   warp 1     MMA issuer
//   warps 2-5  TMEM -> shared memory; then every warp: the sum over the
//              cluster and the epilogue, a row a warp
// ---------------------------------------------------------------------
constexpr int kThreadsFew = 192;
constexpr int kFewPrefetch = 4;     // k-blocks a CTA sends towards L2 ahead of its loads
constexpr int kMaxSplit = 8;        // the portable cluster size

template <int MT, bool GU>
struct FewCfg {
  static constexpr int kNA = GU ? 2 : 1;
  static constexpr int kKps = GU && MT >= 64 ? 1 : 2;       // k-blocks per stage
  static constexpr int kA = kNA * kTileBytes;               // of one k-block
  static constexpr int kB = MT * 128;
  static constexpr int kStage = kKps * (kA + kB) + 2048;    // + the scale tiles
  static constexpr int kStages = (232448 - 1280) / kStage < 6 ? (232448 - 1280) / kStage : 6;
  static constexpr int kSmem = kStages * kStage + 1024 /*align*/ + 256 /*bars*/;
  static constexpr int kAcc = kNA * MT;                     // accumulator columns
  static constexpr int kSf = GU ? 12 : 8;                   // scale columns of a set, two sets
  static constexpr int kCols = kAcc + 2 * kSf <= 64    ? 64
                               : kAcc + 2 * kSf <= 128 ? 128
                               : kAcc + 2 * kSf <= 256 ? 256
                                                       : 512;
  static_assert(kStages >= 3 && kStages * kStage >= kAcc * 512, "the partial sums take the ring");
};

struct FewParams {
  int N, n_kblk;
  int lo[kMaxSeg], hi[kMaxSeg], expert[kMaxSeg];   // the segments that hold rows
  int sf_blk_expert;
  void* y;
  const bf16* resid;
  const bf16* bias;
  uint8_t* sy;
  unsigned* err;
};

template <int MT, int EPI>
__global__ void __launch_bounds__(kThreadsFew, 1)
    gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap tmX,
                        const __grid_constant__ CUtensorMap tmW,
                        const __grid_constant__ CUtensorMap tmSX,
                        const __grid_constant__ CUtensorMap tmSW,
                        const __grid_constant__ FewParams p)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  using C = FewCfg<MT, GU>;
  constexpr int NA = GU ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStage);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::kStages + 2);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * C::kStages,
                 accf = empty0 + 8 * C::kStages, drain = accf + 8;

  griddep_launch();
  const uint32_t w = warp_id();
  const int split = (int)gridDim.x, rank = (int)blockIdx.x;   // the cluster is the x axis
  const int tile = blockIdx.y;
  const int lo = p.lo[blockIdx.z], hi = p.hi[blockIdx.z], expert = p.expert[blockIdx.z];
  // this CTA's stages of the tile, and their first k-block
  const int n_st = (p.n_kblk + C::kKps - 1) / C::kKps;
  const int st0 = rank * n_st / split, st1 = (rank + 1) * n_st / split;
  const int wrow = expert * p.N + tile * 128 * NA;
  const uint32_t base = smem_u32(smem);

  // stage i of this CTA (its empty barrier waited for by the caller)
  auto load = [&](int i) {
    const int s = i % C::kStages, kb = (st0 + i) * C::kKps;
    const int nk = min(C::kKps, p.n_kblk - kb);
    const uint32_t st = base + s * C::kStage, fb = full0 + 8 * s;
    const bool sfs = i == 0 || (kb & 3) == 0;   // a scale tile serves its four k-blocks
    if (elect_one()) {
      mbar_arrive_expect_tx(fb, nk * (C::kA + C::kB) + (sfs ? (NA + 1) * kFp8SfTile : 0));
#pragma unroll
      for (int hk = 0; hk < C::kKps; ++hk) {
        if (hk >= nk) break;
#pragma unroll
        for (int h = 0; h < NA; ++h)
          tma_load_2d(st + (hk * NA + h) * kTileBytes, &tmW, (kb + hk) * 128, wrow + 128 * h, fb);
        tma_load_2d(st + C::kKps * C::kA + hk * C::kB, &tmX, (kb + hk) * 128, 0, fb);
      }
      if (sfs) {
        const uint32_t sf = st + C::kKps * (C::kA + C::kB);
        tma_load_sf(sf, &tmSX, kb >> 2, 0, fb);
#pragma unroll
        for (int h = 0; h < NA; ++h)
          tma_load_sf(sf + (1 + h) * kFp8SfTile, &tmSW, kb >> 2,
                      expert * p.sf_blk_expert + tile * NA + h, fb);
      }
    }
    __syncwarp();
  };

  const int n_it = st1 - st0;
  if (w == 0) {
    if (elect_one()) {
      for (int s = 0; s < C::kStages; ++s) {
        mbar_init(full0 + 8 * s, 1);
        mbar_init(empty0 + 8 * s, 1);
      }
      mbar_init(accf, 1);
      mbar_init(drain, 1);
      fence_barrier_init();
      tma_prefetch_desc(&tmW);
      tma_prefetch_desc(&tmX);
      tma_prefetch_desc(&tmSW);
      tma_prefetch_desc(&tmSX);
      // the weights' first tiles start towards L2 while the previous kernel
      // still runs (a prefetch reads nothing into this CTA: were they being
      // written, L2 holds the new bytes when the loads come)
      for (int i = 0; i < min(kFewPrefetch, min(st1 * C::kKps, p.n_kblk) - st0 * C::kKps); ++i)
        for (int h = 0; h < NA; ++h)
          tma_prefetch_2d(&tmW, (st0 * C::kKps + i) * 128, wrow + 128 * h);
    }
    __syncwarp();
    griddep_wait();
    for (int i = 0; i < min(C::kStages, n_it); ++i) load(i);   // the ring is empty
  } else if (w == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (w == 0) {
    int it = min(C::kStages, n_it);
    for (; it < n_it; ++it) {
      const int s = it % C::kStages, ph = (it / C::kStages) & 1;
      if (!warp_wait(empty0 + 8 * s, ph ^ 1, p.err, kDevWaitEmpty)) break;
      load(it);
    }
    for (int s = 0; s < C::kStages; ++s)   // every fill has landed before the CTA may exit
      if (it > s) warp_wait(full0 + 8 * s, ((it - 1 - s) / C::kStages) & 1, p.err, kDevWaitDrain);
  } else if (w == 1) {
    constexpr uint32_t idesc = idesc_e4m3(128, MT);
    uint32_t set = 0;
    bool ok = true;
    for (int it = 0; it < n_it; ++it) {
      const int s = it % C::kStages, ph = (it / C::kStages) & 1;
      if (!warp_wait_probe(full0 + 8 * s, ph, p.err, kDevWaitFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int kb = (st0 + it) * C::kKps;
      const int nk = min(C::kKps, p.n_kblk - kb);
      const uint32_t st = base + s * C::kStage;
      const bool sfs = it == 0 || (kb & 3) == 0;
      set ^= sfs;
      const uint32_t sfx = tmem + C::kAcc + set * C::kSf, sfw = sfx + 4;
      const uint64_t ad = smem_desc_sw128(st), bd = smem_desc_sw128(st + C::kKps * C::kA);
      if (elect_one()) {
        if (sfs) {
          const uint64_t sf = smem_desc_sf(st + C::kKps * (C::kA + C::kB));
          sf_copy(sfx, sf);
#pragma unroll
          for (int h = 0; h < NA; ++h) sf_copy(sfw + 4 * h, sf + (1 + h) * (kFp8SfTile >> 4));
        }
#pragma unroll
        for (int hk = 0; hk < C::kKps; ++hk) {
          if (hk >= nk) break;
          const uint32_t id = idesc | idesc_scale_byte((kb + hk) & 3);
          // K = 32 steps are 32 bytes, 2 descriptor units, apart
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int h = 0; h < NA; ++h)
              mma_e4m3(tmem + h * MT, ad + (hk * NA + h) * (kTileBytes >> 4) + k * 2,
                       bd + hk * (C::kB >> 4) + k * 2, id, sfw + 4 * h, sfx, (it | hk | k) != 0);
        }
        mma_commit(empty0 + 8 * s);
      }
      __syncwarp();
    }
    if (elect_one()) {
      if (ok) mma_commit(accf);
      mma_commit(drain);
    }
    __syncwarp();
    warp_wait(drain, 0, p.err, kDevWaitDrain);
  }

  if (w != 0) griddep_wait();
  float* part = reinterpret_cast<float*>(smem);   // [NA][MT rows][128 columns], over the ring
  const int wq = (int)(w & 3), n = wq * 32 + (int)lane_id();
  bool ok = true;
  if (w >= 2) {
    if constexpr (EPI == kEpiResid)
      prefetch_resid(p, lo + rank, split, hi, 128, (int)threadIdx.x - 64, tile * 128, 128);
    // every MMA of this CTA has completed, and with them every load
    ok = warp_wait(accf, 0, p.err, kDevWaitAccFull);
    tc_fence_after();
    const uint32_t tb = tmem + ((uint32_t)(wq * 32) << 16);
#pragma unroll 1
    for (int c = (lo & ~15); c < hi; c += 16) {
#pragma unroll
      for (int h = 0; h < NA; ++h) {
        uint32_t r[16];
        tmem_ld16(tb + h * MT + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(h * MT + c + i) * 128 + n] = __uint_as_float(r[i]);
      }
    }
  }
  __syncthreads();
  cluster_sync();   // every CTA's partial sums are in its shared memory

  if (ok) {
    // a warp finishes whole rows, four columns a lane: the sum over the
    // cluster in rank order, and a row's largest needs no other warp. A step's
    // loads are all in flight together: R rows from up to Q CTAs (row by row,
    // 128 rows of an unsplit tile took 5 us; four rows from two CTAs at a time,
    // eight CTAs' sums 2 us more)
    constexpr int kWarps = kThreadsFew / 32;
    const uint32_t own = smem_u32(part) + lane_id() * 16;
    const int ncols = GU ? p.N / 2 : p.N, col = tile * 128 + (int)lane_id() * 4;
    const int step = kWarps * split;
    auto finish = [&](auto r_, auto q_) {
      constexpr int R = decltype(r_)::value, Q = decltype(q_)::value;
      for (int j0 = lo + rank + (int)w * split; j0 < hi; j0 += R * step) {
        uint2 a[R] = {};
        addend4<EPI>(a, p, j0, step, (hi - j0 + step - 1) / step, expert, col, ncols);
        float4 v[Q][NA][R] = {};
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          if (q >= split) break;
          const uint32_t from = mapa_shared(own, q);
#pragma unroll
          for (int h = 0; h < NA; ++h)
#pragma unroll
            for (int i = 0; i < R; ++i)
              if (j0 + i * step < hi) {
                const int at = h * MT + j0 + i * step;
                v[q][h][i] = Q == 1 ? ld_shared4(own + at * 512) : ld_cluster4(from + at * 512);
              }
        }
        float4 t[NA][R];
#pragma unroll
        for (int h = 0; h < NA; ++h)
#pragma unroll
          for (int i = 0; i < R; ++i) {
            t[h][i] = v[0][h][i];
#pragma unroll
            for (int q = 1; q < Q; ++q) {
              t[h][i].x += v[q][h][i].x;
              t[h][i].y += v[q][h][i].y;
              t[h][i].z += v[q][h][i].z;
              t[h][i].w += v[q][h][i].w;
            }
          }
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (j0 + i * step >= hi) break;
          float v[4] = {t[0][i].x, t[0][i].y, t[0][i].z, t[0][i].w};
          if constexpr (GU) {
            v[0] = swiglu1(v[0], t[1][i].x);
            v[1] = swiglu1(v[1], t[1][i].y);
            v[2] = swiglu1(v[2], t[1][i].z);
            v[3] = swiglu1(v[3], t[1][i].w);
          }
          finish4<EPI>(v, a[i], p, j0 + i * step, tile, col, ncols);
        }
      }
    };
    using std::integral_constant;
    if (split == 1)
      finish(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (split == 2)
      finish(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else
      finish(integral_constant<int, 1>{}, integral_constant<int, kMaxSplit>{});
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();   // the peers have read this CTA's partial sums
  if (w == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
}

// ---------------------------------------------------------------------
// Some hundred rows: 256-row tiles would compute rows that are not there, and
// the few-row form loads the activations beside every 128 weight rows. Here a
// CTA pair's M = 256 side is weights, 128 rows (SwiGLU: 128 gate and 128 up
// rows) a CTA, and its N side a unit of up to kRows activation rows, as many as the
// segment has there rounded up to 32, half of them loaded by each CTA. A
// CTA's accumulator then is its own 128 columns of all the unit's rows, and
// the epilogue is the few-row form's. The k-blocks of a tile are split over the
// pairs of a cluster. A stage is as large as the unit's rows make it, so small units
// have more of them in flight.
//   A k-block of 256 rows takes 286 ns, the MMAs' own time 270; of 64 rows 160, the
// weights' loads 135 at 64 bytes a cycle. One k-block a stage took 50 to 130 ns more
// (the handshake of two CTAs costs ~200 a stage). What a tile spends outside its
// k-blocks, 4 to 8.5 us, no other tile on its SM hides: the ring and the partial
// sums take the shared memory of one CTA.
//   warp 0     TMA producer (both CTAs)
//   warp 1     MMA issuer (leader)
//   warps 2-17 TMEM -> shared memory (an unsplit SwiGLU tile: with SwiGLU done); then
//              every warp: the sum over the cluster's pairs and the epilogue, a row
//              a warp (8 warps: 256 rows x 4096 x 512 9.1 us, 16 8.5)
// ---------------------------------------------------------------------
constexpr int kDrainMid = 16;       // warps that empty the accumulators
constexpr int kThreadsMid = 64 + 32 * kDrainMid;
// Rows up to which this form is considered: what the unit table holds, not a
// measured crossover (the pairs' tiles leave places empty above it too: 2500 rows x
// 1024 x 12288 are 40 tiles on 74 pairs, 35 us).
constexpr int kMidRows = 2048;
constexpr int kMidRounds = 1024;    // rows up to which in more than one round of tiles
constexpr int kMidUnits = 48;       // units of a pass: 2048 rows / 64, and two ends a segment

template <bool GU>
struct MidCfg {
  static constexpr int kNA = GU ? 2 : 1;
  static constexpr int kRows = GU ? 192 : 256;              // of a unit: TMEM holds NA x kRows
  static constexpr int kXTiles = GU ? 2 : 3;                // scale tiles that its rows lie in
  static constexpr int kKps = GU ? 1 : 2;                   // k-blocks per stage
  static constexpr int kA = kNA * kTileBytes;               // a k-block, a CTA
  static constexpr int kMaxStages = 6;
  static constexpr int kBody = 225 * 1024;                  // the ring, then the partial sums
  static constexpr int kSmem = kBody + 1024 /*align*/ + 256 /*bars*/;
  static constexpr int kAcc = kNA * kRows;
  static constexpr int kSf = 4 * (kNA + kXTiles);           // scale columns of a set, two sets
  // a stage's bytes: operands (xr activation rows a CTA), then the scale tiles
  __host__ __device__ static constexpr int stage(int xr) { return kKps * (kA + xr * 128) + 2048; }
  static_assert(kAcc + 2 * kSf <= 512 && (kNA + kXTiles) * kFp8SfTile <= 2048 && kSmem <= 232448);
  static_assert(3 * stage(kRows / 2) <= kBody && kNA * kRows * 512 <= kBody);
};

struct MidUnit {
  int m0, expert;   // first row, a multiple of 64
  short lo, hi;     // rows [m0 + lo, m0 + hi) are the segment's
};

struct MidParams {
  int N, n_kblk;
  int sf_blk_expert;
  bool units_first;   // the units of a weight tile run side by side
  void* y;
  const bf16* resid;
  const bf16* bias;
  uint8_t* sy;
  unsigned* err;
  MidUnit unit[kMidUnits];
};

template <int EPI>
__global__ void __launch_bounds__(kThreadsMid, 1)
    gemm_fp8_mid_kernel(const __grid_constant__ CUtensorMap tmX,
                        const __grid_constant__ CUtensorMap tmW,
                        const __grid_constant__ CUtensorMap tmSX,
                        const __grid_constant__ CUtensorMap tmSW,
                        const __grid_constant__ MidParams p)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  using C = MidCfg<GU>;
  constexpr int NA = C::kNA;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBody);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::kMaxStages + 2);
  const uint32_t full0 = smem_u32(bars);               // leader: count 2 (one per CTA) + tx
  const uint32_t empty0 = full0 + 8 * C::kMaxStages;   // each CTA: leader's multicast commit
  const uint32_t accf = empty0 + 8 * C::kMaxStages, drain = accf + 8;   // the same

  griddep_launch();
  const uint32_t w = warp_id();
  const uint32_t cta = cluster_ctarank(), rank = cta & 1, lead_cta = cta & ~1u;
  const uint16_t both = (uint16_t)(3u << lead_cta);
  const int split = (int)gridDim.x >> 1, part_k = (int)(cta >> 1);   // the cluster is the x axis
  // this CTA's 128 output columns, and its rows
  const int blk = (int)(p.units_first ? blockIdx.z : blockIdx.y) * 2 + (int)rank;
  const MidUnit u = p.unit[p.units_first ? blockIdx.y : blockIdx.z];
  const int nr = (u.hi + 31) & ~31;                  // rows the MMAs take
  const int xr = ((nr >> 1) + 31) & ~31;             // rows a CTA loads, in boxes of 32
  // this CTA's stages of the tile, and their first k-block
  const int n_st = (p.n_kblk + C::kKps - 1) / C::kKps, st0 = part_k * n_st / split;
  const int n_it = (part_k + 1) * n_st / split - st0, kb0 = st0 * C::kKps;
  // the ring: as many stages of this unit's size as fit
  const int stage = C::stage(xr), n_ring = min(C::kMaxStages, C::kBody / stage);
  const uint32_t base = smem_u32(smem);
  // scale tiles of the unit's rows, and the scale column of its first (0 or 2)
  const int x_tiles = ((u.m0 & 127) + nr + 127) >> 7, x_col = (u.m0 >> 5) & 3;

  if (threadIdx.x == 0) {
    for (int s = 0; s < n_ring; ++s) {
      mbar_init(full0 + 8 * s, 2);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(accf, 1);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (w == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  const int wrow = u.expert * p.N + blk * 128 * NA;
  if (threadIdx.x == 64) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmSW);
    tma_prefetch_desc(&tmSX);
    // as in the few-row form, while the previous kernel still runs
    for (int i = 0; i < min(kFewPrefetch, min(n_it * C::kKps, p.n_kblk - kb0)); ++i)
      for (int h = 0; h < NA; ++h) tma_prefetch_2d(&tmW, (kb0 + i) * 128, wrow + 128 * h);
  }
  tc_fence_before();
  cluster_sync();   // barriers of both CTAs initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();

  if (w == 0) {
    int it = 0;
    for (int s = 0, ph = 0; it < n_it; ++it) {
      if (!warp_wait_probe(empty0 + 8 * s, ph ^ 1, p.err, kDevWaitEmpty)) break;
      const int kb = kb0 + it * C::kKps, nk = min(C::kKps, p.n_kblk - kb);
      const uint32_t st = base + s * stage, fb = mapa_shared(full0 + 8 * s, lead_cta);
      const bool sfs = it == 0 || (kb & 3) == 0;   // a scale tile serves its four k-blocks
      if (elect_one()) {
        mbar_arrive_expect_tx_cluster(
            fb, nk * (C::kA + xr * 128) + (sfs ? (NA + x_tiles) * kFp8SfTile : 0));
        if (sfs) {
          const uint32_t sf = st + C::kKps * (C::kA + xr * 128);
#pragma unroll
          for (int h = 0; h < NA; ++h)
            tma_load_sf_pair(sf + h * kFp8SfTile, &tmSW, kb >> 2,
                             u.expert * p.sf_blk_expert + blk * NA + h, fb);
          for (int i = 0; i < x_tiles; ++i)
            tma_load_sf_pair(sf + (NA + i) * kFp8SfTile, &tmSX, kb >> 2, (u.m0 >> 7) + i, fb);
        }
        const int x0 = u.m0 + (int)rank * (nr >> 1);
#pragma unroll
        for (int hk = 0; hk < C::kKps; ++hk) {
          if (hk >= nk) break;
          const int kx = (kb + hk) * 128;
#pragma unroll
          for (int h = 0; h < NA; ++h)
            tma_load_2d_pair(st + (hk * NA + h) * kTileBytes, &tmW, kx, wrow + 128 * h, fb);
          const uint32_t xb = st + C::kKps * C::kA + hk * xr * 128;
          for (int i = 0; i < xr; i += 32) tma_load_2d_pair(xb + i * 128, &tmX, kx, x0 + i, fb);
        }
      }
      __syncwarp();
      if (++s == n_ring) s = 0, ph ^= 1;
    }
    // the leader: the last fill of every stage, both CTAs' halves, has landed
    if (rank == 0)
      for (int s = 0; s < n_ring; ++s)
        if (it > s) warp_wait(full0 + 8 * s, ((it - 1 - s) / n_ring) & 1, p.err, kDevWaitDrain);
  } else if (w == 1) {
    if (rank == 0) {
      const uint32_t idesc = idesc_e4m3(256, nr);
      uint32_t set = 0;
      bool ok = true;
      for (int it = 0, s = 0, ph = 0; it < n_it; ++it) {
        if (!warp_wait_probe(full0 + 8 * s, ph, p.err, kDevWaitFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int kb = kb0 + it * C::kKps, nk = min(C::kKps, p.n_kblk - kb);
        const uint32_t st = base + s * stage;
        const bool sfs = it == 0 || (kb & 3) == 0;
        set ^= sfs;
        const uint32_t sfw = tmem + C::kAcc + set * C::kSf, sfx = sfw + 4 * NA;
        const uint64_t ad = smem_desc_sw128(st), bd = smem_desc_sw128(st + C::kKps * C::kA);
        if (elect_one()) {
          if (sfs) {
            const uint64_t sf = smem_desc_sf(st + C::kKps * (C::kA + xr * 128));
            for (int i = 0; i < NA + x_tiles; ++i)
              sf_copy_pair(sfw + 4 * i, sf + i * (kFp8SfTile >> 4));
          }
#pragma unroll
          for (int hk = 0; hk < C::kKps; ++hk) {
            if (hk >= nk) break;
            const uint32_t id = idesc | idesc_scale_byte((kb + hk) & 3);
            // K = 32 steps are 32 bytes, 2 descriptor units, apart
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int h = 0; h < NA; ++h)
                mma_e4m3_pair(tmem + h * C::kRows, ad + (hk * NA + h) * (kTileBytes >> 4) + k * 2,
                              bd + hk * xr * 8 + k * 2, id, sfw + 4 * h, sfx + x_col,
                              (it | hk | k) != 0);
          }
          mma_commit_pair_mc(empty0 + 8 * s, both);
        }
        __syncwarp();
        if (++s == n_ring) s = 0, ph ^= 1;
      }
      if (elect_one()) {
        if (ok) mma_commit_pair_mc(accf, both);
        mma_commit_pair_mc(drain, both);
      }
      __syncwarp();
    }
    // both CTAs: every MMA that writes this CTA's TMEM has completed
    warp_wait(drain, 0, p.err, kDevWaitDrain);
  }

  float* part = reinterpret_cast<float*>(smem);   // [NA][rows][128 columns], over the ring
  bool ok = true;
  if (w >= 2) {
    if constexpr (EPI == kEpiResid)
      prefetch_resid(p, u.m0 + u.lo + part_k, split, u.m0 + u.hi, 32 * kDrainMid,
                     (int)threadIdx.x - 64, blk * 128, 128);
    // every MMA of the pair has completed, and with them every load of both CTAs
    ok = warp_wait(accf, 0, p.err, kDevWaitAccFull);
    tc_fence_after();
    const int wq = (int)(w & 3), n = wq * 32 + (int)lane_id();
    const uint32_t tb = tmem + ((uint32_t)(wq * 32) << 16);
#pragma unroll 1
    for (int c = (u.lo & ~15) + ((int)(w - 2) >> 2) * 16; c < u.hi && ok; c += 4 * kDrainMid) {
      uint32_t r[NA][16];
#pragma unroll
      for (int h = 0; h < NA; ++h) tmem_ld16(tb + h * C::kRows + c, r[h]);
      tmem_ld_wait();
      float* const to = part + c * 128 + n;
      if (GU && split == 1) {   // gate and up of a column are here together
#pragma unroll
        for (int i = 0; i < 16; ++i)
          to[i * 128] = swiglu1(__uint_as_float(r[0][i]), __uint_as_float(r[NA - 1][i]));
      } else {
#pragma unroll
        for (int h = 0; h < NA; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) to[(h * C::kRows + i) * 128] = __uint_as_float(r[h][i]);
      }
    }
  }
  __syncthreads();
  if (split > 1) cluster_sync();   // every pair's partial sums are in its shared memory

  const int ncols = GU ? p.N / 2 : p.N, col = blk * 128 + (int)lane_id() * 4;
  if (ok && blk * 128 < ncols) {   // the last pair's second CTA may be past the columns
    constexpr int kWarps = kThreadsMid / 32;
    const uint32_t own = smem_u32(part) + lane_id() * 16;
    const int step = kWarps * split;
    auto finish = [&](auto r_, auto q_) {
      constexpr int R = decltype(r_)::value, Q = decltype(q_)::value;
      constexpr int NS = Q == 1 ? 1 : NA;   // sums a column: SwiGLU of an unsplit tile is done
      for (int j0 = u.lo + part_k + (int)w * split; j0 < u.hi; j0 += R * step) {
        uint2 a[R] = {};
        addend4<EPI>(a, p, u.m0 + j0, step, (u.hi - j0 + step - 1) / step, u.expert, col, ncols);
        float4 v[Q][NS][R] = {};
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          if (q >= split) break;
          const uint32_t from = mapa_shared(own, 2 * q + rank);
#pragma unroll
          for (int h = 0; h < NS; ++h)
#pragma unroll
            for (int i = 0; i < R; ++i)
              if (j0 + i * step < u.hi) {
                const int at = h * C::kRows + j0 + i * step;
                v[q][h][i] = Q == 1 ? ld_shared4(own + at * 512) : ld_cluster4(from + at * 512);
              }
        }
        float4 t[NS][R];
#pragma unroll
        for (int h = 0; h < NS; ++h)
#pragma unroll
          for (int i = 0; i < R; ++i) {
            t[h][i] = v[0][h][i];
#pragma unroll
            for (int q = 1; q < Q; ++q) {
              t[h][i].x += v[q][h][i].x;
              t[h][i].y += v[q][h][i].y;
              t[h][i].z += v[q][h][i].z;
              t[h][i].w += v[q][h][i].w;
            }
          }
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (j0 + i * step >= u.hi) break;
          float o[4] = {t[0][i].x, t[0][i].y, t[0][i].z, t[0][i].w};
          if constexpr (NS == 2) {
            o[0] = swiglu1(o[0], t[1][i].x);
            o[1] = swiglu1(o[1], t[1][i].y);
            o[2] = swiglu1(o[2], t[1][i].z);
            o[3] = swiglu1(o[3], t[1][i].w);
          }
          finish4<EPI>(o, a[i], p, u.m0 + j0 + i * step, blk, col, ncols);
        }
      }
    };
    using std::integral_constant;
    if (split == 1)
      finish(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (split == 2)
      finish(integral_constant<int, 4 / NA>{}, integral_constant<int, 2>{});
    else
      finish(integral_constant<int, 2 / NA>{}, integral_constant<int, kMaxPairs>{});
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();   // the peers have read this CTA's partial sums, and its TMEM is idle
  if (w == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Row units of segment s in the pair form: blocks of 256 from its first row rounded
// down to 64.
inline int pair_units_of(const SegInfo& seg, int s)
{
  const int lo = seg.off[s], hi = seg.off[s + 1];
  return hi > lo ? (hi - (lo & ~63) + 255) / 256 : 0;
}

// Clusters of 1 to kMaxPairs pairs that can be resident (not every SM has a
// usable partner, and larger clusters leave more SMs out), asked once per kernel
// and device; null where the device refuses the kernel.
template <int EPI, bool SPLIT>
const int* pair_resident(int num_sms)
{
  static std::atomic<uint64_t> attr_set;
  static std::mutex mu;
  static int resident_dev[64][kMaxPairs + 1];
  auto k = gemm_fp8_pair_kernel<EPI, SPLIT>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || !smem_attr_once(k, kSmemPair, attr_set)) return nullptr;
  std::lock_guard<std::mutex> g(mu);
  int* r = resident_dev[dev & 63];
  if (r[0] != 0) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreadsPair);
  cfg.dynamicSmemBytes = kSmemPair;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int s = 1; s <= kMaxPairs; ++s) {
    attr[0].val.clusterDim.x = 2 * s;
    cfg.gridDim = dim3(2 * s);
    if (cudaOccupancyMaxActiveClusters(&r[s], k, &cfg) != cudaSuccess || r[s] <= 0) {
      cudaGetLastError();   // an estimate serves
      r[s] = std::max(1, num_sms / (4 * s));
    }
  }
  r[0] = 1;   // the entries are there
  return r;
}

// split 1: a persistent grid of as many pairs as can be resident at once; more:
// that many pairs a tile, a cluster a tile.
template <int EPI, bool SPLIT>
int launch_pair(const GemmFp8Args& a, const SegInfo& seg, int split, cudaStream_t st,
                std::string* err)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  PairParams p{};
  p.N = a.N;
  p.y = a.y;
  p.resid = static_cast<const bf16*>(a.resid);
  p.bias = static_cast<const bf16*>(a.bias);
  p.sy = a.sy;
  p.err = a.dev_err;
  p.nseg = seg.nseg;
  for (int s = 0; s < seg.nseg; ++s) {
    p.seg_off[s] = seg.off[s];
    p.seg_expert[s] = seg.expert[s];
    p.unit_start[s] = p.n_units;
    p.n_units += pair_units_of(seg, s);
  }
  p.seg_off[seg.nseg] = seg.off[seg.nseg];
  p.unit_start[seg.nseg] = p.n_units;
  p.n_nblk = (a.N + 255) / 256;
  p.n_kblk = fp8_blocks(a.K);
  p.sf_blk_expert = (a.N + 127) / 128;
  p.split = split;
  if ((long)p.n_units * p.n_nblk > 0x3FFFFFFFL) {
    *err = "gemm_fp8: too many output tiles";
    return 1;
  }
  CUtensorMap ma, mb, mbh, msa, msb, msbh;
  const uint64_t wrows = (uint64_t)a.N * a.n_experts, groups = fp8_groups(a.K),
                 wblks = (uint64_t)p.sf_blk_expert * a.n_experts, xblks = (a.M + 127) / 128;
  if (encode_tma_2d(&ma, a.xq, a.M, a.K, 128, 1, err) ||
      encode_tma_2d(&mb, a.wq, wrows, a.K, 128, 1, err) ||
      encode_tma_2d(&mbh, a.wq, wrows, a.K, 64, 1, err) ||
      make_tma_fp8_scales(&msa, a.sx, xblks, groups, 2, err) ||
      make_tma_fp8_scales(&msb, a.sw, wblks, groups, 2, err) ||
      make_tma_fp8_scales(&msbh, a.sw, wblks, groups, 1, err))
    return 2;
  const int* resident = pair_resident<EPI, SPLIT>(a.num_sms);
  if (resident == nullptr) return 2;
  const int tiles = p.n_units * p.n_nblk;
  int ctas;
  if constexpr (SPLIT) {
    p.n_full = tiles;
    ctas = 2 * split * tiles;
  } else {
    // a last round that would leave at least half the pairs idle runs as
    // half-width tiles (a SwiGLU tile holds whole gate and up blocks: it is not
    // split)
    const int pairs = std::min(tiles, resident[1]), rest = tiles % pairs;
    p.n_full = !GU && rest > 0 && 2 * rest <= pairs ? tiles - rest : tiles;
    ctas = 2 * pairs;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreadsPair);
  cfg.dynamicSmemBytes = kSmemPair;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 2 * split;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_pair_kernel<EPI, SPLIT>, ma, mb, mbh, msa, msb, msbh,
                            p) == cudaSuccess
             ? 0
             : 2;
}

// The few-row form's cluster size (how many CTAs share a tile's k-blocks) with
// the least time, and that time in nanoseconds as measured: rounds of the grid
// times (a CTA's stages + its set-up, first loads and epilogue), plus what the
// exchange of the partial sums costs. resident[s]: the clusters of s CTAs that run at once,
// which the layout of the SMs makes fewer than SMs / s for most s.
struct FewPlan {
  int split = 1;
  long ns = -1;
};
inline FewPlan few_plan(long tiles, int n_stages, int stage_ns, int round_ns, const int* resident)
{
  FewPlan best;
  for (int s = 1; s <= kMaxSplit && s <= n_stages; ++s) {
    const long rounds = (tiles + resident[s] - 1) / resident[s];
    const long ns = rounds * ((n_stages + s - 1) / s * (long)stage_ns + round_ns) +
                    (s > 1 ? 400 + 50 * s : 0);
    if (best.ns < 0 || ns < best.ns) best = FewPlan{s, ns};
  }
  return best;
}

// Clusters of each size that can be resident, asked once per kernel and device.
template <int MT, int EPI>
const int* few_resident(int num_sms)
{
  using C = FewCfg<MT, EPI == kEpiSwiglu || EPI == kEpiSwigluFp8>;
  static std::atomic<uint64_t> attr_set;
  static std::mutex mu;
  static int resident_dev[64][kMaxSplit + 1];
  auto k = gemm_fp8_few_kernel<MT, EPI>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || !smem_attr_once(k, C::kSmem, attr_set)) return nullptr;
  std::lock_guard<std::mutex> g(mu);
  int* r = resident_dev[dev & 63];
  if (r[0] != 0) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreadsFew);
  cfg.dynamicSmemBytes = C::kSmem;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int s = 1; s <= kMaxSplit; ++s) {
    attr[0].val.clusterDim.x = s;
    cfg.gridDim = dim3(s);
    if (cudaOccupancyMaxActiveClusters(&r[s], k, &cfg) != cudaSuccess || r[s] <= 0) {
      cudaGetLastError();   // an estimate serves
      r[s] = std::max(1, num_sms / s / 2);
    }
  }
  r[0] = 1;   // the entries are there
  return r;
}

template <int EPI>
int few_tiles(const GemmFp8Args& a)
{
  return EPI == kEpiSwiglu || EPI == kEpiSwigluFp8 ? a.N / 256 : (a.N + 127) / 128;
}

template <int MT, int EPI>
FewPlan few_plan_of(const GemmFp8Args& a, const SegInfo& seg, const int* resident)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  using C = FewCfg<MT, GU>;
  long tiles = 0;
  for (int s = 0; s < seg.nseg; ++s)
    if (seg.off[s + 1] > seg.off[s]) tiles += few_tiles<EPI>(a);
  // a k-block of 128 weight rows: 160 ns; a round's set-up, first loads and
  // epilogue: 2.5 us and 20 ns a row
  const int stage_ns = C::kKps * C::kNA * 160;
  return few_plan(tiles, (fp8_blocks(a.K) + C::kKps - 1) / C::kKps, stage_ns, 2500 + 20 * MT,
                  resident);
}

template <int MT, int EPI>
int launch_few(const GemmFp8Args& a, const SegInfo& seg, const FewPlan& plan, cudaStream_t st,
               std::string* err)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  using C = FewCfg<MT, GU>;
  FewParams p{};
  p.N = a.N;
  p.n_kblk = fp8_blocks(a.K);
  p.sf_blk_expert = (a.N + 127) / 128;
  p.y = a.y;
  p.resid = static_cast<const bf16*>(a.resid);
  p.bias = static_cast<const bf16*>(a.bias);
  p.sy = a.sy;
  p.err = a.dev_err;
  int units = 0;   // launch_rows: a.M <= MT
  for (int s = 0; s < seg.nseg; ++s) {
    if (seg.off[s + 1] <= seg.off[s]) continue;
    p.lo[units] = seg.off[s];
    p.hi[units] = seg.off[s + 1];
    p.expert[units++] = seg.expert[s];
  }
  const int tiles = few_tiles<EPI>(a);
  CUtensorMap mx, mw, msx, msw;
  const uint64_t groups = fp8_groups(a.K);
  if (encode_tma_2d(&mx, a.xq, a.M, a.K, MT, 1, err) ||
      encode_tma_2d(&mw, a.wq, (uint64_t)a.N * a.n_experts, a.K, 128, 1, err) ||
      make_tma_fp8_scales(&msx, a.sx, (a.M + 127) / 128, groups, 1, err) ||
      make_tma_fp8_scales(&msw, a.sw, (uint64_t)p.sf_blk_expert * a.n_experts, groups, 1, err))
    return 2;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreadsFew);
  cfg.gridDim = dim3(plan.split, tiles, units);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = plan.split;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_few_kernel<MT, EPI>, mx, mw, msx, msw, p) == cudaSuccess
             ? 0
             : 2;
}

// Clusters of 1 to kMaxPairs pairs of the form above that can be resident.
template <int EPI>
const int* mid_resident(int num_sms)
{
  using C = MidCfg<EPI == kEpiSwiglu || EPI == kEpiSwigluFp8>;
  static std::atomic<uint64_t> attr_set;
  static std::mutex mu;
  static int resident_dev[64][kMaxPairs + 1];
  auto k = gemm_fp8_mid_kernel<EPI>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || !smem_attr_once(k, C::kSmem, attr_set)) return nullptr;
  std::lock_guard<std::mutex> g(mu);
  int* r = resident_dev[dev & 63];
  if (r[0] != 0) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreadsMid);
  cfg.dynamicSmemBytes = C::kSmem;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int s = 1; s <= kMaxPairs; ++s) {
    attr[0].val.clusterDim.x = 2 * s;
    cfg.gridDim = dim3(2 * s);
    if (cudaOccupancyMaxActiveClusters(&r[s], k, &cfg) != cudaSuccess || r[s] <= 0) {
      cudaGetLastError();   // an estimate serves
      r[s] = std::max(1, num_sms / (4 * s));
    }
  }
  r[0] = 1;   // the entries are there
  return r;
}

struct MidPlan {
  int height = 64, split = 1;   // rows of a unit, pairs a tile
  bool units_first = false;
  bool one_round = false;
  long ns = -1;
};

// The units of height `h`, tallest first (the last round then holds the small
// ones), and how many they are.
inline int mid_units(const SegInfo& seg, int h, MidUnit* unit)
{
  int n = 0;
  for (int s = 0; s < seg.nseg; ++s) {
    const int end = seg.off[s + 1];
    if (end <= seg.off[s]) continue;
    for (int m0 = seg.off[s] & ~63; m0 < end; m0 += h, ++n)
      unit[n] = MidUnit{m0, seg.expert[s], (short)std::max(0, seg.off[s] - m0),
                        (short)std::min(h, end - m0)};
  }
  std::sort(unit, unit + n, [](const MidUnit& a, const MidUnit& b) { return a.hi > b.hi; });
  return n;
}

template <int EPI>
int mid_tiles(const GemmFp8Args& a)
{
  return EPI == kEpiSwiglu || EPI == kEpiSwigluFp8 ? (a.N + 511) / 512 : (a.N + 255) / 256;
}

// Nanoseconds of a k-block of a unit of nr rows, and of its set-up, first loads and
// epilogue, as measured (4096 columns of one unit, K 512 and 4096: 64 rows 4.5 and
// 9.3 us, 128 5.7 and 10.7, 256 8.5 and 16.6; the SwiGLU form, two units of 192 rows x
// 16384: 10.7 and 24.3).
// With many CTAs at it the SwiGLU form's loads count (two weight tiles a k-block):
// 12.3 TB/s into all of the chip's shared memory.
template <bool GU>
inline long mid_kblk_ns(int nr, int ctas)
{
  if (!GU) return std::max(160, 90 + 3 * nr / 4);
  const long bytes = MidCfg<GU>::kA + nr * 64;
  return std::max<long>(std::max(280, 5 * nr / 2), ctas * bytes / 12300);
}
template <bool GU>
inline long mid_unit_ns(int nr)
{
  return GU ? 2800 + 32 * nr : 2700 + 18 * nr;
}

template <int EPI>
MidPlan mid_plan_of(const GemmFp8Args& a, const SegInfo& seg, const int* resident)
{
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  const int n_kblk = fp8_blocks(a.K), tiles = mid_tiles<EPI>(a);
  // every pair of a split tile has a stage: one without would add what its
  // accumulators held
  constexpr int kps = MidCfg<GU>::kKps;
  const int most = std::min(kMaxPairs, (n_kblk + kps - 1) / kps);
  MidPlan best;
  for (int h = 64; h <= MidCfg<GU>::kRows; h += 64) {
    MidUnit unit[kMidUnits];
    const int n = mid_units(seg, h, unit);
    for (int s = 1; s <= most; ++s) {
      // tile i's time, the tiles in order of their units' heights
      const long places = resident[s], all = (long)tiles * n;
      auto time = [&](long i) {
        const int nr = (unit[i / tiles].hi + 31) & ~31;
        const int ctas = 2 * s * (int)std::min(places, all);
        return (n_kblk + s - 1) / s * mid_kblk_ns<GU>(nr, ctas) + mid_unit_ns<GU>(nr);
      };
      // rounds of as many tiles as run at once, each the time of its first; of the
      // last two, the later one's tiles start as the smallest before them end
      long ns = s > 1 ? 1000 + 300 * s : 0, t0 = 0;
      for (; all - t0 > 2 * places; t0 += places) ns += time(t0);
      const long late = all - t0 - places;
      ns += late <= 0 ? time(t0)
                      : std::max({time(t0), time(t0 + places - 1) + time(t0 + places),
                                  time(t0 + places - late) + time(all - 1)});
      if (best.ns < 0 || ns < best.ns) {
        best.height = h;
        best.split = s;
        // A weight tile's units side by side read it from HBM once; one after the
        // other, tallest first, a short last round holds small ones only (two
        // segments, 333 x 24576 x 4096 SwiGLU, 144 tiles on 74 places: 53.5 and 58
        // us; 1000 x 4096 x 12288, 80 tiles: 64 and 52)
        best.units_first = 2 * ((all - 1) % places + 1) > places;
        best.one_round = all <= places;
        best.ns = ns;
      }
    }
  }
  return best;
}

template <int EPI>
int launch_mid(const GemmFp8Args& a, const SegInfo& seg, const MidPlan& plan, cudaStream_t st,
               std::string* err)
{
  using C = MidCfg<EPI == kEpiSwiglu || EPI == kEpiSwigluFp8>;
  MidParams p{};
  p.N = a.N;
  p.n_kblk = fp8_blocks(a.K);
  p.sf_blk_expert = (a.N + 127) / 128;
  p.y = a.y;
  p.resid = static_cast<const bf16*>(a.resid);
  p.bias = static_cast<const bf16*>(a.bias);
  p.sy = a.sy;
  p.err = a.dev_err;
  p.units_first = plan.units_first;
  const int units = mid_units(seg, plan.height, p.unit), tiles = mid_tiles<EPI>(a);
  CUtensorMap mx, mw, msx, msw;
  const uint64_t groups = fp8_groups(a.K);
  if (encode_tma_2d(&mx, a.xq, a.M, a.K, 32, 1, err) ||
      encode_tma_2d(&mw, a.wq, (uint64_t)a.N * a.n_experts, a.K, 128, 1, err) ||
      make_tma_fp8_scales(&msx, a.sx, (a.M + 127) / 128, groups, 1, err) ||
      make_tma_fp8_scales(&msw, a.sw, (uint64_t)p.sf_blk_expert * a.n_experts, groups, 1, err))
    return 2;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreadsMid);
  cfg.gridDim = p.units_first ? dim3(2 * plan.split, units, tiles)
                              : dim3(2 * plan.split, tiles, units);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 2 * plan.split;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, gemm_fp8_mid_kernel<EPI>, mx, mw, msx, msw, p) == cudaSuccess ? 0
                                                                                               : 2;
}

// More than 64 rows: tiles of 256 rows (pairs, one or several a tile), or up to 2048
// rows units of the rows there are, whichever form takes less time by the models
// above (333 rows in two segments x 4096 x 12288: 28 us, in tiles of 256 or
// 128 rows 40; 1000 rows 52 and 62; 100 rows x 6144 x 4096: 13 to 16 and 16 to 21).
// Above 1024 rows only where its tiles all run at once: their epilogues overlap
// nothing, the persistent pairs' do (1512 rows x 1148 x 960 7.4 and 12.3 us, 1418 x
// 4864 x 10592, two rounds, 79 and 67). The models are off by some 5 % where both
// forms are short: 1867 rows x 1024 x 768 with SwiGLU take 7.4 us, pairs 7.0, and
// 1867 x 768 x 1024 8.0, pairs 7.5.
template <int EPI>
int launch_many(const GemmFp8Args& a, const SegInfo& seg, cudaStream_t st, std::string* err)
{
  const long n_st = (fp8_blocks(a.K) + kKps - 1) / kKps;
  long tiles = 0;
  for (int s = 0; s < seg.nseg; ++s) tiles += (long)pair_units_of(seg, s) * ((a.N + 255) / 256);
  const int* one = pair_resident<EPI, false>(a.num_sms);
  if (one == nullptr) return 2;
  // measured: 790 ns a stage of a pair and 5.5 us to start and finish, a last
  // round of half-width tiles half a round (launch_pair); 850 ns and 8.5 us where
  // partial sums meet
  constexpr bool GU = EPI == kEpiSwiglu || EPI == kEpiSwigluFp8;
  int split = 1;
  const long rest = tiles % one[1];
  const long halves = 2 * (tiles / one[1]) +
                      (rest == 0 ? 0 : !GU && tiles > one[1] && 2 * rest <= one[1] ? 1 : 2);
  long pair_ns = halves * n_st * 395 + 5500;
  if (tiles < one[1]) {
    const int* more = pair_resident<EPI, true>(a.num_sms);
    if (more == nullptr) return 2;
    for (int s = 2; s <= kMaxPairs && s <= n_st; ++s) {
      const long ns = (tiles + more[s] - 1) / more[s] * ((n_st + s - 1) / s * 850 + 8500);
      if (ns < pair_ns) {
        pair_ns = ns;
        split = s;
      }
    }
  }
  if (a.M <= kMidRows && mid_tiles<EPI>(a) <= 65535) {
    const int* resident = mid_resident<EPI>(a.num_sms);
    if (resident == nullptr) return 2;
    const MidPlan mid = mid_plan_of<EPI>(a, seg, resident);
    if (mid.ns < pair_ns && (a.M <= kMidRounds || mid.one_round))
      return launch_mid<EPI>(a, seg, mid, st, err);
  }
  return split > 1 ? launch_pair<EPI, true>(a, seg, split, st, err)
                   : launch_pair<EPI, false>(a, seg, 1, st, err);
}

template <int MT, int EPI>
int launch_few_rows(const GemmFp8Args& a, const SegInfo& seg, cudaStream_t st, std::string* err)
{
  const int* resident = few_resident<MT, EPI>(a.num_sms);
  if (resident == nullptr) return 2;
  return launch_few<MT, EPI>(a, seg, few_plan_of<MT, EPI>(a, seg, resident), st, err);
}

template <int EPI>
int launch_rows(const GemmFp8Args& a, const SegInfo& seg, cudaStream_t st, std::string* err)
{
  if (a.M > 64 || few_tiles<EPI>(a) > 65535) return launch_many<EPI>(a, seg, st, err);
  if (a.M <= 16) return launch_few_rows<16, EPI>(a, seg, st, err);
  if (a.M <= 32) return launch_few_rows<32, EPI>(a, seg, st, err);
  return launch_few_rows<64, EPI>(a, seg, st, err);
}

}  // namespace

int gemm_fp8(const GemmFp8Args& a, const SegInfo& seg, cudaStream_t st, std::string* err)
{
  err->clear();
  int rc;
  switch (a.epilogue) {
    case kEpiStore: rc = launch_rows<kEpiStore>(a, seg, st, err); break;
    case kEpiResid: rc = launch_rows<kEpiResid>(a, seg, st, err); break;
    case kEpiSwiglu: rc = launch_rows<kEpiSwiglu>(a, seg, st, err); break;
    case kEpiStoreF32: rc = launch_rows<kEpiStoreF32>(a, seg, st, err); break;
    default: rc = launch_rows<kEpiSwigluFp8>(a, seg, st, err); break;
  }
  if (rc && err->empty()) *err = "gemm_fp8: kernel launch failed";
  return rc;
}

}  // namespace u15

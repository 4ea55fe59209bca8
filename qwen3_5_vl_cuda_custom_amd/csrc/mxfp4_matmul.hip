// Products with MXFP4 weights (format: mxfp4.h): y = x w^T (+ bias) (+ residual), x
// and y bf16, w (N, K) codes and scales, fp32 accumulation, one rounding. The
// weights enter the matrix cores as their exact values in bf16, x as it is.
#include <algorithm>

#include "gemm_tile.h"
#include "mxfp4.h"
#include "mxfp4_rows.h"

namespace {

using namespace q3;

struct MxGemm {
  const bf16* x;
  const uint8_t* w;  // codes
  const uint8_t* s;  // scales
  const bf16* bias;
  const bf16* res;
  bf16* y;
  float* part;  // (gridDim.y, M, N) sums, or null: the block writes y
  int M, N, K;
  int64_t ldx, ldw, lds, ldr, ldc;  // ldw, lds in bytes
  int vec;  // N a multiple of 4, the rows of y, bias and residual in 8-byte pieces
};

__device__ __forceinline__ void store_y(const MxGemm& p, int m, int n, float v) {
  if (p.bias) v += bf2f(p.bias[n]);
  if (p.res) v += bf2f(p.res[m * p.ldr + n]);
  p.y[m * p.ldc + n] = f2bf(v);
}
// Four columns at once (p.vec: every row of y, bias and residual in 8-byte pieces).
__device__ __forceinline__ void store_y4(const MxGemm& p, int m, int n, floatx4 v) {
  if (p.bias) {
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(p.bias + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bf2f(b[e]);
  }
  if (p.res) {
    const bf16x4 b = *reinterpret_cast<const bf16x4*>(p.res + m * p.ldr + n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bf2f(b[e]);
  }
  bf16x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = f2bf(v[e]);
  *reinterpret_cast<bf16x4*>(p.y + m * p.ldc + n) = o;
}

// ------------------------------------------------------------------ more rows
// x through LDS. A block of eight waves, WM along m and 8 / WM along n, forms a tile
// of BN = 16 RT (8 / WM) columns and BM rows over its k range, in stages of BK: every
// load goes global -> LDS past the registers, a ring of NST stages keeps NST - 1 in
// flight, one barrier per stage. Row r of a 16-row group of codes is BK / 2 bytes, row
// m of x 2 BK; their 16-byte chunk c lies at slot c ^ wswz(r), c ^ (m & 15), so that the
// 16 rows of a fragment read use all banks. Scales are loaded as words of four (ALIGNED:
// the rows of scales start at multiples of four bytes), else byte by byte (a load of
// one byte per lane costs as much as one of sixteen: M=32 N=151936 158 -> 113 us without).
// 128 rows run at 1.1 PFLOP/s of the CUs they fill (M=512 N=12288 K=4096: 192 tiles, 67
// us), 32 rows at the loads into LDS (N=4096 K=12288: 11 us for 26.7 MB of weights and
// 98 KB of x per CU, and 3.8 for the sum over 8 ranges).
template <int RT, int BM, int WM, int BK, int NST, bool ALIGNED>
__global__ __launch_bounds__(512) void mx_tile_kernel(const MxGemm p) {
  constexpr int NW = 8, WN = NW / WM, BN = 16 * RT * WN, MT = BM / 16 / WM;
  constexpr int CW = BK / 32, CX = BK / 8;       // 16-byte chunks of a row of codes, of x
  constexpr int WPT = CW / 4, TPW = RT / WM;     // loads of a 16-row group's codes; groups a wave loads
  constexpr int PX = BM * CX / 64 / NW, PW = TPW * WPT;
  constexpr int SB = TPW * 16 * CW;              // scales a wave loads
  constexpr int PS = ALIGNED ? 1 : SB / 64;
  constexpr int PER = PX + PW + PS;
  constexpr int kX = BM * BK * 2, kW = BN * BK / 2, kS = 256 * PS, kStage = kX + kW + NW * kS;  // bytes
  static_assert(BM * CX % (64 * NW) == 0 && RT % WM == 0 && SB <= 256 && SB % 64 == 0, "whole loads per wave");
  __shared__ __attribute__((aligned(1024))) char smem[NST * kStage];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int r = lane & 15, g = lane >> 4;
  const int tiles_n = (p.N + BN - 1) / BN;
  const int tn = blockIdx.x % tiles_n, tm = blockIdx.x / tiles_n;
  const int n0 = tn * BN, m0 = tm * BM;
  const int blocks = p.K / kMxBlock, steps = (blocks + CW - 1) / CW;
  const int t0 = (int)((int64_t)steps * blockIdx.y / gridDim.y), t1 = (int)((int64_t)steps * (blockIdx.y + 1) / gridDim.y);
  const uint32_t lbase = lds_addr(smem);
  auto wswz = [](int row) { return row / (16 / CW) & (CW - 1); };

  // This wave's loads, as byte offsets of stage 0 from the tile's first row.
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * p.ldx, ((int64_t)(min(BM, p.M - m0) - 1) * p.ldx + p.K) * 2);
  const int nrows = min(BN, p.N - n0);
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + (int64_t)n0 * p.ldw, (int64_t)(nrows - 1) * p.ldw + p.K / 2);
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.s + (int64_t)n0 * p.lds, (int64_t)(nrows - 1) * p.lds + blocks);
  const int group0 = RT * wn + TPW * wm;  // first 16-row group it loads
  uint32_t xoff[PX], woff[PW], soff[PS];
  int xc[PX], wc[PW], sb[PS];  // and their first chunk, code chunk (= block), scale
#pragma unroll
  for (int i = 0; i < PX; ++i) {
    const int at = (wave * PX + i) * 64 + lane, m = at / CX;
    xc[i] = at % CX ^ (m & 15);
    xoff[i] = m0 + m < p.M ? (uint32_t)(m * p.ldx * 2 + xc[i] * 16) : kOOB;
  }
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int at = i % WPT * 64 + lane, row = at / CW, n = 16 * (group0 + i / WPT) + row;
    wc[i] = at % CW ^ wswz(row);
    woff[i] = n < nrows ? (uint32_t)(n * p.ldw + wc[i] * 16) : kOOB;
  }
#pragma unroll
  for (int i = 0; i < PS; ++i) {
    const int at = ALIGNED ? 4 * lane : 64 * i + lane, n = 16 * group0 + at / CW;
    sb[i] = at % CW;
    soff[i] = at < SB && n < nrows ? (uint32_t)(n * p.lds + sb[i]) : kOOB;
  }
  auto issue = [&](int t) {
    const uint32_t at = lbase + (uint32_t)((t - t0) % NST) * kStage;
    const int left = t < t1 ? blocks - t * CW : 0;  // blocks from this stage's first on
#pragma unroll
    for (int i = 0; i < PX; ++i)
      dma16(rx, xoff[i] != kOOB && xc[i] < 4 * left ? xoff[i] + (uint32_t)t * (BK * 2) : kOOB,
            at + (wave * PX + i) * 1024);
#pragma unroll
    for (int i = 0; i < PW; ++i)
      dma16(rw, woff[i] != kOOB && wc[i] < left ? woff[i] + (uint32_t)t * (BK / 2) : kOOB,
            at + kX + (group0 * WPT + i) * 1024);
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const uint32_t off = soff[i] != kOOB && sb[i] < left ? soff[i] + (uint32_t)t * CW : kOOB;
      if constexpr (ALIGNED) dma4(rs, off, at + kX + kW + wave * kS);
      else dma1(rs, off, at + kX + kW + wave * kS + 256 * i);
    }
  };

  floatx4 acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{};
#pragma unroll 1
  for (int i = 0; i < NST - 1; ++i) issue(t0 + i);
  for (int t = t0; t < t1; ++t) {
    vm_wait<(NST - 2) * PER>();                                       // this wave's part of stage t has landed
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // every wave's; nobody reads stage t - 1 any more
    issue(t + NST - 1);
    const char* st = smem + ((t - t0) % NST) * kStage;
#pragma unroll
    for (int h = 0; h < CW / 4; ++h) {  // 128 k
      u32x4 w[RT];
      float s[RT];
      const int c = 4 * h + g;  // this lane's block
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int from = wn + WN * (i / TPW), at = (i % TPW * 16 + r) * CW + c;  // the wave that loaded it, and where
        w[i] = *reinterpret_cast<const u32x4*>(st + kX + (RT * wn + i) * (16 * BK / 2) + r * (BK / 2) +
                                               ((c ^ wswz(r)) << 4));
        const char* sp = st + kX + kW + from * kS;
        s[i] = mx_scale(ALIGNED ? *reinterpret_cast<const uint8_t*>(sp + at) : *reinterpret_cast<const uint32_t*>(sp + 4 * at));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bf16x8 x[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int m = 16 * (MT * wm + j) + r;
          x[j] = *reinterpret_cast<const bf16x8*>(st + m * (BK * 2) + (((4 * c + e) ^ r) << 4));
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const bf16x8 a = mx_bf16x8(w[i][e], s[i]);
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[i][j] = mfma16x16x32(a, x[j], acc[i][j]);
        }
      }
    }
  }
  vm_wait<0>();  // the ring's last loads (zeros) have landed, and every wave has read its last stage
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  // The sums through LDS, so that a wave stores runs of a row.
  constexpr int LD = BN + 4;
  static_assert(BM * LD * 4 <= NST * kStage, "the tile's sums");
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      *reinterpret_cast<floatx4*>(sums + (16 * (MT * wm + j) + r) * LD + 16 * (RT * wn + i) + 4 * g) = acc[i][j];
  __syncthreads();
  float* part = p.part ? p.part + (int64_t)blockIdx.y * p.M * p.N : nullptr;
  if (p.vec) {
    for (int at = threadIdx.x; at < BM * BN / 4; at += 64 * NW) {
      const int m = m0 + at / (BN / 4), n = n0 + at % (BN / 4) * 4;
      if (m >= p.M || n >= p.N) continue;
      const floatx4 v = *reinterpret_cast<const floatx4*>(sums + (m - m0) * LD + n - n0);
      if (part) *reinterpret_cast<floatx4*>(part + (int64_t)m * p.N + n) = v;
      else store_y4(p, m, n, v);
    }
  } else {
    for (int at = threadIdx.x; at < BM * BN; at += 64 * NW) {
      const int m = m0 + at / BN, n = n0 + at % BN;
      if (m >= p.M || n >= p.N) continue;
      const float v = sums[(m - m0) * LD + n - n0];
      if (part) part[(int64_t)m * p.N + n] = v;
      else store_y(p, m, n, v);
    }
  }
}

// y from the k ranges' sums, added in their order.
__global__ __launch_bounds__(256) void mx_sum_kernel(const MxGemm p, int parts) {
  const int64_t mn = (int64_t)p.M * p.N, t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p.vec) {
    if (4 * t >= mn) return;
    floatx4 v{};
#pragma unroll 8
    for (int k = 0; k < parts; ++k) v += *reinterpret_cast<const floatx4*>(p.part + k * mn + 4 * t);
    store_y4(p, (int)(4 * t / p.N), (int)(4 * t % p.N), v);
  } else {
    if (t >= mn) return;
    float v = 0.f;
#pragma unroll 8
    for (int k = 0; k < parts; ++k) v += p.part[k * mn + t];
    store_y(p, (int)(t / p.N), (int)(t % p.N), v);
  }
}

// How a product runs: whole weight rows per block and 64 rows of x (kRows, mxfp4_rows.hip), x through LDS in tiles of
// 32, 64 or 128 rows, or the weights expanded to bf16 for the bf16 GEMM.
enum Form { kRows, kTile32, kTile64, kTile128, kExpand };

struct Plan {
  Form form;
  int bn, bm, parts;  // tile, and ranges of k whose sums are added by mx_sum_kernel
};

// Estimates, us. kRows: every block streams all of its rows of x from the L2 (75 KB a us and CU; fewer where x does
// not stay in it and many blocks read) and then its weights (18 KB), and stores: N=4096 K=4096, 64 rows 13 (measured
// 12.3), N=24576 25 (23.2), N=4096 K=12288 31 (29.6); 616 rows, N=393 K=7232 28 (27.8).
double rows_us(int64_t M, int64_t N, int64_t K) {
  const int64_t r = mx_rows_per_block(M, N, false), blocks = q3_cdiv(N, r) * q3_cdiv(M, kMxRowsMax);
  const double x = 2.0 * (double)M * (double)K;
  const double rate = blocks <= 64 || x <= 2e6 ? 75e3 : x <= 16e6 ? 45e3 : 30e3;
  return 1.5 + (double)q3_cdiv(blocks, 256) *
                   (2 + 0.03 * (double)r + (double)K * ((M <= 32 ? 64 : 128) / rate + 0.53 * (double)r / 18e3));
}
// Tiles: a fixed part (more where N is no multiple of four: single stores), each stage of k, and the sum over ranges:
// 32 rows, N=4096 K=12288 14 (12.8); 64 rows, N=12288 K=4096 18 (18.5); 512 rows, N=12288 K=4096 67 (67).
double tile_us(const Plan& g, int64_t M, int64_t N, int64_t K) {
  const int64_t blocks = q3_cdiv(N, g.bn) * q3_cdiv(M, g.bm) * g.parts;
  const bool big = g.form == kTile128;
  const double stage = big ? (blocks > 128 ? 1.85 : 1.4) : g.form == kTile64 ? 2.3 : 0.8;
  return (big ? 8 : 5) + (N % 4 == 0 ? 0 : big ? 10 : 3) + (g.parts > 1 ? 4 : 0) +
         (double)q3_cdiv(blocks, 256) * (double)q3_cdiv(q3_cdiv(K, big ? 128 : 256), g.parts) * stage;
}
// The expansion moves 2.53 bytes a weight at 5.5 TB/s, the product runs at 1.3 PFLOP/s.
double expand_us(int64_t M, int64_t N, int64_t K) {
  const double nk = (double)N * (double)K;
  return 16 + nk * 2.53 / 5.5e6 + 2 * (double)M * nk / 1.3e9;
}

// kRows up to 16 rows, where x is little. Above, the least estimate; the expansion only from 65 rows and one round of
// tiles on. Measured (us), rows / tiles / expanded: 32 rows, N=4096 K=4096 8.4 / 9.6 / -, K=12288 17.4 / 12.8 / -,
// N=12288 K=4096 11.2 / 14.1 / -; 64 rows, N=1024 K=4096 11.5 / 10.0 / -, N=4096 12.3 / 14.5 / -, N=12288 16.0 / 18.5 / -;
// 136 rows, N=1114 K=416 6.5 / 31.5 / 22; 616, N=393 K=7232 27.8 / 26.6 / 59; 3018, N=78 K=512 6.3 / 21.7 / 13.8; 3102,
// N=667 K=9024 108 / 65 / 82; 469, N=9936 K=224 30 / 19 / 23; N=12288 K=4096, 256 rows - / 45 / 77, 512 - / 67 / 98, 777 - / 126 / 115.
// (kernels/mxfp4.py, _expands, tells from the tiles and the workspace whether a product expands.)
Plan plan_of(int64_t M, int64_t N, int64_t K) {
  const Plan rows{kRows, 0, 0, 1};
  if (M <= 16) return rows;
  Plan g = M <= 32 ? Plan{kTile32, 128, 32, 1} : M <= 64 ? Plan{kTile64, 256, 64, 1} : Plan{kTile128, 256, 128, 1};
  const int64_t tiles = q3_cdiv(N, g.bn) * q3_cdiv(M, g.bm);
  g.parts = (int)std::max<int64_t>(1, std::min<int64_t>(256 / tiles, q3_cdiv(K, 256) / 2));
  double us = tile_us(g, M, N, K);
  if (M > 64 && tiles > 256 && expand_us(M, N, K) < us) {
    g = {kExpand, 0, 0, 1};
    us = expand_us(M, N, K);
  }
  return q3_cdiv(M, kMxRowsMax) <= 65535 && rows_us(M, N, K) < us ? rows : g;
}

template <int RT, int BM, int WM, int BK, int NST>
void launch_tile(const MxGemm& p, const Plan& g, hipStream_t st) {
  const dim3 grid((unsigned)(q3_cdiv(p.N, g.bn) * q3_cdiv(p.M, g.bm)), (unsigned)g.parts);
  if (p.K % 128 == 0 && p.lds % 4 == 0 && q3_aligned(p.s, 4))  // whole words of scales
    hipLaunchKernelGGL((mx_tile_kernel<RT, BM, WM, BK, NST, true>), grid, dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((mx_tile_kernel<RT, BM, WM, BK, NST, false>), grid, dim3(512), 0, st, p);
}

}  // namespace

extern "C" {

int64_t q3_matmul_mxfp4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan g = plan_of(M, N, K);
  if (g.form == kExpand) return N * K * 2;  // the weights in bf16
  return g.parts > 1 ? g.parts * M * N * (int64_t)sizeof(float) : 0;
}

int q3_matmul_mxfp4(const void* x, const void* w_codes, const void* w_scales, const void* bias, const void* residual,
                    void* y, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t lds, int64_t ldr,
                    int64_t ldc, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  Q3_REQUIRE(x && w_codes && w_scales && y, Q3_ERR_NULL);
  Q3_REQUIRE(M >= 0 && N >= 0 && K >= kMxBlock && K % kMxBlock == 0, Q3_ERR_SHAPE);
  Q3_REQUIRE(M < (1ll << 31) && N < (1ll << 31) - 256, Q3_ERR_SHAPE);
  // The rows of a tile are addressed with 32-bit offsets.
  Q3_REQUIRE(ldw < (1ll << 22) && lds < (1ll << 22) && ldx < (1ll << 22), Q3_ERR_UNSUPPORTED);
  Q3_REQUIRE(ldx >= K && ldw >= K / 2 && lds >= K / kMxBlock && ldc >= N && (!residual || ldr >= N), Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16, Q3_ERR_DTYPE);
  if (M == 0 || N == 0) return Q3_OK;
  Q3_REQUIRE(q3_aligned(x, 16) && q3_aligned(w_codes, 16) && ldx % 8 == 0 && ldw % 16 == 0, Q3_ERR_ALIGN);
  const int64_t need = q3_matmul_mxfp4_workspace_bytes(M, N, K);
  Q3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Q3_ERR_WORKSPACE);
  Q3_REQUIRE(need == 0 || q3_aligned(workspace, 16), Q3_ERR_ALIGN);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Plan g = plan_of(M, N, K);
  if (g.form == kRows) {
    MxRows p{};
    p.x = static_cast<const bf16*>(x);
    p.w[0] = static_cast<const uint8_t*>(w_codes);
    p.s[0] = static_cast<const uint8_t*>(w_scales);
    p.bias[0] = static_cast<const bf16*>(bias);
    p.n[0] = (int)N;
    p.nseg = 1;
    p.res = static_cast<const bf16*>(residual);
    p.y = static_cast<bf16*>(y);
    p.M = (int)M, p.K = (int)K;
    p.ldx = ldx, p.ldw = ldw, p.lds = lds, p.ldr = ldr, p.ldc = ldc;
    return mx_rows(p, false, st);
  }
  if (g.form == kExpand) {
    Q3_REQUIRE(ldw == K / 2 && lds == K / kMxBlock, Q3_ERR_UNSUPPORTED);
    const int rc = mx_expand(w_codes, w_scales, static_cast<bf16*>(workspace), N * K, st);
    if (rc != Q3_OK) return rc;
    return q3_matmul(x, workspace, bias, residual, y, M, N, K, ldx, K, ldr, ldc, dtype, nullptr, 0, stream);
  }
  MxGemm p{static_cast<const bf16*>(x), static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales),
           static_cast<const bf16*>(bias), static_cast<const bf16*>(residual), static_cast<bf16*>(y),
           g.parts > 1 ? static_cast<float*>(workspace) : nullptr, (int)M, (int)N, (int)K, ldx, ldw, lds, ldr, ldc, 0};
  p.vec = N % 4 == 0 && q3_aligned(y, 8) && ldc % 4 == 0 && (!bias || q3_aligned(bias, 8)) &&
          (!residual || (q3_aligned(residual, 8) && ldr % 4 == 0));
  if (g.form == kTile32)
    launch_tile<1, 32, 1, 256, 2>(p, g, st);
  else if (g.form == kTile64)
    launch_tile<2, 64, 1, 256, 2>(p, g, st);
  else
    launch_tile<4, 128, 2, 128, 3>(p, g, st);
  Q3_LAUNCH_CHECK();
  if (g.parts > 1) {
    hipLaunchKernelGGL(mx_sum_kernel, dim3((unsigned)q3_cdiv(p.vec ? M * N / 4 : M * N, 256)), dim3(256), 0, st, p,
                       g.parts);
    Q3_LAUNCH_CHECK();
  }
  return Q3_OK;
}

}  // extern "C"

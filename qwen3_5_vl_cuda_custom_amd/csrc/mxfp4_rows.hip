// Products by whole weight rows, 64 rows of x at a time (decode steps, and small weights)
// with MXFP4 weights (format: mxfp4.h): one
// launch for a single weight, for the weights of several projections side by side, or
// for SwiGLU's gate and up, with the RMSNorm of the rows fused in if asked for.
//   y = x w^T (+ bias) (+ residual),  y = silu(x g^T) * (x u^T),  x or norm(x)
// bf16 rows and outputs, fp32 sums, one rounding.
//
// Bound by the stream of weights. Every CU owns whole weight rows (all of k), so no
// sums pass between blocks; codes, scales and x go global -> LDS past the registers in
// stages of 512 k, a ring of up to six stages per block keeps the loads in flight, one
// barrier per stage. A wave takes a quarter of a stage: lane (i = l % 16, g = l /
// 16) reads the 16 bytes of block g of that quarter of weight row i and its scale, and
// the 32 values of x's row i at the same k, and forms four products of 16x16x32 (k
// permuted alike in both). The 4 waves' sums meet in LDS, in wave order. Past 32 rows a
// stage is 256 k, and two waves take a half of it each for one half of the rows.
// The norm: x becomes bf16(x * norm weight) on its way into the product, each lane keeps
// the sum of x^2 over the k it sees, and the sums are scaled by rsqrt(sum / K + eps).
//
// Measured (us; an empty kernel takes 2): one row, N=K=4096 5.1, N=12288 K=4096 7.6 (3.5
// TB/s), N=24576 12.8 (4.2 TB/s), N=4096 K=12288 9.7, N=151936 K=4096 54 (6.1 TB/s); 32
// rows, where each CU also reads all of x from the L2, 8.4, 11.2, 16.5, 17.4 and 97; 64
// rows 12.3, 16.0, 23.2, 29.6 and 143.
#include <algorithm>

#include "gemm_tile.h"
#include "mxfp4.h"
#include "mxfp4_rows.h"

namespace {

using namespace q3;

constexpr int kWaves = 4;
constexpr int kMaxGroups = 6;       // 16-row groups of a block (gate and up: 4 of each)
constexpr int kNormMaxK = 8192;     // the norm weight is held in LDS
// Every block normalises all rows, which costs as much as a launch of its own for 32 (gate and up, N=12288 K=4096: 16.5 us
// without, 20 with; 64 rows 23 and 31).
constexpr int kNormMaxRows = 32;

// RG: 16-row groups of weights, XR: rows of x in LDS. AL: the rows of scales start at multiples of four bytes and are
// whole words (K a multiple of 128), so a lane loads four scales; else one, into a word of its own.
template <int RG, int XR, bool SW, bool NORM, bool AL>
struct RowsShape {
  static constexpr int KS = XR <= 32 ? 512 : 256;                    // k of a stage
  static constexpr int WK = KS / 128, WM = kWaves / WK;              // waves along k, and along the tiles of x
  static constexpr int RGT = SW ? 2 * RG : RG;
  static constexpr int MT = XR > 16 ? XR / 16 : 1, MW = MT / WM;     // 16-row tiles of x, and those of a wave
  static constexpr int CW = KS / 32, CX = KS / 8;                    // 16-byte chunks of a row's codes, of a row of x
  // Loads per wave and stage: codes (GW per group), scales, x.
  static constexpr int GW = 16 * CW / 64, PW = (RGT * GW + 3) / 4;
  static constexpr int GS = AL ? 1 : GW, PS = (RGT * GS + 3) / 4, PX = XR * CX / 64 / kWaves;
  static constexpr int PER = PW + PS + PX;
  static constexpr int kW = PW * 4096, kS = PS * 1024, kX = XR * KS * 2, kSlot = kW + kS + kX;  // bytes
  static constexpr int kNorm = NORM ? kNormMaxK * 2 : 0;
  // Stages of the ring. Where x takes little of the LDS, up to six, but no more than lets two blocks run on a CU, the
  // next one's first loads under the last one's sums (one row, us, 4 stages / 6 / 8, half the LDS: N=4096 K=12288 10.5 /
  // 9.3 / 9.4, N=6144 K=4096 6.3 / 6.0 / 6.0; N=12288 9.2 with 8 in the whole LDS, 7.4 in half, N=151936 75 / 62).
  // Else up to four (16 rows, N=12288: 9.2 with 4, 10.4 in half the LDS). Three at least where x is small (N=24576, 13.9
  // with 2).
  static constexpr int kLds = (XR < 16 ? 78 : 156) * 1024 - kNorm;
  static constexpr int NS = std::max(XR < 16 ? 3 : 2, std::min(XR < 16 ? 6 : 4, kLds / kSlot));
  static_assert(NS * kSlot + kNorm <= 156 * 1024 && (NS - 2) * PER < 64, "the ring, and the count of its loads");
  static_assert(XR * CX % (64 * kWaves) == 0 && MT % WM == 0, "whole loads and tiles per wave");
  static_assert(WK * RGT * MT * 1024 <= NS * kSlot, "the waves' sums");
};

template <int RG, int XR, bool SW, bool NORM, bool AL>
__global__ __launch_bounds__(64 * kWaves) void mx_rows_kernel(const MxRows p) {
  typedef RowsShape<RG, XR, SW, NORM, AL> S;
  constexpr int RGT = S::RGT, MT = S::MT, MW = S::MW, NS = S::NS, KS = S::KS, CW = S::CW, CX = S::CX, WK = S::WK;
  __shared__ __attribute__((aligned(1024))) char smem[NS * S::kSlot + S::kNorm];
  __shared__ float s_sq[NORM ? WK * 16 * MT : 1];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, wk = wave % WK, wm = wave / WK;
  int seg = 0;
#pragma unroll
  for (int j = 1; j < kMxRowsSegments; ++j)
    if (j < p.nseg && (int)blockIdx.x >= p.bstart[j]) seg = j;
  seg = __builtin_amdgcn_readfirstlane(seg);
  const int n0 = ((int)blockIdx.x - p.bstart[seg]) * p.r, rows = min(p.r, p.n[seg] - n0);
  const int blocks = p.K / kMxBlock, steps = (p.K + KS - 1) / KS;
  const uint32_t lbase = lds_addr(smem);

  const int64_t wbytes = (int64_t)(rows - 1) * p.ldw + p.K / 2, sbytes = (int64_t)(rows - 1) * p.lds + blocks;
  const int m0 = blockIdx.y * XR, M = min(p.M - m0, XR);  // this block's rows of x
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + m0 * p.ldx, ((int64_t)(M - 1) * p.ldx + p.K) * 2);

  // This wave's loads, as byte offsets at k = 0, and their k. Row r of 16 keeps its 16-byte chunk c at slot c ^ wswz(r)
  // (x: c ^ (r & 15)), so the 16 rows of a fragment read use all banks.
  auto wswz = [](int r) { return r / (16 / CW) & (CW - 1); };
  // Codes: load d of the stage is part d % GW of group d / GW.
  uint32_t woff[S::PW];
  int wc[S::PW];
  __amdgpu_buffer_rsrc_t rw[S::PW];
#pragma unroll
  for (int u = 0; u < S::PW; ++u) {
    const int d = 4 * u + wave, q = d / S::GW, r = d % S::GW * (64 / CW) + lane / CW;
    const int row = 16 * (q < RG ? q : q - RG) + r;
    wc[u] = lane % CW ^ wswz(r);
    woff[u] = q < RGT && row < rows ? (uint32_t)(row * p.ldw + 16 * wc[u]) : kOOB;
    rw[u] = make_rsrc((SW && q >= RG ? p.w[1] : p.w[seg]) + (int64_t)n0 * p.ldw, wbytes);
  }
  // Scales: load d is the 16 rows of group d, a word (four blocks) per lane; or, one block per lane, part d % GS of
  // group d / GS.
  uint32_t soff[S::PS];
  const int sb = AL ? 4 * (lane % (CW / 4)) : lane % CW;
  __amdgpu_buffer_rsrc_t rs[S::PS];
#pragma unroll
  for (int v = 0; v < S::PS; ++v) {
    const int d = 4 * v + wave, q = d / S::GS, r = AL ? lane / (CW / 4) : d % S::GS * (64 / CW) + lane / CW;
    const int row = 16 * (q < RG ? q : q - RG) + r;
    soff[v] = q < RGT && r < 16 && row < rows ? (uint32_t)(row * p.lds + sb) : kOOB;
    rs[v] = make_rsrc((SW && q >= RG ? p.s[1] : p.s[seg]) + (int64_t)n0 * p.lds, sbytes);
  }
  uint32_t xoff[S::PX];
  int xc[S::PX];
#pragma unroll
  for (int u = 0; u < S::PX; ++u) {
    const int m = (4 * u + wave) * (64 / CX) + lane / CX;
    xc[u] = lane % CX ^ (m & 15);
    xoff[u] = m < M ? (uint32_t)(m * p.ldx * 2 + 16 * xc[u]) : kOOB;
  }
  auto issue = [&](int t, int slot) {
    const uint32_t at = lbase + (uint32_t)slot;
    const int left = blocks - CW * t;  // blocks from this stage's first on (none past the last stage)
#pragma unroll
    for (int u = 0; u < S::PX; ++u)
      dma16(rx, xoff[u] != kOOB && xc[u] < 4 * left ? xoff[u] + (uint32_t)t * (KS * 2) : kOOB,
            at + S::kW + S::kS + (4 * u + wave) * 1024);
#pragma unroll
    for (int v = 0; v < S::PS; ++v)
      if constexpr (AL)
        dma4(rs[v], soff[v] != kOOB && sb < left ? soff[v] + (uint32_t)t * (KS / 32) : kOOB,
             at + S::kW + (4 * v + wave) * 256);
      else
        dma1(rs[v], soff[v] != kOOB && sb < left ? soff[v] + (uint32_t)t * (KS / 32) : kOOB,
             at + S::kW + (4 * v + wave) * 256);
#pragma unroll
    for (int u = 0; u < S::PW; ++u)
      dma16_nt(rw[u], woff[u] != kOOB && wc[u] < left ? woff[u] + (uint32_t)t * (KS / 2) : kOOB,
               at + (4 * u + wave) * 1024);
  };
  if constexpr (NORM) {  // before the first stage: its wait covers these
    const __amdgpu_buffer_rsrc_t rn = make_rsrc(p.nw, (int64_t)p.K * 2);
    for (int d = wave; d < (p.K + 511) / 512; d += kWaves)
      dma16(rn, (uint32_t)(d * 1024 + 16 * lane), lbase + (uint32_t)(NS * S::kSlot + d * 1024));
  }

  floatx4 acc[RGT][MW];
#pragma unroll
  for (int q = 0; q < RGT; ++q)
#pragma unroll
    for (int t = 0; t < MW; ++t) acc[q][t] = floatx4{};
  float sq[MW];
#pragma unroll
  for (int t = 0; t < MW; ++t) sq[t] = 0.f;

#pragma unroll 1
  for (int t = 0; t < NS - 1; ++t) issue(t, t * S::kSlot);
  int cur = 0, next = (NS - 1) * S::kSlot;  // slots of stage t and of stage t + NS - 1
  for (int t = 0; t < steps; ++t) {
    vm_wait<(NS - 2) * S::PER>();                                     // this wave's part of stage t has landed
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // every wave's; nobody reads stage t - 1 any more
    issue(t + NS - 1, next);
    const char* st = smem + cur;
    next = cur;
    cur = cur == (NS - 1) * S::kSlot ? 0 : cur + S::kSlot;
    u32x4 w[RGT];
    float s[RGT];
#pragma unroll
    for (int q = 0; q < RGT; ++q) {
      w[q] = *reinterpret_cast<const u32x4*>(st + (16 * q + i) * (KS / 2) + (((4 * wk + g) ^ wswz(i)) << 4));
      const int at = i * CW + 4 * wk + g;
      s[q] = mx_scale(AL ? *reinterpret_cast<const uint8_t*>(st + S::kW + q * 256 + at)
                         : *reinterpret_cast<const uint32_t*>(st + S::kW + (q * 16 * CW + at) * 4));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bf16x8 x[MW];
#pragma unroll
      for (int j = 0; j < MW; ++j) {
        const int m = 16 * (MW * wm + j) + (XR < 16 ? i % XR : i);  // fewer rows: repeated, the copies' sums are not used
        x[j] = *reinterpret_cast<const bf16x8*>(st + S::kW + S::kS + m * (KS * 2) +
                                                (((16 * wk + 4 * g + e) ^ (m & 15)) << 4));
      }
      if constexpr (NORM) {
        const bf16x8 nw = *reinterpret_cast<const bf16x8*>(smem + NS * S::kSlot + 2 * (t * KS + 128 * wk + 32 * g + 8 * e));
#pragma unroll
        for (int j = 0; j < MW; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float f = bf2f(x[j][k]);
            sq[j] += f * f;
            x[j][k] = f2bf(f * bf2f(nw[k]));
          }
      }
#pragma unroll
      for (int q = 0; q < RGT; ++q) {
        const bf16x8 a = mx_bf16x8(w[q][e], s[q]);
#pragma unroll
        for (int j = 0; j < MW; ++j) acc[q][j] = mfma16x16x32(a, x[j], acc[q][j]);
      }
    }
  }
  vm_wait<0>();  // the ring's last loads (zeros) have landed, and every wave has read its last stage
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  floatx4* sums = reinterpret_cast<floatx4*>(smem);
#pragma unroll
  for (int q = 0; q < RGT; ++q)
#pragma unroll
    for (int j = 0; j < MW; ++j) sums[((wk * RGT + q) * MT + MW * wm + j) * 64 + lane] = acc[q][j];
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < MW; ++j) {
      float v = sq[j];
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      if (g == 0) s_sq[(wk * MT + MW * wm + j) * 16 + i] = v;
    }
  }
  __syncthreads();
  // Element e of lane l in (group q, tile j) is weight row 16 q + 4 (l / 16) + e, row 16 j + l % 16 of x.
  for (int it = tid; it < RG * MT * 64; it += 64 * kWaves) {
    const int l = it & 63, j = it / 64 % MT, q = it / (64 * MT);
    const int m = 16 * j + (l & 15), row = 16 * q + 4 * (l >> 4);
    if (m >= M || row >= rows) continue;
    auto total = [&](int group) {
      floatx4 v = sums[(group * MT + j) * 64 + l];
#pragma unroll
      for (int k = 1; k < WK; ++k) v += sums[((k * RGT + group) * MT + j) * 64 + l];
      return v;
    };
    floatx4 v = total(q);
    float norm = 1.f;
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) sum += s_sq[k * MT * 16 + m];
      norm = rsqrtf(sum / (float)p.K + p.eps);
      v *= norm;
    }
    if constexpr (SW) {
      floatx4 u = total(RG + q);
      if constexpr (NORM) u *= norm;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = silu_mul(v[e], u[e]);
    }
    const int col = p.col[seg] + n0 + row;
    const bf16* bias = p.bias[seg] ? p.bias[seg] + n0 + row : nullptr;
    const bf16* res = p.res ? p.res + (int64_t)(m0 + m) * p.ldr + col : nullptr;
    bf16* y = p.y + (int64_t)(m0 + m) * p.ldc + col;
    if (p.vec && row + 3 < rows) {  // 8-byte pieces: n0, the columns and the strides are multiples of four
      if (bias) {
        const bf16x4 b = *reinterpret_cast<const bf16x4*>(bias);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += bf2f(b[e]);
      }
      if (res) {
        const bf16x4 b = *reinterpret_cast<const bf16x4*>(res);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += bf2f(b[e]);
      }
      *reinterpret_cast<bf16x4*>(y) = bf16x4{f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (row + e >= rows) break;
        float o = v[e];
        if (bias) o += bf2f(bias[e]);
        if (res) o += bf2f(res[e]);
        y[e] = f2bf(o);
      }
    }
  }
}

template <int RG, int XR, bool SW>
void launch_form(const MxRows& p, dim3 grid, bool words, hipStream_t st) {
  const dim3 block(64 * kWaves);
  if constexpr (!SW)
    if (!words) {  // a single weight without the norm
      hipLaunchKernelGGL((mx_rows_kernel<RG, XR, false, false, false>), grid, block, 0, st, p);
      return;
    }
  if constexpr (XR <= kNormMaxRows)
    if (p.nw) {
      hipLaunchKernelGGL((mx_rows_kernel<RG, XR, SW, true, true>), grid, block, 0, st, p);
      return;
    }
  hipLaunchKernelGGL((mx_rows_kernel<RG, XR, SW, false, true>), grid, block, 0, st, p);
}
template <int XR, bool SW>
void launch_groups(const MxRows& p, int blocks, bool words, hipStream_t st) {
  const dim3 grid((unsigned)blocks, (unsigned)q3_cdiv(p.M, XR));
  switch ((p.r + 15) / 16) {
    case 1: launch_form<1, XR, SW>(p, grid, words, st); break;
    case 2: launch_form<2, XR, SW>(p, grid, words, st); break;
    case 3: launch_form<3, XR, SW>(p, grid, words, st); break;
    case 4: launch_form<4, XR, SW>(p, grid, words, st); break;
    default:
      if constexpr (!SW) launch_form<6, XR, SW>(p, grid, words, st);
  }
}
template <bool SW>
void launch_rows(const MxRows& p, int blocks, bool words, hipStream_t st) {
  if (p.M <= 4) launch_groups<4, SW>(p, blocks, words, st);
  else if (p.M <= 16) launch_groups<16, SW>(p, blocks, words, st);
  else if (p.M <= 32) launch_groups<32, SW>(p, blocks, words, st);
  else launch_groups<64, SW>(p, blocks, words, st);
}

// Whether the scales are whole words.
bool words_of(const MxRows& p) {
  bool ok = p.K % 128 == 0 && p.lds % 4 == 0;
  for (int j = 0; j < p.nseg; ++j) ok = ok && q3_aligned(p.s[j], 4);
  return ok;
}

}  // namespace

namespace q3 {

int64_t mx_rows_per_block(int64_t M, int64_t N, bool swiglu) {
  const int64_t chunks = q3_cdiv(M, kMxRowsMax);
  int64_t most = 16 * (swiglu ? 4 : kMaxGroups);
  if (M <= 4 && N > 256 * most) most = 64;  // then two blocks fit a CU: N=151936 K=4096 62 -> 54 us
  const int64_t rounds = q3_cdiv(N * chunks, 256 * most);
  int64_t r = 4;
  while (r < most && q3_cdiv(N, r) * chunks > 256 * rounds) r += 4;
  return r;
}

int mx_rows(MxRows p, bool swiglu, hipStream_t st) {
  int64_t total = 0;
  for (int j = 0; j < p.nseg; ++j) {
    p.col[j] = (int)total;
    total += p.n[j];
  }
  // The fewest rows per block (whole 8-byte pieces of y) that give every CU one block, or an equal number of them
  // where even the largest block does not cover N.
  int r = (int)mx_rows_per_block(p.M, total, swiglu);
  auto blocks = [&](int rows) {
    int64_t n = 0;
    for (int j = 0; j < p.nseg; ++j) n += q3_cdiv(p.n[j], rows);
    return n;
  };
  const int64_t rounds = q3_cdiv(q3_cdiv(total, r), 256);
  while (p.nseg > 1 && r < 64 && blocks(r) > 256 * rounds) r += 4;
  p.r = r;
  int64_t grid = 0;
  for (int j = 0; j < p.nseg; ++j) {
    p.bstart[j] = (int)grid;
    grid += q3_cdiv(p.n[j], r);
  }
  p.vec = q3_aligned(p.y, 8) && p.ldc % 4 == 0 && (!p.res || (q3_aligned(p.res, 8) && p.ldr % 4 == 0));
  for (int j = 0; j < p.nseg; ++j) p.vec = p.vec && p.col[j] % 4 == 0 && (!p.bias[j] || q3_aligned(p.bias[j], 8));
  if (swiglu)
    launch_rows<true>(p, (int)grid, true, st);
  else
    launch_rows<false>(p, (int)grid, words_of(p), st);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // namespace q3

namespace {

// Arguments of the two entry points but the weights.
int check_rows(const void* x, const void* norm_weight, const void* y, int64_t M, int64_t K, int64_t N, int64_t ldx,
               int64_t ldc, int dtype) {
  Q3_REQUIRE(x && y, Q3_ERR_NULL);
  Q3_REQUIRE(M >= 0 && K >= kMxBlock && K % kMxBlock == 0 && N >= 0 && ldx >= K && ldc >= N, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16, Q3_ERR_DTYPE);
  Q3_REQUIRE(M <= kMxRowsMax && K % 128 == 0 && K < (1 << 23) && ldx < (1 << 22) && N < (1ll << 31) - 256 &&
                 (!norm_weight || (K <= kNormMaxK && M <= kNormMaxRows)),
             Q3_ERR_UNSUPPORTED);
  return q3_aligned(x, 16) && ldx % 8 == 0 && q3_aligned(norm_weight, 16) ? Q3_OK : Q3_ERR_ALIGN;
}

bool weight_ok(const void* codes, const void* scales) { return q3_aligned(codes, 16) && q3_aligned(scales, 4); }

MxRows rows_of(const void* x, const void* norm_weight, float eps, void* y, int64_t M, int64_t K, int64_t ldx, int64_t ldc) {
  MxRows p{};
  p.x = static_cast<const bf16*>(x);
  p.nw = static_cast<const bf16*>(norm_weight);
  p.eps = eps;
  p.y = static_cast<bf16*>(y);
  p.M = (int)M;
  p.K = (int)K;
  p.ldx = ldx;
  p.ldw = K / 2;
  p.lds = K / kMxBlock;
  p.ldc = ldc;
  return p;
}

}  // namespace

extern "C" {

int q3_matmul_segments_mxfp4(const void* x, const void* norm_weight, float eps, const void* const* codes,
                             const void* const* scales, const void* const* bias, const int64_t* n, int64_t nseg,
                             void* y, int64_t M, int64_t K, int64_t ldx, int64_t ldc, int dtype, void* stream) {
  Q3_REQUIRE(codes && scales && n, Q3_ERR_NULL);
  Q3_REQUIRE(nseg >= 1 && nseg <= kMxRowsSegments, Q3_ERR_SHAPE);
  int64_t total = 0;
  for (int j = 0; j < nseg; ++j) {
    Q3_REQUIRE(codes[j] && scales[j], Q3_ERR_NULL);
    Q3_REQUIRE(n[j] >= 1 && n[j] < (1ll << 31), Q3_ERR_SHAPE);
    total += n[j];
  }
  const int rc = check_rows(x, norm_weight, y, M, K, total, ldx, ldc, dtype);
  if (rc != Q3_OK || M == 0) return rc;
  MxRows p = rows_of(x, norm_weight, eps, y, M, K, ldx, ldc);
  p.nseg = (int)nseg;
  for (int j = 0; j < nseg; ++j) {
    Q3_REQUIRE(weight_ok(codes[j], scales[j]), Q3_ERR_ALIGN);
    p.w[j] = static_cast<const uint8_t*>(codes[j]);
    p.s[j] = static_cast<const uint8_t*>(scales[j]);
    p.bias[j] = bias ? static_cast<const bf16*>(bias[j]) : nullptr;
    p.n[j] = (int)n[j];
  }
  return mx_rows(p, false, static_cast<hipStream_t>(stream));
}

int q3_matmul_swiglu_mxfp4(const void* x, const void* norm_weight, float eps, const void* g_codes, const void* g_scales,
                           const void* u_codes, const void* u_scales, void* y, int64_t M, int64_t N, int64_t K,
                           int64_t ldx, int64_t ldc, int dtype, void* stream) {
  Q3_REQUIRE(g_codes && g_scales && u_codes && u_scales, Q3_ERR_NULL);
  const int rc = check_rows(x, norm_weight, y, M, K, N, ldx, ldc, dtype);
  if (rc != Q3_OK || M == 0 || N == 0) return rc;
  Q3_REQUIRE(weight_ok(g_codes, g_scales) && weight_ok(u_codes, u_scales), Q3_ERR_ALIGN);
  MxRows p = rows_of(x, norm_weight, eps, y, M, K, ldx, ldc);
  p.nseg = 1;
  p.n[0] = (int)N;
  p.w[0] = static_cast<const uint8_t*>(g_codes);
  p.s[0] = static_cast<const uint8_t*>(g_scales);
  p.w[1] = static_cast<const uint8_t*>(u_codes);
  p.s[1] = static_cast<const uint8_t*>(u_scales);
  return mx_rows(p, true, static_cast<hipStream_t>(stream));
}

}  // extern "C"

// Products of many MXFP8 rows: tiles of BM rows of x and BN weight rows through LDS
// (format and matrix instruction: mxfp8.h).
//
// Codes go global -> LDS past the registers (buffer loads with the lds flag), a stage of
// 128 k (one matrix instruction's) at a time, 128 bytes a row; scales, a word a row and
// stage, the same way. Row r keeps its 16-byte chunk c at slot c ^ (r & 7) ^ (r >> 3 & 1),
// so the 16 rows of a fragment read use all banks. A wave holds the stage's TN weight
// fragments and takes the TM fragments of x (columns, below) one after the other, each
// read three columns ahead, TN products to a column. Before the last two columns every
// fragment of the stage has been read: there the stage barrier stands, the next stage's
// fragments are read between the products after it, each weight fragment once its last
// product has issued.
//
// With two slots (256 x 256 tiles fill the LDS) a stage's weight slot is free once every
// wave has the fragments, after the first column: a second barrier there lets the weights
// after next, which come from further away than x, set out most of a stage earlier.
#include <algorithm>

#include "gemm_tile.h"
#include "mxfp8.h"
#include "mxfp8_tile.h"

namespace {

using namespace q3;

struct TileArgs {
  Mx8Args a;
  int64_t slx, slw;  // bytes between rows of scales: whole words
  int N;             // columns of y
  int tiles_m, tiles_n;
  int kt;            // stages of a block
  float* part;       // fp32 partial sums (splits, M, N), or null
};

// A uniform pointer or number in scalar registers (a select can leave it in vector ones).
__device__ __forceinline__ int pin(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* pin(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}

// Eight columns of y from n on (of its segment; `left` of them exist), the row's m.
__device__ __forceinline__ void finish8(const Mx8Args& p, int seg, int64_t m, int n, int col, int left, bool vec,
                                        bool plain, float (&v)[8]) {
  if (plain) {
    const bf16* bias = p.bias[seg];
    if (bias) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) v[e] += bf2f(bias[n + e]);
    }
    if (p.act) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = mx8_act(v[e], p.act);
    }
    if (p.res) {
      const bf16* r = p.res + m * p.ldr + col;
      if (vec && left >= 8) {
        const bf16x8 b = *reinterpret_cast<const bf16x8*>(r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bf2f(b[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) v[e] += bf2f(r[e]);
      }
    }
  }
  if (p.yc) {  // whole blocks of 32 columns: the four lanes of one are neighbours
    uint32_t byte;
    const u32x2 c = mx8_quantize8(v, byte);
    *reinterpret_cast<u32x2*>(p.yc + m * p.ldc + col) = c;
    if ((col & 31) == 0) p.ys[m * (p.ldc / kMx8Block) + col / kMx8Block] = (uint8_t)byte;
    return;
  }
  bf16* y = p.y + m * p.ldc + col;
  if (vec && left >= 8) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f2bf(v[e]);
    *reinterpret_cast<bf16x8*>(y) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) y[e] = f2bf(v[e]);
  }
}

// Whether y and the residual go in 16-byte pieces (segment starts: multiples of eight columns).
__device__ __forceinline__ bool vec_of(const Mx8Args& p, int col0) {
  return col0 % 8 == 0 && p.ldc % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 &&
         (!p.res || (p.ldr % 8 == 0 && (reinterpret_cast<uintptr_t>(p.res) & 15) == 0));
}

template <int BM, int BN, int WM, int WN, int NS, bool SW>
__global__ __launch_bounds__(WM* WN * 64) void mx8_tile_kernel(const TileArgs t) {
  constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  constexpr int BN_OUT = SW ? BN / 2 : BN;
  constexpr int PX = BM / 8 / NW, PW = BN / 8 / NW, PS = ((BM + BN) / 64 + NW - 1) / NW;  // loads per wave and stage
  constexpr bool EARLY = NS == 2;  // the weights' slot is released by a barrier of its own
  constexpr int NSS = NS + 2;      // slots of scales
  constexpr int kX = BM * 128, kW = BN * 128, kS = PS * NW * 256, kLds = NS * (kX + kW) + NSS * kS;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NW % 2 == 0, "whole loads per wave, one swizzle per lane");
  static_assert(TM % 4 == 0 && WTN % (SW ? 64 : 16) == 0 && kLds <= 160 * 1024, "wave tiles");
  __shared__ __attribute__((aligned(1024))) char smem[kLds];

  const Mx8Args& p = t.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN, l16 = lane & 15, q4 = lane >> 4;
  const int K = p.K;

  // This block's tile: the tiles of one XCD are neighbours, four of them along m.
  const int pid = xcd_remap(blockIdx.x, t.tiles_m * t.tiles_n);
  const int group = pid / (4 * t.tiles_n), size_m = min(t.tiles_m - 4 * group, 4);
  const int in = pid - group * 4 * t.tiles_n;
  const int m0 = __builtin_amdgcn_readfirstlane((4 * group + in % size_m) * BM);
  int tn = __builtin_amdgcn_readfirstlane(in / size_m), seg = 0, col0 = 0;
#pragma unroll
  for (int j = 0; j + 1 < kMx8Segments; ++j) {
    const int nt = (p.n[j] + BN_OUT - 1) / BN_OUT;
    if (seg == j && j + 1 < p.nseg && tn >= nt) tn -= nt, col0 += p.n[j], seg = j + 1;
  }
  seg = pin(seg), tn = pin(tn), col0 = pin(col0);
  const int n0 = tn * BN_OUT, rows_n = pin(min(BN_OUT, p.n[seg] - n0)), rows_m = pin(min(BM, p.M - m0));
  const int k_first = blockIdx.z * t.kt, nk = min(t.kt, (K + 127) / 128 - k_first);  // stages

  const __amdgpu_buffer_rsrc_t rx = make_rsrc(pin(p.x + (int64_t)m0 * K), rows_m * K);
  const uint8_t* const wa = pin(p.w[SW ? 0 : seg] + (int64_t)n0 * K);  // SwiGLU: gate's, and up's
  const uint8_t* const wb = SW ? pin(p.w[1] + (int64_t)n0 * K) : wa;
  const uint8_t* const sa = pin(p.ws[SW ? 0 : seg] + n0 * t.slw);
  const uint8_t* const sb = SW ? pin(p.ws[1] + n0 * t.slw) : sa;
  auto swz = [](int r) { return (r & 7) ^ ((r >> 3) & 1); };
  // Load i of this wave fills rows 8 (wave + NW i) .. + 7 of the tile.
  const int lrow = lane >> 3, dc = (lane & 7) ^ swz(wave * 8 + lrow);
  uint32_t xoff[PX], woff[PW];
#pragma unroll
  for (int i = 0; i < PX; ++i) xoff[i] = (uint32_t)(((wave + NW * i) * 8 + lrow) * K);
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int r = (wave + NW * i) * 8 + lrow;
    woff[i] = (uint32_t)((SW ? (r >> 6) * 32 + (r & 31) : r) * K);  // SwiGLU: 32 gate rows, the same 32 up rows, ...
  }
  // Scales: load s of this wave is the rows 64 (wave + NW s) .. + 63 of x, then of the weights (SwiGLU: of gate, of up).
  uint32_t soff[PS];
  const uint8_t* sp[PS];
  int sbytes[PS];
#pragma unroll
  for (int s = 0; s < PS; ++s) {
    const int e = (wave + NW * s) * 64;
    const bool of_x = e < BM, up = SW && e - BM >= BN_OUT;
    const int row = (of_x ? e : up ? e - BM - BN_OUT : e - BM) + lane;
    sp[s] = pin(of_x ? p.xs + m0 * t.slx : up ? sb : sa);
    sbytes[s] = pin(of_x ? rows_m * (int)t.slx : rows_n * (int)t.slw);
    soff[s] = e < BM + BN ? (uint32_t)(row * (int)(of_x ? t.slx : t.slw)) : kOOB;
  }
  const uint32_t lbase = lds_addr(smem);
  constexpr int kW0 = NS * kX, kS0 = kW0 + NS * kW;
  // Byte of a row at which the lane's chunk of stage kt lies; past the row's end, and past the block's stages, past
  // every resource too.
  auto kofs = [&](int kt) {
    const int k = (k_first + kt) * 128 + dc * 16;
    return kt < nk && k < K ? (uint32_t)k : kOOB;
  };
  auto dma_x = [&](int kt, int i) {
    dma16(rx, xoff[i] + kofs(kt), lbase + (uint32_t)(kt % NS * kX + (wave + NW * i) * 1024));
  };
  auto dma_w = [&](int kt, int i) {
    const bool up = SW && ((wave + NW * i) & 4);
    dma16(make_rsrc(SW ? pin(up ? wb : wa) : wa, rows_n * K), woff[i] + kofs(kt), lbase + (uint32_t)(kW0 + kt % NS * kW + (wave + NW * i) * 1024));
  };
  auto dma_s = [&](int kt, int s) {
    dma4(make_rsrc(sp[s], sbytes[s]), kt < nk && soff[s] != kOOB ? soff[s] + (uint32_t)(k_first + kt) * 4 : kOOB,
         lbase + (uint32_t)(kS0 + kt % NSS * kS + (wave + NW * s) * 256));
  };
  // d-th load of what is issued in the columns before the stage barrier: scales, weights (and with more slots x)
  constexpr int ND = PS + PW + (EARLY ? 0 : PX);
  auto dma = [&](int kt, int d) {
    if (d < PS) dma_s(kt, d);
    else if (d < PS + PW) dma_w(kt, d - PS);
    else dma_x(kt, d - PS - PW);
  };

  floatx4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = floatx4{};
  i32x8 fw[TN], fx[4];
  int sw[TN], sx[4];
  const int rn = wn * WTN, rm = wm * WTM;
  auto frag = [&](const char* slot, int r) {
    const char* row = slot + r * 128;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(row + ((q4 ^ swz(r)) << 4));
    const i32x4 hi = *reinterpret_cast<const i32x4*>(row + (((4 + q4) ^ swz(r)) << 4));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto rd_w = [&](int kt, int i) {
    const int r = rn + 16 * i + l16, e = SW ? (r >> 5 & 1) * BN_OUT + (r >> 6) * 32 + (r & 31) : r;
    fw[i] = frag(smem + kW0 + kt % NS * kW, r);
    sw[i] = *reinterpret_cast<const uint8_t*>(smem + kS0 + kt % NSS * kS + (BM + e) * 4 + q4);
  };
  auto rd_x = [&](int kt, int j) {
    const int r = rm + 16 * j + l16;
    fx[j & 3] = frag(smem + kt % NS * kX, r);
    sx[j & 3] = *reinterpret_cast<const uint8_t*>(smem + kS0 + kt % NSS * kS + r * 4 + q4);
  };
  auto mf = [&](int i, int j) { acc[i][j] = mfma_mx8(fw[i], fx[j & 3], acc[i][j], sw[i], sx[j & 3]); };

  constexpr int kAhead = EARLY ? 2 : NS - 1;  // stages issued before the loop
#pragma unroll
  for (int s = 0; s < kAhead; ++s) {
#pragma unroll
    for (int d = 0; d < ND; ++d) dma(s, d);
    if constexpr (EARLY) {
#pragma unroll
      for (int i = 0; i < PX; ++i) dma_x(s, i);
    }
  }
  vm_wait<(kAhead - 1) * (PX + PW + PS)>();  // stage 0 has landed
  __syncthreads();

  auto main = [&](auto active_c) {
    constexpr bool A = decltype(active_c)::value;  // a wave without rows loads and waits only
    if constexpr (A) {
#pragma unroll
      for (int i = 0; i < TN; ++i) rd_w(0, i);
#pragma unroll
      for (int j = 0; j < 3; ++j) rd_x(0, j);
    }
    for (int kt = 0; kt < nk; ++kt) {
      const int next = kt + kAhead;  // the stage whose loads go out
      int d = 0;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < TM - 2; ++j) {
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          if constexpr (A) {
            mf(i, j);
            if (i == 0 && j + 3 < TM) rd_x(kt, j + 3);
          }
          constexpr int slots = TN * (TM - 2) - (EARLY ? TN : 0), gap = slots / ND > 0 ? slots / ND : 1;
          const int at = j * TN + i - (EARLY ? TN : 0);
          if (at >= 0 && at % gap == gap - 1 && d < ND) dma(next, d++);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (EARLY && j == 0) asm volatile("s_barrier" ::: "memory");  // every wave holds the weights' fragments
      }
#pragma unroll
      for (; d < ND; ++d) dma(next, d);
      // Stage kt + 1 has landed and every fragment of stage kt is in registers, in every wave.
      vm_wait<EARLY ? PS + PW : (NS - 2) * (PX + PW + PS)>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (A) {
        rd_x(kt + 1, 0);
        rd_x(kt + 1, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          mf(i, TM - 2);
          if (EARLY && i < PX) dma_x(next, i);
          mf(i, TM - 1);
          rd_w(kt + 1, i);
          __builtin_amdgcn_sched_barrier(0);
        }
        rd_x(kt + 1, 2);
      }
      if constexpr (EARLY) {
#pragma unroll
        for (int i = A ? TN : 0; i < PX; ++i) dma_x(next, i);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (rm < rows_m) main(std::true_type{});
  else main(std::false_type{});
  vm_wait<0>();  // the loads past the last stage (zeros) have landed

  // Epilogue: the accumulators through LDS in fp32, up to RP rows at a time, so that a lane then has eight columns of a
  // row. 16-byte chunk c of row r lies at c ^ (r & 15).
  constexpr int RP0 = kLds / (BN_OUT * 4), RP = RP0 >= BM ? BM : RP0 >= 128 ? 128 : RP0 >= 64 ? 64 : 32;
  static_assert(RP0 >= 32 && BN_OUT % 64 == 0, "epilogue");
  constexpr int C8 = BN_OUT / 8;
  float* lds = reinterpret_cast<float*>(smem);
  auto slot = [](int r, int c) { return r * BN_OUT + ((c ^ (r & 15)) << 2); };
  const bool vec = vec_of(p, col0);
#pragma unroll
  for (int r0 = 0; r0 < BM; r0 += RP) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int r = rm + 16 * j - r0;
      if (r < 0 || r >= RP) continue;
#pragma unroll
      for (int o = 0; o < (SW ? TN / 2 : TN); ++o) {
        floatx4 v;
        if constexpr (SW) {
          const int g = 4 * (o / 2) + o % 2;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = silu_mul(acc[g][j][e], acc[g + 2][j][e]);
        } else {
          v = acc[o][j];
        }
        *reinterpret_cast<floatx4*>(lds + slot(r + l16, ((SW ? rn / 2 : rn) + 16 * o) / 4 + q4)) = v;
      }
    }
    __syncthreads();
    const int items = min(RP, rows_m - r0) * C8;
    for (int it = tid; it < items; it += NW * 64) {
      const int r = it / C8, c = it % C8, left = rows_n - 8 * c;
      if (left <= 0) continue;
      const floatx4 a = *reinterpret_cast<const floatx4*>(lds + slot(r, 2 * c));
      const floatx4 b = *reinterpret_cast<const floatx4*>(lds + slot(r, 2 * c + 1));
      float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      const int64_t m = m0 + r0 + r;
      const int n = n0 + 8 * c;
      if (t.part) {
        float* o = t.part + ((int64_t)blockIdx.z * p.M + m) * t.N + col0 + n;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) o[e] = v[e];
      } else {
        finish8(p, seg, m, n, col0 + n, left, vec, !SW, v);
      }
    }
  }
}

// Rows of scales copied to whole words, zeros behind: x's, then each weight's.
struct PadArgs {
  const uint8_t* s[1 + kMx8Segments];
  int64_t rows[1 + kMx8Segments];
  uint8_t* out;
  int kb, ld;
};
__global__ __launch_bounds__(256) void mx8_pad_scales_kernel(const PadArgs a) {
  const int j = blockIdx.y;
  uint8_t* out = a.out;
  const uint8_t* s = a.s[0];
  int64_t rows = a.rows[0];
#pragma unroll
  for (int u = 1; u <= kMx8Segments; ++u)
    if (j >= u) out += rows * a.ld, s = a.s[u], rows = a.rows[u];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * a.ld; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / a.ld;
    const int b = (int)(i - r * a.ld);
    out[i] = b < a.kb ? s[r * a.kb + b] : 0;
  }
}

int tiles_of(const Mx8Args& a, int bn) {
  int64_t n = 0;
  for (int j = 0; j < a.nseg; ++j) n += q3_cdiv(a.n[j], bn);
  return (int)n;
}

template <int BM, int BN, int WM, int WN, int NS, bool SW>
void launch_tile(TileArgs t, int splits, hipStream_t st) {
  t.tiles_m = (int)q3_cdiv(t.a.M, BM);
  t.tiles_n = tiles_of(t.a, SW ? BN / 2 : BN);
  hipLaunchKernelGGL((mx8_tile_kernel<BM, BN, WM, WN, NS, SW>), dim3((unsigned)(t.tiles_m * t.tiles_n), 1, (unsigned)splits),
                     dim3(WM * WN * 64), 0, st, t);
}

template <bool SW>
void launch_form(const TileArgs& t, int form, int splits, hipStream_t st) {
  if (form == 0) launch_tile<256, 256, 2, 4, 2, SW>(t, splits, st);
  else if (form == 1) launch_tile<128, 256, 2, 4, 3, SW>(t, splits, st);
  else launch_tile<128, 128, 2, 2, 2, SW>(t, splits, st);
}

struct Plan {
  int form;
  bool pad;
};
Plan plan_of(const Mx8Args& a, bool swiglu) {
  Plan p;
  p.pad = a.K % 128 != 0;
  const int out = swiglu ? 2 : 1;
  p.form = q3_cdiv(a.M, 256) * tiles_of(a, 256 / out) >= 200 ? 0 : q3_cdiv(a.M, 128) * tiles_of(a, 256 / out) >= 200 ? 1 : 2;
  return p;
}

}  // namespace

namespace q3 {

int64_t mx8_tile_workspace(const Mx8Args& a, bool swiglu) {
  const Plan plan = plan_of(a, swiglu);
  if (!plan.pad) return 0;
  int64_t rows = a.M;
  for (int j = 0; j < (swiglu ? 2 : a.nseg); ++j) rows += a.n[swiglu ? 0 : j];
  return rows * (q3_cdiv(a.K, 128) * 4);
}

int mx8_tile(const Mx8Args& a, int64_t N, bool swiglu, void* workspace, hipStream_t st) {
  const Plan plan = plan_of(a, swiglu);
  TileArgs t{};
  t.a = a;
  t.N = (int)N;
  t.kt = (int)q3_cdiv(a.K, 128);
  t.slx = t.slw = a.K / kMx8Block;
  if (plan.pad) {
    PadArgs p{};
    p.kb = a.K / kMx8Block;
    p.ld = 4 * t.kt;
    p.out = static_cast<uint8_t*>(workspace);
    uint8_t* out = p.out;
    const int weights = swiglu ? 2 : a.nseg;
    for (int j = -1; j < weights; ++j) {
      const int64_t rows = j < 0 ? a.M : a.n[swiglu ? 0 : j];
      p.s[j + 1] = j < 0 ? a.xs : a.ws[j];
      p.rows[j + 1] = rows;
      (j < 0 ? t.a.xs : t.a.ws[j]) = out;
      out += rows * p.ld;
    }
    hipLaunchKernelGGL(mx8_pad_scales_kernel, dim3(256, 1 + weights), dim3(256), 0, st, p);
    Q3_LAUNCH_CHECK();
    t.slx = t.slw = p.ld;
  }
  if (swiglu) launch_form<true>(t, plan.form, 1, st);
  else launch_form<false>(t, plan.form, 1, st);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // namespace q3

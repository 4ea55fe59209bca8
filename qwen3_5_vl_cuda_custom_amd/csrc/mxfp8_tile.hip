// Products of many MXFP8 rows: tiles of BM rows of x and BN weight rows through LDS
// (format and matrix instruction: mxfp8.h).
//
// Codes go global -> LDS past the registers (buffer loads with the lds flag), a stage of
// 128 k (one matrix instruction's) at a time, 128 bytes a row. Row r keeps its 16-byte
// chunk c at slot c ^ (r & 7), which leaves the fragments' reads without bank conflicts
// (with r >> 3 in the exclusive or as well, 3.5 cycles each were counted). The instructions
// of a full chip run at 3.5 to 3.75 PFLOP/s with nothing else to do (the clock falls to
// 2.0 GHz), and no branch stands in the loops: the compiler moves products past one.
//
// 256 x 256 tiles, eight waves of 128 x 64: a wave holds the stage's TN weight fragments and
// takes the TM fragments of x (columns, below) one after the other, each read three columns
// ahead, TN products to a column. Before the last two columns every fragment of the stage
// has been read: there the stage barrier stands, the next stage's fragments are read between
// the products after it, each weight fragment once its last product has issued. The two slots
// fill the LDS; a stage's weight slot is free once every wave has the fragments, after the
// first column: a second barrier there lets the weights after next, which come from further
// away than x, set out most of a stage earlier. Gate and up of 4096 rows, N 12288, K 4096:
// 316 us and 5 for the scales, 2.61 PFLOP/s; N 4096, K 12288 154 us, 2.68 PFLOP/s. What is
// left is the clock, the loads of codes beside the products, and the barriers.
//
// Smaller tiles, four waves of 128 x 64 or 64 x 64 for 128 x 256 and 128 x 128: one wave a SIMD
// has the registers for two stages' fragments. It reads all of the next stage's between the
// products of this one, so a slot is free at the barrier where its stage begins, and three or
// four slots stay under way. Waves that read as above, eight to a tile of 128 x 256, took 3 %
// longer for SwiGLU of 611 rows, N 12288, and for 128 x 128 and 1000 rows, N = K = 4096, 20 %;
// tiles of 256 x 256 take 86 and 52 us there, these 64 to 67 and 24 to 26: 64 and 32 stages of
// 0.6 and 0.3 us of products, the waits for codes between them, and 7.6 us of a tile with one
// stage alone (launch, first loads, epilogue).
//
// Scales are laid out anew first, by a kernel of their own: the scales of 64 rows and four
// stages are 1 KB as the instruction's lanes take them, word l of a stage lane l's block
// of rows l % 16, + 16, + 32, + 48 (the instruction picks the byte). A load brings a stage
// of them, and three words a stage are all that a wave reads. As rows of bytes their loads
// cost a line per row and the reads twelve bytes a stage: 2 % more for 4096 x 4096 x 12288.
// For small products the launch costs more (2.7 to 4 us), and 128 x 128 tiles take the
// scales by rows (RAW), 16 bytes, four stages', of a row at a time (both ways: form_of).
#include "gemm_tile.h"
#include "mxfp8.h"
#include "mxfp8_tile.h"

namespace {

using namespace q3;

struct TileArgs {
  Mx8Args a;
  const uint8_t* xs;                // scales of x, and of each weight (SwiGLU: of both), laid out as above
  const uint8_t* ws[kMx8Segments];
  int tiles_m, tiles_n, gm;
};

// Eight columns of y from col on (`left` of them exist, or less than one), the row's m (`in`: it exists); the lanes ^ 16,
// ^ 32 and ^ 48 hold the other columns of 32. PLAIN: with bias, activation and residual, the last eight values in `res`
// where all go in 16-byte pieces (`vec`).
template <bool PLAIN>
__device__ __forceinline__ void finish8(const Mx8Args& p, int64_t m, bool in, int col, int left, bool vec,
                                        const float (&bias)[8], const bf16x8& res, float (&v)[8]) {
  if (PLAIN) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias[e];
    mx8_act(v, p.act);
    if (p.res) {
      if (vec) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bf2f(res[e]);
      } else if (in) {
        const bf16* r = p.res + m * p.ldr + col;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) v[e] += bf2f(r[e]);
      }
    }
  }
  if (p.yc) {  // whole blocks of 32 columns
    uint32_t byte;
    const u32x2 c = mx8_quantize8<16>(v, byte);
    if (!in || left <= 0) return;
    *reinterpret_cast<u32x2*>(p.yc + m * p.ldc + col) = c;
    if ((col & 31) == 0) p.ys[m * (p.ldc / kMx8Block) + col / kMx8Block] = (uint8_t)byte;
    return;
  }
  if (!in) return;
  bf16* y = p.y + m * p.ldc + col;
  if (vec) {
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

// The product with byte bi and bj of the scale words.
__device__ __forceinline__ floatx4 mfma_of(i32x8 a, i32x8 b, floatx4 c, int sa, int sb, int bi, int bj) {
#define Q3_MX8_MFMA(I, J) \
  if (bi == I && bj == J) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, sa, J, sb);
#define Q3_MX8_ROW(I) Q3_MX8_MFMA(I, 0) Q3_MX8_MFMA(I, 1) Q3_MX8_MFMA(I, 2) Q3_MX8_MFMA(I, 3)
  Q3_MX8_ROW(0) Q3_MX8_ROW(1) Q3_MX8_ROW(2) Q3_MX8_ROW(3)
#undef Q3_MX8_ROW
#undef Q3_MX8_MFMA
  return c;
}

template <int BM, int BN, int WM, int WN, int NS, bool SW, bool RAW>
__global__ __launch_bounds__(WM* WN * 64) void mx8_tile_kernel(const TileArgs t) {
  constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  constexpr int BN_OUT = SW ? BN / 2 : BN;
  constexpr int GX = BM / 64, GS = (BM + BN) / 64, PS = (GS + NW - 1) / NW;  // groups of 64 rows; loads of scales
  constexpr int PX = BM / 8 / NW, PW = BN / 8 / NW;                          // loads of codes per wave and stage
  constexpr bool PIPE = NW == 4;  // one wave a SIMD: room for two stages' fragments in registers
  constexpr int kX = BM * 128, kW = BN * 128, kS = RAW ? (BM + BN) * 16 : PS * NW * 256;
  constexpr int kLds = NS * (kX + kW) + 4 * kS;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NW % 2 == 0, "whole loads per wave, one swizzle per lane");
  static_assert(PIPE || (NW == 8 && NS == 2), "the two loops");
  static_assert(!RAW || (PIPE && GS == NW && NS <= 4), "scales by rows: a wave to 64 rows");
  static_assert(TM % 4 == 0 && TN == 4 && kLds <= 160 * 1024, "wave tiles");
  __shared__ __attribute__((aligned(1024))) char smem[kLds];

  const Mx8Args& p = t.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN, l16 = lane & 15, q4 = lane >> 4;
  const int K = p.K;

  // This block's tile: the tiles of one XCD are neighbours, t.gm of them along m.
  const int pid = xcd_remap(blockIdx.x, t.tiles_m * t.tiles_n);
  const int group = pid / (t.gm * t.tiles_n), size_m = min(t.tiles_m - t.gm * group, t.gm);
  const int in = pid - group * t.gm * t.tiles_n;
  const int m0 = __builtin_amdgcn_readfirstlane((t.gm * group + in % size_m) * BM);
  int tn = __builtin_amdgcn_readfirstlane(in / size_m), seg = 0, col0 = 0;
#pragma unroll
  for (int j = 0; j + 1 < kMx8Segments; ++j) {
    const int nt = (p.n[j] + BN_OUT - 1) / BN_OUT;
    if (seg == j && j + 1 < p.nseg && tn >= nt) tn -= nt, col0 += p.n[j], seg = j + 1;
  }
  seg = mx8_pin(seg), tn = mx8_pin(tn), col0 = mx8_pin(col0);
  const int n0 = tn * BN_OUT, rows_n = mx8_pin(min(BN_OUT, p.n[seg] - n0)), rows_m = mx8_pin(min(BM, p.M - m0));
  const int nk = (K + 127) / 128, groups_k = (K + 511) / 512;  // stages, and groups of four

  const __amdgpu_buffer_rsrc_t rx = make_rsrc(mx8_pin(p.x + (int64_t)m0 * K), rows_m * K);
  const uint8_t* const wa = mx8_pin(p.w[SW ? 0 : seg] + (int64_t)n0 * K);  // SwiGLU: gate's, and up's
  const uint8_t* const wb = SW ? mx8_pin(p.w[1] + (int64_t)n0 * K) : wa;
  auto swz = [](int r) { return r & 7; };
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
  // Scales: load s of this wave is a stage of 64 rows, x's and then the weights' (by rows: four stages of 16 rows).
  const uint8_t* sp[PS];
  int sbytes[PS];
  const int kb = K / kMx8Block;
  if constexpr (RAW) {  // by rows: this wave's 64
    const uint8_t* of = p.xs + (int64_t)(m0 + 64 * wave) * kb;
    int rows = rows_m - 64 * wave;
    if (64 * wave >= BM) {
      const int first = (SW ? 32 : 64) * (wave - BM / 64);
      of = p.ws[SW ? 0 : seg] + (int64_t)(n0 + first) * kb;
      rows = rows_n - first;
    }
    sp[0] = mx8_pin(of);
    sbytes[0] = mx8_pin(max(rows, 0) * kb);
  } else {
#pragma unroll
    for (int s = 0; s < PS; ++s) {
      const int e = wave + NW * s;
      const bool of_x = e < GX;
      const int g = of_x ? m0 / 64 + e : (SW ? 2 * n0 : n0) / 64 + e - GX;
      // 64-row groups that exist: of all rows, SwiGLU 32 of each weight to a group
      const int all = of_x ? (p.M + 63) / 64 : SW ? (p.n[0] + 31) / 32 : (p.n[seg] + 63) / 64;
      sp[s] = mx8_pin((of_x ? t.xs : t.ws[seg]) + (int64_t)g * groups_k * 1024);
      sbytes[s] = mx8_pin(e < GS && g < all ? groups_k * 1024 : 0);
    }
  }
  const uint32_t lbase = lds_addr(smem);
  constexpr int kW0 = NS * kX, kS0 = kW0 + NS * kW;
  // Byte of a row at which the lane's chunk of stage kt lies; past the row's end past every resource too.
  auto kofs = [&](int kt) {
    const int k = kt * 128 + dc * 16;
    return k < K ? (uint32_t)k : kOOB;
  };
  // Load i of stage kt's codes, into a slot.
  auto dma_x = [&](int kt, int slot, int i) __attribute__((always_inline)) {
    dma16(rx, xoff[i] + kofs(kt), lbase + (uint32_t)(slot * kX + (wave + NW * i) * 1024));
  };
  auto dma_w = [&](int kt, int slot, int i) __attribute__((always_inline)) {
    const bool up = SW && ((wave + NW * i) & 4);
    dma16(make_rsrc(SW ? mx8_pin(up ? wb : wa) : wa, rows_n * K), woff[i] + kofs(kt),
          lbase + (uint32_t)(kW0 + slot * kW + (wave + NW * i) * 1024));
  };
  auto dma_s = [&](int kt, int s) {
    if constexpr (RAW) {
      // 16 of the wave's rows: 16 bytes, the scales of four stages, of the group of stages after kt's
      const int g = (kt >> 2) + 1, u = kt & 3, row = 16 * u + (lane >> 2), st = 4 * g + (lane & 3);
      const uint8_t* of = sp[0];
      int at = row;
      if (SW && wave >= BM / 64 && u >= 2) of = p.ws[1] + (int64_t)(n0 + 32 * (wave - BM / 64)) * kb, at = row - 32;
      dma4(make_rsrc(mx8_pin(of), sbytes[0]), st < nk ? (uint32_t)(at * kb + 4 * st) : kOOB,
           lbase + (uint32_t)(kS0 + (g & 3) * kS + (64 * wave + 16 * u) * 16));
      return;
    }
    dma4(make_rsrc(sp[s], sbytes[s]), kt < nk ? (uint32_t)(kt * 256 + lane * 4) : kOOB,
         lbase + (uint32_t)(kS0 + (kt & 3) * kS + (wave + NW * s) * 256));
  };
  constexpr int kAll = PS + PW + PX;
  // Load d of them.
  auto dma = [&](int kt, int slot, int d) __attribute__((always_inline)) {
    if (d < PS) dma_s(kt, d);
    else if (d < PS + PW) dma_w(kt, slot, d - PS);
    else dma_x(kt, slot, d - PS - PW);
  };

  floatx4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = floatx4{};
  const int rn = wn * WTN, rm = wm * WTM;

  if constexpr (RAW) {
#pragma unroll
    for (int s = -4; s < 0; ++s) dma_s(s, 0);  // the first four stages'
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) {
#pragma unroll
    for (int d = 0; d < kAll; ++d) dma(s, s, d);
  }
  vm_wait<(NS - 1) * kAll>();  // stage 0 has landed
  __syncthreads();

  if constexpr (PIPE) {
    i32x8 pw[2][TN], px[2][TM];
    int zw[2][RAW ? TN : 1], zx[2][RAW ? TM : TM / 4];
    const char* const xrow = smem + (rm + l16) * 128;
    const char* const wrow = smem + kW0 + (rn + l16) * 128;
    const int c0 = (q4 ^ (l16 & 7)) << 4, c1 = ((4 + q4) ^ (l16 & 7)) << 4;
    // Read number n of a stage in slot `at`, to fragments g: the weights', then x's.
    auto read = [&](int g, int n, int at_x, int at_w) __attribute__((always_inline)) {
      const bool w = n < 2 * TN;
      const int f = w ? n / 2 : n / 2 - TN;
      const char* const from = (w ? wrow + at_w : xrow + at_x) + f * 2048 + (n & 1 ? c1 : c0);
      const i32x4 v = *reinterpret_cast<const i32x4*>(from);
      i32x8& to = w ? pw[g][f] : px[g][f];
#pragma unroll
      for (int e = 0; e < 4; ++e) to[4 * (n & 1) + e] = v[e];
    };
    auto read_s = [&](int g, int kt) __attribute__((always_inline)) {
      if constexpr (RAW) {
        const uint8_t* const z = reinterpret_cast<const uint8_t*>(smem) + kS0 + (kt >> 2 & 3) * kS + (kt & 3) * 4 + l16 * 16 + q4;
#pragma unroll
        for (int i = 0; i < TN; ++i) zw[g][i] = z[(BM + rn + 16 * i) * 16];
#pragma unroll
        for (int j = 0; j < TM; ++j) zx[g][j] = z[(rm + 16 * j) * 16];
      } else {
        const char* const z = smem + kS0 + (kt & 3) * kS + lane * 4;
        zw[g][0] = *reinterpret_cast<const int*>(z + (GX + rn / 64) * 256);
#pragma unroll
        for (int j = 0; j < TM / 4; ++j) zx[g][j] = *reinterpret_cast<const int*>(z + (rm / 64 + j) * 256);
      }
    };
    read_s(0, 0);
#pragma unroll
    for (int n = 0; n < 2 * (TN + TM); ++n) read(0, n, 0, 0);
    int cur = 0;  // slot of the stage at hand
    auto stage = [&](auto parity, int kt) __attribute__((always_inline)) {
      constexpr int G = decltype(parity)::value;
      const int nxt = cur + 1 == NS ? 0 : cur + 1;
      // Stage kt + 1 has landed, and every wave holds stage kt: its slot is free.
      vm_wait<(NS - 2) * kAll>();
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      constexpr int kReads = 2 * (TN + TM), kMf = TN * TM;
      int n = 0, d = 0;
#pragma unroll
      for (int m = 0; m < kMf; ++m) {
        acc[m % TN][m / TN] =
            RAW ? mfma_of(pw[G][m % TN], px[G][m / TN], acc[m % TN][m / TN], zw[G][RAW ? m % TN : 0], zx[G][RAW ? m / TN : 0], 0, 0)
                : mfma_of(pw[G][m % TN], px[G][m / TN], acc[m % TN][m / TN], zw[G][0], zx[G][RAW ? 0 : m / TN / 4], m % TN, m / TN & 3);
        if (m == 0) read_s(G ^ 1, kt + 1);
        for (; n < kReads && n * (kMf - 4) < (m + 1) * kReads; ++n) read(G ^ 1, n, nxt * kX, nxt * kW);
        for (; d < kAll && d * (kMf - 2) < m * kAll; ++d) dma(kt + NS, cur, d);
        __builtin_amdgcn_sched_barrier(0);
      }
      cur = nxt;
    };
    for (int kt = 0; kt < nk; kt += 2) {  // an odd last stage's partner is zeros
      stage(std::integral_constant<int, 0>{}, kt);
      stage(std::integral_constant<int, 1>{}, kt + 1);
    }
#pragma unroll
    for (int i = 0; i < TN; ++i)  // (the accumulators stay where they are: without this they are copied around each turn)
#pragma unroll
      for (int j = 0; j < TM; ++j) asm volatile("" : "+a"(acc[i][j]));
    __builtin_amdgcn_s_waitcnt(0xc07f);
  } else {
    i32x8 fw[TN], fx[4];
    int sw, sx[TM / 4], sw_next, sx_next[TM / 4];  // a stage's words of scales
    auto frag = [&](const char* slot, int r) {
      const char* row = slot + r * 128;
      const i32x4 lo = *reinterpret_cast<const i32x4*>(row + ((q4 ^ swz(r)) << 4));
      const i32x4 hi = *reinterpret_cast<const i32x4*>(row + (((4 + q4) ^ swz(r)) << 4));
      return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto rd_w = [&](int kt, int i) { fw[i] = frag(smem + kW0 + kt % NS * kW, rn + 16 * i + l16); };
    auto rd_x = [&](int kt, int j) { fx[j & 3] = frag(smem + kt % NS * kX, rm + 16 * j + l16); };
    auto rd_s = [&](int kt) {
      const char* s = smem + kS0 + (kt & 3) * kS + lane * 4;
      sw_next = *reinterpret_cast<const int*>(s + (GX + rn / 64) * 256);
#pragma unroll
      for (int g = 0; g < TM / 4; ++g) sx_next[g] = *reinterpret_cast<const int*>(s + (rm / 64 + g) * 256);
    };
    auto take_s = [&]() {
      sw = sw_next;
#pragma unroll
      for (int g = 0; g < TM / 4; ++g) sx[g] = sx_next[g];
    };
    auto mf = [&](int i, int j) { acc[i][j] = mfma_of(fw[i], fx[j & 3], acc[i][j], sw, sx[j / 4], i, j & 3); };
    auto main = [&](auto active_c) {
      constexpr bool A = decltype(active_c)::value;  // a wave without rows loads and waits only
      if constexpr (A) {
        rd_s(0);
        take_s();
#pragma unroll
        for (int i = 0; i < TN; ++i) rd_w(0, i);
#pragma unroll
        for (int j = 0; j < 3; ++j) rd_x(0, j);
        // Nothing is left under way here, so that the loop's waits are counted from its own loads (lgkmcnt 0).
        __builtin_amdgcn_s_waitcnt(0xc07f);
      }
      for (int kt = 0; kt < nk; ++kt) {
        const int next = kt + NS;  // the stage whose loads go out
        int d = 0;                 // scales and weights, after the first column
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < TM - 2; ++j) {
#pragma unroll
          for (int i = 0; i < TN; ++i) {
            if constexpr (A) {
              mf(i, j);
              if (i == 0 && j + 3 < TM) rd_x(kt, j + 3);
            }
            constexpr int gap = TN * (TM - 3) / (PS + PW);
            const int at = (j - 1) * TN + i;
            if (at >= 0 && at % gap == gap - 1 && d < PS + PW) dma(next, kt % NS, d++);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (j == 0) {  // every wave holds the weights' fragments (read before the last one of x)
            asm volatile("s_waitcnt lgkmcnt(2)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (; d < PS + PW; ++d) dma(next, kt % NS, d);
        // Stage kt + 1 has landed (later ones may not have) and every fragment of stage kt is in registers, in every wave.
        vm_wait<PS + PW>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (A) {
          rd_s(kt + 1);
          rd_x(kt + 1, 0);
          rd_x(kt + 1, 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < TN; ++i) {
            mf(i, TM - 2);
            if (i < PX) dma_x(next, kt % NS, i);
            mf(i, TM - 1);
            rd_w(kt + 1, i);
            __builtin_amdgcn_sched_barrier(0);
          }
          rd_x(kt + 1, 2);
          take_s();
        }
#pragma unroll
        for (int i = A ? TN : 0; i < PX; ++i) dma_x(next, kt % NS, i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (rm < rows_m) main(std::true_type{});
    else main(std::false_type{});
  }
  vm_wait<0>();  // the loads past the last stage (zeros) have landed: the LDS may go to another block

  // Epilogue: lane (l16, q4) holds columns 4 q4 .. + 3 of row l16 of its products; of two neighbouring products the lane
  // rows change places (permlane16), and it holds eight: 16-byte pieces, four of them 64 bytes of a row. The residuals of
  // four rows of products are under way before the first is used. (Through the LDS, fp32 and whole rows: 1 us more of
  // 8.7 for a 128 x 128 tile with one stage, and 3 to 6 of 175 to 327 us for 4096 rows.)
  constexpr int OP = (SW ? TN / 2 : TN) / 2, JB = 4;
  const int c0 = (SW ? rn / 2 : rn) + 16 * (q4 & 1) + 8 * (q4 >> 1);
  const bool vec = vec_of(p, col0);
  float bias[OP][8] = {};
  if (!SW && p.bias[seg]) {
    const bf16* const b = p.bias[seg] + n0 + c0;
    const bool pieces = (reinterpret_cast<uintptr_t>(p.bias[seg]) & 15) == 0;
#pragma unroll
    for (int o = 0; o < OP; ++o) {
      const int left = rows_n - c0 - 32 * o;
      if (pieces && left >= 8) {
        const bf16x8 u = *reinterpret_cast<const bf16x8*>(b + 32 * o);
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[o][e] = bf2f(u[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) bias[o][e] = bf2f(b[32 * o + e]);
      }
    }
  }
#pragma unroll
  for (int jb = 0; jb < TM; jb += JB) {
    bf16x8 res[JB][OP];
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int o = 0; o < OP; ++o) {
        const int r = rm + 16 * (jb + j) + l16, c = c0 + 32 * o;
        res[j][o] = bf16x8{};
        if (!SW && p.res && vec && r < rows_m && c + 8 <= rows_n)
          res[j][o] = *reinterpret_cast<const bf16x8*>(p.res + (int64_t)(m0 + r) * p.ldr + col0 + n0 + c);
      }
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int o = 0; o < OP; ++o) {
        const int r = rm + 16 * (jb + j) + l16, c = c0 + 32 * o, left = rows_n - c;
        floatx4 a = acc[2 * o][jb + j], b = acc[2 * o + 1][jb + j];
        if constexpr (SW) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] = silu_mul(acc[0][jb + j][e], acc[2][jb + j][e]);
            b[e] = silu_mul(acc[1][jb + j][e], acc[3][jb + j][e]);
          }
        }
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = a[e], y = b[e];
          const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y),
                                                          false, false);
          v[e] = __builtin_bit_cast(float, (uint32_t)s[0]);
          v[4 + e] = __builtin_bit_cast(float, (uint32_t)s[1]);
        }
        finish8<!SW>(p, m0 + r, r < rows_m, col0 + n0 + c, left, vec && left >= 8, bias[o], res[j][o], v);
      }
  }
}

// Scales of 64 rows and four stages as the kernel above takes them (the file's head), zeros past the last row and block;
// SwiGLU: 32 rows of gate, then the same of up. A wave lays out 64 rows of 16 stages: lane l holds 16 bytes of row l at a
// time, and the words of four stages are a transposition between the lanes l % 16 + 16 e and the bytes.
struct LayArgs {
  const uint8_t *s[1 + kMx8Segments], *s2;  // x's, each weight's (rows, kb); up's
  int rows[1 + kMx8Segments], first[1 + kMx8Segments];  // of each; the first wave of each
  uint8_t* out[1 + kMx8Segments];
  int kb, groups_k, nb, mats, waves;  // blocks of 32 k, groups of four stages, waves along k, matrices
};

// Words s of lane l, row l's four stages, to words s: byte e that of block l / 16 of row 16 e + l % 16.
__device__ __forceinline__ void mx8_turn(uint32_t (&w)[4]) {
  // 4 x 4 bytes: words s, bytes q to words q, bytes s; and back
  auto bytes = [](uint32_t (&v)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u), b = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u), d = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
    v[0] = __builtin_amdgcn_perm(c, a, 0x05040100u), v[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    v[2] = __builtin_amdgcn_perm(d, b, 0x05040100u), v[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
  };
  bytes(w);
  // words q of the lanes 16 e + .. to words e of the lanes 16 q + ..
  const auto p = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), q = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const auto u = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false), v = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
  w[0] = u[0], w[1] = u[1], w[2] = v[0], w[3] = v[1];
  bytes(w);
}

__global__ __launch_bounds__(256) void mx8_lay_scales_kernel(const LayArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6))), lane = threadIdx.x & 63;
  if (wave >= a.waves) return;
  int j = 0;
#pragma unroll
  for (int u = 1; u <= kMx8Segments; ++u)
    if (u < a.mats && wave >= a.first[u]) j = u;
  const int at = wave - a.first[j], g = at / a.nb, g0 = at % a.nb * 4;  // 64 rows, first group of four stages
  const bool pair = j == 1 && a.s2;
  const int row = pair ? g * 32 + (lane & 31) : g * 64 + lane;
  // Every address lies in the matrix; what is past its rows or a row's end becomes zero after the loads.
  const uint8_t* src = (pair && lane >= 32 ? a.s2 : a.s[j]) + (int64_t)min(row, a.rows[j] - 1) * a.kb;
  const int end = row < a.rows[j] ? a.kb : 0, c0 = g0 * 16;
  uint32_t w[4][4];
  if (a.kb % 16 == 0) {
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(4)));
    words v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const words*>(src + min(c0 + 16 * i, a.kb - 16));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int s = 0; s < 4; ++s) w[i][s] = c0 + 16 * i < end ? v[i][s] : 0;
  } else if (a.kb % 4 == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i / 4][i % 4] = *reinterpret_cast<const uint32_t*>(src + min(c0 + 4 * i, a.kb - 4));
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c0 + 4 * i >= end) w[i / 4][i % 4] = 0;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      w[i / 4][i % 4] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = c0 + 4 * i + e;
        const uint32_t v = src[min(c, a.kb - 1)];
        w[i / 4][i % 4] |= c < end ? v << (8 * e) : 0;
      }
    }
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(a.out[j]) + ((int64_t)g * a.groups_k + g0) * 256 + lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (g0 + i >= a.groups_k) break;
    mx8_turn(w[i]);
#pragma unroll
    for (int s = 0; s < 4; ++s) out[i * 256 + s * 64] = w[i][s];
  }
}

int64_t tiles_of(const Mx8Args& a, int bn) {
  int64_t n = 0;
  for (int j = 0; j < a.nseg; ++j) n += q3_cdiv(a.n[j], bn);
  return n;
}

template <int BM, int BN, int WM, int WN, int NS, bool SW, bool RAW = false>
void launch_tile(TileArgs t, hipStream_t st) {
  t.tiles_m = (int)q3_cdiv(t.a.M, BM);
  t.tiles_n = (int)tiles_of(t.a, SW ? BN / 2 : BN);
  // The tiles along m in even groups of at most 1024 rows: a remainder of one tile read the weights once more for itself
  // (SwiGLU of 611 rows, N 12288: 4 + 1 tiles 77 us, 5 71.5). Groups of 768 to 2048 rows: within 2 %.
  constexpr int kGroup = 1024 / BM;
  t.gm = (int)q3_cdiv(t.tiles_m, q3_cdiv(t.tiles_m, kGroup));
  hipLaunchKernelGGL((mx8_tile_kernel<BM, BN, WM, WN, NS, SW, RAW>), dim3((unsigned)(t.tiles_m * t.tiles_n)),
                     dim3(WM * WN * 64), 0, st, t);
}

// Forms: tiles of 256 x 256, 128 x 256, 128 x 128, and of the last size with the scales by rows.
constexpr int kFormBM[4] = {256, 128, 128, 128}, kFormBN[4] = {256, 256, 128, 128}, kFormThreads[4] = {512, 256, 256, 256};

template <bool SW>
void launch_form(const TileArgs& t, int form, hipStream_t st) {
  if (form == 0) launch_tile<256, 256, 2, 4, 2, SW>(t, st);
  else if (form == 1) launch_tile<128, 256, 1, 4, 3, SW>(t, st);
  else if (form == 2) launch_tile<128, 128, 2, 2, 4, SW>(t, st);
  else launch_tile<128, 128, 2, 2, 4, SW, true>(t, st);
}

// The form that costs least, by launches + rounds x (first loads and epilogue + stages x a stage), in 10 ns: fitted to one,
// two and four full rounds (a block on each of the 256 CUs) of K 128 to 12288, within 8 %; a last round of few tiles counts
// three quarters of a full one, as fewer blocks get their loads sooner. Measured with each form forced, in us, 256 x 256,
// 128 x 256, 128 x 128 laid out and by rows: 4096 rows, N 4096, K 4096 62, 71, 81, 86; 2048 rows 48, 38, 45, 45; 1024 rows
// 46, 32, 24.5, 24, K 1152 22, 18, 14, 12, K 12288 111, 67, 55, 56; 4096 rows, N 4304 (a seventeenth tile) 94, 93, 96, 102,
// K 1152 43, 50, 49, 48. Scales by rows want whole words of them.
int form_of(const Mx8Args& a, bool swiglu) {
  const int64_t out = swiglu ? 2 : 1, stages = q3_cdiv(a.K, 128);
  auto cost = [&](int bm, int bn, int64_t launches, int64_t fixed, int64_t stage) {
    // (past 2^32 tiles, more than a launch takes, any count will do)
    const int64_t tiles = std::min<int64_t>(q3_cdiv(a.M, bm) * tiles_of(a, (int)(bn / out)), 1ll << 32), rest = tiles % 256;
    return launches * 1024 + (tiles / 256 * 1024 + (rest ? 768 + rest : 0)) * (fixed + stages * stage);
  };
  const int64_t costs[4] = {cost(256, 256, 760, 800, 138), cost(128, 256, 750, 730, 75), cost(128, 128, 430, 540, 43),
                            cost(128, 128, 230, 540, 49)};
  int best = 0;
  for (int j = 1; j < (a.K % 128 == 0 ? 4 : 3); ++j)
    if (costs[j] < costs[best]) best = j;
  return best;
}

// Bytes of laid out scales of n rows.
int64_t laid_bytes(int64_t n, int64_t K) { return q3_cdiv(n, 64) * q3_cdiv(K, 512) * 1024; }

// The scales of t's operands laid out in the workspace.
int lay_scales(TileArgs& t, bool swiglu, void* workspace, hipStream_t st) {
  const Mx8Args& a = t.a;
  LayArgs l{};
  l.kb = a.K / kMx8Block;
  l.groups_k = (int)q3_cdiv(a.K, 512);
  l.nb = (int)q3_cdiv(l.groups_k, 4);
  l.mats = 1 + a.nseg;
  l.s2 = swiglu ? a.ws[1] : nullptr;
  uint8_t* out = static_cast<uint8_t*>(workspace);
  int64_t waves = 0;
  for (int j = 0; j < l.mats; ++j) {
    l.s[j] = j ? a.ws[j - 1] : a.xs;
    l.rows[j] = j ? a.n[j - 1] : a.M;
    l.first[j] = (int)waves;
    l.out[j] = out;
    (j ? t.ws[j - 1] : t.xs) = out;
    const int64_t groups = j && swiglu ? q3_cdiv(l.rows[j], 32) : q3_cdiv(l.rows[j], 64);
    waves += groups * l.nb;
    out += groups * l.groups_k * 1024;
  }
  Q3_REQUIRE(mx8_grid_ok(q3_cdiv(waves, 4), 256), Q3_ERR_UNSUPPORTED);
  l.waves = (int)waves;
  hipLaunchKernelGGL(mx8_lay_scales_kernel, dim3((unsigned)q3_cdiv(waves, 4)), dim3(256), 0, st, l);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // namespace

namespace q3 {

int mx8_tile_form(const Mx8Args& a, bool swiglu) { return form_of(a, swiglu); }

int64_t mx8_tile_workspace(const Mx8Args& a, bool swiglu) {
  if (form_of(a, swiglu) == 3) return 0;
  int64_t bytes = laid_bytes(a.M, a.K);
  if (swiglu) return bytes + laid_bytes(2 * q3_cdiv(a.n[0], 32) * 32, a.K);
  for (int j = 0; j < a.nseg; ++j) bytes += laid_bytes(a.n[j], a.K);
  return bytes;
}

int mx8_tile(const Mx8Args& a, bool swiglu, void* workspace, hipStream_t st) {
  TileArgs t{};
  t.a = a;
  const int form = form_of(a, swiglu);
  Q3_REQUIRE(mx8_grid_ok(q3_cdiv(a.M, kFormBM[form]) * tiles_of(a, kFormBN[form] / (swiglu ? 2 : 1)), kFormThreads[form]),
             Q3_ERR_UNSUPPORTED);
  if (form < 3)
    if (const int rc = lay_scales(t, swiglu, workspace, st)) return rc;
  if (swiglu) launch_form<true>(t, form, st);
  else launch_form<false>(t, form, st);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // namespace q3

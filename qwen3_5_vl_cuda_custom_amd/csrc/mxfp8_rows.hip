// Products of MXFP8 rows with MXFP8 weights by whole weight rows, up to 64 rows of x to
// a block (format and matrix instruction: mxfp8.h):
//   y = act(x w^T (+ bias)) (+ residual),  y = silu(x g^T) * (x u^T)
// over one weight, or the weights of several projections side by side; y in bf16 or in
// eight bits again.
//
// A block owns whole weight rows, all of k, so no sums pass between blocks: its four waves
// take a quarter of the k each and their sums meet in LDS, in wave order. The weight is the
// instruction's first operand, so lane l holds columns 4 (l / 16) .. + 3 of y's row l % 16.
#include "gemm_tile.h"
#include "mxfp8.h"

namespace {

using namespace q3;

constexpr int kWaves = 4;

// The block's sums (wave, group, tile of x; lane l: columns 4 (l / 16) .. + 3 of y's row l % 16), joined in wave order,
// finished and stored: rows [m0, m0 + M) of y, `rows` columns from n0 of weight seg, which starts at column col0. Four
// columns of a row per lane; the eight lanes of 32 columns are neighbours.
template <int RG, int MT, bool SW>
__device__ __forceinline__ void finish_block(const Mx8Args& p, const floatx4* sums, int seg, int m0, int M, int n0, int rows,
                                             int col0) {
  constexpr int RGT = SW ? 2 * RG : RG;
  for (int it = threadIdx.x; it < RG * MT * 64; it += 64 * kWaves) {
    const int m = it / (4 * RG), c = it % (4 * RG), at = (m & 15) + 16 * (c & 3);
    if (m >= M || 4 * c >= rows) continue;
    auto total = [&](int g) {
      floatx4 v = sums[(g * MT + m / 16) * 64 + at];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += sums[((w * RGT + g) * MT + m / 16) * 64 + at];
      return v;
    };
    floatx4 v = total(c / 4);
    if constexpr (SW) {
      const floatx4 u = total(RG + c / 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = silu_mul(v[e], u[e]);
    }
    const int left = rows - 4 * c, n = n0 + 4 * c, col = col0 + n;
    const int64_t row = m0 + m;
    const bool vec = p.vec && left >= 4;  // whole 8-byte pieces
    if (!SW) {
      if (const bf16* b = p.bias[seg]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) v[e] += bf2f(b[n + e]);
      }
      float u[4] = {v[0], v[1], v[2], v[3]};
      mx8_act(u, p.act);
      v = floatx4{u[0], u[1], u[2], u[3]};
    }
    if (p.res) {
      const bf16* r = p.res + row * p.ldr + col;
      if (vec) {
        const bf16x4 b = *reinterpret_cast<const bf16x4*>(r);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += bf2f(b[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) v[e] += bf2f(r[e]);
      }
    }
    if (p.yc) {  // the columns are whole blocks
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, mx8_magnitude(v[e]));
#pragma unroll
      for (int o = 1; o < 8; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      const uint32_t byte = mx8_scale_byte(top);
      const uint32_t codes = byte == 255 ? 0 : mx8_pack4(v[0], v[1], v[2], v[3], mx8_scale(byte));
      *reinterpret_cast<uint32_t*>(p.yc + row * p.ldc + col) = codes;
      if ((c & 7) == 0) p.ys[row * (p.ldc / kMx8Block) + col / kMx8Block] = (uint8_t)byte;
    } else {
      bf16* y = p.y + row * p.ldc + col;
      if (vec) {
        *reinterpret_cast<bf16x4*>(y) = bf16x4{f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) y[e] = f2bf(v[e]);
      }
    }
  }
}

// Weight and block of it that block b of the grid takes, and y's column at which the weight starts.
__device__ __forceinline__ int segment_of_block(const Mx8Args& p, int rows, int& b, int& col0) {
  int seg = 0;
  col0 = 0;
#pragma unroll
  for (int j = 0; j + 1 < kMx8Segments; ++j) {
    const int nb = (p.n[j] + rows - 1) / rows;
    if (seg == j && j + 1 < p.nseg && b >= nb) b -= nb, col0 += p.n[j], seg = j + 1;
  }
  b = __builtin_amdgcn_readfirstlane(b);
  col0 = __builtin_amdgcn_readfirstlane(col0);
  return __builtin_amdgcn_readfirstlane(seg);
}

// Any K and any alignment of the rows of scales, up to 64 rows: fragments and scales straight into registers.
// RG: 16-row groups of weights (SwiGLU: of each of the two), MT: 16-row tiles of x.
template <int RG, int MT, bool SW>
__global__ __launch_bounds__(64 * kWaves) void mx8_rows_kernel(const Mx8Args p) {
  constexpr int RGT = SW ? 2 * RG : RG;
  __shared__ floatx4 sums[kWaves * RGT * MT * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  int b = blockIdx.x, col0;
  const int seg = segment_of_block(p, 16 * RG, b, col0);
  const int n0 = b * 16 * RG, rows = min(16 * RG, p.n[seg] - n0), K = p.K, kb = K / kMx8Block;
  const int M = p.M;

  __amdgpu_buffer_rsrc_t rw[2], rs[2];
#pragma unroll
  for (int u = 0; u < (SW ? 2 : 1); ++u) {
    rw[u] = make_rsrc(p.w[SW ? u : seg] + (int64_t)n0 * K, (int64_t)rows * K);
    rs[u] = make_rsrc(p.ws[SW ? u : seg] + (int64_t)n0 * kb, (int64_t)rows * kb);
  }
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x, (int64_t)M * K);
  const __amdgpu_buffer_rsrc_t rxs = make_rsrc(p.xs, (int64_t)M * kb);

  // Row `row`'s 16 bytes at k and at k + 64, and the scale of block s: zeros past the row's end and the last row.
  auto frag = [&](__amdgpu_buffer_rsrc_t r, int row, int k) {
    const int off = row * K + k;
    const i32x4 lo = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k < K ? off : (int)kOOB, 0, 0));
    const i32x4 hi =
        __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k + 64 < K ? off + 64 : (int)kOOB, 0, 0));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto scale = [&](__amdgpu_buffer_rsrc_t r, int row, int s) {
    return (int)__builtin_amdgcn_raw_buffer_load_b8(r, s < kb ? row * kb + s : (int)kOOB, 0, 0);
  };

  floatx4 acc[RGT][MT];
#pragma unroll
  for (int g = 0; g < RGT; ++g)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[g][j] = floatx4{};
  for (int c = wave; c * 128 < K; c += kWaves) {
    i32x8 w[RGT], x[MT];
    int sw[RGT], sx[MT];
#pragma unroll
    for (int g = 0; g < RGT; ++g) {
      const int u = g >= RG ? 1 : 0, row = 16 * (g - u * RG) + i;
      w[g] = frag(rw[u], row, c * 128 + 16 * q);
      sw[g] = scale(rs[u], row, c * 4 + q);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      x[j] = frag(rx, 16 * j + i, c * 128 + 16 * q);
      sx[j] = scale(rxs, 16 * j + i, c * 4 + q);
    }
#pragma unroll
    for (int g = 0; g < RGT; ++g)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[g][j] = mfma_mx8(w[g], x[j], acc[g][j], sw[g], sx[j]);
  }
#pragma unroll
  for (int g = 0; g < RGT; ++g)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[((wave * RGT + g) * MT + j) * 64 + lane] = acc[g][j];
  __syncthreads();

  finish_block<RG, MT, SW>(p, sums, seg, 0, M, n0, rows, col0);
}

// The same with K a multiple of 128, fed by a ring of stages of 512 k: codes (whole row pieces) go global -> LDS past the
// registers, up to four stages ahead, one barrier a stage. Row r keeps its 16-byte chunk c at slot c ^ (r & 15). A wave takes
// a quarter of a stage, one matrix instruction for each group and tile. Scales come 64 bytes of a row at a time, four
// stages' (as 16 bytes with every stage, a line each for the same lines again, they cost 3 of 21 us at 32 rows of K 12288).
// XR: rows of x in LDS. Weights past the last cache: one row, N = K = 4096 6.5 us (17.3 MB; 4.1 with a row of one
// stage, 4.3 with no weight read: the rest is launch, first loads and the sums), SwiGLU of N 12288 22.5 us (104 MB, 4.6
// TB/s; weights in the last cache 18.9), 32 rows, N 4096, K 12288 18.3 us (15.8), N 151936 131 us (4.9 TB/s).
template <int RG, int XR, bool SW>
struct RingShape {
  static constexpr int RGT = SW ? 2 * RG : RG, MT = XR > 16 ? XR / 16 : 1;
  static constexpr int PW = 2 * RGT, PX = XR / 8, PER = PW + PX;  // loads of a wave and stage: weights, x
  static constexpr int kW = RGT * 8192, kX = XR * 512, kSlot = kW + kX;
  static constexpr int kS = (RGT + MT) * 1024;  // four stages' scales, two slots
  // As many stages as leave room for two blocks on a CU where x is small, the next one's first loads under the last one's
  // sums; else as the LDS holds.
  static constexpr int kLds = (XR <= 8 && 3 * kSlot + 2 * kS <= 80 * 1024 ? 80 : 160) * 1024 - 2 * kS;
  static constexpr int NS = kLds / kSlot >= 5 ? 5 : kLds / kSlot;  // the loads run at most one slot of scales ahead
  static_assert(NS >= 2 && (NS - 2) * PER < 64 && kWaves * RGT * MT * 1024 <= NS * kSlot, "the ring, and the waves' sums");
};

template <int RG, int XR, bool SW>
__global__ __launch_bounds__(64 * kWaves) void mx8_ring_kernel(const Mx8Args p) {
  typedef RingShape<RG, XR, SW> S;
  constexpr int RGT = S::RGT, MT = S::MT, NS = S::NS, kS0 = NS * S::kSlot;
  __shared__ __attribute__((aligned(1024))) char smem[kS0 + 2 * S::kS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  int b = blockIdx.x, col0, part = 0;
  if constexpr (XR == 64) {
    const int parts = (p.M + 63) / 64;
    if (parts > 1) {  // blocks of the same weight rows are neighbours on one XCD
      const int pid = xcd_remap(b, gridDim.x);
      b = pid / parts;
      part = pid - b * parts;
    }
  }
  const int seg = segment_of_block(p, p.r, b, col0);
  const int n0 = b * p.r, rows = __builtin_amdgcn_readfirstlane(min(p.r, p.n[seg] - n0));
  const int m0 = XR == 64 ? mx8_pin(64 * part) : 0, M = XR == 64 ? mx8_pin(min(p.M - m0, 64)) : p.M;
  const int K = p.K, kb = K / kMx8Block, steps = (K + 511) / 512;
  const uint32_t lbase = lds_addr(smem);

  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * K, (int64_t)M * K);
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.w[SW ? 0 : seg] + (int64_t)n0 * K, (int64_t)rows * K);
  const __amdgpu_buffer_rsrc_t rb = SW ? make_rsrc(p.w[1] + (int64_t)n0 * K, (int64_t)rows * K) : ra;
  // Scales, four stages of 16 rows a load: the groups' (SwiGLU: gate's, then up's), x's tiles'. What lies past a row's end
  // is not used.
  constexpr int kSL = (RGT + MT + kWaves - 1) / kWaves;
  const uint8_t* sp[kSL];
  int sbytes[kSL];
#pragma unroll
  for (int u = 0; u < kSL; ++u) {
    const int d = u * kWaves + wave, g = SW && d >= RG ? d - RG : d, left = 16 * (d >= RGT ? d - RGT : g);
    const uint8_t* of = p.ws[SW ? 0 : seg] + (int64_t)n0 * kb;
    if (SW && d >= RG) of = p.ws[1] + (int64_t)n0 * kb;
    if (d >= RGT) of = p.xs + (int64_t)m0 * kb;
    sp[u] = mx8_pin(of + (int64_t)left * kb);
    sbytes[u] = mx8_pin(max(((d >= RGT ? M : rows) - left) * kb, 0));
  }
  const uint32_t soff = (uint32_t)((lane >> 2) * kb + (lane & 3) * 16);
  // A load of codes is two rows: load u of this wave rows 8 u + lr of x or of the groups. Its chunk, and offset at k = 0,
  // for even and odd u.
  const int lr = 2 * wave + (lane >> 5);
  int kof[2];
  uint32_t off0[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    kof[h] = 16 * ((lane & 31) ^ (8 * h + lr));
    off0[h] = (uint32_t)((8 * h + lr) * K + kof[h]);
  }
  auto issue = [&](int t, int at0) {
    const uint32_t at = lbase + (uint32_t)at0, k = (uint32_t)t * 512;
    if (t % 4 == 0) {
#pragma unroll
      for (int u = 0; u < kSL; ++u)
        if (u * kWaves + wave < RGT + MT)
          dma16(make_rsrc(sp[u], sbytes[u]), soff + (uint32_t)t * 16,
                lbase + (uint32_t)(kS0 + (t / 4 & 1) * S::kS + (u * kWaves + wave) * 1024));
    }
    const bool in[2] = {(int)k + kof[0] < K, (int)k + kof[1] < K};
#pragma unroll
    for (int u = 0; u < S::PX; ++u)
      dma16(rx, in[u & 1] ? off0[u & 1] + (uint32_t)(u / 2 * 16 * K) + k : kOOB, at + S::kW + (4 * u + wave) * 1024);
#pragma unroll
    for (int u = 0; u < S::PW; ++u) {
      const int g = u / 2;
      dma16_nt(SW && g >= RG ? rb : ra, in[u & 1] ? off0[u & 1] + (uint32_t)((g < RG ? g : g - RG) * 16 * K) + k : kOOB,
               at + (4 * u + wave) * 1024);
    }
  };

  floatx4 acc[RGT][MT];
#pragma unroll
  for (int g = 0; g < RGT; ++g)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[g][j] = floatx4{};
#pragma unroll 1
  for (int t = 0; t < NS - 1; ++t) issue(t, t * S::kSlot);
  int cur = 0, next = (NS - 1) * S::kSlot;  // slots of stage t and of stage t + NS - 1
  for (int t = 0; t < steps; ++t) {
    vm_wait<(NS - 2) * S::PER>();                                    // this wave's part of stage t has landed
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // every wave's; nobody reads stage t - 1 any more
    issue(t + NS - 1, next);
    const char* st = smem + cur;
    next = cur;
    cur = cur == (NS - 1) * S::kSlot ? 0 : cur + S::kSlot;
    const bool in = t * 16 + 4 * wave + q < kb;  // past the row's end codes are 0, scales may be anything
    auto frag = [&](const char* row, int r) {
      const i32x4 lo = *reinterpret_cast<const i32x4*>(row + (((8 * wave + q) ^ r) << 4));
      const i32x4 hi = *reinterpret_cast<const i32x4*>(row + (((8 * wave + 4 + q) ^ r) << 4));
      return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    const char* const ss = smem + kS0 + (t / 4 & 1) * S::kS + (t & 3) * 16 + 4 * wave + q;
    auto scale = [&](int row) {
      const int v = *reinterpret_cast<const uint8_t*>(ss + row * 64);
      return in ? v : 0;
    };
    i32x8 x[MT];
    int sx[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int r = XR < 16 ? i % XR : i;  // fewer rows: repeated, the copies' sums are not used
      x[j] = frag(st + S::kW + (16 * j + r) * 512, r);
      sx[j] = scale(16 * (RGT + j) + r);
    }
#pragma unroll
    for (int g = 0; g < RGT; ++g) {
      const i32x8 w = frag(st + (16 * g + i) * 512, i);
      const int sw = scale(16 * g + i);
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[g][j] = mfma_mx8(w, x[j], acc[g][j], sw, sx[j]);
    }
  }
  vm_wait<0>();  // the ring's last loads (zeros) have landed, and every wave has read its last stage
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  floatx4* sums = reinterpret_cast<floatx4*>(smem);
#pragma unroll
  for (int g = 0; g < RGT; ++g)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[((wave * RGT + g) * MT + j) * 64 + lane] = acc[g][j];
  __syncthreads();
  finish_block<RG, MT, SW>(p, sums, seg, m0, M, n0, rows, col0);
}

template <int XR, bool SW>
void launch_ring(const Mx8Args& p, unsigned blocks, hipStream_t st) {
  const dim3 grid(blocks), block(64 * kWaves);
  constexpr int most = (XR <= 8 ? 8 : XR <= 32 ? 6 : 4) / (SW ? 2 : 1);  // groups
  const int rg = (p.r + 15) / 16;
  if (rg == 1) hipLaunchKernelGGL((mx8_ring_kernel<1, XR, SW>), grid, block, 0, st, p);
  else if (rg == 2) hipLaunchKernelGGL((mx8_ring_kernel<2, XR, SW>), grid, block, 0, st, p);
  else if (rg == 3 && most >= 3) hipLaunchKernelGGL((mx8_ring_kernel<most >= 3 ? 3 : 2, XR, SW>), grid, block, 0, st, p);
  else if (rg == 4 && most >= 4) hipLaunchKernelGGL((mx8_ring_kernel<most >= 4 ? 4 : 2, XR, SW>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((mx8_ring_kernel<most >= 6 ? 6 : 2, XR, SW>), grid, block, 0, st, p);
}

template <int RG, bool SW>
void launch_tiles(const Mx8Args& p, unsigned blocks, hipStream_t st) {
  const dim3 block(64 * kWaves);
  if (p.M <= 16)
    hipLaunchKernelGGL((mx8_rows_kernel<RG, 1, SW>), dim3(blocks), block, 0, st, p);
  else if (p.M <= 32)
    hipLaunchKernelGGL((mx8_rows_kernel<RG, 2, SW>), dim3(blocks), block, 0, st, p);
  else
    hipLaunchKernelGGL((mx8_rows_kernel<RG, 4, SW>), dim3(blocks), block, 0, st, p);
}

}  // namespace

namespace q3 {

// Few rows, or rows of which every 64 with up to 64 weight rows (SwiGLU: 32 of each) a block give each CU one block at
// most. What the blocks read is what bounds them, and tiles share more of it, but start slower and a tile alone has a
// CU's share of the loads. One round against tiles, us: 100 rows, N 4096, K 4096 12.6 and 29.7, K 12288 24.5 and 69 (tiles
// of that time), 256 rows, N 4096, K 4096 over weights past the last cache 16.3 and 28. Two rounds, the same: 512 rows 30.2
// and 28.3, N = K = 2048, 640 rows 17.4 and 14.1, 128 rows, N 12288 27.3 and 31.1; with weights in the last cache 512 rows
// 27 and 20.
bool mx8_rows_takes(const Mx8Args& p, bool swiglu) {
  if (p.M <= 64) return true;
  int64_t blocks = 0;
  for (int j = 0; j < p.nseg; ++j) blocks += q3_cdiv(p.n[j], swiglu ? 32 : 64);
  return mx8_rows_ring(p) && blocks * q3_cdiv(p.M, 64) <= 256;
}

int mx8_rows(const Mx8Args& args, bool swiglu, hipStream_t st) {
  Mx8Args p = args;
  int64_t N = 0;
  p.vec = q3_aligned(p.y, 8) && p.ldc % 4 == 0 && (!p.res || (q3_aligned(p.res, 8) && p.ldr % 4 == 0));
  for (int j = 0; j < p.nseg; ++j) {
    p.vec = p.vec && (j == 0 || N % 4 == 0);
    N += p.n[j];
  }
  auto blocks = [&](int rows) {
    int64_t n = 0;
    for (int j = 0; j < p.nseg; ++j) n += q3_cdiv(p.n[j], rows);
    return n;
  };
  if (mx8_rows_ring(p)) {
    // The fewest rows a block (whole 8-byte pieces of y, or whole blocks of 32 in eight bits) that give every CU one block,
    // or an equal number of them where even the largest block does not cover N. One row of K 4096, us by rows a block:
    // N 12288 13.2 (48), 24576 24.9, 25.6, 26.3 and 23.1 (16, 32, 64, 96), 49152 45.1, 44.8, 46.1 and 43.1; 32 rows, N
    // 49152 77.9, 57.5, 49.6 and 49.2. (N 151936 would be 8 % faster in blocks of 32, two on a CU: 121 against 131.)
    // Measured for bf16 outputs; whole blocks of 32 fill the CUs less evenly. SwiGLU of K 4096 in bf16 and in eight bits,
    // us: one row, N 9728 18.1 (244 blocks of 40) and 20.9 (152 of 64), N 12288 21.1 (256 of 48) and 22.9 (192 of 64), N
    // 22016 34.8 (501 of 44) and 40.5 (344 of 64); 32 rows 20.6 and 24.6 (304 of 32), 23.0 and 27.0 (384 of 32), 38.5 and 40.8.
    const int unit = p.yc ? 32 : 4;
    int most = 16 * (p.M <= 8 ? (swiglu ? 4 : 6) : p.M <= 32 ? (swiglu ? 3 : 6) : swiglu ? 2 : 4);
    most = most / unit * unit;
    const int64_t parts = q3_cdiv(p.M, 64), rounds = q3_cdiv(N * parts, 256 * most);
    int r = unit;
    while (r < most && blocks(r) * parts > 256 * rounds) r += unit;
    p.r = r;
    Q3_REQUIRE(mx8_grid_ok(blocks(r) * parts, 64 * kWaves), Q3_ERR_UNSUPPORTED);
    const unsigned n = (unsigned)(blocks(r) * parts);
    if (swiglu) {
      if (p.M <= 8) launch_ring<8, true>(p, n, st);
      else if (p.M <= 16) launch_ring<16, true>(p, n, st);
      else if (p.M <= 32) launch_ring<32, true>(p, n, st);
      else launch_ring<64, true>(p, n, st);
    } else {
      if (p.M <= 8) launch_ring<8, false>(p, n, st);
      else if (p.M <= 16) launch_ring<16, false>(p, n, st);
      else if (p.M <= 32) launch_ring<32, false>(p, n, st);
      else launch_ring<64, false>(p, n, st);
    }
    Q3_LAUNCH_CHECK();
    return Q3_OK;
  }
  // 32 weight rows a block where the output's blocks of 32 ask for it, or where that still gives every CU two blocks.
  const bool wide = p.yc || blocks(32) >= 512;
  Q3_REQUIRE(mx8_grid_ok(blocks(wide ? 32 : 16), 64 * kWaves), Q3_ERR_UNSUPPORTED);
  const unsigned n = (unsigned)blocks(wide ? 32 : 16);
  if (swiglu) {
    if (wide) launch_tiles<2, true>(p, n, st);
    else launch_tiles<1, true>(p, n, st);
  } else {
    if (wide) launch_tiles<2, false>(p, n, st);
    else launch_tiles<1, false>(p, n, st);
  }
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // namespace q3

// Products of MXFP8 rows with MXFP8 weights by whole weight rows, 64 rows of x at a
// time (format and matrix instruction: mxfp8.h):
//   y = act(x w^T (+ bias)) (+ residual),  y = silu(x g^T) * (x u^T)
// over one weight, or the weights of several projections side by side; y in bf16 or in
// eight bits again.
//
// A block owns 16 or 32 weight rows and all of k, so no sums pass between blocks: its
// four waves take every fourth 128 k each and their sums meet in LDS, in wave order. The
// weight is the instruction's first operand, so lane l holds columns 4 (l / 16) .. + 3 of
// y's row l % 16.
#include "gemm_tile.h"
#include "mxfp8.h"

namespace {

using namespace q3;

constexpr int kWaves = 4;

// RG: 16-row groups of weights (SwiGLU: of each of the two), MT: 16-row tiles of x.
template <int RG, int MT, bool SW>
__global__ __launch_bounds__(64 * kWaves) void mx8_rows_kernel(const Mx8Args p) {
  constexpr int RGT = SW ? 2 * RG : RG;
  __shared__ floatx4 sums[kWaves * RGT * MT * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, q = lane >> 4;
  int seg = 0, b = blockIdx.x, col0 = 0;  // weight, its block, the column of y at which it starts
#pragma unroll
  for (int j = 0; j + 1 < kMx8Segments; ++j) {
    const int nb = (p.n[j] + 16 * RG - 1) / (16 * RG);
    if (seg == j && j + 1 < p.nseg && b >= nb) b -= nb, col0 += p.n[j], seg = j + 1;
  }
  seg = __builtin_amdgcn_readfirstlane(seg);
  const int n0 = b * 16 * RG, rows = min(16 * RG, p.n[seg] - n0), K = p.K, kb = K / kMx8Block;
  const int m0 = blockIdx.y * 16 * MT, M = min(p.M - m0, 16 * MT);

  __amdgpu_buffer_rsrc_t rw[2], rs[2];
#pragma unroll
  for (int u = 0; u < (SW ? 2 : 1); ++u) {
    rw[u] = make_rsrc(p.w[SW ? u : seg] + (int64_t)n0 * K, (int64_t)rows * K);
    rs[u] = make_rsrc(p.ws[SW ? u : seg] + (int64_t)n0 * kb, (int64_t)rows * kb);
  }
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (int64_t)m0 * K, (int64_t)M * K);
  const __amdgpu_buffer_rsrc_t rxs = make_rsrc(p.xs + (int64_t)m0 * kb, (int64_t)M * kb);

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

  // Four columns of a row per lane; the eight lanes of 32 columns are neighbours.
  for (int it = tid; it < RG * MT * 64; it += 64 * kWaves) {
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
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= left) break;
      if (!SW) {
        if (p.bias[seg]) v[e] += bf2f(p.bias[seg][n + e]);
        v[e] = mx8_act(v[e], p.act);
      }
      if (p.res) v[e] += bf2f(p.res[row * p.ldr + col + e]);
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
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) p.y[row * p.ldc + col + e] = f2bf(v[e]);
    }
  }
}

template <int RG, bool SW>
void launch_tiles(const Mx8Args& p, unsigned blocks, hipStream_t st) {
  const dim3 block(64 * kWaves);
  if (p.M <= 16)
    hipLaunchKernelGGL((mx8_rows_kernel<RG, 1, SW>), dim3(blocks), block, 0, st, p);
  else if (p.M <= 32)
    hipLaunchKernelGGL((mx8_rows_kernel<RG, 2, SW>), dim3(blocks), block, 0, st, p);
  else
    hipLaunchKernelGGL((mx8_rows_kernel<RG, 4, SW>), dim3(blocks, (unsigned)q3_cdiv(p.M, 64)), block, 0, st, p);
}

}  // namespace

namespace q3 {

int mx8_rows(const Mx8Args& p, bool swiglu, hipStream_t st) {
  auto blocks = [&](int rows) {
    int64_t n = 0;
    for (int j = 0; j < p.nseg; ++j) n += q3_cdiv(p.n[j], rows);
    return (unsigned)n;
  };
  // 32 weight rows a block where the output's blocks of 32 ask for it, or where that still gives every CU two blocks.
  const bool wide = p.yc || blocks(32) >= 512;
  if (swiglu) {
    if (wide) launch_tiles<2, true>(p, blocks(32), st);
    else launch_tiles<1, true>(p, blocks(16), st);
  } else {
    if (wide) launch_tiles<2, false>(p, blocks(32), st);
    else launch_tiles<1, false>(p, blocks(16), st);
  }
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // namespace q3

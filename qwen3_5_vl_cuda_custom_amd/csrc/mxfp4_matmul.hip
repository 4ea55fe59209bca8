// Products with MXFP4 weights (format: mxfp4.h): y = x w^T (+ bias) (+ residual), x
// and y bf16, w (N, K) codes and scales, fp32 accumulation, one rounding. The
// weights enter the matrix cores as their exact values in bf16, x as it is.
#include <algorithm>

#include "gemm_tile.h"
#include "mxfp4.h"

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
};

__device__ __forceinline__ void store_y(const MxGemm& p, int m, int n, float v) {
  if (p.bias) v += bf2f(p.bias[n]);
  if (p.res) v += bf2f(p.res[m * p.ldr + n]);
  p.y[m * p.ldc + n] = f2bf(v);
}

// ------------------------------------------------------------------ few rows (decode)
// Bound by the weight stream. A wave takes RT groups of 16 weight rows and every
// eighth 128-value step of its block's k range: lane (r = l % 16, g = l / 16) loads
// the 16 bytes of block 4 step + g of weight row r, one scale, and the 32 values of
// x's row r at the same k (MT tiles of 16 rows), and forms 4 products of 16x16x32
// per tile pair (k permuted alike in both). The eight waves' sums meet in LDS, in
// wave order.
constexpr int kGemvWaves = 8;

template <int MT, int RT>
__global__ __launch_bounds__(64 * kGemvWaves) void mx_gemv_kernel(const MxGemm p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * RT);
  const int blocks = p.K / kMxBlock, steps = (blocks + 3) / 4;
  const int t0 = (int)((int64_t)steps * blockIdx.y / gridDim.y), t1 = (int)((int64_t)steps * (blockIdx.y + 1) / gridDim.y);

  struct Step {
    u32x4 w[RT];
    uint32_t s[RT];
    bf16x8 x[MT][4];
  };
  auto load = [&](int t, Step& d) {
    const int kb = 4 * t + g;
    const bool in = kb < blocks && t < t1;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t n = min(n0 + 16 * i + r, p.N - 1);
      d.w[i] = u32x4{};
      d.s[i] = 0;
      if (in) {
        d.w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.w + n * p.ldw + kb * 16));
        d.s[i] = p.s[n * p.lds + kb];
      }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int m = 16 * j + r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d.x[j][e] = bf16x8{};
        if (in && m < p.M) d.x[j][e] = *reinterpret_cast<const bf16x8*>(p.x + m * p.ldx + kb * 32 + 8 * e);
      }
    }
  };
  floatx4 acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = floatx4{};
  Step cur, nxt;
  load(t0 + wave, cur);
  for (int t = t0 + wave; t < t1; t += kGemvWaves) {
    load(t + kGemvWaves, nxt);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const float s = mx_scale(cur.s[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bf16x8 w = mx_bf16x8(cur.w[i][e], s);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma16x16x32(w, cur.x[j][e], acc[i][j]);
      }
    }
    cur = nxt;
  }

  __shared__ floatx4 s_acc[kGemvWaves][RT * MT][64];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) s_acc[wave][i * MT + j][lane] = acc[i][j];
  __syncthreads();
  for (int q = wave; q < RT * MT; q += kGemvWaves) {
    floatx4 v = s_acc[0][q][lane];
#pragma unroll
    for (int k = 1; k < kGemvWaves; ++k) v += s_acc[k][q][lane];
    const int m = 16 * (q % MT) + r, n = n0 + 16 * (q / MT) + 4 * g;
    if (m >= p.M) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= p.N) break;
      if (p.part)
        p.part[((int64_t)blockIdx.y * p.M + m) * p.N + n + e] = v[e];
      else
        store_y(p, m, n + e, v[e]);
    }
  }
}

// y from the k ranges' sums, added in their order.
__global__ __launch_bounds__(256) void mx_gemv_sum_kernel(const MxGemm p, int parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, mn = (int64_t)p.M * p.N;
  if (i >= mn) return;
  float v = 0.f;
  for (int k = 0; k < parts; ++k) v += p.part[k * mn + i];
  store_y(p, (int)(i / p.N), (int)(i % p.N), v);
}

constexpr int64_t kGemvMaxRows = 32;

struct GemvPlan {
  int rt, parts;
};

GemvPlan gemv_plan(int64_t M, int64_t N, int64_t K) {
  GemvPlan g{M > 4 ? 4 : 1, 1};
  const int64_t tiles = q3_cdiv(N, 16 * g.rt), steps = q3_cdiv(K, 128);
  while (tiles * g.parts < 256 && steps / (2 * g.parts) >= kGemvWaves && g.rt > 1) g.parts *= 2;
  return g;
}

}  // namespace

extern "C" {

int64_t q3_matmul_mxfp4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (M > kGemvMaxRows) return N * K * 2;  // the weights in bf16
  const GemvPlan g = gemv_plan(M, N, K);
  return g.parts > 1 ? g.parts * M * N * (int64_t)sizeof(float) : 0;
}

int q3_matmul_mxfp4(const void* x, const void* w_codes, const void* w_scales, const void* bias, const void* residual,
                    void* y, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t lds, int64_t ldr,
                    int64_t ldc, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  Q3_REQUIRE(x && w_codes && w_scales && y, Q3_ERR_NULL);
  Q3_REQUIRE(M >= 0 && N >= 0 && K >= kMxBlock && K % kMxBlock == 0, Q3_ERR_SHAPE);
  Q3_REQUIRE(M < (1ll << 31) && N < (1ll << 31) - 256 && K < (1ll << 30), Q3_ERR_SHAPE);
  Q3_REQUIRE(ldx >= K && ldw >= K / 2 && lds >= K / kMxBlock && ldc >= N && (!residual || ldr >= N), Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16, Q3_ERR_DTYPE);
  if (M == 0 || N == 0) return Q3_OK;
  Q3_REQUIRE(q3_aligned(x, 16) && q3_aligned(w_codes, 16) && ldx % 8 == 0 && ldw % 16 == 0, Q3_ERR_ALIGN);
  const int64_t need = q3_matmul_mxfp4_workspace_bytes(M, N, K);
  Q3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Q3_ERR_WORKSPACE);
  Q3_REQUIRE(need == 0 || q3_aligned(workspace, 16), Q3_ERR_ALIGN);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (M > kGemvMaxRows) {
    Q3_REQUIRE(ldw == K / 2 && lds == K / kMxBlock, Q3_ERR_UNSUPPORTED);
    const int rc = mx_expand(w_codes, w_scales, static_cast<bf16*>(workspace), N * K, st);
    if (rc != Q3_OK) return rc;
    return q3_matmul(x, workspace, bias, residual, y, M, N, K, ldx, K, ldr, ldc, dtype, nullptr, 0, stream);
  }
  const GemvPlan g = gemv_plan(M, N, K);
  MxGemm p{static_cast<const bf16*>(x), static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales),
           static_cast<const bf16*>(bias), static_cast<const bf16*>(residual), static_cast<bf16*>(y),
           g.parts > 1 ? static_cast<float*>(workspace) : nullptr, (int)M, (int)N, (int)K, ldx, ldw, lds, ldr, ldc};
  const dim3 grid((unsigned)q3_cdiv(N, 16 * g.rt), (unsigned)g.parts), block(64 * kGemvWaves);
  if (g.rt == 1)
    hipLaunchKernelGGL((mx_gemv_kernel<1, 1>), grid, block, 0, st, p);
  else if (M <= 16)
    hipLaunchKernelGGL((mx_gemv_kernel<1, 4>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((mx_gemv_kernel<2, 4>), grid, block, 0, st, p);
  Q3_LAUNCH_CHECK();
  if (g.parts > 1) {
    hipLaunchKernelGGL(mx_gemv_sum_kernel, dim3((unsigned)q3_cdiv(M * N, 256)), dim3(256), 0, st, p, g.parts);
    Q3_LAUNCH_CHECK();
  }
  return Q3_OK;
}

}  // extern "C"

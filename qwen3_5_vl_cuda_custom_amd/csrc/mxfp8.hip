// MXFP8 rows: quantisation, back to bf16 / fp32, and the RMSNorm of a sum whose
// output is in eight bits. The format and its arithmetic: mxfp8.h.
//
// All are bound by memory: eight values (a 16-byte load of bf16, 8 bytes of
// codes) per lane and piece, so the four lanes of a block exchange their largest
// magnitude with two lane shuffles and nothing but a row's sum goes through LDS.
// The norm with its sum of 16384 x 4096 bf16 takes 84 us over inputs past the last cache
// (472 MB, 5.6 TB/s), 77 where part of them stays in it, one row 2.8, 777 rows of 2048
// fp32 values 3.8; rows of more than 8192 values, whose kernel reads them twice (the
// second time from the caches in part), 4096 x 12288 86 us (354 MB, 4.1 TB/s). Back to
// bf16 16384 x 4096 31 us (203 MB); 1000 x 4096 bf16 to eight bits 4.3 (3.1 out of the
// last cache), as columns of wider rows 4.5; 16384 rows 32.8 and 34.8.
#include "mxfp8.h"

namespace {

using namespace q3;

// Pieces of eight values a lane has in flight. With 1, 2 and 4, us: 32 rows of 4096 bf16 to eight bits 2.3, 2.4, 3.0, 1000
// rows 3.3, 3.3, 3.8, 16384 rows 30.3, 29.4, 30.3; back, 4096 rows 9.0, 6.5, 6.9.
constexpr int kPieces = 2;

// x: rows of 8 cols8 values, ldx apart (CONTIG: no gap, piece i is values [8i, 8i + 8)).
template <typename T, bool CONTIG>
__global__ __launch_bounds__(256) void mx8_quantize_kernel(const T* __restrict__ x, u32x2* __restrict__ codes,
                                                           uint8_t* __restrict__ scales, int64_t pieces, int cols8,
                                                           int64_t ldx) {
  const int64_t base = (int64_t)blockIdx.x * (256 * kPieces) + threadIdx.x;
  float v[kPieces][8];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    // the pieces of a block are whole lane groups: past the end all four repeat the last one's block
    const int64_t i = min(base + u * 256, pieces - 4 + (threadIdx.x & 3));
    const T* p = CONTIG ? x + i * 8 : x + (i / cols8) * ldx + (i % cols8) * 8;
    mx8_load8<T>(p, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t i = base + u * 256;
    uint32_t byte;
    const u32x2 c = mx8_quantize8(v[u], byte);
    if (i < pieces) {
      codes[i] = c;
      if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void mx8_dequantize_kernel(const u32x2* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, T* __restrict__ y,
                                                             int64_t pieces) {
  const int64_t base = (int64_t)blockIdx.x * (256 * kPieces) + threadIdx.x;
  u32x2 c[kPieces];
  uint32_t b[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t i = min(base + u * 256, pieces - 1);
    c[u] = codes[i];
    b[u] = scales[i >> 2];
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t i = base + u * 256;
    if (i >= pieces) return;
    const float s = mx8_scale(b[u]);
    if constexpr (sizeof(T) == 2) {
      bf16x8 v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[u][h], s, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[u][h], s, true);
        v[4 * h] = lo[0], v[4 * h + 1] = lo[1], v[4 * h + 2] = hi[0], v[4 * h + 3] = hi[1];
      }
      __builtin_nontemporal_store(v, reinterpret_cast<bf16x8*>(y) + i);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        floatx4 v;
        v[0] = __builtin_amdgcn_cvt_scalef32_f32_fp8((int)c[u][h], s, 0);
        v[1] = __builtin_amdgcn_cvt_scalef32_f32_fp8((int)c[u][h], s, 1);
        v[2] = __builtin_amdgcn_cvt_scalef32_f32_fp8((int)c[u][h], s, 2);
        v[3] = __builtin_amdgcn_cvt_scalef32_f32_fp8((int)c[u][h], s, 3);
        __builtin_nontemporal_store(v, reinterpret_cast<floatx4*>(y) + 2 * i + h);
      }
    }
  }
}

struct NormArgs {
  const void *x, *r, *w;  // rows ldx and ldr apart (r may be null), weight (8 cols8)
  void* h;                // the sum, packed, where there is an r
  u32x2* codes;           // packed
  uint8_t* scales;
  int64_t first, ldx, ldr;  // the launch's first row
  int cols8;              // pieces of a row, a multiple of four
  float eps;
};

// h = x + r, rounded to T as a stored sum is; y = h / sqrt(mean(h^2) + eps) * w in
// fp32, quantised from there. A block of 256 threads per row. P > 0: a thread's P
// pieces (t, t + 256, ...) stay in registers; P = 0, any length: the row is read twice.
template <typename T, int P>
__global__ __launch_bounds__(256) void mx8_norm_kernel(const NormArgs a) {
  __shared__ float sums[4];
  const int64_t row = a.first + blockIdx.x;
  const int t = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.ldr : nullptr;
  const T* w = static_cast<const T*>(a.w);
  T* h = a.h ? static_cast<T*>(a.h) + row * a.cols8 * 8 : nullptr;
  u32x2* codes = a.codes + row * a.cols8;
  uint8_t* scales = a.scales + row * (a.cols8 / 4);

  auto load = [&](int i, float (&v)[8]) {
    mx8_load8<T>(x + 8 * i, v);
    if (r) {
      float u[8];
      mx8_load8<T>(r + 8 * i, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = to_f<T>(from_f<T>(v[e] + u[e]));
    }
  };
  auto finish = [&](int i, const float (&v)[8], const float (&g)[8], float rstd) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = v[e] * rstd * g[e];
    uint32_t byte;
    const u32x2 c = mx8_quantize8(y, byte);
    if (i < a.cols8) {
      codes[i] = c;
      if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
  };
  auto total = [&](float s) {
    s = wave_sum(s);
    if ((t & 63) == 0) sums[t >> 6] = s;
    __syncthreads();
    return sums[0] + sums[1] + sums[2] + sums[3];
  };
  const int blocks = (a.cols8 + 255) / 256;  // pieces of a thread
  // past the row's end the four lanes of a block all repeat the last block's pieces
  auto piece = [&](int u) { return min(t + 256 * u, a.cols8 - 4 + (t & 3)); };

  float s = 0.f;
  if constexpr (P > 0) {
    float v[P][8], g[P][8];
#pragma unroll
    for (int u = 0; u < P; ++u) {
      load(piece(u), v[u]);
      mx8_load8<T>(w + 8 * piece(u), g[u]);
    }
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const bool in = t + 256 * u < a.cols8;
      if (in && h) mx8_store8<T>(h + 8 * (t + 256 * u), v[u]);
      float q = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) q += v[u][e] * v[u][e];
      s += in ? q : 0.f;
    }
    const float rstd = rsqrtf(total(s) / (float)(a.cols8 * 8) + a.eps);
#pragma unroll
    for (int u = 0; u < P; ++u) finish(t + 256 * u, v[u], g[u], rstd);
  } else {
    for (int u = 0; u < blocks; ++u) {
      const int i = t + 256 * u;
      float v[8];
      if (i >= a.cols8) break;
      load(i, v);
      if (h) mx8_store8<T>(h + 8 * i, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e] * v[e];
    }
    const float rstd = rsqrtf(total(s) / (float)(a.cols8 * 8) + a.eps);
    for (int u = 0; u < blocks; ++u) {
      float v[8], g[8];
      load(piece(u), v);
      mx8_load8<T>(w + 8 * piece(u), g);
      finish(t + 256 * u, v, g, rstd);
    }
  }
}

// Rows of one launch (a block of 256 threads each).
constexpr int64_t kLaunchRows = (1 << 24) - 1;

template <typename T>
void launch_norm(const NormArgs& a, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)rows), block(256);
  const int p = (a.cols8 + 255) / 256;
  if (p <= 1) hipLaunchKernelGGL((mx8_norm_kernel<T, 1>), grid, block, 0, st, a);
  else if (p <= 2) hipLaunchKernelGGL((mx8_norm_kernel<T, 2>), grid, block, 0, st, a);
  else if (p <= 4) hipLaunchKernelGGL((mx8_norm_kernel<T, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((mx8_norm_kernel<T, 0>), grid, block, 0, st, a);
}

}  // namespace

extern "C" {

int q3_mxfp8_quantize(const void* x, void* codes, void* scales, int64_t rows, int64_t cols, int64_t ldx, int dtype,
                      void* stream) {
  Q3_REQUIRE(x && codes && scales, Q3_ERR_NULL);
  Q3_REQUIRE(rows >= 0 && cols >= 0 && cols % kMx8Block == 0 && cols < (1ll << 31) && ldx >= cols, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F32, Q3_ERR_DTYPE);
  const int64_t size = dtype == Q3_BF16 ? 2 : 4;
  Q3_REQUIRE(q3_aligned(x, 16) && ldx * size % 16 == 0 && q3_aligned(codes, 8), Q3_ERR_ALIGN);
  if (rows == 0 || cols == 0) return Q3_OK;
  const int64_t pieces = rows * (cols / 8), blocks = q3_cdiv(pieces, 256 * kPieces);
  Q3_REQUIRE(mx8_grid_ok(blocks, 256), Q3_ERR_UNSUPPORTED);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(256);
  u32x2* c = static_cast<u32x2*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  const int cols8 = (int)(cols / 8);
  const bool contig = ldx == cols || rows == 1;
  if (dtype == Q3_BF16) {
    const bf16* p = static_cast<const bf16*>(x);
    if (contig) hipLaunchKernelGGL((mx8_quantize_kernel<bf16, true>), grid, block, 0, st, p, c, s, pieces, cols8, ldx);
    else hipLaunchKernelGGL((mx8_quantize_kernel<bf16, false>), grid, block, 0, st, p, c, s, pieces, cols8, ldx);
  } else {
    const float* p = static_cast<const float*>(x);
    if (contig) hipLaunchKernelGGL((mx8_quantize_kernel<float, true>), grid, block, 0, st, p, c, s, pieces, cols8, ldx);
    else hipLaunchKernelGGL((mx8_quantize_kernel<float, false>), grid, block, 0, st, p, c, s, pieces, cols8, ldx);
  }
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

int q3_mxfp8_dequantize(const void* codes, const void* scales, void* y, int64_t n, int dtype, void* stream) {
  Q3_REQUIRE(codes && scales && y, Q3_ERR_NULL);
  Q3_REQUIRE(n >= 0 && n % kMx8Block == 0, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F32, Q3_ERR_DTYPE);
  Q3_REQUIRE(q3_aligned(codes, 8) && q3_aligned(y, 16), Q3_ERR_ALIGN);
  if (n == 0) return Q3_OK;
  const int64_t pieces = n / 8, blocks = q3_cdiv(pieces, 256 * kPieces);
  Q3_REQUIRE(mx8_grid_ok(blocks, 256), Q3_ERR_UNSUPPORTED);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(256);
  const u32x2* c = static_cast<const u32x2*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (dtype == Q3_BF16)
    hipLaunchKernelGGL((mx8_dequantize_kernel<bf16>), grid, block, 0, st, c, s, static_cast<bf16*>(y), pieces);
  else
    hipLaunchKernelGGL((mx8_dequantize_kernel<float>), grid, block, 0, st, c, s, static_cast<float*>(y), pieces);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

int q3_add_rmsnorm_mxfp8(const void* x, const void* residual, const void* weight, void* sum, void* codes, void* scales,
                         int64_t rows, int64_t cols, int64_t ldx, int64_t ldr, float eps, int dtype, void* stream) {
  Q3_REQUIRE(x && weight && codes && scales && (!residual == !sum), Q3_ERR_NULL);
  Q3_REQUIRE(rows >= 0 && cols >= kMx8Block && cols % kMx8Block == 0 && ldx >= cols && (!residual || ldr >= cols),
             Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F32, Q3_ERR_DTYPE);
  Q3_REQUIRE(rows < (1ll << 31) && cols < (1 << 24), Q3_ERR_UNSUPPORTED);
  const int64_t size = dtype == Q3_BF16 ? 2 : 4;
  Q3_REQUIRE(q3_aligned(x, 16) && ldx * size % 16 == 0 && q3_aligned(residual, 16) && (!residual || ldr * size % 16 == 0) &&
                 q3_aligned(weight, 16) && q3_aligned(sum, 16) && q3_aligned(codes, 8),
             Q3_ERR_ALIGN);
  if (rows == 0) return Q3_OK;
  NormArgs a{};
  a.x = x, a.r = residual, a.w = weight, a.h = sum;
  a.codes = static_cast<u32x2*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.ldx = ldx, a.ldr = ldr;
  a.cols8 = (int)(cols / 8);
  a.eps = eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (a.first = 0; a.first < rows; a.first += kLaunchRows) {
    const int64_t n = std::min(kLaunchRows, rows - a.first);
    if (dtype == Q3_BF16) launch_norm<bf16>(a, n, st);
    else launch_norm<float>(a, n, st);
    Q3_LAUNCH_CHECK();
  }
  return Q3_OK;
}

}  // extern "C"

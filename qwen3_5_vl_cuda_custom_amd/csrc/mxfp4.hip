// MXFP4 rows: quantisation, back to bf16 / fp32, and the write of new key and
// value rows into a 4-bit KV cache. The format and its arithmetic: mxfp4.h.
//
// All three are bound by memory: eight values (a 16-byte load or store of bf16,
// 4 bytes of codes) per lane and piece, so the four lanes of a block exchange
// their largest magnitude with two lane shuffles and nothing goes through LDS. A lane has
// four pieces in flight where rows are long. Measured: quantising 12288 x 4096 fp32 40 us
// (228 MB, 5.7 TB/s), back to bf16 20 us (127 MB, 6.4 TB/s); 256 x 128 bf16 2.6 and 2.4 us;
// writing 4 x 512 new rows of 8 heads x 128 (K and V) 5.9 us, one row 1.9 us.
#include "mxfp4.h"

namespace {

using namespace q3;

// Pieces of eight values a lane has in flight.
constexpr int kPieces = 4;

// x: rows of `cols` values, ldx apart (CONTIG: no gap, piece i is values [8i, 8i + 8)).
template <typename T, bool CONTIG>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, uint32_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, int64_t pieces, int cols8,
                                                          int64_t ldx) {
  const int64_t base = (int64_t)blockIdx.x * (256 * kPieces) + threadIdx.x;
  float v[kPieces][8];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    // the pieces of a block are whole lane groups: past the end all four repeat the last one's block
    const int64_t i = min(base + u * 256, pieces - 4 + (threadIdx.x & 3));
    const T* p = CONTIG ? x + i * 8 : x + (i / cols8) * ldx + (i % cols8) * 8;
    mx_load8<T>(p, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t i = base + u * 256;
    uint32_t byte;
    const uint32_t c = mx_quantize8(v[u], byte);
    if (i < pieces) {
      codes[i] = c;
      if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
  }
}

struct ExpandArgs {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  void* y;
  int n0, n1;           // planes (i, j) of each source, at i * stride + j * stride bytes
  int64_t cst[2][2], sst[2][2];
  int64_t run;          // values of a plane; y is (source, n0, n1, run)
  const int* lens;      // if set: plane (i, j) of `run` values has lens[i] + len_add rows of `row` values in use
  int len_add;
  int64_t row;
};

// K's and V's caches in one launch (grid z), rows in use only.
template <typename T>
__global__ __launch_bounds__(256) void mx_expand_kernel(const ExpandArgs a) {
  const int plane = blockIdx.y, i0 = plane / a.n1, i1 = plane - i0 * a.n1, kv = blockIdx.z;
  int64_t end = a.run, used = a.run, fresh = a.run;
  if (a.lens) {
    fresh = max((int64_t)a.lens[i0], (int64_t)0) * a.row >> 3;
    const int64_t rows = max((int64_t)a.lens[i0] + a.len_add, (int64_t)0);
    used = min(a.run, rows * a.row);
    end = min(a.run, (rows + 63) / 64 * 64 * a.row);
  }
  const int64_t pieces = end >> 3, last = (used >> 3) - 1;
  const int64_t base = (int64_t)blockIdx.x * (256 * kPieces) + threadIdx.x;
  if (base - threadIdx.x >= pieces) return;
  const uint32_t* c = reinterpret_cast<const uint32_t*>((kv ? a.codes[1] : a.codes[0]) + i0 * (kv ? a.cst[1][0] : a.cst[0][0]) +
                                                        i1 * (kv ? a.cst[1][1] : a.cst[0][1]));
  const uint8_t* s = (kv ? a.scales[1] : a.scales[0]) + i0 * (kv ? a.sst[1][0] : a.sst[0][0]) +
                     i1 * (kv ? a.sst[1][1] : a.sst[0][1]);
  T* o = static_cast<T*>(a.y) + ((int64_t)kv * a.n0 * a.n1 + plane) * a.run;
  uint32_t w[kPieces], b[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t i = base + u * 256;
    w[u] = b[u] = 0;
    if (i <= last) {
      w[u] = c[i];
      b[u] = s[i >> 2];
      if (kv && b[u] == 255 && i >= fresh) w[u] = b[u] = 0;
    }
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const int64_t i = base + u * 256;
    if (i >= pieces) return;
    const bf16x8 v = mx_bf16x8(w[u], mx_scale(b[u]));
    if constexpr (sizeof(T) == 2) {
      // past the L2 (12288 x 4096 there and back 68 -> 61 us; the same for codes or loads was slower)
      __builtin_nontemporal_store(v, reinterpret_cast<bf16x8*>(o) + i);
    } else {
      floatx4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = bf2f(v[e]);
        hi[e] = bf2f(v[4 + e]);
      }
      reinterpret_cast<floatx4*>(o)[2 * i] = lo;
      reinterpret_cast<floatx4*>(o)[2 * i + 1] = hi;
    }
  }
}

int launch_expand(const ExpandArgs& a, int sources, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)q3_cdiv(a.run / 8, 256 * kPieces), (unsigned)(a.n0 * a.n1), (unsigned)sources);
  if (dtype == Q3_BF16)
    hipLaunchKernelGGL((mx_expand_kernel<bf16>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((mx_expand_kernel<float>), grid, dim3(256), 0, st, a);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

struct AppendArgs {
  const void* x[2];        // k, v: (B, S, Hkv, D)
  uint8_t* codes[2];       // (B, Hkv, cap, D / 2), rows packed
  uint8_t* scales[2];      // (B, Hkv, cap, D / 32), rows packed
  int64_t xs[2][3];        // (b, s, h) strides, elements
  int64_t cst[2][2], sst[2][2];  // (b, h) strides, bytes
  const int* lens;
  int S, Hkv, D8;
  int64_t cap;
  int64_t pieces;  // B * S * 2 * Hkv * D / 8
};

// One piece per lane, ordered (token, k | v, head, piece of the row): a row is
// D / 8 lanes, a multiple of four, so a block's lanes are neighbours. I: the type
// that the pieces are counted in; 64 bits where 32 do not hold them (a whole cache
// of 34 GB quantised at once), as their divisions cost several times as much.
template <typename T, typename I>
__global__ __launch_bounds__(256) void mx_append_kernel(const AppendArgs a) {
  const int64_t t = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
  const I i = (I)min(t, a.pieces - 4 + (threadIdx.x & 3));
  I r = i / (uint32_t)a.D8;
  const uint32_t j = (uint32_t)(i % (uint32_t)a.D8);
  const uint32_t h = (uint32_t)(r % (uint32_t)a.Hkv);
  r /= (uint32_t)a.Hkv;
  const int kv = (int)(r & 1);
  r >>= 1;
  const uint32_t s = (uint32_t)(r % (uint32_t)a.S), b = (uint32_t)(r / (uint32_t)a.S);
  const T* x = static_cast<const T*>(kv ? a.x[1] : a.x[0]);
  float v[8];
  mx_load8<T>(x + b * (kv ? a.xs[1][0] : a.xs[0][0]) + s * (kv ? a.xs[1][1] : a.xs[0][1]) +
                  h * (kv ? a.xs[1][2] : a.xs[0][2]) + 8 * j,
              v);
  uint32_t byte;
  const uint32_t c = mx_quantize8(v, byte);
  const int64_t at = (int64_t)a.lens[b] + s;
  if (t >= a.pieces || at < 0 || at >= a.cap) return;
  uint8_t* cp = (kv ? a.codes[1] : a.codes[0]) + b * (kv ? a.cst[1][0] : a.cst[0][0]) +
                h * (kv ? a.cst[1][1] : a.cst[0][1]);
  uint8_t* sp = (kv ? a.scales[1] : a.scales[0]) + b * (kv ? a.sst[1][0] : a.sst[0][0]) +
                h * (kv ? a.sst[1][1] : a.sst[0][1]);
  reinterpret_cast<uint32_t*>(cp)[at * a.D8 + j] = c;
  if ((j & 3) == 0) sp[at * (a.D8 >> 2) + (j >> 2)] = (uint8_t)byte;
}

template <typename T>
void launch_quantize(const void* x, void* codes, void* scales, int64_t rows, int64_t cols, int64_t ldx,
                     hipStream_t st) {
  const int64_t pieces = rows * (cols / 8);
  const dim3 grid((unsigned)q3_cdiv(pieces, 256 * kPieces));
  auto* c = static_cast<uint32_t*>(codes);
  auto* s = static_cast<uint8_t*>(scales);
  if (ldx == cols || rows == 1)
    hipLaunchKernelGGL((mx_quantize_kernel<T, true>), grid, dim3(256), 0, st, static_cast<const T*>(x), c, s, pieces,
                       (int)(cols / 8), ldx);
  else
    hipLaunchKernelGGL((mx_quantize_kernel<T, false>), grid, dim3(256), 0, st, static_cast<const T*>(x), c, s, pieces,
                       (int)(cols / 8), ldx);
}

}  // namespace

namespace q3 {

int mx_expand(const void* codes, const void* scales, bf16* y, int64_t n, hipStream_t st) {
  ExpandArgs a{};
  a.codes[0] = static_cast<const uint8_t*>(codes);
  a.scales[0] = static_cast<const uint8_t*>(scales);
  a.y = y;
  a.n0 = a.n1 = 1;
  a.run = n;
  return launch_expand(a, 1, Q3_BF16, st);
}

int mx_expand_cache(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, bf16* y,
                    int64_t B, int64_t Hkv, int64_t rows, int64_t D, const int64_t* cst, const int64_t* sst,
                    const int* lens, int len_add, hipStream_t st) {
  ExpandArgs a{};
  a.codes[0] = static_cast<const uint8_t*>(k_codes);
  a.codes[1] = static_cast<const uint8_t*>(v_codes);
  a.scales[0] = static_cast<const uint8_t*>(k_scales);
  a.scales[1] = static_cast<const uint8_t*>(v_scales);
  a.y = y;
  a.n0 = (int)B;
  a.n1 = (int)Hkv;
  for (int i = 0; i < 4; ++i) {
    a.cst[i / 2][i % 2] = cst[i];
    a.sst[i / 2][i % 2] = sst[i];
  }
  a.run = rows * D;
  a.lens = lens;
  a.len_add = len_add;
  a.row = D;
  return launch_expand(a, 2, Q3_BF16, st);
}

}  // namespace q3

extern "C" {

int q3_mxfp4_quantize(const void* x, void* codes, void* scales, int64_t rows, int64_t cols, int64_t ldx, int dtype,
                      void* stream) {
  Q3_REQUIRE(x && codes && scales, Q3_ERR_NULL);
  Q3_REQUIRE(rows >= 0 && cols >= 0 && cols % kMxBlock == 0 && cols < (1ll << 31) && ldx >= cols, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F32, Q3_ERR_DTYPE);
  if (rows == 0 || cols == 0) return Q3_OK;
  Q3_REQUIRE(rows <= (1ll << 40) / cols, Q3_ERR_SHAPE);
  const int64_t es = dtype == Q3_BF16 ? 2 : 4;
  Q3_REQUIRE(q3_aligned(x, 16) && q3_aligned(codes, 4) && (rows == 1 || ldx * es % 16 == 0), Q3_ERR_ALIGN);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == Q3_BF16)
    launch_quantize<bf16>(x, codes, scales, rows, cols, ldx, st);
  else
    launch_quantize<float>(x, codes, scales, rows, cols, ldx, st);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

int q3_mxfp4_dequantize(const void* codes, const void* scales, void* y, int64_t n0, int64_t n1, int64_t run,
                        const int64_t* strides, int dtype, void* stream) {
  Q3_REQUIRE(codes && scales && y && strides, Q3_ERR_NULL);
  Q3_REQUIRE(n0 >= 0 && n1 >= 0 && run >= 0 && run % kMxBlock == 0 && run <= (1ll << 40), Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F32, Q3_ERR_DTYPE);
  if (n0 == 0 || n1 == 0 || run == 0) return Q3_OK;
  Q3_REQUIRE(n0 <= 65535 && n1 <= 65535 && n0 * n1 <= 65535, Q3_ERR_UNSUPPORTED);
  Q3_REQUIRE(q3_aligned(codes, 4) && q3_aligned(y, 16) && strides[0] % 4 == 0 && strides[1] % 4 == 0, Q3_ERR_ALIGN);
  ExpandArgs a{};
  a.codes[0] = static_cast<const uint8_t*>(codes);
  a.scales[0] = static_cast<const uint8_t*>(scales);
  a.y = y;
  a.n0 = (int)n0;
  a.n1 = (int)n1;
  for (int i = 0; i < 2; ++i) {
    a.cst[0][i] = strides[i];
    a.sst[0][i] = strides[2 + i];
  }
  a.run = run;
  return launch_expand(a, 1, dtype, static_cast<hipStream_t>(stream));
}

int q3_kv_append_mxfp4(const void* k, const void* v, void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                       const int* kv_lens, int64_t B, int64_t S, int64_t Hkv, int64_t D, int64_t cap,
                       const int64_t* strides, int dtype, void* stream) {
  Q3_REQUIRE(k && v && k_codes && k_scales && v_codes && v_scales && kv_lens && strides, Q3_ERR_NULL);
  Q3_REQUIRE(B >= 0 && S >= 0 && Hkv >= 1 && D >= 1 && cap >= 0, Q3_ERR_SHAPE);
  Q3_REQUIRE(dtype == Q3_BF16 || dtype == Q3_F32, Q3_ERR_DTYPE);
  Q3_REQUIRE(D % kMxBlock == 0 && D <= 256, Q3_ERR_UNSUPPORTED);
  if (B == 0 || S == 0) return Q3_OK;
  Q3_REQUIRE(B < (1ll << 31) && S < (1ll << 31) && Hkv < (1ll << 20) && cap < (1ll << 31), Q3_ERR_SHAPE);
  const int64_t per_token = 2 * Hkv * (D / 8);
  Q3_REQUIRE(B * S < (1ll << 38) / per_token, Q3_ERR_SHAPE);  // the grid: 2^30 blocks
  const int64_t es = dtype == Q3_BF16 ? 2 : 4;
  bool ok = q3_aligned(k, 16) && q3_aligned(v, 16) && q3_aligned(k_codes, 4) && q3_aligned(v_codes, 4);
  for (int i = 0; i < 6; ++i) ok = ok && strides[i] * es % 16 == 0;
  for (int i : {6, 7, 10, 11}) ok = ok && strides[i] % 4 == 0;
  Q3_REQUIRE(ok, Q3_ERR_ALIGN);
  AppendArgs a{};
  a.x[0] = k;
  a.x[1] = v;
  a.codes[0] = static_cast<uint8_t*>(k_codes);
  a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scales[0] = static_cast<uint8_t*>(k_scales);
  a.scales[1] = static_cast<uint8_t*>(v_scales);
  for (int kv = 0; kv < 2; ++kv) {
    for (int i = 0; i < 3; ++i) a.xs[kv][i] = strides[3 * kv + i];
    for (int i = 0; i < 2; ++i) {
      a.cst[kv][i] = strides[6 + 4 * kv + i];
      a.sst[kv][i] = strides[8 + 4 * kv + i];
    }
  }
  a.lens = kv_lens;
  a.S = (int)S;
  a.Hkv = (int)Hkv;
  a.D8 = (int)(D / 8);
  a.cap = cap;
  a.pieces = B * S * per_token;
  const bool wide = a.pieces >= (1ll << 31);
  const int64_t blocks = q3_cdiv(a.pieces, 256);  // a launch has less than 2^32 threads along x
  const dim3 grid((unsigned)(wide ? 1 << 23 : blocks), (unsigned)(wide ? q3_cdiv(blocks, 1 << 23) : 1));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == Q3_BF16 && !wide)
    hipLaunchKernelGGL((mx_append_kernel<bf16, uint32_t>), grid, dim3(256), 0, st, a);
  else if (dtype == Q3_BF16)
    hipLaunchKernelGGL((mx_append_kernel<bf16, uint64_t>), grid, dim3(256), 0, st, a);
  else if (!wide)
    hipLaunchKernelGGL((mx_append_kernel<float, uint32_t>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((mx_append_kernel<float, uint64_t>), grid, dim3(256), 0, st, a);
  Q3_LAUNCH_CHECK();
  return Q3_OK;
}

}  // extern "C"

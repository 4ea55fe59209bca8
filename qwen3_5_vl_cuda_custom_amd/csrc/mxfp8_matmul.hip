// Products of MXFP8 rows with MXFP8 weights: the entry points.
#include "mxfp8.h"
#include "mxfp8_tile.h"

namespace {

using namespace q3;

struct Call {
  Mx8Args a;
  int64_t N = 0;  // columns of y
};

// Arguments of every form but the weights; y or (y_codes, y_scales).
int check(Call& c, const void* x_codes, const void* x_scales, const void* residual, void* y, void* y_codes,
          void* y_scales, int64_t M, int64_t K, int64_t ldr, int64_t ldc, int act) {
  Mx8Args& a = c.a;
  Q3_REQUIRE(x_codes && x_scales && (y ? !y_codes && !y_scales : y_codes && y_scales), Q3_ERR_NULL);
  Q3_REQUIRE(M >= 0 && K >= kMx8Block && K % kMx8Block == 0, Q3_ERR_SHAPE);
  if (y) Q3_REQUIRE(ldc >= c.N, Q3_ERR_SHAPE);
  else Q3_REQUIRE(c.N % kMx8Block == 0, Q3_ERR_SHAPE);
  Q3_REQUIRE(!residual || ldr >= c.N, Q3_ERR_SHAPE);
  Q3_REQUIRE(act >= kMx8None && act <= kMx8Silu, Q3_ERR_UNSUPPORTED);
  Q3_REQUIRE(K < (1 << 23) && c.N < (1ll << 31) - 256 && M < (1ll << 31) - 256, Q3_ERR_UNSUPPORTED);
  Q3_REQUIRE(q3_aligned(x_codes, 16) && q3_aligned(x_scales, 4) && (y || q3_aligned(y_codes, 8)), Q3_ERR_ALIGN);
  a.x = static_cast<const uint8_t*>(x_codes);
  a.xs = static_cast<const uint8_t*>(x_scales);
  a.res = static_cast<const bf16*>(residual);
  a.y = static_cast<bf16*>(y);
  a.yc = static_cast<uint8_t*>(y_codes);
  a.ys = static_cast<uint8_t*>(y_scales);
  a.M = (int)M;
  a.K = (int)K;
  a.act = act;
  a.ldr = ldr;
  a.ldc = y ? ldc : c.N;
  return Q3_OK;
}

int weight(Mx8Args& a, int j, const void* codes, const void* scales, const void* bias, int64_t n) {
  Q3_REQUIRE(codes && scales, Q3_ERR_NULL);
  Q3_REQUIRE(n >= 0 && n < (1ll << 31) - 256, Q3_ERR_SHAPE);
  Q3_REQUIRE(q3_aligned(codes, 16) && q3_aligned(scales, 4), Q3_ERR_ALIGN);
  a.w[j] = static_cast<const uint8_t*>(codes);
  a.ws[j] = static_cast<const uint8_t*>(scales);
  a.bias[j] = static_cast<const bf16*>(bias);
  a.n[j] = (int)n;
  return Q3_OK;
}

int64_t workspace_of(const Mx8Args& a, bool swiglu) { return mx8_rows_takes(a, swiglu) ? 0 : mx8_tile_workspace(a, swiglu); }

int launch(const Call& c, bool swiglu, void* workspace, int64_t workspace_bytes, void* stream) {
  if (c.a.M == 0 || c.N == 0) return Q3_OK;
  const int64_t need = workspace_of(c.a, swiglu);
  Q3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), Q3_ERR_WORKSPACE);
  Q3_REQUIRE(q3_aligned(workspace, 16), Q3_ERR_ALIGN);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return mx8_rows_takes(c.a, swiglu) ? mx8_rows(c.a, swiglu, st) : mx8_tile(c.a, swiglu, workspace, st);
}

// The sizes of a call that there may be, as its form goes by them.
bool sizes(Mx8Args& a, int64_t M, const int64_t* n, int64_t nseg, int64_t K) {
  if (!n || nseg < 1 || nseg > kMx8Segments || M <= 0 || K < kMx8Block || K % kMx8Block) return false;
  int64_t N = 0;
  for (int j = 0; j < nseg; ++j) {
    if (n[j] < 1 || n[j] >= (1ll << 31) - 256) return false;
    a.n[j] = (int)n[j];
    N += n[j];
  }
  if (N >= (1ll << 31) - 256 || M >= (1ll << 31) - 256 || K >= (1 << 23)) return false;
  a.nseg = (int)nseg;
  a.M = (int)M;
  a.K = (int)K;
  return true;
}

}  // namespace

extern "C" {

int64_t q3_matmul_mxfp8_workspace_bytes(int64_t M, const int64_t* n, int64_t nseg, int64_t K, int swiglu) {
  Mx8Args a{};
  return sizes(a, M, n, nseg, K) ? workspace_of(a, swiglu != 0) : 0;
}

int q3_matmul_mxfp8_form(int64_t M, const int64_t* n, int64_t nseg, int64_t K, int swiglu) {
  Mx8Args a{};
  if (!sizes(a, M, n, nseg, K)) return Q3_ERR_SHAPE;
  if (mx8_rows_takes(a, swiglu != 0)) return mx8_rows_ring(a) ? 1 : 0;
  return 2 + mx8_tile_form(a, swiglu != 0);
}

int q3_matmul_mxfp8(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales,
                    const void* bias, const void* residual, void* y, void* y_codes, void* y_scales, int64_t M,
                    int64_t N, int64_t K, int64_t ldr, int64_t ldc, int act, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  Call c{};
  c.N = N;
  if (const int rc = weight(c.a, 0, w_codes, w_scales, bias, N)) return rc;
  c.a.nseg = 1;
  if (const int rc = check(c, x_codes, x_scales, residual, y, y_codes, y_scales, M, K, ldr, ldc, act)) return rc;
  return launch(c, false, workspace, workspace_bytes, stream);
}

int q3_matmul_segments_mxfp8(const void* x_codes, const void* x_scales, const void* const* w_codes,
                             const void* const* w_scales, const void* const* bias, const int64_t* n, int64_t nseg,
                             void* y, int64_t M, int64_t K, int64_t ldc, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  Q3_REQUIRE(w_codes && w_scales && n && y, Q3_ERR_NULL);
  Q3_REQUIRE(nseg >= 1 && nseg <= kMx8Segments, Q3_ERR_SHAPE);
  Call c{};
  for (int j = 0; j < nseg; ++j) {
    Q3_REQUIRE(n[j] >= 1, Q3_ERR_SHAPE);
    if (const int rc = weight(c.a, j, w_codes[j], w_scales[j], bias ? bias[j] : nullptr, n[j])) return rc;
    c.N += n[j];
  }
  c.a.nseg = (int)nseg;
  if (const int rc = check(c, x_codes, x_scales, nullptr, y, nullptr, nullptr, M, K, 0, ldc, kMx8None)) return rc;
  return launch(c, false, workspace, workspace_bytes, stream);
}

int q3_matmul_swiglu_mxfp8(const void* x_codes, const void* x_scales, const void* g_codes, const void* g_scales,
                           const void* u_codes, const void* u_scales, void* y, void* y_codes, void* y_scales,
                           int64_t M, int64_t N, int64_t K, int64_t ldc, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  Call c{};
  c.N = N;
  if (const int rc = weight(c.a, 0, g_codes, g_scales, nullptr, N)) return rc;
  if (const int rc = weight(c.a, 1, u_codes, u_scales, nullptr, N)) return rc;
  c.a.nseg = 1;
  if (const int rc = check(c, x_codes, x_scales, nullptr, y, y_codes, y_scales, M, K, 0, ldc, kMx8None)) return rc;
  return launch(c, true, workspace, workspace_bytes, stream);
}

}  // extern "C"

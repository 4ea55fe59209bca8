// The product of up to 64 rows with MXFP4 weights (mxfp4_rows.hip).
#pragma once

#include "q3_common.h"

namespace q3 {

constexpr int kMxRowsMax = 64;       // rows of x
constexpr int kMxRowsSegments = 4;   // weights side by side

struct MxRows {
  const bf16* x;
  const bf16* nw;  // RMSNorm weight, or null
  float eps;
  const uint8_t *w[kMxRowsSegments], *s[kMxRowsSegments];  // codes and scales (SwiGLU: gate, up)
  const bf16* bias[kMxRowsSegments];
  int n[kMxRowsSegments];       // rows of each weight
  int nseg;
  const bf16* res;
  bf16* y;
  int M, K;
  int64_t ldx, ldw, lds, ldr, ldc;  // ldw, lds in bytes
  // set by mx_rows
  int bstart[kMxRowsSegments], col[kMxRowsSegments];  // first block and column of each weight
  int r, vec;                                         // weight rows of a block; whether y, bias, residual go in 8-byte pieces
};

// Whether the kernel takes a product (K a multiple of 128, whole words of scales).
bool mx_rows_ok(int64_t M, int64_t K, const void* scales, int64_t lds);
int mx_rows(MxRows p, bool swiglu, hipStream_t st);

}  // namespace q3

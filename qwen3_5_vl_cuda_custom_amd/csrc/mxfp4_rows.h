// Products by whole MXFP4 weight rows (mxfp4_rows.hip).
#pragma once

#include "q3_common.h"

namespace q3 {

constexpr int kMxRowsMax = 64;       // rows of x per block
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

// Any M (64 rows per block), K a multiple of 32 below 2^23; of 128 with whole words of scales for several weights,
// SwiGLU and the norm.
int mx_rows(MxRows p, bool swiglu, hipStream_t st);
// Weight rows a block takes.
int64_t mx_rows_per_block(int64_t M, int64_t N, bool swiglu);

}  // namespace q3

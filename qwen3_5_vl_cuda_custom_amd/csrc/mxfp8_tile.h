// Products of many MXFP8 rows (mxfp8_tile.hip).
#pragma once

#include "mxfp8.h"

namespace q3 {

int64_t mx8_tile_workspace(const Mx8Args& a, bool swiglu);
// Tiles of 256 x 256 (0), 128 x 256 (1), 128 x 128 (2), and of the last size with the scales by rows (3).
int mx8_tile_form(const Mx8Args& a, bool swiglu);
// workspace: mx8_tile_workspace bytes, 16-byte aligned.
int mx8_tile(const Mx8Args& a, bool swiglu, void* workspace, hipStream_t st);

}  // namespace q3

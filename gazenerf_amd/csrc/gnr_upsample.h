// gnr_upsample.h -- what the 8-bit upsampler (gnr_upsample8.hip) shares with the fp32 one (gnr_upsample.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/gnr.h"

namespace gnr {

struct UpDims {
    int n_blocks, ch[GNR_UPSAMPLE_MAX_BLOCKS + 1], side[GNR_UPSAMPLE_MAX_BLOCKS + 1];
};
int up_dims(const GnrUpsampleProblem* p, UpDims* d);                                // checks the problem; non-zero + gnr_last_error()
void up_rgb(const float* in, float* out, int batch, int S, hipStream_t st);         // out <- blur(bilinear2x(in)), 3 channels; in != out

}  // namespace gnr

// Launchers of rows_general.cu: rows of any width up to 8178, 16-byte aligned pointers,
// codes and their stride multiples of 8.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace fmhc {

// Arguments as launch_rms_fwd's; `norm` false: x itself goes into codes.  False (and
// nothing launched) for rows that are too wide.
bool launch_general_fwd(const void *x, int dtype, const void *res, const void *w, int pdt, float eps, void *y,
                        void *total, float *rstd, void *codes, int64_t stride, float *scales, bool norm,
                        int64_t rows, int C, cudaStream_t s);
// Partials [C] of grad_w that the backward writes (0 for rows that are too wide).
int general_bwd_parts(int64_t rows, int C);
bool launch_general_bwd(const void *g, int dtype, const void *gt, const void *x, const float *rstd, const void *w,
                        int pdt, void *gx, float *part, int64_t rows, int C, cudaStream_t s);

}  // namespace fmhc

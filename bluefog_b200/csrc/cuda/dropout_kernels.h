// Dropout from a counter-based generator, joined with a residual stream (see dropout_kernels.cu).
#pragma once
#include <cuda_runtime.h>

namespace bfb {

enum DropoutType : int { kDropF32 = 0, kDropF16 = 1, kDropBF16 = 2 };

// out[i] = (keep(i) ? factor * x[i] : 0) + residual[i] for i < n.  residual may be null, out may be x or residual.  keep(i):
// the 16-bit word i % 8 of the Philox4x32-10 block with key key[0] and counter (i / 8, site << 16 above it, key[1]) is at least
// `threshold`.  All pointers 16-byte aligned; key: two 64-bit words on the device.
cudaError_t LaunchDropoutAdd(const void* x, const void* residual, void* out, long long n, int type, unsigned int threshold,
                             float factor, const long long* key, unsigned int site, cudaStream_t stream);

}  // namespace bfb

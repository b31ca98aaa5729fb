// The driver's tensor-map encoder, looked up once per process (gemm_tc.cu); null where the
// driver has none.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

namespace snl {
PFN_cuTensorMapEncodeTiled tensor_map_encoder();
}  // namespace snl

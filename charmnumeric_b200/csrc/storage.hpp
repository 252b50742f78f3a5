// Fills, copies and tiles of arrays of the storage types (storage.cu); the other types' are in kernels.cu.
#pragma once
#include <cstdint>

#include <cuda_runtime.h>

#include "kernels.hpp"

namespace cn {

cudaError_t launch_storage_fill(void* base, int dtype, const StridedView& v, const int64_t ext[3], double value, cudaStream_t s);
cudaError_t launch_storage_copy(void* dst, const StridedView& dv, const void* src, const StridedView& sv, const int64_t ext[3], int dtype,
                                cudaStream_t s);
cudaError_t launch_storage_tile(void* dst, const int64_t dst_shape[3], int64_t dst_row_begin, int64_t dst_rows, const void* src,
                                const int64_t src_shape[3], int dtype, cudaStream_t s);

}  // namespace cn

// What the translation units of libvteb200.so share: the error text, the device and the driver entry points of
// vteb200_shim.cu.  Nothing here is part of the C ABI.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace vteb_shim {

int report(int code, const char* fmt, ...);                  // sets vteb_last_error_string() and returns `code`
int report_rt(cudaError_t e, const char* what);
int report_drv(CUresult r, const char* what);
int device_index();                                          // -1 before vteb_init
int encode_tiled(CUtensorMap* map, CUtensorMapDataType type, cuuint32_t rank, void* base, const cuuint64_t* dims,
                 const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle);

}  // namespace vteb_shim

// op_check.h — host-side checks shared by the operator entry points (internal to libtsd_b200).
#pragma once
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/tsd.h"

namespace tsd {

// ggml type numbers the 4-bit and norm operators take (include/tsd_ops.h); bytes of one element, 0 for any other.
inline int float_size(int type) {
    return type == 0 ? 4 : (type == 1 || type == 30) ? 2 : 0;
}

inline bool aligned(const void * p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The status of a call whose launches gave e. A refused launch is reported here and nowhere else: the runtime's last
// error, which calls that ask for it would take for their own, is cleared.
inline int launch_status(const char * fn, cudaError_t e) {
    if (e == cudaSuccess) return TSD_OK;
    cudaGetLastError();
    fprintf(stderr, "%s: %s\n", fn, cudaGetErrorString(e));
    return TSD_ERR_CUDA;
}

// Makes the device that owns the operands current for the duration of a call. Null pointers are
// passed over. rc: TSD_OK, TSD_ERR_ARG if a pointer is not CUDA memory or the operands lie on
// different devices (a launch would fault on them), TSD_ERR_CUDA if the driver cannot tell.
class OperandDevice {
public:
    int rc = TSD_OK;
    explicit OperandDevice(std::initializer_list<const void *> ptrs);
    ~OperandDevice();
    OperandDevice(const OperandDevice &) = delete;
    OperandDevice & operator=(const OperandDevice &) = delete;

private:
    int prev_ = -1;   // device to restore, or -1
};

}  // namespace tsd

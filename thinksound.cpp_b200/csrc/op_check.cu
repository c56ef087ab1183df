// op_check.cu — which device an operator call runs on (see op_check.h).
#include "op_check.h"

namespace tsd {

namespace {
typedef CUresult (*PFN_pointerAttr_t)(void *, CUpointer_attribute, CUdeviceptr);
PFN_pointerAttr_t pointer_attr_fn() {
    static const PFN_pointerAttr_t fn = [] {
        void * p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuPointerGetAttribute", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        if (!ok) cudaGetLastError();   // no driver: leave no error behind for the next call
        return ok ? reinterpret_cast<PFN_pointerAttr_t>(p) : nullptr;
    }();
    return fn;
}
}  // namespace

OperandDevice::OperandDevice(std::initializer_list<const void *> ptrs) {
    const PFN_pointerAttr_t attr = pointer_attr_fn();
    int cur = 0;
    if (!attr || cudaGetDevice(&cur) != cudaSuccess) {
        cudaGetLastError();
        rc = TSD_ERR_CUDA;
        return;
    }
    int dev = -1;
    for (const void * p : ptrs) {
        if (!p) continue;
        int d = -1;
        if (attr(&d, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, reinterpret_cast<CUdeviceptr>(p)) != CUDA_SUCCESS || d < 0 ||
            (dev >= 0 && d != dev)) {
            rc = TSD_ERR_ARG;
            return;
        }
        dev = d;
    }
    if (dev >= 0 && dev != cur) {
        if (cudaSetDevice(dev) != cudaSuccess) {
            cudaGetLastError();
            rc = TSD_ERR_CUDA;
            return;
        }
        prev_ = cur;
    }
}

OperandDevice::~OperandDevice() {
    if (prev_ >= 0) cudaSetDevice(prev_);
}

}  // namespace tsd

// The seam between the executor (psk_exec.cu) and the head's losses (psk_head.cu). Internal to the library.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string>
#include "../../include/presk_cuda.h"

namespace psk {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct HeadContext {
    psk_exec *e; // for its buffers (psk_exec_alloc, psk_exec_free)
    cudaStream_t stream;
    EncodeTiledFn encode;
    int sms;
    uint32_t *status, *ovf; // the executor's status word; this launch's flag of the overflow guard
    bool guarded;
    int64_t kernels = 0;    // kernels launched
    double flops = 0;
    std::string error;
};

// PSK_OP_HEAD_XENT, PSK_OP_HEAD_DISTILL and their _VJP; the table's pointers without the operands' offsets.
int head_run(HeadContext &x, const psk_launch *l, void *const *table);

} // namespace psk

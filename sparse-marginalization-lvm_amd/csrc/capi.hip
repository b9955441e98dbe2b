// ABI bookkeeping for libsparsemarg_hip.so.
#include "common.hpp"

namespace smlvm {
thread_local int g_last_hip_error = 0;
}

extern "C" int smlvm_abi_version(void) { return SMLVM_ABI_VERSION; }

extern "C" int smlvm_last_hip_error(void) { return smlvm::g_last_hip_error; }

extern "C" const char* smlvm_error_string(int code)
{
    switch (code) {
        case SMLVM_OK: return "ok";
        case SMLVM_ERR_INVALID: return "invalid argument";
        case SMLVM_ERR_UNSUPPORTED: return "size not supported by the gfx950 kernels";
        case SMLVM_ERR_HIP: return "HIP launch failed (see smlvm_last_hip_error)";
        case SMLVM_ERR_WORKSPACE: return "workspace missing or too small";
        default: return "unknown error";
    }
}

extern "C" int smlvm_stream_capture_id(void* stream, uint64_t* id)
{
    if (!id) return SMLVM_ERR_INVALID;
    *id = 0;
    if (!stream) return SMLVM_OK;   // (the default stream is never captured; asking it costs 60 us while it is busy)
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long got = 0;
    const hipError_t e = hipStreamGetCaptureInfo((hipStream_t)stream, &status, &got);
    if (e != hipSuccess) {
        smlvm::g_last_hip_error = (int)e;
        return SMLVM_ERR_HIP;
    }
    *id = status == hipStreamCaptureStatusActive ? (uint64_t)got : 0;
    return SMLVM_OK;
}

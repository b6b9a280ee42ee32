// entry_checks.h -- what the entry points on caller-owned device memory check
// before they launch anything (internal).
#pragma once

#include "../../include/moonlight_kernels.h"
#include "device_context.h"
#include "mlh_host.h"

namespace mlh {

inline int refuse(const char *what, const std::string &why, int status = kErrArgs) {
    set_last_error(std::string(what) + ": " + why);
    return status;
}

// One pointer of a call: its name, how its values are aligned, whether it may
// be null.
struct Pointer {
    const void *ptr;
    const char *name;
    unsigned align;
    bool optional;
};

template <int N>
inline int check_pointers(const char *what, const Pointer (&list)[N]) {
    for (const Pointer &p : list) {
        if (!p.ptr && !p.optional) return refuse(what, std::string(p.name) + " is null");
        if ((uintptr_t)p.ptr % p.align)
            return refuse(what, std::string(p.name) + " is not aligned to its values");
    }
    return kOk;
}

// The library stream of the current device, on which every pointer has to be
// memory of that device (a kernel that is given another address faults).
template <int N>
inline int check_device(const char *what, const Pointer (&list)[N], hipStream_t *stream) {
    DeviceContext *ctx = context();
    if (!ctx) return kErrDevice;
    for (const Pointer &p : list) {
        if (!p.ptr) continue;
        hipPointerAttribute_t at;
        const hipError_t e = hipPointerGetAttributes(&at, p.ptr);
        if (e != hipSuccess) (void)hipGetLastError();
        if (e != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged))
            return refuse(what, std::string(p.name) + " is not device memory");
        if (at.device != ctx->device)
            return refuse(what, std::string(p.name) + " is memory of device " +
                                    std::to_string(at.device) + ", the current device is " +
                                    std::to_string(ctx->device));
    }
    *stream = ctx->stream;
    return kOk;
}

inline int finish(int status, const char *what) {
    if (status == kErrArgs) return refuse(what, "invalid arguments");
    if (status == kErrLaunch) set_last_error(std::string(what) + ": kernel launch failed");
    if (status == kErrSize) set_last_error(std::string(what) + ": too many blocks for one launch");
    return status;
}

// Types of values that are not codes.
inline bool type_ok(int type) { return type == MLK_F32 || type == MLK_BF16; }
inline unsigned size_of(int type) { return type == MLK_BF16 ? 2 : 4; }

}  // namespace mlh

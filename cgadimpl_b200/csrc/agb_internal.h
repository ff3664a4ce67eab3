// agb_internal.h -- what the library's translation units share on the host: error reporting, the launch counter,
// device properties and the address of the device status word.  Everything is defined in agb_cuda.cu; nothing here
// is part of the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "agb/agb.h"

#define AGB_HIDDEN __attribute__((visibility("hidden")))

namespace agb_int {

// Stores the message for agb_last_error() on this thread and returns `code`.
AGB_HIDDEN int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
AGB_HIDDEN int cuda_fail(cudaError_t e, const char* what);
// After a kernel launch: the launch's error, else counts it.
AGB_HIDDEN int after_launch(const char* what);
AGB_HIDDEN int check_ptr(const void* p, const char* name, int elem, bool required = true);

struct Device {
    int sms, smem_optin, smem_per_sm;
    int* status;          // the device status word that agb_device_status() reads
};
// Properties of the current device.
AGB_HIDDEN int device(Device* out);
AGB_HIDDEN bool pdl_enabled();

}  // namespace agb_int

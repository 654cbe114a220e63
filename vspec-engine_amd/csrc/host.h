// host.h -- host helpers of paged_kv.hip that the other C entries of the library use.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "vspec_rocm.h"

namespace vkv {

// The reason that vspec_rocm_last_error() gives, kept per host thread.
void host_error(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
// Geometry that every kernel takes; `decode` adds the attention kernels' limits.
int host_check_kv(const VspecPagedKV* kv, const char* who, bool decode);
// Grow-only workspace of the current device, or null when it cannot be allocated.
void* host_workspace(size_t bytes);
int host_num_cus();

}  // namespace vkv

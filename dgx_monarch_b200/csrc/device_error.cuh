// The error word, one a device and translation unit.  Kernels OR a kErr* bit
// into it when a bounded wait expires; the host reads all units' words with
// dgxm_device_error().  (A single one would need relocatable device code.)
#pragma once

#include "common.h"

namespace dgxm {

static __device__ int g_device_error = 0;
static const ErrorWord g_device_error_word(&g_device_error);

static __device__ __forceinline__ void report_device_error(int bits) { atomicOr(&g_device_error, bits); }

}  // namespace dgxm

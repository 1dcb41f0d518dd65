// SPDX-License-Identifier: BSD-3-Clause
// What the library's translation units share of the runtime: the error
// message of the calling thread, the current device and its streams.
// Defined in runtime.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xtc_hip {
namespace core {

// Sets the thread's message (printf form) and returns 1.
int fail(const char* fmt, ...);
// Whether xtc_hip_init has run.
bool ready();
// `stream`, or the library stream where it is null.
hipStream_t pick_stream(void* stream);

// `bytes` of scratch of stream `s` for partial sums (xtc_hip_matmul's), or null where
// there is none: the stream is being captured (a graph must not keep the address
// of a buffer that a later call replaces) or the memory cannot be had; the call
// then sums in one part.
float* partial_sums(size_t bytes, hipStream_t s);

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace core
}  // namespace xtc_hip

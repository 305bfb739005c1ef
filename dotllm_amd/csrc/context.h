// context.h -- what the entry points outside backend.hip need of a context.
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/llmdot_hip.h"

namespace llmdot {

// Sets the calling thread's error message and returns the code.
int ctx_fail(int code, const std::string& msg);
int ctx_device(const llmdot_hip_ctx* ctx);
hipStream_t ctx_stream(const llmdot_hip_ctx* ctx);
// An object that uses the context's stream until it is dropped; false once the
// context has been destroyed.  The last drop after llmdot_hip_destroy releases
// the context.
bool ctx_hold(llmdot_hip_ctx* ctx);
void ctx_drop(llmdot_hip_ctx* ctx);

}  // namespace llmdot

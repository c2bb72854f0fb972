// What the C entry points in mlq_abi.hip share with those in other files.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <string>

namespace mlq {

// Record the calling thread's error message and return `code`.
int abi_fail(int code, const std::string& msg);
int abi_hip_fail(hipError_t e, const char* what);
// Set the library up on `device` and make it the thread's current one.
int abi_device(int device);
hipStream_t abi_stream(int device, void* stream);
bool abi_capturing(hipStream_t s);
// [p, p + bytes) lies inside one allocation on `device`.
int abi_device_ptr(const void* p, int device, const char* caller, const char* what, size_t bytes);

}  // namespace mlq

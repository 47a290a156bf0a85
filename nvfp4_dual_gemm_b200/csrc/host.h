// host.h — host state of the library (dual_gemm.cu) that its other translation
// units use: the thread's error message, the device's properties and error
// word, and tensor-map encoding.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "nvfp4_dual_gemm.h"

namespace nvfp4dg {

// Device error word bits (role whose bounded wait expired).
constexpr unsigned kErrProducer = 1u << 0;
constexpr unsigned kErrMma = 1u << 1;
constexpr unsigned kErrEpilogue = 1u << 2;
constexpr unsigned kErrDrain = 1u << 3;

struct HostDevice {
  int id;
  int sms;
  unsigned* err;  // the device's error word
};

// The current device (an sm_100 one, or a status is returned).
int host_device(HostDevice* out);

// Message of the calling thread's last failure; both failure forms return the
// status to hand to the caller.
void host_clear_error();
int host_fail(int code, const std::string& msg);
int host_cuda_fail(cudaError_t e, const char* what);

// Byte view of `layers` matrices, `layer_bytes` apart, of `rows` rows of
// `row_bytes` bytes, `pitch` apart; boxes of 128 bytes x `box_rows` rows with
// the 128-byte swizzle.  3-D, or 2-D for `layers` = 0 (one matrix).  Needs
// host_device() first.
int host_byte_map(const void* ptr, long long rows, long long row_bytes,
                  long long pitch, int box_rows, long long layers,
                  long long layer_bytes, CUtensorMap* out);

// NVFP4DG_FLAG_SYNC_CHECK: waits for `stream` and reads the error word.
int host_sync_check(cudaStream_t stream);

// How two row-major matrices of `rows` rows of `bytes` bytes lie (pitches in
// bytes; NULL overlaps nothing).  Of matrices with different pitches whose
// ranges meet, no row is looked at: they count as overlapping.
enum class Overlap { kNone, kSame, kPart };
inline Overlap host_overlap(const void* p, long long p_pitch, const void* q,
                            long long q_pitch, long long rows,
                            long long bytes) {
  if (p == nullptr || q == nullptr || rows < 1 || bytes < 1)
    return Overlap::kNone;
  const unsigned long long a = reinterpret_cast<uintptr_t>(p);
  const unsigned long long b = reinterpret_cast<uintptr_t>(q);
  if (a == b && (rows == 1 || p_pitch == q_pitch)) return Overlap::kSame;
  const unsigned long long row = bytes, pitch = p_pitch;
  if (a + (rows - 1) * p_pitch + row <= b || b + (rows - 1) * q_pitch + row <= a)
    return Overlap::kNone;
  if (p_pitch == q_pitch) {  // columns of one wider matrix?
    const unsigned long long d = a < b ? (b - a) % pitch : (a - b) % pitch;
    if (d >= row && pitch - d >= row) return Overlap::kNone;
  }
  return Overlap::kPart;
}

// Whether the `bytes` bytes from p meet a row of the matrix m.
inline bool host_meets(const void* p, long long bytes, const void* m,
                       long long pitch, long long rows, long long row) {
  if (p == nullptr || m == nullptr || bytes < 1 || rows < 1 || row < 1)
    return false;
  const unsigned long long a = reinterpret_cast<uintptr_t>(p);
  const unsigned long long b = reinterpret_cast<uintptr_t>(m);
  const unsigned long long total = (rows - 1) * pitch + row;
  if (a >= b + total || a + bytes <= b) return false;
  if (rows == 1 || a < b) return true;
  const unsigned long long in = (a - b) % pitch;  // from its row's start
  return in < static_cast<unsigned long long>(row) ||
         (in + bytes > static_cast<unsigned long long>(pitch) &&
          a - b - in + pitch < total);
}

// Runs a C entry point's body: no C++ exception leaves it.
template <typename F>
int host_guarded(F body) {
  try {
    return body();
  } catch (...) {
    return NVFP4DG_ERR_CUDA;  // out of host memory
  }
}

}  // namespace nvfp4dg

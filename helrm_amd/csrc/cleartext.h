// cleartext.h -- internal declarations of the operators that train and score
// the model in the clear (layer norm, gated feed-forward block, softmax cross
// entropy against a table).  Not part of the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <stdexcept>
#include <string>
#include "plan.h"

// The element types of an operator's tensors, as the C ABI numbers them.
enum DType { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
inline int dtype_size(int t) { return t == DT_F32 ? 4 : 2; }

// Records the message GetLastError() returns; the value is -1 (runtime.hip).
int report_error(const char* what);

namespace clr {

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };
inline void require(bool ok, const char* what) { if (!ok) throw Error(what); }
inline void check_hip(hipError_t e, const char* what) {
  if (e != hipSuccess) throw Error(std::string("HIP error: ") + hipGetErrorString(e) + " at " + what);
}
template <class F> int guarded(F&& f) {
  try {
    (void)hipGetLastError();   // (of an earlier call, an allocation that failed say: not this one's)
    f();
    check_hip(hipGetLastError(), "a kernel launch");
    return 0;
  }
  catch (const std::exception& e) { return report_error(e.what()); }
  catch (...) { return report_error("unknown error"); }
}
// Workgroups of a launch: one of 2^32 threads or more runs what is left of them beyond, and reports no error.
inline unsigned groups_of(long groups, int threads) {
  require(groups * threads < 1L << 32, "more threads than a launch has");
  return (unsigned)groups;
}
// f(first, n) for up to 2^31 threads' workgroups at a time
template <class F> void in_launches(long groups, int threads, F&& f) {
  const long most = (1L << 31) / threads;
  for (long first = 0; first < groups; first += most) f(first, (unsigned)(groups - first < most ? groups - first : most));
}
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// f(T{}) with T the C++ type of a DType
template <class F> void with_type(int t, F&& f) {
  if (t == DT_F32) f(float{});
  else if (t == DT_BF16) f(__bf16{});
  else f(_Float16{});
}

}  // namespace clr

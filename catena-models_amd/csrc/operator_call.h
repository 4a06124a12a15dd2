// What the entry points of the operators over device memory share: the device
// of their operands, the launch, and checks of layouts.
#pragma once

#include <initializer_list>

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The device that every one of the pointers lies on; the calling thread's
// device for the length of an operator and back again after it.
class OperatorDevice {
 public:
  ~OperatorDevice() {
    if (before_ >= 0) hipSetDevice(before_);
  }
  int enter(std::initializer_list<const void*> pointers, hipStream_t stream) {
    int device = -1;
    for (const void* p : pointers) {
      if (!p) continue;
      hipPointerAttribute_t at;
      if (hipPointerGetAttributes(&at, p) != hipSuccess ||
          (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
        hipGetLastError();
        return fail(CQ35_EINVAL, "%p is not device memory", p);
      }
      if (device >= 0 && at.device != device)
        return fail(CQ35_EINVAL, "operands lie on devices %d and %d", device, at.device);
      device = at.device;
    }
    hipDevice_t of = 0;
    if (stream) {
      HIP_TRY(hipStreamGetDevice(stream, &of));
      if ((int)of != device) return fail(CQ35_EINVAL, "the stream is device %d's, the operands device %d's", (int)of, device);
    }
    int now = -1;
    HIP_TRY(hipGetDevice(&now));
    if (now != device) {
      HIP_TRY(hipSetDevice(device));
      before_ = now;
    }
    return CQ35_OK;
  }

 private:
  int before_ = -1;
};

template <typename Args>
int launch_operator(const char* what, void (*kernel)(Args), dim3 grid, int threads, size_t lds, hipStream_t stream,
                    Args args) {
  void* list[] = {&args};
  const hipError_t e = hipLaunchKernel((const void*)kernel, grid, dim3((unsigned)threads), list, lds, stream);
  if (e != hipSuccess) {
    hipGetLastError();
    return fail(CQ35_EDEVICE, "%s: %s", what, hipGetErrorString(e));
  }
  return CQ35_OK;
}

// Whether dimensions of the given lengths and strides (elements) address
// every element once: in some order each stride covers what lies inside it.
struct Dim {
  int64_t length, stride;
};
template <int N>
bool distinct(const Dim (&dims)[N], int64_t inner) {
  Dim by[N];
  int n = 0;
  for (const Dim& d : dims)
    if (d.length > 1) {
      int i = n++;
      for (; i > 0 && by[i - 1].stride > d.stride; --i) by[i] = by[i - 1];
      by[i] = d;
    }
  int64_t extent = inner;
  for (int i = 0; i < n; ++i) {
    if (by[i].stride < extent || by[i].stride > INT64_MAX / 4 / by[i].length) return false;
    extent += (by[i].length - 1) * by[i].stride;
  }
  return true;
}

}  // namespace

// What every operator class behind the C ABI is made of.
#pragma once
#include <math.h>

#include "runtime.h"

struct vkl_op {
  vkl_device *dev;
  vkl_command *cmd;
  bool inited = false;
  cudaEvent_t e0 = nullptr, e1 = nullptr;
  bool timed = false;
  vkl_op(vkl_device *d, vkl_command *c) : dev(d), cmd(c) {}
  virtual int init() = 0;
  virtual ~vkl_op() {
    if (e0) cudaEventDestroy(e0);
    if (e1) cudaEventDestroy(e1);
  }
  int base_init() {
    if (!dev || !cmd) return vkl::fail(VKL_INVALID_ARGUMENT, "op: null device or command");
    VKL_CUDA(cudaEventCreate(&e0));
    VKL_CUDA(cudaEventCreate(&e1));
    inited = true;
    return VKL_OK;
  }
  int enter(const char *who) {
    if (!inited) return vkl::fail(VKL_FAILED_PRECONDITION, "%s: init() was not called", who);
    VKL_OKAY(vkl::recording(cmd, who));
    VKL_CUDA(cudaEventRecord(e0, cmd->stream));
    return VKL_OK;
  }
  // Op::time(): device microseconds of the last run, 0 before the first.
  virtual int elapsed(uint64_t *usec) {
    *usec = 0;
    if (!timed) return VKL_OK;
    float ms = 0.f;
    const cudaError_t e = cudaEventElapsedTime(&ms, e0, e1);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return vkl::fail(VKL_FAILED_PRECONDITION, "op_time: the op's last run has not finished (wait on its command first)");
    }
    *usec = (uint64_t)llroundf(ms * 1000.f);
    return VKL_OK;
  }
  int leave() {
    VKL_CUDA(cudaEventRecord(e1, cmd->stream));
    timed = true;
    return VKL_OK;
  }
};

namespace vkl {
inline int need_dense(const vkl_tensor *t, const char *who) {
  if (!t) return vkl::fail(VKL_INVALID_ARGUMENT, "%s: null tensor", who);
  if (!t->dense()) return vkl::fail(VKL_UNIMPLEMENTED, "%s: strided views are not supported by this op", who);
  return VKL_OK;
}
template <class T>
int as(vkl_op *op, T **out, const char *who) {
  if (!op) return vkl::fail(VKL_INVALID_ARGUMENT, "%s: null op", who);
  T *t = dynamic_cast<T *>(op);
  if (!t) return vkl::fail(VKL_INVALID_ARGUMENT, "%s: handle is another kind of op", who);
  *out = t;
  return VKL_OK;
}
}  // namespace vkl

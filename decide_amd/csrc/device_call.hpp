// What the operators on device arrays share: a checked call on a context's
// device and stream.
#pragma once

#include <exception>

#include "block_check.hpp"
#include "ctx.hpp"

// The context's device for the duration of a call; the caller's current one
// comes back after it.
struct OnDevice {
  int before = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    if (before == device) before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// check() gives a blockchk::Refusal, launch() a hipError_t. No C++ exception
// (an allocation that fails while a message is built) leaves the C entry point.
template <class Check, class Launch>
int device_call(dn_ctx *c, const char *op, Check check, Launch launch) {
  if (!c) return DN_INVALID_ARG;
  try {
    c->err.clear();
    const blockchk::Refusal r = check();
    if (r.code) return dnh::fail(c, r.code, r.msg);
    const OnDevice on(c->device);
    HIPCHK(c, "hipSetDevice", on.err);
    HIPCHK(c, op, launch());
    return DN_OK;
  } catch (const std::exception &) {
    return DN_OUT_OF_MEMORY;
  }
}

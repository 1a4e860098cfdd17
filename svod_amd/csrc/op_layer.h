// What the op layer's files share: the records of what the last op did, the checks of descriptors and addresses, the device of a
// call's stream and whether it has kernels.
#pragma once
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>

#include "../../include/svodk.h"

namespace svodk {
namespace op {

// ---- per-thread records: ops::chosen (tk/src/ops/mod.rs:83-118) and the last error.
// A record is kept as the static strings it is made of: its text is written when it is asked for, not on every call.
struct Chosen {
  const char *op = nullptr, *family = nullptr, *cfg = nullptr;  // a kernel's family and config, or no family:
  int why = 0;                                                  // the graph, and why
};
inline thread_local Chosen g_chosen;
inline thread_local std::string g_chosen_text;
inline thread_local std::string g_error;

inline const char *fallback_name(int why) {
  switch (why) {
    case SVODK_GRAPH_TARGET: return "Target";
    case SVODK_GRAPH_DTYPE: return "Dtype";
    case SVODK_GRAPH_SYMBOLIC: return "Symbolic";
    case SVODK_GRAPH_SHAPE: return "Shape";
    case SVODK_GRAPH_CONFIG: return "Config";
    default: return "?";
  }
}

// ran_graph (mod.rs:115-118).
inline int ran_graph(const char *op, int why) {
  g_chosen = {op, nullptr, nullptr, why};
  return why;
}

// ran (mod.rs:110-113).
inline void ran(const char *op, const char *family, const char *cfg) { g_chosen = {op, family, cfg, 0}; }

inline std::string chosen_text() {
  const Chosen &c = g_chosen;
  if (c.op == nullptr) return "";
  if (c.family == nullptr) return std::string("Graph { op: \"") + c.op + "\", why: " + fallback_name(c.why) + " }";
  return std::string("Kernel { op: \"") + c.op + "\", family: \"" + c.family + "\", cfg: \"" + c.cfg + "\" }";
}

inline int fail(int status, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  g_error = buf;
  return status;
}

inline const char *dtype_name(int32_t d) {
  switch (d) {
    case SVODK_BF16: return "BFloat16";
    case SVODK_F16: return "Float16";
    case SVODK_F32: return "Float32";
    case SVODK_I32: return "Int32";
    case SVODK_I64: return "Int64";
    case SVODK_BOOL: return "Bool";
    case SVODK_E4M3: return "Float8E4M3";
    case SVODK_E8M0: return "Float8E8M0";
    default: return "?";
  }
}

inline size_t dtype_bytes(int32_t d) {
  switch (d) {
    case SVODK_BF16:
    case SVODK_F16: return 2;
    case SVODK_F32:
    case SVODK_I32: return 4;
    case SVODK_I64: return 8;
    case SVODK_BOOL: return 1;
    default: return 0;
  }
}

inline std::string fmt_shape(const svodk_tensor *t) {
  std::string s = "[";
  for (int i = 0; i < t->rank; i++) {
    if (i) s += ", ";
    s += std::to_string((long long)t->shape[i]);
  }
  return s + "]";
}

inline bool well_formed(const svodk_tensor *t) {
  if (t == nullptr || t->rank < 0 || t->rank > 4 || dtype_bytes(t->dtype) == 0) return false;
  for (int i = 0; i < t->rank; i++)
    if (t->shape[i] < 0) return false;
  return true;
}

inline int64_t numel(const svodk_tensor *t) {
  int64_t n = 1;
  for (int i = 0; i < t->rank; i++) n *= t->shape[i];
  return n;
}

inline bool same_shape(const svodk_tensor *a, const svodk_tensor *b) {
  if (a->rank != b->rank) return false;
  for (int i = 0; i < a->rank; i++)
    if (a->shape[i] != b->shape[i]) return false;
  return true;
}

inline bool is_int(int32_t d) { return d == SVODK_I32 || d == SVODK_I64; }

// What the kernels assume of a device address: 16-bit tensors are read and written in 128-bit pieces
// (and filled into LDS 16 bytes a lane), integers and masks at their element's size.
inline size_t alignment_of(const svodk_tensor *t) {
  return (t->dtype == SVODK_BF16 || t->dtype == SVODK_F16) ? 16 : dtype_bytes(t->dtype);
}

// The first of `tensors` (nulls skipped) whose address is off its alignment, or -1.
inline int misaligned(const svodk_tensor *const *tensors, int n) {
  for (int i = 0; i < n; i++) {
    const svodk_tensor *t = tensors[i];
    if (t != nullptr && t->data != nullptr && ((uintptr_t)t->data & (alignment_of(t) - 1)) != 0) return i;
  }
  return -1;
}

// launch::aliasing (tk/src/launch.rs:227-246): no parameter the kernel writes
// shares memory with another.  Here a parameter is a byte range.
struct Span {
  const char *name;
  const void *data;
  size_t bytes;
  bool written;
};

inline int check_aliasing(const char *op, const Span *spans, int n) {
  for (int i = 0; i < n; i++) {
    for (int j = i + 1; j < n; j++) {
      const Span &a = spans[i], &b = spans[j];
      if (!(a.written || b.written) || a.data == nullptr || b.data == nullptr || a.bytes == 0 || b.bytes == 0) continue;
      const char *a0 = (const char *)a.data, *b0 = (const char *)b.data;
      if (a0 < b0 + b.bytes && b0 < a0 + a.bytes)
        return fail(SVODK_ERR_LAUNCH, "%s: parameters %s and %s share memory", op, a.name, b.name);
    }
  }
  return 0;
}

// The device of the caller's stream is the current one for the length of a call: what is asked of a device (has it kernels,
// its compute units, its scratch, a kernel's function) is then asked of the one that runs the launch.  The default streams
// are the current device's own; on another stream it takes 0.1 us (a norm's call 3.9 -> 4.0).
class OnDeviceOf {
 public:
  explicit OnDeviceOf(void *hip_stream) {
    const hipStream_t stream = (hipStream_t)hip_stream;
    if (stream == nullptr || stream == hipStreamLegacy || stream == hipStreamPerThread) return;
    int of = -1, now = -1;
    if (hipStreamGetDevice(stream, &of) != hipSuccess || hipGetDevice(&now) != hipSuccess)
      (void)hipGetLastError();  // no stream: the launch says so
    else if (of != now && hipSetDevice(of) == hipSuccess)
      back_ = now;
  }
  OnDeviceOf(const OnDeviceOf &) = delete;
  ~OnDeviceOf() {
    if (back_ >= 0) (void)hipSetDevice(back_);
  }

 private:
  int back_ = -1;
};

// ---- the target: ops::supported / planner (mod.rs:161-197), without the cost probes.
// The library is built for gfx950 alone; any other device has no kernels.
inline bool device_is_gfx950(int device) {
  hipDeviceProp_t prop;
  if (hipGetDeviceProperties(&prop, device) != hipSuccess) return false;
  return std::strncmp(prop.gcnArchName, "gfx950", 6) == 0;
}

inline bool current_device_has_kernels() {
  int device = -1;
  if (hipGetDevice(&device) != hipSuccess || device < 0) {
    (void)hipGetLastError();
    return false;
  }
  // 0 unknown, 1 yes, 2 no; two threads that both find it unknown ask the runtime twice and store the same answer.
  static std::atomic<int> known[64];
  if (device >= 64) return device_is_gfx950(device);
  int state = known[device].load(std::memory_order_acquire);
  if (state == 0) {
    state = device_is_gfx950(device) ? 1 : 2;
    known[device].store(state, std::memory_order_release);
  }
  return state == 1;
}

// The compute units of the current device (256 on an MI355X), asked once a device.
inline int current_device_units() {
  int device = -1;
  if (hipGetDevice(&device) != hipSuccess || device < 0) {
    (void)hipGetLastError();
    return 256;
  }
  static std::atomic<int> known[64];
  int units = device < 64 ? known[device].load(std::memory_order_acquire) : 0;
  if (units == 0) {
    if (hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || units <= 0) {
      (void)hipGetLastError();
      units = 256;
    }
    if (device < 64) known[device].store(units, std::memory_order_release);
  }
  return units;
}

// ---- shape gates (tk/src/ops/shape.rs).
// gate (L92-99): a target with kernels, every operand the same 16-bit type the
// target has a matrix core for: gfx950 has one for bf16 and for f16, and both have kernels here.
inline int gate(bool has_target, const int32_t *dtypes, int n) {
  if (!has_target) return SVODK_GRAPH_TARGET;
  if (n <= 0) return SVODK_GRAPH_DTYPE;
  const int32_t first = dtypes[0];
  if (!(first == SVODK_BF16 || first == SVODK_F16)) return SVODK_GRAPH_DTYPE;
  for (int i = 0; i < n; i++)
    if (dtypes[i] != first) return SVODK_GRAPH_DTYPE;
  return 0;
}

}  // namespace op
}  // namespace svodk

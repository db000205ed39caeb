// Checks of the arrays that a call is given.
#pragma once
#include "common.h"

namespace tf {

// The arrays of one call: on the GPU that is current, and no output shares memory with another array.
struct Operands {
  const char* what;
  int device = -1;
  bool ok = true;
  struct Range { uintptr_t from, to; bool written; };
  Range range[12];
  int n = 0;
  explicit Operands(const char* w) : what(w) { if (cudaGetDevice(&device) != cudaSuccess) { cudaGetLastError(); device = 0; } }
  int fail(const char* name, const char* why) { if (ok) set_error("%s: %s %s", what, name, why); ok = false; return -1; }
  // size < 0: any
  void add(const DLArray* a, const char* name, int64_t size, bool written, bool may_miss = false) {
    if (!ok) return;
    if (!a) { if (!may_miss) fail(name, "is missing"); return; }
    if (a->ctx.device_type != kGPU) { fail(name, "is not on the GPU"); return; }
    if (a->ctx.device_id != device) { fail(name, "is on another GPU than the current one"); return; }
    const int64_t count = numel(a);
    if (size >= 0 && count != size) { fail(name, "does not have the size the other arrays ask for"); return; }
    if (count && !a->data) { fail(name, "has no memory"); return; }
    if (count && (reinterpret_cast<uintptr_t>(a->data) & 3)) { fail(name, "is not aligned to its elements"); return; }
    const Range r{(uintptr_t)a->data, (uintptr_t)a->data + sizeof(float) * (uintptr_t)count, written};
    for (int i = 0; i < n; ++i)
      if ((written || range[i].written) && r.from < range[i].to && range[i].from < r.to) { fail(name, "shares memory with another array of the call, and one of the two is written"); return; }
    range[n++] = r;
  }
};

}  // namespace tf

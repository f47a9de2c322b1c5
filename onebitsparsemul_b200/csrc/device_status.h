// What a device's kernels have noted since the last look, and what is said of it. Plain C++, also compiled by a host test.
#pragma once
#include <stdio.h>

#include "../../include/onebit_sparse_tensor.h"

namespace ob {

// A bounded wait that gave up leaves its code in its kernel's wait word, a batch that named something outside its tensors leaves
// a mark in a word of its own: neither can hide the other. 0: nothing.
struct DeviceStatus {
  int tensor_memory_wait = 0, decode_wait = 0, few_token_wait = 0, attend_wait = 0, attend_many_wait = 0;
  int append_batch = 0, attend_batch = 0, attend_many_batch = 0;
};

// The status code and a sentence. A wait that gave up comes first: then results are unusable, while a bad batch only lacks what it
// named wrongly.
inline int describe(const DeviceStatus& s, char* text, size_t size) {
  const struct { int code; const char* kernel; const char* what; } waits[] = {
      {s.tensor_memory_wait, "tensor-memory", "role code"}, {s.decode_wait, "decode", "code"}, {s.few_token_wait, "few-token", "code"},
      {s.attend_wait, "few-row cache attention", "code"}, {s.attend_many_wait, "cache attention", "code"}};
  const char* batch = s.append_batch ? "cache append: a page number or a sequence offset is outside its range (that page was not written)"
                      : s.attend_batch || s.attend_many_batch
                          ? "cache attention: a page number or a sequence offset is outside its range (those tokens were left out)"
                          : nullptr;
  for (const auto& w : waits)
    if (w.code != 0) {
      snprintf(text, size, "a bounded wait inside the %s kernel gave up (%s %d)%s%s", w.kernel, w.what, w.code, batch ? "; " : "", batch ? batch : "");
      return ONEBIT_ERR_DEVICE_WAIT;
    }
  if (!batch) return ONEBIT_OK;
  snprintf(text, size, "%s", batch);
  return ONEBIT_ERR_BATCH;
}

}  // namespace ob

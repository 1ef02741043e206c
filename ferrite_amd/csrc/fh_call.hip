// Entry points of many arguments called with an array of them (fh_call): one conversion for a binding instead of one an argument.
#include <string.h>
#include "fh_common.h"

extern "C" int fh_call(int entry, const int64_t* v) {
  auto p = [&](int i) { return (void*)(uintptr_t)v[i]; };
  auto ip = [&](int i) { return (const int32_t*)(uintptr_t)v[i]; };
  auto fp = [&](int i) { return (const float*)(uintptr_t)v[i]; };
  auto n = [&](int i) { return (int)v[i]; };
  if (!v) return fh::fail(FH_EINVAL, "fh_call: null pointer");
  switch (entry) {
    case FH_CALL_ROPE_APPEND_PAGED: {
      double eps;
      memcpy(&eps, v + 10, 8);
      return fh_rope_append_paged(p(0), n(1), v[2], v[3], n(4), n(5), n(6), n(7), fp(8), fp(9), (float)eps, n(11), fp(12), fp(13), v[14], ip(15), ip(16), ip(17),
                                  v[18], v[19], n(20), p(21), n(22), v[23], p(24), n(25), v[26], p(27));
    }
    case FH_CALL_ATTENTION_PAGED:
      return fh_attention_paged(p(0), n(1), v[2], p(3), n(4), v[5], v[6], n(7), n(8), n(9), n(10), ip(11), ip(12), ip(13), v[14], v[15], n(16), v[17], p(18),
                                n(19), v[20], p(21), (size_t)v[22], p(23));
    case FH_CALL_LORA:
      return fh_lora(p(0), n(1), v[2], v[3], v[4], p(5), p(6), n(7), n(8), n(9), n(10), (const int64_t*)(uintptr_t)v[11], fp(12), ip(13), p(14), v[15], p(16),
                     n(17), v[18], p(19), (size_t)v[20], p(21));
    default: return fh::fail(FH_EINVAL, "fh_call: no such entry point");
  }
}

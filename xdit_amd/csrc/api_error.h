// The thread-local error message behind xdit_attn_last_error and checks that the files with entry points share.
#pragma once
#include <algorithm>
#include <cstdint>

#include "../../include/xdit_amd_attn.h"

namespace xdit {

void api_clear_error();
__attribute__((format(printf, 2, 3))) int api_fail(int code, const char* fmt, ...);  // returns `code`
int api_check_tensor(const char* name, const void* p, const xdit_strides& st, int esize, int D);  // a (B, H, S, D) tensor that the attention kernels can address

// Whether no two rows of `C` elements share one: going from the smallest stride up, each has to step over all that those below it reach.
struct Axis { int64_t n, stride; };
template <int N>
bool rows_apart(int64_t C, Axis (&axes)[N]) {
  std::sort(axes, axes + N, [](const Axis& a, const Axis& b) { return a.stride < b.stride; });
  __int128 reach = C;
  for (const Axis& a : axes) {
    if (a.n <= 1) continue;
    if (a.stride < reach) return false;
    reach += (__int128)a.stride * (a.n - 1);
  }
  return true;
}

}  // namespace xdit

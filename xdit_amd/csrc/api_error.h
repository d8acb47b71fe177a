// The thread-local error message behind xdit_attn_last_error, for the files that hold entry points.
#pragma once

namespace xdit {

void api_clear_error();
__attribute__((format(printf, 2, 3))) int api_fail(int code, const char* fmt, ...);  // returns `code`

}  // namespace xdit

// What the translation units that export C entry points share: the calling thread's error text (engine.hip).
#pragma once
#include <string>

namespace mz {
// Records the text mz_last_error() returns to this thread and hands `code` back.
int api_fail(int code, const std::string &msg);
// MZ_OK, or MZ_ERR_HIP with the error of the launches since the last hipGetLastError.
int api_launch_status(const char *fn);
}  // namespace mz

// What scmiac_last_error() returns next on this thread; gives `code` back.
#pragma once
namespace scmiac {
int api_fail(int code, const char* message);
}  // namespace scmiac

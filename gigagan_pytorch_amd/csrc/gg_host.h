// gg_host.h — the host-side helpers that the library's translation units share (defined in gg_api.hip).
#pragma once

// records the text that gg_last_error() returns (thread-local) and returns `code`
__attribute__((visibility("hidden"))) int gg_fail(int code, const char* fmt, ...);
// 0, or the launch error of this thread as a positive hipError_t
__attribute__((visibility("hidden"))) int gg_check_launch();

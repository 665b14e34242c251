// What the C-ABI translation units share.
#pragma once
#include <stdint.h>

namespace sa {

// Sets the calling thread's message (sa_last_error) and returns `code`.
int fail(int code, const char *fmt, ...);

// The number of a launch whose workgroups count their arrivals (arrives_last): its upper 56 bits, no two in a process alike.
// The first one depends on the time the process took it and on where it lies in memory, so that memory which another
// process left behind holds none of them.
uint64_t next_launch_tag();

// Workgroups of 256 that a launch can have (its threads have 32 bits).
constexpr int64_t kMostGroups256 = (1 << 24) - 1;

}  // namespace sa

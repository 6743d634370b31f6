// What the library's translation units share on the host side (defined in api.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <string>

#include "../../include/tcu_scope.h"

namespace tcu {

// stores the message for tcu_last_error() of this host thread and returns `code`
int report_failure(int code, const std::string &message);
// "lookback_poll_limit" and "test_mute_partition" of tcu_set_option
unsigned shared_poll_limit();
unsigned shared_mute_partition();
// the check behind every entry point: a launch the runtime rejected becomes TCU_ERR_RUNTIME
int launch_outcome(const char *what, unsigned long launches_before, int rc);

// x * y, false if it does not fit size_t
inline bool product_fits(size_t x, size_t y, size_t *out) { return !__builtin_mul_overflow(x, y, out); }

}  // namespace tcu

// What the host parts of the C ABI share.  Host code only.
#pragma once

namespace pplx_amd {

// Makes `message` the calling thread's last failure (pplx_a2a_last_error) and returns `status`.
int report_failure(int status, const char *message);

}  // namespace pplx_amd

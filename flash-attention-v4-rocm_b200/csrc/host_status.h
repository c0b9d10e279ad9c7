// What the library's translation units share on the host.
#pragma once
#include <cstdint>

namespace fav4 {

// Address of the current device's status word (see fav4_bshd_pipeline_status), and the time limit of
// the kernels' waits; null on a CUDA error.
uint32_t* pipeline_status_word();
uint64_t pipeline_wait_limit_ns();

}  // namespace fav4

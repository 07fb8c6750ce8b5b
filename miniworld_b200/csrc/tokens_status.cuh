// Where the token operators' kernels leave the code of a bounded wait that gave up.
#pragma once

namespace trimul {

__device__ int tokens_status;  // 0, or the code of the first such wait (it stays until the host has read it)

}  // namespace trimul

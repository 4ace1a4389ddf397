// Who has shares of a unit of the 8-bit decode: warp `first`, and `more` warps after it.  Plain C++, shared by kernels and tests.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LTCA_HOST_DEVICE __host__ __device__
#else
#define LTCA_HOST_DEVICE
#endif

namespace ltca {

// Whether an entry of the table names warps that there are.  An entry that was never written - its warp gave up a wait and said so
// in the status word - holds whatever the scratch held before, and no address or number of turns may come of that.
LTCA_HOST_DEVICE inline bool shares_are_there(int32_t first, int32_t more, int32_t warps) {
    return first >= 0 && more >= 0 && first < warps && more < warps - first;
}

}  // namespace ltca

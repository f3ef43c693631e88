// Host functions of linear_sm100.cu.
#pragma once

namespace mr {

// Device status word of K13 (0, or MR_ERR_TIMEOUT); synchronizes.
int linear_status(int reset);

}  // namespace mr

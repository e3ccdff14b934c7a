// The wgrad instantiations of linear.h (one translation unit for each product: they compile side by side).
#include "linear.h"

int lin_wgrad(const LinParams& p, int tile, hipStream_t s) { return lin_tile<float, EPI_WGRAD>(p, tile, s); }

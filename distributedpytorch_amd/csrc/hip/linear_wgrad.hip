// The wgrad instantiations of linear.h (one translation unit for each product: they compile side by side).
#include "linear.h"

int lin_wgrad(const LinParams& p, int tile, bool f32, hipStream_t s) {      // (the gradient is fp32)
  return f32 ? lin_tile<float, 3, EPI_WGRAD>(p, tile, s) : lin_tile<float, 1, EPI_WGRAD>(p, tile, s);
}

// The fprop instantiations of linear.h (one translation unit for each product: they compile side by side).
#include "linear.h"

int lin_fprop(const LinParams& p, int tile, bool f32, hipStream_t s) {
  return f32 ? lin_tile<float, 3, EPI_FPROP>(p, tile, s) : lin_tile<bf16_t, 1, EPI_FPROP>(p, tile, s);
}

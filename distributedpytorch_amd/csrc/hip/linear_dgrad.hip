// The dgrad instantiations of linear.h (one translation unit for each product: they compile side by side).
#include "linear.h"

int lin_dgrad(const LinParams& p, int tile, hipStream_t s) {
  return p.parts == 3 ? lin_tile<float, EPI_DGRAD>(p, tile, s) : lin_tile<bf16_t, EPI_DGRAD>(p, tile, s);
}

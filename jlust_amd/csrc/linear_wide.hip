// linear_wide.hip -- the dense products of 32- and 64-bit values.
#include "tile_kernel.hpp"

namespace jlust {

template int plan_tile_product<float>(TileArgs *, bool, bool, int *, size_t *, double *);
template int launch_tile_product<float>(const TileArgs &, bool, bool, int, hipStream_t);
template int plan_tile_product<double>(TileArgs *, bool, bool, int *, size_t *, double *);
template int launch_tile_product<double>(const TileArgs &, bool, bool, int, hipStream_t);

int preload_linear_wide()
{
    JLUST_PRELOAD_KERNEL((tile_product_kernel<double, true, true, 128, 128, 2, 2>));
    return JLUST_STATUS_SUCCESS;
}

}  // namespace jlust

// linear_half.hip -- the dense products of 16-bit values.
#include "tile_kernel.hpp"

namespace jlust {

template int plan_tile_product<_Float16>(TileArgs *, bool, bool, int *, size_t *, double *);
template int launch_tile_product<_Float16>(const TileArgs &, bool, bool, int, hipStream_t);
template int plan_tile_product<__bf16>(TileArgs *, bool, bool, int *, size_t *, double *);
template int launch_tile_product<__bf16>(const TileArgs &, bool, bool, int, hipStream_t);

TileForm tile_form(int shape)
{
    return {TILE_SHAPES[shape].bm, TILE_SHAPES[shape].bn, shape >= COPY_256 && shape <= COPY_128};
}

int preload_linear_half()
{
    JLUST_PRELOAD_KERNEL((tile_product_kernel<__bf16, true, true, 128, 128, 2, 2>));
    return JLUST_STATUS_SUCCESS;
}

}  // namespace jlust

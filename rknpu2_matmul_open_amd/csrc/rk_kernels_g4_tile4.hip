// Tiles of G4 products with 4 groups in a piece of 128 k.
#include "rk_kernels_g4_tile.h"

int rkk::launch_g4_tiles4(hipStream_t st, const rkh_g4_args& g, const rkk::G4Route& r) { return launch_tiles<4>(st, g, r); }

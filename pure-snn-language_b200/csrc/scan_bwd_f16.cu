// scan_bwd_f16.cu - the leaky scan's gradient tile kernels for f16
#define SNN_SCAN_TILE_LAUNCH
#include "scan_tile.h"

template void snnb_scan::launch_tiles<true, __half>(int, bool, int, bool, const Plan&, ScanArgs&, cudaStream_t);

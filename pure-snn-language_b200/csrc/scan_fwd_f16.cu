// scan_fwd_f16.cu - the leaky scan's forward tile kernels for f16
#define SNN_SCAN_TILE_LAUNCH
#include "scan_tile.h"

template void snnb_scan::launch_tiles<false, __half>(int, bool, int, bool, const Plan&, ScanArgs&, cudaStream_t);

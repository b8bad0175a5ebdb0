// scan_fwd_f32.cu - the leaky scan's forward tile kernels for f32
#define SNN_SCAN_TILE_LAUNCH
#include "scan_tile.h"

template void snnb_scan::launch_tiles<false, float>(int, bool, int, bool, const Plan&, ScanArgs&, cudaStream_t);

// scan_bwd_bf16.cu - the leaky scan's gradient tile kernels for bf16
#define SNN_SCAN_TILE_LAUNCH
#include "scan_tile.h"

template void snnb_scan::launch_tiles<true, __nv_bfloat16>(int, bool, int, bool, const Plan&, ScanArgs&, cudaStream_t);

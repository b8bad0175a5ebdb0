// elem.h - element types of the device-tensor operators: loads widened to f32,
// stores rounded once (to nearest even).
#pragma once
#include <algorithm>
#include <atomic>
#include <utility>
#include <vector>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.h"

namespace snnb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

inline int elem_size(int32_t type) { return type == SNN_F32 ? 4 : 2; }
inline bool elem_type_ok(int32_t type) { return type == SNN_F32 || type == SNN_BF16 || type == SNN_F16; }

// f(T()) with the C++ type of an element type code
template <typename F>
void with_elem(int32_t type, F&& f) {
    if (type == SNN_F32) f(float());
    else if (type == SNN_BF16) f(__nv_bfloat16());
    else if (type == SNN_F16) f(__half());
    else throw Error(SNN_ERR_ARG, "element type must be SNN_F32, SNN_BF16 or SNN_F16");
}

// Whether runs of `width` elements, one for each index of dimensions {count, stride},
// lie apart (each stride clears what the smaller ones span)
inline bool apart(std::vector<std::pair<int64_t, int64_t>> dims, int64_t width) {
    for (const auto& d : dims)
        if (d.first == 0) return true;
    std::sort(dims.begin(), dims.end(), [](auto& a, auto& b) { return a.second < b.second; });
    for (const auto& [count, stride] : dims) {
        if (count <= 1) continue;
        if (stride < width) return false;
        width += (count - 1) * stride;
    }
    return true;
}

// the current device's multiprocessors (looked up once per device)
inline int device_sms() {
    static std::atomic<int> sms[64];
    int dev = 0;
    SNN_CUDA(cudaGetDevice(&dev));
    SNN_REQUIRE(dev >= 0 && dev < 64, SNN_ERR_ARG, "device ordinal above 63");
    if (!sms[dev]) {
        int n = 0;
        SNN_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        sms[dev] = n;
    }
    return sms[dev];
}

}  // namespace snnb

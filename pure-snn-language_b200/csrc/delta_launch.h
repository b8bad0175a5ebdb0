// delta_launch.h - the launches of one element type (included by a file for each)
#pragma once
#include "delta_grads.h"
#include "delta_prep.h"
#include "delta_scan.h"

namespace snnb_delta {
template <typename T, typename F>
void by_dim(int kdim, F&& f) {
    if (kdim <= 64) f(std::integral_constant<int, 64>());
    else f(std::integral_constant<int, 128>());
}
template <typename F>
void by_warps(int warps, F&& f) {
    if (warps == 8) f(std::integral_constant<int, 8>());
    else if (warps == 4) f(std::integral_constant<int, 4>());
    else if (warps == 2) f(std::integral_constant<int, 2>());
    else f(std::integral_constant<int, 1>());
}
template <typename T>
void launch_prep_of(const DeltaArgs& A, cudaStream_t st) {
    using P = typename PathOf<T>::P;
    by_dim<T>(A.kdim, [&](auto kd) {
        constexpr int KD = decltype(kd)::value;
        constexpr auto* kernel = k_delta_prep<P, KD>;
        set_smem<kernel>(prep_smem<P, KD>());
        kernel<<<dim3((unsigned)A.slots, (unsigned)A.heads), PREP, prep_smem<P, KD>(), st>>>(A);
    });
    SNN_CUDA(cudaGetLastError());
}
template <typename T>
void launch_scan_of(const DeltaArgs& A, int warps, cudaStream_t st) {
    using P = typename PathOf<T>::P;
    by_dim<T>(A.kdim, [&](auto kd) {
        by_warps(warps, [&](auto nw) {
            constexpr int KD = decltype(kd)::value, NW = decltype(nw)::value;
            using S = Stage<P, KD, NW, P::OUT>;
            constexpr auto* kernel = k_delta_scan<P, KD, NW>;
            set_smem<kernel>(S::SMEM);
            const int tiles = (A.vdim + S::VW - 1) / S::VW;
            DeltaArgs B = A;
            B.tiles = tiles;
            const dim3 grid((unsigned)std::min<long long>(A.items, 1 << 30), (unsigned)A.heads,
                            (unsigned)(A.only ? tiles + (A.kdim + S::VW - 1) / S::VW : tiles));
            kernel<<<grid, NW * 32, S::SMEM, st>>>(B);
        });
    });
    SNN_CUDA(cudaGetLastError());
}
template <typename T>
void launch_grads_of(const DeltaArgs& A, int warps, cudaStream_t st) {
    using P = typename PathOf<T>::P;
    by_dim<T>(A.kdim, [&](auto kd) {
        constexpr int KD = decltype(kd)::value;
        by_warps(warps, [&](auto nw) {
            constexpr int NW = decltype(nw)::value;
            using S = Stage<P, KD, NW, P::PIECES>;
            constexpr auto* kernel = k_delta_back<P, KD, NW>;
            set_smem<kernel>(S::SMEM);
            const dim3 grid((unsigned)std::min<long long>(A.n_seq, 1 << 30), (unsigned)A.heads,
                            (unsigned)((A.vdim + S::VW - 1) / S::VW));
            kernel<<<grid, NW * 32, S::SMEM, st>>>(A);
            SNN_CUDA(cudaGetLastError());
        });
        if (!A.slots) return;
        constexpr auto* kernel = k_delta_grads<T, KD>;
        set_smem<kernel>(GradTile<T, KD>::BYTES);
        kernel<<<dim3((unsigned)A.slots, (unsigned)A.hk), GRADS, GradTile<T, KD>::BYTES, st>>>(A);
        SNN_CUDA(cudaGetLastError());
    });
}
}  // namespace snnb_delta

#define SNN_DELTA_LAUNCHES(T)                                                                        \
    template <> DeltaSizes delta_sizes<T>() {                                                        \
        return {PathOf<T>::P::SQUARES, (int)sizeof(PathOf<T>::P::KE), (int)sizeof(Kept<T>::K), Kept<T>::PLANES};                                   \
    }                                                                                                \
    template <> void launch_prep<T>(const DeltaArgs& A, cudaStream_t st) { launch_prep_of<T>(A, st); } \
    template <> void launch_scan<T>(const DeltaArgs& A, int warps, cudaStream_t st) { launch_scan_of<T>(A, warps, st); } \
    template <> void launch_grads<T>(const DeltaArgs& A, int warps, cudaStream_t st) { launch_grads_of<T>(A, warps, st); }

// Launches of the power-of-two block-scaled FP8 GEMM (gemm_e8m0.cuh).
#include "gemm_e8m0.cuh"
#include "gemm_launch.cuh"
#include "qgemm_internal.h"

namespace qgemm {

namespace {

// `cluster` CTAs a cluster (1: no clusters, or fixed by the kernel).
template <typename... KArgs>
cudaError_t launch_e8(void (*kernel)(KArgs...), bool (&configured)[64], int smem, long long ctas, int threads, int cluster,
                      cudaStream_t stream, KArgs... args) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int TM, int S>
cudaError_t launch_small_one(const CUtensorMap& ta, const CUtensorMap& tb, const E8m0Params& p, cudaStream_t stream) {
    static bool configured[64] = {};
    return launch_e8(gemm_e8m0_small_kernel<TM, S>, configured, E8SmallSmem<TM>::kDynamicBytes,
                     static_cast<long long>(p.m_tiles) * p.n_tiles * S, kE8Threads, S, stream, ta, tb, p);
}

template <int TM>
cudaError_t launch_small(int slices, const CUtensorMap& ta, const CUtensorMap& tb, const E8m0Params& p, cudaStream_t stream) {
    switch (slices) {
        case 1: return launch_small_one<TM, 1>(ta, tb, p, stream);
        case 2: return launch_small_one<TM, 2>(ta, tb, p, stream);
        case 4: return launch_small_one<TM, 4>(ta, tb, p, stream);
        case 8: return launch_small_one<TM, 8>(ta, tb, p, stream);
        default: return cudaErrorInvalidValue;
    }
}

template <int OUT, int BN>
cudaError_t launch_pair_one(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const E8m0Params& p,
                            int clusters, cudaStream_t stream) {
    constexpr int smem = E8PairSmem<BN>::kDynamicBytes;
    static_assert(smem <= 227 * 1024, "dynamic shared memory of one CTA");
    static bool configured[64] = {};
    return launch_e8(gemm_e8m0_pair_kernel<OUT, BN>, configured, smem, 2ll * clusters, kE8Threads, 1, stream, ta, tb, tc, p);
}

template <int BN>
cudaError_t launch_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const E8m0Params& p,
                        int clusters, cudaStream_t stream) {
    switch (p.out) {
        case OUT_F32: return launch_pair_one<OUT_F32, BN>(ta, tb, tc, p, clusters, stream);
        case OUT_BF16: return launch_pair_one<OUT_BF16, BN>(ta, tb, tc, p, clusters, stream);
        case OUT_F16: return launch_pair_one<OUT_F16, BN>(ta, tb, tc, p, clusters, stream);
        default: return cudaErrorInvalidValue;
    }
}

template <int S>
cudaError_t launch_pair_split(const CUtensorMap& ta, const CUtensorMap& tb, const E8m0Params& p, cudaStream_t stream) {
    static_assert(E8PairKSmem::kDynamicBytes <= 227 * 1024, "dynamic shared memory of one CTA");
    static bool configured[64] = {};
    return launch_e8(gemm_e8m0_pair_split_kernel<S>, configured, E8PairKSmem::kDynamicBytes,
                     static_cast<long long>(p.m_tiles) * p.n_tiles * 2 * S, kE8Threads, 2 * S, stream, ta, tb, p);
}

}  // namespace

cudaError_t launch_e8m0_pair(int tile_n, int slices, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                             const E8m0Params& p, int clusters, cudaStream_t stream) {
    if (slices == 2 && tile_n == 128) return launch_pair_split<2>(ta, tb, p, stream);
    if (slices != 1) return cudaErrorInvalidValue;
    return tile_n == 256 ? launch_pair<256>(ta, tb, tc, p, clusters, stream) : launch_pair<128>(ta, tb, tc, p, clusters, stream);
}

cudaError_t launch_e8m0_small(int tokens_per_tile, int slices, const CUtensorMap& ta, const CUtensorMap& tb,
                              const E8m0Params& p, cudaStream_t stream) {
    switch (tokens_per_tile) {
        case 16: return launch_small<16>(slices, ta, tb, p, stream);
        case 32: return launch_small<32>(slices, ta, tb, p, stream);
        case 64: return launch_small<64>(slices, ta, tb, p, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace qgemm

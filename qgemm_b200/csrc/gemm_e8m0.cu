// Launches of the power-of-two block-scaled FP8 GEMM (gemm_e8m0.cuh).
#include "gemm_e8m0.cuh"
#include "gemm_launch.cuh"
#include "qgemm_internal.h"

namespace qgemm {

namespace {

template <int TM, int S>
cudaError_t launch_small_one(const CUtensorMap& ta, const CUtensorMap& tb, const E8m0Params& p, cudaStream_t stream) {
    auto kernel = gemm_e8m0_small_kernel<TM, S>;
    constexpr int smem = E8SmallSmem<TM>::kDynamicBytes;
    static bool configured[64] = {};
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
    cfg.gridDim = dim3(static_cast<unsigned>(p.m_tiles) * static_cast<unsigned>(p.n_tiles) * S);
    cfg.blockDim = dim3(kE8Threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (S > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = S;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, ta, tb, p);
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

template <int OUT>
cudaError_t launch_pair_one(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const E8m0Params& p,
                            int clusters, cudaStream_t stream) {
    auto kernel = gemm_e8m0_pair_kernel<OUT>;
    constexpr int smem = E8PairSmem::kDynamicBytes;
    static_assert(smem <= 227 * 1024, "dynamic shared memory of one CTA");
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    return launch_pdl(kernel, dim3(2 * clusters), dim3(kE8PairThreads), smem, stream, ta, tb, tc, p);
}

}  // namespace

cudaError_t launch_e8m0_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const E8m0Params& p,
                             int clusters, cudaStream_t stream) {
    switch (p.out) {
        case OUT_F32: return launch_pair_one<OUT_F32>(ta, tb, tc, p, clusters, stream);
        case OUT_BF16: return launch_pair_one<OUT_BF16>(ta, tb, tc, p, clusters, stream);
        case OUT_F16: return launch_pair_one<OUT_F16>(ta, tb, tc, p, clusters, stream);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_e8m0_small(int tokens_per_tile, int slices, const CUtensorMap& ta, const CUtensorMap& tb,
                              const E8m0Params& p, cudaStream_t stream) {
    switch (tokens_per_tile) {
        case 16: return launch_small<16>(slices, ta, tb, p, stream);
        case 32: return launch_small<32>(slices, ta, tb, p, stream);
        case 64: return launch_small<64>(slices, ta, tb, p, stream);
        case 128: return launch_small<128>(slices, ta, tb, p, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace qgemm

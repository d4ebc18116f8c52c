// q4_device.cuh -- what the kernels that read 4-bit weights share on the device.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "q4.h"

namespace telmo {

// A product behind the kernel that makes its planes is launched while that one still runs
// (programmatic stream serialisation) and waits where it first needs them; weights it reads before
// (200 rows of f32, 1024 -> 4096: 18.5 us without, 16.8 with; 1500 rows: 39.0 and 36.7).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Adds a launch's attributes: a cluster of `cluster` blocks, and such a start.
inline void add_attributes(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int cluster, bool early) {
    cfg.attrs = attr;
    cfg.numAttrs = 0;
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    if (early) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
}

// Codes 2 p and 2 p + 1 of a word less their zero point, as two exact operands; `base` is
// code_base of the zero point: a pair of 128 + zero (bf16) or 1024 + zero (fp16).
template <bool BF16>
__device__ __forceinline__ uint32_t code_base(uint32_t zero) {
    return (BF16 ? 0x43004300u : 0x64006400u) | (zero * 0x00010001u);
}
template <bool BF16>
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int p, uint32_t base) {
    // Codes are stored with their top bit flipped, which the exclusive or undoes.
    const uint32_t v = ((word >> (4 * p)) & 0x000f000fu) ^ (BF16 ? 0x43084308u : 0x64086408u);
    if (BF16) {
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                         *reinterpret_cast<const __nv_bfloat162*>(&base));
        return *reinterpret_cast<const uint32_t*>(&d);
    }
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&base));
    return *reinterpret_cast<const uint32_t*>(&d);
}

__device__ __forceinline__ float q4_act(float v, int act) {
    if (act == kActRelu) return v < 0.0f ? 0.0f : v;  // a NaN stays one
    if (act == kActSilu) return mul_sigmoid(v, v);
    return v;
}

__device__ __forceinline__ float q4_load(const void* c, int type, int64_t at) {
    if (type == kQ4F32) return static_cast<const float*>(c)[at];
    if (type == kQ4BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(c)[at]);
    return __half2float(static_cast<const __half*>(c)[at]);
}
__device__ __forceinline__ void q4_store(void* c, int type, int64_t at, float v) {
    if (type == kQ4F32) static_cast<float*>(c)[at] = v;
    else if (type == kQ4BF16) static_cast<__nv_bfloat16*>(c)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(c)[at] = __float2half_rn(v);
}

}  // namespace telmo

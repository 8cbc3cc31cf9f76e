// What the accumulated-weight kernels share.
#pragma once

#include "paged.cuh"

namespace jfb {
namespace paged {

struct MassParams {
    View view;
    const void * q;
    const float * lse;
    const float * mass_in;
    float * mass_out;
    uint64_t q_stride;
    uint32_t heads;
    float scale;
};

// The tcgen05 kernel of paged_mass_tc.cu.
jfb_status launch_mass_tc(const jfb_paged_cache & cache, const CUtensorMap & k, MassParams p, const Device & device, cudaStream_t s);

}  // namespace paged
}  // namespace jfb

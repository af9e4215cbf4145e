// Arguments of beam search's kernels (beam.hip).
#pragma once

#include "lrmoe_device.h"
#include "lrmoe_internal.h"
#include "paged.h"

namespace lrmoe {

constexpr int kBeamMax = LRMOE_BEAM_MAX;
constexpr int kForkTensors = LRMOE_FORK_TENSORS;

struct BeamArgs {
    int groups, beams, vocab;
    const void* logits;
    int64_t stride;   // of a row, in elements
    const float* scores;
    const uint8_t* finished;
    int64_t* tokens;
    int32_t* parents;
    float* scores_out;
    float2* sums;     // scratch: a slice's maximum and sum of exponentials
    uint2* best;      // scratch: a slice's best values and their tokens
};
hipError_t launch_beam_select(BeamArgs a, int type, void* workspace, hipStream_t stream);
size_t beam_workspace_bytes(int groups, int beams, int vocab);

struct ForkTensor {
    uint8_t* base;
    int64_t stride, bytes;   // of a row
    int width;               // bytes of an access: what base, stride and bytes are multiples of
    int first;               // workgroup at which the tensor begins
};
struct ForkRowsArgs {
    int rows, tensors;
    const int32_t* parents;
    ForkTensor t[kForkTensors];
};
hipError_t launch_fork_rows(ForkRowsArgs a, hipStream_t stream);

}  // namespace lrmoe

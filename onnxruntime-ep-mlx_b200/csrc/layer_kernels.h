// Internal argument blocks and launchers of the decoder-layer operators (include/b200_layer.h).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "b200_layer.h"

namespace b200 {

// Every launcher takes checked parameters, enqueues on `stream` and counts its launches.
cudaError_t launch_skip_rms_norm(const B200SkipRmsNormParams& p, int num_sms, cudaStream_t stream);

size_t rotary_append_workspace(const B200RotaryAppendParams& p);
cudaError_t launch_rotary_append(const B200RotaryAppendParams& p, int num_sms, cudaStream_t stream);

size_t shared_prefix_workspace(const B200SharedPrefixParams& p, int num_sms);
cudaError_t launch_shared_prefix(const B200SharedPrefixParams& p, int num_sms, cudaStream_t stream);

}  // namespace b200

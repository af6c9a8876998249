// Launches under the stage timing of mlxvs_profile (engine.cpp), for the other
// host files.
#pragma once

#include <hip/hip_runtime.h>

namespace mlxvs::detail {

// Throws if no GPU is there.
void need_device();

// run(args, s), bracketed by events if stage timing is on; throws
// std::runtime_error on a HIP error.
void launch_stage(hipStream_t s, const char* stage, hipError_t (*run)(const void*, hipStream_t),
                  const void* args);

template <typename Args, hipError_t (*Run)(const Args&, hipStream_t)>
void launch_stage(hipStream_t s, const char* stage, const Args& a) {
  launch_stage(s, stage,
               [](const void* p, hipStream_t q) { return Run(*static_cast<const Args*>(p), q); },
               &a);
}

}  // namespace mlxvs::detail

// ifr_losses.h -- launch interface of the preference and policy losses (ifr_losses.hip) used by ifr_api.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ifr.h"

namespace ifr {

int launch_preference(const ifr_preference &p, hipStream_t s);
size_t policy_workspace(const ifr_policy &p);
int launch_policy(const ifr_policy &p, void *ws, hipStream_t s);

}  // namespace ifr

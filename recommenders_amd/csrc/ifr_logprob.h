// ifr_logprob.h -- launch interface of the catalogue log-probabilities (ifr_logprob.hip) used by ifr_api.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/ifr.h"

namespace ifr {

struct LogprobGrad {
    const float *lse, *dlogp;
    int64_t ld_dlogp;
    void *dX, *dV;
    int64_t ld_dx, ld_dv;
    float *dibase;
};

size_t logprob_workspace(const ifr_catalogue &c);
int launch_logprob(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, float *logp, int64_t ld_logp, float *lse,
                   void *ws, hipStream_t s);
size_t logprob_backward_workspace(const ifr_catalogue &c, int64_t m, bool want_dx, bool want_dv, bool want_db);
int launch_logprob_backward(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, const LogprobGrad &g, void *ws,
                            hipStream_t s);

}  // namespace ifr

// MhContext and the argument checks shared by the translation units of
// include/moebius_hip.h.
#pragma once

#include "../../include/moebius_hip.h"
#include "capi_guard.hpp"
#include "common.hpp"
#include "kernels.hpp"

struct MhContext {
    mh::Context ctx;
    explicit MhContext(int dev) : ctx(dev) {}
};

namespace mh {
namespace capi {

inline mh::Context &C(MhContext *c) {
    if (!c) mh::fail(mh::kInvalidArgument, "context is NULL");
    HIP_CHECK(hipSetDevice(c->ctx.device));
    return c->ctx;
}

inline mh::WeightType wtype(uint32_t dt) {
    if (dt == MH_DTYPE_F32) return mh::kF32;
    if (dt == MH_DTYPE_F16) return mh::kF16;
    mh::fail(mh::kInvalidArgument, "unknown weight dtype");
}

inline int dim(uint32_t v, const char *what) {
    if (v > (1u << 30)) mh::fail(mh::kInvalidArgument, std::string(what) + " too large");
    return int(v);
}

}  // namespace capi
}  // namespace mh

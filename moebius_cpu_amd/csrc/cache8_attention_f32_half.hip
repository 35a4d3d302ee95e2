// The attention over a cache in 8 bits, instantiated.
#include "cache8_attention.hpp"

namespace mh {
namespace c8a {

void launch_f32_half(Context &ctx, const Args &a, int nq, int waves, int dt) {
    if (waves) rows_shared<float, 1, 1>(ctx, a, waves, dt);
    else rows_alone<float, 1>(ctx, a, nq, dt);
}

}  // namespace c8a
}  // namespace mh

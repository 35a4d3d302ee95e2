// The attention over a cache in 8 bits, instantiated.
#include "cache8_attention.hpp"

namespace mh {
namespace c8a {

void launch_f32_half(Context &ctx, const Args &a, int nq, int waves, int dt) {
    launch_all<float, 1>(ctx, a, nq, waves, dt);
}

}  // namespace c8a
}  // namespace mh

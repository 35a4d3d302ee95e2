// The attention over a cache in 8 bits, instantiated.
#include "cache8_attention.hpp"

namespace mh {
namespace c8a {

void launch_f16_half(Context &ctx, const Args &a, int waves, int dt) { rows_shared<_Float16, 1, 1>(ctx, a, waves, dt); }

}  // namespace c8a
}  // namespace mh

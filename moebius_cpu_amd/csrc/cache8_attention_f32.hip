// The attention over a cache in 8 bits, instantiated.
#include "cache8_attention.hpp"

namespace mh {
namespace c8a {

void launch_f32(Context &ctx, const Args &a, int nq, int dt) { launch_rows_dt<float, 2>(ctx, a, nq, dt); }

}  // namespace c8a
}  // namespace mh

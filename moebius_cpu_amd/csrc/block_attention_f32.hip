// Instantiations of block_attention.hpp: f32 storage, f32 products.
#include "block_attention.hpp"

namespace mh {
namespace battn {

void launch_f32(Context &ctx, const Args &a, int wr, int dt, bool vec) { launch_mode<float, kF32>(ctx, a, wr, dt, vec); }

}  // namespace battn
}  // namespace mh

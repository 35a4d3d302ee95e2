// Instantiations of block_attention.hpp: f32 storage, f16 products (FAST contexts).
#include "block_attention.hpp"

namespace mh {
namespace battn {

void launch_f32_half(Context &ctx, const Args &a, int wr, int dt, bool vec) { launch_mode<float, kHalf>(ctx, a, wr, dt, vec); }

}  // namespace battn
}  // namespace mh

// Instantiations of block_attention.hpp: f16 storage, f16 products.
#include "block_attention.hpp"

namespace mh {
namespace battn {

void launch_f16(Context &ctx, const Args &a, int wr, int dt, bool vec) { launch_mode<_Float16, kHalf>(ctx, a, wr, dt, vec); }

}  // namespace battn
}  // namespace mh

// The mirrored pass of decaying linear attention: gradients of the values and of the state.
#include "decay_pass.h"

namespace mm {
namespace dattn {
void launch_pass_mirrored(const Pass& p, hipStream_t s) { launch_pass<true>(p, s); }
}  // namespace dattn
}  // namespace mm

// tlk_gau_f32.hip -- the gated attention unit's forward kernels (tlk_gau.hpp) for float.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int forward<float>(Args, int, void *, hipStream_t);
}  // namespace gau
}  // namespace tlk

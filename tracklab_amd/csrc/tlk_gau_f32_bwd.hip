// tlk_gau_f32_bwd.hip -- the gated attention unit's backward kernels (tlk_gau.hpp) for float.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int backward<float>(Args, const BwdIo &, int, hipStream_t);
}  // namespace gau
}  // namespace tlk

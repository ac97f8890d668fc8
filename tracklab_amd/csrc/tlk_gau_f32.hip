// tlk_gau_f32.hip -- the gated attention unit's kernels (tlk_gau.hpp) for float.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int forward<float>(Args, int, void *, hipStream_t);
template int backward<float>(Args, const BwdIo &, int, hipStream_t);
}  // namespace gau
}  // namespace tlk

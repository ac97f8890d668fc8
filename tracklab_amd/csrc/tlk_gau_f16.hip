// tlk_gau_f16.hip -- the gated attention unit's forward kernels (tlk_gau.hpp) for _Float16.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int forward<_Float16>(Args, int, void *, hipStream_t);
}  // namespace gau
}  // namespace tlk

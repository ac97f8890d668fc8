// tlk_gau_f16_bwd.hip -- the gated attention unit's backward kernels (tlk_gau.hpp) for _Float16.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int backward<_Float16>(Args, const BwdIo &, int, hipStream_t);
}  // namespace gau
}  // namespace tlk

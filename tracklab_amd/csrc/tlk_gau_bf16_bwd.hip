// tlk_gau_bf16_bwd.hip -- the gated attention unit's backward kernels (tlk_gau.hpp) for __bf16.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int backward<__bf16>(Args, const BwdIo &, int, hipStream_t);
}  // namespace gau
}  // namespace tlk

// tlk_gau_bf16.hip -- the gated attention unit's forward kernels (tlk_gau.hpp) for __bf16.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int forward<__bf16>(Args, int, void *, hipStream_t);
}  // namespace gau
}  // namespace tlk

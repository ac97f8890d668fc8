// tlk_gau_bf16.hip -- the gated attention unit's kernels (tlk_gau.hpp) for __bf16.
#include "tlk_gau_host.hpp"

namespace tlk {
namespace gau {
template int forward<__bf16>(Args, int, void *, hipStream_t);
template int backward<__bf16>(Args, const BwdIo &, int, hipStream_t);
}  // namespace gau
}  // namespace tlk

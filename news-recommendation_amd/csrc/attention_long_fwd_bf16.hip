// attention of any length, forward, on bf16 tensors
#include "attention_long_fwd.h"

namespace nr {
namespace al {
template int run_fwd<__bf16>(const Args&, bool, bool, int, unsigned, hipStream_t);
}  // namespace al
}  // namespace nr

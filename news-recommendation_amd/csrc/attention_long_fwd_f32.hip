// attention of any length, forward, on fp32 tensors
#include "attention_long_fwd.h"

namespace nr {
namespace al {
template int run_fwd<float>(const Args&, bool, bool, int, unsigned, hipStream_t);
}  // namespace al
}  // namespace nr

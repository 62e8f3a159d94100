// attention of any length, backward, on fp32 tensors
#include "attention_long_bwd.h"

namespace nr {
namespace al {
template int run_bwd<float>(Args, const BwdPlan&, bool, bool, bool, hipStream_t);
}  // namespace al
}  // namespace nr

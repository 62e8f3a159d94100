// attention of any length, backward, on bf16 tensors
#include "attention_long_bwd.h"

namespace nr {
namespace al {
template int run_bwd<__bf16>(Args, const BwdPlan&, bool, bool, bool, hipStream_t);
}  // namespace al
}  // namespace nr

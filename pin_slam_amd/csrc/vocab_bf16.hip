// The label head's kernels for bfloat16 inputs (vocab_run.h).
#include "vocab_run.h"

namespace pin {
template int v_run_typed<PIN_BF16>(const VocabPlan&, int, hipStream_t);
int pin_warm_vocab_bf16() {
    hipFuncAttributes at;
    return hipFuncGetAttributes(&at, reinterpret_cast<const void*>(&vocab_prepare_kernel<PIN_BF16>)) == hipSuccess ? 0 : -1;
}
}  // namespace pin

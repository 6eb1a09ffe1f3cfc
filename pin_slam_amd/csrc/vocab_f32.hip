// The label head's kernels for float32 inputs (vocab_run.h).
#include "vocab_run.h"

namespace pin {
template int v_run_typed<PIN_F32>(const VocabPlan&, int, hipStream_t);
int pin_warm_vocab_f32() {
    hipFuncAttributes at;
    return hipFuncGetAttributes(&at, reinterpret_cast<const void*>(&vocab_prepare_kernel<PIN_F32>)) == hipSuccess ? 0 : -1;
}
}  // namespace pin

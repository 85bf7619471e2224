// Gated projections of fp16 operands.
#include "gated_run.hpp"

namespace trnblas {

template int gated_gemm_run<_Float16>(const GroupedArgs&, bool, hipStream_t);

}  // namespace trnblas

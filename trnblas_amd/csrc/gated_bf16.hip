// Gated projections of bf16 operands.
#include "gated_run.hpp"

namespace trnblas {

template int gated_gemm_run<__bf16>(const GroupedArgs&, bool, hipStream_t);

}  // namespace trnblas

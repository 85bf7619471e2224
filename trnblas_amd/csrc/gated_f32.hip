// Gated projections of fp32 operands.
#include "gated_run.hpp"

namespace trnblas {

template int gated_gemm_run<float>(const GroupedArgs&, bool, hipStream_t);

}  // namespace trnblas

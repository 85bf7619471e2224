// The grouped products of fp32 operands.
#include "grouped_run.hpp"

namespace trnblas {

template int grouped_gemm_run<float>(const GroupedArgs&, bool, hipStream_t);
template int grouped_rank_k_run<float>(const GroupedArgs&, hipStream_t);

}  // namespace trnblas

// The grouped products of f16 operands.
#include "grouped_run.hpp"

namespace trnblas {

template int grouped_gemm_run<_Float16>(const GroupedArgs&, bool, hipStream_t);
template int grouped_rank_k_run<_Float16>(const GroupedArgs&, hipStream_t);

}  // namespace trnblas

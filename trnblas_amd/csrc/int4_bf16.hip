// Products of 4-bit integer weights with bf16 rows, and with fp32 rows as three bf16 pieces.
#include "int4_run.hpp"

namespace trnblas {

template int int4_gemm_run<__bf16>(const GroupedArgs&, const Int4Args&, int, bool, hipStream_t);

}  // namespace trnblas

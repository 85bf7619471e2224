// Products of 4-bit integer weights with fp16 rows.
#include "int4_run.hpp"

namespace trnblas {

template int int4_gemm_run<_Float16>(const GroupedArgs&, const Int4Args&, int, bool, hipStream_t);

}  // namespace trnblas

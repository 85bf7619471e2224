// Products of 4-bit integer weights with many bf16 rows.
#include "int4_tile_run.hpp"

namespace trnblas {

template int int4_tile_run<__bf16>(const GroupedArgs&, const Int4Args&, int, bool, int, hipStream_t);

}  // namespace trnblas

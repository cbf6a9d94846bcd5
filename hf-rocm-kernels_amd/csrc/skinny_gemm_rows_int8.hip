// Row-split kernel for int8 codes, on row-major weights dealt out in 4-row units: instantiations of skinny_gemm_rows_impl.h.
#include "skinny_gemm_rows_impl.h"

namespace hfrk {

int launch_rows_int8_kernel(const GemmArgs& args, int act_loads, int row_tiles, int lds_bytes, hipStream_t stream) {
    if (!rows_variant_exists(act_loads, row_tiles) || lds_bytes != rows_lds_bytes(row_tiles, act_loads)) return HFRK_INVALID_CONFIG;
    switch (act_loads) {
#define HFRK_ROWS_CASE(MA_)                                                                                        \
    case MA_:                                                                                                      \
        return row_tiles == 1 ? launch_rows_one<MA_, 1, false, false, kRowsUnits, true>(args, lds_bytes, stream)   \
                              : launch_rows_one<MA_, 2, false, false, kRowsUnits, true>(args, lds_bytes, stream);
        HFRK_ROWS_CASE(1)
        HFRK_ROWS_CASE(2)
        HFRK_ROWS_CASE(3)
        HFRK_ROWS_CASE(4)
#undef HFRK_ROWS_CASE
        case 6: return launch_rows_one<6, 2, false, false, kRowsUnits, true>(args, lds_bytes, stream);
        case 8: return launch_rows_one<8, 2, false, false, kRowsUnits, true>(args, lds_bytes, stream);
    }
    return HFRK_INVALID_CONFIG;
}

}  // namespace hfrk

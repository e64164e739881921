#define GLP_ROWS_XT kF32
#include "op_rows.cuh"

#define GLP_ROWS_XT kF16
#include "op_rows.cuh"

#define GLP_ROWS_XT kBF16
#include "op_rows.cuh"

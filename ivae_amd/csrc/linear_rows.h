// Interface of linear_rows.hip.
#pragma once
#include "linear.h"

bool rows_serve(const LinArgs& A, int dtype);           // whether a forward product has few enough rows
struct RowsPlan { int nf, len, splits; };               // 16 nf weight rows a block; the summed index in `splits` parts of `len`
RowsPlan rows_plan(const LinArgs& A);
size_t rows_ws(const LinArgs& A);
hipError_t linear_rows_forward(const LinArgs& A, int dtype, hipStream_t st);

// Copies between matrices whose rows differ in width, for operands that the vector kernels cannot take as they lie.
#pragma once
#include "pf_common.h"

// dst [halves][to_rows][to_width] = src [halves][rows][width] (contiguous), zeros where src has nothing; elements of `size` 2 or 4 bytes, to_width * size a
// multiple of 16, dst on a boundary of 16 bytes
void pf_rows_widen(const void* src, int64_t rows, int64_t width, void* dst, int64_t to_rows, int64_t to_width, int halves, int size, hipStream_t st);
// dst [rows][width] (contiguous) = the first columns of src [rows][ld], 16-bit elements
void pf_rows_narrow(const void* src, int64_t ld, void* dst, int64_t rows, int64_t width, hipStream_t st);

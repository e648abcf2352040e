// Interface of linear_pack.hip.
#pragma once
#include "linear.h"

enum { FLIP_NONE, FLIP_ROWS, FLIP_COLS };

struct PackArgs {
    const void* src;            // (rows, cols), row stride ld
    const float* pre;           // or null: (rows, cols) saved pre-activations; the values become act'(pre) src
    void* out;                  // or null: (rows, ldo) of the same type, or for fp32 three bf16 matrices `plane` elements apart, each in
                                // columns of 32 values and `rows` rows (linear_big.h)
    bool pair;                  // 16-bit types: two matrices `plane` elements apart, values times `scale` rounded, and what that rounding left times `up`
    float scale, up;
    uint2* range;               // fp32: of each block, whether the parts of a value of it lost bits, and the largest finite magnitude (its bits)
    float* colsum;              // or null: (row blocks, cols) sums over the rows
    int64_t rows, ld, ldo, plane;
    int cols;
    int act;
    float slope;
    int flip;                   // fp32: every second run of 32 rows (FLIP_ROWS) or columns (FLIP_COLS) with its sign turned
    int group, blocks_x, blocks;    // set by the launcher
};
int pack_row_blocks(int64_t rows, int64_t width, bool colsum, int dtype);  // of a job with ldo = width: rows of its colsum
int pack_blocks(int64_t rows, int64_t width, bool colsum, int dtype);      // ... and all of its blocks
hipError_t launch_packs(const PackArgs* const* P, int n, int dtype, hipStream_t st);    // up to three in one launch; null: none

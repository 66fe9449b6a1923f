// Internal interface of the dense and expert products over fp16 / bf16 weights.
#pragma once

#include "common.hpp"

namespace aeon355 {

// Where a product's result goes.
enum ProductMode : int {
    kProductRows = 0,     // y[position][n] in the operands' type, after activation and residual
    kProductDraws = 1,    // contrib[draw][n] fp32 = weight[draw] * (W h + b)
    kProductPartial = 2,  // partial[split][matrix][token][n] fp32, without epilogue; several are joined by a second launch
};

struct ProductArgs {
    const uint16_t* x;        // [x_rows][x_stride]
    long x_stride;
    const int32_t* rows;      // row of x per position (null: the position itself)
    int x_rows;
    const uint16_t* w[2];     // [experts][n][w_stride]; w[1] only for the gated form
    long w_stride;
    long expert_stride;
    const uint16_t* bias[2];  // [experts][n], nullable
    int n, k;
    int pair;                 // 1: two matrices, y = swiglu(gate, up)
    int activation;
    float limit;
    const int32_t* offsets;   // [experts + 1], null for a dense product (one list of all positions)
    int experts;
    int positions;
    int mode;
    const uint16_t* residual;  // [positions][residual_stride], nullable
    long residual_stride;
    uint16_t* y;               // [positions][y_stride]
    long y_stride;
    float* wide;               // kProductDraws / kProductPartial
    const int32_t* draws;      // kProductDraws: draw of a position
    const float* draw_weights; // by draw
    int draw_count;
    int split_steps;           // kProductPartial: 64-column steps of one share of K
};

}  // namespace aeon355

// Products of two operands that both hold the contraction along their rows, with what a layer does to its sums behind them: the
// gated dense layer and the product of 8-bit integers (ptl_rows_mm.inc).
#pragma once
#include "ptl_common.hpp"

namespace ptl {

enum GateAct : int { GATE_SIGMOID = 0, GATE_SILU = 1, GATE_GELU = 2, GATE_RELU = 3 };

struct RowsArgs {
    const char *w, *x;  // rows of weights, rows of tokens
    int row_b;          // bytes of a row of either
    int outs, tokens;   // gated: 2 x outs rows of weights
    void *y;            // tokens x outs
    void *hidden;       // gated: tokens x 2 outs (NULL: not wanted)
    const void *bias;   // of the weights' rows (NULL: none)
    const float *w_scale, *x_scale;  // integers: of the weights' rows, of the tokens (NULL: 1)
    const char *zeros;  // 16 zero bytes
    int act;
    int tiles_w, tiles_t;
};

// The activation of a gated layer and its derivative.  e = exp(-|v|) is at most 1: nothing overflows, and 1 - s keeps the bits of
// small values.
__device__ inline float gate_sigmoid(float v, float &rest) {  // rest = 1 - sigmoid
    const float e = expf(-fabsf(v)), r = 1.f / (1.f + e), s = e * r;
    rest = v < 0.f ? r : s;
    return v < 0.f ? s : r;
}
constexpr float GATE_C = 0.7978845608028654f, GATE_C3 = 0.044715f;  // sqrt(2 / pi)
__device__ inline float gate_act(float g, int act) {
    float rest;
    if (act == GATE_RELU) return g > 0.f ? g : (g != g ? g : 0.f);
    if (act == GATE_SIGMOID) return gate_sigmoid(g, rest);
    if (act == GATE_SILU) return g * gate_sigmoid(g, rest);
    return g * gate_sigmoid(2.f * GATE_C * g * fmaf(GATE_C3 * g, g, 1.f), rest);  // (1 + tanh(u)) / 2 = sigmoid(2 u)
}
__device__ inline float gate_act_back(float g, int act, float &f) {  // f: the activation itself
    float rest, s;
    if (act == GATE_RELU) {
        f = g > 0.f ? g : (g != g ? g : 0.f);
        return g > 0.f ? 1.f : (g != g ? g : 0.f);
    }
    if (act == GATE_SIGMOID) {
        f = s = gate_sigmoid(g, rest);
        return s * rest;
    }
    if (act == GATE_SILU) {
        s = gate_sigmoid(g, rest);
        f = g * s;
        return s + f * rest;
    }
    s = gate_sigmoid(2.f * GATE_C * g * fmaf(GATE_C3 * g, g, 1.f), rest);
    f = g * s;
    // (far from 0 the slope of s is 0, whatever the square of g grows to)
    const float slope = s * rest;
    return slope > 0.f ? s + g * slope * 2.f * GATE_C * fmaf(3.f * GATE_C3 * g, g, 1.f) : (g != g ? g : s);
}

// 0: launched, 2: HIP error.
template <typename T>
int rows_gated(RowsArgs &a);  // T: tensors and products
template <typename OUT>
int rows_int8(RowsArgs &a);

}  // namespace ptl

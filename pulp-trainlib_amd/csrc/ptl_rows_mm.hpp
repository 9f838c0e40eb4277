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
    int parts;   // 32 x 32 tiles: workgroups that share a tile's k, each with sums of its own in ...
    void *part;  // ... parts x tiles x 16 x 64 (the lanes' accumulators)
};

// The activations of a gated layer, all but the last as m sigmoid(p): silu m = p = x, sigmoid m = 1, p = x, and gelu m = x,
// p = 2 sqrt(2 / pi) (x + 0.044715 x^3), since (1 + tanh(u)) / 2 = sigmoid(2 u).  Which one it is decides uniform constants and
// selects, not branches: a tile has 32768 outputs a compute unit, at expf(), a division and a branch each 10 us of 200 (4096 tokens,
// 2048 -> 5632 in fp16), this way 2.
struct Gate {
    float k1, k3;  // gelu: p = x (k1 + k3 x^2)
    bool one, relu, gelu;
    __device__ inline Gate(int act) {
        gelu = act == GATE_GELU;
        k1 = gelu ? 1.5957691216057308f : 1.f;
        k3 = gelu ? 0.07135481627260025f : 0.f;  // 0.044715 k1
        one = act == GATE_SIGMOID;
        relu = act == GATE_RELU;
    }
    // sigmoid(p) and 1 - sigmoid(p): exp(-|p|) is at most 1, nothing overflows and small values keep their bits.  log2(e) is the sum of
    // two floats, so that the exponent is formed to 2^-24 of itself.
    __device__ static inline float sigmoid(float p, float &rest) {
        const float n = -fabsf(p), e = __builtin_amdgcn_exp2f(fmaf(n, 1.44269502f, n * 1.92596299e-8f));
        const float r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
        rest = p < 0.f ? r : s;
        return p < 0.f ? s : r;
    }
    // Infinities take the limits: the product that gives gelu's p would be 0 times infinity in the others, and at -inf the sigmoid's 0
    // meets the lowest finite value.  GELU: 0 or 1 where it is known which, -1 otherwise.
    template <int GELU>
    __device__ inline float power(float x) const {
        if constexpr (GELU == 0) return x;
        const float p = x * fmaf(k3 * x, x, k1);
        return GELU == 1 || gelu ? p : x;
    }
    __device__ inline float factor(float x) const { return one ? 1.f : fmaxf(x, -3.402823466e38f); }
    template <int GELU = -1>
    __device__ inline float act(float x) const {
        float rest;
        const float s = sigmoid(power<GELU>(x), rest), f = factor(x) * s;
        return relu ? (x < 0.f ? 0.f : x) : f;
    }
    // The derivative; f: the activation itself.
    __device__ inline float back(float x, float &f) const {
        float rest;
        const float s = sigmoid(power<-1>(x), rest), slope = s * rest;  // of sigmoid, to p
        f = relu ? (x < 0.f ? 0.f : x) : factor(x) * s;
        // d p / d x = k1 + 3 k3 x^2; far from 0 the slope is 0, whatever that grows to
        const float d = slope > 0.f ? slope * (one ? 1.f : x * fmaf(3.f * k3 * x, x, k1)) : (x != x ? x : 0.f);
        return relu ? (x > 0.f ? 1.f : x != x ? x : 0.f) : one ? d : s + d;
    }
};

// Both products behind the gradients of a gated layer's pre-activations (dw or dx NULL: not wanted).  x and w have rows of `cols` values
// (in and more), dh of `pitch` (rows and more), all of whole 16-byte pieces; what dh has beyond `rows` is 0.  low: what dh lost when it was
// rounded, GRAD_LOW times, in the same layout (NULL: the products are of dh as it is).  The plan comes first: it says in how many parts k of
// dx and of dw is taken and what workspace their sums need, `ws`, which a call has in hand before its first launch.
constexpr float GRAD_LOW = 2048.f;
struct GradParts {
    int parts[2];
    size_t bytes;
};
template <typename T>
int gated_products_plan(GradParts &p, bool dw, bool dx, bool low, int ns, int in, int rows);
template <typename T>
int gated_products(const GradParts &parts, float *ws, const T *x, const T *w, const T *dh, const T *low, T *dw, T *dx, int ns, int in, int rows, int cols,
                   int pitch);
// Copies of n_x rows of x and n_w rows of w (either may be 0), whose rows have `bytes`, to rows of `pitch` bytes (in whole 16-byte pieces)
// with zeros behind them, one behind the other.
void rows_copy(const void *w, size_t n_w, const void *x, size_t n_x, void *to, int bytes, int pitch);

// 0: launched, 2: HIP error.
template <typename T>
int rows_gated(RowsArgs &a);  // T: tensors and products
template <typename OUT>
int rows_int8(RowsArgs &a);

}  // namespace ptl

// Orthogonalisation of matrices: what the host hands the kernels and how a matrix's share of the workspace is laid out.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace nnb {

constexpr int kOrthoTile = 64;           // matrices are padded with zeros to whole tiles
constexpr int kOrthoItems = 20;          // matrices (or equal batches of them) per group of launches
constexpr int kOrthoMaxSteps = 16;
constexpr int kOrthoSegment = 3;         // Newton-Schulz steps between two looks at the matrix itself
constexpr int kOrthoNormParts = 256;     // partial sums of squares per matrix

constexpr int ortho_padded(int v) { return (v + kOrthoTile - 1) / kOrthoTile * kOrthoTile; }

// One matrix, or `batch` equal ones.  X is the matrix laid on its long side: m <= n, transposed if rows > cols.
struct OrthoItem {
    const void *x;               // the matrix, or the gradient of an optimiser step
    void *out;                   // the result, or the new weights
    const void *weight;          // optimiser step only: weights, momentum before and after (contiguous)
    const float *momentum;
    float *momentum_out;
    long long x_rs, x_cs, x_bs;  // strides of x and out in elements: row, column, batch
    long long o_rs, o_cs, o_bs;
    size_t ws;                   // offset of the first matrix's area, a multiple of 256
    size_t ws_stride;            // bytes of one matrix's area
    int rows, cols, batch, type;
    float scale;                 // optimiser step: lr * max(1, rows / cols)^(1/2)
};

struct OrthoGroup {
    OrthoItem item[kOrthoItems];
    int first[kOrthoItems + 1];  // first block of every item in the launch at hand
    int count;
    unsigned char *ws;
};

// Areas of one matrix's workspace.  "Planes" are a hi and a lo half per value: value * 2^k = hi + lo.
struct OrthoArea {
    int m, n, mp, np;
    size_t parts, x, xt[2], sq[6], bytes;
};
enum OrthoSquare { SQ_A0 = 0, SQ_A1 = 1, SQ_T = 2, SQ_P = 3, SQ_Q0 = 4, SQ_Q1 = 5 };

__host__ __device__ inline OrthoArea ortho_area(int rows, int cols) {
    OrthoArea a;
    a.m = rows < cols ? rows : cols;
    a.n = rows < cols ? cols : rows;
    a.mp = ortho_padded(a.m);
    a.np = ortho_padded(a.n);
    const size_t wide = (size_t)a.mp * a.np * 4, square = (size_t)a.mp * a.mp * 4;
    size_t o = 0;
    a.parts = o; o += kOrthoNormParts * sizeof(double);
    a.x = o; o += wide;
    for (int i = 0; i < 2; ++i) { a.xt[i] = o; o += wide; }
    for (int i = 0; i < 6; ++i) { a.sq[i] = o; o += square; }
    a.bytes = o;
    return a;
}

struct OrthoParams {
    int type;                    // nnb_dtype of x, out and weight
    int muon;                    // 1: optimiser step
    int steps;
    float coef[kOrthoMaxSteps][3];
    double eps;
    float mu, decay;             // optimiser step: momentum, 1 - lr * weight_decay
    int nesterov;
};

}  // namespace nnb

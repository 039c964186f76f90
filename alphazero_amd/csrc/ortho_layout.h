// Orthogonalisation of matrices: what the host hands the kernels and how a matrix's share of the workspace is laid out.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace nnb {

constexpr int kOrthoPad = 64;            // matrices are padded with zeros to a multiple of this
constexpr int kOrthoItems = 20;          // matrices (or equal batches of them) per group of launches
constexpr int kOrthoMaxSteps = 16;
constexpr int kOrthoSegment = 3;         // Newton-Schulz steps between two looks at the matrix itself
// Matrices up to this side take all products of a segment in one launch, a block each, where all of a call are as small;
// their squares' diagonals are held apart in float32, there and beside larger ones.
constexpr int kOrthoSegmentRows = 128;
// Squares of up to so many rows take the products of lo halves along: they cost little there (launches), and the plain
// float32 form is the more accurate the smaller the matrix (200 x 3000: 2.2e-6 of the result without, 2.0e-6 with, plain
// 1.8e-6; 777 x 1501: 1.6e-6, 1.5e-6, plain 3.0e-6; three of them 304 us without, 332 with).
constexpr int kOrthoLoRows = 512;
constexpr int kOrthoNormParts = 1024;    // partial sums of squares per matrix at most

__host__ __device__ constexpr int ortho_padded(int v) { return (v + kOrthoPad - 1) / kOrthoPad * kOrthoPad; }
__host__ __device__ constexpr int ortho_min(int a, int b) { return a < b ? a : b; }
__host__ __device__ constexpr int ortho_max(int a, int b) { return a > b ? a : b; }

// One matrix, or `batch` equal ones.
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

// What the products need of an item.
struct OrthoShape {
    size_t ws, ws_stride;
    int rows, cols, batch, splits;
};

// A block looks for its item in two rounds of reads: the head of the group, then the item.
template <typename Item> struct OrthoGroupOf {
    int blocks;                  // of the launch at hand (blockIdx.x)
    int first[kOrthoItems];      // first block of every item; behind the last one INT32_MAX
    int count;
    unsigned char *ws;
    Item item[kOrthoItems];
};
typedef OrthoGroupOf<OrthoItem> OrthoGroup;
typedef OrthoGroupOf<OrthoShape> OrthoShapes;

// Areas of one matrix's workspace.  X is the matrix laid on its long side (m <= n, transposed if rows > cols).  A matrix
// [R][K] of float32-faithful operands (value * 2^k = hi + lo, two halves) takes 4 R K bytes: units of 16 rows x 32 k,
// [R / 16][K / 32], 1 KB of hi and 1 KB of lo halves, each in the order in which a 16 x 16 x 32 matrix instruction takes
// them: lane l holds k 8 (l / 16) .. + 7 of row l % 16.
struct OrthoArea {
    int m, n, mp, np;
    int sub;                     // side of the sub-tiles X X^T is made of: 64 (128 x 128 tiles) or 32 (64 x 64 tiles)
    int sub_tiles;               // of those on and above the diagonal
    int splits;                  // parts that the long side is cut into for X X^T
    int parts_used;              // partial sums of squares
    bool apart;                  // squares hold zeros on their diagonals, which lie beside them in float32
    size_t parts, x, xt0, sq0, diag0, partial, bytes;
    size_t wide, square;         // bytes of an m x n and of an m x m matrix
    __host__ __device__ size_t xt(int i) const { return xt0 + i * wide; }
    __host__ __device__ size_t sq(int i) const { return sq0 + i * square; }
    __host__ __device__ size_t diag_of(int i) const { return diag0 + i * mp * sizeof(float); }
};
enum OrthoSquare { SQ_A0 = 0, SQ_A1 = 1, SQ_T = 2, SQ_P = 3, SQ_Q0 = 4, SQ_Q1 = 5 };

__host__ __device__ constexpr int ortho_triangle(int t) { return t * (t + 1) / 2; }

// Parts that the long side is cut into for X X^T: enough to give every CU two blocks, at least 256 each (a tile takes 1024
// whole in 12.8 us; in four parts 7.4, and adding those up 4.1).
inline int ortho_splits(int rows, int cols) {
    const int mp = ortho_padded(ortho_min(rows, cols)), np = ortho_padded(ortho_max(rows, cols));
    const int tiles = ortho_triangle(mp > 256 ? (mp + 127) / 128 : mp / 64);
    return ortho_max(1, ortho_min(512 / tiles, np / 256));
}

__host__ __device__ inline OrthoArea ortho_area(int rows, int cols, int splits) {
    OrthoArea a;
    a.m = rows < cols ? rows : cols;
    a.n = rows < cols ? cols : rows;
    a.mp = ortho_padded(a.m);
    a.np = ortho_padded(a.n);
    a.sub = a.mp > 256 ? 64 : 32;
    a.sub_tiles = ortho_triangle(a.mp / a.sub);
    a.splits = splits;
    a.apart = a.mp <= kOrthoSegmentRows;
    const long long count = (long long)rows * cols;
    a.parts_used = (int)(count / 4096 < 1 ? 1 : count / 4096 < kOrthoNormParts ? count / 4096 : kOrthoNormParts);
    a.wide = (size_t)a.mp * a.np * 4;
    a.square = (size_t)a.mp * a.mp * 4;
    size_t o = 0;
    a.parts = o; o += (size_t)kOrthoNormParts * sizeof(double);
    a.x = o; o += a.wide;
    a.xt0 = o; o += 2 * a.wide;
    a.sq0 = o; o += 6 * a.square;
    a.diag0 = o; o += 6 * a.mp * sizeof(float);
    a.partial = o;
    if (a.splits > 1) o += (size_t)a.splits * a.sub_tiles * a.sub * a.sub * sizeof(float);
    a.bytes = o;
    return a;
}
inline OrthoArea ortho_area(int rows, int cols) { return ortho_area(rows, cols, ortho_splits(rows, cols)); }

// A small matrix stays in one block's LDS from its first to its last step: X <- a X + (b A + c A^2) X as it is written.
constexpr int kOrthoSmallRows = 64, kOrthoSmallCols = 192;
struct OrthoSmallStep {
    float a_scale;               // 2^(k_A - 2 k_X)
    float b, c;                  // b 2^(k_B - k_A), c 2^(k_B - 2 k_A)
    float ax, y_scale;           // a 2^(k_B), 2^(k_X' - k_B - k_X); the last step's k_X' is 0
};
struct OrthoSmallSteps {
    float pow_kx;                // 2^(k_X) at the start
    OrthoSmallStep step[kOrthoMaxSteps];
};
__host__ __device__ inline bool ortho_is_small(int rows, int cols) {
    return ortho_min(rows, cols) <= kOrthoSmallRows && ortho_max(rows, cols) <= kOrthoSmallCols;
}
struct OrthoSegmentStep {
    float a, b, c;               // P = a I + b A + c A^2, times 2^(k_P), 2^(k_P - k_A), 2^(k_P - 2 k_A)
    float t_scale, a_scale;      // T = P A, A <- T P: 2^(k_out - k_f - k_g)
    float q_scale;               // Q <- P Q
};
struct OrthoSegmentSteps {
    int count;
    OrthoSegmentStep step[kOrthoSegment];
};

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

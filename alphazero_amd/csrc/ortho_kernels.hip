// Orthogonalisation by Newton-Schulz products, and the optimiser step built on it.
//
// X (m x n, m <= n, divided by its Frobenius norm) goes through k steps X <- p(A) X with A = X X^T and
// p(A) = a I + b A + c A^2.  p(A) commutes with A, so the steps can run on the m x m matrices alone: A <- p(A) A p(A),
// Q <- p(A) Q, and X is touched only to form A (X X^T) and to apply the product of the polynomials (Q X).  Rounding
// errors in A grow by up to a^2 a step in the directions of small singular values, so A is formed afresh from X after
// every kOrthoSegment = 3 steps: five steps (3 + 2) are as accurate as five plain ones (normal numbers, error over the
// result's size against the plain float32 form's: 200 x 3000 2.0e-6 / 1.8e-6, 1024 x 11520 1.5e-6 / 5.1e-6, 128 x 2048
// 5e-7 / 1.6e-6; one segment of five on a square matrix 1.6e-5 / 1.8e-6).
// All m x m matrices are symmetric: where a product is a launch, half of their tiles are computed and the other half
// mirrored.  Up to kOrthoSegmentRows rows their diagonals are held apart in float32 whichever kernel multiplies (beside
// a large matrix 100 x 130 is off by 7e-7 of the result, as alone; with the diagonals among the halves 2.1e-6).
//
// Arithmetic: every operand is value * 2^k = hi + lo, two halves (22 bits), and a product is three matrix
// instructions (hi lo + lo hi + hi hi) into float32.  The exponents k keep every entry below 2^15: the host bounds
// the matrices' spectral norms from the coefficients, an entry never exceeds them.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "lds_loads.h"
#include "mfma_tiles.h"
#include "numeric_types.h"

namespace nnb {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The item a block works on, and the block's index within it.
template <typename Group> __device__ __forceinline__ int find_item(const Group &g, int block, int &local) {
    int item = 0, start = 0;                             // without branches: one wait for all reads
#pragma unroll
    for (int i = 1; i < kOrthoItems; ++i) {
        const bool behind = block >= g.first[i];
        item += behind;
        start = behind ? g.first[i] : start;
    }
    local = block - start;
    return item;
}

// Consecutive logical blocks on one XCD (hardware deals blocks to the eight XCDs in turn), so that its L2 holds what
// neighbours share.
template <typename Group> __device__ __forceinline__ int xcd_block(const Group &g) {
    const unsigned total = g.blocks, each = total / 8, extra = total % 8, xcd = blockIdx.x % 8;
    return xcd * each + (xcd < extra ? xcd : extra) + blockIdx.x / 8;
}

// What is orthogonalised: the matrix itself, or the optimiser's new momentum (with Nesterov's look-ahead the gradient
// plus the new momentum's next share).
__device__ __forceinline__ float update_of(const OrthoParams &p, float g, float m_new) {
    if (!p.muon) return g;
    return p.nesterov ? g + p.mu * m_new : m_new;
}

// N consecutive elements in wide accesses; global memory takes them at any element's alignment.
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[N]; };

// Elements c .. c + N - 1 of a row of `cols`, zeros past its end.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T *row, long long cs, int c, int cols, float (&v)[N]) {
    if (cs == 1 && c + N <= cols) {
        const Pack<T, N> q = *reinterpret_cast<const Pack<T, N> *>(row + c);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = to_f32(q.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = c + e < cols ? to_f32(row[(c + e) * cs]) : 0.f;
    }
}

// Sum of squares of u, in double (a gradient's squares leave float32's range long before the gradient does), as partial
// sums that the next kernel adds in a fixed order; the optimiser step's new momentum is written on the way.  Bound by
// memory: 1024 x 11520 in float32 12.5 us (3.8 TB/s), 27.5 with the momentum (5.2 TB/s).
// The part `local` of a matrix, by 256 threads; all of the block meet here, those behind the last part too.
template <typename T>
__device__ __forceinline__ void norm_part(const OrthoGroup &g, const OrthoParams &p, const OrthoItem &it, int local, int tid, double *wave_sum) {
    constexpr int N = 16 / sizeof(T);
    const OrthoArea a = ortho_area(it.rows, it.cols, 1);
    const bool live = local < it.batch * a.parts_used;
    const int b = it.batch == 1 ? 0 : local / a.parts_used, part = local - b * a.parts_used;
    // a matrix without gaps is one long row
    const bool flat = it.x_cs == 1 && (it.x_rs == it.cols || it.rows == 1);
    const int rows = flat ? 1 : it.rows, cols = flat ? it.rows * it.cols : it.cols;
    const int per_row = (cols - 1) / N + 1;
    const unsigned total = (unsigned)rows * (unsigned)per_row;
    const T *x = static_cast<const T *>(it.x) + b * it.x_bs;
    double sum = 0.0;
    for (unsigned i = part * 256 + tid; live && i < total; i += a.parts_used * 256) {
        const unsigned r = flat ? 0 : i / per_row;
        const int c = (int)(i - r * per_row) * N;
        float v[N];
        load_row<T, N>(x + r * it.x_rs, it.x_cs, c, cols, v);
        if (p.muon) {                                            // flat
            float m[N];
            load_row<float, N>(it.momentum, 1, c, cols, m);
#pragma unroll
            for (int e = 0; e < N; ++e) m[e] = p.mu * m[e] + v[e];
            if (c + N <= cols) {
                Pack<float, N> q;
#pragma unroll
                for (int e = 0; e < N; ++e) q.v[e] = m[e];
                *reinterpret_cast<Pack<float, N> *>(it.momentum_out + c) = q;
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (c + e < cols) it.momentum_out[c + e] = m[e];
            }
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = update_of(p, v[e], m[e]);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum += (double)v[e] * (double)v[e];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((tid & 63) == 0) wave_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0 && live)
        reinterpret_cast<double *>(g.ws + it.ws + b * it.ws_stride + a.parts)[part] =
            (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
}
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoGroup g, OrthoParams p) {
    __shared__ double wave_sum[4];
    int local;
    const OrthoItem &it = g.item[find_item(g, blockIdx.x, local)];
    norm_part<T>(g, p, it, local, threadIdx.x, wave_sum);
}

__device__ __forceinline__ half8 pack_hi(const float (&v)[8], half8 &lo) {
    half8 hi;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (f16_t)v[e];
        lo[e] = (f16_t)(v[e] - (float)hi[e]);
    }
    return hi;
}

// sum[j] += a 16 x 16 block of 32 products: hi + lo halves of F's rows times those of N blocks of G's rows.
template <int N> __device__ __forceinline__ void add_to(half8 fh, half8 fl, const half8 (&gh)[N], const half8 (&gl)[N], f32x4 (&sum)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl, gh[j], sum[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh, gl[j], sum[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh, gh[j], sum[j], 0, 0, 0);
}
// The same from zero.
// The matrix unit aligns the products of an instruction, and the sum they are added to, to the largest of them and cuts
// off what lies more than 3 bits below that one's last place.  In a running sum this takes away from every product once
// the sum has grown (a diagonal entry of X X^T lost 2e-6 of itself over 2048 columns); from zero, with the small cross
// products first, what is cut is small against the stage's own sum.  ALL: the product of the lo halves too, which
// reaches 2^-22 of the whole and matters where one product makes up an entry, as on the diagonals of the squares.
template <int N, bool ALL>
__device__ __forceinline__ void add_products(half8 fh, half8 fl, const half8 (&gh)[N], const half8 (&gl)[N], f32x4 (&sum)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (ALL)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl, gl[j], sum[j], 0, 0, 0);
    add_to<N>(fh, fl, gh, gl, sum);
}

// Where lane l of unit (row block rb, k block kb) of a matrix with K columns finds its hi halves; the lo ones lie 1 KB on.
__device__ __forceinline__ size_t unit_offset(int rb, int kb, int k) { return ((size_t)rb * (k / 32) + kb) * 2048; }

// The numbers of a wave's tile in LDS (S x S, rows of `stride` floats) as hi + lo units of a matrix with K columns, the
// tile's first row being r0 and its first column c0: as they stand, or (TURNED) its transpose, whose first row is c0.
// change(v, row, column, unit, its number): last word on eight numbers of a row before they are rounded.
template <int S, bool TURNED, typename F>
__device__ __forceinline__ void emit_units(const float *tile, int stride, unsigned char *dst, int r0, int c0, int k, F &&change) {
    const int lane = threadIdx.x & 63;
    if (TURNED) { const int t = r0; r0 = c0; c0 = t; }
#pragma unroll
    for (int u = 0; u < S / 16 * (S / 32); ++u) {
        const int rb = u / (S / 32), kb = u % (S / 32);
        const int r = rb * 16 + (lane & 15), c = kb * 32 + (lane >> 4) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = TURNED ? tile[(c + e) * stride + r] : tile[r * stride + c + e];
        unsigned char *at = dst + unit_offset(r0 / 16 + rb, c0 / 32 + kb, k) + lane * 16;
        change(v, r0 + r, c0 + c, at, u);
        half8 lo;
        *reinterpret_cast<half8 *>(at) = pack_hi(v, lo);
        *reinterpret_cast<half8 *>(at + 1024) = lo;
    }
}
// Keeps the diagonal in float32 on the way; a square held apart (OrthoArea::apart) has zeros there in its units.
struct KeepDiagonal {
    float *diag;
    bool apart;
    __device__ __forceinline__ void operator()(float (&v)[8], int r, int c, unsigned char *, int) const {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (r == c + e) {
                diag[r] = v[e];
                if (apart) v[e] = 0.f;
            }
    }
};
struct Unchanged {
    __device__ __forceinline__ void operator()(float (&)[8], int, int, unsigned char *, int) const {}
};

// u / (|u| + eps) * 2^kx as units, X and its transpose, zero-padded.  One block per 64 x 64 tile.  Bound by memory:
// 1024 x 11520 in float32 26 us (5.5 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoGroup g, OrthoParams p, float pow_kx) {
    constexpr int N = 16 / sizeof(T), kStride = 68;
    __shared__ float tile[64 * kStride];
    __shared__ double wave_sum[4];
    int local;
    const OrthoItem &it = g.item[find_item(g, xcd_block(g), local)];
    const OrthoArea a = ortho_area(it.rows, it.cols, 1);
    const int rt = ortho_padded(it.rows) / 64, ct = ortho_padded(it.cols) / 64;
    const int b = local / (rt * ct), t = local % (rt * ct), r0 = t / ct * 64, c0 = t % ct * 64;
    unsigned char *area = g.ws + it.ws + b * it.ws_stride;
    const T *x = static_cast<const T *>(it.x) + b * it.x_bs;
    const int c = threadIdx.x % (64 / N) * N, rr = threadIdx.x / (64 / N);
    float u[16 / N][N];
#pragma unroll
    for (int i = 0; i < 16 / N; ++i) {
        const int r = r0 + rr + i * (256 / (64 / N));
        if (r < it.rows) {
            load_row<T, N>(x + r * it.x_rs, it.x_cs, c0 + c, it.cols, u[i]);
            if (p.muon) {
                float m[N];
                load_row<float, N>(it.momentum_out + (size_t)r * it.cols, 1, c0 + c, it.cols, m);
#pragma unroll
                for (int e = 0; e < N; ++e) u[i][e] = update_of(p, u[i][e], m[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) u[i][e] = 0.f;
        }
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.parts_used; i += 256) sum += reinterpret_cast<const double *>(area + a.parts)[i];
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    const double norm = sqrt((wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3])) + p.eps;
    const double scale = (double)pow_kx / norm;                  // leaves float32's range for very small matrices
#pragma unroll
    for (int i = 0; i < 16 / N; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
            tile[(rr + i * (256 / (64 / N))) * kStride + c + e] = (float)((double)u[i][e] * scale);
    __syncthreads();
    const bool tall = it.rows > it.cols;
    // each wave a 32 x 32 quarter, both ways round
    const int wave = threadIdx.x >> 6, qr = wave / 2 * 32, qc = wave % 2 * 32;
    const float *q = tile + qr * kStride + qc;
    emit_units<32, false>(q, kStride, area + (tall ? a.xt(0) : a.x), r0 + qr, c0 + qc, tall ? a.mp : a.np, Unchanged{});
    emit_units<32, true>(q, kStride, area + (tall ? a.x : a.xt(0)), r0 + qr, c0 + qc, tall ? a.np : a.mp, Unchanged{});
}

enum OrthoStage { STAGE_GRAM, STAGE_POLY, STAGE_MUL, STAGE_APPLY, STAGE_FINISH };

// Index of sub-tile (i, j), i <= j, of a symmetric matrix of `side` sub-tiles a side.
__device__ __forceinline__ int sub_tile(int i, int j, int side) { return i * side - i * (i - 1) / 2 + j - i; }

struct StageArgs {
    int f, g[2], out[2];         // squares: factors and result (MUL: up to two with the same first factor, by blockIdx.y;
                                 // POLY: A and P; GRAM: A; APPLY, FINISH: Q)
    int whole[2];                // POLY, MUL: the result is the segment's last Q, which keeps its diagonal in the units
    int xt;                      // which transposed planes APPLY / FINISH read (APPLY writes the other one)
    float out_scale[2];          // 2^(k_out - k_f - k_g); FINISH: 2^(-k_f - k_g)
    float a, b, c;               // POLY: coefficients, times 2^(k_out), 2^(k_out - k_A), 2^(k_out - 2 k_A)
};

// C = F G^T over K, both factors in units.  A block computes a tile of WR x WC sub-tiles (16 TB squared, one wave each)
// with KG groups of such waves that share K; a stage is 32 of K per group, brought to LDS by the loads themselves into a
// ring of RING stages; a wave reads a stage's operands into registers while it multiplies the one before, a read or a load
// behind every second product (of small tiles every product), and all waves meet once per stage.
//
// What bounds it: a CU takes in at most 64 bytes a clock (54 measured from L2, 18 to 24 from behind it), a 128 x 128
// tile loads 32 KB a stage for 768 clocks of products, and the two overlap only where several blocks share a CU: of 1024 x
// 1024 x 11520, loads alone take 50 us, products alone 46, both 73 with two blocks of four waves per CU.  One block per
// CU is slower whatever it gains in reuse or depth (97 us with a ring of five stages, 85 with 128 x 256 tiles on eight
// waves).  Reads and loads between the products, not in front of them, take X X^T of that size from 45 to 40 us and a
// product of squares (1024) from 12.2 to 11.4, and change nothing here.
template <int TB_, int WR_, int WC_, int KG_, int RING_> struct Shape {
    static constexpr int TB = TB_, WR = WR_, WC = WC_, KG = KG_, RING = RING_, kSub = 16 * TB, kRows = WR * kSub, kCols = WC * kSub,
                         kWaves = WR * WC * KG, kThreads = 64 * kWaves, kUnits = (WR + WC) * TB;
};
typedef Shape<4, 2, 2, 1, 2> LargeTile;                          // 128 x 128
typedef Shape<2, 2, 2, 1, 3> SmallTile;                          // 64 x 64, three blocks per CU
typedef Shape<2, 2, 2, 2, 4> LoneTile;                           // 64 x 64, two groups of waves, one block per CU

// Tiles of rows x cols that hold anything on or above the diagonal of an m x m matrix, and the tile of index `tile`.
template <typename S> __host__ __device__ inline int tiles_a_side(int mp) { return (mp + S::kRows - 1) / S::kRows; }
template <typename S> __host__ __device__ inline int upper_tiles(int mp) {
    static_assert(S::kRows == S::kCols, "");
    return ortho_triangle(tiles_a_side<S>(mp));
}

// What the squares of a call have in common: more than kOrthoLoRows rows or fewer each, all over kOrthoSegmentRows; or
// nothing, and every block looks at its own matrix.  (Looking costs 1024 x 11520 alone 1.4 %, three of 1501 x 777 2.4.)
enum OrthoKind { KIND_LARGE, KIND_MIDDLE, KIND_MIXED };

template <typename T, int STAGE, typename S, int KIND>
__device__ __forceinline__ void product(const OrthoShapes &g, const OrthoParams &p, const StageArgs &s, const OrthoGroup *items) {
    constexpr int TB = S::TB, RING = S::RING, kSub = S::kSub, kStride = kSub + 4, kUnits = S::kUnits, kGroup = S::WR * S::WC;
    constexpr bool symmetric = STAGE == STAGE_GRAM || STAGE == STAGE_POLY || STAGE == STAGE_MUL;
    constexpr int kStageBytes = S::KG * kUnits * 2048, kRingBytes = RING * kStageBytes, kOutBytes = kGroup * kSub * kStride * 4;
    constexpr int kPerWave = 2 * kUnits / kGroup;                // loads of 1 KB per stage: its group's, for its k
    static_assert(2 * kUnits % kGroup == 0, "whole loads");
    __shared__ __attribute__((aligned(16))) unsigned char lds[kRingBytes > kOutBytes ? kRingBytes : kOutBytes];
    int local;
    const int index = find_item(g, xcd_block(g), local);
    const OrthoShape &it = g.item[index];
    const OrthoArea a = ortho_area(it.rows, it.cols, it.splits);
    const int mt = tiles_a_side<S>(a.mp), nt = (a.np + S::kCols - 1) / S::kCols;
    const int tiles = symmetric ? upper_tiles<S>(a.mp) : mt * nt;
    int part = 0;
    if (STAGE == STAGE_GRAM && a.splits > 1) { part = local / tiles % a.splits; local = local / (tiles * a.splits) * tiles + local % tiles; }
    const int batch = it.batch == 1 ? 0 : local / tiles;
    int ti = 0, tj = local - batch * tiles;
    if (symmetric) {
        while (tj >= mt - ti) tj -= mt - ti++;
        tj += ti;
    } else {
        ti = tj % mt;
        tj /= mt;
    }
    unsigned char *area = g.ws + it.ws + batch * it.ws_stride;
    const int which = STAGE == STAGE_MUL ? blockIdx.y : 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = wave / kGroup, in_group = wave % kGroup, wr = in_group / S::WC, wc = in_group % S::WC;
    const int r0 = ti * S::kRows + wr * kSub, c0 = tj * S::kCols + wc * kSub;
    // What the matrix unit does not see: POLY's lower terms, and where the diagonals are held apart the products with them,
    // F G = O_F O_G + D_F O_G + O_F D_G + D_F D_G (POLY: both factors are A).  Small tiles read their part of the factors
    // while they wait for the first operands (five matrices of up to 515 rows, one step: 155 us without, 132 so).
    constexpr bool kRest = STAGE == STAGE_POLY || STAGE == STAGE_MUL, kAhead = kRest && TB == 2 && KIND == KIND_MIXED;
    constexpr int kTileUnits = kSub / 16 * (kSub / 32);
    struct Part { half8 f[2], g[2]; float df, dg[8]; };          // of a unit: hi and lo halves, diagonals
    Part ahead[kAhead ? kTileUnits : 1];
    const bool apart = kRest && KIND == KIND_MIXED && a.apart;
    const int f_square = s.f, g_square = STAGE == STAGE_MUL ? s.g[which] : s.f;
    auto read_part = [&](Part &part, int r, int c, size_t at) {
        auto units = [&](int square, half8 (&to)[2]) {
            const unsigned char *from = area + a.sq(square) + at;
            to[0] = *reinterpret_cast<const half8 *>(from), to[1] = *reinterpret_cast<const half8 *>(from + 1024);
        };
        if (STAGE == STAGE_POLY || apart) units(f_square, part.f);
        if (!apart) return;
        if (STAGE == STAGE_MUL) units(g_square, part.g);
        part.df = reinterpret_cast<const float *>(area + a.diag_of(f_square))[r];
        const f32x4 *dg = reinterpret_cast<const f32x4 *>(area + a.diag_of(g_square) + c * sizeof(float));
#pragma unroll
        for (int e = 0; e < 8; ++e) part.dg[e] = dg[e / 4][e % 4];
    };
    if constexpr (kAhead) {
        if (kg == 0 && r0 <= c0 && c0 < a.mp)
#pragma unroll
            for (int u = 0; u < kTileUnits; ++u) {
                const int rb = u / (kSub / 32), kb = u % (kSub / 32);
                read_part(ahead[u], r0 + rb * 16 + (lane & 15), c0 + kb * 32 + (lane >> 4) * 8,
                          unit_offset(r0 / 16 + rb, c0 / 32 + kb, a.mp) + lane * 16);
            }
    }
    f32x4 acc[TB][TB] = {};
    {
        const int kdim = STAGE == STAGE_GRAM ? a.np : a.mp, k_units = kdim / 32;
        int k0 = 0, k1 = k_units;                                // a multiple of 64: whole stages, an even number of 32s
        if (STAGE == STAGE_GRAM) {
            k0 = (int)((long long)(k_units / 4) * part / a.splits) * 4;
            k1 = part + 1 == a.splits ? k_units : (int)((long long)(k_units / 4) * (part + 1) / a.splits) * 4;
        }
        const unsigned char *f = area + (STAGE == STAGE_GRAM ? a.x : a.sq(s.f));
        const unsigned char *h = STAGE == STAGE_GRAM ? f : STAGE == STAGE_POLY ? f : STAGE == STAGE_MUL ? area + a.sq(s.g[which])
                                                                                            : area + a.xt(s.xt);
        const int f_rows = a.mp / 16 - 1, h_rows = (symmetric ? a.mp : a.np) / 16 - 1;
        const unsigned char *source[kPerWave];                   // this wave's kilobytes of a stage; past the end the last rows again
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int d = in_group * kPerWave + i, u = d / 2;
            source[i] = uniform((u < S::WR * TB ? f + unit_offset(ortho_min(ti * S::WR * TB + u, f_rows), k0 + kg, kdim)
                                                : h + unit_offset(ortho_min(tj * S::WC * TB + u - S::WR * TB, h_rows), k0 + kg, kdim)) +
                                d % 2 * 1024);
        }
        const int stages = (k1 - k0) / S::KG;
        auto issue = [&](int t, int slot, int i) {
            load_to_lds(source[i] + (size_t)t * (S::KG * 2048), lane * 16,
                        lds + slot * kStageBytes + kg * kUnits * 2048 + (in_group * kPerWave + i) * 1024);
        };
        half8 fh[2][TB], fl[2][TB], hh[2][TB], hl[2][TB];
        auto fragment = [&](int slot, auto to, auto which_read) {     // read r of 4 * TB
            constexpr int B = to, R = which_read, I = R / 4;
            const unsigned char *base = lds + slot * kStageBytes + kg * kUnits * 2048 + lane * 16;
            const unsigned char *fu = base + (wr * TB + I) * 2048, *hu = base + ((S::WR + wc) * TB + I) * 2048;
            if constexpr (R % 4 == 0) fl[B][I] = *reinterpret_cast<const half8 *>(fu + 1024);
            if constexpr (R % 4 == 1) hh[B][I] = *reinterpret_cast<const half8 *>(hu);
            if constexpr (R % 4 == 2) fh[B][I] = *reinterpret_cast<const half8 *>(fu);
            if constexpr (R % 4 == 3) hl[B][I] = *reinterpret_cast<const half8 *>(hu + 1024);
        };
        // Every stage's sum from zero, smallest products first, added up by the vector pipe (see add_products).  On large
        // tiles a row of blocks at a time; the four blocks of small ones together, since a block's products wait for each
        // other, and added while the next stage multiplies (three 832 x 832 x 832: 17.0 us by rows, 16.1 so).
        constexpr bool kFromZero = STAGE == STAGE_POLY || STAGE == STAGE_MUL || STAGE == STAGE_GRAM;
        auto run = [&](auto with_lo) __attribute__((always_inline)) {
            constexpr bool kAll = with_lo;                       // products of lo halves too (see add_products)
            f32x4 sum[2][TB][TB] = {};
            auto nothing = [](auto) {};
            constexpr int kMemory = 4 * TB + kPerWave, kEvery = 3 * TB * TB / kMemory;      // reads and loads of a step
            static_assert(kMemory * kEvery == 3 * TB * TB && (4 * TB) == 2 * kPerWave, "between the products, two reads and a load in turn");
            auto multiply_with = [&](auto from, auto &&between) {    // between(n), n < kMemory, behind every kEvery products
                constexpr int B = from;
                if constexpr (TB == 2) {
                    f32x4 (&to)[TB][TB] = kFromZero ? sum[B] : acc;
                    if constexpr (kFromZero)
#pragma unroll
                        for (int i = 0; i < TB * TB; ++i) to[i / TB][i % TB] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if constexpr (kAll)
#pragma unroll
                        for (int i = 0; i < TB * TB; ++i)
                            to[i / TB][i % TB] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[B][i / TB], hl[B][i % TB], to[i / TB][i % TB], 0, 0, 0);
                    static_for<3 * TB * TB>([&](auto index) {
                        constexpr int N = index, P = N / (TB * TB), I = N / TB % TB, J = N % TB;
                        to[I][J] = __builtin_amdgcn_mfma_f32_16x16x32_f16(P == 0 ? fl[B][I] : fh[B][I], P == 1 ? hl[B][J] : hh[B][J], to[I][J], 0, 0, 0);
                        asm volatile("" : "+v"(to[I][J]));           // holds it between the reads and loads around it
                        if constexpr (N % kEvery == kEvery - 1) between(std::integral_constant<int, N / kEvery>{});
                    });
                    if constexpr (kFromZero)
#pragma unroll
                        for (int i = 0; i < TB * TB; ++i) acc[i / TB][i % TB] += sum[1 - B][i / TB][i % TB];
                } else {
                    static_for<TB>([&](auto row) {
                        constexpr int I = row;
                        f32x4 (&to)[TB] = kFromZero ? sum[0][I & 1] : acc[I];
                        if constexpr (kFromZero) {
#pragma unroll
                            for (int j = 0; j < TB; ++j) to[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                            if constexpr (kAll)
#pragma unroll
                                for (int j = 0; j < TB; ++j) to[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[B][I], hl[B][j], to[j], 0, 0, 0);
                        }
                        static_for<3 * TB>([&](auto index) {
                            constexpr int P = index / TB, J = index % TB, N = (I * 3 + P) * TB + J;
                            to[J] = __builtin_amdgcn_mfma_f32_16x16x32_f16(P == 0 ? fl[B][I] : fh[B][I], P == 1 ? hl[B][J] : hh[B][J], to[J], 0, 0, 0);
                            asm volatile("" : "+v"(to[J]));
                            if constexpr (N % kEvery == kEvery - 1) between(std::integral_constant<int, N / kEvery>{});
                        });
                        if constexpr (kFromZero && I > 0)
#pragma unroll
                            for (int j = 0; j < TB; ++j) acc[I - 1][j] += sum[0][(I - 1) & 1][j];
                    });
                    if constexpr (kFromZero)
#pragma unroll
                        for (int j = 0; j < TB; ++j) acc[TB - 1][j] += sum[0][(TB - 1) & 1][j];
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            auto multiply = [&](auto from) { multiply_with(from, nothing); };
            auto add_last = [&](auto from) {
                constexpr int B = from;
                if constexpr (TB == 2 && kFromZero)
#pragma unroll
                    for (int i = 0; i < TB; ++i)
#pragma unroll
                        for (int j = 0; j < TB; ++j) acc[i][j] += sum[B][i][j];
            };
            constexpr int kInFlight = (RING - 2) * kPerWave;         // a wave's loads behind the stage it waits for
            // behind the last stage the last again, never read: so many loads are in flight behind a stage throughout
            auto at_most = [&](int t) { return t < stages ? t : stages - 1; };
            constexpr std::integral_constant<int, 0> even{};
            constexpr std::integral_constant<int, 1> odd{};
#pragma unroll
            for (int t = 0; t < RING - 1; ++t)
#pragma unroll
                for (int d = 0; d < kPerWave; ++d) issue(at_most(t), t, d);
            wait_and_meet<kInFlight>();
#pragma unroll
            for (int d = 0; d < kPerWave; ++d) issue(at_most(RING - 1), RING - 1, d);
            static_for<4 * TB>([&](auto r) { fragment(0, even, r); });
            int slot = 0;
            auto step = [&](int t, auto from, auto to) {             // multiplies stage t, reads stage t + 1
                const int next = slot + 1 == RING ? 0 : slot + 1;
                wait_and_meet<kInFlight>();
                const int ahead = at_most(t + RING);
                multiply_with(from, [&](auto n) {
                    constexpr int N = n;
                    if constexpr (N % 3 == 2) issue(ahead, slot, N / 3);
                    else fragment(next, to, std::integral_constant<int, N - N / 3>{});
                });
                slot = next;
            };
            // pairs of stages, for the two sets of registers; an odd last one by itself
            int t = 0;
            for (; t + 2 < stages; t += 2) {
                step(t, even, odd);
                step(t + 1, odd, even);
            }
            if (t + 1 < stages) {
                step(t, even, odd);
                multiply(odd);
                add_last(odd);
            } else {
                multiply(even);
                add_last(even);
            }
        };
        // The matrix chooses, not the launch: its precision does not depend on what else is in the call.
        if constexpr (STAGE == STAGE_POLY || STAGE == STAGE_MUL) {
            if (KIND == KIND_MIDDLE || (KIND == KIND_MIXED && a.mp <= kOrthoLoRows)) run(std::true_type{});
            else run(std::false_type{});
        } else {
            run(std::false_type{});
        }
    }

    // The groups' sums meet in the first one's registers, its results in LDS, every wave's in its own part (free once all
    // waves have read their last operands and their last loads have landed).
    wait_and_meet<0>();
    float *mine = reinterpret_cast<float *>(lds) + in_group * kSub * kStride;
    static_assert(S::KG <= 2, "");
    if (S::KG == 2) {
        f32x4 *sums = reinterpret_cast<f32x4 *>(lds) + in_group * TB * TB * 64 + lane;
        if (kg == 1)
#pragma unroll
            for (int i = 0; i < TB * TB; ++i) sums[i * 64] = acc[i / TB][i % TB];
        __syncthreads();
        if (kg == 0)
#pragma unroll
            for (int i = 0; i < TB * TB; ++i) acc[i / TB][i % TB] += sums[i * 64];
        __syncthreads();
        if (kg == 1) return;
    }
    // behind the padding, or below the diagonal, where the mirror image of another sub-tile goes
    if (r0 >= a.mp || c0 >= (symmetric ? a.mp : a.np) || (symmetric && r0 > c0)) return;
    if (STAGE == STAGE_GRAM && a.splits > 1) {
        f32x4 *partials = reinterpret_cast<f32x4 *>(area + a.partial) + ((size_t)part * a.sub_tiles + sub_tile(r0 / kSub, c0 / kSub, a.mp / kSub)) * TB * TB * 64 + lane;
#pragma unroll
        for (int i = 0; i < TB * TB; ++i) partials[i * 64] = acc[i / TB][i % TB];
        return;
    }
    const float out_scale = STAGE == STAGE_POLY ? s.c : s.out_scale[which];
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mine[(16 * i + 4 * (lane >> 4) + e) * kStride + 16 * j + (lane & 15)] = acc[i][j][e] * out_scale;
    if constexpr (symmetric) {
        unsigned char *dst = area + a.sq(s.out[which]);
        if constexpr (STAGE == STAGE_POLY || STAGE == STAGE_MUL) {
            float *d_out = reinterpret_cast<float *>(area + a.diag_of(s.out[which]));
            const bool whole = s.whole[which];
            auto add_rest = [&](float (&v)[8], int r, int c, unsigned char *at, int u) {
                float *keep = mine + (r - r0) * kStride + c - c0;         // for the mirror image
                Part part;
                if constexpr (kAhead) part = ahead[u];
                else read_part(part, r, c, at - dst);
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (float)part.f[0][e] + (float)part.f[1][e];
                if constexpr (STAGE == STAGE_POLY) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += s.b * f[e] + (r == c + e ? s.a : 0.f);
                }
                if (apart) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float g_e = STAGE == STAGE_MUL ? (float)part.g[0][e] + (float)part.g[1][e] : f[e];
                        v[e] += out_scale * (part.df * g_e + f[e] * part.dg[e]);
                        if (r == c + e) {
                            v[e] += out_scale * (part.df * part.dg[e]) + (STAGE == STAGE_POLY ? s.b * part.df : 0.f);
                            d_out[r] = v[e];
                            if (!whole) v[e] = 0.f;
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) keep[e] = v[e];
            };
            if (STAGE == STAGE_POLY || apart) emit_units<kSub, false>(mine, kStride, dst, r0, c0, a.mp, add_rest);
            else emit_units<kSub, false>(mine, kStride, dst, r0, c0, a.mp, Unchanged{});
        } else {
            if (r0 == c0)
                emit_units<kSub, false>(mine, kStride, dst, r0, c0, a.mp, KeepDiagonal{reinterpret_cast<float *>(area + a.diag_of(s.out[0])), a.apart});
            else
                emit_units<kSub, false>(mine, kStride, dst, r0, c0, a.mp, Unchanged{});
        }
        if (r0 != c0) emit_units<kSub, true>(mine, kStride, dst, r0, c0, a.mp, Unchanged{});
    } else if constexpr (STAGE == STAGE_APPLY) {
        emit_units<kSub, false>(mine, kStride, area + a.x, r0, c0, a.np, Unchanged{});
        emit_units<kSub, true>(mine, kStride, area + a.xt(1 - s.xt), r0, c0, a.mp, Unchanged{});
    } else {
        const OrthoItem &o = items->item[index];
        const bool tall = o.rows > o.cols;                       // then the tile is the transpose of the result's
        T *out = static_cast<T *>(o.out) + batch * o.o_bs;
        const int ur0 = tall ? c0 : r0, uc0 = tall ? r0 : c0;
#pragma unroll 2
        for (int q = lane; q < kSub * kSub / 4; q += 64) {
            const int i = q / (kSub / 4), j = q % (kSub / 4) * 4, ur = ur0 + i, uc = uc0 + j;
            if (ur >= o.rows || uc >= o.cols) continue;
            float v[4], w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = tall ? mine[(j + e) * kStride + i] : mine[i * kStride + j + e];
            if (p.muon) {
                load_row<T, 4>(static_cast<const T *>(o.weight) + (size_t)ur * o.cols, 1, uc, o.cols, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = w[e] * p.decay - o.scale * v[e];
            }
            T *to = out + ur * o.o_rs;
            if (o.o_cs == 1 && uc + 4 <= o.cols) {
                Pack<T, 4> r;
#pragma unroll
                for (int e = 0; e < 4; ++e) r.v[e] = from_f32<T>(v[e]);
                *reinterpret_cast<Pack<T, 4> *>(to + uc) = r;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (uc + e < o.cols) to[(uc + e) * o.o_cs] = from_f32<T>(v[e]);
            }
        }
    }
}

template <int STAGE, typename S, int KIND>
__global__ __launch_bounds__(S::kThreads, 2) void ortho_product_kernel(OrthoShapes g, OrthoParams p, StageArgs s) {
    product<float, STAGE, S, KIND>(g, p, s, nullptr);
}
template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads, 2) void ortho_finish_kernel(OrthoShapes g, OrthoParams p, StageArgs s, OrthoGroup items) {
    product<T, STAGE_FINISH, S, KIND_MIXED>(g, p, s, &items);
}

// Adds up the parts of X X^T, one block of four waves per sub-tile (16 TB squared), and lays it out both ways round.
// Bound by latency: 1024 x 1024 in 14 parts 8.5 us, 128 x 128 in 8 parts 4.1.
template <int TB>
__global__ __launch_bounds__(256) void ortho_reduce_kernel(OrthoShapes g, StageArgs s) {
    constexpr int kSub = 16 * TB, kStride = kSub + 4, kEach = TB * TB / 4;
    __shared__ float tile[kSub * kStride];
    int local;
    const OrthoShape &it = g.item[find_item(g, blockIdx.x, local)];
    const OrthoArea a = ortho_area(it.rows, it.cols, it.splits);
    const int batch = it.batch == 1 ? 0 : local / a.sub_tiles, index = local - batch * a.sub_tiles, side = a.mp / kSub;
    int ti = 0, tj = index;
    while (tj >= side - ti) tj -= side - ti++;
    tj += ti;
    unsigned char *area = g.ws + it.ws + batch * it.ws_stride;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const f32x4 *partials = reinterpret_cast<const f32x4 *>(area + a.partial) + ((size_t)index * TB * TB + wave * kEach) * 64 + lane;
    f32x4 sum[kEach] = {};
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k)
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum[i] += partials[((size_t)k * a.sub_tiles * TB * TB + i) * 64];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int b = wave * kEach + i;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            tile[(16 * (b / TB) + 4 * (lane >> 4) + e) * kStride + 16 * (b % TB) + (lane & 15)] = sum[i][e] * s.out_scale[0];
    }
    __syncthreads();
    // a wave takes a quarter of the units, each way round
    unsigned char *dst = area + a.sq(s.out[0]);
    const KeepDiagonal keep{reinterpret_cast<float *>(area + a.diag_of(s.out[0])), a.apart};       // (off the diagonal nothing is kept)
    constexpr int kQuarter = kSub / 2;
    const int qr = wave / 2 * kQuarter, qc = wave % 2 * kQuarter;
    if constexpr (kQuarter >= 32) {
        const float *q = tile + qr * kStride + qc;
        emit_units<kQuarter, false>(q, kStride, dst, ti * kSub + qr, tj * kSub + qc, a.mp, keep);
        if (ti != tj) emit_units<kQuarter, true>(q, kStride, dst, ti * kSub + qr, tj * kSub + qc, a.mp, Unchanged{});
    } else {
        if (wave == 0) emit_units<kSub, false>(tile, kStride, dst, ti * kSub, tj * kSub, a.mp, keep);
        if (wave == 1 && ti != tj) emit_units<kSub, true>(tile, kStride, dst, ti * kSub, tj * kSub, a.mp, Unchanged{});
    }
}

// ------------------------------------------------------------------------------------- matrices in one block's LDS
//
// A square's results come four rows of one column to a lane: eight bytes of hi and of lo halves of the transposed
// matrix's units, which for a symmetric matrix is the matrix.
//
// A square M is kept as D + O: its diagonal in float32, the units hold the rest with zeros there, and
//     F G = D_F D_G + D_F O_G + O_F D_G + O_F O_G
// of which only the last goes through the matrix unit.  The diagonal is what is large in these matrices: in the products
// it costs halves their last bits and makes the matrix unit cut off the small ones (see add_products), errors that the
// recursion on A then multiplies (100 x 130 of normal numbers: 2.4e-6 of the result's size with the diagonal in the units).

// Address of lane (row r, k .. k + 3) in units of a matrix with K columns.
__device__ __forceinline__ int unit_bytes(int r, int k, int kdim) {
    return ((r / 16) * (kdim / 32) + k / 32) * 2048 + ((k % 32 / 8) * 16 + r % 16) * 16 + k % 8 * 2;
}
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void put4(unsigned char *unit, f32x4 v) {
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = (f16_t)v[e];
        lo[e] = (f16_t)(v[e] - (float)hi[e]);
    }
    *reinterpret_cast<half4 *>(unit) = hi;
    *reinterpret_cast<half4 *>(unit + 1024) = lo;
}
__device__ __forceinline__ f32x4 get4(const unsigned char *unit) {
    const half4 hi = *reinterpret_cast<const half4 *>(unit), lo = *reinterpret_cast<const half4 *>(unit + 1024);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)hi[e] + (float)lo[e];
    return v;
}
// Four rows r .. r + 3 of column c of a square with K columns, as D + O in units and a float32 diagonal.
__device__ __forceinline__ void put_square(unsigned char *units, float *diag, int r, int c, int kdim, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (r + e == c) {
            diag[c] = v[e];
            v[e] = 0.f;
        }
    put4(units + unit_bytes(c, r, kdim), v);
}
// acc += rows rb of F times rows cb .. cb + N - 1 (blocks of 16) of G, both units with K columns, k_units of 32 of them.
template <int N>
__device__ __forceinline__ void multiply_units(const unsigned char *f, const unsigned char *g, int rb, int cb, int kdim, int k_units,
                                               f32x4 (&acc)[N]) {
    const int lane = threadIdx.x & 63, ku = kdim / 32;
    for (int k = 0; k < k_units; ++k) {
        const unsigned char *fu = f + (rb * ku + k) * 2048 + lane * 16;
        const half8 fh = *reinterpret_cast<const half8 *>(fu), fl = *reinterpret_cast<const half8 *>(fu + 1024);
        half8 gh[N], gl[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const unsigned char *gu = g + ((cb + j) * ku + k) * 2048 + lane * 16;
            gh[j] = *reinterpret_cast<const half8 *>(gu);
            gl[j] = *reinterpret_cast<const half8 *>(gu + 1024);
        }
        add_to<N>(fh, fl, gh, gl, acc);
    }
}

// A whole matrix (m <= 64, n <= NP) in one block of sixteen waves: the twenty launches of the long way would cost a small
// matrix several times what it computes.  What bounds it is the chain of a step: three products, each behind a barrier.
// So a wave has one block of 16 of a square, its parts of A and X stay in float32 registers, blocks of padding are left
// out, and X Y's tiles come out of the matrix unit both ways round, for the two orders of units they are stored in
// (128 x 32, five steps: 28.0 us with two blocks to a wave, values read back from LDS and halves scattered, now 21.5).
// Beside larger matrices their norms are taken in the same launch, four parts to a block (the step of the network with
// two launches 536 us, so 516).
template <typename T, int NP>
__global__ __launch_bounds__(1024) void ortho_small_kernel(OrthoGroup g, OrthoParams p, OrthoSmallSteps steps) {
    constexpr int M = kOrthoSmallRows, kWide = M * NP * 4, kSquare = M * M * 4, TN = NP / 64;
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * kWide + 2 * kSquare + 2 * M * 4];
    unsigned char *x = lds, *xt = lds + kWide, *sq_a = lds + 2 * kWide, *sq_b = sq_a + kSquare;
    float *diag_a = reinterpret_cast<float *>(sq_b + kSquare), *diag_b = diag_a + M;
    int batch;
    const OrthoItem &it = g.item[find_item(g, blockIdx.x, batch)];
    if (!ortho_is_small(it.rows, it.cols)) {
        norm_part<T>(g, p, it, batch * 4 + threadIdx.x / 256, threadIdx.x % 256, reinterpret_cast<double *>(lds) + threadIdx.x / 256 * 4);
        return;
    }
    const bool tall = it.rows > it.cols;
    const int m = tall ? it.cols : it.rows, n = tall ? it.rows : it.cols;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const T *src = static_cast<const T *>(it.x) + batch * it.x_bs;
    const long long rs = tall ? it.x_cs : it.x_rs, cs = tall ? it.x_rs : it.x_cs;
    // X is u or its transpose; a thread takes eight columns of a row
    constexpr int kPer = (M * NP / 8 + 1023) / 1024;
    float u[kPer][8];
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const int at = q * 1024 + tid, i = at / (NP / 8), j = at % (NP / 8) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = 0.f;
            if (i < m && j + e < n) {                            // (i >= 64 behind the last part)
                v = to_f32(src[i * rs + (j + e) * cs]);
                if (p.muon) {
                    const size_t o = tall ? (size_t)(j + e) * it.cols + i : (size_t)i * it.cols + j + e;
                    const float m_new = p.mu * it.momentum[o] + v;
                    it.momentum_out[o] = m_new;
                    v = update_of(p, v, m_new);
                }
            }
            u[q][e] = v;
            sum += (double)v * (double)v;
        }
    }
    double *wave_sum = reinterpret_cast<double *>(sq_a);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) wave_sum[wave] = sum;
    __syncthreads();
    double norm = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w) norm += wave_sum[w];
    const double scale = (double)steps.pow_kx / (sqrt(norm) + p.eps);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        const int at = q * 1024 + tid, i = at / (NP / 8), j = at % (NP / 8) * 8;
        if (i >= M) break;
        float v[8];
        half8 lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)((double)u[q][e] * scale);
        const half8 hi = pack_hi(v, lo);
        unsigned char *row = x + unit_bytes(i, j, NP);
        *reinterpret_cast<half8 *>(row) = hi;
        *reinterpret_cast<half8 *>(row + 1024) = lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            unsigned char *turned = xt + unit_bytes(j + e, i, M);
            *reinterpret_cast<f16_t *>(turned) = hi[e];
            *reinterpret_cast<f16_t *>(turned + 1024) = lo[e];
        }
    }
    __syncthreads();
    // This wave's block (rb, cb) of a square and its TN blocks of X: (rb, nb + j).  A lane holds four rows of a column, of
    // X's blocks turned round four columns of a row too.  What lies behind m, n rounded up to 32 is zero and left out.
    const int rb = wave / 4, cb = wave % 4, nb = wave % 4 * TN, mk = (m + 31) / 32, nk = (n + 31) / 32;
    const int row = rb * 16 + (lane >> 4) * 4, col = cb * 16 + (lane & 15), turned_row = rb * 16 + (lane & 15);
    const bool in_square = rb < 2 * mk && cb < 2 * mk, diagonal = rb == cb;
    auto x_col = [&](int j) { return (nb + j) * 16 + (lane & 15); };
    auto x_turned_col = [&](int j) { return (nb + j) * 16 + (lane >> 4) * 4; };
    f32x4 own_x[TN], own_turned[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        own_x[j] = get4(xt + unit_bytes(x_col(j), row, M));
        own_turned[j] = get4(x + unit_bytes(turned_row, x_turned_col(j), NP));
    }
    for (int s = 0; s < p.steps; ++s) {
        const OrthoSmallStep &st = steps.step[s];
        f32x4 own_a[1] = {};
        if (in_square) {
            multiply_units<1>(x, x, rb, cb, NP, nk, own_a);
            own_a[0] *= st.a_scale;
            if (diagonal) put_square(sq_a, diag_a, row, col, M, own_a[0]);
            else put4(sq_a + unit_bytes(col, row, M), own_a[0]);
        }
        __syncthreads();
        if (in_square) {
            f32x4 b[1] = {};
            multiply_units<1>(sq_a, sq_a, rb, cb, M, mk, b);
            f32x4 off = own_a[0];
            if (diagonal)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row + e == col) off[e] = 0.f;
            const f32x4 df = *reinterpret_cast<const f32x4 *>(diag_a + row);
            b[0] = own_a[0] * st.b + (b[0] + df * own_a[0] + off * diag_a[col]) * st.c;
            if (diagonal) put_square(sq_b, diag_b, row, col, M, b[0]);
            else put4(sq_b + unit_bytes(col, row, M), b[0]);
        }
        __syncthreads();
        f32x4 y[TN] = {}, turned[TN] = {};
        if (rb < 2 * mk) {
#pragma unroll 1
            for (int k = 0; k < mk; ++k) {
                const unsigned char *fu = sq_b + (rb * (M / 32) + k) * 2048 + lane * 16;
                const half8 fh = *reinterpret_cast<const half8 *>(fu), fl = *reinterpret_cast<const half8 *>(fu + 1024);
                half8 gh[TN], gl[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const unsigned char *gu = xt + ((nb + j) * (M / 32) + k) * 2048 + lane * 16;
                    gh[j] = *reinterpret_cast<const half8 *>(gu), gl[j] = *reinterpret_cast<const half8 *>(gu + 1024);
                }
                add_to<TN>(fh, fl, gh, gl, y);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    turned[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(gh[j], fl, turned[j], 0, 0, 0);
                    turned[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(gl[j], fh, turned[j], 0, 0, 0);
                    turned[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(gh[j], fh, turned[j], 0, 0, 0);
                }
            }
            const f32x4 db = *reinterpret_cast<const f32x4 *>(diag_b + row);
            const float db_turned = diag_b[turned_row];
#pragma unroll
            for (int j = 0; j < TN; ++j) {                              // (a + D_B) X + O_B X
                own_x[j] = y[j] = ((db + st.ax) * own_x[j] + y[j]) * st.y_scale;
                own_turned[j] = ((db_turned + st.ax) * own_turned[j] + turned[j]) * st.y_scale;
            }
        }
        if (s + 1 < p.steps) {
            __syncthreads();                                            // everybody has read the old X
            if (rb < 2 * mk)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    put4(xt + unit_bytes(x_col(j), row, M), own_x[j]);
                    put4(x + unit_bytes(turned_row, x_turned_col(j), NP), own_turned[j]);
                }
            __syncthreads();
            continue;
        }
        T *out = static_cast<T *>(it.out) + batch * it.o_bs;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = row + e, c = x_col(j);
                if (i >= m || c >= n) continue;
                const int ur = tall ? c : i, uc = tall ? i : c;
                float v = y[j][e];
                if (p.muon) v = to_f32(static_cast<const T *>(it.weight)[(size_t)ur * it.cols + uc]) * p.decay - it.scale * v;
                out[ur * it.o_rs + uc * it.o_cs] = from_f32<T>(v);
            }
    }
}

// All products of a segment for a matrix with m <= 128 in one block, a wave per B x B blocks of 16: A comes from memory, Q
// goes there.  The units of A (then T, then the next A) and of P stay in LDS, Q's are read back from memory; every wave
// keeps its own part of A, P and Q in float32 registers, so that the products with the diagonals cost two operations per
// element: read back from the units, they and the conversions took most of the time (128 x 128, three steps: 43.5 us, now
// 29.4; their matrix instructions alone 12).
template <int MP, int B>
__global__ __launch_bounds__(MP / 16 / B * (MP / 16 / B) * 64) void ortho_segment_kernel(OrthoShapes g, OrthoSegmentSteps steps, int a_from,
                                                                                      int q_to) {
    constexpr int kSquare = MP * MP * 4, kSide = MP / 16 / B;
    __shared__ __attribute__((aligned(16))) unsigned char sq_a[kSquare], sq_p[kSquare];
    __shared__ __attribute__((aligned(16))) float diag_a[MP], diag_t[MP], diag_p[MP], diag_q[2][MP];
    int batch;
    const OrthoShape &it = g.item[find_item(g, blockIdx.x, batch)];
    const OrthoArea area = ortho_area(it.rows, it.cols, it.splits);
    if (area.mp != MP) return;                                           // the other size's launch takes it
    unsigned char *ws = g.ws + it.ws + batch * it.ws_stride;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rb = wave / kSide * B, cb = wave % kSide * B;              // this wave's first blocks
    const bool diagonal = rb == cb;                                      // its blocks i, i hold the diagonal
    auto row = [&](int i) { return (rb + i) * 16 + (lane >> 4) * 4; };
    auto col = [&](int j) { return (cb + j) * 16 + (lane & 15); };
    auto at = [&](int i, int j) { return unit_bytes(col(j), row(i), MP); };
    typedef f32x4 Part[B][B];
    Part own_a, own_p, own_q, acc;
    auto store = [&](unsigned char *to, float *diag, const Part &v) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) {
                if (diagonal && i == j) put_square(to, diag, row(i), col(j), MP, v[i][j]);
                else put4(to + at(i, j), v[i][j]);
            }
    };
    // acc = scale F G
    auto product = [&](const unsigned char *f, const float *diag_f, const Part &own_f, const unsigned char *h, const float *diag_h,
                       const Part &own_h, float scale) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int k = 0; k < MP / 32; ++k) {
            half8 fh[B], fl[B], gh[B], gl[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const unsigned char *fu = f + ((rb + i) * (MP / 32) + k) * 2048 + lane * 16, *gu = h + ((cb + i) * (MP / 32) + k) * 2048 + lane * 16;
                fh[i] = *reinterpret_cast<const half8 *>(fu), fl[i] = *reinterpret_cast<const half8 *>(fu + 1024);
                gh[i] = *reinterpret_cast<const half8 *>(gu), gl[i] = *reinterpret_cast<const half8 *>(gu + 1024);
            }
#pragma unroll
            for (int i = 0; i < B; ++i) add_to<B>(fh[i], fl[i], gh, gl, acc[i]);
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const f32x4 df = *reinterpret_cast<const f32x4 *>(diag_f + row(i));
#pragma unroll
            for (int j = 0; j < B; ++j) {
                f32x4 of = own_f[i][j];
                if (diagonal && i == j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (row(i) + e == col(j)) of[e] = 0.f;
                acc[i][j] = (acc[i][j] + df * own_h[i][j] + of * diag_h[col(j)]) * scale;
            }
        }
    };
    const float *diag = reinterpret_cast<const float *>(ws + area.diag_of(a_from));
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
        for (int j = 0; j < B; ++j) {
            own_a[i][j] = get4(ws + area.sq(a_from) + at(i, j));
            if (diagonal && i == j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row(i) + e == col(j)) own_a[i][j][e] = diag[col(j)];
        }
    store(sq_a, diag_a, own_a);
    __syncthreads();
    // Q alternates between two places so that the last one, whole, is q_to
    int q = (steps.count & 1) ? q_to : (q_to == SQ_Q0 ? SQ_Q1 : SQ_Q0);
    auto store_q = [&](bool last) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) own_q[i][j] = acc[i][j];
        if (!last) {
            store(ws + area.sq(q), diag_q[q == SQ_Q1], own_q);
            return;
        }
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) put4(ws + area.sq(q) + at(i, j), own_q[i][j]);
    };
    for (int s = 0; s < steps.count; ++s) {
        const OrthoSegmentStep &st = steps.step[s];
        const bool last = s + 1 == steps.count;
        product(sq_a, diag_a, own_a, sq_a, diag_a, own_a, st.c);
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) {
                acc[i][j] += own_a[i][j] * st.b;
                if (diagonal && i == j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] += row(i) + e == col(j) ? st.a : 0.f;
                own_p[i][j] = acc[i][j];
            }
        store(sq_p, diag_p, own_p);
        if (s == 0) store_q(last);                                       // the first step's P is Q
        __syncthreads();
        if (s > 0) {
            product(sq_p, diag_p, own_p, ws + area.sq(q), diag_q[q == SQ_Q1], own_q, st.q_scale);
            q = q == SQ_Q0 ? SQ_Q1 : SQ_Q0;
            store_q(last);
        }
        if (last) break;
        product(sq_p, diag_p, own_p, sq_a, diag_a, own_a, st.t_scale);
        __syncthreads();                                                 // everybody has read A
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) own_a[i][j] = acc[i][j];
        store(sq_a, diag_t, own_a);                                      // T
        __syncthreads();
        product(sq_a, diag_t, own_a, sq_p, diag_p, own_p, st.a_scale);
        __syncthreads();                                                 // everybody has read T
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) own_a[i][j] = acc[i][j];
        store(sq_a, diag_a, own_a);
        __syncthreads();
    }
}

// Largest magnitudes on [0, rho]: of p, of l p(l) and of l p(l)^2, p(l) = c0 + c1 l + c2 l^2.  They lie at the ends or where a
// derivative vanishes: p', p + l p' = c0 + 2 c1 l + 3 c2 l^2, and p + 2 l p' = c0 + 3 c1 l + 5 c2 l^2 (or p itself, a zero).
void polynomial_bounds(const float *c, double rho, double &p_max, double &lp_max, double &lpp_max) {
    p_max = lp_max = lpp_max = 0.0;
    auto at = [&](double l) {
        if (!(l >= 0.0 && l <= rho)) return;
        const double v = std::fabs(c[0] + c[1] * l + c[2] * l * l);
        p_max = std::fmax(p_max, v);
        lp_max = std::fmax(lp_max, l * v);
        lpp_max = std::fmax(lpp_max, l * v * v);
    };
    auto roots = [&](double q0, double q1, double q2) {          // of q0 + q1 l + q2 l^2
        if (q2 == 0.0) { if (q1 != 0.0) at(-q0 / q1); return; }
        const double d = q1 * q1 - 4.0 * q2 * q0;
        if (d < 0.0) return;
        at((-q1 + std::sqrt(d)) / (2.0 * q2));
        at((-q1 - std::sqrt(d)) / (2.0 * q2));
    };
    at(0.0);
    at(rho);
    roots(c[1], 2.0 * c[2], 0.0);
    roots(c[0], 2.0 * c[1], 3.0 * c[2]);
    roots(c[0], 3.0 * c[1], 5.0 * c[2]);
}

// Largest k <= 14 with bound * 2^k <= 2^15 (halves reach 2^16: the rest is room for rounding).
int exponent_for(double bound) {
    int k = 14;
    while (k > -60 && bound * std::ldexp(1.0, k) > 32768.0) --k;
    return k;
}

}  // namespace

bool ortho_coefficients_ok(const OrthoParams &p) {
    double rho = 1.0, q = 1.0;
    for (int i = 0; i < p.steps; ++i) {
        double pm, lp, lpp;
        polynomial_bounds(p.coef[i], rho * 1.001, pm, lp, lpp);
        if (i % kOrthoSegment == 0) q = 1.0;
        q *= pm;
        // beyond these bounds the halves would run out of range; a sequence that converges stays far below
        if (!(q <= 4096.0) || !(lpp <= 4096.0) || !(lp <= 4096.0)) return false;
        rho = std::fmax(lpp, 1e-6);
    }
    return true;
}

namespace {

template <typename S> int all_tiles(const OrthoArea &a) {
    return (a.mp + S::kRows - 1) / S::kRows * ((a.np + S::kCols - 1) / S::kCols);
}

// The small matrices of the group, and the others' norms.
void launch_small(hipStream_t st, OrthoGroup &g, const OrthoParams &p) {
    OrthoSmallSteps steps = {};
    double rho = 1.0;
    int kx = exponent_for(1.0), blocks = 0, widest = 0;
    steps.pow_kx = (float)std::ldexp(1.0, kx);
    for (int i = 0; i < p.steps; ++i) {
        const float *c = p.coef[i];
        double p_max, lp_max, lpp_max;
        polynomial_bounds(c, rho * 1.001, p_max, lp_max, lpp_max);
        // |b l + c l^2| <= |p| + |a|
        const int ka = exponent_for(rho), kb = exponent_for(p_max + std::fabs(c[0]));
        const int kn = i + 1 < p.steps ? exponent_for(std::sqrt(std::fmax(lpp_max, 1e-6))) : 0;
        OrthoSmallStep &s = steps.step[i];
        s.a_scale = (float)std::ldexp(1.0, ka - 2 * kx);
        s.b = (float)std::ldexp(c[1], kb - ka);
        s.c = (float)std::ldexp(c[2], kb - 2 * ka);
        s.ax = (float)std::ldexp(c[0], kb);
        s.y_scale = (float)std::ldexp(1.0, kn - kb - kx);
        kx = kn;
        rho = std::fmax(lpp_max, 1e-6);
    }
    for (int i = 0; i < g.count; ++i) {
        const OrthoItem &it = g.item[i];
        g.first[i] = blocks;
        if (ortho_is_small(it.rows, it.cols)) {
            blocks += it.batch;
            widest = ortho_max(widest, ortho_max(it.rows, it.cols));
        } else {
            blocks += (it.batch * ortho_area(it.rows, it.cols, 1).parts_used + 3) / 4;
        }
    }
    for (int i = g.count; i < kOrthoItems; ++i) g.first[i] = INT32_MAX;
    g.blocks = blocks;
    with_dtype(p.type, [&](auto type) {
        typedef decltype(type) T;
        if (widest <= 64) ortho_small_kernel<T, 64><<<blocks, 1024, 0, st>>>(g, p, steps);
        else if (widest <= 128) ortho_small_kernel<T, 128><<<blocks, 1024, 0, st>>>(g, p, steps);
        else ortho_small_kernel<T, kOrthoSmallCols><<<blocks, 1024, 0, st>>>(g, p, steps);
    });
}

}  // namespace

void launch_orthogonalize(hipStream_t st, OrthoGroup &g, const OrthoParams &p) {
    int smalls = 0;                                              // they come first
    while (smalls < g.count && ortho_is_small(g.item[smalls].rows, g.item[smalls].cols)) ++smalls;
    if (smalls) {
        launch_small(st, g, p);
        if (smalls == g.count) return;
        std::copy(g.item + smalls, g.item + g.count, g.item);
        g.count -= smalls;
    }
    bool segments = true;
    for (int i = 0; i < g.count; ++i) segments &= ortho_min(g.item[i].rows, g.item[i].cols) <= kOrthoSegmentRows;
    OrthoShapes shapes = {};
    shapes.count = g.count;
    shapes.ws = g.ws;
    auto with_tile = [](int k, auto &&f) {
        if (k == 0) f(LargeTile{});
        else if (k == 1) f(SmallTile{});
        else f(LoneTile{});
    };
    long long upper[2] = {}, full[2] = {};
    int smallest = INT32_MAX, largest = 0;
    bool any64 = false, any128 = false, gram_of[2] = {}, reduce_of[2] = {};
    for (int i = 0; i < g.count; ++i) {
        const OrthoItem &it = g.item[i];
        const OrthoArea a = ortho_area(it.rows, it.cols);
        shapes.item[i] = {it.ws, it.ws_stride, it.rows, it.cols, it.batch, a.splits};
        for (int k = 0; k < 2; ++k)
            with_tile(k, [&](auto shape) {
                typedef decltype(shape) S;
                upper[k] += (long long)it.batch * upper_tiles<S>(a.mp);
                full[k] += (long long)it.batch * all_tiles<S>(a);
            });
        smallest = ortho_min(smallest, a.mp);
        largest = ortho_max(largest, a.mp);
        any64 |= a.mp == 64;
        any128 |= a.mp == 128;
        gram_of[a.sub == 64] = true;
        reduce_of[a.sub == 64] |= a.splits > 1;
    }
    // Large tiles where they give most CUs at least one; where even small ones give no CU two, two groups share each
    // (one product of squares: 1024, 136 small tiles, 13.9 us with two groups, 17.1 without; 832 three times, 273 tiles,
    // 22.4 and 16.4.  Q X of 832 x 1536 three times, 252 large tiles: 27.7, 31.8 on small ones).
    auto pick = [](const long long (&n)[2]) { return n[0] >= 200 ? 0 : n[1] > 256 ? 1 : 2; };
    const int kind = smallest > kOrthoLoRows ? KIND_LARGE : smallest > kOrthoSegmentRows && largest <= kOrthoLoRows ? KIND_MIDDLE : KIND_MIXED;
    const int symmetric_tile = pick(upper), full_tile = pick(full);
    auto blocks = [&](auto &group, auto per_matrix) {
        int n = 0;
        for (int i = 0; i < g.count; ++i) {
            group.first[i] = n;
            n += g.item[i].batch * per_matrix(ortho_area(g.item[i].rows, g.item[i].cols));
        }
        for (int i = g.count; i < kOrthoItems; ++i) group.first[i] = INT32_MAX;
        group.blocks = n;
        return n;
    };
    auto squares = [&] {
        int n = 0;
        with_tile(symmetric_tile, [&](auto tile) { n = blocks(shapes, [](const OrthoArea &a) { return upper_tiles<decltype(tile)>(a.mp); }); });
        return n;
    };
    auto whole = [&] {
        int n = 0;
        with_tile(full_tile, [&](auto tile) {
            typedef decltype(tile) S;
            n = blocks(shapes, [](const OrthoArea &a) { return all_tiles<S>(a); });
        });
        return n;
    };
    auto launch = [&](auto stage, int tile, dim3 grid, const StageArgs &s) {
        constexpr int STAGE = stage;
        with_tile(tile, [&](auto shape) {
            typedef decltype(shape) S;
            auto of_kind = [&](auto k) { ortho_product_kernel<STAGE, S, k><<<grid, S::kThreads, 0, st>>>(shapes, p, s); };
            if constexpr (STAGE == STAGE_POLY || STAGE == STAGE_MUL) {
                if (kind == KIND_LARGE) of_kind(std::integral_constant<int, KIND_LARGE>{});
                else if (kind == KIND_MIDDLE) of_kind(std::integral_constant<int, KIND_MIDDLE>{});
                else of_kind(std::integral_constant<int, KIND_MIXED>{});
            } else {
                of_kind(std::integral_constant<int, KIND_MIXED>{});
            }
        });
    };
    auto gram = [&](const StageArgs &s) {
        for (int large = 0; large < 2; ++large) {
            if (!gram_of[large]) continue;
            auto mine = [&](const OrthoArea &a) { return (a.sub == 64) == (large == 1); };
            int n = blocks(shapes, [&](const OrthoArea &a) {
                return !mine(a) ? 0 : (large ? upper_tiles<LargeTile>(a.mp) : upper_tiles<SmallTile>(a.mp)) * a.splits; });
            launch(std::integral_constant<int, STAGE_GRAM>{}, large ? 0 : 1, n, s);
            if (!reduce_of[large]) continue;
            n = blocks(shapes, [&](const OrthoArea &a) { return mine(a) && a.splits > 1 ? a.sub_tiles : 0; });
            if (large) ortho_reduce_kernel<4><<<n, 256, 0, st>>>(shapes, s);
            else ortho_reduce_kernel<2><<<n, 256, 0, st>>>(shapes, s);
        }
    };
    with_dtype(p.type, [&](auto type) {
        typedef decltype(type) T;
        int n = blocks(g, [](const OrthoArea &a) { return a.parts_used; });
        if (!smalls) ortho_norm_kernel<T><<<n, 256, 0, st>>>(g, p);
        double rho = 1.0;                       // bound of A's largest eigenvalue
        int kx = exponent_for(1.0), xt = 0;
        n = blocks(g, [](const OrthoArea &a) { return a.mp / 64 * (a.np / 64); });
        ortho_split_kernel<T><<<n, 256, 0, st>>>(g, p, (float)std::ldexp(1.0, kx));
        for (int s0 = 0; s0 < p.steps; s0 += kOrthoSegment) {
            const int len = p.steps - s0 < kOrthoSegment ? p.steps - s0 : kOrthoSegment;
            StageArgs s = {};
            int ka = exponent_for(rho), kq = 0, cur = SQ_A0, q = SQ_P;
            s.out[0] = cur;
            s.out_scale[0] = (float)std::ldexp(1.0, ka - 2 * kx);
            gram(s);
            n = squares();
            double q_max = 1.0;
            OrthoSegmentSteps all = {};
            all.count = len;
            const int a_from = cur;
            for (int i = 0; i < len; ++i) {
                const float *c = p.coef[s0 + i];
                double p_max, lp_max, lpp_max;
                polynomial_bounds(c, rho * 1.001, p_max, lp_max, lpp_max);
                // the first step's P is the segment's Q
                const int kp = exponent_for(p_max), pout = i == 0 ? SQ_Q0 : SQ_P;
                s.f = cur; s.out[0] = pout; s.whole[0] = len == 1;
                s.a = (float)std::ldexp(c[0], kp); s.b = (float)std::ldexp(c[1], kp - ka); s.c = (float)std::ldexp(c[2], kp - 2 * ka);
                all.step[i].a = s.a; all.step[i].b = s.b; all.step[i].c = s.c;
                if (!segments) launch(std::integral_constant<int, STAGE_POLY>{}, symmetric_tile, n, s);
                q_max *= p_max;
                // T = P A and Q <- P Q in one launch, then A <- T P
                int pair = 0;
                s.f = pout;
                const int kt = exponent_for(lp_max);
                if (i + 1 < len) {
                    s.g[pair] = cur; s.out[pair] = SQ_T; s.whole[pair] = 0;
                    s.out_scale[pair++] = all.step[i].t_scale = (float)std::ldexp(1.0, kt - kp - ka);
                }
                if (i == 0) {
                    q = SQ_Q0; kq = kp;
                } else {
                    const int kn = exponent_for(q_max), next = q == SQ_Q0 ? SQ_Q1 : SQ_Q0;
                    s.g[pair] = q; s.out[pair] = next; s.whole[pair] = i + 1 == len;
                    s.out_scale[pair++] = all.step[i].q_scale = (float)std::ldexp(1.0, kn - kp - kq);
                    q = next; kq = kn;
                }
                if (pair && !segments)
                    launch(std::integral_constant<int, STAGE_MUL>{}, symmetric_tile == 2 && n * pair > 256 ? 1 : symmetric_tile, dim3(n, pair), s);
                if (i + 1 < len) {
                    const int kn = exponent_for(lpp_max), next = cur == SQ_A0 ? SQ_A1 : SQ_A0;
                    s.f = SQ_T; s.g[0] = pout; s.out[0] = next; s.whole[0] = 0;
                    s.out_scale[0] = all.step[i].a_scale = (float)std::ldexp(1.0, kn - kt - kp);
                    if (!segments) launch(std::integral_constant<int, STAGE_MUL>{}, symmetric_tile, dim3(n, 1), s);
                    cur = next; ka = kn;
                }
                rho = std::fmax(lpp_max, 1e-6);
            }
            if (segments) {
                n = blocks(shapes, [](const OrthoArea &) { return 1; });
                if (any64) ortho_segment_kernel<64, 1><<<n, 1024, 0, st>>>(shapes, all, a_from, q);
                if (any128) ortho_segment_kernel<128, 2><<<n, 1024, 0, st>>>(shapes, all, a_from, q);
            }
            s.f = q; s.xt = xt;
            n = whole();
            if (s0 + len < p.steps) {
                const int kn = exponent_for(std::sqrt(rho));
                s.out_scale[0] = (float)std::ldexp(1.0, kn - kq - kx);
                launch(std::integral_constant<int, STAGE_APPLY>{}, full_tile, n, s);
                kx = kn;
                xt = 1 - xt;
            } else {
                s.out_scale[0] = (float)std::ldexp(1.0, -kq - kx);
                with_tile(full_tile, [&](auto shape) {
                    typedef decltype(shape) S;
                    ortho_finish_kernel<T, S><<<n, S::kThreads, 0, st>>>(shapes, p, s, g);
                });
            }
        }
    });
}

}  // namespace nnb

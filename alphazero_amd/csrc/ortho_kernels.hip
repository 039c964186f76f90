// Orthogonalisation by Newton-Schulz products, and the optimiser step built on it.
//
// X (m x n, m <= n, divided by its Frobenius norm) goes through k steps X <- p(A) X with A = X X^T and
// p(A) = a I + b A + c A^2.  p(A) commutes with A, so the steps can run on the m x m matrices alone: A <- p(A) A p(A),
// Q <- p(A) Q, and X is touched only to form A (X X^T) and to apply the product of the polynomials (Q X).  Rounding
// errors in A grow by up to a^2 a step in the directions of small singular values, so A is formed afresh from X after
// every kOrthoSegment = 3 steps: five steps (3 + 2) are as accurate as five plain ones (float32, 256 x 1024 of
// normal numbers: 3e-6 of the result's size against 2e-6; one segment of five on a square matrix: 1.6e-5 against 1.8e-6).
// All m x m matrices are symmetric: half of their tiles are computed, the other half mirrored.
//
// Arithmetic: every operand is value * 2^k = hi + lo, two halves (22 bits), and a product is three matrix
// instructions (hi lo + lo hi + hi hi) into float32.  The exponents k keep every entry below 2^15: the host bounds
// the matrices' spectral norms from the coefficients, an entry never exceeds them.
#include <hip/hip_runtime.h>
#include <stdint.h>

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
    int i = 0;
    while (i + 1 < g.count && block >= g.first[i + 1]) ++i;
    local = block - g.first[i];
    return i;
}

// Consecutive logical blocks on one XCD (hardware deals blocks to the eight XCDs in turn), so that its L2 holds what
// neighbours share.
__device__ __forceinline__ int xcd_block() {
    const int total = gridDim.x, each = total / 8, extra = total % 8, xcd = blockIdx.x % 8;
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
// sums that the next kernel adds in a fixed order; the optimiser step's new momentum is written on the way.
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoGroup g, OrthoParams p) {
    constexpr int N = 16 / sizeof(T);
    int local;
    const OrthoItem &it = g.item[find_item(g, blockIdx.x, local)];
    const OrthoArea a = ortho_area(it.rows, it.cols);
    const int b = local / a.parts_used, part = local % a.parts_used;
    // a matrix without gaps is one long row
    const bool flat = it.x_cs == 1 && (it.x_rs == it.cols || it.rows == 1);
    const int rows = flat ? 1 : it.rows, cols = flat ? it.rows * it.cols : it.cols;
    const int per_row = (cols - 1) / N + 1;
    const unsigned total = (unsigned)rows * (unsigned)per_row;
    const T *x = static_cast<const T *>(it.x) + b * it.x_bs;
    double sum = 0.0;
    for (unsigned i = part * 256 + threadIdx.x; i < total; i += a.parts_used * 256) {
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
    __shared__ double wave_sum[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        reinterpret_cast<double *>(g.ws + it.ws + b * it.ws_stride + a.parts)[part] =
            (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
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

// Where lane l of unit (row block rb, k block kb) of a matrix with K columns finds its hi halves; the lo ones lie 1 KB on.
__device__ __forceinline__ size_t unit_offset(int rb, int kb, int k) { return ((size_t)rb * (k / 32) + kb) * 2048; }

// The numbers of a wave's tile in LDS (S x S, rows of `stride` floats) as hi + lo units of a matrix with K columns, the
// tile's first row being r0 and its first column c0: as they stand, or (TURNED) its transpose, whose first row is c0.
// change(v, row, column, unit): last word on eight numbers of a row before they are rounded.
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
        change(v, r0 + r, c0 + c, at);
        half8 lo;
        *reinterpret_cast<half8 *>(at) = pack_hi(v, lo);
        *reinterpret_cast<half8 *>(at + 1024) = lo;
    }
}
struct Unchanged {
    __device__ __forceinline__ void operator()(float (&)[8], int, int, unsigned char *) const {}
};

// u / (|u| + eps) * 2^kx as units, X and its transpose, zero-padded.  One block per 64 x 64 tile.
template <typename T>
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoGroup g, OrthoParams p, float pow_kx) {
    constexpr int N = 16 / sizeof(T), kStride = 68;
    __shared__ float tile[64 * kStride];
    __shared__ double wave_sum[4];
    int local;
    const OrthoItem &it = g.item[find_item(g, xcd_block(), local)];
    const OrthoArea a = ortho_area(it.rows, it.cols);
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

enum OrthoStage { STAGE_GRAM, STAGE_REDUCE, STAGE_POLY, STAGE_MUL, STAGE_APPLY, STAGE_FINISH };

struct StageArgs {
    int f, g[2], out[2];         // squares: factors and result (MUL: up to two with the same first factor, by blockIdx.y;
                                 // POLY: A and P; GRAM: A; APPLY, FINISH: Q)
    int xt;                      // which transposed planes APPLY / FINISH read (APPLY writes the other one)
    float out_scale[2];          // 2^(k_out - k_f - k_g); FINISH: 2^(-k_f - k_g)
    float a, b, c;               // POLY: coefficients, times 2^(k_out), 2^(k_out - k_A), 2^(k_out - 2 k_A)
};

// C = F G^T over K, both factors in units.  A block computes a tile of 32 * TB squared with 2 x 2 waves; a stage is 32 of K,
// brought to LDS by the loads themselves into a ring of RING stages; a wave reads a stage's operands into registers
// while it multiplies the one before, and all waves meet once per stage.  48 matrix instructions (TB = 4) stand against
// 16 LDS reads.
template <typename T, int STAGE, int TB, int RING>
__device__ __forceinline__ void product(const OrthoShapes &g, const OrthoParams &p, const StageArgs &s, const OrthoGroup *items) {
    constexpr int kTile = 32 * TB, kSub = 16 * TB, kStride = kSub + 4, kUnits = 4 * TB;
    constexpr bool symmetric = STAGE == STAGE_GRAM || STAGE == STAGE_REDUCE || STAGE == STAGE_POLY || STAGE == STAGE_MUL;
    constexpr int kRingBytes = STAGE == STAGE_REDUCE ? 0 : RING * kUnits * 2048, kOutBytes = 4 * kSub * kStride * 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[kRingBytes > kOutBytes ? kRingBytes : kOutBytes];
    int local;
    const int index = find_item(g, xcd_block(), local);
    const OrthoShape &it = g.item[index];
    const OrthoArea a = ortho_area(it.rows, it.cols);
    const int mt = (a.mp + kTile - 1) / kTile, nt = (a.np + kTile - 1) / kTile;
    const int tiles = symmetric ? ortho_triangle(mt) : mt * nt;
    int part = 0;
    if (STAGE == STAGE_GRAM) { part = local / tiles % a.splits; local = local / (tiles * a.splits) * tiles + local % tiles; }
    const int batch = local / tiles, tile = local % tiles;
    int ti = 0, tj;
    if (symmetric) {
        int t = tile;
        while (t >= mt - ti) { t -= mt - ti; ++ti; }
        tj = ti + t;
    } else {
        ti = tile % mt;
        tj = tile / mt;
    }
    unsigned char *area = g.ws + it.ws + batch * it.ws_stride;
    const int which = STAGE == STAGE_MUL ? blockIdx.y : 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / 2 * kSub, wc = wave % 2 * kSub;
    f32x4 acc[TB][TB] = {};
    f32x4 *partials = reinterpret_cast<f32x4 *>(area + a.partial) + ((size_t)tile * 4 + wave) * TB * TB * 64 + lane;
    const size_t partial_stride = (size_t)tiles * 4 * TB * TB * 64;

    if constexpr (STAGE == STAGE_REDUCE) {
        for (int k = 0; k < a.splits; ++k)
#pragma unroll
            for (int i = 0; i < TB * TB; ++i) acc[i / TB][i % TB] += partials[k * partial_stride + i * 64];
    } else {
        const int kdim = STAGE == STAGE_GRAM ? a.np : a.mp, k_units = kdim / 32;
        int k0 = 0, k1 = k_units;                                // an even number of k-steps
        if (STAGE == STAGE_GRAM) {
            k0 = (int)((long long)(k_units / 2) * part / a.splits) * 2;
            k1 = (int)((long long)(k_units / 2) * (part + 1) / a.splits) * 2;
        }
        const unsigned char *f = area + (STAGE == STAGE_GRAM ? a.x : a.sq(s.f));
        const unsigned char *h = STAGE == STAGE_GRAM ? f : STAGE == STAGE_POLY ? f : STAGE == STAGE_MUL ? area + a.sq(s.g[which])
                                                                                            : area + a.xt(s.xt);
        const int f_rows = a.mp / 16 - 1, h_rows = (symmetric ? a.mp : a.np) / 16 - 1;
        const unsigned char *source[TB];                         // this wave's units of a stage; past the end the last again
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int u = wave * TB + i;
            source[i] = uniform(u < 2 * TB ? f + unit_offset(ortho_min(ti * 2 * TB + u, f_rows), k0, kdim)
                                           : h + unit_offset(ortho_min(tj * 2 * TB + u - 2 * TB, h_rows), k0, kdim));
        }
        const int stages = k1 - k0;
        auto issue = [&](int t, int slot) {
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    load_to_lds(source[i] + (size_t)t * 2048 + j * 1024, lane * 16, lds + (slot * kUnits + wave * TB + i) * 2048 + j * 1024);
        };
        half8 fh[2][TB], fl[2][TB], hh[2][TB], hl[2][TB];
        auto fragments = [&](int slot, auto to) {
            constexpr int B = to;
            const unsigned char *base = lds + slot * kUnits * 2048 + lane * 16;
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const unsigned char *fu = base + (wave / 2 * TB + i) * 2048, *hu = base + (2 * TB + wave % 2 * TB + i) * 2048;
                fh[B][i] = *reinterpret_cast<const half8 *>(fu);
                fl[B][i] = *reinterpret_cast<const half8 *>(fu + 1024);
                hh[B][i] = *reinterpret_cast<const half8 *>(hu);
                hl[B][i] = *reinterpret_cast<const half8 *>(hu + 1024);
            }
        };
        auto multiply = [&](auto from) {
            constexpr int B = from;
            // the three products of an entry stand TB * TB instructions apart: none waits for the one before
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[B][i], hh[B][j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[B][i], hl[B][j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[B][i], hh[B][j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        constexpr int kInFlight = (RING - 2) * 2 * TB;           // a wave's loads behind the stage it waits for
        auto meet = [&](bool all_issued) {
            if (all_issued) wait_and_meet<kInFlight>();
            else wait_and_meet<0>();
        };
        constexpr std::integral_constant<int, 0> even{};
        constexpr std::integral_constant<int, 1> odd{};
#pragma unroll
        for (int t = 0; t < RING - 1; ++t)
            if (t < stages) issue(t, t);
        meet(RING - 1 <= stages);
        if (RING - 1 < stages) issue(RING - 1, RING - 1);
        fragments(0, even);
        int slot = 0;
        auto step = [&](int t, auto from, auto to) {             // multiplies stage t, reads stage t + 1
            const int next = slot + 1 == RING ? 0 : slot + 1;
            meet(t + RING <= stages);
            if (t + RING < stages) issue(t + RING, slot);
            fragments(next, to);
            multiply(from);
            slot = next;
        };
        int t = 0;
        for (; t + 2 < stages; t += 2) {
            step(t, even, odd);
            step(t + 1, odd, even);
        }
        step(t, even, odd);
        multiply(odd);
        if (STAGE == STAGE_GRAM && a.splits > 1) {
#pragma unroll
            for (int i = 0; i < TB * TB; ++i) partials[part * partial_stride + i * 64] = acc[i / TB][i % TB];
            return;
        }
    }

    // A wave's results meet in its own part of LDS (free once all waves have read their last operands).
    __syncthreads();
    float *mine = reinterpret_cast<float *>(lds) + wave * kSub * kStride;
    const float out_scale = STAGE == STAGE_POLY ? s.c : s.out_scale[which];
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mine[(16 * i + 4 * (lane >> 4) + e) * kStride + 16 * j + (lane & 15)] = acc[i][j][e] * out_scale;
    const int r0 = ti * kTile + wr, c0 = tj * kTile + wc;
    if (r0 >= a.mp || c0 >= (symmetric ? a.mp : a.np)) return;   // behind the padding
    if constexpr (symmetric) {
        unsigned char *dst = area + a.sq(s.out[which]);
        if constexpr (STAGE == STAGE_POLY) {
            const unsigned char *from = area + a.sq(s.f);
            auto add_lower = [&](float (&v)[8], int r, int c, unsigned char *at) {
                const half8 hi = *reinterpret_cast<const half8 *>(from + (at - dst)), lo = *reinterpret_cast<const half8 *>(from + (at - dst) + 1024);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += s.b * ((float)hi[e] + (float)lo[e]) + (r == c + e ? s.a : 0.f);
            };
            emit_units<kSub, false>(mine, kStride, dst, r0, c0, a.mp, add_lower);
            if (ti != tj) emit_units<kSub, true>(mine, kStride, dst, r0, c0, a.mp, add_lower);
        } else {
            emit_units<kSub, false>(mine, kStride, dst, r0, c0, a.mp, Unchanged{});
            if (ti != tj) emit_units<kSub, true>(mine, kStride, dst, r0, c0, a.mp, Unchanged{});
        }
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

template <int STAGE, int TB, int RING>
__global__ __launch_bounds__(256, 2) void ortho_product_kernel(OrthoShapes g, OrthoParams p, StageArgs s) {
    product<float, STAGE, TB, RING>(g, p, s, nullptr);
}
template <typename T, int TB, int RING>
__global__ __launch_bounds__(256, 2) void ortho_finish_kernel(OrthoShapes g, OrthoParams p, StageArgs s, OrthoGroup items) {
    product<T, STAGE_FINISH, TB, RING>(g, p, s, &items);
}

// Largest magnitudes on [0, rho]: of p, of l p(l) and of l p(l)^2.
void polynomial_bounds(const float *c, double rho, double &p_max, double &lp_max, double &lpp_max) {
    p_max = lp_max = lpp_max = 0.0;
    for (int i = 0; i <= 4096; ++i) {
        const double l = rho * i / 4096.0, v = std::fabs(c[0] + c[1] * l + c[2] * l * l);
        p_max = std::fmax(p_max, v);
        lp_max = std::fmax(lp_max, l * v);
        lpp_max = std::fmax(lpp_max, l * v * v);
    }
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

void launch_orthogonalize(hipStream_t st, OrthoGroup &g, const OrthoParams &p) {
    OrthoShapes shapes = {};
    shapes.count = g.count;
    shapes.ws = g.ws;
    long long symmetric128 = 0, full128 = 0;
    bool reduce = false, large_gram = false;
    for (int i = 0; i < g.count; ++i) {
        const OrthoItem &it = g.item[i];
        const OrthoArea a = ortho_area(it.rows, it.cols);
        shapes.item[i] = {it.ws, it.ws_stride, it.rows, it.cols, it.batch};
        const int mt = (a.mp + 127) / 128, nt = (a.np + 127) / 128;
        symmetric128 += (long long)it.batch * ortho_triangle(mt);
        full128 += (long long)it.batch * mt * nt;
        reduce |= a.splits > 1;
        large_gram |= a.tile == 128;
    }
    // Tiles of 128 need half the LDS traffic, tiles of 64 give four times the blocks: 128 where they fill the chip.
    const int symmetric_tile = symmetric128 >= 200 ? 128 : 64, full_tile = full128 >= 200 ? 128 : 64;
    auto blocks = [&](auto &group, auto per_matrix) {
        int n = 0;
        for (int i = 0; i < g.count; ++i) {
            group.first[i] = n;
            n += g.item[i].batch * per_matrix(ortho_area(g.item[i].rows, g.item[i].cols), g.item[i]);
        }
        group.first[g.count] = n;
        return n;
    };
    auto squares = [&] {
        return blocks(shapes, [&](const OrthoArea &a, const OrthoItem &) { return ortho_triangle((a.mp + symmetric_tile - 1) / symmetric_tile); });
    };
    auto whole = [&] {
        return blocks(shapes, [&](const OrthoArea &a, const OrthoItem &) { return (a.mp + full_tile - 1) / full_tile * ((a.np + full_tile - 1) / full_tile); });
    };
    auto launch = [&](auto stage, bool large, dim3 grid, const StageArgs &s) {
        constexpr int STAGE = stage;
        if (grid.x == 0) return;
        if (large) ortho_product_kernel<STAGE, 4, 2><<<grid, 256, 0, st>>>(shapes, p, s);
        else ortho_product_kernel<STAGE, 2, 4><<<grid, 256, 0, st>>>(shapes, p, s);
    };
    auto gram = [&](const StageArgs &s) {
        for (int large = 0; large < 2; ++large) {
            auto mine = [&](const OrthoArea &a) { return (a.tile == 128) == (large == 1); };
            int n = blocks(shapes, [&](const OrthoArea &a, const OrthoItem &) {
                return mine(a) ? ortho_triangle((a.mp + a.tile - 1) / a.tile) * a.splits : 0; });
            launch(std::integral_constant<int, STAGE_GRAM>{}, large, n, s);
            n = blocks(shapes, [&](const OrthoArea &a, const OrthoItem &) {
                return mine(a) && a.splits > 1 ? ortho_triangle((a.mp + a.tile - 1) / a.tile) : 0; });
            launch(std::integral_constant<int, STAGE_REDUCE>{}, large, n, s);
        }
    };
    with_dtype(p.type, [&](auto type) {
        typedef decltype(type) T;
        int n = blocks(g, [](const OrthoArea &a, const OrthoItem &) { return a.parts_used; });
        ortho_norm_kernel<T><<<n, 256, 0, st>>>(g, p);
        double rho = 1.0;                       // bound of A's largest eigenvalue
        int kx = exponent_for(1.0), xt = 0;
        n = blocks(g, [](const OrthoArea &a, const OrthoItem &) { return a.mp / 64 * (a.np / 64); });
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
            for (int i = 0; i < len; ++i) {
                const float *c = p.coef[s0 + i];
                double p_max, lp_max, lpp_max;
                polynomial_bounds(c, rho * 1.001, p_max, lp_max, lpp_max);
                // the first step's P is the segment's Q
                const int kp = exponent_for(p_max), pout = i == 0 ? SQ_Q0 : SQ_P;
                s.f = cur; s.out[0] = pout;
                s.a = (float)std::ldexp(c[0], kp); s.b = (float)std::ldexp(c[1], kp - ka); s.c = (float)std::ldexp(c[2], kp - 2 * ka);
                launch(std::integral_constant<int, STAGE_POLY>{}, symmetric_tile == 128, n, s);
                q_max *= p_max;
                // T = P A and Q <- P Q in one launch, then A <- T P
                int pair = 0;
                s.f = pout;
                const int kt = exponent_for(lp_max);
                if (i + 1 < len) {
                    s.g[pair] = cur; s.out[pair] = SQ_T;
                    s.out_scale[pair++] = (float)std::ldexp(1.0, kt - kp - ka);
                }
                if (i == 0) {
                    q = SQ_Q0; kq = kp;
                } else {
                    const int kn = exponent_for(q_max), next = q == SQ_Q0 ? SQ_Q1 : SQ_Q0;
                    s.g[pair] = q; s.out[pair] = next;
                    s.out_scale[pair++] = (float)std::ldexp(1.0, kn - kp - kq);
                    q = next; kq = kn;
                }
                if (pair) launch(std::integral_constant<int, STAGE_MUL>{}, symmetric_tile == 128, dim3(n, pair), s);
                if (i + 1 < len) {
                    const int kn = exponent_for(lpp_max), next = cur == SQ_A0 ? SQ_A1 : SQ_A0;
                    s.f = SQ_T; s.g[0] = pout; s.out[0] = next;
                    s.out_scale[0] = (float)std::ldexp(1.0, kn - kt - kp);
                    launch(std::integral_constant<int, STAGE_MUL>{}, symmetric_tile == 128, dim3(n, 1), s);
                    cur = next; ka = kn;
                }
                rho = std::fmax(lpp_max, 1e-6);
            }
            s.f = q; s.xt = xt;
            n = whole();
            if (s0 + len < p.steps) {
                const int kn = exponent_for(std::sqrt(rho));
                s.out_scale[0] = (float)std::ldexp(1.0, kn - kq - kx);
                launch(std::integral_constant<int, STAGE_APPLY>{}, full_tile == 128, n, s);
                kx = kn;
                xt = 1 - xt;
            } else {
                s.out_scale[0] = (float)std::ldexp(1.0, -kq - kx);
                if (full_tile == 128) ortho_finish_kernel<T, 4, 2><<<n, 256, 0, st>>>(shapes, p, s, g);
                else ortho_finish_kernel<T, 2, 4><<<n, 256, 0, st>>>(shapes, p, s, g);
            }
        }
    });
}

}  // namespace nnb

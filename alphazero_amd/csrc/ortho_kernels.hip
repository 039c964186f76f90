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
#include "mfma_tiles.h"
#include "numeric_types.h"

namespace nnb {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));

// The item a block works on, and the block's index within it.
__device__ __forceinline__ int find_item(const OrthoGroup &g, int block, int &local) {
    int i = 0;
    while (i + 1 < g.count && block >= g.first[i + 1]) ++i;
    local = block - g.first[i];
    return i;
}

// u of element (r, c): the matrix itself, or what the optimiser orthogonalises (the new momentum, with Nesterov's
// look-ahead the gradient plus the new momentum's next share)
template <typename T>
__device__ __forceinline__ float update_of(const OrthoParams &p, float g, float m_new) {
    if (!p.muon) return g;
    return p.nesterov ? g + p.mu * m_new : m_new;
}

// Sum of squares of u, in double (a gradient's squares leave float32's range long before the gradient does), as
// partial sums that the next kernel adds in a fixed order; the optimiser step's new momentum is written on the way.
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoGroup g, OrthoParams p) {
    int local;
    const OrthoItem &it = g.item[find_item(g, blockIdx.x, local)];
    const OrthoArea a = ortho_area(it.rows, it.cols);
    const int b = local / kOrthoNormParts, part = local % kOrthoNormParts;
    const long long total = (long long)it.rows * it.cols;
    const T *x = static_cast<const T *>(it.x) + b * it.x_bs;
    double sum = 0.0;
    for (long long i = (long long)part * 256 + threadIdx.x; i < total; i += 256 * kOrthoNormParts) {
        const int r = (int)(i / it.cols), c = (int)(i % it.cols);
        const float gr = to_f32(x[r * it.x_rs + c * it.x_cs]);
        float m_new = 0.f;
        if (p.muon) {
            m_new = p.mu * it.momentum[i] + gr;
            it.momentum_out[i] = m_new;
        }
        const float u = update_of<T>(p, gr, m_new);
        sum += (double)u * (double)u;
    }
    __shared__ double part_sum[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        reinterpret_cast<double *>(g.ws + it.ws + b * it.ws_stride + a.parts)[part] =
            (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
}

struct Planes {
    f16_t *hi, *lo;
};
__device__ __forceinline__ Planes planes(unsigned char *area, size_t offset, size_t count) {
    f16_t *p = reinterpret_cast<f16_t *>(area + offset);
    return {p, p + count};
}
__device__ __forceinline__ void split(float y, f16_t &hi, f16_t &lo) {
    hi = (f16_t)y;
    lo = (f16_t)(y - (float)hi);
}

// u / (|u| + eps) * 2^kx as planes, row-major and transposed, zero-padded to whole tiles.
template <typename T>
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoGroup g, OrthoParams p, float pow_kx) {
    __shared__ float tile[64][65];
    __shared__ double part_sum[4];
    int local;
    const OrthoItem &it = g.item[find_item(g, blockIdx.x, local)];
    const OrthoArea a = ortho_area(it.rows, it.cols);
    const int rt = ortho_padded(it.rows) / 64, ct = ortho_padded(it.cols) / 64;
    const int b = local / (rt * ct), t = local % (rt * ct), r0 = t / ct * 64, c0 = t % ct * 64;
    unsigned char *area = g.ws + it.ws + b * it.ws_stride;
    double sum = reinterpret_cast<const double *>(area + a.parts)[threadIdx.x];
    static_assert(kOrthoNormParts == 256, "one partial sum per thread");
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part_sum[threadIdx.x >> 6] = sum;
    const T *x = static_cast<const T *>(it.x) + b * it.x_bs;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int r = r0 + e / 64, c = c0 + e % 64;
        float u = 0.f;
        if (r < it.rows && c < it.cols) {
            const float gr = to_f32(x[r * it.x_rs + c * it.x_cs]);
            u = update_of<T>(p, gr, p.muon ? it.momentum_out[(long long)r * it.cols + c] : 0.f);
        }
        tile[e / 64][e % 64] = u;
    }
    __syncthreads();
    const double norm = sqrt((part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3])) + p.eps;
    const double scale = (double)pow_kx / norm;
    const bool tall = it.rows > it.cols;
    const size_t count = (size_t)a.mp * a.np;
    const Planes straight = planes(area, tall ? a.xt[0] : a.x, count), turned = planes(area, tall ? a.x : a.xt[0], count);
    const int ld_s = ct * 64, ld_t = rt * 64;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int i = e / 64, j = e % 64;
        f16_t hi, lo;
        split((float)((double)tile[i][j] * scale), hi, lo);
        const size_t o = (size_t)(r0 + i) * ld_s + c0 + j;
        straight.hi[o] = hi; straight.lo[o] = lo;
        split((float)((double)tile[j][i] * scale), hi, lo);
        const size_t q = (size_t)(c0 + i) * ld_t + r0 + j;
        turned.hi[q] = hi; turned.lo[q] = lo;
    }
}

enum OrthoStage { STAGE_GRAM, STAGE_POLY, STAGE_MUL, STAGE_APPLY, STAGE_FINISH };

struct StageArgs {
    int f, g, out;               // squares: factors and result (MUL), A and P (POLY), A (GRAM), Q (APPLY, FINISH)
    int xt;                      // which transposed planes APPLY / FINISH read (APPLY writes the other one)
    float out_scale;             // 2^(k_out - k_f - k_g); FINISH: 2^(-k_f - k_g)
    float a, b, c;               // POLY: coefficients, times 2^(k_out), 2^(k_out - k_A), 2^(k_out - 2 k_A)
};

// C = F G^T over K, both factors K-contiguous planes, one 64 x 64 tile per block, four waves of 32 x 32.
template <typename T, int STAGE>
__global__ __launch_bounds__(256) void ortho_product_kernel(OrthoGroup g, OrthoParams p, StageArgs s) {
    __shared__ u32x4 lds[4][256];                 // F hi, F lo, G hi, G lo: 64 rows x 32 k, in fragment order
    int local;
    const OrthoItem &it = g.item[find_item(g, blockIdx.x, local)];
    const OrthoArea a = ortho_area(it.rows, it.cols);
    constexpr bool symmetric = STAGE == STAGE_GRAM || STAGE == STAGE_POLY || STAGE == STAGE_MUL;
    const int mt = a.mp / 64, nt = a.np / 64;
    const int per = symmetric ? mt * (mt + 1) / 2 : mt * nt;
    const int batch = local / per;
    int t = local % per, ti = 0, tj;
    if (symmetric) {
        while (t >= mt - ti) { t -= mt - ti; ++ti; }
        tj = ti + t;
    } else {
        ti = t % mt;
        tj = t / mt;
    }
    unsigned char *area = g.ws + it.ws + batch * it.ws_stride;
    const size_t wide = (size_t)a.mp * a.np, square = (size_t)a.mp * a.mp;
    const int kdim = STAGE == STAGE_GRAM ? a.np : a.mp;
    Planes f, h;
    if (STAGE == STAGE_GRAM) { f = planes(area, a.x, wide); h = f; }
    else if (STAGE == STAGE_POLY) { f = planes(area, a.sq[s.f], square); h = f; }
    else if (STAGE == STAGE_MUL) { f = planes(area, a.sq[s.f], square); h = planes(area, a.sq[s.g], square); }
    else { f = planes(area, a.sq[s.f], square); h = planes(area, a.xt[s.xt], wide); }

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
    const size_t fo = (size_t)(ti * 64 + tid / 4) * kdim + tid % 4 * 8, ho = (size_t)(tj * 64 + tid / 4) * kdim + tid % 4 * 8;
    const int slot = (tid / 64) * 64 + (tid % 4) * 16 + (tid / 4) % 16;
    f32x4 acc[2][2] = {};
    for (int k = 0; k < kdim; k += 32) {
        const u32x4 v0 = *reinterpret_cast<const u32x4 *>(f.hi + fo + k), v1 = *reinterpret_cast<const u32x4 *>(f.lo + fo + k);
        const u32x4 v2 = *reinterpret_cast<const u32x4 *>(h.hi + ho + k), v3 = *reinterpret_cast<const u32x4 *>(h.lo + ho + k);
        __syncthreads();
        lds[0][slot] = v0; lds[1][slot] = v1; lds[2][slot] = v2; lds[3][slot] = v3;
        __syncthreads();
        half8 fh[2], fl[2], hh[2], hl[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fh[i] = as_half8(lds[0][wr * 4 + i * 64 + lane]); fl[i] = as_half8(lds[1][wr * 4 + i * 64 + lane]);
            hh[i] = as_half8(lds[2][wc * 4 + i * 64 + lane]); hl[i] = as_half8(lds[3][wc * 4 + i * 64 + lane]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[i], hh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[i], hl[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[i], hh[j], acc[i][j], 0, 0, 0);
            }
    }
    const float keep = p.decay;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = ti * 64 + wr + 16 * i + 4 * (lane >> 4) + e, c = tj * 64 + wc + 16 * j + (lane & 15);
                const float v = acc[i][j][e];
                if (symmetric) {
                    if (r > c) continue;
                    const size_t o = (size_t)r * a.mp + c, q = (size_t)c * a.mp + r;
                    float y = v * s.out_scale;
                    if (STAGE == STAGE_POLY) {
                        const float av = (float)f.hi[o] + (float)f.lo[o];
                        y = (r == c ? s.a : 0.f) + s.b * av + s.c * v;
                    }
                    const Planes d = planes(area, a.sq[s.out], square);
                    f16_t hi, lo;
                    split(y, hi, lo);
                    d.hi[o] = hi; d.lo[o] = lo;
                    d.hi[q] = hi; d.lo[q] = lo;
                } else if (STAGE == STAGE_APPLY) {
                    const Planes d = planes(area, a.x, wide), dt = planes(area, a.xt[1 - s.xt], wide);
                    f16_t hi, lo;
                    split(v * s.out_scale, hi, lo);
                    const size_t o = (size_t)r * a.np + c, q = (size_t)c * a.mp + r;
                    d.hi[o] = hi; d.lo[o] = lo;
                    dt.hi[q] = hi; dt.lo[q] = lo;
                } else {
                    if (r >= a.m || c >= a.n) continue;
                    const bool tall = it.rows > it.cols;
                    const int ur = tall ? c : r, uc = tall ? r : c;
                    const float o = v * s.out_scale;
                    T *out = static_cast<T *>(it.out) + batch * it.o_bs + ur * it.o_rs + uc * it.o_cs;
                    if (p.muon) {
                        const float w = to_f32(static_cast<const T *>(it.weight)[(long long)ur * it.cols + uc]);
                        *out = from_f32<T>(w * keep - it.scale * o);
                    } else {
                        *out = from_f32<T>(o);
                    }
                }
            }
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
    auto blocks = [&](auto per_matrix) {
        int n = 0;
        for (int i = 0; i < g.count; ++i) {
            g.first[i] = n;
            n += g.item[i].batch * per_matrix(ortho_area(g.item[i].rows, g.item[i].cols));
        }
        g.first[g.count] = n;
        return n;
    };
    auto symmetric = [](const OrthoArea &a) { const int t = a.mp / 64; return t * (t + 1) / 2; };
    auto full = [](const OrthoArea &a) { return a.mp / 64 * (a.np / 64); };
    with_dtype(p.type, [&](auto type) {
        typedef decltype(type) T;
        int n = blocks([](const OrthoArea &) { return kOrthoNormParts; });
        ortho_norm_kernel<T><<<n, 256, 0, st>>>(g, p);
        double rho = 1.0;                       // bound of A's largest eigenvalue
        int kx = exponent_for(1.0);
        n = blocks(full);
        ortho_split_kernel<T><<<n, 256, 0, st>>>(g, p, (float)std::ldexp(1.0, kx));
        int xt = 0;
        for (int s0 = 0; s0 < p.steps; s0 += kOrthoSegment) {
            const int len = p.steps - s0 < kOrthoSegment ? p.steps - s0 : kOrthoSegment;
            StageArgs s = {};
            int ka = exponent_for(rho), kq = 0, cur = SQ_A0, q = SQ_P;
            s.out = cur;
            s.out_scale = (float)std::ldexp(1.0, ka - 2 * kx);
            n = blocks(symmetric);
            ortho_product_kernel<T, STAGE_GRAM><<<n, 256, 0, st>>>(g, p, s);
            double q_max = 1.0;
            for (int i = 0; i < len; ++i) {
                const float *c = p.coef[s0 + i];
                double p_max, lp_max, lpp_max;
                polynomial_bounds(c, rho * 1.001, p_max, lp_max, lpp_max);
                // the first step's P is the segment's Q
                const int kp = exponent_for(p_max), pout = i == 0 ? SQ_Q0 : SQ_P;
                s.f = cur; s.out = pout;
                s.a = (float)std::ldexp(c[0], kp); s.b = (float)std::ldexp(c[1], kp - ka); s.c = (float)std::ldexp(c[2], kp - 2 * ka);
                n = blocks(symmetric);
                ortho_product_kernel<T, STAGE_POLY><<<n, 256, 0, st>>>(g, p, s);
                q_max *= p_max;
                if (i == 0) {
                    q = SQ_Q0; kq = kp;
                } else {
                    const int kn = exponent_for(q_max), next = q == SQ_Q0 ? SQ_Q1 : SQ_Q0;
                    s.f = SQ_P; s.g = q; s.out = next;
                    s.out_scale = (float)std::ldexp(1.0, kn - kp - kq);
                    ortho_product_kernel<T, STAGE_MUL><<<n, 256, 0, st>>>(g, p, s);
                    q = next; kq = kn;
                }
                if (i + 1 < len) {
                    const int kt = exponent_for(lp_max), next = cur == SQ_A0 ? SQ_A1 : SQ_A0;
                    s.f = pout; s.g = cur; s.out = SQ_T;
                    s.out_scale = (float)std::ldexp(1.0, kt - kp - ka);
                    ortho_product_kernel<T, STAGE_MUL><<<n, 256, 0, st>>>(g, p, s);
                    const int kn = exponent_for(lpp_max);
                    s.f = SQ_T; s.g = pout; s.out = next;
                    s.out_scale = (float)std::ldexp(1.0, kn - kt - kp);
                    ortho_product_kernel<T, STAGE_MUL><<<n, 256, 0, st>>>(g, p, s);
                    cur = next; ka = kn;
                }
                rho = std::fmax(lpp_max, 1e-6);
            }
            s.f = q; s.xt = xt;
            n = blocks(full);
            if (s0 + len < p.steps) {
                const int kn = exponent_for(std::sqrt(rho));
                s.out_scale = (float)std::ldexp(1.0, kn - kq - kx);
                ortho_product_kernel<T, STAGE_APPLY><<<n, 256, 0, st>>>(g, p, s);
                kx = kn;
                xt = 1 - xt;
            } else {
                s.out_scale = (float)std::ldexp(1.0, -kq - kx);
                ortho_product_kernel<T, STAGE_FINISH><<<n, 256, 0, st>>>(g, p, s);
            }
        }
    });
}

}  // namespace nnb

// 4-bit floats with shared scales ("MX4"): quantisation, its inverse, and a linear layer on them.
//
// A row of K numbers is cut into blocks of 32.  A block shares the scale 2^e, e = floor(log2 max|x|) - 2 clamped to
// [-127, 127], stored as the byte e + 127; an element is the e2m1 code of x / 2^e: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6
// for codes 0..7, to nearest with ties to the even code, beyond 6 to 6.  A block that holds an infinity or a NaN gets
// the scale byte 255 and reads as NaN.
//
// Codes: [rows][Kp/2] bytes, Kp = K padded with zeros to k-steps of 128, element 2i in the low half of byte i.
// Scales: one 256-byte word block per 16 rows and four k-steps, in the order the matrix instruction wants them: lane
// l = 16 * (k-block within the step) + (row within the 16) holds four bytes, one per k-step, so a fragment's scales
// for 512 elements are one coalesced load and the instruction picks the byte itself.  (Scales in row order cost a cache
// line per row and fetch; the codes' own traffic is what the large product waits for.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "mfma_tiles.h"
#include "numeric_types.h"

namespace nnb {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------- quantisation

// Scale byte of a block whose largest magnitude has the float32 bits `top` (sign cleared).
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}

// Eight consecutive elements of a block -> eight codes.  `byte` is the block's scale (not 255).
__device__ __forceinline__ uint32_t encode8(const float (&v)[8], uint32_t byte) {
    // 2^(byte - 127); 2^-127 is below the normal range
    const float scale = __builtin_bit_cast(float, byte ? byte << 23 : 0x00400000u);
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}

// Eight elements in one or two wide accesses; global memory takes them at any element's alignment.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Pack8 { T v[8]; };

// x [rows][cols] (any strides) -> codes, scales.  A block takes 16 rows x 512 elements, a wave four of the rows, a lane
// eight elements of each, so that four lanes share a scale; the sixteen rows' scale bytes meet in LDS and leave as one
// word block.  row_count (may be null): live rows, read on the device.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T *__restrict__ x, long long rows, int cols, int kp,
                                                           long long row_stride, long long col_stride,
                                                           const int32_t *__restrict__ row_count,
                                                           uint32_t *__restrict__ codes, uint32_t *__restrict__ scales) {
    __shared__ uint32_t bytes[64];
    if (row_count) rows = *row_count < rows ? *row_count : rows;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int words = mx4_scale_words(kp);
    const long long tasks = (rows + 15) / 16 * words;
    for (long long t = blockIdx.x; t < tasks; t += gridDim.x) {
        const long long row0 = t / words * 16 + wave * 4;
        const int k = (int)(t % words) * 512 + lane * 8;
        const T *p = x + row0 * row_stride + k * col_stride;
        Pack8<T> q[4];
        if (col_stride == 1 && k + 8 <= cols) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row0 + i < rows) q[i] = *reinterpret_cast<const Pack8<T> *>(p + i * row_stride);
                else q[i] = {};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    q[i].v[j] = row0 + i < rows && k + j < cols ? p[i * row_stride + j * col_stride] : T(0.f);
        }
        uint8_t *b = reinterpret_cast<uint8_t *>(bytes);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[8];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = to_f32(q[i].v[j]);
                const uint32_t m = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;       // magnitudes order as integers
                top = m > top ? m : top;
            }
            top = max(top, (uint32_t)__shfl_xor((int)top, 1));
            top = max(top, (uint32_t)__shfl_xor((int)top, 2));
            const uint32_t byte = scale_byte(top);
            if (row0 + i < rows && k < kp) codes[((row0 + i) * kp + k) >> 3] = byte == 255 ? 0 : encode8(v, byte);
            if ((lane & 3) == i) b[((lane >> 2 & 3) * 16 + wave * 4 + i) * 4 + (lane >> 4)] = (uint8_t)byte;
        }
        __syncthreads();
        if (threadIdx.x < 64) scales[t * 64 + lane] = bytes[lane];
        __syncthreads();
    }
}

__device__ __forceinline__ float mx4_value(uint32_t code, float scale) {
    const uint32_t m = code & 7;
    const float size = m < 2 ? 0.5f * (float)m : __builtin_ldexpf(1.f + 0.5f * (float)(m & 1), (int)(m >> 1) - 1);
    return (code & 8 ? -size : size) * scale;
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, long long rows, int cols,
                                                             int kp, T *__restrict__ out) {
    const int groups = kp >> 3;
    const long long total = rows * groups, stride = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const long long row = i / groups;
        const int k = (int)(i - row * groups) * 8;
        if (k >= cols) continue;
        const uint32_t c = codes[i], byte = scales[mx4_scale_at(row, k >> 5, kp)];
        const float scale = __builtin_bit_cast(float, byte == 255 ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
        Pack8<T> q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q.v[j] = from_f32<T>(mx4_value(c >> (4 * j), scale));
        T *p = out + row * cols + k;
        if (k + 8 <= cols) {
            *reinterpret_cast<Pack8<T> *>(p) = q;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < cols) p[j] = q.v[j];
        }
    }
}

// ----------------------------------------------------------------------------------------------- linear layer
//
// y [rows][n] = x [rows][K] * w [n][K]^T (+ bias, ReLU), both in MX4, on v_mfma_scale_f32_16x16x128_f8f6f4: lane l of a
// 16 x 128 fragment holds the 32 elements (one scale block) l/16 of row l%16.  The weights are the instruction's first
// operand, so a lane ends up with four consecutive features of one row: one store.

__device__ __forceinline__ f32x4 mfma_mx4(i32x4 w, i32x4 x, f32x4 acc, int w_scale, int x_scale, int step) {
    const i32x8 w8 = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
    const i32x8 x8 = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
    // 4 = e2m1; the byte of the scale word is part of the instruction
    switch (step) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc, 4, 4, 0, w_scale, 0, x_scale);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc, 4, 4, 1, w_scale, 1, x_scale);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc, 4, 4, 2, w_scale, 2, x_scale);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc, 4, 4, 3, w_scale, 3, x_scale);
    }
}

// Bias, ReLU, rounding and store of the four features c .. c + 3 of row r.
template <typename T> struct alignas(4 * sizeof(T)) Pack4 { T v[4]; };
template <typename T>
__device__ __forceinline__ void store_features(const Mx4Linear &a, long long r, int c, f32x4 acc, const float (&bias)[4]) {
    Pack4<T> q;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v = acc[e] + bias[e];
        if (a.relu) v = v < 0.f ? 0.f : v;                   // NaN stays NaN
        q.v[e] = from_f32<T>(v);
    }
    T *p = static_cast<T *>(a.y) + r * a.y_stride + c;
    if (a.wide && c + 4 <= a.n) {
        *reinterpret_cast<Pack4<T> *>(p) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < a.n) p[e] = q.v[e];
    }
}
__device__ __forceinline__ void load_bias(const Mx4Linear &a, int c, float (&bias)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = a.bias && c + e < a.n ? load_as_f32(a.bias, a.bias_type, c + e) : 0.f;
}

// Large products.  A block computes (WX * TX * 16) rows x (WW * TW * 16) features with WX x WW waves; a stage is 256
// elements (128 bytes) of every row, brought to LDS by the loads themselves, two stages in turn.  A row's eight 16-byte
// chunks lie at chunk ^ (row & 7): a fragment read then touches every bank group once.
#define LDS_PTR(p) (__attribute__((address_space(3))) uint32_t *)(p)
#define GLOBAL_PTR(p) (const __attribute__((address_space(1))) uint32_t *)(p)

template <typename T, int WX, int WW, int TX, int TW>
__global__ __launch_bounds__(WX *WW * 64, 1) void mx4_tile_kernel(Mx4Linear a) {
    constexpr int kRows = WX * TX * 16, kFeatures = WW * TW * 16, kWaves = WX * WW;
    constexpr int kLoads = (kRows + kFeatures) / 8 / kWaves;         // 1 KB (8 rows x 128 bytes) each, per wave and stage
    static_assert((kRows + kFeatures) % (8 * kWaves) == 0, "whole loads per wave");
    __shared__ i32x4 lds[2][(kRows + kFeatures) * 8];
    const long long rows = a.row_count && *a.row_count < a.rows ? *a.row_count : a.rows;

    // Tiles in groups of eight row tiles walked feature tile by feature tile; consecutive tiles of the walk on one
    // XCD (blocks go to the eight XCDs in turn), so that its L2 holds what they share.
    const int xt = (int)((a.rows + kRows - 1) / kRows), wt = (a.n + kFeatures - 1) / kFeatures;
    int tile = blockIdx.x;
    {
        const int total = xt * wt, each = total / 8, extra = total % 8, xcd = tile % 8;
        tile = xcd * each + (xcd < extra ? xcd : extra) + tile / 8;
    }
    const int group = tile / (8 * wt), in_group = tile - group * 8 * wt;
    const int height = xt - group * 8 < 8 ? xt - group * 8 : 8;
    const long long row0 = (long long)(group * 8 + in_group % height) * kRows;
    const int col0 = in_group / height * kFeatures;
    if (row0 >= rows) return;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = a.kp / 128, stages = (steps + 1) / 2;
    const uint32_t cs = a.kp / 2;
    const int chunk = (lane & 7) ^ (lane >> 3);
    const uint8_t *xbase = a.x_codes + row0 * cs, *wbase = a.w_codes + (size_t)col0 * cs;
    uint32_t offset[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        int r = (wave * kLoads + j) * 8 + (lane >> 3);
        const bool is_x = r < kRows;
        // rows and features past the end repeat the last one; their results are not stored
        const long long left = is_x ? rows - row0 : (long long)(a.n - col0);
        if (!is_x) r -= kRows;
        r = r < left ? r : (int)left - 1;
        offset[j] = (uint32_t)r * cs + chunk * 16;
    }
    auto issue = [&](int t) {
        // an odd number of k-steps: the last stage's second half would lie behind the row; it fetches the first half again
        const uint32_t k = t * 128 - (2 * t + 2 > steps && chunk >= 4 ? 64 : 0);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint8_t *base = (wave * kLoads + j) * 8 < kRows ? xbase : wbase;
            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(base + (size_t)(offset[j] + k)),
                                             LDS_PTR(&lds[t & 1][(wave * kLoads + j) * 64]), 16, 0, 0);
        }
    };
    const int wx = wave % WX * TX * 16, ww = wave / WX * TW * 16;    // this wave's first row and feature in the tile
    const int words = mx4_scale_words(a.kp);
    const uint32_t *xs[TX], *ws[TW];
#pragma unroll
    for (int i = 0; i < TX; ++i) {
        long long r = row0 + wx + i * 16;
        r = r < rows ? r : rows - 1;
        xs[i] = reinterpret_cast<const uint32_t *>(a.x_scales) + (r / 16 * words) * 64 + lane;
    }
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        int c = col0 + ww + i * 16;
        c = c < a.n ? c : a.n - 1;
        ws[i] = reinterpret_cast<const uint32_t *>(a.w_scales) + ((size_t)(c / 16) * words) * 64 + lane;
    }
    // where this lane finds chunk l/16 (first step of a stage; the second one's is the same with bit 6 of the byte address
    // flipped) of row l%16 of a fragment
    const int read0 = (lane & 15) * 8 + ((lane >> 4) ^ (lane & 7));

    f32x4 acc[TX][TW] = {};
    int sx[TX], sw[TW], sx_next[TX], sw_next[TW];
    auto load_scales = [&](int word) {
#pragma unroll
        for (int i = 0; i < TX; ++i) sx_next[i] = (int)xs[i][word * 64];
#pragma unroll
        for (int i = 0; i < TW; ++i) sw_next[i] = (int)ws[i][word * 64];
    };
    // Every load this wave has issued has landed, and after the barrier everybody's; nobody reads the other buffer any
    // more.  The wait is the builtin so that the compiler knows of it and adds none between the next stage's loads and
    // the products.
    auto meet = [&] {
        __builtin_amdgcn_s_waitcnt(0x0070);                  // vmcnt(0) lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    };
    auto compute = [&](int t, int s, int step_of_word) {
        i32x4 xf[TX], wf[TW];
        const i32x4 *base = lds[t & 1];
#pragma unroll
        for (int i = 0; i < TX; ++i) xf[i] = base[(wx + i * 16) * 8 + (read0 ^ (s * 4))];
#pragma unroll
        for (int i = 0; i < TW; ++i) wf[i] = base[(kRows + ww + i * 16) * 8 + (read0 ^ (s * 4))];
#pragma unroll
        for (int i = 0; i < TX; ++i)
#pragma unroll
            for (int j = 0; j < TW; ++j) acc[i][j] = mfma_mx4(wf[j], xf[i], acc[i][j], sw[j], sx[i], step_of_word);
    };
    issue(0);
    load_scales(0);
    for (int t = 0; t < stages; t += 2) {
        meet();
#pragma unroll
        for (int i = 0; i < TX; ++i) sx[i] = sx_next[i];
#pragma unroll
        for (int i = 0; i < TW; ++i) sw[i] = sw_next[i];
        if (t + 1 < stages) issue(t + 1);
        compute(t, 0, 0);
        if (2 * t + 1 < steps) compute(t, 1, 1);
        if (t + 1 < stages) {
            meet();
            if (t + 2 < stages) {
                issue(t + 2);
                load_scales(t / 2 + 1);
            }
            compute(t + 1, 0, 2);
            if (2 * t + 3 < steps) compute(t + 1, 1, 3);
        }
    }
#pragma unroll
    for (int j = 0; j < TW; ++j) {
        const int c = col0 + ww + j * 16 + (lane >> 4) * 4;
        if (c >= a.n) continue;
        float bias[4];
        load_bias(a, c, bias);
#pragma unroll
        for (int i = 0; i < TX; ++i) {
            const long long r = row0 + wx + i * 16 + (lane & 15);
            if (r < rows) store_features<T>(a, r, c, acc[i][j], bias);
        }
    }
}

// Few rows: a block computes RT * 16 rows x 16 features, its eight waves take every eighth word (512 elements) of K
// with fragments straight from memory and add up in LDS in a fixed order.  FUSED (at most 16 rows, kMx4FusedElements
// elements): x comes as numbers and every block quantises them into LDS for itself, which saves a launch.
constexpr int kMx4FusedElements = 65536;
constexpr int kRowsWaves = 8;

template <typename T, int RT, typename X, bool FUSED>
__global__ __launch_bounds__(kRowsWaves * 64) void mx4_rows_kernel(Mx4Linear a, const X *__restrict__ x, int cols,
                                                                  long long row_stride, long long col_stride) {
    __shared__ f32x4 part[kRowsWaves][RT][64];
    __shared__ uint32_t xcodes[FUSED ? kMx4FusedElements / 8 : 1];
    __shared__ uint8_t xbytes[FUSED ? kMx4FusedElements / 32 : 1];
    const long long rows = a.row_count && *a.row_count < a.rows ? *a.row_count : a.rows;
    const long long row0 = (long long)blockIdx.y * (RT * 16);
    if (row0 >= rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kb = lane >> 4;
    const int col0 = blockIdx.x * 16;
    const int steps = a.kp / 128, words = mx4_scale_words(a.kp);
    const size_t cs = a.kp / 2;
    const int c = col0 + r16 < a.n ? col0 + r16 : a.n - 1;
    const uint8_t *wc = a.w_codes + c * cs + kb * 16;
    const uint32_t *ws = reinterpret_cast<const uint32_t *>(a.w_scales) + (size_t)blockIdx.x * words * 64 + lane;
    const uint8_t *xc[RT];
    const uint32_t *xs[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const long long r = row0 + i * 16 + r16 < rows ? row0 + i * 16 + r16 : rows - 1;
        const long long tile = row0 + i * 16 < rows ? row0 / 16 + i : (rows - 1) / 16;
        if (FUSED) {
            xc[i] = reinterpret_cast<const uint8_t *>(xcodes) + r * cs + kb * 16;
        } else {
            xc[i] = a.x_codes + r * cs + kb * 16;
            xs[i] = reinterpret_cast<const uint32_t *>(a.x_scales) + tile * words * 64 + lane;
        }
    }
    i32x4 wf[4];
    int wsc = 0;
    auto load_w = [&](int word) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int step = word * 4 + s < steps ? word * 4 + s : steps - 1;        // the tail repeats the last step, unused
            wf[s] = *reinterpret_cast<const i32x4 *>(wc + (size_t)step * 64);
        }
        wsc = (int)ws[(size_t)word * 64];
    };
    if (wave < words) load_w(wave);
    if (FUSED) {
        const int per_row = a.kp / 8, total = (int)rows * per_row;
        for (int i = threadIdx.x; i < (total + 3) / 4 * 4; i += kRowsWaves * 64) {
            const int r = i / per_row, k = (i - r * per_row) * 8;
            const X *p = x + r * row_stride + k * col_stride;
            float v[8];
            if (col_stride == 1 && k + 8 <= cols) {
                const Pack8<X> q = *reinterpret_cast<const Pack8<X> *>(p);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = to_f32(q.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = k + j < cols ? to_f32(p[j * col_stride]) : 0.f;
            }
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
            top = max(top, (uint32_t)__shfl_xor((int)top, 1));
            top = max(top, (uint32_t)__shfl_xor((int)top, 2));
            const uint32_t byte = scale_byte(top);
            xcodes[i] = byte == 255 ? 0 : encode8(v, byte);
            if ((i & 3) == 0) xbytes[i >> 2] = (uint8_t)byte;
        }
        __syncthreads();
    }
    f32x4 acc[RT] = {};
    for (int word = wave; word < words; word += kRowsWaves) {
        i32x4 w4[4], xf[RT][4];
        int sx[RT][4];
        const int sw = wsc;
#pragma unroll
        for (int s = 0; s < 4; ++s) w4[s] = wf[s];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int step = word * 4 + s < steps ? word * 4 + s : steps - 1;
                xf[i][s] = *reinterpret_cast<const i32x4 *>(xc[i] + (size_t)step * 64);
                if (FUSED) sx[i][s] = (int)xbytes[(int)(r16 < rows ? r16 : rows - 1) * (a.kp / 32) + step * 4 + kb];
            }
            if (!FUSED) sx[i][0] = (int)xs[i][(size_t)word * 64];
        }
        if (word + kRowsWaves < words) load_w(word + kRowsWaves);
        static_for<4>([&](auto s) {
            if (word * 4 + s < steps) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    if (FUSED) acc[i] = mfma_mx4(w4[s], xf[i][s], acc[i], sw >> (8 * s), sx[i][s], 0);
                    else acc[i] = mfma_mx4(w4[s], xf[i][s], acc[i], sw, sx[i][0], s);
                }
            }
        });
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave < RT) {
        f32x4 sum = part[0][wave][lane];
#pragma unroll
        for (int w = 1; w < kRowsWaves; ++w) sum += part[w][wave][lane];
        const long long r = row0 + wave * 16 + r16;
        const int cf = col0 + kb * 4;
        if (r < rows && cf < a.n) {
            float bias[4];
            load_bias(a, cf, bias);
            store_features<T>(a, r, cf, sum, bias);
        }
    }
}

}  // namespace

void launch_mx4_quantize(hipStream_t st, int type, long long rows, int cols, const void *x, long long row_stride,
                         long long col_stride, const int32_t *row_count, uint8_t *codes, uint8_t *scales) {
    const int kp = mx4_padded(cols);
    const long long tasks = (rows + 15) / 16 * mx4_scale_words(kp);
    with_dtype(type, [&](auto t) {
        typedef decltype(t) T;
        mx4_quantize_kernel<T><<<(int)(tasks < 16384 ? tasks : 16384), 256, 0, st>>>(
            static_cast<const T *>(x), rows, cols, kp, row_stride, col_stride, row_count,
            reinterpret_cast<uint32_t *>(codes), reinterpret_cast<uint32_t *>(scales));
    });
}

void launch_mx4_dequantize(hipStream_t st, int type, long long rows, int cols, const uint8_t *codes, const uint8_t *scales,
                           void *out) {
    const int kp = mx4_padded(cols);
    const long long blocks = (rows * (kp / 8) + 255) / 256;
    with_dtype(type, [&](auto t) {
        typedef decltype(t) T;
        mx4_dequantize_kernel<T><<<(int)(blocks < 16384 ? blocks : 16384), 256, 0, st>>>(
            reinterpret_cast<const uint32_t *>(codes), scales, rows, cols, kp, static_cast<T *>(out));
    });
}

bool mx4_linear_fuses(long long rows, int cols) { return rows <= 16 && rows * mx4_padded(cols) <= kMx4FusedElements; }

void launch_mx4_linear(hipStream_t st, Mx4Linear a, const Mx4Rows *x) {
    with_dtype(a.y_type, [&](auto t) {
        typedef decltype(t) T;
        a.wide = reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0 && a.y_stride % 4 == 0;
        const unsigned features = (unsigned)((a.n + 15) / 16);
        if (x) {
            with_dtype(x->type, [&](auto u) {
                typedef decltype(u) X;
                mx4_rows_kernel<T, 1, X, true><<<dim3(features, 1), kRowsWaves * 64, 0, st>>>(
                    a, static_cast<const X *>(x->x), x->cols, x->row_stride, x->col_stride);
            });
        } else if (a.rows <= 16) {
            mx4_rows_kernel<T, 1, float, false><<<dim3(features, 1), kRowsWaves * 64, 0, st>>>(a, nullptr, 0, 0, 0);
        } else if (a.rows <= 256) {
            mx4_rows_kernel<T, 4, float, false><<<dim3(features, (unsigned)((a.rows + 63) / 64)), kRowsWaves * 64, 0, st>>>(
                a, nullptr, 0, 0, 0);
        } else {
            auto tiles = [&](int r, int f) { return (a.rows + r - 1) / r * ((a.n + f - 1) / f); };
            if (tiles(256, 256) >= 256)
                mx4_tile_kernel<T, 2, 2, 8, 8><<<(unsigned)tiles(256, 256), 256, 0, st>>>(a);
            else
                mx4_tile_kernel<T, 2, 2, 4, 4><<<(unsigned)tiles(128, 128), 256, 0, st>>>(a);
        }
    });
}

}  // namespace nnb

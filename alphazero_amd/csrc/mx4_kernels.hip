// 4-bit floats with shared scales ("MX4"): quantisation, its inverse, and a linear layer on them.
//
// A row of K numbers is cut into blocks of 32.  A block shares the scale 2^e, e = floor(log2 max|x|) - 2 clamped to
// [-127, 127], stored as the byte e + 127; an element is the e2m1 code of x / 2^e: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6
// for codes 0..7, to nearest with ties to the even code, beyond 6 to 6.  A block that holds an infinity or a NaN gets
// the scale byte 255 and reads as NaN.  Rows are padded with zeros to a multiple of 128 elements (kMx4Pad), one
// k-step of v_mfma_scale_f32_16x16x128_f8f6f4: codes [rows][Kp/2] (element 2i in the low half of byte i), scales
// [rows][Kp/32].
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

template <typename T> struct alignas(16) Pack8 { T v[8]; };

// x [rows][cols] (any strides) -> codes, scales.  `lanes` (16, 32 or 64) consecutive lanes walk one row, eight elements
// each, so four lanes share a block and a wave covers 64 / lanes rows; `wide`: a lane's eight elements are 16 / 32
// aligned bytes.  row_count (may be null): live rows, read on the device.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T *__restrict__ x, long long rows, int cols, int kp,
                                                           long long row_stride, long long col_stride, int lanes, bool wide,
                                                           const int32_t *__restrict__ row_count,
                                                           uint32_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    if (row_count) rows = *row_count < rows ? *row_count : rows;
    const int lane = threadIdx.x & 63;
    const int rows_per_wave = 64 / lanes;
    const int segments = (kp + lanes * 8 - 1) / (lanes * 8);
    const long long row_groups = (rows + rows_per_wave - 1) / rows_per_wave;
    const long long tasks = row_groups * segments;
    const long long waves = (long long)gridDim.x * 4;
    for (long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); t < tasks; t += waves) {
        const long long row = t / segments * rows_per_wave + lane / lanes;
        const int k = (int)(t % segments) * lanes * 8 + (lane % lanes) * 8;
        const bool live = row < rows && k < kp;
        float v[8];
        const T *p = x + row * row_stride + k * col_stride;
        if (wide && live && k + 8 <= cols) {
            const Pack8<T> q = *reinterpret_cast<const Pack8<T> *>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(q.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = live && k + i < cols ? to_f32(p[i * col_stride]) : 0.f;
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t m = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;      // magnitudes order as integers
            top = m > top ? m : top;
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        const uint32_t byte = scale_byte(top);
        const uint32_t c = byte == 255 ? 0 : encode8(v, byte);
        if (live) {
            codes[(row * kp + k) >> 3] = c;
            if ((lane & 3) == 0) scales[(row * kp + k) >> 5] = (uint8_t)byte;
        }
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
                                                             int kp, bool wide, T *__restrict__ out) {
    const int groups = kp >> 3;
    const long long total = rows * groups, stride = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const long long row = i / groups;
        const int k = (int)(i - row * groups) * 8;
        if (k >= cols) continue;
        const uint32_t c = codes[i], byte = scales[i >> 2];
        const float scale = __builtin_bit_cast(float, byte == 255 ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
        Pack8<T> q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q.v[j] = from_f32<T>(mx4_value(c >> (4 * j), scale));
        T *p = out + row * cols + k;
        if (wide && k + 8 <= cols) {
            *reinterpret_cast<Pack8<T> *>(p) = q;
        } else {
            for (int j = 0; j < 8 && k + j < cols; ++j) p[j] = q.v[j];
        }
    }
}

// ----------------------------------------------------------------------------------------------- linear layer

// y [rows][n] = x [rows][K] * w [n][K]^T (+ bias, ReLU), both in MX4.  One wave per 16 rows x 64 columns, fragments
// straight from memory: lane l of a 16x16x128 tile holds the 32 elements (one scale block) l/16 of row l%16.
template <typename T>
__global__ __launch_bounds__(256) void mx4_linear_kernel(Mx4Linear a) {
    const long long rows = a.row_count && *a.row_count < a.rows ? *a.row_count : a.rows;
    const int lane = threadIdx.x & 63, r16 = lane & 15, kb = lane >> 4;
    const long long row0 = (long long)blockIdx.x * 64 + (threadIdx.x >> 6) * 16;
    const int col0 = blockIdx.y * 64;
    if (row0 >= rows) return;
    const size_t cs = a.kp / 2, ss = a.kp / 32;
    const long long xr = row0 + r16 < rows ? row0 + r16 : rows - 1;
    const uint8_t *xc = a.x_codes + xr * cs + kb * 16;
    const uint8_t *xs = a.x_scales + xr * ss + kb;
    const uint8_t *wc[4], *ws[4];
    for (int j = 0; j < 4; ++j) {
        const int c = col0 + 16 * j + r16 < a.n ? col0 + 16 * j + r16 : a.n - 1;
        wc[j] = a.w_codes + c * cs + kb * 16;
        ws[j] = a.w_scales + c * ss + kb;
    }
    f32x4 acc[4] = {};
    for (int k = 0; k < a.kp / 128; ++k) {
        const i32x4 x4 = *reinterpret_cast<const i32x4 *>(xc + 64 * k);
        const i32x8 xf = __builtin_shufflevector(x4, x4, 0, 1, 2, 3, -1, -1, -1, -1);
        const int xsc = xs[4 * k];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const i32x4 w4 = *reinterpret_cast<const i32x4 *>(wc[j] + 64 * k);
            const i32x8 wf = __builtin_shufflevector(w4, w4, 0, 1, 2, 3, -1, -1, -1, -1);
            acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xf, wf, acc[j], 4, 4, 0, xsc, 0, (int)ws[j][4 * k]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = col0 + 16 * j + r16;
        if (c >= a.n) continue;
        const float bias = a.bias ? load_as_f32(a.bias, a.bias_type, c) : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long r = row0 + 4 * kb + i;
            if (r >= rows) continue;
            float v = acc[j][i] + bias;
            if (a.relu) v = v < 0.f ? 0.f : v;               // NaN stays NaN
            static_cast<T *>(a.y)[r * a.y_stride + c] = from_f32<T>(v);
        }
    }
}

int grid_for(long long waves_of_work) {
    const long long blocks = (waves_of_work + 3) / 4;
    return (int)(blocks < 4096 ? blocks : 4096);
}

}  // namespace

void launch_mx4_quantize(hipStream_t st, int type, long long rows, int cols, const void *x, long long row_stride,
                         long long col_stride, const int32_t *row_count, uint8_t *codes, uint8_t *scales) {
    const int kp = mx4_padded(cols);
    const int lanes = kp >= 512 ? 64 : kp >= 256 ? 32 : 16;
    const long long tasks = (rows + 64 / lanes - 1) / (64 / lanes) * ((kp + lanes * 8 - 1) / (lanes * 8));
    with_dtype(type, [&](auto t) {
        typedef decltype(t) T;
        const bool wide = col_stride == 1 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && row_stride * sizeof(T) % 16 == 0;
        mx4_quantize_kernel<T><<<grid_for(tasks), 256, 0, st>>>(static_cast<const T *>(x), rows, cols, kp, row_stride,
                                                                col_stride, lanes, wide, row_count,
                                                                reinterpret_cast<uint32_t *>(codes), scales);
    });
}

void launch_mx4_dequantize(hipStream_t st, int type, long long rows, int cols, const uint8_t *codes, const uint8_t *scales,
                           void *out) {
    const int kp = mx4_padded(cols);
    with_dtype(type, [&](auto t) {
        typedef decltype(t) T;
        const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && cols * sizeof(T) % 16 == 0;
        mx4_dequantize_kernel<T><<<grid_for((rows * (kp / 8) + 63) / 64), 256, 0, st>>>(
            reinterpret_cast<const uint32_t *>(codes), scales, rows, cols, kp, wide, static_cast<T *>(out));
    });
}

void launch_mx4_linear(hipStream_t st, const Mx4Linear &a) {
    const dim3 grid((unsigned)((a.rows + 63) / 64), (unsigned)((a.n + 63) / 64));
    with_dtype(a.y_type, [&](auto t) { mx4_linear_kernel<decltype(t)><<<grid, 256, 0, st>>>(a); });
}

}  // namespace nnb

// 4-bit floats with shared scales ("MX4"): quantisation, its inverse, and a linear layer on them.
//
// A row of K numbers is cut into blocks of 32.  A block shares the scale 2^e, e = floor(log2 max|x|) - 2 clamped to
// [-127, 127], stored as the byte e + 127; an element is the e2m1 code of x / 2^e: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6
// for codes 0..7, to nearest with ties to the even code, beyond 6 to 6.  A block that holds an infinity or a NaN gets
// the scale byte 255 and reads as NaN.
//
// Layout: units of 32 rows x 256 elements (rows and K are padded with zeros), 4096 bytes of codes and 256 of scales each,
// [row / 32][k / 256], in the order in which v_mfma_scale_f32_32x32x64_f8f6f4 takes them: lane l = 32 * half + row of k-step s
// holds the 32 elements (one block) 64 s + 32 half of its row, 16 bytes at (64 s + l) * 16 (element 2i in the low half of
// byte i), and their scale is byte s of word l.  A unit is contiguous, so whole kilobytes move between memory and LDS
// whatever K is (rows of a power-of-two length would all start on the same memory channels), a fragment is one
// conflict-free LDS read, and its four k-steps' scales one word.
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

template <typename T, int N> struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) PackN { T v[N]; };
// Eight elements in one or two wide accesses; global memory takes them at any element's alignment.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Pack8 { T v[8]; };

// x [rows][cols] (any strides) -> codes, scales.  A block makes one unit: a thread eight elements of four rows, so that
// four lanes share a scale; codes and scales meet in LDS and leave in whole lines.  row_count (may be null): live rows,
// read on the device.  Bound by memory: 4096 x 11520 halves 26 us, 4.6 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T *__restrict__ x, long long rows, int cols, int kp,
                                                           long long row_stride, long long col_stride,
                                                           const int32_t *__restrict__ row_count,
                                                           uint4 *__restrict__ codes, uint32_t *__restrict__ scales) {
    __shared__ uint4 unit[256];
    __shared__ uint32_t bytes[64];
    if (row_count) rows = *row_count < rows ? *row_count : rows;
    const int units = kp / 256;
    const long long tasks = (rows + 31) / 32 * units;
    const int group = threadIdx.x & 31, r0 = threadIdx.x >> 5;  // eight elements of the 256, rows r0, r0 + 8, + 16, + 24
    for (long long t = blockIdx.x; t < tasks; t += gridDim.x) {
        const long long row0 = t / units * 32 + r0;
        const int k = (int)(t % units) * 256 + group * 8;
        const T *p = x + row0 * row_stride + k * col_stride;
        Pack8<T> q[4];
        if (col_stride == 1 && k + 8 <= cols) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row0 + 8 * i < rows) q[i] = *reinterpret_cast<const Pack8<T> *>(p + 8 * i * row_stride);
                else q[i] = {};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    q[i].v[j] = row0 + 8 * i < rows && k + j < cols ? p[8 * i * row_stride + j * col_stride] : T(0.f);
        }
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
            const int lane = (group >> 2 & 1) * 32 + r0 + 8 * i, step = group >> 3;
            reinterpret_cast<uint32_t *>(unit)[(step * 64 + lane) * 4 + (group & 3)] = byte == 255 ? 0 : encode8(v, byte);
            if ((group & 3) == i) reinterpret_cast<uint8_t *>(bytes)[lane * 4 + step] = (uint8_t)byte;
        }
        __syncthreads();
        codes[t * 256 + threadIdx.x] = unit[threadIdx.x];
        if (threadIdx.x < 64) scales[t * 64 + threadIdx.x] = bytes[threadIdx.x];
        __syncthreads();
    }
}

// A block turns one unit back into numbers: its 16-byte blocks meet in LDS row by row, then every lane writes 16 bytes of
// a row's 256 columns.  Bound by memory: 4096 x 11520 to float32 35 us, 6.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint4 *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                             long long rows, int cols, int kp, bool aligned, T *__restrict__ out) {
    constexpr int kPack = 16 / sizeof(T), kRowLanes = 256 / kPack;
    __shared__ uint4 blocks[32][9];
    __shared__ uint8_t bytes[256];
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const int units = kp / 256, tid = threadIdx.x;
    const long long tasks = (rows + 31) / 32 * units;
    for (long long t = blockIdx.x; t < tasks; t += gridDim.x) {
        const long long row0 = t / units * 32;
        const int k0 = (int)(t % units) * 256;
        blocks[tid & 31][tid >> 5] = codes[t * 256 + tid];           // piece (k-step, half) = tid / 32 of row tid % 32
        bytes[tid] = scales[t * 256 + tid];
        __syncthreads();
        const int k = tid % kRowLanes * kPack, block = k >> 5;
#pragma unroll 4
        for (int r = tid / kRowLanes; r < 32; r += 256 / kRowLanes) {
            if (row0 + r >= rows || k0 + k >= cols) continue;
            const uint32_t byte = bytes[((block & 1) * 32 + r) * 4 + (block >> 1)];
            const float scale = __builtin_bit_cast(float, byte ? byte << 23 : 0x00400000u);
            const uint8_t *c = reinterpret_cast<const uint8_t *>(&blocks[r][block]) + (k & 31) / 2;
            PackN<T, kPack> q;
#pragma unroll
            for (int e = 0; e < kPack; e += 4) {
                const uint32_t pair = *reinterpret_cast<const uint16_t *>(c + e / 2);
                const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(pair, scale, 0);
                const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(pair, scale, 1);
                const float v[4] = {a[0], a[1], b[0], b[1]};
#pragma unroll
                for (int j = 0; j < 4; ++j) q.v[e + j] = from_f32<T>(byte == 255 ? __builtin_nanf("") : v[j]);
            }
            T *p = out + (row0 + r) * cols + k0 + k;
            if (aligned) {
                *reinterpret_cast<PackN<T, kPack> *>(p) = q;
            } else {
#pragma unroll
                for (int j = 0; j < kPack; ++j)
                    if (k0 + k + j < cols) p[j] = q.v[j];
            }
        }
        __syncthreads();
    }
}

// ----------------------------------------------------------------------------------------------- linear layer
//
// y [rows][n] = x [rows][K] * w [n][K]^T (+ bias, ReLU), both in MX4.  The weights are the matrix instructions' first
// operand, so a lane ends up with four consecutive features of one row: one store.

__device__ __forceinline__ i32x8 operand(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// 32 x 32 x 64: lane l holds the 32 elements (one block) l/32 of row l%32; 4 = e2m1; the byte of the scale words is
// part of the instruction.
template <int BYTE>
__device__ __forceinline__ f32x16 mfma_mx4_32(i32x4 w, i32x4 x, f32x16 acc, int w_scale, int x_scale) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(x), acc, 4, 4, BYTE, w_scale, BYTE, x_scale);
}
// 16 x 16 x 128: block l/16 of row l%16.
template <int W_BYTE, int X_BYTE>
__device__ __forceinline__ f32x4 mfma_mx4_16(i32x4 w, i32x4 x, f32x4 acc, int w_scale, int x_scale) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), acc, 4, 4, W_BYTE, w_scale, X_BYTE, x_scale);
}

// Bias, ReLU, rounding and store of the N features c .. c + N - 1 of row r.
template <typename T, int N>
__device__ __forceinline__ void store_features(const Mx4Linear &a, long long r, int c, const float *sum, const float (&bias)[N]) {
    const float least = a.relu ? 0.f : -__builtin_inff();
    PackN<T, N> q;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float v = sum[e] + bias[e];
        q.v[e] = from_f32<T>(v < least ? least : v);         // NaN stays NaN
    }
    T *p = static_cast<T *>(a.y) + r * a.y_stride + c;
    if (a.wide && c + N <= a.n) {
        *reinterpret_cast<PackN<T, N> *>(p) = q;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < a.n) p[e] = q.v[e];
    }
}

// Large products on 32 x 32 x 64 tiles (measured alone: 6.5 PFLOP/s with one wave per SIMD, 16 x 16 x 128 3.6).  A block
// of WX x WW waves computes (WX * TX * 32) rows x (WW * TW * 32) features.  A stage is 256 elements of every row, one unit per 32
// rows, brought to LDS by the loads themselves into a ring of RING stages.  Operands are read from LDS AHEAD k-steps
// before they multiply; all waves meet once per stage, when its last operands are in registers: from then on its place in
// the ring is free for the stage RING further on, and the next one's operands are read while the last AHEAD k-steps
// multiply.
// What bounds it: 8192 x 8192 x 8192 takes 292 us (profiles/operators_kernel_stats.csv; boxes differ by a tenth), at which
// the power cap holds the clock: in a row of products alone, where one box took 329, codes of zero took 212, and 291 without
// the loads (68 KB a stage for 2048 clocks of products; touching lines ahead of them saved nothing).  4096 rows of
// 11520 -> 1024 take 33.3 us on 128 x 128 tiles: 4 of it to store, the rest some 1350 clocks for each of the 45 stages, in which
// the products are 512 and the 96 KB of operands out of LDS 768 at 128 B a clock; what keeps these from overlapping is not
// known (29 us without the loads; four waves with half the reads 38).

template <typename T, int WX, int WW, int TX, int TW, int RING, int AHEAD>
__global__ __launch_bounds__(WX *WW * 64, 1) void mx4_tile_kernel(Mx4Linear a) {
    constexpr int kWaves = WX * WW, kRows = WX * TX * 32, kFeatures = WW * TW * 32;
    constexpr int kXUnits = WX * TX, kUnits = kXUnits + WW * TW;     // per stage, of 4 KB; a wave loads kPerWave of them
    constexpr int kPerWave = kUnits / kWaves;
    constexpr int kScaleLoads = kUnits / 4;                          // 1 KB: the scales of four units
    constexpr int kInFlight = (RING - 2) * 4 * kPerWave;             // a wave's loads of codes behind the stage it waits for
    static_assert(kXUnits % 4 == 0 && kUnits % 4 == 0 && kUnits % kWaves == 0 && kScaleLoads <= kWaves, "");
    __shared__ i32x4 lds[RING][kUnits][256];
    __shared__ i32x4 lds_scales[RING][kUnits][16];
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
    const int stages = a.kp / 256;
    // Unit u of the tile: kXUnits of x, then the weights'.  Rows and features past the end repeat the last unit; their
    // results are not stored.
    const long long x_unit0 = row0 / 32, w_unit0 = col0 / 32;
    const int x_left = (int)((rows + 31) / 32 - x_unit0 < kXUnits ? (rows + 31) / 32 - x_unit0 : kXUnits) - 1;
    const int w_left = ((a.n + 31) / 32 - (int)w_unit0 < kUnits - kXUnits ? (a.n + 31) / 32 - (int)w_unit0 : kUnits - kXUnits) - 1;
    auto unit_at = [&](int u) {                                      // units of its tensor before it
        const int i = u < kXUnits ? u : u - kXUnits, left = u < kXUnits ? x_left : w_left;
        return ((u < kXUnits ? x_unit0 : w_unit0) + (i < left ? i : left)) * stages;
    };
    const uint8_t *codes[kPerWave];                                  // this wave's units: wave * kPerWave + i
#pragma unroll
    for (int i = 0; i < kPerWave; ++i) {
        const int u = wave * kPerWave + i;
        codes[i] = (u < kXUnits ? a.x_codes : a.w_codes) + unit_at(u) * 4096;
    }
    const bool loads_scales = wave < kScaleLoads;                    // one load more for the first waves
    const int sload = loads_scales ? wave : 0;
    const uint8_t *scales = (sload * 4 < kXUnits ? a.x_scales : a.w_scales) + unit_at(sload * 4) * 256;
    const uint32_t soffset = (uint32_t)(unit_at(sload * 4 + (lane >> 4)) - unit_at(sload * 4)) * 256 + (lane & 15) * 16;
    constexpr int kLoads = 4 * kPerWave + 1;                         // of a stage, the last one of scales
    auto issue_one = [&](int t, int slot, int n) {
        if (n < 4 * kPerWave)
            load_to_lds(codes[n / 4] + (size_t)t * 4096 + n % 4 * 1024, lane * 16, &lds[slot][wave * kPerWave + n / 4][n % 4 * 64]);
        else if (kScaleLoads == kWaves || loads_scales)
            load_to_lds(scales + (size_t)t * 256, soffset, &lds_scales[slot][sload * 4][0]);
    };
    auto issue = [&](int t, int slot) {
#pragma unroll
        for (int n = 0; n < kLoads; ++n) issue_one(t, slot, n);
    };
    const int ux = wave % WX * TX, uw = kXUnits + wave / WX * TW;    // this wave's first units in the tile

    constexpr int kBuffers = AHEAD == 1 ? 2 : 4;                     // of operands, by k-step
    f32x16 acc[TX][TW] = {};
    i32x4 xf[kBuffers][TX], wf[kBuffers][TW];
    int sx[2][TX], sw[2][TW];
    auto fragments = [&](int slot, auto s) {
        constexpr int S = s;
#pragma unroll
        for (int i = 0; i < TW; ++i) wf[S % kBuffers][i] = lds[slot][uw + i][S * 64 + lane];
#pragma unroll
        for (int i = 0; i < TX; ++i) xf[S % kBuffers][i] = lds[slot][ux + i][S * 64 + lane];
    };
    auto fragment_scales = [&](int slot, int to) {
#pragma unroll
        for (int i = 0; i < TW; ++i) sw[to][i] = reinterpret_cast<const int *>(lds_scales[slot][uw + i])[lane];
#pragma unroll
        for (int i = 0; i < TX; ++i) sx[to][i] = reinterpret_cast<const int *>(lds_scales[slot][ux + i])[lane];
    };
    // The loads of the stage to come have landed (those of later ones may be on their way), this wave has read what it
    // needs of the present one, and after the barrier so have all.
    auto meet = [&](bool all_issued) {
        if (!all_issued) wait_and_meet<0>();
        else if (loads_scales) wait_and_meet<kInFlight + RING - 2>();
        else wait_and_meet<kInFlight>();
    };
    // A k-step's products, with between(n) behind product n.  They stay where they are: nothing orders a matrix instruction
    // and a load by itself.
    auto multiply_with = [&](auto s, auto &&between) {
        constexpr int S = s;
#pragma unroll
        for (int i = 0; i < TX; ++i)
#pragma unroll
            for (int j = 0; j < TW; ++j) {
                acc[i][j] = mfma_mx4_32<S>(wf[S % kBuffers][j], xf[S % kBuffers][i], acc[i][j], sw[0][j], sx[0][i]);
                if constexpr (TX * TW >= 4) asm volatile("" : "+a"(acc[i][j]));
                else asm volatile("" : "+v"(acc[i][j]));
                between(i * TW + j);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](auto s) { multiply_with(s, [](int) {}); };
    // Where a wave has many products and many loads, the loads go out one behind every second product of the last k-step
    // (the stage's place is free from there on) and of the next stage's first: in a row they stop the wave until the
    // memory pipe has taken them all.
    constexpr bool kSpread = TX * TW >= 16;
    constexpr int kFirst = TX * TW / 2;                              // loads of the last k-step
    static_assert(!kSpread || (RING == 2 && AHEAD == 1 && kLoads == TX * TW + 1), "one behind every second product, one more in front");
#pragma unroll
    for (int t = 0; t < RING - 1; ++t)
        if (t < stages) issue(t, t);
    meet(RING - 1 <= stages);
    if (RING - 1 < stages) {
#pragma unroll
        for (int n = 0; n < (kSpread ? kFirst : kLoads); ++n) issue_one(RING - 1, RING - 1, n);
    }
    static_for<AHEAD>([&](auto s) { fragments(0, s); });
    fragment_scales(0, 0);
    int slot = 0;
    for (int t = 0; t + 1 < stages; ++t) {
        const int next = slot + 1 == RING ? 0 : slot + 1;
        static_for<4>([&](auto s) {
            constexpr int S = s;
            if constexpr (S == 4 - AHEAD) {
                meet(!kSpread && t + RING <= stages);
                fragment_scales(next, 1);
            }
            if constexpr (S + AHEAD < 4) fragments(slot, std::integral_constant<int, S + AHEAD>{});
            else fragments(next, std::integral_constant<int, S + AHEAD - 4>{});
            if constexpr (kSpread && S == 3) {                       // behind the last stage the last again, never read
                const int ahead = t + 2 < stages ? t + 2 : stages - 1;
                multiply_with(s, [&](int n) { if (n % 2) issue_one(ahead, slot, n / 2); });
            } else if constexpr (kSpread && S == 0) {                // the rest of the stage begun one step ago
                multiply_with(s, [&](int n) {
                    if (n == 0) issue_one(t + 1, next, kFirst);
                    else if (n % 2) issue_one(t + 1, next, kFirst + 1 + n / 2);
                });
            } else {
                if constexpr (!kSpread && S == 4 - AHEAD)
                    if (t + RING < stages) issue(t + RING, slot);
                multiply(s);
            }
        });
#pragma unroll
        for (int i = 0; i < TX; ++i) sx[0][i] = sx[1][i];
#pragma unroll
        for (int i = 0; i < TW; ++i) sw[0][i] = sw[1][i];
        slot = next;
    }
    static_for<4>([&](auto s) {
        constexpr int S = s;
        if constexpr (S + AHEAD < 4) fragments(slot, std::integral_constant<int, S + AHEAD>{});
        multiply(s);
    });

    // Results leave through LDS (free once all waves are past their last fragment; every wave has its own part), 32 rows
    // at a time, so that a row's features are stored in whole cache lines: straight from the accumulators a lane would
    // write four features of its own row (measured on 8192 x 8192 outputs in bfloat16: 140 us for the stores alone).
    // Loops stay rolled where they can: this code runs once per tile, and what it costs is fetching its instructions.
    constexpr int kWidth = TW * 32, kStride = kWidth + 4, kPack = 16 / sizeof(T), kRowLanes = kWidth / kPack;
    static_assert((kWaves * 32 * kStride + kFeatures) * 4 <= (int)sizeof(lds), "the waves' parts and the bias fit");
    wait_and_meet<0>();
    float *mine = reinterpret_cast<float *>(lds) + wave * 32 * kStride;
    float *bias = reinterpret_cast<float *>(lds) + kWaves * 32 * kStride;
    if ((int)threadIdx.x < kFeatures) {
        const int c = col0 + threadIdx.x;
        bias[threadIdx.x] = a.bias && c < a.n ? load_as_f32(a.bias, a.bias_type, c) : 0.f;
    }
    __syncthreads();
    const int f0 = lane % kRowLanes * kPack, c = col0 + wave / WX * kWidth + f0;
    float b[kPack];
#pragma unroll
    for (int e = 0; e < kPack; ++e) b[e] = bias[wave / WX * kWidth + f0 + e];
#pragma unroll
    for (int i = 0; i < TX; ++i) {
#pragma unroll
        for (int j = 0; j < TW; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x4 v = {acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
                *reinterpret_cast<f32x4 *>(&mine[(lane & 31) * kStride + j * 32 + e * 8 + (lane >> 5) * 4]) = v;
            }
#pragma unroll 2
        for (int q = 0; q < 32 * kRowLanes / 64; ++q) {
            const int in_tile = q * (64 / kRowLanes) + lane / kRowLanes;
            const long long r = row0 + (ux + i) * 32 + in_tile;
            if (r < rows) store_features<T, kPack>(a, r, c, &mine[in_tile * kStride + f0], b);
        }
    }
}

// Few rows, on 16 x 16 x 128 tiles: a block computes RT * 16 rows x 16 features, its eight waves take every eighth 512
// elements of K with fragments straight from memory and add up in LDS in a fixed order.  FUSED (at most 16 rows,
// kMx4FusedElements elements): x comes as numbers and every block quantises them into LDS for itself, which saves a
// launch.  Bound by latency, from the first weights' arrival to the last join: 1 row of 11520 -> 1024 5.9 us, 3 of them
// the launch.
constexpr int kMx4FusedElements = 65536;
constexpr int kRowsWaves = 8;

template <typename T, int RT, typename X, bool FUSED>
__global__ __launch_bounds__(kRowsWaves * 64) void mx4_rows_kernel(Mx4Linear a, const X *__restrict__ x, int cols,
                                                                  long long row_stride, long long col_stride) {
    __shared__ f32x4 part[kRowsWaves][RT][64];
    __shared__ uint32_t xcodes[FUSED ? kMx4FusedElements / 8 : 1];
    __shared__ uint8_t xbytes[FUSED ? kMx4FusedElements / 32 : 1];
    const long long rows = a.row_count && *a.row_count < a.rows ? *a.row_count : a.rows;
    const int feature_tiles = (a.n + 15) / 16;
    const long long row0 = (long long)(blockIdx.x / feature_tiles) * (RT * 16);
    if (row0 >= rows) return;
    // A wave's loop bounds have to be scalar values: matrix instructions ignore the lane mask, so a branch around one must
    // be a real branch.
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, kb = lane >> 4;
    const int col0 = blockIdx.x % feature_tiles * 16;
    const int words = a.kp / 256, chunks = (words + 1) / 2;
    // This lane's block of a k-step of 128 within a unit: k-step kb / 2 (of 64) of its half of the unit, half kb % 2, so
    // 16 bytes at `at` (+ 2048 for the unit's second half) and scale bytes kb / 2 and 2 + kb / 2 of one word.
    auto at = [&](int first) { return (kb >> 1) * 1024 + ((kb & 1) * 32 + (first & 16) + r16) * 16; };
    auto word_at = [&](int first) { return (kb & 1) * 32 + (first & 16) + r16; };
    const int shift = 8 * (kb >> 1);
    const uint8_t *wc = a.w_codes + (size_t)(col0 / 32) * words * 4096 + at(col0);
    const uint32_t *ws = reinterpret_cast<const uint32_t *>(a.w_scales) + (size_t)(col0 / 32) * words * 64 + word_at(col0);
    const uint8_t *xc[RT];
    const uint32_t *xs[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (FUSED) {
            xc[i] = reinterpret_cast<const uint8_t *>(xcodes) + (r16 < rows ? r16 : rows - 1) * (a.kp / 2) + kb * 16;
        } else {
            const long long first = row0 + i * 16 < rows ? row0 + i * 16 : (rows - 1) / 16 * 16;
            xc[i] = a.x_codes + first / 32 * words * 4096 + at((int)(first & 16));
            xs[i] = reinterpret_cast<const uint32_t *>(a.x_scales) + first / 32 * words * 64 + word_at((int)(first & 16));
        }
    }
    i32x4 wf[4];
    int wsc[2] = {};
    auto unit_of = [&](int chunk, int s) { return (size_t)(chunk * 2 + s / 2 < words ? chunk * 2 + s / 2 : words - 1); };
    auto load_w = [&](int chunk) {                   // two units; behind the last one the last again, unused
#pragma unroll
        for (int s = 0; s < 4; ++s) wf[s] = *reinterpret_cast<const i32x4 *>(wc + unit_of(chunk, s) * 4096 + (s & 1) * 2048);
#pragma unroll
        for (int s = 0; s < 2; ++s) wsc[s] = (int)ws[unit_of(chunk, 2 * s) * 64];
    };
    if (wave < chunks) load_w(wave);
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
    for (int chunk = wave; chunk < chunks; chunk += kRowsWaves) {
        i32x4 w4[4], xf[RT][4];
        int sx[RT][4];
        const int sw[2] = {wsc[0] >> shift, wsc[1] >> shift};
#pragma unroll
        for (int s = 0; s < 4; ++s) w4[s] = wf[s];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (FUSED) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int step = (int)unit_of(chunk, s) * 2 + (s & 1);
                    xf[i][s] = *reinterpret_cast<const i32x4 *>(xc[i] + step * 64);
                    sx[i][s] = (int)xbytes[(int)(r16 < rows ? r16 : rows - 1) * (a.kp / 32) + step * 4 + kb];
                }
            } else {
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    xf[i][s] = *reinterpret_cast<const i32x4 *>(xc[i] + unit_of(chunk, s) * 4096 + (s & 1) * 2048);
#pragma unroll
                for (int s = 0; s < 2; ++s) sx[i][s] = (int)xs[i][unit_of(chunk, 2 * s) * 64] >> shift;
            }
        }
        if (chunk + kRowsWaves < chunks) load_w(chunk + kRowsWaves);
        static_for<4>([&](auto s) {
            constexpr int S = s, BYTE = 2 * (S & 1);
            if (chunk * 2 + S / 2 < words) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    if (FUSED) acc[i] = mfma_mx4_16<BYTE, 0>(w4[S], xf[i][S], acc[i], sw[S / 2], sx[i][S]);
                    else acc[i] = mfma_mx4_16<BYTE, BYTE>(w4[S], xf[i][S], acc[i], sw[S / 2], sx[i][S / 2]);
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
            float v[4], bias[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = sum[e];
                bias[e] = a.bias && cf + e < a.n ? load_as_f32(a.bias, a.bias_type, cf + e) : 0.f;
            }
            store_features<T, 4>(a, r, cf, v, bias);
        }
    }
}

}  // namespace

void launch_mx4_quantize(hipStream_t st, int type, long long rows, int cols, const void *x, long long row_stride,
                         long long col_stride, const int32_t *row_count, uint8_t *codes, uint8_t *scales) {
    const int kp = mx4_padded(cols);
    const long long tasks = (rows + 31) / 32 * (kp / 256);
    with_dtype(type, [&](auto t) {
        typedef decltype(t) T;
        mx4_quantize_kernel<T><<<(int)(tasks < 16384 ? tasks : 16384), 256, 0, st>>>(
            static_cast<const T *>(x), rows, cols, kp, row_stride, col_stride, row_count,
            reinterpret_cast<uint4 *>(codes), reinterpret_cast<uint32_t *>(scales));
    });
}

void launch_mx4_dequantize(hipStream_t st, int type, long long rows, int cols, const uint8_t *codes, const uint8_t *scales,
                           void *out) {
    const int kp = mx4_padded(cols);
    const long long tasks = (rows + 31) / 32 * (kp / 256);
    with_dtype(type, [&](auto t) {
        typedef decltype(t) T;
        mx4_dequantize_kernel<T><<<(int)(tasks < 16384 ? tasks : 16384), 256, 0, st>>>(
            reinterpret_cast<const uint4 *>(codes), scales, rows, cols, kp,
            cols * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0, static_cast<T *>(out));
    });
}

namespace {

// Which kernel multiplies: the cheapest by a model of the time in microseconds, fitted to 178 sizes of 17 to 8192 rows, 64 to
// 8192 features and 100 to 16384 columns, 70 of them random, each run in all four forms with a float32 or bfloat16 result
// (profiles/mx4_forms.txt).  The model is off by 8 % of the rows kernel's time in the mean, 4 of the small tiles' and 6 of the
// large ones', by 37 at worst; what it picks takes 0.5 % more than the fastest form in the mean, and 11 at most but for one
// size of 30.  Measured, rows / one / two / large:
//       64 rows of 8192 -> 8192   12.6 / 18.8 / 24.1 / 45.9   rows        64 rows of 1024 -> 8192    5.2 /  6.1 /  7.1 / 13.5   rows
//      256 rows of 8192 -> 8192   42.4 / 20.1 / 25.6 / 49.2   one       2048 rows of 1024 -> 8192   93.5 / 27.3 / 21.8 / 22.5   two
//     2048 rows of 8192 -> 8192    -   / 95.8 / 82.5 / 69.5   large     4096 rows of 4096 -> 4096    157 / 51.7 / 46.9 / 42.7   large
// The rows kernel and the tiles add a row's products in different orders, but all forms of each in one: with `order_rows`
// the choice between the two goes by that count, so that a row's results do not depend on how many come with it.

// As few rows per block (16, 32, 64) as still leave at most a block per CU (128 rows of 11520 -> 1024: 7.2 / 6.2 / 7.6 us with
// 16 / 32 / 64 rows, 64 rows 4.8 / 5.6 / 7.3).
int rows_per_block(long long rows, int n) {
    const long long feature_tiles = (n + 15) / 16;
    if (rows <= 16 || (rows + 15) / 16 * feature_tiles <= 256) return 16;
    return rows <= 32 || (rows + 31) / 32 * feature_tiles <= 256 ? 32 : 64;
}

// Blocks of 64 rows x 16 features, each CU's in turn, the columns' part of a short row hidden behind the latency of its reads;
// or the rows' way from memory to the eight XCDs, where few features leave every XCD almost all of them to read.
double rows_cost(long long rows, int n, int kp) {
    const int per_block = rows_per_block(rows, n), feature_tiles = (n + 15) / 16;
    const double blocks = (double)((rows + per_block - 1) / per_block) * feature_tiles;
    const double compute = std::max(1.0, blocks / 256) * (per_block / 64.0) * std::max(1.35, kp / 1660.0);
    return 2.4 + std::max(compute, (double)rows * kp / 2 * std::min(8, feature_tiles) / 4.6e6);
}

// A tile form: `at_once` tiles of `side` squared work together, which takes a time per stage of 256 elements and one for
// the results, both the longer the more of the tiles there are (a crowd shares memory and power; two blocks a CU, its pipes).
struct TileCost {
    int side, at_once, crowd;                // crowd: 1 linear, 2 quadratic in the share of tiles that are there
    double start, stage, crowded_stage, end, store, f32_store, narrow, narrow_store;
};
constexpr TileCost kOnePerCu = {128, 256, 1, 2.4, 0.43, 0.14, 1.8, 2.0, 0.45, 1.7, 2.3};     // eight waves, ring of four stages
constexpr TileCost kTwoPerCu = {128, 512, 2, 3.9, 0.56, 0.50, 1.0, 3.6, 0.50, 0.8, 7.0};     // four waves, two stages each
constexpr TileCost kLarge = {256, 256, 1, 5.4, 1.10, 0.50, 6.4, 4.4, 0.80, 5.2, 2.8};

double tile_cost(const TileCost &c, long long rows, int n, int kp, bool f32, bool wide) {
    const double tiles = (double)((rows + c.side - 1) / c.side) * ((n + c.side - 1) / c.side);
    const double rounds = std::ceil(tiles / c.at_once), share = tiles / (rounds * c.at_once);
    const double stages = kp / 256 * (c.stage + c.crowded_stage * (c.crowd == 2 ? share * share : share));
    const double stores = c.end + c.store * share * (f32 ? 1.0 + c.f32_store : 1.0) + (wide ? 0.0 : c.narrow + c.narrow_store * share);
    return c.start + rounds * (stages + stores);
}

Mx4Form cheapest_tiles(long long rows, int n, int kp, bool f32, bool wide, double &cost) {
    const double one = tile_cost(kOnePerCu, rows, n, kp, f32, wide), two = tile_cost(kTwoPerCu, rows, n, kp, f32, wide),
                 large = tile_cost(kLarge, rows, n, kp, f32, wide);
    cost = std::min(one, std::min(two, large));
    return cost == one ? MX4_ONE_PER_CU : cost == two ? MX4_TWO_PER_CU : MX4_LARGE;
}

bool rows_form(long long rows, int n, int kp, bool f32, bool wide) {
    double tiles;
    cheapest_tiles(rows, n, kp, f32, wide, tiles);
    return rows <= 16 || rows_cost(rows, n, kp) <= tiles;
}

template <typename T> void launch_product(hipStream_t st, const Mx4Linear &a) {
    auto tiles = [&](int r, int f) { return (a.rows + r - 1) / r * ((a.n + f - 1) / f); };
    switch (mx4_form(a.rows, a.n, a.kp, sizeof(T) == 4, a.wide, a.order_rows)) {
    case MX4_ROWS: {
        auto of_rows = [&](auto rt) {
            constexpr int RT = rt;
            mx4_rows_kernel<T, RT, float, false><<<(unsigned)tiles(RT * 16, 16), kRowsWaves * 64, 0, st>>>(a, nullptr, 0, 0, 0);
        };
        const int per_block = rows_per_block(a.rows, a.n);
        if (per_block == 16) of_rows(std::integral_constant<int, 1>{});
        else if (per_block == 32) of_rows(std::integral_constant<int, 2>{});
        else of_rows(std::integral_constant<int, 4>{});
        break;
    }
    case MX4_LARGE: mx4_tile_kernel<T, 2, 2, 4, 4, 2, 1><<<(unsigned)tiles(256, 256), 256, 0, st>>>(a); break;
    case MX4_TWO_PER_CU: mx4_tile_kernel<T, 2, 2, 2, 2, 2, 2><<<(unsigned)tiles(128, 128), 256, 0, st>>>(a); break;
    case MX4_ONE_PER_CU: mx4_tile_kernel<T, 4, 2, 1, 2, 4, 3><<<(unsigned)tiles(128, 128), 512, 0, st>>>(a); break;
    }
}

}  // namespace

Mx4Form mx4_form(long long rows, int n, int kp, bool f32, bool wide, long long order_rows) {
    double cost;
    const bool by_rows = order_rows > 0 ? rows_form(order_rows, n, kp, f32, wide) : rows_form(rows, n, kp, f32, wide);
    return by_rows ? MX4_ROWS : cheapest_tiles(rows, n, kp, f32, wide, cost);
}

bool mx4_linear_fuses(long long rows, int cols, int n, long long order_rows) {
    return rows <= 16 && rows * mx4_padded(cols) <= kMx4FusedElements &&
           (order_rows <= 0 || rows_form(order_rows, n, mx4_padded(cols), true, true));
}

void launch_mx4_linear(hipStream_t st, Mx4Linear a, const Mx4Rows *x) {
    with_dtype(a.y_type, [&](auto t) {
        typedef decltype(t) T;
        a.wide = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_stride * sizeof(T) % 16 == 0;
        if (x) {
            with_dtype(x->type, [&](auto u) {
                typedef decltype(u) X;
                mx4_rows_kernel<T, 1, X, true><<<(unsigned)((a.n + 15) / 16), kRowsWaves * 64, 0, st>>>(
                    a, static_cast<const X *>(x->x), x->cols, x->row_stride, x->col_stride);
            });
        } else {
            launch_product<T>(st, a);
        }
    });
}

}  // namespace nnb

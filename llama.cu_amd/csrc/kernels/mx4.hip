// Rows to microscaled 4-bit numbers (mx4.h) and back, and rows as the products with 4-bit weights take them.
//
// A block of 32 has the scale 2^(floor(log2 max |x|) - 2), so that its largest number lies in 4 .. 8 of it, held to 2^-127 at least; a
// number goes to the nearest code, ties to the even one, and beyond 6 to 6: the conversion instruction's own rounding, the only one there
// is.  The exponent is the largest magnitude's exponent field less two: magnitudes are compared as integers, under which infinities and
// NaN are the largest, and a block that holds one has the scale 255.  A lane takes 8 neighbours (a load of 16 bytes), four lanes a block.
//
// Bound by memory: a bfloat16 number is 2 bytes read and 17 / 32 written.  28672 x 4096: quantised in 53 to 58 us and read back in 58 to 61, 5.1 to 5.6 TB/s, what a large copy
// reaches; one row of 4096 1.7 us each way, which is the launch.
#include "mx4.h"
#include "rows.h"

constexpr int MX4_THREADS = 256, MX4_UNIT = 8;

// Eight numbers of a row from `at` on, zeros behind its end; WIDE: 16-byte loads are allowed.
template <class T, bool WIDE>
__device__ __forceinline__ void mx4_fetch(const T *__restrict__ row, int at, int k, Pack<T, MX4_UNIT> &v) {
    if (WIDE && at + MX4_UNIT <= k) {
        v = *(const Pack<T, MX4_UNIT> *)(row + at);
    } else {
#pragma unroll
        for (int i = 0; i < MX4_UNIT; ++i) v.v[i] = at + i < k ? row[at + i] : from_f32<T>(0.f);
    }
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t magnitude(bf16_t x) { return (uint32_t)(x.bits & 0x7fffu) << 16; }

// units: 8 numbers each, `row_units` to a row (a multiple of 32: rows are filled up to 256 numbers).
template <class T, bool WIDE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_quantize_kernel(const T *__restrict__ x, size_t ldx, int k, uint32_t units, uint32_t row_units, uint32_t *__restrict__ codes, uint8_t *__restrict__ scales,
                    uint8_t *__restrict__ by_pair, size_t rows) {
    const uint32_t u = blockIdx.x * MX4_THREADS + threadIdx.x;
    if (u >= units) return;                                        // (units are whole waves' halves: a block's four lanes go together)
    const uint32_t row = u / row_units, at = (u - row * row_units) * MX4_UNIT;
    Pack<T, MX4_UNIT> v;
    mx4_fetch<T, WIDE>(x + row * ldx, at, k, v);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < MX4_UNIT; ++i) most = max(most, magnitude(v.v[i]));
    most = max(most, (uint32_t)__builtin_amdgcn_mov_dpp((int)most, 0xB1, 0xF, 0xF, true));      // the lane beside
    most = max(most, (uint32_t)__builtin_amdgcn_mov_dpp((int)most, 0x4E, 0xF, 0xF, true));      // and the two lanes away
    const uint32_t field = most >> 23, e = field == 255 ? 255u : (uint32_t)max((int)field - 2, 0);
    const float scale = __uint_as_float(e ? e << 23 : 0x00400000u);
    uint32_t out = 0;
    if constexpr (sizeof(T) == 2) {
#define PAIR(I) out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(mx4_bf16x2, (uint32_t)v.v[2 * I].bits | (uint32_t)v.v[2 * I + 1].bits << 16), scale, I)
        PAIR(0); PAIR(1); PAIR(2); PAIR(3);
#undef PAIR
    } else {
#define PAIR(I) out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v.v[2 * I], v.v[2 * I + 1], scale, I)
        PAIR(0); PAIR(1); PAIR(2); PAIR(3);
#undef PAIR
    }
    codes[u] = e == 255 ? 0u : out;
    if ((threadIdx.x & 3) == 0) {
        scales[u >> 2] = (uint8_t)e;
        const uint32_t block = at / MX4_BLOCK;
        if (by_pair) by_pair[(block / 8 * rows + row) * 8 + mx4_scale_place(block % 8)] = (uint8_t)e;
    }
}

template <class T, bool WIDE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_values_kernel(const uint8_t *__restrict__ codes, size_t ldc, const uint8_t *__restrict__ scales, size_t lds, int k, uint32_t units, uint32_t row_units,
                  T *__restrict__ y, size_t ldy) {
    const uint32_t u = blockIdx.x * MX4_THREADS + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / row_units, at = (u - row * row_units) * MX4_UNIT;
    uint32_t c = 0;
    const uint8_t *from = codes + row * ldc + at / 2;
    if (WIDE) c = *(const uint32_t *)from;
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) c |= (uint32_t)from[i] << 8 * i;
    const float scale = mx4_scale(scales[row * lds + at / MX4_BLOCK]);
    T *to = y + row * ldy + at;
    Pack<T, MX4_UNIT> v;
    if constexpr (sizeof(T) == 2) {
        const mx4_u32x4 b = mx4_to_bf16(c, scale);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v.v[2 * i].bits = (uint16_t)b[i]; v.v[2 * i + 1].bits = (uint16_t)(b[i] >> 16); }
    } else {
#define PAIR(I) { const mx4_f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, I); v.v[2 * I] = p.x; v.v[2 * I + 1] = p.y; }
        PAIR(0) PAIR(1) PAIR(2) PAIR(3)
#undef PAIR
    }
    if (WIDE && at + MX4_UNIT <= (uint32_t)k) {
        *(Pack<T, MX4_UNIT> *)to = v;
    } else {
#pragma unroll
        for (int i = 0; i < MX4_UNIT; ++i)
            if (at + i < (uint32_t)k) to[i] = v.v[i];
    }
}

// Rows for the products: bfloat16, filled up with zeros to a multiple of 256, and 16-byte aligned.  float32 rows become three planes of bfloat16 one
// behind the other whose sum they are (each takes the next eight bits of the mantissa, cut off and not rounded, so that nothing passes into the
// exponent and what is left is exact): three products with 32-bit sums are then a product of 32-bit rows.  What lies below bfloat16's smallest is
// lost, 2^-133; infinities and NaN are the first plane's alone.
template <class T, bool WIDE>
__global__ void __launch_bounds__(MX4_THREADS)
mx4_rows_kernel(const T *__restrict__ x, size_t ldx, int k, uint32_t units, uint32_t row_units, uint32_t *__restrict__ out) {
    const uint32_t u = blockIdx.x * MX4_THREADS + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / row_units, unit = u - row * row_units;
    Pack<T, MX4_UNIT> v;
    mx4_fetch<T, WIDE>(x + row * ldx, unit * MX4_UNIT, k, v);
    if constexpr (sizeof(T) == 2) {
        mx4_u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = (uint32_t)v.v[2 * i].bits | (uint32_t)v.v[2 * i + 1].bits << 16;
        *(mx4_u32x4 *)(out + (size_t)u * 4) = o;
    } else {
        uint32_t *to = out + ((size_t)row * 3 * row_units + unit) * 4;
#pragma unroll
        for (int plane = 0; plane < 3; ++plane) {
            mx4_u32x4 o;
#pragma unroll
            for (int i = 0; i < MX4_UNIT; ++i) {
                const uint32_t bits = __float_as_uint(v.v[i]);
                // (a NaN whose mantissa's upper bits are zeros would become an infinity)
                const uint32_t top = (bits & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : bits & 0xffff0000u;
                o[i / 2] = i & 1 ? o[i / 2] | top : top >> 16;
                v.v[i] = (bits & 0x7f800000u) == 0x7f800000u ? 0.f : v.v[i] - __uint_as_float(top);
            }
            *(mx4_u32x4 *)(to + (size_t)plane * row_units * 4) = o;
        }
    }
}

static bool mx4_wide(const void *p, long long ld, int type) { return (uintptr_t)p % 16 == 0 && ld * (type == LCU_BF16 ? 2 : 4) % 16 == 0; }

// What is one of `rows` rows of `k` numbers, filled up to `row_units` units: the number of units, or 0 where they are too many for one launch.
static uint32_t mx4_units(long long rows, long long row_units) {
    const long long units = rows * row_units;
    return units > 0 && units < 1ll << 31 ? (uint32_t)units : 0u;
}

// Scales [rows, lds], whole pairs of macro-steps, as the products in tiles read them: [pairs][rows][8].
__global__ void __launch_bounds__(MX4_THREADS)
mx4_by_pair_kernel(const uint8_t *__restrict__ scales, size_t lds, size_t rows, int pairs, uint8_t *__restrict__ out) {
    const size_t row = (size_t)blockIdx.x * MX4_THREADS + threadIdx.x;
    if (row >= rows) return;
    for (int p = blockIdx.y; p < pairs; p += gridDim.y) {
        uint8_t s[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) s[mx4_scale_place(b)] = scales[row * lds + 8 * p + b];
        uint64_t all = 0;
#pragma unroll
        for (int b = 0; b < 8; ++b) all |= (uint64_t)s[b] << 8 * b;
        *(uint64_t *)(out + ((size_t)p * rows + row) * 8) = all;
    }
}

// The number of the capture into a graph that a stream is in, 0: none.
LCU_API int lcu_capture_id(hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (stream && hipStreamGetCaptureInfo(stream, &status, &id) != hipSuccess) (void)hipGetLastError();
    return status == hipStreamCaptureStatusNone ? 0 : (int)(id % 0x7fffffff) + 1;
}

// scales: [rows, lds] bytes, 8 pairs of them in every row; out: [pairs][rows][8], 8-byte aligned.
LCU_API int lcu_mx4_by_pair(const void *scales, long long lds, long long rows, int pairs, void *out, hipStream_t stream) {
    if (rows <= 0 || pairs <= 0) return LCU_OK;
    const long long groups = (rows + MX4_THREADS - 1) / MX4_THREADS;
    if (!scales || !out || (uintptr_t)out % 8 || (rows > 1 && lds < 8 * (long long)pairs) || groups > 0x7fffffff) return LCU_BAD_ARGUMENT;
    mx4_by_pair_kernel<<<dim3((unsigned)groups, (unsigned)min(pairs, 256)), dim3(MX4_THREADS), 0, stream>>>((const uint8_t *)scales, (size_t)lds, (size_t)rows, pairs, (uint8_t *)out);
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

// x: [rows, ldx] of `type`; codes: [rows][kp / 2], scales: [rows][kp / 32] with kp = k rounded up to 256, codes 4-byte aligned; by_pair: null, or the scales once more as the products in
// tiles read them, [kp / 256][rows][8], a row's eight as in mx4.h.
LCU_API int lcu_mx4_quantize(const void *x, long long ldx, int type, long long rows, int k, void *codes, void *scales, void *by_pair, hipStream_t stream) {
    if (rows <= 0 || k <= 0) return LCU_OK;
    const long long row_units = ((long long)k + MX4_PAIR - 1) / MX4_PAIR * (MX4_PAIR / MX4_UNIT);
    const uint32_t units = mx4_units(rows, row_units);
    if (!units || !x || !codes || !scales || (uintptr_t)codes % 4 || (rows > 1 && ldx < k) || (type != LCU_BF16 && type != LCU_F32)) return LCU_BAD_ARGUMENT;
    const dim3 grid((units + MX4_THREADS - 1) / MX4_THREADS), block(MX4_THREADS);
    const bool wide = mx4_wide(x, ldx, type);
#define GO(T, WIDE) mx4_quantize_kernel<T, WIDE><<<grid, block, 0, stream>>>((const T *)x, (size_t)ldx, k, units, (uint32_t)row_units, (uint32_t *)codes, (uint8_t *)scales, (uint8_t *)by_pair, (size_t)rows)
    if (type == LCU_BF16) { if (wide) GO(bf16_t, true); else GO(bf16_t, false); }
    else { if (wide) GO(float, true); else GO(float, false); }
#undef GO
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

// codes: [rows, ldc] bytes, scales: [rows, lds] bytes, whole blocks of 32 in both; y: [rows, ldy] of `type`.
LCU_API int lcu_mx4_values(const void *codes, long long ldc, const void *scales, long long lds, long long rows, int k, void *y, long long ldy, int type,
                           hipStream_t stream) {
    if (rows <= 0 || k <= 0) return LCU_OK;
    const long long row_units = ((long long)k + MX4_UNIT - 1) / MX4_UNIT;
    const uint32_t units = mx4_units(rows, row_units);
    if (!units || !codes || !scales || !y || (rows > 1 && (ldc < (k + 1) / 2 || lds < 1 || ldy < k)) || (type != LCU_BF16 && type != LCU_F32)) return LCU_BAD_ARGUMENT;
    const dim3 grid((units + MX4_THREADS - 1) / MX4_THREADS), block(MX4_THREADS);
    const bool wide = mx4_wide(y, ldy, type) && (uintptr_t)codes % 4 == 0 && ldc % 4 == 0;
#define GO(T, WIDE) mx4_values_kernel<T, WIDE><<<grid, block, 0, stream>>>((const uint8_t *)codes, (size_t)ldc, (const uint8_t *)scales, (size_t)lds, k, units, (uint32_t)row_units, (T *)y, (size_t)ldy)
    if (type == LCU_BF16) { if (wide) GO(bf16_t, true); else GO(bf16_t, false); }
    else { if (wide) GO(float, true); else GO(float, false); }
#undef GO
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

// x: [rows, ldx] of `type`; out: [rows][planes][kp] bfloat16, kp = k rounded up to 256, planes 1 (bfloat16) or 3 (float32), 16-byte aligned.
LCU_API int lcu_mx4_rows(const void *x, long long ldx, int type, long long rows, int k, void *out, hipStream_t stream) {
    if (rows <= 0 || k <= 0) return LCU_OK;
    const long long row_units = ((long long)k + MX4_PAIR - 1) / MX4_PAIR * (MX4_PAIR / MX4_UNIT);
    const uint32_t units = mx4_units(rows, row_units);
    if (!units || !x || !out || (uintptr_t)out % 16 || (rows > 1 && ldx < k) || (type != LCU_BF16 && type != LCU_F32)) return LCU_BAD_ARGUMENT;
    const dim3 grid((units + MX4_THREADS - 1) / MX4_THREADS), block(MX4_THREADS);
    const bool wide = mx4_wide(x, ldx, type);
#define GO(T, WIDE) mx4_rows_kernel<T, WIDE><<<grid, block, 0, stream>>>((const T *)x, (size_t)ldx, k, units, (uint32_t)row_units, (uint32_t *)out)
    if (type == LCU_BF16) { if (wide) GO(bf16_t, true); else GO(bf16_t, false); }
    else { if (wide) GO(float, true); else GO(float, false); }
#undef GO
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

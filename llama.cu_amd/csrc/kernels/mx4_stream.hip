// Y[M, N] = X[M, K] * W[N, K]^T with W in microscaled 4-bit numbers (mx4.h), 32-bit sums: the kernels that stream W past up to 64 rows.
//
// A workgroup takes NT tiles of 16 features (for SwiGLU the gate rows of a tile and the up rows that meet them) and 16 MT rows; its eight waves (four where there are more workgroups than
// the card holds at once) share out K in pairs of macro-steps (256 k) and add their partial sums through LDS in a fixed order.  Rows of bfloat16: the codes become bfloat16
// in registers, exactly and with their scale, two a conversion, in the order in which the matrix instruction of 16 x 16 x 32 wants its operand.  Rows of
// float32 come as three planes of bfloat16 whose sum they are, each multiplied with the same codes.  Rows in 4 bits: the scaled instruction of 16 x 16 x 128
// takes both sides' codes and scales as they are.
//
// Bound by memory where the weight is large, by the latency of a wave's chain of loads where it is not (a wave has K / 8, of which two pairs of macro-steps are on their way; K is
// split over the waves of one workgroup and no further, so that no second launch adds the parts).  One row: 6144 x 4096 4.8 us (2.8 TB/s), 128256 x 4096 45 to 48 (5.8 to 6.2 TB/s); 8 rows:
// 28672 x 4096 with the activation 14.6 to 16 us (3.9 to 4.3 TB/s), 57344 x 8192 46 to 49 (5.1 to 5.4).  Rows in float32 and in 4 bits, weights out of memory, the gap between launches and the rows' planes
// included: 6144 x 4096 one row 9.7 and 6.2 us, 28672 x 4096 four rows in float32 24, eight in 4 bits 18, 4104 x 11008 four rows in float32 18, 4096 x 14336 twelve in 4 bits 14.  Beyond 8 rows every workgroup's reading of
// all rows out of the L2 caches weighs more and the products in tiles take over.
#include "mx4.h"
#include "mx4/matrix.h"
#include "gate_act.h"
#include "quad_rows.h"
#include "../shared/per_device.h"

enum { MX4_EPI_BF16 = 0, MX4_EPI_F32 = 1, MX4_EPI_SWIGLU = 2, MX4_EPI_SWIGLU_F32 = 3 };

constexpr int MX4_WAVES = 8, MX4_MAX_LDX = 1 << 24;

// What a kernel needs to know of the weight and of where the sums go.
struct Mx4Args {
    const uint8_t *codes, *scales;
    int pairs, macros;              // pairs of macro-steps in W; macro-steps that count
    void *y;
    long long ldy;
    int M, N;                       // rows and features (SwiGLU: both halves)
    int wide_out;                   // four neighbours may be stored at once
};

// Where the tiles of a workgroup stand: a lane's rows of W.
template <int NT, int EPI>
__device__ __forceinline__ void mx4_rows_of(const Mx4Args &a, int l16, int (&row)[NT]) {
    const int last = (a.N + 15) / 16 * 16 - 1;
#pragma unroll
    for (int n = 0; n < NT; ++n)
        row[n] = min(EPI >= MX4_EPI_SWIGLU ? (int)blockIdx.x * 16 + l16 + n * (a.N / 2) : ((int)blockIdx.x * NT + n) * 16 + l16, last);
}

// The waves' sums, added and stored: acc[n][m] of lane (g, c) are features 4 g .. + 3 of tile n and row token(c) of tile m.
template <int NT, int MT, int EPI, class Token>
__device__ __forceinline__ void mx4_finish(const Mx4Args &a, int row0, mx4_f32x4 (&acc)[NT][MT], mx4_f32x4 (*red)[NT * MT][WAVE], Token token) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) red[wave][n * MT + m][lane] = acc[n][m];
    __syncthreads();
    auto total = [&](int t) {
        mx4_f32x4 v = red[0][t][lane];
        for (int w = 1; w < waves; ++w) v += red[w][t][lane];
        return v;
    };
    constexpr bool SWIGLU = EPI >= MX4_EPI_SWIGLU, F32 = EPI == MX4_EPI_F32 || EPI == MX4_EPI_SWIGLU_F32;
    const int cols = SWIGLU ? a.N / 2 : a.N;
    for (int t = wave; t < (SWIGLU ? MT : NT * MT); t += waves) {
        const int m = t % MT, row = row0 + 16 * m + token(c), col = (SWIGLU ? (int)blockIdx.x : (int)blockIdx.x * NT + t / MT) * 16 + 4 * g;
        mx4_f32x4 v = total(t);
        if constexpr (SWIGLU) {
            const mx4_f32x4 up = total(MT + m);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = gate_up<GATE_SILU>(v[i], up[i], 0.f, 0.f);
        }
        if (row >= a.M || col >= cols) continue;
        if constexpr (F32) {
            float *to = (float *)a.y + row * a.ldy + col;
            if (a.wide_out && col + 4 <= cols) *(mx4_f32x4 *)to = v;
            else
                for (int i = 0; i < 4 && col + i < cols; ++i) to[i] = v[i];
        } else {
            bf16_t *to = (bf16_t *)a.y + row * a.ldy + col;
            if (a.wide_out && col + 4 <= cols) *(uint2 *)to = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
            else
                for (int i = 0; i < 4 && col + i < cols; ++i) to[i] = from_f32<bf16_t>(v[i]);
        }
    }
}

// X: [M, ldx] bfloat16, a row's PLANES planes `plane` numbers apart; LOADS: loads of 128 k of a tile's rows (quad_rows.h).
template <int NT, int MT, int PLANES, int EPI, int LOADS>
__global__ void __launch_bounds__(MX4_WAVES *WAVE)
mx4_stream_kernel(const bf16_t *__restrict__ X, int ldx, int plane, Mx4Args a) {
    constexpr int AHEAD = 2;                         // pairs of macro-steps of W on their way
    __shared__ mx4_f32x4 red[MX4_WAVES][NT * MT][WAVE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int pairs = (a.macros + 1) / 2, per = (pairs + waves - 1) / waves, p0 = min(pairs, wave * per), p1 = min(pairs, p0 + per);
    const int row0 = blockIdx.y * 16 * MT, rows = min(a.M - row0, 16 * MT);
    int at[NT];
    mx4_rows_of<NT, EPI>(a, l16, at);
    const uint8_t *wc[NT], *ws[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        wc[n] = a.codes + mx4_row_codes(at[n], a.pairs) + g * 256;
        ws[n] = a.scales + mx4_row_scales(at[n], a.pairs);
    }
    // a buffer that ends with the last row's k: rows beyond it read zeros
    const __amdgpu_buffer_rsrc_t xb = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t *>(X) + (size_t)row0 * ldx, 0, (uint32_t)((rows - 1) * ldx + (PLANES - 1) * plane + a.macros * 128) * 2u, 0x00020000);
    const uint32_t place = (uint32_t)(quad_load_row(0, lane) * ldx + quad_k(lane)) * 2u, four = 8u * ldx;
    mx4_f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = mx4_f32x4{0.f, 0.f, 0.f, 0.f};
    mx4_u32x4 code[AHEAD][NT][2], b[MT * PLANES][LOADS];
    uint32_t scale[AHEAD][NT];                       // of the lane's odd or even blocks
    auto fetch_w = [&](int u, int p) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            scale[u][n] = *(const uint32_t *)(ws[n] + (size_t)p * MX4_PAIR_SCALES + 4 * (g & 1));
#pragma unroll
            for (int h = 0; h < 2; ++h) code[u][n][h] = __builtin_nontemporal_load((const mx4_u32x4 *)(wc[n] + (size_t)p * MX4_PAIR_CODES + 1024 * h));
        }
    };
    auto fetch_x = [&](int m, int plane_of, int s) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            b[m * PLANES + plane_of][i] = __builtin_bit_cast(mx4_u32x4, __builtin_amdgcn_raw_buffer_load_b128(xb, place + (4 * m + i) * four + 2u * plane_of * plane + 256u * s, 0, 0));
    };
    auto fetch_all_x = [&](int s) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < PLANES; ++q) fetch_x(m, q, s);
    };
    // the last matrix instructions' wait, which the compiler leaves a state short behind the branches of the loop
    auto wait_for_sums = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) asm volatile("s_nop 3" : "+v"(acc[n][MT - 1]));
    };
    auto macro_step = [&](int u, int h, int s, int next) {
        mx4_u32x4 w[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float sc = mx4_scale((scale[u][n] >> 8 * (2 * h + (g >> 1))) & 255u);      // block 4 h + g
#pragma unroll
            for (int j = 0; j < 4; ++j) w[n][j] = mx4_to_bf16(code[u][n][h][j], sc);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < PLANES; ++q) {
                mx4_u32x4 x[4];
                quad_operands<LOADS>(b[m * PLANES + q], x);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[n][m] = mx4_multiply_16(w[n][j], x[j], acc[n][m]);
                if (next < a.macros) fetch_x(m, q, next);
            }
        wait_for_sums();
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (p0 + u < p1) fetch_w(u, p0 + u);
    if (p0 < p1) fetch_all_x(2 * p0);
    for (int p = p0; p < p1; p += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (p + u >= p1) break;
            const int s = 2 * (p + u);
            macro_step(u, 0, s, s + 1);
            if (s + 1 < a.macros) macro_step(u, 1, s + 1, p + u + 1 < p1 ? s + 2 : a.macros);
            if (p + u + AHEAD < p1) fetch_w(u, p + u + AHEAD);
        }
    }
    mx4_finish<NT, MT, EPI>(a, row0, acc, red, [](int c) { return quad_row(c); });
}

// X in 4 bits: codes [M, ldx] bytes and scales [M, lds] bytes, whole macro-steps of 128 k.
template <int NT, int MT, int EPI>
__global__ void __launch_bounds__(MX4_WAVES *WAVE)
mx4_stream4_kernel(const uint8_t *__restrict__ X, int ldx, const uint8_t *__restrict__ XS, int lds, Mx4Args a) {
    __shared__ mx4_f32x4 red[MX4_WAVES][NT * MT][WAVE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int per = (a.macros + waves - 1) / waves, s0 = min(a.macros, wave * per), s1 = min(a.macros, s0 + per);
    const int row0 = blockIdx.y * 16 * MT;
    int at[NT];
    mx4_rows_of<NT, EPI>(a, l16, at);
    const uint8_t *wc[NT], *ws[NT], *xc[MT], *xs[MT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        wc[n] = a.codes + mx4_row_codes(at[n], a.pairs) + g * 256;
        ws[n] = a.scales + mx4_row_scales(at[n], a.pairs);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const size_t row = min(row0 + 16 * m + l16, a.M - 1);       // (rows behind the last are multiplied and not stored)
        xc[m] = X + row * ldx + g * 16;
        xs[m] = XS + row * lds;
    }
    mx4_f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = mx4_f32x4{0.f, 0.f, 0.f, 0.f};
    // W comes from memory, four macro-steps on their way; the rows from the L2 caches, two
    constexpr int AHEAD_W = 4, AHEAD_X = 2;
    mx4_u32x4 w[AHEAD_W][NT], x[AHEAD_X][MT];
    uint32_t wscale[AHEAD_W][NT], xscale[AHEAD_X][MT];
    auto fetch_w = [&](int u, int s) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            w[u][n] = __builtin_nontemporal_load((const mx4_u32x4 *)(wc[n] + (size_t)s * 1024));
            wscale[u][n] = *(const uint32_t *)(ws[n] + (size_t)(s >> 1) * MX4_PAIR_SCALES + 4 * (g & 1)) >> 8 * (2 * (s & 1) + (g >> 1));      // block 4 (s & 1) + g
        }
    };
    auto fetch_x = [&](int u, int s) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            x[u][m] = *(const mx4_u32x4 *)(xc[m] + (size_t)s * 64);
            xscale[u][m] = *(const uint32_t *)(xs[m] + (size_t)s * 4);
        }
    };
#pragma unroll
    for (int u = 0; u < AHEAD_W; ++u)
        if (s0 + u < s1) fetch_w(u, s0 + u);
#pragma unroll
    for (int u = 0; u < AHEAD_X; ++u)
        if (s0 + u < s1) fetch_x(u, s0 + u);
    for (int s = s0; s < s1; s += AHEAD_W) {
#pragma unroll
        for (int u = 0; u < AHEAD_W; ++u) {
            if (s + u >= s1) break;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    acc[n][m] = mx4_multiply_codes_16<0>(w[u][n], x[u % AHEAD_X][m], acc[n][m], wscale[u][n], xscale[u % AHEAD_X][m] >> 8 * g);
#pragma unroll
            for (int n = 0; n < NT; ++n) asm volatile("s_nop 7" : "+v"(acc[n][MT - 1]));      // (the last products' wait, which the compiler leaves short behind a branch)
            if (s + u + AHEAD_W < s1) fetch_w(u, s + u + AHEAD_W);
            if (s + u + AHEAD_X < s1) fetch_x(u % AHEAD_X, s + u + AHEAD_X);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) asm volatile("s_nop 15" : "+v"(acc[n][m]));      // (the last products are there before they are read, whatever lies between)
    mx4_finish<NT, MT, EPI>(a, row0, acc, red, [](int c) { return c; });
}

// How many workgroups of eight waves the current device holds at once (more than any launch has, where it does not say).
static long long mx4_held(const void *kernel, LcuPerDevice &known) {
    constexpr long long UNKNOWN = 1ll << 40;
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess) device = -1;
    const long long held = known.get(device, [kernel](int of) {
        int each = 0, units = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, MX4_WAVES * WAVE, 0) != hipSuccess || hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, of) != hipSuccess) return 0ll;
        return (long long)each * units;
    }, UNKNOWN);
    if (held == UNKNOWN) (void)hipGetLastError();
    return held;
}

// codes, scales: W in the products' order, [ceil(N / 16)][pairs] blocks, 16-byte aligned.  x_kind: 1 bfloat16 rows [M, ldx]; 3 float32 rows as
// planes [M][3][ldx / 3]; 4 codes [M, ldx] bytes with scales xs [M, lds] bytes; all of
// them in whole macro-steps of 128 k, zeros behind K.  epi: MX4_EPI_*; SwiGLU: N counts gate and up rows.
LCU_API int lcu_mx4_stream(const void *x, long long ldx, int x_kind, const void *xs, long long lds, const void *codes, const void *scales, int pairs, void *y, long long ldy,
                           int M, int N, int K, int epi, hipStream_t stream) {
    if (M <= 0 || N <= 0) return LCU_OK;
    const int macros = (K + 127) / 128, cols = epi >= MX4_EPI_SWIGLU ? N / 2 : N, elem = epi == MX4_EPI_F32 || epi == MX4_EPI_SWIGLU_F32 ? 4 : 2;
    if (K <= 0 || pairs < (macros + 1) / 2 || ldy < cols || epi < 0 || epi > MX4_EPI_SWIGLU_F32 || (epi >= MX4_EPI_SWIGLU && N % 2) || !x || !codes || !scales || !y ||
        ((uintptr_t)x | (uintptr_t)codes) % 16 || (uintptr_t)scales % 8 || ldx < 0 || ldx >= MX4_MAX_LDX)
        return LCU_BAD_ARGUMENT;
    if (x_kind == 1 ? ldx % 8 || ldx < 128ll * macros : x_kind == 3 ? ldx % 24 || ldx < 3ll * macros * 128
        : x_kind == 4 ? ldx % 16 || lds % 4 || !xs || (uintptr_t)xs % 4 || lds >= MX4_MAX_LDX || (M > 1 && (ldx < 64ll * macros || lds < 4ll * macros)) : true)
        return LCU_BAD_ARGUMENT;
    const Mx4Args a = {(const uint8_t *)codes, (const uint8_t *)scales, pairs, macros, y, ldy, M, N, ((uintptr_t)y | (uintptr_t)(ldy * elem)) % (4 * elem) == 0};
    const int tiles = (cols + 15) / 16, work = x_kind == 4 ? macros : (macros + 1) / 2;
    // two tiles of features a workgroup where there are many, and more than four rows are read for them (us, one tile / two, weights out of memory: 16384 x 2048 16 rows 9.5 / 8.1, 28672 x 4096
    // 16 rows 24.8 / 20.6, 128256 x 4096 8 rows 61.8 / 51.6; one row 45.3 / 47.9; 4096 x 14336 8 rows 12.4 / 14.7)
    const bool pairs_of = x_kind == 1 && M > 4 && M <= 16 && N > 8192 && epi < MX4_EPI_SWIGLU;
    auto grid = [&](int nt, int mt) { return dim3(epi >= MX4_EPI_SWIGLU ? tiles : (tiles + nt - 1) / nt, (M + 16 * mt - 1) / (16 * mt)); };
    if ((M + 15) / 16 > 65535) return LCU_BAD_ARGUMENT;
    // Eight waves a workgroup, four where the card does not hold all workgroups of eight at once: half as many waves then go through twice the K each, and there are fewer rounds, the last of
    // them fuller (us, eight / four: 28672 x 4096 with the activation, 8 rows, 17.7 / 15.6; 128256 x 4096, one row, 55.7 / 48.1; 57344 x 8192 50.7 / 46.4; held at once: 6144 x 4096 5.5 / 6.5,
    // 4096 x 14336 11.3 / 14.9).  Over 595 shapes and kinds of rows 1.01 times the best of two to eight waves.
    auto block = [&](dim3 g, long long held) { return dim3(min((long long)g.x * g.y > held ? MX4_WAVES / 2 : MX4_WAVES, work) * WAVE); };
#define RUN(NT, MT, KERNEL, ...)                                                      \
    do {                                                                              \
        static LcuPerDevice held;                                                     \
        const dim3 g = grid(NT, MT);                                                  \
        KERNEL<<<g, block(g, mx4_held((const void *)KERNEL, held)), 0, stream>>>(__VA_ARGS__); \
    } while (0)
#define GO(NT, MT, PLANES, EPI, LOADS) RUN(NT, MT, (mx4_stream_kernel<NT, MT, PLANES, EPI, LOADS>), (const bf16_t *)x, (int)ldx, (int)(PLANES == 3 ? ldx / 3 : 0), a)
#define GO4(NT, MT, EPI) RUN(NT, MT, (mx4_stream4_kernel<NT, MT, EPI>), (const uint8_t *)x, (int)ldx, (const uint8_t *)xs, (int)lds, a)
#define ROWS(NT, EPI)                                      \
    do {                                                   \
        if (x_kind == 4) {                                 \
            if (M <= 16) GO4(NT, 1, EPI);                  \
            else if (M <= 32) GO4(NT, 2, EPI);             \
            else GO4(NT, 4, EPI);                          \
        } else if (x_kind == 3) {                          \
            if (M <= 4) GO(NT, 1, 3, EPI, 1);              \
            else if (M <= 16) GO(NT, 1, 3, EPI, 4);        \
            else GO(NT, NT == 1 ? 2 : 1, 3, EPI, 4);       \
        } else {                                           \
            if (M <= 4) GO(NT, 1, 1, EPI, 1);              \
            else if (M <= 8) GO(NT, 1, 1, EPI, 2);         \
            else if (M <= 16) GO(NT, 1, 1, EPI, 4);        \
            else if (M <= 32) GO(NT, 2, 1, EPI, 4);        \
            else GO(NT, 4, 1, EPI, 4);                     \
        }                                                  \
    } while (0)
    if (epi == MX4_EPI_SWIGLU) ROWS(2, MX4_EPI_SWIGLU);
    else if (epi == MX4_EPI_SWIGLU_F32) ROWS(2, MX4_EPI_SWIGLU_F32);
    else if (pairs_of) { if (epi == MX4_EPI_BF16) ROWS(2, MX4_EPI_BF16); else ROWS(2, MX4_EPI_F32); }
    else if (epi == MX4_EPI_BF16) ROWS(1, MX4_EPI_BF16);
    else ROWS(1, MX4_EPI_F32);
#undef RUN
#undef GO
#undef GO4
#undef ROWS
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

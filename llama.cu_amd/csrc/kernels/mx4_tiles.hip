// Y[M, N] = X[M, K] * W[N, K]^T with W in microscaled 4-bit numbers (mx4.h), 32-bit sums: many rows, in tiles.
//
// A workgroup has a tile of F features and T tokens.  Both operands come by loads that write into LDS themselves, in rings of their own of SF and ST
// steps; a wave multiplies 32 FT features and 32 TT tokens.  One barrier a step, in the middle of it: the products of a step's last slice, and then of
// each slice, run while the next slice is read, so the matrix cores have work on both sides of the barrier.
//
//   rows in bfloat16   a step is 64 k.  A lane reads a block of 32 codes of a feature at once, a step's worth, and makes the operands of the four
//                      slices (32 x 32 x 16) out of it as they are needed; W takes a quarter of the LDS and of its bandwidth that bfloat16 would.
//                      The waves stand four by features and two by tokens, since every wave converts its own features' codes.
//   rows in float32    come as three planes of bfloat16 whose sum they are, and a step takes all three: the features' operands are made once for them.  (As rows of three times the
//                      k, with W gone through three times: 37 x 4104 x 11008 31.3 us, so 26.4; 1600 x 6144 x 4096 223 us, so 211.)
//   rows in 4 bits     a step is 256 k, a slice 64 (32 x 32 x 64, scaled); the scales, four bytes a lane and step, come into registers.  Steps of 128 k, which the rings hold more of,
//                      took a tenth longer: half a line a row and load.
//
// The rings are waited for by counting their own loads (MtShape::LEFT).  The scales come into registers a step ahead, and waits are for everything asked for before: the compiler's wait for a
// step's scales is one for all loads of the steps before the last.  So a load has a step's time, also in rings of four stages, whose count alone would leave it two.
//
// Which tile: the largest that fills the card, and where none does slices of K beside each other, whose sums a second launch adds (the rule and its figures stand where the kernel is
// chosen).  Rows in 4 bits have waves of 128 x 128 and one a SIMD, which read half of what waves of 64 x 128 do out of LDS a product (8192 x 28672 with 4,096 rows 480 us, so 430).
// Many rows are bound by the matrix cores at the clock that the power limit leaves, and by what waves wait for each other: 28672 x 4096 with the activation, 2,048 rows in bfloat16 371 to 390 us
// (1.23 to 1.30 PFLOP/s; the library's bfloat16 product alone 354 to 399): matrix cores busy 64 % of the time at 1.6 to 1.8 GHz, a quarter of the waves' time waiting for loads; 8192 x 28672, 4,096
// rows in 4 bits 412 to 430 us (4.5 to 4.7 PFLOP/s), 65 % at 1.6 to 1.7 GHz, a fifth.  Few rows by the loads' latency: 4096 x 14336, 64 rows in 4 bits 9.5 to 10.9 us and 3.9 for the slices' sums
// (matrix cores 5 % busy, 57 % of the waves' time waiting for loads); 28672 x 4096, 24 rows, with the activation 18.4 us; 4104 x 11008, 37 rows in float32 20.4 us and 4 (30 %, 25 %).
#include <type_traits>
#include "mx4.h"
#include "mx4/matrix.h"
#include "gate_act.h"

enum { MT_EPI_BF16 = 0, MT_EPI_F32 = 1, MT_EPI_SWIGLU = 2, MT_EPI_SWIGLU_F32 = 3 };

template <int LEFT>
__device__ __forceinline__ void mt_wait_loads() {
    static_assert(LEFT >= 0 && LEFT < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt((LEFT & 15) | ((LEFT >> 4) << 14) | (7 << 4) | (15 << 8));
}

// FOUR: rows in 4 bits.  SF, ST: steps of features and of tokens that the rings hold.  P: planes of a row that a step takes, one product each with the same features.
template <bool FOUR_, int FT_, int TT_, int WF_, int WT_, int SF_, int ST_, int P_ = 1> struct MtShape {
    static constexpr bool FOUR = FOUR_;
    static constexpr int FT = FT_, TT = TT_, WF = WF_, WT = WT_, SF = SF_, ST = ST_, P = P_, TOKENS = TT * P, SLICES = 4;
    static constexpr int WAVES = WF * WT, THREADS = WAVES * WAVE, F = 32 * FT * WF, T = 32 * TT * WT;
    static constexpr int FP = FOUR ? 8 : 2, TP = 8;                    // pieces (16 bytes) of a row a stage
    static constexpr int STEP_CODES = 256 * FP;                        // bytes of a tile of 16 features a step
    static constexpr int LF = F * FP / WAVE / WAVES, LT = P * T * TP / WAVE / WAVES;       // loads of a wave a stage
    static constexpr int LDS = SF * F * FP + ST * P * T * TP;              // pieces
    // Loads that may be on their way when a step begins: the rings' that are asked for behind the last of the step's own stages (a turn asks for tokens and then for features, and of the first step's
    // stages the features, further ahead, come first).  Scales' loads are not counted, wherever the compiler puts them among these: more of them on their way make the wait longer, never shorter.
    static constexpr int LEFT = (SF > ST ? LF : 0) + (ST - 2) * (LF + LT);
    static_assert(FT % 2 == 0 && F * FP % (WAVE * WAVES) == 0 && T * P * TP % (WAVE * WAVES) == 0 && (P == 1 || !FOUR) && SF >= ST && ST >= 2 && LDS * 16 <= 160 * 1024, "whole loads, and room for the stages");
};

// Where piece c of row r stands among the row's in LDS: sixteen neighbouring rows' pieces c lie in sixteen places that are read at once (c ^ (r & 7), in eight: four
// cycles a read more).
__device__ __forceinline__ int mt_place(int r, int c) { return c ^ (r >> 1 & 7); }

template <class S> struct MtFrags { mx4_u32x4 f[S::FT], t[S::TOKENS]; };

// The scales of a step: FOUR: of the lane's row its four blocks', a byte a slice; else the byte of its one block.
template <class S> struct MtScales { uint32_t f[S::FT], t[S::FOUR ? S::TT : 1]; };

__device__ __forceinline__ void mt_read(mx4_u32x4 &to, const mx4_u32x4 *from) {
    to = *from;
    __builtin_amdgcn_sched_barrier(0);
}

// The last slice of one step's products while the first of the next is read, and so on through that step's slices but the last, whose operands are in
// registers in the end.  nf, nt: the next step's stages; df, dt: the stages that the loads of a later step go to (parameters of one function with
// __restrict__: else the compiler lets every read from LDS wait for every load in flight).  codes: the step's codes of bfloat16 rows' features.
template <class S, class IssueT, class IssueF>
__device__ __forceinline__ void mt_turn(const mx4_u32x4 *__restrict__ nf, const mx4_u32x4 *__restrict__ nt, mx4_u32x4 *__restrict__ df, mx4_u32x4 *__restrict__ dt, IssueT &&issue_t,
                                        IssueF &&issue_f, const int (&at_f)[S::SLICES], const int (&at_t)[S::SLICES], MtFrags<S> (&op)[2], mx4_u32x4 (&codes)[S::FT],
                                        const MtScales<S> &before, const MtScales<S> &now, mx4_f32x16 (&acc)[S::FT][S::TT]) {
    auto slice = [&](auto number) {
        constexpr int s = decltype(number)::value, PRODUCTS = S::FT * S::TOKENS, used = (s + S::SLICES - 1) % S::SLICES;         // the slice that is multiplied
        MtFrags<S> &use = op[(s + 1) & 1], &get = op[s & 1];
#pragma unroll
        for (int i = 0; i < PRODUCTS; ++i) {
            const int f = i / S::TT % S::FT, t = i % S::TT, p = i / (S::FT * S::TT);
            if constexpr (S::FOUR) {
                const MtScales<S> &sc = s == 0 ? before : now;
                acc[f][t] = mx4_multiply_codes_32<used>(use.f[f], use.t[t], acc[f][t], sc.f[f], sc.t[t]);
            } else {
                acc[f][t] = mx4_multiply_32(use.f[f], use.t[p * S::TT + t], acc[f][t]);
            }
            __builtin_amdgcn_sched_barrier(0);
            {
                // the tokens' loads in the first slice where they are wanted in the next step, the features' behind them; else all spread over all slices but the last
                constexpr int FIRST = S::ST == 2 ? PRODUCTS : PRODUCTS * (S::SLICES - 1) * S::LT / (S::LT + S::LF), REST = PRODUCTS * (S::SLICES - 1) - FIRST;
                const int n = s * PRODUCTS + i;
                if (n < FIRST) {
#pragma unroll
                    for (int l = n * S::LT / FIRST; l < (n + 1) * S::LT / FIRST; ++l) { issue_t(dt, l); __builtin_amdgcn_sched_barrier(0); }
                } else if (n < FIRST + REST) {
#pragma unroll
                    for (int l = (n - FIRST) * S::LF / REST; l < (n - FIRST + 1) * S::LF / REST; ++l) { issue_f(df, l); __builtin_amdgcn_sched_barrier(0); }
                }
            }
            if constexpr (S::FOUR) {
                constexpr int READS = S::FT + S::TT;
                const int r0 = i * READS / PRODUCTS, r1 = (i + 1) * READS / PRODUCTS;
#pragma unroll
                for (int r = r0; r < r1; ++r) {
                    if (r < S::TT) mt_read(get.t[r], nt + at_t[s] + 32 * S::TP * r);
                    else mt_read(get.f[r - S::TT], nf + at_f[s] + 32 * S::FP * (r - S::TT));
                }
            } else {
                constexpr int READS = S::TOKENS + (s == 0 ? S::FT : 0);
                const int r0 = i * READS / PRODUCTS, r1 = (i + 1) * READS / PRODUCTS;
#pragma unroll
                for (int r = r0; r < r1; ++r) {
                    if (s == 0 && r < S::FT) mt_read(codes[r], nf + at_f[0] + 32 * S::FP * r);
                    else {
                        const int x = r - (s == 0 ? S::FT : 0);
                        mt_read(get.t[x], nt + at_t[s] + (x / S::TT * S::T + 32 * (x % S::TT)) * S::TP);
                    }
                }
                // the next slice's features, in the second half of this one's products
                constexpr int HALF = PRODUCTS / 2;
                if (i >= HALF) {
                    const int f0 = (i - HALF) * S::FT / (PRODUCTS - HALF), f1 = (i + 1 - HALF) * S::FT / (PRODUCTS - HALF);
#pragma unroll
                    for (int x = f0; x < f1; ++x) {
                        get.f[x] = mx4_to_bf16(codes[x][s], mx4_scale(now.f[x]));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };
    slice(std::integral_constant<int, 0>{});
    slice(std::integral_constant<int, 1>{});
    slice(std::integral_constant<int, 2>{});
    slice(std::integral_constant<int, 3>{});
}

struct MtArgs {
    const void *x, *xs;             // rows (bfloat16, or codes) and the codes' scales
    uint32_t ldx, lds, x_bytes, xs_bytes;     // bytes from row to row, and of the scales from a pair of macro-steps to the next (a row's are 8 bytes); of the whole
    const uint8_t *codes, *scales;
    uint32_t codes_bytes, scales_bytes;
    int pairs;
    void *y;
    long long ldy;
    int M, N, steps, slices;
    int wide_out;
    int each;                       // steps of a slice of K; slice i's sums go to the i-th plane of y
    long long plane;
};

template <class S, int EPI>
__global__ void __launch_bounds__(S::THREADS, 1)
mx4_tiles_kernel(MtArgs a) {
    extern __shared__ __attribute__((aligned(16))) mx4_u32x4 mt_lds[];
    constexpr int FT = S::FT, TT = S::TT;
    constexpr bool FOUR = S::FOUR, SWIGLU = EPI >= MT_EPI_SWIGLU, OUT32 = EPI == MT_EPI_F32 || EPI == MT_EPI_SWIGLU_F32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, hi = lane >> 5;
    const int wf = wave % S::WF, wt = wave / S::WF;
    // ---- which tile and slice: workgroups go to the eight dies in turn; a die takes a run of a slice's tiles, those of a few feature tiles side by side (17 tiles in 12 slices
    // by tiles alone, 3 a die and none for the last two: 41 us, so 35)
    const int t_tiles = (a.M + S::T - 1) / S::T, f_tiles = (a.N + S::F - 1) / S::F, tiles = t_tiles * f_tiles, items = tiles * a.slices;
    const int run = (items + 7) / 8, item = blockIdx.x % 8 * run + blockIdx.x / 8;
    if ((int)blockIdx.x / 8 >= run || item >= items) return;
    const int slice_k = item / tiles, of_slice = item - slice_k * tiles, ft0 = of_slice / t_tiles, tt0 = of_slice - ft0 * t_tiles, half_n = a.N / 2;
    const int first = slice_k * a.each, steps = min(a.steps - first, a.each);
    // row r of the tile's features in W (SwiGLU: in turns 32 gate rows and the up rows that meet them)
    auto feature = [&](int r) { return SWIGLU ? (r / 32 & 1) * half_n + ft0 * (S::F / 2) + r / 64 * 32 + r % 32 : ft0 * S::F + r; };
    const __amdgpu_buffer_rsrc_t wb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.codes), 0, a.codes_bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t sb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.scales), 0, a.scales_bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t xb = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(a.x), 0, a.x_bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t xsb = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(a.xs), 0, a.xs_bytes, 0x00020000);
    // ---- the loads of a stage: load i of wave w brings the 64 pieces from (i * WAVES + w) * 64 on
    uint32_t from_f[S::LF], from_t[S::LT];
#pragma unroll
    for (int i = 0; i < S::LF; ++i) {
        const int chunk = i * S::WAVES + wave;
        // a stage is [tile of 16][step's blocks][feature]
        const int tile = FOUR ? chunk / 2 : chunk * 2 + lane / 32, block = FOUR ? chunk % 2 * 4 + lane / 16 : lane / 16 & 1, row = feature(tile * 16 + lane % 16);
        from_f[i] = (uint32_t)mx4_row_codes(row, a.pairs) + block * 256;
    }
#pragma unroll
    for (int i = 0; i < S::LT; ++i) {
        const int r = (i * S::WAVES + wave) * (WAVE / S::TP) + lane / S::TP;
        from_t[i] = (uint32_t)(tt0 * S::T + r % S::T) * a.ldx + (S::P > 1 ? (uint32_t)(r / S::T) * (a.ldx / S::P) : 0u) + 16u * mt_place(r, lane % S::TP);
    }
    mx4_u32x4 *const lds_f = mt_lds, *const lds_t = mt_lds + S::SF * S::F * S::FP;
    // (a later step than there are: the last once more, which nobody reads)
    auto issue_f = [&](mx4_u32x4 *dst, int w_step, int i) {
        auto *to = (__attribute__((address_space(3))) void *)(dst + (i * S::WAVES + wave) * WAVE);
        const uint32_t from = from_f[i] + (uint32_t)w_step * S::STEP_CODES;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, to, 16, from, 0, 0, 0);
    };
    auto issue_t = [&](mx4_u32x4 *dst, int step, int i) {
        auto *to = (__attribute__((address_space(3))) void *)(dst + (i * S::WAVES + wave) * WAVE);
        const uint32_t from = from_t[i] + (uint32_t)(first + min(step, steps - 1)) * (16u * S::TP);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, to, 16, from, 0, 0, 0);
    };
    // ---- where the lane's operands stand in a stage
    int at_f[S::SLICES], at_t[S::SLICES];
#pragma unroll
    for (int s = 0; s < S::SLICES; ++s) {
        at_f[s] = l32 / 16 * (16 * S::FP) + ((FOUR ? s * 2 : 0) + hi) * 16 + l32 % 16;
        at_t[s] = l32 * S::TP + mt_place(l32, FOUR ? 2 * s + hi : 4 * hi + s);
    }
    const int of_f = wf * 32 * FT * S::FP, of_t = wt * 32 * TT * S::TP;
    uint32_t sf[FT], st[TT];
#pragma unroll
    for (int f = 0; f < FT; ++f) sf[f] = (uint32_t)mx4_row_scales(feature(wf * 32 * FT + 32 * f + l32), a.pairs) + 4 * hi;
#pragma unroll
    for (int t = 0; t < TT; ++t) st[t] = (uint32_t)(tt0 * S::T + wt * 32 * TT + 32 * t + l32) * 8u + 4u * hi;
    auto fetch_scales = [&](MtScales<S> &to, int step, int w_step) {
        if constexpr (FOUR) {
#pragma unroll
            for (int f = 0; f < FT; ++f) to.f[f] = __builtin_amdgcn_raw_buffer_load_b32(sb, sf[f] + (uint32_t)w_step * MX4_PAIR_SCALES, 0, 0);
#pragma unroll
            for (int t = 0; t < TT; ++t) to.t[t] = __builtin_amdgcn_raw_buffer_load_b32(xsb, st[t] + (uint32_t)step * a.lds, 0, 0);
        } else {
#pragma unroll
            for (int f = 0; f < FT; ++f) to.f[f] = __builtin_amdgcn_raw_buffer_load_b8(sb, sf[f] + (uint32_t)(w_step >> 2) * MX4_PAIR_SCALES + (w_step & 3), 0, 0);
        }
    };
    mx4_f32x16 acc[FT][TT];
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[f][t][i] = 0.f;
    MtFrags<S> op[2];
    mx4_u32x4 codes[FT];
    MtScales<S> before, now, next;
#pragma unroll
    for (int f = 0; f < FT; ++f) {
        op[1].f[f] = codes[f] = mx4_u32x4{0u, 0u, 0u, 0u};
        before.f[f] = 0;
    }
#pragma unroll
    for (int t = 0; t < S::TOKENS; ++t) {
        op[1].t[t] = mx4_u32x4{0u, 0u, 0u, 0u};
        before.t[FOUR ? t : 0] = 0;
    }
    // the features' ring's step (behind the last one: the first, which nobody reads)
    int wf_step = first;
    auto next_w = [&](int s) { return s + 1 == a.steps ? 0 : s + 1; };
    // what SF - 1 turns before the first would have asked for, in the turns' order
    int s_step = wf_step;
    fetch_scales(next, first, s_step);
#pragma unroll
    for (int j = 1 - S::SF; j < 0; ++j) {
        if (j + S::ST - 1 >= 0) {
#pragma unroll
            for (int i = 0; i < S::LT; ++i) { issue_t(lds_t + (j + S::ST - 1) * S::P * S::T * S::TP, j + S::ST - 1, i); __builtin_amdgcn_sched_barrier(0); }
        }
#pragma unroll
        for (int i = 0; i < S::LF; ++i) { issue_f(lds_f + (j + S::SF - 1) * S::F * S::FP, wf_step, i); __builtin_amdgcn_sched_barrier(0); }
        wf_step = next_w(wf_step);
    }
    int rf = 0, rt = 0, df = S::SF - 1, dt = S::ST - 1;
    for (int t = 0; t < steps; ++t) {
        now = next;
        s_step = next_w(s_step);
        fetch_scales(next, first + min(t + 1, steps - 1), s_step);
        mt_wait_loads<S::LEFT>();                              // this step's stages are there
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        mt_turn<S>(lds_f + rf * S::F * S::FP + of_f, lds_t + rt * S::P * S::T * S::TP + of_t, lds_f + df * S::F * S::FP, lds_t + dt * S::P * S::T * S::TP,
                   [&](mx4_u32x4 *dst, int i) { issue_t(dst, t + S::ST - 1, i); }, [&](mx4_u32x4 *dst, int i) { issue_f(dst, wf_step, i); }, at_f, at_t, op, codes, before, now, acc);
        before = now;
        wf_step = next_w(wf_step);
        rf = rf + 1 == S::SF ? 0 : rf + 1;
        rt = rt + 1 == S::ST ? 0 : rt + 1;
        df = df + 1 == S::SF ? 0 : df + 1;
        dt = dt + 1 == S::ST ? 0 : dt + 1;
    }
    // the last slice
#pragma unroll
    for (int i = 0; i < FT * S::TOKENS; ++i) {
        const int f = i / TT % FT, t = i % TT, p = i / (FT * TT);
        if constexpr (FOUR) acc[f][t] = mx4_multiply_codes_32<3>(op[1].f[f], op[1].t[t], acc[f][t], before.f[f], before.t[t]);
        else acc[f][t] = mx4_multiply_32(op[1].f[f], op[1].t[p * TT + t], acc[f][t]);
    }
    mt_wait_loads<0>();                                        // (the copies that nobody reads have landed before LDS is used otherwise)
    __syncthreads();
    // ---- out: a wave turns 32 tokens at a time through LDS of its own, and stores whole rows of its features
    constexpr int OUT_F = SWIGLU ? 16 * FT : 32 * FT, ELEM = OUT32 ? 4 : 2, PITCH = OUT_F * ELEM + 16, CH = OUT_F * ELEM / 16;
    static_assert(S::WAVES * 32 * PITCH <= S::LDS * 16, "room for the waves' rows");
    char *mine = (char *)mt_lds + wave * 32 * PITCH, *const y = (char *)a.y + (size_t)slice_k * a.plane * ELEM;
    const int out_n = SWIGLU ? half_n : a.N, f0 = (SWIGLU ? ft0 * (S::F / 2) : ft0 * S::F) + wf * OUT_F;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
        for (int f = 0; f < (SWIGLU ? FT / 2 : FT); ++f)
#pragma unroll
            for (int q = 0; q < 4; ++q) {                      // features 32 f + 8 q + 4 hi ..
                char *to = mine + l32 * PITCH + (32 * f + 8 * q + 4 * hi) * ELEM;
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = SWIGLU ? gate_up<GATE_SILU>(acc[2 * f % FT][t][4 * q + e], acc[(2 * f + 1) % FT][t][4 * q + e], 0.f, 0.f) : acc[f][t][4 * q + e];
                if constexpr (OUT32) *(mx4_f32x4 *)to = mx4_f32x4{o[0], o[1], o[2], o[3]};
                else *(uint2 *)to = make_uint2(pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3]));
            }
        const int tok0 = tt0 * S::T + wt * 32 * TT + 32 * t;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (a.wide_out) {
#pragma unroll
            for (int x = 0; x < 32 * CH / WAVE; ++x) {
                const int i = x * WAVE + lane, row = i / CH, c = i % CH, col = f0 + c * (16 / ELEM);
                const mx4_u32x4 v = *(const mx4_u32x4 *)(mine + row * PITCH + c * 16);
                if (tok0 + row < a.M && col < out_n) *(mx4_u32x4 *)(y + ((size_t)(tok0 + row) * a.ldy + col) * ELEM) = v;
            }
        } else {
            for (int i = lane; i < 32 * OUT_F; i += WAVE) {
                const int row = i / OUT_F, col = f0 + i % OUT_F;
                if (tok0 + row >= a.M || col >= out_n) continue;
                if constexpr (OUT32) ((float *)y)[(size_t)(tok0 + row) * a.ldy + col] = *(const float *)(mine + row * PITCH + i % OUT_F * 4);
                else ((uint16_t *)y)[(size_t)(tok0 + row) * a.ldy + col] = *(const uint16_t *)(mine + row * PITCH + i % OUT_F * 2);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// The planes of the slices' sums, added up, and the epilogue: four columns a thread.
template <int EPI>
__global__ void __launch_bounds__(256)
mx4_join_kernel(const float *__restrict__ planes, int slices, long long plane, int N, int M, long long ldp, void *__restrict__ y, long long ldy, int wide_out) {
    constexpr bool SWIGLU = EPI >= MT_EPI_SWIGLU, OUT32 = EPI == MT_EPI_F32 || EPI == MT_EPI_SWIGLU_F32;
    const int cols = SWIGLU ? N / 2 : N, fours = (cols + 3) / 4;
    const long long at = blockIdx.x * 256ll + threadIdx.x;
    if (at >= (long long)M * fours) return;
    const int row = (int)(at / fours), col = (int)(at - (long long)row * fours) * 4, n = min(4, cols - col);
    auto sum = [&](int c, float (&v)[4]) {
        const float *from = planes + row * ldp + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = 0.f;
        if (c % 4 == 0) {
#pragma unroll 4
            for (int s = 0; s < slices; ++s) {
                const mx4_f32x4 p = *(const mx4_f32x4 *)(from + s * plane);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += p[e];
            }
        } else {
            for (int s = 0; s < slices; ++s)
                for (int e = 0; e < n; ++e) v[e] += from[s * plane + e];
        }
    };
    float v[4];
    sum(col, v);
    if constexpr (SWIGLU) {
        float up[4];
        sum(col + cols, up);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gate_up<GATE_SILU>(v[e], up[e], 0.f, 0.f);
    }
    if constexpr (OUT32) {
        float *to = (float *)y + row * ldy + col;
        if (wide_out) *(mx4_f32x4 *)to = mx4_f32x4{v[0], v[1], v[2], v[3]};
        else
            for (int e = 0; e < n; ++e) to[e] = v[e];
    } else {
        bf16_t *to = (bf16_t *)y + row * ldy + col;
        if (wide_out) *(uint2 *)to = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
        else
            for (int e = 0; e < n; ++e) to[e] = from_f32<bf16_t>(v[e]);
    }
}

template <class S, int EPI>
static int mt_go(const MtArgs &a, int slices, hipStream_t stream) {
    const long long items = (long long)((a.M + S::T - 1) / S::T) * ((a.N + S::F - 1) / S::F) * slices;
    if (items > 0x7ffffff0) return LCU_BAD_ARGUMENT;
    constexpr int bytes = S::LDS * 16;
    static unsigned long long asked = 0;                       // a bit a device
    int device = 0;
    if (bytes > 64 * 1024 && hipGetDevice(&device) == hipSuccess && !(asked >> (device & 63) & 1)) {      // more LDS than a launch gets unasked
        const hipError_t e = hipFuncSetAttribute((const void *)mx4_tiles_kernel<S, EPI>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return (int)e;
        asked |= 1ull << (device & 63);
    }
    mx4_tiles_kernel<S, EPI><<<dim3((unsigned)((items + 7) / 8 * 8)), dim3(S::THREADS), bytes, stream>>>(a);
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

// Arguments as lcu_mx4_stream's, but that the scales of rows in 4 bits come by pairs of macro-steps (256 k): [pairs][lds bytes], 8 bytes a row; rows in 4 bits in whole pairs.  shape: by x_kind, tiles of features x tokens:
// 1: 0 128 x 128, 1 256 x 256, 2 128 x 64, 3 256 x 128, 4 256 x 32; 3: 0 128 x 64, 1 256 x 64, 2 256 x 32; 4: 0 128 x 128, 1 256 x 256, 2 128 x 64, 3 128 x 256.  slices: of K, each of which has workgroups of its own; with more than one, planes has room for slices x M x N floats (N
// rounded up to four),
// 16-byte aligned.  A load's place is 32 bits: a call takes rows and weights of less than 4 GiB each (the rows of the last tile beyond their end too).
LCU_API int lcu_mx4_tiles(const void *x, long long ldx, int x_kind, const void *xs, long long lds, const void *codes, const void *scales, int pairs, void *y, long long ldy,
                          int M, int N, int K, int epi, int shape, int slices, void *planes, hipStream_t stream) {
    if (M <= 0 || N <= 0) return LCU_OK;
    const int macros = (K + 127) / 128, cols = epi >= MT_EPI_SWIGLU ? N / 2 : N, elem = epi == MT_EPI_F32 || epi == MT_EPI_SWIGLU_F32 ? 4 : 2;
    const long long w_rows = (N + 15) / 16 * 16, row_bytes = x_kind == 4 ? ldx : ldx * 2, limit = 1ll << 32;
    if (K <= 0 || pairs < (macros + 1) / 2 || ldy < cols || epi < 0 || epi > MT_EPI_SWIGLU_F32 || (epi >= MT_EPI_SWIGLU && N % 2) || !x || !codes || !scales || !y ||
        ((uintptr_t)x | (uintptr_t)codes) % 16 || (uintptr_t)scales % 8 || row_bytes <= 0 || row_bytes % 16 || (M + 512ll) * row_bytes >= limit || (w_rows + 512) * pairs * 128 >= limit)
        return LCU_BAD_ARGUMENT;
    if (x_kind == 1 ? ldx < 128ll * macros : x_kind == 3 ? ldx % 768 || ldx < 3ll * macros * 128
        : x_kind == 4 ? !xs || lds % 8 || (uintptr_t)xs % 8 || ldx < 128ll * ((macros + 1) / 2) || lds < 8ll * M || (macros + 1) / 2 * lds + 4096 >= limit : true)
        return LCU_BAD_ARGUMENT;
    MtArgs a = {};
    a.x = x; a.xs = xs;
    a.ldx = (uint32_t)row_bytes; a.lds = (uint32_t)lds;
    a.codes = (const uint8_t *)codes; a.scales = (const uint8_t *)scales;
    a.codes_bytes = (uint32_t)(w_rows * pairs * 128); a.scales_bytes = (uint32_t)(w_rows * pairs * 8);
    a.pairs = pairs; a.y = y; a.ldy = ldy; a.M = M; a.N = N;
    // steps: 256 k in 4 bits, else 64
    const int two = (macros + 1) / 2;
    a.steps = x_kind == 4 ? two : macros * 2;
    a.x_bytes = (uint32_t)((M - 1) * row_bytes + (x_kind == 3 ? row_bytes : (long long)a.steps * 128));
    a.xs_bytes = x_kind == 4 ? (uint32_t)((two - 1) * lds + M * 8ll) : 0u;
    if (slices < 1 || slices > a.steps || (slices > 1 && (!planes || (uintptr_t)planes % 16))) return LCU_BAD_ARGUMENT;
    a.each = (a.steps + slices - 1) / slices;
    a.slices = slices = (a.steps + a.each - 1) / a.each;       // (as many as hold a step)
    const bool wide = ((uintptr_t)y | (uintptr_t)(ldy * elem) | (uintptr_t)(cols * elem)) % 16 == 0;
    a.wide_out = wide;
    if (slices > 1) {
        a.y = planes; a.ldy = (N + 3) / 4 * 4; a.plane = M * a.ldy;             // (rows of whole fours, with 13 columns or 929: else each number went alone, twice the time)
        a.wide_out = true;
    }
#define EPIS(...)                                                                    \
    do {                                                                             \
        typedef MtShape<__VA_ARGS__> S;                                               \
        if (slices > 1 || epi == MT_EPI_F32) rc = mt_go<S, MT_EPI_F32>(a, slices, stream); \
        else if (epi == MT_EPI_BF16) rc = mt_go<S, MT_EPI_BF16>(a, 1, stream);        \
        else if (epi == MT_EPI_SWIGLU) rc = mt_go<S, MT_EPI_SWIGLU>(a, 1, stream);    \
        else rc = mt_go<S, MT_EPI_SWIGLU_F32>(a, 1, stream);                          \
    } while (0)
    int rc = LCU_BAD_ARGUMENT;
    if (x_kind == 4) {
        if (shape == 0) EPIS(true, 2, 2, 2, 2, 4, 4);
        else if (shape == 1) EPIS(true, 4, 4, 2, 2, 3, 2);
        else if (shape == 2) EPIS(true, 2, 1, 2, 2, 3, 3);
        else if (shape == 3) EPIS(true, 2, 2, 2, 4, 3, 3);
    } else if (x_kind == 3) {
        if (shape == 0) EPIS(false, 2, 1, 2, 2, 4, 3, 3);
        else if (shape == 1) EPIS(false, 2, 1, 4, 2, 4, 4, 3);
        else if (shape == 2) EPIS(false, 2, 1, 4, 1, 4, 4, 3);
    } else {
        if (shape == 0) EPIS(false, 2, 2, 2, 2, 4, 4);
        else if (shape == 1) EPIS(false, 2, 4, 4, 2, 4, 3);
        else if (shape == 2) EPIS(false, 2, 1, 2, 2, 4, 4);
        else if (shape == 3) EPIS(false, 2, 4, 4, 1, 4, 3);
        else if (shape == 4) EPIS(false, 2, 1, 4, 1, 3, 3);
    }
#undef EPIS
    if (rc != LCU_OK || slices == 1) return rc;
    const long long threads = (long long)M * ((cols + 3) / 4);
    const int out_wide = ((uintptr_t)y | (uintptr_t)(ldy * elem) | (uintptr_t)(cols * elem)) % (4 * elem) == 0;
    const dim3 grid((unsigned int)((threads + 255) / 256)), block(256);
#define JOIN(EPI) mx4_join_kernel<EPI><<<grid, block, 0, stream>>>((const float *)planes, slices, a.plane, N, M, a.ldy, y, ldy, out_wide)
    if (epi == MT_EPI_BF16) JOIN(MT_EPI_BF16);
    else if (epi == MT_EPI_F32) JOIN(MT_EPI_F32);
    else if (epi == MT_EPI_SWIGLU) JOIN(MT_EPI_SWIGLU);
    else JOIN(MT_EPI_SWIGLU_F32);
#undef JOIN
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

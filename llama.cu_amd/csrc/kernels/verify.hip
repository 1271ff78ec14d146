// Verification of drafted tokens: which of a request's drafts stand, and the token after them.
//
// Request b has the rows starts[b] .. starts[b + 1] - 1 of the target's probabilities p, one more than it has drafts.  Draft i, drawn from q_i (or
// certain, where no q is given), stands if u_i q_i(d_i) < p_i(d_i), that is with the probability min(1, p / q); the first that does not ends the
// run of a drafts that do.  The token after them is drawn from max(p_a - q_a, 0) where a draft was refused (from p_a where that leaves nothing)
// and from p_a where all stand: the first v whose sum C(v) of what precedes it, itself included, is more than u C(V).  Tokens come out distributed as
// the target's are.  Probabilities that are no finite positive numbers count as zero.
//
// Only the row at which the run ends is read (two, with the draft's): first its parts' sums, a workgroup each, in 64 bits and a fixed order; then a
// workgroup a request finds the part, and reads that again to find the token; up to 8,192 tokens one workgroup a request does all.  Bound by memory: 4 or 8 bytes a token of the vocabulary:
// 61 requests of 128,259 tokens 17 us and 4.3 (3.6 TB/s in the first), 1 request 4.2 and 3.9, the launches' own.
#include "common.h"

constexpr int VF_THREADS = 512, VF_MAX_PARTS = 64, VF_MAX_DRAFTS = 1024;

__device__ __forceinline__ float vf_clean(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

// What has become of a request's drafts.
struct VfRun {
    int row, draft, count, taken;     // its first row and draft, how many drafts, how many stand
    bool bad;                         // starts that make no sense
};

__device__ __forceinline__ VfRun vf_place(int rows, const int *__restrict__ starts, int n_drafts, int most) {
    VfRun v;
    const int b = blockIdx.x;
    const long long row = starts[b], count = (long long)starts[b + 1] - row - 1;
    v.row = (int)row;
    v.count = (int)count;
    v.draft = (int)(row - b);
    v.taken = 0;
    v.bad = row < 0 || count < 0 || count > most || row + count >= rows || row - b < 0 || row - b + count > n_drafts;
    return v;
}

// Every thread of the workgroup calls it and gets the answer.
__device__ __forceinline__ VfRun vf_run(const float *__restrict__ p, size_t ldp, int rows, const int *__restrict__ starts, const int *__restrict__ drafts, int n_drafts,
                        const float *__restrict__ q, size_t ldq, const float *__restrict__ accept, int vocab, int most) {
    __shared__ int first;
    VfRun v = vf_place(rows, starts, n_drafts, most);
    if (v.bad) return v;
    if (threadIdx.x == 0) first = v.count;
    __syncthreads();
    for (int i = threadIdx.x; i < v.count; i += VF_THREADS) {
        const int d = drafts[v.draft + i];
        bool stands = false;
        if (d >= 0 && d < vocab) {
            const float pd = vf_clean(p[(size_t)(v.row + i) * ldp + d]), qd = q ? vf_clean(q[(size_t)(v.draft + i) * ldq + d]) : 1.f;
            stands = (double)accept[v.draft + i] * (double)qd < (double)pd;
        }
        if (!stands) atomicMin(&first, i);
    }
    __syncthreads();
    v.taken = first;
    return v;
}

// What is left of the target's probability of token i for the token after the run.
struct VfLeft {
    const float *p, *q;
    int without;                      // the certain draft that was refused, or -1
    __device__ __forceinline__ double operator()(int i) const {
        const double v = vf_clean(p[i]);
        if (i == without) return 0.0;
        if (!q) return v;
        const double left = v - (double)vf_clean(q[i]);
        return left > 0.0 ? left : 0.0;
    }
};
__device__ __forceinline__ VfLeft vf_left(const VfRun &v, const float *p, size_t ldp, const int *drafts, const float *q, size_t ldq) {
    const bool refused = v.taken < v.count;
    return {p + (size_t)(v.row + v.taken) * ldp, refused && q ? q + (size_t)(v.draft + v.taken) * ldq : nullptr, refused && !q ? drafts[v.draft + v.taken] : -1};
}

__device__ __forceinline__ double vf_wave_sum(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
    return v;
}

__device__ __forceinline__ double vf_wave_scan(double v, int lane) {
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) {
        const double up = __shfl_up(v, off, WAVE);
        if (lane >= off) v += up;
    }
    return v;
}

// sums: [requests][parts][2], of what is left and of the target's own.  PARTS: how many of them a workgroup has.
template <int PARTS>
__global__ void __launch_bounds__(VF_THREADS)
vf_sum_kernel(const float *__restrict__ p, size_t ldp, int rows, const int *__restrict__ starts, const int *__restrict__ drafts, int n_drafts, const float *__restrict__ q,
              size_t ldq, const float *__restrict__ accept, int vocab, int most, int parts, double *__restrict__ sums, int *__restrict__ accepted) {
    __shared__ double all[VF_THREADS / WAVE][PARTS][2];
    const VfRun run = vf_run(p, ldp, rows, starts, drafts, n_drafts, q, ldq, accept, vocab, most);
    if (blockIdx.y == 0 && threadIdx.x == 0) accepted[blockIdx.x] = run.bad ? 0 : run.taken;
    if (run.bad) return;
    const VfLeft left = vf_left(run, p, ldp, drafts, q, ldq);
    const int each = (vocab + parts - 1) / parts, part0 = blockIdx.y * PARTS;
    double mine[PARTS], own[PARTS];
    if (each <= 4 * VF_THREADS) {                      // all of a workgroup's loads on their way at once; what they bring is not wanted again, but for one part
        float pv[PARTS][4], qv[PARTS][4];
#pragma unroll
        for (int n = 0; n < PARTS; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int lo = min(vocab, (part0 + n) * each), hi = part0 + n < parts ? min(vocab, lo + each) : lo, i = lo + j * VF_THREADS + (int)threadIdx.x;
                pv[n][j] = i < hi ? __builtin_nontemporal_load(left.p + i) : 0.f;
                qv[n][j] = i < hi && left.q ? __builtin_nontemporal_load(left.q + i) : 0.f;
            }
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
            mine[n] = own[n] = 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int lo = min(vocab, (part0 + n) * each), i = lo + j * VF_THREADS + (int)threadIdx.x;
                const double v = vf_clean(pv[n][j]);
                own[n] += v;
                if (i != left.without) mine[n] += fmax(v - (double)vf_clean(qv[n][j]), 0.0);
            }
        }
    } else {
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
            const int lo = min(vocab, (part0 + n) * each), hi = part0 + n < parts ? min(vocab, lo + each) : lo;
            mine[n] = own[n] = 0.0;
#pragma unroll 4
            for (int i = lo + threadIdx.x; i < hi; i += VF_THREADS) { mine[n] += left(i); own[n] += vf_clean(left.p[i]); }
        }
    }
#pragma unroll
    for (int n = 0; n < PARTS; ++n) {
        mine[n] = vf_wave_sum(mine[n]);
        own[n] = vf_wave_sum(own[n]);
        if ((threadIdx.x & 63) == 0) { all[threadIdx.x >> 6][n][0] = mine[n]; all[threadIdx.x >> 6][n][1] = own[n]; }
    }
    __syncthreads();
    if (threadIdx.x < 2 * PARTS && part0 + (int)threadIdx.x / 2 < parts) {
        double t = 0.0;
        for (int w = 0; w < VF_THREADS / WAVE; ++w) t += all[w][threadIdx.x / 2][threadIdx.x % 2];
        sums[((size_t)blockIdx.x * parts + part0) * 2 + threadIdx.x] = t;
    }
}

// PIECE: neighbouring tokens of the part that a thread has at most, all of them on their way at once.
template <int PIECE>
__global__ void __launch_bounds__(VF_THREADS)
vf_token_kernel(const float *__restrict__ p, size_t ldp, int rows, const int *__restrict__ starts, const int *__restrict__ drafts, int n_drafts, const float *__restrict__ q,
                size_t ldq, const float *__restrict__ final_u, int vocab, int most, const double *__restrict__ sums, int parts, const int *__restrict__ accepted,
                int *__restrict__ tokens) {
    __shared__ double wave_sums[VF_THREADS / WAVE];
    __shared__ int found, last;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    VfRun run = vf_place(rows, starts, n_drafts, most);
    run.taken = accepted[b];
    int *out = tokens + (size_t)b * (most + 1);
    for (int i = threadIdx.x; i <= most; i += VF_THREADS)
        if (run.bad || i != run.taken) out[i] = !run.bad && i < run.taken ? drafts[run.draft + i] : -1;
    if (threadIdx.x == 0) { found = 0x7fffffff; last = -1; }
    if (run.bad) return;
    VfLeft left = vf_left(run, p, ldp, drafts, q, ldq);
    // the parts' sums, a lane each, and what lies before a part: every wave does the same
    static_assert(VF_MAX_PARTS <= WAVE, "a lane a part");
    const double2 mine_of = lane < parts ? ((const double2 *)sums)[(size_t)b * parts + lane] : make_double2(0.0, 0.0);
    double of_part = mine_of.x, reach = vf_wave_scan(of_part, lane), total = __shfl(reach, WAVE - 1, WAVE);
    if (!(total > 0.0)) {                              // nothing is left: the target's own
        left.q = nullptr;
        left.without = -1;
        of_part = mine_of.y;
        reach = vf_wave_scan(of_part, lane);
        total = __shfl(reach, WAVE - 1, WAVE);
    }
    const double goal = (double)final_u[b] * total;
    // the part in which the sum passes the goal, else the last that holds anything
    const unsigned long long passed = __ballot(of_part > 0.0 && reach > goal), holds = __ballot(of_part > 0.0);
    if (!holds) {
        if (threadIdx.x == 0) out[run.taken] = -1;
        return;
    }
    const int part = passed ? __ffsll(passed) - 1 : 63 - __clzll(holds);
    const double before = part > 0 ? __shfl(reach, part > 0 ? part - 1 : 0, WAVE) : 0.0;
    const int each = (vocab + parts - 1) / parts, lo = min(vocab, part * each), hi = min(vocab, lo + each);
    const int piece = (hi - lo + VF_THREADS - 1) / VF_THREADS, from = min(hi, lo + (int)threadIdx.x * piece), to = min(hi, from + piece);
    double v[PIECE], mine = 0.0;
#pragma unroll
    for (int i = 0; i < PIECE; ++i) v[i] = from + i < to ? left(from + i) : 0.0;
#pragma unroll
    for (int i = 0; i < PIECE; ++i) mine += v[i];
    const double scan = vf_wave_scan(mine, lane);
    if (lane == WAVE - 1) wave_sums[wave] = scan;
    __syncthreads();
    double at = before;
    for (int w = 0; w < wave; ++w) at += wave_sums[w];
    at += scan - mine;
    int mine_last = -1, mine_found = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PIECE; ++i) {
        at += v[i];
        if (v[i] > 0.0) {
            mine_last = from + i;
            if (at > goal) mine_found = min(mine_found, from + i);
        }
    }
    // (lanes are in the order of the tokens: a wave's first and last lane that have something have the wave's)
    const unsigned long long founds = __ballot(mine_found < vocab), lasts = __ballot(mine_last >= 0);
    if (founds && lane == __ffsll(founds) - 1) atomicMin(&found, mine_found);
    if (lasts && lane == 63 - __clzll(lasts)) atomicMax(&last, mine_last);
    __syncthreads();
    if (threadIdx.x == 0) out[run.taken] = found < vocab ? found : last;      // (the goal lies a rounding beyond the part: its last)
}

// A vocabulary of up to 512 PIECE tokens: one launch, a workgroup a request.
template <int PIECE>
__global__ void __launch_bounds__(VF_THREADS)
vf_small_kernel(const float *__restrict__ p, size_t ldp, int rows, const int *__restrict__ starts, const int *__restrict__ drafts, int n_drafts, const float *__restrict__ q,
                size_t ldq, const float *__restrict__ accept, const float *__restrict__ final_u, int vocab, int most, int *__restrict__ accepted, int *__restrict__ tokens) {
    __shared__ double wave_sums[VF_THREADS / WAVE];
    __shared__ int found, last;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const VfRun run = vf_run(p, ldp, rows, starts, drafts, n_drafts, q, ldq, accept, vocab, most);
    int *out = tokens + (size_t)b * (most + 1);
    for (int i = threadIdx.x; i <= most; i += VF_THREADS)
        if (run.bad || i != run.taken) out[i] = !run.bad && i < run.taken ? drafts[run.draft + i] : -1;
    if (threadIdx.x == 0) { accepted[b] = run.bad ? 0 : run.taken; found = 0x7fffffff; last = -1; }
    if (run.bad) return;
    VfLeft left = vf_left(run, p, ldp, drafts, q, ldq);
    const int piece = (vocab + VF_THREADS - 1) / VF_THREADS, from = min(vocab, (int)threadIdx.x * piece), to = min(vocab, from + piece);
    double v[PIECE], at = 0.0, mine = 0.0, total = 0.0;
    for (int turn = 0; turn < 2; ++turn) {             // what is left; and where that is nothing the target's own
        mine = 0.0;
#pragma unroll
        for (int i = 0; i < PIECE; ++i) v[i] = from + i < to ? left(from + i) : 0.0;
#pragma unroll
        for (int i = 0; i < PIECE; ++i) mine += v[i];
        const double scan = vf_wave_scan(mine, lane);
        __syncthreads();
        if (lane == WAVE - 1) wave_sums[wave] = scan;
        __syncthreads();
        at = scan - mine;
        total = 0.0;
        for (int w = 0; w < VF_THREADS / WAVE; ++w) {
            if (w == wave) at += total;
            total += wave_sums[w];
        }
        if (total > 0.0) break;
        left.q = nullptr;
        left.without = -1;
    }
    const double goal = (double)final_u[b] * total;
    int mine_last = -1, mine_found = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PIECE; ++i) {
        at += v[i];
        if (v[i] > 0.0) {
            mine_last = from + i;
            if (at > goal) mine_found = min(mine_found, from + i);
        }
    }
    const unsigned long long founds = __ballot(mine_found < vocab), lasts = __ballot(mine_last >= 0);
    if (founds && lane == __ffsll(founds) - 1) atomicMin(&found, mine_found);
    if (lasts && lane == 63 - __clzll(lasts)) atomicMax(&last, mine_last);
    __syncthreads();
    if (threadIdx.x == 0) out[run.taken] = found < vocab ? found : last;
}

// probs: [rows, ldp] float32, drafts, accept: [n_drafts], draft_probs: null or [n_drafts, ldq], starts: [requests + 1], final_u: [requests]; accepted: [requests],
// tokens: [requests, most + 1]; parts: workgroups a request, 1 to 64, of 8,192 tokens at most; sums: [requests][parts][2] doubles
// (one part needs none).
LCU_API int lcu_verify_drafts(const float *probs, long long ldp, int rows, const int *starts, int requests, const int *drafts, int n_drafts, const float *draft_probs,
                              long long ldq, const float *accept, const float *final_u, int vocab, int most, int parts, double *sums, int *accepted, int *tokens,
                              hipStream_t stream) {
    if (requests <= 0) return LCU_OK;
    if (rows < 0 || vocab <= 0 || most < 0 || most > VF_MAX_DRAFTS || n_drafts < 0 || parts < 1 || parts > VF_MAX_PARTS || !probs || !starts || !final_u || !accepted || (parts > 1 && !sums) ||
        !tokens || (n_drafts && (!drafts || !accept)) || (rows > 1 && ldp < vocab) || (draft_probs && n_drafts > 1 && ldq < vocab) ||
        (vocab + parts - 1) / parts > 16 * VF_THREADS)
        return LCU_BAD_ARGUMENT;
    if (parts == 1) {
#define SMALL(PIECE) vf_small_kernel<PIECE><<<dim3(requests), dim3(VF_THREADS), 0, stream>>>(probs, (size_t)ldp, rows, starts, drafts, n_drafts, draft_probs, (size_t)ldq, accept, \
                                                                                         final_u, vocab, most, accepted, tokens)
        if (vocab <= 2 * VF_THREADS) SMALL(2);
        else SMALL(16);
#undef SMALL
        LCU_LAUNCH_CHECK();
        return LCU_OK;
    }
    // few requests: a workgroup a part; many: four of them, whose loads are all on their way at once
#define SUM(PARTS) vf_sum_kernel<PARTS><<<dim3(requests, (parts + PARTS - 1) / PARTS), dim3(VF_THREADS), 0, stream>>>(probs, (size_t)ldp, rows, starts, drafts, n_drafts, draft_probs, \
                                                                                                              (size_t)ldq, accept, vocab, most, parts, sums, accepted)
    if ((long long)requests * parts <= 1024) SUM(1);
    else SUM(4);
#undef SUM
    LCU_LAUNCH_CHECK();
#define GO(PIECE) vf_token_kernel<PIECE><<<dim3(requests), dim3(VF_THREADS), 0, stream>>>(probs, (size_t)ldp, rows, starts, drafts, n_drafts, draft_probs, (size_t)ldq, final_u, vocab, \
                                                                                      most, sums, parts, accepted, tokens)
    const int each = (vocab + parts - 1) / parts;
    if (each <= 4 * VF_THREADS) GO(4);
    else GO(16);
#undef GO
    LCU_LAUNCH_CHECK();
    return LCU_OK;
}

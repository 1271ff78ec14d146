// The distribution that a row's temperature, top_p and top_k leave of its logits: the one that sampling.hip draws from.
//
// With the logits in descending order (equal ones by index), weights w_i = exp((l_i - l_0) / T) and prefix sums c, a draw takes the first
// entry with c_i >= u L, L = min(top_p c_n, c_k): entry i has the share (min(c_i, L) - min(c_{i-1}, L)) / L, so the entry at the cut
// keeps the part of its weight that lies within.  Nothing is sorted.  Rows of up to 8,192 entries: one launch, a row in a workgroup's registers.  Longer ones: five launches (four of few rows), a row cut into parts in those that read or write it:
//   max     the largest logit, where it stands, and the sum of all weights, in one pass with a running maximum;
//   count   a histogram of the distances (l_0 - l) / T, counts alone;
//   write   a bin's weights are known to within its width, so the bins in which the cut can lie are known from the counts, and which entries are kept in full.  Rows
//           without a cut are written.  Of the others what is not kept becomes zero; entries that are, or may be, are gathered;
//   cut     one workgroup a row finds the cut among the gathered entries of those bins, eight bits of their order at a time until few are left, and among these
//           by what precedes each, on sums of 64-bit fixed-point weights (w 2^44: no order of additions changes them), and writes the gathered ones' shares.
// Where more entries are kept than are gathered (a flat row) only those near the cut are, with the exact sum of what lies above, and the
// last launch
//   store   writes the whole row.
// Where even those near the cut are too many (tens of thousands of equal logits) `cut` searches the row itself.
//
// Bound by memory where there are many rows, and each launch's latency where there are few: 320 rows of 128,256 with cuts of every kind 185 us out of memory (max 55, the logits' one
// trip; count 28, out of the last cache; write 62, at a copy's rate; cut 18 to 22; store 14), 5 rows 28 (5.7, 5.9, 10.5, 7 and the gaps between them).
//
// A NaN counts as -inf, which has no share; a row of nothing else becomes zeros.  Infinities of the one sign share alike.  A temperature
// that is not positive leaves the first of the largest logits.
//
// Roundings.  A distance is a 32-bit difference times a 32-bit log2(e) / T: with the constant, the quotient, the difference and the product four times 2^-24 of it at most, by which a weight of
// distance d is off by d ln 2 times as much, and by the exponential's last place (d = 20: 3.3e-6, of a weight of 1e-6).  Four weights are added in 32 bits (a step of 2^-24 each) before sums go on in 64: that costs an addition in 64 bits instead of four.  The sums that
// the cut is searched by have weights cut off below 2^-44 of the largest, 2^-25 of it at most in a row of 2^19: fixed-point sums are the same in any order.
#include "common.h"

constexpr int TP_THREADS = 512, TP_CUT_THREADS = 1024, TP_BINS = 8192, TP_GATHER = 8192, TP_EACH = TP_GATHER / TP_CUT_THREADS, TP_MAX_PARTS = 32, TP_MAX_VOCAB = 1 << 19, TP_SMALL = 8 * TP_CUT_THREADS, TP_FEW = 32;
constexpr double TP_ONE = 17592186044416.0;          // 2^44: 2^19 weights of 1 are 2^63
constexpr float TP_NOTHING = 126.f;                  // the exponential ends at 2^-126
constexpr float TP_LOG2E = 1.44269504088896341f;

struct TpPart {                                      // of a part of a row: its largest logit and where, its smallest, its weights' sum
    double sum;
    float most, least;
    int at, pad;
};
struct TpRow {
    unsigned long long mass_above;                   // of entries kept in full that are not gathered
    unsigned int gathered;
    unsigned int before, upto;                       // how many entries lie in the bins before those in which the cut can lie, and up to the last of them
    int first_bin;                                   // of those bins
    // the cut: which key, which of the equal ones is the last that is kept, and the part that it has, the scale of what is kept whole
    unsigned int border;
    int last, store;                                 // store: the row is yet to be written
    float kept, inv;
};
struct TpEntry { unsigned int key; int at; };

// Up to 64 rows' options in the launch itself.
constexpr int TP_GIVEN = 64;
struct TpOptions { float temperature[TP_GIVEN], top_p[TP_GIVEN]; int top_k[TP_GIVEN]; };

__device__ __forceinline__ unsigned int tp_key(float x) {
    const unsigned int u = x == 0.f ? 0u : __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float tp_logit(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// What a row's options are, and what the parts have found.  Distances are those of the exponents of two: (l_0 - l) / T log2(e).
struct TpCut {
    float most, inv_t, per_bin;                      // inv_t: log2(e) / T; per_bin: bins for one unit of distance
    double sum, limit_p;                             // limit_p: top_p times the sum
    int k, at;
    bool empty, greedy, cuts;
};
// (not below 1e-38: an infinite distance times 0 would be none)
__device__ __forceinline__ float tp_inv_t(float temperature) { return fmaxf(TP_LOG2E / temperature, 1e-38f); }
// (the maximum with 0 makes 0 of what is no number: an infinite logit's distance from itself, and 0 times an infinite 1 / T)
__device__ __forceinline__ float tp_apart(float most, float l, float inv_t) { return fmaxf((most - l) * inv_t, 0.f); }
__device__ __forceinline__ float tp_distance(const TpCut &c, float l) { return tp_apart(c.most, l, c.inv_t); }
__device__ __forceinline__ float tp_weight(float distance) { return __builtin_amdgcn_exp2f(-distance); }
// w 2^44, w at most 1: the mantissa where the exponent puts it
__device__ __forceinline__ unsigned long long tp_fixed(float w) {
    const unsigned int bits = __float_as_uint(w), down = 127u - (bits >> 23);
    return down < 64u ? (unsigned long long)((bits & 0x7fffffu) | 0x800000u) << 21 >> down : 0ull;
}
__device__ __forceinline__ int tp_bin(const TpCut &c, float distance) { return min((int)(distance * c.per_bin), TP_BINS - 1); }
__device__ __forceinline__ float tp_clean(float l) { return fmaxf(l, -INFINITY); }      // (of a NaN and a number the maximum is the number)

// Every lane of a wave calls it and gets the answer: a lane a part (one after the other they are a trip to memory each, 10 us of 31 parts).
__device__ __forceinline__ TpCut tp_row(const TpPart *__restrict__ part, int parts, int vocab, float temperature, float top_p, int top_k) {
    static_assert(TP_MAX_PARTS <= 32, "half a wave");
    const int lane = threadIdx.x & 31;
    const TpPart mine = part[lane < parts ? lane : 0];
    TpCut c;
    c.most = mine.most;
    float least = mine.least;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) { c.most = fmaxf(c.most, __shfl_xor(c.most, off, WAVE)); least = fminf(least, __shfl_xor(least, off, WAVE)); }
    c.inv_t = tp_inv_t(temperature);
    c.at = mine.most == c.most ? mine.at : 0x7fffffff;
    c.sum = lane < parts && mine.most > -INFINITY ? mine.sum * (double)tp_weight(tp_distance(c, mine.most)) : 0.0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) { c.at = min(c.at, __shfl_xor(c.at, off, WAVE)); c.sum += __shfl_xor(c.sum, off, WAVE); }
    c.empty = c.most == -INFINITY;
    c.k = top_k;
    c.greedy = !(temperature > 0.f) || top_k <= 1 || !(top_p > 0.f);
    c.cuts = top_k < vocab || top_p < 1.f;
    c.limit_p = top_p < 1.f ? (double)top_p * c.sum : INFINITY;
    const float reach = fminf(tp_distance(c, least), TP_NOTHING);
    c.per_bin = reach > 0.f ? (float)(TP_BINS - 1) / reach : 0.f;
    return c;
}

// A stretch of a row, at borders of four: f(index, four logits) of every four (WIDE; else one at a time, the others -inf), loads of four such on their way
// at once: with one the row came at 3.4 TB/s.
template <bool WIDE, class F>
__device__ __forceinline__ void tp_fours(const float *__restrict__ row, int lo, int hi, F f) {
    constexpr int AT_ONCE = 4, V = WIDE ? 4 : 1;
    const int step = V * (int)blockDim.x;
    auto load = [&](int i) {
        if constexpr (WIDE) return *(const float4 *)(row + i);
        else return make_float4(row[i], -INFINITY, -INFINITY, -INFINITY);
    };
    auto give = [&](int i, const float4 &v) {
        const float l[4] = {tp_clean(v.x), tp_clean(v.y), tp_clean(v.z), tp_clean(v.w)};
        f(i, l);
    };
    int i = lo + V * (int)threadIdx.x;
    for (; i + (AT_ONCE - 1) * step < hi; i += AT_ONCE * step) {
        float4 v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) v[u] = load(i + u * step);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) give(i + u * step, v[u]);
    }
    for (; i < hi; i += step) give(i, load(i));
}
// f(index, logit) of every entry.
template <bool WIDE, class F>
__device__ __forceinline__ void tp_scan(const float *__restrict__ row, int lo, int hi, F f) {
    tp_fours<WIDE>(row, lo, hi, [&](int i, const float (&l)[4]) {
#pragma unroll
        for (int e = 0; e < (WIDE ? 4 : 1); ++e) f(i + e, l[e]);
    });
}
// The shares of every entry, share(index, logit), to `to`.
template <bool WIDE, class F>
__device__ __forceinline__ void tp_store_shares(const float *__restrict__ row, int lo, int hi, float *__restrict__ to, F share) {
    tp_fours<WIDE>(row, lo, hi, [&](int i, const float (&l)[4]) {
        if constexpr (WIDE) *(float4 *)(to + i) = make_float4(share(i, l[0]), share(i + 1, l[1]), share(i + 2, l[2]), share(i + 3, l[3]));
        else to[i] = share(i, l[0]);
    });
}
__device__ __forceinline__ void tp_stretch(int vocab, int part, int parts, int &lo, int &hi) {
    const int fours = (vocab + 3) / 4, each = (fours + parts - 1) / parts;
    lo = min(vocab, part * each * 4);
    hi = min(vocab, lo + each * 4);
}

template <bool WIDE>
__global__ void __launch_bounds__(TP_THREADS)
tp_max_kernel(const float *__restrict__ logits, size_t ld, int vocab, TpOptions given, const float *__restrict__ temperature, float *__restrict__ options,
              TpPart *__restrict__ part, TpRow *__restrict__ rows, unsigned int *__restrict__ hist) {
    const int r = blockIdx.x, parts = gridDim.y;
    if (options && blockIdx.y == 0 && threadIdx.x == 0) {            // for the launches that follow
        options[r] = given.temperature[r];
        options[gridDim.x + r] = given.top_p[r];
        ((int *)options)[2 * gridDim.x + r] = given.top_k[r];
    }
    int lo, hi;
    tp_stretch(vocab, blockIdx.y, parts, lo, hi);
    if (hist) {                                      // cleared for the next launch
        for (int b = (int)blockIdx.y * TP_THREADS + threadIdx.x; b < TP_BINS; b += TP_THREADS * parts) hist[(size_t)r * TP_BINS + b] = 0u;
        if (blockIdx.y == 0 && threadIdx.x == 0) { rows[r].mass_above = 0; rows[r].gathered = 0; }
    }
    const float inv_t = tp_inv_t(options ? given.temperature[r] : temperature[r]);
    float most = -INFINITY, least = INFINITY;
    double sum = 0.0;
    int at = 0x7fffffff;
    // four at a time: what they add is summed in 32 bits, the sum of it all in 64
    auto four = [&](int i, const float (&l)[4]) {
        const float top = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));
        if (top > most) {
            sum = most > -INFINITY ? sum * (double)tp_weight(tp_apart(top, most, inv_t)) : 0.0;
            most = top;
            at = i + (l[0] == top ? 0 : l[1] == top ? 1 : l[2] == top ? 2 : 3);
        }
        if (most > -INFINITY) {
            float add = 0.f;
#pragma unroll
            for (int e = 0; e < (WIDE ? 4 : 1); ++e) add += tp_weight(tp_apart(most, l[e], inv_t));
            sum += (double)add;
        }
#pragma unroll
        for (int e = 0; e < (WIDE ? 4 : 1); ++e) least = fminf(least, l[e]);
    };
    tp_fours<WIDE>(logits + r * ld, lo, hi, four);
    __shared__ TpPart mine[TP_THREADS / WAVE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float all = wave_max(most);
    int first = most == all ? at : 0x7fffffff;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { first = min(first, __shfl_xor(first, off, WAVE)); least = fminf(least, __shfl_xor(least, off, WAVE)); }
    sum = most > -INFINITY ? (most == all ? sum : sum * (double)tp_weight(tp_apart(all, most, inv_t))) : 0.0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, WAVE);
    if (lane == 0) mine[wave] = {sum, all, least, first, 0};
    __syncthreads();
    if (threadIdx.x == 0) {
        TpPart t = mine[0];
        for (int w = 1; w < TP_THREADS / WAVE; ++w) {
            if (mine[w].most > t.most || (mine[w].most == t.most && mine[w].at < t.at)) { t.most = mine[w].most; t.at = mine[w].at; }
            t.least = fminf(t.least, mine[w].least);
        }
        t.sum = 0.0;
        for (int w = 0; w < TP_THREADS / WAVE; ++w)
            if (mine[w].most > -INFINITY) t.sum += mine[w].most == t.most ? mine[w].sum : mine[w].sum * (double)tp_weight(tp_apart(t.most, mine[w].most, inv_t));
        part[(size_t)r * parts + blockIdx.y] = t;
    }
}

template <bool WIDE>
__global__ void __launch_bounds__(TP_THREADS)
tp_count_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, const float *__restrict__ top_p, const int *__restrict__ top_k,
                const TpPart *__restrict__ part, unsigned int *__restrict__ hist) {
    __shared__ unsigned int count[TP_BINS];
    const int r = blockIdx.x, parts = gridDim.y;
    const TpCut c = tp_row(part + (size_t)r * parts, parts, vocab, temperature[r], top_p[r], top_k[r]);
    if (c.empty || c.greedy || !c.cuts) return;
    for (int b = threadIdx.x; b < TP_BINS; b += TP_THREADS) count[b] = 0u;
    __syncthreads();
    int lo, hi;
    tp_stretch(vocab, blockIdx.y, parts, lo, hi);
    tp_scan<WIDE>(logits + r * ld, lo, hi, [&](int, float l) {
        const float d = tp_distance(c, l);
        if (d <= TP_NOTHING) atomicAdd(&count[tp_bin(c, d)], 1u);
    });
    __syncthreads();
    for (int b = threadIdx.x; b < TP_BINS; b += TP_THREADS)
        if (count[b]) atomicAdd(&hist[(size_t)r * TP_BINS + b], count[b]);
}

// The bins in which the cut can lie, lo to hi, and how many entries lie before and up to them.  Every thread of the workgroup (TP_THREADS) calls it and gets the answer; held: room for
// the counts.
struct TpBracket { int lo, hi; unsigned int before, upto; };
__device__ __forceinline__ TpBracket tp_bracket(const TpCut &c, const unsigned int *__restrict__ hist, uint4 *__restrict__ held) {
    constexpr int FOURS = TP_BINS / TP_THREADS / 4, WAVES = TP_THREADS / WAVE;
    __shared__ unsigned int wave_n[WAVES];
    __shared__ float wave_lo[WAVES], wave_hi[WAVES];
    __shared__ int over[3];                            // the first thread whose bins reach: k entries; top_p of the sum at most, and at least
    __shared__ int bin[3];
    __shared__ unsigned int before[3], upto[3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, me = (int)threadIdx.x;
#pragma unroll
    for (int i = 0; i < FOURS; ++i) held[i * TP_THREADS + threadIdx.x] = ((const uint4 *)hist)[i * TP_THREADS + threadIdx.x];
    if (threadIdx.x < 3) over[threadIdx.x] = TP_THREADS - 1;
    __syncthreads();
    // a bin's weights lie between its borders'.  A ten-thousandth either way is room for the roundings of distances and weights, and for sums in 32 bits: forty additions deep, 2^-24 each
    const float wide = c.per_bin > 0.f ? 1.0f / c.per_bin : 0.f;
    auto walk = [&](unsigned int n_at, float most_at, float least_at, auto f) {
        float most = 0.f, least = 0.f, edge = tp_weight((float)(me * FOURS * 4) * wide);
#pragma unroll 1                                       // (with all of it unrolled: 75 registers, and three workgroups a compute unit instead of four)
        for (int i = 0; i < FOURS; ++i) {
            const uint4 four = held[me * FOURS + i];
            const unsigned int n[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int b = (me * FOURS + i) * 4 + e;
                const float next = tp_weight((float)(b + 1) * wide);
                most += (float)n[e] * edge;
                least += (float)n[e] * next;
                edge = next;
                n_at += n[e];
                f(b, n[e], n_at, most_at + most * 1.0001f, least_at + least * 0.9999f);
            }
        }
    };
    unsigned int n_mine = 0, n_scan;
    float most_mine = 0.f, least_mine = 0.f;
    walk(0u, 0.f, 0.f, [&](int, unsigned int, unsigned int n, float most, float least) { n_mine = n; most_mine = most; least_mine = least; });
    n_scan = n_mine;
    float most_scan = most_mine, least_scan = least_mine;
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) {
        const unsigned int a = __shfl_up(n_scan, off, WAVE);
        const float b = __shfl_up(most_scan, off, WAVE), d = __shfl_up(least_scan, off, WAVE);
        if (lane >= off) { n_scan += a; most_scan += b; least_scan += d; }
    }
    if (lane == WAVE - 1) { wave_n[wave] = n_scan; wave_hi[wave] = most_scan; wave_lo[wave] = least_scan; }
    // (what lies before a thread is the thread before's sum: its own sum less its own part would lose what is small beside that)
    unsigned int n_at = __shfl_up(n_scan, 1, WAVE);
    float most_at = __shfl_up(most_scan, 1, WAVE), least_at = __shfl_up(least_scan, 1, WAVE);
    if (lane == 0) { n_at = 0; most_at = least_at = 0.f; }
    __syncthreads();
    for (int w = 0; w < wave; ++w) { n_at += wave_n[w]; most_at += wave_hi[w]; least_at += wave_lo[w]; }
    // (a wave's first lane that is over has the wave's first; all lanes behind it are over too, and their minima would be taken one after the other)
    auto first_of = [&](bool is_over, int *to) {
        const unsigned long long mask = __ballot(is_over);
        if (mask && lane == __ffsll(mask) - 1) atomicMin(to, me);
    };
    first_of(n_at + n_mine >= (unsigned int)c.k, &over[0]);
    first_of((double)(most_at + most_mine) >= c.limit_p, &over[1]);
    first_of((double)(least_at + least_mine) >= c.limit_p, &over[2]);
    __syncthreads();
    // that thread's bin; its last if there is none at all
    if (me == over[0] || me == over[1] || me == over[2]) {
        int at[3] = {-1, -1, -1};
        unsigned int n_before[3], n_upto[3];
        walk(n_at, most_at, least_at, [&](int b, unsigned int n, unsigned int with, float most, float least) {
            const bool is_over[3] = {with >= (unsigned int)c.k, (double)most >= c.limit_p, (double)least >= c.limit_p}, last = b % (FOURS * 4) == FOURS * 4 - 1;
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (at[i] < 0 && (is_over[i] || last)) { at[i] = b; n_before[i] = with - n; n_upto[i] = with; }
        });
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (me == over[i]) { bin[i] = at[i]; before[i] = n_before[i]; upto[i] = n_upto[i]; }
    }
    __syncthreads();
    const int lo = bin[1] < bin[0] ? 1 : 0, hi = bin[2] < bin[0] ? 2 : 0;
    return {bin[lo], bin[hi], before[lo], upto[hi]};
}

enum { TP_ALL = 0, TP_NEAR = 1, TP_SEARCH = 2 };      // what of a row is gathered: all that is kept, what is near the cut, nothing
template <class B> __device__ __forceinline__ int tp_how(const B &b) { return b.upto <= TP_GATHER ? TP_ALL : b.upto - b.before <= TP_GATHER ? TP_NEAR : TP_SEARCH; }

template <bool WIDE>
__global__ void __launch_bounds__(TP_THREADS)
tp_write_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, const float *__restrict__ top_p, const int *__restrict__ top_k,
                const TpPart *__restrict__ part, const unsigned int *__restrict__ hist, TpRow *__restrict__ rows, TpEntry *__restrict__ entries, float *__restrict__ out) {
    const int r = blockIdx.x, parts = gridDim.y;
    const TpCut c = tp_row(part + (size_t)r * parts, parts, vocab, temperature[r], top_p[r], top_k[r]);
    int lo, hi;
    tp_stretch(vocab, blockIdx.y, parts, lo, hi);
    float *to = out + (size_t)r * vocab;
    if (c.empty || c.greedy) {
        for (int i = lo + threadIdx.x; i < hi; i += TP_THREADS) to[i] = !c.empty && i == c.at ? 1.f : 0.f;
        return;
    }
    const float *row = logits + r * ld;
    if (!c.cuts) {
        const float inv = (float)(1.0 / c.sum);
        tp_store_shares<WIDE>(row, lo, hi, to, [&](int, float l) { return tp_weight(tp_distance(c, l)) * inv; });
        return;
    }
    // every workgroup of a row finds the bins by itself: a launch for them alone took 6 us of 5 rows' 34 and 12 of 320 rows' 163
    __shared__ __attribute__((aligned(16))) TpEntry mine[TP_GATHER / 2];
    static_assert(sizeof(mine) >= TP_BINS * sizeof(unsigned int), "the counts, and then the entries");
    const TpBracket b = tp_bracket(c, hist + (size_t)r * TP_BINS, (uint4 *)mine);
    if (blockIdx.y == 0 && threadIdx.x == 0) { rows[r].before = b.before; rows[r].upto = b.upto; rows[r].first_bin = b.lo; }
    const int how = tp_how(b);
    if (how == TP_SEARCH) return;
    const int from = how == TP_ALL ? 0 : b.lo;
    unsigned long long above = 0;
    // a workgroup's entries come together in LDS first: one place of them all in the row's list (an atomic addition a wave and four entries took 25 us of
    // 31 parts' 39)
    __shared__ unsigned int mine_n, place;
    if (threadIdx.x == 0) mine_n = 0;
    __syncthreads();
    auto flush = [&]() {
        __syncthreads();
        const unsigned int n = mine_n;
        if (threadIdx.x == 0 && n) place = atomicAdd(&rows[r].gathered, n);
        __syncthreads();
        for (unsigned int i = threadIdx.x; i < n; i += TP_THREADS)
            if (place + i < TP_GATHER) entries[(size_t)r * TP_GATHER + place + i] = mine[i];
        __syncthreads();
        if (threadIdx.x == 0) mine_n = 0;
        __syncthreads();
    };
    auto entry = [&](int i, float l) {
        const float d = tp_distance(c, l);
        const int bin = d <= TP_NOTHING ? tp_bin(c, d) : TP_BINS;
        if (bin >= from && bin <= b.hi) mine[atomicAdd(&mine_n, 1u)] = {tp_key(l), i};
        if (bin < from) above += tp_fixed(tp_weight(d));
    };
    // as much of the stretch at a time as fits whatever is kept of it
    for (int at = lo; at < hi; at += TP_GATHER / 2) {
        if (at > lo) flush();
        const int end = min(hi, at + TP_GATHER / 2);
        if (how == TP_ALL)
            tp_store_shares<WIDE>(row, at, end, to, [&](int i, float l) { entry(i, l); return 0.f; });
        else
            tp_scan<WIDE>(row, at, end, entry);
    }
    flush();
    if (how == TP_NEAR) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) above += __shfl_xor(above, off, WAVE);
        if ((threadIdx.x & 63) == 0 && above) atomicAdd(&rows[r].mass_above, above);
    }
}

struct TpSum { unsigned long long mass; unsigned int count; };

// What an entry of key k at index i keeps.
__device__ __forceinline__ float tp_share(const TpRow &t, unsigned int k, int i, float w) {
    if (k < t.border || (k == t.border && i > t.last)) return 0.f;
    if (k == t.border && i == t.last && t.kept >= 0.f) return t.kept;
    return w * t.inv;
}

// What the search for a cut needs of LDS.
struct TpShared {
    unsigned long long mass[256];
    unsigned int count[256], found[2];
    TpSum found_above;
    TpEntry few[TP_FEW];
    unsigned int n_few;
    TpRow cut;
};

// The cut among the entries that `each` goes through (f(key, index, weight)); above: what lies over all of them, base and span: the smallest key of them and how far the largest lies from
// it; left: how many they are, or more than that.  Every thread of the workgroup (256 or more) calls it and gets the answer.
template <class Each>
__device__ __forceinline__ TpRow tp_search(const TpCut &c, TpShared &sh, TpSum above, unsigned int base, unsigned int span, unsigned int left, Each each) {
    const int lane = threadIdx.x & 63;
    // (at least a unit, of which the first entry then has all)
    const unsigned long long limit_p = c.limit_p < 524288.0 ? max(1ull, (unsigned long long)(c.limit_p * TP_ONE)) : ~0ull;
    // the digits of the largest key at which the entries down to it reach one of the limits; `above`: what lies over the keys with the digits so far
    unsigned int border = 0;                           // (less the smallest key)
    bool all = false;                                  // (the limits lie a rounding beyond all there is)
    int open = span ? 32 - __clz(span) : 1;            // bits that are not decided yet
    while (open > 0 && left > TP_FEW) {
        const int shift = max(0, open - 8);
        const unsigned int digits = 1u << (open - shift);       // (the last ones may be fewer than 256: a key above them has been counted)
        __syncthreads();
        if (threadIdx.x < 256) { sh.mass[threadIdx.x] = 0; sh.count[threadIdx.x] = 0; }
        __syncthreads();
        each([&](unsigned int k, int, float w) {
            const unsigned int digit = ((k - base) >> shift) - (border >> shift);       // (border's undecided bits are zeros)
            if (digit < digits && k - base >= border) {
                atomicAdd(&sh.count[digit], 1u);
                atomicAdd(&sh.mass[digit], tp_fixed(w));
            }
        });
        __syncthreads();
        if (threadIdx.x < WAVE) {                      // a wave walks the digits from the largest on, four a lane
            TpSum mine = {0, 0}, digit[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 255 - (4 * lane + e);
                digit[e] = {sh.mass[d], sh.count[d]};
                mine.mass += digit[e].mass; mine.count += digit[e].count;
            }
            TpSum scan = mine;
#pragma unroll
            for (int off = 1; off < WAVE; off <<= 1) {
                const unsigned long long m = __shfl_up(scan.mass, off, WAVE);
                const unsigned int n = __shfl_up(scan.count, off, WAVE);
                if (lane >= off) { scan.mass += m; scan.count += n; }
            }
            TpSum so_far = {above.mass + scan.mass - mine.mass, above.count + scan.count - mine.count};
            int got = -1;
            TpSum got_above = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const TpSum with = {so_far.mass + digit[e].mass, so_far.count + digit[e].count};
                if (got < 0 && digit[e].count && (with.count >= (unsigned int)c.k || with.mass >= limit_p)) { got = 255 - (4 * lane + e); got_above = so_far; }
                so_far = with;
            }
            const unsigned long long reached = __ballot(got >= 0);
            if (reached == 0) {
                if (lane == WAVE - 1) { sh.found[0] = 256; sh.found_above = so_far; }
            } else if (lane == __ffsll((unsigned long long)reached) - 1) {
                sh.found[0] = (unsigned int)got;
                sh.found_above = got_above;
            }
        }
        __syncthreads();
        above = sh.found_above;
        if (sh.found[0] == 256u) { all = true; break; }
        border |= sh.found[0] << shift;
        left = sh.count[sh.found[0]];
        open = shift;
    }
    if (!all && left <= TP_FEW) {                      // a lane an entry: what precedes it, and itself, in one turn (digit by digit to the end: the launch 9.2 us of 5 rows and 24.5 of 320, so 7.0 and 21.9)
        __syncthreads();
        if (threadIdx.x == 0) sh.n_few = 0;
        __syncthreads();
        each([&](unsigned int k, int i, float) {
            if ((unsigned long long)((k - base) ^ border) >> open == 0) {
                const unsigned int place = atomicAdd(&sh.n_few, 1u);
                if (place < TP_FEW) sh.few[place] = {k, i};
            }
        });
        __syncthreads();
        if (threadIdx.x < WAVE) {
            const unsigned int n = min((unsigned int)__builtin_amdgcn_readfirstlane(sh.n_few), (unsigned int)TP_FEW);
            const TpEntry mine = lane < (int)n ? sh.few[lane] : TpEntry{0u, 0x7fffffff};
            const unsigned long long w = lane < (int)n ? tp_fixed(tp_weight(tp_distance(c, tp_logit(mine.key)))) : 0ull;
            TpSum before = above;
            for (unsigned int j = 0; j < n; ++j) {
                const unsigned int k = __builtin_amdgcn_readlane(mine.key, j);
                const int i = __builtin_amdgcn_readlane(mine.at, j);
                const unsigned long long w_j = (unsigned long long)(unsigned int)__builtin_amdgcn_readlane((int)(w >> 32), j) << 32 | (unsigned int)__builtin_amdgcn_readlane((int)w, j);
                if (k > mine.key || (k == mine.key && i < mine.at)) { before.mass += w_j; ++before.count; }
            }
            const unsigned long long with = before.mass + w;
            const bool by_k = before.count + 1 >= (unsigned int)c.k, reached = lane < (int)n && (by_k || with >= limit_p);
            const bool first = reached && before.count < (unsigned int)c.k && before.mass < limit_p;      // (and none before it)
            TpRow t = {};
            t.last = 0x7fffffff;
            t.kept = -1.f;
            if (first) {
                const unsigned long long limit = by_k ? min(limit_p, with) : limit_p, kept = limit - before.mass;
                if (kept < w) t.kept = (float)((double)kept / (double)limit);
                t.border = mine.key;
                t.last = mine.at;
                t.inv = (float)(TP_ONE / (double)limit);
                sh.cut = t;
            }
            if (__ballot(first) == 0) {                // (the limits lie a rounding beyond all there is)
                unsigned long long total = w;
#pragma unroll
                for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, WAVE);
                total += above.mass;
                t.inv = total ? (float)(TP_ONE / (double)total) : 0.f;
                if (lane == 0) sh.cut = t;
            }
        }
        __syncthreads();
        return sh.cut;
    }
    TpRow t = {};
    t.last = 0x7fffffff;
    t.kept = -1.f;                                     // (what is kept whole has its weight's own digits, not those of the sums)
    unsigned long long limit = above.mass;
    if (!all) {
        const unsigned int equal = sh.count[sh.found[0]];                        // of the last digit: all have the key
        border += base;
        const unsigned long long each_mass = tp_fixed(tp_weight(tp_distance(c, tp_logit(border))));
        limit = limit_p;
        if (above.count + equal >= (unsigned int)c.k) limit = min(limit, above.mass + ((unsigned int)c.k - above.count) * each_mass);
        unsigned int rank = each_mass ? (unsigned int)min((limit - above.mass + each_mass - 1) / each_mass, (unsigned long long)equal) : min((unsigned int)c.k - above.count, equal);
        rank = max(1u, rank);
        const unsigned long long kept = limit - above.mass - (unsigned long long)(rank - 1) * each_mass;
        if (kept < each_mass) t.kept = (float)((double)kept / (double)limit);
        t.border = border;
        // the rank-th smallest index among the equal ones (more than a few), eight bits at a time
        unsigned int index = 0;
        left = rank;
        for (int shift = 16; shift >= 0; shift -= 8) {
            __syncthreads();
            if (threadIdx.x < 256) sh.count[threadIdx.x] = 0;
            __syncthreads();
            each([&](unsigned int k, int i, float) {
                if (k == border && (shift == 16 || ((unsigned int)i ^ index) >> (shift + 8) == 0)) atomicAdd(&sh.count[(unsigned int)i >> shift & 255], 1u);
            });
            __syncthreads();
            if (threadIdx.x < WAVE) {
                unsigned int mine = 0, n[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) { n[e] = sh.count[4 * lane + e]; mine += n[e]; }
                unsigned int scan = mine;
#pragma unroll
                for (int off = 1; off < WAVE; off <<= 1) {
                    const unsigned int up = __shfl_up(scan, off, WAVE);
                    if (lane >= off) scan += up;
                }
                unsigned int so_far = scan - mine;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (so_far < left && left <= so_far + n[e]) { sh.found[0] = 4 * lane + e; sh.found[1] = so_far; }
                    so_far += n[e];
                }
            }
            __syncthreads();
            index |= sh.found[0] << shift;
            left -= sh.found[1];
        }
        t.last = (int)index;
    }
    t.inv = limit ? (float)(TP_ONE / (double)limit) : 0.f;
    return t;
}

// A workgroup's part of a row's shares.
template <bool WIDE>
__device__ __forceinline__ void tp_store_row(const float *__restrict__ row, int vocab, const TpCut &c, const TpRow &t, float *__restrict__ to) {
    int lo, hi;
    tp_stretch(vocab, blockIdx.y, gridDim.y, lo, hi);
    tp_store_shares<WIDE>(row, lo, hi, to, [&](int i, float l) {
        const float d = tp_distance(c, l);
        return d <= TP_NOTHING ? tp_share(t, tp_key(l), i, tp_weight(d)) : 0.f;
    });
}

template <bool WIDE>
__global__ void __launch_bounds__(TP_CUT_THREADS)
tp_cut_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, const float *__restrict__ top_p, const int *__restrict__ top_k,
              const TpPart *__restrict__ part, int parts, TpRow *__restrict__ rows, const TpEntry *__restrict__ entries, float *__restrict__ out) {
    // gridDim.y workgroups a row, which all find its cut: with more than one each writes its part of a row that is yet to be written
    __shared__ TpShared sh;
    __shared__ unsigned int key_lo, key_hi;
    __shared__ unsigned long long mass_before;
    const int r = blockIdx.x, lane = threadIdx.x & 63;
    const TpCut c = tp_row(part + (size_t)r * parts, parts, vocab, temperature[r], top_p[r], top_k[r]);
    if (c.empty || c.greedy || !c.cuts) {
        if (threadIdx.x == 0 && gridDim.y == 1) rows[r].store = 0;
        return;
    }
    const TpRow b = rows[r];
    const int how = tp_how(b);
    const float *row = logits + r * ld;
    float *to = out + (size_t)r * vocab;
    const unsigned int gathered = how == TP_SEARCH ? 0u : min(b.gathered, (unsigned int)TP_GATHER);
    unsigned int key[TP_EACH];
    int at[TP_EACH];
#pragma unroll
    for (int e = 0; e < TP_EACH; ++e) {
        const unsigned int i = e * TP_CUT_THREADS + threadIdx.x;
        const TpEntry t = i < gathered ? entries[(size_t)r * TP_GATHER + i] : TpEntry{0u, 0x7fffffff};
        key[e] = t.key;
        at[e] = t.at;
    }
    // What lies in the bins before those of the cut is added up, and only the others are searched (of 8,192 gathered entries all searched: their additions by digits wait for each other).  The digits are
    // those of the distance from the smallest key: the keys' own first digit is the exponent, which nearly all share.
    if (threadIdx.x == 0) { key_lo = 0xffffffffu; key_hi = 0; mass_before = 0; }
    __syncthreads();
    unsigned int lowest = 0xffffffffu, highest = 0, near = 0;         // near: a bit an entry of the thread's
    unsigned long long mass = 0;
#pragma unroll
    for (int e = 0; e < TP_EACH; ++e)
        if (e * TP_CUT_THREADS + threadIdx.x < gathered) {
            const float d = tp_distance(c, tp_logit(key[e]));
            if (tp_bin(c, d) >= b.first_bin) { near |= 1u << e; lowest = min(lowest, key[e]); highest = max(highest, key[e]); }
            else mass += tp_fixed(tp_weight(d));
        }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        lowest = min(lowest, (unsigned int)__shfl_xor(lowest, off, WAVE));
        highest = max(highest, (unsigned int)__shfl_xor(highest, off, WAVE));
        mass += __shfl_xor(mass, off, WAVE);
    }
    if (lane == 0 && highest) { atomicMin(&key_lo, lowest); atomicMax(&key_hi, highest); }
    if (lane == 0 && mass) atomicAdd(&mass_before, mass);
    __syncthreads();
    const bool any = how != TP_SEARCH && key_hi;
    const unsigned int base = any ? key_lo : 0u, span = any ? key_hi - key_lo : ~0u;
    // f(key, index, weight) of every entry that is looked at
    auto each = [&](auto f) {
        if (how == TP_SEARCH) {
            tp_scan<WIDE>(row, 0, vocab, [&](int i, float l) {
                const float d = tp_distance(c, l);
                if (d <= TP_NOTHING) f(tp_key(l), i, tp_weight(d));
            });
        } else {
#pragma unroll
            for (int e = 0; e < TP_EACH; ++e)
                if (near >> e & 1) f(key[e], at[e], tp_weight(tp_distance(c, tp_logit(key[e]))));
        }
    };
    TpRow t = tp_search(c, sh, how == TP_SEARCH ? TpSum{0, 0} : TpSum{how == TP_NEAR ? b.mass_above : mass_before, b.before}, base, span,
                        how == TP_SEARCH ? ~0u : b.upto - b.before, each);
    t.store = how != TP_ALL;
    if (how == TP_ALL) {
        if (blockIdx.y > 0) return;
#pragma unroll
        for (int e = 0; e < TP_EACH; ++e)
            if (e * TP_CUT_THREADS + threadIdx.x < gathered) to[at[e]] = tp_share(t, key[e], at[e], tp_weight(tp_distance(c, tp_logit(key[e]))));
    }
    if (gridDim.y > 1) {
        if (t.store) tp_store_row<WIDE>(row, vocab, c, t, to);
        return;
    }
    if (threadIdx.x == 0) {
        rows[r].border = t.border; rows[r].last = t.last; rows[r].store = t.store;
        rows[r].kept = t.kept; rows[r].inv = t.inv;
    }
}

template <bool WIDE>
__global__ void __launch_bounds__(TP_THREADS)
tp_store_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, const float *__restrict__ top_p, const int *__restrict__ top_k,
                const TpPart *__restrict__ part, const TpRow *__restrict__ rows, float *__restrict__ out) {
    const int r = blockIdx.x, parts = gridDim.y;
    const TpRow t = rows[r];
    if (!t.store) return;
    const TpCut c = tp_row(part + (size_t)r * parts, parts, vocab, temperature[r], top_p[r], top_k[r]);
    tp_store_row<WIDE>(logits + r * ld, vocab, c, t, out + (size_t)r * vocab);
}

// A row of up to 1,024 EACH entries as a whole, in registers: one launch for everything.
template <int EACH>
__global__ void __launch_bounds__(TP_CUT_THREADS)
tp_small_kernel(const float *__restrict__ logits, size_t ld, int vocab, TpOptions given, const float *__restrict__ temperature, const float *__restrict__ top_p,
                const int *__restrict__ top_k, float *__restrict__ out) {
    constexpr int WAVES = TP_CUT_THREADS / WAVE;
    __shared__ TpShared sh;
    __shared__ float wave_most[WAVES];
    __shared__ int wave_at[WAVES];
    __shared__ double wave_sum[WAVES];
    __shared__ unsigned int key_lo, key_hi;
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float t_r = temperature ? temperature[r] : given.temperature[r], p_r = top_p ? top_p[r] : given.top_p[r];
    const int k_r = top_k ? top_k[r] : given.top_k[r];
    const float *row = logits + r * ld;
    float *to = out + (size_t)r * vocab;
    float l[EACH], most = -INFINITY;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = e * TP_CUT_THREADS + threadIdx.x;
        l[e] = i < vocab ? tp_clean(row[i]) : -INFINITY;
        most = fmaxf(most, l[e]);
    }
    most = wave_max(most);
    if (lane == 0) wave_most[wave] = most;
    if (threadIdx.x == 0) { key_lo = 0xffffffffu; key_hi = 0; }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) most = fmaxf(most, wave_most[w]);
    TpCut c;
    c.most = most;
    c.inv_t = tp_inv_t(t_r);
    c.k = k_r;
    c.empty = most == -INFINITY;
    c.greedy = !(t_r > 0.f) || k_r <= 1 || !(p_r > 0.f);
    c.cuts = k_r < vocab || p_r < 1.f;
    int at = 0x7fffffff;
    double sum = 0.0;
    unsigned int lowest = 0xffffffffu, highest = 0;
#pragma unroll
    for (int e = EACH - 1; e >= 0; --e) {
        if (l[e] == most) at = e * TP_CUT_THREADS + threadIdx.x;
        const float d = tp_distance(c, l[e]);
        if (d <= TP_NOTHING) {
            sum += (double)tp_weight(d);
            lowest = min(lowest, tp_key(l[e]));
            highest = max(highest, tp_key(l[e]));
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        at = min(at, __shfl_xor(at, off, WAVE));
        sum += __shfl_xor(sum, off, WAVE);
        lowest = min(lowest, (unsigned int)__shfl_xor(lowest, off, WAVE));
        highest = max(highest, (unsigned int)__shfl_xor(highest, off, WAVE));
    }
    if (lane == 0) {
        wave_at[wave] = at;
        wave_sum[wave] = sum;
        atomicMin(&key_lo, lowest);
        atomicMax(&key_hi, highest);
    }
    __syncthreads();
    c.at = 0x7fffffff;
    c.sum = 0.0;
    for (int w = 0; w < WAVES; ++w) { c.at = min(c.at, wave_at[w]); c.sum += wave_sum[w]; }
    c.limit_p = p_r < 1.f ? (double)p_r * c.sum : INFINITY;
    TpRow t = {};
    t.last = 0x7fffffff;
    t.kept = -1.f;
    t.inv = (float)(1.0 / c.sum);
    if (!c.empty && !c.greedy && c.cuts)
        t = tp_search(c, sh, TpSum{0, 0}, key_lo, key_hi - key_lo, (unsigned int)vocab, [&](auto f) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const float d = tp_distance(c, l[e]);
                if (d <= TP_NOTHING && e * TP_CUT_THREADS + (int)threadIdx.x < vocab) f(tp_key(l[e]), e * TP_CUT_THREADS + (int)threadIdx.x, tp_weight(d));
            }
        });
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = e * TP_CUT_THREADS + threadIdx.x;
        const float d = tp_distance(c, l[e]);
        if (i < vocab) to[i] = c.empty ? 0.f : c.greedy ? (i == c.at ? 1.f : 0.f) : d <= TP_NOTHING ? tp_share(t, tp_key(l[e]), i, tp_weight(d)) : 0.f;
    }
}

// Bytes of scratch memory that lcu_token_probs needs, in whatever state they are (cuts: some row may have a cut).
LCU_API size_t lcu_token_probs_scratch_bytes(int rows, int vocab, int parts, int cuts) {
    if (rows <= 0 || parts <= 0 || vocab <= TP_SMALL) return 0;
    return (size_t)rows * (parts * sizeof(TpPart) + (cuts ? sizeof(TpRow) + TP_BINS * sizeof(unsigned int) + TP_GATHER * sizeof(TpEntry) : 0) + 3 * sizeof(float));
}

// logits: [rows, ld] float32; temperature, top_p, top_k: [rows], on the device, or null and `given` holds the three one after the other on the host (up to 64 rows); out: [rows,
// vocab] float32; parts: workgroups a row, 1 to 32; cuts: 0 if no row has top_k < vocab or top_p < 1; scratch: lcu_token_probs_scratch_bytes bytes, 16-byte aligned.
LCU_API int lcu_token_probs(const float *logits, long long ld, int rows, int vocab, const float *temperature, const float *top_p, const int *top_k, const float *given, float *out,
                            int parts, int cuts, void *scratch, hipStream_t stream) {
    if (rows <= 0) return LCU_OK;
    const bool small = vocab <= TP_SMALL;
    if (vocab <= 0 || vocab > TP_MAX_VOCAB || (rows > 1 && ld < vocab) || parts < 1 || parts > TP_MAX_PARTS || !logits || !out || (!small && (!scratch || (uintptr_t)scratch % 16)) ||
        (given ? rows > TP_GIVEN : !temperature || !top_p || !top_k))
        return LCU_BAD_ARGUMENT;
    TpOptions options;
    if (given) {
        temperature = top_p = nullptr;
        top_k = nullptr;
        for (int r = 0; r < rows; ++r) {
            options.temperature[r] = given[r];
            options.top_p[r] = given[rows + r];
            options.top_k[r] = ((const int *)given)[2 * rows + r];
        }
    }
    if (small) {
#define SMALL(EACH) tp_small_kernel<EACH><<<dim3(rows), dim3(TP_CUT_THREADS), 0, stream>>>(logits, (size_t)ld, vocab, options, temperature, top_p, top_k, out)
        if (vocab <= TP_CUT_THREADS) SMALL(1);
        else if (vocab <= 4 * TP_CUT_THREADS) SMALL(4);
        else SMALL(8);
#undef SMALL
        LCU_LAUNCH_CHECK();
        return LCU_OK;
    }
    char *at = (char *)scratch;
    unsigned int *hist = cuts ? (unsigned int *)at : nullptr;
    at += cuts ? (size_t)rows * TP_BINS * sizeof(unsigned int) : 0;
    TpPart *part = (TpPart *)at;             at += (size_t)rows * parts * sizeof(TpPart);
    TpRow *state = (TpRow *)at;              at += cuts ? (size_t)rows * sizeof(TpRow) : 0;
    TpEntry *entries = (TpEntry *)at;        at += cuts ? (size_t)rows * TP_GATHER * sizeof(TpEntry) : 0;
    float *copied = given ? (float *)at : nullptr;
    if (given) {
        temperature = copied;
        top_p = copied + rows;
        top_k = (const int *)copied + 2 * rows;
    }
    const bool wide = (uintptr_t)logits % 16 == 0 && ld % 4 == 0 && vocab % 4 == 0 && (uintptr_t)out % 16 == 0;
    const dim3 cut(rows, parts), block(TP_THREADS);
    const bool together = parts > 1 && (long long)rows * parts <= 256;            // a compute unit a workgroup: each finds its row's cut by itself, which saves a launch (5 rows)
#define GO(WIDE)                                                                                                                                    \
    do {                                                                                                                                            \
        tp_max_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, options, temperature, copied, part, state, hist);                  \
        LCU_LAUNCH_CHECK();                                                                                                                         \
        if (cuts) {                                                                                                                                 \
            tp_count_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, hist);                      \
            LCU_LAUNCH_CHECK();                                                                                                                     \
        }                                                                                                                                           \
        tp_write_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, hist, state, entries, out);     \
        LCU_LAUNCH_CHECK();                                                                                                                         \
        if (cuts) {                                                                                                                                 \
            tp_cut_kernel<WIDE><<<dim3(rows, together ? parts : 1), dim3(TP_CUT_THREADS), 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, parts, state, entries, out); \
            LCU_LAUNCH_CHECK();                                                                                                                     \
            if (!together) tp_store_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, state, out);               \
            LCU_LAUNCH_CHECK();                                                                                                                     \
        }                                                                                                                                           \
    } while (0)
    if (wide) GO(true);
    else GO(false);
#undef GO
    return LCU_OK;
}

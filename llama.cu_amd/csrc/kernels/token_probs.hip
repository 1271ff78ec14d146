// The distribution that a row's temperature, top_p and top_k leave of its logits: the one that sampling.hip draws from.
//
// With the logits in descending order (equal ones by index), weights w_i = exp((l_i - l_0) / T) and prefix sums c, a draw takes the first
// entry with c_i >= u L, L = min(top_p c_n, c_k): entry i has the share (min(c_i, L) - min(c_{i-1}, L)) / L, so the entry at the cut
// keeps the part of its weight that lies within.  Nothing is sorted.  Four launches, a row cut into parts in the first three:
//   max     the largest logit, where it stands, and the sum of all weights, in one pass with a running maximum;
//   count   a histogram of the distances (l_0 - l) / T, counts alone: a bin's weights are known to within its width, so the bins in which
//           the cut can lie are known from it, and which entries are kept in full;
//   write   rows without a cut are written.  Of the others what is not kept becomes zero; entries that are, or may be, are gathered;
//   cut     one workgroup a row finds the cut among the gathered entries bit by bit of their order, on sums of 64-bit fixed-point
//           weights (w 2^44: no order of additions changes them), and writes their shares.
// Where more entries are kept than are gathered (a flat row) only those near the cut are, with the exact sum of what lies above, and the
// last launch writes the whole row; where even those are too many (tens of thousands of equal logits) it searches the row itself.
//
// A NaN counts as -inf, which has no share; a row of nothing else becomes zeros.  Infinities of the one sign share alike.  A temperature
// that is not positive leaves the first of the largest logits.
#include "common.h"

constexpr int TP_THREADS = 512, TP_CUT_THREADS = 1024, TP_BINS = 8192, TP_GATHER = 8192, TP_EACH = TP_GATHER / TP_CUT_THREADS, TP_MAX_PARTS = 32, TP_MAX_VOCAB = 1 << 19;
constexpr double TP_ONE = 17592186044416.0;          // 2^44: 2^19 weights of 1 are 2^63
constexpr float TP_NOTHING = 104.f;                  // exp(-104) is no 32-bit number any more

struct TpPart {                                      // of a part of a row: its largest logit and where, its smallest but -inf, its weights' sum
    double sum;
    float most, least;
    int at, pad;
};
struct TpRow {
    unsigned long long mass_above;                   // of entries kept in full that are not gathered
    unsigned int gathered, pad;
};
struct TpEntry { unsigned int key; int at; };

__device__ __forceinline__ unsigned int tp_key(float x) {
    const unsigned int u = x == 0.f ? 0u : __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float tp_logit(unsigned int k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// What a row's options are, and what the parts have found.
struct TpCut {
    float most, inv_t, per_bin;                      // per_bin: bins for one unit of distance
    double sum, limit_p;                             // limit_p: top_p times the sum
    int k, at;
    bool empty, greedy, cuts;
};
__device__ __forceinline__ float tp_distance(const TpCut &c, float l) { return l == c.most ? 0.f : (c.most - l) * c.inv_t; }
__device__ __forceinline__ float tp_weight(float distance) { return expf(-distance); }
__device__ __forceinline__ unsigned long long tp_fixed(float w) { return (unsigned long long)((double)w * TP_ONE); }
__device__ __forceinline__ int tp_bin(const TpCut &c, float distance) { return min((int)(distance * c.per_bin), TP_BINS - 1); }
__device__ __forceinline__ float tp_clean(float l) { return l != l ? -INFINITY : l; }

__device__ __forceinline__ TpCut tp_row(const TpPart *__restrict__ part, int parts, int vocab, float temperature, float top_p, int top_k) {
    TpCut c;
    c.most = -INFINITY;
    c.at = 0x7fffffff;
    float least = INFINITY;
    for (int p = 0; p < parts; ++p) {
        if (part[p].most > c.most) { c.most = part[p].most; c.at = part[p].at; }       // (parts in order: the first of equal ones stays)
        least = fminf(least, part[p].least);
    }
    c.inv_t = 1.0f / temperature;
    c.sum = 0.0;
    for (int p = 0; p < parts; ++p)
        if (part[p].most > -INFINITY) c.sum += part[p].sum * (double)tp_weight(tp_distance(c, part[p].most));
    c.empty = c.most == -INFINITY;
    c.k = top_k;
    c.greedy = !(temperature > 0.f) || top_k <= 1 || !(top_p > 0.f);
    c.cuts = top_k < vocab || top_p < 1.f;
    c.limit_p = top_p < 1.f ? (double)top_p * c.sum : INFINITY;
    const float reach = fminf(tp_distance(c, least), TP_NOTHING);
    c.per_bin = reach > 0.f ? (float)(TP_BINS - 1) / reach : 0.f;
    return c;
}

// A stretch of a row, at borders of four: f(index, logit) of every entry.
template <bool WIDE, class F>
__device__ __forceinline__ void tp_scan(const float *__restrict__ row, int lo, int hi, F f) {
    if constexpr (WIDE) {
        for (int i = lo + 4 * (int)threadIdx.x; i < hi; i += 4 * (int)blockDim.x) {
            if (i + 4 <= hi) {
                const float4 v = *(const float4 *)(row + i);
                f(i, tp_clean(v.x)); f(i + 1, tp_clean(v.y)); f(i + 2, tp_clean(v.z)); f(i + 3, tp_clean(v.w));
            } else {
                for (int j = i; j < hi; ++j) f(j, tp_clean(row[j]));
            }
        }
    } else {
        for (int i = lo + (int)threadIdx.x; i < hi; i += (int)blockDim.x) f(i, tp_clean(row[i]));
    }
}
__device__ __forceinline__ void tp_stretch(int vocab, int part, int parts, int &lo, int &hi) {
    const int fours = (vocab + 3) / 4, each = (fours + parts - 1) / parts;
    lo = min(vocab, part * each * 4);
    hi = min(vocab, lo + each * 4);
}

template <bool WIDE>
__global__ void __launch_bounds__(TP_THREADS)
tp_max_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, TpPart *__restrict__ part, TpRow *__restrict__ rows,
              unsigned int *__restrict__ hist) {
    const int r = blockIdx.x, parts = gridDim.y;
    int lo, hi;
    tp_stretch(vocab, blockIdx.y, parts, lo, hi);
    if (hist) {                                      // cleared for the next launch
        for (int b = (int)blockIdx.y * TP_THREADS + threadIdx.x; b < TP_BINS; b += TP_THREADS * parts) hist[(size_t)r * TP_BINS + b] = 0u;
        if (blockIdx.y == 0 && threadIdx.x == 0) { rows[r].mass_above = 0; rows[r].gathered = 0; }
    }
    const float inv_t = 1.0f / temperature[r];
    float most = -INFINITY, least = INFINITY;
    double sum = 0.0;
    int at = 0x7fffffff;
    tp_scan<WIDE>(logits + r * ld, lo, hi, [&](int i, float l) {
        if (l > most) {
            sum = most > -INFINITY ? sum * (double)expf((most - l) * inv_t) : 0.0;
            most = l;
            at = i;
        }
        if (l > -INFINITY) { sum += l == most ? 1.0 : (double)expf((l - most) * inv_t); least = fminf(least, l); }
    });
    __shared__ TpPart mine[TP_THREADS / WAVE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float all = wave_max(most);
    int first = most == all ? at : 0x7fffffff;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { first = min(first, __shfl_xor(first, off, WAVE)); least = fminf(least, __shfl_xor(least, off, WAVE)); }
    sum = most > -INFINITY ? (most == all ? sum : sum * (double)expf((most - all) * inv_t)) : 0.0;
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
            if (mine[w].most > -INFINITY) t.sum += mine[w].most == t.most ? mine[w].sum : mine[w].sum * (double)expf((mine[w].most - t.most) * inv_t);
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

// The bins lo .. hi in which the cut can lie; how many entries lie in the bins before lo and up to hi.
struct TpBracket { int lo, hi; unsigned int before, upto; };

// Every thread of the workgroup calls it and gets the answer.
template <int THREADS>
__device__ TpBracket tp_bracket(const TpCut &c, const unsigned int *__restrict__ hist) {
    constexpr int EACH = TP_BINS / THREADS, WAVES = THREADS / WAVE;
    __shared__ unsigned int wave_n[WAVES];
    __shared__ double wave_lo[WAVES], wave_hi[WAVES];
    __shared__ int found_k, found_lo, found_hi;
    __shared__ unsigned int n_before, n_upto;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) { found_k = found_lo = found_hi = TP_BINS - 1; n_before = n_upto = 0; }
    // a bin's weights lie between its borders': with room for the roundings of the distances and of the weights
    const float wide = c.per_bin > 0.f ? 1.0f / c.per_bin : 0.f;
    unsigned int n[EACH], n_mine = 0;
    double least[EACH], least_mine = 0.0, most_mine = 0.0, most[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int b = (int)threadIdx.x * EACH + e;
        n[e] = hist[b];
        most[e] = n[e] ? (double)n[e] * expf(-(float)b * wide) * 1.0001 : 0.0;
        least[e] = n[e] ? (double)n[e] * expf(-(float)(b + 1) * wide) * 0.9999 : 0.0;
        n_mine += n[e]; most_mine += most[e]; least_mine += least[e];
    }
    unsigned int n_scan = n_mine;
    double most_scan = most_mine, least_scan = least_mine;
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) {
        const unsigned int a = __shfl_up(n_scan, off, WAVE);
        const double b = __shfl_up(most_scan, off, WAVE), d = __shfl_up(least_scan, off, WAVE);
        if (lane >= off) { n_scan += a; most_scan += b; least_scan += d; }
    }
    if (lane == WAVE - 1) { wave_n[wave] = n_scan; wave_hi[wave] = most_scan; wave_lo[wave] = least_scan; }
    __syncthreads();
    unsigned int n_at = n_scan - n_mine;
    double most_at = most_scan - most_mine, least_at = least_scan - least_mine;
    for (int w = 0; w < wave; ++w) { n_at += wave_n[w]; most_at += wave_hi[w]; least_at += wave_lo[w]; }
    const unsigned int n_first = n_at;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int b = (int)threadIdx.x * EACH + e;
        n_at += n[e]; most_at += most[e]; least_at += least[e];
        if (n_at >= (unsigned int)c.k) atomicMin(&found_k, b);
        if (most_at >= c.limit_p) atomicMin(&found_lo, b);
        if (least_at >= c.limit_p) atomicMin(&found_hi, b);
    }
    __syncthreads();
    TpBracket out;
    out.lo = min(found_k, found_lo);
    out.hi = min(found_k, found_hi);
    n_at = n_first;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int b = (int)threadIdx.x * EACH + e;
        if (b == out.lo) n_before = n_at;
        n_at += n[e];
        if (b == out.hi) n_upto = n_at;
    }
    __syncthreads();
    out.before = n_before;
    out.upto = n_upto;
    __syncthreads();
    return out;
}

enum { TP_ALL = 0, TP_NEAR = 1, TP_SEARCH = 2 };      // what of a row is gathered: all that is kept, what is near the cut, nothing
__device__ __forceinline__ int tp_how(const TpBracket &b) { return b.upto <= TP_GATHER ? TP_ALL : b.upto - b.before <= TP_GATHER ? TP_NEAR : TP_SEARCH; }

template <bool WIDE>
__global__ void __launch_bounds__(TP_THREADS)
tp_write_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, const float *__restrict__ top_p, const int *__restrict__ top_k,
                const TpPart *__restrict__ part, TpRow *__restrict__ rows, const unsigned int *__restrict__ hist, TpEntry *__restrict__ entries, float *__restrict__ out) {
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
        if constexpr (WIDE) {
            for (int i = lo + 4 * (int)threadIdx.x; i < hi; i += 4 * TP_THREADS) {
                const float4 v = *(const float4 *)(row + i);
                *(float4 *)(to + i) = make_float4(tp_weight(tp_distance(c, tp_clean(v.x))) * inv, tp_weight(tp_distance(c, tp_clean(v.y))) * inv,
                                                  tp_weight(tp_distance(c, tp_clean(v.z))) * inv, tp_weight(tp_distance(c, tp_clean(v.w))) * inv);
            }
        } else {
            tp_scan<WIDE>(row, lo, hi, [&](int i, float l) { to[i] = tp_weight(tp_distance(c, l)) * inv; });
        }
        return;
    }
    const TpBracket b = tp_bracket<TP_THREADS>(c, hist + (size_t)r * TP_BINS);
    const int how = tp_how(b);
    if (how == TP_SEARCH) return;
    const int from = how == TP_ALL ? 0 : b.lo;
    unsigned long long above = 0;
    tp_scan<WIDE>(row, lo, hi, [&](int i, float l) {
        const float d = tp_distance(c, l);
        const int bin = d <= TP_NOTHING ? tp_bin(c, d) : TP_BINS;
        if (how == TP_ALL) to[i] = 0.f;
        if (bin >= from && bin <= b.hi) {
            const unsigned int place = atomicAdd(&rows[r].gathered, 1u);
            if (place < TP_GATHER) entries[(size_t)r * TP_GATHER + place] = {tp_key(l), i};
        } else if (bin < from) {
            above += tp_fixed(tp_weight(d));
        }
    });
    if (how == TP_NEAR) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) above += __shfl_xor(above, off, WAVE);
        if ((threadIdx.x & 63) == 0 && above) atomicAdd(&rows[r].mass_above, above);
    }
}

struct TpSum { unsigned long long mass; unsigned int count; };

// Sums over the workgroup, for every thread.
__device__ __forceinline__ TpSum tp_total(TpSum v, TpSum *scratch) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { v.mass += __shfl_xor(v.mass, off, WAVE); v.count += __shfl_xor(v.count, off, WAVE); }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    TpSum t = {0, 0};
    for (int w = 0; w < TP_CUT_THREADS / WAVE; ++w) { t.mass += scratch[w].mass; t.count += scratch[w].count; }
    return t;
}

template <bool WIDE>
__global__ void __launch_bounds__(TP_CUT_THREADS)
tp_cut_kernel(const float *__restrict__ logits, size_t ld, int vocab, const float *__restrict__ temperature, const float *__restrict__ top_p, const int *__restrict__ top_k,
              const TpPart *__restrict__ part, int parts, const TpRow *__restrict__ rows, const unsigned int *__restrict__ hist, const TpEntry *__restrict__ entries,
              float *__restrict__ out) {
    __shared__ TpSum scratch[TP_CUT_THREADS / WAVE];
    const int r = blockIdx.x;
    const TpCut c = tp_row(part + (size_t)r * parts, parts, vocab, temperature[r], top_p[r], top_k[r]);
    if (c.empty || c.greedy || !c.cuts) return;
    const TpBracket b = tp_bracket<TP_CUT_THREADS>(c, hist + (size_t)r * TP_BINS);
    const int how = tp_how(b);
    const float *row = logits + r * ld;
    float *to = out + (size_t)r * vocab;
    const unsigned int gathered = how == TP_SEARCH ? 0u : min(rows[r].gathered, (unsigned int)TP_GATHER);
    unsigned int key[TP_EACH];
    int at[TP_EACH];
    unsigned long long fixed[TP_EACH];
#pragma unroll
    for (int e = 0; e < TP_EACH; ++e) {
        const unsigned int i = e * TP_CUT_THREADS + threadIdx.x;
        const TpEntry t = i < gathered ? entries[(size_t)r * TP_GATHER + i] : TpEntry{0u, 0x7fffffff};
        key[e] = t.key;
        at[e] = t.at;
        fixed[e] = i < gathered ? tp_fixed(tp_weight(tp_distance(c, tp_logit(t.key)))) : 0;
    }
    // entries whose place in the order (key, then the lower index) satisfies `in`: their weights and number
    auto sum_of = [&](auto in) {
        TpSum t = {0, 0};
        if (how == TP_SEARCH) {
            tp_scan<WIDE>(row, 0, vocab, [&](int i, float l) {
                const float d = tp_distance(c, l);
                if (d <= TP_NOTHING && in(tp_key(l), i)) { t.mass += tp_fixed(tp_weight(d)); ++t.count; }
            });
        } else {
#pragma unroll
            for (int e = 0; e < TP_EACH; ++e)
                if (e * TP_CUT_THREADS + threadIdx.x < gathered && in(key[e], at[e])) { t.mass += fixed[e]; ++t.count; }
        }
        t = tp_total(t, scratch);
        if (how == TP_NEAR) { t.mass += rows[r].mass_above; t.count += b.before; }
        return t;
    };
    const unsigned long long limit_p = c.limit_p < 524288.0 ? (unsigned long long)(c.limit_p * TP_ONE) : ~0ull;
    auto reached = [&](const TpSum &t) { return t.count >= (unsigned int)c.k || t.mass >= limit_p; };
    // the largest key at which the entries down to it reach one of the limits
    unsigned int border = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned int t = border | 1u << bit;
        if (reached(sum_of([&](unsigned int k, int) { return k >= t; }))) border = t;
    }
    const TpSum above = sum_of([&](unsigned int k, int) { return k > border; }), with = sum_of([&](unsigned int k, int) { return k >= border; });
    const bool all = !reached(with);                   // (the limit lies a rounding beyond all there is)
    const unsigned long long each = with.count > above.count ? (with.mass - above.mass) / (with.count - above.count) : 0;
    unsigned long long limit = with.mass;
    int last = 0x7fffffff;                             // the index of the last of the equal entries that keeps anything
    unsigned long long kept = each;                    // and what it keeps
    if (!all) {
        limit = limit_p;
        if (with.count >= (unsigned int)c.k) limit = min(limit, above.mass + ((unsigned int)c.k - above.count) * each);
        unsigned int rank = each ? (unsigned int)((limit - above.mass + each - 1) / each) : (unsigned int)c.k - above.count;
        rank = max(1u, min(rank, with.count - above.count));
        kept = limit - above.mass - (unsigned long long)(rank - 1) * each;
        if (with.count - above.count > 1) {
            // the rank-th smallest index among them
            unsigned int index = 0;
            for (int bit = 30; bit >= 0; --bit) {
                const unsigned int t = index | 1u << bit;
                if (t >= (unsigned int)vocab) continue;
                TpSum below = sum_of([&](unsigned int k, int i) { return k == border && (unsigned int)i < t; });
                if (how == TP_NEAR) below.count -= b.before;
                if (below.count < rank) index = t;
            }
            last = (int)index;
        } else {
            last = -1;                                  // (a single one: its own index)
        }
    }
    const double inv = limit ? TP_ONE / (double)limit : 0.0;
    const bool part_of_it = kept < each;               // (what is kept whole has its weight's own digits, not those of the sums)
    auto share = [&](unsigned int k, int i, float w) {
        if (!all && (k < border || (k == border && last >= 0 && i > last))) return 0.f;
        if (!all && part_of_it && k == border && (last < 0 || i == last)) return (float)((double)kept / (double)limit);
        return (float)((double)w * inv);
    };
    if (how == TP_ALL) {
#pragma unroll
        for (int e = 0; e < TP_EACH; ++e)
            if (e * TP_CUT_THREADS + threadIdx.x < gathered) to[at[e]] = share(key[e], at[e], tp_weight(tp_distance(c, tp_logit(key[e]))));
    } else {
        tp_scan<WIDE>(row, 0, vocab, [&](int i, float l) {
            const float d = tp_distance(c, l);
            to[i] = d <= TP_NOTHING ? share(tp_key(l), i, tp_weight(d)) : 0.f;
        });
    }
}

// Bytes of scratch memory that lcu_token_probs needs, in whatever state they are (cuts: some row may have a cut).
LCU_API size_t lcu_token_probs_scratch_bytes(int rows, int parts, int cuts) {
    if (rows <= 0 || parts <= 0) return 0;
    return (size_t)rows * (parts * sizeof(TpPart) + (cuts ? sizeof(TpRow) + TP_BINS * sizeof(unsigned int) + TP_GATHER * sizeof(TpEntry) : 0));
}

// logits: [rows, ld] float32; temperature, top_p, top_k: [rows], on the device; out: [rows, vocab] float32; parts: workgroups a row, 1 to 32; cuts: 0 if no row has
// top_k < vocab or top_p < 1; scratch: lcu_token_probs_scratch_bytes(rows, parts, cuts) bytes, 8-byte aligned.
LCU_API int lcu_token_probs(const float *logits, long long ld, int rows, int vocab, const float *temperature, const float *top_p, const int *top_k, float *out, int parts,
                            int cuts, void *scratch, hipStream_t stream) {
    if (rows <= 0) return LCU_OK;
    if (vocab <= 0 || vocab > TP_MAX_VOCAB || (rows > 1 && ld < vocab) || parts < 1 || parts > TP_MAX_PARTS || !logits || !temperature || !top_p || !top_k || !out || !scratch ||
        (uintptr_t)scratch % 8)
        return LCU_BAD_ARGUMENT;
    char *at = (char *)scratch;
    TpPart *part = (TpPart *)at;             at += (size_t)rows * parts * sizeof(TpPart);
    TpRow *state = (TpRow *)at;              at += cuts ? (size_t)rows * sizeof(TpRow) : 0;
    TpEntry *entries = (TpEntry *)at;        at += cuts ? (size_t)rows * TP_GATHER * sizeof(TpEntry) : 0;
    unsigned int *hist = cuts ? (unsigned int *)at : nullptr;
    const bool wide = (uintptr_t)logits % 16 == 0 && ld % 4 == 0 && vocab % 4 == 0 && (uintptr_t)out % 16 == 0;
    const dim3 cut(rows, parts), block(TP_THREADS);
#define GO(WIDE)                                                                                                                                    \
    do {                                                                                                                                            \
        tp_max_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, part, state, hist);                                   \
        LCU_LAUNCH_CHECK();                                                                                                                         \
        if (cuts) {                                                                                                                                 \
            tp_count_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, hist);                      \
            LCU_LAUNCH_CHECK();                                                                                                                     \
        }                                                                                                                                           \
        tp_write_kernel<WIDE><<<cut, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, state, hist, entries, out);     \
        LCU_LAUNCH_CHECK();                                                                                                                         \
        if (cuts) {                                                                                                                                 \
            tp_cut_kernel<WIDE><<<dim3(rows), dim3(TP_CUT_THREADS), 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_p, top_k, part, parts, state, hist, entries, out); \
            LCU_LAUNCH_CHECK();                                                                                                                     \
        }                                                                                                                                           \
    } while (0)
    if (wide) GO(true);
    else GO(false);
#undef GO
    return LCU_OK;
}

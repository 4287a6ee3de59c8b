// One token a row from logits of any vocabulary, after temperature, top-k, top-p and min-p, from a given uniform number.
//
// Definition.  w_i = exp((x_i - max x) / T); the row in the order (x descending, index ascending).  top-k keeps the first k; top-p,
// of those, every entry before which the kept weights sum to at most p of theirs; min-p those with w_i >= min_p.  Each keeps a
// PREFIX of the order, so the kept set is one prefix, described by its last entry.  The draw is the first index (in index order)
// at which the sum of the kept weights exceeds u times their total.
//
// What makes the answer a whole number that every order of summation agrees on: weights are 64-bit integers, w = round(2^44 exp(..)),
// from an exponential in double precision (2^18 of them sum to 2^62), so partial sums are exact whoever adds them, and a comparison
// with a border has the error of the weights alone, 0.6 units: a rounding to nearest, and less than a tenth from the exponential (two of which
// are multiplied for a half in the table below).  In single precision the sums of a row of 10^5 likely
// tokens are off by some 10^-7 of the total, and one draw in a thousand would differ from the definition's.
//
// One workgroup a row, one launch: the largest logit; a histogram of 2048 bins over the 32 nats that weigh anything, in counts and
// weights; the bin in which k or p is crossed, and among its few entries the last kept one; the kept weights by tiles of consecutive
// indices; the tile that u falls into.  A row of 128000 16-bit logits is 256 KB, which its die's L2 keeps for the passes after the
// first: memory's part of 256 such rows (65 MB) is 14 us.  Measured (256 x 128000 bf16, normal logits of deviation 2.5): no filter 40 us,
// top-k 50 56, top-p 0.9 85, both 85, min-p 0.05 34; temperature 0 20; two thirds of the entries equal, top-p 131, and temperature 0
// 257 if they are the largest (their indices meet at one address).  What bounds it is the exponential in double precision of every
// entry that is weighed (for 16-bit logits taken from a table in LDS instead: 120 -> 98 us with top-p when it came in) and the LDS atomics of the histogram.
#include "paged.h"

namespace {

constexpr int NB = 2048, CAP = 1024;                  // histogram bins; entries of the exact selection
constexpr double W1 = 17592186044416.0;               // 2^44: the weight of the largest logit
constexpr double RANGE = 32.0;                        // exp(-31.98) 2^44 < 0.5: entries further from the largest weigh nothing
constexpr int MAX_BINS = 1 << 18;

typedef unsigned long long u64;

// 2^(j / 32): correctly rounded, from 50 decimal digits
__constant__ double EXP2_32[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// (ln 2 / 32)^k / k!
constexpr double LN2_32 = 0.69314718055994530942 / 32.0;
constexpr double L1 = LN2_32, L2 = LN2_32 * LN2_32 / 2.0, L3 = LN2_32 * LN2_32 * LN2_32 / 6.0, L4 = LN2_32 * LN2_32 * LN2_32 * LN2_32 / 24.0,
                 L5 = LN2_32 * LN2_32 * LN2_32 * LN2_32 * LN2_32 / 120.0;

template <typename T> struct Row;                     // 16 bytes of logits at a time
template <> struct Row<float> { static constexpr int E = 4; static __device__ __forceinline__ float get(u32x4 v, int e) { return __uint_as_float(v[e]); } };
template <> struct Row<f16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(u32x4 v, int e) { return (float)__builtin_bit_cast(f16x8, v)[e]; }
};
template <> struct Row<bf16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(u32x4 v, int e) { return __uint_as_float((e & 1) ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16); }
};
// E logits from index i on; -inf behind the row's end.  A NaN may come out: fmaxf and the bins pass it over.
template <typename T> __device__ __forceinline__ u32x4 load_row(const T* row, int i, int n) {
    constexpr int E = Row<T>::E;
    if (i + E <= n) return *reinterpret_cast<const u32x4_any*>(row + i);
    u32x4 v;
    if constexpr (E == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < n ? __float_as_uint(row[i + e]) : 0xff800000u;
    } else {
        const unsigned none = sizeof(T) == 2 && __is_same(T, f16) ? 0xfc00u : 0xff80u;
        const unsigned short* bits = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
        for (int h = 0; h < 4; ++h)
            v[h] = (i + 2 * h < n ? bits[i + 2 * h] : none) | (i + 2 * h + 1 < n ? bits[i + 2 * h + 1] : none) << 16;
    }
    return v;
}
// f(16 bytes, index of the first) for the whole row, every thread its part: U requests in flight while U others are worked on
template <typename T, int NT, typename F> __device__ __forceinline__ void each_load(const T* row, int n, F f) {
    constexpr int E = Row<T>::E, STEP = NT * E, U = 16 / E;
    u32x4 next[U];
    auto ask = [&](int i) {
#pragma unroll
        for (int q = 0; q < U; ++q)
            if (i + q * STEP < n) next[q] = load_row(row, i + q * STEP, n);
    };
    ask(threadIdx.x * E);
    for (int i = threadIdx.x * E; i < n; i += U * STEP) {
        u32x4 v[U];
#pragma unroll
        for (int q = 0; q < U; ++q) v[q] = next[q];
        ask(i + U * STEP);
#pragma unroll
        for (int q = 0; q < U; ++q)
            if (i + q * STEP < n) f(v[q], i + q * STEP);
    }
}
// f(logit, index)
template <typename T, int NT, typename F> __device__ __forceinline__ void each(const T* row, int n, F f) {
    each_load<T, NT>(row, n, [&](u32x4 v, int i) {
#pragma unroll
        for (int e = 0; e < Row<T>::E; ++e) f(Row<T>::get(v, e), i + e);
    });
}

// order-preserving integers of floats
__device__ __forceinline__ unsigned key_of(float x) { const unsigned b = __float_as_uint(x); return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u); }
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

template <typename T, bool TABLE> struct Weigh {
    float mx, bins;                                   // largest logit, bins per unit of logit: both of logits times
    float by;                                         // a power of two, in whose scale neither differences nor bins leave a float's range
    double c, md;                                     // 32 / (T ln 2); the largest logit
    const double* tab;                                // EXP2_32 in LDS: 32 entries, one pair of banks each
    const double* keys;                               // a table of the weights themselves (see real), or NULL
    // how far below the largest, in bins; NB - 1: weighs nothing
    __device__ __forceinline__ float depth(float x) const { return x == mx ? 0.f : fminf(fmaf(x, -by, mx * by) * bins, (float)(NB - 1)); }
    __device__ __forceinline__ int bin(float x) const { return (int)depth(x); }
    // The largest x that lies in bin b or below it (depth falls with x, also as it is rounded), so that telling an entry's bin takes
    // comparisons alone.  The whole wave: its lanes divide the interval by 64 at a time.
    __device__ __forceinline__ float below(int b) const {
        if (b == 0) return INFINITY;
        unsigned lo = key_of(-INFINITY), hi = key_of(mx);          // depth(lo) >= b > depth(hi)
        while (hi - lo > 1) {
            const unsigned step = (hi - lo + 63) / 64, m = min(lo + step * ((threadIdx.x & 63) + 1), hi);
            const int n = __popcll(__ballot(m < hi && depth(of_key(m)) >= (float)b));      // the first n lanes
            lo += step * n;
            hi = min(lo + step, hi);
        }
        return of_key(lo);
    }
    // 2^44 exp((x - max) / T) in double: z = n + f in 32nds of an octave; 2^(f / 32) by the Taylor series of the exponential to the
    // fifth power (f <= 1/2: the next term is 2.2e-15 of the weight, 0.04 of the whole numbers' unit; the term before it, 1.2e-12, would be
    // 22 of them), 2^(n / 32) from the table and the exponent field.  n by adding and taking away 1.5 2^52, in whose low word it stands
    // meanwhile.
    __device__ __forceinline__ double power(double z) const {
        const double t = z + 6755399441055744.0, f = z - (t - 6755399441055744.0);
        double p = fma(f, L5, L4);
        p = fma(p, f, L3);
        p = fma(p, f, L2);
        p = fma(p, f, L1);
        p = fma(p, f, 1.0);
        const int n = (int)__double_as_longlong(t);
        const double w = p * tab[n & 31];
        return __hiloint2double(__double2hiint(w) + ((n >> 5) + 44) * 0x100000, __double2loint(w));
    }
    __device__ __forceinline__ double direct(float x) const { return power(x == mx ? 0.0 : ((double)x - md) * c); }
    // Logits of 16 bits are few: those of 2^-10 .. 2^7 in magnitude, by their first 7 fraction bits, have a table in LDS (17 octaves of two
    // signs), and the three further bits of a half another, by which the first is multiplied.  A logit has one weight, here as there.
    static constexpr int OCTAVES = 17, FIRST = 127 - 10, KEYS = OCTAVES * 128, REST = OCTAVES * 8;
    __device__ __forceinline__ double real(float x) const {
        if constexpr (TABLE) {
            const unsigned b = __float_as_uint(x), m = b & 0x7fffffffu, i = (m >> 16) - (FIRST << 7);
            if (keys && i < (unsigned)KEYS) {
                double w = keys[i + (b >> 31) * KEYS];
                if constexpr (__is_same(T, f16)) {
                    w *= keys[2 * KEYS + (m >> 13 & 7u) + (i >> 7) * 8 + (b >> 31) * REST];
                    w = x == mx ? W1 : w;
                }
                return w;
            }
        }
        return direct(x);
    }
    // (entries that no logit of this row has may lie far above or below its largest: their powers are cut off, not their products)
    template <int NT> __device__ __forceinline__ void fill(double* table) {
        auto far = [&](double z) { return power(fmin(fmax(z, -30000.0), 30000.0)); };
        for (int i = threadIdx.x; i < 2 * KEYS; i += NT) {
            const float x = __uint_as_float(((unsigned)(i % KEYS) + (FIRST << 7)) << 16 | (i >= KEYS ? 0x80000000u : 0u));
            table[i] = x == mx ? W1 : far(((double)x - md) * c);
        }
        if constexpr (__is_same(T, f16))
            for (int i = threadIdx.x; i < 2 * REST; i += NT) {
                const int k = i % REST;
                const double d = (double)(k & 7) * __uint_as_float((unsigned)((k >> 3) + FIRST - 10) << 23);
                table[2 * KEYS + i] = far((i >= REST ? -d : d) * c) * (1.0 / W1);
            }
        keys = table;
    }
    // a whole number in the low bits of the sum with 2^52: rounded to nearest
    static __device__ __forceinline__ u64 whole(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; }
    __device__ __forceinline__ u64 whole(float x) const { return whole(real(x)); }
};
// order (x descending, index ascending) as one ascending integer; -0 counts as 0
__device__ __forceinline__ u64 place(float x, int i) {
    return ((u64)~key_of(x + 0.0f) << 32) | (unsigned)i;
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {     // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}
struct Shared {
    u64 mass[NB];
    unsigned count[NB];
    u64 at[CAP];                                      // the border bin's entries: their places ...
    u64 w[CAP];                                       // ... and weights
    u64 tile[MAX_BINS / 1024];                        // kept weight of 256 E consecutive entries
    double tab[32];
    unsigned lo_key, hi_key;                          // of the border bin's logits
    u64 part[16];
    u64 border;                                       // place of the last kept entry
    u64 before_w, before_n;                           // in front of the bin that a search has found
    unsigned n;                                       // entries listed
    int pick;
};
// inclusive prefix sum over the block; *total: all
template <int NT> __device__ __forceinline__ u64 block_scan(u64 v, Shared& s, u64* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 x = wave_scan(v);
    if (lane == 63) s.part[wave] = x;
    __syncthreads();
    u64 base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { const u64 p = s.part[w]; base += w < wave ? p : 0; all += p; }
    __syncthreads();
    *total = all;
    return base + x;
}

struct Args {
    const void* logits; int64_t ld; int bins;
    const float *u, *temp; const int* top_k; const float *top_p, *min_p;      // per row; NULL: the value below for all
    float temp_all; int top_k_all; float top_p_all, min_p_all;
    int64_t* out;
};

template <int NT> __device__ __forceinline__ void clear_bins(Shared& s) {
    for (int i = threadIdx.x; i < NB; i += NT) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
}
// f(logit) is true for the entries that count: add(bin, weight) for each.  Where a whole wave's 16 bytes hold one value (a mask's, over
// half the vocabulary), whose additions would queue up at one address, it enters once, for all of them.
template <typename T, int NT, typename F> __device__ __forceinline__ void each_run(const T* row, int n, F f) {
    constexpr int E = Row<T>::E;
    each_load<T, NT>(row, n, [&](u32x4 v, int) {
        const unsigned one = __builtin_amdgcn_readfirstlane(v[0]);
        const bool same = v[0] == one && v[1] == one && v[2] == one && v[3] == one && (E == 4 || (one >> 16) == (one & 0xffffu));
        const u64 all = __ballot(1);
        if (__ballot(same) == all) {
            if ((all & ((1ull << (threadIdx.x & 63)) - 1)) == 0) f(Row<T>::get(v, 0), (unsigned)__popcll(all) * E);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) f(Row<T>::get(v, e), 1u);
        }
    });
}
// The first bin at which the running count (COUNT) or weight exceeds `limit`; NB if none does.  s.before_*: the sums in front of it.
template <int NT, bool COUNT> __device__ int crossing(u64 limit, Shared& s, bool weights_too = false) {
    constexpr int PER = NB / NT;
    if (threadIdx.x == 0) s.pick = NB;
    __syncthreads();
    u64 c = 0, w = 0, total;
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        if (COUNT) c += s.count[PER * threadIdx.x + b];
        if (!COUNT || weights_too) w += s.mass[PER * threadIdx.x + b];
    }
    u64 ic = COUNT ? block_scan<NT>(c, s, &total) - c : 0, iw = !COUNT || weights_too ? block_scan<NT>(w, s, &total) - w : 0;
    if ((COUNT ? ic : iw) <= limit && (COUNT ? ic + c : iw + w) > limit) {
        for (int b = PER * threadIdx.x; ; ++b) {
            const u64 nc = ic + (COUNT ? s.count[b] : 0), nw = iw + (!COUNT || weights_too ? s.mass[b] : 0);
            if ((COUNT ? nc : nw) > limit) { s.pick = b; s.before_n = ic; s.before_w = iw; break; }
            ic = nc; iw = nw;
        }
    }
    __syncthreads();
    return s.pick;
}

// The last kept entry of a bin -- COUNT: the `limit`-th after its first; else the last one that no more than `limit` of weight is
// before -- and the bin's weight up to and with it.
struct Found { u64 border, mass; };

// The same among the entries of one value, by their index: entry number limit (COUNT) or limit / weight.  False: the logits in
// (lo, hi] are not all of that value.  Rare (more equal logits than a list holds), hence a call.
template <typename T, int NT, bool COUNT, typename G>
__device__ __attribute__((noinline)) bool search_index(const T* row, int n, const G g, float one, float lo, float hi, u64 limit, Shared& s, Found* f) {
    constexpr int E = Row<T>::E;
    const int lane = threadIdx.x & 63;
    __syncthreads();
    clear_bins<NT>(s);
    bool other = false;
    each_load<T, NT>(row, n, [&](u32x4 v, int i) {
        // a wave's loads are 64 E consecutive entries from a multiple of as many on: of one 512
        unsigned times = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float x = Row<T>::get(v, e);
            times += __popcll(__ballot(x == one));
            other |= x > lo && x <= hi && x != one;
        }
        if (lane == 0 && times) atomicAdd(&s.count[i >> 9], times);
    });
    if (other) s.lo_key = 0;
    __syncthreads();
    if (s.lo_key == 0) return false;
    u64 total, mine = 0;
    for (int b = threadIdx.x; b < NB; b += NT) mine += s.count[b];
    block_scan<NT>(mine, s, &total);
    const u64 w = g.whole(one), nth = min(COUNT ? limit : w ? limit / w : ~0ull, total - 1);
    const int b = crossing<NT, true>(nth, s);
    if (threadIdx.x < 64) {
        unsigned left = (unsigned)(nth - s.before_n);
        for (int c = 0; c < 8; ++c) {
            const int i = b * 512 + c * 64 + lane;
            const bool eq = i < n && (float)row[i] == one;
            const u64 who = __ballot(eq);
            if (eq && __popcll(who & ((1ull << lane) - 1)) == left) s.border = place(one, i);
            const unsigned here = __popcll(who);
            if (left < here) break;
            left -= here;
        }
    }
    __syncthreads();
    f->border = s.border;
    f->mass = (nth + 1) * w;
    return true;
}
// More entries than the list holds: of one value, as a rule.  Of different ones the border's by its digits, 11, 11 and 10 bits of the
// places, then its index.
template <typename T, int NT, bool COUNT, typename G>
__device__ __attribute__((noinline)) Found search_many(const T* row, int n, const G g, float lo, float hi, u64 limit, bool with_mass, Shared& s) {
    Found f;
    for (int i = threadIdx.x * Row<T>::E; i < n && *(volatile unsigned*)&s.hi_key == 0; i += NT * Row<T>::E) {
        const u32x4 v = load_row(row, i, n);
#pragma unroll
        for (int e = 0; e < Row<T>::E; ++e) {
            const float x = Row<T>::get(v, e);
            if (x > lo && x <= hi) s.hi_key = key_of(x + 0.0f);
        }
    }
    __syncthreads();
    if (search_index<T, NT, COUNT>(row, n, g, of_key(s.hi_key), lo, hi, limit, s, &f)) return f;
    u64 prefix = 0, before = 0;
    for (int d = 0; d < 3; ++d) {
        __syncthreads();
        clear_bins<NT>(s);
        const int bits = d < 2 ? 11 : 10, sh = 64 - 11 * d - bits, top = sh + bits;
        each_run<T, NT>(row, n, [&](float x, unsigned times) {
            if (x > lo && x <= hi) {
                const u64 p = place(x, 0);
                if (d == 0 || (p ^ prefix) >> (top & 63) == 0) {
                    const int b = (int)(p >> sh) & ((1 << bits) - 1);
                    if (COUNT) atomicAdd(&s.count[b], times);
                    if (with_mass || !COUNT) atomicAdd(&s.mass[b], g.whole(x) * times);
                }
            }
        });
        __syncthreads();
        const int b = crossing<NT, COUNT>(limit, s, with_mass);
        // (none: everything of this prefix is kept -- its largest place stands for it)
        if (b == NB) { __syncthreads(); return Found{prefix | (d == 0 ? ~0ull : (1ull << top) - 1), before}; }
        prefix |= (u64)b << sh;
        limit -= COUNT ? s.before_n : s.before_w;
        before += s.before_w;
    }
    const float one = of_key(~(unsigned)(prefix >> 32));
    if (threadIdx.x == 0) s.lo_key = ~0u;
    search_index<T, NT, COUNT>(row, n, g, one, INFINITY, INFINITY, limit, s, &f);
    f.mass += before;
    return f;
}
template <typename T, int NT, bool COUNT, typename G>
__device__ __forceinline__ Found select(const T* row, int n, const G& g, int which, u64 limit, bool with_mass, Shared& s) {
    if (threadIdx.x == 0) { s.n = 0; s.border = 0; s.lo_key = ~0u; s.hi_key = 0; }
    __syncthreads();
    const float lo = g.below(which + 1), hi = g.below(which);       // the bin's logits: lo < x <= hi
    // (more than the list holds for sure: they are not put there one by one, which for 85000 equal ones took 30 us)
    bool many = COUNT ? s.count[which] > CAP : s.mass[which] > g.whole(fminf(hi, g.mx)) * CAP;
    if (!many) {
        each<T, NT>(row, n, [&](float x, int i) {
            if (x > lo && x <= hi) {
                const unsigned at = atomicAdd(&s.n, 1u);
                if (at < CAP) s.at[at] = place(x, i);
            }
        });
        __syncthreads();
        many = s.n > CAP;
    }
    if (many) return search_many<T, NT, COUNT>(row, n, g, lo, hi, limit, with_mass, s);
    const unsigned m = s.n;
    // Entry against entry: the others in as many parts as there are threads for, a thread an entry and a part (154 entries: 5 us; one
    // part 10, an entry to a wave 8).  The sums take the histogram's place.
    for (unsigned t = threadIdx.x; t < m; t += NT) {
        if (!COUNT || with_mass) s.w[t] = g.whole(of_key(~(unsigned)(s.at[t] >> 32)));
        s.mass[t] = 0;
    }
    __syncthreads();
    const unsigned wide = (m + 63) & ~63u, parts = max(NT / max(wide, 1u), 1u), per = (m + parts - 1) / parts;
    for (unsigned i = threadIdx.x; i < wide * parts; i += NT) {
        const unsigned part = i / wide, t = i - part * wide, end = min((part + 1) * per, m);
        if (t >= m) continue;
        const u64 me = s.at[t];
        u64 before = 0;
#pragma unroll 4
        for (unsigned j = part * per; j < end; ++j) before += s.at[j] < me ? (COUNT ? 1 : s.w[j]) : 0;
        atomicAdd(&s.mass[t], before);
    }
    __syncthreads();
    u64 sum = 0;
    for (unsigned t = threadIdx.x; t < m; t += NT)
        if (s.mass[t] <= limit) { atomicMax(&s.border, s.at[t]); if (!COUNT || with_mass) sum += s.w[t]; }
    Found f;
    block_scan<NT>(sum, s, &f.mass);
    f.border = s.border;
    return f;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_filtered_kernel(const Args a) {
    constexpr int E = Row<T>::E;
    constexpr bool TABLE = E == 8 && NT == 1024;      // (4352 weights to begin with: not for a short row's sake)
    __shared__ Shared s;
    const int n = a.bins, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const T* row = (const T*)a.logits + r * a.ld;

    // ---- the largest logit --------------------------------------------------------------------------------------------------------
    float top = -INFINITY;
    each<T, NT>(row, n, [&](float x, int) { top = fmaxf(top, x); });
    top = jb_wave_max(top);
    if (lane == 0) s.part[wave] = __float_as_uint(top);
    if (tid < 32) s.tab[tid] = EXP2_32[tid];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) top = fmaxf(top, __uint_as_float((unsigned)s.part[w]));
    __syncthreads();
    const float temp = a.temp ? a.temp[r] : a.temp_all;
    if (top == -INFINITY || !(temp > 0.f)) {          // nothing allowed: -1; temperature 0: the largest
        if (tid == 0) s.pick = 0x7fffffff;
        __syncthreads();
        if (top > -INFINITY) each<T, NT>(row, n, [&](float x, int i) { if (x == top) atomicMin(&s.pick, i); });
        __syncthreads();
        if (tid == 0) a.out[r] = top > -INFINITY ? s.pick : -1;
        return;
    }
    const int k = a.top_k ? a.top_k[r] : a.top_k_all;
    const float p = a.top_p ? a.top_p[r] : a.top_p_all;
    Weigh<T, TABLE> g;
    g.mx = top;
    g.c = 1.0 / (LN2_32 * (double)temp);
    g.md = (double)g.mx;
    // (differences of logits pass a float's range where they are as large as floats get; bins, where the temperature is as small)
    g.by = temp < 0x1p-60f ? 0x1p60f : 0.5f;
    g.bins = (float)((double)NB / RANGE / (double)temp / (double)g.by);
    g.tab = s.tab;
    g.keys = nullptr;
    const double least = fmin((double)(a.min_p ? a.min_p[r] : a.min_p_all), 1.0) * W1;
    const bool by_k = k > 0 && k < n, by_p = p > 0.f && p < 1.f;
    u64 border = ~0ull;
    // entries up to this logit weigh nothing.  (Of a row whose largest logit is infinite only its equals weigh anything.)
    const float zero = g.below(NB - 1);
    if constexpr (TABLE) {
        // where most entries are weighed, and the temperature leaves the rests' powers within a double's range
        __shared__ double keys[2 * (Weigh<T, TABLE>::KEYS + (__is_same(T, f16) ? Weigh<T, TABLE>::REST : 0))];
        if (temp >= 0.002f && (by_p || !(by_k || least > 0.0))) {
            g.template fill<NT>(keys);
            __syncthreads();
        }
    }

    if (by_k || by_p) {
        clear_bins<NT>(s);
        each_run<T, NT>(row, n, [&](float x, unsigned times) {
            if (x > zero) {
                const int b = g.bin(x);
                if (by_k) atomicAdd(&s.count[b], times);
                if (by_p) atomicAdd(&s.mass[b], g.whole(x) * times);
            }
        });
        __syncthreads();
        int kb = NB;
        u64 total = 0, limit = 0, before = 0;
        int pb = NB;
        if (by_p) {                                   // (before the histogram is used up by a search)
            u64 all, mine = 0;
            if (by_k) kb = crossing<NT, true>((u64)k - 1, s);
            const u64 before_n = by_k ? s.before_n : 0;
            __syncthreads();
            constexpr int PER = NB / NT;
#pragma unroll
            for (int b = PER * tid; b < PER * (tid + 1); ++b) mine += b < kb ? s.mass[b] : 0;
            block_scan<NT>(mine, s, &all);
            total = all;
            u64 part = 0;
            if (kb < NB) {
                // the histogram is needed again after the selection, which may clear it: keep this thread's bins
                u64 keep_m[PER];
#pragma unroll
                for (int b = 0; b < PER; ++b) keep_m[b] = s.mass[PER * tid + b];
                const Found f = select<T, NT, true>(row, n, g, kb, (u64)k - 1 - before_n, true, s);
                border = f.border;
                part = f.mass;
                __syncthreads();
#pragma unroll
                for (int b = 0; b < PER; ++b) s.mass[PER * tid + b] = keep_m[b];
                __syncthreads();
            }
            // before <= p total, in whole numbers
            limit = (u64)((double)p * (double)(total + part));
            pb = crossing<NT, false>(limit, s);
            before = s.before_w;
            __syncthreads();
            if (pb < kb || (pb == kb && kb < NB)) {
                const Found f = select<T, NT, false>(row, n, g, pb, limit - before, true, s);
                border = f.border < border ? f.border : border;
            }
        } else {
            kb = crossing<NT, true>((u64)k - 1, s);
            const u64 before_n = s.before_n;
            __syncthreads();
            if (kb < NB) border = select<T, NT, true>(row, n, g, kb, (u64)k - 1 - before_n, false, s).border;
        }
        __syncthreads();
    }

    // ---- the draw: kept weights by index ------------------------------------------------------------------------------------------
    constexpr int TILE = 256 * E;
    const int tiles = (n + TILE - 1) / TILE;
    // what top-k and top-p have kept: x > cut, or x == cut and index <= last
    const float cut = border == ~0ull ? zero : of_key(~(unsigned)(border >> 32));
    const int last = border == ~0ull ? -1 : (int)(unsigned)border;
    // (a little below what min-p leaves, in logits: the weight itself decides)
    float rough = zero;
    if (least > 0.0) {
        const float f = of_key(key_of((float)((double)top + (double)temp * (log(least / W1) - 1e-3)) - fabsf(top) * 0x1p-22f) - 1);     // (and the rounding)
        if (f > zero && f < top) rough = f;
    }
    auto weight = [&](float x) -> u64 {
        const double w = g.real(x);
        return w >= least ? g.whole(w) : 0;
    };
    const bool everything = border == ~0ull && !(least > 0.0);
    // the smallest logit to look at (the one above `zero`, which weighs nothing)
    const float edge = everything ? of_key(key_of(zero) + 1) : fmaxf(cut, rough);
    auto in = [&](float x, int i) { return x > rough && (x > cut || (x == cut && i <= last)); };
    u32x4 next[4];
    auto ask = [&](int t) {
        const int i = t * TILE + lane * E;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (i + q * 64 * E < n) next[q] = load_row(row, i + q * 64 * E, n);
    };
    ask(wave);
    for (int t = wave; t < tiles; t += NT / 64) {
        const int i = t * TILE + lane * E;
        u32x4 v[4];
        u64 w = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = next[q];
        ask(t + NT / 64);
        auto each_kept = [&](auto f) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (i + q * 64 * E < n) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float x = Row<T>::get(v[q], e);
                        if (x >= edge) f(x, i + q * 64 * E + e);
                    }
                }
        };
        // (three forms: no filter 17 us of a row of 128000, the general one 24; top-k 8 with the single comparison in front, 14 without)
        if (everything) each_kept([&](float x, int) { w += g.whole(x); });
        else if (least > 0.0) each_kept([&](float x, int j) { if (in(x, j)) w += weight(x); });
        else each_kept([&](float x, int j) { if (x > cut || j <= last) w += g.whole(x); });
        w = wave_sum(w);
        if (lane == 0) s.tile[t] = w;
    }
    __syncthreads();
    u64 total;
    const u64 mine = tid < tiles ? s.tile[tid] : 0, inc = block_scan<NT>(mine, s, &total);
    const float uf = a.u[r];
    const double ud = uf > 0.f ? (double)uf : 0.0;                 // NaN and less: the first kept token
    u64 goal = (u64)fmin(ud * (double)total, 9.0e18);
    if (goal >= total) goal = total - 1;                           // 1 and more: the last (the largest logit always weighs something)
    if (inc - mine <= goal && inc > goal) { s.pick = tid; s.before_w = inc - mine; }
    __syncthreads();
    // the tile's four parts by four waves, the one whose part it is in by its lanes
    u64 w[E], sum = 0;
    const int i = s.pick * TILE + wave * 64 * E + lane * E;
    if (wave < 4) {
        if (i < n) {
            const u32x4 v = load_row(row, i, n);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = Row<T>::get(v, e);
                w[e] = in(x, i + e) ? weight(x) : 0;
                sum += w[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = 0;
        }
    }
    const u64 upto = wave_scan(sum);
    if (lane == 63) s.part[wave] = upto;
    __syncthreads();
    if (wave < 4) {
        u64 mark = s.before_w + upto - sum;
        for (int q = 0; q < wave; ++q) mark += s.part[q];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (mark <= goal && mark + w[e] > goal) a.out[r] = i + e;
            mark += w[e];
        }
    }
}

}  // namespace

extern "C" int jb_sample_filtered(const jb_sample_filtered_args* a, void* stream) {
    JB_REQUIRE(a, "null pointer");
    JB_REQUIRE(a->dtype == JB_F32 || a->dtype == JB_F16 || a->dtype == JB_BF16, "bad dtype");
    JB_REQUIRE(a->rows >= 0 && a->bins > 0 && (a->ld >= a->bins || a->ld == 0 || a->rows < 2), "bad dims");
    if (a->bins > MAX_BINS) JB_UNSUPPORTED("vocabularies of up to 262144 tokens");
    if (a->rows == 0) return JB_OK;
    JB_REQUIRE(a->logits && a->u && a->tokens, "null pointer");
    hipStream_t s = (hipStream_t)stream;
    constexpr int64_t MOST = 1 << 21;                  // rows of a launch, which holds 2^32 threads
    for (int64_t r = 0; r < a->rows; r += MOST) {
        const unsigned n = (unsigned)(a->rows - r < MOST ? a->rows - r : MOST);
        const char* row = (const char*)a->logits + r * a->ld * (a->dtype == JB_F32 ? 4 : 2);
        auto from = [&](auto* p) { return p ? p + r : p; };
        const Args k = {row, a->ld, a->bins, a->u + r, from(a->temp), from(a->top_k), from(a->top_p), from(a->min_p),
                        a->temp_all, a->top_k_all, a->top_p_all, a->min_p_all, a->tokens + r};
        // rows of up to 16384 tokens: four waves, whose barriers cost less than the other twelve would save
#define JB_GO(T)                                                                  \
    do {                                                                          \
        if (a->bins <= 16384) sample_filtered_kernel<T, 256><<<n, 256, 0, s>>>(k); \
        else sample_filtered_kernel<T, 1024><<<n, 1024, 0, s>>>(k);               \
    } while (0)
        if (a->dtype == JB_F32) JB_GO(float); else if (a->dtype == JB_F16) JB_GO(f16); else JB_GO(bf16);
#undef JB_GO
        JB_CHECK_LAUNCH();
    }
    return JB_OK;
}

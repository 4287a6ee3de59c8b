// One token a row from logits of any vocabulary, after temperature, top-k, top-p and min-p, from a given uniform number.
//
// Definition.  w_i = exp((x_i - max x) / T); the row in the order (x descending, index ascending).  top-k keeps the first k; top-p,
// of those, every entry before which the kept weights sum to at most p of theirs; min-p those with w_i >= min_p.  Each keeps a
// PREFIX of the order, so the kept set is one prefix, described by its last entry.  The draw is the first index (in index order)
// at which the sum of the kept weights exceeds u times their total.
//
// What makes the answer a whole number that every order of summation agrees on: weights are 64-bit integers, w = round(2^44 exp(..)),
// from an exponential in double precision (2^18 of them sum to 2^62), so partial sums are exact whoever adds them, and a comparison
// with a border has the error of the weights alone, 2^-45 of the largest.  In single precision the sums of a row of 10^5 likely
// tokens are off by some 10^-7 of the total, and one draw in a thousand would differ from the definition's.
#include "paged.h"

namespace {

constexpr int NT = 1024, NB = 2048, CAP = 1024;       // threads of a row; histogram bins; entries of the exact selection
constexpr double W1 = 17592186044416.0;               // 2^44: the weight of the largest logit
constexpr double RANGE = 32.0;                        // exp(-31.98) 2^44 < 0.5: entries further from the largest weigh nothing
constexpr int MAX_BINS = 1 << 18;
constexpr double LN2_REST = 1.908214929270587816e-10;   // ln 2 - 2977044471 / 2^32

typedef unsigned long long u64;

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
// NaN counts as a forbidden token; -0 is 0
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
// E logits from index i on; -inf behind the row's end
template <typename T> __device__ __forceinline__ void load_row(const T* row, int i, int n, float (&x)[Row<T>::E]) {
    constexpr int E = Row<T>::E;
    if (i + E <= n) {
        const u32x4 v = *reinterpret_cast<const u32x4_any*>(row + i);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = clean(Row<T>::get(v, e));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = i + e < n ? clean((float)row[i + e]) : -INFINITY;
    }
}

// exp(y) for y <= 0: y = n ln 2 + r, |r| <= ln 2 / 2, exp(r) by its Taylor series to r^13 (the next term: 2^-54).
// Coefficients 1 / k!.
__device__ __forceinline__ double exp_neg(double y) {
    const double n = rint(y * 1.4426950408889634074);
    double r = fma(n, -2977044471.0 / 4294967296.0, y);          // ln 2 = its first 32 bits and the rest: n times the first is exact
    r = fma(n, -LN2_REST, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
struct Weigh {
    float mx, bins;                                   // largest logit; bins per unit of logit
    double inv_t, min_p;
    // entries further below the largest than RANGE temperatures are in the last bin and weigh nothing
    __device__ __forceinline__ int bin(float x) const { return x == mx ? 0 : (int)fminf((mx - x) * bins, (float)(NB - 1)); }
    __device__ __forceinline__ double real(float x) const { return x == mx ? 1.0 : exp_neg(((double)x - (double)mx) * inv_t); }
    // a whole number in the low bits of the sum with 2^52: rounded to nearest
    static __device__ __forceinline__ u64 whole(double w) { return (u64)__double_as_longlong(w * W1 + 4503599627370496.0) & 0xfffffffffffffull; }
};
// order (x descending, index ascending) as one ascending integer
__device__ __forceinline__ u64 place(float x, int i) {
    const unsigned b = __float_as_uint(x), up = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return ((u64)~up << 32) | (unsigned)i;
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
    u64 tile[MAX_BINS / 256];                         // kept weight of 64 E consecutive entries
    u64 part[NT / 64];
    float fpart[NT / 64];
    u64 border;                                       // place of the last kept entry
    u64 before_w; unsigned before_n, n;               // of the border bin; entries listed
    int pick;
};
// inclusive prefix sum over the block; *total: all
__device__ __forceinline__ u64 block_scan(u64 v, Shared& s, u64* total) {
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

// The first bin at which the running sum of `v` (two bins a thread, in order) exceeds `limit`; NB if none does.  s.before_*: the
// sums in front of it.
template <typename V> __device__ int crossing(const V* v, u64 limit, Shared& s, u64* before) {
    if (threadIdx.x == 0) { s.pick = NB; s.before_w = 0; }
    __syncthreads();
    const u64 a = v[2 * threadIdx.x], b = v[2 * threadIdx.x + 1];
    u64 total;
    const u64 inc = block_scan(a + b, s, &total), exc = inc - a - b;
    if (exc <= limit && inc > limit) {
        const bool second = exc + a <= limit;
        s.pick = 2 * threadIdx.x + second;
        s.before_w = exc + (second ? a : 0);
    }
    __syncthreads();
    const int r = s.pick;
    *before = s.before_w;
    __syncthreads();
    return r;
}

template <typename T>
__global__ __launch_bounds__(NT) void sample_filtered_kernel(const Args a) {
    constexpr int E = Row<T>::E, STEP = NT * E;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    const int n = a.bins, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const T* row = (const T*)a.logits + r * a.ld;
    float x[E];

    // ---- the largest logit and its first index ---------------------------------------------------------------------------------
    u64 first = ~0ull;
    for (int i = tid * E; i < n; i += STEP) {
        load_row(row, i, n, x);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (i + e < n) { const u64 p = place(x[e], i + e); first = p < first ? p : first; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const u64 u = __shfl_xor(first, o); first = u < first ? u : first; }
    if (lane == 0) s.part[wave] = first;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) first = s.part[w] < first ? s.part[w] : first;
    __syncthreads();
    const unsigned up = ~(unsigned)(first >> 32);
    const float mx = __uint_as_float(up ^ ((up >> 31) ? 0x80000000u : 0xffffffffu));
    const float temp = a.temp ? a.temp[r] : a.temp_all;
    if (mx == -INFINITY || !(temp > 0.f)) {           // nothing allowed: -1; temperature 0: the largest
        if (tid == 0) a.out[r] = mx == -INFINITY ? -1 : (int64_t)(unsigned)first;
        return;
    }
    const int k = a.top_k ? a.top_k[r] : a.top_k_all;
    const float p = a.top_p ? a.top_p[r] : a.top_p_all;
    Weigh g;
    g.mx = mx; g.inv_t = 1.0 / (double)temp; g.bins = (float)((double)NB / RANGE * g.inv_t); g.min_p = fmin((double)(a.min_p ? a.min_p[r] : a.min_p_all), 1.0);
    const bool by_k = k > 0 && k < n, by_p = p > 0.f && p < 1.f;
    u64 border = ~0ull;

    if (by_k || by_p) {
        for (int i = tid; i < NB; i += NT) { s.mass[i] = 0; s.count[i] = 0; }
        __syncthreads();
        for (int i = tid * E; i < n; i += STEP) {
            load_row(row, i, n, x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int b = g.bin(x[e]);
                if (b < NB - 1) {
                    if (by_k) atomicAdd(&s.count[b], 1u);
                    if (by_p) atomicAdd(&s.mass[b], Weigh::whole(g.real(x[e])));
                }
            }
        }
        __syncthreads();
        u64 before_n = 0, before_w = 0, limit_w = ~0ull;
        int bin = NB;
        // Entries of one bin in exact order: for each, what of its bin comes before it.
        auto list_bin = [&](int which) {
            if (tid == 0) s.n = 0;
            __syncthreads();
            for (int i = tid * E; i < n; i += STEP) {
                load_row(row, i, n, x);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (g.bin(x[e]) == which && i + e < n && x[e] > -INFINITY) {
                        const unsigned at = atomicAdd(&s.n, 1u);
                        if (at < CAP) { s.at[at] = place(x[e], i + e); s.w[at] = Weigh::whole(g.real(x[e])); }
                    }
            }
            __syncthreads();
        };
        // The last kept entry among those of bin `which` whose place is at most `upto`: rank below `rank` and weight before within `limit`.
        // Bins of up to CAP entries are ranked entry against entry; larger ones (many equal logits) are halved by place, 64 times.
        auto select = [&](int which, u64 rank, u64 limit, u64 upto, u64* mass) {
            list_bin(which);
            const unsigned m = s.n;
            if (tid == 0) s.border = 0;
            __syncthreads();
            u64 sum = 0;
            if (m <= CAP) {
                if (tid < m && s.at[tid] <= upto) {
                    const u64 me = s.at[tid];
                    u64 nb = 0, wb = 0;
                    for (unsigned j = 0; j < m; ++j)
                        if (s.at[j] < me) { ++nb; wb += s.w[j]; }
                    if (nb < rank && wb <= limit) { atomicMax(&s.border, me); sum = s.w[tid]; }
                }
                u64 total;
                block_scan(sum, s, &total);
                *mass = total;
                return s.border;
            }
            // the largest place L with  #{place < L} < rank  and  weight{place < L} <= limit  among places <= upto: by bisection
            auto below = [&](u64 L, u64* cnt, u64* wt) {
                u64 c = 0, w = 0;
                for (int i = tid * E; i < n; i += STEP) {
                    load_row(row, i, n, x);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (i + e < n && x[e] > -INFINITY && g.bin(x[e]) == which && place(x[e], i + e) < L) { ++c; w += Weigh::whole(g.real(x[e])); }
                }
                block_scan(c, s, cnt);
                block_scan(w, s, wt);
            };
            u64 L = 0, c, w;
            for (int bit = 63; bit >= 0; --bit) {
                const u64 cand = L | (1ull << bit);
                below(cand, &c, &w);
                if (c < rank && w <= limit) L = cand;
            }
            // L: the largest value for which the entries before it still leave room: every entry at or before L is kept
            if (L > upto) L = upto;
            below(L + (L != ~0ull), &c, &w);
            *mass = w;
            return L;
        };
        u64 mass_k = 0;
        if (by_k) {
            bin = crossing(s.count, (u64)k - 1, s, &before_n);
            if (bin < NB) {
                border = select(bin, (u64)k - before_n, ~0ull, ~0ull, &mass_k);
            }
        }
        if (by_p) {
            // weight of what top-k has left: the bins before its border's, and the border bin's part
            u64 total, all;
            u64 mine = 0;
            for (int b = 2 * tid; b < 2 * tid + 2; ++b) mine += b < bin ? s.mass[b] : 0;
            block_scan(mine, s, &all);
            total = all + (bin < NB ? mass_k : 0);
            // before <= p total, in whole numbers
            limit_w = (u64)((double)p * (double)total);
            const int pb = crossing(s.mass, limit_w, s, &before_w);
            if (pb < bin || (pb == bin && bin < NB)) border = select(pb, ~0ull, limit_w - before_w, border, &mass_k);
        }
    }

    // ---- the draw: kept weights by index ------------------------------------------------------------------------------------------
    const int tiles = (n + 64 * E - 1) / (64 * E);
    auto kept = [&](float v, int i) -> u64 {
        if (i >= n || g.bin(v) >= NB - 1 || place(v, i) > border) return 0;
        const double w = g.real(v);
        return w >= g.min_p ? Weigh::whole(w) : 0;
    };
    for (int t = wave; t < tiles; t += NT / 64) {
        const int i = t * 64 * E + lane * E;
        u64 w = 0;
        if (i < n) {
            load_row(row, i, n, x);
#pragma unroll
            for (int e = 0; e < E; ++e) w += kept(x[e], i + e);
        }
        w = wave_sum(w);
        if (lane == 0) s.tile[t] = w;
    }
    __syncthreads();
    const int per = (tiles + NT - 1) / NT;
    u64 mine = 0, total;
    for (int t = tid * per; t < min(tiles, (tid + 1) * per); ++t) mine += s.tile[t];
    const u64 inc = block_scan(mine, s, &total);
    const float uf = a.u[r];
    const double ud = uf > 0.f ? (double)uf : 0.0;                 // NaN and less: the first kept token
    u64 goal = (u64)fmin(ud * (double)total, 9.0e18);
    if (goal >= total) goal = total - 1;                           // 1 and more: the last (the largest logit always weighs something)
    u64 left = inc - mine;
    if (left <= goal && inc > goal)
        for (int t = tid * per; t < min(tiles, (tid + 1) * per); ++t) {
            if (left + s.tile[t] > goal) { s.pick = t; s.before_w = left; break; }
            left += s.tile[t];
        }
    __syncthreads();
    if (wave == 0) {
        const int i = s.pick * 64 * E + lane * E;
        u64 w[E], sum = 0;
        if (i < n) load_row(row, i, n, x);
#pragma unroll
        for (int e = 0; e < E; ++e) { w[e] = i < n ? kept(x[e], i + e) : 0; sum += w[e]; }
        u64 at = s.before_w + wave_scan(sum) - sum;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (at <= goal && at + w[e] > goal) a.out[r] = i + e;
            at += w[e];
        }
    }
}

}  // namespace

extern "C" int jb_sample_filtered(const jb_sample_filtered_args* a, void* stream) {
    JB_REQUIRE(a, "null pointer");
    JB_REQUIRE(a->dtype == JB_F32 || a->dtype == JB_F16 || a->dtype == JB_BF16, "bad dtype");
    JB_REQUIRE(a->rows >= 0 && a->bins > 0 && (a->ld >= a->bins || a->rows < 2), "bad dims");
    if (a->bins > MAX_BINS) JB_UNSUPPORTED("vocabularies of up to 262144 tokens");
    if (a->rows == 0) return JB_OK;
    JB_REQUIRE(a->logits && a->u && a->tokens, "null pointer");
    const Args k = {a->logits, a->ld, a->bins, a->u, a->temp, a->top_k, a->top_p, a->min_p, a->temp_all, a->top_k_all, a->top_p_all, a->min_p_all, a->tokens};
    static_assert(sizeof(Shared) <= 64 * 1024, "LDS");
    hipStream_t s = (hipStream_t)stream;
    if (a->dtype == JB_F32) sample_filtered_kernel<float><<<(unsigned)a->rows, NT, sizeof(Shared), s>>>(k);
    else if (a->dtype == JB_F16) sample_filtered_kernel<f16><<<(unsigned)a->rows, NT, sizeof(Shared), s>>>(k);
    else sample_filtered_kernel<bf16><<<(unsigned)a->rows, NT, sizeof(Shared), s>>>(k);
    JB_CHECK_LAUNCH();
    return JB_OK;
}

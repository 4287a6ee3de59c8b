// Attention of the newest tokens of many sequences over key / value rows that lie in pages.
//
//   out[t][h] = sum_k softmax_k(scale q[t][h] . K[k][h / G]) V[k][h / G],   k over the positions that t's position sees
//
// A sequence is a row of `table` (its page numbers in order of position) and its length; its queries are its last cu_q[i+1] -
// cu_q[i] positions.  G = n_head / n_kv_head query heads share a key / value head, so a tile of 16 ROWS -- a row is a (token, head
// of the group) pair, heads fastest -- meets one K / V stream, for one new token as for thousands.
#include "paged.h"

namespace {

template <typename T> struct El;
template <> struct El<f16> {
    typedef f16x8 vec;
    static constexpr int E = 8;
    static constexpr unsigned ABS = 0x7fff7fffu, STEP = 0x04000400u;      // of two elements: without the sign; the exponent's lowest bit
    static constexpr float LIFT = 14.f;                                   // see reference_of
    static constexpr float TINY = 0x1p-24f, SPLIT = 0x1p-13f;             // the smallest number; from where on a half of one is exact
    static __device__ __forceinline__ f32x4 mfma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct El<bf16> {
    typedef bf16x8 vec;
    static constexpr int E = 8;
    static constexpr unsigned ABS = 0x7fff7fffu, STEP = 0x00800080u;
    static constexpr float LIFT = 0.f;
    static constexpr float TINY = 0x1p-126f, SPLIT = 0x1p-125f;
    static __device__ __forceinline__ f32x4 mfma(vec a, vec b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct El<float> {
    typedef f32x4 vec;
    static constexpr int E = 4;
    static constexpr unsigned ABS = 0x7fffffffu, STEP = 0x00800000u;
    static constexpr float LIFT = 0.f;
    static __device__ __forceinline__ f32x4 mfma(vec a, vec b, f32x4 c) { return jb_mfma(a, b, c); }
};

// A row's probabilities are 2^(score - m) with m the running maximum less LIFT (scores in units of log2 e).  A half is subnormal below
// 2^-14 and 0 below 2^-25: unlifted, the 8000 keys 18 nats below one other were lost from the values' sum and not from the weights'.  Up to
// 2^14 = a quarter of the largest half they keep their bits down to 2^-28 of the largest.  (What m is exactly does not matter, as a state's
// sum, values and m go together -- but that no probability passes 2^15: far scores, of which 14 is within a rounding or two, go unlifted.)
template <typename T> __device__ __forceinline__ float reference_of(float mx) { return El<T>::LIFT != 0.f && fabsf(mx) < 0x1p20f ? mx - El<T>::LIFT : mx; }

// A probability's exponent is one fused c score - m, while m came from a rounded product: of scores past 2^28 the two are 16 and more
// apart, and the largest probability left the range of a half, past 2^31 that of a float (NaN, or a sum of 0).  From FAR on -- the rounding is
// then half of one -- the product is rounded as m's was, so that the largest score's exponent is 0.
constexpr float FAR = 0x1p24f;
template <int N, typename V> __device__ __forceinline__ void settle(V& s, float c, float m) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float x = s[i] * c;
        asm volatile("" : "+v"(x));              // (or the compiler fuses it all the same)
        s[i] = x - m;
    }
}

// A number's part that is left to the first of two places; what is missing goes to the second.  Both are exact, and of the number's own sign
// unless it is 0, or no larger than the smallest (bf16: normal) one.
template <typename T> __device__ __forceinline__ float half_of(float v) { return fabsf(v) >= El<T>::SPLIT ? v * 0.5f : v == 0.f ? 0.f : v - copysignf(El<T>::TINY, v); }

struct Args {
    const void* q; int64_t q_row, q_head;
    void* out; int64_t o_row, o_head;
    const void *k, *v; int64_t page_stride, row_stride, head_stride;
    const int* table; int64_t table_stride; int max_pages;
    const int *lens, *cu;
    float* part; float* ml;                      // splits' states: [token][head][split][D], [token][head][split][2]
    JbDiv page, group;
    unsigned n_pages;
    int page_shift;                              // ceil(log2 page_size): a row of the cache is (page << page_shift) | row in page
    int n_tokens, n_seq, n_head, n_kv, G, D;
    int func, bc, window;
    int tr;                                      // rows of a tile
    int tiles, splits; unsigned chunk;                    // grid: row tiles per (sequence, kv head), key splits, keys of a split's turn
    unsigned groups; int by_die;                 // order of the workgroups (place_of)
    int aligned;                                 // pages of a multiple of 16 rows, consecutive positions
    float c, c_abs;                              // scale * log2(e); its magnitude, not quite 0 (-inf * 0 is no number)
};

constexpr unsigned BAD = 0xffffffffu;            // a key on a page number that does not exist: nobody sees it
constexpr int KB = 32;                           // keys of a wave's turn

struct Seq { int t0, nq, pos0; const int* table; };      // first query row, queries, position of the first, page numbers
__device__ __forceinline__ Seq seq_of(const Args& a, int i) {
    Seq s;
    s.t0 = min(max(a.cu[i], 0), a.n_tokens);
    s.nq = max(min(a.cu[i + 1], a.n_tokens) - s.t0, 0);
    const int64_t cap = (int64_t)a.max_pages * a.page.d;
    const int len = (int)min((int64_t)max(a.lens[i], 0), min(cap, (int64_t)0x7fff0000));
    s.pos0 = len - s.nq;
    s.table = a.table + (int64_t)i * a.table_stride;
    return s;
}
__device__ __forceinline__ int times(int n, int bc) { return n > 0 ? (n - 1) / bc + 1 : 0; }      // ceil(n / bc), bc as large as it may be
__device__ __forceinline__ int tiles_of(const Args& a, int nq) {
    if (a.func != JB_ATTN_TRANSPOSE_BLOCK) return (int)(((int64_t)nq * a.G + a.tr - 1) / a.tr);
    const int cls = min(a.bc, nq);
    return cls * (int)(((int64_t)times(nq, a.bc) * a.G + a.tr - 1) / a.tr);
}
// Row r of a tile is token j0 + i * js of the chunk, i = (row0 + r) / G, head (row0 + r) % G; the keys that any of its rows
// may see sit at positions kb + x * ks, x < n.
struct Tile { int j0, js, row0, rows, kb, ks, n; };      // rows: rows of this tile's class in all
__device__ __forceinline__ Tile tile_of(const Args& a, const Seq& s, int tile) {
    Tile t;
    if (a.func == JB_ATTN_TRANSPOSE_BLOCK) {             // one residue class of positions modulo bc
        const int per = (int)(((int64_t)times(s.nq, a.bc) * a.G + a.tr - 1) / a.tr);
        t.j0 = tile / per; t.js = a.bc; t.row0 = (tile % per) * a.tr;
        t.rows = times(s.nq - t.j0, a.bc) * a.G;
    } else {
        t.j0 = 0; t.js = 1; t.row0 = tile * a.tr; t.rows = s.nq * a.G;
    }
    t.kb = 0; t.ks = 1; t.n = 0;
    if (t.row0 >= t.rows) return t;
    const int pf = max(s.pos0 + t.j0 + (int)jb_div(t.row0, a.group) * t.js, 0);
    const int pl = s.pos0 + t.j0 + (int)jb_div(min(t.row0 + a.tr, t.rows) - 1, a.group) * t.js;
    if (pl < 0) return t;                                // a length shorter than the chunk: no such positions
    switch (a.func) {
        case JB_ATTN_BLOCK: t.kb = pf - pf % a.bc; t.n = pl + 1 - t.kb; break;
        case JB_ATTN_PREV_BLOCK: t.kb = max(pf / a.bc - 1, 0) * a.bc; t.n = max(pl / a.bc * a.bc - t.kb, 0); break;
        case JB_ATTN_TRANSPOSE_BLOCK: t.ks = a.bc; t.kb = pl % a.bc; t.n = pl / a.bc + 1; break;
        default: t.kb = a.window ? max(pf - a.window + 1, 0) : 0; t.n = pl + 1 - t.kb;
    }
    if (a.aligned && t.n > 0) { t.n += t.kb & 15; t.kb &= ~15; }        // halves of turns begin at multiples of 16
    return t;
}
// The positions [lo, hi) that the query at position p sees (of those its tile walks).
__device__ __forceinline__ void sees(const Args& a, int p, int& lo, int& hi) {
    lo = 0; hi = p + 1;
    if (p < 0) { hi = 0; return; }
    if (a.func == JB_ATTN_BLOCK) lo = p - p % a.bc;
    else if (a.func == JB_ATTN_PREV_BLOCK) { const int b = p / a.bc; hi = b * a.bc; lo = hi - (b > 0 ? a.bc : 0); }
    else if (a.func == JB_ATTN_DENSE && a.window) lo = max(p - a.window + 1, 0);
}
__device__ __forceinline__ int active_splits(const Args& a, int n) {
    return a.splits == 1 ? 1 : min(a.splits, max((int)(((unsigned)n + a.chunk - 1u) / a.chunk), 1));
}

// Workgroup b's work.  Workgroups go round the eight dies by number, and each die has its own L2: b % 8 picks the group of work items
// that share memory -- one token a sequence: a sequence's keys under all heads, whose rows lie side by side; chunks: a head's keys
// under all tiles -- and a die takes a group's items one after the other.  Where that would leave dies idle, or give them sequences of
// different lengths (chunks whose heads are no multiple of eight), the items go round instead.
__device__ __forceinline__ bool place_of(const Args& a, unsigned b, int& tile, int& split, int& kvh, int& si) {
    const unsigned inner = a.tiles == 1 ? a.n_kv : a.tiles;
    unsigned group, item;
    if (a.by_die) { const unsigned r = b >> 3; item = r % inner; group = (r / inner) * 8 + (b & 7); }
    else { item = b % inner; group = b / inner; }
    if (group >= a.groups) return false;
    if (a.tiles == 1) { si = (int)(group % a.n_seq); split = (int)(group / a.n_seq); kvh = (int)item; tile = 0; }
    else { kvh = (int)(group % a.n_kv); group /= a.n_kv; si = (int)(group % a.n_seq); split = (int)(group / a.n_seq); tile = a.tiles - 1 - (int)item; }      // the longest first
    return true;
}

// (page << page_shift) | row in page of a position; BAD where the table names no page.
__device__ __forceinline__ unsigned cache_row(const Args& a, const Seq& s, int pos) {
    const unsigned p = jb_div((unsigned)pos, a.page);
    const unsigned pg = (unsigned)s.table[p];
    return pg < a.n_pages ? (pg << a.page_shift) | ((unsigned)pos - p * a.page.d) : BAD;
}
__device__ __forceinline__ int64_t cache_offset(const Args& a, unsigned row) {
    row = row == BAD ? 0u : row;
    return (int64_t)(row >> a.page_shift) * a.page_stride + (int64_t)(row & ((1u << a.page_shift) - 1u)) * a.row_stride;
}
template <typename T> __device__ __forceinline__ u32x4 load16(const T* p) { return *reinterpret_cast<const u32x4_any*>(p); }

// The A operands of O^T += V^T P^T from the rows themselves: w[i] holds E consecutive channels of key i of the lane's group, the
// operand of tile j wants channel j of all of them.  A lane owns both, so the transposition is a byte permutation per two elements.
__device__ __forceinline__ f16x8 gather(const u32x4 (&w)[8], int j, f16) {
    u32x4 r;
#pragma unroll
    for (int h = 0; h < 4; ++h) r[h] = __builtin_amdgcn_perm(w[2 * h + 1][j >> 1], w[2 * h][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(f16x8, r);
}
__device__ __forceinline__ bf16x8 gather(const u32x4 (&w)[8], int j, bf16) { return __builtin_bit_cast(bf16x8, gather(w, j, f16())); }

template <typename T> __device__ __forceinline__ void store8(T* o, const float* v);
template <> __device__ __forceinline__ void store8(float* o, const float* v) {
    *reinterpret_cast<u32x4_any*>(o) = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
    *reinterpret_cast<u32x4_any*>(o + 4) = __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]});
}
template <typename T> __device__ __forceinline__ void store8(T* o, const float* v) {
    typename El<T>::vec x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (T)v[e];
    *reinterpret_cast<u32x4_any*>(o) = __builtin_bit_cast(u32x4, x);
}

// Values that are no numbers, for the 16 rows of a tile from row0 on that are not in `skip`: where a row sees an infinite value its output is
// infinite, where it sees infinite ones of both signs or a NaN it is no number, whatever else is in the sum (a probability is not 0; one of a
// score of -inf is, and 0 times infinity no number: its key counts all the same, as telling it took 5-10 % of short chunks' time).  The
// matrix products cannot say so: a value a row does not see would reach it as 0 * NaN, and one that it sees meets parts that are 0 -- the low
// part of a probability that has none, a probability that rounds to 0.  So turns that some row does not see whole take such values out of
// the operands, and a tile that has met one, or whose sums are not finite, ends here: one wave looks through the split's values, 64
// keys at a time, for those that are no numbers, and overwrites what they decide.  Channels dc .. dc + 63 for dc = 64 part, + 64 parts, ...
template <typename T>
__device__ void put_infinities(const Args& a, const Seq& s, const Tile& t, int kvh, int split, int n_act, int row0, unsigned skip, int part, int parts) {
    constexpr int E = El<T>::E;
    const int lane = threadIdx.x & 63, my = min(row0 + (lane & 15), t.rows - 1), D = a.D;
    const T* vbase = (const T*)a.v + (int64_t)kvh * a.head_stride;
    int first, end;
    {
        const int p = s.pos0 + t.j0 + (int)jb_div(my, a.group) * t.js;
        sees(a, p, first, end);
        if (t.ks == 1) { first = max(first - t.kb, 0); end -= t.kb; }
        else { first = 0; end = p < 0 ? 0 : p / t.ks + 1; }
    }
    for (int dc = part * 64; dc < D; dc += parts * 64) {
        unsigned pos = 0u, neg = 0u;             // bit r: row r sees such a value of channel dc + lane
        for (unsigned x0 = split * a.chunk; x0 < (unsigned)t.n; x0 += n_act * a.chunk) {
            const int x1 = (int)min(x0 + a.chunk, (unsigned)t.n);
            for (int xb = (int)x0; xb < x1; xb += 64) {
                const unsigned rows = cache_row(a, s, t.kb + min(xb + lane, x1 - 1) * t.ks);         // a key a lane
                bool odd = false;
                if (rows != BAD && xb + lane < x1)
                    for (int d = dc; d < min(dc + 64, D); d += E) {
                        const u32x4 w = load16(vbase + cache_offset(a, rows) + min(d, D - E));
#pragma unroll
                        for (int h = 0; h < 4; ++h) odd |= (((w[h] & El<T>::ABS) + El<T>::STEP) & ~El<T>::ABS) != 0u;
                    }
                for (unsigned long long who = __ballot(odd); who; who &= who - 1) {
                    const int i = __builtin_ctzll(who), x = xb + i;
                    const float v = (float)vbase[cache_offset(a, (unsigned)__builtin_amdgcn_readlane((int)rows, i)) + min(dc + lane, D - 1)];
                    const unsigned who_sees = (unsigned)__ballot(lane < 16 && x >= first && x < end);
                    pos |= v != v || v == INFINITY ? who_sees : 0u;
                    neg |= v != v || v == -INFINITY ? who_sees : 0u;
                }
            }
        }
        if (dc + lane >= D) continue;
        for (int r = 0; r < 16; ++r) {
            const bool up = pos >> r & 1u, down = neg >> r & 1u;
            if (skip >> r & 1u || !(up || down)) continue;
            const float v = up && down ? NAN : up ? INFINITY : -INFINITY;
            const int i = (int)jb_div(row0 + r, a.group), h = kvh * a.G + (row0 + r - i * a.G);
            const int64_t tok = s.t0 + t.j0 + i * t.js;
            if (n_act > 1) a.part[((tok * a.n_head + h) * a.splits + split) * (int64_t)D + dc + lane] = v;
            else ((T*)a.out)[tok * a.o_row + (int64_t)h * a.o_head + dc + lane] = (T)v;
        }
    }
}

// One workgroup per (sequence, kv head, tile of 16 rows, split of the keys).
//
//   S^T = K Q^T     A = 16 keys x 32 channels straight from the cache rows, B = the rows' queries (in registers throughout): a
//                   lane holds, for query row l & 15, the scores of keys (l >> 4) * 4 + r of both 16-key halves -- the softmax
//                   statistics take two cross-lane steps, and the rescaling of the output none.
//   O^T += V^T P^T  the order of a product's inner index is free: slot (g, i) is key (i / 4) * 16 + g * 4 + i % 4, so the B
//                   operand is the lane's own probabilities, and the A operand the lane's own eight value pieces (gather above).
// K and V therefore go from memory to the matrix cores through registers alone.
// In 16 bits the probabilities enter as a high and a low part (two products), off by 2^-16 of themselves in bf16 and 2^-22 in f16 (those
// above 2^-28 of the largest, see reference_of; an absolute 2^-39 below): the output is as near the 64-bit value as its own rounding allows; the products hide behind the memory anyway (one new token: 1 row of 16 used).
// NC slices of 16 E channels cover d_head, each a wave's: heads of up to 128 halfs have four waves side by side on the keys, every
// one with a running maximum and sum of its own, joined through LDS at the end; wider heads NC waves to a turn of 32 keys, which add
// up their parts of the scores through LDS (one barrier a turn).  One wave for a whole head of 480 channels held 512 registers, four
// waves a compute unit, each request waiting for the one before.
// ALIGNED (pages of a multiple of 16 rows, keys at consecutive positions): a 16-key half of a turn lies in one page, so that its rows
// are one scalar address and a lane's constant offset, page numbers come 64 at a time, and the next turn's rows are on their way while
// one is computed.  Otherwise (odd pages, the transpose pattern) every key is looked up by a lane and its address handed round.
// Measured (one new token a sequence; a copy reaches 4.7 TB/s on the card): 64 sequences of 511-8192 keys, 32 heads on 8 of 128 channels,
// bf16 in pages of 16: 260 us, 4.4 TB/s; 16 of 4096-8192 under a head of 480: 39 us in f16, 4.8 TB/s over and over the same cache (4.0 over
// three in turn), 94 us in f32, 4.0 TB/s; 64 of 500-4000, 8 heads of 150: 178 us, 3.8 TB/s.  Bound by memory.  Three waves a SIMD instead of
// two, for which the registers spill: 310, 54, 174 and 289 us.  Keys looked up lane by lane instead of ALIGNED: 251, 43, 125 and 263 us.
template <typename T, int NC> struct Shape {
    static constexpr int WAVES = NC > 4 ? NC : 4, KG = WAVES / NC, CH = 16 * El<T>::E, LDO = CH + 4;     // LDO: rows 4 banks apart
    struct alignas(16) Shared {
        float s[NC > 1 ? 2 : 1][NC > 1 ? WAVES : 1][NC > 1 ? 64 : 1][8];      // parts of the scores, two turns' worth
        float o[KG > 1 ? WAVES : 1][KG > 1 ? 16 : 1][LDO];
        float ml[KG][16][2];
        int odd;
    };
};
template <typename T, int NC, bool ALIGNED>
__global__ __launch_bounds__((Shape<T, NC>::WAVES * 64), 2) void attn_paged_rows_kernel(const Args a) {
    typedef typename El<T>::vec vec;
    typedef Shape<T, NC> Sh;
    constexpr int E = El<T>::E, CH = Sh::CH, KT = 4 * E, NK = CH / KT, KG = Sh::KG;
    __shared__ typename Sh::Shared sh;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    // scalar, so that what depends on the wave branches: matrix instructions run whatever the lanes' mask, also under an empty one
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / NC, cb = wave % NC * CH;
    int tile0, split, kvh, si;
    if (!place_of(a, blockIdx.x, tile0, split, kvh, si)) return;
    const Seq s = seq_of(a, si);
    const int n_tiles = tiles_of(a, s.nq);
    const T* kbase = (const T*)a.k + (int64_t)kvh * a.head_stride;
    const T* vbase = (const T*)a.v + (int64_t)kvh * a.head_stride;
    const int D = a.D, nk = min((D - cb + KT - 1) / KT, NK);       // k-tiles of this slice (none: a slice behind the head's end)
    int flip = 0;
    // a lane's offsets from the row of its half's first key (ALIGNED): fragments' channels are clamped to the head
    // -- bytes, so that an access is a scalar base and a 32-bit offset
    const unsigned rs = (unsigned)a.row_stride * (unsigned)sizeof(T);
    unsigned koff[NK], voff[4];
    if constexpr (ALIGNED) {
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) koff[ks] = c * rs + (unsigned)min(cb + ks * KT + g * E, D - E) * (unsigned)sizeof(T);
#pragma unroll
        for (int r = 0; r < 4; ++r) voff[r] = (g * 4 + r) * rs + (unsigned)min(cb + c * E, D - E) * (unsigned)sizeof(T);
    }

    for (int tile = tile0; tile < n_tiles; tile += a.tiles) {
        const Tile t = tile_of(a, s, tile);
        if (t.row0 >= t.rows) continue;
        const int n_act = active_splits(a, t.n);
        if (split >= n_act) continue;
        const int R = t.row0 + c, my = min(R, t.rows - 1);
        const int qi = (int)jb_div(my, a.group), j = t.j0 + qi * t.js, head = kvh * a.G + (my - qi * a.G);
        const bool row_ok = R < t.rows;
        // the walked keys [xlo, xhi) that the lane's row sees, and those that every row of the tile sees: the first row ends first, the
        // last begins last.  (What rows that are none would add up stays in their own columns.)
        auto walk = [&](int p, int& first, int& end) {
            int lo, hi;
            sees(a, p, lo, hi);
            if (t.ks == 1) { first = max(lo - t.kb, 0); end = hi - t.kb; }
            else { first = 0; end = p < 0 ? 0 : p / t.ks + 1; }
        };
        int xlo, xhi, all_lo, all_hi, unused;
        walk(s.pos0 + j, xlo, xhi);
        if (!row_ok || xhi < xlo) xlo = xhi = 0;
        walk(s.pos0 + t.j0 + (int)jb_div(t.row0, a.group) * t.js, unused, all_hi);
        walk(s.pos0 + t.j0 + (int)jb_div(min(t.row0 + 15, t.rows - 1), a.group) * t.js, all_lo, unused);

        const T* qrow = (const T*)a.q + (int64_t)(s.t0 + j) * a.q_row + (int64_t)head * a.q_head;
        vec qf[NK];
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
            // a fragment that passes the end of the head is read from D - E on, as the keys' is; what an earlier one covers is zeroed
            const int e0 = cb + ks * KT + g * E, at = min(e0, D - E);
            qf[ks] = __builtin_bit_cast(vec, load16(qrow + at));
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (at + e < e0 || !row_ok) qf[ks][e] = (T)0.f;
        }
        f32x4 acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;            // of the lane's row: the reference the same in its four lanes, the sum a part in each
        bool odd = false;                        // values that are no numbers have been taken out of a turn (put_infinities)
        // Channels that a fragment past the head's end has over again meet zeros of the query: out of the keys they go too (an infinite one
        // would be 0 * inf, not the score of -inf that takes its key out)
        const bool tail = NC == 1 ? D < CH : nk > 0 && D - cb < nk * KT;
        auto clear_tail = [&](u32x4 (&kf)[2][NK]) {
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                if (ks < nk - 1) continue;
                const int again = cb + ks * KT + g * E - (D - E);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const unsigned keep = E == 4 ? (again > d ? 0u : ~0u) : again >= 2 * d + 2 ? 0u : again == 2 * d + 1 ? 0xffff0000u : ~0u;
#pragma unroll
                    for (int h = 0; h < 2; ++h) kf[h][ks][d] &= keep;
                }
            }
        };

        // One turn: the scores' parts so far in sc, the values in vf.  gone: bit i, no page holds key i.
        auto turn = [&](f32x4 (&sc)[2], u32x4 (&vf)[8], int xb, int x1, unsigned gone) {
            // scores of keys h * 16 + g * 4 + r, i.e. of slot i = h * 4 + r
            const bool masked = xb + KB > x1 || xb < all_lo || xb + KB > all_hi || __any(gone != 0u);
            unsigned see = 0xffu;
            float p[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = sc[i >> 2][i & 3] * a.c;
            if (masked) {
                see = 0u;
                const unsigned d0 = (unsigned)(xb + g * 4 - xlo), dn = (unsigned)(min(xhi, x1) > xlo ? min(xhi, x1) - xlo : 0);
#pragma unroll
                for (int i = 0; i < 8; ++i) see |= (d0 + (i >> 2) * 16 + (i & 3) < dn ? 1u : 0u) << i;
                see &= ~gone;
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = see >> i & 1u ? p[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, p[i]);
            mx = jb_rows_reduce(mx, [](float u, float v) { return fmaxf(u, v); });
            const float m_new = fmaxf(m, reference_of<T>(mx)), base = m_new == -INFINITY ? 0.f : m_new;
            if (__any(m_new != m)) {
                const float alpha = __builtin_amdgcn_exp2f(m - base);
                l *= alpha;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] *= alpha;
                m = m_new;
            }
            // (fused: the rounding of the running maximum is common to all probabilities, a score's own product is not rounded)
            float c2 = a.c, from = base;
            if (__any(fabsf(base) >= FAR)) { settle<4>(sc[0], c2, from); settle<4>(sc[1], c2, from); c2 = 1.f; from = 0.f; }
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i >> 2][i & 3], c2, -from));
            // Where a turn is masked at all its values are looked at: those that are no numbers leave the operands.
            if (masked) {
                const unsigned left = (unsigned)max(x1 - xb - g * 4, 0);       // keys that are there at all: before the end, on a page
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = see >> i & 1u ? p[i] : 0.f;
                    const unsigned there = (unsigned)((i >> 2) * 16 + (i & 3)) < left && !(gone >> i & 1u) ? 0xffffffffu : 0u;
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const unsigned w = vf[i][h] & there;
                        // the top bit of an element: all of its exponent's are set (an addition carries into it)
                        const unsigned bad = ((w & El<T>::ABS) + El<T>::STEP) & ~El<T>::ABS;
                        vf[i][h] = w & ~(E == 8 ? (bad - (bad >> 15)) | bad : (unsigned)((int)bad >> 31));
                        odd |= bad != 0u && nk > 0;                            // (a slice behind the head's end has loaded none)
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) l += p[i];
            if (nk <= 0) return;
            if constexpr (E == 8) {
                vec ph, pl;
#pragma unroll
                for (int i = 0; i < 8; ++i) { ph[i] = (T)p[i]; pl[i] = (T)(p[i] - (float)ph[i]); }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const vec vt = gather(vf, e, T());
                    acc[e] = El<T>::mfma(vt, ph, acc[e]);
                    acc[e] = El<T>::mfma(vt, pl, acc[e]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, vf[i])[e], p[i], acc[e], 0, 0, 0);
            }
        };
        // the slices' parts of a turn's scores, added up in the same order by all: their statistics are the same bit for bit
        auto add_slices = [&](f32x4 (&sc)[2], bool on) {
            if (on) {
                *reinterpret_cast<f32x4*>(sh.s[flip][wave][lane]) = sc[0];
                *reinterpret_cast<f32x4*>(sh.s[flip][wave][lane] + 4) = sc[1];
            }
            __syncthreads();
            if (on) {
                sc[0] = sc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < NC; ++u) {
                    sc[0] += *reinterpret_cast<const f32x4*>(sh.s[flip][kg * NC + u][lane]);
                    sc[1] += *reinterpret_cast<const f32x4*>(sh.s[flip][kg * NC + u][lane] + 4);
                }
            }
            flip ^= 1;
        };

        for (unsigned x0 = split * a.chunk; x0 < (unsigned)t.n; x0 += n_act * a.chunk) {
            const int x1 = (int)min(x0 + a.chunk, (unsigned)t.n);
            const int turns = (x1 - (int)x0 + KG * KB - 1) / (KG * KB);      // of every wave; the last may hold no keys for some
            if constexpr (ALIGNED) {
                u32x4 kf[2][NK], vf[8];
                unsigned pages = 0;              // lane 2 u + h: the page of half h of the u-th turn of 32
                // where half h of turn u begins (a half behind the last key: the last key's)
                auto half_at = [&](int u, int h) { return t.kb + min((int)x0 + (u * KG + kg) * KB + h * 16, (x1 - 1) & ~15); };
                int64_t row_at[2];               // the halves' first rows: of the turn whose keys, then whose values are asked for
                unsigned gone = 0u;
                auto find = [&](int u) {
                    if ((u & 31) == 0) pages = (unsigned)s.table[jb_div((unsigned)half_at(u + (lane >> 1), lane & 1), a.page)];
                    gone = 0u;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const unsigned pg = (unsigned)__builtin_amdgcn_readlane((int)pages, (u & 31) * 2 + h), at = (unsigned)half_at(u, h);
                        if (pg >= a.n_pages) gone |= 0xfu << (4 * h);
                        row_at[h] = (int64_t)(pg < a.n_pages ? pg : 0u) * a.page_stride + (int64_t)(at - jb_div(at, a.page) * a.page.d) * a.row_stride;
                    }
                };
                auto load_k = [&]() {
#pragma unroll
                    for (int ks = 0; ks < NK; ++ks)
                        if (NC == 1 || ks < nk) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) kf[h][ks] = load16((const char*)(kbase + row_at[h]) + koff[ks]);
                        }
                };
                auto load_v = [&]() {
                    if (NC == 1 || nk > 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) vf[i] = load16((const char*)(vbase + row_at[i >> 2]) + voff[i & 3]);
                    }
                };
                find(0);
                load_k();
                load_v();
                for (int u = 0; u < turns; ++u) {
                    const int xb = (int)x0 + (u * KG + kg) * KB;
                    const bool on = xb < x1;
                    f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
                    if (on) {
                        if (tail) clear_tail(kf);
#pragma unroll
                        for (int ks = 0; ks < NK; ++ks)
                            if (NC == 1 || ks < nk) {
#pragma unroll
                                for (int h = 0; h < 2; ++h) sc[h] = El<T>::mfma(__builtin_bit_cast(vec, kf[h][ks]), qf[ks], sc[h]);
                            }
                    }
                    // the next turn's keys take the registers of this one's, and are on their way while it goes on; its values later
                    // those of this one's
                    const unsigned lost = gone;
                    if (u + 1 < turns) { find(u + 1); load_k(); }
                    if constexpr (NC > 1) add_slices(sc, on);
                    if (on) turn(sc, vf, xb, x1, lost);
                    if (u + 1 < turns) load_v();
                }
            } else {
                int xb = (int)x0 + kg * KB;
                unsigned row = xb < x1 ? cache_row(a, s, t.kb + min(xb + (lane & 31), x1 - 1) * t.ks) : BAD;
                for (int u = 0; u < turns; ++u, xb += KG * KB) {
                    const bool on = xb < x1;     // the wave's turn has keys
                    f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
                    unsigned vrow[8], gone = 0u;
                    u32x4 vf[8];
                    if (on) {
                        u32x4 kf[2][NK];
                        const T* kp[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) kp[h] = kbase + cache_offset(a, __shfl(row, h * 16 + c));
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            vrow[i] = __shfl(row, (i >> 2) * 16 + g * 4 + (i & 3));
                            gone |= (vrow[i] == BAD ? 1u : 0u) << i;
                        }
#pragma unroll
                        for (int ks = 0; ks < NK; ++ks)
                            if (NC == 1 || ks < nk) {
#pragma unroll
                                for (int h = 0; h < 2; ++h) kf[h][ks] = load16(kp[h] + min(cb + ks * KT + g * E, D - E));
                            }
                        if (NC == 1 || nk > 0) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) vf[i] = load16(vbase + cache_offset(a, vrow[i]) + min(cb + c * E, D - E));
                        }
                        // the next turn's rows are looked up meanwhile
                        const int xn = xb + KG * KB;
                        if (xn < x1) row = cache_row(a, s, t.kb + min(xn + (lane & 31), x1 - 1) * t.ks);
                        if (tail) clear_tail(kf);
#pragma unroll
                        for (int ks = 0; ks < NK; ++ks)
                            if (NC == 1 || ks < nk) {
#pragma unroll
                                for (int h = 0; h < 2; ++h) sc[h] = El<T>::mfma(__builtin_bit_cast(vec, kf[h][ks]), qf[ks], sc[h]);
                            }
                    }
                    if constexpr (NC > 1) add_slices(sc, on);
                    if (on) turn(sc, vf, xb, x1, gone);
                }
            }
        }
        l = jb_rows_reduce(l, [](float u, float v) { return u + v; });

        // ---- the rows' states: joined over the waves side by side on the keys, written where they belong --------------------------
        float M = m, L = l, mine = 1.f;
        if constexpr (KG > 1) {
            __syncthreads();                      // the exchange of the previous tile has been read
            if (g == 0 && cb == 0) { sh.ml[kg][c][0] = m; sh.ml[kg][c][1] = l; }
            if (threadIdx.x == 0) sh.odd = 0;
            __syncthreads();
            M = -INFINITY; L = 0.f;
#pragma unroll
            for (int w = 0; w < KG; ++w) M = fmaxf(M, sh.ml[w][c][0]);
            const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < KG; ++w) L += sh.ml[w][c][1] * __builtin_amdgcn_exp2f(sh.ml[w][c][0] - base);
            mine = __builtin_amdgcn_exp2f(m - base);
        }
        const bool counts = row_ok && L > 0.f;    // (a sum that is no number, of the scores, has outputs that are none)
        float zero = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) zero = fmaf(acc[e][r], 0.f, zero);         // or no number
        odd |= counts && zero != 0.f;
        if constexpr (KG > 1) { if (odd) sh.odd = 1; }
        else odd = __syncthreads_or(odd);
        // a state of several is joined with the others' by its own maximum and sum; nothing seen: zeros
        mine *= n_act > 1 ? 1.f : L != 0.f ? 1.f / L : 0.f;
        if (n_act > 1 && wave == 0 && g == 0 && row_ok) {
            float* o = a.ml + (((int64_t)(s.t0 + j) * a.n_head + head) * a.splits + split) * 2;
            o[0] = M; o[1] = L;
        }
        auto put = [&](int64_t tok, int h, int at, const float* v) {
            if (n_act > 1) {
                float* o = a.part + (((tok * a.n_head + h) * a.splits + split) * (int64_t)D + at);
                *reinterpret_cast<u32x4_any*>(o) = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
                if constexpr (E == 8) *reinterpret_cast<u32x4_any*>(o + 4) = __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]});
            } else {
                T* o = (T*)a.out + tok * a.o_row + (int64_t)h * a.o_head + at;
                if constexpr (E == 8) store8<T>(o, v);
                else *reinterpret_cast<u32x4_any*>(o) = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
            }
        };
        // a lane holds pieces g * 4 + r of its row: piece m's channels are min(cb + m * E, D - E) + e
        if constexpr (KG == 1) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v[8];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = acc[e][r] * mine;
                const int d0 = cb + (g * 4 + r) * E;
                if (row_ok && d0 < D) put(s.t0 + j, head, min(d0, D - E), v);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<f32x4*>(&sh.o[wave][c][(g * 4 + r) * E + e]) = f32x4{acc[e][r], acc[e + 1][r], acc[e + 2][r], acc[e + 3][r]} * mine;
            __syncthreads();
            odd = __builtin_amdgcn_readfirstlane(sh.odd);
            const int wr = threadIdx.x >> 4, wc = threadIdx.x & 15, wR = min(t.row0 + wr, t.rows - 1), wi = (int)jb_div(wR, a.group);
#pragma unroll
            for (int u = 0; u < NC; ++u) {
                const int d0 = u * CH + wc * E;
                float v[8];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    v[e] = 0.f;
#pragma unroll
                    for (int w = 0; w < KG; ++w) v[e] += sh.o[w * NC + u][wr][wc * E + e];
                }
                if (t.row0 + wr < t.rows && d0 < D) put(s.t0 + t.j0 + wi * t.js, kvh * a.G + (wR - wi * a.G), min(d0, D - E), v);
            }
        }
        if (odd) {
            __syncthreads();
            put_infinities<T>(a, s, t, kvh, split, n_act, t.row0, ~(unsigned)__ballot(counts), wave, Sh::WAVES);
        }
    }
}

// Chunks: one workgroup of four waves per (sequence, kv head, tile of 128 rows, split of the keys), a wave 32 rows.
//
// The same two products on 32 x 32 x 16 matrix instructions: S^T = K Q^T leaves a lane the scores of 16 of 32 keys for row l & 31, which
// are the B operand of O^T += V^T P^T once slot (h, i) of a k-step s is key 16 s + 8 (i / 4) + 4 h + i % 4.  64 keys at a time go through LDS
// (32 under heads of 129-160 channels, so that two workgroups of them fit a compute unit: 4 x 2048 queries 652 us against 858),
// two buffers, one barrier a turn: half the waves bring the keys' rows, the others the values', transposed on the way by byte
// permutations ([channel][key], so that an operand is one 16-byte read), all asked for a turn ahead.  LDS rows are padded by 16 bytes: the
// 16 lanes of a read phase then hit 16 different groups of four banks.
// The probabilities enter the second product rounded once to 16 bits, which adds an error of the size of the output's own
// rounding (each is off by half a step, and they average); a second product for the rest took 864 us for 707 of the second case below.
// Measured (32 heads on 8 of 128 channels, bf16, pages of 64; the library's product of 16384^3 runs at 1370 TFLOP/s): 4 x 2048 queries behind
// 6144 keys: 1.20-1.26 ms, 760-800 TFLOP/s; 4 x 257-2048 behind 4097-8192: 690-760 us from card to card, 620-690 TFLOP/s; 8 heads of 150, f16,
// 100-1000 queries behind 1000-5000: 118 us, 247 TFLOP/s; 2 heads of 256, f16, 4 x 512-2048 behind 4096-6144: 250 us, 200 TFLOP/s.  Two workgroups
// share a compute unit (one under 256 channels).  By the counters of the second case the matrix units are busy 27 % of the time, the vector
// ALU issues -- the softmax's exponentials, most of all -- 39 %, the LDS is read 24 %: two waves a SIMD overlap little of them, and the
// registers hold no third.  Waves of 64 rows, which halve the LDS reads but leave one wave a SIMD (and its registers spilling): 1.13 ms
// instead of 0.83 for the second case as things then were.
template <typename T> struct Mfma32;
template <> struct Mfma32<f16> { static __device__ __forceinline__ f32x16 go(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); } };
template <> struct Mfma32<bf16> { static __device__ __forceinline__ f32x16 go(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); } };

template <int DP> struct ChunkLds {                                       // bytes
    static constexpr int KT = DP == 160 ? 32 : 64;                        // keys of a turn
    static constexpr int KROW = DP * 2 + 16, VROW = KT * 2 + 16, K = KT * KROW, V = DP * VROW, BUF = K + V;
    static constexpr int OFF = 2 * BUF, ODD = OFF + 3 * KT * 8, GAP = ODD + 4, ALL = GAP + 3 * 4;
};
__device__ __forceinline__ float swap_halves_max(float x) {              // the larger of lanes l and l ^ 32, in both
    float a = x, b = x;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    return fmaxf(a, b);
}

template <typename T, int DP>
__global__ __launch_bounds__(256, (DP <= 160 ? 2 : 1)) void attn_paged_chunk_kernel(const Args a) {
    typedef typename El<T>::vec vec;
    typedef ChunkLds<DP> L;
    constexpr int KT = L::KT, NKS = DP / 16, NDT = DP / 32, PIECES = DP / 8, LPR = PIECES < 16 ? PIECES : 1024 / KT, SETS = (PIECES + LPR - 1) / LPR, OCT = KT / 8;
    constexpr int CREW = PIECES > 8 ? 2 : 1;      // waves that bring the keys' rows, and as many the values': eight pieces a lane and set
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // of the turn computed, the one asked for and the one looked up:
    int64_t* const s_off = reinterpret_cast<int64_t*>(lds + L::OFF);    // [3][KT]: a key's offset in the pool, -1: nowhere
    int* const s_gap = reinterpret_cast<int*>(lds + L::GAP);            // [3]: whether a key is on no page
    int* const s_odd = reinterpret_cast<int*>(lds + L::ODD);            // whether values have been met that are no numbers
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tile0, split, kvh, si;
    if (!place_of(a, blockIdx.x, tile0, split, kvh, si)) return;
    const Seq s = seq_of(a, si);
    const int n_tiles = tiles_of(a, s.nq), D = a.D, NP = (D + 7) / 8;
    const T* kbase = (const T*)a.k + (int64_t)kvh * a.head_stride;
    const T* vbase = (const T*)a.v + (int64_t)kvh * a.head_stride;
    // pieces behind the head's end are zeros throughout (the queries' are too, but 0 * NaN is not)
    if (NP < PIECES)
        for (int i = threadIdx.x; i < 2 * KT * (PIECES - NP); i += 256) {
            const int row = i / (PIECES - NP), pc = NP + i % (PIECES - NP);
            *reinterpret_cast<u32x4*>(lds + row / KT * L::BUF + row % KT * L::KROW + pc * 16) = u32x4{0, 0, 0, 0};
        }

    for (int tile = tile0; tile < n_tiles; tile += a.tiles) {
        const Tile t = tile_of(a, s, tile);
        if (t.row0 >= t.rows) continue;
        const int n_act = active_splits(a, t.n);
        if (split >= n_act) continue;
        auto pos_of = [&](int R) { return s.pos0 + (int)jb_div(R, a.group); };
        auto walk = [&](int p, int& first, int& end) {
            int lo, hi;
            sees(a, p, lo, hi);
            first = max(lo - t.kb, 0); end = max(hi - t.kb, 0);
        };
        vec qf[NKS];
        const int R0 = t.row0 + wave * 32, R = R0 + c, my = min(R, t.rows - 1);
        const int qi = (int)jb_div(my, a.group), head = kvh * a.G + my - qi * a.G;
        const T* qrow = (const T*)a.q + (int64_t)(s.t0 + qi) * a.q_row + (int64_t)head * a.q_head;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int e0 = (ks * 2 + h) * 8, at = min(e0, D - 8);
            vec x = __builtin_bit_cast(vec, load16(qrow + at));
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at + e < e0 || R >= t.rows) x[e] = (T)0.f;
            if (a.c < 0.f) x = -x;                // (the softmax below takes a scale that is not negative)
            qf[ks] = x;
        }
        if (NP * 8 > D) {
            // the channels that the last piece has over again are halved in both: with 0 in one, an infinite key would be 0 * inf there
            vec prev = __builtin_bit_cast(vec, load16(qrow + max(NP * 8 - 16, 0))), last = __builtin_bit_cast(vec, load16(qrow + D - 8));
            const int again = NP * 8 - D;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = a.c < 0.f ? -(float)last[e] : (float)last[e], w = a.c < 0.f ? -(float)prev[e] : (float)prev[e];
                last[e] = (T)(e < again ? v - half_of<T>(v) : v);
                prev[e] = (T)(e >= 8 - again ? half_of<T>(w) : w);
            }
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                if (R < t.rows && ks * 2 + h == NP - 1) qf[ks] = last;
                if (R < t.rows && ks * 2 + h == NP - 2) qf[ks] = prev;
            }
        }
        // the walked keys that the lane's row sees; those that all of the wave's rows see, and any of them (a wave without rows: none)
        int xlo, xhi, all_lo = 0x7fffffff, all_hi = 0, any_lo = 0x7fffffff, any_hi = 0;
        walk(s.pos0 + qi, xlo, xhi);
        if (R >= t.rows || xhi < xlo) xlo = xhi = 0;
        if (R0 < t.rows) {
            walk(pos_of(R0), any_lo, all_hi);
            walk(pos_of(min(R0 + 31, t.rows - 1)), all_lo, any_hi);
        }
        // what every row of the workgroup sees: outside it the values are looked at on their way to LDS
        int wg_lo, wg_hi, unused;
        walk(pos_of(t.row0), unused, wg_hi);
        walk(pos_of(min(t.row0 + a.tr, t.rows) - 1), wg_lo, unused);

        f32x16 acc[NDT];
        float m = -INFINITY, l = 0.f;            // of the lane's row: the reference the same in both its lanes, the sum a part in each
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;

        __syncthreads();
        if (threadIdx.x == 0) *s_odd = 0;
        for (unsigned x0 = split * a.chunk; x0 < (unsigned)t.n; x0 += n_act * a.chunk) {
            const int x1 = (int)min(x0 + a.chunk, (unsigned)t.n), turns = (x1 - (int)x0 + KT - 1) / KT;
            // the first wave: where the keys of turn u are -- their pages asked for early in a turn, used at its end
            auto page_number = [&](int u) { return (unsigned)s.table[jb_div((unsigned)(t.kb + min((int)x0 + u * KT + lane % KT, x1 - 1)), a.page)]; };
            auto look_up = [&](int u, unsigned pg) {
                const int x = (int)x0 + u * KT + lane % KT;
                const unsigned at = (unsigned)(t.kb + min(x, x1 - 1)), in_page = at - jb_div(at, a.page) * a.page.d;
                s_off[u % 3 * KT + lane % KT] = x < x1 && pg < a.n_pages ? (int64_t)pg * a.page_stride + (int64_t)in_page * a.row_stride : -1;
                const bool gap = __any(x < x1 && pg >= a.n_pages);
                if (lane == 0) s_gap[u % 3] = gap;
            };
            // What a lane brings of a turn: of the keys piece `piece` of every eighth row, of the values that piece of the eight keys of an
            // operand.  One sequence of loads for both (a branch around them would have to wait for them at its end).
            u32x4 hold[8 * SETS];
            const bool values = wave >= CREW, works = CREW == 2 || wave < 2;
            const int in_crew = (wave % CREW) * 64 + lane, piece = values ? lane / OCT + 64 / OCT * (wave % CREW) : in_crew % LPR;
            const int key0 = values ? (lane % OCT >> 1) * 16 + (lane & 1) * 4 : in_crew / LPR;
            auto key_of = [&](int q) { return key0 + (values ? (q >> 2) * 8 + (q & 3) : q * OCT); };
            auto ask = [&](int u) {               // turn u's rows into registers (of a key that is none any row will do)
                const int64_t* off = s_off + u % 3 * KT;
                const T* base = values ? vbase : kbase;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const T* row = base + max(off[key_of(q)], (int64_t)0);
#pragma unroll
                    for (int st = 0; st < SETS; ++st) hold[st * 8 + q] = load16(row + min((piece + LPR * st) * 8, D - 8));
                }
            };
            auto put = [&](int u) {               // and from there to LDS
                char* buf = lds + (u & 1) * L::BUF;
                if (!values) {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
#pragma unroll
                        for (int st = 0; st < SETS; ++st)
                            if (piece + LPR * st < NP) *reinterpret_cast<u32x4*>(buf + (key0 + q * OCT) * L::KROW + (piece + LPR * st) * 16) = hold[st * 8 + q];
                } else {
                    const int xb = (int)x0 + u * KT;
                    const bool look = xb < wg_lo || xb + KT > min(wg_hi, x1) || __builtin_amdgcn_readfirstlane(s_gap[u % 3]);
                    if (look) {
                        unsigned odd = 0u;
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const bool none = s_off[u % 3 * KT + key_of(q)] < 0;
#pragma unroll
                            for (int st = 0; st < SETS; ++st)
#pragma unroll
                                for (int d = 0; d < 4; ++d) {
                                    const unsigned w = none ? 0u : hold[st * 8 + q][d], bad = ((w & El<T>::ABS) + El<T>::STEP) & ~El<T>::ABS;
                                    hold[st * 8 + q][d] = w & ~((bad - (bad >> 15)) | bad);
                                    odd |= bad;
                                }
                        }
                        if (odd) *s_odd = 1;
                    }
#pragma unroll
                    for (int st = 0; st < SETS; ++st)
                        if (piece + LPR * st < PIECES) {
                            const u32x4 w[8] = {hold[st * 8], hold[st * 8 + 1], hold[st * 8 + 2], hold[st * 8 + 3], hold[st * 8 + 4], hold[st * 8 + 5], hold[st * 8 + 6], hold[st * 8 + 7]};
                            char* at = buf + L::K + (piece + LPR * st) * 8 * L::VROW + lane % OCT * 16;
#pragma unroll
                            for (int e = 0; e < 8; ++e) *reinterpret_cast<u32x4*>(at + e * L::VROW) = __builtin_bit_cast(u32x4, gather(w, e, f16()));
                        }
                }
            };

            __syncthreads();                      // the buffers of the turns before are free
            if (wave == 0) { look_up(0, page_number(0)); if (turns > 1) look_up(1, page_number(1)); }
            __syncthreads();
            if (works) { ask(0); put(0); }
            __syncthreads();
            for (int u = 0; u < turns; ++u) {
                const bool more = u + 1 < turns;
                // (unconditionally, the last turn's over again at the end: see hold)
                if (works) ask(min(u + 1, turns - 1));
                const unsigned pg = page_number(u + 2);
                const char* buf = lds + (u & 1) * L::BUF;
                const int64_t* off = s_off + u % 3 * KT + h * 4;
                const bool gap = __builtin_amdgcn_readfirstlane(s_gap[u % 3]);
#pragma unroll
                for (int sub = 0; sub < KT / 32; ++sub) {
                    const int xb = (int)x0 + u * KT + sub * 32;
                    if (xb >= min(any_hi, x1) || xb + 32 <= any_lo) continue;         // none of the wave's rows sees any of them
                    f32x16 sc;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
                    for (int ks = 0; ks < NKS; ++ks)
                        sc = Mfma32<T>::go(*reinterpret_cast<const vec*>(buf + (sub * 32 + c) * L::KROW + (ks * 2 + h) * 16), qf[ks], sc);
                    if (xb + 32 > x1 || xb < all_lo || xb + 32 > all_hi || gap) {
                        const int end = min(xhi, x1);
                        const unsigned d0 = (unsigned)(xb + h * 4 - xlo), dn = (unsigned)(end > xlo ? end - xlo : 0);
#pragma unroll
                        for (int r = 0; r < 16; ++r) sc[r] = d0 + (r >> 2) * 8 + (r & 3) < dn ? sc[r] : -INFINITY;
                        if (gap) {                // positions on no page are seen by nobody
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (off[sub * 32 + (r >> 2) * 8 + (r & 3)] < 0) sc[r] = -INFINITY;
                        }
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[r]);
                    const float m_new = fmaxf(m, reference_of<T>(swap_halves_max(mx) * a.c_abs)), base = m_new == -INFINITY ? 0.f : m_new;
                    if (__any(m_new != m)) {
                        const float alpha = __builtin_amdgcn_exp2f(m - base);
                        l *= alpha;
#pragma unroll
                        for (int dt = 0; dt < NDT; ++dt) acc[dt] *= alpha;
                        m = m_new;
                    }
                    float c2 = a.c_abs, from = base;
                    if (__any(fabsf(base) >= FAR)) { settle<16>(sc, c2, from); c2 = 1.f; from = 0.f; }
                    vec pf[2];
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(sc[r], c2, -from));
                        l += p;
                        pf[r >> 3][r & 7] = (T)p;
                    }
#pragma unroll
                    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                        for (int dt = 0; dt < NDT; ++dt) {
                            const vec vt = *reinterpret_cast<const vec*>(buf + L::K + (dt * 32 + c) * L::VROW + ((sub * 2 + s2) * 2 + h) * 16);
                            acc[dt] = Mfma32<T>::go(vt, pf[s2], acc[dt]);
                        }
                }
                if (works && more) put(u + 1);    // into the buffer of the turn before
                if (wave == 0 && u + 2 < turns) look_up(u + 2, pg);
                __syncthreads();
            }
        }

        // ---- states out ---------------------------------------------------------------------------------------------------------
        const int64_t tok = s.t0 + qi;
        const float sum = l + __shfl_xor(l, 32);
        const float mine = n_act > 1 ? 1.f : sum != 0.f ? 1.f / sum : 0.f;
        const bool counts = R < t.rows && sum > 0.f;         // (a sum that is no number, of the scores, has outputs that are none)
        float zero[4] = {0.f, 0.f, 0.f, 0.f};     // or no numbers
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) zero[r & 3] = fmaf(acc[dt][r], 0.f, zero[r & 3]);
        const bool odd = __builtin_amdgcn_readfirstlane(*s_odd) || __any(counts && (zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.f);
        if (R < t.rows) {
            if (n_act > 1 && h == 0) {
                float* o = a.ml + ((tok * a.n_head + head) * a.splits + split) * 2;
                o[0] = m; o[1] = sum;
            }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int pc = dt * 4 + r4;
                    if (pc >= NP) continue;
                    const int at = min(pc * 8, D - 8) + h * 4;
                    if (n_act > 1) {
                        float* o = a.part + (((tok * a.n_head + head) * a.splits + split) * (int64_t)D + at);
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[k] = acc[dt][r4 * 4 + k];
                    } else {
                        T* o = (T*)a.out + tok * a.o_row + (int64_t)head * a.o_head + at;
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[k] = (T)(acc[dt][r4 * 4 + k] * mine);
                    }
                }
        }
        if (__builtin_expect(odd, 0)) {
            __threadfence_block();                // (the rows' other outputs are written)
            const unsigned skip = ~(unsigned)__ballot(counts);
            for (int half = 0; half < 2; ++half) put_infinities<T>(a, s, t, kvh, split, n_act, R0 + half * 16, skip >> (half * 16), 0, 1);
        }
    }
}

// Joins the splits' states of rows that were split: a wave 64 channels of a row of a tile, four a lane, a quarter of the splits each
// sixteen lanes; their weights one a lane.  (A wave a row left 16 waves to read 32 states of 480 channels: 19 us, now 5.)
// U: fours of splits at most; ROWS: rows whose states are asked for together (four: the 150-channel chunks 120 -> 116 us in all).
template <typename T, int U, int ROWS>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(const Args a, int tile_rows) {
    int64_t b = blockIdx.x;
    const int fours = (tile_rows + 3) / 4, wr = (int)(b % fours) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); b /= fours;
    if (wr >= tile_rows) return;
    const int tile0 = (int)(b % a.tiles); b /= a.tiles;
    const int kvh = (int)(b % a.n_kv), si = (int)(b / a.n_kv), lane = threadIdx.x & 63, part_of = lane >> 4;
    const Seq s = seq_of(a, si);
    const int n_tiles = tiles_of(a, s.nq), d0 = blockIdx.y * 64 + (lane & 15) * 4, d = min(d0, a.D - 4);     // (a last piece begins four before the end)
    for (int tile = tile0; tile < n_tiles; tile += a.tiles) {
        const Tile t = tile_of(a, s, tile);
        const int n_act = active_splits(a, t.n);
        if (n_act < 2) continue;
        const int end = min(t.row0 + a.tr, t.rows);
        for (int R0 = t.row0 + wr; R0 < end; R0 += tile_rows * ROWS) {
            f32x4 v[ROWS][U];
            float m[ROWS], l[ROWS];
            int64_t to[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const int R = min(R0 + r * tile_rows, end - 1), i = (int)jb_div(R, a.group), h = kvh * a.G + (R - i * a.G);
                const int64_t tok = s.t0 + t.j0 + i * t.js, state = (tok * a.n_head + h) * a.splits;
                const float *ml = a.ml + state * 2, *part = a.part + state * (int64_t)a.D + d;
                to[r] = tok * a.o_row + (int64_t)h * a.o_head + d;
                m[r] = lane < n_act ? ml[2 * lane] : -INFINITY;
                l[r] = lane < n_act ? ml[2 * lane + 1] : 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u * 4 < n_act) v[r][u] = __builtin_bit_cast(f32x4, *reinterpret_cast<const u32x4_any*>(part + (int64_t)min(u * 4 + part_of, n_act - 1) * a.D));
            }
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (R0 + r * tile_rows >= end) break;
                const float M = jb_wave_max(m[r]), base = M == -INFINITY ? 0.f : M, e = __builtin_amdgcn_exp2f(m[r] - base), L = jb_wave_sum(l[r] * e);
                const float w = L != 0.f ? e / L : 0.f;
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (u * 4 < n_act) {
                        const float wu = __shfl(w, u * 4 + part_of);
                        if (wu != 0.f) o += v[r][u] * wu;                // (a lane behind the last split weighs nothing)
                        else if (u * 4 + part_of < n_act)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[k] += fabsf(v[r][u][k]) < INFINITY ? 0.f : v[r][u][k];      // infinite all the same
                    }
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = jb_rows_reduce(o[k], [](float x, float y) { return x + y; });
                if (part_of == 0 && d0 < a.D) {
                    T* q = (T*)a.out + to[r];
#pragma unroll
                    for (int k = 0; k < 4; ++k) q[k] = (T)o[k];
                }
            }
        }
    }
}

struct Plan { int64_t tiles, range; int tr, splits; unsigned chunk; };       // tr: rows of a tile, 16 the rows kernel's, 128 the chunks'
Plan plan_of(const jb_attn_paged_args* p) {
    Plan w;
    const int64_t G = p->n_head / p->n_kv_head, bc = p->block_ctx, rows = p->max_q * G, streams = (int64_t)p->n_kv_head * p->n_seq;
    w.tr = 16;
    if (p->dtype != JB_F32 && p->attn_func != JB_ATTN_TRANSPOSE_BLOCK && p->d_head <= 256 && rows >= 64)
        w.tr = 128;
    if (p->attn_func == JB_ATTN_TRANSPOSE_BLOCK) w.tiles = (int64_t)(p->max_q < bc ? p->max_q : bc) * (((p->max_q + bc - 1) / bc * G + 15) / 16);
    else w.tiles = (rows + w.tr - 1) / w.tr;
    // 2^20 workgroups fill the chip many times over, and a launch holds 2^32 threads: what max_q asks for beyond is walked by the tiles there are
    const int64_t most_tiles = streams < 1 << 20 ? (1 << 20) / streams : 1;
    if (w.tiles > most_tiles) w.tiles = most_tiles;
    // keys that a tile walks at most
    w.range = p->max_len;
    if (p->attn_func == JB_ATTN_BLOCK || p->attn_func == JB_ATTN_PREV_BLOCK) w.range = bc + w.tr / G + 15;
    else if (p->attn_func == JB_ATTN_TRANSPOSE_BLOCK) w.range = (p->max_len + bc - 1) / bc;
    else if (p->window) w.range = (int64_t)p->window + w.tr / G + 15;
    if (w.range > p->max_len) w.range = p->max_len;
    const int64_t wgs = w.tiles * streams;
    w.splits = 1; w.chunk = 0x7fffffff;
    int64_t chunk = 0;
    // Few tiles: the keys are split, so that every compute unit has two workgroups.  A workgroup costs some 5 us before its first keys
    // are there, so its turn is 256 keys at least (16 sequences of 4096-8192 keys under one head of 480: 39 us; 512 keys: 43, 128: 45) -- a
    // launch too small to fill the chip even so takes 64 (300 keys: 17 us against 27) -- and 2048 at most, which evens out
    // sequences of different lengths (64 of 511-8192 keys: 260 us against 266 unsplit).
    if (w.tr == 16 && wgs < 1024 && w.range > 64) {
        chunk = (wgs * w.range / 512 + 127) / 128 * 128;
        if (chunk > 2048) chunk = 2048;
        if (chunk < 256) chunk = wgs * w.range <= 64 * 256 ? 64 : 256;
    }
    // Chunks: two workgroups a compute unit as well, by the tiles that there can be in all (sequences are rarely as long as the longest:
    // 3 of 100-1000 queries, 5000 keys under 8 heads of 150: 118 us, split for as many tiles as the launch has 168; 1000 queries of one
    // sequence: 80 us; three or four workgroups a unit: 103; one and a half: 95), and 512 keys at least.
    const int64_t filled = (p->n_tokens * G + w.tr - 1) / w.tr + p->n_seq / 2, real = filled * p->n_kv_head < wgs ? filled * p->n_kv_head : wgs;
    if (w.tr > 16 && real < 1024 && w.range > 512) {
        chunk = (real * w.range / 512 + 127) / 128 * 128;
        if (chunk < 512) chunk = 512;
    }
    if (chunk) {
        // the join holds 64 states; a batch padded far beyond its sequences' rows gets fewer, so that 1 GiB holds them
        const int64_t fit = (1ll << 30) / ((int64_t)p->n_tokens * p->n_head * (p->d_head + 2) * 4), most = fit < 1 ? 1 : fit < 64 ? fit : 64;
        if ((w.range + chunk - 1) / chunk > most) chunk = ((w.range + most - 1) / most + 127) / 128 * 128;
        if (w.range > chunk) { w.splits = (int)((w.range + chunk - 1) / chunk); w.chunk = (unsigned)chunk; }
    }
    return w;
}
int64_t workspace_of(const jb_attn_paged_args* p, const Plan& w) {
    return w.splits == 1 ? 0 : (int64_t)p->n_tokens * p->n_head * w.splits * (p->d_head + 2) * 4;
}

int shift_of(int page_size) {                     // ceil(log2 page_size)
    int s = 0;
    while (s < 31 && (1u << s) < (unsigned)page_size) ++s;
    return s;
}
int check_args(const jb_attn_paged_args* a, const char* who) {
    auto bad = [&](const char* what) { jb_set_error(std::string(who) + ": " + what); return (int)JB_ERR_ARG; };
    if (!a) return bad("null pointer");
    if (a->dtype != JB_F32 && a->dtype != JB_F16 && a->dtype != JB_BF16) return bad("bad dtype");
    if (a->attn_func < JB_ATTN_DENSE || a->attn_func > JB_ATTN_PREV_BLOCK) {
        jb_set_error(std::string(who) + ": pages hold the keys of dense, block, transpose and prev layers");
        return JB_ERR_UNSUPPORTED;
    }
    if (a->n_tokens < 0 || a->n_seq < 0 || a->n_head <= 0 || a->n_kv_head <= 0 || a->n_head % a->n_kv_head) return bad("bad dims");
    if (a->d_head < 8 || a->d_head > 512) { jb_set_error(std::string(who) + ": heads of 8 to 512 channels"); return JB_ERR_UNSUPPORTED; }
    if (a->n_pages <= 0 || a->page_size <= 0 || a->max_pages <= 0) return bad("bad dims of the cache");
    if (((uint64_t)a->n_pages << shift_of(a->page_size)) > 0xffffffffull || (int64_t)a->n_pages * a->page_size > 0x7fffffff) return bad("more than 2^31 cache rows");
    if (a->page_stride < 0 || a->row_stride < 0 || a->head_stride < 0 || a->q_row_stride < 0 || a->q_head_stride < 0 || a->table_stride < 0) return bad("negative stride");
    if (a->out_head_stride < a->d_head || a->out_row_stride < a->d_head ||
        !jb_apart(a->d_head, a->n_tokens, a->out_row_stride, a->n_head, a->out_head_stride)) return bad("output rows overlap");
    if (a->attn_func != JB_ATTN_DENSE && a->block_ctx <= 0) return bad("block_ctx required");
    if (a->window < 0 || (a->window && a->attn_func != JB_ATTN_DENSE)) return bad("a window goes with the dense pattern");
    if (a->max_q < 0 || a->max_len < 0 || (int64_t)a->max_q * a->n_head > 0x7fffffff || (int64_t)a->n_tokens * a->n_head > 0x7fffffff) return bad("bad dims");
    return JB_OK;
}

template <typename T, int NC> void launch_rows(const Args& k, int64_t wgs, hipStream_t s) {
    if (k.aligned) attn_paged_rows_kernel<T, NC, true><<<(unsigned)wgs, Shape<T, NC>::WAVES * 64, 0, s>>>(k);
    else attn_paged_rows_kernel<T, NC, false><<<(unsigned)wgs, Shape<T, NC>::WAVES * 64, 0, s>>>(k);
}

template <typename T, int DP> int launch_chunk_of(const Args& k, int64_t wgs, hipStream_t s) {
    constexpr int bytes = ChunkLds<DP>::ALL;
    static bool configured[64] = {};                  // per device (a call that is made twice does no harm)
    int dev = 0;
    JB_HIP(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        JB_HIP(hipFuncSetAttribute((const void*)attn_paged_chunk_kernel<T, DP>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    attn_paged_chunk_kernel<T, DP><<<(unsigned)wgs, 256, bytes, s>>>(k);
    return JB_OK;
}
template <typename T> int launch_chunk(const Args& k, int64_t wgs, hipStream_t s) {
    return k.D <= 64 ? launch_chunk_of<T, 64>(k, wgs, s) : k.D <= 128 ? launch_chunk_of<T, 128>(k, wgs, s)
           : k.D <= 160 ? launch_chunk_of<T, 160>(k, wgs, s) : launch_chunk_of<T, 256>(k, wgs, s);
}
template <> int launch_chunk<float>(const Args&, int64_t, hipStream_t) { return JB_ERR_UNSUPPORTED; }        // (never asked for: plan_of)

}  // namespace

extern "C" int64_t jb_attn_paged_workspace(const jb_attn_paged_args* a) {
    const int rc = check_args(a, __func__);
    if (rc) return rc;
    if (a->n_tokens == 0 || a->n_seq == 0 || a->max_q == 0) return 0;
    return workspace_of(a, plan_of(a));
}

extern "C" int jb_attn_paged(const jb_attn_paged_args* a, void* stream) {
    const int rc = check_args(a, __func__);
    if (rc) return rc;
    if (a->n_tokens == 0 || a->n_seq == 0 || a->max_q == 0) return JB_OK;
    JB_REQUIRE(a->q && a->k && a->v && a->out && a->table && a->lens && a->cu_q, "null pointer");
    const Plan w = plan_of(a);
    const int64_t need = workspace_of(a, w);
    JB_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need && (uintptr_t)a->workspace % 16 == 0), "workspace missing, too small or not aligned");
    const int64_t wgs = w.tiles * a->n_kv_head * a->n_seq;
    constexpr int64_t MOST = 0xffffffffll / 512;       // workgroups of up to 512 threads that a launch holds
    JB_REQUIRE(wgs * w.splits <= MOST, "grid too large");
    Args k = {};
    k.q = a->q; k.q_row = a->q_row_stride; k.q_head = a->q_head_stride;
    k.out = a->out; k.o_row = a->out_row_stride; k.o_head = a->out_head_stride;
    k.k = a->k; k.v = a->v; k.page_stride = a->page_stride; k.row_stride = a->row_stride; k.head_stride = a->head_stride;
    k.table = a->table; k.table_stride = a->table_stride; k.max_pages = a->max_pages;
    k.lens = a->lens; k.cu = a->cu_q;
    k.page = jb_make_div((unsigned)a->page_size);
    k.group = jb_make_div((unsigned)(a->n_head / a->n_kv_head));
    k.n_pages = (unsigned)a->n_pages;
    k.page_shift = shift_of(a->page_size);
    k.n_tokens = a->n_tokens; k.n_seq = a->n_seq; k.n_head = a->n_head; k.n_kv = a->n_kv_head; k.G = a->n_head / a->n_kv_head; k.D = a->d_head;
    k.func = a->attn_func; k.bc = a->block_ctx > 0 ? a->block_ctx : 1; k.window = a->window;
    k.tr = w.tr; k.tiles = (int)w.tiles; k.splits = w.splits; k.chunk = w.chunk;
    k.c = a->scale * 1.44269504088896340736f;
    k.c_abs = fmaxf(fabsf(k.c), 1e-30f);
    // (a lane's offset inside a 16-row half is 32 bits wide)
    k.aligned = w.tr == 16 && a->page_size % 16 == 0 && a->attn_func != JB_ATTN_TRANSPOSE_BLOCK && a->row_stride <= 0x7fffffff / 64 - 512;
    const int64_t inner = w.tiles == 1 ? k.n_kv : w.tiles, groups = wgs * w.splits / inner;
    JB_REQUIRE((groups + 8) * inner <= MOST, "grid too large");
    k.groups = (unsigned)groups; k.by_die = w.tiles == 1 ? groups >= 8 : k.n_kv % 8 == 0;
    const int64_t grid = k.by_die ? (groups + 7) / 8 * 8 * inner : groups * inner;
    if (need) {
        k.part = (float*)a->workspace;
        k.ml = k.part + (int64_t)a->n_tokens * a->n_head * w.splits * a->d_head;
    }
    hipStream_t s = (hipStream_t)stream;
    const int64_t most_rows = (int64_t)a->max_q * k.G;
    // waves that join a tile: 16, each several rows of a chunk (24 tiles under 8 heads, 5 states: 122 us in all; 64 waves, whose beginnings cost
    // as much as a row, 131) -- more where tiles are so few that the waves find room at once (8 tiles, 59 states: 61 -> 51)
    const int64_t room = wgs < 64 ? 1024 / wgs : 16, side = w.tr == 16 ? 16 : room < 128 ? room : 128;
    const int tile_rows = (int)(most_rows < side ? most_rows : side);
    JB_REQUIRE(w.splits == 1 || wgs * ((tile_rows + 3) / 4) <= MOST, "grid too large");
#define JB_ROWS(T, CH)                                                            \
    do {                                                                          \
        if (w.tr > 16) { const int rc2 = launch_chunk<T>(k, grid, s); if (rc2) return rc2; } \
        else if (a->d_head <= 128) launch_rows<T, 128 / CH>(k, grid, s);               \
        else if (a->d_head <= 256) launch_rows<T, 256 / CH>(k, grid, s);          \
        else launch_rows<T, 512 / CH>(k, grid, s);                                \
        JB_CHECK_LAUNCH();                                                        \
        if (w.splits > 1) {                                                       \
            const dim3 g((unsigned)(wgs * ((tile_rows + 3) / 4)), (unsigned)((a->d_head + 63) / 64)); \
            if (w.splits <= 16) attn_paged_join_kernel<T, 4, 4><<<g, 256, 0, s>>>(k, tile_rows); \
            else attn_paged_join_kernel<T, 16, 1><<<g, 256, 0, s>>>(k, tile_rows); \
        }                                                                         \
    } while (0)
    if (a->dtype == JB_F16) JB_ROWS(f16, 128);
    else if (a->dtype == JB_BF16) JB_ROWS(bf16, 128);
    else JB_ROWS(float, 64);
#undef JB_ROWS
    JB_CHECK_LAUNCH();
    return JB_OK;
}

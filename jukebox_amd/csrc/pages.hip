// The pages of a cache: rows written into them, and the control of who holds which (include/jukebox_hip.h).
//
// Nothing here computes: what counts is how few launches and passes the control takes, and that copies keep enough requests in
// flight.  Free pages are those with ref == 0 and are given out from the lowest number on, so that what a call does depends on its
// arguments alone -- not on the order in which workgroups arrive, nor on a list that grew with the history of the cache.  The scan
// this takes is n_pages words by one workgroup (65536 pages: 256 KB), ended as soon as enough pages are found.
#include "paged.h"

namespace {

constexpr int NT = 1024;                              // threads of the planning workgroup
constexpr int MAX_POOLS = 256;                        // pools of one launch: their addresses travel in the kernel's arguments

__device__ __forceinline__ u32x4 load_any(const char* p) { return *reinterpret_cast<const u32x4_any*>(p); }

// ---- rows into pages -------------------------------------------------------------------------------------------------------

struct WriteArgs {
    const char *k, *v; int64_t tok, head;             // bytes
    char *kp, *vp; int64_t page_stride, row_stride, head_stride;
    const int64_t* slots; int64_t n_slots;            // rows of the cache
    JbDiv page, pieces, heads;                        // page size; 16-byte pieces of a head's row; heads
    int row_bytes; unsigned n;                        // n: pieces in all
};
// A thread moves the same 16 bytes of a key and a value row; the last piece of a row that is no multiple of 16 begins 16 bytes
// before its end (what two pieces share is written twice, with the same bytes).
__global__ __launch_bounds__(256) void kv_write_kernel(const WriteArgs a) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= a.n) return;
    const unsigned th = jb_div(i, a.pieces), t = jb_div(th, a.heads), h = th - t * a.heads.d;
    const int at = min((int)(i - th * a.pieces.d) * 16, a.row_bytes - 16);
    const int64_t slot = a.slots[t], src = (int64_t)t * a.tok + (int64_t)h * a.head + at;
    const u32x4 kx = load_any(a.k + src), vx = load_any(a.v + src);
    if (slot < 0 || slot >= a.n_slots) return;
    const unsigned pg = jb_div((unsigned)slot, a.page);
    const int64_t dst = (int64_t)pg * a.page_stride + (int64_t)((unsigned)slot - pg * a.page.d) * a.row_stride + (int64_t)h * a.head_stride + at;
    *reinterpret_cast<u32x4_any*>(a.kp + dst) = kx;
    *reinterpret_cast<u32x4_any*>(a.vp + dst) = vx;
}

// ---- block-wide helpers of the planning workgroup ------------------------------------------------------------------------------

// exclusive prefix sum over the NT threads; *total: the sum.  Ends with the scratch free again.
__device__ __forceinline__ int scan_excl(int v, int* s, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(x, o);
        if (lane >= o) x += u;
    }
    if (lane == 63) s[wave] = x;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { const int sw = s[w]; base += w < wave ? sw : 0; all += sw; }
    __syncthreads();
    *total = all;
    return base + x - v;
}
__device__ __forceinline__ bool any_of(bool x, int* s) {
    if (threadIdx.x == 0) s[0] = 0;
    __syncthreads();
    if (x) s[0] = 1;
    __syncthreads();
    const bool r = s[0] != 0;
    __syncthreads();
    return r;
}
// The `need` lowest pages with ref == 0 into found[]; the number found (fewer than `need` only if there are fewer).
__device__ int find_free(const int* ref, int n_pages, int need, int* found, int* s) {
    int have = 0;
    for (int p0 = 0; p0 < n_pages && have < need; p0 += NT * 4) {
        const int p = p0 + threadIdx.x * 4;
        bool f[4];
        int mine = 0, total;
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[e] = p + e < n_pages && ref[p + e] == 0; mine += f[e]; }
        int at = have + scan_excl(mine, s, &total);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f[e]) { if (at < need) found[at] = p + e; ++at; }
        have += total;
    }
    return min(have, need);
}

// ---- extend ------------------------------------------------------------------------------------------------------------------

struct ExtendArgs {
    int* table; int64_t table_stride; int max_pages;
    int *lens, *ref; const int* cu; int64_t* slots; int* status;
    int* work;                                        // [0] whether it fits; [1 + i] length before; [1 + n + i] first of its new pages; then the new pages
    int n_seq, n_pages, n_tokens;
    JbDiv page;
};
__device__ __forceinline__ int pages_of(int len, const JbDiv& page) { return len > 0 ? (int)jb_div((unsigned)len - 1u, page) + 1 : 0; }

__device__ __forceinline__ void extend_token(const ExtendArgs& a, int t) {
    const int *was = a.work + 1, *first = was + a.n_seq, *found = first + a.n_seq;
    int64_t slot = -1;
    if (a.work[0] && t < a.cu[a.n_seq]) {
        int i = 0, hi = a.n_seq - 1;                  // the last sequence that begins at or before t
        while (i < hi) { const int m = (i + hi + 1) >> 1; if (a.cu[m] <= t) i = m; else hi = m - 1; }
        const int pos = was[i] + (t - a.cu[i]), p = (int)jb_div((unsigned)pos, a.page), had = pages_of(was[i], a.page);
        const int row = pos - p * (int)a.page.d;
        int* entry = a.table + (int64_t)i * a.table_stride + p;
        int pg;
        if (p >= had) {
            pg = found[first[i] + p - had];
            if (row == 0) { *entry = pg; a.ref[pg] = 1; }          // a new page's first token enters it
        } else pg = *entry;
        if ((unsigned)pg < (unsigned)a.n_pages) slot = (int64_t)pg * a.page.d + row;
    }
    a.slots[t] = slot;
}
// TOKENS: the planning workgroup writes the tokens' slots too (few of them: a second launch would cost more).
template <bool TOKENS> __global__ __launch_bounds__(NT) void pages_extend_kernel(const ExtendArgs a) {
    __shared__ int s[NT / 64];
    int *was = a.work + 1, *first = was + a.n_seq, *found = first + a.n_seq;
    bool bad = threadIdx.x == 0 && a.cu[0] != 0;
    int need = 0;
    for (int i0 = 0; i0 < a.n_seq; i0 += NT) {
        const int i = i0 + threadIdx.x;
        int more = 0, total;
        if (i < a.n_seq) {
            const int len = a.lens[i], b = a.cu[i], e = a.cu[i + 1];
            const bool ok = len >= 0 && b >= 0 && e >= b && e <= a.n_tokens && (int64_t)len + (e - b) <= (int64_t)a.max_pages * a.page.d &&
                            (int64_t)len + (e - b) <= 0x7fff0000;
            bad |= !ok;
            if (ok) more = min(pages_of(len + (e - b), a.page) - pages_of(len, a.page), a.n_pages + 1);
            was[i] = len;
        }
        const int at = scan_excl(more, s, &total);
        if (i < a.n_seq) first[i] = need + at;
        // a sum beyond what there is says no more (and must not wrap: n_pages <= 2^20)
        need = min(need + min(total, a.n_pages + 1), a.n_pages + 1);
    }
    const bool wrong = any_of(bad, s);
    const bool fits = !wrong && need <= a.n_pages && find_free(a.ref, a.n_pages, need, found, s) == need;
    if (threadIdx.x == 0) {
        a.work[0] = fits;
        if (!fits) *a.status = wrong ? JB_PAGES_BAD_ARG : JB_PAGES_NONE_FREE;
    }
    if (fits)
        for (int i = threadIdx.x; i < a.n_seq; i += NT) a.lens[i] = was[i] + a.cu[i + 1] - a.cu[i];
    if constexpr (TOKENS) {
        __syncthreads();
        for (int t = threadIdx.x; t < a.n_tokens; t += NT) extend_token(a, t);
    }
}
__global__ __launch_bounds__(256) void pages_slots_kernel(const ExtendArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < a.n_tokens) extend_token(a, t);
}

// ---- free --------------------------------------------------------------------------------------------------------------------

// Whether the m rows lie inside the table and none is named twice; `seen` holds a bit per row afterwards.  Whole block.
__device__ bool rows_fit(const int* rows, int m, int n_seq, unsigned* seen, int* s) {
    for (int i = threadIdx.x; i < (n_seq + 31) / 32; i += blockDim.x) seen[i] = 0u;
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < m; i += blockDim.x) {
        const int r = rows[i];
        if ((unsigned)r >= (unsigned)n_seq) bad = true;
        else bad |= atomicOr(&seen[r >> 5], 1u << (r & 31)) >> (r & 31) & 1u;
    }
    return !any_of(bad, s);
}
// One workgroup a row; each looks at the whole list by itself, so that a wrong one changes nothing.
__global__ __launch_bounds__(256) void pages_free_kernel(int* table, int64_t table_stride, int max_pages, int* lens, int* ref, int n_pages,
                                                         const int* rows, int m, int n_seq, int* status) {
    extern __shared__ unsigned seen[];
    __shared__ int s[NT / 64];
    if (!rows_fit(rows, m, n_seq, seen, s)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) *status = JB_PAGES_BAD_ARG;
        return;
    }
    const int r = rows[blockIdx.x];
    int* row = table + (int64_t)r * table_stride;
    for (int c = threadIdx.x; c < max_pages; c += 256) {
        const int pg = row[c];
        if (pg == -1) continue;
        if ((unsigned)pg < (unsigned)n_pages) atomicSub(ref + pg, 1);
        row[c] = -1;
    }
    if (threadIdx.x == 0) lens[r] = 0;
}

// ---- copies of pages -----------------------------------------------------------------------------------------------------------

struct Pools { char* base[MAX_POOLS]; };
constexpr int CHUNK = 16384;                          // bytes of a workgroup's turn: four 16-byte requests a thread

// Page src[i] of every pool to page dst[i], i < *count (or n); the whole grid.
__device__ void copy_pages(const Pools& p, int n_pools, int64_t page_bytes, int64_t stride, const int* src, const int* dst, int n, int n_pages) {
    const unsigned chunks = (unsigned)((page_bytes + CHUNK - 1) / CHUNK);
    const uint64_t per = (uint64_t)chunks * n_pools, total = per * n;
    for (uint64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const unsigned i = (unsigned)(w / per), x = (unsigned)(w - i * per), pool = x / chunks;
        const int64_t at = (int64_t)(x - pool * chunks) * CHUNK;
        const int a = src[i], b = dst[i];
        if ((unsigned)a >= (unsigned)n_pages || (unsigned)b >= (unsigned)n_pages) continue;
        const char* from = p.base[pool] + (int64_t)a * stride;
        char* to = p.base[pool] + (int64_t)b * stride;
        if (page_bytes >= 16) {
            const int64_t end = min(at + (int64_t)CHUNK, page_bytes);
            u32x4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t o = at + (int64_t)(u * 256 + threadIdx.x) * 16;
                if (o < end) v[u] = load_any(from + min(o, page_bytes - 16));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t o = at + (int64_t)(u * 256 + threadIdx.x) * 16;
                if (o < end) *reinterpret_cast<u32x4_any*>(to + min(o, page_bytes - 16)) = v[u];
            }
        } else if (threadIdx.x < page_bytes) to[threadIdx.x] = from[threadIdx.x];
    }
}
__global__ __launch_bounds__(256) void pages_copy_kernel(const Pools p, int n_pools, int64_t page_bytes, int64_t stride, const int* src, const int* dst,
                                                         int n, int n_pages) {
    copy_pages(p, n_pools, page_bytes, stride, src, dst, n, n_pages);
}

// ---- fork ----------------------------------------------------------------------------------------------------------------------

struct ForkArgs {
    int* table; int64_t table_stride; int max_pages;
    int *lens, *ref; const int *src, *dst; int* status;
    int* work;                                        // [0] fits, [1] copies; [2 + i] new page of pair i or -1; then copies' sources, targets, free pages
    int m, n_seq, n_pages;
    JbDiv page;
};
__global__ __launch_bounds__(NT) void pages_fork_plan_kernel(const ForkArgs a) {
    extern __shared__ unsigned seen[];
    __shared__ int s[NT / 64];
    int *fresh = a.work + 2, *from = fresh + a.m, *to = from + a.m, *found = to + a.m;
    bool wrong = !rows_fit(a.dst, a.m, a.n_seq, seen, s);
    int need = 0;
    if (!wrong) {
        bool bad = false;
        for (int i0 = 0; i0 < a.m; i0 += NT) {
            const int i = i0 + threadIdx.x;
            int more = 0, total, pg = -1;
            if (i < a.m) {
                const int r = a.src[i];
                bad |= a.lens[a.dst[i]] != 0;
                if ((unsigned)r >= (unsigned)a.n_seq || (seen[r >> 5] >> (r & 31) & 1u)) bad = true;
                else {
                    const int n = a.lens[r];
                    if (n < 0 || n > (int64_t)a.max_pages * a.page.d) bad = true;
                    else if (n % (int)a.page.d) { pg = a.table[(int64_t)r * a.table_stride + n / (int)a.page.d]; more = 1; }
                }
            }
            const int at = need + scan_excl(more, s, &total);
            if (i < a.m) {
                fresh[i] = more ? at : -1;
                if (more) from[at] = pg;
            }
            need += total;
        }
        wrong = any_of(bad, s);
    }
    const bool fits = !wrong && find_free(a.ref, a.n_pages, need, found, s) == need;
    __syncthreads();
    if (threadIdx.x == 0) {
        a.work[0] = fits;
        a.work[1] = fits ? need : 0;
        if (!fits) *a.status = wrong ? JB_PAGES_BAD_ARG : JB_PAGES_NONE_FREE;
    }
    if (!fits) return;
    for (int i = threadIdx.x; i < a.m; i += NT) {
        const int at = fresh[i];
        if (at >= 0) { fresh[i] = found[at]; to[at] = found[at]; }
        a.lens[a.dst[i]] = a.lens[a.src[i]];          // no source is a target
    }
}
// The rows (a workgroup a pair, first launch only) and the copies of the part-filled last pages.
__global__ __launch_bounds__(256) void pages_fork_kernel(const ForkArgs a, const Pools p, int n_pools, int64_t page_bytes, int64_t stride, bool rows) {
    if (!a.work[0]) return;
    const int *fresh = a.work + 2, *from = fresh + a.m, *to = from + a.m;
    if (rows)
        for (int i = blockIdx.x; i < a.m; i += gridDim.x) {
            const int full = a.lens[a.src[i]] / (int)a.page.d;
            const int* row = a.table + (int64_t)a.src[i] * a.table_stride;
            int* out = a.table + (int64_t)a.dst[i] * a.table_stride;
            for (int c = threadIdx.x; c < a.max_pages; c += 256) {
                int pg = -1;
                if (c < full) {
                    pg = row[c];
                    if ((unsigned)pg < (unsigned)a.n_pages) atomicAdd(a.ref + pg, 1);
                } else if (c == full && fresh[i] >= 0) {
                    pg = fresh[i];
                    a.ref[pg] = 1;
                }
                out[c] = pg;
            }
        }
    copy_pages(p, n_pools, page_bytes, stride, from, to, a.work[1], a.n_pages);
}

// ---- compact -------------------------------------------------------------------------------------------------------------------

// work: [0] live pages, [1] moves; then the moves' sources, their targets, and for every page its new number.
// The j-th live page at or above the number of live pages goes to the j-th free one below it: sources and targets never overlap.
__global__ __launch_bounds__(NT) void pages_compact_plan_kernel(const int* ref, int n_pages, int* work) {
    __shared__ int s[NT / 64];
    int *src = work + 2, *dst = src + n_pages, *map = dst + n_pages;
    int live = 0, total;
    {
        int mine = 0;
        for (int p = threadIdx.x; p < n_pages; p += NT) mine += ref[p] > 0;
        scan_excl(mine, s, &live);
    }
    int holes = 0, moves = 0;
    for (int p0 = 0; p0 < n_pages; p0 += NT) {
        const int p = p0 + threadIdx.x;
        const bool on = p < n_pages && ref[p] > 0;
        const bool hole = p < live && !on, move = on && p >= live;
        // both kinds in one scan: at most NT of either, and both only in the tile that holds the border
        const int at = scan_excl((hole ? 1 : 0) | (move ? 1 << 16 : 0), s, &total);
        if (hole) dst[holes + (at & 0xffff)] = p;
        if (move) src[moves + (at >> 16)] = p;
        if (p < n_pages) map[p] = p;
        holes += total & 0xffff;
        moves += total >> 16;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < moves; j += NT) map[src[j]] = dst[j];
    if (threadIdx.x == 0) { work[0] = live; work[1] = moves; }
}
__global__ __launch_bounds__(256) void pages_compact_kernel(const int* table, int64_t table_stride, int n_seq, int max_pages, const int* ref, int n_pages,
                                                            int* table_out, int* ref_out, const int* work, const Pools p, int n_pools,
                                                            int64_t page_bytes, int64_t stride, bool control) {
    const int live = work[0], *src = work + 2, *dst = src + n_pages, *map = dst + n_pages;
    if (control) {
        const int64_t cells = (int64_t)n_seq * max_pages, step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
        for (int64_t i = at; i < cells; i += step) {
            const int64_t r = i / max_pages;
            const int pg = table[r * table_stride + (i - r * max_pages)];
            table_out[i] = (unsigned)pg < (unsigned)n_pages ? map[pg] : -1;
        }
        for (int64_t i = at; i < n_pages; i += step) {
            const int n = ref[i];
            if (n > 0) ref_out[map[i]] = n;
            if (i >= live) ref_out[i] = 0;
        }
    }
    copy_pages(p, n_pools, page_bytes, stride, src, dst, work[1], n_pages);
}

int pools_fit(const char* who, const jb_page_pools* p) {
    auto bad = [&](const char* what) { jb_set_error(std::string(who) + ": " + what); return (int)JB_ERR_ARG; };
    if (!p || (p->n_pools > 0 && !p->base)) return bad("null pointer");
    if (p->n_pools < 0 || p->n_pages <= 0 || p->page_bytes <= 0 || p->page_stride < p->page_bytes) return bad("bad dims of the pools");
    for (int i = 0; i < p->n_pools; ++i)
        if (!p->base[i]) return bad("null pool");
    return JB_OK;
}
// f(pools, how many, whether it is the first launch) for every MAX_POOLS of the pools (once at least)
template <typename F> void each_launch(const jb_page_pools* p, F f) {
    int done = 0;
    do {
        Pools k = {};
        const int n = p->n_pools - done < MAX_POOLS ? p->n_pools - done : MAX_POOLS;
        for (int i = 0; i < n; ++i) k.base[i] = (char*)p->base[done + i];
        f(k, n, done == 0);
        done += n;
    } while (done < p->n_pools);
}
// workgroups for up to n pages of each of `pools` pools: eight a compute unit keep the memory busy, each then takes several turns
unsigned copy_grid(int64_t page_bytes, int64_t n, int pools) {
    const int64_t turns = n * pools * ((page_bytes + CHUNK - 1) / CHUNK);
    return (unsigned)(turns < 1 ? 1 : turns > 2048 ? 2048 : turns);
}
constexpr int MAX_PAGES = 1 << 20;                    // sums over NT sequences' pages stay below 2^31
constexpr int MAX_SCAN = 1 << 30;                     // pages that one workgroup scans, whose steps stay below 2^31
constexpr int MAX_SEQS = 1 << 17;                     // rows of a table: a bit each in LDS

}  // namespace

extern "C" int jb_kv_write(const jb_kv_write_args* a, void* stream) {
    JB_REQUIRE(a, "null pointer");
    JB_REQUIRE(a->dtype == JB_F32 || a->dtype == JB_F16 || a->dtype == JB_BF16, "bad dtype");
    JB_REQUIRE(a->n_tokens >= 0 && a->n_kv_head > 0 && a->d_head > 0 && a->n_pages > 0 && a->page_size > 0, "bad dims");
    JB_REQUIRE(a->tok_stride >= 0 && a->tok_head_stride >= 0 && a->page_stride >= 0 && a->row_stride >= 0 && a->head_stride >= 0, "negative stride");
    JB_REQUIRE((int64_t)a->n_pages * a->page_size <= 0x7fffffff, "more than 2^31 cache rows");
    JB_REQUIRE(jb_apart(a->d_head, a->n_pages, a->page_stride, a->page_size, a->row_stride, a->n_kv_head, a->head_stride), "rows of the cache overlap");
    const int e = a->dtype == JB_F32 ? 4 : 2;
    int64_t heads = a->n_kv_head, d = a->d_head;
    if (a->tok_head_stride == d && a->head_stride == d) { d *= heads; heads = 1; }       // the heads of a row lie together on both sides
    if (d * e < 16) JB_UNSUPPORTED("rows of less than 16 bytes");
    JB_REQUIRE(d * e <= 0x7fffffff, "bad dims");
    if (a->n_tokens == 0) return JB_OK;
    JB_REQUIRE(a->k && a->v && a->kpool && a->vpool && a->slots, "null pointer");
    const int64_t pieces = (d * e + 15) / 16, n = pieces * heads * a->n_tokens;
    JB_REQUIRE(n <= 0x7fffffff, "too many rows for one call");
    WriteArgs k = {};
    k.k = (const char*)a->k; k.v = (const char*)a->v; k.tok = a->tok_stride * e; k.head = a->tok_head_stride * e;
    k.kp = (char*)a->kpool; k.vp = (char*)a->vpool;
    k.page_stride = a->page_stride * e; k.row_stride = a->row_stride * e; k.head_stride = a->head_stride * e;
    k.slots = a->slots; k.n_slots = (int64_t)a->n_pages * a->page_size;
    k.page = jb_make_div((unsigned)a->page_size); k.pieces = jb_make_div((unsigned)pieces); k.heads = jb_make_div((unsigned)heads);
    k.row_bytes = (int)(d * e); k.n = (unsigned)n;
    kv_write_kernel<<<(unsigned)((n + 255) / 256), 256, 0, (hipStream_t)stream>>>(k);
    JB_CHECK_LAUNCH();
    return JB_OK;
}

extern "C" int jb_pages_extend(const jb_page_table* t, const int* cu_new, int n_tokens, int64_t* slots, int* work, int* status, void* stream) {
    JB_REQUIRE(t && (t->n_seq == 0 || (t->table && t->lens)) && t->ref && cu_new && work && status && (slots || n_tokens == 0), "null pointer");
    JB_REQUIRE(t->n_seq >= 0 && t->max_pages > 0 && t->n_pages > 0 && t->page_size > 0 && n_tokens >= 0, "bad dims");
    JB_REQUIRE(t->table_stride >= t->max_pages || t->n_seq < 2, "rows of the table overlap");
    JB_REQUIRE((int64_t)t->n_pages * t->page_size <= 0x7fffffff, "more than 2^31 cache rows");
    if (t->n_pages > MAX_PAGES) JB_UNSUPPORTED("more than 1048576 pages");
    if (t->n_seq == 0 && n_tokens == 0) return JB_OK;
    ExtendArgs a = {t->table, t->table_stride, t->max_pages, t->lens, t->ref, cu_new, slots, status, work, t->n_seq, t->n_pages, n_tokens,
                    jb_make_div((unsigned)t->page_size)};
    hipStream_t s = (hipStream_t)stream;
    if (n_tokens <= 2048) pages_extend_kernel<true><<<1, NT, 0, s>>>(a);
    else {
        pages_extend_kernel<false><<<1, NT, 0, s>>>(a);
        pages_slots_kernel<<<(unsigned)((n_tokens + 255) / 256), 256, 0, s>>>(a);
    }
    JB_CHECK_LAUNCH();
    return JB_OK;
}

extern "C" int jb_pages_free(const jb_page_table* t, const int* rows, int n_rows, int* status, void* stream) {
    JB_REQUIRE(t && (t->n_seq == 0 || (t->table && t->lens)) && t->ref && status && (rows || n_rows == 0), "null pointer");
    JB_REQUIRE(t->n_seq >= 0 && t->max_pages > 0 && t->n_pages > 0 && n_rows >= 0, "bad dims");
    JB_REQUIRE(t->table_stride >= t->max_pages || t->n_seq < 2, "rows of the table overlap");
    JB_REQUIRE(t->n_seq <= MAX_SEQS && n_rows <= t->n_seq, "more rows than the table has, or a table of more than 131072");
    if (n_rows == 0) return JB_OK;
    const size_t lds = (size_t)(t->n_seq + 31) / 32 * 4;
    pages_free_kernel<<<(unsigned)n_rows, 256, lds, (hipStream_t)stream>>>(t->table, t->table_stride, t->max_pages, t->lens, t->ref, t->n_pages, rows, n_rows,
                                                                           t->n_seq, status);
    JB_CHECK_LAUNCH();
    return JB_OK;
}

extern "C" int jb_pages_copy(const jb_page_pools* p, const int* src, const int* dst, int n_pairs, void* stream) {
    const int rc = pools_fit(__func__, p);
    if (rc) return rc;
    JB_REQUIRE(n_pairs >= 0 && (n_pairs == 0 || (src && dst)), "null pointer");
    if (n_pairs == 0 || p->n_pools == 0) return JB_OK;
    each_launch(p, [&](const Pools& k, int n, bool) {
        pages_copy_kernel<<<copy_grid(p->page_bytes, n_pairs, n), 256, 0, (hipStream_t)stream>>>(k, n, p->page_bytes, p->page_stride, src, dst, n_pairs, p->n_pages);
    });
    JB_CHECK_LAUNCH();
    return JB_OK;
}

extern "C" int jb_pages_fork(const jb_page_table* t, const jb_page_pools* p, const int* src, const int* dst, int n_pairs, int* work, int* status, void* stream) {
    JB_REQUIRE(t && (t->n_seq == 0 || (t->table && t->lens)) && t->ref && work && status && (n_pairs == 0 || (src && dst)), "null pointer");
    const int rc = pools_fit(__func__, p);
    if (rc) return rc;
    JB_REQUIRE(t->n_seq >= 0 && t->max_pages > 0 && t->n_pages > 0 && t->page_size > 0 && n_pairs >= 0 && t->n_pages == p->n_pages, "bad dims");
    JB_REQUIRE(t->table_stride >= t->max_pages || t->n_seq < 2, "rows of the table overlap");
    JB_REQUIRE((int64_t)t->n_pages * t->page_size <= 0x7fffffff, "more than 2^31 cache rows");
    JB_REQUIRE(t->n_seq <= MAX_SEQS && n_pairs <= t->n_seq, "more pairs than the table has rows, or a table of more than 131072");
    if (t->n_pages > MAX_SCAN) JB_UNSUPPORTED("more than 2^30 pages");
    if (n_pairs == 0) return JB_OK;
    ForkArgs a = {t->table, t->table_stride, t->max_pages, t->lens, t->ref, src, dst, status, work, n_pairs, t->n_seq, t->n_pages, jb_make_div((unsigned)t->page_size)};
    hipStream_t s = (hipStream_t)stream;
    pages_fork_plan_kernel<<<1, NT, (size_t)(t->n_seq + 31) / 32 * 4, s>>>(a);
    JB_CHECK_LAUNCH();
    each_launch(p, [&](const Pools& k, int n, bool first) {
        pages_fork_kernel<<<copy_grid(p->page_bytes, n_pairs, n > 0 ? n : 1), 256, 0, s>>>(a, k, n, p->page_bytes, p->page_stride, first);
    });
    JB_CHECK_LAUNCH();
    return JB_OK;
}

extern "C" int jb_pages_compact(const jb_page_table* t, const jb_page_pools* p, int* table_out, int* ref_out, int* work, void* stream) {
    JB_REQUIRE(t && t->ref && ref_out && work && ((t->table && table_out) || t->n_seq == 0), "null pointer");
    const int rc = pools_fit(__func__, p);
    if (rc) return rc;
    JB_REQUIRE(t->n_seq >= 0 && t->max_pages > 0 && t->n_pages > 0 && t->n_pages == p->n_pages, "bad dims");
    JB_REQUIRE(t->table_stride >= t->max_pages || t->n_seq < 2, "rows of the table overlap");
    JB_REQUIRE(table_out != t->table && ref_out != t->ref, "the outputs are arrays of their own");
    if (t->n_pages > MAX_SCAN) JB_UNSUPPORTED("more than 2^30 pages");
    hipStream_t s = (hipStream_t)stream;
    pages_compact_plan_kernel<<<1, NT, 0, s>>>(t->ref, t->n_pages, work);
    JB_CHECK_LAUNCH();
    each_launch(p, [&](const Pools& k, int n, bool first) {
        pages_compact_kernel<<<copy_grid(p->page_bytes, t->n_pages, n > 0 ? n : 1), 256, 0, s>>>(t->table, t->table_stride, t->n_seq, t->max_pages, t->ref, t->n_pages,
                                                                                                table_out, ref_out, work, k, n, p->page_bytes, p->page_stride, first);
    });
    JB_CHECK_LAUNCH();
    return JB_OK;
}

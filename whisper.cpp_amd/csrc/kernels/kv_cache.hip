// The paged K/V cache's own operations (include/mi355x_kernels.h: mi355x_kv_*).  The bookkeeping is integer work on small arrays and stays on the
// device: pages are found, handed out and given back by the kernels, so a decode loop needs no host round trip between a beam search's choice and
// the next step.  Page numbers do not depend on timing: free pages are taken in ascending order by prefix sums of one workgroup, and the counts change
// by integer atomics whose order does not matter.
#include "kv_cache.h"

// the work area, in ints: flag[4] | start[n_seq] | copied[n_seq] | first[n_seq] | pages[n_pages] | rank[n_pages]
struct kv_work { int * flag, * start, * copied, * first, * pages, * rank; };
__host__ __device__ static inline kv_work kv_work_of(int * w, int n_seq, int n_pages) {
    kv_work r; r.flag = w; r.start = w + 4; r.copied = r.start + n_seq; r.first = r.copied + n_seq; r.pages = r.first + n_seq; r.rank = r.pages + n_pages; return r;
}
extern "C" size_t mi355x_kv_work_bytes(int n_seq, int n_pages) {
    return n_seq < 1 || n_pages < 1 ? 0 : 4 * (4 + 3 * (size_t) n_seq + 2 * (size_t) n_pages);
}

#define KV_WG 1024

// exclusive prefix sum over the workgroup; `total` in every thread.  `part`: KV_WG / 64 ints of LDS
__device__ __forceinline__ int wg_scan(int v, int * part, int & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
    #pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(s, o, 64); if (lane >= o) s += u; }
    __syncthreads();
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int base = 0; total = 0;
    #pragma unroll
    for (int w = 0; w < KV_WG / 64; w++) { const int p = part[w]; if (w < wave) base += p; total += p; }
    return base + s - v;
}

// the last entry i of [0, n) with at[i] <= x, for ascending `at` with at[0] <= x
__device__ __forceinline__ int last_at_most(const int * at, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (at[m] <= x) lo = m; else hi = m; }
    return lo;
}

// the same by a whole wave, for an x that is one of the wave's: 64 entries at a look, one load's latency where a bisection has log2(n)
__device__ __forceinline__ int last_at_most_wave(const int * at, int n, int x) {
    const int lane = threadIdx.x & 63;
    int lo = 0, step = 1;
    while (step * 64 < n) step *= 64;
    for (; step > 0; step /= 64) {
        const int i = (int) min((int64_t) lo + (int64_t) lane * step, (int64_t) n - 1);
        lo = min(lo + max((int) __popcll(__ballot(lo + (int64_t) lane * step < n && at[i] <= x)) - 1, 0) * step, n - 1);
    }
    return lo;
}

// ---------------------------------------------------------------------------------------------------------------
// reset
// ---------------------------------------------------------------------------------------------------------------
struct KvResetArgs { kvc c; };
__global__ void __launch_bounds__(256) k_kv_reset(const KvResetArgs a) {
    const int64_t nt = (int64_t) a.c.n_seq * a.c.max_pages, step = (int64_t) gridDim.x * 256, i0 = (int64_t) blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = i0; i < nt; i += step) a.c.table[i] = -1;
    for (int64_t i = i0; i < a.c.n_seq; i += step) a.c.len[i] = 0;
    for (int64_t i = i0; i < a.c.n_pages; i += step) a.c.ref[i] = 0;
    if (i0 == 0) *a.c.status = 0;
}
extern "C" int mi355x_kv_reset(mi355x_ctx * ctx, const mi355x_kv_cache * c) {
    KvResetArgs a; const int rc = kv_view(c, &a.c);
    if (rc) return rc;
    if (!ctx) return kv_refuse("kv_reset: no context");
    const device_scope scope(ctx);
    int64_t nb = ((int64_t) c->n_seq * c->max_pages + c->n_pages) / 1024 + 1;
    if (nb > 2048) nb = 2048;
    return emit(ctx, "kv_reset", k_kv_reset, dim3((uint32_t) nb), dim3(256), 0, a);
}

// ---------------------------------------------------------------------------------------------------------------
// append: pages first (one workgroup), then the rows.  The pages' part is latency: a list of n entries, one pass over as many counts as
// it takes to find the pages it needs.
// ---------------------------------------------------------------------------------------------------------------
struct KvAppendArgs {
    kvc c;
    const int * seq, * cu;
    const char * k, * v; int64_t k_nb1, k_nb2, v_nb1, v_nb2;
    int n, rows, type_in, bf16;
    int nch, cshift;               // 16-byte pieces of a row of all heads (K or V), log2 of the pieces of one head
    uint32_t div_m;                // ceil(2^32 / (2*nch))
    int rb, row_blocks;            // rows per workgroup, workgroups with rows
};

// returns whether the cache was changed; uniform over the workgroup
__device__ __forceinline__ bool kv_reserve(const KvAppendArgs & a, const kv_work & w, uint32_t * seen, int * part, int * shared) {
    const int tid = threadIdx.x, cap = a.c.max_pages << a.c.shift;
    const int words = (a.c.n_seq + 31) >> 5;
    // the counts of the lowest pages are asked for first: what the entries need is known several loads later
    int low[4];
    #pragma unroll
    for (int e = 0; e < 4; e++) low[e] = a.c.ref[min(tid * 4 + e, a.c.n_pages - 1)];
    for (int i = tid; i < words; i += KV_WG) seen[i] = 0;
    if (tid == 0) shared[0] = shared[1] = 0;
    __syncthreads();
    int need_all = 0, bad = 0;
    for (int base = 0; base < a.n; base += KV_WG) {
        const int i = base + tid;
        int need = 0;
        if (i < a.n) {
            const int s = a.seq[i], r0 = a.cu[i], r1 = a.cu[i + 1];
            int start = -1, copied = -1;
            if (s >= a.c.n_seq || r0 < 0 || r1 < r0 || r1 > a.rows) bad |= MI355X_KV_BAD_ARG;
            else if (s >= 0) {
                const int old = a.c.len[s], more = r1 - r0;
                if ((atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1) bad |= MI355X_KV_BAD_ARG;
                else if (old < 0 || old > cap) bad |= MI355X_KV_BAD_ARG;
                else if (more > cap - old) bad |= MI355X_KV_ROW_FULL;
                else {
                    start = old;
                    need = ((old + more + a.c.mask) >> a.c.shift) - ((old + a.c.mask) >> a.c.shift);
                    if (more > 0 && (old & a.c.mask)) {
                        const int p = a.c.table[(int64_t) s * a.c.max_pages + (old >> a.c.shift)];
                        if (p < 0 || p >= a.c.n_pages) bad |= MI355X_KV_BAD_ARG;
                        else if (a.c.ref[p] > 1) { copied = p; need++; }
                    }
                }
            }
            w.start[i] = start; w.copied[i] = copied;
            if (copied >= 0) shared[1] = 1;                          // some entry copies its last page
        }
        int total;
        const int at = wg_scan(need, part, total);
        if (i < a.n) w.first[i] = need_all + at;
        need_all = total > INT32_MAX - need_all ? INT32_MAX : need_all + total;
    }
    if (bad) atomicOr((unsigned *) &shared[0], (unsigned) bad);
    __syncthreads();
    bad = shared[0];
    // the lowest free pages
    int found = 0;
    if (!bad) {
        for (int base = 0; base < a.c.n_pages && found < need_all; base += KV_WG * 4) {
            const int p0 = base + tid * 4;
            int fr[4], cnt = 0;
            #pragma unroll
            for (int e = 0; e < 4; e++) if (base) low[e] = a.c.ref[min(p0 + e, a.c.n_pages - 1)];
            #pragma unroll
            for (int e = 0; e < 4; e++) { fr[e] = p0 + e < a.c.n_pages && low[e] == 0; cnt += fr[e]; }
            int total, at = wg_scan(cnt, part, total) + found;
            #pragma unroll
            for (int e = 0; e < 4; e++) if (fr[e]) { if (at < need_all) w.pages[at] = p0 + e; at++; }
            found += total;
        }
        if (found < need_all) bad = MI355X_KV_OUT_OF_PAGES;
    }
    if (tid == 0) { w.flag[0] = bad == 0; if (bad) atomicOr((unsigned *) a.c.status, (unsigned) bad); }
    if (bad) return false;
    __syncthreads();                                                 // lists complete, every count read
    for (int j = tid; j < need_all; j += KV_WG) {
        const int i = last_at_most(w.first, a.n, j), s = a.seq[i], old = w.start[i], p = w.pages[j];
        const int col = ((old + a.c.mask) >> a.c.shift) - (w.copied[i] >= 0) + (j - w.first[i]);
        a.c.table[(int64_t) s * a.c.max_pages + col] = p;
        a.c.ref[p] = 1;
    }
    for (int i = tid; i < a.n; i += KV_WG) {
        const int s = a.seq[i];
        if (s < 0) continue;
        if (w.copied[i] >= 0) atomicAdd(&a.c.ref[w.copied[i]], -1);
        a.c.len[s] = w.start[i] + a.cu[i + 1] - a.cu[i];
    }
    return true;
}

// U pieces of 16 bytes (as stored) of each of NT threads, from j0 on, of the `count` pieces of rows r0 ..: first all loads, which do not wait for the rows'
// places, then the stores to the places at[], rounded to the cache's type
template <int NT, int U> struct kv_pieces {
    u32x4_t x[U][2];
    // piece j's row (j / per: exact, j * per < 2^32), V or K, head and piece of the head
    static __device__ __forceinline__ void of(const KvAppendArgs & a, int j, int & r, bool & isv, int & head, int & ch) {
        r = (int) __umulhi((uint32_t) j, a.div_m);
        const int piece = j - r * 2 * a.nch;
        isv = piece >= a.nch;
        const int q = isv ? piece - a.nch : piece;
        head = q >> a.cshift; ch = q & ((1 << a.cshift) - 1);
    }
    __device__ __forceinline__ void load(const KvAppendArgs & a, int r0, int count, int j0) {
        const char * src[U];
        #pragma unroll
        for (int u = 0; u < U; u++) {
            int r, head, ch; bool isv;
            of(a, min(j0 + u * NT, count - 1), r, isv, head, ch);
            src[u] = (isv ? a.v + (r0 + r) * a.v_nb2 + head * a.v_nb1 : a.k + (r0 + r) * a.k_nb2 + head * a.k_nb1) + ch * (a.type_in == MI355X_TYPE_F32 ? 32 : 16);
        }
        #pragma unroll
        for (int u = 0; u < U; u++) x[u][0] = *(const u32x4_t *) src[u];
        if (a.type_in == MI355X_TYPE_F32) {
            #pragma unroll
            for (int u = 0; u < U; u++) x[u][1] = ((const u32x4_t *) src[u])[1];
        }
    }
    __device__ __forceinline__ void store(const KvAppendArgs & a, const int64_t * at, int count, int j0) {
        const bool same = a.type_in == (a.bf16 ? MI355X_TYPE_BF16 : MI355X_TYPE_F16);
        #pragma unroll
        for (int u = 0; u < U; u++) {
            int r, head, ch; bool isv;
            of(a, min(j0 + u * NT, count - 1), r, isv, head, ch);
            if (j0 + u * NT >= count || at[r] < 0) continue;
            u32x4_t y = x[u][0];
            if (!same) {
                char raw[32]; float f[8];
                __builtin_memcpy(raw, &x[u][0], 16); __builtin_memcpy(raw + 16, &x[u][1], 16);
                load8(raw, a.type_in, f);
                if (a.bf16) {
                    bf16x8_t o;
                    #pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = (__bf16) f[e];
                    __builtin_memcpy(&y, &o, 16);
                } else {
                    half8_t o;
                    #pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = (half_t) f[e];
                    __builtin_memcpy(&y, &o, 16);
                }
            }
            *(u32x4_t *) ((isv ? a.c.v : a.c.k) + at[r] + head * a.c.nb_head + ch * 16) = y;
        }
    }
};

// byte offset of packed row r's place in the pools (entry i's, if the row has one), -1 if it belongs to no sequence
__device__ __forceinline__ int64_t kv_place(const KvAppendArgs & a, const kv_work & w, int r, int i) {
    if (r < a.cu[0] || r >= a.cu[a.n]) return -1;
    const int s = a.seq[i];
    if (s < 0) return -1;
    const int at = w.start[i] + r - a.cu[i];
    const int p = a.c.table[(int64_t) s * a.c.max_pages + (at >> a.c.shift)];
    if (p < 0 || p >= a.c.n_pages) return -1;                        // a table that the caller has overwritten
    return p * a.c.nb_page + (at & a.c.mask) * a.c.nb_key;
}

// the places of rows r0 .. r0 + nr - 1: each wave finds the entries of its rows (by turns), then a lane for each row follows it to its page
template <int NT, int ROWS> __device__ __forceinline__ void kv_places(const KvAppendArgs & a, const kv_work & w, int r0, int nr, int64_t * place) {
    constexpr int NW = NT / 64, PER = (ROWS + NW - 1) / NW;
    static_assert(PER <= 64, "a lane for each of a wave's rows");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane * NW + wave;
    int i = 0;
    #pragma unroll
    for (int q = 0; q < PER; q++) if (q * NW + wave < nr) {
        const int found = last_at_most_wave(a.cu, a.n, r0 + q * NW + wave);
        if (lane == q) i = found;
    }
    if (lane < PER && r < nr) place[r] = kv_place(a, w, r0 + r, i);
}

// the rows of entry i's last page that its sequence shared, into the page of its own
template <int NT> __device__ __forceinline__ void kv_copy_shared(const KvAppendArgs & a, const kv_work & w, int i, int tid) {
    const int p = w.copied[i];
    if (p < 0) return;
    const int keys = w.start[i] & a.c.mask, to = a.c.table[(int64_t) a.seq[i] * a.c.max_pages + (w.start[i] >> a.c.shift)];
    if (to < 0 || to >= a.c.n_pages) return;
    const int per = keys << a.cshift;                                // pieces of one head
    for (int j = tid; j < 2 * a.c.Hkv * per; j += NT) {
        const int hv = j / per, q = j - hv * per, head = hv >> 1;
        const int64_t at = head * a.c.nb_head + (q >> a.cshift) * a.c.nb_key + (q & ((1 << a.cshift) - 1)) * 16;
        char * pool = hv & 1 ? a.c.v : a.c.k;
        *(uint4 *) (pool + to * a.c.nb_page + at) = *(const uint4 *) (pool + p * a.c.nb_page + at);
    }
}

__global__ void __launch_bounds__(KV_WG) k_kv_reserve(const KvAppendArgs a) {
    extern __shared__ uint32_t seen[];
    __shared__ int part[KV_WG / 64], shared[2];
    kv_reserve(a, kv_work_of(a.c.work, a.c.n_seq, a.c.n_pages), seen, part, shared);
}

// rows into their pages: rb rows per workgroup, whose places are looked up while the rows are on their way; behind them one workgroup per entry for shared
// last pages.  Bound by HBM (rows in, rows out) once there are enough rows: with the two launches before it (11 us) 17321 rows of 8 heads of 128, 142 MB in
// and out, 43.1 us, of which this is about 32 (4.4 TB/s; 27.5 where the same rows come again and again); four pieces of a thread at a time (eight: 46; places first,
// then the rows: 45, and 300 rows a sequence 15.1 instead of 13.7; a bisection for each row: 32 rows 12.6, so 12.4).
#define KV_U 4
#define KV_RB 16
__global__ void __launch_bounds__(256) k_kv_write(const KvAppendArgs a) {
    const kv_work w = kv_work_of(a.c.work, a.c.n_seq, a.c.n_pages);
    if ((int) blockIdx.x >= a.row_blocks) { if (w.flag[0]) kv_copy_shared<256>(a, w, blockIdx.x - a.row_blocks, threadIdx.x); return; }
    __shared__ int64_t at[KV_RB];
    const int r0 = blockIdx.x * a.rb, nr = min(a.rb, a.rows - r0), count = nr * 2 * a.nch;
    kv_pieces<256, KV_U> p;
    p.load(a, r0, count, threadIdx.x);
    if (w.flag[0] == 0) return;
    kv_places<256, KV_RB>(a, w, r0, nr, at);
    __syncthreads();
    p.store(a, at, count, threadIdx.x);
    for (int j0 = threadIdx.x + KV_U * 256; j0 < count; j0 += KV_U * 256) { p.load(a, r0, count, j0); p.store(a, at, count, j0); }
}

// few rows: pages and rows by one workgroup, without the second launch, as long as that is one batch of loads for each thread (with the truncation before
// it, 20 heads of 64: one row 7.9 us, two launches 11.6; eight rows 11.3, 12.2).  One CU takes too long for more: 32 rows of 20 heads of 64 (10240 pieces)
// 14.9 us by itself, where two launches take 5.3 + 4.9.
#define KV_SMALL_ROWS 256
#define KV_SMALL_PIECES (4 * KV_WG)
__global__ void __launch_bounds__(KV_WG) k_kv_append_small(const KvAppendArgs a) {
    extern __shared__ uint32_t seen[];
    __shared__ int part[KV_WG / 64], shared[2];
    __shared__ int64_t at[KV_SMALL_ROWS];
    const kv_work w = kv_work_of(a.c.work, a.c.n_seq, a.c.n_pages);
    const int count = a.rows * 2 * a.nch;
    kv_pieces<KV_WG, KV_SMALL_PIECES / KV_WG> p;
    p.load(a, 0, count, threadIdx.x);
    if (!kv_reserve(a, w, seen, part, shared)) return;
    __syncthreads();                                                 // table and lists as they are now
    if ((int) threadIdx.x < a.rows) at[threadIdx.x] = kv_place(a, w, threadIdx.x, last_at_most(a.cu, a.n, threadIdx.x));
    if (shared[1]) for (int i = threadIdx.x >> 6; i < a.n; i += KV_WG / 64) kv_copy_shared<64>(a, w, i, threadIdx.x & 63);
    __syncthreads();
    p.store(a, at, count, threadIdx.x);
}

extern "C" int mi355x_kv_append(mi355x_ctx * ctx, const mi355x_kv_cache * c, int n, const int32_t * seq, const int32_t * cu, const mi355x_tensor * k, const mi355x_tensor * v) {
    KvAppendArgs a; memset(&a, 0, sizeof(a));
    const int rc = kv_view(c, &a.c);
    if (rc) return rc;
    if (!ctx || !k || !v) return kv_refuse("kv_append: a NULL argument");
    if (!kv_rows_ok(k, c->head_dim, c->n_head_kv) || !kv_rows_ok(v, c->head_dim, c->n_head_kv) || k->ne[2] != v->ne[2] || k->type != v->type)
        return kv_refuse("kv_append: k and v are [head_dim, n_head_kv, rows] of one type, 16-byte aligned");
    if (n < 0 || n > c->n_seq) return kv_refuse("kv_append: more entries than sequences");
    if (n == 0) return 0;
    if (!seq || !cu || ((uintptr_t) seq | (uintptr_t) cu) % 4) return kv_refuse("kv_append: seq or cu");
    if (!kv_fits(k->ne[2] + n, 256)) return kv_refuse("kv_append: too many rows for one launch");
    const device_scope scope(ctx);
    a.seq = seq; a.cu = cu; a.n = n; a.rows = (int) k->ne[2]; a.type_in = k->type; a.bf16 = c->type == MI355X_TYPE_BF16;
    a.k = (const char *) k->data; a.k_nb1 = k->nb[1]; a.k_nb2 = k->nb[2];
    a.v = (const char *) v->data; a.v_nb1 = v->nb[1]; a.v_nb2 = v->nb[2];
    a.cshift = c->head_dim == 64 ? 3 : 4; a.nch = c->n_head_kv << a.cshift;
    a.div_m = (uint32_t) ((((uint64_t) 1 << 32) + 2 * a.nch - 1) / (2 * a.nch));
    const uint32_t lds = (uint32_t) ((c->n_seq + 31) / 32 * 4);
    if (a.rows > 0 && a.rows <= KV_SMALL_ROWS && (int64_t) a.rows * 2 * a.nch <= KV_SMALL_PIECES)
        return emit(ctx, "kv_append", k_kv_append_small, dim3(1), dim3(KV_WG), lds, a);
    int rc1 = emit(ctx, "kv_reserve", k_kv_reserve, dim3(1), dim3(KV_WG), lds, a);
    if (rc1 || a.rows == 0) return rc1;
    a.rb = 1;
    if (a.rows >= 4096) { a.rb = KV_U * 256 / (2 * a.nch); a.rb = a.rb < 1 ? 1 : a.rb > KV_RB ? KV_RB : a.rb; }
    a.row_blocks = (a.rows + a.rb - 1) / a.rb;
    const double bytes = (double) a.rows * a.nch * 2 * (16 + (k->type == MI355X_TYPE_F32 ? 32 : 16));
    return emit(ctx, "kv_write", k_kv_write, dim3((uint32_t) (a.row_blocks + n)), dim3(256), 0, a, bytes);
}

// ---------------------------------------------------------------------------------------------------------------
// truncate: one workgroup per entry.  An exchange takes each page out of the row, so that a sequence named twice gives a page back once.
// ---------------------------------------------------------------------------------------------------------------
struct KvTruncateArgs { kvc c; const int * seq, * keep; int n; };
__global__ void __launch_bounds__(256) k_kv_truncate(const KvTruncateArgs a) {
    const int s = a.seq[blockIdx.x], keep = a.keep[blockIdx.x];
    if (s < 0) return;
    if (s >= a.c.n_seq || keep < 0) { if (threadIdx.x == 0) atomicOr((unsigned *) a.c.status, MI355X_KV_BAD_ARG); return; }
    __shared__ int held;
    if (threadIdx.x == 0) held = atomicMin(&a.c.len[s], keep);
    __syncthreads();
    if (held <= keep) return;
    const int last = min((int) (((int64_t) held + a.c.mask) >> a.c.shift), a.c.max_pages);
    for (int j = ((keep + a.c.mask) >> a.c.shift) + threadIdx.x; j < last; j += 256) {
        const int p = atomicExch(&a.c.table[(int64_t) s * a.c.max_pages + j], -1);
        if (p >= 0 && p < a.c.n_pages) atomicAdd(&a.c.ref[p], -1);
    }
}
extern "C" int mi355x_kv_truncate(mi355x_ctx * ctx, const mi355x_kv_cache * c, int n, const int32_t * seq, const int32_t * keep) {
    KvTruncateArgs a; const int rc = kv_view(c, &a.c);
    if (rc) return rc;
    if (!ctx || n < 0 || (n > 0 && (!seq || !keep || ((uintptr_t) seq | (uintptr_t) keep) % 4))) return kv_refuse("kv_truncate: arguments");
    if (!kv_fits(n, 256)) return kv_refuse("kv_truncate: too many entries for one launch");
    const device_scope scope(ctx);
    a.seq = seq; a.keep = keep; a.n = n;
    return emit(ctx, "kv_truncate", k_kv_truncate, dim3((uint32_t) n), dim3(256), 0, a);
}

// ---------------------------------------------------------------------------------------------------------------
// fork: a workgroup owns `cols` columns of the table.  It reads all sources' entries into LDS before it writes any destination's, so rows may
// change places; every workgroup comes to the same verdict over the list by itself.
// ---------------------------------------------------------------------------------------------------------------
struct KvForkArgs { kvc c; const int * src, * dst; int n, cshift; };
__global__ void __launch_bounds__(256) k_kv_fork(const KvForkArgs a) {
    extern __shared__ int lds[];
    __shared__ int verdict;
    const int tid = threadIdx.x, words = (a.c.n_seq + 31) >> 5, cols = 1 << a.cshift, c0 = blockIdx.x << a.cshift;
    uint32_t * seen = (uint32_t *) lds; int * snap = lds + words, * slen = snap + (a.n << a.cshift);
    for (int i = tid; i < words; i += 256) seen[i] = 0;
    if (tid == 0) verdict = 0;
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < a.n; i += 256) {
        const int d = a.dst[i], s = a.src[i];
        if (d >= a.c.n_seq || s >= a.c.n_seq) bad = 1;
        else if (d >= 0) {
            if ((atomicOr(&seen[d >> 5], 1u << (d & 31)) >> (d & 31)) & 1) bad = 1;
            if (blockIdx.x == 0) slen[i] = s >= 0 ? a.c.len[s] : 0;
        }
    }
    if (bad) verdict = 1;
    for (int j = tid; j < a.n << a.cshift; j += 256) {
        const int i = j >> a.cshift, col = c0 + (j & (cols - 1)), s = a.src[i];
        snap[j] = s >= 0 && s < a.c.n_seq && col < a.c.max_pages ? a.c.table[(int64_t) s * a.c.max_pages + col] : -1;
    }
    __syncthreads();
    if (verdict) { if (blockIdx.x == 0 && tid == 0) atomicOr((unsigned *) a.c.status, MI355X_KV_BAD_ARG); return; }
    for (int j = tid; j < a.n << a.cshift; j += 256) {
        const int i = j >> a.cshift, col = c0 + (j & (cols - 1)), d = a.dst[i];
        if (d < 0 || col >= a.c.max_pages) continue;
        int * e = &a.c.table[(int64_t) d * a.c.max_pages + col];
        const int was = *e, is = snap[j];
        if (was == is) continue;
        *e = is;
        if (was >= 0 && was < a.c.n_pages) atomicAdd(&a.c.ref[was], -1);
        if (is >= 0 && is < a.c.n_pages) atomicAdd(&a.c.ref[is], 1);
    }
    if (blockIdx.x == 0) for (int i = tid; i < a.n; i += 256) if (a.dst[i] >= 0) a.c.len[a.dst[i]] = slen[i];
}
extern "C" int mi355x_kv_fork(mi355x_ctx * ctx, const mi355x_kv_cache * c, int n, const int32_t * src, const int32_t * dst) {
    KvForkArgs a; const int rc = kv_view(c, &a.c);
    if (rc) return rc;
    if (!ctx || n < 0 || n > 8192 || (n > 0 && (!src || !dst || ((uintptr_t) src | (uintptr_t) dst) % 4))) return kv_refuse("kv_fork: arguments");
    if (n == 0) return 0;
    const device_scope scope(ctx);
    a.src = src; a.dst = dst; a.n = n;
    // 8 columns (32 bytes of a row) per workgroup; fewer where the list is so long that they would not fit beside it in 128 KB
    a.cshift = 3;
    const size_t fixed = ((size_t) c->n_seq + 31) / 32 * 4 + (size_t) n * 4;
    while (a.cshift > 0 && fixed + ((size_t) n << a.cshift) * 4 > 128 * 1024) a.cshift--;
    const size_t lds = fixed + ((size_t) n << a.cshift) * 4;         // <= 128 KB
    const int64_t blocks = ((int64_t) c->max_pages + (1 << a.cshift) - 1) >> a.cshift;
    if (!kv_fits(blocks, 256)) return kv_refuse("kv_fork: the table is too wide for one launch");
    static std::atomic<uint64_t> allowed{0};
    const int rl = kv_allow_lds(ctx, (const void *) k_kv_fork, (uint32_t) lds, allowed);
    if (rl) return rl;
    return emit(ctx, "kv_fork", k_kv_fork, dim3((uint32_t) blocks), dim3(256), (uint32_t) lds, a);
}

// ---------------------------------------------------------------------------------------------------------------
// compact: the held pages' ranks (one workgroup, 5 us for 10000), then pages and table.  Bound by HBM: every held page is read and written once.  Half a
// gigabyte in and out: 91 us = 5.0 TB/s.
// ---------------------------------------------------------------------------------------------------------------
struct KvCompactArgs { kvc a, b; int cshift, slices, table_blocks; };
__global__ void __launch_bounds__(KV_WG) k_kv_rank(const KvCompactArgs a) {
    __shared__ int part[KV_WG / 64];
    const kv_work w = kv_work_of(a.a.work, a.a.n_seq, a.a.n_pages);
    int used = 0;
    for (int base = 0; base < a.a.n_pages; base += KV_WG * 4) {
        const int p0 = base + threadIdx.x * 4;
        int held[4], cnt = 0;
        #pragma unroll
        for (int e = 0; e < 4; e++) held[e] = a.a.ref[min(p0 + e, a.a.n_pages - 1)];
        #pragma unroll
        for (int e = 0; e < 4; e++) { held[e] = p0 + e < a.a.n_pages && held[e] > 0; cnt += held[e]; }
        int total, at = wg_scan(cnt, part, total) + used;
        #pragma unroll
        for (int e = 0; e < 4; e++) if (p0 + e < a.a.n_pages) { w.rank[p0 + e] = held[e] ? at : -1; if (held[e]) w.pages[at++] = p0 + e; }
        used += total;
    }
    if (threadIdx.x == 0) {
        w.flag[1] = used <= a.b.n_pages ? used : -1;
        if (used > a.b.n_pages) atomicOr((unsigned *) a.b.status, MI355X_KV_OUT_OF_PAGES);
    }
}
#define KV_SLICE 1024             // 16-byte pieces per workgroup
// slice `slice` of page `p` to page r of the new pool
__device__ __forceinline__ void kv_move(const KvCompactArgs & a, int p, int r, int slice) {
    const int64_t from = p * a.a.nb_page, to = r * a.b.nb_page;
    const int per = a.a.Hkv << (a.a.shift + a.cshift);               // pieces of a page in one pool
    // every load before the first store, and none under a condition: one that might not happen is not asked for before its store (99 and 18 us)
    u32x4_t x[KV_SLICE / 256];
    char * dst[KV_SLICE / 256];
    #pragma unroll
    for (int e = 0; e < KV_SLICE / 256; e++) {
        const int j0 = slice * KV_SLICE + e * 256 + threadIdx.x, j1 = min(j0, 2 * per - 1);
        const bool isv = j1 >= per;
        const int j = isv ? j1 - per : j1, ch = j & ((1 << a.cshift) - 1), row = j >> a.cshift, key = row & a.a.mask, head = row >> a.a.shift;
        x[e] = *(const u32x4_t *) ((isv ? a.a.v : a.a.k) + from + head * a.a.nb_head + key * a.a.nb_key + ch * 16);
        dst[e] = j0 < 2 * per ? (isv ? a.b.v : a.b.k) + to + head * a.b.nb_head + key * a.b.nb_key + ch * 16 : nullptr;
    }
    #pragma unroll
    for (int e = 0; e < KV_SLICE / 256; e++) if (dst[e]) *(u32x4_t *) dst[e] = x[e];
}
__global__ void __launch_bounds__(256) k_kv_compact(const KvCompactArgs a) {
    const kv_work w = kv_work_of(a.a.work, a.a.n_seq, a.a.n_pages);
    const int used = w.flag[1];
    if (used < 0) return;
    if ((int) blockIdx.x < a.table_blocks) {
        const int64_t step = (int64_t) a.table_blocks * 256, i0 = (int64_t) blockIdx.x * 256 + threadIdx.x, nt = (int64_t) a.b.n_seq * a.b.max_pages;
        for (int64_t i = i0; i < nt; i += step) {
            const int64_t s = i / a.b.max_pages, col = i - s * a.b.max_pages;
            const int p = col < a.a.max_pages ? a.a.table[s * a.a.max_pages + col] : -1;
            a.b.table[i] = p >= 0 && p < a.a.n_pages ? w.rank[p] : -1;
        }
        for (int64_t i = i0; i < a.b.n_seq; i += step) a.b.len[i] = a.a.len[i];
        for (int64_t i = i0; i < a.b.n_pages; i += step) a.b.ref[i] = i < used ? a.a.ref[w.pages[i]] : 0;
        return;
    }
    const int64_t blk = blockIdx.x - a.table_blocks;
    const int r = (int) (blk / a.slices), slice = (int) (blk - (int64_t) r * a.slices);
    if (r >= used) return;
    kv_move(a, w.pages[r], r, slice);
}

// few pages and few slices: every workgroup ranks the pages for itself, without the first launch (822 pages, 4 MB in and out: 4.1 us, two launches
// 7.1); with more than 16 slices for each CU the ranks would be made again and again
#define KV_SMALL_PAGES 2048
#define KV_SMALL_SLICES 4096
__global__ void __launch_bounds__(256) k_kv_compact_small(const KvCompactArgs a) {
    constexpr int PER = KV_SMALL_PAGES / 256;
    __shared__ int rank[KV_SMALL_PAGES], sum[4], mine;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, p0 = tid * PER;
    int ref[PER], cnt = 0;
    #pragma unroll
    for (int e = 0; e < PER; e++) ref[e] = a.a.ref[min(p0 + e, a.a.n_pages - 1)];
    #pragma unroll
    for (int e = 0; e < PER; e++) { if (p0 + e >= a.a.n_pages) ref[e] = 0; cnt += ref[e] > 0; }
    int at = cnt;
    #pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(at, o, 64); if (lane >= o) at += u; }
    if (lane == 63) sum[wave] = at;
    __syncthreads();
    int used = 0;
    at -= cnt;
    #pragma unroll
    for (int w = 0; w < 4; w++) { if (w < wave) at += sum[w]; used += sum[w]; }
    if (used > a.b.n_pages) { if (blockIdx.x == 0 && tid == 0) atomicOr((unsigned *) a.b.status, MI355X_KV_OUT_OF_PAGES); return; }
    const int blk = (int) blockIdx.x - a.table_blocks, r = blk / a.slices;
    if (blk >= 0) {
        if (r >= used) return;
        #pragma unroll
        for (int e = 0; e < PER; e++) if (ref[e] > 0 && at++ == r) mine = p0 + e;
        __syncthreads();
        kv_move(a, mine, r, blk - r * a.slices);
        return;
    }
    #pragma unroll
    for (int e = 0; e < PER; e++) {
        rank[p0 + e] = ref[e] > 0 ? at : -1;
        if (ref[e] > 0) { if (blockIdx.x == 0) a.b.ref[at] = ref[e]; at++; }
    }
    __syncthreads();
    const int64_t step = (int64_t) a.table_blocks * 256, i0 = (int64_t) blockIdx.x * 256 + tid, nt = (int64_t) a.b.n_seq * a.b.max_pages;
    for (int64_t i = i0; i < nt; i += step) {
        const int64_t s = i / a.b.max_pages, col = i - s * a.b.max_pages;
        const int p = col < a.a.max_pages ? a.a.table[s * a.a.max_pages + col] : -1;
        a.b.table[i] = p >= 0 && p < a.a.n_pages ? rank[p] : -1;
    }
    for (int64_t i = i0; i < a.b.n_seq; i += step) a.b.len[i] = a.a.len[i];
    for (int64_t i = used + i0; i < a.b.n_pages; i += step) a.b.ref[i] = 0;
}
extern "C" int mi355x_kv_compact(mi355x_ctx * ctx, const mi355x_kv_cache * from, const mi355x_kv_cache * to) {
    KvCompactArgs a; int rc = kv_view(from, &a.a);
    if (!rc) rc = kv_view(to, &a.b);
    if (rc) return rc;
    if (!ctx) return kv_refuse("kv_compact: no context");
    if (from->type != to->type || from->head_dim != to->head_dim || from->n_head_kv != to->n_head_kv || from->page_size != to->page_size || from->n_seq != to->n_seq || to->max_pages < from->max_pages)
        return kv_refuse("kv_compact: the caches differ in type, dims or sequences, or the new table is narrower");
    if (from->k == to->k || from->k == to->v || from->v == to->k || from->v == to->v || from->table == to->table || from->len == to->len || from->ref == to->ref || from->work == to->work)
        return kv_refuse("kv_compact: the new cache has to be other memory");
    const device_scope scope(ctx);
    a.cshift = from->head_dim == 64 ? 3 : 4;
    const int64_t per = (int64_t) 2 * from->n_head_kv * from->page_size << a.cshift;
    a.slices = (int) ((per + KV_SLICE - 1) / KV_SLICE);
    const int64_t entries = (int64_t) to->n_seq * to->max_pages + to->n_pages;
    int64_t tb = entries / 2048 + 1;
    a.table_blocks = (int) (tb > 1024 ? 1024 : tb);
    const int64_t pages = from->n_pages < to->n_pages ? from->n_pages : to->n_pages;     // at most so many are held and fit
    const int64_t blocks = a.table_blocks + pages * a.slices;
    if (per > INT32_MAX || !kv_fits(blocks, 256)) return kv_refuse("kv_compact: pools too large for one launch");
    if (from->n_pages <= KV_SMALL_PAGES && pages * a.slices <= KV_SMALL_SLICES) {
        a.table_blocks = (int) (entries / 256 + 1 > 1024 ? 1024 : entries / 256 + 1);
        return emit(ctx, "kv_compact", k_kv_compact_small, dim3((uint32_t) (a.table_blocks + pages * a.slices)), dim3(256), 0, a);
    }
    rc = emit(ctx, "kv_rank", k_kv_rank, dim3(1), dim3(KV_WG), 0, a);
    return rc ? rc : emit(ctx, "kv_compact", k_kv_compact, dim3((uint32_t) blocks), dim3(256), 0, a);
}

// Attention of one new token per stream over the paged K/V cache (include/mi355x_kernels.h: mi355x_attn_paged).
//     o = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q.k_j - max)
// Bound by the bytes of the keys and values, which every K/V head's workgroups read once for all the query heads that share it: up to 16 of them are
// the columns of one matrix product, so that grouped heads cost no more reads and no more instructions than single ones.
//
//   k_attn_paged   a workgroup = one K/V head (x 16 query heads) x the keys of one query, or a run of the keys of several (paged_split_of); its waves take
//                  tiles of 32 keys in turn, each with its own running maximum and sum, and are joined in LDS at the end.
//                  S^T = K.Q^T and O^T = V^T.P^T on v_mfma_f32_16x16x32: a lane owns ONE head (column), so the softmax statistics are
//                  scalars of the lane and the P fragment feeds the second product straight from the registers (the order of the 32 keys inside the
//                  product is the same for both operands).  K goes from memory to registers as the operand lies (64 consecutive bytes of a key per
//                  instruction and 4 lanes), V through an area of LDS that belongs to the wave, read back transposed: no barrier in the loop, and the
//                  next tile's 8 or 16 KB are on their way while one is computed.  974 MB of BF16 keys: 175 us = 5.6 TB/s (a loop that only
//                  reads reaches 6.2 on this card, a copy 4.9); 351 MB in 64 queries of 1 .. 8192 keys: 81 us (a run for each wave instead of each workgroup: 80 to 83).
//   k_attn_join    joins the parts of one query and head where the keys were split.
// The same kernel serves packed sequences of few rows (attn_packed.hip says when): a tile's 16 columns are then (query, head) pairs, each with its own
// range of keys.
//
// F32 queries are split into NT terms of the cache's type (2 x 11 or 3 x 8 bits), the weights likewise: the products are exact, the sums F32.  16-bit queries
// take one term; the weights are then rounded to 16 bits, half a step of the result's own type (the sum of the weights is of the unrounded ones, in F32): an F16 or BF16
// result is off by 2^-11 or 2^-8 either way.  Over a BF16 cache a step of F32 queries is thus finer than the same model's prompt (attn_packed.hip: one term).
#include "kv_cache.h"

#define TILE 32                        // keys of a tile: one 16x16x32 product over keys
#define MIN_RUN 8                      // tiles of a run at least: two for each wave
#define OVERHEAD 6                     // tiles: of a query in a run, see cost_of
#define NEG_BIG (-__FLT_MAX__)         // the running maximum's start, no more than any score: exp2(x - NEG_BIG) of a masked x = -inf is 0, not NaN

struct PagedArgs {
    kvc c;
    const int * seq;
    const char * q; int64_t q_nb1, q_nb2;
    char * o; int64_t o_nb1, o_nb2;
    float * part_o, * part_ml; int * meta;     // where the keys are split: records [unit][W + n][rec_rows][D], [..][2]; n + 1 sums of costs and the cost of a run
    float c2;                          // scale * log2(e)
    int q_type, o_type, window;
    int G, H, groups;                  // query heads per K/V head, query heads, sets of 16 query heads per K/V head
    int W, rec_rows;                   // workgroups of a unit (K/V head x set of 16 query heads), 0: one for each query; rows of a record
    const int * cu_q, * cu_k;          // packed rows: as in PackedArgs
    int n, rows_q, rows_k, causal;
    int lds_main;                      // bytes of LDS in front of the sums
    int qt, hg;                        // queries of a tile of 16 rows, heads of the group that each has there: qt * hg <= 16
};

// the keys that query i sees, as [lo, hi)
struct paged_span { int s, lo, hi; };
__device__ __forceinline__ int tiles_of(const paged_span & p) { return p.hi > p.lo ? (p.hi + TILE - 1) / TILE - p.lo / TILE : 0; }
// in two steps, so that what depends on the sequence alone can be asked for along with its length
__device__ __forceinline__ int held_of(const PagedArgs & a, int s) { return a.c.len[min(max(s, 0), a.c.n_seq - 1)]; }
__device__ __forceinline__ paged_span span_of(const PagedArgs & a, int s, int held) {
    paged_span r;
    r.s = s;
    const int64_t cap = (int64_t) a.c.max_pages << a.c.shift;
    r.hi = s < 0 || s >= a.c.n_seq || held < 0 ? 0 : held > cap ? (int) cap : held;
    r.lo = a.window > 0 && r.hi > a.window ? r.hi - a.window : 0;
    return r;
}
// what a query costs a run of the split: its tiles, and about as much as OVERHEAD tiles for its start and end
__device__ __forceinline__ int cost_of(int tiles) { return tiles > 0 ? tiles + OVERHEAD : 0; }

// F32 values as NT terms of a 16-bit type: x = t0 + t1 (+ t2), each the rounding of what the ones before leave
template <typename O, int NT> __device__ __forceinline__ void split8(const float * f, typename O::vec8 * t) {
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        float r = f[e];
        #pragma unroll
        for (int n = 0; n < NT; n++) { t[n][e] = (typename O::elem) r; if (n + 1 < NT) r -= (float) t[n][e]; }
    }
}

// what a 16-byte piece's number in a V row of LDS is changed by (exclusive-or): the eight keys that one half of a transposing read touches lie in
// different banks
template <int D> __device__ __forceinline__ int v_swap(int key) { return D == 128 ? (key & 7) << 1 : (key >> 1 & 3) << 1; }

enum { SMALL_PAGES, BIG_PAGES, ROWS };                   // where K and V lie: pages of fewer than 32 keys; 32 and more (a tile lies in one); packed rows

// (registers: 64 dims and 16-bit queries fit four waves to a SIMD, if only just)
template <typename O, int D, int NT, int SRC, bool PACKED>
__global__ void __launch_bounds__(512, D == 64 && NT == 1 && !PACKED ? 4 : 2) k_attn_paged(const PagedArgs a) {
    typedef typename O::vec8 vec8;
    constexpr int KK = D / 32;                           // 32-dim pieces of a key
    constexpr int NV = D / 16;                           // V loads of a tile; 16-dim blocks of the result
    constexpr int RPL = 512 / D;                         // V rows per load
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, nl = lane & 15, g4 = lane >> 4, waves = blockDim.x >> 6;
    const int units = a.c.Hkv * a.groups, unit = blockIdx.x % units, w = blockIdx.x / units, grp = unit % a.groups, hk = unit / a.groups;
    int i = w;                                           // the query; packed: the first query row of this workgroup
    paged_span sp;
    int nq = 1, k0 = 0, own = 0;                         // packed: queries here, the keys' first row, the first query's own key
    if (PACKED) {
        packed_job job;
        if (!packed_find(a, i, job)) return;
        int L = 0;
        sp.s = -1;
        if (SRC == ROWS) {
            k0 = a.cu_k[job.i]; const int k1 = a.cu_k[job.i + 1];
            if (k0 >= 0 && k1 <= a.rows_k && k1 > k0) L = k1 - k0;
        } else {
            sp.s = a.seq ? a.seq[job.i] : job.i;
            if (sp.s >= 0 && sp.s < a.c.n_seq) { const int64_t cap = (int64_t) a.c.max_pages << a.c.shift; const int len = a.c.len[sp.s]; L = len < 0 ? 0 : len > cap ? (int) cap : len; }
        }
        const int q0 = job.tile * a.qt;
        nq = min(a.qt, job.nq - q0); own = L - job.nq + q0; i = job.r0 + q0;
        sp.lo = a.window > 0 ? max(own - a.window + 1, 0) : 0;
        sp.hi = a.causal ? min(own + nq, L) : L;
    }
    // Split keys: the queries' costs, one after the other, are cut into W equal runs; a run may end one query, hold others and begin the next.
    int p = 0, p1 = 0;
    int * pre = (int *) (lds + a.lds_main);              // sums of the costs of the queries before i
    if (!PACKED && a.W) {
        for (int j = threadIdx.x; j < a.n; j += blockDim.x) {
            const int sj = a.seq ? a.seq[j] : j;
            pre[j + 1] = cost_of(tiles_of(span_of(a, sj, held_of(a, sj))));
        }
        if (threadIdx.x == 0) pre[0] = 0;
        __syncthreads();
        if (wave == 0) {
            int carry = 0;
            for (int base = 0; base < a.n; base += 64) {
                int v = base + lane < a.n ? pre[base + lane + 1] : 0;
                #pragma unroll
                for (int d = 1; d < 64; d <<= 1) { const int u = __shfl_up(v, d, 64); if (lane >= d) v += u; }
                if (base + lane < a.n) pre[base + lane + 1] = v + carry;
                carry += __shfl(v, 63, 64);
            }
        }
        __syncthreads();
        const int total = pre[a.n], per = max((total + a.W - 1) / a.W, MIN_RUN);
        if (blockIdx.x == 0) for (int j = threadIdx.x; j < a.n + 2; j += blockDim.x) a.meta[j] = j <= a.n ? pre[j] : per;
        p = min((int64_t) w * per, (int64_t) total); p1 = min(p + per, total);
        if (p >= p1) return;
        int lo = 0, hi = a.n;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (pre[mid] <= p) lo = mid; else hi = mid; }
        i = lo;
    }
    const int g0 = grp * 16, rows = PACKED ? nq * a.hg : min(16, a.G - g0), h0 = hk * a.G + g0;
    // a lane's places in its wave's V area: where it puts row r (key RPL r + lane / (D / 8); the change by the key's bit 2 is one of r's), and where it reads
    // dims 16 d of key 4 g4 + nl / 4 (exclusive-or with d << 5)
    const int wkey = lane / (D / 8), rkey = 4 * g4 + (nl >> 2);
    const uint32_t v_put = lds_at(lds) + wave * (TILE * D * 2) + wkey * (D * 2) + ((lane % (D / 8)) ^ v_swap<D>(wkey)) * 16;
    const uint32_t v_get = lds_at(lds) + wave * (TILE * D * 2) + rkey * (D * 2) + (((nl >> 1) & 1) ^ v_swap<D>(rkey)) * 16 + (nl & 1) * 8;
    // row r of the 16: query i + r / hg, head h0 + r % hg (one query: head h0 + r)
    auto q_of = [&](int r) { return PACKED ? r / a.hg : 0; };
    auto h_of = [&](int r) { return PACKED ? r - r / a.hg * a.hg : r; };
    const bool here = nl < rows && g0 + h_of(nl) < a.G;
    const int ql = min(q_of(nl), nq - 1);
    auto v_row = [&](uint32_t put, int r) { return (LDS u32x4_t *) (size_t) ((put ^ (D == 128 ? (r & 1) << 7 : 0)) + r * RPL * (D * 2)); };
    bool bad = false;
    for (;;) {                                           // the parts of queries in this run
    const int seq = PACKED ? sp.s : a.seq ? a.seq[i] : i, held = PACKED ? 0 : held_of(a, seq);
    const int * row = a.c.table + (int64_t) min(max(seq, 0), a.c.n_seq - 1) * a.c.max_pages;
    // the page of each key of a tile, in lane key & 31, as the table has it
    auto ask_pages = [&](int t) { return SRC == ROWS ? 0 : row[min((int64_t) (t * TILE + (lane & 31)) >> a.c.shift, (int64_t) a.c.max_pages - 1)]; };
    int pg = 0;
    const bool early = !PACKED && !a.W && a.window == 0;             // the wave's first tile does not depend on the length
    if (early) pg = ask_pages(wave);

    // Q^T as the second operand: lane (head nl, dims 32 kk + 8 g4 ..)
    vec8 qf[NT][KK];
    #pragma unroll
    for (int kk = 0; kk < KK; kk++) {
        float f[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };
        if (here) load8(a.q + (int64_t) (i + q_of(nl)) * a.q_nb2 + (int64_t) (h0 + h_of(nl)) * a.q_nb1 + (32 * kk + 8 * g4) * (a.q_type == MI355X_TYPE_F32 ? 4 : 2), a.q_type, f);
        vec8 t[NT];
        split8<O, NT>(f, t);
        #pragma unroll
        for (int n = 0; n < NT; n++) qf[n][kk] = t[n];
    }
    if (!PACKED) sp = span_of(a, seq, held);
    const int t_first = sp.lo / TILE, t_all = tiles_of(sp);
    int t0 = t_first, t1 = t_first + t_all;
    if (!PACKED && a.W) {
        const int at = pre[i] + OVERHEAD;                            // where its tiles begin
        t0 = t_first + max(p - at, 0); t1 = t_first + max(min(p1, pre[i + 1]) - at, 0);
    }
    const bool whole = t1 - t0 == t_all;
    // the keys that lane nl's row sees are first .. last
    const int last = PACKED && a.causal ? min(own + ql, sp.hi - 1) : sp.hi - 1, first = PACKED && a.window > 0 ? max(own + ql - a.window + 1, 0) : sp.lo;
    const char * kb = a.c.k + hk * a.c.nb_head, * vb = a.c.v + hk * a.c.nb_head;
    // keys outside the span are replaced by the nearest inside (of the same tile): what no row sees is not read
    auto key_of = [&](int t, int kl) { return min(max(t * TILE + kl, sp.lo), sp.hi - 1); };
    auto checked = [&](int t, int pg) {
        const int key = t * TILE + (lane & 31);
        bad |= SRC != ROWS && key >= sp.lo && key < sp.hi && (unsigned) pg >= (unsigned) a.c.n_pages;
        return SRC == ROWS ? 0 : min(max(pg, 0), a.c.n_pages - 1);
    };
    auto place = [&](int t, int key, int pg) -> int64_t {
        if (SRC == ROWS) return (int64_t) ((uint64_t) (uint32_t) (k0 + key) * (uint32_t) a.c.nb_key);
        const int p = SRC == BIG_PAGES ? __builtin_amdgcn_readfirstlane(pg) : __shfl(pg, key - t * TILE, 64);
        return (int64_t) ((uint64_t) (uint32_t) p * (uint32_t) a.c.nb_page + (uint64_t) (uint32_t) (key & a.c.mask) * (uint32_t) a.c.nb_key);
    };
    vec8 kr[2][KK]; u32x4_t vr[NV];
    auto fetch_k = [&](int t, int pg) {
        #pragma unroll
        for (int b = 0; b < 2; b++) {
            const char * at = kb + place(t, key_of(t, 16 * b + nl), pg) + 16 * g4;
            #pragma unroll
            for (int kk = 0; kk < KK; kk++) kr[b][kk] = *(const vec8 *) (at + 64 * kk);
        }
    };
    auto fetch_v = [&](int t, int pg) {
        #pragma unroll
        for (int r = 0; r < NV; r++) {
            vr[r] = *(const u32x4_t *) (vb + place(t, key_of(t, r * RPL + lane / (D / 8)), pg) + (lane % (D / 8)) * 16);
        }
    };

    floatx4 o[NV];
    #pragma unroll
    for (int d = 0; d < NV; d++) o[d] = floatx4{ 0, 0, 0, 0 };
    float m = NEG_BIG, l = 0.0f;
    int t = t0 + wave;
    if (t < t1) {
        if (!early) pg = ask_pages(t);
        pg = checked(t, pg);
        fetch_k(t, pg);
        fetch_v(t, pg);
        pg = ask_pages(t + waves);
        for (; t < t1; t += waves) {
            const bool more = t + waves < t1;
            uint32_t put = v_put, get = v_get;
            asm volatile("" : "+v"(put), "+v"(get));                 // the places are made again in each step: kept for all steps they would cost a wave per SIMD in registers
            floatx4 s[2], rest[2];                                   // the first terms' products, and the others'
            #pragma unroll
            for (int b = 0; b < 2; b++) {
                s[b] = rest[b] = floatx4{ 0, 0, 0, 0 };
                #pragma unroll
                for (int n = NT - 1; n > 0; n--)
                    #pragma unroll
                    for (int kk = 0; kk < KK; kk++) rest[b] = O::mfma16(kr[b][kk], qf[n][kk], rest[b]);
                #pragma unroll
                for (int kk = 0; kk < KK; kk++) s[b] = O::mfma16(kr[b][kk], qf[0][kk], s[b]);
            }
            if (more) { pg = checked(t + waves, pg); fetch_k(t + waves, pg); }
            // V into this wave's area.  Zero times an infinity or a NaN is none: where some row does not see all of the tile, they are taken out here,
            // and counted over the keys that each row sees below (rare: the next V tile waits for it).
            bool odd = false;
            if (PACKED && (t * TILE + TILE - 1 > (a.causal ? own : sp.hi - 1) || (a.window > 0 && t * TILE < own + nq - a.window))) {
                uint32_t nf = 0;
                #pragma unroll
                for (int r = 0; r < NV; r++) nf |= not_finite8<O>(vr[r]);
                odd = __any(nf != 0);
            }
            if (PACKED && odd) {
                #pragma unroll
                for (int r = 0; r < NV; r++) {
                    u32x4_t x = vr[r], kind = { 0, 0, 0, 0 };
                    take_apart<O>(x, kind);
                    *v_row(put, r) = x;
                }
            } else {
                if (!PACKED && (t * TILE < sp.lo || t * TILE + TILE > sp.hi)) {                      // rows that stand for none: their weight is zero, which an infinity would not obey
                    #pragma unroll
                    for (int r = 0; r < NV; r++) {
                        const int key = t * TILE + r * RPL + wkey;
                        if (key < sp.lo || key >= sp.hi) vr[r] = u32x4_t{ 0, 0, 0, 0 };
                    }
                }
                #pragma unroll
                for (int r = 0; r < NV; r++) *v_row(put, r) = vr[r];
            }
            if (more && !odd) {
                fetch_v(t + waves, pg);
                pg = ask_pages(t + 2 * waves);
            }
            // softmax: element r of block b is key 16 b + 4 g4 + r of head nl
            float x[8], top = NEG_BIG;
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = t * TILE + 16 * (e >> 2) + 4 * g4 + (e & 3);
                // (an infinite key: the first term's sign is the query's, the others' need not be)
                if (NT > 1) s[e >> 2][e & 3] += __builtin_amdgcn_fmed3f(rest[e >> 2][e & 3], -0x1p126f, 0x1p126f);
                x[e] = key >= first && key <= last ? s[e >> 2][e & 3] * a.c2 : -INFINITY;
                top = fmaxf(top, x[e]);
            }
            top = fmaxf(top, lane_xor16(top));
            top = fmaxf(top, lane_xor32(top));
            if (__any(top > m)) {
                const float mn = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - mn);
                m = mn; l *= alpha;
                #pragma unroll
                for (int d = 0; d < NV; d++)
                    #pragma unroll
                    for (int r = 0; r < 4; r++) o[d][r] *= alpha;
            }
            // F16 weights are held times 2^15, so that small ones do not fall below its range; the factor cancels against the sum's
            // (added to the difference, which is small where weights are not: m - 15 is another number than it says from 2^24 on)
            float p[8];
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const float d = x[e] - m;
                p[e] = __builtin_amdgcn_exp2f(__is_same(O, f16_ops) ? d + 15.0f : d);
                l += p[e];
            }
            vec8 pf[NT];
            split8<O, NT>(p, pf);
            // V^T as the first operand: this 16-lane group's keys 4 g4 + {0..3} and 16 + 4 g4 + {0..3}, dims 16 d + {0..15}
            auto v_frag = [&](int d) {
                vec8 vf;
                #pragma unroll
                for (int b = 0; b < 2; b++) {
                    const short4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS short4_t *) (size_t) ((get ^ d << 5) + 16 * b * (D * 2)));
                    __builtin_memcpy((char *) &vf + 8 * b, &r, 8);
                }
                return vf;
            };
            #pragma unroll
            for (int d = 0; d < NV; d++) {
                const vec8 vf = v_frag(d);
                #pragma unroll
                for (int n = NT - 1; n >= 0; n--) o[d] = O::mfma16(vf, pf[n], o[d]);
            }
            if (PACKED && odd) {
                #pragma unroll
                for (int r = 0; r < NV; r++) {
                    u32x4_t x = vr[r], kind = { 0, 0, 0, 0 };
                    take_apart<O>(x, kind);
                    *v_row(put, r) = kind;
                }
                vec8 seen;
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = t * TILE + 16 * (e >> 2) + 4 * g4 + (e & 3);
                    seen[e] = (typename O::elem) (key >= first && key <= last ? 1.0f : 0.0f);
                }
                #pragma unroll
                for (int d = 0; d < NV; d++) {
                    const floatx4 cnt = O::mfma16(v_frag(d), seen, floatx4{ 0, 0, 0, 0 });
                    #pragma unroll
                    for (int r = 0; r < 4; r++) o[d][r] += put_back(cnt[r]);
                }
                if (more) {
                    fetch_v(t + waves, pg);
                    pg = ask_pages(t + 2 * waves);
                }
            }
        }
    }
    l += lane_xor16(l);
    l += lane_xor32(l);

    // a NaN among row h's sums of dims d .., where the row's weights are numbers: the values decide (kinds_of)
    auto settle = [&](int h, int d, floatx4 & r) {
        const int own_h = own + q_of(h), k_last = PACKED && a.causal ? min(own_h, sp.hi - 1) : sp.hi - 1, k_first = PACKED && a.window > 0 ? max(own_h - a.window + 1, 0) : sp.lo;
        uint32_t kinds[4] = { 0, 0, 0, 0 };
        #pragma unroll 1
        for (int key = max(k_first, t0 * TILE); key <= min(k_last, t1 * TILE - 1); key++) {
            if (SRC == ROWS) kinds_of<O>(a.c.v + hk * a.c.nb_head + (int64_t) (k0 + key) * a.c.nb_key + d * 2, kinds);
            else kinds_of<O>(a.c.v + hk * a.c.nb_head + min(max(row[key >> a.c.shift], 0), a.c.n_pages - 1) * a.c.nb_page + (key & a.c.mask) * a.c.nb_key + d * 2, kinds);
        }
        #pragma unroll
        for (int n = 0; n < 4; n++) if (kinds[n]) r[n] = kinds_value(kinds[n]);
    };
    // join the waves: their (m, l) and O^T over the dead V areas, dim-major for the writer's runs
    __syncthreads();
    float * ml = (float *) lds, * ol = ml + waves * 32;
    if (g4 == 0) { ml[wave * 32 + nl] = m; ml[wave * 32 + 16 + nl] = l; }
    #pragma unroll
    for (int d = 0; d < NV; d++) *(floatx4 *) (ol + (wave * 16 + nl) * (D + 4) + 16 * d + 4 * g4) = o[d];
    __syncthreads();
    for (int j = threadIdx.x; j < rows * (D / 4); j += blockDim.x) {
        const int h = j / (D / 4), d = j % (D / 4) * 4;
        if (PACKED && g0 + h_of(h) >= a.G) continue;
        float M = NEG_BIG, L = 0.0f;
        for (int w = 0; w < waves; w++) M = fmaxf(M, ml[w * 32 + h]);
        floatx4 r = { 0, 0, 0, 0 };
        for (int w = 0; w < waves; w++) {
            const float f = __builtin_amdgcn_exp2f(ml[w * 32 + h] - M);
            L += f * ml[w * 32 + 16 + h];
            const floatx4 x = *(const floatx4 *) (ol + (w * 16 + h) * (D + 4) + d);
            #pragma unroll
            for (int e = 0; e < 4; e++) r[e] += f * x[e];
        }
        const float all = r[0] + r[1] + r[2] + r[3];
        if (__builtin_expect(all != all && L == L, 0)) settle(h, d, r);
        if (whole) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            store4(a.o + (int64_t) (i + q_of(h)) * a.o_nb2 + (int64_t) (h0 + h_of(h)) * a.o_nb1 + d * (a.o_type == MI355X_TYPE_F32 ? 4 : 2), a.o_type, r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv);
        } else {                                         // w + i is another one for every part: the next has a larger w, a larger i or both
            const int64_t rec = ((int64_t) unit * (a.W + a.n) + w + i) * a.rec_rows + h;
            *(floatx4 *) (a.part_o + rec * D + d) = r;
            if (d == 0) { a.part_ml[rec * 2] = M; a.part_ml[rec * 2 + 1] = L; }
        }
    }
    if (PACKED || !a.W) break;
    p = min(p1, pre[i + 1]);
    if (p >= p1) break;
    do i++; while (pre[i + 1] == pre[i]);                // (p < the sum of all: there is one with tiles)
    __syncthreads();
    }
    if (SRC != ROWS && __any(bad) && lane == 0) atomicOr((unsigned *) a.c.status, MI355X_KV_BAD_ARG);
}

// the factor of a part whose maximum is so far below the whole's: never zero, which would make a NaN of an infinity in the part
__device__ __forceinline__ float part_weight(float below) { return fmaxf(__builtin_amdgcn_exp2f(below), 0x1p-126f); }

// Joins the parts of one query and head, where it has several; zeros where it has none.  D/4 threads take a part's sums, 1024/D parts at a time.
template <int D, int NT>
__global__ void __launch_bounds__(NT) k_attn_join(const PagedArgs a) {
    constexpr int L4 = D / 4, NG = NT / L4;
    __shared__ float red[NG][D + 4], lsum[NG], top[NG];
    const int h = blockIdx.x % a.H, i = blockIdx.x / a.H, g = threadIdx.x / L4, d = threadIdx.x % L4 * 4;
    const int p0 = a.meta[i], p1 = a.meta[i + 1], per = a.meta[a.n + 1];
    const int w0 = (p0 + OVERHEAD) / per, n = p1 > p0 ? (p1 - 1) / per - w0 + 1 : 0;
    if (n == 1) return;                                              // written as a whole
    const int hk = h / a.G, unit = hk * a.groups + (h - hk * a.G) / 16;
    const int64_t rec = ((int64_t) unit * (a.W + a.n) + w0 + i) * a.rec_rows + (h - hk * a.G) % 16;
    float M = NEG_BIG, L = 0.0f;
    floatx4 r = { 0, 0, 0, 0 };
    for (int s0 = g; s0 < n; s0 += 4 * NG) {                         // four parts at a time: all of their loads at once
        float m[4], l[4]; floatx4 x[4];
        #pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t k = rec + (int64_t) min(s0 + u * NG, n - 1) * a.rec_rows;
            m[u] = a.part_ml[k * 2]; l[u] = a.part_ml[k * 2 + 1]; x[u] = *(const floatx4 *) (a.part_o + k * D + d);
        }
        #pragma unroll
        for (int u = 0; u < 4; u++) {
            if (s0 + u * NG >= n) break;
            const float mn = fmaxf(M, m[u]), f0 = part_weight(M - mn), f1 = part_weight(m[u] - mn);
            M = mn; L = L * f0 + l[u] * f1;
            #pragma unroll
            for (int e = 0; e < 4; e++) r[e] = r[e] * f0 + x[u][e] * f1;
        }
    }
    *(floatx4 *) &red[g][d] = r;
    if (d == 0) { top[g] = M; lsum[g] = L; }
    __syncthreads();
    if (g > 0) return;
    float T = top[0];
    #pragma unroll
    for (int w = 1; w < NG; w++) T = fmaxf(T, top[w]);
    L = 0.0f;
    #pragma unroll
    for (int e = 0; e < 4; e++) r[e] = 0.0f;
    #pragma unroll
    for (int w = 0; w < NG; w++) {
        const float f = part_weight(top[w] - T);
        const floatx4 x = *(const floatx4 *) &red[w][d];
        L += f * lsum[w];
        #pragma unroll
        for (int e = 0; e < 4; e++) r[e] += f * x[e];
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    store4(a.o + (int64_t) i * a.o_nb2 + (int64_t) h * a.o_nb1 + d * (a.o_type == MI355X_TYPE_F32 ? 4 : 2), a.o_type, r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv);
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
// Whether and how the keys are split.  A workgroup takes a query's keys (of one K/V head) alone where there are at most 1024 of them (448 keys, 8 heads of
// 64: 7.3 us, where a second launch alone is 4), or where every CU has two such workgroups and none reads more than half a megabyte (32 x 1500, 20 heads of
// 64: 48.6 us; split 52.1.  64 x 1 .. 2048, 8 heads of 128, a megabyte: 33.4; split 26.5).  Beyond that the costs of all queries are cut into as many
// equal runs as workgroups of four waves fit the chip at once (two to a CU: 178 to 243 registers at 128 dims): every CU has the same to do, however the lengths differ, and
// no workgroup starts late (2 x 100001 .. 131072 keys, 8 heads of 128: 175 us; three to a CU, in two rounds: 191).
#define CHIP_RUNS (2 * 256)
struct paged_split { int W, rec_rows; size_t floats, bytes; };
static paged_split paged_split_of(const mi355x_kv_cache * c, int64_t n, int64_t n_head, int max_len) {
    paged_split r = { 0, 0, 0, 0 };
    const int64_t cap = (int64_t) c->max_pages * c->page_size, len = max_len > 0 && max_len < cap ? max_len : cap, G = n_head / c->n_head_kv, units = c->n_head_kv * ((G + 15) / 16);
    if (len <= 1024 || (n * units >= CHIP_RUNS && len * c->head_dim <= 131072) || n > 4096 || n * (cap / TILE + 1 + OVERHEAD) > INT32_MAX / 2) return r;   // (the last: sums of costs are 32 bits)
    r.W = units < CHIP_RUNS ? (int) (CHIP_RUNS / units) : 1;
    r.rec_rows = (int) (G < 16 ? G : 16);
    r.floats = (size_t) units * (r.W + n) * r.rec_rows;
    r.bytes = (r.floats * (c->head_dim + 2) + n + 2) * 4;
    return r;
}
extern "C" size_t mi355x_attn_paged_work_bytes(const mi355x_kv_cache * c, int n, int n_head, int max_len) {
    if (!c || n < 1 || n_head < 1 || c->n_head_kv < 1 || n_head % c->n_head_kv || c->page_size < 1 || c->max_pages < 1 || c->head_dim < 1) return 0;
    return paged_split_of(c, n, n_head, max_len).bytes;
}

template <typename O, int D, int NT, int SRC, bool PACKED>
static int launch_as(mi355x_ctx * ctx, PagedArgs & a, int64_t blocks, int threads) {
    const uint32_t v = (uint32_t) (threads / 64 * TILE * D * 2), j = (uint32_t) (threads / 64 * (32 + 16 * (D + 4)) * 4);
    a.lds_main = (int) (v > j ? v : j);
    const uint32_t lds = (uint32_t) a.lds_main + (a.W ? (a.n + 1) * 4 : 0);
    static std::atomic<uint64_t> allowed{0};
    const int rl = kv_allow_lds(ctx, (const void *) k_attn_paged<O, D, NT, SRC, PACKED>, lds, allowed);
    return rl ? rl : emit(ctx, PACKED ? "attn_packed" : "attn_paged", k_attn_paged<O, D, NT, SRC, PACKED>, dim3((uint32_t) blocks), dim3(threads), lds, a);
}
template <typename O, int D, int NT>
static int launch_paged(mi355x_ctx * ctx, PagedArgs & a) {
    const int64_t blocks = (int64_t) (a.W ? a.W : a.n) * a.c.Hkv * a.groups;
    const int threads = a.W || (int64_t) a.n * a.c.Hkv * a.groups > ctx->n_cu ? 256 : 512;
    return a.c.shift >= 5 ? launch_as<O, D, NT, BIG_PAGES, false>(ctx, a, blocks, threads) : launch_as<O, D, NT, SMALL_PAGES, false>(ctx, a, blocks, threads);
}
template <typename O, int D>
static int launch_few(mi355x_ctx * ctx, PagedArgs & a, bool paged) {
    const int64_t blocks = ((int64_t) a.rows_q / a.qt + a.n) * a.c.Hkv * a.groups;
    if (!kv_fits(blocks, 512)) return kv_refuse("attn_packed: too many rows for one launch");
    if (!paged) return launch_as<O, D, 1, ROWS, true>(ctx, a, blocks, 512);
    return a.c.shift >= 5 ? launch_as<O, D, 1, BIG_PAGES, true>(ctx, a, blocks, 512) : launch_as<O, D, 1, SMALL_PAGES, true>(ctx, a, blocks, 512);
}
int mi355x_attn_few_rows(mi355x_ctx * ctx, const PackedArgs & p, int type, int dim, bool paged) {
    PagedArgs a; memset(&a, 0, sizeof(a));
    a.c = p.c; a.c.Hkv = p.Hkv; a.seq = p.seq;
    a.q = p.q; a.q_nb1 = p.q_nb1; a.q_nb2 = p.q_nb2; a.q_type = p.q_type;
    a.o = p.o; a.o_nb1 = p.o_nb1; a.o_nb2 = p.o_nb2; a.o_type = p.o_type;
    a.c2 = p.flip ? -p.c2 : p.c2; a.window = p.window; a.G = p.G; a.H = p.G * p.Hkv; a.groups = (p.G + 15) / 16;
    a.cu_q = p.cu_q; a.cu_k = p.cu_k; a.n = p.n; a.rows_q = p.rows_q; a.rows_k = p.rows_k; a.causal = p.causal;
    a.hg = p.G < 16 ? p.G : 16; a.qt = 16 / a.hg;
    if (dim == 64) return type == MI355X_TYPE_F16 ? launch_few<f16_ops, 64>(ctx, a, paged) : launch_few<bf16_ops, 64>(ctx, a, paged);
    return type == MI355X_TYPE_F16 ? launch_few<f16_ops, 128>(ctx, a, paged) : launch_few<bf16_ops, 128>(ctx, a, paged);
}

extern "C" int mi355x_attn_paged(mi355x_ctx * ctx, const mi355x_kv_cache * c, const mi355x_attn_paged_desc * d) {
    PagedArgs a; memset(&a, 0, sizeof(a));
    const int rc = kv_view(c, &a.c);
    if (rc) return rc;
    if (!ctx || !d) return kv_refuse("attn_paged: a NULL argument");
    const int64_t H = d->q.ne[1], n = d->q.ne[2];
    if (H < 1 || H > 32768 || H % c->n_head_kv) return kv_refuse("attn_paged: the query heads are no multiple of the K/V heads");
    if (!kv_rows_ok(&d->q, c->head_dim, H) || !kv_rows_ok(&d->dst, c->head_dim, H) || d->dst.ne[2] != n) return kv_refuse("attn_paged: q and dst are [head_dim, n_head, n], F32 / F16 / BF16, 16-byte aligned");
    if (n > INT32_MAX / 32768 || !kv_fits(n * H, n > 4096 ? 512 : 1024)) return kv_refuse("attn_paged: too many queries");      // (a workgroup for each query and head at most; 1024 threads: k_attn_join)
    if (!d->seq && n > c->n_seq) return kv_refuse("attn_paged: more queries than sequences");
    if ((uintptr_t) d->seq % 4 || d->window < 0 || d->max_len < 0) return kv_refuse("attn_paged: seq, window or max_len");
    if (n == 0) return 0;
    const device_scope scope(ctx);
    a.seq = d->seq;
    a.q = (const char *) d->q.data; a.q_nb1 = d->q.nb[1]; a.q_nb2 = d->q.nb[2]; a.q_type = d->q.type;
    a.o = (char *) d->dst.data; a.o_nb1 = d->dst.nb[1]; a.o_nb2 = d->dst.nb[2]; a.o_type = d->dst.type;
    a.c2 = d->scale * 1.4426950408889634f; a.window = d->window;
    a.H = (int) H; a.G = (int) (H / c->n_head_kv); a.groups = (a.G + 15) / 16;
    a.n = (int) n;
    const paged_split sp = paged_split_of(c, n, H, d->max_len);
    a.W = sp.W; a.rec_rows = sp.rec_rows;
    if (sp.bytes) {
        if (!d->work || d->work_bytes < sp.bytes || (uintptr_t) d->work % 16) return kv_refuse("attn_paged: the work area is missing, too small or misaligned");
        a.part_o = (float *) d->work;
        a.part_ml = a.part_o + sp.floats * c->head_dim;
        a.meta = (int *) (a.part_ml + sp.floats * 2);
    }
    const bool f16 = c->type == MI355X_TYPE_F16, one = d->q.type == c->type;
    int e;
    if (c->head_dim == 64) e = f16 ? (one ? launch_paged<f16_ops, 64, 1>(ctx, a) : launch_paged<f16_ops, 64, 2>(ctx, a))
                                   : (one ? launch_paged<bf16_ops, 64, 1>(ctx, a) : launch_paged<bf16_ops, 64, 3>(ctx, a));
    else                   e = f16 ? (one ? launch_paged<f16_ops, 128, 1>(ctx, a) : launch_paged<f16_ops, 128, 2>(ctx, a))
                                   : (one ? launch_paged<bf16_ops, 128, 1>(ctx, a) : launch_paged<bf16_ops, 128, 3>(ctx, a));
    if (e || !a.W) return e;
    // a workgroup for each query and head: 256 threads take 8 (128 dims) or 16 parts at a time, 1024 threads where a query has many
    const dim3 grid((uint32_t) (n * H));
    if (a.W / a.n >= 16) return c->head_dim == 64 ? emit(ctx, "attn_join", k_attn_join<64, 1024>, grid, dim3(1024), 0, a) : emit(ctx, "attn_join", k_attn_join<128, 1024>, grid, dim3(1024), 0, a);
    return c->head_dim == 64 ? emit(ctx, "attn_join", k_attn_join<64, 256>, grid, dim3(256), 0, a) : emit(ctx, "attn_join", k_attn_join<128, 256>, grid, dim3(256), 0, a);
}

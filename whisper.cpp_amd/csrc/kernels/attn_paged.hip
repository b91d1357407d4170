// Attention of one new token per stream over the paged K/V cache (include/mi355x_kernels.h: mi355x_attn_paged).
//     o = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q.k_j - max)
// Bound by the bytes of the keys and values, which every K/V head's workgroups read once for all the query heads that share it: up to 16 of them are
// the columns of one matrix product, so that grouped heads cost no more reads and no more instructions than single ones.
//
//   k_attn_paged   a workgroup = one query x one K/V head (x 16 query heads) x one share of the keys; its waves take the share's tiles of 32 keys in
//                  turn, each with its own running maximum and sum, and are joined in LDS at the end.
//                  S^T = K.Q^T and O^T = V^T.P^T on v_mfma_f32_16x16x32: a lane owns ONE head (column), so the softmax statistics are
//                  scalars of the lane and the P fragment feeds the second product straight from the registers (the order of the 32 keys inside the
//                  product is the same for both operands).  K goes from memory to registers as the operand lies (64 consecutive bytes of a key per
//                  instruction and 4 lanes), V through an area of LDS that belongs to the wave, read back transposed: no barrier in the loop, and the
//                  next tile's 16 KB are on their way while one is computed.
//   k_attn_join    joins the shares of one head where the keys were split.
//
// F32 queries are split into NT terms of the cache's type (2 x 11 or 3 x 8 bits), the weights likewise: the products are exact, the sums F32.  16-bit queries
// take one term; the weights are then rounded to 16 bits, half a step of the result's own type.
#include "kv_cache.h"

#define TILE 32                        // keys of a tile: one 16x16x32 product over keys
#define NEG_BIG (-3.0e38f)             // the running maximum's start: exp2(x - NEG_BIG) of a masked x = -inf is 0, not NaN

struct PagedArgs {
    kvc c;
    const int * seq;
    const char * q; int64_t q_nb1, q_nb2;
    char * o; int64_t o_nb1, o_nb2;
    float * part_o, * part_ml;         // [query][head][share][D], [..][2]: where the keys are split
    float c2;                          // scale * log2(e)
    int q_type, o_type, window;
    int G, H, groups;                  // query heads per K/V head, query heads, sets of 16 query heads per K/V head
    int shares, min_tiles;
    const int * cu_q, * cu_k;          // packed rows: as in PackedArgs
    int n, rows_q, rows_k, causal;
    int qt, hg;                        // queries of a tile of 16 rows, heads of the group that each has there: qt * hg <= 16
};

// the keys that query i sees, as [lo, hi), and the tiles of one share
struct paged_span { int s, lo, hi, per; };
__device__ __forceinline__ int tiles_of(const paged_span & p) { return p.hi > p.lo ? (p.hi + TILE - 1) / TILE - p.lo / TILE : 0; }
__device__ __forceinline__ paged_span span_of(const PagedArgs & a, int i) {
    paged_span r;
    r.s = a.seq ? a.seq[i] : i;
    int len = 0;
    if (r.s >= 0 && r.s < a.c.n_seq) len = a.c.len[r.s];
    const int64_t cap = (int64_t) a.c.max_pages << a.c.shift;
    r.hi = len < 0 ? 0 : len > cap ? (int) cap : len;
    r.lo = a.window > 0 && r.hi > a.window ? r.hi - a.window : 0;
    const int tiles = tiles_of(r);
    r.per = max((tiles + a.shares - 1) / a.shares, a.min_tiles);
    return r;
}
__device__ __forceinline__ int shares_of(const paged_span & p) { return (tiles_of(p) + p.per - 1) / p.per; }

// F32 values as NT terms of a 16-bit type: x = t0 + t1 (+ t2), each the rounding of what the ones before leave
template <typename O, int NT> __device__ __forceinline__ void split8(const float * f, typename O::vec8 * t) {
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        float r = f[e];
        #pragma unroll
        for (int n = 0; n < NT; n++) { t[n][e] = (typename O::elem) r; if (n + 1 < NT) r -= (float) t[n][e]; }
    }
}

// a 16-byte piece's place in a V row of LDS: the eight keys that one half of a transposing read touches lie in different banks
template <int D> __device__ __forceinline__ int v_piece(int key, int piece) {
    return D == 128 ? piece ^ ((key & 7) << 1) : piece ^ (((key >> 1) & 3) << 1);
}

enum { SMALL_PAGES, BIG_PAGES, ROWS };                   // where K and V lie: pages of fewer than 32 keys; 32 and more (a tile lies in one); packed rows

template <typename O, int D, int NT, int SRC, bool PACKED>
__global__ void __launch_bounds__(512, 2) k_attn_paged(const PagedArgs a) {
    typedef typename O::vec8 vec8;
    constexpr int KK = D / 32;                           // 32-dim pieces of a key
    constexpr int NV = D / 16;                           // V loads of a tile; 16-dim blocks of the result
    constexpr int RPL = 512 / D;                         // V rows per load
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, nl = lane & 15, g4 = lane >> 4, waves = blockDim.x >> 6;
    const int unit = blockIdx.x, grp = unit % a.groups, hk = unit / a.groups % a.c.Hkv, share = blockIdx.y;
    int i = unit / a.groups / a.c.Hkv;                   // the query; packed: the first query row of this workgroup
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
        sp.per = 1 << 30;
    } else sp = span_of(a, i);
    const int t0 = sp.lo / TILE + share * sp.per, t1 = tiles_of(sp) ? min(t0 + sp.per, (sp.hi + TILE - 1) / TILE) : t0;
    const int g0 = grp * 16, rows = PACKED ? nq * a.hg : min(16, a.G - g0), h0 = hk * a.G + g0;
    if (t0 >= t1 && (share > 0 || a.shares > 1)) return;             // (an empty sequence: k_attn_join writes its zeros, or this workgroup below)
    char * vl = lds + wave * (TILE * D * 2);
    // row r of the 16: query i + r / hg, head h0 + r % hg (one query: head h0 + r).  The keys that lane nl's row sees are first .. last.
    auto q_of = [&](int r) { return PACKED ? r / a.hg : 0; };
    auto h_of = [&](int r) { return PACKED ? r - r / a.hg * a.hg : r; };
    const bool here = nl < rows && g0 + h_of(nl) < a.G;
    const int ql = min(q_of(nl), nq - 1);
    const int last = PACKED && a.causal ? min(own + ql, sp.hi - 1) : sp.hi - 1, first = PACKED && a.window > 0 ? max(own + ql - a.window + 1, 0) : sp.lo;

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
    const int * row = a.c.table + (int64_t) max(sp.s, 0) * a.c.max_pages;
    const char * kb = a.c.k + hk * a.c.nb_head, * vb = a.c.v + hk * a.c.nb_head;
    // the page of each key of a tile, in lane key & 31.  Keys outside the span are replaced by the nearest inside: what no row sees is not read.
    bool bad = false;
    auto pages_of = [&](int t) {
        if (SRC == ROWS) return 0;
        const int key = min(max(t * TILE + (lane & 31), sp.lo), sp.hi - 1);
        int p = row[key >> a.c.shift];
        bad |= (unsigned) p >= (unsigned) a.c.n_pages;
        return min(max(p, 0), a.c.n_pages - 1);
    };
    auto place = [&](int key, int kl, int pg) -> int64_t {           // kl: the key's number in the tile
        if (SRC == ROWS) return (int64_t) (k0 + key) * a.c.nb_key;
        const int p = SRC == BIG_PAGES ? __builtin_amdgcn_readfirstlane(pg) : __shfl(pg, kl, 64);
        return p * a.c.nb_page + (key & a.c.mask) * a.c.nb_key;
    };
    vec8 kr[2][KK]; u32x4_t vr[NV];
    auto fetch_k = [&](int t, int pg) {
        #pragma unroll
        for (int b = 0; b < 2; b++) {
            const int key = min(max(t * TILE + 16 * b + nl, sp.lo), sp.hi - 1);
            const char * at = kb + place(key, 16 * b + nl, pg) + 16 * g4;
            #pragma unroll
            for (int kk = 0; kk < KK; kk++) kr[b][kk] = *(const vec8 *) (at + 64 * kk);
        }
    };
    auto fetch_v = [&](int t, int pg) {
        #pragma unroll
        for (int r = 0; r < NV; r++) {
            const int kl = r * RPL + lane / (D / 8), key = min(max(t * TILE + kl, sp.lo), sp.hi - 1);
            vr[r] = *(const u32x4_t *) (vb + place(key, kl, pg) + (lane % (D / 8)) * 16);
        }
    };

    floatx4 o[NV];
    #pragma unroll
    for (int d = 0; d < NV; d++) o[d] = floatx4{ 0, 0, 0, 0 };
    float m = NEG_BIG, l = 0.0f;
    int t = t0 + wave;
    if (t < t1) {
        int pg = pages_of(t);
        fetch_k(t, pg);
        fetch_v(t, pg);
        pg = pages_of(min(t + waves, t1 - 1));
        for (; t < t1; t += waves) {
            const bool more = t + waves < t1;
            floatx4 s[2];
            #pragma unroll
            for (int b = 0; b < 2; b++) {
                s[b] = floatx4{ 0, 0, 0, 0 };
                #pragma unroll
                for (int n = NT - 1; n >= 0; n--)
                    #pragma unroll
                    for (int kk = 0; kk < KK; kk++) s[b] = O::mfma16(kr[b][kk], qf[n][kk], s[b]);
            }
            if (more) fetch_k(t + waves, pg);
            // V into this wave's area.  Zero times an infinity or a NaN is none: where some row does not see all of the tile, they are taken out here,
            // and counted over the keys that each row sees below (rare: the next V tile waits for it).
            bool odd = false;
            if (PACKED && (t * TILE + TILE - 1 > (a.causal ? own : sp.hi - 1) || (a.window > 0 && t * TILE < own + nq - a.window))) {
                uint32_t nf = 0;
                #pragma unroll
                for (int r = 0; r < NV; r++) nf |= not_finite8<O>(vr[r]);
                odd = __any(nf != 0);
            }
            auto put_v = [&](int what) {                             // 0: as it is, 1: without what is not finite, 2: what that was
                #pragma unroll
                for (int r = 0; r < NV; r++) {
                    const int kl = r * RPL + lane / (D / 8);
                    u32x4_t x = vr[r], kind = { 0, 0, 0, 0 };
                    if (what) take_apart<O>(x, kind);
                    *(u32x4_t *) (vl + kl * (D * 2) + v_piece<D>(kl, lane % (D / 8)) * 16) = what == 2 ? kind : x;
                }
            };
            if (PACKED && odd) put_v(1); else put_v(0);
            if (more && !odd) {
                fetch_v(t + waves, pg);
                pg = pages_of(min(t + 2 * waves, t1 - 1));
            }
            // softmax: element r of block b is key 16 b + 4 g4 + r of head nl
            float x[8], top = NEG_BIG;
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = t * TILE + 16 * (e >> 2) + 4 * g4 + (e & 3);
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
            const float shift = sizeof(typename O::elem) == 2 && __is_same(O, f16_ops) ? m - 15.0f : m;
            float p[8];
            #pragma unroll
            for (int e = 0; e < 8; e++) { p[e] = __builtin_amdgcn_exp2f(x[e] - shift); l += p[e]; }
            vec8 pf[NT];
            split8<O, NT>(p, pf);
            // V^T as the first operand: this 16-lane group's keys 4 g4 + {0..3} and 16 + 4 g4 + {0..3}, dims 16 d + {0..15}
            auto v_frag = [&](int d) {
                vec8 vf;
                #pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int key = 16 * b + 4 * g4 + (nl >> 2);
                    const char * at = vl + key * (D * 2) + v_piece<D>(key, 2 * d + ((nl >> 1) & 1)) * 16 + (nl & 1) * 8;
                    const short4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t *) at);
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
                put_v(2);
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
                    pg = pages_of(min(t + 2 * waves, t1 - 1));
                }
            }
        }
    }
    if (SRC != ROWS && __any(bad) && lane == 0) atomicOr((unsigned *) a.c.status, MI355X_KV_BAD_ARG);
    l += lane_xor16(l);
    l += lane_xor32(l);

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
        if (a.shares == 1) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            store4(a.o + (int64_t) (i + q_of(h)) * a.o_nb2 + (int64_t) (h0 + h_of(h)) * a.o_nb1 + d * (a.o_type == MI355X_TYPE_F32 ? 4 : 2), a.o_type, r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv);
        } else {
            const int64_t rec = ((int64_t) i * a.H + h0 + h) * a.shares + share;
            *(floatx4 *) (a.part_o + rec * D + d) = r;
            if (d == 0) { a.part_ml[rec * 2] = M; a.part_ml[rec * 2 + 1] = L; }
        }
    }
}

// one workgroup = one query x one head: D/4 threads per share
template <int D>
__global__ void __launch_bounds__(256) k_attn_join(const PagedArgs a) {
    constexpr int L4 = D / 4, NG = 256 / L4;
    __shared__ float red[NG][D + 4];
    __shared__ float lsum[NG];
    const int h = blockIdx.x % a.H, i = blockIdx.x / a.H, g = threadIdx.x / L4, d = threadIdx.x % L4 * 4;
    const paged_span sp = span_of(a, i);
    const int n = shares_of(sp);
    const int64_t rec = ((int64_t) i * a.H + h) * a.shares;
    float M = NEG_BIG;
    for (int s = 0; s < n; s++) M = fmaxf(M, a.part_ml[(rec + s) * 2]);
    float L = 0.0f;
    floatx4 r = { 0, 0, 0, 0 };
    for (int s = g; s < n; s += NG) {
        const float f = __builtin_amdgcn_exp2f(a.part_ml[(rec + s) * 2] - M);
        const floatx4 x = *(const floatx4 *) (a.part_o + (rec + s) * D + d);
        L += f * a.part_ml[(rec + s) * 2 + 1];
        #pragma unroll
        for (int e = 0; e < 4; e++) r[e] += f * x[e];
    }
    *(floatx4 *) &red[g][d] = r;
    if (d == 0) lsum[g] = L;
    __syncthreads();
    if (g > 0) return;
    for (int w = 1; w < NG; w++) {
        L += lsum[w];
        const floatx4 x = *(const floatx4 *) &red[w][d];
        #pragma unroll
        for (int e = 0; e < 4; e++) r[e] += x[e];
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    store4(a.o + (int64_t) i * a.o_nb2 + (int64_t) h * a.o_nb1 + d * (a.o_type == MI355X_TYPE_F32 ? 4 : 2), a.o_type, r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv);
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
// shares of the keys: enough workgroups for the chip, of at least 512 keys each
static int paged_shares(const mi355x_kv_cache * c, int n, int n_head, int max_len) {
    const int64_t cap = (int64_t) c->max_pages * c->page_size;
    int64_t len = max_len > 0 && max_len < cap ? max_len : cap;
    const int G = n_head / c->n_head_kv;
    const int64_t units = (int64_t) n * c->n_head_kv * ((G + 15) / 16);
    int64_t by_len = (len + 511) / 512, by_units = 2048 / (units > 0 ? units : 1);
    if (by_units < 1) by_units = 1;
    int64_t s = by_len < by_units ? by_len : by_units;
    if (s < (len + 2047) / 2048) s = (len + 2047) / 2048;            // ragged batches: one long sequence must not be one workgroup's
    return (int) (s > 256 ? 256 : s < 1 ? 1 : s);
}
extern "C" size_t mi355x_attn_paged_work_bytes(const mi355x_kv_cache * c, int n, int n_head, int max_len) {
    if (!c || n < 1 || n_head < 1 || c->n_head_kv < 1 || n_head % c->n_head_kv || c->page_size < 1 || c->max_pages < 1 || c->head_dim < 1) return 0;
    const int s = paged_shares(c, n, n_head, max_len);
    return s == 1 ? 0 : (size_t) n * n_head * s * (c->head_dim + 2) * 4;
}

template <typename O, int D, int NT, int SRC, bool PACKED>
static int launch_as(mi355x_ctx * ctx, const PagedArgs & a, int64_t blocks, int threads) {
    const uint32_t v = (uint32_t) (threads / 64 * TILE * D * 2), j = (uint32_t) (threads / 64 * (32 + 16 * (D + 4)) * 4), lds = v > j ? v : j;
    static std::atomic<uint64_t> allowed{0};
    const int rl = kv_allow_lds(ctx, (const void *) k_attn_paged<O, D, NT, SRC, PACKED>, lds, allowed);
    return rl ? rl : emit(ctx, PACKED ? "attn_packed" : "attn_paged", k_attn_paged<O, D, NT, SRC, PACKED>, dim3((uint32_t) blocks, (uint32_t) a.shares), dim3(threads), lds, a);
}
template <typename O, int D, int NT>
static int launch_paged(mi355x_ctx * ctx, const PagedArgs & a, int n, int threads) {
    const int64_t blocks = (int64_t) n * a.c.Hkv * a.groups;
    return a.c.shift >= 5 ? launch_as<O, D, NT, BIG_PAGES, false>(ctx, a, blocks, threads) : launch_as<O, D, NT, SMALL_PAGES, false>(ctx, a, blocks, threads);
}
template <typename O, int D>
static int launch_few(mi355x_ctx * ctx, const PagedArgs & a, bool paged) {
    const int64_t blocks = ((int64_t) a.rows_q / a.qt + a.n) * a.c.Hkv * a.groups;
    if (blocks > INT32_MAX) return kv_refuse("attn_packed: too many rows for one launch");
    if (!paged) return launch_as<O, D, 1, ROWS, true>(ctx, a, blocks, 512);
    return a.c.shift >= 5 ? launch_as<O, D, 1, BIG_PAGES, true>(ctx, a, blocks, 512) : launch_as<O, D, 1, SMALL_PAGES, true>(ctx, a, blocks, 512);
}
int mi355x_attn_few_rows(mi355x_ctx * ctx, const PackedArgs & p, int type, int dim, bool paged) {
    PagedArgs a; memset(&a, 0, sizeof(a));
    a.c = p.c; a.c.Hkv = p.Hkv; a.seq = p.seq;
    a.q = p.q; a.q_nb1 = p.q_nb1; a.q_nb2 = p.q_nb2; a.q_type = p.q_type;
    a.o = p.o; a.o_nb1 = p.o_nb1; a.o_nb2 = p.o_nb2; a.o_type = p.o_type;
    a.c2 = p.flip ? -p.c2 : p.c2; a.window = p.window; a.G = p.G; a.H = p.G * p.Hkv; a.groups = (p.G + 15) / 16; a.shares = 1; a.min_tiles = 1 << 30;
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
    if (n > INT32_MAX / 32768 || n * H > INT32_MAX / 8) return kv_refuse("attn_paged: too many queries");
    if (!d->seq && n > c->n_seq) return kv_refuse("attn_paged: more queries than sequences");
    if ((uintptr_t) d->seq % 4 || d->window < 0 || d->max_len < 0) return kv_refuse("attn_paged: seq, window or max_len");
    if (n == 0) return 0;
    const device_scope scope(ctx);
    a.seq = d->seq;
    a.q = (const char *) d->q.data; a.q_nb1 = d->q.nb[1]; a.q_nb2 = d->q.nb[2]; a.q_type = d->q.type;
    a.o = (char *) d->dst.data; a.o_nb1 = d->dst.nb[1]; a.o_nb2 = d->dst.nb[2]; a.o_type = d->dst.type;
    a.c2 = d->scale * 1.4426950408889634f; a.window = d->window;
    a.H = (int) H; a.G = (int) (H / c->n_head_kv); a.groups = (a.G + 15) / 16;
    a.shares = paged_shares(c, (int) n, (int) H, d->max_len);
    a.min_tiles = a.shares == 1 ? 1 << 30 : 8;
    const size_t need = a.shares == 1 ? 0 : (size_t) n * H * a.shares * (c->head_dim + 2) * 4;
    if (need) {
        if (!d->work || d->work_bytes < need || (uintptr_t) d->work % 16) return kv_refuse("attn_paged: the work area is missing, too small or misaligned");
        a.part_o = (float *) d->work;
        a.part_ml = a.part_o + (size_t) n * H * a.shares * c->head_dim;
    }
    const int threads = a.shares == 1 ? 512 : 256;
    const bool f16 = c->type == MI355X_TYPE_F16, one = d->q.type == c->type;
    int e;
    if (c->head_dim == 64) e = f16 ? (one ? launch_paged<f16_ops, 64, 1>(ctx, a, (int) n, threads) : launch_paged<f16_ops, 64, 2>(ctx, a, (int) n, threads))
                                   : (one ? launch_paged<bf16_ops, 64, 1>(ctx, a, (int) n, threads) : launch_paged<bf16_ops, 64, 3>(ctx, a, (int) n, threads));
    else                   e = f16 ? (one ? launch_paged<f16_ops, 128, 1>(ctx, a, (int) n, threads) : launch_paged<f16_ops, 128, 2>(ctx, a, (int) n, threads))
                                   : (one ? launch_paged<bf16_ops, 128, 1>(ctx, a, (int) n, threads) : launch_paged<bf16_ops, 128, 3>(ctx, a, (int) n, threads));
    if (e || a.shares == 1) return e;
    const dim3 grid((uint32_t) (n * H));
    return c->head_dim == 64 ? emit(ctx, "attn_join", k_attn_join<64>, grid, dim3(256), 0, a) : emit(ctx, "attn_join", k_attn_join<128>, grid, dim3(256), 0, a);
}

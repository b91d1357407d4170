// Causal attention of packed sequences with grouped heads (include/mi355x_kernels.h: mi355x_attn_packed), over their own keys or over the paged cache.
//     o_r = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q_r.k_j - max),   j <= L - Q + r   (and j > L - Q + r - window)
// Bound by the matrix cores (4 D flop per row and key) and by the exponentials (one per row and key, a quarter of the VALU's rate): at 128 dims a
// 32 x 64 tile is 1024 cycles of matrix instructions beside ~930 of vector work, at 64 dims 512 beside ~900.
//
//   k_attn_packed  a workgroup = up to 256 rows of one K/V head: a row is (query, head of the group), query-major, so that grouped heads share every K/V
//                  tile and the causal edge stays as narrow as one query's.  8 waves x 32 rows, 64-key tiles that all waves share in LDS.
//                  S^T = K.Q^T and O^T = V^T.P^T on v_mfma_f32_32x32x16: a lane owns one row, so maximum, sum and rescaling are the lane's own scalars,
//                  and P goes from registers to the second product.  K and V rows lie in LDS as they come, 16-byte pieces permuted so that neither the
//                  row reads (K) nor the transposing reads (V) meet in a bank.  The two waves of a SIMD run half a step apart, one in the matrix products
//                  (PV of the tile before, QK of this one) while the other is in the softmax: 8192 rows, 32 / 8 heads of 128, BF16: 595 us = 923
//                  TFLOP/s (both waves in step, and LDS rows at 8-byte addresses: 1555 us).
// A masked weight is an exact zero, but zero times an infinity or a NaN is none: where a tile that is masked in part holds such values, they are taken
// out on the way into LDS and counted over the keys that a row sees, so that a row never meets what it does not see.
#include "kv_cache.h"

#define KT 64                          // keys of a tile

struct PackedArgs {
    kvc c;                             // PAGED: the cache.  Otherwise k, v and their strides in nb_key (rows) and nb_head
    const char * q; int64_t q_nb1, q_nb2;
    char * o; int64_t o_nb1, o_nb2;
    const int * cu_q, * cu_k, * seq;
    float c2; int flip;                // |scale| * log2(e), at least 1e-37; whether the scale is negative (the queries change sign)
    int n, rows_q, rows_k, q_type, o_type, causal, window;
    int G, Hkv, qt;                    // query heads per K/V head; queries of a workgroup
};

// slot -> (sequence, tile of its rows): sequence i has the slots cu[i]/qt + i .. cu[i+1]/qt + i, at least as many as its tiles, found by bisection
struct packed_job { int i, r0, nq, L, tile; };
__device__ __forceinline__ bool packed_find(const PackedArgs & a, int slot, packed_job & j) {
    int lo = 0, hi = a.n;
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (a.cu_q[m] / a.qt + m <= slot) lo = m; else hi = m; }
    j.i = lo;
    j.r0 = a.cu_q[lo]; const int r1 = a.cu_q[lo + 1];
    if (j.r0 < 0 || r1 > a.rows_q || r1 <= j.r0) return false;
    j.nq = r1 - j.r0;
    const int tiles = (j.nq + a.qt - 1) / a.qt, t = slot - (j.r0 / a.qt + lo);
    if (t < 0 || t >= tiles) return false;
    j.tile = tiles - 1 - t;                                          // the rows with most keys first
    return true;
}

template <typename O, int D> __device__ __forceinline__ int k_piece(int key, int piece) { return D == 128 ? piece ^ (key & 15) : piece ^ ((key >> 1) & 7); }
template <int D> __device__ __forceinline__ int v_slot(int key, int piece) { return D == 128 ? piece ^ ((key & 3) << 2) : piece ^ (((key >> 1) & 1) << 2); }

// bit 15 of each half: whether it is an infinity or a NaN
template <typename O> __device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
    return ((w & 0x7FFF7FFFu) + (__is_same(O, f16_ops) ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
template <typename O> __device__ __forceinline__ uint32_t not_finite8(u32x4_t w) { return not_finite2<O>(w[0]) | not_finite2<O>(w[1]) | not_finite2<O>(w[2]) | not_finite2<O>(w[3]); }

// infinities and NaNs out of eight values: zeros in their places, and what they were as numbers of the type: 1 (inf), 128 (-inf), 16384 (NaN)
template <typename O> __device__ __forceinline__ void take_apart(u32x4_t & v, u32x4_t & kind) {
    constexpr bool F = __is_same(O, f16_ops);
    #pragma unroll
    for (int w = 0; w < 4; w++)
        #pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const uint32_t x = v[w] >> h & 0xFFFF, top = F ? 0x7C00 : 0x7F80;
            if ((x & top) != top) continue;
            kind[w] |= ((x & 0x7FFF) != top ? (F ? 0x7400u : 0x4680u) : x & 0x8000 ? (F ? 0x5800u : 0x4300u) : (F ? 0x3C00u : 0x3F80u)) << h;
            v[w] &= ~(0xFFFFu << h);
        }
}

#define SLOTS 3                        // K tiles t .. t+2, V tiles t-1 .. t+1 are in use at a time

template <typename O, int D, bool PAGED>
__global__ void __launch_bounds__(512, 2) k_attn_packed(const PackedArgs a) {
    typedef typename O::vec8 vec8;
    typedef typename O::elem elem;
    constexpr int KK = D / 16, NI = D / 32;
    constexpr int PCS = D / 8;                                        // 16-byte pieces of a row
    constexpr int NL = KT * PCS / 512, RPL = 512 / PCS;               // pieces per thread and tile, K and V each; keys that lie between them
    constexpr int TILE_B = KT * D * 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];                                     // SLOTS K tiles, SLOTS V tiles, SLOTS tiles of what was taken out of V
    __shared__ int odd[SLOTS];                                        // t + 1: something was taken out of V tile t
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hf = lane >> 5;
    const int hk = blockIdx.x % a.Hkv, slot = blockIdx.x / a.Hkv;
    packed_job job;
    if (!packed_find(a, slot, job)) return;
    int k0 = 0, L = 0;
    const int * row = nullptr;
    if (PAGED) {
        const int s = a.seq ? a.seq[job.i] : job.i;
        if (s >= 0 && s < a.c.n_seq) {
            const int64_t cap = (int64_t) a.c.max_pages << a.c.shift;
            const int len = a.c.len[s];
            L = len < 0 ? 0 : len > cap ? (int) cap : len;
            row = a.c.table + (int64_t) s * a.c.max_pages;
        }
    } else {
        k0 = a.cu_k[job.i]; const int k1 = a.cu_k[job.i + 1];
        if (k0 >= 0 && k1 <= a.rows_k && k1 > k0) L = k1 - k0;
    }
    // this lane's row
    const int q_base = job.tile * a.qt, nrow = min(a.qt, job.nq - q_base) * a.G, r = wave * 32 + (lane & 31);
    const int rc = min(r, nrow - 1), qi = q_base + rc / a.G, g = rc - rc / a.G * a.G;
    const int off = L - job.nq;                                       // row qi's own key is off + qi
    const int last = a.causal ? min(off + qi, L - 1) : L - 1;         // the last key it sees (-1: none)
    const int first = a.window > 0 ? max(off + qi - a.window + 1, 0) : 0;
    // the same for the wave's first and last row and for the workgroup's: uniform
    const int wr0 = min(wave * 32, nrow - 1), wr1 = min(wave * 32 + 31, nrow - 1), wq0 = q_base + wr0 / a.G, wq1 = q_base + wr1 / a.G, bq1 = q_base + (nrow - 1) / a.G;
    const int w_last_min = a.causal ? min(off + wq0, L - 1) : L - 1, w_last = a.causal ? min(off + wq1, L - 1) : L - 1;
    const int w_first = a.window > 0 ? max(off + wq0 - a.window + 1, 0) : 0, w_first_max = a.window > 0 ? max(off + wq1 - a.window + 1, 0) : 0;
    const int b_last_min = a.causal ? min(off + q_base, L - 1) : L - 1, b_last = a.causal ? min(off + bq1, L - 1) : L - 1;
    const int b_first = a.window > 0 ? max(off + q_base - a.window + 1, 0) : 0, b_first_max = a.window > 0 ? max(off + bq1 - a.window + 1, 0) : 0;
    const int T0 = b_first / KT, T = b_last >= b_first && L > 0 ? b_last / KT + 1 - T0 : 0;          // tiles T0 .. T0 + T - 1
    // tiles that this wave's rows see nothing of are passed over; the rest of its tiles are t_lo .. t_hi - 1
    const int t_lo = max(w_first / KT - T0, 0), t_hi = wave * 32 < nrow && w_last >= w_first ? min(w_last / KT + 1 - T0, T) : 0;

    vec8 qf[KK];
    {
        const char * qp = a.q + (int64_t) (job.r0 + qi) * a.q_nb2 + (int64_t) (hk * a.G + g) * a.q_nb1;
        #pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            float f[8];
            load8(qp + (16 * kk + 8 * hf) * (a.q_type == MI355X_TYPE_F32 ? 4 : 2), a.q_type, f);
            #pragma unroll
            for (int e = 0; e < 8; e++) qf[kk][e] = (elem) (a.flip ? -f[e] : f[e]);
        }
    }
    floatx16 o[NI], s[2];
    vec8 pf[4];
    #pragma unroll
    for (int i = 0; i < NI; i++)
        #pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // staging: thread -> key tid / PCS (+ RPL), piece tid % PCS.  Keys outside what the workgroup sees are replaced by the nearest inside: never read.
    const int skey = tid / PCS, spc = tid % PCS;
    const char * kb = a.c.k + hk * a.c.nb_head + spc * 16, * vb = a.c.v + hk * a.c.nb_head + spc * 16;
    bool bad = false;
    u32x4_t kr[NL], vr[NL];
    int pg_k[NL], pg_v[NL], pg_n[NL];                                 // pages of the K tile and of the V tile that are fetched next, and of the tile behind
    auto key_of = [&](int t, int e) { return min(max((T0 + t) * KT + skey + e * RPL, b_first), b_last); };
    auto page_of = [&](int t, int * pg) {
        if (PAGED) {
            #pragma unroll
            for (int e = 0; e < NL; e++) pg[e] = row[key_of(t, e) >> a.c.shift];
        }
    };
    auto place = [&](int t, int e, const int * pg) -> int64_t {
        const int key = key_of(t, e);
        if (!PAGED) return (int64_t) (k0 + key) * a.c.nb_key;
        bad |= (unsigned) pg[e] >= (unsigned) a.c.n_pages;
        return min(max(pg[e], 0), a.c.n_pages - 1) * a.c.nb_page + (key & a.c.mask) * a.c.nb_key;
    };
    auto fetch_k = [&](int t, const int * pg) {
        #pragma unroll
        for (int e = 0; e < NL; e++) kr[e] = *(const u32x4_t *) (kb + place(t, e, pg));
    };
    auto fetch_v = [&](int t, const int * pg) {
        #pragma unroll
        for (int e = 0; e < NL; e++) vr[e] = *(const u32x4_t *) (vb + place(t, e, pg));
    };
    auto put_k = [&](int t) {
        char * kl = lds + t % SLOTS * TILE_B;
        #pragma unroll
        for (int e = 0; e < NL; e++) *(u32x4_t *) (kl + (skey + e * RPL) * (D * 2) + k_piece<O, D>(skey + e * RPL, spc) * 16) = kr[e];
    };
    auto put_v = [&](int t) {
        char * vl = lds + (SLOTS + t % SLOTS) * TILE_B;
        const bool edge = (T0 + t) * KT + KT - 1 > b_last_min || (T0 + t) * KT < b_first_max;         // masked in part for some row
        #pragma unroll
        for (int e = 0; e < NL; e++) {
            const int at = (skey + e * RPL) * (D * 2) + v_slot<D>(skey + e * RPL, spc) * 16;
            if (edge) {
                u32x4_t kind = { 0, 0, 0, 0 };
                if (not_finite8<O>(vr[e])) { take_apart<O>(vr[e], kind); odd[t % SLOTS] = t + 1; }    // every writer writes the same; what an older tile left does not match
                *(u32x4_t *) (vl + SLOTS * TILE_B + at) = kind;
            }
            *(u32x4_t *) (vl + at) = vr[e];
        }
    };
    auto part = [&](int t) { return (T0 + t) * KT + KT - 1 > w_last_min || (T0 + t) * KT < w_first_max; };

    // S^T = K.Q^T: element e of block b is key 32 b + (e & 3) + 8 (e >> 2) + 4 hf of the tile
    auto qk = [&](int t) {
        const char * kl = lds + t % SLOTS * TILE_B;
        #pragma unroll
        for (int b = 0; b < 2; b++)
            #pragma unroll
            for (int e = 0; e < 16; e++) s[b][e] = 0.0f;
        vec8 kf[2][2];                                                // the next products' operands are read while these run
        auto get = [&](int kk) {
            #pragma unroll
            for (int b = 0; b < 2; b++) {
                const int key = b * 32 + (lane & 31);
                kf[kk & 1][b] = *(const vec8 *) (kl + key * (D * 2) + k_piece<O, D>(key, kk * 2 + hf) * 16);
            }
        };
        get(0);
        #pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 1 < KK) get(kk + 1);
            #pragma unroll
            for (int b = 0; b < 2; b++) s[b] = O::mfma32(kf[kk & 1][b], qf[kk], s[b]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // V^T's operand for keys 16 c .. +15 (this lane's 16-lane group: 16 c + 4 hf + {0..3} and + 8), dims 32 i .. +31
    auto v_frag = [&](const char * vl, int c, int i) {
        const int li = lane & 15;
        vec8 vf;
        #pragma unroll
        for (int b = 0; b < 2; b++) {
            const int key = 16 * c + 4 * hf + (li >> 2) + 8 * b;
            const char * at = vl + key * (D * 2) + v_slot<D>(key, 4 * i + 2 * ((lane >> 4) & 1) + ((li >> 1) & 1)) * 16 + (li & 1) * 8;
            const short4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t *) at);
            __builtin_memcpy((char *) &vf + 8 * b, &x, 8);
        }
        return vf;
    };
    // O^T += V^T.P^T
    auto pv = [&](int t) {
        const char * vl = lds + (SLOTS + t % SLOTS) * TILE_B;
        vec8 vf[2][NI];
        #pragma unroll
        for (int i = 0; i < NI; i++) vf[0][i] = v_frag(vl, 0, i);
        #pragma unroll
        for (int c = 0; c < 4; c++) {
            #pragma unroll
            for (int i = 0; i < NI; i++) if (c + 1 < 4) vf[(c + 1) & 1][i] = v_frag(vl, c + 1, i);
            #pragma unroll
            for (int i = 0; i < NI; i++) o[i] = O::mfma32(vf[c & 1][i], pf[c], o[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_amdgcn_readfirstlane(odd[t % SLOTS]) != t + 1) return;
        // what was taken out of this tile, for the rows that see it: over the visible keys, how many of each kind
        const int hi = last - (T0 + t) * KT - 4 * hf, lo = first - (T0 + t) * KT - 4 * hf;
        #pragma unroll
        for (int i = 0; i < NI; i++) {
            floatx16 cnt;
            #pragma unroll
            for (int e = 0; e < 16; e++) cnt[e] = 0.0f;
            #pragma unroll
            for (int c = 0; c < 4; c++) {
                vec8 seen;
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int k = 16 * c + (e & 3) + 8 * (e >> 2);
                    seen[e] = (elem) (k > hi || k < lo ? 0.0f : 1.0f);
                }
                cnt = O::mfma32(v_frag(vl + SLOTS * TILE_B, c, i), seen, cnt);
                __builtin_amdgcn_sched_barrier(0);
            }
            #pragma unroll
            for (int e = 0; e < 16; e++) {
                const int n = (int) cnt[e];                           // NaNs x 16384 + (-inf)s x 128 + (+inf)s, at most 64 of each
                o[i][e] += ((n & 127) ? INFINITY : 0.0f) + ((n & 0x3F80) ? -INFINITY : 0.0f) + (n >= 16384 ? NAN : 0.0f);
            }
        }
    };
    // P^T from S^T, with the running maximum and sum.  The maximum follows only when a row's grows by more than 2^8 in its weights, so that O is
    // hardly ever rescaled; F16 weights are held times 2^7 (2^15 at most), so that small ones do not fall below its range.  Both cancel against the sum.
    auto softmax = [&](int t) {
        if (part(t)) {
            const int hi = last - (T0 + t) * KT - 4 * hf, lo = first - (T0 + t) * KT - 4 * hf;
            #pragma unroll
            for (int b = 0; b < 2; b++)
                #pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int k = 32 * b + (e & 3) + 8 * (e >> 2);
                    if (k > hi || k < lo) s[b][e] = -INFINITY;
                }
        }
        float top = fmaxf(s[0][0], s[0][1]);
        #pragma unroll
        for (int e = 2; e < 32; e += 2) top = fmaxf(fmaxf(top, s[e >> 4][e & 15]), s[(e + 1) >> 4][(e + 1) & 15]);
        top = fmaxf(top, lane_xor32(top));
        if (__any((top - m) * a.c2 > 8.0f)) {
            const float mn = fmaxf(m, top), alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * a.c2);
            m = mn; l *= alpha;
            #pragma unroll
            for (int i = 0; i < NI; i++)
                #pragma unroll
                for (int e = 0; e < 16; e++) o[i][e] *= alpha;
        }
        const float mc = (m == -INFINITY ? 0.0f : m * a.c2) - (__is_same(O, f16_ops) ? 7.0f : 0.0f);
        float sum = 0.0f;
        #pragma unroll
        for (int b = 0; b < 2; b++)
            #pragma unroll
            for (int e = 0; e < 16; e++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], a.c2, -mc));
                sum += p;
                pf[2 * b + (e >> 3)][e & 7] = (elem) p;
            }
        l += sum;
    };

    if (T > 0) {
        // Two groups of four waves, one of each on every SIMD, half a step apart: while one runs the matrix products of a step (PV of the tile before, QK
        // of this one), the other runs the softmax and brings tiles in.  A barrier ends each half step.
        const bool second = wave >= 4;
        if (tid < SLOTS) odd[tid] = 0;
        page_of(0, pg_k);
        page_of(min(1, T - 1), pg_n);
        fetch_k(0, pg_k);
        fetch_v(0, pg_k);
        put_k(0);
        fetch_k(min(1, T - 1), pg_n);
        __syncthreads();                                              // odd[] cleared
        put_v(0);
        put_k(1);
        #pragma unroll
        for (int e = 0; e < NL; e++) pg_v[e] = pg_n[e];               // V tile 1, K tile 2 next
        page_of(min(2, T - 1), pg_k);
        fetch_v(min(1, T - 1), pg_v);
        fetch_k(min(2, T - 1), pg_k);
        page_of(min(3, T - 1), pg_n);
        __syncthreads();
        if (second) __syncthreads();
        for (int t = 0; t < T; t++) {
            if (t > t_lo && t <= t_hi) pv(t - 1);
            if (t >= t_lo && t < t_hi) qk(t);
            __syncthreads();
            if (t + 2 < T) put_k(t + 2);
            if (t + 1 < T) put_v(t + 1);
            if (t + 3 < T) {
                #pragma unroll
                for (int e = 0; e < NL; e++) { pg_v[e] = pg_k[e]; pg_k[e] = pg_n[e]; }
                fetch_k(t + 3, pg_k);
                page_of(min(t + 4, T - 1), pg_n);
                fetch_v(t + 2, pg_v);
            } else if (t + 2 < T) fetch_v(t + 2, pg_k);
            if (t >= t_lo && t < t_hi) softmax(t);
            if (!second || t + 1 < T) __syncthreads();
        }
        if (t_hi == T && t_hi > t_lo) pv(T - 1);
    }
    if (PAGED && __any(bad) && lane == 0) atomicOr((unsigned *) a.c.status, MI355X_KV_BAD_ARG);
    l += lane_xor32(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (r < nrow) {
        char * op = a.o + (int64_t) (job.r0 + qi) * a.o_nb2 + (int64_t) (hk * a.G + g) * a.o_nb1;
        #pragma unroll
        for (int i = 0; i < NI; i++)
            #pragma unroll
            for (int e = 0; e < 4; e++)
                store4(op + (32 * i + 8 * e + 4 * hf) * (a.o_type == MI355X_TYPE_F32 ? 4 : 2), a.o_type, o[i][4*e] * inv, o[i][4*e+1] * inv, o[i][4*e+2] * inv, o[i][4*e+3] * inv);
    }
}

template <typename O, int D, bool PAGED>
static int launch_packed(mi355x_ctx * ctx, const PackedArgs & a, int64_t blocks) {
    static std::atomic<uint64_t> allowed{0};
    const uint32_t lds = 3 * SLOTS * KT * D * 2;
    const int rl = kv_allow_lds(ctx, (const void *) k_attn_packed<O, D, PAGED>, lds + 1024, allowed);
    if (rl) return rl;
    return emit(ctx, "attn_packed", k_attn_packed<O, D, PAGED>, dim3((uint32_t) blocks), dim3(512), lds, a);
}

extern "C" int mi355x_attn_packed(mi355x_ctx * ctx, const mi355x_attn_packed_desc * d) {
    if (!ctx || !d) return kv_refuse("attn_packed: a NULL argument");
    PackedArgs a; memset(&a, 0, sizeof(a));
    int type, dim; int64_t Hkv;
    if (d->cache) {
        const int rc = kv_view(d->cache, &a.c);
        if (rc) return rc;
        type = d->cache->type; dim = d->cache->head_dim; Hkv = d->cache->n_head_kv;
        if (!d->seq && d->n > d->cache->n_seq) return kv_refuse("attn_packed: more entries than sequences");
    } else {
        type = d->k.type; dim = (int) d->k.ne[0]; Hkv = d->k.ne[1];
        if ((type != MI355X_TYPE_F16 && type != MI355X_TYPE_BF16) || (d->k.ne[0] != 64 && d->k.ne[0] != 128) || Hkv < 1 || Hkv > 32768) return kv_refuse("attn_packed: k and v are F16 or BF16, [64 or 128, n_head_kv, rows]");
        if (!kv_rows_ok(&d->k, dim, Hkv) || !kv_rows_ok(&d->v, dim, Hkv) || d->v.type != type || d->v.ne[2] != d->k.ne[2]) return kv_refuse("attn_packed: v has another shape or type than k, or they are misaligned");
        if (d->k.nb[1] != d->v.nb[1] || d->k.nb[2] != d->v.nb[2]) return kv_refuse("attn_packed: k and v have other strides");
        a.c.k = (char *) d->k.data; a.c.v = (char *) d->v.data; a.c.nb_head = d->k.nb[1]; a.c.nb_key = d->k.nb[2];
        a.rows_k = (int) d->k.ne[2];
    }
    const int64_t H = d->q.ne[1], rows = d->q.ne[2];
    if (H < 1 || H % Hkv || H / Hkv > 128) return kv_refuse("attn_packed: the query heads are no multiple (up to 128) of the K/V heads");
    if (!kv_rows_ok(&d->q, dim, H) || !kv_rows_ok(&d->dst, dim, H) || d->dst.ne[2] != rows) return kv_refuse("attn_packed: q and dst are [head_dim, n_head, rows], F32 / F16 / BF16, 16-byte aligned");
    if (d->n < 0 || d->window < 0 || d->max_q < 0) return kv_refuse("attn_packed: n, window or max_q");
    if (d->n == 0 || rows == 0) return 0;
    if (!d->cu_q || ((uintptr_t) d->cu_q | (uintptr_t) d->cu_k | (uintptr_t) d->seq) % 4) return kv_refuse("attn_packed: cu_q, cu_k or seq");
    const device_scope scope(ctx);
    a.q = (const char *) d->q.data; a.q_nb1 = d->q.nb[1]; a.q_nb2 = d->q.nb[2]; a.q_type = d->q.type;
    a.o = (char *) d->dst.data; a.o_nb1 = d->dst.nb[1]; a.o_nb2 = d->dst.nb[2]; a.o_type = d->dst.type;
    a.cu_q = d->cu_q; a.cu_k = d->cu_k ? d->cu_k : d->cu_q; a.seq = d->seq;
    a.c2 = fmaxf(fabsf(d->scale) * 1.4426950408889634f, 1e-37f); a.flip = d->scale < 0.0f; a.n = d->n; a.rows_q = (int) rows; a.causal = d->causal != 0; a.window = d->window;
    a.G = (int) (H / Hkv); a.Hkv = (int) Hkv; a.qt = 256 / a.G;
    const int64_t blocks = (rows / a.qt + d->n) * Hkv;
    if (blocks > INT32_MAX) return kv_refuse("attn_packed: too many rows for one launch");
    const bool f16 = type == MI355X_TYPE_F16, paged = d->cache != nullptr;
    if (dim == 64) return f16 ? (paged ? launch_packed<f16_ops, 64, true>(ctx, a, blocks) : launch_packed<f16_ops, 64, false>(ctx, a, blocks))
                              : (paged ? launch_packed<bf16_ops, 64, true>(ctx, a, blocks) : launch_packed<bf16_ops, 64, false>(ctx, a, blocks));
    return f16 ? (paged ? launch_packed<f16_ops, 128, true>(ctx, a, blocks) : launch_packed<f16_ops, 128, false>(ctx, a, blocks))
               : (paged ? launch_packed<bf16_ops, 128, true>(ctx, a, blocks) : launch_packed<bf16_ops, 128, false>(ctx, a, blocks));
}

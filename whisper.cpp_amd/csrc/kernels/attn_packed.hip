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
//                  (PV of the tile before, QK of this one) while the other is in the softmax: 8192 rows, 32 / 8 heads of 128, BF16: 552 us = 997
//                  TFLOP/s (531 to 588 by card; both waves in step, and LDS rows at 8-byte addresses: 1555 us).
// Queries and weights are rounded to K's and V's type, which the matrix instructions take: half a step of 16 bits in each weight, whose sum is kept unrounded in 32, as
// are maximum and result.  A second term of each weight would be the products with V once more, half as much matrix work again in a kernel that is bound by it.
// What the rounding makes of infinities is put right by the writer (kinds_of).
// A masked weight is an exact zero, but zero times an infinity or a NaN is none: where a tile that is masked in part holds such values, they are taken
// out on the way into LDS and counted over the keys that a row sees, so that a row never meets what it does not see.
#include "kv_cache.h"

// what a 16-byte piece's number in its row is changed by (exclusive-or): the rows that an instruction reads together lie in different banks
template <int D> __device__ __forceinline__ int k_swap(int key) { return D == 128 ? key & 15 : key >> 1 & 7; }
template <int D> __device__ __forceinline__ int v_swap(int key) { return D == 128 ? (key & 3) << 2 : (key >> 1 & 1) << 2; }

template <typename O, int D, bool PAGED, int NW, int KG>
__global__ void __launch_bounds__(64 * NW, 2) k_attn_packed(const PackedArgs a) {
    typedef typename O::vec8 vec8;
    typedef typename O::elem elem;
    constexpr int KK = D / 16, NI = D / 32;
    constexpr int PCS = D / 8;                                        // 16-byte pieces of a row
    constexpr int KT = NW == 8 || KG == 2 ? 64 : 32;                     // keys of a tile
    constexpr int KA = NW == 8 ? 2 : 1, VA = KA - 1;                  // tiles that K and V are in LDS ahead of the step that they are written in
    constexpr int SLOTS = NW == 8 ? 3 : 1;                            // in use at a time: K tiles t .. t+2, V tiles t-1 .. t+1 (one of each where all waves are in step)
    constexpr int NL = KT * PCS / (64 * NW), RPL = 64 * NW / PCS;               // pieces per thread and tile, K and V each; keys that lie between them
    constexpr int TILE_B = KT * D * 2;
    constexpr int NB = KT / 32 / KG, NC = 2 * NB;                     // 32-key blocks of S and 16-key chunks of P that a wave has of a tile
    extern __shared__ __attribute__((aligned(1024))) char lds[];      // SLOTS K tiles, SLOTS V tiles, SLOTS tiles of what was taken out of V, odd[SLOTS]
    int * odd = (int *) (lds + 3 * SLOTS * TILE_B);                   // t + 1: something was taken out of V tile t
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
    // this lane's row; which half of each tile's keys this wave takes (KG 2)
    const int rw = wave % (NW / KG), k_off = wave / (NW / KG) * 32;
    const int q_base = job.tile * a.qt, nrow = min(a.qt, job.nq - q_base) * a.G, r = rw * 32 + (lane & 31);
    const int rc = min(r, nrow - 1), qi = q_base + rc / a.G, g = rc - rc / a.G * a.G;
    const int off = L - job.nq;                                       // row qi's own key is off + qi
    const int last = a.causal ? min(off + qi, L - 1) : L - 1;         // the last key it sees (-1: none)
    const int first = a.window > 0 ? max(off + qi - a.window + 1, 0) : 0;
    // the same for the wave's first and last row and for the workgroup's: uniform
    const int wr0 = min(rw * 32, nrow - 1), wr1 = min(rw * 32 + 31, nrow - 1), wq0 = q_base + wr0 / a.G, wq1 = q_base + wr1 / a.G, bq1 = q_base + (nrow - 1) / a.G;
    const int w_last_min = a.causal ? min(off + wq0, L - 1) : L - 1, w_last = a.causal ? min(off + wq1, L - 1) : L - 1;
    const int w_first = a.window > 0 ? max(off + wq0 - a.window + 1, 0) : 0, w_first_max = a.window > 0 ? max(off + wq1 - a.window + 1, 0) : 0;
    const int b_last_min = a.causal ? min(off + q_base, L - 1) : L - 1, b_last = a.causal ? min(off + bq1, L - 1) : L - 1;
    const int b_first = a.window > 0 ? max(off + q_base - a.window + 1, 0) : 0, b_first_max = a.window > 0 ? max(off + bq1 - a.window + 1, 0) : 0;
    const int T0 = b_first / KT, T = b_last >= b_first && L > 0 ? b_last / KT + 1 - T0 : 0;          // tiles T0 .. T0 + T - 1
    // tiles that this wave's rows see nothing of are passed over; the rest of its tiles are t_lo .. t_hi - 1
    const int t_lo = max(w_first / KT - T0, 0), t_hi = rw * 32 < nrow && w_last >= w_first ? min(w_last / KT + 1 - T0, T) : 0;

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
    floatx16 o[NI], s[NB];
    vec8 pf[NC];
    #pragma unroll
    for (int i = 0; i < NI; i++)
        #pragma unroll
        for (int e = 0; e < 16; e++) o[i][e] = 0.0f;
    constexpr float lift = __is_same(O, f16_ops) ? 7.0f : 0.0f;
    float m = -INFINITY, l = 0.0f, mc = -lift;
    bool big = false;                                                 // some row's maximum is so large that the scores meet it before their products with c2 are made

    // staging: thread -> key tid / PCS (+ RPL), piece tid % PCS.  A tile's keys behind the last are other rows of the pool or the last row again: no
    // row sees them, and what of their values is not finite is taken out below.  A tile's places are made once, for its keys, and kept for its values.
    const int skey = tid / PCS, spc = tid % PCS;
    const char * kb = a.c.k + hk * a.c.nb_head + spc * 16, * vb = a.c.v + hk * a.c.nb_head + spc * 16;
    if (!PAGED) { kb += k0 * a.c.nb_key; vb += k0 * a.c.nb_key; }
    bool bad = false;
    u32x4_t kr[NL], vr[NL];
    int pg[NL];                                                       // pages of the tile whose places are made next
    int64_t at_k[NL], at_v[NL];                                       // places of the K tile and of the V tile that are fetched next
    const uint32_t nb_key = (uint32_t) a.c.nb_key, nb_page = (uint32_t) a.c.nb_page;
    auto ask = [&](int t) {
        if (PAGED) {
            #pragma unroll
            for (int e = 0; e < NL; e++) pg[e] = row[min(((T0 + t) * KT + skey + e * RPL) >> a.c.shift, a.c.max_pages - 1)];
        }
    };
    auto make = [&](int t) {
        #pragma unroll
        for (int e = 0; e < NL; e++) {
            const int key = (T0 + t) * KT + skey + e * RPL;
            if (PAGED) {
                bad |= (unsigned) pg[e] >= (unsigned) a.c.n_pages && key >= b_first && key <= b_last;     // (a page that no row sees may be gone)
                at_k[e] = (int64_t) ((uint64_t) (uint32_t) min(max(pg[e], 0), a.c.n_pages - 1) * nb_page + (uint64_t) (uint32_t) (key & a.c.mask) * nb_key);
            } else at_k[e] = (int64_t) ((uint64_t) (uint32_t) min(key, L - 1) * nb_key);
        }
    };
    auto keep = [&]() {
        #pragma unroll
        for (int e = 0; e < NL; e++) at_v[e] = at_k[e];
    };
    auto fetch_k = [&]() {
        #pragma unroll
        for (int e = 0; e < NL; e++) kr[e] = *(const u32x4_t *) (kb + at_k[e]);
    };
    auto fetch_v = [&](const int64_t * at) {
        #pragma unroll
        for (int e = 0; e < NL; e++) vr[e] = *(const u32x4_t *) (vb + at[e]);
    };
    const int k_put = skey * (D * 2) + (spc ^ k_swap<D>(skey)) * 16, v_put = skey * (D * 2) + (spc ^ v_swap<D>(skey)) * 16;     // (the same for keys RPL apart)
    auto put_k = [&](int t) {
        #pragma unroll
        for (int e = 0; e < NL; e++) *(u32x4_t *) (lds + t % SLOTS * TILE_B + k_put + e * RPL * (D * 2)) = kr[e];
    };
    auto put_v = [&](int t) {
        char * vl = lds + (SLOTS + t % SLOTS) * TILE_B + v_put;
        const bool edge = (T0 + t) * KT + KT - 1 > b_last_min || (T0 + t) * KT < b_first_max;         // masked in part for some row
        #pragma unroll
        for (int e = 0; e < NL; e++) {
            const int at = e * RPL * (D * 2);
            if (edge) {
                u32x4_t kind = { 0, 0, 0, 0 };
                if (not_finite8<O>(vr[e])) { take_apart<O>(vr[e], kind); odd[t % SLOTS] = t + 1; }    // every writer writes the same; what an older tile left does not match
                *(u32x4_t *) (vl + SLOTS * TILE_B + at) = kind;
            }
            *(u32x4_t *) (vl + at) = vr[e];
        }
    };
    // a lane's places in a K tile (key lane & 31, piece 2 kk + hf: exclusive-or with kk << 5) and in a V tile (4 hf + (lane & 15) / 4, half a piece of dims
    // 32 i + 16 (lane / 16 & 1) ..: exclusive-or with i << 6)
    const int li = lane & 15, key0 = 4 * hf + (li >> 2);
    const uint32_t k_lane = (lane & 31) * (D * 2) + (hf ^ k_swap<D>(lane & 31)) * 16;
    const uint32_t v_lane = key0 * (D * 2) + ((2 * ((lane >> 4) & 1) + ((li >> 1) & 1)) ^ v_swap<D>(key0)) * 16 + (li & 1) * 8;
    auto part = [&](int t) { return (T0 + t) * KT + KT - 1 > w_last_min || (T0 + t) * KT < w_first_max; };

    // S^T = K.Q^T: element e of block b is key k_off + 32 b + (e & 3) + 8 (e >> 2) + 4 hf of the tile
    auto qk = [&](int t) {
        const uint32_t kl = lds_at(lds) + t % SLOTS * TILE_B + k_off * (D * 2) + k_lane;
        #pragma unroll
        for (int b = 0; b < NB; b++)
            #pragma unroll
            for (int e = 0; e < 16; e++) s[b][e] = 0.0f;
        vec8 kf[4][NB];                                               // the next products' operands are read while these run
        auto get = [&](int kk) {
            #pragma unroll
            for (int b = 0; b < NB; b++) {
                kf[kk & 3][b] = *(const LDS vec8 *) (size_t) ((kl ^ kk << 5) + b * 32 * (D * 2));
            }
        };
        get(0); get(1); get(2);
        #pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 3 < KK) get(kk + 3);
            #pragma unroll
            for (int b = 0; b < NB; b++) s[b] = O::mfma32(kf[kk & 3][b], qf[kk], s[b]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // V^T's operand for keys k_off + 16 c .. +15 (this lane's 16-lane group: 4 hf + {0..3} and + 8 of them), dims 32 i .. +31
    auto v_frag = [&](uint32_t vl, int c, int i) {
        vec8 vf;
        #pragma unroll
        for (int b = 0; b < 2; b++) {
            const short4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS short4_t *) (size_t) ((vl ^ i << 6) + (16 * c + 8 * b) * (D * 2)));
            __builtin_memcpy((char *) &vf + 8 * b, &x, 8);
        }
        return vf;
    };
    // O^T += V^T.P^T
    auto pv = [&](int t) {
        const uint32_t vl = lds_at(lds) + (SLOTS + t % SLOTS) * TILE_B + k_off * (D * 2) + v_lane;
        vec8 vf[2][NI];
        #pragma unroll
        for (int i = 0; i < NI; i++) vf[0][i] = v_frag(vl, 0, i);
        #pragma unroll
        for (int c = 0; c < NC; c++) {
            #pragma unroll
            for (int i = 0; i < NI; i++) if (c + 1 < NC) vf[(c + 1) & 1][i] = v_frag(vl, c + 1, i);
            #pragma unroll
            for (int i = 0; i < NI; i++) o[i] = O::mfma32(vf[c & 1][i], pf[c], o[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_amdgcn_readfirstlane(odd[t % SLOTS]) != t + 1) return;
        // what was taken out of this tile, for the rows that see it: over the visible keys, how many of each kind
        const int hi = last - (T0 + t) * KT - k_off - 4 * hf, lo = first - (T0 + t) * KT - k_off - 4 * hf;
        #pragma unroll
        for (int i = 0; i < NI; i++) {
            floatx16 cnt;
            #pragma unroll
            for (int e = 0; e < 16; e++) cnt[e] = 0.0f;
            #pragma unroll
            for (int c = 0; c < NC; c++) {
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
                o[i][e] += put_back(cnt[e]);
            }
        }
    };
    // P^T from S^T, with the running maximum and sum.  The maximum follows only when a row's grows by more than 2^8 in its weights, so that O is
    // hardly ever rescaled; F16 weights are held times 2^7 (2^15 at most), so that small ones do not fall below its range.  Both cancel against the sum.
    auto softmax = [&](int t) {
        if (part(t)) {
            const int hi = last - (T0 + t) * KT - k_off - 4 * hf, lo = first - (T0 + t) * KT - k_off - 4 * hf;
            #pragma unroll
            for (int b = 0; b < NB; b++)
                #pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int k = 32 * b + (e & 3) + 8 * (e >> 2);
                    if (k > hi || k < lo) s[b][e] = -INFINITY;
                }
        }
        float top = fmaxf(s[0][0], s[0][1]);
        #pragma unroll
        for (int e = 2; e < 16 * NB; e += 2) top = fmaxf(fmaxf(top, s[e >> 4][e & 15]), s[(e + 1) >> 4][(e + 1) & 15]);
        top = fmaxf(top, lane_xor32(top));
        if (__any((top - m) * a.c2 > 8.0f)) {
            const float mn = fmaxf(m, top), alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * a.c2);
            m = mn; l *= alpha;
            #pragma unroll
            for (int i = 0; i < NI; i++)
                #pragma unroll
                for (int e = 0; e < 16; e++) o[i][e] *= alpha;
            // m * c2 is rounded before the scores' products meet it: no more than F32 scores are off by themselves, and within 2^+-0.07 up to 2^20, but beyond
            // the range of the weights' type (F16 from 2^24 on, any type from 2^31 on) for larger ones.  Those take the difference first.
            mc = m == -INFINITY ? 0.0f : m * a.c2;
            big = __any(fabsf(mc) > 0x1p20f);
            mc = (big ? 0.0f : mc) - lift;
        }
        if (__builtin_expect(big, 0)) {
            const float m0 = m == -INFINITY ? 0.0f : m;
            #pragma unroll
            for (int e = 0; e < 16 * NB; e++) s[e >> 4][e & 15] -= m0;
        }
        float sum = 0.0f;
        #pragma unroll
        for (int b = 0; b < NB; b++)
            #pragma unroll
            for (int e = 0; e < 16; e++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], a.c2, -mc));
                sum += p;
                pf[2 * b + (e >> 3)][e & 7] = (elem) p;
            }
        l += sum;
    };

    if (T > 0) {
        // Eight waves: two groups of four, one wave of each on every SIMD, half a step apart: while one runs the matrix products of a step (PV of the tile
        // before, QK of this one), the other runs the softmax and brings tiles in.  A barrier ends each half step.  Four waves: all in step, another
        // workgroup of the CU fills the gaps.
        const bool second = NW == 8 && wave >= 4;
        if (tid < SLOTS) odd[tid] = 0;
        ask(0); make(0);
        ask(min(1, T - 1));
        fetch_k();
        if (VA == 1) fetch_v(at_k);
        put_k(0);
        keep(); make(min(1, T - 1));
        if (KA == 2) {
            ask(min(2, T - 1));
            fetch_k();
            __syncthreads();                                          // odd[] cleared
            put_v(0);
            put_k(1);
            keep(); make(min(2, T - 1));
        }
        ask(min(KA + 1, T - 1));
        fetch_v(at_v);                                                // V tile VA, K tile KA next
        fetch_k();
        __syncthreads();
        if (second) __syncthreads();
        for (int t = 0; t < T; t++) {
            if (NW == 8) __builtin_amdgcn_s_setprio(1);
            if (t > t_lo && t <= t_hi) pv(t - 1);
            if (t >= t_lo && t < t_hi) qk(t);
            if (NW == 8) __builtin_amdgcn_s_setprio(0);
            __syncthreads();
            if (t + KA < T) put_k(t + KA);
            if (t + VA < T) put_v(t + VA);
            // the places of K's tile of the step before are V's now.  Pages: the next places first, for a wait for the page numbers behind the loads of V
            // would be one for those (piece over a cache: 90 us, so 80).  Rows: no such wait, and no copy of the places (long, grouped: 558 us, so 546)
            if (PAGED) {
                keep();
                if (t + KA + 1 < T) make(t + KA + 1);
                if (t + VA + 1 < T) fetch_v(at_v);
            } else {
                if (t + VA + 1 < T) fetch_v(at_k);
                if (t + KA + 1 < T) make(t + KA + 1);
            }
            if (t + KA + 1 < T) {
                fetch_k();
                ask(min(t + KA + 2, T - 1));
            }
            if (t >= t_lo && t < t_hi) softmax(t);
            if (!second || t + 1 < T) __syncthreads();
        }
        if (t_hi == T && t_hi > t_lo) pv(T - 1);
    }
    if (PAGED && __any(bad) && lane == 0) atomicOr((unsigned *) a.c.status, MI355X_KV_BAD_ARG);
    l += lane_xor32(l);
    if (KG == 2) {                                                    // the second half of the keys joins the first, over the dead tiles: [m, l, o ..][wave, lane]
        constexpr int RS = 32 * NW;                                   // records are laid lane by lane
        float * rec = (float *) lds + (wave % (NW / 2)) * 64 + lane;
        __syncthreads();
        if (wave >= NW / 2) {
            rec[0] = m; rec[RS] = l;
            #pragma unroll
            for (int i = 0; i < NI; i++)
                #pragma unroll
                for (int e = 0; e < 16; e++) rec[(2 + 16 * i + e) * RS] = o[i][e];
        }
        __syncthreads();
        if (wave >= NW / 2) return;
        const float mo = rec[0], mn = fmaxf(m, mo);
        const float f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * a.c2), f1 = mo == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mo - mn) * a.c2);
        l = l * f0 + rec[RS] * f1;
        #pragma unroll
        for (int i = 0; i < NI; i++)
            #pragma unroll
            for (int e = 0; e < 16; e++) o[i][e] = o[i][e] * f0 + rec[(2 + 16 * i + e) * RS] * f1;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (r < nrow) {
        const int os = a.o_type == MI355X_TYPE_F32 ? 4 : 2;
        char * op = a.o + (int64_t) (job.r0 + qi) * a.o_nb2 + (int64_t) (hk * a.G + g) * a.o_nb1;
        float all = 0.0f;
        #pragma unroll
        for (int i = 0; i < NI; i++)
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y0 = o[i][4*e] * inv, y1 = o[i][4*e+1] * inv, y2 = o[i][4*e+2] * inv, y3 = o[i][4*e+3] * inv;
                all += y0 + y1 + y2 + y3;
                store4(op + (32 * i + 8 * e + 4 * hf) * os, a.o_type, y0, y1, y2, y3);
            }
        if (__builtin_expect(all != all && l == l, 0)) {              // some may be NaN that are not: the values decide (kinds_of)
            #pragma unroll 1
            for (int d = 4 * hf; d < D; d += 8) {
                const char * at = a.c.v + hk * a.c.nb_head + d * 2;
                uint32_t kinds[4] = { 0, 0, 0, 0 };
                #pragma unroll 1
                for (int key = first; key <= last; key++) {
                    if (PAGED) kinds_of<O>(at + min(max(row[key >> a.c.shift], 0), a.c.n_pages - 1) * a.c.nb_page + (key & a.c.mask) * a.c.nb_key, kinds);
                    else kinds_of<O>(at + (int64_t) (k0 + key) * a.c.nb_key, kinds);
                }
                #pragma unroll
                for (int n = 0; n < 4; n++) if (kinds[n]) store1(op + (d + n) * os, a.o_type, kinds_value(kinds[n]));
            }
        }
    }
}

template <typename O, int D, bool PAGED, int NW, int KG>
static int launch_packed_as(mi355x_ctx * ctx, PackedArgs & a, int64_t Hkv) {
    static std::atomic<uint64_t> allowed{0};
    a.qt = 32 * NW / KG / a.G;
    if (a.qt < 1) return kv_refuse("attn_packed: a group of more heads than a workgroup has rows");      // (launch_packed chooses a form that has them)
    const int64_t blocks = ((int64_t) a.rows_q / a.qt + a.n) * Hkv;
    if (!kv_fits(blocks, 64 * NW)) return kv_refuse("attn_packed: too many rows for one launch");
    const uint32_t lds = (NW == 8 ? 3 * 3 * 64 : KG == 2 ? 3 * 64 : 3 * 32) * D * 2 + 16;
    const int rl = kv_allow_lds(ctx, (const void *) k_attn_packed<O, D, PAGED, NW, KG>, lds, allowed);
    if (rl) return rl;
    return emit(ctx, "attn_packed", k_attn_packed<O, D, PAGED, NW, KG>, dim3((uint32_t) blocks), dim3(64 * NW), lds, a);
}
// Which form a call gets, by what the host knows (rows, sequences, an upper bound of the rows and of the keys of one); us for BF16, [sequences] x [rows]
// (+ [keys before them]), [query heads]/[K/V heads]:
//   few rows, workgroups of 16 rows no more than CUs, some hundred keys: attn_paged.hip's kernel, whose eight waves take the keys in turn
//       1 x 5 + 8192, 32/8 of 128: 77 (143 here);  1 x 32 + 1500, 20/20 of 64: 13.5 (36);  but 32 x 8 + 1000, 32/8: 50 (29)
//   64 dims: four waves, 128 rows (8 x 1500, 20/20: 101; eight waves 122); where that leaves CUs idle, 64 rows and two waves on each tile's keys
//       (1 x 1500, 20/20: 25; 38.  1 x 4096, 20/20: 82; 100)
//   128 dims: eight waves, 256 rows (1 x 8192, 32/8: 565; four waves 661).  Up to 768 keys the start and the end of a workgroup weigh more than its
//       loop: four waves, two workgroups to a CU (64 x 128, 32/8: 51; 64.  32 x 512: 157; 167.  8 x 1024: 120; 118).  Few workgroups: two waves on each
//       tile's keys (1 x 8192, 8/8, whose last rows' workgroups are twice the mean: 205; 250.  2 x 256 + 8192, 32/8: 177; 253), but not where that makes
//       a second round of workgroups of equal length (4 x 512 + 2048 of a window, 32/8: 133; 96)
template <typename O, int D, bool PAGED>
static int launch_packed(mi355x_ctx * ctx, PackedArgs & a, int64_t Hkv, int max_q, int64_t keys) {
    const int64_t rows = (int64_t) a.rows_q * a.G;                   // query x head of a group
    const int64_t few = (int64_t) a.n * Hkv * ((max_q * (int64_t) a.G + 15) / 16);   // workgroups of 16 rows
    if (max_q > 0 && (int64_t) max_q * a.G <= 256 && few <= ctx->n_cu && keys >= 256) return mi355x_attn_few_rows(ctx, a, __is_same(O, f16_ops) ? MI355X_TYPE_F16 : MI355X_TYPE_BF16, D, PAGED);
    const int64_t wide = rows * Hkv / 256;                           // workgroups of 256 rows, if all were full
    const bool pairs = a.G <= 64;                                    // four waves, two on each tile's keys: 64 rows, which have to hold a group's heads
    if constexpr (D == 64) {
        if (wide < 512 && keys >= 128 && pairs) return launch_packed_as<O, D, PAGED, 4, 2>(ctx, a, Hkv);
        return launch_packed_as<O, D, PAGED, 4, 1>(ctx, a, Hkv);
    } else {
        const int64_t per = (rows + a.n - 1) / a.n;                  // of one sequence on the average
        const bool wedge = a.causal && a.window == 0 && keys <= 2 * (a.rows_q / a.n);
        if (wide <= (wedge ? ctx->n_cu : ctx->n_cu / 2) && keys >= 256) return per <= 64 && pairs ? launch_packed_as<O, D, PAGED, 4, 2>(ctx, a, Hkv) : launch_packed_as<O, D, PAGED, 8, 2>(ctx, a, Hkv);
        return keys <= 768 ? launch_packed_as<O, D, PAGED, 4, 1>(ctx, a, Hkv) : launch_packed_as<O, D, PAGED, 8, 1>(ctx, a, Hkv);
    }
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
        if (d->k.nb[1] < 0 || d->k.nb[2] < 0 || d->k.nb[2] > UINT32_MAX) return kv_refuse("attn_packed: k's strides");
        a.c.k = (char *) d->k.data; a.c.v = (char *) d->v.data; a.c.nb_head = d->k.nb[1]; a.c.nb_key = d->k.nb[2];
        a.rows_k = (int) d->k.ne[2];
    }
    const int64_t H = d->q.ne[1], rows = d->q.ne[2];
    if (H < 1 || H % Hkv || H / Hkv > 128) return kv_refuse("attn_packed: the query heads are no multiple (up to 128) of the K/V heads");
    if (!kv_rows_ok(&d->q, dim, H) || !kv_rows_ok(&d->dst, dim, H) || d->dst.ne[2] != rows) return kv_refuse("attn_packed: q and dst are [head_dim, n_head, rows], F32 / F16 / BF16, 16-byte aligned");
    if (d->n < 0 || d->window < 0 || d->max_q < 0 || !isfinite(d->scale)) return kv_refuse("attn_packed: n, window, max_q or scale");
    if (d->n == 0 || rows == 0) return 0;
    if (!d->cu_q || ((uintptr_t) d->cu_q | (uintptr_t) d->cu_k | (uintptr_t) d->seq) % 4) return kv_refuse("attn_packed: cu_q, cu_k or seq");
    const device_scope scope(ctx);
    a.q = (const char *) d->q.data; a.q_nb1 = d->q.nb[1]; a.q_nb2 = d->q.nb[2]; a.q_type = d->q.type;
    a.o = (char *) d->dst.data; a.o_nb1 = d->dst.nb[1]; a.o_nb2 = d->dst.nb[2]; a.o_type = d->dst.type;
    a.cu_q = d->cu_q; a.cu_k = d->cu_k ? d->cu_k : d->cu_q; a.seq = d->seq;
    a.c2 = fmaxf(fabsf(d->scale) * 1.4426950408889634f, 1e-37f); a.flip = d->scale < 0.0f; a.n = d->n; a.rows_q = (int) rows; a.causal = d->causal != 0; a.window = d->window;
    a.G = (int) (H / Hkv); a.Hkv = (int) Hkv;
    const bool f16 = type == MI355X_TYPE_F16, paged = d->cache != nullptr;
    if (paged ? a.window >= (int64_t) d->cache->max_pages * d->cache->page_size : a.window >= a.rows_k) a.window = 0;      // no key lies before it
    const int64_t keys = paged ? (int64_t) d->cache->max_pages * d->cache->page_size : a.rows_k / d->n;       // of a sequence, as far as the host knows
    if (dim == 64) return f16 ? (paged ? launch_packed<f16_ops, 64, true>(ctx, a, Hkv, d->max_q, keys) : launch_packed<f16_ops, 64, false>(ctx, a, Hkv, d->max_q, keys))
                              : (paged ? launch_packed<bf16_ops, 64, true>(ctx, a, Hkv, d->max_q, keys) : launch_packed<bf16_ops, 64, false>(ctx, a, Hkv, d->max_q, keys));
    return f16 ? (paged ? launch_packed<f16_ops, 128, true>(ctx, a, Hkv, d->max_q, keys) : launch_packed<f16_ops, 128, false>(ctx, a, Hkv, d->max_q, keys))
               : (paged ? launch_packed<bf16_ops, 128, true>(ctx, a, Hkv, d->max_q, keys) : launch_packed<bf16_ops, 128, false>(ctx, a, Hkv, d->max_q, keys));
}

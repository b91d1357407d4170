// Internal header of the paged K/V cache: what kv_cache.hip, attn_paged.hip and attn_packed.hip share.
#pragma once
#include "common.h"
#include <math.h>
#include <atomic>

// the calling thread's device is the context's for the length of a call, and the caller's again afterwards
struct device_scope {
    int prev = -1; bool changed = false;
    explicit device_scope(const mi355x_ctx * ctx) {
        if (hipGetDevice(&prev) == hipSuccess && prev != ctx->device) changed = hipSetDevice(ctx->device) == hipSuccess;
    }
    ~device_scope() { if (changed) (void) hipSetDevice(prev); }
};

// a cache as kernels see it
struct kvc {
    char * k, * v;
    int64_t nb_key, nb_head, nb_page;
    int * table, * len, * ref, * status, * work;
    int n_pages, n_seq, max_pages, shift, mask, Hkv;
};

static inline int kv_refuse(const char * what) { mi355x_set_error("%s", what); return MI355X_E_UNSUPPORTED; }

// a launch has at most 2^32 - 1 threads: looked at before the first launch of a call, so that none is done by half
static inline bool kv_fits(int64_t blocks, int64_t threads) { return blocks <= UINT32_MAX / threads; }

// argument checks of every call that takes a cache; fills `o`
static inline int kv_view(const mi355x_kv_cache * c, kvc * o) {
    if (!c) return kv_refuse("kv cache: NULL");
    if (c->type != MI355X_TYPE_F16 && c->type != MI355X_TYPE_BF16) return kv_refuse("kv cache: type is neither F16 nor BF16");
    if (c->head_dim != 64 && c->head_dim != 128) return kv_refuse("kv cache: head_dim is neither 64 nor 128");
    if (c->n_head_kv < 1 || (int64_t) c->n_head_kv * c->head_dim > 32768) return kv_refuse("kv cache: n_head_kv");
    if (c->page_size < 1 || c->page_size > 4096 || (c->page_size & (c->page_size - 1))) return kv_refuse("kv cache: page_size is not a power of two up to 4096");
    if (c->n_pages < 1 || c->n_seq < 1 || c->n_seq > 262144 || c->max_pages < 1 || (int64_t) c->max_pages * c->page_size > INT32_MAX / 2) return kv_refuse("kv cache: n_pages, n_seq or max_pages");
    if (!c->k || !c->v || !c->table || !c->len || !c->ref || !c->status || !c->work) return kv_refuse("kv cache: a NULL pointer");
    if (((uintptr_t) c->k | (uintptr_t) c->v | (uintptr_t) c->nb_key | (uintptr_t) c->nb_head | (uintptr_t) c->nb_page) % 16) return kv_refuse("kv cache: pools and strides need 16-byte alignment");
    if (((uintptr_t) c->table | (uintptr_t) c->len | (uintptr_t) c->ref | (uintptr_t) c->status | (uintptr_t) c->work) % 4) return kv_refuse("kv cache: misaligned tables");
    const int64_t row = c->head_dim * 2;
    if (c->nb_key < row || c->nb_head < row || c->nb_page < row) return kv_refuse("kv cache: strides smaller than a row");
    if (c->nb_key > UINT32_MAX || c->nb_page > UINT32_MAX) return kv_refuse("kv cache: strides of 4 GiB and more");
    o->k = (char *) c->k; o->v = (char *) c->v; o->nb_key = c->nb_key; o->nb_head = c->nb_head; o->nb_page = c->nb_page;
    o->table = c->table; o->len = c->len; o->ref = c->ref; o->status = c->status; o->work = (int *) c->work;
    o->n_pages = c->n_pages; o->n_seq = c->n_seq; o->max_pages = c->max_pages;
    o->shift = __builtin_ctz((unsigned) c->page_size); o->mask = c->page_size - 1; o->Hkv = c->n_head_kv;
    return 0;
}

// a tensor of rows of heads: [head_dim, heads, rows]
static inline bool kv_rows_ok(const mi355x_tensor * t, int dim, int64_t heads) {
    const int ts = t->type == MI355X_TYPE_F32 ? 4 : t->type == MI355X_TYPE_F16 || t->type == MI355X_TYPE_BF16 ? 2 : 0;
    return ts && t->ne[0] == dim && t->ne[1] == heads && t->ne[2] >= 0 && t->ne[2] < INT32_MAX && t->ne[3] == 1 && t->nb[0] == ts &&
           (t->data || t->ne[2] == 0) && ((uintptr_t) t->data | (uintptr_t) t->nb[1] | (uintptr_t) t->nb[2]) % 16 == 0;
}

// more than 64 KB of dynamic LDS has to be allowed once per kernel and device; `done`: a bit per device
static inline int kv_allow_lds(mi355x_ctx * ctx, const void * f, uint32_t lds, std::atomic<uint64_t> & done) {
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (lds <= 64 * 1024 || (done.load(std::memory_order_relaxed) & bit)) return 0;
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, 158 * 1024);
    if (e != hipSuccess) { mi355x_set_error("dynamic LDS of %u bytes refused: %s", lds, hipGetErrorString(e)); return (int) e; }
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

#ifdef __HIPCC__
struct PackedArgs;
// attn_paged.hip: packed sequences of few rows (up to 16 rows of a K/V head at a time, every wave its own tiles of the keys)
int mi355x_attn_few_rows(mi355x_ctx * ctx, const PackedArgs & a, int type, int dim, bool paged);

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short  short4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// the two 16-bit types: conversions (round to nearest even) and the matrix instructions on them
struct f16_ops {
    typedef half8_t vec8;
    typedef half_t  elem;
    static __device__ __forceinline__ floatx4  mfma16(vec8 a, vec8 b, floatx4 c)  { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ floatx16 mfma32(vec8 a, vec8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
struct bf16_ops {
    typedef bf16x8_t vec8;
    typedef __bf16   elem;
    static __device__ __forceinline__ floatx4  mfma16(vec8 a, vec8 b, floatx4 c)  { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ floatx16 mfma32(vec8 a, vec8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// LDS by its 32-bit address
#define LDS __attribute__((address_space(3)))
__device__ __forceinline__ uint32_t lds_at(char * p) { return (uint32_t) (size_t) (LDS char *) p; }

// eight consecutive elements of F32 / F16 / BF16 memory as floats, and back
__device__ __forceinline__ void load8(const char * p, int type, float * f) {
    if (type == MI355X_TYPE_F32) {
        const float4 a = ((const float4 *) p)[0], b = ((const float4 *) p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else if (type == MI355X_TYPE_F16) {
        const half8_t a = *(const half8_t *) p;
        #pragma unroll
        for (int e = 0; e < 8; e++) f[e] = (float) a[e];
    } else {
        const bf16x8_t a = *(const bf16x8_t *) p;
        #pragma unroll
        for (int e = 0; e < 8; e++) f[e] = (float) a[e];
    }
}
__device__ __forceinline__ void store4(char * p, int type, float a, float b, float c, float d) {
    if (type == MI355X_TYPE_F32) *(float4 *) p = make_float4(a, b, c, d);
    else if (type == MI355X_TYPE_F16) { half4_t h; h[0] = (half_t) a; h[1] = (half_t) b; h[2] = (half_t) c; h[3] = (half_t) d; *(half4_t *) p = h; }
    else { typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4))); bf16x4_t h; h[0] = (__bf16) a; h[1] = (__bf16) b; h[2] = (__bf16) c; h[3] = (__bf16) d; *(bf16x4_t *) p = h; }
}

__device__ __forceinline__ void store1(char * p, int type, float a) {
    if (type == MI355X_TYPE_F32) *(float *) p = a;
    else if (type == MI355X_TYPE_F16) *(half_t *) p = (half_t) a;
    else *(__bf16 *) p = (__bf16) a;
}

// ---- packed rows (attn_packed.hip, and attn_paged.hip's kernel for few rows) ----
struct PackedArgs {
    kvc c;                             // PAGED: the cache.  Otherwise k, v and their strides in nb_key (rows) and nb_head
    const char * q; int64_t q_nb1, q_nb2;
    char * o; int64_t o_nb1, o_nb2;
    const int * cu_q, * cu_k, * seq;
    float c2; int flip;                // |scale| * log2(e), at least 1e-37; whether the scale is negative (the queries change sign)
    int n, rows_q, rows_k, q_type, o_type, causal, window;
    int G, Hkv, qt;                    // query heads per K/V head; queries of a workgroup
};

// slot -> (sequence, tile of its rows): sequence i has the slots cu[i]/qt + i .. cu[i+1]/qt + i, at least as many as its tiles.  A wave looks at 64
// sequences at a time: one load's latency where a bisection has log2(n) of them.
struct packed_job { int i, r0, nq, tile; };
template <typename A> __device__ __forceinline__ bool packed_find(const A & a, int slot, packed_job & j) {
    const int lane = threadIdx.x & 63;
    int lo = 0, step = 1;
    while (step * 64 < a.n) step *= 64;                              // coarse to fine: every `step`-th sequence behind lo
    for (; step > 0; step /= 64) {
        const int i = (int) min((int64_t) lo + (int64_t) lane * step, (int64_t) a.n);
        const unsigned long long m = __ballot(i < a.n && a.cu_q[i] / a.qt + i <= slot);
        lo += max((int) __popcll(m) - 1, 0) * step;                  // (a count is unsigned: no sequence begins at or before the slot, 0 - 1)
    }
    j.i = lo;
    j.r0 = a.cu_q[lo]; const int r1 = a.cu_q[lo + 1];
    if (j.r0 < 0 || r1 > a.rows_q || r1 <= j.r0) return false;
    j.nq = r1 - j.r0;
    const int tiles = (j.nq + a.qt - 1) / a.qt, t = slot - (j.r0 / a.qt + lo);
    if (t < 0 || t >= tiles) return false;
    j.tile = tiles - 1 - t;                                          // the rows with most keys first
    return true;
}

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

// what a count over visible keys of the numbers above adds to a sum (at most 64 of each kind)
__device__ __forceinline__ float put_back(float count) {
    const int n = (int) count;
    return ((n & 127) ? INFINITY : 0.0f) + ((n & 0x3F80) ? -INFINITY : 0.0f) + (n >= 16384 ? NAN : 0.0f);
}

// ---- infinities among the values that a row sees ----
// In the products, weights have 16 bits (or are sums of such terms): a weight below their range times an infinity is a NaN where it should be an infinity, and so are
// two terms of one weight that have other signs.  The kernels leave it at that, and the writer of a result that came out a NaN, though the row's weights are numbers,
// looks at the values itself: a bit for an infinity, a negative one, a NaN among four values (`at`: 8 bytes)
template <typename O> __device__ __forceinline__ void kinds_of(const char * at, uint32_t * kinds) {
    const uint32_t top = __is_same(O, f16_ops) ? 0x7C00 : 0x7F80;
    const uint2 w = *(const uint2 *) at;
    #pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t x = (e < 2 ? w.x : w.y) >> 16 * (e & 1) & 0xFFFF;
        if ((x & top) == top) kinds[e] |= (x & 0x7FFF) != top ? 4u : x & 0x8000 ? 2u : 1u;
    }
}
__device__ __forceinline__ float kinds_value(uint32_t kinds) { return kinds == 1 ? INFINITY : kinds == 2 ? -INFINITY : NAN; }

#endif

// Appending keys and values to a paged cache, queries and keys rotated by their positions on the way.
//
// Mathematics: each pair (a, b) of a rotated head becomes (a cos - b sin, b cos + a sin) in float32, rounded once; the
// rest of the head and the values are copied.  The cosines and sines come from float32 tables made once by the caller, so
// far positions lose nothing to an angle computed in 32 bits.
//
// What bounds it: bytes.  Every element is read once and written once, and a token of 32 query and 2 x 8 key-value heads of
// 128 16-bit elements is 24 KB of traffic against 0.5 KB of table: one CTA per token, a thread keeps one place inside the
// head (and its cosines and sines in registers) and walks over the heads.
#include "paged.cuh"

namespace enc {
namespace {

constexpr int THREADS = 128;

struct AppendArgs {
    const void *k, *v, *q;
    void *q_out, *k_cache, *v_cache;
    const float *cos, *sin;
    const int32_t *seq_ids, *positions, *block_table;
    int64_t sk_t, sk_h, sv_t, sv_h, sq_t, sq_h, so_t, so_h, s_cos;
    int64_t ck_p, ck_h, ck_t, cv_p, cv_h, cv_t, s_table;
    int64_t num_seqs, num_pages, num_positions, capacity;
    int q_heads, kv_heads, head_dim, rot_dim;
    bool angles_aligned;  // rows of cos and sin start on 16 bytes
    FastDiv page_size;
};

template <int N> __device__ __forceinline__ void load_floats(const float *p, bool aligned, float (&f)[N]) {
    if (N % 4 == 0 && aligned) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const float4 x = *reinterpret_cast<const float4 *>(p + 4 * i);
            f[4 * i] = x.x; f[4 * i + 1] = x.y; f[4 * i + 2] = x.z; f[4 * i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = p[i];
    }
}

// N neighbouring elements: one 16-byte vector, or single elements where rows are not aligned for that.
template <typename T, int N, bool VEC> struct Elems {
    T e[N];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = p[i];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = e[i];
    }
    __device__ __forceinline__ void get(float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = to_f32(e[i]);
    }
    __device__ __forceinline__ void set(const float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = from_f32<T>(f[i]);
    }
};
template <typename T, int N> struct Elems<T, N, true> {
    uint4 v;
    __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = v; }
    __device__ __forceinline__ void get(float (&f)[N]) const { Pack<T>::unpack(v, f); }
    __device__ __forceinline__ void set(const float (&f)[N]) { v = Pack<T>::pack(f); }
};

// Bytes in flight are what a CTA's short life is about, so registers are capped for as many CTAs as that leaves without spills
// (5016 float32 tokens of 18 heads of 64, pairs of neighbours: 15.0 us at 8 CTAs per SM, 12.7 at 12).
template <typename T, bool INTERLEAVED> constexpr int append_ctas_per_sm() { return sizeof(T) == 4 ? (INTERLEAVED ? 12 : 10) : 8; }

// One CTA per token.  VEC: 16-byte vectors (NV elements); else single elements.  An item is one place inside a head: a pair
// of vectors that turn together (one vector of neighbouring pairs when INTERLEAVED), or a vector that is copied.  The loads
// of a thread's first UN heads and of its first value vector are under way before the token's position, its page and its
// angles have arrived: they are the longest chain (index -> page number, position -> cosines).
template <typename T, bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, append_ctas_per_sm<T, INTERLEAVED>()) append_kernel(AppendArgs a) {
    constexpr int NV = VEC ? Pack<T>::N : (INTERLEAVED ? 2 : 1);  // elements of an item's vector
    constexpr int UN = 3;                                         // heads in flight per thread
    constexpr int NC = INTERLEAVED ? NV / 2 : NV;                 // angles of an item
    constexpr int CV = VEC ? NV : 1;                              // elements of a copied vector
    using Vec = Elems<T, NV, VEC>;
    using Copy = Elems<T, CV, VEC>;
    const int64_t t = blockIdx.x;
    const int turning = INTERLEAVED ? a.rot_dim / NV : a.rot_dim / 2 / NV;
    const int items = turning + (a.head_dim - a.rot_dim) / CV;
    const int nx = items < THREADS ? items : THREADS, ny = THREADS / nx;
    const int x = threadIdx.x % nx, y = threadIdx.x / nx;
    const int heads = a.kv_heads + (a.q ? a.q_heads : 0);  // key heads first, then query heads
    const int vh = a.head_dim / CV, values = a.kv_heads * vh;
    const T *k = reinterpret_cast<const T *>(a.k) + t * a.sk_t, *v = reinterpret_cast<const T *>(a.v) + t * a.sv_t;
    const T *q = reinterpret_cast<const T *>(a.q) + t * a.sq_t;
    T *qo = reinterpret_cast<T *>(a.q_out) + t * a.so_t;
    grid_dependency_wait();
    const int seq = a.seq_ids[t], pos = a.positions[t];

    Vec u[UN], w[UN];
    auto load = [&](int it, int h0) {
        const bool turn = it < turning;
        const int off = turn ? it * NV : a.rot_dim + (it - turning) * CV;
#pragma unroll
        for (int j = 0; j < UN; ++j) {
            const int h = h0 + j * ny;
            if (h >= heads) continue;
            const T *src = h < a.kv_heads ? k + h * a.sk_h : q + (h - a.kv_heads) * a.sq_h;
            if (VEC || turn) u[j].load(src + off);
            else reinterpret_cast<Copy &>(u[j]).load(src + off);
            if (!INTERLEAVED && turn) w[j].load(src + off + a.rot_dim / 2);
        }
    };
    auto value = [&](int i) {
        Copy c;
        c.load(v + (i / vh) * a.sv_h + (i % vh) * CV);
        return c;
    };
    const bool mine = y < ny;
    if (mine) load(x, y);
    Copy first_value;
    if (threadIdx.x < values) first_value = value(threadIdx.x);

    if (seq < 0) return;  // padding
    int64_t page = 0;
    int row = 0;
    bool ok = seq < a.num_seqs && pos >= 0 && pos < a.capacity && (a.rot_dim == 0 || pos < a.num_positions);
    if (ok) {
        const uint32_t pi = a.page_size.div((uint32_t)pos);
        row = pos - (int)(pi * a.page_size.d);
        page = a.block_table[seq * a.s_table + pi];
        ok = page >= 0 && page < a.num_pages;
    }
    if (!ok) {
        if (threadIdx.x == 0) atomicExch(&g_bad_index, 1u);
        return;
    }
    T *kc = reinterpret_cast<T *>(a.k_cache) + page * a.ck_p + row * a.ck_t;
    T *vc = reinterpret_cast<T *>(a.v_cache) + page * a.cv_p + row * a.cv_t;

    if (mine) {
        for (int it = x; it < items; it += THREADS) {
            const bool turn = it < turning;
            const int off = turn ? it * NV : a.rot_dim + (it - turning) * CV, off2 = off + a.rot_dim / 2;
            float cs[NC], sn[NC];
            if (turn) {
                load_floats<NC>(a.cos + pos * a.s_cos + it * NC, a.angles_aligned, cs);
                load_floats<NC>(a.sin + pos * a.s_cos + it * NC, a.angles_aligned, sn);
            }
            for (int h0 = y; h0 < heads; h0 += ny * UN) {
                if (it != x || h0 != y) load(it, h0);
#pragma unroll
                for (int j = 0; j < UN; ++j) {
                    const int h = h0 + j * ny;
                    if (h >= heads) continue;
                    T *dst = h < a.kv_heads ? kc + h * a.ck_h : qo + (h - a.kv_heads) * a.so_h;
                    if (!turn) {
                        reinterpret_cast<const Copy &>(u[j]).store(dst + off);
                        continue;
                    }
                    float fu[NV], fw[NV];
                    u[j].get(fu);
                    if (!INTERLEAVED) w[j].get(fw);
#pragma unroll
                    for (int e = 0; e < NC; ++e) {
                        float &lo = INTERLEAVED ? fu[(2 * e) % NV] : fu[e], &hi = INTERLEAVED ? fu[(2 * e + 1) % NV] : fw[e];
                        const float x0 = lo, x1 = hi;
                        lo = fmaf(x0, cs[e], -(x1 * sn[e]));
                        hi = fmaf(x1, cs[e], x0 * sn[e]);
                    }
                    u[j].set(fu);
                    u[j].store(dst + off);
                    if (!INTERLEAVED) {
                        w[j].set(fw);
                        w[j].store(dst + off2);
                    }
                }
            }
        }
    }
    for (int i = threadIdx.x; i < values; i += THREADS)  // values: plain copies
        (i < THREADS ? first_value : value(i)).store(vc + (i / vh) * a.cv_h + (i % vh) * CV);
}

template <typename T>
int launch_append(const AppendArgs &a, int64_t tokens, bool interleaved, bool vec, cudaStream_t st) {
    const dim3 grid((unsigned)tokens);
    note_indexed_launch();
    if (vec && interleaved) launch_overlapped(append_kernel<T, true, true>, grid, dim3(THREADS), 0, st, a);
    else if (vec) launch_overlapped(append_kernel<T, true, false>, grid, dim3(THREADS), 0, st, a);
    else if (interleaved) launch_overlapped(append_kernel<T, false, true>, grid, dim3(THREADS), 0, st, a);
    else launch_overlapped(append_kernel<T, false, false>, grid, dim3(THREADS), 0, st, a);
    return check_launch("enc_append_kv");
}

}  // namespace

unsigned int take_bad_index_append() { return take_bad_index_word(); }
int append_variants() { return 1; }
void append_variant_info(int, char *out, size_t n) { snprintf(out, n, "one CTA of %d threads per token", THREADS); }

}  // namespace enc

extern "C" int enc_append_kv(const enc_paged_cache *cache, const enc_append_args *args, int dtype, int variant, void *stream) {
    ENC_PROLOGUE();
    using namespace enc;
    const char *me = "enc_append_kv";
    if (!cache || !args) return fail(ENC_ERR_BAD_ARG, "%s: NULL cache or arguments", me);
    const enc_append_args &g = *args;
    const int64_t tokens = g.tokens, q_heads = g.q_heads, rot_dim = g.rot_dim;
    const bool interleaved = g.interleaved != 0;
    if (!is_float_dtype(dtype)) return fail(ENC_ERR_BAD_ARG, "%s: dtype %d is not float16, bfloat16 or float32", me, dtype);
    if (variant >= append_variants()) return fail(ENC_ERR_BAD_ARG, "%s: variant %d out of range", me, variant);
    const int bad = check_cache(*cache, me);
    if (bad) return bad;
    if (tokens < 0 || q_heads < 0) return fail(ENC_ERR_BAD_ARG, "%s: negative size", me);
    if (rot_dim < 0 || rot_dim > cache->head_dim || rot_dim % 2) return fail(ENC_ERR_BAD_ARG, "%s: rot_dim %lld must be even and at most head_dim %lld", me, (long long)rot_dim, (long long)cache->head_dim);
    if ((g.q != nullptr) != (g.q_out != nullptr)) return fail(ENC_ERR_BAD_ARG, "%s: q and q_out go together", me);
    if (tokens == 0) return ENC_OK;
    if (tokens > 0x7fffffffLL || q_heads > 0xffff) return fail(ENC_ERR_UNSUPPORTED, "%s: more than 2^31-1 tokens or 65535 query heads", me);
    if (!g.k || !g.v || !g.seq_ids || !g.positions) return fail(ENC_ERR_BAD_ARG, "%s: NULL tensor", me);
    if (rot_dim > 0 && (!g.cos || !g.sin)) return fail(ENC_ERR_BAD_ARG, "%s: rot_dim %lld without cos and sin", me, (long long)rot_dim);
    // (with no pages or no sequences nothing can be in range: the kernel reports every token that is not padding)
    if ((!cache->k || !cache->v || !cache->block_table) && cache->num_pages > 0 && cache->num_seqs > 0 && cache->table_width > 0)
        return fail(ENC_ERR_BAD_ARG, "%s: NULL cache tensor", me);
    AppendArgs a{};
    a.k = g.k; a.v = g.v; a.q = g.q; a.q_out = g.q_out; a.k_cache = cache->k; a.v_cache = cache->v;
    a.cos = g.cos; a.sin = g.sin; a.seq_ids = g.seq_ids; a.positions = g.positions; a.block_table = cache->block_table;
    a.sk_t = g.k_stride_token; a.sk_h = g.k_stride_head; a.sv_t = g.v_stride_token; a.sv_h = g.v_stride_head;
    a.sq_t = g.q_stride_token; a.sq_h = g.q_stride_head; a.so_t = g.o_stride_token; a.so_h = g.o_stride_head; a.s_cos = g.stride_cos;
    a.ck_p = cache->k_stride_page; a.ck_h = cache->k_stride_head; a.ck_t = cache->k_stride_token;
    a.cv_p = cache->v_stride_page; a.cv_h = cache->v_stride_head; a.cv_t = cache->v_stride_token;
    a.s_table = cache->stride_table;
    a.num_seqs = cache->num_seqs; a.num_pages = cache->num_pages; a.num_positions = g.num_positions;
    a.capacity = paged_capacity(*cache);
    a.q_heads = (int)q_heads; a.kv_heads = (int)cache->kv_heads; a.head_dim = (int)cache->head_dim; a.rot_dim = (int)rot_dim;
    a.page_size = FastDiv((uint32_t)cache->page_size);
    a.angles_aligned = aligned16(g.cos) && aligned16(g.sin) && g.stride_cos % 4 == 0;
    // 16-byte vectors where every row starts on 16 bytes and no vector straddles the rotated part or its halves
    const int nv = 16 / (int)dtype_size(dtype);
    bool vec = cache->head_dim % nv == 0 && rot_dim % (interleaved ? nv : 2 * nv) == 0 && aligned16(g.k) && aligned16(g.v) &&
               aligned16(cache->k) && aligned16(cache->v) && (!g.q || (aligned16(g.q) && aligned16(g.q_out)));
    for (int64_t s : {a.sk_t, a.sk_h, a.sv_t, a.sv_h, a.ck_p, a.ck_h, a.ck_t, a.cv_p, a.cv_h, a.cv_t}) vec = vec && s % nv == 0;
    if (g.q) for (int64_t s : {a.sq_t, a.sq_h, a.so_t, a.so_h}) vec = vec && s % nv == 0;
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ENC_F16: return launch_append<__half>(a, tokens, interleaved, vec, st);
        case ENC_BF16: return launch_append<__nv_bfloat16>(a, tokens, interleaved, vec, st);
        default: return launch_append<float>(a, tokens, interleaved, vec, st);
    }
}

// Attention of one new token per sequence over a paged key-value cache: the CUDA-core kernel, the join of split rows and the
// entry points.  Mathematics, bound and split are in paged_attention.cuh.
#include "paged_attention.cuh"

#include <type_traits>

namespace enc {
using namespace paged;
namespace {

// ---- join ------------------------------------------------------------------------------------------
// One CTA per (run, row): where a run's last piece begins a row group, the pieces of that group are that piece and the first
// pieces of the runs after it.  Two passes over the pieces' statistics (maximum, then weights), then the weighted sum.
template <typename T, int ROWS> __global__ void __launch_bounds__(THREADS) join_kernel(PagedArgs a) {
    __shared__ float red[WARPS], part[WARPS][MAX_HEAD_DIM];
    grid_dependency_wait();
    const int4 h = a.headers[blockIdx.x];
    const int rows = h.y & 255, first_head = h.y >> 8, r = blockIdx.y;
    if (r >= rows) return;
    const int n = h.z - (int)blockIdx.x + 1;  // pieces
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t stride = a.head_dim + 2;
    auto piece = [&](int i) { return slot_of(a, blockIdx.x + i, i == 0 ? 1 : 0, ROWS) + r * stride; };
    float m = -INFINITY;
    for (int i = threadIdx.x; i < n; i += THREADS) m = fmaxf(m, piece(i)[a.head_dim]);
    m = warp_max(m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, red[w]);
    __syncthreads();
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, x[MAX_HEAD_DIM / 32];
#pragma unroll
    for (int i = 0; i < MAX_HEAD_DIM / 32; ++i) x[i] = 0.0f;
    for (int i = warp; i < n; i += WARPS) {  // a warp takes every WARPS-th piece, its lanes the elements
        const float *p = piece(i);
        const float c = fast_exp2(p[a.head_dim] - base);
        l = fmaf(p[a.head_dim + 1], c, l);
#pragma unroll
        for (int j = 0; j < MAX_HEAD_DIM / 32; ++j)
            if (lane + 32 * j < a.head_dim) x[j] = fmaf(p[lane + 32 * j], c, x[j]);
    }
    if (lane == 0) red[warp] = l;
#pragma unroll
    for (int j = 0; j < MAX_HEAD_DIM / 32; ++j)
        if (lane + 32 * j < a.head_dim) part[warp][lane + 32 * j] = x[j];
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) l += red[w];
    const int64_t seq = h.x;
    T *o = reinterpret_cast<T *>(a.o) + seq * a.so_s + (first_head + r) * a.so_h;
    for (int d = threadIdx.x; d < a.head_dim; d += THREADS) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) y += part[w][d];
        o[d] = from_f32<T>(l == 0.0f ? 0.0f : __fdiv_rn(y, l));
    }
    if (threadIdx.x == 0 && a.lse) a.lse[seq * a.q_heads + first_head + r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ---- CUDA-core kernel: any head_dim up to 256, any dtype, any strides ----------------------------------
// Eight lanes share a key, four keys per warp at a time; a lane owns CH groups of four neighbouring elements of the head and
// keeps its part of q and O for ROWS query rows in registers, with statistics of its own per group of eight lanes.  K and V
// go straight from memory to registers.
template <typename T, bool VEC> __device__ __forceinline__ void load4(const T *p, int d, int head_dim, float (&f)[4]) {
    if (VEC) {
        if (sizeof(T) == 4) {
            const float4 x = *reinterpret_cast<const float4 *>(p + d);
            f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
        } else {
            struct alignas(8) H { T e[4]; };
            const H x = *reinterpret_cast<const H *>(p + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = to_f32(x.e[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = d + e < head_dim ? to_f32(p[d + e]) : 0.0f;
    }
}

template <typename T, int CH, int ROWS, bool VEC> __global__ void __launch_bounds__(THREADS) paged_simple_kernel(PagedArgs a) {
    __shared__ float so[WARPS * ROWS * MAX_HEAD_DIM], sm[WARPS][ROWS], sl[WARPS][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l8 = lane & 7, sub = lane >> 3;
    const int D = a.head_dim;
    grid_dependency_wait();
    walk_run<T, ROWS>(a, [&](int64_t seq, int kv_head, int first_head, int rows, int first, int skip, int keys, int t0, int t1, float *slot) {
        const T *qb = reinterpret_cast<const T *>(a.q) + seq * a.sq_s, *kb = reinterpret_cast<const T *>(a.k) + kv_head * a.sk_h;
        const T *vb = reinterpret_cast<const T *>(a.v) + kv_head * a.sv_h;
        float q[ROWS][CH][4], o[ROWS][CH][4], m[ROWS], l[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int d = (c * 8 + l8) * 4;
                if (r < rows && d < D) load4<T, VEC>(qb + (first_head + r) * a.sq_h, d, D, q[r][c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    q[r][c][e] = r < rows && d < D ? q[r][c][e] * a.scale : 0.0f;
                    o[r][c][e] = 0.0f;
                }
            }
        }
        const int stop = t1 * TILE < keys ? t1 * TILE : keys;
        for (int j0 = t0 * TILE + warp * 4; j0 < stop; j0 += 4 * WARPS) {  // the same trip count for the whole warp
            const int j = j0 + sub;
            int64_t page = 0;
            int row = 0;
            const bool in = j < stop && j >= skip && locate(a, seq, first + j, page, row);
            float k[CH][4], v[CH][4];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int d = (c * 8 + l8) * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) k[c][e] = v[c][e] = 0.0f;
                if (in && d < D) {
                    load4<T, VEC>(kb + page * a.sk_p + row * a.sk_t, d, D, k[c]);
                    load4<T, VEC>(vb + page * a.sv_p + row * a.sv_t, d, D, v[c]);
                }
            }
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                float s = 0.0f;
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s = fmaf(q[r][c][e], k[c][e], s);
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                if (!in) s = -INFINITY;
                if (s > m[r]) {
                    const float c0 = m[r] == -INFINITY ? 0.0f : fast_exp2(m[r] - s);
                    m[r] = s;
                    l[r] *= c0;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[r][c][e] *= c0;
                }
                const float p = in ? fast_exp2(s - (m[r] == -INFINITY ? 0.0f : m[r])) : 0.0f;
                l[r] += p;
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[r][c][e] = fmaf(p, v[c][e], o[r][c][e]);
            }
        }
        // join the four groups of lanes, then hand the warp's result over
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float mw = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 8));
            mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, 16));
            const float c0 = fast_exp2(m[r] - (mw == -INFINITY ? 0.0f : mw));
            float lw = l[r] * c0;
            lw += __shfl_xor_sync(0xffffffffu, lw, 8);
            lw += __shfl_xor_sync(0xffffffffu, lw, 16);
            if (lane == 0) {
                sm[warp][r] = mw;
                sl[warp][r] = lw;
            }
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = o[r][c][e] * c0;
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    const int d = (c * 8 + l8) * 4 + e;
                    if (sub == 0 && d < D) so[(warp * ROWS + r) * MAX_HEAD_DIM + d] = x;
                }
        }
        __syncthreads();
        write_piece<T, ROWS>(a, so, ROWS * MAX_HEAD_DIM, MAX_HEAD_DIM, sm, sl, rows, seq, first_head, slot, 0, D);
        __syncthreads();
    });
}

// ---- host ------------------------------------------------------------------------------------------
enum { V_TENSOR = 0, V_CORES = 1, VARIANTS = 2 };

// The tensor-core kernels take 16-bit types, head dimensions they are instantiated for, and 16-byte rows in the cache.
bool tensor_ok(const enc_paged_cache &c, int dtype) {
    if (dtype_size(dtype) != 2 || mma_ctas_per_sm(c.head_dim) == 0 || !aligned16(c.k) || !aligned16(c.v)) return false;
    for (int64_t s : {c.k_stride_page, c.k_stride_head, c.k_stride_token, c.v_stride_page, c.v_stride_head, c.v_stride_token})
        if (s % 8) return false;
    return true;
}

struct Plan {
    int variant, rows, row_groups, grid;
    int64_t work;
};

// Which kernel, how many query rows it takes at a time, how many CTAs, and the bytes for pieces.
void make_plan(const enc_paged_cache &c, int64_t q_heads, int dtype, int variant, Plan &p) {
    const int group = (int)(q_heads / c.kv_heads);
    p.variant = variant >= 0 ? variant : tensor_ok(c, dtype) ? V_TENSOR : V_CORES;
    p.rows = p.variant == V_TENSOR ? mma_rows(group) : group == 1 ? 1 : c.head_dim > 128 ? 2 : 4;
    const int per_sm = p.variant == V_TENSOR ? mma_ctas_per_sm(c.head_dim) : 4;
    p.row_groups = (int)cdiv(group, p.rows);
    const int64_t most = c.num_seqs * c.kv_heads * p.row_groups * cdiv(paged_capacity(c), TILE);  // tiles if every row is full
    const int64_t fill = (int64_t)device_props().sm_count * per_sm;
    p.grid = (int)(most < fill ? (most > 0 ? most : 1) : fill);
    // sequences of one tile are never cut
    p.work = paged_capacity(c) <= TILE ? 0 : (int64_t)p.grid * 16 + 2 * (int64_t)p.grid * p.rows * (c.head_dim + 2) * 4;
}

template <typename T, int ROWS> void launch_join(const PagedArgs &a, int grid, cudaStream_t st) {
    const int rows = a.group < ROWS ? a.group : ROWS;
    if (a.headers) launch_overlapped(join_kernel<T, ROWS>, dim3(grid, rows), dim3(THREADS), 0, st, a);
}

template <typename T, int CH, int ROWS>
void launch_simple(const PagedArgs &a, int grid, bool vec, cudaStream_t st) {
    if (vec) launch_overlapped(paged_simple_kernel<T, CH, ROWS, true>, dim3(grid), dim3(THREADS), 0, st, a);
    else launch_overlapped(paged_simple_kernel<T, CH, ROWS, false>, dim3(grid), dim3(THREADS), 0, st, a);
    launch_join<T, ROWS>(a, grid, st);
}

template <typename T> int launch_paged(const PagedArgs &a, const Plan &p, cudaStream_t st) {
    note_indexed_launch();
    if constexpr (sizeof(T) == 2) {
        if (p.variant == V_TENSOR) {
            const int rc = launch_mma(a, std::is_same<T, __half>::value ? ENC_F16 : ENC_BF16, p.grid, st);
            if (rc != ENC_OK) return rc;
            if (p.rows == 8) launch_join<T, 8>(a, p.grid, st);
            else launch_join<T, 16>(a, p.grid, st);
            return check_launch("enc_paged_attention");
        }
    }
    const int nv = 4;
    bool vec = a.head_dim % nv == 0;
    for (const void *x : {a.q, a.k, a.v}) vec = vec && reinterpret_cast<uintptr_t>(x) % (nv * sizeof(T)) == 0;
    for (int64_t s : {a.sq_s, a.sq_h, a.sk_p, a.sk_h, a.sk_t, a.sv_p, a.sv_h, a.sv_t}) vec = vec && s % nv == 0;
    if (a.head_dim > 128) {
        if (p.rows == 1) launch_simple<T, 8, 1>(a, p.grid, vec, st);
        else launch_simple<T, 8, 2>(a, p.grid, vec, st);
    } else if (a.head_dim > 64) {
        if (p.rows == 1) launch_simple<T, 4, 1>(a, p.grid, vec, st);
        else launch_simple<T, 4, 4>(a, p.grid, vec, st);
    } else {
        if (p.rows == 1) launch_simple<T, 2, 1>(a, p.grid, vec, st);
        else launch_simple<T, 2, 4>(a, p.grid, vec, st);
    }
    return check_launch("enc_paged_attention");
}

int check_paged(const enc_paged_cache *c, int64_t q_heads, int dtype, int variant, const char *me) {
    if (!c) return fail(ENC_ERR_BAD_ARG, "%s: NULL cache", me);
    if (!is_float_dtype(dtype)) return fail(ENC_ERR_BAD_ARG, "%s: dtype %d is not float16, bfloat16 or float32", me, dtype);
    if (variant >= VARIANTS) return fail(ENC_ERR_BAD_ARG, "%s: variant %d out of range", me, variant);
    const int bad = check_cache(*c, me);
    if (bad) return bad;
    if (c->head_dim > MAX_HEAD_DIM) return fail(ENC_ERR_UNSUPPORTED, "%s: head_dim %lld > %d", me, (long long)c->head_dim, MAX_HEAD_DIM);
    if (q_heads < 1 || q_heads % c->kv_heads) return fail(ENC_ERR_BAD_ARG, "%s: %lld query heads over %lld kv heads", me, (long long)q_heads, (long long)c->kv_heads);
    if (q_heads > 0xffff) return fail(ENC_ERR_UNSUPPORTED, "%s: more than 65535 query heads", me);
    if (variant == V_TENSOR && !tensor_ok(*c, dtype))
        return fail(ENC_ERR_UNSUPPORTED, "%s: variant %d needs float16 or bfloat16, another head_dim, or 16-byte aligned cache rows", me, variant);
    return 0;
}

}  // namespace

unsigned int take_bad_index_paged_mma();
unsigned int take_bad_index_paged_attention() { return take_bad_index_word() | take_bad_index_paged_mma(); }
int paged_attention_variants() { return VARIANTS; }
void paged_attention_variant_info(int v, char *out, size_t n) {
    if (v == V_TENSOR) snprintf(out, n, "mma m16n8k16, 16 keys by 8 or 16 query rows per warp and step, keys and values through a cp.async ring");
    else snprintf(out, n, "CUDA cores, eight lanes per key, keys and values straight to registers");
}

}  // namespace enc

extern "C" int64_t enc_paged_attention_work_bytes(const enc_paged_cache *cache, int64_t q_heads, int dtype, int variant) {
    using namespace enc;
    if (check_paged(cache, q_heads, dtype, variant, "enc_paged_attention_work_bytes")) return -1;
    Plan p;
    make_plan(*cache, q_heads, dtype, variant, p);
    return p.work;
}

extern "C" int enc_paged_attention(const enc_paged_cache *cache, const void *q, void *o, float *lse, const int32_t *seq_lens,
                                   int64_t q_heads, int64_t q_stride_seq, int64_t q_stride_head, int64_t o_stride_seq,
                                   int64_t o_stride_head, float sm_scale, int64_t window, void *work, int64_t work_bytes,
                                   int dtype, int variant, void *stream) {
    ENC_PROLOGUE();
    using namespace enc;
    const char *me = "enc_paged_attention";
    const int bad = check_paged(cache, q_heads, dtype, variant, me);
    if (bad) return bad;
    if (window < 0) return fail(ENC_ERR_BAD_ARG, "%s: negative window", me);
    if (cache->num_seqs == 0) return ENC_OK;
    if (!q || !o || !seq_lens) return fail(ENC_ERR_BAD_ARG, "%s: NULL tensor", me);
    if ((!cache->k || !cache->v || !cache->block_table) && paged_capacity(*cache) > 0 && cache->num_pages > 0)
        return fail(ENC_ERR_BAD_ARG, "%s: NULL cache tensor", me);
    Plan p;
    make_plan(*cache, q_heads, dtype, variant, p);
    if (p.work > 0 && (!work || work_bytes < p.work || !aligned16(work)))
        return fail(ENC_ERR_BAD_ARG, "%s: needs %lld bytes of 16-byte aligned workspace, got %lld", me, (long long)p.work, (long long)work_bytes);
    PagedArgs a{};
    a.q = q; a.k = cache->k; a.v = cache->v; a.o = o; a.lse = lse;
    a.block_table = cache->block_table; a.seq_lens = seq_lens;
    a.headers = p.work ? reinterpret_cast<int4 *>(work) : nullptr;
    a.slots = p.work ? reinterpret_cast<float *>(reinterpret_cast<char *>(work) + (int64_t)p.grid * 16) : nullptr;
    a.sq_s = q_stride_seq; a.sq_h = q_stride_head; a.so_s = o_stride_seq; a.so_h = o_stride_head;
    a.sk_p = cache->k_stride_page; a.sk_h = cache->k_stride_head; a.sk_t = cache->k_stride_token;
    a.sv_p = cache->v_stride_page; a.sv_h = cache->v_stride_head; a.sv_t = cache->v_stride_token;
    a.s_table = cache->stride_table;
    a.num_seqs = cache->num_seqs; a.num_pages = cache->num_pages; a.capacity = paged_capacity(*cache); a.window = window;
    a.q_heads = (int)q_heads; a.head_dim = (int)cache->head_dim; a.group = (int)(q_heads / cache->kv_heads);
    a.row_groups = p.row_groups; a.units = (int)cache->kv_heads * p.row_groups;
    a.whole = cache->page_size % 16 == 0;
    a.min_run = 1;
    a.scale = sm_scale * LOG2E;
    a.page_size = FastDiv((uint32_t)cache->page_size);
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ENC_F16: return launch_paged<__half>(a, p, st);
        case ENC_BF16: return launch_paged<__nv_bfloat16>(a, p, st);
        default: return launch_paged<float>(a, p, st);
    }
}

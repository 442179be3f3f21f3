// Attention of one new token per sequence over a paged key-value cache: the CUDA-core kernel, the join of split rows and the
// entry points.  Mathematics, bound and split are in paged_attention.cuh.
#include "paged_attention.cuh"

#include <type_traits>

namespace enc {
using namespace paged;
namespace {

// ---- join ------------------------------------------------------------------------------------------
// Where a run's last piece begins a row group, the pieces of that group are that piece and the first pieces of the runs after
// it.  A CTA looks through its share of the headers.  Rows cut into few pieces (up to JOIN_FEW) go to a warp each, all rows
// of the CTA's headers side by side; rows cut into many (one long sequence has one per run) take the whole CTA, its warps
// every JOIN_WARPS-th piece and then their results.  Lanes hold four neighbouring elements each; JOIN_DEEP pieces are in
// flight per warp, because each is a trip to L2; one pass with a running maximum.
constexpr int JOIN_WARPS = 8, JOIN_DEEP = 4, JOIN_FEW = 4 * JOIN_DEEP, JOIN_HEADERS = 64;

struct Partial {
    float x[4], m, l;
};
// Elements d .. d + 3 of the pieces first, first + step, ... of a row, joined.  pieces: piece 0 of the row's first run.
__device__ __forceinline__ Partial join_pieces(const float *pieces, int64_t piece_stride, int ml_at, int d, int first, int n, int step) {
    Partial s = {{0.0f, 0.0f, 0.0f, 0.0f}, -INFINITY, 0.0f};
    for (int i = first; i < n; i += JOIN_DEEP * step) {
        float4 y[JOIN_DEEP];
        float2 ml[JOIN_DEEP];
#pragma unroll
        for (int u = 0; u < JOIN_DEEP; ++u) {
            const int p = i + u * step;
            ml[u] = make_float2(-INFINITY, 0.0f);
            y[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (p < n) {
                const float *at = pieces + (p == 0 ? 1 : 2 * p) * piece_stride;
                y[u] = *reinterpret_cast<const float4 *>(at + d);
                ml[u] = *reinterpret_cast<const float2 *>(at + ml_at);
            }
        }
        float top = s.m;
#pragma unroll
        for (int u = 0; u < JOIN_DEEP; ++u) top = fmaxf(top, ml[u].x);
        const float base = top == -INFINITY ? 0.0f : top, down = fast_exp2(s.m - base);
        s.m = top;
        s.l *= down;
#pragma unroll
        for (int e = 0; e < 4; ++e) s.x[e] *= down;
#pragma unroll
        for (int u = 0; u < JOIN_DEEP; ++u) {
            const float w = fast_exp2(ml[u].x - base);
            s.l = fmaf(ml[u].y, w, s.l);
            s.x[0] = fmaf(y[u].x, w, s.x[0]); s.x[1] = fmaf(y[u].y, w, s.x[1]);
            s.x[2] = fmaf(y[u].z, w, s.x[2]); s.x[3] = fmaf(y[u].w, w, s.x[3]);
        }
    }
    return s;
}
template <typename T> __device__ __forceinline__ void write_row(const PagedArgs &a, int64_t seq, int head, int d, const Partial &s) {
    store4<T>(reinterpret_cast<T *>(a.o) + seq * a.so_s + head * a.so_h, d, a.head_dim, s.x, s.l);
    if (d == 0 && a.lse) a.lse[seq * a.q_heads + head] = s.l == 0.0f ? -INFINITY : (s.m + log2f(s.l)) * LN2;
}

template <typename T, int ROWS> __global__ void __launch_bounds__(JOIN_WARPS * 32, 4) join_kernel(PagedArgs a, int grid) {
    __shared__ int4 header[JOIN_HEADERS];
    __shared__ Partial parts[JOIN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int stride = (int)slot_stride(a.head_dim), width = stride - 4;  // floats of a row, elements
    grid_dependency_wait();
    for (int h0 = blockIdx.x; h0 < grid; h0 += JOIN_HEADERS * gridDim.x) {
        const int left = (grid - h0 + (int)gridDim.x - 1) / (int)gridDim.x, count = left < JOIN_HEADERS ? left : JOIN_HEADERS;
        __syncthreads();
        if (threadIdx.x < count) {
            const int id = h0 + threadIdx.x * gridDim.x, runs = a.headers[grid].x;
            int4 h = a.headers[id];
            if (id >= runs) h.y = 0;  // behind the last run with tiles nothing was written
            h.w = h.z - id + 1;       // pieces
            header[threadIdx.x] = h;
        }
        __syncthreads();
        auto pieces_of = [&](int k, int r) { return slot_of(a, h0 + (int64_t)k * gridDim.x, 0, ROWS) + r * stride; };
        for (int it = blockIdx.y * JOIN_WARPS + warp; it < count * ROWS; it += gridDim.y * JOIN_WARPS) {
            const int k = it / ROWS, r = it % ROWS;
            const int4 h = header[k];
            if (r >= (h.y & 255) || h.w > JOIN_FEW) continue;
            for (int d = lane * 4; d < width; d += 128)
                write_row<T>(a, h.x, (h.y >> 8) + r, d, join_pieces(pieces_of(k, r), ROWS * stride, stride - 4, d, 0, h.w, 1));
        }
        for (int k = 0; k < count; ++k) {
            const int4 h = header[k];
            if ((h.y & 255) == 0 || h.w <= JOIN_FEW) continue;
            for (int r = blockIdx.y; r < (h.y & 255); r += gridDim.y)
                for (int d0 = 0; d0 < width; d0 += 128) {
                    const int d = d0 + lane * 4;
                    if (d < width) parts[warp][lane] = join_pieces(pieces_of(k, r), ROWS * stride, stride - 4, d, warp, h.w, JOIN_WARPS);
                    __syncthreads();
                    if (warp == 0 && d < width) {
                        Partial s = parts[0][lane];
#pragma unroll
                        for (int w = 1; w < JOIN_WARPS; ++w) s.m = fmaxf(s.m, parts[w][lane].m);
                        const float base = s.m == -INFINITY ? 0.0f : s.m;
                        s.l = s.x[0] = s.x[1] = s.x[2] = s.x[3] = 0.0f;
#pragma unroll
                        for (int w = 0; w < JOIN_WARPS; ++w) {
                            const Partial &p = parts[w][lane];
                            const float c = fast_exp2(p.m - base);
                            s.l = fmaf(p.l, c, s.l);
#pragma unroll
                            for (int e = 0; e < 4; ++e) s.x[e] = fmaf(p.x[e], c, s.x[e]);
                        }
                        write_row<T>(a, h.x, (h.y >> 8) + r, d, s);
                    }
                    __syncthreads();
                }
        }
    }
}

// ---- CUDA-core kernel: any head_dim up to 256, any dtype, any strides ----------------------------------
// Eight lanes share a key, four keys per warp at a time; a lane owns CH groups of four neighbouring elements of the head and
// keeps its part of q and O for ROWS query rows in registers, with statistics of its own per group of eight lanes.  K and V
// go straight from memory to registers, KEYS keys per group at once: a step is a trip to memory, so what is in flight per
// trip is what counts.
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

constexpr int cores_ctas_per_sm(int ch, int rows) { return ch * rows <= 2 ? 4 : ch * rows <= 8 ? 3 : 2; }

template <typename T, int CH, int ROWS, bool VEC> __global__ void __launch_bounds__(THREADS, cores_ctas_per_sm(CH, ROWS)) paged_simple_kernel(PagedArgs a) {
    constexpr int KEYS = CH <= 2 ? 4 : CH == 4 ? 2 : 1;
    __shared__ __align__(16) float so[WARPS * ROWS * MAX_HEAD_DIM];
    __shared__ float sm[WARPS][ROWS], sl[WARPS][ROWS];
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
        // KEYS keys per group of lanes and step, all of their loads under way together; their pages are looked up a step ahead
        const int stop = t1 * TILE < keys ? t1 * TILE : keys;
        int64_t place_page[KEYS];
        int place_row[KEYS];
        uint32_t there = 0;
        auto look_up = [&](int j0) {
            there = 0;
#pragma unroll
            for (int u = 0; u < KEYS; ++u) {
                const int j = j0 + 4 * u + sub;
                place_page[u] = 0;
                place_row[u] = 0;
                if (j < stop && j >= skip && locate(a, seq, first + j, place_page[u], place_row[u])) there |= 1u << u;
            }
        };
        const int start = t0 * TILE + warp * 4 * KEYS;
        look_up(start);
        for (int j0 = start; j0 < stop; j0 += 4 * KEYS * WARPS) {  // the same trip count for the whole warp
            float k[KEYS][CH][4], v[KEYS][CH][4];
            const uint32_t in = there;
#pragma unroll
            for (int u = 0; u < KEYS; ++u)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int d = (c * 8 + l8) * 4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[u][c][e] = v[u][c][e] = 0.0f;
                    if ((in >> u & 1) && d < D) {
                        load4<T, VEC>(kb + place_page[u] * a.sk_p + place_row[u] * a.sk_t, d, D, k[u][c]);
                        load4<T, VEC>(vb + place_page[u] * a.sv_p + place_row[u] * a.sv_t, d, D, v[u][c]);
                    }
                }
            look_up(j0 + 4 * KEYS * WARPS);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                float s[KEYS], top = m[r];
#pragma unroll
                for (int u = 0; u < KEYS; ++u) {
                    s[u] = 0.0f;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[u] = fmaf(q[r][c][e], k[u][c][e], s[u]);
                    s[u] += __shfl_xor_sync(0xffffffffu, s[u], 1);
                    s[u] += __shfl_xor_sync(0xffffffffu, s[u], 2);
                    s[u] += __shfl_xor_sync(0xffffffffu, s[u], 4);
                    if (!(in >> u & 1)) s[u] = -INFINITY;
                    top = fmaxf(top, s[u]);
                }
                if (top > m[r]) {
                    const float down = m[r] == -INFINITY ? 0.0f : fast_exp2(m[r] - top);
                    m[r] = top;
                    l[r] *= down;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[r][c][e] *= down;
                }
                const float base = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
                for (int u = 0; u < KEYS; ++u) {
                    const float p = fast_exp2(s[u] - base);
                    l[r] += p;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[r][c][e] = fmaf(p, v[u][c][e], o[r][c][e]);
                }
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
enum { V_RING = 0, V_CORES = 1, VARIANTS = 2 };

// The ring kernels take the head dimensions they are instantiated for, and 16-byte rows in the cache.
bool ring_ok(const enc_paged_cache &c, int dtype) {
    // (an empty cache has no address that a copy could name)
    if (ring_ctas_per_sm(dtype, c.head_dim) == 0 || !c.k || !c.v || !aligned16(c.k) || !aligned16(c.v)) return false;
    for (int64_t s : {c.k_stride_page, c.k_stride_head, c.k_stride_token, c.v_stride_page, c.v_stride_head, c.v_stride_token})
        if (s % (16 / (int64_t)dtype_size(dtype))) return false;
    return true;
}

struct Plan {
    int variant, rows, row_groups, long_runs, grid;
    int64_t work;
    bool by_rows;
};

// Which kernel, how many query rows it takes at a time, how many CTAs, and the bytes for pieces.
void make_plan(const enc_paged_cache &c, int64_t q_heads, int dtype, int variant, Plan &p) {
    const int group = (int)(q_heads / c.kv_heads);
    p.variant = variant >= 0 ? variant : ring_ok(c, dtype) ? V_RING : V_CORES;
    p.rows = p.variant == V_RING ? ring_rows(dtype, group) : group == 1 ? 1 : c.head_dim > 128 ? 2 : 4;
    const int ch = c.head_dim > 128 ? 8 : c.head_dim > 64 ? 4 : 2;
    const int per_sm = p.variant == V_RING ? ring_ctas_per_sm(dtype, c.head_dim) : cores_ctas_per_sm(ch, p.rows);
    p.row_groups = (int)cdiv(group, p.rows);
    const int64_t units = c.num_seqs * c.kv_heads * p.row_groups, row_tiles = cdiv(paged_capacity(c), TILE);
    p.by_rows = row_tiles <= ROW_TILES;
    const int64_t most = p.by_rows ? units : units * row_tiles;  // the line's length if every row is full
    const int64_t fill = (int64_t)device_props().sm_count * per_sm;
    p.long_runs = (int)(most < fill ? (most > 0 ? most : 1) : fill);
    // Short runs even out the SMs (see paged_attention.cuh) but cost two microseconds each: measured at 48 x 32 kv heads (664
    // tiles a CTA at most) 685 us without, 637 with two per long run, 618 with six; at 64 x 8 (110 tiles) 105, 102, 140.  With
    // fewer rows than CTAs every short run is a piece that the join has to fetch (2 x 4: 101 us without, 120 with two).
    const int shorts = p.variant != V_RING || p.by_rows || units < fill || most < 64 * fill ? 0 : most < 256 * fill ? 2 : 6;
    p.grid = p.long_runs * (1 + shorts);
    p.work = p.by_rows ? 0 : (int64_t)(p.grid + 1) * 16 + 2 * (int64_t)p.grid * p.rows * slot_stride((int)c.head_dim) * 4;
}

template <typename T, int ROWS> void launch_join(const PagedArgs &a, int grid, cudaStream_t st) {
    if (!a.headers) return;
    // CTAs side by side for the rows of a group where groups are cut into many pieces, so few of them have a header at all
    const int most = 4 * device_props().sm_count;
    const bool many = a.num_seqs * a.units * JOIN_FEW < grid;
    launch_overlapped(join_kernel<T, ROWS>, dim3((unsigned)(grid < most ? grid : most), many ? (unsigned)(a.group < ROWS ? a.group : ROWS) : 1u), dim3(JOIN_WARPS * 32), 0, st, a, grid);
}

template <typename T, int CH, int ROWS>
void launch_simple(const PagedArgs &a, int grid, bool vec, cudaStream_t st) {
    if (vec) launch_overlapped(paged_simple_kernel<T, CH, ROWS, true>, dim3(grid), dim3(THREADS), 0, st, a);
    else launch_overlapped(paged_simple_kernel<T, CH, ROWS, false>, dim3(grid), dim3(THREADS), 0, st, a);
    launch_join<T, ROWS>(a, grid, st);
}

template <typename T> int launch_paged(const PagedArgs &a, const Plan &p, cudaStream_t st) {
    note_indexed_launch();
    if (p.variant == V_RING) {
        const int dtype = std::is_same<T, float>::value ? ENC_F32 : std::is_same<T, __half>::value ? ENC_F16 : ENC_BF16;
        const int rc = launch_ring(a, dtype, p.grid, st);
        if (rc != ENC_OK) return rc;
        if constexpr (sizeof(T) == 4) {
            if (p.rows == 1) launch_join<T, 1>(a, p.grid, st);
            else launch_join<T, 4>(a, p.grid, st);
        } else {
            if (p.rows == 8) launch_join<T, 8>(a, p.grid, st);
            else launch_join<T, 16>(a, p.grid, st);
        }
        return check_launch("enc_paged_attention");
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
    if ((double)c->num_seqs * (double)q_heads * (double)cdiv(paged_capacity(*c), TILE) >= 2147400000.0)  // (room for a run more)
        return fail(ENC_ERR_UNSUPPORTED, "%s: %lld sequences of up to %lld keys with %lld heads pass 2^31 tiles of %d keys", me,
                    (long long)c->num_seqs, (long long)paged_capacity(*c), (long long)q_heads, TILE);
    if (variant == V_RING && !ring_ok(*c, dtype))
        return fail(ENC_ERR_UNSUPPORTED, "%s: variant %d needs another head_dim, or 16-byte aligned cache rows", me, variant);
    return 0;
}

}  // namespace

unsigned int take_bad_index_paged_ring();
unsigned int take_bad_index_paged_attention() { return take_bad_index_word() | take_bad_index_paged_ring(); }
int paged_attention_variants() { return VARIANTS; }
void paged_attention_variant_info(int v, char *out, size_t n) {
    if (v == V_RING) snprintf(out, n, "keys and values through a cp.async ring per warp, 16 keys a step; 16-bit types by mma m16n8k16, float32 on CUDA cores");
    else snprintf(out, n, "CUDA cores, eight lanes per key, keys and values straight to registers");
}

}  // namespace enc

extern "C" int64_t enc_paged_attention_work_bytes(const enc_paged_cache *cache, int64_t q_heads, int dtype, int variant) {
    using namespace enc;
    if (check_paged(cache, q_heads, dtype, variant < 0 ? -1 : V_CORES, "enc_paged_attention_work_bytes") || variant >= VARIANTS) return -1;
    int64_t most = 0;
    for (int v = 0; v < VARIANTS; ++v) {
        if ((variant >= 0 && v != variant) || (v == V_RING && ring_ctas_per_sm(dtype, cache->head_dim) == 0)) continue;
        Plan p;
        make_plan(*cache, q_heads, dtype, v, p);
        if (p.work > most) most = p.work;
    }
    return most;
}

extern "C" int enc_paged_attention(const enc_paged_cache *cache, const enc_paged_attention_args *args, int dtype, int variant, void *stream) {
    ENC_PROLOGUE();
    using namespace enc;
    const char *me = "enc_paged_attention";
    if (!args) return fail(ENC_ERR_BAD_ARG, "%s: NULL arguments", me);
    const enc_paged_attention_args &g = *args;
    const int64_t q_heads = g.q_heads;
    const int bad = check_paged(cache, q_heads, dtype, variant, me);
    if (bad) return bad;
    if (g.window < 0) return fail(ENC_ERR_BAD_ARG, "%s: negative window", me);
    if (cache->num_seqs == 0) return ENC_OK;
    if (!g.q || !g.o || !g.seq_lens) return fail(ENC_ERR_BAD_ARG, "%s: NULL tensor", me);
    if ((!cache->k || !cache->v || !cache->block_table) && paged_capacity(*cache) > 0 && cache->num_pages > 0)
        return fail(ENC_ERR_BAD_ARG, "%s: NULL cache tensor", me);
    Plan p;
    make_plan(*cache, q_heads, dtype, variant, p);
    if (p.work > 0 && (!g.work || g.work_bytes < p.work || !aligned16(g.work)))
        return fail(ENC_ERR_BAD_ARG, "%s: needs %lld bytes of 16-byte aligned workspace, got %lld", me, (long long)p.work, (long long)g.work_bytes);
    PagedArgs a{};
    a.q = g.q; a.k = cache->k; a.v = cache->v; a.o = g.o; a.lse = g.lse;
    a.block_table = cache->block_table; a.seq_lens = g.seq_lens;
    a.headers = p.work ? reinterpret_cast<int4 *>(g.work) : nullptr;
    a.slots = p.work ? reinterpret_cast<float *>(reinterpret_cast<char *>(g.work) + (int64_t)(p.grid + 1) * 16) : nullptr;
    a.sq_s = g.q_stride_seq; a.sq_h = g.q_stride_head; a.so_s = g.o_stride_seq; a.so_h = g.o_stride_head;
    a.sk_p = cache->k_stride_page; a.sk_h = cache->k_stride_head; a.sk_t = cache->k_stride_token;
    a.sv_p = cache->v_stride_page; a.sv_h = cache->v_stride_head; a.sv_t = cache->v_stride_token;
    a.s_table = cache->stride_table;
    a.num_seqs = cache->num_seqs; a.num_pages = cache->num_pages; a.capacity = paged_capacity(*cache); a.window = g.window;
    a.q_heads = (int)q_heads; a.head_dim = (int)cache->head_dim; a.group = (int)(q_heads / cache->kv_heads);
    a.row_groups = p.row_groups; a.units = (int)cache->kv_heads * p.row_groups;
    a.whole = cache->page_size % 16 == 0;
    a.long_runs = p.long_runs;
    a.by_rows = p.by_rows;
    a.scale = (float)(g.sm_scale * 1.4426950408889634);
    a.page_size = FastDiv((uint32_t)cache->page_size);
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ENC_F16: return launch_paged<__half>(a, p, st);
        case ENC_BF16: return launch_paged<__nv_bfloat16>(a, p, st);
        default: return launch_paged<float>(a, p, st);
    }
}

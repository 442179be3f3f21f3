// Attention of one new token per sequence over a paged key-value cache: the kernels with a ring per warp, for rows of 16-byte
// vectors.  Mathematics, bound and split are in paged_attention.cuh.
//
// Each warp has a ring of its own in shared memory and walks its keys without CTA barriers: 16 keys and 16 values per stage,
// 16-byte asynchronous copies, rows padded by 16 bytes so that ldmatrix meets no bank twice.  The ring runs on across the
// pieces of a run: the next row's keys are on their way while a finished one is joined and written.
//
// 16-bit types.  The query heads that share a kv head are the columns of an m16n8k16 product: S^T = K Q^T over 16 keys per warp
// and step, and O^T += V^T P^T over the same 16 keys, 8 heads at a time (two column blocks for 9 to 16).  With the keys as rows
// nothing is padded up to 16 but the keys themselves: against queries as rows the matrix instructions and the registers of O
// and Q halve for groups of up to 8 heads.  P^T needs the layout of S^T transposed: one movmatrix per 8 x 8 block.  The
// kernel is bound by HBM as long as a warp's step (365 instructions on 8 KB, 24 of them products) stays short; the tensor
// pipe's rate does not matter.  What the matrix instruction buys is that the work per key hardly grows with the number of
// query heads.  tcgen05 would need 128 rows of keys or queries to fill its smallest tile.
//
// P is fed as the sum of two 16-bit numbers, P = hi + lo, in two products: the weights keep 16 or more bits instead of 8 or 11
// and the output is as exact as a float32 product rounded once.
//
// The maximum that weights are taken relative to moves only when a score passes it by SLACK powers of two, so nearly all
// steps need neither the reduction over the keys nor the rescaling; l and O use the same reference, so the result is the
// same.  In fp16 the reference is kept 14 powers of two below the maximum it was taken from, so that weights down to 2^-28 of
// the largest are normal numbers, and it moves as soon as a weight would pass 2^15.
//
// float32.  CUDA cores (CoreRows): four query rows at a time, eight lanes to a key.
//
// Measured (a pass among others, inputs of 0.5 to 4 GB beyond L2): bf16, 48 sequences of 2000 to 8192 keys, 32 heads of 128
// with keys of their own: 610 us, 6.57 TB/s; 64 of 1 to 4096 keys, 32 heads over 8: 102 us, 5.1 TB/s, of which 23 us do not
// grow with the batch (two launches, the first loads, the uneven ends, the join); 2 of 100000 and 131072 keys, 32 over 4,
// fp16: 93 us, 5.1 TB/s.
#include <type_traits>

#include "paged_attention.cuh"

namespace enc {
namespace paged {
namespace {

template <typename T, int D, int STAGES> struct Ring {
    static constexpr int PITCH = (int)sizeof(T) * D + 16;  // bytes of a key or value row
    static constexpr int HALF = 16 * PITCH;                // 16 keys (or values)
    static constexpr int WARP = STAGES * 2 * HALF;
    static constexpr int TOTAL = WARPS * WARP;
};
// Floats of a row of partial results: 4 more than a multiple of 16, so that the 8 elements x 4 row pairs that a warp writes
// at a time (TensorRows) meet 32 banks.
__host__ __device__ constexpr int part_stride(int dims) { return dims + 4; }

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t &>(x);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 x = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t &>(x);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t x);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t x) { return __half22float2(reinterpret_cast<const __half2 &>(x)); }

// The runs of a CTA: its own block's first, then the runs of blocks that have not started, which it claims from the hardware's
// queue (clusterlaunchcontrol: a claimed block never starts).  One claim is under way while a run is worked on; after a run
// without tiles (there are none behind it) or a refusal no cursor claims more.  CLAIMS answers are kept: between the warps'
// loading cursors lie at most STAGES tiles and two pieces, and a run has at least one tile.
constexpr int CLAIMS = 16;
struct Claims {
    uint4 answer[CLAIMS];
    uint64_t arrived[CLAIMS];
    uint32_t gave_up;
};
__device__ __forceinline__ void claim(Claims &c, int i) {  // by one thread; i counts the CTA's runs
    sm100::fence_proxy_async();
    sm100::mbar_expect_tx(&c.arrived[i % CLAIMS], sizeof(uint4));
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(&c.answer[i % CLAIMS])), "r"(smem_u32(&c.arrived[i % CLAIMS])) : "memory");
}
// The i-th run's number, or -1 when there is none left (or the answer did not come within the bound of every wait).
__device__ __forceinline__ int claimed(Claims &c, int i) {
    if (!sm100::mbar_wait(&c.arrived[i % CLAIMS], (i / CLAIMS) & 1, &c.gave_up)) {
        atomicExch(&g_bad_index, 2u);
        return -1;
    }
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .pred P;\n\t.reg .b128 A;\n\tld.shared.b128 A, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 P, A;\n\tselp.u32 %0, 1, 0, P;\n\tmov.u32 %1, 0;\n\t"
        "@P clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, A;\n\t}"
        : "=r"(ok), "=r"(x) : "r"(smem_u32(&c.answer[i % CLAIMS])) : "memory");
    return ok ? (int)x : -1;
}

// A place in the CTA's runs: a tile of one unit (kv head and row group) of one sequence.
struct Cursor {
    int64_t seq;
    int left, end;           // tiles (by rows: row groups) left in the run, the line's tile behind it
    int run;                 // its number; -1: all done
    int unit, t, tiles, keys, first, skip;

    __device__ __forceinline__ void read_keys(const PagedArgs &a) {
        keys = keys_of(a, seq, first, skip);
        tiles = tiles_of(keys);
    }
    // Goes to run `id`, which may be empty.
    __device__ __forceinline__ void start(const PagedArgs &a, const Line &line, const int (&before)[THREADS], int id) {
        run = id;
        int begin, at;
        line.run(a, id, begin, end);
        left = end - begin;
        if (left <= 0) return;
        find_tile(a, before, begin, seq, at);
        read_keys(a);
        const int weight = weight_of(a, keys);
        unit = at / weight;
        t = at - unit * weight;
    }
    // One tile on, inside the run.
    __device__ __forceinline__ void next(const PagedArgs &a) {
        if (!a.by_rows) --left;
        if (++t < tiles) return;
        t = 0;
        if (a.by_rows) --left;
        if (++unit < a.units || left <= 0) return;
        unit = 0;
        do {  // (left > 0: a sequence with keys follows)
            ++seq;
            read_keys(a);
        } while (keys == 0);
    }
};
// The runs that a warp's loading cursor has entered and its finishing cursor has not: at most one per stage, and one.
template <int STAGES> struct RunQueue {
    Cursor at[STAGES + 2];
};

// What a warp does with 16 keys and values of its ring for up to ROWS query rows: the queries, O, the maximum and the sum.
//   16-bit types: matrix instructions.  Columns are query rows, NQ blocks of eight.
template <typename T, int D, int NQ> struct TensorRows {
    static constexpr int ROWS = 8 * NQ, KS = D / 16, PITCH = 2 * D + 16;  // KS: steps of the first product
    static constexpr float LOWER = std::is_same<T, __half>::value ? 14.0f : 0.0f, SLACK = std::is_same<T, __half>::value ? 15.0f : 16.0f;
    uint32_t q[KS][NQ][2];
    float o[KS][NQ][4], m[NQ][2], l[NQ][2];  // O^T: rows i * 16 + lr (+ 8) of the head, columns lc, lc + 1 of the query block
    int lane, lr, lc;                        // this thread's row (and row + 8) and first column in accumulators

    __device__ __forceinline__ explicit TensorRows(int lane_) : lane(lane_), lr(lane_ >> 2), lc((lane_ & 3) * 2) { clear(); }
    __device__ __forceinline__ void clear() {  // nothing seen yet
#pragma unroll
        for (int b = 0; b < NQ; ++b) {
            m[b][0] = m[b][1] = -INFINITY;
            l[b][0] = l[b][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[i][b][x] = 0.0f;
        }
    }
    __device__ __forceinline__ void ask_queries(const PagedArgs &a, const T *qp, int rows) {
#pragma unroll
        for (int b = 0; b < NQ; ++b) {
            const T *p = qp + (b * 8 + lr) * a.sq_h + lc;
            const bool there = b * 8 + lr < rows;
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) {
                uint32_t v = 0;
                if (there && a.q_pairs) v = *reinterpret_cast<const uint32_t *>(p + i * 8);
                else if (there) v = (uint32_t)*reinterpret_cast<const uint16_t *>(p + i * 8) | (uint32_t)*reinterpret_cast<const uint16_t *>(p + i * 8 + 1) << 16;
                q[i / 2][b][i % 2] = v;
            }
        }
    }
    // The keys from `skip` on, `left` of them.
    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t ks, uint32_t vs, int left, int skip) {
        float s[NQ][4];
        {
            float odd[NQ][4] = {};  // two chains of products, added at the end
#pragma unroll
            for (int b = 0; b < NQ; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[b][x] = 0.0f;
            const uint32_t kaddr = ks + (lane & 15) * PITCH + (lane >> 4) * 16;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t k[4];
                ldsm4(k, kaddr + i * 32);
#pragma unroll
                for (int b = 0; b < NQ; ++b) mma16816<T>(i & 1 ? odd[b] : s[b], k, q[i][b][0], q[i][b][1]);
            }
#pragma unroll
            for (int b = 0; b < NQ; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[b][x] = (s[b][x] + odd[b][x]) * a.scale;
        }
        if (left < 16) {
#pragma unroll
            for (int b = 0; b < NQ; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (lr + (x >> 1) * 8 >= left) s[b][x] = -INFINITY;
        }
        if (skip > 0) {  // keys in front of the window
#pragma unroll
            for (int b = 0; b < NQ; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (lr + (x >> 1) * 8 < skip) s[b][x] = -INFINITY;
        }
        bool over = false;
#pragma unroll
        for (int b = 0; b < NQ; ++b) over |= fmaxf(s[b][0], s[b][2]) > m[b][0] + SLACK || fmaxf(s[b][1], s[b][3]) > m[b][1] + SLACK;
        if (__any_sync(0xffffffffu, over)) {  // rare after the first keys of a row
#pragma unroll
            for (int b = 0; b < NQ; ++b) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float top = fmaxf(s[b][c], s[b][c + 2]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) - LOWER;
                    if (top > m[b][c]) {
                        const float down = m[b][c] == -INFINITY ? 0.0f : fast_exp2(m[b][c] - top);
                        m[b][c] = top;
                        l[b][c] *= down;
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            o[i][b][c] *= down;
                            o[i][b][c + 2] *= down;
                        }
                    }
                }
            }
        }
        uint32_t hi[NQ][2], lo[NQ][2];  // P^T as the right operand of the second product
#pragma unroll
        for (int b = 0; b < NQ; ++b) {
            const float base0 = m[b][0] == -INFINITY ? 0.0f : m[b][0], base1 = m[b][1] == -INFINITY ? 0.0f : m[b][1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float p0 = fast_exp2(s[b][2 * h] - base0), p1 = fast_exp2(s[b][2 * h + 1] - base1);
                l[b][0] += p0;
                l[b][1] += p1;
                const uint32_t x = pack2<T>(p0, p1);
                const float2 r = unpack2<T>(x);
                hi[b][h] = transpose8x8(x);
                lo[b][h] = transpose8x8(pack2<T>(p0 - r.x, p1 - r.y));
            }
        }
        const uint32_t vaddr = vs + ((lane & 7) + (lane >> 4) * 8) * PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint32_t v[4];
            ldsm4_trans(v, vaddr + i * 32);
#pragma unroll
            for (int b = 0; b < NQ; ++b) {
                mma16816<T>(o[i][b], v, hi[b][0], hi[b][1]);
                mma16816<T>(o[i][b], v, lo[b][0], lo[b][1]);
            }
        }
    }
    // This warp's maxima and sums; O as it is.
    __device__ __forceinline__ void finish(float *sm, float *sl) {
#pragma unroll
        for (int b = 0; b < NQ; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                l[b][c] += __shfl_xor_sync(0xffffffffu, l[b][c], 4);
                l[b][c] += __shfl_xor_sync(0xffffffffu, l[b][c], 8);
                l[b][c] += __shfl_xor_sync(0xffffffffu, l[b][c], 16);
                if (lr == 0) {
                    sm[b * 8 + lc + c] = m[b][c];
                    sl[b * 8 + lc + c] = l[b][c];
                }
            }
    }
    // Elements d0 .. d0 + dims - 1 of O, a row every `stride` floats.
    __device__ __forceinline__ void put(float *part, int stride, int d0, int dims, int rows) const {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            if (i * 16 < d0 || i * 16 >= d0 + dims) continue;
#pragma unroll
            for (int b = 0; b < NQ; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = b * 8 + lc + (x & 1);
                    if (r < rows) part[r * stride + i * 16 - d0 + lr + (x >> 1) * 8] = o[i][b][x];
                }
        }
    }
};

//   float32: CUDA cores, so that nothing is rounded below 32 bits.  Eight lanes share a key, four keys at a time; a lane owns CH
// groups of four neighbouring elements of the head, and each group of eight lanes has statistics of its own.
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 x;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
    return x;
}
template <int D, int R> struct CoreRows {
    static constexpr int ROWS = R, CH = D / 32, PITCH = 4 * D + 16;
    float4 q[R][CH], o[R][CH];
    float m[R], l[R];
    int lane, l8, sub;

    __device__ __forceinline__ explicit CoreRows(int lane_) : lane(lane_), l8(lane_ & 7), sub(lane_ >> 3) { clear(); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c) o[r][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    __device__ __forceinline__ void ask_queries(const PagedArgs &a, const float *qp, int rows) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const float *p = qp + r * a.sq_h + (c * 8 + l8) * 4;
                q[r][c] = r < rows ? make_float4(p[0], p[1], p[2], p[3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
    }
    __device__ __forceinline__ void step(const PagedArgs &a, uint32_t ks, uint32_t vs, int left, int skip) {
        float s[4][R];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float4 k[CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) k[c] = lds4(ks + (u * 4 + sub) * PITCH + (c * 8 + l8) * 16);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float x = 0.0f;
#pragma unroll
                for (int c = 0; c < CH; ++c) x = fmaf(q[r][c].w, k[c].w, fmaf(q[r][c].z, k[c].z, fmaf(q[r][c].y, k[c].y, fmaf(q[r][c].x, k[c].x, x))));
                s[u][r] = x;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float x = s[u][r];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                const int key = u * 4 + sub;
                s[u][r] = key < left && key >= skip ? x * a.scale : -INFINITY;
                top = fmaxf(top, s[u][r]);
            }
            if (top > m[r]) {
                const float down = m[r] == -INFINITY ? 0.0f : fast_exp2(m[r] - top);
                m[r] = top;
                l[r] *= down;
#pragma unroll
                for (int c = 0; c < CH; ++c) o[r][c] = make_float4(o[r][c].x * down, o[r][c].y * down, o[r][c].z * down, o[r][c].w * down);
            }
            const float base = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                s[u][r] = fast_exp2(s[u][r] - base);
                l[r] += s[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const float4 v = lds4(vs + (u * 4 + sub) * PITCH + (c * 8 + l8) * 16);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    o[r][c].x = fmaf(s[u][r], v.x, o[r][c].x);
                    o[r][c].y = fmaf(s[u][r], v.y, o[r][c].y);
                    o[r][c].z = fmaf(s[u][r], v.z, o[r][c].z);
                    o[r][c].w = fmaf(s[u][r], v.w, o[r][c].w);
                }
            }
    }
    __device__ __forceinline__ void finish(float *sm, float *sl) {  // joins the four groups of lanes
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float down = fast_exp2(m[r] - (top == -INFINITY ? 0.0f : top));
            auto both = [&](float x) {
                x *= down;
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                return x + __shfl_xor_sync(0xffffffffu, x, 16);
            };
            const float sum = both(l[r]);
#pragma unroll
            for (int c = 0; c < CH; ++c) o[r][c] = make_float4(both(o[r][c].x), both(o[r][c].y), both(o[r][c].z), both(o[r][c].w));
            if (lane == 0) {
                sm[r] = top;
                sl[r] = sum;
            }
        }
    }
    __device__ __forceinline__ void put(float *part, int stride, int d0, int dims, int rows) const {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int d = (c * 8 + l8) * 4 - d0;
            if (sub != 0 || d < 0 || d >= dims) continue;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < rows) *reinterpret_cast<float4 *>(part + r * stride + d) = o[r][c];
        }
    }
};

template <typename T, int D, int STAGES, int CTAS, typename Math, bool WHOLE> __global__ void __launch_bounds__(THREADS, CTAS) paged_ring_kernel(PagedArgs a) {
    using R = Ring<T, D, STAGES>;
    constexpr int NV = 16 / (int)sizeof(T), CHUNKS = D / NV;  // 16-byte chunks of a row
    constexpr int ROWS = Math::ROWS;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sm[WARPS][ROWS], sl[WARPS][ROWS];
    float *so = reinterpret_cast<float *>(smem + R::TOTAL);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t ring = smem_u32(smem) + warp * R::WARP;
    __shared__ Claims claims;
    __shared__ RunQueue<STAGES> queue[WARPS];
    __shared__ int before[THREADS];
    const bool more = (int)gridDim.x > a.long_runs;  // there are runs to claim
    if (threadIdx.x == 0 && more) {
        for (int i = 0; i < CLAIMS; ++i) sm100::mbar_init(&claims.arrived[i], 1);
        claims.gave_up = 0;
        sm100::fence_barrier_init();
    }
    grid_dependency_wait();
    const Line line = make_line(a, before);  // (its barriers order the initialisation above, too)
    if (threadIdx.x == 0 && more) claim(claims, 0);

    Cursor load, at;       // the tile that is loaded next, the tile that is worked on next
    int entered = 0, finished = 0, answers = 0;  // runs that either has entered; claims looked at
    bool queue_left = false;                     // the last run claimed had no tiles: others like it may wait
    auto keep = [&]() {    // the loading cursor has entered a run (or come to the end)
        if (lane == 0) queue[warp].at[entered % (STAGES + 2)] = load;
        ++entered;
        __syncwarp();
    };
    // Moves the loading cursor, at the end of its run, to the CTA's next.  The thread that learns of a run with tiles asks for
    // the next.
    auto next_run = [&]() {
        const int id = more ? claimed(claims, answers) : -1;
        ++answers;
        load.run = -1;
        if (id >= 0) {
            load.start(a, line, before, id);
            queue_left = load.left <= 0;
            if (queue_left) {
                if (line.any_empty && id < a.long_runs) write_empty_rows<T>(a, id);
                load.run = -1;
            } else if (threadIdx.x == 0) {
                claim(claims, answers);
            }
        }
        keep();
    };
    auto follow = [&]() {  // the finishing cursor enters the next run that the loading one has entered: what the run owes besides its tiles
        at = queue[warp].at[finished % (STAGES + 2)];
        ++finished;
        if (at.run < 0) return;
        if (threadIdx.x == 0 && a.headers) a.headers[at.run].y = 0;
        if (line.any_empty && at.run < a.long_runs) write_empty_rows<T>(a, at.run);
    };
    load.start(a, line, before, blockIdx.x);
    if (load.left > 0) {
        keep();
        follow();
    } else {
        if (line.any_empty && (int)blockIdx.x < a.long_runs) write_empty_rows<T>(a, blockIdx.x);
        next_run();
        follow();
    }
    // Page number that the next copies need, read one tile ahead.  WHOLE: pages are whole multiples of 16 keys and so is the
    // first key, so a warp's 16 keys lie in one page and their rows at one distance; otherwise every lane looks up its key.
    int page = 0;
    auto read_page = [&]() {
        if (load.run < 0) return;
        const int j = load.t * TILE + warp * 16 + (WHOLE ? 0 : lane & 15);
        if (j < load.keys) page = a.block_table[load.seq * a.s_table + a.page_size.div((uint32_t)(load.first + j))];
    };
    auto issue = [&](int stage, bool ahead) {  // the copies of one tile's 16 keys and values, then one step on
        if (load.run >= 0) {
            const int j0 = load.t * TILE + warp * 16, n = load.keys - j0;  // keys of the 16 that exist
            const int kv_head = a.row_groups == 1 ? load.unit : load.unit / a.row_groups;
            const T *kb = reinterpret_cast<const T *>(a.k) + kv_head * a.sk_h, *vb = reinterpret_cast<const T *>(a.v) + kv_head * a.sv_h;
            const uint32_t dst = ring + stage * 2 * R::HALF;
            const bool ok = page >= 0 && page < a.num_pages;
            const uint32_t pos = (uint32_t)(load.first + j0 + (WHOLE ? 0 : lane & 15));
            const int in_page = (int)(pos - a.page_size.div(pos) * a.page_size.d);
            if (n > 0 && !ok && (WHOLE ? lane == 0 : (lane & 15) < n)) atomicExch(&g_bad_index, 1u);
            const int skip = WHOLE && load.t == 0 && warp == 0 ? load.skip : 0;
            if (WHOLE && n >= 16 && skip == 0 && ok) {  // all of a page's 16 keys: no tests
                const T *k = kb + page * a.sk_p + in_page * a.sk_t, *v = vb + page * a.sv_p + in_page * a.sv_t;
                if constexpr (32 % CHUNKS == 0) {  // the same place of the row in every step: one pointer each, moved on
                    constexpr int ROWS_A_STEP = 32 / CHUNKS;
                    const T *kp = k + (lane / CHUNKS) * a.sk_t + lane % CHUNKS * NV, *vp = v + (lane / CHUNKS) * a.sv_t + lane % CHUNKS * NV;
                    const uint32_t to = dst + lane / CHUNKS * R::PITCH + lane % CHUNKS * 16;
#pragma unroll
                    for (int i = 0; i < CHUNKS / 2; ++i) {
                        cp_async16(to + i * ROWS_A_STEP * R::PITCH, kp);
                        cp_async16(to + i * ROWS_A_STEP * R::PITCH + R::HALF, vp);
                        kp += ROWS_A_STEP * a.sk_t;
                        vp += ROWS_A_STEP * a.sv_t;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < CHUNKS / 2; ++i) {
                        const int idx = i * 32 + lane, r = idx / CHUNKS, c = idx - r * CHUNKS;
                        cp_async16(dst + r * R::PITCH + c * 16, k + (r * a.sk_t + c * NV));
                        cp_async16(dst + R::HALF + r * R::PITCH + c * 16, v + (r * a.sv_t + c * NV));
                    }
                }
            } else if (n > 0) {
                const T *row = nullptr;  // of key lane & 15; lanes 0-15: the key rows, 16-31: the value rows
                if (ok && (lane & 15) < n && (lane & 15) >= skip) {
                    const int64_t at = in_page + (WHOLE ? lane & 15 : 0);
                    row = lane < 16 ? kb + page * a.sk_p + at * a.sk_t : vb + page * a.sv_p + at * a.sv_t;
                }
#pragma unroll
                for (int i = 0; i < CHUNKS / 2; ++i) {
                    const int idx = i * 32 + lane, r = idx / CHUNKS, c = idx - r * CHUNKS;
                    const T *k = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), r));
                    const T *v = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), 16 + r));
                    cp_async16(dst + r * R::PITCH + c * 16, k ? k + c * NV : reinterpret_cast<const T *>(a.k), k ? 16 : 0);
                    cp_async16(dst + R::HALF + r * R::PITCH + c * 16, v ? v + c * NV : reinterpret_cast<const T *>(a.v), v ? 16 : 0);
                }
            }
            load.next(a);
            if (load.left <= 0) next_run();
            if (ahead) read_page();
        }
        cp_async_commit();
    };
    Math math(lane);
    int64_t seq = 0;
    int first_head = 0, rows = 0, t0 = 0, stage = 0, discarded = 0;
    auto begin_piece = [&]() {  // the finishing cursor stands at a piece's first tile: asks for its queries
        seq = at.seq;
        t0 = at.t;
        const int kv_head = a.row_groups == 1 ? at.unit : at.unit / a.row_groups, rg = at.unit - kv_head * a.row_groups;
        rows = a.group - rg * ROWS < ROWS ? a.group - rg * ROWS : ROWS;
        first_head = kv_head * a.group + rg * ROWS;
        const T *qp = reinterpret_cast<const T *>(a.q) + seq * a.sq_s + (int64_t)first_head * a.sq_h;
        math.ask_queries(a, qp, rows);
    };
    if (at.run >= 0) begin_piece();
    for (bool prime = true;;) {
        if (prime) {  // fill the ring
            prime = false;
            // One tile after the other would wait for one page number after the other: lane s asks for that of the s-th tile from
            // here, as far as they are the same run's and sequence's (WHOLE: a warp needs one number a tile).
            int early = 0, known = 0;
            if (WHOLE && load.run >= 0) {
                const int t = load.t + lane, ahead = t / load.tiles, j = (t - ahead * load.tiles) * TILE + warp * 16;
                const bool same = lane < STAGES && (a.by_rows ? ahead < load.left : lane < load.left) && load.unit + ahead < a.units;
                if (same && j < load.keys) early = a.block_table[load.seq * a.s_table + a.page_size.div((uint32_t)(load.first + j))];
                known = __popc(__ballot_sync(0xffffffffu, same));
            }
#pragma unroll 1
            for (int s = 0; s < STAGES; ++s) {
                const int number = __shfl_sync(0xffffffffu, early, s);
                if (s < known) page = number;
                else if (s == known) read_page();
                issue(stage + s < STAGES ? stage + s : stage + s - STAGES, s >= known);
            }
            if (known >= STAGES) read_page();
        }
        if (at.run < 0) {
            // Runs without tiles are at the queue's end and wait for nothing; taken off it, a bounded number by each CTA, they
            // cost a claim instead of the start of a block.  All cursors stand here, so they go on together.
            if (!queue_left || discarded++ == 32) break;
            queue_left = false;
            __syncthreads();
            if (threadIdx.x == 0) claim(claims, answers);
            next_run();
            follow();
            prime = at.run >= 0;
            if (prime) begin_piece();
            continue;
        }
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const int left = at.keys - (at.t * TILE + warp * 16);  // keys of this warp's 16 that exist
        if (left > 0) {
            const uint32_t ks = ring + stage * 2 * R::HALF, vs = ks + R::HALF;
            math.step(a, ks, vs, left, WHOLE && at.t == 0 && warp == 0 ? at.skip : 0);
        }
        __syncwarp();
        issue(stage, true);
        stage = stage + 1 == STAGES ? 0 : stage + 1;

        const int t1 = at.t + 1, tiles = at.tiles, run = at.run;
        const int done = at.end - at.left + 1;  // tiles of the line up to here
        at.next(a);
        if (t1 < tiles && at.left > 0) continue;
        // the piece ends here: hand this warp's part over, join the warps' parts, write; the next piece's queries are under way
        // meanwhile
        math.finish(sm[warp], sl[warp]);
        float *slot = nullptr;
        if (t0 > 0) {
            slot = slot_of(a, run, 0, ROWS);
        } else if (t1 < tiles) {
            slot = slot_of(a, run, 1, ROWS);
            if (threadIdx.x == 0) a.headers[run] = make_int4((int)seq, rows | (first_head << 8), line.run_of(a, done - t1 + tiles - 1), 0);
        }
        const int64_t old_seq = seq;
        const int old_head = first_head, old_rows = rows, stride = part_stride(a.merge_dims);
        if (at.left <= 0) follow();
        if (at.run >= 0) begin_piece();
        for (int d0 = 0; d0 < D; d0 += a.merge_dims) {
            math.put(so + warp * a.merge_rows * stride, stride, d0, a.merge_dims, old_rows);
            __syncthreads();
            write_piece<T, ROWS>(a, so, a.merge_rows * stride, stride, sm, sl, old_rows, old_seq, old_head, slot, d0, a.merge_dims);
            __syncthreads();
        }
        math.clear();
    }
    cp_async_wait<0>();
}

// Shared memory of a CTA so that CTAS of them fit an SM (228 KB, 1 KB of it taken per CTA, and a little static).
constexpr int budget(int ctas, int rows) { return (228 * 1024) / ctas - 1024 - (2304 + 32 * rows); }

template <typename T, int D, int STAGES, int CTAS, typename Math> int launch(PagedArgs a, int grid, cudaStream_t st) {
    using R = Ring<T, D, STAGES>;
    constexpr int ROWS = Math::ROWS;
    static_assert(R::TOTAL + WARPS * ROWS * part_stride(D / 2) * 4 <= budget(CTAS, ROWS), "partial results of half a head must fit");
    auto kern = a.whole ? paged_ring_kernel<T, D, STAGES, CTAS, Math, true> : paged_ring_kernel<T, D, STAGES, CTAS, Math, false>;
    a.merge_rows = a.group < ROWS ? a.group : ROWS;
    a.merge_dims = R::TOTAL + WARPS * a.merge_rows * part_stride(D) * 4 <= budget(CTAS, ROWS) ? D : D / 2;
    const int smem = R::TOTAL + WARPS * a.merge_rows * part_stride(a.merge_dims) * 4;
    static OncePerDevice opted[2];
    const int rc = opted[a.whole].opt_in(kern, R::TOTAL + WARPS * ROWS * part_stride(D) * 4, "enc_paged_attention");
    if (rc != ENC_OK) return rc;
    launch_overlapped(kern, dim3(grid), dim3(THREADS), smem, st, a);
    return check_launch("enc_paged_attention");
}

template <typename T, int D, int STAGES1, int STAGES2, int CTAS> int launch_tensor(const PagedArgs &a, int grid, cudaStream_t st) {
    return ring_rows(ENC_F16, a.group) == 8 ? launch<T, D, STAGES1, CTAS, TensorRows<T, D, 1>>(a, grid, st)
                                            : launch<T, D, STAGES2, CTAS, TensorRows<T, D, 2>>(a, grid, st);
}
template <typename T> int launch_tensor_dim(const PagedArgs &a, int grid, cudaStream_t st) {
    switch (a.head_dim) {
        case 32: return launch_tensor<T, 32, 4, 4, 3>(a, grid, st);
        case 64: return launch_tensor<T, 64, 3, 3, 3>(a, grid, st);
        case 96: return launch_tensor<T, 96, 3, 3, 2>(a, grid, st);
        case 128: return launch_tensor<T, 128, 3, 2, 2>(a, grid, st);
        default: return launch_tensor<T, 256, 2, 2, 1>(a, grid, st);
    }
}
template <int D, int STAGES, int CTAS> int launch_cores(const PagedArgs &a, int grid, cudaStream_t st) {
    return ring_rows(ENC_F32, a.group) == 1 ? launch<float, D, STAGES, CTAS, CoreRows<D, 1>>(a, grid, st) : launch<float, D, STAGES, CTAS, CoreRows<D, 4>>(a, grid, st);
}

}  // namespace

int ring_ctas_per_sm(int dtype, int64_t d) {
    if (dtype == ENC_F32) return d == 32 || d == 64 ? 2 : d == 128 ? 1 : 0;
    switch (d) {
        case 32: case 64: return 3;
        case 96: case 128: return 2;
        case 256: return 1;
    }
    return 0;
}

int launch_ring(const PagedArgs &args, int dtype, int grid, cudaStream_t st) {
    PagedArgs a = args;
    a.q_pairs = reinterpret_cast<uintptr_t>(a.q) % 4 == 0 && a.sq_s % 2 == 0 && a.sq_h % 2 == 0;
    if (ring_ctas_per_sm(dtype, a.head_dim) == 0) return fail(ENC_ERR_UNSUPPORTED, "enc_paged_attention: no ring kernel for head_dim %d", a.head_dim);
    if (dtype == ENC_F16) return launch_tensor_dim<__half>(a, grid, st);
    if (dtype == ENC_BF16) return launch_tensor_dim<__nv_bfloat16>(a, grid, st);
    return a.head_dim == 32 ? launch_cores<32, 4, 2>(a, grid, st) : a.head_dim == 64 ? launch_cores<64, 3, 2>(a, grid, st) : launch_cores<128, 2, 1>(a, grid, st);
}

}  // namespace paged

unsigned int take_bad_index_paged_ring() { return take_bad_index_word(); }

}  // namespace enc

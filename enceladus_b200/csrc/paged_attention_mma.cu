// Attention of one new token per sequence over a paged key-value cache: the tensor-core kernel for 16-bit types.
// Mathematics, bound and split are in paged_attention.cuh.
//
// The up to 16 query heads that share a kv head are the rows of an m16n8k16 product: S = Q K^T over 16 keys per warp and step,
// O += P V with P taken from S's registers.  The unit is bound by HBM, so the tensor pipe's rate does not matter (at 6.5 TB/s
// an SM has about 350 cycles for 16 keys of 128 elements, and spends 48 of these instructions on them); what the matrix
// instruction buys is that the work per key no longer grows with the number of query heads.  tcgen05 would need 128 query rows
// to fill its smallest tile, and its operands would still come through shared memory.
//
// Each warp has a ring of its own in shared memory and walks its keys without CTA barriers: 16 keys and 16 values per stage,
// 16-byte asynchronous copies, rows padded by 16 bytes so that ldmatrix meets no bank twice.  The ring runs on across the
// pieces of a run: the next row's keys are on their way while a finished one is joined and written.
//
// P is fed as the sum of two 16-bit numbers, P = hi + lo, in two products: the weights keep 16 or more bits instead of 8 or 11
// and the output is as exact as a float32 product rounded once.  In fp16 the maximum is kept 14 powers of two lower, so that
// weights down to 2^-28 of the largest are still normal numbers.
#include <type_traits>

#include "paged_attention.cuh"

namespace enc {
namespace paged {
namespace {

template <int D, int STAGES> struct Ring {
    static constexpr int PITCH = 2 * D + 16;             // bytes of a key or value row
    static constexpr int HALF = 16 * PITCH;              // 16 keys (or values)
    static constexpr int WARP = STAGES * 2 * HALF;
    static constexpr int TOTAL = WARPS * WARP;
    static constexpr int O_STRIDE = D + 8;               // floats of a row of partial results
};

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

// A place in the CTA's run: a tile of one unit (kv head and row group) of one sequence.
struct Cursor {
    int64_t left, seq;  // tiles left in the run
    int unit, t, tiles, keys, first, skip;

    __device__ __forceinline__ void start(const PagedArgs &a, const Run &run) {
        left = run.end - run.begin;
        if (left <= 0) return;
        seq = run.seq;
        keys = keys_of(a, seq, first, skip);
        tiles = (int)tiles_of(keys);
        unit = (int)(run.at / tiles);
        t = (int)(run.at - (int64_t)unit * tiles);
    }
    __device__ __forceinline__ void next(const PagedArgs &a) {
        --left;
        if (++t < tiles) return;
        t = 0;
        if (++unit < a.units || left <= 0) return;
        unit = 0;
        do {  // (left > 0: a sequence with keys follows)
            ++seq;
            keys = keys_of(a, seq, first, skip);
        } while (keys == 0);
        tiles = (int)tiles_of(keys);
    }
};

template <typename T, int D, int STAGES, int CTAS, bool WHOLE> __global__ void __launch_bounds__(THREADS, CTAS) paged_mma_kernel(PagedArgs a) {
    using R = Ring<D, STAGES>;
    constexpr int KS = D / 16, CHUNKS = D / 8;  // steps of the first product; 16-byte chunks of a row
    constexpr float LOWER = std::is_same<T, __half>::value ? 14.0f : 0.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sm[WARPS][MMA_ROWS], sl[WARPS][MMA_ROWS];
    float *so = reinterpret_cast<float *>(smem + R::TOTAL);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t ring = smem_addr(smem) + warp * R::WARP;
    const int qr = lane >> 2, qc = (lane & 3) * 2;  // this thread's row (and row + 8) and first column in accumulators
    grid_dependency_wait();
    const Run run = find_run(a);
    if (threadIdx.x == 0 && a.headers) a.headers[blockIdx.x].y = 0;

    Cursor load, at;
    load.start(a, run);
    at = load;
    // Page number that the next copies need, read one tile ahead.  WHOLE: pages are whole multiples of 16 keys and so is the
    // first key, so a warp's 16 keys lie in one page and their rows at one distance; otherwise every lane looks up its key.
    int page = 0;
    auto read_page = [&]() {
        if (load.left <= 0) return;
        const int j = load.t * TILE + warp * 16 + (WHOLE ? 0 : lane & 15);
        if (j < load.keys) page = a.block_table[load.seq * a.s_table + a.page_size.div((uint32_t)(load.first + j))];
    };
    auto issue = [&](int stage) {  // the copies of one tile's 16 keys and values, then one step on
        if (load.left > 0) {
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
                    const T *kp = k + (lane / CHUNKS) * a.sk_t + lane % CHUNKS * 8, *vp = v + (lane / CHUNKS) * a.sv_t + lane % CHUNKS * 8;
                    const uint32_t to = dst + lane / CHUNKS * R::PITCH + lane % CHUNKS * 16;
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        cp_async16(to + i * ROWS_A_STEP * R::PITCH, kp);
                        cp_async16(to + i * ROWS_A_STEP * R::PITCH + R::HALF, vp);
                        kp += ROWS_A_STEP * a.sk_t;
                        vp += ROWS_A_STEP * a.sv_t;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        const int idx = i * 32 + lane, r = idx / CHUNKS, c = idx - r * CHUNKS;
                        cp_async16(dst + r * R::PITCH + c * 16, k + (r * a.sk_t + c * 8));
                        cp_async16(dst + R::HALF + r * R::PITCH + c * 16, v + (r * a.sv_t + c * 8));
                    }
                }
            } else if (n > 0) {
                const T *row = nullptr;  // of key lane & 15; lanes 0-15: the key rows, 16-31: the value rows
                if (ok && (lane & 15) < n && (lane & 15) >= skip) {
                    const int64_t at = in_page + (WHOLE ? lane & 15 : 0);
                    row = lane < 16 ? kb + page * a.sk_p + at * a.sk_t : vb + page * a.sv_p + at * a.sv_t;
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const int idx = i * 32 + lane, r = idx / CHUNKS, c = idx - r * CHUNKS;
                    const T *k = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), r));
                    const T *v = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), 16 + r));
                    cp_async16(dst + r * R::PITCH + c * 16, k ? k + c * 8 : reinterpret_cast<const T *>(a.k), k ? 16 : 0);
                    cp_async16(dst + R::HALF + r * R::PITCH + c * 16, v ? v + c * 8 : reinterpret_cast<const T *>(a.v), v ? 16 : 0);
                }
            }
            load.next(a);
            read_page();
        }
        cp_async_commit();
    };
    read_page();
#pragma unroll
    for (int s = 0; s < STAGES; ++s) issue(s);

    uint32_t q[KS][4];
    float o[D / 8][4], m[2], l[2];
    bool fresh = true;
    int64_t seq = 0;
    int first_head = 0, rows = 0, t0 = 0, stage = 0;
    while (at.left > 0) {
        if (fresh) {  // a new piece: its queries, and nothing seen yet
            fresh = false;
            seq = at.seq;
            t0 = at.t;
            const int kv_head = a.row_groups == 1 ? at.unit : at.unit / a.row_groups, rg = at.unit - kv_head * a.row_groups;
            rows = a.group - rg * MMA_ROWS < MMA_ROWS ? a.group - rg * MMA_ROWS : MMA_ROWS;
            first_head = kv_head * a.group + rg * MMA_ROWS;
            const T *qp = reinterpret_cast<const T *>(a.q) + seq * a.sq_s + (int64_t)first_head * a.sq_h;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = qr + (x & 1) * 8, d = i * 16 + (x >> 1) * 8 + qc;
                    uint32_t v = 0;
                    if (r < rows) {
                        const T *p = qp + r * a.sq_h + d;
                        v = (uint32_t)*reinterpret_cast<const uint16_t *>(p) | (uint32_t)*reinterpret_cast<const uint16_t *>(p + 1) << 16;
                    }
                    q[i][x] = v;
                }
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
        }
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const int left = at.keys - (at.t * TILE + warp * 16);  // keys of this warp's 16 that exist
        if (left > 0) {
            const uint32_t ks = ring + stage * 2 * R::HALF, vs = ks + R::HALF;
            float s[2][4] = {};
            const uint32_t kaddr = ks + ((lane & 7) + (lane >> 4) * 8) * R::PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t b[4];
                ldsm4(b, kaddr + i * 32);
                mma16816<T>(s[0], q[i], b[0], b[1]);
                mma16816<T>(s[1], q[i], b[2], b[3]);
            }
            uint32_t hi[4], lo[4];  // P as the left operand of the second product
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[0][x] *= a.scale;
                s[1][x] *= a.scale;
            }
            if (left < 16) {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if ((x >> 2) * 8 + qc + (x & 1) >= left) s[x >> 2][x & 3] = -INFINITY;
            }
            if (at.skip > 0 && at.t == 0 && warp == 0) {  // keys in front of the window
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if ((x >> 2) * 8 + qc + (x & 1) < at.skip) s[x >> 2][x & 3] = -INFINITY;
            }
            bool grew = false;
            float up[2] = {1.0f, 1.0f}, base[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && rows <= 8) continue;  // the lower eight rows hold no queries
                float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) - LOWER;
                if (top > m[h]) {
                    up[h] = m[h] == -INFINITY ? 0.0f : fast_exp2(m[h] - top);
                    m[h] = top;
                    grew = true;
                }
                base[h] = m[h] == -INFINITY ? 0.0f : m[h];
            }
            if (__any_sync(0xffffffffu, grew)) {  // rare after the first keys of a row
#pragma unroll
                for (int h = 0; h < 2; ++h) l[h] *= up[h];
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[i][x] *= up[x >> 1];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && rows <= 8) {
                    hi[1] = hi[3] = lo[1] = lo[3] = 0;
                    continue;
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p0 = fast_exp2(s[n][2 * h] - base[h]), p1 = fast_exp2(s[n][2 * h + 1] - base[h]);
                    l[h] += p0 + p1;
                    const uint32_t x = pack2<T>(p0, p1);
                    const float2 r = unpack2<T>(x);
                    hi[2 * n + h] = x;
                    lo[2 * n + h] = pack2<T>(p0 - r.x, p1 - r.y);
                }
            }
            const uint32_t vaddr = vs + (lane & 15) * R::PITCH + (lane >> 4) * 16;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t b[4];
                ldsm4_trans(b, vaddr + i * 32);
                mma16816<T>(o[2 * i], hi, b[0], b[1]);
                mma16816<T>(o[2 * i + 1], hi, b[2], b[3]);
                mma16816<T>(o[2 * i], lo, b[0], b[1]);
                mma16816<T>(o[2 * i + 1], lo, b[2], b[3]);
            }
        }
        __syncwarp();
        issue(stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;

        const int t1 = at.t + 1, tiles = at.tiles;
        const int64_t done = run.end - at.left + 1;  // tiles of the line up to here
        at.next(a);
        if (t1 < tiles && at.left > 0) continue;
        // the piece ends here: hand this warp's part over, join the warps' parts, write
        fresh = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int r = qr + 8 * h;
            if (r < rows) {
                if ((lane & 3) == 0) {
                    sm[warp][r] = m[h];
                    sl[warp][r] = l[h];
                }
                float *p = so + (warp * a.merge_rows + r) * R::O_STRIDE + qc;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2 *>(p + i * 8) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
            }
        }
        float *slot = nullptr;
        if (t0 > 0) {
            slot = slot_of(a, blockIdx.x, 0, MMA_ROWS);
        } else if (t1 < tiles) {
            slot = slot_of(a, blockIdx.x, 1, MMA_ROWS);
            if (threadIdx.x == 0) a.headers[blockIdx.x] = make_int4((int)seq, rows | (first_head << 8), (int)((done - t1 + tiles - 1) / run.run), 0);
        }
        __syncthreads();
        write_piece<T, MMA_ROWS>(a, so, a.merge_rows * R::O_STRIDE, R::O_STRIDE, sm, sl, rows, seq, first_head, slot);
        __syncthreads();
    }
    cp_async_wait<0>();
    write_empty_rows<T>(a);
}

template <typename T, int D, int STAGES, int CTAS> int launch(PagedArgs a, int grid, cudaStream_t st) {
    using R = Ring<D, STAGES>;
    auto kern = a.whole ? paged_mma_kernel<T, D, STAGES, CTAS, true> : paged_mma_kernel<T, D, STAGES, CTAS, false>;
    a.merge_rows = a.group < MMA_ROWS ? a.group : MMA_ROWS;
    const int smem = R::TOTAL + WARPS * a.merge_rows * R::O_STRIDE * 4;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(ENC_ERR_LAUNCH, "enc_paged_attention: cannot opt in to %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    launch_overlapped(kern, dim3(grid), dim3(THREADS), smem, st, a);
    return check_launch("enc_paged_attention");
}

template <typename T> int launch_dim(const PagedArgs &a, int grid, cudaStream_t st) {
    switch (a.head_dim) {
        case 32: return launch<T, 32, 4, 2>(a, grid, st);
        case 64: return launch<T, 64, 4, 2>(a, grid, st);
        case 80: return launch<T, 80, 3, 2>(a, grid, st);
        case 96: return launch<T, 96, 2, 2>(a, grid, st);
        case 128: return launch<T, 128, 2, 2>(a, grid, st);
        case 256: return launch<T, 256, 2, 1>(a, grid, st);
    }
    return fail(ENC_ERR_UNSUPPORTED, "enc_paged_attention: no tensor-core kernel for head_dim %d", a.head_dim);
}

}  // namespace

int mma_ctas_per_sm(int64_t d) {
    switch (d) {
        case 32: case 64: case 80: case 96: case 128: return 2;
        case 256: return 1;
    }
    return 0;
}

int launch_mma(const PagedArgs &a, int dtype, int grid, cudaStream_t st) {
    return dtype == ENC_F16 ? launch_dim<__half>(a, grid, st) : launch_dim<__nv_bfloat16>(a, grid, st);
}

}  // namespace paged

unsigned int take_bad_index_paged_mma() { return take_bad_index_word(); }

}  // namespace enc

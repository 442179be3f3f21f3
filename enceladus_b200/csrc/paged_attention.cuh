// Attention of one new token per sequence over a paged key-value cache, split over the cache's length and joined.
//
// Mathematics: for a query row, s_j = q . k_j * sm_scale * log2(e); one pass over the keys keeps the running maximum m, the
// sum l = sum_j 2^(s_j - m) and O = sum_j 2^(s_j - m) v_j, all float32.  Two pieces (m1, l1, O1), (m2, l2, O2) of a row join
// to m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m) and the same for O, in any split.  o = O / l,
// lse = (m + log2 l) ln 2.  A piece whose scores are all -inf has m = -inf and counts with weight zero.
//
// What bounds it: each key and value is read once and used by the query heads that share it, a handful of operations per
// byte, so the bound is HBM bandwidth; with few or short sequences, latency.
//
// Split: the work is a line of 64-key tiles (sequence by sequence, kv head by kv head), dealt out in equal contiguous
// runs over a grid that fills the GPU once.  Every CTA finds its run from seq_lens by a scan over the batch, so ragged
// lengths, one long sequence and many short ones all load every SM alike, and nothing about the lengths has to reach
// the host.  A row that ends inside a run is finished there; the up to two pieces of a run that belong to rows cut by
// its ends go to a workspace and a second, overlapped launch joins them in order (no atomics: the result does not depend
// on timing).
#pragma once

#include "paged.cuh"

namespace enc {
namespace paged {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int TILE = 64;          // keys of a tile
constexpr int MAX_HEAD_DIM = 256;

struct PagedArgs {
    const void *q, *k, *v;
    void *o;
    float *lse;
    const int32_t *block_table, *seq_lens;
    int4 *headers;   // per CTA: the row group that its last piece begins {first query row, rows, last CTA of it, -}
    float *slots;    // per CTA two pieces of `rows` x (head_dim + 2) floats: O, m, l
    int64_t sq_s, sq_h, so_s, so_h, sk_p, sk_h, sk_t, sv_p, sv_h, sv_t, s_table;
    int64_t num_seqs, num_pages, capacity, window;
    int q_heads, head_dim, group, row_groups;  // query rows per kv head; row groups (of the kernel's row count) per kv head
    int units;                                 // row groups per sequence: kv_heads * row_groups
    bool whole;                                // pages are whole multiples of 16 keys
    int min_run;                               // tiles a run has at least
    bool q_pairs;                              // query elements can be read two at a time
    int merge_rows, merge_dims;                // rows and elements of a warp's part that shared memory holds at a time
    float scale;                               // sm_scale * log2(e)
    FastDiv page_size;
};

// ---- schedule ------------------------------------------------------------------------------------
// The keys that sequence b's row reads: `first` is the first one's position, the result how many.  Where pages are whole
// multiples of 16 keys, `first` is rounded down to 16 and the `skip` (< 16) keys in front of the window are read but
// not used.
static __device__ __forceinline__ int keys_of(const PagedArgs &a, int64_t b, int &first, int &skip) {
    int n = a.seq_lens[b];
    if (n < 0 || n > a.capacity) {
        atomicExch(&g_bad_index, 1u);
        n = n < 0 ? 0 : (int)a.capacity;
    }
    const int begin = a.window > 0 && n > a.window ? n - (int)a.window : 0;
    first = a.whole ? begin & ~15 : begin;
    skip = begin - first;
    return n - first;
}
static __device__ __forceinline__ int64_t tiles_of(int keys) { return (keys + TILE - 1) / TILE; }

struct Run {
    int64_t seq, at;      // first sequence, first tile inside the sequence's units
    int64_t begin, end;   // tiles on the line
    int64_t run;          // tiles of a full run
};

// Every thread of the CTA returns the CTA's run of tiles.  The sequences are dealt to the threads in contiguous pieces;
// the thread whose piece holds the run's first tile finds the sequence.
static __device__ __forceinline__ Run find_run(const PagedArgs &a) {
    __shared__ int64_t warp_total[WARPS], found[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t per = (a.num_seqs + THREADS - 1) / THREADS;
    const int64_t b0 = threadIdx.x * per, b1 = b0 + per < a.num_seqs ? b0 + per : a.num_seqs;
    int64_t mine = 0;
    int first, skip;
    for (int64_t b = b0; b < b1; ++b) mine += tiles_of(keys_of(a, b, first, skip));
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) warp_total[warp] = upto;
    __syncthreads();
    int64_t total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += warp_total[w];
        total += warp_total[w];
    }
    total *= a.units;
    Run r;
    r.run = (total + gridDim.x - 1) / gridDim.x;
    if (r.run < a.min_run) r.run = a.min_run;
    r.begin = blockIdx.x * r.run;
    r.end = r.begin + r.run < total ? r.begin + r.run : total;
    r.seq = r.at = 0;
    if (r.begin >= r.end) return r;  // (the same for all threads: begin and end depend on the block alone)
    if (before * a.units <= r.begin && r.begin < (before + mine) * a.units) {
        int64_t at = r.begin - before * a.units;
        for (int64_t b = b0; b < b1; ++b) {
            const int64_t t = tiles_of(keys_of(a, b, first, skip)) * a.units;
            if (at < t) {
                found[0] = b;
                found[1] = at;
                break;
            }
            at -= t;
        }
    }
    __syncthreads();
    r.seq = found[0];
    r.at = found[1];
    return r;
}

static __device__ __forceinline__ float *slot_of(const PagedArgs &a, int64_t cta, int which, int rows) {
    return a.slots + (2 * cta + which) * rows * (int64_t)(a.head_dim + 2);
}

// A piece's rows, one partial result per warp in shared memory (O unnormalised, rows `stride` apart, m and l),
// joined and written (elements d0 .. d0 + dims - 1 of the head, `so` starting at d0): to the output when the piece is the whole row, to `slot` otherwise.
template <typename T, int ROWS>
static __device__ __forceinline__ void write_piece(const PagedArgs &a, const float *so, int warp_stride, int stride, const float (*sm)[ROWS], const float (*sl)[ROWS],
                                            int rows, int64_t seq, int first_head, float *slot, int d0, int dims) {
    T *o = reinterpret_cast<T *>(a.o) + seq * a.so_s;
    for (int i = threadIdx.x; i < rows * dims; i += THREADS) {
        const int r = i / dims, e = i - r * dims, d = d0 + e;
        float m = sm[0][r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) m = fmaxf(m, sm[w][r]);
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float c = fast_exp2(sm[w][r] - base);
            l = fmaf(sl[w][r], c, l);
            x = fmaf(so[w * warp_stride + r * stride + e], c, x);
        }
        if (slot) {
            slot[r * (a.head_dim + 2) + d] = x;
            if (d == 0) {
                slot[r * (a.head_dim + 2) + a.head_dim] = m;
                slot[r * (a.head_dim + 2) + a.head_dim + 1] = l;
            }
        } else {
            o[(first_head + r) * a.so_h + d] = from_f32<T>(l == 0.0f ? 0.0f : __fdiv_rn(x, l));
            if (d == 0 && a.lse) a.lse[seq * a.q_heads + first_head + r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
        }
    }
}

// The rows of sequences without keys, dealt over the grid: zero, lse -inf.
template <typename T> __device__ __forceinline__ void write_empty_rows(const PagedArgs &a) {
    T *o = reinterpret_cast<T *>(a.o);
    for (int64_t b = blockIdx.x; b < a.num_seqs; b += gridDim.x) {  // rows without keys
        int first, skip;
        if (keys_of(a, b, first, skip) > 0) continue;
        for (int i = threadIdx.x; i < a.q_heads * a.head_dim; i += THREADS) {
            const int h = i / a.head_dim, d = i - h * a.head_dim;
            o[b * a.so_s + h * a.so_h + d] = from_f32<T>(0.0f);
            if (d == 0 && a.lse) a.lse[b * a.q_heads + h] = -INFINITY;
        }
    }
}

// Walks over the CTA's run: process(seq, kv head, first query head, rows, first key, keys to skip, keys, tile range, slot or NULL) per
// piece.  Also writes the header that the join reads, and the rows of sequences without keys.
template <typename T, int ROWS, typename F> __device__ __forceinline__ void walk_run(const PagedArgs &a, F process) {
    const Run run = find_run(a);
    if (threadIdx.x == 0 && a.headers) a.headers[blockIdx.x].y = 0;
    int64_t seq = run.seq, at = run.at;
    for (int64_t pos = run.begin; pos < run.end;) {
        int first, skip;
        const int keys = keys_of(a, seq, first, skip);
        const int64_t tiles = tiles_of(keys);
        if (at >= tiles * a.units) {
            at -= tiles * a.units;  // (zero: a sequence's tiles are walked to their end)
            ++seq;
            continue;
        }
        const int unit = (int)(at / tiles), t0 = (int)(at - unit * tiles);
        const int t1 = tiles - t0 < run.end - pos ? (int)tiles : t0 + (int)(run.end - pos);
        const int kv_head = unit / a.row_groups, rg = unit - kv_head * a.row_groups;
        const int rows = a.group - rg * ROWS < ROWS ? a.group - rg * ROWS : ROWS;
        const int first_head = kv_head * a.group + rg * ROWS;
        float *slot = nullptr;
        if (t0 > 0) {
            slot = slot_of(a, blockIdx.x, 0, ROWS);
        } else if (t1 < tiles) {
            slot = slot_of(a, blockIdx.x, 1, ROWS);
            if (threadIdx.x == 0) a.headers[blockIdx.x] = make_int4((int)seq, rows | (first_head << 8), (int)((pos + tiles - 1) / run.run), 0);
        }
        process(seq, kv_head, first_head, rows, first, skip, keys, t0, t1, slot);
        pos += t1 - t0;
        at += t1 - t0;
    }
    write_empty_rows<T>(a);
}

// Where key `pos` of sequence seq lives: its page and its row in it; false (and the error word) if the page is out of range.
static __device__ __forceinline__ bool locate(const PagedArgs &a, int64_t seq, int pos, int64_t &page, int &row) {
    const uint32_t pi = a.page_size.div((uint32_t)pos);
    row = pos - (int)(pi * a.page_size.d);
    page = a.block_table[seq * a.s_table + pi];
    if (page >= 0 && page < a.num_pages) return true;
    atomicExch(&g_bad_index, 1u);
    return false;
}


// Tensor-core kernels (paged_attention_mma.cu): whether there is one for this head_dim, CTAs per SM, and the launch.
int mma_ctas_per_sm(int64_t head_dim);                       // 0: none
inline int mma_rows(int group) { return group <= 8 ? 8 : 16; }  // query rows that a CTA takes at a time
int launch_mma(const PagedArgs &a, int dtype, int grid, cudaStream_t st);

}  // namespace paged
}  // namespace enc

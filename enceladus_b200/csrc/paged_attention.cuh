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
// Split: the work is a line of 64-key tiles (sequence by sequence, kv head by kv head), cut into runs.  Every CTA finds its
// runs from seq_lens by a scan over the batch, so ragged lengths, one long sequence and many short ones all load every
// SM alike, and nothing about the lengths has to reach the host.  A row that ends inside a run is finished there; the up to
// two pieces of a run that belong to rows cut by its ends go to a workspace and a second, overlapped launch joins them in
// order (no atomics: the result does not depend on timing).
//
// Where no row can have more than ROW_TILES tiles, rows are not cut at all: the line counts rows, and there is nothing to join
// (one sequence of 130 keys: the same 10.5 us on the device, but 14.0 instead of 18.5 us a call from the host).
//
// Equal runs are not equal times: SMs differ by up to 1.3 in the bandwidth they get (measured per SM with equal runs: 500 to
// 663 us at 48 x 32 kv heads).  So the runs come in two lengths: as many long ones as CTAs fit the GPU, 60% of the work, and
// several times as many short ones that the ring kernel's CTAs claim as they get free (680 -> 617 us).
#pragma once

#include "paged.cuh"

namespace enc {
namespace paged {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int TILE = 64;          // keys of a tile
constexpr int ROW_TILES = 4;      // rows of at most so many tiles are not cut
constexpr int MAX_HEAD_DIM = 256;

struct PagedArgs {
    const void *q, *k, *v;
    void *o;
    float *lse;
    const int32_t *block_table, *seq_lens;
    int4 *headers;   // per run: the row group that its last piece begins {sequence, rows and first head, last run of it, -};
                     // behind the last run's, how many runs have tiles
    float *slots;    // per run two pieces, see slot_of
    int64_t sq_s, sq_h, so_s, so_h, sk_p, sk_h, sk_t, sv_p, sv_h, sv_t, s_table;
    int64_t num_seqs, num_pages, capacity, window;
    int q_heads, head_dim, group, row_groups;  // query rows per kv head; row groups (of the kernel's row count) per kv head
    int units;                                 // row groups per sequence: kv_heads * row_groups
    bool by_rows;                              // rows are not cut: the line counts row groups instead of tiles
    bool whole;                                // pages are whole multiples of 16 keys
    int long_runs;                             // runs of the first kind; the grid's other runs are short ones
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
static __device__ __forceinline__ int tiles_of(int keys) { return (keys + TILE - 1) / TILE; }
// What a sequence's row group takes up on the line: its tiles, or one where rows are not cut (a.by_rows).
static __device__ __forceinline__ int weight_of(const PagedArgs &a, int keys) { return a.by_rows ? keys > 0 : tiles_of(keys); }

// The line of tiles, as every CTA computes it (below 2^31 tiles: the host refuses more, and 32-bit divisions are several times
// as fast as 64-bit ones).
struct Line {
    int total, long_run, shorts_at, share;  // tiles; where the short runs begin and how many tiles they divide
    int shorts;
    bool any_empty;                         // some sequence has no keys

    // A run's tiles; none if there are fewer tiles than runs, and then none in the runs behind it either.
    __device__ __forceinline__ void run(const PagedArgs &a, int id, int &begin, int &end) const {
        int64_t b, e;
        if (id < a.long_runs) {
            b = (int64_t)id * long_run;
            e = b + long_run;
        } else {  // the first `more` short runs have a tile more than the others
            const int k = id - a.long_runs, least = share / shorts, more = share - least * shorts;
            b = (int64_t)shorts_at + (int64_t)k * least + (k < more ? k : more);
            e = b + least + (k < more);
        }
        begin = (int)(b < total ? b : total);
        end = (int)(e < total ? e : total);
    }
    __device__ __forceinline__ int run_of(const PagedArgs &a, int tile) const {
        if (tile < shorts_at) return tile / long_run;
        const int least = share / shorts, more = share - least * shorts, x = tile - shorts_at, wide = more * (least + 1);
        return a.long_runs + (x < wide ? x / (least + 1) : more + (x - wide) / least);
    }
    __device__ __forceinline__ int runs(const PagedArgs &a) const { return total > 0 ? run_of(a, total - 1) + 1 : 0; }
};

// The sequences are dealt to the threads in contiguous pieces; `before`[i] (shared) becomes the tiles in front of thread i's
// piece.
static __device__ __forceinline__ Line make_line(const PagedArgs &a, int (&before)[THREADS]) {
    __shared__ int warp_total[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t per = (a.num_seqs + THREADS - 1) / THREADS;
    const int64_t b0 = threadIdx.x * per, b1 = b0 + per < a.num_seqs ? b0 + per : a.num_seqs;
    int mine = 0;
    int first, skip;
    bool empty = false;
    for (int64_t b = b0; b < b1; ++b) {
        const int keys = keys_of(a, b, first, skip);
        empty |= keys == 0;
        mine += weight_of(a, keys) * a.units;
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) warp_total[warp] = upto;
    Line r;
    r.any_empty = __syncthreads_or(empty);
    int front = upto - mine;
    r.total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) front += warp_total[w];
        r.total += warp_total[w];
    }
    before[threadIdx.x] = front;
    r.shorts = (int)gridDim.x - a.long_runs;
    r.long_run = r.shorts > 0 ? r.total / 4 * 3 / a.long_runs : (r.total + a.long_runs - 1) / a.long_runs;
    if (r.long_run < 1) r.long_run = 1;
    r.shorts_at = r.long_run * a.long_runs;
    r.share = r.total - r.shorts_at > r.shorts ? r.total - r.shorts_at : r.shorts;  // at least a tile each, to the last
    if (threadIdx.x == 0 && a.headers) a.headers[gridDim.x].x = r.runs(a);  // for the join (the same from every block)
    __syncthreads();
    return r;
}

// The sequence that holds a tile of the line (tile < total), and the tile's place among the sequence's.  By a whole warp.
static __device__ __forceinline__ void find_tile(const PagedArgs &a, const int (&before)[THREADS], int tile, int64_t &seq, int &at) {
    const int lane = threadIdx.x & 31;
    unsigned behind = 0;  // pieces that begin at the tile or in front of it
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) behind += before[lane + 32 * i] <= tile;
    const int piece = (int)__reduce_add_sync(0xffffffffu, behind) - 1;
    at = tile - before[piece];
    seq = piece * ((a.num_seqs + THREADS - 1) / THREADS);
    for (;; ++seq) {
        int first, skip;
        const int t = weight_of(a, keys_of(a, seq, first, skip)) * a.units;
        if (at < t) return;
        at -= t;
    }
}

// Elements e .. e + 3 of an output row of n: x / l, rounded once.
template <typename T> __device__ __forceinline__ void store4(T *o, int e, int n, const float (&x)[4], float l) {
    const float inverse = l == 0.0f ? 0.0f : __frcp_rn(l);
    T y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = from_f32<T>(l == 0.0f ? 0.0f : x[i] * inverse);
    if (e + 4 <= n && reinterpret_cast<uintptr_t>(o + e) % (4 * sizeof(T)) == 0) {
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(o + e) = reinterpret_cast<const uint4 &>(y);
        else *reinterpret_cast<uint2 *>(o + e) = reinterpret_cast<const uint2 &>(y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (e + i < n) o[e + i] = y[i];
    }
}

// A run's two pieces: `rows` rows of O (rounded up to four elements), then m and l.
__host__ __device__ inline int64_t slot_stride(int head_dim) { return (head_dim + 3) / 4 * 4 + 4; }
static __device__ __forceinline__ float *slot_of(const PagedArgs &a, int64_t run, int which, int rows) {
    return a.slots + (2 * run + which) * rows * slot_stride(a.head_dim);
}

// A piece's rows, one partial result per warp in shared memory (O unnormalised, rows `stride` floats apart, m and l), joined and
// written (elements d0 .. d0 + dims - 1 of the head, `so` starting at d0): to the output when the piece is the whole row, to
// `slot` otherwise.  A warp per row, four neighbouring elements per lane; stride is a multiple of 4.
template <typename T, int ROWS>
__device__ __forceinline__ void write_piece(const PagedArgs &a, const float *so, int warp_stride, int stride, const float (*sm)[ROWS], const float (*sl)[ROWS],
                                            int rows, int64_t seq, int first_head, float *slot, int d0, int dims) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < rows; r += WARPS) {
        float m = sm[0][r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) m = fmaxf(m, sm[w][r]);
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, c[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            c[w] = fast_exp2(sm[w][r] - base);
            l = fmaf(sl[w][r], c[w], l);
        }
        T *o = reinterpret_cast<T *>(a.o) + seq * a.so_s + (first_head + r) * a.so_h + d0;
        float *p = slot + r * slot_stride(a.head_dim);
        for (int e = lane * 4; e < dims; e += 128) {
            float x[4] = {};
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float4 y = *reinterpret_cast<const float4 *>(so + w * warp_stride + r * stride + e);
                x[0] = fmaf(y.x, c[w], x[0]); x[1] = fmaf(y.y, c[w], x[1]);
                x[2] = fmaf(y.z, c[w], x[2]); x[3] = fmaf(y.w, c[w], x[3]);
            }
            if (slot) *reinterpret_cast<float4 *>(p + d0 + e) = make_float4(x[0], x[1], x[2], x[3]);
            else store4<T>(o, e, dims, x, l);
        }
        if (lane == 0 && d0 == 0) {
            if (slot) *reinterpret_cast<float2 *>(p + slot_stride(a.head_dim) - 4) = make_float2(m, l);
            else if (a.lse) a.lse[seq * a.q_heads + first_head + r] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
        }
    }
}

// The rows of sequences without keys, dealt over the long runs (which all have a block of their own): zero, lse -inf.
template <typename T> __device__ __forceinline__ void write_empty_rows(const PagedArgs &a, int id) {
    T *o = reinterpret_cast<T *>(a.o);
    for (int64_t b = id; b < a.num_seqs; b += a.long_runs) {
        int first, skip;
        if (keys_of(a, b, first, skip) > 0) continue;
        for (int i = threadIdx.x; i < a.q_heads * a.head_dim; i += THREADS) {
            const int h = i / a.head_dim, d = i - h * a.head_dim;
            o[b * a.so_s + h * a.so_h + d] = from_f32<T>(0.0f);
            if (d == 0 && a.lse) a.lse[b * a.q_heads + h] = -INFINITY;
        }
    }
}

// Walks over the CTA's run: process(seq, kv head, first query head, rows, first key, keys to skip, keys, tile range, slot or
// NULL) per piece.  Also writes the header that the join reads, and the rows of sequences without keys.
template <typename T, int ROWS, typename F> __device__ __forceinline__ void walk_run(const PagedArgs &a, F process) {
    __shared__ int before[THREADS];
    const Line line = make_line(a, before);
    int pos, end, at = 0;
    int64_t seq = 0;
    line.run(a, blockIdx.x, pos, end);
    if (threadIdx.x == 0 && a.headers) a.headers[blockIdx.x].y = 0;
    if (pos < end) find_tile(a, before, pos, seq, at);
    while (pos < end) {
        int first, skip;
        const int keys = keys_of(a, seq, first, skip), tiles = tiles_of(keys), weight = weight_of(a, keys);
        if (at >= weight * a.units) {
            at -= weight * a.units;  // (zero: a sequence is walked to its end)
            ++seq;
            continue;
        }
        const int unit = at / weight, t0 = at - unit * weight;  // (by rows: 0)
        const int t1 = a.by_rows || tiles - t0 < end - pos ? tiles : t0 + (end - pos);
        const int kv_head = unit / a.row_groups, rg = unit - kv_head * a.row_groups;
        const int rows = a.group - rg * ROWS < ROWS ? a.group - rg * ROWS : ROWS;
        const int first_head = kv_head * a.group + rg * ROWS;
        float *slot = nullptr;
        if (t0 > 0) {
            slot = slot_of(a, blockIdx.x, 0, ROWS);
        } else if (t1 < tiles) {
            slot = slot_of(a, blockIdx.x, 1, ROWS);
            if (threadIdx.x == 0) a.headers[blockIdx.x] = make_int4((int)seq, rows | (first_head << 8), line.run_of(a, pos + tiles - 1), 0);
        }
        process(seq, kv_head, first_head, rows, first, skip, keys, t0, t1, slot);
        pos += a.by_rows ? 1 : t1 - t0;
        at += a.by_rows ? 1 : t1 - t0;
    }
    if (line.any_empty) write_empty_rows<T>(a, blockIdx.x);
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


// The ring kernels (paged_attention_ring.cu): CTAs per SM for a type and head_dim, 0 where there is none, the query rows that a
// CTA takes at a time, and the launch.
int ring_ctas_per_sm(int dtype, int64_t head_dim);
inline int ring_rows(int dtype, int group) { return dtype == ENC_F32 ? (group == 1 ? 1 : 4) : group <= 8 ? 8 : 16; }
int launch_ring(const PagedArgs &a, int dtype, int grid, cudaStream_t st);

}  // namespace paged
}  // namespace enc

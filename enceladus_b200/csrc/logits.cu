// Penalties for repeated tokens, biases and grammar masks on logits, one pass.
//
// Mathematics per row and token t (float32, one rounding at the store): a token of the history is divided by the repetition
// penalty where positive and multiplied where not; one that was generated n > 0 times loses frequency * n + presence; the
// row's biases are added; a token whose mask bit is clear becomes -inf whatever it was.
//
// What bounds it: bytes, the logits read once and written once.  Few tokens of a row are penalised, but they are scattered over
// it, and whatever is done for one lane of a warp costs the warp.  So everything but the stream is done on compacted lists.
// A CTA owns a stretch of one row's vocabulary.  It streams the stretch through the mask, which waits for nothing but the
// logits.  Meanwhile it searches the row's history for tokens of the stretch (a comparison per token; a warp's finds take
// their places in a queue by a prefix sum), counts the queue in shared memory (integer atomics, so the order does not
// matter) and lists each token when it is first counted; the list is worked off over what was streamed and is still in L2.
// Nothing the size of the vocabulary besides the logits touches memory.
// Measured at 256 x 131072 float32 with histories up to 8192: penalties inside the stream 145 us, the list before the stream 131,
// after it 102, queue and list 85 (of which the stream alone is 39).  A fourth CTA per SM (counts of 16 bits, 32 registers a
// thread) 87.  A second launch with a hash table per row 98 (its scattered reads and writes go to memory again), a cluster per
// row that counts each token once over distributed shared memory 235 (common tokens queue up at one CTA).
#include <type_traits>

#include "paged.cuh"

namespace enc {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr uint32_t IN_PROMPT = 1u << 31, HAS_BIAS = 1u << 30;          // above the count, which the history's length bounds
constexpr uint32_t COUNT = HAS_BIAS - 1;
constexpr int AHEAD = 8;                                               // tokens of the history per thread and round
constexpr int STAGED = 512;                                            // biases that shared memory holds

struct LogitsArgs {
    const void *in;
    void *out;
    const int32_t *tokens, *lens, *prompt_lens, *bias_ids, *mask;
    const float *repetition, *frequency, *presence, *bias_values;
    int64_t vocab, s_in, s_out, s_tokens, s_bias, s_mask;
    int history, biases;
};

// A vector with -inf in place of the elements whose bits are clear.
template <typename T> __device__ __forceinline__ uint4 masked(uint4 x, uint32_t bits) {
    uint32_t *w = reinterpret_cast<uint32_t *>(&x);
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bits >> i & 1 ? w[i] : 0xff800000u;
    } else {
        const uint32_t low = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t keep = (bits >> (2 * i) & 1 ? 0xffffu : 0u) | (bits >> (2 * i + 1) & 1 ? 0xffff0000u : 0u);
            w[i] = (w[i] & keep) | (low & ~keep);
        }
    }
    return x;
}

// A stretch of a row, cut so that the input's vectors are aligned whatever the row's address: with `skew` elements of the row's
// first vector in front of the row, stretch i starts at token i * tile - skew.  A thread has VPT vectors of it.
template <typename T, int VPT> struct Stretch {
    static constexpr int NV = Pack<T>::N, TILE = VPT * THREADS * NV;
    const T *in;
    T *out;
    const int32_t *mask;
    int skew, vocab, v0;  // v0: the stretch's first token; negative in a skewed row's first stretch
    bool aligned_out;     // the input's vectors are vectors of the output too
    bool inside;          // and all of them lie in the row
    uint4 x[VPT];
    uint32_t bits[VPT];   // the mask's

    __device__ __forceinline__ Stretch(const LogitsArgs &a, int64_t row, int i) {
        in = reinterpret_cast<const T *>(a.in) + row * a.s_in;
        out = reinterpret_cast<T *>(a.out) + row * a.s_out;
        mask = a.mask ? a.mask + row * a.s_mask : nullptr;
        skew = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
        vocab = (int)a.vocab;
        v0 = i * TILE - skew;
        aligned_out = reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T) == skew;
        inside = v0 >= 0 && v0 + TILE <= vocab && aligned_out;
    }
    __device__ __forceinline__ int token(int j) const { return v0 + (j * THREADS + (int)threadIdx.x) * NV; }
    __device__ __forceinline__ void load() {
        if (inside) {
            const T *p = in + v0 + (int)threadIdx.x * NV;
#pragma unroll
            for (int j = 0; j < VPT; ++j) x[j] = *reinterpret_cast<const uint4 *>(p + j * THREADS * NV);
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int t = token(j);
                if (t >= 0 && t + NV <= vocab) {
                    x[j] = *reinterpret_cast<const uint4 *>(in + t);
                } else {
                    T *e = reinterpret_cast<T *>(&x[j]);
#pragma unroll
                    for (int i = 0; i < NV; ++i) e[i] = t + i >= 0 && t + i < vocab ? in[t + i] : from_f32<T>(0.0f);
                }
            }
        }
        if (!mask) return;
        if (skew == 0) {  // a vector's bits lie in one word
#pragma unroll
            for (int j = 0; j < VPT; ++j) bits[j] = token(j) < vocab ? (uint32_t)mask[token(j) >> 5] >> (token(j) & 31) : 0u;
        } else {          // in two, perhaps; bits in front of the row and behind it do not matter
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int t = token(j), first = t < 0 ? 0 : t, last = t + NV - 1 < vocab ? t + NV - 1 : vocab - 1;
                bits[j] = 0;
                if (first > last) continue;
                const uint32_t lo = mask[first >> 5], hi = mask[last >> 5];
                bits[j] = t < 0 ? lo << -t : __funnelshift_r(lo, hi, t & 31);
            }
        }
    }
    __device__ __forceinline__ void store() {
        if (mask) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) x[j] = masked<T>(x[j], bits[j]);
        }
        if (inside) {
            T *p = out + v0 + (int)threadIdx.x * NV;
#pragma unroll
            for (int j = 0; j < VPT; ++j) *reinterpret_cast<uint4 *>(p + j * THREADS * NV) = x[j];
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int t = token(j);
                if (aligned_out && t >= 0 && t + NV <= vocab) {
                    *reinterpret_cast<uint4 *>(out + t) = x[j];
                } else {
                    const T *e = reinterpret_cast<const T *>(&x[j]);
#pragma unroll
                    for (int i = 0; i < NV; ++i)
                        if (t + i >= 0 && t + i < vocab) out[t + i] = e[i];
                }
            }
        }
    }
};

// VPT 16-byte vectors per thread: a stretch of VPT * THREADS vectors.
template <typename T, int VPT> __global__ void __launch_bounds__(THREADS, 3) logits_kernel(LogitsArgs a) {
    constexpr int NV = Pack<T>::N, TILE = VPT * THREADS * NV;
    extern __shared__ __align__(16) uint32_t seen[];              // [TILE] what was counted per token
    uint16_t *list = reinterpret_cast<uint16_t *>(seen + TILE);   // [TILE] the tokens with something counted
    __shared__ uint16_t queue[THREADS * AHEAD];                   // finds of a round: place in the stretch, QUEUE_PROMPT
    __shared__ int bias_id[STAGED], listed, queued;
    __shared__ float bias_value[STAGED], penalty[3];
    constexpr uint16_t QUEUE_PROMPT = 0x8000;
    static_assert(TILE <= QUEUE_PROMPT, "a place and a flag in 16 bits");
    const int lane = threadIdx.x & 31;
    const int64_t row = blockIdx.y;
    Stretch<T, VPT> st(a, row, blockIdx.x);
    const int vocab = st.vocab, v0 = st.v0;
    if (v0 >= vocab) return;
    const int lo = v0 < 0 ? 0 : v0, hi = v0 + TILE < vocab ? v0 + TILE : vocab;  // tokens of the stretch
    const int32_t *tok = a.tokens + row * a.s_tokens, *ids = a.bias_ids + row * a.s_bias;
    const float *values = a.bias_values + row * a.s_bias;
    const int history = a.tokens ? a.history : 0;
    const bool reports = blockIdx.x == 0;  // one CTA per row reports what is out of range
    grid_dependency_wait();
    // Everything that the search needs and the logits themselves are asked for at once: a stretch takes a few microseconds, and
    // one round trip to memory after the other would be most of them.
    int token[AHEAD];
    const bool quads = aligned16(tok) && history % 4 == 0;
    auto load_tokens = [&](int i0) {  // AHEAD neighbouring tokens from i0 on, in fours
#pragma unroll
        for (int u = 0; u < AHEAD; u += 4) {
            if (quads) {
                int4 x = make_int4(0, 0, 0, 0);
                if (i0 + u < history) x = *reinterpret_cast<const int4 *>(tok + i0 + u);
                token[u] = x.x; token[u + 1] = x.y; token[u + 2] = x.z; token[u + 3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) token[u + e] = i0 + u + e < history ? tok[i0 + u + e] : 0;
            }
        }
    };
    load_tokens(threadIdx.x * AHEAD);
    int n = 0, prompt = 0;
    if (a.tokens) {
        n = a.lens[row];
        prompt = a.prompt_lens[row];
    }
    for (int i = threadIdx.x; i < a.biases && i < STAGED; i += THREADS) {
        bias_id[i] = ids[i];
        bias_value[i] = values[i];
    }
    if (threadIdx.x < 3 && a.tokens) penalty[threadIdx.x] = (threadIdx.x == 0 ? a.repetition : threadIdx.x == 1 ? a.frequency : a.presence)[row];
    st.load();
#pragma unroll
    for (int i = 0; i < TILE / 4 / THREADS; ++i) reinterpret_cast<uint4 *>(seen)[i * THREADS + threadIdx.x] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) listed = queued = 0;
    __syncthreads();
    bool bad = n < 0 || n > history || prompt < 0 || prompt > n;
    n = n < 0 ? 0 : n > history ? history : n;
    auto note = [&](int at, bool add, uint32_t what) {
        const uint32_t before = add ? atomicAdd(&seen[at], what) : atomicOr(&seen[at], what);
        if (before == 0) list[atomicAdd(&listed, 1)] = (uint16_t)at;
    };
    for (int r0 = 0; r0 < n; r0 += THREADS * AHEAD) {
        const int i0 = r0 + threadIdx.x * AHEAD;
        unsigned found = 0;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if ((unsigned)(token[u] - lo) < (unsigned)(hi - lo)) found |= 1u << u;
        const int here = n - i0;  // tokens of the AHEAD that count
        const unsigned valid = here >= AHEAD ? (1u << AHEAD) - 1 : here > 0 ? (1u << here) - 1 : 0u;
        found &= valid;
        if (reports) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) bad |= (valid >> u & 1) && (unsigned)token[u] >= (unsigned)vocab;
        }
        int before = __popc(found);  // inclusive prefix sum over the warp, one reservation per warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += y;
        }
        int at = 0;
        if (lane == 31 && before > 0) at = atomicAdd(&queued, before);
        at = __shfl_sync(0xffffffffu, at, 31) + before - __popc(found);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (found >> u & 1) queue[at++] = (uint16_t)(token[u] - v0) | (i0 + u < prompt ? QUEUE_PROMPT : 0);
        if (r0 + THREADS * AHEAD < n) load_tokens(i0 + THREADS * AHEAD);  // the next round's
        __syncthreads();
        const int in_queue = queued;
        for (int i = threadIdx.x; i < in_queue; i += THREADS) {
            const int q = queue[i];
            note(q & (QUEUE_PROMPT - 1), !(q & QUEUE_PROMPT), q & QUEUE_PROMPT ? IN_PROMPT : 1u);
        }
        if (r0 + THREADS * AHEAD < n) {
            __syncthreads();
            if (threadIdx.x == 0) queued = 0;
            __syncthreads();
        }
    }
    for (int i = threadIdx.x; i < a.biases; i += THREADS) {
        const int t = i < STAGED ? bias_id[i] : ids[i];
        if ((unsigned)(t - lo) < (unsigned)(hi - lo)) note(t - v0, false, HAS_BIAS);
        else if (t < -1 || t >= vocab) bad = true;
    }
    if (bad && reports) atomicExch(&g_bad_index, 1u);
    st.store();
    __syncthreads();
    // the list; its logits were read just now (in place, what was streamed over them is the same value, or -inf where -inf stays)
    if (listed == 0) return;
    const float rep = penalty[0], freq = penalty[1], pres = penalty[2];  // (not looked at without a history)
    for (int i0 = threadIdx.x - lane; i0 < listed; i0 += THREADS) {  // a warp's 32 of the list
        const bool there = i0 + lane < listed;
        const int at = there ? list[i0 + lane] : 0, t = v0 + at;
        const uint32_t w = seen[at], made = w & COUNT;
        const bool allowed = there && (!st.mask || ((st.mask[t >> 5] >> (t & 31)) & 1));
        float f = allowed ? to_f32(st.in[t]) : 0.0f;
        if (made || (w & IN_PROMPT)) f = f > 0.0f ? __fdiv_rn(f, rep) : f * rep;
        if (made) f -= fmaf(freq, (float)made, pres);
        // a token with biases: the warp searches them together and adds what it finds in their order
        for (unsigned biased = __ballot_sync(0xffffffffu, allowed && (w & HAS_BIAS)); biased; biased &= biased - 1) {
            const int who = __ffs(biased) - 1, wanted = __shfl_sync(0xffffffffu, t, who);
            float b = 0.0f;
            for (int e0 = 0; e0 < a.biases; e0 += 32) {
                const int e = e0 + lane;
                const int id = e >= a.biases ? -1 : e < STAGED ? bias_id[e] : ids[e];
                for (unsigned hits = __ballot_sync(0xffffffffu, id == wanted); hits; hits &= hits - 1) {
                    const int hit = e0 + __ffs(hits) - 1;
                    b += hit < STAGED ? bias_value[hit] : values[hit];
                }
            }
            if (lane == who) f += b;
        }
        if (allowed) st.out[t] = from_f32<T>(f);
    }
}

template <typename T, int VPT> int launch_tile(const LogitsArgs &a, int64_t rows, cudaStream_t st) {
    constexpr int NV = Pack<T>::N, TILE = VPT * THREADS * NV, SMEM = TILE * 6;
    static OncePerDevice opted;
    const int rc = opted.opt_in(logits_kernel<T, VPT>, SMEM, "enc_penalize_logits");
    if (rc != ENC_OK) return rc;
    // a skewed row may need one stretch more
    launch_overlapped(logits_kernel<T, VPT>, dim3((unsigned)cdiv(a.vocab + NV - 1, TILE), (unsigned)rows), dim3(THREADS), SMEM, st, a);
    return check_launch("enc_penalize_logits");
}

template <typename T> int launch_logits(const LogitsArgs &a, int64_t rows, cudaStream_t st) {
    note_indexed_launch();
    constexpr int VPT = 8192 / THREADS / Pack<T>::N;
    return rows * cdiv(a.vocab, 8192) >= device_props().sm_count ? launch_tile<T, VPT>(a, rows, st) : launch_tile<T, 1>(a, rows, st);
}

}  // namespace

unsigned int take_bad_index_logits() { return take_bad_index_word(); }
int logits_variants() { return 1; }
void logits_variant_info(int, char *out, size_t n) { snprintf(out, n, "cta_threads=%d, a stretch of the vocabulary per CTA", THREADS); }

}  // namespace enc

extern "C" int enc_penalize_logits(const enc_logits_args *args, int dtype, int variant, void *stream) {
    ENC_PROLOGUE();
    using namespace enc;
    const char *me = "enc_penalize_logits";
    if (!args) return fail(ENC_ERR_BAD_ARG, "%s: NULL arguments", me);
    const enc_logits_args &g = *args;
    const int64_t rows = g.rows, vocab = g.vocab, history = g.history, num_biases = g.num_biases;
    if (!is_float_dtype(dtype)) return fail(ENC_ERR_BAD_ARG, "%s: dtype %d is not float16, bfloat16 or float32", me, dtype);
    if (variant >= logits_variants()) return fail(ENC_ERR_BAD_ARG, "%s: variant %d out of range", me, variant);
    if (rows < 0 || vocab < 0 || history < 0 || num_biases < 0) return fail(ENC_ERR_BAD_ARG, "%s: negative size", me);
    const int given = !!g.tokens + !!g.lens + !!g.prompt_lens + !!g.repetition + !!g.frequency + !!g.presence;
    if (given != 0 && given != 6 && !(given == 5 && !g.tokens && history == 0))
        return fail(ENC_ERR_BAD_ARG, "%s: tokens, lens, prompt_lens, repetition, frequency and presence come together", me);
    if (num_biases > 0 && (!g.bias_ids || !g.bias_values)) return fail(ENC_ERR_BAD_ARG, "%s: biases without ids or values", me);
    if (g.mask && g.stride_mask < cdiv(vocab, 32)) return fail(ENC_ERR_BAD_ARG, "%s: %lld mask words a row do not cover %lld tokens", me, (long long)g.stride_mask, (long long)vocab);
    if (rows == 0 || vocab == 0) return ENC_OK;
    if (!g.logits || !g.out) return fail(ENC_ERR_BAD_ARG, "%s: NULL tensor", me);
    if (rows > 65535 || vocab > 0x3fffffffLL || history > (int64_t)COUNT || num_biases > 0x3fffffffLL)
        return fail(ENC_ERR_UNSUPPORTED, "%s: more than 65535 rows, or 2^30-1 tokens, history or biases", me);
    LogitsArgs a{};
    a.in = g.logits; a.out = g.out; a.tokens = g.tokens; a.lens = g.lens; a.prompt_lens = g.prompt_lens; a.bias_ids = g.bias_ids; a.mask = g.mask;
    a.repetition = g.repetition; a.frequency = g.frequency; a.presence = g.presence; a.bias_values = g.bias_values;
    a.vocab = vocab; a.s_in = g.stride_in; a.s_out = g.stride_out; a.s_tokens = g.stride_tokens; a.s_bias = g.stride_bias; a.s_mask = g.stride_mask;
    a.history = (int)history; a.biases = (int)num_biases;
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ENC_F16: return launch_logits<__half>(a, rows, st);
        case ENC_BF16: return launch_logits<__nv_bfloat16>(a, rows, st);
        default: return launch_logits<float>(a, rows, st);
    }
}

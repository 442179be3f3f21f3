// Penalties for repeated tokens, biases and grammar masks on logits, one pass.
//
// Mathematics per row and token t (float32, one rounding at the store): a token of the history is divided by the repetition
// penalty where positive and multiplied where not; one that was generated n > 0 times loses frequency * n + presence; the
// row's biases are added; a token whose mask bit is clear becomes -inf whatever it was.
//
// What bounds it: bytes, the logits read once and written once.  A CTA owns a stretch of one row's vocabulary: it counts the
// history's tokens that fall into the stretch in shared memory (integer atomics, so the order does not matter), then streams
// the stretch; a count word of zero leaves the logit as it is, which is nearly all of them.  Nothing the size of the
// vocabulary besides the logits touches memory.
#include "paged.cuh"

namespace enc {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_TILE = 8192;                                         // tokens of a stretch at most (32 KB of counts)
constexpr uint32_t IN_PROMPT = 1u << 31, HAS_BIAS = 1u << 30;          // above the count, which the history's length bounds
constexpr uint32_t COUNT = HAS_BIAS - 1;

struct LogitsArgs {
    const void *in;
    void *out;
    const int32_t *tokens, *lens, *prompt_lens, *bias_ids, *mask;
    const float *repetition, *frequency, *presence, *bias_values;
    int64_t vocab, s_in, s_out, s_tokens, s_bias, s_mask;
    int history, biases, tile;
};

template <typename T> __global__ void __launch_bounds__(THREADS) logits_kernel(LogitsArgs a) {
    extern __shared__ uint32_t seen[];
    grid_dependency_wait();
    const int64_t row = blockIdx.y;
    const int v0 = blockIdx.x * a.tile, v1 = a.vocab - v0 < a.tile ? (int)a.vocab : v0 + a.tile;
    for (int i = threadIdx.x; i < v1 - v0; i += THREADS) seen[i] = 0;
    __syncthreads();
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    const bool reports = blockIdx.x == 0;  // one CTA per row reports what is out of range
    if (a.tokens) {
        int n = a.lens[row], prompt = a.prompt_lens[row];
        if (n < 0 || n > a.history || prompt < 0 || prompt > n) {
            if (reports && threadIdx.x == 0) atomicExch(&g_bad_index, 1u);
            n = n < 0 ? 0 : n > a.history ? a.history : n;
        }
        rep = a.repetition[row];
        freq = a.frequency[row];
        pres = a.presence[row];
        const int32_t *tok = a.tokens + row * a.s_tokens;
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const int t = tok[i];
            if (t >= v0 && t < v1) {
                if (i < prompt) atomicOr(&seen[t - v0], IN_PROMPT);
                else atomicAdd(&seen[t - v0], 1u);
            } else if (reports && (t < 0 || t >= a.vocab)) {
                atomicExch(&g_bad_index, 1u);
            }
        }
    }
    const int32_t *ids = a.bias_ids + row * a.s_bias;
    const float *values = a.bias_values + row * a.s_bias;
    for (int i = threadIdx.x; i < a.biases; i += THREADS) {
        const int t = ids[i];
        if (t >= v0 && t < v1) atomicOr(&seen[t - v0], HAS_BIAS);
        else if (reports && (t < -1 || t >= a.vocab)) atomicExch(&g_bad_index, 1u);
    }
    __syncthreads();
    const T *in = reinterpret_cast<const T *>(a.in) + row * a.s_in;
    T *out = reinterpret_cast<T *>(a.out) + row * a.s_out;
    const int32_t *mask = a.mask ? a.mask + row * a.s_mask : nullptr;
    for (int t = v0 + threadIdx.x; t < v1; t += THREADS) {
        float x = to_f32(in[t]);
        const uint32_t w = seen[t - v0];
        if (w) {
            const uint32_t n = w & COUNT;
            if (n || (w & IN_PROMPT)) x = x > 0.0f ? __fdiv_rn(x, rep) : x * rep;
            if (n) x -= fmaf(freq, (float)n, pres);
            if (w & HAS_BIAS) {
                float b = 0.0f;
                for (int i = 0; i < a.biases; ++i)
                    if (ids[i] == t) b += values[i];
                x += b;
            }
        }
        if (mask && !((mask[t >> 5] >> (t & 31)) & 1)) x = -INFINITY;
        out[t] = from_f32<T>(x);
    }
}

template <typename T> int launch_logits(LogitsArgs a, int64_t rows, cudaStream_t st) {
    note_indexed_launch();
    a.tile = MAX_TILE;
    launch_overlapped(logits_kernel<T>, dim3((unsigned)cdiv(a.vocab, a.tile), (unsigned)rows), dim3(THREADS), a.tile * sizeof(uint32_t), st, a);
    return check_launch("enc_penalize_logits");
}

}  // namespace

unsigned int take_bad_index_logits() { return take_bad_index_word(); }
int logits_variants() { return 1; }
void logits_variant_info(int, char *out, size_t n) { snprintf(out, n, "cta_threads=%d, counts of the history in shared memory", THREADS); }

}  // namespace enc

extern "C" int enc_penalize_logits(const void *logits, void *out, int64_t rows, int64_t vocab, int64_t stride_in, int64_t stride_out,
                                   const int32_t *tokens, int64_t history, int64_t stride_tokens, const int32_t *lens,
                                   const int32_t *prompt_lens, const float *repetition, const float *frequency,
                                   const float *presence, const int32_t *bias_ids, const float *bias_values, int64_t num_biases,
                                   int64_t stride_bias, const int32_t *mask, int64_t stride_mask, int dtype, int variant, void *stream) {
    ENC_PROLOGUE();
    using namespace enc;
    const char *me = "enc_penalize_logits";
    if (!is_float_dtype(dtype)) return fail(ENC_ERR_BAD_ARG, "%s: dtype %d is not float16, bfloat16 or float32", me, dtype);
    if (variant >= logits_variants()) return fail(ENC_ERR_BAD_ARG, "%s: variant %d out of range", me, variant);
    if (rows < 0 || vocab < 0 || history < 0 || num_biases < 0) return fail(ENC_ERR_BAD_ARG, "%s: negative size", me);
    const int given = !!tokens + !!lens + !!prompt_lens + !!repetition + !!frequency + !!presence;
    if (given != 0 && given != 6 && !(given == 5 && !tokens && history == 0))
        return fail(ENC_ERR_BAD_ARG, "%s: tokens, lens, prompt_lens, repetition, frequency and presence come together", me);
    if (num_biases > 0 && (!bias_ids || !bias_values)) return fail(ENC_ERR_BAD_ARG, "%s: biases without ids or values", me);
    if (mask && stride_mask < cdiv(vocab, 32)) return fail(ENC_ERR_BAD_ARG, "%s: %lld mask words a row do not cover %lld tokens", me, (long long)stride_mask, (long long)vocab);
    if (rows == 0 || vocab == 0) return ENC_OK;
    if (!logits || !out) return fail(ENC_ERR_BAD_ARG, "%s: NULL tensor", me);
    if (rows > 65535 || vocab > 0x3fffffffLL || history > (int64_t)COUNT || num_biases > 0x3fffffffLL)
        return fail(ENC_ERR_UNSUPPORTED, "%s: more than 65535 rows, or 2^30-1 tokens, history or biases", me);
    LogitsArgs a{};
    a.in = logits; a.out = out; a.tokens = tokens; a.lens = lens; a.prompt_lens = prompt_lens; a.bias_ids = bias_ids; a.mask = mask;
    a.repetition = repetition; a.frequency = frequency; a.presence = presence; a.bias_values = bias_values;
    a.vocab = vocab; a.s_in = stride_in; a.s_out = stride_out; a.s_tokens = stride_tokens; a.s_bias = stride_bias; a.s_mask = stride_mask;
    a.history = (int)history; a.biases = (int)num_biases;
    cudaStream_t st = as_stream(stream);
    switch (dtype) {
        case ENC_F16: return launch_logits<__half>(a, rows, st);
        case ENC_BF16: return launch_logits<__nv_bfloat16>(a, rows, st);
        default: return launch_logits<float>(a, rows, st);
    }
}

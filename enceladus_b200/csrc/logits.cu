// Penalties for repeated tokens, biases and grammar masks on logits, one pass.
//
// Mathematics per row and token t (float32, one rounding at the store): a token of the history is divided by the repetition
// penalty where positive and multiplied where not; one that was generated n > 0 times loses frequency * n + presence; the
// row's biases are added; a token whose mask bit is clear becomes -inf whatever it was.
//
// What bounds it: bytes, the logits read once and written once.  A CTA owns a stretch of one row's vocabulary.  It streams the
// stretch through the mask, which waits for nothing but the logits, and counts the history's tokens that fall into it in
// shared memory meanwhile (integer atomics, so the order does not matter).  The tokens that something happens to are few but
// scattered, and a warp that met them while streaming would walk through the penalties for one lane nearly every time (900
// instructions a warp at 256 x 131072): so the thread that counts a token first puts it on a list, and the list is worked off
// at the end with every lane busy, over what was streamed.  Nothing the size of the vocabulary besides the logits touches
// memory.
#include "paged.cuh"

namespace enc {
namespace {

constexpr int THREADS = 512;
constexpr uint32_t IN_PROMPT = 1u << 31, HAS_BIAS = 1u << 30;          // above the count, which the history's length bounds
constexpr uint32_t COUNT = HAS_BIAS - 1;

struct LogitsArgs {
    const void *in;
    void *out;
    const int32_t *tokens, *lens, *prompt_lens, *bias_ids, *mask;
    const float *repetition, *frequency, *presence, *bias_values;
    int64_t vocab, s_in, s_out, s_tokens, s_bias, s_mask;
    int history, biases;
};

__device__ __forceinline__ float load_l2(const float *p) { return __ldcg(p); }
__device__ __forceinline__ __half load_l2(const __half *p) { return __ldcg(p); }
__device__ __forceinline__ __nv_bfloat16 load_l2(const __nv_bfloat16 *p) { return __ldcg(p); }

// The logit of a token that its count word says something about.
__device__ __forceinline__ float changed(float x, uint32_t w, float rep, float freq, float pres, const int32_t *ids, const float *values, int biases, int t) {
    const uint32_t n = w & COUNT;
    if (n || (w & IN_PROMPT)) x = x > 0.0f ? __fdiv_rn(x, rep) : x * rep;
    if (n) x -= fmaf(freq, (float)n, pres);
    if (w & HAS_BIAS) {
        float b = 0.0f;
        for (int i = 0; i < biases; ++i)
            if (ids[i] == t) b += values[i];
        x += b;
    }
    return x;
}

// VPT 16-byte vectors per thread: a stretch of VPT * THREADS vectors.  Stretches are cut so that the input's vectors are
// aligned whatever the row's address: with `skew` elements of the row's first vector in front of the row, stretch i starts at
// token i * TILE - skew.
template <typename T, int VPT> __global__ void __launch_bounds__(THREADS, 3) logits_kernel(LogitsArgs a) {
    constexpr int NV = Pack<T>::N, TILE = VPT * THREADS * NV;
    extern __shared__ __align__(16) uint32_t seen[];             // [TILE] what was counted per token
    uint16_t *list = reinterpret_cast<uint16_t *>(seen + TILE);  // [TILE] the tokens with something counted
    __shared__ int listed;
    const int64_t row = blockIdx.y;
    const T *in = reinterpret_cast<const T *>(a.in) + row * a.s_in;
    T *out = reinterpret_cast<T *>(a.out) + row * a.s_out;
    const int skew = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T)), vocab = (int)a.vocab;
    const int v0 = (int)blockIdx.x * TILE - skew;  // token of seen[0]; negative in a skewed row's first stretch
    if (v0 >= vocab) return;
    const int lo = v0 < 0 ? 0 : v0, hi = v0 + TILE < vocab ? v0 + TILE : vocab;  // tokens of the stretch
    const bool aligned_out = reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T) == skew;
    const int32_t *mask = a.mask ? a.mask + row * a.s_mask : nullptr;
    const int32_t *tok = a.tokens + row * a.s_tokens;
    const int history = a.tokens ? a.history : 0, h4 = aligned16(tok) ? history / 4 : 0;
    grid_dependency_wait();
    // Everything that the counting needs and the logits themselves are asked for at once: a stretch takes a few microseconds,
    // and one round trip to memory after the other would be most of them.
    constexpr int UN = 2;  // vectors of the history in flight per thread
    const int4 nothing = make_int4(-1, -1, -1, -1);
    int4 token[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) token[u] = (int)threadIdx.x + u * THREADS < h4 ? reinterpret_cast<const int4 *>(tok)[threadIdx.x + u * THREADS] : nothing;
    int n = 0, prompt = 0;
    if (a.tokens) {
        n = a.lens[row];
        prompt = a.prompt_lens[row];
    }
    uint4 x[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int t = v0 + (j * THREADS + (int)threadIdx.x) * NV;
        if (t >= 0 && t + NV <= vocab) {
            x[j] = ld_stream(in + t);
        } else {
            T *e = reinterpret_cast<T *>(&x[j]);
#pragma unroll
            for (int i = 0; i < NV; ++i) e[i] = t + i >= 0 && t + i < vocab ? in[t + i] : from_f32<T>(0.0f);
        }
    }
#pragma unroll
    for (int i = 0; i < TILE / 4 / THREADS; ++i) reinterpret_cast<uint4 *>(seen)[i * THREADS + threadIdx.x] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const bool reports = blockIdx.x == 0;  // one CTA per row reports what is out of range
    bool bad = n < 0 || n > history || prompt < 0 || prompt > n;
    n = n < 0 ? 0 : n > history ? history : n;
    auto count = [&](int t, int i) {
        if ((unsigned)(t - lo) < (unsigned)(hi - lo)) {
            const uint32_t before = i < prompt ? atomicOr(&seen[t - v0], IN_PROMPT) : atomicAdd(&seen[t - v0], 1u);
            if (before == 0) list[atomicAdd(&listed, 1)] = (uint16_t)(t - v0);
        } else if (reports) {
            bad |= (unsigned)t >= (unsigned)vocab;
        }
    };
    for (int i = threadIdx.x; i < h4 && 4 * i < n; i += UN * THREADS) {
        if (i >= UN * THREADS) {
#pragma unroll
            for (int u = 0; u < UN; ++u) token[u] = i + u * THREADS < h4 ? reinterpret_cast<const int4 *>(tok)[i + u * THREADS] : nothing;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int at = 4 * (i + u * THREADS);
            if (at < n) count(token[u].x, at);
            if (at + 1 < n) count(token[u].y, at + 1);
            if (at + 2 < n) count(token[u].z, at + 2);
            if (at + 3 < n) count(token[u].w, at + 3);
        }
    }
    for (int i = 4 * h4 + threadIdx.x; i < n; i += THREADS) count(tok[i], i);
    const int32_t *ids = a.bias_ids + row * a.s_bias;
    const float *values = a.bias_values + row * a.s_bias;
    for (int i = threadIdx.x; i < a.biases; i += THREADS) {
        const int t = ids[i];
        if ((unsigned)(t - lo) < (unsigned)(hi - lo)) {
            if (atomicOr(&seen[t - v0], HAS_BIAS) == 0) list[atomicAdd(&listed, 1)] = (uint16_t)(t - v0);
        } else if (t < -1 || t >= vocab) {
            bad = true;
        }
    }
    if (bad && reports) atomicExch(&g_bad_index, 1u);

    // the stream
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int t = v0 + (j * THREADS + (int)threadIdx.x) * NV;
        if (t + NV <= 0 || t >= vocab) continue;
        if (mask) {  // NV bits from bit t on; bits in front of the row and behind it do not matter
            uint32_t allowed;
            if (skew == 0) {
                allowed = (uint32_t)mask[t >> 5] >> (t & 31);
            } else {
                const int first = t < 0 ? 0 : t, last = t + NV - 1 < vocab ? t + NV - 1 : vocab - 1;
                const uint32_t w0 = mask[first >> 5], w1 = mask[last >> 5];
                allowed = t < 0 ? w0 << -t : __funnelshift_r(w0, w1, t & 31);
            }
            float f[NV];
            Pack<T>::unpack(x[j], f);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (!((allowed >> i) & 1)) f[i] = -INFINITY;
            x[j] = Pack<T>::pack(f);
        }
        if (aligned_out && t >= 0 && t + NV <= vocab) {
            *reinterpret_cast<uint4 *>(out + t) = x[j];
        } else {
            const T *e = reinterpret_cast<const T *>(&x[j]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (t + i >= 0 && t + i < vocab) out[t + i] = e[i];
        }
    }
    __syncthreads();
    // the list; its logits come from L2 (in place, what was streamed over them is the same value, or -inf where -inf stays)
    if (listed == 0) return;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.tokens) {
        rep = a.repetition[row];
        freq = a.frequency[row];
        pres = a.presence[row];
    }
    for (int i = threadIdx.x; i < listed; i += THREADS) {
        const int at = list[i], t = v0 + at;
        const bool allowed = !mask || ((mask[t >> 5] >> (t & 31)) & 1);
        if (allowed) out[t] = from_f32<T>(changed(to_f32(load_l2(in + t)), seen[at], rep, freq, pres, ids, values, a.biases, t));
    }
}

template <typename T, int VPT> void launch_tile(const LogitsArgs &a, int64_t rows, cudaStream_t st) {
    constexpr int NV = Pack<T>::N, TILE = VPT * THREADS * NV;
    constexpr int SMEM = TILE * 6;
    cudaFuncSetAttribute(logits_kernel<T, VPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    // a skewed row may need one stretch more
    launch_overlapped(logits_kernel<T, VPT>, dim3((unsigned)cdiv(a.vocab + NV - 1, TILE), (unsigned)rows), dim3(THREADS), SMEM, st, a);
}

template <typename T> int launch_logits(const LogitsArgs &a, int64_t rows, cudaStream_t st) {
    note_indexed_launch();
    constexpr int VPT = 8192 / THREADS / Pack<T>::N;
    if (rows * cdiv(a.vocab, 8192) >= device_props().sm_count) launch_tile<T, VPT>(a, rows, st);
    else launch_tile<T, 1>(a, rows, st);
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

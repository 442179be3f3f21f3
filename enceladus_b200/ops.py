"""The kernel set: `@jit` kernel definitions and their host wrappers.

Each wrapper has the signature and behaviour of the reference example of the same name
(examples/01_vector_add.py ... examples/10_cumsum.py): it accepts NumPy arrays or torch CUDA tensors,
allocates its outputs with `new_empty`/`new_zeros` and launches `kernel[grid](...)` with the same
arguments.  The kernel bodies are not executed — each launch is served by the hand-written CUDA kernel
registered under the kernel's name — so a body here is only a statement of what that kernel computes.
A user's own copy of a reference example works the same way after `import enceladus_b200 as enceladus`.
"""

from __future__ import annotations

import math

import numpy as np

import enceladus_b200 as enceladus
import enceladus_b200.language as tl
from enceladus_b200 import _native as N
from enceladus_b200.runtime import lane
from enceladus_b200.configs import attention_configs, matmul_configs


# ---- 01 vector add -----------------------------------------------------------------------------
@enceladus.jit
def add_kernel(x_ptr, y_ptr, out_ptr, n, BLOCK: tl.constexpr):
    """out[i] = x[i] + y[i] for i < n."""


def add(x, y, block: int = 1024):
    """Returns `x + y` for two contiguous arrays of the same shape and dtype."""
    out = enceladus.new_empty(x)
    n = int(np.prod(x.shape))
    add_kernel[(enceladus.cdiv(n, block),)](x, y, out, n, BLOCK=block)
    return out


# ---- 02 softmax --------------------------------------------------------------------------------
@enceladus.jit
def softmax_kernel(out_ptr, in_ptr, stride_in, stride_out, n_cols, BLOCK: tl.constexpr):
    """One row per program: exp(x - max(x)) / sum(exp(x - max(x))) in float32, stored in the input dtype."""


def softmax(x):
    """Returns the softmax of each row of a 2D array, in the input dtype.

    The rows can be strided, but the elements within a row must be contiguous.
    """
    m, n = x.shape
    out = enceladus.new_empty(x)
    softmax_kernel[(m,)](out, x, enceladus.element_strides(x)[0], enceladus.element_strides(out)[0], n,
                         BLOCK=enceladus.next_power_of_2(n))
    return out


# ---- 03 layernorm ------------------------------------------------------------------------------
@enceladus.jit
def layernorm_kernel(x_ptr, y_ptr, w_ptr, b_ptr, mean_ptr, rstd_ptr, stride_x, stride_y, n_cols, eps,
                     BLOCK: tl.constexpr):
    """One row per program: mean, centred variance, rstd = 1/sqrt(var+eps); y = (x-mean)*rstd*w + b."""


def layernorm(x, w, b, eps: float = 1e-5, block: int | None = None):
    """Returns `(y, mean, rstd)` for a 2D input normalized over its last dimension."""
    m, n = x.shape
    y = enceladus.new_empty(x)
    mean = enceladus.new_empty(x, (m,), np.float32)
    rstd = enceladus.new_empty(x, (m,), np.float32)
    block = block or min(1024, enceladus.next_power_of_2(n))
    stride_x, stride_y = enceladus.element_strides(x)[0], enceladus.element_strides(y)[0]
    layernorm_kernel[(m,)](x, y, w, b, mean, rstd, stride_x, stride_y, n, eps, BLOCK=block)
    return y, mean, rstd


# ---- 05 fused GELU -----------------------------------------------------------------------------
@enceladus.jit
def fused_gelu_kernel(x_ptr, bias_ptr, out_ptr, n, n_cols, scale, BLOCK: tl.constexpr):
    """t = x*scale + bias[i % n_cols]; out = 0.5*t*(1 + erf(t/sqrt(2)))."""


def fused_gelu(x, bias, scale: float, block: int = 1024):
    """Returns `gelu(x * scale + bias)` for a contiguous 2D `x` and a bias per column."""
    out = enceladus.new_empty(x)
    n = int(np.prod(x.shape))
    fused_gelu_kernel[(enceladus.cdiv(n, block),)](x, bias, out, n, x.shape[-1], scale, BLOCK=block)
    return out


@enceladus.jit
def tanh_gelu_kernel(x_ptr, out_ptr, n, BLOCK: tl.constexpr):
    """out = 0.5*x*(1 + tanh(0.7978845608*(x + 0.044715*x^3))), elementwise."""


def tanh_gelu(x, block: int = 1024):
    """Returns the tanh-form GELU of a contiguous array of any shape."""
    out = enceladus.new_empty(x)
    n = int(np.prod(x.shape))
    tanh_gelu_kernel[(enceladus.cdiv(n, block),)](x, out, n, BLOCK=block)
    return out


# ---- 06 rmsnorm --------------------------------------------------------------------------------
@enceladus.jit
def rmsnorm_kernel(x_ptr, w_ptr, out_ptr, stride_x, stride_out, n_cols, eps, BLOCK: tl.constexpr):
    """One row per program: x * (1/sqrt(mean(x^2) + eps)) * w."""


def rmsnorm(x, w, eps: float = 1e-6):
    """Returns RMSNorm of each row of a 2D array, in the input dtype."""
    m, n = x.shape
    out = enceladus.new_empty(x)
    rmsnorm_kernel[(m,)](x, w, out, enceladus.element_strides(x)[0], enceladus.element_strides(out)[0], n, eps,
                         BLOCK=enceladus.next_power_of_2(n))
    return out


# ---- 04 / 07 matmul ----------------------------------------------------------------------------
@enceladus.jit
def matmul_desc_kernel(a_ptr, b_ptr, c_ptr, M, N, K, stride_am, stride_bk, stride_cm, BM: tl.constexpr,
                       BN: tl.constexpr, BK: tl.constexpr):
    """C = A @ B with float32 accumulation; out-of-range tile elements read as zero, are not stored."""


@enceladus.jit
def matmul_bias_gelu_kernel(a_ptr, b_ptr, bias_ptr, c_ptr, M, N, K, stride_am, stride_bk, stride_cm,
                            BM: tl.constexpr, BN: tl.constexpr, BK: tl.constexpr):
    """C = gelu_erf(A @ B + bias[None, :]) with the epilogue applied to the float32 accumulator."""


def matmul_desc(a, b, c=None, bm: int = 128, bn: int = 256, bk: int = 64, num_warps: int = 4,
                dot_backend: str = "auto"):
    """Returns `a @ b` in the input dtype. `a`, `b`, and `c` must be row-major."""
    (m, k), (_, n) = a.shape, b.shape
    if c is None:
        c = enceladus.new_empty(a, (m, n))
    grid = (enceladus.cdiv(n, bn), enceladus.cdiv(m, bm))
    sa, sb, sc = (enceladus.element_strides(t)[0] for t in (a, b, c))
    matmul_desc_kernel[grid](a, b, c, m, n, k, sa, sb, sc, BM=bm, BN=bn, BK=bk, num_warps=num_warps,
                             dot_backend=dot_backend)
    return c


matmul = matmul_desc


def matmul_bias_gelu(a, b, bias, c=None, bm: int = 128, bn: int = 256, bk: int = 64, dot_backend: str = "auto"):
    """Returns `gelu(a @ b + bias)` in the input dtype."""
    (m, k), (_, n) = a.shape, b.shape
    if c is None:
        c = enceladus.new_empty(a, (m, n))
    grid = (enceladus.cdiv(n, bn), enceladus.cdiv(m, bm))
    sa, sb, sc = (enceladus.element_strides(t)[0] for t in (a, b, c))
    matmul_bias_gelu_kernel[grid](a, b, bias, c, m, n, k, sa, sb, sc, BM=bm, BN=bn, BK=bk, dot_backend=dot_backend)
    return c


matmul_desc_tuned = enceladus.autotune(configs=matmul_configs("float16"), key=["M", "N", "K"])(matmul_desc_kernel)


def matmul_tuned(a, b, c=None):
    """Returns `a @ b` using the fastest tile variant for this shape and dtype."""
    (m, k), (_, n) = a.shape, b.shape
    if c is None:
        c = enceladus.new_empty(a, (m, n))
    grid = lambda meta: (enceladus.cdiv(n, meta["BN"]), enceladus.cdiv(m, meta["BM"]))  # noqa: E731
    sa, sb, sc = (enceladus.element_strides(t)[0] for t in (a, b, c))
    matmul_desc_tuned[grid](a, b, c, m, n, k, sa, sb, sc)
    return c


# ---- integer matmul (benchmarks/bench_matmul.py:100-131) ------------------------------------------
@enceladus.jit
def int8_matmul_kernel(a_ptr, b_ptr, c_ptr, M, N, K, BM: tl.constexpr, BN: tl.constexpr, BK: tl.constexpr):
    """C[int32] = A @ B for dense row-major integer A [M, K] and B [K, N]: int32 accumulation, exact, products
    and sums wrap modulo 2^32 (an integer `tl.dot` per K block)."""


def int_matmul(a, b, c=None, bm: int = 128, bn: int = 256, bk: int = 128):
    """Returns the exact int32 product of two contiguous integer matrices (int8, uint8, int16 or int32)."""
    (m, k), (_, n) = a.shape, b.shape
    if c is None:
        c = enceladus.new_empty(a, (m, n), np.int32)
    int8_matmul_kernel[(enceladus.cdiv(n, bn), enceladus.cdiv(m, bm))](a, b, c, m, n, k, BM=bm, BN=bn, BK=bk)
    return c


# ---- 08 flash attention ------------------------------------------------------------------------
@enceladus.jit
def attention_kernel(q_ptr, k_ptr, v_ptr, o_ptr, sm_scale, N_CTX, stride_h, stride_m, HEAD_DIM: tl.constexpr,
                     BLOCK_M: tl.constexpr, BLOCK_N: tl.constexpr, CAUSAL: tl.constexpr):
    """softmax(q k^T * sm_scale [causal]) v per (batch, head): base-2 online softmax in float32, the
    probabilities rounded to the input dtype before the second product."""


@enceladus.jit
def attention_lse_kernel(q_ptr, k_ptr, v_ptr, o_ptr, lse_ptr, sm_scale, N_CTX, stride_h, stride_m,
                         HEAD_DIM: tl.constexpr, BLOCK_M: tl.constexpr, BLOCK_N: tl.constexpr,
                         CAUSAL: tl.constexpr):
    """attention_kernel plus lse[b*h, i] = ln2 * (m_i + log2 l_i) of the running statistics, float32."""


def _check_qkv(q, k, v):
    if not (tuple(q.shape) == tuple(k.shape) == tuple(v.shape)) or len(q.shape) != 4:
        raise ValueError("q, k, and v must all have shape (batch, heads, seq_len, head_dim)")
    if q.shape[-1] not in (16, 32, 64, 128):
        raise ValueError(f"head_dim must be 16, 32, 64, or 128, not {q.shape[-1]}")


def attention(q, k, v, causal: bool = False, sm_scale: float | None = None, o=None, block_m: int = 128,
              block_n: int = 128, num_warps: int = 4, return_lse: bool = False):
    """Returns `softmax(q @ k^T * sm_scale) @ v` for contiguous (batch, heads, seq, dim) inputs.

    With `return_lse=True`, also returns the float32 log-sum-exp of the scaled scores, shape
    (batch, heads, seq).
    """
    _check_qkv(q, k, v)
    z, h, n, d = q.shape
    o = enceladus.new_empty(q) if o is None else o
    scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    grid = (enceladus.cdiv(n, block_m), z * h)
    if return_lse:
        lse = enceladus.new_empty(q, (z, h, n), np.float32)
        attention_lse_kernel[grid](q, k, v, o, lse, scale, n, n * d, d, HEAD_DIM=d, BLOCK_M=block_m,
                                   BLOCK_N=block_n, CAUSAL=causal, num_warps=num_warps, dot_warps=(num_warps, 1))
        return o, lse
    attention_kernel[grid](q, k, v, o, scale, n, n * d, d, HEAD_DIM=d, BLOCK_M=block_m, BLOCK_N=block_n,
                           CAUSAL=causal, num_warps=num_warps, dot_warps=(num_warps, 1))
    return o


attention_tuned_kernel = enceladus.autotune(configs=attention_configs("float16", 128),
                                            key=["N_CTX", "HEAD_DIM", "CAUSAL"])(attention_kernel)


def attention_tuned(q, k, v, causal: bool = False, sm_scale: float | None = None, o=None):
    """Returns the same result as `attention`, using the fastest tile variant for the shape."""
    _check_qkv(q, k, v)
    z, h, n, d = q.shape
    o = enceladus.new_empty(q) if o is None else o
    scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    grid = lambda meta: (enceladus.cdiv(n, meta["BLOCK_M"]), z * h)  # noqa: E731
    attention_tuned_kernel[grid](q, k, v, o, scale, n, n * d, d, HEAD_DIM=d, CAUSAL=causal)
    return o


# ---- 09 histogram ------------------------------------------------------------------------------
@enceladus.jit
def histogram_kernel(x_ptr, hist_ptr, n, lo, inv_width, NUM_BINS: tl.constexpr, BLOCK: tl.constexpr):
    """hist[floor((float(x) - lo) * inv_width)] += 1 for every in-range element."""


def histogram(x, num_bins: int, lo: float, hi: float, block: int = 1024):
    """Returns the `int32` counts of `x` in `num_bins` equal bins over `[lo, hi)`."""
    hist = enceladus.new_zeros(x, (num_bins,), np.int32)
    n = int(np.prod(x.shape))
    histogram_kernel[(enceladus.cdiv(n, block),)](x, hist, n, float(lo), num_bins / (hi - lo),
                                                  NUM_BINS=num_bins, BLOCK=block)
    return hist


# ---- 10 cumsum ---------------------------------------------------------------------------------
@enceladus.jit
def cumsum_kernel(out_ptr, in_ptr, n_rows, n_cols, stride_in, stride_out, REVERSE: tl.constexpr,
                  BLOCK_M: tl.constexpr, BLOCK_N: tl.constexpr):
    """Inclusive scan of each row (suffix sums when REVERSE); narrow integers sum in int32."""


def cumsum(x, reverse: bool = False):
    """Returns the cumulative sum of each row of a 2D array, or of a 1D array of any length.

    Integers narrower than 32 bits sum in `int32`; int32 sums wrap modulo 2**32.
    """
    flat = len(x.shape) == 1
    m, n = (1, x.shape[0]) if flat else x.shape
    dt = enceladus.element_dtype(x)
    out = enceladus.new_empty(x, dtype=np.int32 if dt.kind in "iub" and dt.itemsize < 4 else dt)
    block_n = enceladus.next_power_of_2(n)
    block_m = max(1, min(16, 4096 // block_n))
    si = n if flat else enceladus.element_strides(x)[0]
    so = n if flat else enceladus.element_strides(out)[0]
    cumsum_kernel[(enceladus.cdiv(m, block_m),)](out, x, m, n, si, so, REVERSE=reverse, BLOCK_M=block_m,
                                                 BLOCK_N=block_n)
    return out


# ---- the decoding step: paged key-value cache, attention of one new token, logits -----------------------
# A step runs once per generated token and its kernels can be as short as a few microseconds.  So a call on torch tensors tries
# the short way first (runtime/lane.py), which takes every valid call on the current device; what it does not take (NumPy arrays,
# another device, a forced variant, empty or wrong arguments) is checked here and goes through `kernel[grid](...)`.
def _strides(x):
    """Strides in elements."""
    try:
        return x.stride()
    except AttributeError:
        return enceladus.element_strides(x)


def _short(kernel, name: str, *args):
    """The result of a call that went the short way, or NotImplemented."""
    way = lane.get()
    if way is None or kernel.variant is not None or kernel.interpret is not None:
        return NotImplemented
    r = getattr(way, name)(*args)
    if type(r) is int:  # an enc_status: raises
        N.check(r)
    return r


def _no_overlap(x, st, what: str) -> None:
    """Refuses an output whose elements share memory (an expanded view), where writes would meet."""
    if 0 in st and any(n > 1 and s == 0 for n, s in zip(x.shape, st)):
        raise ValueError(f"{what} is written, so its elements can't share memory (a stride is 0)")


def _check_cache(k_cache, v_cache, block_table):
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must both have shape (pages, kv_heads, page_size, head_dim), but got "
                         f"{tuple(shape)} and {tuple(v_cache.shape)}")
    if len(block_table.shape) != 2:
        raise ValueError(f"block_table must have shape (sequences, pages per sequence), not {tuple(block_table.shape)}")
    ks, vs, ts = _strides(k_cache), _strides(v_cache), _strides(block_table)
    if ks[3] != 1 or vs[3] != 1 or ts[1] != 1:
        for x, st, what in ((k_cache, ks, "k_cache"), (v_cache, vs, "v_cache"), (block_table, ts, "block_table")):
            if x.shape[-1] > 1 and st[-1] != 1 and 0 not in x.shape:
                raise ValueError(f"the last dimension of {what} must be contiguous")
    return ks, vs, ts[0]


def _check_heads(x, what: str, rows: int, head_dim: int, heads: int | None = None):
    """Strides of a (rows, heads, head_dim) array with contiguous heads."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} must have shape ({rows}, {'heads' if heads is None else heads}, {head_dim}), not {tuple(shape)}")
    st = _strides(x)
    if st[2] != 1 and head_dim > 1 and 0 not in shape:
        raise ValueError(f"the last dimension of {what} must be contiguous")
    return st


def _check_row(x, what: str, n: int) -> None:
    shape = x.shape
    if len(shape) != 1 or shape[0] != n or (n > 1 and _strides(x)[0] != 1):
        raise ValueError(f"{what} must be contiguous with shape ({n},), not {tuple(shape)}")


@enceladus.jit
def append_kv_kernel(k_ptr, v_ptr, q_ptr, q_out_ptr, k_cache_ptr, v_cache_ptr, block_table_ptr, seq_ids_ptr, positions_ptr, cos_ptr,
                     sin_ptr, n_seqs, table_width, stride_table, n_pages, n_positions, stride_k_token, stride_k_head, stride_v_token,
                     stride_v_head, stride_q_token, stride_q_head, stride_o_token, stride_o_head, stride_cos, stride_kp, stride_kh,
                     stride_kt, stride_vp, stride_vh, stride_vt, Q_HEADS: tl.constexpr, KV_HEADS: tl.constexpr,
                     HEAD_DIM: tl.constexpr, ROT_DIM: tl.constexpr, PAGE_SIZE: tl.constexpr, INTERLEAVED: tl.constexpr):
    """One token per program: k and v go to row positions[t] % PAGE_SIZE of page block_table[seq_ids[t], positions[t] // PAGE_SIZE];
    the first ROT_DIM elements of every k and q head turn in pairs by cos / sin of the token's position, in float32."""


def append_kv(k, v, k_cache, v_cache, block_table, seq_ids, positions, cos=None, sin=None, q=None, q_out=None,
              interleaved: bool = False):
    """Appends one key and value per token to a paged cache, in place, and returns the rotated `q` (None without `q`).

    `k` and `v` have shape (tokens, kv_heads, head_dim), `q` (tokens, q_heads, head_dim); slices of one fused
    projection will do, only the heads' elements must be contiguous. The caches have shape (pages, kv_heads,
    page_size, head_dim) with any strides: a cache laid out token by token is passed as `cache.transpose(1, 2)`.
    Token `t` is token `positions[t]` of sequence `seq_ids[t]`, whose pages `block_table[seq_ids[t]]` lists; a
    negative `seq_ids[t]` marks padding, for which nothing is written. All index arrays are int32. Prompts and
    single tokens mix freely, but no two tokens of a call may be the same token of a sequence, nor two sequences
    write to one shared page.

    `cos` and `sin`, float32 of shape (positions, rot_dim / 2), turn the first `rot_dim` elements of each query and
    key head: elements `(i, i + rot_dim / 2)` together, or `(2i, 2i + 1)` when `interleaved`. Without them nothing
    turns. `q_out` may be `q`. A sequence, position or page out of range is skipped, and `synchronize()` raises
    `CudaError`.
    """
    r = _short(append_kv_kernel, "append_kv", k, v, k_cache, v_cache, block_table, seq_ids, positions, cos, sin, q, q_out, interleaved)
    if r is not NotImplemented:
        return r
    ks, vs, st = _check_cache(k_cache, v_cache, block_table)
    pages, kv_heads, page_size, d = k_cache.shape
    tokens = k.shape[0]
    k_st, v_st = _check_heads(k, "k", tokens, d, kv_heads), _check_heads(v, "v", tokens, d, kv_heads)
    _check_row(seq_ids, "seq_ids", tokens)
    _check_row(positions, "positions", tokens)
    _no_overlap(k_cache, ks, "k_cache")
    _no_overlap(v_cache, vs, "v_cache")
    q_st = o_st = (0, 0, 0)
    q_heads = 0
    if q is not None:
        q_st, q_heads = _check_heads(q, "q", tokens, d), q.shape[1]
        if q_out is None:
            q_out = enceladus.new_empty(q)
        o_st = _check_heads(q_out, "q_out", tokens, d, q_heads)
        _no_overlap(q_out, o_st, "q_out")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    n_positions = rot_dim = cos_st = 0
    if cos is not None:
        shape = cos.shape
        if len(shape) != 2 or shape != sin.shape or 2 * shape[1] > d:
            raise ValueError(f"cos and sin must both have shape (positions, rot_dim / 2) with rot_dim <= {d}, but got "
                             f"{tuple(cos.shape)} and {tuple(sin.shape)}")
        c = _strides(cos)
        if c != _strides(sin) or (shape[1] > 1 and c[1] != 1):
            raise ValueError("cos and sin must have the same strides and contiguous rows")
        n_positions, rot_dim, cos_st = shape[0], 2 * shape[1], c[0]
        if not rot_dim:
            cos = sin = None
    seqs, width = block_table.shape
    append_kv_kernel[(tokens,)](k, v, q, q_out, k_cache, v_cache, block_table, seq_ids, positions, cos, sin, seqs, width, st, pages,
                                n_positions, k_st[0], k_st[1], v_st[0], v_st[1], q_st[0], q_st[1],
                                o_st[0], o_st[1], cos_st, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], Q_HEADS=q_heads,
                                KV_HEADS=kv_heads, HEAD_DIM=d, ROT_DIM=rot_dim, PAGE_SIZE=page_size, INTERLEAVED=interleaved)
    return q_out


@enceladus.jit
def paged_attention_kernel(q_ptr, k_cache_ptr, v_cache_ptr, o_ptr, lse_ptr, block_table_ptr, seq_lens_ptr, sm_scale, window, table_width,
                           stride_table, n_pages, stride_qs, stride_qh, stride_os, stride_oh, stride_kp, stride_kh, stride_kt,
                           stride_vp, stride_vh, stride_vt, Q_HEADS: tl.constexpr, KV_HEADS: tl.constexpr, HEAD_DIM: tl.constexpr,
                           PAGE_SIZE: tl.constexpr):
    """softmax(q k^T * sm_scale) v of one query token per sequence over the sequence's keys in a paged cache: base-2 online
    softmax in float32, the probabilities not rounded; lse = ln2 * (m + log2 l)."""


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, sm_scale: float | None = None, window: int = 0, o=None,
                    return_lse: bool = False):
    """Returns `softmax(q @ k^T * sm_scale) @ v` for one new token per sequence over a paged cache, in the input dtype.

    `q` has shape (sequences, q_heads, head_dim), head_dim at most 256; the caches and `block_table` are those of
    `append_kv`, with `q_heads` a multiple of the cache's heads. Sequence `s` looks at its first `seq_lens[s]` (int32)
    tokens, or the last `window` of them when `window` is positive. `o` may be `q`. A sequence of length zero gives
    zeros, and so does a row whose weights are all zero. What the cache holds past a sequence's length or in front of its window doesn't
    matter; an infinite value among those that do can make its column NaN.

    With `return_lse=True`, also returns the float32 log-sum-exp of the scaled scores, shape (sequences, q_heads):
    -inf for a row without keys. A length or page out of range is cut or skipped, and `synchronize()` raises `CudaError`.
    """
    r = _short(paged_attention_kernel, "paged_attention", q, k_cache, v_cache, block_table, seq_lens, sm_scale, window, o, return_lse)
    if r is not NotImplemented:
        return r
    ks, vs, st = _check_cache(k_cache, v_cache, block_table)
    pages, kv_heads, page_size, d = k_cache.shape
    seqs = q.shape[0]
    q_st = _check_heads(q, "q", seqs, d)
    q_heads = q.shape[1]
    if kv_heads == 0 or q_heads == 0 or q_heads % kv_heads:
        raise ValueError(f"the query heads must be a multiple of the cache's heads, but got {q_heads} and {kv_heads}")
    if not 1 <= d <= 256:
        raise ValueError(f"head_dim must be from 1 to 256, not {d}")
    if block_table.shape[0] != seqs:
        raise ValueError(f"block_table has {block_table.shape[0]} rows, but q has {seqs}")
    _check_row(seq_lens, "seq_lens", seqs)
    if window < 0:
        raise ValueError(f"window can't be negative, but got {window}")
    if o is None:
        o = enceladus.new_empty(q)
    o_st = _check_heads(o, "o", seqs, d, q_heads)
    _no_overlap(o, o_st, "o")
    scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    lse = enceladus.new_empty(q, (seqs, q_heads), np.float32) if return_lse else None
    paged_attention_kernel[(seqs,)](q, k_cache, v_cache, o, lse, block_table, seq_lens, scale, window, block_table.shape[1], st, pages,
                                    q_st[0], q_st[1], o_st[0], o_st[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], Q_HEADS=q_heads,
                                    KV_HEADS=kv_heads, HEAD_DIM=d, PAGE_SIZE=page_size)
    return (o, lse) if return_lse else o


@enceladus.jit
def penalize_logits_kernel(logits_ptr, out_ptr, tokens_ptr, lens_ptr, prompt_lens_ptr, repetition_ptr, frequency_ptr, presence_ptr,
                           bias_ids_ptr, bias_values_ptr, mask_ptr, vocab, stride_in, stride_out, history, stride_tokens, n_biases,
                           stride_bias, stride_mask):
    """One row per program: penalties for the tokens of the row's history, biases, then -inf where the mask bit is clear."""


def penalize_logits(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
                    bias_ids=None, bias_values=None, mask=None, out=None):
    """Returns `logits` (rows, vocab) with penalties, biases and a grammar mask applied, in the input dtype.

    The first `lens[r]` of `tokens[r]` are row `r`'s history, the first `prompt_lens[r]` of them its prompt (int32).
    In this order, in float32: a logit whose token is in the history is divided by `repetition[r]` if positive and
    multiplied by it otherwise; one whose token was generated (is behind the prompt) `n > 0` times loses
    `frequency[r] * n + presence[r]`; `bias_values[r, i]` (float32) is added to token `bias_ids[r, i]` (int32; -1: an
    unused place; a token that occurs twice gets both); a token whose bit in `mask` is clear becomes -inf, whatever
    it was: bit `t % 32` of word `mask[r, t // 32]` (int32) is set for a token that is allowed. A row that allows
    nothing is -inf throughout.

    The history's arrays come together, the biases' too, and each part can be left out. `out` may be `logits`.
    A token, bias id or length out of range is ignored or cut, and `synchronize()` raises `CudaError`.
    """
    r = _short(penalize_logits_kernel, "penalize_logits", logits, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values,
               mask, out)
    if r is not NotImplemented:
        return r
    if len(logits.shape) != 2:
        raise ValueError(f"logits must have shape (rows, vocab), not {tuple(logits.shape)}")
    m, n = logits.shape

    def rows_of(x, what, cols=None):
        shape = x.shape
        if len(shape) != 2 or shape[0] != m or (cols is not None and shape[1] != cols):
            raise ValueError(f"{what} must have shape ({m}, {'...' if cols is None else cols}), not {tuple(shape)}")
        st = _strides(x)
        if st[1] != 1 and shape[1] > 1:
            raise ValueError(f"the rows of {what} must be contiguous")
        return st[0]

    si = rows_of(logits, "logits")
    past = (tokens, lens, prompt_lens, repetition, frequency, presence)
    history = stride_tokens = n_biases = stride_bias = stride_mask = 0
    if tokens is not None:
        if lens is None or prompt_lens is None or repetition is None or frequency is None or presence is None:
            raise ValueError("tokens, lens, prompt_lens, repetition, frequency and presence go together")
        stride_tokens, history = rows_of(tokens, "tokens"), tokens.shape[1]
        _check_row(lens, "lens", m)
        _check_row(prompt_lens, "prompt_lens", m)
        _check_row(repetition, "repetition", m)
        _check_row(frequency, "frequency", m)
        _check_row(presence, "presence", m)
    elif any(x is not None for x in past):
        raise ValueError("tokens, lens, prompt_lens, repetition, frequency and presence go together")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if bias_ids is not None:
        stride_bias, n_biases = rows_of(bias_ids, "bias_ids"), bias_ids.shape[1]
        if rows_of(bias_values, "bias_values", n_biases) != stride_bias and m > 1:
            raise ValueError("bias_ids and bias_values must have the same strides")
    if mask is not None:
        stride_mask = rows_of(mask, "mask", enceladus.cdiv(n, 32))
        if m == 1:  # the stride of a single row means nothing
            stride_mask = mask.shape[1]
    if out is None:
        out = enceladus.new_empty(logits)
    so = rows_of(out, "out", n)
    _no_overlap(out, (so,), "out")
    penalize_logits_kernel[(m,)](logits, out, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, mask,
                                 n, si, so, history, stride_tokens, n_biases, stride_bias, stride_mask)
    return out

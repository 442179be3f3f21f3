"""The decoding step's operators without a GPU: what the wrappers and the C ABI refuse before anything is launched."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from enceladus_b200 import _native as N
from enceladus_b200 import ops
from enceladus_b200.runtime import registry


@pytest.fixture(scope="module")
def lib():
    from enceladus_b200 import build

    build.build()
    return N.load()


def cache(**kw):
    c = dict(k=16, v=16, block_table=16, num_pages=4, page_size=16, kv_heads=2, head_dim=64, num_seqs=3, table_width=17, stride_table=17,
             k_stride_page=2048, k_stride_head=1024, k_stride_token=64, v_stride_page=2048, v_stride_head=1024, v_stride_token=64)
    c.update(kw)
    return N.paged_cache(*(c[n] or 0 for n in N.PAGED_CACHE_FIELDS))


def pack(what, fields, values):
    return what(*(values[n] or 0 for n in fields))


def append(lib, c, *, k=16, v=16, q=None, q_out=None, cos=None, sin=None, ids=16, pos=16, tokens=2, q_heads=0, rot=0, n_pos=0, dtype=N.F32,
           variant=-1):
    args = pack(N.append_args, N.APPEND_FIELDS, dict(
        k=k, v=v, q=q, q_out=q_out, cos=cos, sin=sin, seq_ids=ids, positions=pos, tokens=tokens, q_heads=q_heads, rot_dim=rot, interleaved=0,
        num_positions=n_pos, k_stride_token=128, k_stride_head=64, v_stride_token=128, v_stride_head=64, q_stride_token=256,
        q_stride_head=64, o_stride_token=256, o_stride_head=64, stride_cos=32))
    return lib.enc_append_kv(c, args, dtype, variant, None)


def attend(lib, c, *, q=16, o=16, lens=16, q_heads=4, window=0, work=None, nbytes=0, dtype=N.F32, variant=-1):
    args = pack(N.paged_attention_args, N.PAGED_ATTENTION_FIELDS, dict(
        q=q, o=o, lse=None, seq_lens=lens, work=work, work_bytes=nbytes, q_heads=q_heads, q_stride_seq=256, q_stride_head=64, o_stride_seq=256,
        o_stride_head=64, window=window, sm_scale=0.125))
    return lib.enc_paged_attention(c, args, dtype, variant, None)


def logits(lib, *, x=16, out=16, rows=2, vocab=100, past=(None,) * 6, history=0, ids=None, values=None, biases=0, mask=None, words=4,
           dtype=N.F32, variant=-1):
    args = pack(N.logits_args, N.LOGITS_FIELDS, dict(
        logits=x, out=out, **dict(zip(("tokens", "lens", "prompt_lens", "repetition", "frequency", "presence"), past)), bias_ids=ids,
        bias_values=values, mask=mask, rows=rows, vocab=vocab, stride_in=vocab, stride_out=vocab, history=history, stride_tokens=history,
        num_biases=biases, stride_bias=biases, stride_mask=words))
    return lib.enc_penalize_logits(args, dtype, variant, None)


def test_structs_match_the_header():
    import re

    text = (N.LIB_PATH.parents[2] / "include" / "enceladus_b200.h").read_text()
    assert ctypes.sizeof(ctypes.c_void_p) == 8
    for name, fields, size in (("enc_paged_cache", N.PAGED_CACHE_FIELDS, len(cache())), ("enc_append_args", N.APPEND_FIELDS, len(N.append_args(*[0] * 22))),
                               ("enc_paged_attention_args", N.PAGED_ATTENTION_FIELDS, len(N.paged_attention_args(*[0] * 13))),
                               ("enc_logits_args", N.LOGITS_FIELDS, len(N.logits_args(*[0] * 20)))):
        end = text.index("} " + name + ";")
        body = re.sub(r"/\*.*?\*/", "", text[text.rindex("typedef struct {", 0, end):end], flags=re.S)
        assert re.findall(r"\b\*?(\w+)\s*[,;]", body) == list(fields), name
        assert size == 8 * len(fields), name  # pointers, 64-bit integers and a double: no padding
    assert N.ERR_BAD_INDEX == 6 and "ENC_ERR_BAD_INDEX = 6" in text
    for name in ("APPEND_KV", "PAGED_ATTENTION", "LOGITS"):
        assert f"ENC_K_{name} = {getattr(N, 'K_' + name)}" in text


def test_append_refusals(lib):
    bad = N.ERR_BAD_ARG
    assert append(lib, None) == bad
    assert append(lib, cache(), dtype=N.I32) == bad
    assert append(lib, cache(), variant=99) == bad
    assert append(lib, cache(), k=None) == bad and append(lib, cache(), ids=None) == bad and append(lib, cache(), pos=None) == bad
    assert append(lib, cache(), q=16) == bad and "go together" in N.last_error()
    assert append(lib, cache(), rot=64) == bad and "without cos" in N.last_error()
    for rot in (-2, 3, 66):
        assert append(lib, cache(), rot=rot, cos=16, sin=16) == bad
    assert append(lib, cache(), tokens=-1) == bad
    for kw in (dict(page_size=0), dict(num_pages=-1), dict(kv_heads=0), dict(head_dim=0), dict(num_seqs=-1), dict(table_width=-1),
               dict(k=None), dict(block_table=None)):
        assert append(lib, cache(**kw)) == bad, kw
    for kw in (dict(page_size=2**31), dict(num_pages=2**31), dict(table_width=2**31), dict(head_dim=2**16)):
        assert append(lib, cache(**kw)) == N.ERR_UNSUPPORTED, kw
    assert append(lib, cache(), tokens=2**31) == N.ERR_UNSUPPORTED
    assert append(lib, cache(), tokens=0) == N.OK
    lib.enc_test_fail_next(N.ERR_LAUNCH)
    assert append(lib, cache(), tokens=0) == N.ERR_LAUNCH


def test_attention_refusals(lib):
    bad = N.ERR_BAD_ARG
    assert attend(lib, None) == bad
    assert attend(lib, cache(), dtype=N.I8) == bad
    assert attend(lib, cache(), variant=99) == bad
    assert attend(lib, cache(), q_heads=3) == bad and attend(lib, cache(), q_heads=0) == bad
    assert attend(lib, cache(), window=-1) == bad
    assert attend(lib, cache(), q=None) == bad and attend(lib, cache(), o=None) == bad and attend(lib, cache(), lens=None) == bad
    assert attend(lib, cache(head_dim=257)) == N.ERR_UNSUPPORTED
    assert attend(lib, cache(head_dim=0)) == bad
    assert attend(lib, cache(num_seqs=0), q=None) == N.OK
    size = lib.enc_paged_attention_work_bytes(cache(), 4, N.F32, -1)
    # the answer depends on the GPU's size; without one the library assumes a B200
    assert size > 0
    assert attend(lib, cache(), work=16, nbytes=size - 1) == bad and "workspace" in N.last_error()
    assert attend(lib, cache(), work=8, nbytes=size) == bad
    assert lib.enc_paged_attention_work_bytes(cache(table_width=4), 4, N.F32, -1) == 0  # a tile per row: nothing is cut
    assert lib.enc_paged_attention_work_bytes(None, 4, N.F32, -1) == -1
    assert lib.enc_paged_attention_work_bytes(cache(), 3, N.F32, -1) == -1


def test_logits_refusals(lib):
    bad = N.ERR_BAD_ARG
    assert logits(lib, dtype=N.I32) == bad
    assert logits(lib, variant=99) == bad
    assert logits(lib, rows=-1) == bad and logits(lib, vocab=-1) == bad
    assert logits(lib, x=None) == bad and logits(lib, out=None) == bad
    assert logits(lib, past=(16, 16, 16, 16, 16, None), history=4) == bad and "come together" in N.last_error()
    assert logits(lib, biases=3) == bad and logits(lib, biases=3, ids=16) == bad
    assert logits(lib, mask=16, words=3) == bad and "do not cover" in N.last_error()
    assert logits(lib, rows=65536) == N.ERR_UNSUPPORTED
    assert logits(lib, rows=0) == N.OK and logits(lib, vocab=0) == N.OK


def test_variants_are_described(lib):
    for k in (N.K_APPEND_KV, N.K_PAGED_ATTENTION, N.K_LOGITS):
        assert N.num_variants(k) >= 1 and all(N.variant_info(k, v) for v in range(N.num_variants(k)))


def test_registry_and_definitions_agree():
    for name in ("append_kv_kernel", "paged_attention_kernel", "penalize_logits_kernel"):
        k = getattr(ops, name)
        assert registry.lookup(name, tuple(k.arg_names)).name == name


def arrays():
    f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    i = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    return f, i


def test_append_wrapper_refusals():
    f, i = arrays()
    good = dict(k=f(3, 2, 64), v=f(3, 2, 64), k_cache=f(4, 2, 16, 64), v_cache=f(4, 2, 16, 64), block_table=i(2, 4), seq_ids=i(3), positions=i(3))
    for change, match in ((dict(k=f(3, 2, 32)), "k must have shape"), (dict(v=f(2, 2, 64)), "v must have shape"), (dict(k=f(3, 1, 64)), "k must have shape"),
                          (dict(v_cache=f(4, 2, 16, 32)), "both have shape"), (dict(k_cache=f(4, 2, 16), v_cache=f(4, 2, 16)), "both have shape"),
                          (dict(block_table=i(2)), "block_table must have shape"), (dict(block_table=i(4, 2).T), "contiguous"),
                          (dict(k_cache=f(4, 2, 64, 16).swapaxes(2, 3)), "contiguous"), (dict(k=f(3, 64, 2).swapaxes(1, 2)), "contiguous"),
                          (dict(seq_ids=i(2)), "seq_ids must"), (dict(positions=i(6)[::2]), "positions must"),
                          (dict(q_out=f(3, 4, 64)), "q_out without q"), (dict(q=f(3, 4, 32)), "q must have"), (dict(q=f(3, 4, 64), q_out=f(3, 2, 64)), "q_out must"),
                          (dict(cos=f(9, 32)), "go together"), (dict(cos=f(9, 33), sin=f(9, 33)), "rot_dim <= 64"), (dict(cos=f(9, 32), sin=f(8, 32)), "cos and sin"),
                          (dict(cos=f(9, 32), sin=f(9, 64)[:, ::2]), "same strides"),
                          (dict(k_cache=np.broadcast_to(f(1, 2, 16, 64), (4, 2, 16, 64))), "share memory")):
        with pytest.raises(ValueError, match=match):
            ops.append_kv(**{**good, **change})
    with pytest.raises(TypeError, match="`positions_ptr` must be"):
        registry._need(torch.int32, positions_ptr=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError, match="share one element type"):
        registry._float_code("x", k_ptr=torch.zeros(1), v_ptr=torch.zeros(1, dtype=torch.float16))
    with pytest.raises(TypeError, match="share one element type"):
        registry._float_code("x", k_ptr=torch.zeros(1, dtype=torch.float64))


def test_attention_wrapper_refusals():
    f, i = arrays()
    good = dict(q=f(2, 4, 64), k_cache=f(4, 2, 16, 64), v_cache=f(4, 2, 16, 64), block_table=i(2, 4), seq_lens=i(2))
    for change, match in ((dict(q=f(2, 3, 64)), "multiple"), (dict(q=f(2, 4, 32)), "q must have shape"), (dict(q=f(2, 0, 64)), "multiple"),
                          (dict(block_table=i(3, 4)), "block_table has 3 rows"), (dict(seq_lens=i(3)), "seq_lens must"), (dict(window=-1), "window"),
                          (dict(o=f(2, 4, 32)), "o must have shape"), (dict(q=f(2, 64, 4).swapaxes(1, 2)), "contiguous"),
                          (dict(o=np.broadcast_to(f(1, 4, 64), (2, 4, 64))), "share memory"),
                          (dict(q=f(2, 4, 300), k_cache=f(4, 2, 16, 300), v_cache=f(4, 2, 16, 300)), "from 1 to 256"),
                          (dict(k_cache=f(4, 0, 16, 64), v_cache=f(4, 0, 16, 64)), "multiple")):
        with pytest.raises(ValueError, match=match):
            ops.paged_attention(**{**good, **change})


def test_logits_wrapper_refusals():
    f, i = arrays()
    past = dict(tokens=i(2, 9), lens=i(2), prompt_lens=i(2), repetition=f(2), frequency=f(2), presence=f(2))
    for change, match in ((dict(logits=f(100)), "logits must have shape"), (dict(logits=f(100, 2).T), "contiguous"), (dict(tokens=i(2, 9)), "go together"),
                          (dict(**{**past, "lens": i(3)}), "lens must"), (dict(**{**past, "tokens": i(3, 9)}), "tokens must"),
                          (dict(bias_ids=i(2, 3)), "go together"), (dict(bias_ids=i(2, 3), bias_values=f(2, 4)), "bias_values must"),
                          (dict(mask=i(2, 3)), "mask must"), (dict(mask=i(1, 4)), "mask must"), (dict(out=f(2, 99)), "out must"),
                          (dict(out=np.broadcast_to(f(1, 100), (2, 100))), "share memory")):
        with pytest.raises(ValueError, match=match):
            ops.penalize_logits(**{"logits": f(2, 100), **change})


def test_missing_arrays_are_refused_unless_optional(monkeypatch):
    """None stands only for the arrays that a kernel can go without."""
    from enceladus_b200.runtime import jit

    ad = registry.lookup("penalize_logits_kernel", tuple(ops.penalize_logits_kernel.arg_names))
    bound = {p: None for p in ad.params}
    with pytest.raises(TypeError, match="`logits_ptr` must be"):
        jit.launch(ad, bound, (1, 1, 1), -1, None)
    assert ad.optional == frozenset(ad.array_list) - {"logits_ptr", "out_ptr"}
    soft = registry.lookup("softmax_kernel", tuple(ops.softmax_kernel.arg_names))
    assert not soft.optional


def test_explain_names_the_entry_point_and_leaves_out_what_is_absent(lib, capsys):
    f, _ = arrays()
    x = f(2, 100)
    text = ops.penalize_logits_kernel.explain(x, x, *[None] * 9, 100, 100, 100, 0, 0, 0, 0, 0, grid=(2,))
    assert "enc_penalize_logits" in text and "logits_ptr" in text and "mask_ptr" not in text
    assert "enc_paged_attention" in jit_entry("paged_attention_kernel") and "enc_append_kv" in jit_entry("append_kv_kernel")


def jit_entry(name):
    from enceladus_b200.runtime import jit

    return jit._ENTRY_POINTS[getattr(ops, name).adapter().kernel_id]

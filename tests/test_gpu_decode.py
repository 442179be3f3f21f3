"""The operators of a decoding step against plain implementations in 64 bits.

Tolerances are derived, not tuned: an output may be off by half a step of its type (`half_step`) plus what float32
arithmetic on the way can lose, which each check writes out as a multiple of U = 2^-24 (one float32 rounding) times the sum of
the magnitudes that were added.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

import enceladus_b200 as enceladus
from enceladus_b200 import _native as N
from enceladus_b200 import ops

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24
TINY = {F16: 2.0**-25, BF16: 0.0, F32: 0.0}  # half of fp16's smallest step: its subnormals are in reach of these values


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(got, want, bound):
    """|got - want| <= bound elementwise, with the non-finite values in the same places."""
    got = got.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = (got - want).abs()[fine] - bound.expand_as(want)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"off by {float(over.max()):.3e} more than the bound"


# ---- cache -------------------------------------------------------------------------------------------------------
def make_cache(g, pages, heads, page, dim, dtype, layout="nhd", fill=None):
    shape = (pages, page, heads, dim) if layout == "nhd" else (pages, heads, page, dim)
    t = randn(g, *shape, dtype=dtype) if fill is None else torch.full(shape, fill, device="cuda", dtype=dtype)
    return t.transpose(1, 2) if layout == "nhd" else t


def tables(n, rot):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * freq
    return a.cos().float(), a.sin().float()


def rotate64(x, cos, sin, rot, interleaved):
    """The rotation in 64 bits, and the sum of the magnitudes that each element adds."""
    x = x.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2 : rot])
    want, size = x.clone(), x.abs()
    ia, ib = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    want[..., ia], want[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = (a * c).abs() + (b * s).abs()
    size[..., ib] = (b * c).abs() + (a * s).abs()
    return want, size


def check_append(dtype, seq_list, *, page=16, heads=(8, 2), dim=64, rot=64, interleaved=False, layout="nhd", pad=0, offset=0, seed=0,
                 inplace=False):
    """Appends tokens (sequence, position) of `seq_list` plus padding and checks q_out and every place of both caches."""
    g = gen(seed)
    hq, hk = heads
    width = max(p for _, p in seq_list) // page + 1
    seqs = max(s for s, _ in seq_list) + 1
    used = sorted({(s, p // page) for s, p in seq_list})
    pages = len(used) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((seqs, width), -7, dtype=torch.int32)
    for i, (s, p) in enumerate(used):
        table[s, p] = order[i]
    kc, vc = make_cache(g, pages, hk, page, dim, dtype, layout), make_cache(g, pages, hk, page, dim, dtype, layout)
    n = len(seq_list) + pad
    fused = randn(g, n, offset + (hq + 2 * hk) * dim, dtype=dtype)[:, offset:]  # `offset` elements before q: another alignment
    q, k, v = (x.unflatten(1, (-1, dim)) for x in fused.split([hq * dim, hk * dim, hk * dim], 1))
    order2 = torch.randperm(n, generator=torch.Generator().manual_seed(seed + 1)).tolist()
    tok = [(seq_list + [(-1, 123456)] * pad)[i] for i in order2]
    ids, pos = ints([s for s, _ in tok]), ints([p for _, p in tok])
    cos, sin = tables(width * page, rot) if rot else (None, None)
    q_before, kc_before, vc_before = q.clone(), kc.clone(), vc.clone()
    q_out = q if inplace else randn(g, n, hq, dim, dtype=dtype)
    out_before = q_out.clone()
    got = ops.append_kv(k, v, kc, vc, table.cuda(), ids, pos, cos=cos, sin=sin, q=q, q_out=q_out, interleaved=interleaved)
    assert got is q_out
    enceladus.synchronize()
    live = torch.tensor([s >= 0 for s, _ in tok], device="cuda")
    place = pos[live].long()
    if rot:
        rows = lambda x: rotate64(x[live], cos[place], sin[place], rot, interleaved)  # noqa: E731
    else:
        rows = lambda x: (x[live].double(), x[live].double().abs())  # noqa: E731
    qw, qs = rows(q_before)
    # a product and a fused multiply-add (2 roundings of what is added), then the store's rounding
    bound = lambda w, s: (half_step(dtype) * w.abs() + 3 * U * s + TINY[dtype]) * (1 + 1e-6)  # noqa: E731
    within(q_out[live], qw, bound(qw, qs))
    assert torch.equal(q_out[~live], out_before[~live])
    kw, ksz = rows(k)
    want_k, want_v, size = kc_before.double(), vc_before.double(), torch.zeros_like(kc_before, dtype=torch.float64)
    for i, (s, p) in enumerate([t for t in tok if t[0] >= 0]):
        at = int(table[s, p // page])
        want_k[at, :, p % page], size[at, :, p % page] = kw[i], ksz[i]
        want_v[at, :, p % page] = v[live][i].double()
    touched = size.abs().sum(-1, keepdim=True) > 0
    within(kc, want_k, torch.where(touched, bound(want_k, size), 0.0))
    within(vc, want_v, torch.zeros_like(want_v))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_append_ragged_prompts(dtype, interleaved, layout):
    tokens = [(0, p) for p in range(37)] + [(1, p) for p in range(5, 6)] + [(2, p) for p in range(100, 133)]
    check_append(dtype, tokens, interleaved=interleaved, layout=layout, pad=3, page=16)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("dim,rot,offset,page", [(128, 128, 0, 64), (128, 32, 0, 1), (64, 16, 8, 24), (80, 80, 0, 16), (96, 50, 0, 16), (33, 32, 1, 5),
                                                 (64, 64, 3, 16), (256, 256, 0, 16), (1, 0, 0, 16), (128, 0, 0, 16), (300, 300, 0, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_sizes_and_alignments(dtype, dim, rot, offset, page, interleaved):
    check_append(dtype, [(0, 0), (0, 1), (1, 70), (3, page), (3, page + 1)], dim=dim, rot=rot, offset=offset, page=page, interleaved=interleaved, seed=dim)


@pytest.mark.parametrize("heads", [(1, 1), (32, 8), (7, 7), (71, 1), (5, 5)])
def test_append_heads(heads):
    check_append(BF16, [(i, 3 * i) for i in range(9)], heads=heads, dim=128, rot=128, pad=2)


def test_append_far_positions():
    check_append(BF16, [(0, 1_000_000), (1, 131_071), (1, 131_072)], page=128, dim=128, rot=128)


def test_append_in_place_and_without_queries():
    check_append(F16, [(0, p) for p in range(20)], inplace=True, pad=2)
    g = gen(1)
    kc, vc = make_cache(g, 2, 3, 16, 64, F16), make_cache(g, 2, 3, 16, 64, F16)
    k, v = randn(g, 4, 3, 64, dtype=F16), randn(g, 4, 3, 64, dtype=F16)
    assert ops.append_kv(k, v, kc, vc, ints([[1]]), ints([0, 0, -1, 0]), ints([0, 5, 2, 15])) is None
    enceladus.synchronize()
    for i, p in ((0, 0), (1, 5), (3, 15)):
        assert torch.equal(kc[1, :, p], k[i]) and torch.equal(vc[1, :, p], v[i])


def test_append_out_of_range_is_skipped_and_reported():
    g = gen(2)
    kc, vc = make_cache(g, 4, 2, 16, 64, BF16), make_cache(g, 4, 2, 16, 64, BF16)
    k, v, q = randn(g, 1, 2, 64, dtype=BF16), randn(g, 1, 2, 64, dtype=BF16), randn(g, 1, 4, 64, dtype=BF16)
    cos, sin = tables(40, 64)
    k0, v0 = kc.clone(), vc.clone()
    table = ints([[0, 1, 4, 2**31 - 1], [2, -1, 0, -2**31]])
    for seq, pos in ((2, 0), (2**31 - 1, 0), (0, -1), (0, -2**31), (0, 64), (0, 2**31 - 1), (0, 32), (0, 48), (1, 16), (1, 48), (1, 41)):
        ops.append_kv(k, v, kc, vc, table, ints([seq]), ints([pos]), cos=cos, sin=sin, q=q)
        with pytest.raises(enceladus.CudaError, match="out of range") as e:
            enceladus.synchronize()
        assert e.value.status == N.ERR_BAD_INDEX
        assert torch.equal(kc, k0) and torch.equal(vc, v0), (seq, pos)
    enceladus.synchronize()  # reported once
    ops.append_kv(k, v, kc, vc, table, ints([-5]), ints([2**31 - 1]), cos=cos, sin=sin, q=q)
    enceladus.synchronize()
    assert torch.equal(kc, k0)


# ---- attention -----------------------------------------------------------------------------------------------------
def attend64(q, kc, vc, table, lens, scale, window):
    """o, lse in 64 bits, and two bounds: on the float32 error of o before it is rounded, and on that of lse.

    A score is a sum of D products: (D + 3) U of the sum of their magnitudes, in bits (base 2).  A weight 2^x is off by that
    times ln 2, by ex2.approx (2^-22), by the rounding of x (U |x|, and |x| below the scores' spread), by the split of a
    weight into two 16-bit parts (2^-16) and by the factors 2^(m - m') of rescaling and joining (a few 2^-22 each, at most one
    per key or piece).  Sums over n keys add n U."""
    b, hq, d = q.shape
    hk, page = kc.shape[1], kc.shape[2]
    o = torch.zeros(b, hq, d, device="cuda", dtype=torch.float64)
    lse = torch.full((b, hq), -math.inf, device="cuda", dtype=torch.float64)
    eo, el = torch.zeros_like(o), torch.zeros(b, hq, device="cuda", dtype=torch.float64)
    for i, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        pg = table[i, : -(-n // page)].long()
        for h in range(hk):
            k = kc[pg, h].reshape(-1, d)[lo:n].double()
            v = vc[pg, h].reshape(-1, d)[lo:n].double()
            rows = slice(h * hq // hk, (h + 1) * hq // hk)
            s = q[i, rows].double() @ k.T * scale
            size = (q[i, rows].double().abs() @ k.abs().T * abs(scale)).amax(1, keepdim=True)  # magnitudes: the scale's sign is no part
            top = s.amax(1, keepdim=True)
            p = (s - top).exp()
            total = p.sum(1, keepdim=True)
            w = p / total
            o[i, rows] = w @ v
            lse[i, rows] = (top + total.log())[:, 0]
            es = (d + 3) * U * size + U * ((top - s.amin(1, keepdim=True)) + s.abs().amax(1, keepdim=True)) * 2
            rel = es + 40 * 2.0**-22 + 2.0**-16 + (n - lo + 8) * U
            eo[i, rows] = 2 * rel * (w @ v.abs())
            el[i, rows] = (es + 40 * 2.0**-22 + (n - lo + 8) * U + 4 * U * lse[i, rows, None].abs())[:, 0]
    return o, lse, eo, el


def make_attention(dtype, lens, *, heads=(8, 2), dim=64, page=16, layout="nhd", seed=0, spread=1.0, garbage=math.nan, extra=1):
    """q, caches and table: every place that no sequence owns holds `garbage`, unused table entries are out of range."""
    g = gen(seed)
    hq, hk = heads
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need) + extra), 2**31 - 1, dtype=torch.int32)
    kc, vc = make_cache(g, pages, hk, page, dim, dtype, layout, garbage), make_cache(g, pages, hk, page, dim, dtype, layout, garbage)
    at = 0
    for i, n in enumerate(lens):
        for j in range(need[i]):
            pg = order[at]
            table[i, j] = pg
            m = min(page, n - j * page)
            kc[pg, :, :m] = randn(g, hk, m, dim, dtype=dtype) * spread
            vc[pg, :, :m] = randn(g, hk, m, dim, dtype=dtype)
            at += 1
    return randn(g, len(lens), hq, dim, dtype=dtype), kc, vc, table.cuda()


def check_attention(dtype, lens, *, window=0, scale=None, variants=True, **kw):
    q, kc, vc, table = make_attention(dtype, lens, **kw)
    d = q.shape[-1]
    o64, lse64, eo, el = attend64(q, kc, vc, table, lens, d**-0.5 if scale is None else scale, window)
    bound = half_step(dtype) * o64.abs() * (1 + 1e-6) + eo * 1.01 + TINY[dtype]
    o, lse = ops.paged_attention(q, kc, vc, table, ints(lens), sm_scale=scale, window=window, return_lse=True)
    enceladus.synchronize()
    within(o, o64, bound)
    within(lse, lse64, el)
    if not variants:
        return
    for variant in range(N.num_variants(N.K_PAGED_ATTENTION)):
        ops.paged_attention_kernel.variant = variant
        try:
            o2, lse2 = ops.paged_attention(q, kc, vc, table, ints(lens), sm_scale=scale, window=window, return_lse=True)
        except NotImplementedError:
            continue
        finally:
            ops.paged_attention_kernel.variant = None
        enceladus.synchronize()
        within(o2, o64, bound)
        within(lse2, lse64, el)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [64], [65], [1, 0, 63, 64, 65, 127, 0], [1000, 1, 257], [16, 32, 48]], ids=str)
def test_attention_lengths(dtype, lens):
    check_attention(dtype, lens, dim=128)
    check_attention(dtype, lens, dim=64, page=64, layout="hnd")


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("heads", [(1, 1), (2, 1), (3, 3), (5, 1), (12, 4), (16, 1), (17, 1), (33, 1), (14, 2), (32, 8), (71, 1)], ids=str)
def test_attention_head_groups(dtype, heads):
    check_attention(dtype, [130, 0, 1, 700], heads=heads, dim=128, seed=heads[0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("dim", [1, 7, 16, 20, 32, 48, 64, 80, 96, 112, 128, 160, 192, 200, 256])
def test_attention_head_dims(dtype, dim):
    check_attention(dtype, [300, 17], dim=dim, heads=(6, 2), seed=dim)


@pytest.mark.parametrize("page", [1, 2, 5, 16, 24, 31, 64, 100, 256])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_attention_page_sizes(page, layout):
    check_attention(BF16, [333, 100, 1, 0, 99, 257], page=page, layout=layout, dim=128, seed=page)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 100, 1000, 2**31 - 1, 2**40])
def test_attention_windows(dtype, window):
    check_attention(dtype, [0, 1, 64, 65, 163, 164, 165, 900, 1500], window=window, dim=64, page=24, variants=window == 100)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("page", [16, 24])
def test_attention_what_lies_in_front_of_the_window_is_not_read(dtype, page):
    """Pages that the window has left are gone from the table, and keys in front of it on its first page are NaN."""
    lens, window = [500, 77, 16 * 20, 65], 70
    for dim in (64, 128):
        q, kc, vc, table = make_attention(dtype, lens, dim=dim, page=page, seed=dim)
        o64, lse64, eo, el = attend64(q, kc, vc, table, lens, dim**-0.5, window)
        for i, n in enumerate(lens):
            lo = max(0, n - window)
            at = int(table[i, lo // page])
            kc[at, :, : lo % page] = math.nan
            vc[at, :, : lo % page] = math.inf
            table[i, : lo // page] = -1
        o, lse = ops.paged_attention(q, kc, vc, table, ints(lens), window=window, return_lse=True)
        enceladus.synchronize()
        within(o, o64, half_step(dtype) * o64.abs() * (1 + 1e-6) + eo * 1.01 + TINY[dtype])
        within(lse, lse64, el)


def test_attention_over_an_empty_cache():
    """No pages, or no columns: rows without keys are zero; a length that nothing can hold is cut and reported."""
    for dtype in (BF16, F32):
        q = randn(gen(8), 2, 4, 64, dtype=dtype)
        for pages, columns in ((0, 3), (2, 0), (0, 0)):
            kc = torch.zeros(pages, 2, 16, 64, device="cuda", dtype=dtype)
            table = torch.zeros(2, columns, device="cuda", dtype=torch.int32)
            o, lse = ops.paged_attention(q, kc, kc.clone(), table, ints([0, 0]), return_lse=True)
            enceladus.synchronize()
            assert not o.any() and (lse == -math.inf).all()
            ops.paged_attention(q, kc, kc.clone(), table, ints([0, 5]))
            with pytest.raises(enceladus.CudaError, match="out of range"):
                enceladus.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_long_rows_are_split(dtype):
    check_attention(dtype, [40_000], heads=(8, 1), dim=128, page=64, garbage=0.0)
    check_attention(dtype, [20_000, 3, 0, 9_999], heads=(4, 4), dim=64, page=32, garbage=0.0)


def test_attention_many_sequences():
    r = np.random.default_rng(0)
    lens = [int(x) for x in r.integers(0, 150, 700)]
    check_attention(BF16, lens, heads=(4, 2), dim=64, page=16, variants=False, garbage=0.0)


@pytest.mark.parametrize("columns", [200, 900])
@pytest.mark.parametrize("longest", [0, 1, 40, 3000])
def test_attention_wide_tables(columns, longest):
    """Tables far wider than the lengths need: the grid is sized for rows that the lengths do not fill."""
    r = np.random.default_rng(columns + longest)
    lens = [int(x) for x in r.integers(0, longest + 1, 170)]
    for dim, heads in ((64, (6, 3)), (128, (4, 4))):
        check_attention(BF16, lens, heads=heads, dim=dim, page=16, variants=False, garbage=0.0, extra=columns, seed=longest)


def test_attention_many_long_rows():
    r = np.random.default_rng(1)
    lens = [int(x) for x in r.integers(1, 6000, 100)]
    check_attention(F16, lens, heads=(8, 8), dim=64, page=32, variants=False, garbage=0.0, extra=200, window=4000)
    check_attention(BF16, lens, heads=(36, 4), dim=64, page=24, variants=False, garbage=0.0, extra=200)


def test_attention_large_launches_side_by_side():
    """Launches large enough to claim runs from one another's blocks, on three streams at once and captured: the same bits."""
    r = np.random.default_rng(2)
    lens = [int(x) for x in r.integers(0, 3000, 160)]
    q, kc, vc, table = make_attention(BF16, lens, heads=(16, 4), dim=64, page=16, garbage=0.0, extra=300)
    n = ints(lens)
    first = ops.paged_attention(q, kc, vc, table, n)
    o64, _, eo, _ = attend64(q, kc, vc, table, lens, 0.125, 0)
    within(first, o64, half_step(BF16) * o64.abs() * (1 + 1e-6) + eo * 1.01)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.paged_attention(q, kc, vc, table, n)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(18):
        with torch.cuda.stream(streams[i % 3]):
            if i % 3 == 2:
                graph.replay()
            else:
                got.append(ops.paged_attention(q, kc, vc, table, n))
    torch.cuda.synchronize()
    assert torch.equal(first, captured) and all(torch.equal(first, x) for x in got)
    enceladus.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_attention_growing_scores(dtype):
    """Scores spread over many powers of two, so that the running maximum moves and most weights are tiny."""
    check_attention(dtype, [700, 64], dim=128, spread=6.0)
    check_attention(dtype, [700, 64], dim=128, scale=-0.5)
    check_attention(dtype, [700, 64], dim=128, scale=0.0)


def test_attention_small_weights_count_in_fp16():
    """One key far above 20000 others of weight 2^-13 each: together they outweigh it."""
    n, d = 20_001, 64
    q = torch.zeros(1, 1, d, device="cuda", dtype=F16)
    q[..., 0] = 1
    kc = torch.zeros(1, 1, n, d, device="cuda", dtype=F16)
    vc = torch.zeros_like(kc)
    kc[0, 0, 0, 0] = 13 * math.log(2)
    vc[0, 0, 1:, 1] = 1
    vc[0, 0, 0, 2] = 1
    table, lens = ints([[0]]), [n]
    o64, lse64, eo, el = attend64(q, kc, vc, table, lens, 1.0, 0)
    for cut in (1.0, 2.0):  # at 2.0 the others weigh 2^-26 each
        o64, lse64, eo, el = attend64(q, kc, vc, table, lens, cut, 0)
        o, lse = ops.paged_attention(q, kc, vc, table, ints(lens), sm_scale=cut, return_lse=True)
        within(o, o64, half_step(F16) * o64.abs() * (1 + 1e-6) + eo * 1.01 + TINY[F16])
        within(lse, lse64, el)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_attention_infinities(dtype):
    """Keys that score -inf weigh nothing; a row of only such keys is zero with lse -inf; NaN stays in its row."""
    g = gen(3)
    n, d = 200, 64
    kc, vc = randn(g, 1, 2, n, d, dtype=dtype), randn(g, 1, 2, n, d, dtype=dtype)
    q = randn(g, 1, 2, d, dtype=dtype)
    q[..., 0] = 1
    kc[0, 0, ::2, 0] = -math.inf
    kc[0, 1, :, 0] = -math.inf
    args = (ints([[0]]), ints([n]))
    o, lse = ops.paged_attention(q, kc, vc, *args, return_lse=True)
    some = torch.arange(1, n, 2, device="cuda")
    k2, v2 = kc[:, :1, some].contiguous(), vc[:, :1, some].contiguous()
    o64, lse64, eo, el = attend64(q[:, :1], k2, v2, args[0], [len(some)], d**-0.5, 0)
    within(o[:, :1], o64, half_step(dtype) * o64.abs() * (1 + 1e-6) + eo * 1.01 + TINY[dtype])
    within(lse[:, :1], lse64, el)
    assert not o[0, 1].any() and float(lse[0, 1]) == -math.inf
    q[0, 0, 3] = math.nan
    o, lse = ops.paged_attention(q, kc, vc, *args, return_lse=True)
    assert torch.isnan(o[0, 0]).all() and torch.isnan(lse[0, 0]) and not o[0, 1].any()


def test_attention_strided_arguments():
    """q and o as slices of larger arrays, a table with a row stride, caches inside one [2, ...] pool, odd strides."""
    g = gen(4)
    lens = [90, 33]
    for dtype, dim, pad in ((BF16, 64, 0), (BF16, 64, 3), (F32, 64, 1)):
        pool = randn(g, 8, 2, 16, 3, dim + pad, dtype=dtype)[..., :dim]
        kc, vc = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
        table = torch.randperm(8, device="cuda", generator=g, dtype=torch.int32).repeat(2).reshape(2, 8)[:, :7]
        qkv = randn(g, 2, 12 * (dim + pad), dtype=dtype).unflatten(1, (12, dim + pad))[..., :dim]
        q = qkv[:, 2:8]
        out = torch.full((2, 9, dim), 7.0, device="cuda", dtype=dtype)
        o64, _, eo, _ = attend64(q, kc, vc, table, lens, dim**-0.5, 0)
        ops.paged_attention(q, kc, vc, table, ints(lens), o=out[:, 3:])
        within(out[:, 3:], o64, half_step(dtype) * o64.abs() * (1 + 1e-6) + eo * 1.01)
        assert (out[:, :3] == 7.0).all()
    shared = ints([[0, 1]]).expand(3, 2)  # every sequence on the same pages
    kc, vc, q = randn(g, 2, 2, 16, 64, dtype=BF16), randn(g, 2, 2, 16, 64, dtype=BF16), randn(g, 3, 2, 64, dtype=BF16)
    o64, _, eo, _ = attend64(q, kc, vc, shared, [32, 7, 20], 0.125, 0)
    within(ops.paged_attention(q, kc, vc, shared, ints([32, 7, 20])), o64, half_step(BF16) * o64.abs() * (1 + 1e-6) + eo * 1.01)
    enceladus.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("lens", [[130, 0, 1, 200], [20_000, 3, 0, 9_999]], ids=str)
@pytest.mark.parametrize("variant", [None, *range(2)])
def test_attention_output_over_the_queries(dtype, lens, variant):
    """o may be q, for rows of one piece, of many and of none: the same bits as with an output of its own."""
    q, kc, vc, table = make_attention(dtype, lens, heads=(12, 2), dim=64, garbage=0.0)
    ops.paged_attention_kernel.variant = variant
    try:
        want = ops.paged_attention(q, kc, vc, table, ints(lens))
        assert ops.paged_attention(q, kc, vc, table, ints(lens), o=q) is q
    finally:
        ops.paged_attention_kernel.variant = None
    enceladus.synchronize()
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_attention_scales_of_any_sign(dtype, scale):
    check_attention(dtype, [300, 0, 17, 900], scale=scale, dim=128)


def test_attention_out_of_range_is_reported():
    q, kc, vc, table = make_attention(BF16, [100, 40], dim=64)
    for lens, page in (([8 * 16 + 1, 1], None), ([-1, 1], None), ([2**31 - 1, 1], None), ([100, 40], -1), ([100, 40], kc.shape[0])):
        bad = table.clone()
        if page is not None:
            bad[1, 1] = page
        ops.paged_attention(q, kc, vc, bad, ints(lens))
        with pytest.raises(enceladus.CudaError, match="enc_paged_attention"):
            enceladus.synchronize()
    ops.paged_attention(q, kc, vc, table, ints([100, 40]))
    enceladus.synchronize()


def test_attention_offsets_past_32_bits():
    """A pool whose element offsets pass 2^32: the sequence's pages sit at both ends."""
    page, dim, dtype = 64, 128, BF16
    pages = 2**32 // (page * dim) + 3  # one head: 8.6 GB per cache
    if torch.cuda.mem_get_info()[0] < 20 * 2**30:
        pytest.skip("needs 20 GB of device memory")
    kc = torch.empty(pages, 1, page, dim, device="cuda", dtype=dtype)
    vc = torch.empty_like(kc)
    g = gen(5)
    chosen = [pages - 1, 0, pages - 2]
    table = ints([chosen])
    k, v = randn(g, 3 * page, 1, dim, dtype=dtype), randn(g, 3 * page, 1, dim, dtype=dtype)
    ops.append_kv(k, v, kc, vc, table, ints([0] * 3 * page), ints(list(range(3 * page))))
    for i, p in enumerate(chosen):
        assert torch.equal(kc[p, 0], k[i * page : (i + 1) * page, 0]) and torch.equal(vc[p, 0], v[i * page : (i + 1) * page, 0])
    q = randn(g, 1, 4, dim, dtype=dtype)
    o64, _, eo, _ = attend64(q, kc, vc, table, [3 * page], dim**-0.5, 0)
    within(ops.paged_attention(q, kc, vc, table, ints([3 * page])), o64, half_step(dtype) * o64.abs() * (1 + 1e-6) + eo * 1.01)
    enceladus.synchronize()


def test_attention_is_the_same_every_time_and_on_other_streams():
    lens = [3000, 1, 0, 777, 5000]
    q, kc, vc, table = make_attention(BF16, lens, heads=(32, 8), dim=128, garbage=0.0)
    first = ops.paged_attention(q, kc, vc, table, ints(lens))
    n = ints(lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append(ops.paged_attention(q, kc, vc, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in got)


def test_attention_captured_graphs_follow_the_lengths():
    """Two graphs captured from one set of tensors, replayed on two streams at once with lengths that change between replays."""
    lens = [1000, 5, 0, 64]
    q, kc, vc, table = make_attention(BF16, [4000] * 4, heads=(8, 2), dim=128, garbage=0.0)
    n = ints(lens)
    q2 = q * 2
    ops.paged_attention(q, kc, vc, table, n)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (q, q2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.paged_attention(x, kc, vc, table, n, return_lse=True))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for now in ([1000, 5, 0, 64], [4000, 4000, 1, 0], [0, 0, 0, 0], [1, 2, 3, 4]):
        n.copy_(ints(now))
        torch.cuda.synchronize()
        for _ in range(3):
            for gr, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        for x, (o, lse) in zip((q, q2), outs):
            o64, lse64, eo, el = attend64(x, kc, vc, table, now, 128**-0.5, 0)
            within(o, o64, half_step(BF16) * o64.abs() * (1 + 1e-6) + eo * 1.01)
            within(lse, lse64, el)
    enceladus.synchronize()


# ---- logits --------------------------------------------------------------------------------------------------------
def logits64(x, tokens, lens, prompts, rep, freq, pres, ids, values, mask):
    """The definition in 64 bits, row by row, and the sum of the magnitudes met on the way."""
    y = x.double().clone()
    size = y.abs()
    for r in range(y.shape[0]):
        row = y[r]
        if tokens is not None:
            n, m = int(lens[r]), int(prompts[r])
            past = tokens[r, :n].long()
            seen = torch.unique(past)
            old = row[seen]
            row[seen] = torch.where(old > 0, old / float(rep[r]), old * float(rep[r]))
            size[r, seen] += row[seen].abs()
            made = torch.bincount(past[m:], minlength=y.shape[1])
            drop = made.double() * float(freq[r]) + (made > 0) * float(pres[r])
            row -= drop
            size[r] += drop.abs() + (made * float(freq[r])).abs()
        if ids is not None:
            for t, v in zip(ids[r].tolist(), values[r].tolist()):
                if t >= 0:
                    row[t] += v
                    size[r, t] += 2 * abs(v)
        if mask is not None:
            t = torch.arange(y.shape[1], device="cuda")
            row[((mask[r].long()[t // 32] >> (t % 32)) & 1) == 0] = -math.inf
    return y, size


def make_logits(dtype, rows, vocab, history, biases, mask, seed=0):
    g = gen(seed)
    x = (randn(g, rows, vocab) * 4).to(dtype)
    lens = torch.randint(0, history + 1, (rows,), device="cuda", generator=g, dtype=torch.int32)
    lens[0] = history
    prompts = (lens.double() * torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)).int()
    tokens = (torch.rand(rows, history, device="cuda", generator=g).pow(3) * vocab).int().clamp_(max=vocab - 1)
    tokens[torch.arange(history, device="cuda") >= lens[:, None]] = -9  # past the length: anything
    u = lambda lo, hi: torch.rand(rows, device="cuda", generator=g) * (hi - lo) + lo  # noqa: E731
    ids = values = bits = None
    if biases:
        ids = torch.randint(-1, vocab, (rows, biases), device="cuda", generator=g, dtype=torch.int32)
        ids[:, biases // 2 :] = ids[:, : biases - biases // 2].clone()  # tokens with several biases
        values = randn(g, rows, biases) * 5
    if mask:
        bits = torch.randint(-(2**31), 2**31, (rows, -(-vocab // 32)), device="cuda", generator=g, dtype=torch.int32)
        bits[-1] = 0  # a row that allows nothing
        bits[rows // 2] = -1
    return x, tokens, lens, prompts, u(0.7, 1.6), u(-0.5, 0.5), u(-1.0, 1.0), ids, values, bits


def check_logits(x, *rest, out=None):
    want, size = logits64(x, *rest)
    names = ("tokens", "lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values", "mask")
    got = ops.penalize_logits(x, **dict(zip(names, rest)), out=out)
    enceladus.synchronize()
    # at most six float32 operations plus one per bias; a bias adds its own magnitude to `size`
    steps = 6 + (0 if rest[6] is None else rest[6].shape[1])
    fine = torch.where(torch.isfinite(want), want, 0.0)
    within(got, want, (half_step(x.dtype) * fine.abs() + steps * U * size + TINY[x.dtype]) * (1 + 1e-6))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 31), (3, 33), (2, 8192), (2, 8193), (5, 50001), (1, 131072), (70, 1000)])
def test_logits_shapes(dtype, rows, vocab):
    check_logits(*make_logits(dtype, rows, vocab, 300, 7, True, seed=vocab))
    check_logits(*make_logits(dtype, rows, vocab, 1, 0, False, seed=vocab))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (0, 3), (2, 5), (0, 8)])
def test_logits_strided_and_in_place(dtype, offset, pad):
    x, *rest = make_logits(dtype, 4, 20011, 900, 40, True)
    wide = torch.full((4, offset + 20011 + pad), 3.0, device="cuda", dtype=dtype)
    view = wide[:, offset : offset + 20011]
    view.copy_(x)
    check_logits(view, *rest)
    check_logits(x, *rest, out=view)  # input and output aligned differently
    view.copy_(x)
    check_logits(view, *rest, out=view)
    assert (wide[:, :offset] == 3.0).all() and (wide[:, offset + 20011 :] == 3.0).all()


def test_logits_parts_alone():
    x, tokens, lens, prompts, rep, freq, pres, ids, values, mask = make_logits(F32, 3, 5000, 200, 20, True)
    past = (tokens, lens, prompts, rep, freq, pres)
    none = (None,) * 6
    check_logits(x, *past, None, None, None)
    check_logits(x, *none, ids, values, None)
    check_logits(x, *none, None, None, mask)
    check_logits(x, *none, None, None, None)
    check_logits(x, *past, ids, values, None)
    check_logits(x, tokens[:, :0], lens * 0, prompts * 0, rep, freq, pres, ids, values, mask)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_logits_extreme_values(dtype):
    """-inf and the type's lowest value stay what they are where nothing touches them; NaN and inf in masked places vanish."""
    x, tokens, lens, prompts, rep, freq, pres, ids, values, mask = make_logits(dtype, 4, 1000, 100, 0, True)
    low = torch.finfo(dtype).min
    x[:, ::7], x[:, 1::7], x[:, 2::7], x[:, 3::7] = -math.inf, low, math.nan, math.inf
    untouched = torch.ones_like(x, dtype=torch.bool)
    for r in range(4):
        untouched[r, tokens[r, : int(lens[r])].long()] = False
    got = ops.penalize_logits(x, tokens, lens, prompts, rep, freq, pres, mask=mask)
    t = torch.arange(1000, device="cuda")
    allowed = ((mask[:, t // 32] >> (t % 32)) & 1) == 1
    assert (got[~allowed] == -math.inf).all()
    same = allowed & untouched
    assert torch.equal(torch.nan_to_num(got[same], nan=5.0), torch.nan_to_num(x[same], nan=5.0))
    assert torch.equal(torch.isnan(got[same]), torch.isnan(x[same]))
    enceladus.synchronize()


def test_logits_one_token_repeated_and_long_history():
    vocab, n = 40_000, 30_000
    x = randn(gen(6), 2, vocab)
    tokens = torch.full((2, n), 39_999, device="cuda", dtype=torch.int32)
    tokens[1] = torch.arange(n, device="cuda", dtype=torch.int32)
    f = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    check_logits(x, tokens, ints([n, n]), ints([1, 0]), f(1.3, 1.1), f(0.001, 0.25), f(0.5, 0.125), None, None, None)


def test_logits_out_of_range_is_reported():
    x, tokens, lens, prompts, rep, freq, pres, ids, values, _ = make_logits(F32, 2, 100, 10, 4, False)
    want = ops.penalize_logits(x, tokens, lens, prompts, rep, freq, pres, ids, values)
    enceladus.synchronize()
    for what in ("token", "negative", "len", "prompt", "bias"):
        a = [t.clone() for t in (tokens, lens, prompts, ids)]
        if what == "token":
            a[0][0, 0] = 100
        elif what == "negative":
            a[0][0, 0] = -1
        elif what == "len":
            a[1][1] = 11
        elif what == "prompt":
            a[2][0] = 11
        else:
            a[3][1, 0] = -2
        ops.penalize_logits(x, a[0], a[1], a[2], rep, freq, pres, a[3], values)
        with pytest.raises(enceladus.CudaError, match="enc_penalize_logits"):
            enceladus.synchronize()
    assert torch.equal(want, ops.penalize_logits(x, tokens, lens, prompts, rep, freq, pres, ids, values))
    enceladus.synchronize()


# ---- together ------------------------------------------------------------------------------------------------------
def test_numpy_arguments():
    r = np.random.default_rng(0)
    kc, vc = r.standard_normal((4, 2, 8, 32)).astype(np.float32), r.standard_normal((4, 2, 8, 32)).astype(np.float32)
    k, v, q = (r.standard_normal((3, h, 32)).astype(np.float32) for h in (2, 2, 4))
    table = np.array([[2, 1], [0, 3]], np.int32)
    ids, pos = np.array([0, 1, 0], np.int32), np.array([9, 4, 10], np.int32)
    k0 = kc.copy()
    assert ops.append_kv(k, v, kc, vc, table, ids, pos) is None
    assert np.array_equal(kc[1, :, 1], k[0]) and np.array_equal(kc[0, :, 4], k[1]) and np.array_equal(vc[1, :, 2], v[2])
    changed = np.zeros(kc.shape[:3], bool)
    changed[1, :, 1] = changed[0, :, 4] = changed[1, :, 2] = True
    assert np.array_equal(kc[~changed], k0[~changed])
    lens = np.array([11, 5], np.int32)
    o, lse = ops.paged_attention(q[:2], kc, vc, table, lens, return_lse=True)
    dev = [torch.from_numpy(x).cuda() for x in (q[:2], kc, vc, table, lens)]
    o2, lse2 = ops.paged_attention(*dev, return_lse=True)
    assert np.array_equal(o, o2.cpu().numpy()) and np.array_equal(lse, lse2.cpu().numpy())
    x = r.standard_normal((2, 100)).astype(np.float32)
    past = (np.array([[1, 2, 2], [5, 5, 5]], np.int32), np.array([3, 2], np.int32), np.array([1, 0], np.int32),
            *(np.full(2, c, np.float32) for c in (1.2, 0.5, 0.25)))
    y = ops.penalize_logits(x, *past)
    y2 = ops.penalize_logits(*(torch.from_numpy(t).cuda() for t in (x, *past)))
    assert np.array_equal(y, y2.cpu().numpy())


def general(kernel):
    """The kernel's calls go through `kernel[grid](...)` while this is in force."""
    class Way:
        def __enter__(self):
            kernel.variant = N.VARIANT_AUTO

        def __exit__(self, *_):
            kernel.variant = None

    return Way()


def test_a_process_may_begin_with_a_captured_step():
    """Nothing has to run before the first capture: no allocation, no set-up that a capture would refuse."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from enceladus_b200 import ops
import enceladus_b200 as enceladus
z = lambda *s, t=torch.bfloat16: torch.ones(*s, device="cuda", dtype=t)
kc, vc, k, v, q, qo = z(400, 4, 16, 128), z(400, 4, 16, 128), z(8, 4, 128), z(8, 4, 128), z(8, 16, 128), z(8, 16, 128)
kc2, q2 = z(400, 4, 16, 64, t=torch.float32), z(8, 4, 64, t=torch.float32)
i = lambda x: x.to(torch.int32)
table = i(torch.arange(400, device="cuda").reshape(8, 50))
ids, pos, lens, x = i(torch.arange(8, device="cuda")), i(z(8) * 699), i(z(8) * 700), z(8, 50000)
tok, one = i(z(8, 40)), z(8, t=torch.float32)
cos = z(800, 64, t=torch.float32)
out = torch.empty_like(x)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.append_kv(k * 3, v * 3, kc, vc, table, ids, pos, cos=cos, sin=cos * 0, q=q, q_out=qo)
    o = ops.paged_attention(qo, kc, vc, table, lens)
    o2 = ops.paged_attention(q2, kc2, kc2, table, lens)
    o3 = ops.paged_attention(qo, kc, vc, table, lens + 1)
    ops.penalize_logits(x, tok, ids * 0 + 40, ids * 0, one * 2, one, one, out=out)
graph.replay()
enceladus.synchronize()
# 699 is 700 in bfloat16 (steps of 4): the new token lies in page 43, slot 12, the first behind the length
assert (pos == 700).all() and (kc[table[:, 43].long(), :, 12] == 3).all() and (kc == 3).sum() == 8 * 4 * 128
# without it every value is 1: a mean of ones, whose two sums of 700 and whose division round in float32
assert (o == 1).all() and ((o2 - 1).abs() <= (2 * 700 + 4) * 2.0 ** -24).all(), (o, o2)
# with it its score leads by 2 * 128 / sqrt(128) = 22.6, and the 700 ones move the result by 2e-7 from 3
assert (o3 == 3).all(), o3
assert (out[:, 1] == 0.5 - 41).all() and (out[:, 2:] == 1).all()
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_short_way_and_the_launch_path_agree():
    """Every valid call on device tensors goes the short way, with the launch path's bits; nothing else does."""
    from enceladus_b200.runtime import lane

    way = lane.get()
    assert way is not None, "enc_torch_lane.so is not built"
    g = gen(9)
    for dtype in (BF16, F16, F32):
        q, kc, vc, table = make_attention(dtype, [300, 0, 41], dim=64, garbage=0.0)
        n = ints([300, 0, 41])
        for scale, window in ((None, 0), (0.3, 100), (1, 2**40)):
            args = (q, kc, vc, table, n, scale, window, None, True)
            assert way.paged_attention(*args) is not NotImplemented
            a = ops.paged_attention(q, kc, vc, table, n, sm_scale=scale, window=window, return_lse=True)
            with general(ops.paged_attention_kernel):
                b = ops.paged_attention(q, kc, vc, table, n, sm_scale=scale, window=window, return_lse=True)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        k, v, cos, sin = randn(g, 3, 2, 64, dtype=dtype), randn(g, 3, 2, 64, dtype=dtype), *tables(400, 48)
        ids, pos = ints([0, -1, 2]), ints([299, 0, 40])
        for interleaved in (False, True):
            for rot in ((cos, sin), (None, None)):
                caches = [kc.clone(), vc.clone()], [kc.clone(), vc.clone()]
                outs = [torch.zeros_like(q) for _ in range(2)]
                assert way.append_kv(k, v, *caches[0], table, ids, pos, *rot, q, outs[0], interleaved) is outs[0]
                with general(ops.append_kv_kernel):
                    assert ops.append_kv(k, v, *caches[1], table, ids, pos, *rot, q=q, q_out=outs[1], interleaved=interleaved) is outs[1]
                assert torch.equal(outs[0], outs[1]) and all(torch.equal(x, y) for x, y in zip(*caches))
        assert way.append_kv(k, v, kc, vc, table, ids, pos, None, None, None, None, False) is None
        x, *rest = make_logits(dtype, 3, 777, 50, 5, True)
        for parts in (rest, [*rest[:6], None, None, None], [None] * 6 + rest[6:], [None] * 9):
            assert way.penalize_logits(x, *parts, None) is not NotImplemented
            names = ("tokens", "lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values", "mask")
            a = ops.penalize_logits(x, **dict(zip(names, parts)))
            with general(ops.penalize_logits_kernel):
                b = ops.penalize_logits(x, **dict(zip(names, parts)))
            assert torch.equal(a, b)
        enceladus.synchronize()

        bad_k = k.double()
        for args in ((bad_k, v, kc, vc, table, ids, pos), (k, v[:2], kc, vc, table, ids, pos), (k, v, kc, vc[:1], table, ids, pos),
                     (k, v, kc, vc, table.long(), ids, pos), (k, v, kc, vc, table, ids.long(), pos), (k, v, kc, vc, table, ids, pos[:2]),
                     (k.cpu(), v, kc, vc, table, ids, pos), (k, v, kc[:1].expand_as(kc), vc, table, ids, pos), (k, v, kc.transpose(2, 3), vc, table, ids, pos),
                     (None, v, kc, vc, table, ids, pos), (k.cpu().float().numpy(), v, kc, vc, table, ids, pos), (k[:0], v[:0], kc, vc, table, ids[:0], pos[:0])):
            assert way.append_kv(*args, cos, sin, None, None, False) is NotImplemented
        for extra in ((cos, None, q, None), (cos.double(), sin.double(), q, None), (cos[:, ::2], sin[:, ::2], q, None), (cos, sin, None, q), (cos, sin, q, q[:2]),
                      (cos, sin, q, q[:, :1].expand_as(q)), (*tables(9, 66), q, None)):
            assert way.append_kv(k, v, kc, vc, table, ids, pos, *extra, False) is NotImplemented
        for args in ((q[:, :3], kc, vc, table, n), (q[:2], kc, vc, table, n), (q, kc, vc, table[:2], n), (q, kc, vc, table, n.long()), (q, kc, vc, table, n[:2]),
                     (q.cpu(), kc, vc, table, n), (q.transpose(0, 1), kc, vc, table, n), (q[..., :32], kc, vc, table, n)):
            assert way.paged_attention(*args, None, 0, None, False) is NotImplemented
        for extra in (("x", 0, None, False), (None, -1, None, False), (None, 1.5, None, False), (None, 2**70, None, False), (None, 0, q[:2], False)):
            assert way.paged_attention(q, kc, vc, table, n, *extra) is NotImplemented
        assert way.penalize_logits(x, *rest[:5], None, *rest[6:], None) is NotImplemented
        assert way.penalize_logits(x, None, *rest[1:], None) is NotImplemented
        assert way.penalize_logits(x, *rest[:8], rest[8][:, 1:], None) is NotImplemented
        assert way.penalize_logits(x, *rest, x[:, :5]) is NotImplemented
        assert way.penalize_logits(x.t(), *[None] * 10) is NotImplemented
        assert way.penalize_logits(x) is NotImplemented
    with pytest.raises(ValueError, match="go together"):
        ops.penalize_logits(x, *rest[:5])
    with pytest.raises(TypeError, match="must be int32"):
        ops.paged_attention(q, kc, vc, table, n.long())
    lib = N.load()
    lib.enc_test_fail_next(N.ERR_LAUNCH)
    with pytest.raises(enceladus.CudaError, match="injected"):
        ops.paged_attention(q, kc, vc, table, n)
    with pytest.raises(NotImplementedError, match="head_dim"):  # an error of the library's own, worded there
        with general(ops.paged_attention_kernel):
            ops.paged_attention_kernel[(1,)](q, kc, vc, q, None, table, n, 1.0, 0, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, Q_HEADS=2, KV_HEADS=2,
                                             HEAD_DIM=300, PAGE_SIZE=16)


def decode_step(w, x, kc, vc, table, ids, pos, lens, cos, sin, past, mask):
    """One layer and a head, made of the framework's operators only."""
    b, hid = x.shape
    hq, hk, d = w["heads"]
    qkv = ops.matmul(ops.rmsnorm(x, w["norm"]), w["qkv"]).reshape(b, hq + 2 * hk, d)
    q = ops.append_kv(qkv[:, hq : hq + hk], qkv[:, hq + hk :], kc, vc, table, ids, pos, cos=cos, sin=sin, q=qkv[:, :hq])
    o = ops.paged_attention(q, kc, vc, table, lens)
    x = ops.add(x, ops.matmul(o.reshape(b, hq * d), w["out"]))
    x = ops.add(x, ops.matmul(ops.matmul_bias_gelu(ops.rmsnorm(x, w["norm"]), w["up"], w["bias"]), w["down"]))
    logits = ops.matmul(ops.rmsnorm(x, w["norm"]), w["vocab"])
    return ops.softmax(ops.penalize_logits(logits, *past, mask=mask))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_decoding_steps_match_attention_over_the_whole_sequence(dtype):
    """Three sequences generated token by token, eagerly and as one replayed graph; the last step's probabilities against
    the same model run over whole sequences in 64 bits with the dense causal definition."""
    g = gen(7)
    hq, hk, d, hid, vocab, steps = 4, 2, 64, 128, 500, 40
    w = {"heads": (hq, hk, d), "norm": (1 + randn(g, hid) * 0.1).to(dtype), "qkv": (randn(g, hid, (hq + 2 * hk) * d) * hid**-0.5).to(dtype),
         "out": (randn(g, hq * d, hid) * hid**-0.5).to(dtype), "up": (randn(g, hid, 256) * hid**-0.5).to(dtype),
         "bias": (randn(g, 256) * 0.1).to(dtype), "down": (randn(g, 256, hid) * 0.05).to(dtype), "vocab": (randn(g, hid, vocab) * hid**-0.5).to(dtype)}
    inputs = randn(g, steps, 3, hid, dtype=dtype)
    cos, sin = tables(64, d)
    table = ints([[5, 0, 3], [1, 2, 7], [6, 4, 8], [-1, -1, -1]])
    ids = ints([0, 1, 2, -1])  # the batch is padded to four
    f = lambda v: torch.full((4,), v, device="cuda")  # noqa: E731
    tokens = torch.randint(0, vocab, (4, 30), device="cuda", generator=g, dtype=torch.int32)
    past = (tokens, ints([30, 10, 0, 0]), ints([5, 10, 0, 0]), f(1.2), f(0.3), f(0.2))
    mask = torch.randint(-(2**31), 2**31, (4, 16), device="cuda", generator=g, dtype=torch.int32)
    results = []
    for captured in (False, True):
        kc, vc = make_cache(g, 9, hk, 16, d, dtype, fill=math.nan), make_cache(g, 9, hk, 16, d, dtype, fill=math.nan)
        x, pos, lens = torch.zeros(4, hid, device="cuda", dtype=dtype), ints([0, 0, 0, 0]), ints([1, 1, 1, 0])
        if captured:
            scratch = (kc.clone(), vc.clone())
            decode_step(w, x, *scratch, table, ids, pos, lens, cos, sin, past, mask)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                probs = decode_step(w, x, kc, vc, table, ids, pos, lens, cos, sin, past, mask)
        for t in range(steps):
            x[:3] = inputs[t]
            if captured:
                graph.replay()
            else:
                probs = decode_step(w, x, kc, vc, table, ids, pos, lens, cos, sin, past, mask)
            pos[:3] += 1
            lens[:3] += 1
        results.append(probs[:3].clone())
        enceladus.synchronize()
    assert torch.equal(results[0], results[1])

    norm = lambda z: z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w["norm"].double()  # noqa: E731
    x = inputs.double().transpose(0, 1)  # (3, steps, hid)
    qkv = (norm(x) @ w["qkv"].double()).reshape(3, steps, hq + 2 * hk, d)
    turn = lambda z: torch.stack([rotate64(s, cos[:steps], sin[:steps], d, False)[0] for s in z])  # noqa: E731
    q, k, v = turn(qkv[:, :, :hq]), turn(qkv[:, :, hq : hq + hk]), qkv[:, :, hq + hk :]
    k, v = k.repeat_interleave(hq // hk, 2), v.repeat_interleave(hq // hk, 2)
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) * d**-0.5
    s.masked_fill_(torch.ones(steps, steps, device="cuda").triu(1).bool(), -math.inf)
    o = torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).reshape(3, steps, hq * d)
    x = x + o @ w["out"].double()
    x = x + torch.nn.functional.gelu(norm(x) @ w["up"].double() + w["bias"].double()) @ w["down"].double()
    logits = (norm(x) @ w["vocab"].double())[:, -1]
    want = logits64(logits, *[t[:3] for t in past], None, None, mask[:3])[0].softmax(-1)
    # The step rounds to its type about ten times in a row; roundings of relative size h on values of order one move a logit by
    # about h * sqrt(10) * (a few standard deviations), and a probability by that relative to itself: 32 h covers it.
    assert float(((results[0].double() - want).abs() / (want + 1e-4)).max()) <= 32 * half_step(dtype) + 1e-4

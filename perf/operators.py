"""The operators of a decoding step as they are measured: appending to a paged key-value cache with the position
rotation on the way, attention of one new token over that cache, and the penalties, biases and grammar masks that the
logits pass through before they are sampled.

`own` chooses who computes: False, the plain forms below (elementary torch operations in 32 bits, rounded once at the
end); True, the calls that a user makes of `enceladus_b200.ops`.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # One request generating: its new token's q, k and v out of the fused projection.  Latency is all there is.
        {"name": "append_one", "op": "append", "dtype": "bf16", "tokens": 1, "seqs": 1, "pad": 0, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot_dim": 128, "page": 16, "layout": "nhd", "interleaved": False, "context": 700},
        # A full decoding batch, padded to the size it is captured at: one token of each of 250 requests, six idle rows.
        {"name": "append_batch", "op": "append", "dtype": "f16", "tokens": 250, "seqs": 250, "pad": 6, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot_dim": 128, "page": 16, "layout": "hnd", "interleaved": False, "context": 4096},
        # Prompts of nine requests entering the cache in one pass, the largest job.
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "tokens": 32768, "seqs": 9, "pad": 0, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "rot_dim": 128, "page": 64, "layout": "hnd", "interleaved": False, "context": 0},
        # A small full-precision model with neighbouring pairs rotated, half of each head left as it is, odd sizes.
        {"name": "append_f32_odd", "op": "append", "dtype": "f32", "tokens": 5003, "seqs": 7, "pad": 13, "q_heads": 12, "kv_heads": 3,
         "head_dim": 64, "rot_dim": 32, "page": 24, "layout": "nhd", "interleaved": True, "context": 999},
        # One short conversation: the smallest attention.
        {"name": "attend_one", "op": "attend", "dtype": "bf16", "seqs": 1, "shortest": 130, "longest": 130, "empty": 0, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "layout": "nhd", "window": 0, "lse": False},
        # An ordinary serving batch: ragged lengths, two rows idle.
        {"name": "attend_batch", "op": "attend", "dtype": "bf16", "seqs": 64, "shortest": 1, "longest": 4096, "empty": 2, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "layout": "nhd", "window": 0, "lse": False},
        # Few requests over long documents: few rows, so the length has to be split.
        {"name": "attend_long", "op": "attend", "dtype": "f16", "seqs": 2, "shortest": 100000, "longest": 131072, "empty": 0, "q_heads": 32,
         "kv_heads": 4, "head_dim": 128, "page": 64, "layout": "hnd", "window": 0, "lse": True},
        # The largest: every head with keys of its own (the shapes of the dense attention benchmark, one token at its end).
        {"name": "attend_heads", "op": "attend", "dtype": "bf16", "seqs": 48, "shortest": 2000, "longest": 8192, "empty": 0, "q_heads": 32,
         "kv_heads": 32, "head_dim": 128, "page": 32, "layout": "hnd", "window": 0, "lse": False},
        # Full precision, head_dim 64, pages of an odd size, only the last thousand keys seen, the statistics returned.
        {"name": "attend_f32_window", "op": "attend", "dtype": "f32", "seqs": 33, "shortest": 1, "longest": 5000, "empty": 1, "q_heads": 16,
         "kv_heads": 4, "head_dim": 64, "page": 24, "layout": "nhd", "window": 1000, "lse": True},
        # One request: penalties over a short history, a handful of biases.
        {"name": "logits_one", "op": "logits", "dtype": "f32", "rows": 1, "vocab": 32000, "history": 200, "biases": 4, "mask": False},
        # Structured output in bf16 over an odd vocabulary: grammar masks on every row, no biases.
        {"name": "logits_grammar", "op": "logits", "dtype": "bf16", "rows": 48, "vocab": 50001, "history": 1500, "biases": 0, "mask": True},
        # The largest: a full batch over a wide vocabulary, long histories, biases and masks.
        {"name": "logits_batch", "op": "logits", "dtype": "f32", "rows": 256, "vocab": 131072, "history": 8192, "biases": 64, "mask": True},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logits"])
    dtype = rng.choice(["bf16", "f16", "bf16", "f32"])
    if op == "logits":
        vocab = _spread(rng, 500, 140000)
        rows = _spread(rng, 1, min(256, 33000000 // vocab))
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "history": _spread(rng, 1, 8192), "biases": rng.choice([0, 3, 64]),
                "mask": rng.random() < 0.6}
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16, 32])
    group = rng.choice([g for g in (1, 2, 4, 5, 7, 8, 16) if g * kv_heads <= 64])
    c = {"op": op, "dtype": dtype, "q_heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": rng.choice([32, 64, 64, 128, 128, 128, 256]),
         "page": rng.choice([16, 16, 32, 64, 128, 1, 24]), "layout": rng.choice(["nhd", "hnd"])}
    width = c["head_dim"] * SIZE[dtype]
    if op == "append":
        most = 360000000 // ((c["q_heads"] + 2 * kv_heads) * width)
        tokens = _spread(rng, 1, min(32768, most))
        seqs = tokens if tokens <= 256 and rng.random() < 0.5 else rng.randint(1, min(16, tokens))
        return {**c, "tokens": tokens, "seqs": seqs, "pad": rng.choice([0, 0, 5]), "rot_dim": rng.choice([c["head_dim"], c["head_dim"], c["head_dim"] // 2]),
                "interleaved": rng.random() < 0.3, "context": _spread(rng, 1, 100000)}
    most = 2000000000 // (kv_heads * width)  # keys in all
    seqs = _spread(rng, 1, 128)
    longest = _spread(rng, 1, min(131072, max(1, most // seqs)))
    return {**c, "seqs": seqs, "shortest": rng.randint(1, longest), "longest": longest, "empty": rng.choice([0, 0, min(1, seqs - 1)]),
            "window": rng.choice([0, 0, 0, _spread(rng, 1, 4096)]), "lse": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(c):
    """Key counts of the sequences of an attention case: spread evenly from the shortest to the longest, the idle ones zero."""
    n = c["seqs"] - c["empty"]
    step = (c["longest"] - c["shortest"]) / max(1, n - 1)
    return [0] * c["empty"] + [c["longest"] - int(round(i * step)) for i in range(n)]


def _histories(c):
    """Token counts of the rows of a logits case."""
    return [max(1, c["history"] - (i * c["history"]) // c["rows"]) for i in range(c["rows"])]


def _counts(c):
    """New tokens of each sequence of an append case, the first ones longer."""
    s, t = c["seqs"], c["tokens"]
    if s == t:
        return [1] * s
    weight = [s - i for i in range(s)]
    got = [1 + (t - s) * w // sum(weight) for w in weight]
    got[0] += t - sum(got)
    return got


def _spans(c):
    """(tokens already in the cache, new tokens) of each sequence of an append case."""
    rnd = random.Random(c["tokens"])
    return [(rnd.randint(0, c["context"]), n) for n in _counts(c)]


def _cache(c, pages, g):
    """A page pool [pages, kv_heads, page, head_dim]; laid out token by token (nhd) or head by head (hnd)."""
    shape = (pages, c["page"], c["kv_heads"], c["head_dim"]) if c["layout"] == "nhd" else (pages, c["kv_heads"], c["page"], c["head_dim"])
    t = torch.randn(shape, device="cuda", dtype=TYPES[c["dtype"]], generator=g)
    return t.transpose(1, 2) if c["layout"] == "nhd" else t


def prepare(case, seed):
    c, rnd = case, random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": c}
    if c["op"] == "append":
        page = c["page"]
        spans = _spans(c)
        rnd.shuffle(spans)
        width = -(-max(f + n for f, n in spans) // page)
        # Only the pages that the call writes are in the pool: those of the earlier context all name page 0.
        table, pages = [], 1
        for f, n in spans:
            a, b = f // page, (f + n - 1) // page
            table.append((a, b, pages))
            pages += b - a + 1
        order = torch.randperm(pages - 1, device="cuda", generator=g, dtype=torch.int32) + 1
        s["block_table"] = torch.zeros(c["seqs"], width, dtype=torch.int32, device="cuda")
        for i, (a, b, p) in enumerate(table):
            s["block_table"][i, a:b + 1] = order[p - 1:p + b - a]
        seq_ids = [i for i, (_, n) in enumerate(spans) for _ in range(n)] + [-1] * c["pad"]
        positions = [f + j for f, n in spans for j in range(n)] + [0] * c["pad"]
        s["seq_ids"], s["positions"] = ints(seq_ids), ints(positions)
        heads, d = c["q_heads"] + 2 * c["kv_heads"], c["head_dim"]
        qkv = torch.randn(len(seq_ids), heads, d, device="cuda", dtype=TYPES[c["dtype"]], generator=g)  # the fused projection's output
        s["q"], s["k"], s["v"] = qkv.split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)
        s["q_out"] = torch.zeros(len(seq_ids), c["q_heads"], d, device="cuda", dtype=TYPES[c["dtype"]])
        s["k_cache"], s["v_cache"] = _cache(c, pages, g), _cache(c, pages, g)
        freq = 10000.0 ** (-torch.arange(0, c["rot_dim"], 2, device="cuda", dtype=torch.float64) / c["rot_dim"])
        angle = torch.arange(width * page, device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif c["op"] == "attend":
        lens = _lengths(c)
        rnd.shuffle(lens)
        need = [-(-n // c["page"]) for n in lens]
        order = torch.randperm(max(1, sum(need)), device="cuda", generator=g, dtype=torch.int32)
        s["block_table"] = torch.full((c["seqs"], max(1, max(need))), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            s["block_table"][i, :n] = order[at:at + n]
            at += n
        s["seq_lens"] = ints(lens)
        s["k_cache"], s["v_cache"] = _cache(c, max(1, sum(need)), g), _cache(c, max(1, sum(need)), g)
        s["q"] = torch.randn(c["seqs"], c["q_heads"], c["head_dim"], device="cuda", dtype=TYPES[c["dtype"]], generator=g)
    else:
        r, n, v = c["rows"], c["history"], c["vocab"]
        lens = _histories(c)
        rnd.shuffle(lens)
        s["logits"] = (torch.randn(r, v, device="cuda", generator=g) * 4).to(TYPES[c["dtype"]])
        s["tokens"] = (torch.rand(r, n, device="cuda", generator=g).pow(3) * v).int().clamp_(max=v - 1)  # the common ones come often
        s["lens"], s["prompt_lens"] = ints(lens), ints([x // 2 for x in lens])
        uniform = lambda lo, hi: torch.rand(r, device="cuda", generator=g) * (hi - lo) + lo  # noqa: E731
        s["repetition"], s["frequency"], s["presence"] = uniform(1.0, 1.5), uniform(0.0, 0.5), uniform(-0.5, 1.0)
        s["bias_ids"] = s["bias_values"] = s["mask"] = None
        if c["biases"]:
            s["bias_ids"] = torch.randint(-1, v, (r, c["biases"]), device="cuda", dtype=torch.int32, generator=g)  # -1: an unused place
            s["bias_values"] = torch.randn(r, c["biases"], device="cuda", generator=g) * 5
        if c["mask"]:
            words = lambda: torch.randint(-2**31, 2**31, (r, -(-v // 32)), device="cuda", dtype=torch.int32, generator=g)  # noqa: E731
            s["mask"] = words() & words()  # a quarter of the vocabulary allowed
            s["mask"][::2] = -1  # every other request free
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------
def _append_plain(s):
    c = s["case"]
    page, r = c["page"], c["rot_dim"]
    live = (s["seq_ids"] >= 0).nonzero()[:, 0]
    seq, pos = s["seq_ids"][live].long(), s["positions"][live].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def rotated(x):
        x = x[live].float()
        turn, rest = x[..., :r], x[..., r:]
        if c["interleaved"]:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turn[..., :r // 2], turn[..., r // 2:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, rest), -1).to(TYPES[c["dtype"]])

    at = s["block_table"][seq, pos // page].long()
    s["k_cache"][at, :, pos % page] = rotated(s["k"])
    s["v_cache"][at, :, pos % page] = s["v"][live]
    s["q_out"][live] = rotated(s["q"])
    return [s["q_out"], s["k_cache"], s["v_cache"]]


def _attend_plain(s):
    c = s["case"]
    b, hk, d = c["seqs"], c["kv_heads"], c["head_dim"]
    pages = s["block_table"].clamp(min=0).long()
    gathered = lambda cache: cache[pages].permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d).float()  # noqa: E731
    q = s["q"].float().reshape(b, hk, -1, d)
    scores = torch.matmul(q, gathered(s["k_cache"]).transpose(2, 3)) / math.sqrt(d)
    at = torch.arange(scores.shape[-1], device="cuda")
    lens = s["seq_lens"].long()[:, None]
    seen = at < lens
    if c["window"]:
        seen &= at >= lens - c["window"]
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    values = gathered(s["v_cache"]).masked_fill(~seen.transpose(2, 3), 0.0)
    o = torch.where(total > 0, torch.matmul(p, values) / total, 0.0)
    o = o.reshape(b, -1, d).to(TYPES[c["dtype"]])
    return [o, (top + torch.log(total)).reshape(b, -1)] if c["lse"] else [o]


def _logits_plain(s):
    c = s["case"]
    x = s["logits"].float()
    at = torch.arange(s["tokens"].shape[1], device="cuda")
    valid = at < s["lens"][:, None]
    made = valid & (at >= s["prompt_lens"][:, None])
    ids = s["tokens"].long()
    seen = torch.zeros_like(x).scatter_add_(1, ids, valid.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, ids, made.float())
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        used = s["bias_ids"] >= 0
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].clamp(min=0).long(), torch.where(used, s["bias_values"], 0.0))
    if s["mask"] is not None:
        token = torch.arange(c["vocab"], device="cuda")
        allowed = (s["mask"][:, token // 32] >> (token % 32)) & 1
        x = x.masked_fill(allowed == 0, -math.inf)
    return [x.to(TYPES[c["dtype"]])]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "logits": _logits_plain}[c["op"]](s)
    from enceladus_b200 import ops

    if c["op"] == "append":
        ops.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_ids"], s["positions"], cos=s["cos"], sin=s["sin"],
                      q=s["q"], q_out=s["q_out"], interleaved=c["interleaved"])
        return [s["q_out"], s["k_cache"], s["v_cache"]]
    if c["op"] == "attend":
        o = ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], window=c["window"], return_lse=c["lse"])
        return list(o) if c["lse"] else [o]
    return [ops.penalize_logits(s["logits"], s["tokens"], s["lens"], s["prompt_lens"], s["repetition"], s["frequency"], s["presence"],
                                bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"])]


# ---- what one pass cannot do without -----------------------------------------------------------------------------
def work(case):
    c = case
    size = SIZE[c["dtype"]]
    if c["op"] == "append":
        heads = c["q_heads"] + 2 * c["kv_heads"]
        tables = 4 * c["rot_dim"] + 12  # the angle's cosines and sines, the token's sequence, position and page
        return {"bytes": c["tokens"] * (2 * heads * c["head_dim"] * size + tables), "flops": c["tokens"] * (c["q_heads"] + c["kv_heads"]) * 3 * c["rot_dim"]}
    if c["op"] == "attend":
        keys = [min(n, c["window"]) if c["window"] else n for n in _lengths(c)]
        rows = c["seqs"] * c["q_heads"]
        return {"bytes": sum(keys) * 2 * c["kv_heads"] * c["head_dim"] * size + 2 * rows * c["head_dim"] * size + (4 * rows if c["lse"] else 0)
                + sum(4 * -(-n // c["page"]) for n in keys) + 4 * c["seqs"], "flops": 4 * sum(keys) * c["q_heads"] * c["head_dim"]}
    values = c["rows"] * c["vocab"]
    return {"bytes": 2 * values * size + 4 * sum(_histories(c)) + 20 * c["rows"] + 8 * c["rows"] * c["biases"] + (c["rows"] * -(-c["vocab"] // 32) * 4 if c["mask"] else 0),
            "flops": 2 * values}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "append":
        r, half = c["rot_dim"], c["rot_dim"] // 2
        q_out, k_cache, v_cache = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
        # the rotation as a product of complex numbers, pair by pair, from the cosines and sines that the call is given
        pairs = torch.arange(half, device="cuda")
        one, two = (2 * pairs, 2 * pairs + 1) if c["interleaved"] else (pairs, pairs + half)
        seqs, place = s["seq_ids"].tolist(), s["positions"].long()
        turn = torch.complex(s["cos"].double(), s["sin"].double())[place][:, None, :]

        def turned(x):
            x = x.double()
            z = torch.complex(x[..., one], x[..., two]) * turn
            x[..., one], x[..., two] = z.real, z.imag
            return x

        k, q, v = turned(s["k"]), turned(s["q"]), s["v"].double()
        for seq in sorted(set(seqs) - {-1}):
            mine = (s["seq_ids"] == seq).nonzero().flatten()
            where, row = s["block_table"][seq, place[mine] // c["page"]].long(), place[mine] % c["page"]
            k_cache.transpose(1, 2).index_put_((where, row), k[mine])
            v_cache.transpose(1, 2).index_put_((where, row), v[mine])
            q_out[mine] = q[mine]
        return [q_out, k_cache, v_cache]
    if c["op"] == "attend":
        b, h, d = s["q"].shape
        o = torch.zeros(b, h, d, device="cuda", dtype=torch.float64)
        lse = torch.full((b, h), -math.inf, device="cuda", dtype=torch.float64)
        group = h // c["kv_heads"]
        for i, n in enumerate(s["seq_lens"].tolist()):
            if not n:
                continue
            mine = s["block_table"][i, :-(-n // c["page"])].long()
            for j in range(c["kv_heads"]):
                k = s["k_cache"][mine, j].reshape(-1, d)[:n].double()
                v = s["v_cache"][mine, j].reshape(-1, d)[:n].double()
                if c["window"]:
                    k, v = k[-c["window"]:], v[-c["window"]:]
                mine_q = slice(j * group, (j + 1) * group)
                score = s["q"][i, mine_q].double() @ k.T * d ** -0.5
                lse[i, mine_q] = torch.logsumexp(score, 1)
                o[i, mine_q] = (score - lse[i, mine_q, None]).exp() @ v
        return [o, lse] if c["lse"] else [o]
    x = s["logits"].double()
    bits = torch.arange(32, device="cuda", dtype=torch.int32)
    for i, (n, m) in enumerate(zip(s["lens"].tolist(), s["prompt_lens"].tolist())):
        row, history = x[i], s["tokens"][i, :n].long()
        before = torch.bincount(history, minlength=c["vocab"]).bool()
        made = torch.bincount(history[m:], minlength=c["vocab"]).double()
        rep = s["repetition"][i].double()
        row[before & (row > 0)] /= rep
        row[before & (s["logits"][i] <= 0)] *= rep
        row -= made * s["frequency"][i].double() + made.clamp(max=1) * s["presence"][i].double()
        if s["bias_ids"] is not None:
            used = s["bias_ids"][i] >= 0
            row.index_add_(0, s["bias_ids"][i][used].long(), s["bias_values"][i][used].double())
        if s["mask"] is not None:
            allowed = ((s["mask"][i][:, None] >> bits) & 1).flatten()[:c["vocab"]]
            row[allowed == 0] = -math.inf
    return [x]

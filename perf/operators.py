"""The operators of a serving step over a paged compressed cache, as cases that can be timed.

A step of a batch of requests: the pages, slots and positions of its tokens
from the requests' lengths (`plan`), the norm of each query and key head with
the position rotation (`rope`), keys and values quantized into their pages and
read back as a later prefill reads them (`store`), and one new token per
request attending over its pages (`decode`).

Where `own` is false `run()` computes them in elementary torch operations in
32 bits; where it is true it makes the library's calls.  `listed()` holds the
fixed cases, `draw()` more of the same ranges, `exact()` the same results in
64-bit arithmetic, written apart from the plain forms.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the bookkeeping of one decode step: 64 requests, a token each, some pages full, some requests done
        {"name": "plan_decode_64", "kind": "plan", "requests": 64, "page": 64, "ctx": 8192, "chunk": 1, "done": 0.05,
         "pad": 0},
        # a step that mixes long prompt chunks with decodes, small pages
        {"name": "plan_chunks_512", "kind": "plan", "requests": 512, "page": 16, "ctx": 4096, "chunk": 1000,
         "done": 0.1, "pad": 500},
        # the heads of 16 decoding requests, out of the fused projection's rows
        {"name": "rope_decode_16", "kind": "rope", "tokens": 16, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": False, "norm": True, "far": 32768, "dtype": "bf16"},
        # a prompt chunk of 8,192 tokens
        {"name": "rope_prompt_8192", "kind": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "norm": True, "far": 8192, "dtype": "bf16"},
        # neighbouring pairs, half of each head rotated, positions near a million
        {"name": "rope_pairs_1037", "kind": "rope", "tokens": 1037, "heads": 16, "kv_heads": 8, "dim": 64, "rot": 32,
         "interleaved": True, "norm": False, "far": 1000000, "dtype": "f16"},
        # one token of each of 16 requests into its page
        {"name": "store_decode_16", "kind": "store", "mode": "pqo", "bits": 3, "tokens": 16, "kv_heads": 8,
         "dim": 128, "page": 64, "pad": 0, "dtype": "bf16"},
        # a prompt chunk padded to its launch size
        {"name": "store_prompt_8000", "kind": "store", "mode": "pqo", "bits": 4, "tokens": 8000, "kv_heads": 8,
         "dim": 128, "page": 64, "pad": 192, "dtype": "bf16"},
        # a ragged chunk with the sketch of the keys' residuals
        {"name": "store_tq_2047", "kind": "store", "mode": "tq", "bits": 3, "tokens": 2047, "kv_heads": 8,
         "dim": 128, "page": 32, "pad": 0, "dtype": "f16"},
        # one short conversation: latency
        {"name": "decode_one_700", "kind": "decode", "mode": "pqo", "bits": 3, "batch": 1, "ctx": 700, "ragged": False,
         "heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a serving batch of 16 requests of different lengths
        {"name": "decode_batch16", "kind": "decode", "mode": "pqo", "bits": 4, "batch": 16, "ctx": 16384,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # TQ records with the correction of the logits, an odd batch, small pages
        {"name": "decode_tq3_batch23", "kind": "decode", "mode": "tq", "bits": 3, "batch": 23, "ctx": 6001,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "f16"},
        # a full server: many requests of every length
        {"name": "decode_batch128", "kind": "decode", "mode": "pqo", "bits": 3, "batch": 128, "ctx": 8192,
         "ragged": True, "heads": 16, "kv_heads": 8, "dim": 128, "page": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "store", "store", "decode", "decode", "decode"])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    dim, dtype = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "plan":
        return {"kind": kind, "requests": _log(rng, 1, 512), "page": page, "ctx": _log(rng, 64, 8192),
                "chunk": rng.choice([1, 1, _log(rng, 2, 1000)]), "done": rng.choice([0.0, 0.05, 0.2]),
                "pad": rng.choice([0, _log(rng, 1, 500)])}
    if kind == "rope":
        dim = rng.choice([32, 64, 96, 128, 128, 256])
        heads = kv_heads * group
        most = 8192 * 40 * 128 * 2 // ((heads + kv_heads) * dim * SIZE[dtype])
        return {"kind": kind, "tokens": _log(rng, 1, min(16384, most)), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.4,
                "norm": rng.random() < 0.7, "far": _log(rng, 1, 1000000), "dtype": dtype}
    mode, bits = rng.choice(["pqo", "pqo", "pq", "tq"]), rng.choice([3, 4])
    if kind == "store":
        most = 8192 * 8 * 128 * 2 // (kv_heads * dim * SIZE[dtype] * (4 if mode == "tq" else 1))
        return {"kind": kind, "mode": mode, "bits": bits, "tokens": _log(rng, 1, min(most, 16384)),
                "kv_heads": kv_heads, "dim": dim, "page": page, "pad": rng.choice([0, _log(rng, 1, 300)]),
                "dtype": dtype}
    batch = _log(rng, 1, 160)
    most = 16 * 16384 * 8 * 128 // (batch * kv_heads * dim)
    return {"kind": kind, "mode": mode, "bits": bits, "batch": batch, "ctx": _log(rng, 1, min(32768, most)),
            "ragged": rng.random() < 0.7, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype}


# ---------------------------------------------------------------- inputs

EPS = 1e-6
SIGNS = 0xB1A6D4B2  # bit j: element j of a rotated block is negated


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _table(name):
    """Centroids and boundaries of the cache's codebooks of 2, 3 and 4 bits, f32 values."""
    if name == 2:
        return np.float32([-2.1573, -0.7434, 0.7434, 2.1573]), np.float32([-1.0385, 0.0, 1.0385])
    if name == 3:
        return (np.float32([-2.1573, -1.3336, -0.7434, -0.2428, 0.2428, 0.7434, 1.3336, 2.1573]),
                np.float32([-1.7455, -1.0385, -0.4931, 0.0, 0.4931, 1.0385, 1.7455]))
    r, n = np.float32(2.1573), np.arange(16, dtype=np.float32)
    step = np.float32(np.float32(2) * r) / np.float32(15)
    return -r + n * step, -r + (n[:15] + np.float32(0.5)) * step


def _codebook(case):
    """The centroids and boundaries of a case's codes, and the outer centroid that scales go by."""
    cent, bounds = _table(case["bits"] if case["mode"] == "pqo" else case["bits"] - 1)
    return cent, bounds, _table(case["bits"])[0].max()


def _dev(a):
    return torch.as_tensor(np.ascontiguousarray(a), device="cuda")


def _sign_row():
    return torch.tensor([-1.0 if (SIGNS >> j) & 1 else 1.0 for j in range(32)], device="cuda")


INV32 = float(np.float32(1) / np.sqrt(np.float32(32)))
DEC32 = float(np.float32(INV32) * np.sqrt(np.float32(32)))


def _wht(x):
    """Walsh-Hadamard transform of the last axis (32), nearest pairs first."""
    shape = x.shape
    x = x.reshape(-1, 32)
    for_pairs = x.reshape(-1, 16, 2)
    x = torch.stack((for_pairs[..., 0] + for_pairs[..., 1], for_pairs[..., 0] - for_pairs[..., 1]), -1).reshape(-1, 8, 2, 2)
    x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), -2).reshape(-1, 4, 2, 4)
    x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), -2).reshape(-1, 2, 2, 8)
    x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), -2).reshape(-1, 1, 2, 16)
    x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), -2)
    return x.reshape(shape)


def _encode(case, x):
    """Records of x [..., d]: packed codes [..., d * bits / 8] and f16 scales [..., d / 32], negative for "pqo".
    Every step is one f32 operation, as the record format has them."""
    cent, bounds, outer = _codebook(case)
    bits, d = case["bits"], x.shape[-1]
    r = _wht(x.float().reshape(*x.shape[:-1], d // 32, 32)) * (_sign_row() * INV32)
    s = (r.abs().amax(-1) * float(np.float32(1.0 / float(outer)))).clamp_min(float(np.float32(1e-10)))
    codes = torch.bucketize(r / s[..., None], _dev(bounds)).reshape(*x.shape[:-1], d // 8, 8)
    word = (codes << (torch.arange(8, device="cuda") * bits)).sum(-1)
    packed = ((word[..., None] >> (torch.arange(bits, device="cuda") * 8)) & 255).to(torch.uint8)
    half = s.to(torch.float16)
    return packed.reshape(*x.shape[:-1], d * bits // 8), (-half if case["mode"] == "pqo" else half)


def _codes(case, packed):
    """The codes [..., d] of packed records."""
    bits = case["bits"]
    byte = packed.reshape(*packed.shape[:-1], -1, bits).to(torch.int32)
    word = (byte << (torch.arange(bits, device="cuda", dtype=torch.int32) * 8)).sum(-1, dtype=torch.int32)
    codes = (word[..., None] >> (torch.arange(8, device="cuda", dtype=torch.int32) * bits)) & ((1 << bits) - 1)
    return codes.reshape(*packed.shape[:-1], -1)


def _decode(case, packed, scales):
    """The values [..., d] that records stand for, in f32, step by step as the record format has them."""
    cent = _dev(_codebook(case)[0])
    c = cent[_codes(case, packed)].reshape(*scales.shape, 32) * (_sign_row() * DEC32)
    y = (_wht(c) * INV32) * scales.float().abs()[..., None]
    return y.reshape(*packed.shape[:-1], -1)


def _activations(gen, tokens, heads, dim):
    """N(0, 1) with four channels of each head eight times as large, as key caches have them."""
    x = torch.randn((tokens, heads, dim), generator=gen, device="cuda")
    ch = torch.rand((heads, dim), generator=gen, device="cuda").argsort(1)[:, :4]
    return x * torch.ones((heads, dim), device="cuda").scatter_(1, ch, 8.0)


def _lengths(case, seed):
    b, ctx = case["batch"], case["ctx"]
    if not case["ragged"]:
        return np.full(b, ctx)
    return np.random.default_rng(seed).integers(max(1, ctx // 8), ctx + 1, size=b)


def _pools(case, pages, filled):
    """A layer's pages: codes, scales and, for "tq", signs and norms; `filled` tokens' worth of records drawn."""
    h, ps, d, bits = case["kv_heads"], case["page"], case["dim"], case["bits"]
    k, v = (torch.zeros((pages, h, ps, d * bits // 8), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, h, ps, d // 32), dtype=torch.float16, device="cuda") for _ in range(2))
    p = {"k": k, "ks": ks, "v": v, "vs": vs}
    if case["mode"] == "tq":
        p["signs"] = torch.zeros((pages, h, ps, d // 8), dtype=torch.uint8, device="cuda")
        p["norms"] = torch.zeros((pages, h, ps), dtype=torch.float16, device="cuda")
    if filled is not None:
        step = max(1, (1 << 25) // (h * ps * d))
        for at in range(0, pages, step):
            n = min(step, pages - at)
            for codes, scales in ((k, ks), (v, vs)):
                x = _activations(filled, n * ps, h, d).reshape(n, ps, h, d).transpose(1, 2)
                codes[at:at + n], scales[at:at + n] = _encode(case, x)
        if case["mode"] == "tq":
            p["signs"].random_(0, 256, generator=filled)
            p["norms"].copy_(torch.rand((pages, h, ps), generator=filled, device="cuda") * (0.03 * d ** 0.5) + 0.01 * d ** 0.5)
    return p


def _own_layer(p):
    import turboquant_amd as tq
    return tq.PagedLayer(p["k"], p["ks"].view(torch.int16), p["v"], p["vs"].view(torch.int16), p.get("signs"),
                         p["norms"].view(torch.int16) if "norms" in p else None)


def prepare(case, seed):
    return {"case": case, **globals()["_prepare_" + case["kind"]](case, seed)}


def _step_tokens(c):
    """The token rows that a step is launched for: what its requests bring as a rule, and more."""
    return int(c["requests"] * (1 if c["chunk"] == 1 else 1 + 0.17 * c["chunk"])) + c["pad"]


def _prepare_plan(c, seed):
    rng = np.random.default_rng(seed)
    b, ps = c["requests"], c["page"]
    lens = rng.integers(0, c["ctx"] + 1, size=b)
    new = np.where(rng.random(b) < 0.1, 0, 1)
    if c["chunk"] > 1:  # a third of the requests bring a chunk of a prompt
        new = np.where(rng.random(b) < 0.33, rng.integers(1, c["chunk"] + 1, size=b), new)
    new = np.where(rng.random(b) < c["done"], -1, new)
    held = -(-lens // ps)
    width = -(-(c["ctx"] + c["chunk"]) // ps)
    pages = b * width
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((b, width), -1, np.int32)
    table[np.arange(width)[None] < held[:, None]] = ids[:held.sum()]
    free = np.concatenate((ids[held.sum():], np.zeros(held.sum(), np.int32)))
    return {"kv_lens": _dev(lens.astype(np.int32)), "new_lens": _dev(new.astype(np.int32)), "table": _dev(table),
            "free": _dev(free), "free_count": _dev(np.int32([pages - held.sum()])), "tokens": _step_tokens(c),
            "kv_out": torch.zeros(b, dtype=torch.int32, device="cuda"),
            "free_out": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_rope(c, seed):
    g = _gen(seed)
    hq, hk, d, t = c["heads"], c["kv_heads"], c["dim"], c["tokens"]
    rows = torch.randn((t, (hq + 2 * hk) * d), generator=g, device="cuda").mul_(1.7).to(DTYPES[c["dtype"]])
    last = torch.randint(0, c["far"] + 1, (1,), generator=g, device="cuda")
    positions = (last + torch.arange(t, device="cuda") % 4096).to(torch.int32)
    freq = 1e6 ** (-np.arange(c["rot"] // 2) / max(1, c["rot"] // 2))
    w = [torch.rand(d, generator=g, device="cuda").add_(0.5).to(DTYPES[c["dtype"]]) for _ in range(2)]
    return {"q": rows[:, :hq * d].view(t, hq, d), "k": rows[:, hq * d:(hq + hk) * d].view(t, hk, d),
            "positions": positions, "inv_freq": _dev(freq.astype(np.float32)),
            "wq": w[0] if c["norm"] else None, "wk": w[1] if c["norm"] else None}


def _prepare_store(c, seed):
    g = _gen(seed)
    h, d, ps, t = c["kv_heads"], c["dim"], c["page"], c["tokens"]
    rows = torch.cat([_activations(g, t + c["pad"], h, d), _activations(g, t + c["pad"], h, d)], 1).to(DTYPES[c["dtype"]])
    pages = -(-t // ps) + 3
    # runs of a few requests in pages in any order, one run after the other's last page
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(t, device="cuda") + (5 if t + 5 <= (pages - 1) * ps else 0)
    slots = torch.full((t + c["pad"],), -1, dtype=torch.int64, device="cuda")
    slots[:t] = order[at // ps] * ps + at % ps
    p = _pools(c, pages, None)
    s = {"k": rows[:, :h], "v": rows[:, h:], "slots": slots, "pools": p, "rmat": None,
         "out": [torch.zeros((t + c["pad"], h, d), dtype=DTYPES[c["dtype"]], device="cuda") for _ in range(2)]}
    if c["mode"] == "tq":
        s["rmat"] = torch.randint(-2 ** 31, 2 ** 31, (d * d // 32,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    if own:
        s["layer"] = _own_layer(p)
    return s


def _prepare_decode(c, seed):
    g = _gen(seed)
    lens = _lengths(c, seed)
    ps, b, d = c["page"], c["batch"], c["dim"]
    held = -(-lens // ps)
    pages = int(held.sum()) + 2
    ids = np.random.default_rng(seed + 1).permutation(pages).astype(np.int32)
    width = -(-c["ctx"] // ps)
    table = np.full((b, width), -1, np.int32)
    table[np.arange(width)[None] < held[:, None]] = ids[:held.sum()]
    p = _pools(c, pages, g)
    s = {"q": torch.randn((b, c["heads"], d), generator=g, device="cuda").to(DTYPES[c["dtype"]]), "pools": p,
         "table": _dev(table), "lens": _dev(lens.astype(np.int32)), "rmat": None}
    if c["mode"] == "tq":
        s["rmat"] = torch.randint(-2 ** 31, 2 ** 31, (d * d // 32,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    if own:
        import turboquant_amd as tq
        s["layer"] = _own_layer(p)
        s["ws"] = tq.AttentionWorkspace(b, c["heads"], c["kv_heads"], d, c["ctx"])
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state, state["case"])


def _outliers(case):
    import turboquant_amd as tq
    return tq.cache.OUTLIER_ALL if case["mode"] == "pqo" else 0


def _own_plan(s, c):
    import turboquant_amd as tq
    p = tq.paged_plan(s["kv_lens"], s["new_lens"], s["table"], s["free"], s["free_count"], c["page"], s["tokens"],
                      kv_lens_out=s["kv_out"], free_count_out=s["free_out"])
    return {"slots": p.slots, "positions": p.positions, "starts": p.starts, "lens": p.kv_lens, "free": p.free_count,
            "table": s["table"], "stack": s["free"]}


def _own_rope(s, c):
    import turboquant_amd as tq
    return tq.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["wq"], s["wk"], EPS, c["interleaved"])


def _own_store(s, c):
    import turboquant_amd as tq
    tq.paged_store(s["layer"], s["slots"], s["k"], s["v"], c["bits"], _outliers(c), sign_matrix=s["rmat"])
    out = dict(zip("kv", tq.paged_load(s["layer"], s["slots"], c["bits"], _outliers(c), out=s["out"])))
    if c["mode"] == "tq":
        out.update(signs=s["pools"]["signs"], norms=s["pools"]["norms"])
    return out


def _own_decode(s, c):
    import turboquant_amd as tq
    return tq.paged_decode_attention(s["q"], s["layer"], s["table"], s["lens"], c["bits"], c["ctx"], c["dim"] ** -0.5,
                                     s["ws"], _outliers(c), sign_matrix=s["rmat"])


def _ceil(a, b):
    return (a + (b - 1)) // b


def _plain_plan(s, c):
    ps, (b, width), tokens = c["page"], s["table"].shape, s["tokens"]
    lens, new, table, stack = s["kv_lens"].long(), s["new_lens"].long(), s["table"], s["free"]
    col = torch.arange(width, device="cuda")[None]
    # requests that are done give their pages back first
    held = _ceil(lens, ps)
    back = torch.where(new < 0, held, 0)
    to = (s["free_count"].long() + back.cumsum(0) - back)[:, None] + col
    to = torch.where(col < back[:, None], to, stack.numel())
    grown = torch.cat((stack, stack[:1])).scatter(0, to.reshape(-1), table.reshape(-1))
    stack.copy_(grown[:-1])
    avail = s["free_count"].long() + back.sum()
    # what each request needs, and whether it can have it
    n = new.clamp_min(0)
    ends = n.cumsum(0)
    room = (lens + n <= width * ps) & (ends <= tokens)
    need = torch.where(room, _ceil(lens + n, ps) - held, 0)
    taken = need.cumsum(0)
    fits = room & ((need == 0) | (taken <= avail))
    # its new pages, from the top of the stack down
    j = col - held[:, None]
    new_page = (j >= 0) & (j < torch.where(fits, need, 0)[:, None])
    pick = (avail - 1 - (taken - need))[:, None] - j
    table.copy_(torch.where(new_page, stack[pick.clamp(0, stack.numel() - 1)], table))
    after = torch.where(new < 0, 0, torch.where(fits, lens + n, lens)).to(torch.int32)
    free = (avail - torch.where(fits, need, 0).sum()).to(torch.int32).reshape(1)
    # its tokens
    i = torch.arange(tokens, device="cuda")
    owner = (i[:, None] >= ends[None]).sum(1)
    own_by = owner.clamp_max(b - 1)
    pos = lens[own_by] + i - (ends - n)[own_by]
    live = (owner < b) & fits[own_by]
    page = table[own_by, (pos // ps).clamp(0, width - 1)].long()
    slots = torch.where(live, page * ps + pos % ps, -1)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32)
    return {"slots": slots, "positions": torch.where(live, pos, -1).to(torch.int32), "starts": starts, "lens": after,
            "free": free, "table": table, "stack": stack}


def _plain_rope(s, c):
    rot, angle = c["rot"], s["positions"].double()[:, None] * s["inv_freq"].double()[None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def one(x, w):
        y = x.float()
        if w is not None:
            y = y / ((y * y).mean(-1, keepdim=True) + EPS).sqrt() * w.float()
        r, rest = y[..., :rot], y[..., rot:]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((r, rest), -1).to(x.dtype)

    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _rows_of(words, d):
    """The +-1 matrix whose row j is d / 32 words of `words`, a set bit for -1."""
    bits = (words.reshape(d, d // 32, 1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    return 1.0 - 2.0 * bits.reshape(d, d).float()


def _plain_store(s, c):
    p, ps, d = s["pools"], c["page"], c["dim"]
    rows = (s["slots"] >= 0).nonzero()[:, 0]
    slots = s["slots"][rows]
    page, off = slots // ps, slots % ps
    k = s["k"][rows]
    p["k"][page, :, off], p["ks"][page, :, off] = _encode(c, k)
    p["v"][page, :, off], p["vs"][page, :, off] = _encode(c, s["v"][rows])
    back = _decode(c, p["k"][page, :, off], p["ks"][page, :, off])
    s["out"][0][rows] = back.to(s["out"][0].dtype)
    s["out"][1][rows] = _decode(c, p["v"][page, :, off], p["vs"][page, :, off]).to(s["out"][1].dtype)
    out = {"k": s["out"][0], "v": s["out"][1]}
    if c["mode"] == "tq":
        # the sketch's sums run in element order, one f32 rounding a step, which fixes its bits
        r, m = k.float() - back, _rows_of(s["rmat"], d)
        norm, prod = torch.zeros_like(r[..., 0]), torch.zeros_like(r)
        for j in range(d):
            norm = norm + r[..., j] * r[..., j]
            prod = prod + r[..., j:j + 1] * m[:, j]
        inv = float(np.float32(1) / np.sqrt(np.float32(d)))
        bits = (prod * inv >= 0).to(torch.uint8).reshape(*prod.shape[:-1], d // 8, 8)
        byte = (bits << torch.arange(8, device="cuda", dtype=torch.uint8)).sum(-1, dtype=torch.uint8)
        p["signs"][page, :, off], p["norms"][page, :, off] = byte, norm.sqrt().to(torch.float16)
        out.update(signs=p["signs"], norms=p["norms"])
    return out


def _plain_decode(s, c):
    p, ps, d, hk = s["pools"], c["page"], c["dim"], c["kv_heads"]
    b, hq = s["q"].shape[:2]
    t = torch.arange(c["ctx"], device="cuda")
    seen = t[None] < s["lens"][:, None]
    page = torch.where(seen, s["table"][:, t // ps], 0).long()
    off = (t % ps)[None].expand_as(page)
    k = _decode(c, p["k"][page, :, off], p["ks"][page, :, off]).permute(0, 2, 3, 1).contiguous()
    q = s["q"].float().reshape(b, hk, hq // hk, d)
    x = torch.matmul(q, k)
    del k
    if c["mode"] == "tq":
        rq = (torch.matmul(q, _rows_of(s["rmat"], d).t().contiguous())) * d ** -0.5
        bit = (p["signs"][page, :, off][..., None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
        sign = (2.0 * bit.flatten(-2).float() - 1.0).permute(0, 2, 3, 1).contiguous()
        norm = p["norms"][page, :, off].float().permute(0, 2, 1)[:, :, None]
        x = x + torch.matmul(rq, sign) * norm * (math.sqrt(math.pi / 2) / math.sqrt(d))
        del sign, bit
    x = torch.where(seen[:, None, None], x * d ** -0.5, -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.where(seen[:, None, None], torch.exp(x - torch.where(top > -math.inf, top, 0.0)), 0.0)
    v = _decode(c, p["v"][page, :, off], p["vs"][page, :, off]).permute(0, 2, 1, 3).contiguous()
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w, v) / torch.where(total > 0, total, 1.0)
    return out.reshape(b, hq, d).to(s["q"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "plan":
        # per request its length and new length in, length and start out; per token a slot and a position
        tokens = _step_tokens(c)
        return {"bytes": c["requests"] * 16 + tokens * 12, "flops": tokens * 4}
    d, size = c["dim"], SIZE[c["dtype"]]
    if c["kind"] == "rope":
        n = c["tokens"] * (c["heads"] + c["kv_heads"]) * d
        return {"bytes": 2 * n * size, "flops": n * (6 if c["norm"] else 3)}
    rec = d * c["bits"] // 8 + d // 16
    sketch = d // 8 + 2 if c["mode"] == "tq" else 0
    if c["kind"] == "store":
        n = 2 * c["tokens"] * c["kv_heads"]  # stored, and read back
        return {"bytes": n * (2 * d * size + 2 * rec) + n // 2 * sketch, "flops": n * d * 16 + (n * d * d if sketch else 0)}
    tokens = int(_lengths(c, 0).sum())
    return {"bytes": tokens * c["kv_heads"] * (2 * rec + sketch) + 2 * c["batch"] * c["heads"] * d * size,
            "flops": tokens * c["heads"] * d * (6 if sketch else 4)}


# ---------------------------------------------------------------- the same in 64 bits
# Records are defined by 32-bit steps, so `store` has its values from those steps, one element of numpy at a time;
# what is computed from records is 64-bit.

def exact(case, seed):
    if case["kind"] == "plan":
        return None
    return globals()["_exact_" + case["kind"]](prepare(case, seed), case)


def _exact_rope(s, c):
    pos, freq = s["positions"].cpu().numpy().astype(np.float64), s["inv_freq"].cpu().numpy().astype(np.float64)
    turn = np.exp(1j * (pos[:, None] * freq[None]))
    n = c["rot"] // 2

    def one(x, w):
        y = x.double().cpu().numpy()
        if w is not None:
            y = y * w.double().cpu().numpy() / np.sqrt(np.square(y).mean(-1, keepdims=True) + EPS)
        first, second = (np.arange(n) * 2, np.arange(n) * 2 + 1) if c["interleaved"] else (np.arange(n), np.arange(n) + n)
        z = (y[..., first] + 1j * y[..., second]) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _hadamard():
    i = np.arange(32)
    return np.where(np.vectorize(lambda v: bin(v).count("1") & 1)(i[:, None] & i[None]), -1.0, 1.0)


def _bits(bytes_):
    """The bits of bytes, the lowest first, as 64-bit zeros and ones."""
    return torch.stack([bytes_.bitwise_and(1 << i).ne(0) for i in range(8)], -1).flatten(-2).double()


def _values(c, packed, scales):
    """What records stand for, in 64 bits."""
    codes = torch.matmul(_bits(packed).reshape(*packed.shape[:-1], -1, c["bits"]), _dev(2.0 ** np.arange(c["bits"])))
    cent = _dev(_codebook(c)[0].astype(np.float64))[codes.long()].reshape(*scales.shape, 32) * _sign_row().double()
    y = torch.matmul(cent, _dev(_hadamard())) / math.sqrt(32.0)
    return (y * scales.double().abs()[..., None]).reshape(*packed.shape[:-1], -1)


def _f32_steps(c, x):
    """x [..., 32] through a record: f32 steps held in 64 bits, then the stored value in 64 bits."""
    f = lambda a: a.astype(np.float32).astype(np.float64)  # noqa: E731
    cent, bounds, outer = (np.asarray(a, np.float64) for a in _codebook(c))
    sign = np.array([-1.0 if (SIGNS >> j) & 1 else 1.0 for j in range(32)])
    r, i = x, np.arange(32)
    for h in (1, 2, 4, 8, 16):
        r = f(np.where(i & h, r[..., i ^ h] - r, r + r[..., i ^ h]))
    r = f(r * (sign * INV32))
    s = np.maximum(f(np.abs(r).max(-1) * float(np.float32(1.0 / float(outer)))), float(np.float32(1e-10)))
    v = f(r / s[..., None])
    scale = s.astype(np.float16).astype(np.float64)
    y = (cent[np.searchsorted(bounds, v, side="left")] * sign) @ _hadamard()
    return y / math.sqrt(32.0) * scale[..., None]


def _exact_store(s, c):
    out = {}
    live = s["slots"].cpu().numpy() >= 0
    for name in "kv":
        x = s[name].double().cpu().numpy()
        y = _f32_steps(c, x.reshape(*x.shape[:-1], -1, 32)).reshape(x.shape)
        out[name] = np.where(live[:, None, None], y, 0.0)
    if c["mode"] == "tq":
        slots = s["slots"].cpu().numpy()[live]
        norms = np.zeros(tuple(s["pools"]["norms"].shape))
        norms[slots // c["page"], :, slots % c["page"]] = np.sqrt(np.square(s["k"].double().cpu().numpy() - out["k"]).sum(-1))[live]
        out.update(signs=None, norms=norms)  # a sign is that of an f32 sum
    return out


def _exact_decode(s, c):
    p, ps, d, hk = s["pools"], c["page"], c["dim"], c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    m = _rows_of(s["rmat"], d).double() if c["mode"] == "tq" else None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][b, :-(-n // ps)].long()
        rec = {name: t[pages].transpose(0, 1).flatten(1, 2)[:, :n] for name, t in p.items()}
        k, v = _values(c, rec["k"], rec["ks"]), _values(c, rec["v"], rec["vs"])
        q = s["q"][b].double().reshape(hk, -1, d)
        x = torch.matmul(q, k.transpose(1, 2).contiguous())
        if m is not None:
            bit = _bits(rec["signs"])
            rq = torch.matmul(q, m.t().contiguous()) / math.sqrt(d)
            x = x + torch.matmul(rq, (2 * bit - 1).transpose(1, 2).contiguous()) * rec["norms"].double()[:, None] * math.sqrt(math.pi / 2 / d)
        out[b] = torch.matmul(torch.softmax(x / math.sqrt(d), -1), v).reshape(-1, d)
    return out

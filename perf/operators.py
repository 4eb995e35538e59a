"""Cases that time the paged-cache operators of the kernel level: q/k norm with rotation
(`qora_qk_norm_rope`), append to a paged KV cache (`qora_paged_append`) and attention over
it (`qora_paged_attention`).

`own` false: `run` computes each operator in elementary torch operations, in 32 bits,
rounded once at the end. `own` true: `run` calls the entry points of the framework.

Layout shared by the cases. Rows are tokens, row-major [rows][heads][head_dim]; q, k and v
are views of one joined row (as a joined projection writes them) where a case says so.
Sequence s owns the rows q_start[s] .. q_start[s+1]-1, which are its newest positions: with
n of them and kv_len[s] = L positions in all, row i of the sequence sits at L - n + i.
Position p of sequence s lies in page table[s][p // page_size], slot p % page_size; a
page is [slot][head][head_dim] ("slot") or [head][slot][head_dim] ("head")."""
import importlib
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
WORK = 64 << 20  # bytes of scratch a serving program sets aside once for the attention


# ------------------------------------------------------------------ cases
def listed():
    heads = {"q_heads": 16, "kv_heads": 4, "dim": 128}
    return [
        # one new token of one request: what counts is the call itself
        {"name": "norm rope 1 row f32", "op": "norm", **heads, "act": "f32", "rows": 1, "rot": 64, "gains": True, "top": 65536},
        # a long prompt's q and k out of the joined projection, an odd number of rows
        {"name": "norm rope 8191 rows bf16", "op": "norm", **heads, "act": "bf16", "rows": 8191, "rot": 64, "gains": True, "top": 65536},
        # a batched decode step: 32 requests, one row each, far-apart positions
        {"name": "append 32 tokens f32 to f16", "op": "append", **heads, "act": "f32", "kv": "f16", "page": 16, "layout": "head",
         "seqs": 32, "new_min": 1, "new_max": 1, "old_min": 100, "old_max": 4000, "rot": 64, "gains": False, "lens": 1, "top": 65536},
        # one ragged chunk of a prompt into the reference's cache type
        {"name": "append 509 rows f32 to f32", "op": "append", **heads, "act": "f32", "kv": "f32", "page": 16, "layout": "head",
         "seqs": 1, "new_min": 509, "new_max": 509, "old_min": 1531, "old_max": 1531, "rot": 64, "gains": False, "lens": 2, "top": 65536},
        # prompts of several requests in one pass, with the norms of q and k
        {"name": "append 5 prompts bf16", "op": "append", **heads, "act": "bf16", "kv": "bf16", "page": 64, "layout": "slot",
         "seqs": 5, "new_min": 700, "new_max": 2600, "old_min": 0, "old_max": 0, "rot": 64, "gains": True, "lens": 3, "top": 65536},
        # single-token form, one request with a 32K-token cache
        {"name": "one token over 32K f32/f16", "op": "attend", **heads, "act": "f32", "kv": "f16", "page": 64, "layout": "head",
         "seqs": 1, "new_min": 1, "new_max": 1, "old_min": 32767, "old_max": 32767, "window": 0, "lens": 4},
        # a batched decode step over ragged short caches of the reference's type
        {"name": "32 tokens ragged f32/f32", "op": "attend", **heads, "act": "f32", "kv": "f32", "page": 16, "layout": "head",
         "seqs": 32, "new_min": 1, "new_max": 1, "old_min": 60, "old_max": 4000, "window": 0, "lens": 5},
        # a large batch of requests, one token each
        {"name": "128 tokens ragged f16", "op": "attend", **heads, "act": "f16", "kv": "f16", "page": 16, "layout": "slot",
         "seqs": 128, "new_min": 1, "new_max": 1, "old_min": 200, "old_max": 8000, "window": 0, "lens": 6},
        # the next chunk of a long prompt over what is cached of it
        {"name": "512 rows over 8K f32/f16", "op": "attend", **heads, "act": "f32", "kv": "f16", "page": 64, "layout": "head",
         "seqs": 1, "new_min": 512, "new_max": 512, "old_min": 7680, "old_max": 7680, "window": 0, "lens": 7},
        # a prompt on the reference's cache type, odd length
        {"name": "prompt 1021 f32/f32", "op": "attend", **heads, "act": "f32", "kv": "f32", "page": 16, "layout": "head",
         "seqs": 1, "new_min": 1021, "new_max": 1021, "old_min": 0, "old_max": 0, "window": 0, "lens": 8},
        # chunks and single tokens of different requests in one pass, sliding window
        {"name": "mixed chunks bf16 window", "op": "attend", **heads, "act": "bf16", "kv": "bf16", "page": 32, "layout": "slot",
         "seqs": 8, "new_min": 1, "new_max": 900, "old_min": 0, "old_max": 5000, "window": 2000, "lens": 9},
        # a whole long prompt at once
        {"name": "prompt 8192 f16", "op": "attend", **heads, "act": "f16", "kv": "f16", "page": 64, "layout": "slot",
         "seqs": 1, "new_min": 8192, "new_max": 8192, "old_min": 0, "old_max": 0, "window": 0, "lens": 10},
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attend", "attend", "attend"])
    dim = rng.choice([128, 128, 128, 64])
    kv_heads, group = rng.choice([4, 4, 2, 8, 1]), rng.choice([4, 4, 1, 2, 3, 8])
    c = {"op": op, "q_heads": kv_heads * min(group, 16 // kv_heads), "kv_heads": kv_heads, "dim": dim}
    c["act"], kv = rng.choice([("f32", "f16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "norm":
        return {**c, "rows": _log(rng, 1, 8191), "rot": rng.choice([dim // 2, dim // 2, dim // 4]), "gains": rng.random() < 0.6, "top": 65536}
    c.update(kv=kv, page=rng.choice([16, 16, 32, 64, 128, 8, 20]), layout=rng.choice(["slot", "head"]), lens=rng.randrange(1 << 20))
    if op == "append":
        seqs = _log(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8000 // seqs))
        old = _log(rng, 1, min(4000, 128000 // seqs))
        return {**c, "seqs": seqs, "new_min": max(1, new // 3), "new_max": new, "old_min": old // 8, "old_max": old, "rot": rng.choice([dim // 2, dim // 2, dim // 4]),
                "gains": rng.random() < 0.4, "top": 65536}
    # single tokens, a few tokens (as checked drafts are), chunks; no more than the largest listed cases ask for
    kind = rng.choice(["token", "token", "few", "chunk", "chunk"])
    seqs = _log(rng, 1, {"token": 128, "few": 32, "chunk": 8}[kind])
    new = {"token": 1, "few": rng.randint(2, 12), "chunk": _log(rng, 13, 4000 // seqs)}[kind]
    old = _log(rng, 1, min(32000, {"token": 250000 // seqs, "few": 60000 // seqs, "chunk": (1 << 25) // (seqs * new)}[kind]))
    window = _log(rng, 16, 8000) if rng.random() < 0.25 else 0
    return {**c, "seqs": seqs, "new_min": max(1, new // 4), "new_max": new, "old_min": old // 6, "old_max": old, "window": window}


def _lengths(case):
    """(new rows, cached positions in all) of each sequence."""
    r = random.Random(case["lens"])
    new = [r.randint(case["new_min"], case["new_max"]) for _ in range(case["seqs"])]
    return new, [n + r.randint(case["old_min"], case["old_max"]) for n in new]


# ------------------------------------------------------------------ inputs
def _tables(g, top, rot):
    inv = 10000.0 ** (-torch.arange(rot, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, hq, hk, d = TYPES[case["act"]], case["q_heads"], case["kv_heads"], case["dim"]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    st = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if case["op"] == "norm":
        rows = case["rows"]
        st["qkv"] = (rand(rows, (hq + 2 * hk) * d) * (0.5 + 1.5 * torch.rand(rows, 1, generator=g, device="cuda"))).to(t)
        st["pos"] = torch.randint(0, case["top"], (1,), generator=g, device="cuda", dtype=torch.int32) if rows == 1 else (
            torch.arange(rows, device="cuda", dtype=torch.int32) + torch.randint(0, case["top"] - rows, (1,), generator=g, device="cuda", dtype=torch.int32))
        st["q_out"], st["k_out"] = (torch.empty(rows, h * d, dtype=t, device="cuda") for h in (hq, hk))
    else:
        new, total = _lengths(case)
        rows, ps, seqs = sum(new), case["page"], case["seqs"]
        need = [-(-x // ps) for x in total]
        pages, wide = sum(need) + max(1, sum(need) // 8), max(need)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        first = torch.tensor([sum(need[:s]) for s in range(seqs)], device="cuda")[:, None] + torch.arange(wide, device="cuda")[None]
        st["table"] = torch.where(torch.arange(wide, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None], order[first.clamp(max=pages - 1)], 0).to(torch.int32)
        start = [sum(new[:s]) for s in range(seqs + 1)]
        st["start"], st["len"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (start, total))
        shape = (pages, ps, hk, d) if case["layout"] == "slot" else (pages, hk, ps, d)
        st["kp"], st["vp"] = (rand(*shape).to(TYPES[case["kv"]]) for _ in range(2))
        st["rows"], st["pages"], st["longest"], st["most"], st["wide"] = rows, pages, max(total), max(new), wide
        if case["op"] == "append":
            st["qkv"] = (rand(rows, (hq + 2 * hk) * d) * 1.5).to(t)
            st["q_out"] = torch.empty(rows, hq * d, dtype=t, device="cuda")
        else:
            st["q"] = (rand(rows, hq * d) * 1.5).to(t)
            st["out"] = torch.empty(rows, hq * d, dtype=t, device="cuda")
            st["lse"] = torch.empty(rows, hq, dtype=torch.float32, device="cuda")
            st["work"] = torch.empty(WORK, dtype=torch.uint8, device="cuda")
    if case["op"] != "attend":
        st["cos"], st["sin"] = _tables(g, case["top"], case["rot"])
        if case["gains"]:
            st["q_gain"], st["k_gain"] = (1.0 + 0.2 * rand(d) for _ in range(2))
    return st


# ------------------------------------------------------------------ plain forms
def _norm_rope(x, gain, cos, sin, rot):
    """x [rows][heads][dim] f32, cos/sin [rows][rot]: the norm (with a gain), then the rotation."""
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
    a, b, c, s = x[..., :rot], x[..., rot:2 * rot], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * rot:]], -1)


def _places(st):
    """Of each row: its sequence and its position there."""
    rows = torch.arange(st["rows"], device="cuda", dtype=torch.int32)
    s = torch.bucketize(rows, st["start"][1:], right=True)
    n = st["start"][1:] - st["start"][:-1]
    return s, (st["len"] - n)[s] + rows - st["start"][s]


def _by_slot(st, pages):
    return pages if st["case"]["layout"] == "slot" else pages.transpose(1, 2)


def _plain_norm(st):
    c = st["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    x = st["qkv"][:, :(hq + hk) * d].float().view(-1, hq + hk, d)
    cos, sin = st["cos"][st["pos"].long()], st["sin"][st["pos"].long()]
    q, k = (_norm_rope(y, st.get(g), cos, sin, c["rot"]) for y, g in ((x[:, :hq], "q_gain"), (x[:, hq:], "k_gain")))
    return {"q": q.to(st["q_out"].dtype).flatten(1), "k": k.to(st["k_out"].dtype).flatten(1)}


def _plain_append(st):
    c = st["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    x = st["qkv"].float().view(-1, hq + 2 * hk, d)
    s, p = _places(st)
    cos, sin = st["cos"][p.long()], st["sin"][p.long()]
    q, k = (_norm_rope(y, st.get(g), cos, sin, c["rot"]) for y, g in ((x[:, :hq], "q_gain"), (x[:, hq:hq + hk], "k_gain")))
    page, slot = st["table"][s, (p // c["page"]).long()].long(), (p % c["page"]).long()
    _by_slot(st, st["kp"])[page, slot] = k.to(st["kp"].dtype)
    _by_slot(st, st["vp"])[page, slot] = x[:, hq + hk:].to(st["vp"].dtype)
    return {"q": q.to(st["q_out"].dtype).flatten(1), "k_pages": st["kp"], "v_pages": st["vp"]}


def _plain_attend(st):
    c = st["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    at = torch.arange(st["longest"], device="cuda")
    page = st["table"][:, at // c["page"]].long()
    k, v = (_by_slot(st, x)[page, at % c["page"]].float() for x in (st["kp"], st["vp"]))  # [seqs][positions][heads][dim]
    n = (st["start"][1:] - st["start"][:-1]).long()
    i = torch.arange(st["most"], device="cuda")
    row = (st["start"][:-1].long()[:, None] + i).clamp(max=st["rows"] - 1)
    q = st["q"].float().view(-1, hk, hq // hk, d)[row]  # [seqs][new][kv heads][group][dim]
    x = torch.einsum("snhgd,slhd->shgnl", q, k) / math.sqrt(d)
    p = (st["len"].long() - n)[:, None] + i  # [seqs][new]
    seen = (at <= p[..., None]) & (i < n[:, None])[..., None]
    if c["window"]:
        seen &= at > p[..., None] - c["window"]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    o = torch.einsum("shgnl,slhd->snhgd", w, v) / torch.where(total > 0, total, torch.ones_like(total)).permute(0, 3, 1, 2, 4)
    lse = (top + torch.log(total)).permute(0, 3, 1, 2, 4)
    s, at = _places(st)
    i = (at - (st["len"] - n)[s]).long()
    return {"out": o[s, i].to(st["out"].dtype).flatten(1), "lse": lse[s, i].flatten(1)}


# ------------------------------------------------------------------ the framework's calls
def _own_norm(st):
    eng, c = importlib.import_module("qora-llm_b200").engine, st["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    x, wide = st["qkv"], (hq + 2 * hk) * d
    eng.qk_norm_rope(x.data_ptr(), x.data_ptr() + hq * d * x.element_size(), st["q_out"].data_ptr(), st["k_out"].data_ptr(),
                     c["rows"], hq, hk, d, st["pos"].data_ptr(), st["cos"].data_ptr(), st["sin"].data_ptr(), c["top"], c["rot"],
                     st["q_gain"].data_ptr() if c["gains"] else None, st["k_gain"].data_ptr() if c["gains"] else None, EPS,
                     dtype=c["act"], q_stride=wide, k_stride=wide, stream=st["stream"])
    return {"q": st["q_out"], "k": st["k_out"]}


def _strides(c):
    hk, d, ps = c["kv_heads"], c["dim"], c["page"]
    return (ps * hk * d, d, hk * d) if c["layout"] == "slot" else (ps * hk * d, ps * d, d)  # page, head, slot


def _own_append(st):
    eng, c = importlib.import_module("qora-llm_b200").engine, st["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    x, wide, e = st["qkv"], (hq + 2 * hk) * d, st["qkv"].element_size()
    at = x.data_ptr()
    eng.paged_append(at + hq * d * e, at + (hq + hk) * d * e, st["rows"], hk, d, st["kp"].data_ptr(), st["vp"].data_ptr(), st["pages"], c["page"],
                     st["start"].data_ptr(), st["len"].data_ptr(), st["table"].data_ptr(), st["wide"], c["seqs"],
                     q_ptr=at, q_out_ptr=st["q_out"].data_ptr(), q_heads=hq, cos_ptr=st["cos"].data_ptr(), sin_ptr=st["sin"].data_ptr(),
                     rope_rows=c["top"], rope_half_dim=c["rot"], q_gamma_ptr=st["q_gain"].data_ptr() if c["gains"] else None,
                     k_gamma_ptr=st["k_gain"].data_ptr() if c["gains"] else None, eps=EPS, dtype=c["act"], kv_dtype=c["kv"],
                     q_stride=wide, k_stride=wide, v_stride=wide, page_strides=_strides(c), stream=st["stream"])
    return {"q": st["q_out"], "k_pages": st["kp"], "v_pages": st["vp"]}


def _own_attend(st):
    eng, c = importlib.import_module("qora-llm_b200").engine, st["case"]
    eng.paged_attention(st["q"].data_ptr(), st["out"].data_ptr(), st["rows"], c["q_heads"], c["kv_heads"], c["dim"],
                        st["kp"].data_ptr(), st["vp"].data_ptr(), st["pages"], c["page"],
                        st["start"].data_ptr(), st["len"].data_ptr(), st["table"].data_ptr(), st["wide"], c["seqs"], st["most"],
                        st["work"].data_ptr(), WORK, window=c["window"], lse_ptr=st["lse"].data_ptr(),
                        dtype=c["act"], kv_dtype=c["kv"], page_strides=_strides(c), stream=st["stream"])
    return {"out": st["out"], "lse": st["lse"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "append": _own_append, "attend": _own_attend}[op](state)
    return {"norm": _plain_norm, "append": _plain_append, "attend": _plain_attend}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def _attended(n, total, window):
    """Pairs of a new row and a position that it attends to, and the positions that any row attends to."""
    pairs = 0
    for i in range(n):
        p = total - n + i + 1
        pairs += min(p, window) if window else p
    return pairs, min(total, window + n - 1) if window else total


def work(case):
    hq, hk, d, e = case["q_heads"], case["kv_heads"], case["dim"], SIZE[case["act"]]
    if case["op"] == "norm":
        rows, rot = case["rows"], case["rot"]
        return {"bytes": rows * (2 * (hq + hk) * d * e + 8 * rot + 4), "flops": rows * (hq + hk) * d * 8}
    new, total = _lengths(case)
    rows, meta = sum(new), 4 * (2 * case["seqs"] + 1)
    if case["op"] == "append":
        rot = case["rot"]
        return {"bytes": rows * (hq * d * 2 * e + 2 * hk * d * (e + SIZE[case["kv"]]) + 8 * rot + 4) + meta, "flops": rows * (hq + hk) * d * 8}
    pairs, seen = (sum(x) for x in zip(*(_attended(n, t, case["window"]) for n, t in zip(new, total))))
    return {"bytes": rows * hq * (2 * d * e + 4) + seen * 2 * hk * d * SIZE[case["kv"]] + -(-seen // case["page"]) * 4 + meta,
            "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------------ the definition, in 64 bits
def _turned(x, gain, pos, st, rot):
    """x [heads][dim] rows at positions pos, 64 bits, one pair of elements at a time."""
    x = x.double()
    if gain is not None:
        x = gain.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    z = torch.complex(x[..., :rot], x[..., rot:2 * rot])
    z = z * torch.complex(st["cos"].double()[pos], st["sin"].double()[pos])[:, None]
    y = x.clone()
    y[..., :rot], y[..., rot:2 * rot] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm":
        x, pos = st["qkv"].view(-1, hq + 2 * hk, d), st["pos"].long()
        return {"q": _turned(x[:, :hq], st.get("q_gain"), pos, st, case["rot"]).flatten(1),
                "k": _turned(x[:, hq:hq + hk], st.get("k_gain"), pos, st, case["rot"]).flatten(1)}
    new, total = _lengths(case)
    ps, table, row = case["page"], st["table"].tolist(), 0
    if case["op"] == "append":
        x, qs, kp, vp = st["qkv"].view(-1, hq + 2 * hk, d), [], st["kp"].double(), st["vp"].double()
        for s, (n, t) in enumerate(zip(new, total)):
            pos = torch.arange(t - n, t, device="cuda")
            y = x[row:row + n]
            qs.append(_turned(y[:, :hq], st.get("q_gain"), pos, st, case["rot"]))
            k, v = _turned(y[:, hq:hq + hk], st.get("k_gain"), pos, st, case["rot"]), y[:, hq + hk:].double()
            page, slot = torch.tensor(table[s], device="cuda")[pos // ps], pos % ps
            for pool, z in ((kp, k), (vp, v)):
                if case["layout"] == "slot":
                    pool[page, slot] = z
                else:
                    pool[page, :, slot] = z
            row += n
        return {"q": torch.cat(qs).flatten(1), "k_pages": kp, "v_pages": vp}
    out = torch.zeros(st["rows"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((st["rows"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for s, (n, t) in enumerate(zip(new, total)):
        page = torch.tensor(table[s][: -(-t // ps)], device="cuda")
        for h in range(hk):
            pick = (lambda pool: pool[page, :, h] if case["layout"] == "slot" else pool[page, h])  # noqa: E731
            k, v = (pick(pool).reshape(-1, d)[:t].double() for pool in (st["kp"], st["vp"]))
            for i in range(0, n, 2048):
                m = min(2048, n - i)
                p = torch.arange(t - n + i, t - n + i + m, device="cuda")[:, None]
                j = torch.arange(t, device="cuda")[None]
                hide = j > p
                if case["window"]:
                    hide = hide | (j <= p - case["window"])
                for a in range(h * (hq // hk), (h + 1) * (hq // hk)):
                    z = (st["q"].view(-1, hq, d)[row + i:row + i + m, a].double() @ k.T) * d ** -0.5
                    z[hide] = -math.inf
                    lse[row + i:row + i + m, a] = torch.logsumexp(z, 1)
                    out[row + i:row + i + m, a] = torch.softmax(z, 1) @ v
        row += n
    return {"out": out.flatten(1), "lse": lse.flatten(1)}

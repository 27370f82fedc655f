"""Workloads of the batched-serving operators: the paged KV-cache append, attention over the paged
cache with a shared prefix, and the residual norm with int8 output.

Each case names an operator (`op`) and its sizes.  `run` computes it in its plain form (elementary
torch operations in 32 bits, one rounding at the end) or, where `own` is true, through the g4b package.

A batch of sequences is described by `seqs`, `new_lo`..`new_hi` (tokens a sequence appends in this step),
`past_lo`..`past_hi` (tokens of its own that it holds already, behind the shared prefix) and `prefix`
(tokens of the prefix that all sequences share); the ragged lengths are drawn from `ragged`.
"""
import os
import random
import sys

import torch

own = False

EPS = 1e-6
DEV = "cuda"
_DT = {"f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def _attn(name, op, heads, kv_heads, hd, page, seqs, new, past, prefix=0, window=0, dtype="f16", ragged=1):
    return {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": page, "seqs": seqs,
            "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "prefix": prefix,
            "window": window, "dtype": dtype, "ragged": ragged}


def _norm(name, rows, dim, dtype, post=True):
    return {"name": name, "op": "norm_i8", "rows": rows, "dim": dim, "dtype": dtype, "post": post}


def listed():
    return [
        # one user's next token: the smallest append, where latency counts
        _attn("append one token", "append", 16, 8, 256, 64, 1, (1, 1), (776, 776)),
        # a decode step of 64 sequences behind a system prompt, q|k|v straight from an f32 GEMM
        _attn("append decode batch", "append", 16, 8, 256, 64, 64, (1, 1), (0, 1500), prefix=1000, dtype="f32"),
        # the prompts of five new requests, ragged, in one step
        _attn("append prompts", "append", 16, 8, 256, 64, 5, (300, 1600), (0, 100)),
        # one user's next token over a short conversation, no prefix
        _attn("attend one token", "attend", 16, 8, 256, 64, 1, (1, 1), (700, 700)),
        # a decode step of unrelated conversations of very different lengths
        _attn("attend decode ragged", "attend", 16, 8, 256, 64, 48, (1, 1), (5, 4000)),
        # many users of one long document or system prompt, with short conversations of their own
        _attn("attend long prefix", "attend", 16, 8, 256, 64, 64, (1, 1), (20, 1000), prefix=16384),
        # the same with 8 query heads on one KV head of 128, small pages, a prefix that ends inside a page
        _attn("attend hd128 small pages", "attend", 8, 1, 128, 16, 128, (1, 1), (1, 300), prefix=8011),
        # prompt chunks behind a prefix on a sliding-window layer
        _attn("attend chunks window", "attend", 16, 8, 256, 32, 3, (1400, 2300), (0, 1200), prefix=2048, window=1024),
        # a full-attention layer with 16 query heads on one KV head of 512
        _attn("attend hd512", "attend", 16, 1, 512, 64, 32, (1, 1), (10, 500), prefix=4096),
        # one token's norm between two GEMMs
        _norm("norm one row", 1, 3840, "f16"),
        # a decode batch, activations as f32
        _norm("norm decode batch", 64, 3840, "f32"),
        # a prefill chunk
        _norm("norm prefill", 8192, 3840, "f16"),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


_HEADS = ((16, 8, 256), (8, 1, 128), (4, 2, 512), (16, 1, 512), (8, 4, 256), (6, 2, 128))


def draw(rng):
    most = {op: {k: max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")} for op in
            ("append", "attend", "norm_i8")}
    while True:
        c = _drawn(rng)
        if all(v <= most[c["op"]][k] for k, v in work(c).items()):      # nothing costs more than the listed cases
            return c


def _drawn(rng):
    op = rng.choice(("append", "attend", "attend", "norm_i8"))
    if op == "norm_i8":
        c = _norm("", _log(rng, 1, 8192), 16 * _log(rng, 4, 960), rng.choice(("f16", "f32")), rng.random() < 0.7)
    else:
        heads, kv_heads, hd = rng.choice(_HEADS)
        page = rng.choice((16, 32, 64, 128))
        prefix = 0 if rng.random() < 0.3 else _log(rng, 17, 12000)
        window = 0 if rng.random() < 0.6 else _log(rng, 33, 4096)
        if rng.random() < 0.6:      # a decode step, perhaps with a few proposed tokens
            seqs, new, past = _log(rng, 1, 64), (1, rng.choice((1, 1, 4))), (0, _log(rng, 10, 2000))
        else:                       # prompt chunks
            seqs, new, past = _log(rng, 1, 4), (1, _log(rng, 40, 1500)), (0, _log(rng, 10, 1000))
        c = _attn("", op, heads, kv_heads, hd, page, seqs, new, past, prefix, window, rng.choice(("f16", "f32")),
                  rng.randrange(1 << 20))
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------- shapes
def _lengths(case):
    """(new tokens, total length with the prefix) of each sequence: plain integers of the case."""
    r = random.Random(case["ragged"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    return new, [case["prefix"] + p + n for p, n in zip(past, new)]


def _pages(case):
    """Pages of the prefix and of the longest sequence's own part."""
    _, total = _lengths(case)
    pg = case["page"]
    return -(-case["prefix"] // pg), -(-(max(total) - case["prefix"]) // pg)


def work(case):
    if case["op"] == "norm_i8":
        n = case["rows"] * case["dim"]
        xb = 2 if case["dtype"] == "f16" else 4
        return {"bytes": n * (xb + 4 + 4 + 1) + case["rows"] * 4 + case["dim"] * 4 * (2 if case["post"] else 1),
                "flops": 12 * n}
    new, total = _lengths(case)
    nh, nkv, hd, tokens = case["heads"], case["kv_heads"], case["hd"], sum(new)
    if case["op"] == "append":
        xb = 2 if case["dtype"] == "f16" else 4
        positions = set()
        for n, t in zip(new, total):
            positions.update(range(t - n, t))
        n = tokens * (nh + 2 * nkv) * hd
        return {"bytes": n * (xb + 2) + len(positions) * hd * 8, "flops": 10 * n}
    w, prefix = case["window"], case["prefix"]
    seen = sum(min(p + 1, w) if w else p + 1 for n, t in zip(new, total) for p in range(t - n, t))
    first = [max(0, t - n - w + 1) if w else 0 for n, t in zip(new, total)]
    keys = max(0, prefix - min(first)) + sum(t - max(prefix, f) for t, f in zip(total, first))
    return {"bytes": keys * nkv * hd * 4 + tokens * nh * hd * 4, "flops": 4 * hd * nh * seen}


# ----------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device=DEV, dtype=dtype)  # noqa: E731
    if case["op"] == "norm_i8":
        m, d = case["rows"], case["dim"]
        s = {"x": randn(m, d, dtype=_DT[case["dtype"]]), "h": 3 * randn(m, d), "w": 1 + 0.1 * randn(d),
             "w_post": 1 + 0.1 * randn(d) if case["post"] else None, "scl": 0.75}
        s["h"][:, :: 97] *= 2        # a few channels of a residual stream are larger than the others
        s["h_out"] = torch.empty_like(s["h"])
        s["values"] = torch.empty((m, d), dtype=torch.float16, device=DEV)
        return s
    new, total = _lengths(case)
    nh, nkv, hd, page, prefix = case["heads"], case["kv_heads"], case["hd"], case["page"], case["prefix"]
    seqs, tokens = case["seqs"], sum(new)
    np_, no = _pages(case)
    n_pages = np_ + seqs * no + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    t32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s = {"q_start": t32(start), "kv_len": t32(total), "tokens": tokens,
         "prefix_len": t32([prefix]) if prefix else None, "prefix_table": order[:np_].contiguous() if prefix else None,
         "table": order[np_:np_ + seqs * no].reshape(seqs, no).contiguous(), "window": case["window"], "heads": nh,
         "seq_of": torch.repeat_interleave(torch.arange(seqs, device=DEV), t32(new).long(), output_size=tokens)}
    s["pos"] = (s["kv_len"].long() - s["q_start"][1:].long())[s["seq_of"]] + torch.arange(tokens, device=DEV)
    s["longest_new"], s["own_lo"] = max(new), prefix
    if case["op"] == "append":
        s["qkv"] = randn(tokens, (nh + 2 * nkv) * hd, dtype=_DT[case["dtype"]])
        s["qnw"], s["knw"] = (1 + 0.1 * randn(hd)) * hd ** -0.25, (1 + 0.1 * randn(hd))
        inv = 10000.0 ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
        ang = torch.arange((np_ + no) * page, device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = (f(torch.cat((ang, ang), 1)).float() for f in (torch.cos, torch.sin))
        s["kc"] = torch.zeros(n_pages, nkv, page, hd, device=DEV, dtype=torch.float16)
        s["vc"] = torch.zeros_like(s["kc"])
        s["q_out"] = torch.empty(tokens, nh * hd, device=DEV, dtype=torch.float16)
    else:
        # normed keys and values; queries whose norm weights keep scores at a standard deviation of about 4
        s["kc"] = randn(n_pages, nkv, page, hd, dtype=torch.float16)
        s["vc"] = randn(n_pages, nkv, page, hd, dtype=torch.float16)
        s["q"] = randn(tokens, nh * hd, dtype=torch.float16) * (4 * hd ** -0.5)
        s["out"] = torch.empty_like(s["q"])
    return s


def _package():
    """The g4b package of this tree (the working folder is its root)."""
    root = os.path.join(os.getcwd(), "gemma4-12b-snapdragonx2elite_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import g4b.ops
    import g4b.paged
    return g4b


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"] = case["op"]
    if own:
        s["g4b"] = _package()
        if case["op"] != "norm_i8":
            # a serving step plans its batch once; every layer's append and attention use that plan
            s["plan"] = s["g4b"].paged.PagedPlan(s["tokens"], case["seqs"], case["heads"], case["kv_heads"],
                                                 case["hd"], case["page"], s["table"].shape[1],
                                                 prefix_pages=0 if s["prefix_table"] is None else s["prefix_table"].numel(),
                                                 window=case["window"], device=DEV)
            s["plan"].update(s["q_start"], s["kv_len"], s["prefix_len"])
    return s


# -------------------------------------------------------------------------------------------- run
def run(s):
    if own:
        return {"append": _own_append, "attend": _own_attend, "norm_i8": _own_norm}[s["op"]](s)
    return {"append": _plain_append, "attend": _plain_attend, "norm_i8": _plain_norm}[s["op"]](s)


def _own_append(s):
    nkv, hd, nq = s["kc"].shape[1], s["kc"].shape[3], s["heads"] * s["kc"].shape[3]
    s["plan"].append(s["qkv"], s["qnw"], s["knw"], s["cos"], s["sin"], s["kc"], s["vc"], s["table"],
                     koff=nq, voff=nq + nkv * hd, q_out=s["q_out"])
    return s["q_out"], s["kc"], s["vc"]


def _own_attend(s):
    return s["plan"].attend(s["q"], s["kc"], s["vc"], s["table"], prefix_table=s["prefix_table"], out=s["out"])


def _own_norm(s):
    a8, sa = s["g4b"].ops.rows_normadd_i8(s["x"], s["h"], s["w"], w_post=s["w_post"], scl=s["scl"], h_out=s["h_out"])
    # the values the int8 codes stand for
    return s["h_out"], torch.mul(a8, sa[:, None], out=s["values"]), sa


def _rms(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin


def _plain_append(s):
    kc, vc = s["kc"], s["vc"]
    nkv, page, hd = kc.shape[1:]
    n = s["pos"].numel()
    x = s["qkv"].float().view(n, -1, hd)
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    s["q_out"].copy_(_rotate(_rms(x[:, :s["heads"]]) * s["qnw"], cos, sin).view(n, -1))
    at = s["pos"] - s["own_lo"]      # every new token lies behind the prefix
    rows = s["table"].long()[s["seq_of"], at // page]
    kc[rows, :, at % page] = _rotate(_rms(x[:, s["heads"]:s["heads"] + nkv]) * s["knw"], cos, sin).half()
    vc[rows, :, at % page] = _rms(x[:, s["heads"] + nkv:]).half()
    return s["q_out"], kc, vc


def _plain_attend(s):
    kc, vc, table = s["kc"], s["vc"], s["table"].long()
    nkv, page, hd = kc.shape[1:]
    seqs, nh, width, tokens = table.shape[0], s["heads"], s["longest_new"], s["q"].shape[0]
    grp = nh // nkv
    # the queries of each sequence, padded to the longest: rows [seq, kv head, token x group]
    index = s["q_start"][:-1, None].long() + torch.arange(width, device=DEV)
    live = index < s["q_start"][1:, None]
    index = torch.where(live, index, torch.zeros_like(index))
    q = s["q"].float().view(tokens, nkv, grp, hd)[index].permute(0, 2, 1, 3, 4).reshape(seqs, nkv, width * grp, hd)
    pos = torch.where(live, s["pos"][index], torch.full_like(index, -1))[:, None, :, None].expand(seqs, 1, width, grp)
    pos = pos.reshape(seqs, 1, width * grp, 1)
    gather = lambda c, t: c[t].float().transpose(-4, -3).reshape(*t.shape[:-1], nkv, -1, hd)  # noqa: E731
    ok, ov = gather(kc, table), gather(vc, table)                     # [seq, kv head, own keys, hd]
    scores = q @ ok.transpose(-1, -2)
    at = s["own_lo"] + torch.arange(ok.shape[2], device=DEV)
    if s["prefix_table"] is not None:
        pt = s["prefix_table"].long()
        pk, pv = gather(kc, pt), gather(vc, pt)                       # [kv head, prefix keys, hd]
        pk, pv = pk[:, :s["own_lo"]], pv[:, :s["own_lo"]]
        rows = q.transpose(0, 1).reshape(nkv, seqs * width * grp, hd)
        ps = (rows @ pk.transpose(-1, -2)).view(nkv, seqs, width * grp, -1).transpose(0, 1)
        scores = torch.cat((ps, scores), -1)
        at = torch.cat((torch.arange(s["own_lo"], device=DEV), at))
    hidden = at > pos
    if s["window"]:
        hidden = hidden | (at <= pos - s["window"])
    scores = scores.masked_fill_(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    n_pre = at.numel() - ok.shape[2]
    out = p[..., n_pre:] @ ov
    if n_pre:
        pr = p[..., :n_pre].transpose(0, 1).reshape(nkv, seqs * width * grp, n_pre)
        out = out + (pr @ pv).view(nkv, seqs, width * grp, hd).transpose(0, 1)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    out = out.view(seqs, nkv, width, grp, hd).permute(0, 2, 1, 3, 4).reshape(seqs, width, nh * hd)
    s["out"].copy_(out[s["seq_of"], torch.arange(tokens, device=DEV) - s["q_start"].long()[s["seq_of"]]])
    return s["out"]


def _plain_norm(s):
    x = s["x"].float()
    if s["w_post"] is not None:
        x = _rms(x) * s["w_post"]
    torch.mul(s["h"] + x, s["scl"], out=s["h_out"])
    y = _rms(s["h_out"]) * s["w"]
    sa = torch.clamp(y.abs().amax(-1) / 127, min=1e-12)
    a8 = torch.round(y * (1 / sa)[:, None]).clamp(-127, 127).to(torch.int8)
    return s["h_out"], torch.mul(a8, sa[:, None], out=s["values"]), sa


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """The definitions, one sequence (or one block of rows) at a time, in 64 bits."""
    s = _inputs(case, seed)
    f64 = torch.float64
    if case["op"] == "norm_i8":
        outs = []
        for x, h in zip(s["x"].split(1024), s["h"].split(1024)):
            x, h = x.to(f64), h.to(f64)
            if s["w_post"] is not None:
                x = x / (x.pow(2).mean(1, True) + EPS).sqrt() * s["w_post"].to(f64)
            h = (h + x) * s["scl"]
            y = h / (h.pow(2).mean(1, True) + EPS).sqrt() * s["w"].to(f64)
            sa = (y.abs().max(1).values / 127).clamp(min=1e-12)
            outs.append((h, (y / sa[:, None]).round().clamp(-127, 127) * sa[:, None], sa))
        return tuple(torch.cat(o) for o in zip(*outs))
    new, total = _lengths(case)
    nkv, page, hd = s["kc"].shape[1:]
    nh, prefix, window = case["heads"], case["prefix"], case["window"]
    if case["op"] == "append":
        kc, vc, q_out = s["kc"].to(f64), s["vc"].to(f64), torch.zeros(s["tokens"], nh, hd, dtype=f64, device=DEV)
        t0 = 0
        for b in range(case["seqs"]):
            x = s["qkv"][t0:t0 + new[b]].to(f64).reshape(new[b], -1, hd)
            x = x / (x.pow(2).mean(-1, True) + EPS).sqrt()
            at = torch.arange(total[b] - new[b], total[b], device=DEV)
            c, sn = s["cos"][at].to(f64)[:, None, :], s["sin"][at].to(f64)[:, None, :]

            def turn(v):
                lo, hi = v.chunk(2, -1)
                return torch.cat((lo * c[..., :hd // 2] - hi * sn[..., :hd // 2],
                                  hi * c[..., hd // 2:] + lo * sn[..., hd // 2:]), -1)

            q_out[t0:t0 + new[b]] = turn(x[:, :nh] * s["qnw"].to(f64))
            own_at = at - prefix
            page_of = s["table"][b].long().index_select(0, own_at // page)
            kc[page_of, :, own_at % page] = turn(x[:, nh:nh + nkv] * s["knw"].to(f64))
            vc[page_of, :, own_at % page] = x[:, nh + nkv:]
            t0 += new[b]
        return q_out.reshape(s["tokens"], nh * hd), kc, vc
    out = torch.zeros(s["tokens"], nh, hd, dtype=f64, device=DEV)

    def rows_of(cache, pages, n):
        """The first n positions that these pages hold, [n, kv head, hd]."""
        return cache[pages.long()].permute(0, 2, 1, 3).reshape(-1, nkv, hd)[:n].to(f64)

    t0 = 0
    for b in range(case["seqs"]):
        k = rows_of(s["kc"], s["table"][b], total[b] - prefix)
        v = rows_of(s["vc"], s["table"][b], total[b] - prefix)
        if prefix:
            k = torch.cat((rows_of(s["kc"], s["prefix_table"], prefix), k))
            v = torch.cat((rows_of(s["vc"], s["prefix_table"], prefix), v))
        for i in range(0, new[b], 256):
            n = min(256, new[b] - i)
            p0 = total[b] - new[b] + i
            lo = max(0, p0 - window + 1) if window else 0
            kk, vv = k[lo:p0 + n], v[lo:p0 + n]
            q = s["q"][t0 + i:t0 + i + n].to(f64).reshape(n, nkv, nh // nkv, hd)
            sc = torch.einsum("tkgd,jkd->kgtj", q, kk)
            j, p = torch.arange(lo, p0 + n, device=DEV), torch.arange(p0, p0 + n, device=DEV)[:, None]
            see = (j <= p) & (j > p - window) if window else j <= p
            w = torch.softmax(torch.where(see, sc, torch.tensor(float("-inf"), dtype=f64, device=DEV)), -1)
            out[t0 + i:t0 + i + n] = torch.einsum("kgtj,jkd->tkgd", w, vv).reshape(n, nh, hd)
        t0 += new[b]
    return out.reshape(s["tokens"], nh * hd)

"""Timed cases of the int8 transformer-decoder operators: RMSNorm -> int8, the W8A8 product, the paged int8 cache and the
attention over it. `run` computes a case with elementary torch operations, or (own = True) with the library's kernels.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SZ = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token of a decoder as wide as the encoder (1024): pure latency
        {"name": "norm 1x1024 bf16", "op": "norm", "n": 1, "d": 1024, "dt": "bf16", "group": 0, "res": True},
        # a ragged batch of f32 activations, quantised per 128 columns for the ternary product
        {"name": "norm 613x4096 f32 g128", "op": "norm", "n": 613, "d": 4096, "dt": "f32", "group": 128, "res": True},
        # a stacked prefill
        {"name": "norm 16384x4096 bf16", "op": "norm", "n": 16384, "d": 4096, "dt": "bf16", "group": 0, "res": True},
        # one token through a square projection: the weights' bytes
        {"name": "product 1x4096x4096 bf16", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "dt": "bf16", "act": "store",
         "bias": False},
        # a decode batch through a feed-forward's first product
        {"name": "product 37x8192x2048 f16", "op": "gemm", "m": 37, "n": 8192, "k": 2048, "dt": "f16", "act": "silu",
         "bias": True},
        # an utterance's frames through a feed-forward's second product (4096 -> 1024), f32 as in the encoder
        {"name": "product 1500x1024x4096 f32", "op": "gemm", "m": 1500, "n": 1024, "k": 4096, "dt": "f32",
         "act": "store", "bias": True},
        # a stacked prefill through a wide product: the tensor cores
        {"name": "product 8192x16384x4096 bf16", "op": "gemm", "m": 8192, "n": 16384, "k": 4096, "dt": "bf16",
         "act": "store", "bias": False},
        # one new token of each of 64 sequences, most of them into a page that is already started
        {"name": "cache 64x1 bf16", "op": "cache", "seqs": 64, "new": 1, "past": 2000, "ragged": True, "heads": 8,
         "hd": 128, "page": 64, "dt": "bf16"},
        # the keys and values of a stacked prefill
        {"name": "cache 8x2048 bf16", "op": "cache", "seqs": 8, "new": 2048, "past": 300, "ragged": True, "heads": 8,
         "hd": 128, "page": 64, "dt": "bf16"},
        # one hypothesis's token over 30 s of context, heads of 64, no sharing
        {"name": "attend 1x1 over 1500 f16", "op": "attend", "seqs": 1, "new": 1, "past": 1499, "ragged": False,
         "heads": 16, "kv": 16, "hd": 64, "page": 32, "dt": "f16", "window": 0},
        # a decode batch over long ragged contexts, four query heads to a key head
        {"name": "attend 64x1 over 16k bf16", "op": "attend", "seqs": 64, "new": 1, "past": 16000, "ragged": True,
         "heads": 32, "kv": 8, "hd": 128, "page": 64, "dt": "bf16", "window": 0},
        # a chunk of a ragged prefill over what is cached already
        {"name": "attend 4x2048 over 4k bf16", "op": "attend", "seqs": 4, "new": 2048, "past": 2000, "ragged": True,
         "heads": 32, "kv": 8, "hd": 128, "page": 64, "dt": "bf16", "window": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dt = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["norm", "gemm", "cache", "attend", "gemm", "attend"])
    if op == "norm":
        group = rng.choice([0, 0, 128])
        d = _log(rng, 65, 8192)
        if group:
            d = max(1, round(d / group)) * group
        n = _log(rng, 1, 16384)
        n = max(1, min(n, 16384 * 4096 // d // (2 if dt == "f32" else 1)))
        return {"op": op, "n": n, "d": d, "dt": dt, "group": group, "res": rng.random() < 0.7}
    if op == "gemm":
        m, n, k = _log(rng, 1, 8192), _log(rng, 17, 16384), 16 * _log(rng, 4, 1024)
        m = max(1, min(m, (1 << 38) // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "dt": dt, "act": rng.choice(["store", "silu"]),
                "bias": rng.random() < 0.5}
    heads, hd, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    seqs = _log(rng, 1, 96)
    new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    if op == "cache":
        new = max(1, min(new, 16384 // seqs))
        return {"op": op, "seqs": seqs, "new": new, "past": rng.choice([0, _log(rng, 1, 4000)]), "ragged": True,
                "heads": heads, "hd": hd, "page": page, "dt": dt}
    share = rng.choice([1, 2, 3, 4, 8])
    while heads * share > 32:
        share = max(1, share // 2)
        heads = min(heads, 32 // share)
    past = _log(rng, 1, 16000)
    new = max(1, min(new, 8192 // seqs))
    past = max(0, min(past, 8000000 // (seqs * heads)))
    if new > 1:  # the work of the largest listed chunk at most
        past = min(past, 4000)
        new = max(1, min(new, 65536 // (seqs * heads * share) * 4, 2048))
    return {"op": op, "seqs": seqs, "new": new, "past": past, "ragged": rng.random() < 0.7, "heads": heads * share,
            "kv": heads, "hd": hd, "page": page, "dt": dt, "window": rng.choice([0, 0, 0, _log(rng, 16, 2048)])}


# ------------------------------------------------------------------------------------------------------ the inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _acts(g, n, d):
    """Activations: unit normal, with a few channels that are much larger, as residual streams have them."""
    x = _randn(g, n, d)
    x *= 1.0 + 15.0 * (torch.rand(d, generator=g, device=DEV) < 0.01)
    return x


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _lengths(case):
    """Host lists (past, new) of each sequence: part of the case, the same for every seed."""
    s = case["seqs"]
    if not case["ragged"]:
        return [case["past"]] * s, [case["new"]] * s
    r = torch.Generator().manual_seed(1000003 * case["past"] + 1009 * case["new"] + s)
    u = torch.rand(s, generator=r).tolist()
    w = torch.rand(s, generator=r).tolist()
    past = [int(case["past"] * (0.25 + 0.75 * a)) for a in u]
    new = [max(1, int(case["new"] * (0.5 + 0.5 * b))) for b in w]
    return past, new


def _table(case, lens, g):
    """A page table: the sequences' pages lie scattered over the pool, as an allocator leaves them; -1 behind the last."""
    page = case["page"]
    need = torch.tensor([-(-n // page) for n in lens])
    total = max(1, int(need.sum()))
    width = max(1, int(need.max()))
    ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(width)[None]
    at = (first[:, None] + col).clamp(max=total - 1).to(DEV)
    return torch.where((col < need[:, None]).to(DEV), ids[at], _int(-1)), total


def _codes(g, pages, heads, page, hd):
    """A pool of codes and scales as a run of writes leaves it: normal values, each (page, head) scaled to its largest."""
    scale = (2.8 + 0.8 * torch.rand((pages, heads), generator=g, device=DEV)) / 127.0
    c = torch.empty((pages, heads, page, hd), dtype=torch.int8, device=DEV)
    step = max(1, (1 << 27) // (heads * page * hd))
    for at in range(0, pages, step):
        v = torch.randn((min(step, pages - at), heads, page, hd), generator=g, device=DEV, dtype=torch.float16)
        v = v / scale[at:at + step, :, None, None].half()
        c[at:at + step] = v.round().clamp(-127, 127).to(torch.int8)
    return c, scale


def _cu(n):
    return [0] + torch.cumsum(torch.tensor(n), 0).tolist()


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["op"] == "norm":
        n, d, dt = case["n"], case["d"], DT[case["dt"]]
        st["x"] = _acts(g, n, d).to(dt)
        st["v"] = (0.5 * _randn(g, n, d)).to(dt) if case["res"] else None
        st["gamma"] = 1.0 + 0.2 * _randn(g, d)
    elif case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        st["x"] = (_randn(g, m, k) * 36.0).round().clamp(-127, 127).to(torch.int8)
        st["sx"] = 0.01 + 0.05 * torch.rand((m, 1), generator=g, device=DEV)
        st["w"] = (_randn(g, n, k) * 36.0).round().clamp(-127, 127).to(torch.int8)
        st["sw"] = (0.5 + torch.rand(n, generator=g, device=DEV)) / (1.3 * 36.0 * math.sqrt(k))
        st["bias"] = 0.5 * _randn(g, n) if case["bias"] else None
    else:
        past, new = _lengths(case)
        lens = [a + b for a, b in zip(past, new)]
        heads = case["heads"] if case["op"] == "cache" else case["kv"]
        st["table"], pages = _table(case, lens, g)
        st["kc"], st["ks"] = _codes(g, pages, heads, case["page"], case["hd"])
        st["vc"], st["vs"] = _codes(g, pages, heads, case["page"], case["hd"])
        st["cu"], st["total"] = _int(_cu(new)), sum(new)
        st["start"], st["lens"] = _int(past), _int(lens)
        dt, hd = DT[case["dt"]], case["hd"]
        if case["op"] == "cache":
            st["k"] = _randn(g, st["total"], heads, hd).to(dt)
            st["v"] = _randn(g, st["total"], heads, hd).to(dt)
            # what is read back: from the first position of the first page that is written
            first = [p // case["page"] * case["page"] for p in past]
            count = [n - f for n, f in zip(lens, first)]
            st["rstart"], st["rcu"], st["rtotal"] = _int(first), _int(_cu(count)), sum(count)
        else:
            st["q"] = _randn(g, st["total"], case["heads"], hd).to(dt)
            st["most"], st["longest"] = max(new), max(lens)
    return st


# ------------------------------------------------------------------------------------------------ the plain forms

def _of(cu, total):
    """(sequence, place within it) of each stacked row."""
    row = torch.arange(total, device=DEV)
    seq = torch.searchsorted(cu.long(), row, right=True) - 1
    return seq, row - cu.long()[seq]


def _norm(st, case):
    x = st["x"].double()
    h = (x if st["v"] is None else x + st["v"].double()).float()
    d = h.shape[1]
    ms = h.double().square().mean(-1, keepdim=True)
    y = h * (1.0 / (ms + 1e-6).sqrt()).float() * st["gamma"]
    y = y.view(h.shape[0], -1, case["group"] or d)
    top = y.abs().amax(-1, keepdim=True)
    s = torch.where(top == 0, torch.ones_like(top), top / torch.full_like(top, 127.0))
    code = (y * (1.0 / s)).round().clamp(-127, 127)
    # codes are given as the values that they stand for, in 16 bits
    out = {"values": (code * s).view(h.shape).to(_sixteen(case)), "scales": s.squeeze(-1)}
    if st["v"] is not None:
        out["res"] = h.to(st["x"].dtype)
    return out


def _sixteen(case):
    return torch.bfloat16 if case["dt"] == "bf16" else torch.float16


def _gemm(st, case):
    # sums of up to 16384 products of 127 x 127 pass 24 bits: f32 sums round, by less than their own type shows
    y = (st["x"].float() @ st["w"].float().t()) * (st["sx"] * st["sw"][None])
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    return y.to(DT[case["dt"]])


def _write(codes, scale, x, st, case):
    """One of K and V: the touched pages' codes and scales are replaced."""
    page, table, start, cu = case["page"], st["table"].long(), st["start"].long(), st["cu"].long()
    seq, i = _of(cu, st["total"])
    pos = start[seq] + i
    pid, slot = table[seq, pos // page], pos % page
    x = x.float()
    top = torch.zeros_like(scale)
    top.index_reduce_(0, pid, x.abs().amax(-1), "amax")
    new = torch.where(top == 0, top, (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126))
    # a page that holds earlier tokens of its sequence keeps at least its scale
    part = start % page
    held = torch.zeros(scale.shape[0], dtype=torch.long, device=DEV)
    at = table[torch.arange(len(start), device=DEV), (start // page).clamp(max=table.shape[1] - 1)]
    some = (part > 0) & (cu[1:] > cu[:-1])
    held[at[some]] = part[some]
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEV)
    touched[pid] = True
    old = torch.where((held > 0)[:, None], scale, torch.zeros_like(scale))
    s = torch.where(touched[:, None], torch.maximum(old, new), scale)
    p = at[some]
    ratio = torch.where(s[p] > 0, old[p] / s[p], torch.ones_like(s[p]))
    again = (codes[p].float() * ratio[:, :, None, None]).round()
    keep = torch.arange(page, device=DEV)[None, None, :, None] < held[p][:, None, None, None]
    codes[p] = torch.where(keep, again.to(torch.int8), codes[p])
    sp = s[pid][:, :, None]
    code = torch.where(sp > 0, (x * (1.0 / sp)).round().clamp(-127, 127), torch.zeros_like(x))
    codes[pid, :, slot] = code.to(torch.int8)
    scale.copy_(s)


def _read(codes, scale, st, case):
    seq, i = _of(st["rcu"], st["rtotal"])
    pos = st["rstart"].long()[seq] + i
    pid = st["table"].long()[seq, pos // case["page"]]
    return (codes[pid, :, pos % case["page"]].float() * scale[pid][:, :, None]).to(DT[case["dt"]])


def _cache(st, case):
    _write(st["kc"], st["ks"], st["k"], st, case)
    _write(st["vc"], st["vs"], st["v"], st, case)
    return {"k": _read(st["kc"], st["ks"], st, case), "v": _read(st["vc"], st["vs"], st, case), "ks": st["ks"],
            "vs": st["vs"]}


def _dense(codes, scale, st, case):
    """The sequences' keys or values, padded: [sequence, head, position, hd]."""
    pid = st["table"].long().clamp(min=0)
    x = codes[pid].float() * scale[pid][:, :, :, None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :st["longest"]]


def _attend(st, case):
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    most, share = st["most"], heads // kv
    seq, i = _of(st["cu"], st["total"])
    q = torch.zeros((case["seqs"], most, heads, hd), device=DEV)
    q[seq, i] = st["q"].float()
    q = q.view(-1, most, kv, share, hd).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [sequence, kv, query x share, hd]
    s = (q @ _dense(st["kc"], st["ks"], st, case).transpose(-1, -2)) / math.sqrt(hd)
    lens = st["lens"].long()
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    pos = (lens - n)[:, None] + torch.arange(most, device=DEV)[None]
    key = torch.arange(st["longest"], device=DEV)
    seen = key <= pos[:, :, None]
    if case["window"]:
        seen &= key > pos[:, :, None] - case["window"]
    s.masked_fill_(~seen.repeat_interleave(share, 1)[:, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s @ _dense(st["vc"], st["vs"], st, case)) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(-1, kv, most, share, hd).permute(0, 2, 1, 3, 4).reshape(-1, most, heads, hd)
    return o[seq, i].to(DT[case["dt"]])


def _own_cache(st):
    from voxrt_b200.cache import KvCache

    if "handle" not in st:  # what a program keeps: the pool's handle
        st["handle"] = KvCache(st["kc"], st["vc"], st["ks"], st["vs"])
    return st["handle"]


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from voxrt_b200 import kernels as K

        if op == "norm":
            r = torch.empty_like(st["x"]) if case["res"] else None
            a = K.rms_quant(st["x"], st["gamma"], group=case["group"] or None, eps=1e-6, v=st["v"], x_res=r)
            out = {"values": K.dequantize(a, _sixteen(case)), "scales": a.scales}
            if r is not None:
                out["res"] = r
            return out
        if op == "gemm":
            y = torch.empty((case["m"], case["n"]), dtype=DT[case["dt"]], device=DEV)
            return K.gemm_i8(K.Int8Matrix(st["w"], st["sw"]), K.QuantAct(st["x"], st["sx"], case["k"]), y,
                             bias=st["bias"], ep=K.Epilogue.Silu if case["act"] == "silu" else K.Epilogue.Store)
        c = _own_cache(st)
        if op == "cache":
            c.write(st["k"], st["v"], st["table"], st["start"], st["cu"])
            k, v = c.read(st["table"], st["rstart"], st["rcu"], st["rtotal"], DT[case["dt"]])
            return {"k": k, "v": v, "ks": c.ks, "vs": c.vs}
        return c.attend(st["q"], st["table"], st["lens"], st["cu"], causal=True, window=case["window"])
    return {"norm": _norm, "gemm": _gemm, "cache": _cache, "attend": _attend}[op](st, case)


# ------------------------------------------------------------------------------------------------- the work, exactly

def work(case):
    b = SZ[case["dt"]]
    if case["op"] == "norm":
        n, d = case["n"], case["d"]
        groups = d // (case["group"] or d)
        # x (and v in, the sum out), the codes written and read back, the values written
        return {"bytes": n * d * ((3 if case["res"] else 1) * b + 1 + 1 + 2) + 8 * n * groups + 4 * d,
                "flops": 9.0 * n * d}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * b + 4 * (m + n + (n if case["bias"] else 0)), "flops": 2.0 * m * n * k}
    past, new = _lengths(case)
    if case["op"] == "cache":
        row = case["heads"] * case["hd"]
        held = sum(p % case["page"] for p in past)
        # the new values in and their codes out; a started page's codes in; all that is read back in and out
        return {"bytes": 2 * row * (sum(new) * (b + 1) + held + (sum(new) + held) * (1 + b)),
                "flops": 2.0 * row * sum(new) * 6}
    w = case["window"] or 1 << 60
    keys = sum(sum(min(p + i + 1, w) for i in range(n)) for p, n in zip(past, new))
    held = sum(min(p + n, w + n) for p, n in zip(past, new))
    return {"bytes": 2 * held * case["kv"] * case["hd"] + 2 * sum(new) * case["heads"] * case["hd"] * b,
            "flops": 4.0 * keys * case["heads"] * case["hd"]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        h = st["x"].double()
        if st["v"] is not None:
            h += st["v"].double()
        y = h / (h.pow(2).sum(1, keepdim=True) / case["d"] + 1e-6).sqrt() * st["gamma"].double()
        parts = y.reshape(case["n"], -1, case["group"] or case["d"])
        s = parts.abs().max(2).values / 127
        v = (parts / s[..., None]).round() * s[..., None]
        out = {"values": v.reshape(y.shape), "scales": s}
        if st["v"] is not None:
            out["res"] = h
        return out
    if case["op"] == "gemm":
        if 2.0 * case["m"] * case["n"] * case["k"] > 1e14:
            return None
        y = torch.mm(st["x"].double(), st["w"].double().T)
        y *= st["sx"].double()
        y *= st["sw"].double()
        if case["bias"]:
            y += st["bias"].double()
        return y * torch.sigmoid(y) if case["act"] == "silu" else y
    past, new = _lengths(case)
    page, at, outs = case["page"], 0, []
    if case["op"] == "cache":
        got = {"k": [], "v": [], "ks": st["ks"].double(), "vs": st["vs"].double()}
        for s, (p, n) in enumerate(zip(past, new)):
            ids = st["table"][s].tolist()
            for name, codes, scales in (("k", st["kc"], got["ks"]), ("v", st["vc"], got["vs"])):
                x = st[name][at:at + n].double()
                for j in range(p // page, (p + n - 1) // page + 1):
                    lo, hi = max(p, j * page), min(p + n, (j + 1) * page)
                    part = x[lo - p:hi - p]
                    top = part.abs().amax((0, 2)) / 127
                    held = lo - j * page
                    was = scales[ids[j]].clone()
                    now = torch.maximum(top, was) if held else top
                    scales[ids[j]] = now
                    if held:
                        c = codes[ids[j], :, :held].double() * (was / now)[:, None, None]
                        got[name].append((c.round() * now[:, None, None]).transpose(0, 1))
                    got[name].append((part / now[:, None]).round() * now[:, None])
            at += n
        return {**got, "k": torch.cat(got["k"]), "v": torch.cat(got["v"])}
    share, hd = case["heads"] // case["kv"], case["hd"]
    for s, (p, n) in enumerate(zip(past, new)):
        length = p + n
        ids = st["table"][s, :-(-length // page)].long()
        k, v = ((c[ids].double() * f[ids].double()[:, :, None, None]).transpose(0, 1).reshape(case["kv"], -1, hd)
                [:, :length] for c, f in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
        key = torch.arange(length, device=DEV)
        for lo in range(0, n, 256):
            hi = min(n, lo + 256)
            q = st["q"][at + lo:at + hi].double().reshape(hi - lo, case["kv"], share, hd)
            e = torch.einsum("ngsd,gkd->gsnk", q, k) * hd ** -0.5
            pos = torch.arange(p + lo, p + hi, device=DEV)[:, None]
            hide = (key > pos) | (key <= pos - (case["window"] or 1 << 60))
            o = torch.einsum("gsnk,gkd->ngsd", torch.softmax(e.masked_fill(hide, -math.inf), -1), v)
            outs.append(o.reshape(hi - lo, case["heads"], hd))
        at += n
    return torch.cat(outs)

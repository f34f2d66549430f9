"""Serving operators of a compressed, bounded key/value cache, as measured work.

The cache.  Pages of `ps` slots (a multiple of 16) hold K and V of every kv
head as FP8 E4M3 codes, [pages][nkv][ps][d], with one FP32 scale, a power of
two, per block of 16 slots and head, [pages][nkv][ps/16]: a slot's value is
code * scale.  A block's scale is 2^e with the smallest e in [-64, 120] for
which its largest finite magnitude is at most 448 * 2^e.

write    New rows of K and V go to the slots [len - new, len) of their
         sequences.  A block that holds older rows keeps at least its old
         scale; when that has to grow, the older codes are rounded to it.
decode   One query per sequence and head over the visible slots: from the
         sequence's start on, and within `window` slots of the newest one
         or within `prefix` slots of the start.  s = scale * q.k, then
         cap * tanh(s / cap) when cap > 0, then - slope * (newest - slot),
         softmax, times V.  With accumulation, every slot's weights, summed
         over the kv head's group of queries, are added to its counter.
evict    Per sequence and kv head: the newest `recent` slots and, of the
         others, those with the largest counters (ties: the lowest slot)
         are kept, `budget` in all, moved in order to other pages and
         quantized anew in their new blocks.
packed   Prefill of several documents packed row after row, a document's
         queries being its last rows: causal, or within `prefix` rows of the
         document's start; `window`, cap and slope as in decode, the
         distance taken as its magnitude.

`run` computes each in 32 bits with elementary operations, or, with `own`,
through the framework's entry points.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode step's append, 64 sequences of a continuous batch
        dict(name="write_step", op="write", B=64, lo=16, hi=1024, new=1, nkv=8, d=128, ps=16,
             t="bf16", pick=4),
        # the rows of eight prompts entering the cache after their prefill
        dict(name="write_prompts", op="write", B=8, lo=512, hi=4096, new=0, nkv=8, d=128, ps=16,
             t="f32", pick=5),
        # one sequence at a short context: the smallest decode, launch-bound
        dict(name="decode_4k", op="decode", B=1, lo=4097, hi=4097, nq=32, nkv=8, d=128, ps=16,
             t="f32", cap=0.0, slopes=False, prefix=0, window=0, starts=False, acc=False, pick=1),
        # a sliding-window layer of a capped model, its first slots kept visible
        dict(name="decode_window", op="decode", B=1, lo=32769, hi=32769, nq=8, nkv=4, d=256,
             ps=16, t="bf16", cap=50.0, slopes=False, prefix=20, window=1024, starts=False,
             acc=False, pick=2),
        # a continuous batch whose weights are counted for eviction
        dict(name="decode_batch", op="decode", B=64, lo=512, hi=32768, nq=32, nkv=8, d=128, ps=16,
             t="bf16", cap=0.0, slopes=False, prefix=0, window=0, starts=False, acc=True, pick=4),
        # long contexts, a distance bias, several documents in a sequence
        dict(name="decode_long", op="decode", B=32, lo=8192, hi=131072, nq=64, nkv=8, d=128,
             ps=16, t="f32", cap=0.0, slopes=True, prefix=0, window=0, starts=True, acc=False,
             pick=5),
        # one sequence brought back to its budget
        dict(name="evict_one", op="evict", B=1, lo=4351, hi=4351, budget=4096, recent=256, nkv=8,
             d=128, ps=16, pick=1),
        # a batch of long sequences brought down to a budget
        dict(name="evict_batch", op="evict", B=16, lo=8192, hi=32768, budget=4096, recent=512,
             nkv=8, d=128, ps=16, pick=3),
        # one short prompt: latency
        dict(name="packed_short", op="packed", B=1, lo=77, hi=77, past=0, nq=32, nkv=8, d=128,
             t="bf16", cap=30.0, slopes=False, prefix=0, window=0, pick=1),
        # ragged documents packed together, a distance bias
        dict(name="packed_docs", op="packed", B=24, lo=60, hi=4000, past=0, nq=32, nkv=8, d=128,
             t="bf16", cap=0.0, slopes=True, prefix=0, window=0, pick=7),
        # a capped sliding-window layer, head size 256, a second part of a prompt
        dict(name="packed_window", op="packed", B=2, lo=4096, hi=4096, past=1000, nq=8, nkv=4,
             d=256, t="f16", cap=50.0, slopes=False, prefix=0, window=1024, pick=1),
        # one long prompt with a prefix that all its rows see
        dict(name="packed_long", op="packed", B=1, lo=16384, hi=16384, past=0, nq=32, nkv=8, d=128,
             t="bf16", cap=0.0, slopes=False, prefix=500, window=0, pick=1),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "evict", "packed"])
    nkv, group, d = rng.choice([(8, 4, 128), (4, 2, 256), (8, 8, 128), (2, 4, 64), (1, 8, 128),
                                (4, 1, 64), (5, 4, 128)])
    ps = rng.choice([16, 16, 32, 64])
    pick = rng.randrange(1 << 20)
    if op == "write":
        B = _logint(rng, 1, 64)
        one = rng.random() < 0.5
        hi = _logint(rng, 16, 24000 // B + 16)
        return dict(op=op, B=B, lo=max(1, hi // 8), hi=hi, new=1 if one else 0, nkv=nkv, d=d,
                    ps=ps, t=rng.choice(list(TYPES)), pick=pick)
    if op == "decode":
        B = _logint(rng, 1, 64)
        hi = _logint(rng, 20, min(131072, 2000000 // B))
        return dict(op=op, B=B, lo=max(1, hi // rng.choice([1, 4, 64])), hi=hi, nq=nkv * group,
                    nkv=nkv, d=d, ps=ps, t=rng.choice(list(TYPES)),
                    cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3,
                    prefix=rng.choice([0, 4, 37]), window=rng.choice([0, 0, 1024, 4000]),
                    starts=rng.random() < 0.3, acc=rng.random() < 0.4, pick=pick)
    if op == "evict":
        B = _logint(rng, 1, 16)
        hi = _logint(rng, 300, 32768)
        budget = _logint(rng, 64, max(64, hi // 2))
        return dict(op=op, B=B, lo=max(1, hi // 3), hi=hi, budget=budget,
                    recent=rng.choice([0, 1, budget // 8, budget // 2]), nkv=nkv, d=d, ps=ps,
                    pick=pick)
    B = _logint(rng, 1, 24)
    hi = _logint(rng, 8, 12000 // B)
    return dict(op=op, B=B, lo=max(1, hi // rng.choice([1, 8])), hi=hi,
                past=rng.choice([0, 0, 333, 1000]), nq=nkv * group, nkv=nkv, d=d,
                t=rng.choice(["bf16", "f16"]), cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                slopes=rng.random() < 0.3, prefix=rng.choice([0, 0, 60, 500]),
                window=rng.choice([0, 0, 256, 1024]), pick=pick)


def lengths(case):
    """The case's sequence lengths (part of the case, not of the seed)."""
    r = random.Random(case["pick"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def starts_of(case):
    """First visible slot of each sequence: its newest document's start."""
    lens = lengths(case)
    if not case["starts"]:
        return [0] * len(lens)
    r = random.Random(case["pick"] + 1)
    return [r.randint(0, n // 4) for n in lens]


def visible(case):
    """Visible slots of each sequence (decode)."""
    out = []
    for n, st in zip(lengths(case), starts_of(case)):
        if case["window"] > 0:
            lo = max(st, n - case["window"])
            out.append(n - lo + max(0, min(lo, st + case["prefix"]) - st))
        else:
            out.append(n - st)
    return out


def pairs(case):
    """Visible (query, key) pairs of the packed case, per head."""
    tot = 0
    for n in lengths(case):
        k = n + case["past"]
        w, pr = case["window"], min(case["prefix"], k)
        for p in range(case["past"], k):
            lo = max(0, p - w + 1) if w > 0 else 0
            tot += p + 1 - lo + (min(lo, pr) + max(0, pr - p - 1))
    return tot


def work(case):
    op, nkv, d = case["op"], case["nkv"], case["d"]
    if op == "write":
        rows = case["B"] if case["new"] else sum(lengths(case))
        el = 4 if case["t"] == "f32" else 2
        return {"bytes": rows * nkv * d * 2 * (el + 1) + 2 * 4 * nkv * max(case["B"], rows // 16),
                "flops": 4 * rows * nkv * d}
    if op == "decode":
        v, n = sum(visible(case)), sum(lengths(case))
        el = 4 if case["t"] == "f32" else 2
        b = v * nkv * (2 * d + 0.5) + 2 * case["B"] * case["nq"] * d * el
        if case["acc"]:
            b += 2 * 4 * n * nkv
        return {"bytes": b, "flops": 4 * v * case["nq"] * d}
    if op == "evict":
        n = sum(lengths(case))
        kept = sum(min(x, case["budget"]) for x in lengths(case))
        return {"bytes": nkv * (4 * n + kept * (2 * 2 * d + 4 + 4 + 1)), "flops": nkv * n}
    t = sum(lengths(case))
    k = t + case["past"] * case["B"]
    return {"bytes": 2 * (2 * t * case["nq"] * d + 2 * k * nkv * d),
            "flops": 4 * pairs(case) * case["nq"] * d}


# ---------------------------------------------------------------- the cache's format

def block_scale(amax):
    """2^e, e the smallest in [-64, 120] with amax <= 448 * 2^e."""
    m, x = torch.frexp(amax)  # amax = m * 2^x, m in [0.5, 1); 448 = 0.875 * 2^9
    e = x - 9 + (m > 0.875).to(x.dtype)
    e = torch.where(amax > 0, e, torch.full_like(e, -64)).clamp(-64, 120)
    return torch.ldexp(torch.ones_like(amax), e)


def amax_of(x):
    """Largest finite magnitude of [..., 16, d] blocks."""
    a = x.abs()
    return torch.where(torch.isfinite(a), a, torch.zeros_like(a)).amax(dim=(-2, -1))


def codes_of(x, scale):
    """FP8 codes of [..., 16, d] under their blocks' scales."""
    return (x / scale[..., None, None]).clamp(-448.0, 448.0).to(E4M3)


def as_blocks(x, ps):
    """[pages][nkv][ps][d] as [pages][nkv][ps/16][16][d]."""
    p, h, _, d = x.shape
    return x.reshape(p, h, ps // 16, 16, d)


def make_pool(g, pages, nkv, ps, d, spread):
    """A pool of plausible rows: normal values, their size varying by block."""
    codes = torch.empty(pages, nkv, ps, d, dtype=torch.uint8, device=DEV)
    scale = torch.empty(pages, nkv, ps // 16, device=DEV)
    step = max(1, (1 << 27) // (nkv * ps * d))
    for p in range(0, pages, step):
        q = min(pages, p + step)
        x = torch.randn(q - p, nkv, ps // 16, 16, d, device=DEV, generator=g)
        x *= torch.exp(spread * torch.randn(q - p, nkv, ps // 16, 1, 1, device=DEV, generator=g))
        s = block_scale(amax_of(x))
        codes[p:q] = codes_of(x, s).view(torch.uint8).view(q - p, nkv, ps, d)
        scale[p:q] = s
    return codes, scale


def tables(g, needs, extra=3):
    """Shuffled page tables: [B][max pages], and the number of pages."""
    total = sum(needs) + extra
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    bt = torch.zeros(len(needs), max(1, max(needs)), dtype=torch.int32, device=DEV)
    i = 0
    for b, m in enumerate(needs):
        bt[b, :m] = perm[i:i + m]
        i += m
    return bt, total


# ---------------------------------------------------------------- prepare

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = {"case": case}
    op, nkv, d = case["op"], case["nkv"], case["d"]
    lens = lengths(case)
    st["lens"] = lens
    if op == "packed":
        _prepare_packed(case, g, st)
        return st
    ps = case["ps"]
    bt, pages = tables(g, [(n + ps - 1) // ps for n in lens])
    st["bt"] = bt
    if op == "write":
        new = [1] * len(lens) if case["new"] else list(lens)
        st["new"] = new
        k, ks = make_pool(g, pages, nkv, ps, d, 0.3)
        v, vs = make_pool(g, pages, nkv, ps, d, 0.3)
        st.update(k=k, v=v, k_scale=ks, v_scale=vs)
        rows = sum(new)
        big = torch.exp(0.5 * torch.randn(rows, nkv, 1, device=DEV, generator=g))
        st["k_rows"] = (torch.randn(rows, nkv, d, device=DEV, generator=g) * big).to(TYPES[case["t"]])
        st["v_rows"] = torch.randn(rows, nkv, d, device=DEV, generator=g).to(TYPES[case["t"]])
    elif op == "decode":
        nq, B = case["nq"], len(lens)
        k, ks = make_pool(g, pages, nkv, ps, d, 0.2)
        v, vs = make_pool(g, pages, nkv, ps, d, 0.2)
        st.update(k=k, v=v, k_scale=ks, v_scale=vs)
        st["q"] = torch.randn(B, nq, d, device=DEV, generator=g).to(TYPES[case["t"]])
        st["o"] = torch.empty(B, nq, d, device=DEV, dtype=TYPES[case["t"]])
        st["slopes"] = (torch.exp2(-8.0 * torch.arange(1, nq + 1, device=DEV) / nq)
                        if case["slopes"] else None)
        st["starts"] = starts_of(case)
        if case["acc"]:
            st["weight"] = torch.rand(pages, nkv, ps, device=DEV, generator=g)
            st["weight_out"] = torch.zeros(pages, nkv, ps, device=DEV)
    else:
        k, ks = make_pool(g, pages, nkv, ps, d, 0.3)
        v, vs = make_pool(g, pages, nkv, ps, d, 0.3)
        w = torch.rand(pages, nkv, ps, device=DEV, generator=g)
        w = torch.where(w < 0.9, (w * 64).floor() / 64, 20 * w * w)  # with ties, as unread slots have
        st.update(k=k, v=v, k_scale=ks, v_scale=vs, weight=w)
        bt2, pages2 = tables(g, [(min(n, case["budget"]) + ps - 1) // ps for n in lens])
        st["dst_bt"] = bt2
        st["dst"] = dict(k=torch.zeros(pages2, nkv, ps, d, dtype=torch.uint8, device=DEV),
                         v=torch.zeros(pages2, nkv, ps, d, dtype=torch.uint8, device=DEV),
                         k_scale=torch.zeros(pages2, nkv, ps // 16, device=DEV),
                         v_scale=torch.zeros(pages2, nkv, ps // 16, device=DEV),
                         weight=torch.zeros(pages2, nkv, ps, device=DEV))
        st["kept"] = torch.empty(len(lens), nkv, case["budget"], dtype=torch.int32, device=DEV)
    if own:
        import molot_b200 as mb
        plan = mb.F8Plan()
        if op == "write":
            plan.build(nkv, nkv, d, lens, new_lens=st["new"])
        elif op == "decode":
            plan.build(case["nq"], nkv, d, lens, starts=st["starts"],
                       prefix=[case["prefix"]] * len(lens), window=case["window"])
        else:
            plan.build(nkv, nkv, d, lens)
        st["plan"] = plan
        st["layer"] = mb.F8Layer(st["k"], st["v"], st["k_scale"], st["v_scale"], bt,
                                 weight=st.get("weight"))
        if op == "evict":
            x = st["dst"]
            st["dst_layer"] = mb.F8Layer(x["k"], x["v"], x["k_scale"], x["v_scale"], st["dst_bt"],
                                         weight=x["weight"])
    return st


def _prepare_packed(case, g, st):
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    t, tk = sum(st["lens"]), sum(st["lens"]) + case["past"] * len(st["lens"])
    ty = TYPES[case["t"]]
    if case["past"]:
        q = torch.randn(t, nq, d, device=DEV, generator=g).to(ty)
        kv = torch.randn(tk, 2 * nkv, d, device=DEV, generator=g).to(ty)
        st.update(q=q, k=kv[:, :nkv], v=kv[:, nkv:])
    else:  # the three parts of one projection's output
        qkv = torch.randn(t, nq + 2 * nkv, d, device=DEV, generator=g).to(ty)
        st.update(q=qkv[:, :nq], k=qkv[:, nq:nq + nkv], v=qkv[:, nq + nkv:])
    st["o"] = torch.empty(t, nq, d, device=DEV, dtype=ty)
    st["lse"] = torch.empty(t, nq, device=DEV)
    st["slopes"] = (torch.exp2(-8.0 * torch.arange(1, nq + 1, device=DEV) / nq)
                    if case["slopes"] else None)
    if own:
        import molot_b200 as mb
        plan = mb.PackedPlan()
        plan.build(nq, nkv, d, st["lens"], k_lens=[n + case["past"] for n in st["lens"]],
                   prefix=[case["prefix"]] * len(st["lens"]), window=case["window"])
        st["plan"] = plan


# ---------------------------------------------------------------- run

def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        plan = st["plan"]
        if op == "write":
            plan.write(st["layer"], st["k_rows"], st["v_rows"])
            return _write_out(st)
        if op == "decode":
            plan.decode(st["layer"], st["q"], st["o"], case["d"] ** -0.5, softcap=case["cap"],
                        slopes=st["slopes"], weight_out=st.get("weight_out"))
            return (st["o"], st["weight_out"]) if case["acc"] else (st["o"],)
        if op == "evict":
            plan.evict(st["layer"], st["dst_layer"], case["budget"], case["recent"], st["kept"])
            return _evict_out(st)
        plan.attend(st["q"], st["k"], st["v"], st["o"], case["d"] ** -0.5, softcap=case["cap"],
                    slopes=st["slopes"], lse=st["lse"])
        return st["o"], st["lse"]
    if op == "write":
        _plain_write(st)
        return _write_out(st)
    if op == "decode":
        return _plain_decode(st)
    if op == "evict":
        _plain_evict(st)
        return _evict_out(st)
    return _plain_packed(st)


def _write_out(st):
    return st["k"].view(E4M3), st["k_scale"], st["v"].view(E4M3), st["v_scale"]


def _evict_out(st):
    x = st["dst"]
    return (st["kept"], x["k"].view(E4M3), x["k_scale"], x["v"].view(E4M3), x["v_scale"],
            x["weight"])


def _plain_write(st):
    case, bt = st["case"], st["bt"].long()
    ps, row = case["ps"], 0
    for b, (n, m) in enumerate(zip(st["lens"], st["new"])):
        n0 = n - m
        b0, b1 = n0 // 16, (n + 15) // 16
        idx = torch.arange(b0, b1, device=DEV)
        page, sub = bt[b][idx * 16 // ps], (idx * 16 % ps) // 16
        for pool, sc, rows in (("k", "k_scale", "k_rows"), ("v", "v_scale", "v_rows")):
            blocks, scales = as_blocks(st[pool], ps), st[sc]
            old = blocks[page, :, sub].view(E4M3).float()  # [nb][nkv][16][d]
            so = scales[page, :, sub]  # [nb][nkv]
            nb, nkv, _, d = old.shape
            x = torch.zeros(nb * 16, nkv, d, device=DEV)
            x[n0 - b0 * 16:n - b0 * 16] = st[rows][row:row + m].float()
            x = x.view(nb, 16, nkv, d).transpose(1, 2)
            s = block_scale(amax_of(x))
            if n0 > b0 * 16:  # the first block holds older rows
                s[0] = torch.maximum(s[0], so[0])
            slot = (idx * 16)[:, None] + torch.arange(16, device=DEV)
            is_new = ((slot >= n0) & (slot < n))[:, None, :, None]
            val = torch.where(is_new, x, old * so[..., None, None])
            c = codes_of(val, s).view(torch.uint8)
            past = (slot >= n)[:, None, :, None]  # slots past the end keep their bytes
            blocks[page, :, sub] = torch.where(past, old.to(E4M3).view(torch.uint8), c)
            scales[page, :, sub] = s
        row += m


def _rows(st, b, n, pool, sc):
    """Values of a sequence's first n slots, [nkv][n][d]."""
    case = st["case"]
    ps = case["ps"]
    m = (n + ps - 1) // ps
    p = st["bt"][b, :m].long()
    x = as_blocks(st[pool][p], ps).view(E4M3).float() * st[sc][p][..., None, None]
    return x.permute(1, 0, 2, 3, 4).reshape(x.shape[1], m * ps, case["d"])[:, :n]


def _plain_decode(st):
    case = st["case"]
    nq, nkv, ps = case["nq"], case["nkv"], case["ps"]
    out = torch.zeros(len(st["lens"]), nq, case["d"], device=DEV)
    wout = torch.zeros_like(st["weight"]) if case["acc"] else None
    for b, n in enumerate(st["lens"]):
        k, v = _rows(st, b, n, "k", "k_scale"), _rows(st, b, n, "v", "v_scale")
        q = st["q"][b].float().view(nkv, nq // nkv, -1)
        s = torch.matmul(q, k.transpose(1, 2)) * case["d"] ** -0.5
        if case["cap"] > 0:
            s = case["cap"] * torch.tanh(s / case["cap"])
        t = torch.arange(n, device=DEV)
        if case["slopes"]:
            s = s - st["slopes"].view(nkv, -1, 1) * (n - 1 - t)
        first = st["starts"][b]
        see = t >= first
        if case["window"] > 0:
            see = see & ((n - 1 - t < case["window"]) | (t < first + case["prefix"]))
        s = s.masked_fill(~see, -math.inf)
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = p / p.sum(dim=-1, keepdim=True)
        out[b] = torch.matmul(p, v).view(nq, -1)
        if case["acc"]:
            page = st["bt"][b][t // ps].long()
            wout[page, :, t % ps] = st["weight"][page, :, t % ps] + p.sum(dim=1).t()
    out = out.to(TYPES[case["t"]])
    return (out, wout) if case["acc"] else (out,)


def _plain_evict(st):
    case, x = st["case"], st["dst"]
    ps, nkv, d, budget = case["ps"], case["nkv"], case["d"], case["budget"]
    st["kept"].fill_(-1)
    head = torch.arange(nkv, device=DEV)[:, None]
    for b, n in enumerate(st["lens"]):
        t = torch.arange(n, device=DEV)
        w = st["weight"][st["bt"][b][t // ps].long(), :, t % ps].t()  # [nkv][n]
        if n <= budget:
            keep = t.expand(nkv, n)
        else:
            old = n - case["recent"]
            order = torch.sort(w[:, :old], dim=1, descending=True, stable=True)[1]
            keep = torch.cat([order[:, :budget - case["recent"]].sort(dim=1)[0],
                              t[old:].expand(nkv, -1)], dim=1)
        m = keep.shape[1]
        st["kept"][b, :, :m] = keep.int()
        nb = (m + 15) // 16
        j = torch.arange(m, device=DEV)
        x["weight"][st["dst_bt"][b][j // ps].long(), :, j % ps] = w.gather(1, keep).t()
        idx = torch.arange(nb, device=DEV)
        page, sub = st["dst_bt"][b][idx * 16 // ps].long(), (idx * 16 % ps) // 16
        for pool, sc in (("k", "k_scale"), ("v", "v_scale")):
            val = torch.zeros(nkv, nb * 16, d, device=DEV)
            val[:, :m] = _rows(st, b, n, pool, sc)[head, keep]
            val = val.view(nkv, nb, 16, d).transpose(0, 1)
            s = block_scale(amax_of(val))
            c = codes_of(val, s).view(torch.uint8)
            blocks = as_blocks(x[pool], ps)
            live = (idx[:, None] * 16 + torch.arange(16, device=DEV) < m)[:, None, :, None]
            blocks[page, :, sub] = torch.where(live, c, blocks[page, :, sub])
            x[sc][page, :, sub] = s


def _plain_packed(st):
    case = st["case"]
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    t, past = sum(st["lens"]), case["past"]
    out = torch.zeros(t, nq, d, device=DEV)
    lse = torch.full((t, nq), -math.inf, device=DEV)
    qs = ks = 0
    for n in st["lens"]:
        m = n + past
        k = st["k"][ks:ks + m].float().transpose(0, 1)
        v = st["v"][ks:ks + m].float().transpose(0, 1)
        step = max(1, (1 << 28) // (nq * m))
        for r in range(0, n, step):
            e = min(n, r + step)
            q = st["q"][qs + r:qs + e].float().view(e - r, nkv, nq // nkv, d).permute(1, 2, 0, 3)
            s = torch.matmul(q, k[:, None].transpose(2, 3)) * d ** -0.5
            if case["cap"] > 0:
                s = case["cap"] * torch.tanh(s / case["cap"])
            pos = torch.arange(past + r, past + e, device=DEV)[:, None]
            tt = torch.arange(m, device=DEV)
            if case["slopes"]:
                s = s - st["slopes"].view(nkv, -1, 1, 1) * (pos - tt).abs()
            see = tt <= pos
            if case["window"] > 0:
                see = see & (pos - tt < case["window"])
            see = see | (tt < case["prefix"])
            s = s.masked_fill(~see, -math.inf)
            mx = s.amax(dim=-1, keepdim=True)
            p = torch.exp(s - mx)
            l = p.sum(dim=-1, keepdim=True)
            o = torch.matmul(p, v[:, None]) / l
            out[qs + r:qs + e] = o.permute(2, 0, 1, 3).reshape(e - r, nq, d)
            lse[qs + r:qs + e] = (mx + torch.log(l))[..., 0].permute(2, 0, 1).reshape(e - r, nq)
        qs += n
        ks += m
    return out.to(TYPES[case["t"]]), lse


# ---------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions in 64 bits, one sequence and kv head at a time."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"write": _exact_write, "decode": _exact_decode, "evict": _exact_evict,
            "packed": _exact_packed}[case["op"]](case, st)


def _round_e4m3(x):
    """Nearest E4M3 value, ties to the even mantissa, saturating; in float64."""
    a = x.abs().clamp(max=448.0)
    ex = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a))))
    ex = torch.where(torch.exp2(ex) > a, ex - 1, ex)
    ex = torch.where(torch.exp2(ex + 1) <= a, ex + 1, ex).clamp(min=-6)
    quantum = torch.exp2(ex - 3)
    return torch.copysign(torch.round(a / quantum) * quantum, x)


def _exp_of(amax):
    """The smallest e in [-64, 120] with amax <= 448 * 2^e."""
    e = torch.ceil(torch.log2((amax / 448.0).clamp(min=2.0 ** -64))).clamp(-64, 120)
    e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
    return torch.where((amax <= 448.0 * torch.exp2(e - 1)) & (e > -64), e - 1, e)


def _exact_write(case, st):
    ps, nkv, d = case["ps"], case["nkv"], case["d"]
    outs = []
    for pool, sc, rows in (("k", "k_scale", "k_rows"), ("v", "v_scale", "v_rows")):
        codes = st[pool].view(E4M3).double()
        scale = st[sc].double()
        row = 0
        for b, (n, m) in enumerate(zip(st["lens"], st["new"])):
            n0 = n - m
            new = st[rows][row:row + m].double()
            row += m
            lo = n0 // 16 * 16
            slots = torch.arange(lo, n, device=DEV)
            page = st["bt"][b].long()[slots // ps]
            old = codes[page, :, slots % ps] * scale[page, :, (slots % ps) // 16][..., None]
            val = old.clone()
            val[n0 - lo:] = new
            nb = (n - lo + 15) // 16
            a = torch.zeros(nb * 16, nkv, dtype=torch.float64, device=DEV)
            a[n0 - lo:n - lo] = new.abs().amax(dim=-1)
            e = _exp_of(a.view(nb, 16, nkv).amax(dim=1))
            if n0 > lo:
                e[0] = torch.maximum(e[0], torch.log2(scale[page[0], :, (lo % ps) // 16]).round())
            s = torch.exp2(e).repeat_interleave(16, dim=0)[:n - lo]
            codes[page, :, slots % ps] = _round_e4m3(val / s[..., None])
            scale[page, :, (slots % ps) // 16] = s
        outs += [codes, scale]
    return tuple(outs)


def _head64(st, b, slots, h, pool, sc):
    ps = st["case"]["ps"]
    page = st["bt"][b].long()[slots // ps]
    c = st[pool][page, h, slots % ps].view(E4M3).double()
    return c * st[sc][page, h, (slots % ps) // 16].double()[:, None]


def _exact_decode(case, st):
    nq, nkv, d, ps = case["nq"], case["nkv"], case["d"], case["ps"]
    G = nq // nkv
    out = torch.zeros(len(st["lens"]), nq, d, dtype=torch.float64, device=DEV)
    wout = torch.zeros(st["weight"].shape, dtype=torch.float64, device=DEV) if case["acc"] else None
    for b, n in enumerate(st["lens"]):
        first = st["starts"][b]
        sees = range(first, n)
        if case["window"] > 0:
            lo = max(first, n - case["window"])
            sees = list(range(first, min(lo, first + case["prefix"]))) + list(range(lo, n))
            sl = torch.tensor(sees, device=DEV)
        else:
            sl = torch.arange(first, n, device=DEV)
        full = torch.arange(n, device=DEV)
        for h in range(nkv):
            k = _head64(st, b, sl, h, "k", "k_scale")
            s = st["q"][b, h * G:(h + 1) * G].double() @ k.T / math.sqrt(d)
            if case["cap"] > 0:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if case["slopes"]:
                s = s - st["slopes"][h * G:(h + 1) * G].double()[:, None] * (n - 1 - sl).double()
            p = torch.softmax(s, dim=1)
            out[b, h * G:(h + 1) * G] = p @ _head64(st, b, sl, h, "v", "v_scale")
            if case["acc"]:
                page = st["bt"][b].long()[full // ps]
                w = st["weight"][page, h, full % ps].double()
                w[sl] += p.sum(dim=0)
                wout[page, h, full % ps] = w
    return (out, wout) if case["acc"] else (out,)


def _exact_evict(case, st):
    ps, nkv, d, budget, recent = (case[x] for x in ("ps", "nkv", "d", "budget", "recent"))
    x = st["dst"]
    kept = torch.full_like(st["kept"], -1)
    kc, vc = (torch.zeros(x[p].shape, dtype=torch.float64, device=DEV) for p in ("k", "v"))
    kss, vss = (torch.zeros(x[p].shape, dtype=torch.float64, device=DEV)
                for p in ("k_scale", "v_scale"))
    wo = torch.zeros(x["weight"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["lens"]):
        page_of = st["bt"][b].long()
        for h in range(nkv):
            t = torch.arange(n, device=DEV)
            w = st["weight"][page_of[t // ps], h, t % ps].double()
            if n > budget:
                # rank by (weight, lower slot first) through one sort of distinct pairs
                old = n - recent
                ww = w[:old].tolist()
                best = sorted(range(old), key=lambda i: (-ww[i], i))[:budget - recent]
                t = torch.tensor(sorted(best) + list(range(old, n)), device=DEV)
            m = len(t)
            kept[b, h, :m] = t.int()
            j = torch.arange(m, device=DEV)
            dp = st["dst_bt"][b].long()[j // ps]
            wo[dp, h, j % ps] = w[t]
            for pool, sc, c, s in (("k", "k_scale", kc, kss), ("v", "v_scale", vc, vss)):
                val = _head64(st, b, t, h, pool, sc)
                nb = (m + 15) // 16
                a = torch.zeros(nb * 16, dtype=torch.float64, device=DEV)
                a[:m] = val.abs().amax(dim=1)
                e = torch.exp2(_exp_of(a.view(nb, 16).amax(dim=1))).repeat_interleave(16)[:m]
                c[dp, h, j % ps] = _round_e4m3(val / e[:, None])
                s[dp, h, (j % ps) // 16] = e
    return kept, kc, kss, vc, vss, wo


def _exact_packed(case, st):
    nq, nkv, d, past = case["nq"], case["nkv"], case["d"], case["past"]
    t = sum(st["lens"])
    out = torch.empty(t, nq, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(t, nq, dtype=torch.float64, device=DEV)
    qs = ks = 0
    for n in st["lens"]:
        m = n + past
        for h in range(nq):
            k = st["k"][ks:ks + m, h * nkv // nq].double()
            v = st["v"][ks:ks + m, h * nkv // nq].double()
            for r in range(0, n, 4096):
                e = min(n, r + 4096)
                s = st["q"][qs + r:qs + e, h].double() @ k.T / math.sqrt(d)
                if case["cap"] > 0:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                gap = (torch.arange(past + r, past + e, device=DEV)[:, None]
                       - torch.arange(m, device=DEV)[None, :])
                if case["slopes"]:
                    s = s - st["slopes"][h].double() * gap.abs()
                hide = gap < 0
                if case["window"] > 0:
                    hide |= gap >= case["window"]
                hide[:, :min(m, case["prefix"])] = False
                s[hide] = -math.inf
                z = torch.logsumexp(s, dim=1)
                out[qs + r:qs + e, h] = torch.exp(s - z[:, None]) @ v
                lse[qs + r:qs + e, h] = z
        qs += n
        ks += m
    return out, lse

"""The 8-bit block-scaled paged cache on the GPU against its definition in
64 bits: writing (exact), decode attention (every mask and score modifier),
weight counters, eviction (exact), refusals."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# Unit roundoff of the outputs' type (24, 8 and 11 significant bits).
U_OUT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# Rounding of the softmax weights before their product with V: split in two
# halves for float32, one FP16 value otherwise.
U_P = {"float32": 2.0 ** -20, "bfloat16": 2.0 ** -10, "float16": 2.0 ** -10}
# Relative error of a weight from its score: FP32 sums of 256 products, the
# base-2 exponential, the cap's tanh (scores here stay below 64 in size).
U_S = 8e-6


def e4m3(torch, x):
    """Nearest E4M3 value of float64 x, ties to even, saturating at 448."""
    a = x.abs().clamp(max=448.0)
    ex = torch.floor(torch.log2(a.clamp(min=2.0 ** -20))).clamp(min=-6)
    q = torch.exp2(ex - 3)
    return torch.copysign(torch.round(a / q) * q, x)


def scale_of(torch, amax):
    e = torch.ceil(torch.log2((amax / 448.0).clamp(min=2.0 ** -64))).clamp(max=120)
    e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
    return torch.exp2(e)


class Cache:
    """Pools on the GPU and their values in float64, slot by slot."""

    def __init__(self, mb, torch, lens, nkv, d, ps, seed, spare=3, weight=True):
        g = torch.Generator().manual_seed(seed)
        need = [max(1, math.ceil(n / ps)) for n in lens]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=g).int()
        self.bt = torch.zeros(len(lens), max(need) + 1, dtype=torch.int32)
        i = 0
        for b, m in enumerate(need):
            self.bt[b, :m] = perm[i:i + m]
            i += m
        # every byte that is not written holds NaN codes
        self.k = torch.full((pages, nkv, ps, d), 0x7F, dtype=torch.uint8, device="cuda")
        self.v = torch.full_like(self.k, 0xFF)
        self.ks = torch.full((pages, nkv, ps // 16), 1.0, device="cuda")
        self.vs = torch.full_like(self.ks, 1.0)
        self.w = torch.zeros(pages, nkv, ps, device="cuda") if weight else None
        self.torch, self.lens, self.nkv, self.d, self.ps = torch, lens, nkv, d, ps
        self.layer = mb.F8Layer(self.k, self.v, self.ks, self.vs, self.bt.cuda(), weight=self.w)

    def slots(self, b, n):
        t = np.arange(n)
        return self.bt[b].numpy()[t // self.ps].astype(np.int64), t % self.ps

    def values(self, b, n, which):
        """float64 [n][nkv][d] of a sequence's first n slots."""
        page, sub = self.slots(b, n)
        codes, sc = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        c = codes.view(self.torch.float8_e4m3fn).float().double().cpu()[page, :, sub]
        return c * sc.double().cpu()[page, :, sub // 16][..., None]

    def counters(self, b, n, w=None):
        page, sub = self.slots(b, n)
        return (self.w if w is None else w).double().cpu()[page, :, sub]


def fill(mb, torch, c, nq, seed, dtype, spread=0.3):
    """Writes whole sequences of random rows."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(c.lens)
    k = torch.randn(rows, c.nkv, c.d, generator=g) * torch.exp(
        spread * torch.randn(rows, c.nkv, 1, generator=g))
    v = torch.randn(rows, c.nkv, c.d, generator=g)
    k, v = k.to(dtype), v.to(dtype)
    plan = mb.F8Plan()
    plan.build(nq, c.nkv, c.d, c.lens, new_lens=c.lens)
    plan.write(c.layer, k.cuda(), v.cuda())
    plan.close()
    return k.double(), v.double()


# ---------------------------------------------------------------- write

@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("lens,nkv,d,ps", [
    ([1, 15, 16, 17, 0, 100, 333], 8, 128, 16),
    ([40, 7, 65], 4, 256, 32),
    ([129, 1, 64], 3, 64, 64),
], ids=["d128", "d256", "d64"])
def test_write_whole(mb, torch_cuda, dtype, lens, nkv, d, ps):
    """Whole sequences: codes and scales are exact."""
    torch = torch_cuda
    c = Cache(mb, torch, lens, nkv, d, ps, seed=1)
    k, v = fill(mb, torch, c, nkv, 2, getattr(torch, dtype))
    row = 0
    for b, n in enumerate(lens):
        for rows, which in ((k, "k"), (v, "v")):
            got = c.values(b, n, which)
            for t0 in range(0, n, 16):
                x = rows[row + t0:row + min(n, t0 + 16)]
                s = scale_of(torch, x.abs().amax(dim=(0, 2)))[None, :, None]
                assert torch.equal(got[t0:t0 + 16], e4m3(torch, x / s) * s), (b, t0, which)
        row += n


def test_write_token_by_token_matches_definition(mb, torch_cuda):
    """One row a step, magnitudes growing and shrinking: a block's scale only
    grows while it fills, and its older codes are rounded to the new scale."""
    torch = torch_cuda
    nkv, d, ps, n = 2, 64, 16, 50
    c = Cache(mb, torch, [n], nkv, d, ps, seed=3)
    g = torch.Generator().manual_seed(4)
    mag = torch.exp2(torch.randint(-12, 13, (n, nkv, 1), generator=g).double())
    k = (torch.randn(n, nkv, d, generator=g).double() * mag).float()
    v = (torch.randn(n, nkv, d, generator=g).double() / mag).float()
    k[20] = 0
    plan = mb.F8Plan()
    want = {"k": torch.zeros(n, nkv, d).double(), "v": torch.zeros(n, nkv, d).double()}
    cur = {}
    for t in range(n):
        plan.build(nkv, nkv, d, [t + 1])
        plan.write(c.layer, k[t:t + 1].cuda(), v[t:t + 1].cuda())
        for which, rows in (("k", k), ("v", v)):
            s = scale_of(torch, rows[t].double().abs().amax(dim=-1))
            if t % 16:
                s = torch.maximum(s, cur[which])
            cur[which] = s
            lo = t // 16 * 16
            want[which][t] = rows[t].double()
            blk = want[which][lo:t + 1]
            want[which][lo:t + 1] = e4m3(torch, blk / s[None, :, None]) * s[None, :, None]
    plan.close()
    for which in ("k", "v"):
        assert torch.equal(c.values(0, n, which), want[which]), which


def test_write_chunks_strides_and_counters(mb, torch_cuda):
    """Parts of a prompt out of a wider projection; the new slots' counters
    become zero, the others keep theirs; slots past the end keep their bytes."""
    torch = torch_cuda
    nkv, d, ps = 2, 128, 32
    lens, old = [70, 21], [33, 5]
    c = Cache(mb, torch, lens, nkv, d, ps, seed=5)
    c.w.fill_(2.0)
    qkv = torch.randn(sum(lens) - sum(old), 4 + 2 * nkv, d, device="cuda").bfloat16()
    full = torch.randn(sum(old), nkv, d, device="cuda").bfloat16()
    plan = mb.F8Plan()
    plan.build(nkv, nkv, d, old, new_lens=old)
    plan.write(c.layer, full, full)
    c.w.fill_(2.0)
    plan.build(nkv, nkv, d, lens, new_lens=[a - b for a, b in zip(lens, old)])
    k, v = qkv[:, 4:4 + nkv], qkv[:, 4 + nkv:]
    assert not k.is_contiguous()
    plan.write(c.layer, k, v)
    plan.close()
    row = 0
    for b, (n, m) in enumerate(zip(lens, old)):
        got = c.values(b, n, "k")[m:]
        x = k[row:row + n - m].double().cpu()
        row += n - m
        # half a step of the block's largest magnitude covers any scale the
        # partly filled block ends with
        assert torch.all((got - x).abs() <= x.abs() / 16 + 2.0 ** -9 * 8 * 2)
        w = c.counters(b, n)
        assert torch.all(w[:m] == 2) and torch.all(w[m:] == 0)
        page, sub = c.slots(b, ((n + ps - 1) // ps) * ps)
        assert torch.all(c.k.cpu()[page, :, sub][n:] == 0x7F)


def test_write_special_values(mb, torch_cuda):
    """Infinities saturate and set no scale, NaN stays NaN, zeros and the
    largest and smallest magnitudes keep within the scale's range."""
    torch = torch_cuda
    nkv, d = 1, 64
    c = Cache(mb, torch, [16 * 5], nkv, d, 16, seed=6)
    k = torch.zeros(80, nkv, d)
    k[0, 0, 0], k[0, 0, 1], k[0, 0, 2], k[0, 0, 3] = math.inf, -math.inf, math.nan, 448.0
    k[16, 0, 0] = 3.4e38
    k[32, 0, 0] = 1e-38
    k[48, 0, :2] = torch.tensor([448.5, -1.0])
    plan = mb.F8Plan()
    plan.build(1, 1, d, [80], new_lens=[80])
    plan.write(c.layer, k.cuda(), torch.zeros_like(k).cuda())
    plan.close()
    x = c.values(0, 80, "k")[:, 0]
    assert x[0, :2].tolist() == [448.0, -448.0] and x[0, 2].isnan() and x[0, 3] == 448.0
    assert x[16, 0] == e4m3(torch, k[16, 0, 0].double() / 2.0 ** 120) * 2.0 ** 120
    assert x[32, 0] == 0 and torch.all(x[64:] == 0)
    assert x[48, :2].tolist() == [448.0, -1.0]  # scale 2, 448.5 / 2 rounds to 224
    page, sub = c.slots(0, 80)
    assert c.ks.cpu()[page, 0, sub // 16][::16].tolist() == [1.0, 2.0 ** 120, 2.0 ** -64, 2.0,
                                                             2.0 ** -64]


# ---------------------------------------------------------------- decode

def decode_ref(torch, c, q, b, n, scale, cap, slopes, first, prefix, window):
    """float64 o, lse, weights [nq][n], and sum p |v| for the error bound."""
    nq = q.shape[1]
    G = nq // c.nkv
    k, v = c.values(b, n, "k"), c.values(b, n, "v")
    t = torch.arange(n)
    see = (t >= first) & ((window <= 0) | (n - 1 - t < window) | (t < first + prefix))
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    o, lse, ps, av = [], [], [], []
    for h in range(nq):
        s = (k[:, h // G] @ q[b, h].double()) * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - slopes[h].double() * (n - 1 - t)
        s = torch.where(see, s, -math.inf)
        if not bool(see.any()):
            p, z = torch.zeros(n).double(), torch.tensor(-math.inf).double()
        else:
            z = torch.logsumexp(s, 0)
            p = torch.exp(s - z)
        o.append(p @ v[:, h // G])
        av.append(p @ v[:, h // G].abs())
        lse.append(z)
        ps.append(p)
    return torch.stack(o), torch.stack(lse), torch.stack(ps), torch.stack(av)


CASES = {
    "ragged": dict(lens=[1, 15, 16, 17, 100, 1000, 333, 0], nq=32, nkv=8, d=128, ps=16),
    "long": dict(lens=[9000, 3], nq=8, nkv=2, d=128, ps=32),
    "window_sinks": dict(lens=[900, 40, 5, 257], nq=8, nkv=4, d=256, ps=16, window=100, prefix=20),
    "window_one": dict(lens=[33, 1, 200], nq=4, nkv=4, d=64, ps=64, window=1),
    "cap": dict(lens=[500, 77], nq=16, nkv=2, d=128, ps=16, cap=5.0),
    "bias": dict(lens=[700, 2, 31], nq=12, nkv=4, d=64, ps=16, bias=True),
    "documents": dict(lens=[400, 64, 17, 30], nq=10, nkv=2, d=128, ps=16, starts=[123, 64, 16, 0],
                      prefix=3, window=50),
    "all": dict(lens=[1500, 260], nq=32, nkv=8, d=128, ps=16, starts=[100, 7], prefix=40,
                window=600, cap=20.0, bias=True),
    "group16": dict(lens=[300, 90], nq=16, nkv=1, d=128, ps=16, cap=30.0),
    "group9": dict(lens=[210], nq=18, nkv=2, d=64, ps=16, bias=True),
    "group3_d256": dict(lens=[130, 48], nq=9, nkv=3, d=256, ps=16),
}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("name", CASES)
def test_decode(mb, torch_cuda, name, dtype):
    torch = torch_cuda
    cs = dict(dict(window=0, prefix=0, cap=0.0, bias=False, starts=None), **CASES[name])
    lens, nq, nkv, d = cs["lens"], cs["nq"], cs["nkv"], cs["d"]
    ty = getattr(torch, dtype)
    c = Cache(mb, torch, lens, nkv, d, cs["ps"], seed=11)
    fill(mb, torch, c, nq, 12, torch.float32)
    c.w.copy_(torch.rand(c.w.shape, generator=torch.Generator().manual_seed(1)))
    g = torch.Generator().manual_seed(13)
    q = torch.randn(len(lens), nq, d, generator=g).to(ty)
    slopes = torch.exp2(-torch.arange(1, nq + 1).float() / 2) if cs["bias"] else None
    scale = d ** -0.5
    plan = mb.F8Plan()
    plan.build(nq, nkv, d, lens, starts=cs["starts"], prefix=[cs["prefix"]] * len(lens),
               window=cs["window"])
    o = torch.full((len(lens), nq, d), math.nan, device="cuda", dtype=ty)
    lse = torch.full((len(lens), nq), math.nan, device="cuda")
    wout = torch.full_like(c.w, math.nan)
    sl = None if slopes is None else slopes.cuda()
    plan.decode(c.layer, q.cuda(), o, scale, softcap=cs["cap"], slopes=sl, lse=lse,
                weight_out=wout)
    o2 = torch.empty_like(o)
    plan.decode(c.layer, q.cuda(), o2, scale, softcap=cs["cap"], slopes=sl)
    assert torch.equal(o, o2)  # counting changes nothing
    w2 = c.w.clone()
    lay2 = mb.F8Layer(c.k, c.v, c.ks, c.vs, c.bt.cuda(), weight=w2)
    plan.decode(lay2, q.cuda(), o2, scale, softcap=cs["cap"], slopes=sl, weight_out=w2)
    plan.close()
    for b, n in enumerate(lens):
        first = cs["starts"][b] if cs["starts"] else 0
        want, z, p, av = decode_ref(torch, c, q, b, n, scale, cs["cap"], slopes, first,
                                    cs["prefix"], cs["window"])
        got = o[b].double().cpu()
        tol = U_OUT[dtype] * want.abs() + (U_P[dtype] + 2 * U_S) * av
        assert torch.all((got - want).abs() <= tol + 1e-30), (b, n)
        zg = lse[b].double().cpu()
        if n == 0 or first == n:
            assert torch.all(zg == -math.inf) and torch.all(got == 0)
        else:
            assert torch.all((zg - z).abs() <= U_S + 2.0 ** -23 * z.abs()), (b, n)
        if n:
            w = c.counters(b, n) + p.view(nkv, nq // nkv, n).sum(dim=1).t()
            for pool in (wout, w2):
                gw = c.counters(b, n, pool)
                assert torch.all((gw - w).abs() <= 4 * U_S * nq / nkv + 2.0 ** -22 * w), (b, n)


def test_decode_masked_slots_hold_anything(mb, torch_cuda):
    """NaN rows outside the visible slots (before the start, between prefix
    and window, past the end of a block) leave the output untouched; blocks
    whose scales differ by 2^40 keep FP32 accuracy."""
    torch = torch_cuda
    n, nq, nkv, d = 600, 8, 2, 128
    c = Cache(mb, torch, [n], nkv, d, 16, seed=21)
    g = torch.Generator().manual_seed(22)
    k = torch.randn(n, nkv, d, generator=g)
    v = torch.randn(n, nkv, d, generator=g)
    v[300:420] *= 2.0 ** 40
    v[500:520] *= 2.0 ** -40
    first, prefix, window = 37, 10, 290
    seen = torch.zeros(n, dtype=torch.bool)
    seen[first:first + prefix] = True
    seen[n - window:] = True
    k[~seen], v[~seen] = math.nan, math.nan
    plan = mb.F8Plan()
    plan.build(nq, nkv, d, [n], new_lens=[n])
    plan.write(c.layer, k.cuda(), v.cuda())
    q = torch.randn(1, nq, d, generator=g)
    # heads 0..3 look away from the large rows, the others see all alike
    plan.build(nq, nkv, d, [n], starts=[first], prefix=[prefix], window=window)
    o = torch.empty(1, nq, d, device="cuda")
    for bias in (0.0, 1.0):  # 1: the newest rows outweigh those of 2^40 by far
        slopes = torch.full((nq,), bias)
        plan.decode(c.layer, q.cuda(), o, d ** -0.5, slopes=slopes.cuda())
        want, _, _, av = decode_ref(torch, c, q, 0, n, d ** -0.5, 0.0, slopes, first, prefix,
                                    window)
        assert torch.all((o[0].double().cpu() - want).abs() <= (U_P["float32"] + 2 * U_S) * av)
    plan.close()


def test_decode_other_stream_and_strided_queries(mb, torch_cuda):
    torch = torch_cuda
    lens, nq, nkv, d = [321, 64], 8, 2, 64
    c = Cache(mb, torch, lens, nkv, d, 16, seed=31)
    fill(mb, torch, c, nq, 32, torch.float16)
    qkv = torch.randn(2, nq + 2 * nkv, d, device="cuda", dtype=torch.float16)
    plan = mb.F8Plan()
    plan.build(nq, nkv, d, lens)
    o = torch.empty(2, nq, d, device="cuda", dtype=torch.float16)
    plan.decode(c.layer, qkv[:, :nq].contiguous(), o, 0.125)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o2 = torch.zeros_like(o)
    side.wait_stream(torch.cuda.current_stream())
    plan.decode(c.layer, qkv[:, :nq], o2, 0.125, stream=side)
    side.synchronize()
    assert torch.equal(o, o2)
    plan.close()


# ---------------------------------------------------------------- evict

@pytest.mark.parametrize("lens,budget,recent,nkv,d,ps", [
    ([300, 40, 33, 0, 64], 48, 8, 2, 128, 16),
    ([1000, 65], 64, 64, 3, 64, 32),
    ([777, 17], 100, 0, 4, 256, 16),
    ([5000, 2100], 1025, 129, 2, 64, 64),
    ([20], 1, 1, 1, 128, 16),
    ([20], 1, 0, 1, 128, 16),
])
def test_evict(mb, torch_cuda, lens, budget, recent, nkv, d, ps):
    """Kept slots, their counters, codes and scales are exact."""
    torch = torch_cuda
    c = Cache(mb, torch, lens, nkv, d, ps, seed=41)
    fill(mb, torch, c, nkv, 42, torch.float32, spread=1.5)
    g = torch.Generator().manual_seed(43)
    w = torch.rand(c.w.shape, generator=g)
    w = torch.where(w < 0.7, torch.floor(w * 8) / 8, w * 9)  # many ties, zeros among them
    w.view(-1)[::37] = -0.0
    c.w.copy_(w)
    dst = Cache(mb, torch, [min(n, budget) for n in lens], nkv, d, ps, seed=44)
    plan = mb.F8Plan()
    plan.build(nkv, nkv, d, lens)
    kept = torch.full((len(lens), nkv, budget), 7, dtype=torch.int32, device="cuda")
    plan.evict(c.layer, dst.layer, budget, recent, kept)
    plan.close()
    for b, n in enumerate(lens):
        m = min(n, budget)
        w = c.counters(b, n)
        kv, vv = c.values(b, n, "k"), c.values(b, n, "v")
        gk, gv, gw = dst.values(b, m, "k"), dst.values(b, m, "v"), dst.counters(b, m)
        for h in range(nkv):
            keep = list(range(n))
            if n > budget:
                best = sorted(range(n - recent), key=lambda t: (-float(w[t, h]), t))
                keep = sorted(best[:budget - recent]) + list(range(n - recent, n))
            assert kept[b, h].tolist() == keep + [-1] * (budget - m), (b, h)
            assert torch.equal(gw[:, h], w[keep, h])
            for x, got in ((kv, gk), (vv, gv)):
                x = x[keep, h]
                for t0 in range(0, m, 16):
                    blk = x[t0:t0 + 16]
                    s = scale_of(torch, blk.abs().amax())
                    assert torch.equal(got[t0:t0 + 16, h], e4m3(torch, blk / s) * s), (b, h, t0)


def test_evict_unordered_counters(mb, torch_cuda):
    """NaN counters go first, infinite ones last, negative ones in order."""
    torch = torch_cuda
    n, budget = 40, 36
    c = Cache(mb, torch, [n], 1, 64, 16, seed=51)
    fill(mb, torch, c, 1, 52, torch.float32)
    vals = torch.arange(n).float() - 20.0
    vals[5], vals[30], vals[31] = math.inf, math.nan, -math.inf
    page, sub = c.slots(0, n)
    w = c.w.cpu()
    w[page, 0, sub] = vals
    c.w.copy_(w)
    dst = Cache(mb, torch, [budget], 1, 64, 16, seed=53)
    plan = mb.F8Plan()
    plan.build(1, 1, 64, [n])
    kept = torch.zeros(1, 1, budget, dtype=torch.int32, device="cuda")
    plan.evict(c.layer, dst.layer, budget, 0, kept)
    plan.close()
    assert kept[0, 0].tolist() == [t for t in range(n) if t not in (30, 31, 0, 1)]


# ---------------------------------------------------------------- refusals

def test_refusals(mb, torch_cuda):
    torch = torch_cuda
    nq, nkv, d, lens = 4, 2, 64, [40]
    c = Cache(mb, torch, lens, nkv, d, 16, seed=61)
    q = torch.zeros(1, nq, d, device="cuda")
    o = torch.zeros_like(q)
    plan = mb.F8Plan()
    with pytest.raises(ValueError):
        plan.decode(c.layer, q, o, 1.0)  # not built

    def refused(status, *args, **kw):
        with pytest.raises(mb.MolotError) as e:
            plan.build(*args, **kw)
        assert e.value.status == status

    refused(mb.ERR_INVALID, 3, 2, d, lens)
    refused(mb.ERR_UNSUPPORTED, 4, 2, 96, lens)
    refused(mb.ERR_UNSUPPORTED, 130, 2, d, lens)
    refused(mb.ERR_INVALID, 4, 2, d, [-1])
    refused(mb.ERR_INVALID, 4, 2, d, [5], new_lens=[6])
    refused(mb.ERR_INVALID, 4, 2, d, [5], starts=[6])
    refused(mb.ERR_INVALID, 4, 2, d, [5], prefix=[-1])
    refused(mb.ERR_INVALID, 4, 2, d, [])
    with pytest.raises(ValueError):
        plan.build(4, 2, d, [5, 6], starts=[0])
    plan.build(nq, nkv, d, lens)
    for bad in (dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=math.nan)):
        with pytest.raises(mb.MolotError) as e:
            plan.decode(c.layer, q, o, 1.0, **bad)
        assert e.value.status == mb.ERR_INVALID
    with pytest.raises(ValueError):
        plan.decode(c.layer, q.half(), o, 1.0)
    with pytest.raises(ValueError):
        plan.decode(c.layer, q[:, :2], o, 1.0)
    with pytest.raises(ValueError):
        plan.decode(c.layer, q, o.transpose(1, 2).contiguous().transpose(1, 2), 1.0)
    no_w = mb.F8Layer(c.k, c.v, c.ks, c.vs, c.bt.cuda())
    with pytest.raises(mb.MolotError):
        plan.decode(no_w, q, o, 1.0, weight_out=c.w)
    narrow = mb.F8Layer(c.k, c.v, c.ks, c.vs, c.bt[:, :2].contiguous().cuda())
    with pytest.raises(mb.MolotError) as e:
        plan.decode(narrow, q, o, 1.0)  # 32 of 40 slots
    assert e.value.status == mb.ERR_INVALID
    kept = torch.zeros(1, nkv, 8, dtype=torch.int32, device="cuda")
    for budget, recent in ((8, 9), (8, -1)):
        with pytest.raises(mb.MolotError):
            plan.evict(c.layer, c.layer, budget, recent, kept)
    with pytest.raises(ValueError):
        plan.evict(c.layer, c.layer, 9, 1, kept)
    with pytest.raises(mb.MolotError):
        plan.evict(no_w, c.layer, 8, 1, kept)
    rows = torch.zeros(1, nkv, d, device="cuda")
    with pytest.raises(ValueError):
        plan.write(c.layer, rows, rows.half())
    with pytest.raises(ValueError):
        plan.write(c.layer, rows.double(), rows.double())
    with pytest.raises(ValueError):
        mb.F8Layer(c.k, c.v, c.ks[:, :, :0], c.vs, c.bt.cuda())
    with pytest.raises(ValueError):
        mb.F8Layer(c.k.int(), c.v, c.ks, c.vs, c.bt.cuda())
    with pytest.raises(ValueError):
        mb.F8Layer(c.k, c.v, c.ks, c.vs, c.bt.long().cuda())
    plan.close()


def test_serving_loop(mb, torch_cuda):
    """The operators as a server runs them: packed prefill of two prompts,
    their rows into the pager's pools, decode steps that count weights, an
    eviction into new pages, decode over what was kept -- against the same
    loop in float64 over the cache's own values."""
    torch = torch_cuda
    nq, nkv, d, ps, budget = 8, 2, 64, 16, 64
    ty = torch.bfloat16
    g = torch.Generator().manual_seed(71)
    prompts = [90, 37]
    pager = mb.Pager(1, nkv, d, ps, 40, 8, 12, dtype="f8b")
    seqs = [pager.add(n) for n in prompts]
    qkv = torch.randn(sum(prompts), nq + 2 * nkv, d, generator=g).to(ty).cuda()
    q, k, v = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    packed = mb.PackedPlan()
    packed.build(nq, nkv, d, prompts)
    o = torch.empty(sum(prompts), nq, d, device="cuda", dtype=ty)
    packed.attend(q, k, v, o, d ** -0.5, softcap=30.0)
    assert torch.isfinite(o).all()
    plan = mb.F8Plan()
    bt, lens = pager.tables(seqs)
    layer = pager.f8_layer(0, torch.from_numpy(bt).cuda())
    plan.build(nq, nkv, d, lens, new_lens=lens)
    plan.write(layer, k, v)

    def view():
        c = Cache.__new__(Cache)
        c.torch, c.nkv, c.d, c.ps = torch, nkv, d, ps
        c.bt = torch.from_numpy(bt)
        c.k, c.v = pager.layer_pools(0)
        c.ks, c.vs, c.w = pager.layer_blocks(0)
        return c

    sums = [torch.zeros(int(n), nkv).double() for n in lens]
    for step in range(6):
        for s in seqs:
            pager.grow(s)
        bt, lens = pager.tables(seqs)
        layer = pager.f8_layer(0, torch.from_numpy(bt).cuda())
        x = torch.randn(2, nq + 2 * nkv, d, generator=g).to(ty).cuda()
        plan.build(nq, nkv, d, lens)
        plan.write(layer, x[:, nq:nq + nkv], x[:, nq + nkv:])
        o = torch.empty(2, nq, d, device="cuda", dtype=ty)
        plan.decode(layer, x[:, :nq], o, d ** -0.5, softcap=30.0, weight_out=layer.tensors[4])
        c = view()
        for b in range(2):
            n = int(lens[b])
            want, _, p, av = decode_ref(torch, c, x[:, :nq].cpu(), b, n, d ** -0.5, 30.0, None, 0,
                                        0, 0)
            tol = U_OUT["bfloat16"] * want.abs() + (U_P["bfloat16"] + 2 * U_S) * av
            assert torch.all((o[b].double().cpu() - want).abs() <= tol)
            sums[b] = torch.cat([sums[b], torch.zeros(1, nkv).double()])
            sums[b] += p.view(nkv, nq // nkv, n).sum(dim=1).t()
            assert torch.all((c.counters(b, n) - sums[b]).abs() <= 1e-3)
    # the longer sequence is brought down to its budget in pages of its own
    s_new = [pager.add(min(int(n), budget)) for n in lens]
    bt2, lens2 = pager.tables(s_new)
    dst = pager.f8_layer(0, torch.from_numpy(bt2).cuda())
    kept = torch.empty(2, nkv, budget, dtype=torch.int32, device="cuda")
    plan.evict(layer, dst, budget, 16, kept)
    for s in seqs:
        pager.free(s)
    plan.build(nq, nkv, d, lens2)
    o = torch.empty(2, nq, d, device="cuda", dtype=ty)
    plan.decode(dst, x[:, :nq], o, d ** -0.5)
    bt = bt2
    c = view()
    for b in range(2):
        want, _, _, av = decode_ref(torch, c, x[:, :nq].cpu(), b, int(lens2[b]), d ** -0.5, 0.0,
                                    None, 0, 0, 0)
        tol = U_OUT["bfloat16"] * want.abs() + (U_P["bfloat16"] + 2 * U_S) * av
        assert torch.all((o[b].double().cpu() - want).abs() <= tol)
    plan.close()
    packed.close()
    pager.close()

"""The 8-bit cache at lengths and batches where a decode is shared out in
each of its ways (clusters, ranges that end with the segments, ranges that
straddle them), at pool offsets beyond 32 bits, and evictions whose keys do
not fit on chip; against the definition in 64 bits on the GPU."""
import math

import pytest

pytestmark = pytest.mark.gpu

U_P = 2.0 ** -20  # weights split in two FP16 parts
U_S = 8e-6        # relative error of a weight from its score


def pools(torch, pages, nkv, ps, d, g, weight=False):
    """Random codes and scales (any byte but the two NaN codes)."""
    k = torch.randint(0, 126, (pages, nkv, ps, d), dtype=torch.uint8, device="cuda", generator=g)
    v = torch.randint(0, 126, (pages, nkv, ps, d), dtype=torch.uint8, device="cuda", generator=g)
    k = k // 2 + 128 * (k & 1)  # both signs, below 2
    v = v // 2 + 128 * (v & 1)
    ks = torch.exp2(torch.randint(-2, 2, (pages, nkv, ps // 16), device="cuda",
                                  generator=g).float())
    vs = torch.exp2(torch.randint(-2, 2, (pages, nkv, ps // 16), device="cuda",
                                  generator=g).float())
    return k, v, ks, vs


def rows(torch, codes, scale, bt, b, n, h, ps):
    t = torch.arange(n, device="cuda")
    page = bt[b].long()[t // ps]
    c = codes[page, h, t % ps].view(torch.float8_e4m3fn).double()
    return c * scale[page, h, (t % ps) // 16].double()[:, None]


@pytest.mark.parametrize("lens,nq,nkv,d,ps", [
    ([4097], 32, 8, 128, 16),                                  # clusters
    ([66 * 16, 3, 0, 500], 8, 4, 256, 16),                     # clusters, ragged
    ([40001], 8, 2, 128, 32),                                  # ranges that end with the segments
    ([30000, 29000, 1], 4, 2, 64, 16),
    ([17 * i % 2900 + 1 for i in range(60)], 16, 8, 128, 16),  # ranges that straddle segments
    ([3000, 0, 1, 2500, 15] * 20, 20, 5, 64, 48),
    ([2000] * 40, 8, 4, 256, 16),
    ([1500, 700] * 30, 32, 2, 128, 16),                        # two head groups
], ids=str)
def test_decode_shares(mb, torch_cuda, lens, nq, nkv, d, ps):
    torch = torch_cuda
    g = torch.Generator(device="cuda")
    g.manual_seed(sum(lens))
    need = [max(1, math.ceil(n / ps)) for n in lens]
    pages = sum(need) + 2
    k, v, ks, vs = pools(torch, pages, nkv, ps, d, g)
    perm = torch.randperm(pages, device="cuda", generator=g).int()
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    i = 0
    for b, m in enumerate(need):
        bt[b, :m] = perm[i:i + m]
        i += m
    q = torch.randn(len(lens), nq, d, device="cuda", generator=g)
    o = torch.full_like(q, math.nan)
    lse = torch.full((len(lens), nq), math.nan, device="cuda")
    plan = mb.F8Plan()
    plan.build(nq, nkv, d, lens)
    layer = mb.F8Layer(k, v, ks, vs, bt)
    plan.decode(layer, q, o, d ** -0.5, lse=lse)
    first = o.clone()
    plan.decode(layer, q, o, d ** -0.5, lse=lse)
    assert torch.equal(o, first)  # the merge does not depend on who comes last
    plan.check()
    plan.close()
    G = nq // nkv
    for b, n in enumerate(lens):
        if n == 0:
            assert torch.all(o[b] == 0) and torch.all(lse[b] == -math.inf)
            continue
        for h in range(nkv):
            kk, vv = rows(torch, k, ks, bt, b, n, h, ps), rows(torch, v, vs, bt, b, n, h, ps)
            s = q[b, h * G:(h + 1) * G].double() @ kk.T * d ** -0.5
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            want, av = p @ vv, p @ vv.abs()
            got = o[b, h * G:(h + 1) * G].double()
            assert torch.all((got - want).abs() <= 2.0 ** -23 * want.abs() + (U_P + 2 * U_S) * av)
            zg = lse[b, h * G:(h + 1) * G].double()
            assert torch.all((zg - z).abs() <= U_S + 2.0 ** -22 * z.abs())


def test_offsets_beyond_32_bits(mb, torch_cuda):
    """Pages whose codes lie past 4 GB of their pool: written, attended to,
    evicted from and to."""
    torch = torch_cuda
    nkv, d, ps, pages, n, budget = 8, 256, 64, 40000, 200, 90
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    k = torch.zeros(pages, nkv, ps, d, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 32
    ks = torch.ones(pages, nkv, ps // 16, device="cuda")
    vs = torch.ones_like(ks)
    w = torch.rand(pages, nkv, ps, device="cuda", generator=g)
    bt = torch.tensor([[39999, 35001, 39000, 33333]], dtype=torch.int32, device="cuda")
    bt2 = torch.tensor([[39998, 34000]], dtype=torch.int32, device="cuda")
    kr = torch.randn(n, nkv, d, device="cuda", generator=g)
    vr = torch.randn(n, nkv, d, device="cuda", generator=g)
    plan = mb.F8Plan()
    plan.build(nkv, nkv, d, [n], new_lens=[n])
    plan.write(mb.F8Layer(k, v, ks, vs, bt), kr, vr)
    src = mb.F8Layer(k, v, ks, vs, bt, weight=w)
    q = torch.randn(1, nkv, d, device="cuda", generator=g)
    o = torch.empty_like(q)
    plan.decode(src, q, o, d ** -0.5)
    kept = torch.empty(1, nkv, budget, dtype=torch.int32, device="cuda")
    plan.evict(src, mb.F8Layer(k, v, ks, vs, bt2, weight=w), budget, 10, kept)
    plan.check()
    plan.close()
    for h in range(nkv):
        kk, vv = rows(torch, k, ks, bt, 0, n, h, ps), rows(torch, v, vs, bt, 0, n, h, ps)
        assert torch.all((kk - kr[:, h].double()).abs() <= kr[:, h].double().abs() / 16 + 2.0 ** -9)
        p = torch.softmax(q[0, h].double() @ kk.T * d ** -0.5, 0)
        want, av = p @ vv, p @ vv.abs()
        assert torch.all((o[0, h].double() - want).abs() <= 2.0 ** -23 * want.abs()
                         + (U_P + 2 * U_S) * av)
        moved = rows(torch, k, ks, bt2, 0, budget, h, ps)
        keep = kept[0, h].long()
        assert torch.all(keep[1:] > keep[:-1])
        # a row may be rounded once more, under a larger scale
        assert torch.all((moved - kk[keep]).abs() <= kk[keep].abs() / 16 + 2.0 ** -9)


@pytest.mark.parametrize("n,budget,recent", [(60000, 1000, 77), (60000, 59990, 0),
                                             (49153, 4096, 4095), (131072, 65536, 1)])
def test_evict_many(mb, torch_cuda, n, budget, recent):
    """More candidates than a CTA holds on chip; half of the counters tie."""
    torch = torch_cuda
    nkv, d, ps = 2, 64, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(n + budget)
    need, need2 = math.ceil(n / ps), math.ceil(budget / ps)
    k, v, ks, vs = pools(torch, need + need2, nkv, ps, d, g)
    w = torch.rand(need + need2, nkv, ps, device="cuda", generator=g)
    w = torch.where(w < 0.5, (w * 16).floor(), w)
    perm = torch.randperm(need + need2, device="cuda", generator=g).int()
    bt, bt2 = perm[:need].view(1, -1).contiguous(), perm[need:].view(1, -1).contiguous()
    t = torch.arange(n, device="cuda")
    before = w.clone()
    plan = mb.F8Plan()
    plan.build(nkv, nkv, d, [n])
    kept = torch.empty(1, nkv, budget, dtype=torch.int32, device="cuda")
    plan.evict(mb.F8Layer(k, v, ks, vs, bt, weight=w), mb.F8Layer(k, v, ks, vs, bt2, weight=w),
               budget, recent, kept)
    plan.close()
    j = torch.arange(budget, device="cuda")
    for h in range(nkv):
        c = before[bt[0].long()[t // ps], h, t % ps]
        order = torch.sort(c[:n - recent], descending=True, stable=True)[1][:budget - recent]
        want = torch.cat([order.sort()[0], t[n - recent:]])
        assert torch.equal(kept[0, h].long(), want)
        assert torch.equal(w[bt2[0].long()[j // ps], h, j % ps], c[want])


def test_bounded_wait_is_reported(mb, torch_cuda):
    """A decode whose copies are withheld gives up, reports it once, and
    leaves the plan usable (nothing is in flight, nothing faults)."""
    torch = torch_cuda
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    n, nkv, d, ps = 300, 2, 64, 16
    k, v, ks, vs = pools(torch, 19, nkv, ps, d, g)
    bt = torch.arange(19, dtype=torch.int32, device="cuda").view(1, -1)
    layer = mb.F8Layer(k, v, ks, vs, bt)
    q = torch.randn(1, 4, d, device="cuda", generator=g)
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    plan = mb.F8Plan()
    plan.build(4, nkv, d, [n])
    plan.decode(layer, q, o, 0.125)
    plan.check()
    mb.debug_withhold_next(1_000_000)
    plan.decode(layer, q, o2, 0.125)
    with pytest.raises(mb.MolotError) as e:
        plan.check()
    assert e.value.status == mb.ERR_TIMEOUT
    plan.check()
    plan.decode(layer, q, o2, 0.125)
    plan.check()
    assert torch.equal(o, o2)
    plan.close()

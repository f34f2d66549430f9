"""Packed-document prefill attention on the GPU against its definition in 64
bits, at the masks and sizes where it can go wrong, and its refusals."""
import math

import pytest

pytestmark = pytest.mark.gpu

U_OUT = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # unit roundoff (8 and 11 significant bits)
# Weights are rounded to the operands' type before their product with V.
U_P = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# Relative error of a weight from its score (FP32 sums, exponential, cap).
U_S = 2e-5


def reference(torch, q, k, v, q_lens, k_lens, prefix, window, scale, cap, slopes):
    """float64 o, lse, and sum p |v| for the error bound."""
    T, nq, d = q.shape
    nkv = k.shape[1]
    o = torch.zeros(T, nq, d, dtype=torch.float64, device=q.device)
    av = torch.zeros_like(o)
    lse = torch.full((T, nq), -math.inf, dtype=torch.float64, device=q.device)
    q0 = k0 = 0
    for m, n, pre in zip(q_lens, k_lens, prefix):
        if m and n:
            pos = torch.arange(n - m, n, device=q.device)[:, None]
            t = torch.arange(n, device=q.device)[None, :]
            see = t <= pos
            if window > 0:
                see = see & (pos - t < window)
            see = see | (t < pre)
            some = see.any(dim=1)
            for h in range(nq):
                kk = k[k0:k0 + n, h * nkv // nq].double()
                vv = v[k0:k0 + n, h * nkv // nq].double()
                s = q[q0:q0 + m, h].double() @ kk.T * scale
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    s = s - slopes[h].double() * (pos - t).abs()
                s = torch.where(see, s, -math.inf)
                z = torch.logsumexp(s, 1)
                p = torch.where(some[:, None], torch.exp(s - z[:, None]), 0.0)
                o[q0:q0 + m, h] = p @ vv
                av[q0:q0 + m, h] = p @ vv.abs()
                lse[q0:q0 + m, h] = z
        q0 += m
        k0 += n
    return o, lse, av


CASES = {
    "one_token": dict(q=[1], nq=8, nkv=2, d=128),
    "short": dict(q=[77], nq=4, nkv=1, d=128, cap=30.0),
    "tile_edges": dict(q=[127, 128, 129, 255, 256, 257, 1, 64, 65], nq=4, nkv=2, d=128),
    "d64": dict(q=[300, 5, 0, 700], nq=6, nkv=2, d=64, bias=True),
    "d256": dict(q=[200, 333], nq=4, nkv=2, d=256, cap=50.0),
    "past": dict(q=[40, 1, 130], k=[500, 129, 130], nq=8, nkv=2, d=128),
    "fewer_keys": dict(q=[50, 300], k=[20, 170], nq=4, nkv=4, d=64),
    "no_keys": dict(q=[20, 30], k=[0, 64], nq=2, nkv=1, d=128),
    "window": dict(q=[1000, 300], nq=4, nkv=2, d=128, window=100),
    "window_one": dict(q=[270], nq=2, nkv=2, d=64, window=1),
    "window_past": dict(q=[150], k=[1400], nq=4, nkv=1, d=256, window=333),
    "prefix": dict(q=[500, 20, 300], nq=4, nkv=2, d=128, prefix=[130, 50, 0]),
    "prefix_window": dict(q=[900, 700], nq=4, nkv=2, d=128, prefix=[10, 260], window=128),
    "prefix_negative": dict(q=[100], k=[30], nq=2, nkv=1, d=64, prefix=[12]),
    "bias_cap_all": dict(q=[400, 129], k=[700, 129], nq=8, nkv=2, d=128, prefix=[150, 7],
                         window=200, cap=10.0, bias=True),
    "window_unlimited": dict(q=[100, 40], k=[30, 200], nq=4, nkv=2, d=64, window=2 ** 31 - 1),
    "group1": dict(q=[190], nq=3, nkv=3, d=128),
    "group8": dict(q=[190, 33], nq=16, nkv=2, d=128, bias=True),
    "group5": dict(q=[140], nq=5, nkv=1, d=64),
}


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("name", CASES)
def test_packed(mb, torch_cuda, name, dtype):
    torch = torch_cuda
    cs = CASES[name]
    q_lens = cs["q"]
    k_lens = cs.get("k", q_lens)
    nq, nkv, d = cs["nq"], cs["nkv"], cs["d"]
    prefix = cs.get("prefix", [0] * len(q_lens))
    window, cap = cs.get("window", 0), cs.get("cap", 0.0)
    ty = getattr(torch, dtype)
    g = torch.Generator().manual_seed(5)
    T, K = sum(q_lens), sum(k_lens)
    q = (2 * torch.randn(T, nq, d, generator=g)).to(ty).cuda()
    kv = torch.randn(K, 2 * nkv, d, generator=g).to(ty).cuda()
    k, v = kv[:, :nkv], kv[:, nkv:]
    slopes = torch.exp2(-torch.arange(1, nq + 1).float()).cuda() if cs.get("bias") else None
    plan = mb.PackedPlan()
    plan.build(nq, nkv, d, q_lens, k_lens=k_lens, prefix=prefix, window=window)
    o = torch.full((T, nq, d), math.nan, device="cuda", dtype=ty)
    lse = torch.full((T, nq), math.nan, device="cuda")
    plan.attend(q, k, v, o, d ** -0.5, softcap=cap, slopes=slopes, lse=lse)
    o2 = torch.full_like(o, math.nan)
    plan.attend(q, k, v, o2, d ** -0.5, softcap=cap, slopes=slopes)
    plan.close()
    assert torch.equal(o, o2)
    want, z, av = reference(torch, q, k, v, q_lens, k_lens, prefix, window, d ** -0.5, cap, slopes)
    tol = U_OUT[dtype] * want.abs() + (U_P[dtype] + 2 * U_S) * av + 1e-30
    err = (o.double() - want).abs()
    assert torch.all(err <= tol), float((err / tol).max())
    empty = z == -math.inf
    assert torch.all(lse.double()[empty] == -math.inf) and torch.all(o[empty] == 0)
    assert torch.all((lse.double() - z).abs()[~empty] <= (U_S + 2.0 ** -22 * z.abs())[~empty])


def test_packed_ignores_what_it_may_not_see(mb, torch_cuda):
    """NaN and infinities in rows that the mask hides, and in the neighbouring
    documents, leave a document's outputs as they are."""
    torch = torch_cuda
    nq, nkv, d = 4, 2, 128
    lens, window = [200, 300, 90], 64
    g = torch.Generator().manual_seed(6)
    T = sum(lens)
    q = torch.randn(T, nq, d, generator=g).bfloat16().cuda()
    k = torch.randn(T, nkv, d, generator=g).bfloat16().cuda()
    v = torch.randn(T, nkv, d, generator=g).bfloat16().cuda()
    plan = mb.PackedPlan()
    plan.build(nq, nkv, d, lens, window=window)
    o = torch.empty(T, nq, d, device="cuda", dtype=torch.bfloat16)
    plan.attend(q, k, v, o, d ** -0.5)
    k2, v2 = k.clone(), v.clone()
    for x, val in ((k2, math.nan), (v2, math.nan)):
        x[:200] = val
        x[490:] = val
    k2[200:230], v2[200:230] = math.inf, -math.inf
    o2 = torch.empty_like(o)
    plan.attend(q, k2, v2, o2, d ** -0.5)
    plan.close()
    # rows of the middle document whose window starts at 230 or later
    assert torch.equal(o[230 + window - 1:490], o2[230 + window - 1:490])


def test_packed_infinite_and_large_scores(mb, torch_cuda):
    """Scores far beyond the exponential's range, and a cap that tames them."""
    torch = torch_cuda
    T, nq, nkv, d = 200, 2, 1, 64
    g = torch.Generator().manual_seed(8)
    q = (300 * torch.randn(T, nq, d, generator=g)).bfloat16().cuda()
    k = (300 * torch.randn(T, nkv, d, generator=g)).bfloat16().cuda()
    v = torch.randn(T, nkv, d, generator=g).bfloat16().cuda()
    plan = mb.PackedPlan()
    plan.build(nq, nkv, d, [T])
    o = torch.empty(T, nq, d, device="cuda", dtype=torch.bfloat16)
    plan.attend(q, k, v, o, 1.0, softcap=40.0)
    want, _, av = reference(torch, q, k, v, [T], [T], [0], 0, 1.0, 40.0, None)
    assert torch.all((o.double() - want).abs() <= U_OUT["bfloat16"] * want.abs()
                     + (U_P["bfloat16"] + 2 * U_S) * av)
    plan.attend(q, k, v, o, 1.0)  # the softmax picks one row
    best = (q.double().transpose(0, 1) @ k[:, 0].double().T)
    best = best.masked_fill(torch.ones(T, T, device="cuda").triu(1).bool(), -math.inf).argmax(-1)
    assert torch.equal(o.transpose(0, 1), v[:, 0][best])
    plan.close()


def test_packed_refusals(mb, torch_cuda):
    torch = torch_cuda
    plan = mb.PackedPlan()
    q = torch.zeros(5, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(5, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        plan.attend(q, k, k, q.clone(), 1.0)

    def refused(status, *args, **kw):
        with pytest.raises(mb.MolotError) as e:
            plan.build(*args, **kw)
        assert e.value.status == status

    refused(mb.ERR_INVALID, 3, 2, 64, [5])
    refused(mb.ERR_UNSUPPORTED, 4, 2, 80, [5])
    refused(mb.ERR_INVALID, 4, 2, 64, [-5])
    refused(mb.ERR_INVALID, 4, 2, 64, [5], k_lens=[-1])
    refused(mb.ERR_INVALID, 4, 2, 64, [5], prefix=[-1])
    refused(mb.ERR_INVALID, 4, 2, 64, [])
    with pytest.raises(ValueError):
        plan.build(4, 2, 64, [5], k_lens=[5, 5])
    plan.build(4, 2, 64, [5])
    o = torch.zeros_like(q)
    with pytest.raises(mb.MolotError) as e:
        plan.attend(q.float(), k.float(), k.float(), o.float(), 1.0)
    assert e.value.status == mb.ERR_UNSUPPORTED
    for cap in (-1.0, math.inf, math.nan):
        with pytest.raises(mb.MolotError) as e:
            plan.attend(q, k, k, o, 1.0, softcap=cap)
        assert e.value.status == mb.ERR_INVALID
    with pytest.raises(ValueError):
        plan.attend(q, k.half(), k.half(), o, 1.0)
    with pytest.raises(ValueError):
        plan.attend(q[:4], k, k, o[:4], 1.0)
    wide = torch.zeros(5, 2, 66, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        plan.attend(q, wide[:, :, :64], k, o, 1.0)  # heads not contiguous
    odd = torch.zeros(5 * 132, device="cuda", dtype=torch.bfloat16).view(5, 132)
    with pytest.raises(mb.MolotError) as e:  # rows 264 bytes apart
        plan.attend(q, odd[:, :128].view(5, 2, 64), k, o, 1.0)
    assert e.value.status == mb.ERR_INVALID
    plan.close()

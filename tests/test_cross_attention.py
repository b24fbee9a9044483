"""nn_ops.cross_attention: the kernels against 64-bit computations of the definition on the same bf16 inputs, their refusals on the CPU.

Bounds, element by element, from the roundings alone (h = 2^-8, half a step of bf16 relative to the value; e = (D + 8) 2^-24 max_j scale sum_d |q_d k_d|, the fp32
sums of a score, which exp turns into a relative error of P):
  O:   P is rounded to bf16 where it meets v and in the row sum: 2 (h + e) sum_j P |v|, and the result's rounding h |O|            =: T_O
  dv:  P carries the forward's row sum (h), its own rounding (h) and 2 e: 2 (h + e) sum_r P |dO| + h |dv|
  dS = P (dP - delta): 2 (h + e) |dS| + P sum_d |dO| T_O (delta reads the rounded O) + P (D + 2) 2^-24 sum_d |dO v|                =: T_S
  dq:  scale sum_j T_S |k| + h |dq|;   dk: scale sum_r T_S |q| + h |dk|
each times 1.05 for second-order terms and the fp32 additions of the long sums."""
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
BF = torch.bfloat16
HALF = 2.0 ** -8


def valid_keys(B, Nk, lens, mask, device):
    v = torch.ones(B, Nk, dtype=torch.bool, device=device)
    if lens is not None:
        v &= torch.arange(Nk, device=device)[None] < lens.long()[:, None]
    return v if mask is None else v & mask


def oracle(q, k, v, g=None, lens=None, mask=None, scale=None):
    """float64 O (, dq, dk, dv) and their bounds, sample by sample and head by head, on the valid keys only"""
    B, Nq, H, D = q.shape
    G = H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    ok = valid_keys(B, k.shape[1], lens, mask, q.device)
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=q.device)  # noqa: E731
    O, TO, dQ, TQ, dK, TK, dV, TV = z(q), z(q), z(q), z(q), z(k), z(k), z(v), z(v)
    for b in range(B):
        at = ok[b].nonzero()[:, 0]
        if not len(at):
            continue
        for h in range(H):
            Q, K, V = q[b, :, h].double(), k[b, at, h // G].double(), v[b, at, h // G].double()
            S = Q @ K.t() * scale
            P = torch.softmax(S, 1)
            e = (D + 8) * 2.0 ** -24 * (Q.abs() @ K.abs().t() * scale).amax(1, keepdim=True)
            o = P @ V
            to = 2 * (HALF + e) * (P @ V.abs()) + HALF * o.abs()
            O[b, :, h], TO[b, :, h] = o, to
            if g is None:
                continue
            Y = g[b, :, h].double()
            dP = Y @ V.t()
            delta = (Y * o).sum(1, keepdim=True)
            dS = P * (dP - delta)
            TS = 2 * (HALF + e) * dS.abs() + P * ((Y.abs() * to).sum(1, keepdim=True) + (D + 2) * 2.0 ** -24 * (Y.abs() @ V.abs().t()))
            dQ[b, :, h], TQ[b, :, h] = scale * dS @ K, scale * TS @ K.abs()
            for dst, val in ((dK, scale * dS.t() @ Q), (TK, scale * TS.t() @ Q.abs()), (dV, P.t() @ Y), (TV, 2 * ((HALF + e) * P).t() @ Y.abs())):
                dst[b, at, h // G] += val
    if g is None:
        return O, TO
    return (O, dQ, dK, dV), (TO, TQ + HALF * dQ.abs(), TK + HALF * dK.abs(), TV + HALF * dV.abs())


def within(name, got, want, tol):
    assert got.shape == want.shape and got.dtype == BF
    off = (got.double() - want).abs()
    bad = ~(off <= 1.05 * tol + 1e-30)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / (tol + 1e-30))[bad].max()):.3g} of the bound, " \
                          f"first at {[int(x) for x in bad.nonzero()[0]]}"


def both(q, k, v, lens=None, mask=None, scale=None, g=None):
    """the kernels' outputs and gradients against the oracle's"""
    from imagefolder_amd import nn_ops
    g = torch.randn(q.shape, device=q.device).to(BF) if g is None else g
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    y = nn_ops.cross_attention(q, k, v, kv_lens=lens, key_mask=mask, scale=scale)
    assert nn_ops.IMPL["cross_attention"] == "hip"
    grads = torch.autograd.grad(y, (q, k, v), g)
    with torch.no_grad():
        assert torch.equal(nn_ops.cross_attention(q, k, v, kv_lens=lens, key_mask=mask, scale=scale), y)
        want, tol = oracle(q, k, v, g, lens, mask, scale)
    for name, a, w, t in zip(("O", "dq", "dk", "dv"), (y.detach(),) + grads, want, tol):
        within(name, a, w, t)
    return y.detach(), grads


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 257, 12, 12, 64), (1, 1, 5000, 8, 2, 128), (3, 5, 63, 4, 4, 32), (2, 130, 65, 6, 2, 96), (2, 129, 300, 4, 1, 80),
          (1, 700, 1000, 2, 2, 128), (2, 33, 64, 3, 3, 40), (1, 2, 9001, 2, 1, 64), (4, 77, 2, 4, 2, 16), (8, 16, 128, 2, 2, 24), (1, 1500, 31, 8, 1, 64),
          (9, 257, 256, 8, 8, 64), (1, 3, 4097, 16, 1, 128), (2, 1, 1025, 16, 1, 96), (1, 17, 700, 1, 1, 112),
          # the backward in one block, its rows whole and split, at the ends of its sizes
          (2, 40, 128, 6, 2, 128), (1, 1000, 127, 2, 1, 120), (1, 700, 100, 5, 1, 56), (3, 31, 1, 2, 2, 128), (2, 65, 288, 4, 4, 64), (1, 900, 289, 2, 2, 64),
          (1, 800, 281, 3, 1, 32), (2, 33, 129, 3, 3, 8), (1, 2100, 33, 2, 2, 96), (1, 600, 97, 24, 4, 128), (70, 100, 200, 1, 1, 48)]


@gpu
@pytest.mark.parametrize("case", ["plain", "lens", "mask", "both"])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,D", SHAPES)
def test_against_64_bits(B, Nq, Nk, H, Hk, D, case):
    gen = torch.Generator(device="cuda").manual_seed(Nq * Nk + D)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF)  # noqa: E731
    q, k, v, g = r(B, Nq, H, D) * 2, r(B, Nk, Hk, D), r(B, Nk, Hk, D), r(B, Nq, H, D)
    lens = mask = None
    if case in ("lens", "both"):
        lens = torch.randint(0, Nk + 1, (B,), generator=gen, device="cuda", dtype=torch.int64 if D % 3 else torch.int32)
        if B > 1:
            lens[0], lens[-1] = 0, Nk
        else:
            lens[0] = max(1, Nk - 70)
    if case in ("mask", "both"):
        mask = torch.rand(B, Nk, generator=gen, device="cuda") < 0.6
        if B > 1:
            mask[1] = False
        if Nk > 200:
            mask[0, 64:192] = False         # whole tiles without a key
    y, grads = both(q, k, v, lens, mask, g=g)
    empty = ~valid_keys(B, Nk, lens, mask, "cuda")
    assert float(grads[1][empty].abs().sum()) == 0 and float(grads[2][empty].abs().sum()) == 0
    assert float(y[empty.all(1)].abs().sum()) == 0 and float(grads[0][empty.all(1)].abs().sum()) == 0


@gpu
@pytest.mark.parametrize("Nq,Nk,D", [(1, 333, 64), (200, 333, 64), (200, 260, 64), (90, 120, 128), (900, 70, 96)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(BF).min])
def test_what_lies_in_masked_places_reaches_nothing(Nq, Nk, D, bad):
    from imagefolder_amd import nn_ops
    B, H, Hk = 3, 4, 2
    torch.manual_seed(5)
    q, k, v, g = (torch.randn(*s, device="cuda").to(BF) for s in ((B, Nq, H, D), (B, Nk, Hk, D), (B, Nk, Hk, D), (B, Nq, H, D)))
    lens = torch.tensor([Nk // 3, 0, Nk], device="cuda")
    mask = torch.rand(B, Nk, device="cuda") < 0.5
    ok = valid_keys(B, Nk, lens, mask, "cuda")
    results = []
    for fill in (0.0, bad):
        kk, vv = (torch.where(ok[:, :, None, None], t, torch.full_like(t, fill)).requires_grad_(True) for t in (k, v))
        qq = q.clone().requires_grad_(True)
        y = nn_ops.cross_attention(qq, kk, vv, kv_lens=lens, key_mask=mask)
        results.append((y.detach(),) + torch.autograd.grad(y, (qq, kk, vv), g))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert all(bool(t.isfinite().all()) for t in results[1])


@gpu
def test_lengths_outside_the_keys_are_clamped():
    from imagefolder_amd import nn_ops
    q, k, v = (torch.randn(4, n, 2, 32, device="cuda").to(BF) for n in (7, 90, 90))
    for dt in (torch.int32, torch.int64):
        a = nn_ops.cross_attention(q, k, v, kv_lens=torch.tensor([-3, 91, 2 ** 31 - 1, 90], device="cuda", dtype=dt))
        b = nn_ops.cross_attention(q, k, v, kv_lens=torch.tensor([0, 90, 90, 90], device="cuda", dtype=dt))
        assert torch.equal(a, b) and float(a[0].abs().sum()) == 0


@gpu
def test_without_keys_queries_or_samples():
    from imagefolder_amd import nn_ops
    for B, Nq, Nk in ((0, 3, 4), (2, 0, 5), (2, 3, 0), (2, 0, 0)):
        q, k, v = (torch.randn(B, n, 4, 64, device="cuda").to(BF).requires_grad_(True) for n in (Nq, Nk, Nk))
        y = nn_ops.cross_attention(q, k, v)
        assert y.shape == q.shape and float(y.abs().sum()) == 0
        for t, d in zip((q, k, v), torch.autograd.grad(y, (q, k, v), torch.ones_like(y))):
            assert d.shape == t.shape and float(d.abs().sum()) == 0


@gpu
@pytest.mark.parametrize("Nq", [1, 150])
def test_extreme_scores(Nq):
    """one key far ahead of the others, scores whose exponentials leave fp32, equal scores"""
    torch.manual_seed(Nq)
    B, Nk, H, D = 2, 500, 2, 64
    k, v = torch.randn(B, Nk, H, D, device="cuda").to(BF), torch.randn(B, Nk, H, D, device="cuda").to(BF)
    q = torch.randn(B, Nq, H, D, device="cuda").to(BF)
    g = torch.randn(B, Nq, H, D, device="cuda").to(BF)
    from imagefolder_amd import nn_ops
    # scores of the order of 1e4: e of the bounds is then a few percent, which they take into account
    both(q * 16, k * 16, v, scale=4.0, g=g)
    # ascending and descending keys: the running maximum moves at every tile, or never
    ramp = torch.arange(Nk, device="cuda")[None, :, None, None] / 16
    for sign in (1, -1):
        kk = torch.zeros(B, Nk, H, D, device="cuda")
        kk[..., :1] = sign * ramp
        qq = torch.ones(B, Nq, H, D, device="cuda").to(BF)
        both(qq, kk.to(BF), v, scale=1.0, g=g)
    # zero queries: the mean of the values, and no gradient for the keys through equal scores
    y = nn_ops.cross_attention(torch.zeros_like(q), k, v)
    want = v.double().mean(1)[:, None].expand(B, Nq, H, D)
    within("mean", y, want, 2 * HALF * v.double().abs().mean(1)[:, None].expand_as(want) + HALF * want.abs())
    # infinite scores: as the softmax of the definition (nan where inf meets inf), and -inf is a key that is not there
    kk = k.clone()
    kk[:, 7] = 0
    kk[:, 7, :, 0] = float("-inf")
    qq = q.abs() + 1
    y = nn_ops.cross_attention(qq, kk, v)
    drop = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
    drop[:, 7] = False
    assert torch.equal(y, nn_ops.cross_attention(qq, k, v, key_mask=drop))
    assert bool(nn_ops.cross_attention(qq, -kk, v).isnan().any())


@gpu
@pytest.mark.parametrize("Nk,D", [(50, 64), (50, 128), (400, 64), (400, 128)])
def test_the_smallest_scale(Nk, D):
    """scores that are all but equal: the mean of the values; lse / scale, where the backward's products begin, is log(Nk) 2^64 then.  An accumulator that begins
    there loses q k^T beside it, which is 2^-50 of it: P = exp(0) / Nk up to 2^-22, and the gradients are those of the oracle"""
    torch.manual_seed(Nk + D)
    q, k, v, g = (torch.randn(2, n, 2, D, device="cuda").to(BF) for n in (70, Nk, Nk, 70))
    both(q, k, v, scale=2.0 ** -64, g=g)


@gpu
def test_strides_alignment_and_broadcasts():
    from imagefolder_amd import nn_ops
    torch.manual_seed(0)
    B, Nq, Nk, H, D = 3, 70, 150, 4, 64
    packed = torch.randn(B, Nk, 2, H, D, device="cuda").to(BF)
    head_major = torch.randn(B, H, Nq, D, device="cuda").to(BF)
    both(head_major.transpose(1, 2), packed[:, :, 0], packed[:, :, 1])
    # one set of keys for every sample, one head's values for every head
    both(head_major.transpose(1, 2), packed[:1, :, 0].expand(B, Nk, H, D), packed[:, :, 1, :1].expand(B, Nk, H, D))
    # rows that do not begin at 16 bytes, elements that do not lie side by side, every other token
    odd = torch.randn(B * Nq * H * D + 1, device="cuda").to(BF)[1:].view(B, Nq, H, D)
    both(odd, packed[:, :, 0], packed[:, :, 1])
    both(torch.randn(B, Nq, D, H, device="cuda").to(BF).transpose(2, 3), torch.randn(B, 2 * Nk, H, D + 4, device="cuda").to(BF)[:, ::2, :, :D], packed[:, :, 1])
    # gradients that arrive expanded or transposed
    q, k, v = (t.detach().requires_grad_(True) for t in (head_major.transpose(1, 2), packed[:, :, 0], packed[:, :, 1]))
    y = nn_ops.cross_attention(q, k, v)
    a = torch.autograd.grad(y.sum(), (q, k, v), retain_graph=True)
    b = torch.autograd.grad(y, (q, k, v), torch.ones_like(y), retain_graph=True)
    c = torch.autograd.grad(y.transpose(1, 2), (q, k, v), torch.ones(B, H, Nq, D, device="cuda").to(BF))
    assert all(torch.equal(x, y_) and torch.equal(x, z) for x, y_, z in zip(a, b, c))


@gpu
def test_same_bits_from_run_to_run():
    from imagefolder_amd import nn_ops
    for B, Nq, Nk, H, Hk, D in ((2, 300, 700, 8, 2, 64), (1, 2, 6000, 8, 8, 128), (3, 900, 257, 4, 4, 64), (2, 700, 90, 16, 4, 96)):
        q, k, v, g = (torch.randn(B, n, h, D, device="cuda").to(BF).requires_grad_(True) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
        runs = []
        for _ in range(3):
            y = nn_ops.cross_attention(q, k, v)
            runs.append((y.detach(),) + torch.autograd.grad(y, (q, k, v), g.detach()))
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@gpu
def test_gradients_against_differences():
    """inputs on a grid of 1/16 and steps of 1/8 along -1, 0, 1 are exact in bf16: what parts the kernels' differences from their gradient are the roundings of
    the two results (T_O) over the step, the gradient's own bound, and the third derivative, which the 64-bit oracle gives at the same points"""
    from imagefolder_amd import nn_ops
    torch.manual_seed(2)
    B, Nq, Nk, H, Hk, D, h = 2, 40, 90, 4, 2, 64, 0.125
    grid = lambda *s: (torch.randint(-24, 25, s, device="cuda") / 16).to(BF)  # noqa: E731
    x = [grid(B, Nq, H, D), grid(B, Nk, Hk, D), grid(B, Nk, Hk, D)]
    g = torch.randn(B, Nq, H, D, device="cuda").to(BF)
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(nn_ops.cross_attention(*leaves), leaves, g)
    want, tol = oracle(*x, g)
    for i in range(3):
        d = torch.randint(-1, 2, x[i].shape, device="cuda").to(BF)
        at = lambda s: [t + s * h * d if j == i else t for j, t in enumerate(x)]  # noqa: E731
        mine = sum(s * float((nn_ops.cross_attention(*at(s)).double() * g.double()).sum()) for s in (1, -1)) / (2 * h)
        exact, bounds = zip(*(oracle(*at(s)) for s in (1, -1)))
        true = sum(s * float((o * g.double()).sum()) for s, o in zip((1, -1), exact)) / (2 * h)
        slope = float((grads[i].double() * d.double()).sum())
        rounding = sum(float((t * g.double().abs()).sum()) for t in bounds) / (2 * h)
        third = abs(true - float((want[1 + i] * d.double()).sum()))
        assert abs(mine - slope) <= 1.05 * (rounding + float((tol[1 + i] * d.double().abs()).sum())) + third


@gpu
def test_oracle_gradients_against_differences():
    torch.manual_seed(3)
    x = [torch.randn(2, n, 2, 8, dtype=torch.float64, device="cuda") for n in (5, 9, 9)]
    g = torch.randn(2, 5, 2, 8, dtype=torch.float64, device="cuda")
    lens = torch.tensor([9, 4], device="cuda")
    want, _ = oracle(*x, g, lens)
    for i in range(3):
        d, h = torch.randn_like(x[i]), 1e-5
        f = [float((oracle(*[t + s * h * d if j == i else t for j, t in enumerate(x)], lens=lens)[0] * g).sum()) for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - float((want[1 + i] * d).sum())) <= 1e-7


@gpu
def test_past_32_bits_of_elements():
    """keys and values whose last ones lie behind 2^31 elements; only those are ahead of the rest"""
    from imagefolder_amd import nn_ops
    Nk, H, D = 2 ** 31 // (64 * 128) + 40, 64, 128
    k, v = torch.zeros(1, Nk, H, D, dtype=BF, device="cuda"), torch.zeros(1, Nk, H, D, dtype=BF, device="cuda")
    q = torch.ones(1, 1, H, D, dtype=BF, device="cuda")
    k[0, -3:] = 4.0
    v[0, -3:] = torch.randn(3, H, D, device="cuda").to(BF)
    y = nn_ops.cross_attention(q, k, v)
    want = v[0, -3:].double().mean(0)[None, None]          # (the others' weight: 2.6e5 exp(-45))
    within("O", y, want, 2 * HALF * v[0, -3:].double().abs().mean(0)[None, None] + HALF * want.abs())
    y = nn_ops.cross_attention(q.expand(1, 40, H, D), k, v)
    within("O", y, want.expand(1, 40, H, D), (2 * HALF * v[0, -3:].double().abs().mean(0)[None, None] + HALF * want.abs()).expand(1, 40, H, D))


@gpu
@pytest.mark.parametrize("Nq,Nk", [(60, 130), (1, 3000)])
def test_in_graphs_and_on_another_stream(Nq, Nk):
    from imagefolder_amd import nn_ops
    B, H, Hk, D = 2, 8, 2, 64
    q, k, v = (torch.randn(B, n, h, D, device="cuda").to(BF).requires_grad_(True) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk)))
    g = torch.randn(B, Nq, H, D, device="cuda").to(BF)
    lens = torch.tensor([Nk, Nk // 2], device="cuda")

    def step():
        y = nn_ops.cross_attention(q, k, v, kv_lens=lens)
        return (y.detach(),) + torch.autograd.grad(y, (q, k, v), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, step()))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:                   # two graphs, each with workspaces of its own
        with torch.cuda.graph(graph):
            outs.append(step())
    for n in range(4):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            k.mul_(-1)
            lens[0] = Nk - 17 * n
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@gpu
def test_two_streams_at_once():
    from imagefolder_amd import nn_ops
    sizes = ((4, 300, 500, 8, 2, 64), (2, 900, 100, 8, 8, 128), (3, 64, 257, 12, 12, 64), (2, 1, 5000, 16, 4, 128))
    for size in sizes:
        B, Nq, Nk, H, Hk, D = size
        jobs = [tuple(torch.randn(B, n, h, D, device="cuda").to(BF).requires_grad_(True) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk))) for _ in range(2)]
        g = torch.randn(B, Nq, H, D, device="cuda").to(BF)

        def step(job):
            y = nn_ops.cross_attention(*job)
            return (y.detach(),) + torch.autograd.grad(y, job, g)

        want = [step(j) for j in jobs]
        streams = [torch.cuda.Stream() for _ in jobs]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(4):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(step(jobs[i]))
        torch.cuda.synchronize()
        for w, runs in zip(want, got):
            assert all(torch.equal(a, b) for r in runs for a, b in zip(w, r))


@gpu
def test_some_of_the_gradients_and_views_of_lengths_and_masks():
    from imagefolder_amd import nn_ops
    torch.manual_seed(9)
    B, Nq, Nk, H, D = 3, 40, 90, 2, 64
    q, k, v, g = (torch.randn(B, n, H, D, device="cuda").to(BF) for n in (Nq, Nk, Nk, Nq))
    lens = torch.tensor([90, 5, 7, 5, 33, 5], device="cuda", dtype=torch.int32)[::2]
    mask = (torch.rand(1, Nk, device="cuda") < 0.7).expand(B, Nk)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(nn_ops.cross_attention(*leaves, kv_lens=lens.contiguous(), key_mask=mask.contiguous()), leaves, g)
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        (d,) = torch.autograd.grad(nn_ops.cross_attention(*args, kv_lens=lens, key_mask=mask), (args[i],), g)
        assert torch.equal(d, want[i])
    one = q.clone().requires_grad_(True)            # one tensor in all three places: its gradients add up
    y = nn_ops.cross_attention(one, one, one)
    parts = [t.clone().requires_grad_(True) for t in (q, q, q)]
    z = nn_ops.cross_attention(*parts)
    (d,) = torch.autograd.grad(y, (one,), g)
    a, b, c = (t.double() for t in torch.autograd.grad(z, parts, g))
    # two additions in bf16, in whatever order: each rounds at most half a step of a sum that is at most the sum of the parts' sizes
    assert torch.equal(y, z) and bool(((d.double() - (a + b + c)).abs() <= 2.05 * HALF * (a.abs() + b.abs() + c.abs())).all())


@gpu
@pytest.mark.parametrize("Nq", [1, 33])
def test_more_samples_than_a_grid_dimension_of_16_bits(Nq):
    B, Nk, D = 70001, 3, 8
    gen = torch.Generator(device="cuda").manual_seed(Nq)
    q, k, v, g = (torch.randn(B, n, 1, D, generator=gen, device="cuda").to(BF).requires_grad_(True) for n in (Nq, Nk, Nk, Nq))
    from imagefolder_amd import nn_ops
    y = nn_ops.cross_attention(q, k, v)
    grads = torch.autograd.grad(y, (q, k, v), g.detach())
    for b in (0, 1, 65535, 65536, 70000):
        part = [t.detach()[b:b + 1] for t in (q, k, v, g)]
        want, tol = oracle(*part)
        for name, a, w, t in zip(("O", "dq", "dk", "dv"), (y.detach(),) + grads, want, tol):
            within(name, a[b:b + 1], w, t)


@gpu
@pytest.mark.parametrize("N,H,D", [(257, 3, 32), (130, 2, 128), (65, 4, 96), (50, 2, 8)])
def test_packed_self_attention_of_other_head_widths(N, H, D):
    """nn_ops.attention_qkvpacked and its twin of the fused blocks take head widths other than 64 through these kernels"""
    from imagefolder_amd import nn_ops, ops_dense
    torch.manual_seed(D)
    qkv = torch.randn(2, N, 3 * H * D, device="cuda").to(BF).requires_grad_(True)
    g = torch.randn(2, N, H * D, device="cuda").to(BF)
    for entry in (nn_ops.attention_qkvpacked, ops_dense.attention_qkvpacked):
        y = entry(qkv, H)
        assert nn_ops.IMPL["attention"] == "hip (xq_xattn_forward / xq_xattn_backward)"
        (dx,) = torch.autograd.grad(y, (qkv,), g)
        q, k, v = qkv.detach().view(2, N, 3, H, D).unbind(2)
        want, tol = oracle(q, k, v, g.view(2, N, H, D))
        within("O", y.detach().view(2, N, H, D), want[0], tol[0])
        for i, part in enumerate(dx.view(2, N, 3, H, D).unbind(2)):
            within("qkv"[i], part, want[1 + i], tol[1 + i])


@gpu
def test_packed_self_attention_of_an_empty_batch():
    from imagefolder_amd import nn_ops
    for B, N in ((0, 5), (2, 0)):
        qkv = torch.zeros(B, N, 3 * 2 * 32, device="cuda", dtype=BF, requires_grad=True)
        y = nn_ops.attention_qkvpacked(qkv, 2)
        assert y.shape == (B, N, 64)
        (dx,) = torch.autograd.grad(y, (qkv,), torch.zeros_like(y))
        assert dx.shape == qkv.shape


@gpu
def test_autocast_casts_fp32():
    from imagefolder_amd import nn_ops
    from imagefolder_amd._lib import XqError
    q, k, v = (torch.randn(2, n, 4, 64, device="cuda", requires_grad=True) for n in (30, 50, 50))
    with torch.autocast("cuda", torch.bfloat16):
        y = nn_ops.cross_attention(q, k, v)
    assert y.dtype == BF and torch.equal(y, nn_ops.cross_attention(q.to(BF), k.to(BF), v.to(BF)))
    y.float().sum().backward()
    assert all(t.grad.dtype == torch.float32 and bool(t.grad.isfinite().all()) for t in (q, k, v))
    with pytest.raises(XqError, match="bf16"):
        nn_ops.cross_attention(q, k, v)


@gpu
def test_a_decoder_layer_of_the_three_operators():
    """codes -> embedding -> dropout -> attention to an encoder's states -> dropout + residual, forward and backward, against the same chain in float64 with
    the kernels' masks.  Bounds on norms: the chain rounds to bf16 in six places on the way (embedding, dropout, P, O; dS, dq, dO on the way back), each at most
    2^-8 of what it rounds: 8 * 2^-8 covers them."""
    from imagefolder_amd import nn_ops
    torch.manual_seed(11)
    B, N, M, H, D, V = 4, 60, 45, 4, 64, 500
    W = H * D
    table = (torch.randn(V, W, device="cuda") / 8).requires_grad_(True)
    states = torch.randn(B, M, 2, H, D, device="cuda").to(BF).requires_grad_(True)
    codes = torch.randint(0, V, (B, N), device="cuda")
    lens = torch.tensor([45, 1, 0, 30], device="cuda")
    keys = [torch.tensor([9, i], device="cuda") for i in range(2)]
    e = nn_ops.embedding(codes, table, scale=W ** 0.5 / 2, padding_idx=0, dtype=BF)
    x = nn_ops.dropout(e, 0.1, key=keys[0])
    o = nn_ops.cross_attention(x.view(B, N, H, D), states[:, :, 0], states[:, :, 1], kv_lens=lens)
    y = nn_ops.dropout(o.reshape(B, N, W), 0.2, key=keys[1], residual=x.float())
    g = torch.randn(B, N, W, device="cuda")
    grads = torch.autograd.grad(y, (table, states), g)
    assert [nn_ops.IMPL[n] for n in ("embedding", "dropout", "cross_attention")] == ["hip"] * 3
    f1, f2 = (nn_ops.dropout(torch.ones(B, N, W, device="cuda"), p, key=k).double() for p, k in ((0.1, keys[0]), (0.2, keys[1])))
    t64, s64 = table.detach().double().requires_grad_(True), states.detach().double().requires_grad_(True)
    x64 = torch.where((codes == 0)[..., None], t64.detach()[codes], t64[codes]) * (W ** 0.5 / 2) * f1
    q64 = x64.view(B, N, H, D).transpose(1, 2)
    k64, v64 = s64[:, :, 0].transpose(1, 2), s64[:, :, 1].transpose(1, 2)
    ok = (torch.arange(M, device="cuda")[None] < lens[:, None])[:, None, None]
    s = (q64 @ k64.transpose(2, 3) * D ** -0.5).masked_fill(~ok, -1e300)
    o64 = ((torch.softmax(s, -1) * ok) @ v64).transpose(1, 2).reshape(B, N, W)
    y64 = x64 + o64 * f2
    want = torch.autograd.grad(y64, (t64, s64), g.double())
    for a, b in ((y.detach(), y64.detach()), (grads[0], want[0]), (grads[1], want[1])):
        assert float((a.double() - b).norm()) <= 8 * HALF * float(b.norm())
    assert float(grads[0][0].abs().sum()) == 0 and float(grads[1][2].abs().sum()) == 0


# ---- refusals and the CPU ------------------------------------------------------------------------------------------------------------------

def test_refusals():
    import ctypes
    from imagefolder_amd import _lib, nn_ops, ops_seq
    from imagefolder_amd._lib import XqError
    t = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)  # noqa: E731
    good = dict(q=t(2, 3, 4, 16), k=t(2, 5, 2, 16), v=t(2, 5, 2, 16))
    for kw, what in ((dict(q=t(3, 4, 16)), "heads, head dim"), (dict(k=t(2, 6, 2, 16)), "go together"), (dict(k=t(1, 5, 2, 16), v=t(1, 5, 2, 16)), "go together"),
                     (dict(q=t(2, 3, 4, 8)), "go together"), (dict(q=t(2, 3, 5, 16)), "evenly"), (dict(k=t(2, 5, 0, 16), v=t(2, 5, 0, 16)), "evenly"),
                     (dict(kv_lens=torch.zeros(3, dtype=torch.int32)), "kv_lens"), (dict(kv_lens=torch.zeros(2)), "kv_lens"),
                     (dict(key_mask=torch.zeros(2, 5)), "key_mask"), (dict(key_mask=torch.zeros(2, 4, dtype=torch.bool)), "key_mask"), (dict(scale=0.0), "scale"),
                     (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=2.0 ** -65), "scale"), (dict(scale=2.0 ** 65), "scale"),
                     (dict(q=t(2, 3, 4, 16, dt=torch.float32)), "bf16"), (dict(v=t(2, 5, 2, 16, dt=torch.float16)), "bf16"),
                     (dict(kv_lens=torch.zeros(2, dtype=torch.int32, device="meta")), "one device")):
        with pytest.raises(XqError, match=what):
            ops_seq.cross_attention(**{**good, **kw})
    # a scale held in a tensor is read at every call
    t = torch.tensor(0.5)
    assert ops_seq.check_cross_attention(**good, kv_lens=None, key_mask=None, scale=t) == 0.5
    t.fill_(0.25)
    assert ops_seq.check_cross_attention(**good, kv_lens=None, key_mask=None, scale=t) == 0.25
    t = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)  # noqa: E731
    for D in (12, 136, 0):
        with pytest.raises(XqError, match="head dim"):
            ops_seq.cross_attention(t(2, 3, 4, D), t(2, 5, 2, D), t(2, 5, 2, D))
    with pytest.raises(XqError, match="evenly"):
        nn_ops.cross_attention(t(2, 3, 5, 16), good["k"], good["v"])
    l, one = _lib.lib(), ctypes.c_void_p(16)
    st = (ctypes.c_int64 * 9)(*[64] * 9)
    f = ctypes.c_float

    def fwd(q=one, k=one, v=one, B=2, Nq=3, Nk=5, H=4, Hk=2, D=16, strides=st, scale=0.25, out=one, ws=None, nbytes=0):
        return l.xq_xattn_forward(q, k, v, B, Nq, Nk, H, Hk, D, strides, None, 0, None, f(scale), out, None, ws, nbytes, None)

    def bwd(q=one, B=2, Nq=3, Nk=5, H=4, Hk=2, D=16, strides=st, gstrides=st, scale=0.25, out=one, lse=one, dq=one, ws=one, nbytes=1 << 20):
        return l.xq_xattn_backward(q, one, one, out, one, lse, B, Nq, Nk, H, Hk, D, strides, None, 0, None, f(scale), dq, one, one, gstrides, ws, nbytes, None)

    def err():
        return l.xq_last_error().decode()

    odd = (ctypes.c_int64 * 9)(*[64, 64, 64, 64, 60, 64, 64, 64, 64])
    for call in (fwd, bwd):
        assert call(H=5) == -1 and "evenly" in err()
        assert call(D=12) == -1 and "multiple of 8" in err()
        assert call(D=136) == -1 and call(B=-1) == -1 and call(Hk=0) == -1
        assert call(scale=0.0) == -1 and call(scale=float("nan")) == -1 and "scale" in err()
        assert call(scale=2.0 ** -65) == -1 and call(scale=2.0 ** 65) == -1 and "scale" in err()
        assert call(q=None) == -1 and "null" in err()
        assert call(q=ctypes.c_void_p(8)) == -1 and "q has to be" in err()
        assert call(strides=odd) == -1 and "k has to be" in err()
        assert call(out=ctypes.c_void_p(24)) == -1 and "16-byte" in err()
        assert call(Nq=2 ** 30, B=4) == -1 and "too many" in err()
        assert call(B=0, q=None, strides=None) == 0
    assert bwd(gstrides=odd) == -1 and "dk has to be" in err()
    for i, name in enumerate(("dq", "dq", "dq", "dk", "dk", "dk", "dv", "dv", "dv")):
        wide = (ctypes.c_int64 * 9)(*[0 if j == i else 64 for j in range(9)])
        assert bwd(gstrides=wide) == -1 and f"{name} has a stride of 0" in err()
    assert bwd(lse=None) == -1 and bwd(dq=None) == -1
    need = l.xq_xattn_backward_workspace_bytes(2, 3, 400, 4, 2, 16)
    assert need >= 2 * 3 * 4 * 4 and bwd(Nk=400, nbytes=need - 1) == -2 and "too small" in err()
    need = l.xq_xattn_backward_workspace_bytes(2, 900, 5, 4, 2, 16)          # the rows split over blocks
    assert need >= 2 * 2 * 2 * 2 * 5 * 16 * 4 and bwd(Nq=900, nbytes=need - 1) == -2 and "too small" in err()
    assert l.xq_xattn_backward_workspace_bytes(2, 3, 5, 4, 2, 16) == 0
    need = l.xq_xattn_forward_workspace_bytes(1, 1, 8192, 8, 8, 128)
    assert need > 0 and fwd(B=1, Nq=1, Nk=8192, H=8, Hk=8, D=128, ws=one, nbytes=need - 1) == -2
    assert l.xq_xattn_forward_workspace_bytes(64, 256, 257, 12, 12, 64) == 0
    assert l.xq_xattn_forward_workspace_bytes(1, 1, 8192, 8, 3, 128) == 0 and l.xq_xattn_backward_workspace_bytes(1, 1, 1, 1, 1, 9) == 0


def test_on_the_cpu_it_is_the_definition():
    from imagefolder_amd import nn_ops
    torch.manual_seed(1)
    q, k, v = (torch.randn(3, n, h, 16, requires_grad=True) for n, h in ((4, 6), (9, 2), (9, 2)))
    lens, mask = torch.tensor([9, 0, 4]), torch.rand(3, 9) < 0.7
    y = nn_ops.cross_attention(q, k, v, kv_lens=lens, key_mask=mask)
    g = torch.randn_like(y)
    grads = torch.autograd.grad(y, (q, k, v), g)
    want, _ = oracle(q.detach(), k.detach(), v.detach(), g, lens, mask)
    for a, b in zip((y.detach(),) + grads, want):
        assert float((a.double() - b).abs().max()) <= 1e-5
    assert float(nn_ops.cross_attention(q, k[:, :0], v[:, :0]).abs().sum()) == 0

"""nn_ops.dropout and nn_ops.embedding: the kernels against plain 64-bit computations of the same definition, their refusals on the CPU.

Tolerances (none is fitted to a run): a result computed in fp32 and rounded once to type T is off by at most eps_T / 2 of its value plus the fp32 part: one
rounding of the factor and one of the product (fmaf: none more) for dropout, i.e. 2 * 2^-24 relative; for a gradient row of c summands at most
(c + 2) * 2^-24 * scale * sum |g| (c - 1 additions, the products with the scale, any order)."""
import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def philox(block, stream, seed):
    """Philox4x32-10 over an array of counter blocks -> (len, 4) uint32"""
    m = np.uint64(0xFFFFFFFF)
    block = np.asarray(block, dtype=np.uint64)
    c = [block & m, block >> np.uint64(32), np.full_like(block, stream & 0xFFFFFFFF), np.full_like(block, (stream >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & m, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1).astype(np.uint32)


def factors(first, n, p, key):
    """the factor of elements first .. first + n (first a multiple of 8) in 64 bits"""
    t = int(round(65536 * p))
    w = philox(np.arange(first // 8, first // 8 + (n + 7) // 8), int(key[1]), int(key[0]))
    u16 = np.stack((w & 0xFFFF, w >> 16), -1).reshape(-1)[:n]
    return np.where(u16 >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0, 0.0)


def test_generator_against_the_published_answers():
    # Random123's known answers for philox4x32-10: zeros, ones, digits of pi (counter 0x85a308d3_243f6a88 etc.)
    assert philox([0], 0, 0)[0].tolist() == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([2 ** 64 - 1], 2 ** 64 - 1, 2 ** 64 - 1)[0].tolist() == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x85A308D3243F6A88], 0x0370734413198A2E, 0x299F31D0A4093822)[0].tolist() == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def close(got, want, types=(), rel=2.0 ** -23):
    """want: float64; got within the roundings of its type"""
    want = torch.as_tensor(want, dtype=torch.float64, device=got.device)
    tol = want.abs() * (HALF[got.dtype] * (1 + 2.0 ** -8) + rel) + 1e-38
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (got[bad][:4], want[bad][:4])


def new_key(a, b):
    return torch.tensor([a, b], dtype=torch.int64, device="cuda")


@gpu
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 2047, 4099, 1000003])
@pytest.mark.parametrize("kind,res", [(BF, None), (F32, None), (BF, BF), (BF, F32), (F32, F32)])
def test_dropout_and_its_gradient(n, kind, res):
    from imagefolder_amd import nn_ops
    torch.manual_seed(n)
    key = new_key(-3 + n, 2 ** 40 + n)
    p = 0.3 if n % 2 else 0.81
    x = torch.randn(n, device="cuda").to(kind).requires_grad_(True)
    r = None if res is None else torch.randn(n, device="cuda").to(res).requires_grad_(True)
    f = torch.from_numpy(factors(0, n, p, key.tolist())).cuda()
    y = nn_ops.dropout(x, p, key=key, residual=r)
    assert y.dtype == (res or kind) and nn_ops.IMPL["dropout"] == "hip"
    if r is None:
        close(y.detach(), x.detach().double() * f)
        assert bool((y.detach()[f == 0] == 0).all())
    else:
        want = x.detach().double() * f + r.detach().double()
        # the sum: its own rounding, and the factor's on the product
        tol = want.abs() * HALF[y.dtype] * (1 + 2.0 ** -7) + (x.detach().double() * f).abs() * 2.0 ** -23 + 1e-38
        assert bool(((y.detach().double() - want).abs() <= tol).all())
    g = torch.randn(n, device="cuda").to(y.dtype)
    grads = torch.autograd.grad(y, [x] if r is None else [x, r], g)
    assert grads[0].dtype == kind
    close(grads[0], g.double() * f)
    if r is not None:
        assert torch.equal(grads[1], g)


@gpu
@pytest.mark.parametrize("p", [2.0 ** -17 - 1e-9, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1.0])
def test_dropout_at_the_ends_of_p(p):
    from imagefolder_amd import nn_ops
    n = 100000
    x = torch.randn(n, device="cuda")
    key = new_key(5, 6)
    f = factors(0, n, p, (5, 6))
    close(nn_ops.dropout(x, p, key=key), x.double() * torch.from_numpy(f).cuda())
    if p == 1.0:
        assert not f.any()
    if p < 2.0 ** -17:
        assert (f == 1).all()


@gpu
def test_dropout_drops_infinities_and_nan():
    from imagefolder_amd import nn_ops
    n = 4096
    f = torch.from_numpy(factors(0, n, 0.5, (1, 2))).cuda()
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.where(f == 0, torch.full((n,), bad, device="cuda"), torch.ones(n, device="cuda"))
        y = nn_ops.dropout(x, 0.5, key=new_key(1, 2))
        assert bool((y == torch.where(f == 0, 0.0, 2.0)).all())
        r = torch.ones(n, device="cuda")
        assert bool((nn_ops.dropout(x, 0.5, key=new_key(1, 2), residual=r) == torch.where(f == 0, 1.0, 3.0)).all())


@gpu
@pytest.mark.parametrize("kind", [BF, F32])
def test_dropout_of_other_memory_orders(kind):
    """the mask goes by an element's place in memory; the result lies as a dense x does"""
    from imagefolder_amd import nn_ops
    key, p = new_key(11, 12), 0.4
    base = torch.randn(3, 10, 6, 7, device="cuda").to(kind)
    dense = [base, base.contiguous(memory_format=torch.channels_last), base.permute(2, 0, 3, 1), base.flatten()[1:], base.flatten()[1:].view(-1, 1).t(), base[:1, 2:3]]
    for x in dense:
        y = nn_ops.dropout(x, p, key=key)
        f = torch.from_numpy(factors(0, x.numel(), p, (11, 12))).cuda()
        in_memory = torch.as_strided(x, (x.numel(),), (1,), x.storage_offset())
        assert [s for s, n in zip(y.stride(), y.shape) if n > 1] == [s for s, n in zip(x.stride(), x.shape) if n > 1]
        close(torch.as_strided(y, (x.numel(),), (1,), y.storage_offset()), in_memory.double() * f)
    # with holes or overlaps: as its contiguous copy
    for x in (base[:, ::2], base.expand(2, *base.shape)[:, :, :, 1:], base[0, 0, 0, :1].expand(9)):
        assert torch.equal(nn_ops.dropout(x, p, key=key), nn_ops.dropout(x.contiguous(), p, key=key))
    # a residual and a gradient that lie in another order than x
    x = base.contiguous(memory_format=torch.channels_last).requires_grad_(True)
    r = torch.randn(3, 10, 6, 7, device="cuda")
    y = nn_ops.dropout(x, p, key=key, residual=r)
    f = nn_ops.dropout(torch.ones_like(x.detach(), dtype=F32), p, key=key)
    assert torch.allclose(y, r + x.detach().float() * f, rtol=0, atol=1e-6 * float(y.detach().abs().max()))
    g = torch.randn(3, 10, 6, 7, device="cuda")
    (dx,) = torch.autograd.grad(y, [x], g, retain_graph=True)
    close(dx, g.double() * f.double())
    (dx,) = torch.autograd.grad(y.sum(), [x])          # an expanded gradient
    close(dx, f.double())


@gpu
def test_dropout_gradient_against_differences():
    from imagefolder_amd import nn_ops
    n, key = 5000, new_key(3, 4)
    x, d, g = (torch.randn(n, device="cuda") for _ in range(3))
    xr = x.clone().requires_grad_(True)
    y = nn_ops.dropout(xr, 0.25, key=key)
    (dx,) = torch.autograd.grad(y, [xr], g)
    h = 2.0 ** -4
    diff = (nn_ops.dropout(x + h * d, 0.25, key=key).double() - nn_ops.dropout(x - h * d, 0.25, key=key).double()) / (2 * h)
    # the map is linear: what is left are the roundings of x + h d and of the two results (each 2^-24 of values below 8) over 2 h, against g
    assert abs(float((diff * g.double()).sum() - (dx.double() * d.double()).sum())) <= 4 * 8 * 2.0 ** -24 / (2 * h) * float(g.abs().sum())


@gpu
def test_dropout_keys():
    from imagefolder_amd import nn_ops
    x = torch.ones(100000, device="cuda")
    torch.manual_seed(7)
    a, b = nn_ops.dropout(x, 0.5), nn_ops.dropout(x, 0.5)
    torch.manual_seed(7)
    c = nn_ops.dropout(x, 0.5)
    assert torch.equal(a, c) and not torch.equal(a, b)
    # 100000 fair draws: 6 standard deviations of the mean factor
    assert abs(float(a.mean()) - 1.0) < 6 / 100000 ** 0.5
    assert torch.equal(nn_ops.dropout(x, 0.5, training=False), x) and torch.equal(nn_ops.dropout(x, 0.0, residual=x), 2 * x)
    # a key that changes between the passes is an error, not another mask
    key, xr = new_key(1, 1), x.clone().requires_grad_(True)
    y = nn_ops.dropout(xr, 0.5, key=key)
    key[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@gpu
def test_dropout_past_32_bits_of_elements():
    from imagefolder_amd import nn_ops
    n = 2 ** 32 + 19
    x = torch.ones(n, dtype=BF, device="cuda")
    y = nn_ops.dropout(x, 0.5, key=new_key(8, 9))
    for first in (0, 2 ** 31 - 8, 2 ** 32 - 8, 2 ** 32 + 16):
        m = min(64, n - first)
        assert np.array_equal(y[first:first + m].double().cpu().numpy(), factors(first, m, 0.5, (8, 9)))


@gpu
def test_dropout_in_a_graph_and_on_another_stream():
    from imagefolder_amd import nn_ops
    x = torch.randn(70001, device="cuda").requires_grad_(True)
    g = torch.randn(70001, device="cuda")
    key = new_key(21, 0)

    def step(k):
        y = nn_ops.dropout(x, 0.3, key=k)
        return (y,) + torch.autograd.grad(y, [x], g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step(key)]
        step(None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, step(key)))
    graph, fresh = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(key)
    with torch.cuda.graph(fresh):
        drawn = step(None)
    seen = []
    for k in range(4):
        key[1] = k
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(key)))
        fresh.replay()
        torch.cuda.synchronize()
        y, dx = (t.detach().clone() for t in drawn)
        assert torch.equal(y == 0, dx == 0)
        seen.append(y)
    assert not any(torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])


# ---- embedding -----------------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("D", [1, 3, 8, 12, 100, 768, 1032])
@pytest.mark.parametrize("wt,yt", [(F32, F32), (F32, BF), (BF, BF), (BF, F32)])
def test_embedding_rows(D, wt, yt):
    from imagefolder_amd import nn_ops
    torch.manual_seed(D)
    V = 301
    w = torch.randn(V, D, device="cuda").to(wt)
    for shape, it in (((1,), torch.int64), ((5, 7), torch.int32), ((2, 3, 401), torch.int64), ((0,), torch.int64)):
        idx = torch.randint(0, V, shape, device="cuda").to(it)
        y = nn_ops.embedding(idx, w, scale=1.7, dtype=yt)
        assert y.shape == (*shape, D) and y.dtype == yt
        close(y, w.double()[idx.long()] * float(np.float32(1.7)))
    assert torch.equal(nn_ops.embedding(idx, w), w[idx.long()])


@gpu
def test_embedding_of_strange_indices_and_views():
    from imagefolder_amd import nn_ops
    w = torch.randn(50, 24, device="cuda")
    idx = torch.tensor([3, -1, 49, 50, -2 ** 40, 2 ** 40, 0], device="cuda")
    y = nn_ops.embedding(idx, w)
    ok = (idx >= 0) & (idx < 50)
    assert torch.equal(y[ok], w[idx[ok]]) and bool(y[~ok].isnan().all())
    # strided indices, a table that is a view (columns of a wider one: copied; rows from an odd offset: unaligned)
    wide = torch.randn(51, 48, device="cuda")
    i2 = torch.randint(0, 50, (6, 10), device="cuda")
    assert torch.equal(nn_ops.embedding(i2.t()[::2], wide[:50, :24]), wide[:50, :24][i2.t()[::2]])
    odd = torch.randn(50 * 24 + 1, device="cuda")[1:].view(50, 24)
    assert torch.equal(nn_ops.embedding(i2, odd), odd[i2])


def indices(kind, N, V, gen):
    if kind == "same":
        return torch.full((N,), V - 1, device="cuda")
    if kind == "skewed":                                # one row takes half of them, a few the next quarter
        i = torch.randint(0, V, (N,), generator=gen, device="cuda")
        u = torch.rand(N, generator=gen, device="cuda")
        return torch.where(u < 0.5, torch.full_like(i, V // 3), torch.where(u < 0.75, i % min(V, 5), i))
    i = torch.randint(0, V, (N,), generator=gen, device="cuda")
    return i.sort().values if kind == "sorted" else i


def check_gradient(idx, g, V, scale, dw, skip=None):
    N, D = g.reshape(-1, g.shape[-1]).shape
    i, g64 = idx.reshape(-1).long(), g.reshape(N, D).double()
    ok = (i >= 0) & (i < V)
    if skip is not None:
        ok &= i != skip
    i, g64 = i[ok], g64[ok]
    # on the host: 64-bit sums of runs of the sorted tokens
    order = np.argsort(i.cpu().numpy(), kind="stable")
    rows, first = np.unique(i.cpu().numpy()[order], return_index=True)
    want, size = np.zeros((V, D)), np.zeros((V, D))
    if len(rows):
        sorted64 = g64.cpu().numpy()[order]
        want[rows], size[rows] = np.add.reduceat(sorted64, first), np.add.reduceat(np.abs(sorted64), first)
    want, size = torch.from_numpy(want * scale).cuda(), torch.from_numpy(size * abs(scale)).cuda()
    count = torch.bincount(i, minlength=V).double()[:, None]
    tol = (count + 2) * 2.0 ** -24 * size + want.abs() * HALF[dw.dtype] * (1 + 2.0 ** -7) + 1e-38
    off = (dw.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert bool((dw[count[:, 0] == 0] == 0).all())


@gpu
@pytest.mark.parametrize("kind", ["uniform", "sorted", "skewed", "same"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 8), (3, 2, 5), (513, 2, 768), (2048, 256, 16), (2049, 257, 33), (5000, 1000, 100), (33000, 8192, 64), (70001, 65537, 8),
                                   (300, 2 ** 20, 4), (4097, 40000, 1)])
def test_embedding_gradient(kind, N, V, D):
    from imagefolder_amd import nn_ops
    gen = torch.Generator(device="cuda").manual_seed(N + V)
    idx = indices(kind, N, V, gen)
    w = torch.randn(V, D, generator=gen, device="cuda").requires_grad_(True)
    y = nn_ops.embedding(idx, w, scale=0.5)
    g = torch.randn(N, D, generator=gen, device="cuda")
    (dw,) = torch.autograd.grad(y, [w], g, retain_graph=True)
    check_gradient(idx, g, V, 0.5, dw)
    (again,) = torch.autograd.grad(y, [w], g)
    assert torch.equal(dw, again)


@gpu
@pytest.mark.parametrize("wt,yt", [(F32, F32), (F32, BF), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("D", [7, 64, 200])
def test_embedding_gradient_types_padding_and_strange_indices(wt, yt, D):
    from imagefolder_amd import nn_ops
    gen = torch.Generator(device="cuda").manual_seed(D)
    V, N = 700, 9000
    for it in (torch.int64, torch.int32):
        idx = indices("skewed", N, V, gen).to(it).view(90, 100)
        idx[0, :5] = torch.tensor([-1, 700, -2 ** 31, 2 ** 31 - 1, 701], device="cuda").to(it)
        w = torch.randn(V, D, generator=gen, device="cuda").to(wt).requires_grad_(True)
        for pad in (None, V // 3, -1):
            y = nn_ops.embedding(idx, w, scale=2.0, padding_idx=pad, dtype=yt)
            g = torch.randn(90, 100, D, generator=gen, device="cuda").to(yt)
            (dw,) = torch.autograd.grad(y, [w], g)
            assert dw.dtype == wt
            check_gradient(idx, g, V, 2.0, dw, skip=None if pad is None else pad % V)
    # a gradient that is a view, and an expanded one
    y = nn_ops.embedding(idx[1:], w, dtype=yt)
    wide = torch.randn(89, 100, 2 * D, generator=gen, device="cuda").to(yt)
    (dw,) = torch.autograd.grad(y, [w], wide[..., ::2], retain_graph=True)
    check_gradient(idx[1:], wide[..., ::2], V, 1.0, dw)
    (dw,) = torch.autograd.grad(y.sum(), [w])
    check_gradient(idx[1:], torch.ones_like(y.detach()), V, 1.0, dw)


@gpu
def test_embedding_gradient_of_many_tokens_and_of_none():
    from imagefolder_amd import nn_ops
    gen = torch.Generator(device="cuda").manual_seed(1)
    for kind, V in (("uniform", 30000), ("same", 3), ("skewed", 2 ** 18)):
        N, D = 1200001, 8                               # more than one tile of tokens to a slice
        idx = indices(kind, N, V, gen)
        w = torch.zeros(V, D, device="cuda", requires_grad=True)
        g = torch.randn(N, D, generator=gen, device="cuda")
        (dw,) = torch.autograd.grad(nn_ops.embedding(idx, w), [w], g)
        check_gradient(idx, g, V, 1.0, dw)
    w = torch.randn(9, 5, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(nn_ops.embedding(torch.zeros(0, 4, dtype=torch.int64, device="cuda"), w), [w], torch.zeros(0, 4, 5, device="cuda"))
    assert torch.equal(dw, torch.zeros(9, 5, device="cuda"))


@gpu
def test_embedding_gradient_against_differences():
    from imagefolder_amd import nn_ops
    idx = torch.randint(0, 40, (300,), device="cuda")
    w, d = torch.randn(40, 16, device="cuda"), torch.randn(40, 16, device="cuda")
    g = torch.randn(300, 16, device="cuda")
    wr = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(nn_ops.embedding(idx, wr, scale=3.0), [wr], g)
    h = 2.0 ** -4
    diff = (nn_ops.embedding(idx, w + h * d, scale=3.0).double() - nn_ops.embedding(idx, w - h * d, scale=3.0).double()) / (2 * h)
    # linear in w: roundings of w + h d and of the products (values below 32), over 2 h, against g
    assert abs(float((diff * g.double()).sum() - (dw.double() * d.double()).sum())) <= 4 * 32 * 2.0 ** -24 / (2 * h) * float(g.abs().sum())


@gpu
def test_embedding_past_32_bits_of_elements():
    from imagefolder_amd import nn_ops
    V, D = 2 ** 20, 2056                               # 2^31.006 elements in the table and in its gradient
    w = torch.zeros(V, D, dtype=BF, device="cuda")
    w[-1] = 3.0
    w.requires_grad_(True)
    idx = torch.tensor([V - 1, 0, V - 1], device="cuda")
    y = nn_ops.embedding(idx, w)
    assert bool((y.detach()[0] == 3).all()) and bool((y.detach()[1] == 0).all())
    (dw,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert bool((dw[-1] == 2).all()) and bool((dw[0] == 1).all()) and float(dw[1:-1].abs().max()) == 0.0


@gpu
def test_embedding_in_a_graph_and_on_another_stream():
    from imagefolder_amd import nn_ops
    V, N, D = 3000, 20000, 48
    w = torch.randn(V, D, device="cuda", requires_grad=True)
    idx = torch.randint(0, V, (N,), device="cuda")
    g = torch.randn(N, D, device="cuda")

    def step():
        y = nn_ops.embedding(idx, w, scale=2.0)
        return (y,) + torch.autograd.grad(y, [w], g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        idx.copy_(torch.randint(0, V, (N,), device="cuda") if k % 2 else torch.full((N,), k, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


# ---- refusals and the CPU ------------------------------------------------------------------------------------------------------------------

def test_refusals():
    from imagefolder_amd import _lib, nn_ops, ops_seq
    from imagefolder_amd._lib import XqError
    x = torch.zeros(8)
    for kw, what in (({"x": x.half()}, "type"), ({"p": 1.5}, r"\[0, 1\]"), ({"p": float("nan")}, r"\[0, 1\]"), ({"residual": torch.zeros(4)}, "shape"),
                     ({"residual": x.bfloat16()}, "residual of type"), ({"key": torch.zeros(2)}, "int64"), ({"key": torch.zeros(3, dtype=torch.int64)}, "two values"),
                     ({"key": torch.zeros(2, dtype=torch.int64, device="meta")}, "one device")):
        with pytest.raises(XqError, match=what):
            ops_seq.dropout(**{"x": x, "p": 0.5, "key": torch.zeros(2, dtype=torch.int64), **kw})
    with pytest.raises(XqError, match="MI355X"):
        nn_ops.dropout(x, 0.5, key=torch.zeros(2, dtype=torch.int64))
    w, idx = torch.zeros(4, 6), torch.zeros(3, dtype=torch.int64)
    for kw, what in (({"weight": torch.zeros(4)}, "rows, width"), ({"weight": torch.zeros(0, 4)}, "rows, width"), ({"weight": w.half()}, "bf16 / fp32"),
                     ({"dtype": torch.float16}, "bf16 / fp32"), ({"idx": idx.float()}, "int64 / int32"), ({"padding_idx": 4}, "padding_idx"),
                     ({"padding_idx": -5}, "padding_idx"), ({"idx": idx.to("meta")}, "one device")):
        with pytest.raises(XqError, match=what):
            ops_seq.embedding(**{"idx": idx, "weight": w, **kw})
    # the C entry points, before anything touches a device
    import ctypes
    l, one = _lib.lib(), ctypes.c_void_p(16)

    def err():
        return l.xq_last_error().decode()

    assert l.xq_dropout(one, 1, None, -1, 0.5, one, one, 1, None) == -1 and "negative" in err()
    assert l.xq_dropout(one, 1, None, 8, 1.01, one, one, 1, None) == -1 and "[0, 1]" in err()
    assert l.xq_dropout(one, 1, None, 8, float("nan"), one, one, 1, None) == -1
    assert l.xq_dropout(None, 1, None, 8, 0.5, one, one, 1, None) == -1 and "null" in err()
    assert l.xq_dropout(one, 1, None, 8, 0.5, None, one, 1, None) == -1 and "null" in err()
    assert l.xq_dropout(one, 1, None, 8, 0.5, ctypes.c_void_p(4), one, 1, None) == -1 and "aligned" in err()
    assert l.xq_dropout(None, 1, None, 0, 0.5, None, None, 1, None) == 0
    assert l.xq_embedding_forward(one, 1, one, 0, 4, 0, 8, 1.0, one, 0, None) == -1 and "V=0" in err()
    assert l.xq_embedding_forward(one, 1, one, 0, 4, 2 ** 20 + 1, 8, 1.0, one, 0, None) == -1 and "2^20" in err()
    assert l.xq_embedding_forward(one, 1, None, 0, 4, 8, 8, 1.0, one, 0, None) == -1 and "null" in err()
    assert l.xq_embedding_forward(None, 1, None, 0, 0, 8, 8, 1.0, None, 0, None) == 0
    need = l.xq_embedding_backward_workspace_bytes(1000, 64, 8)
    assert need >= 1000 * 12 and l.xq_embedding_backward_workspace_bytes(0, 64, 8) == 0 and l.xq_embedding_backward_workspace_bytes(5, 2 ** 21, 8) == 0
    assert l.xq_embedding_backward(one, 1, one, 0, 1000, 64, 8, 1.0, -1, one, 0, one, need - 1, None) == -2 and "too small" in err()
    assert l.xq_embedding_backward(one, 1, one, 0, 1000, 64, 8, 1.0, -1, one, 0, None, need, None) == -1 and "null" in err()
    assert l.xq_embedding_backward(one, 1, one, 0, 2 ** 31, 64, 8, 1.0, -1, one, 0, one, need, None) == -1 and "2^31" in err()
    assert l.xq_embedding_backward(one, 1, one, 0, 1000, 64, 0, 1.0, -1, one, 0, one, need, None) == -1


def test_on_the_cpu_they_are_the_plain_operators():
    from imagefolder_amd import nn_ops
    x = torch.randn(1000, requires_grad=True)
    torch.manual_seed(3)
    y = nn_ops.dropout(x, 0.5, residual=torch.ones(1000))
    torch.manual_seed(3)
    assert torch.equal(y, torch.nn.functional.dropout(x, 0.5) + 1)
    w = torch.randn(6, 4, requires_grad=True)
    idx = torch.tensor([[1, 5], [2, 1]])
    y = nn_ops.embedding(idx, w, scale=2.0, padding_idx=5)
    assert torch.equal(y, w[idx] * 2)
    (dw,) = torch.autograd.grad(y.sum(), [w])
    assert torch.equal(dw, torch.tensor([0., 4., 2., 0., 0., 0.])[:, None].expand(6, 4))


# ---- the framework's own paths -------------------------------------------------------------------------------------------------------------

@gpu
def test_cnn_block_with_the_counter_based_dropout(monkeypatch):
    """ResnetBlock(dropout > 0): off by default (the module's own dropout); on, a bf16 training step runs on the kernel, channels-last, and its gradient is that of the same
    block with the mask as a constant factor (what the block computes is the same operators on the same values: equal bits)"""
    from imagefolder_amd import nn_ops
    from imagefolder_amd.cnn import ResnetBlock
    torch.manual_seed(4)
    block = ResnetBlock(128, 128, dropout=0.25).cuda().train()
    x = torch.randn(2, 128, 16, 16, device="cuda").to(BF).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    nn_ops.IMPL.pop("dropout", None)
    with torch.autocast("cuda", torch.bfloat16):
        block(x)
    assert "dropout" not in nn_ops.IMPL
    monkeypatch.setattr(nn_ops, "COUNTER_DROPOUT", True)
    seen = {}
    own = nn_ops.dropout

    def spy(t, p, *a, **k):
        seen["key"] = torch.tensor([3, 4], device="cuda")
        seen["like"] = t.detach()
        return own(t, p, key=seen["key"])

    monkeypatch.setattr(nn_ops, "dropout", spy)
    with torch.autocast("cuda", torch.bfloat16):
        y = block(x)
    assert nn_ops.IMPL["dropout"] == "hip"
    g = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, block.conv1.weight, block.conv2.weight], g)
    keep = own(torch.ones_like(seen["like"], dtype=F32), 0.25, key=seen["key"])
    assert seen["like"].stride() == keep.stride() and 0.2 < float((keep == 0).float().mean()) < 0.3

    class Fixed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return (t.float() * keep).to(t.dtype)

        @staticmethod
        def backward(ctx, d):
            return (d.float() * keep).to(d.dtype)

    monkeypatch.setattr(nn_ops, "module_dropout", lambda m, t: Fixed.apply(t))
    with torch.autocast("cuda", torch.bfloat16):
        z = block(x)
    want = torch.autograd.grad(z, [x, block.conv1.weight, block.conv2.weight], g)
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(got, want))
    block.eval()
    nn_ops.IMPL.pop("dropout", None)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        block(x)
    assert "dropout" not in nn_ops.IMPL


@gpu
def test_level_embedding_of_the_tokenizer_runs_on_the_lookup():
    from imagefolder_amd import nn_ops
    from imagefolder_amd.dino_enc.dinov2 import DINOv2Encoder
    torch.manual_seed(0)
    enc = DINOv2Encoder(in_channels=3, num_latent_tokens=16, product_quant=1, model_name="vit_base_patch14_dinov2.lvd142m", pretrained=False, abs_pos_embed=True,
                        tuning_method="full",
                        model_kwargs={'img_size': 64, 'patch_size': 8, 'drop_path_rate': 0.0, 'embed_dim': 64, 'depth': 2, 'num_heads': 1}).cuda()
    nn_ops.IMPL.pop("embedding", None)
    seq = enc._assemble(torch.randn(2, 64, 64, device="cuda"))
    assert nn_ops.IMPL["embedding"] == "hip"
    g = torch.randn_like(seq)
    (dw,) = torch.autograd.grad(seq, [enc.lvl_embed.weight], g)
    check_gradient(enc.lvl1LC, g.sum(0, keepdim=True), enc.lvl_embed.weight.shape[0], 1.0, dw)


@gpu
def test_an_embedding_module_of_another_kind_runs_as_it_is():
    from imagefolder_amd import nn_ops
    torch.manual_seed(4)
    idx = torch.randint(0, 9, (3, 5), device="cuda")
    for kw in (dict(dtype=torch.float16), dict(dtype=torch.float64), dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        m = torch.nn.Embedding(9, 16, device="cuda", **kw)
        nn_ops.IMPL.pop("embedding", None)
        y = nn_ops.module_embedding(m, idx)
        assert "embedding" not in nn_ops.IMPL and torch.equal(y, m(idx)) and y.dtype == m.weight.dtype
    m = torch.nn.Embedding(9, 16, padding_idx=2, device="cuda")
    y = nn_ops.module_embedding(m, idx)
    assert nn_ops.IMPL["embedding"] == "hip" and torch.equal(y, m(idx))
    (dw,) = torch.autograd.grad(y, (m.weight,), torch.ones_like(y))
    want = torch.bincount(idx.reshape(-1), minlength=9).float()
    want[2] = 0
    assert torch.equal(dw, want[:, None].expand(9, 16))


@gpu
def test_second_derivatives_are_refused():
    from imagefolder_amd import nn_ops
    w = torch.randn(9, 16, device="cuda", requires_grad=True)
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    q = torch.randn(1, 4, 2, 8, device="cuda").bfloat16().requires_grad_(True)
    packed = torch.randn(1, 4, 3 * 2 * 8, device="cuda").bfloat16().requires_grad_(True)
    key = torch.tensor([1, 2], device="cuda")
    idx = torch.tensor([1, 1, 3], device="cuda")
    for leaf, f in ((w, lambda t: nn_ops.embedding(idx, t)), (x, lambda t: nn_ops.dropout(t, 0.5, key=key)), (q, lambda t: nn_ops.cross_attention(t, t, t)),
                    (packed, lambda t: nn_ops.attention_qkvpacked(t, 2))):
        y = f(leaf)
        plain, = torch.autograd.grad(y.float().square().sum(), (leaf,), retain_graph=True)
        again, = torch.autograd.grad(y.float().square().sum(), (leaf,), create_graph=True)
        assert torch.equal(plain, again.detach())
        with pytest.raises(RuntimeError, match="twice"):
            again.float().sum().backward()


@gpu
def test_embedding_and_dropout_on_two_streams_at_once():
    from imagefolder_amd import nn_ops
    jobs = []
    for seed in range(2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        idx = torch.randint(0, 5000, (20000,), generator=gen, device="cuda")
        idx[::3] = 7 + seed                       # a frequent row: its pieces meet in the workspace
        jobs.append((torch.randn(5000, 64, generator=gen, device="cuda").requires_grad_(True), idx, torch.randn(20000, 64, generator=gen, device="cuda"),
                     torch.tensor([seed, 5], device="cuda")))

    def step(w, idx, g, key):
        y = nn_ops.dropout(nn_ops.embedding(idx, w), 0.3, key=key)
        return (y.detach(),) + torch.autograd.grad(y, (w,), g)

    want = [step(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*jobs[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(w, r))

"""Calls at the edges of what nn_ops.cross_attention, dropout, embedding and the packed attention of other head widths take: empty ones, sizes past the kernels' limits,
transforms of autograd other than reverse mode, modules with hooks."""
import subprocess
import sys

import pytest
import torch

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32

# (B, Nq, Nk): nothing on one side, sizes on both sides of where the contracted axis is split over blocks
EMPTY = [(b, nq, nk) for n in (1, 448, 449, 480, 481, 5000) for b, nq, nk in ((0, 3, n), (0, n, 3), (2, 0, n), (2, n, 0), (0, n, n), (0, 0, n), (0, n, 0))]


def test_workspaces_of_empty_calls():
    """in a process of its own: a division by zero ends the process"""
    code = ("from imagefolder_amd import _lib\nl = _lib.lib()\n"
            f"for B, Nq, Nk in {EMPTY!r}:\n"
            "    for H, Hk, D in ((4, 4, 64), (8, 2, 128), (1, 1, 8)):\n"
            "        f, b = (fn(B, Nq, Nk, H, Hk, D) for fn in (l.xq_xattn_forward_workspace_bytes, l.xq_xattn_backward_workspace_bytes))\n"
            "        assert f == 0, (B, Nq, Nk, H, f)\n"
            "        assert b <= 4 * B * H * Nq + 256, (B, Nq, Nk, H, b)\n"          # delta alone
            "print('done')")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0 and "done" in r.stdout, (r.returncode, r.stderr[-500:])


@gpu
@pytest.mark.parametrize("B,Nq,Nk", EMPTY)
def test_attention_of_empty_calls(B, Nq, Nk):
    from imagefolder_amd import nn_ops
    q, k, v = (torch.randn(B, n, 4, 64, device="cuda").to(BF).requires_grad_(True) for n in (Nq, Nk, Nk))
    y = nn_ops.cross_attention(q, k, v)
    assert y.shape == q.shape and not y.any()
    for t, d in zip((q, k, v), torch.autograd.grad(y, (q, k, v), torch.ones_like(y))):
        assert d.shape == t.shape and not d.any()


@gpu
@pytest.mark.parametrize("N", [448, 449, 481, 5000])
def test_packed_attention_of_an_empty_batch(N):
    from imagefolder_amd import nn_ops, ops_dense
    for entry in (nn_ops.attention_qkvpacked, ops_dense.attention_qkvpacked):
        qkv = torch.zeros(0, N, 3 * 2 * 32, device="cuda", dtype=BF, requires_grad=True)
        y = entry(qkv, 2)
        assert y.shape == (0, N, 64)
        assert torch.autograd.grad(y, (qkv,), torch.zeros_like(y))[0].shape == qkv.shape


def test_no_vector_arithmetic_in_inline_asm():
    """The compiler places no wait between a matrix instruction and inline asm that reads its result: what computes on vector registers is written with builtins"""
    import pathlib
    import re
    csrc = pathlib.Path(__file__).resolve().parents[1] / "imagefolder_amd" / "csrc"
    sources = sorted(csrc.glob("*.hip")) + sorted(csrc.glob("*.hpp"))
    assert len(sources) > 10
    found = [f"{p.name}: {m.group(0)[:60]}" for p in sources for m in re.finditer(r'\basm\s*(?:volatile\s*)?\(\s*"[^"]*\bv_\w+', p.read_text())]
    assert not found, found


# ---- transforms of autograd other than reverse mode -----------------------------------------------------------------------------------------

def copying_launch(monkeypatch):
    """stands for the kernels on the CPU: the result's memory gets the (first) input's -> the names launched"""
    import ctypes
    from imagefolder_amd import ops_seq
    calls = []

    def launch(name, device, *args):
        calls.append(name)
        if name == "xq_dropout":
            ctypes.memmove(args[6], args[0], 4 * args[3])
        elif name == "xq_embedding_forward":
            ctypes.memmove(args[8], args[2], 4 * args[4] * args[6])
        else:
            B, Nq, _, H, _, D = args[3:9]
            ctypes.memmove(args[14], args[0], 2 * B * Nq * H * D)

    monkeypatch.setattr(ops_seq, "_launch", launch)
    return calls


def forward_calls():
    from imagefolder_amd import ops_seq
    key, idx = torch.tensor([1, 2]), torch.arange(5)
    k = torch.randn(1, 7, 2, 8).to(BF)
    return (("dropout", torch.randn(40), lambda t: ops_seq.dropout(t, 0.5, key=key)),
            ("dropout + residual", torch.randn(40), lambda t: ops_seq.dropout(t, 0.5, key=key, residual=t)),
            ("embedding", torch.randn(5, 8), lambda t: ops_seq.embedding(idx, t)),
            ("cross_attention", torch.randn(1, 3, 2, 8).to(BF), lambda t: ops_seq.cross_attention(t, k, k)))


@pytest.mark.parametrize("i", range(4))
def test_a_tangent_is_refused_not_lost(i, monkeypatch):
    """forward-mode differentiation: the operators have no formula for it, so that a dual tensor is an error with and without gradients, as long as a level is open"""
    from torch.autograd import forward_ad
    calls = copying_launch(monkeypatch)
    name, x, f = forward_calls()[i]
    assert torch.equal(f(x), x) and len(calls) == 1, name
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not dual.requires_grad
        with pytest.raises(RuntimeError, match="jvp"):
            f(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
            f(dual)
        assert torch.equal(f(x), x)                    # no tangent on it
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("i", range(4))
def test_a_trace_records_the_call(i, monkeypatch):
    calls = copying_launch(monkeypatch)
    name, x, f = forward_calls()[i]
    traced = torch.jit.trace(f, (x,), check_trace=False)
    other = torch.randn(x.shape).to(x.dtype)
    before = len(calls)
    assert torch.equal(traced(other), other) and len(calls) == before + 1, name


@gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls(grad):
    """a traced program computes each call anew, on its own inputs"""
    from imagefolder_amd import nn_ops
    key, idx = torch.tensor([1, 2], device="cuda"), torch.arange(5, device="cuda")
    k = torch.randn(1, 70, 2, 8, device="cuda").to(BF)
    for x, f in ((torch.randn(4000, device="cuda"), lambda t: nn_ops.dropout(t, 0.5, key=key)),
                 (torch.randn(5, 8, device="cuda"), lambda t: nn_ops.embedding(idx, t, scale=3.0)),
                 (torch.randn(1, 3, 2, 8, device="cuda").to(BF), lambda t: nn_ops.cross_attention(t, k, k)),
                 (torch.randn(2, 9, 3 * 2 * 32, device="cuda").to(BF), lambda t: nn_ops.attention_qkvpacked(t, 2))):
        traced = torch.jit.trace(f, (x.clone().requires_grad_(grad),), check_trace=False)
        for _ in range(3):
            other = torch.randn(x.shape, device="cuda").to(x.dtype)
            assert torch.equal(traced(other), f(other))


# ---- infinities ------------------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("Nk,D", [(50, 32), (50, 64), (50, 96), (50, 128), (200, 32), (200, 64), (300, 64), (300, 96), (300, 128)])
@pytest.mark.parametrize("Nq,G", [(1, 1), (31, 1), (32, 1), (33, 1), (65, 1), (300, 1), (11, 3), (11, 5), (50, 8), (700, 2)])
def test_a_key_at_minus_infinity_has_zero_gradients(Nk, D, Nq, G):
    """its score is -inf and its P 0 in every row, whatever the number of rows: dk and dv are those of a call where it is masked (dq = dS k is 0 x inf there)"""
    from imagefolder_amd import nn_ops
    torch.manual_seed(Nq + D)
    B, Hk = 2, 2
    q = torch.randn(B, Nq, Hk * G, D, device="cuda").abs().add(0.5).to(BF).requires_grad_(True)
    k, v = (torch.randn(B, Nk, Hk, D, device="cuda").to(BF).requires_grad_(True) for _ in range(2))
    g = torch.randn(B, Nq, Hk * G, D, device="cuda").to(BF)
    bad = k.detach().clone()
    bad[:, 7] = 0
    bad[:, 7, :, 0] = float("-inf")
    bad.requires_grad_(True)
    there = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
    there[:, 7] = False
    y, want = nn_ops.cross_attention(q, bad, v), nn_ops.cross_attention(q, k, v, key_mask=there)
    assert torch.equal(y, want)
    got, ref = torch.autograd.grad(y, (bad, v), g), torch.autograd.grad(want, (k, v), g)
    for a, b in zip(got, ref):
        assert not a[:, 7].any() and torch.equal(a, b)


# ---- more than one call of the kernels takes ---------------------------------------------------------------------------------------------------

def packed(B, N, H, D, **kw):
    from types import SimpleNamespace
    return SimpleNamespace(**{**dict(is_cuda=True, dtype=BF, shape=torch.Size((B, N, 3 * H * D)), dim=lambda: 3), **kw})


@pytest.mark.parametrize("B,N,H,D", [(32768, 49, 16, 32), (29127, 128, 16, 32), (29128, 128, 16, 32), (26214, 129, 16, 8), (26215, 129, 16, 8), (466033, 1, 1, 128), (466034, 1, 1, 128),
                                     (2, 268434432, 1, 8), (2, 268434433, 1, 8), (1, 1, 21845, 128), (1, 1, 21846, 128), (0, 70000, 3, 32), (4, 0, 3, 32)])
def test_packed_attention_takes_what_its_kernels_take(B, N, H, D):
    """the dispatch and the C entry's own limits say the same (its workspace query checks them); the library takes the rest"""
    from imagefolder_amd import _lib, ops_seq
    l = _lib.lib()
    assert l.xq_xattn_forward_workspace_bytes(1, 1, 1, 1, 1, 9) == 0 and "head dim 9" in l.xq_last_error().decode()
    for fn in (l.xq_xattn_forward_workspace_bytes, l.xq_xattn_backward_workspace_bytes):
        fn(B, N, N, H, H, D)
    refused = "too many rows" in l.xq_last_error().decode()
    if 3 * H * D <= 1 << 23:
        assert ops_seq.packed_attention_supported(packed(B, N, H, D), H) == (not refused)
    else:
        assert not ops_seq.packed_attention_supported(packed(B, N, H, D), H)


def test_packed_attention_leaves_other_forms_to_the_library():
    from imagefolder_amd import ops_seq
    assert ops_seq.packed_attention_supported(packed(2, 50, 4, 32), 4)
    for t, H in ((packed(2, 50, 4, 32, dtype=torch.float16), 4), (packed(2, 50, 4, 32, is_cuda=False), 4), (packed(2, 50, 4, 32, dim=lambda: 4), 4), (packed(2, 50, 4, 36), 4),
                 (packed(2, 50, 4, 136), 4), (packed(2, 50, 4, 32), 5), (packed(2, 50, 1, 2), 2)):
        assert not ops_seq.packed_attention_supported(t, H)


@gpu
def test_packed_attention_of_more_windows_than_one_call_takes():
    from imagefolder_amd import nn_ops, ops_dense
    torch.manual_seed(3)
    B, N, H, D = 32768, 3, 16, 8
    qkv = torch.randn(B, N, 3 * H * D, device="cuda").to(BF).requires_grad_(True)
    for entry in (nn_ops.attention_qkvpacked, ops_dense.attention_qkvpacked):
        y = entry(qkv, H)
        (dx,) = torch.autograd.grad(y, (qkv,), torch.ones_like(y))
        assert y.shape == (B, N, H * D) and dx.shape == qkv.shape and bool(dx.isfinite().all())
        for b in (0, B // 2, B - 1):
            q, k, v = qkv.detach()[b].double().view(N, 3, H, D).permute(1, 2, 0, 3)
            p = torch.softmax(q @ k.transpose(1, 2) * D ** -0.5, -1)
            # P rounded to bf16 where it meets v and in the row sum, the result once
            tol = 1.05 * (2 * 2.0 ** -8 * (p @ v.abs()) + 2.0 ** -8 * (p @ v).abs()) + 1e-6
            assert bool(((y.detach()[b].double().view(N, H, D).transpose(0, 1) - p @ v).abs() <= tol).all())


def test_the_limit_of_table_rows_is_the_kernels():
    from imagefolder_amd import _lib, ops_seq
    l = _lib.lib()
    assert l.xq_embedding_backward_workspace_bytes(5, ops_seq.MAX_ROWS, 8) > 0 and l.xq_embedding_backward_workspace_bytes(5, ops_seq.MAX_ROWS + 1, 8) == 0


@gpu
@pytest.mark.parametrize("more", [0, 1])
def test_an_embedding_module_of_many_rows(more):
    from imagefolder_amd import nn_ops, ops_seq
    V = ops_seq.MAX_ROWS + more
    m = torch.nn.Embedding(V, 4, device="cuda")
    idx = torch.tensor([[0, V - 1, 5], [5, 5, 0]], device="cuda")
    nn_ops.IMPL.pop("embedding", None)
    y = nn_ops.module_embedding(m, idx)
    assert ("embedding" in nn_ops.IMPL) == (more == 0) and torch.equal(y, m(idx))
    (dw,) = torch.autograd.grad(y.sum(), (m.weight,))
    assert dw[:, 0].nonzero()[:, 0].tolist() == [0, 5, V - 1] and dw[[0, 5, V - 1], 0].tolist() == [2, 3, 1]


# ---- modules that something hangs on -----------------------------------------------------------------------------------------------------------

def hung(make, x):
    """(a module, what its call adds) for each way of hanging something on a module's call; `seen` tells that it ran"""
    seen = []

    class Own(type(make())):
        def forward(self, t):
            seen.append("subclass")
            return super().forward(t)

    m = make()
    m.register_forward_hook(lambda *a: seen.append("hook"))
    yield m, seen
    m = make()
    m.register_forward_pre_hook(lambda *a: seen.append("pre"))
    yield m, seen
    m = make()
    m.__class__ = Own
    yield m, seen
    m = make()
    inner = m.forward
    m.forward = lambda t: (seen.append("own"), inner(t))[1]
    yield m, seen
    m = make()
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: seen.append("global"))
    try:
        yield m, seen
    finally:
        handle.remove()


def dropouts_and_lookups(device):
    idx = torch.randint(0, 9, (3, 5), device=device)
    x = torch.randn(3, 40, device=device)
    return ((lambda: torch.nn.Embedding(9, 16, device=device), idx, "module_embedding", "embedding"), (lambda: torch.nn.Dropout(0.5), x, "module_dropout", "dropout"))


@pytest.mark.parametrize("which", [0, 1])
def test_what_hangs_on_a_module_runs(which, monkeypatch):
    """on the CPU, with the dispatch's own look at the device (x.is_cuda) left out of the way: what is asked is the module"""
    from imagefolder_amd import nn_ops
    monkeypatch.setattr(nn_ops, "COUNTER_DROPOUT", True)
    make, x, entry, _ = dropouts_and_lookups("cpu")[which]
    assert nn_ops._runs_plainly(make(), type(make()))
    for m, seen in hung(make, x):
        assert not nn_ops._runs_plainly(m, type(make()))
        seen.clear()
        getattr(nn_ops, entry)(m, x)
        assert len(seen) == 1
    assert nn_ops._runs_plainly(make(), type(make()))
    for kind in ("register_full_backward_hook", "register_full_backward_pre_hook"):
        m = make()
        getattr(m, kind)(lambda *a: None)
        assert not nn_ops._runs_plainly(m, type(make()))


@gpu
@pytest.mark.parametrize("which", [0, 1])
def test_what_hangs_on_a_module_runs_on_the_gpu(which, monkeypatch):
    from imagefolder_amd import nn_ops
    monkeypatch.setattr(nn_ops, "COUNTER_DROPOUT", True)
    make, x, entry, name = dropouts_and_lookups("cuda")[which]
    nn_ops.IMPL.pop(name, None)
    for m, seen in hung(make, x):
        seen.clear()
        getattr(nn_ops, entry)(m, x)
        assert len(seen) == 1 and name not in nn_ops.IMPL
    getattr(nn_ops, entry)(make(), x)
    assert nn_ops.IMPL[name] == "hip"


@gpu
def test_a_module_that_is_no_embedding_in_its_place():
    from imagefolder_amd import nn_ops

    class Sum(torch.nn.Module):                         # a table without `weight`
        def __init__(self):
            super().__init__()
            self.a, self.b = (torch.nn.Embedding(9, 4, device="cuda") for _ in range(2))

        def forward(self, idx):
            return self.a(idx) + self.b(idx)

    m, idx = Sum(), torch.randint(0, 9, (3, 5), device="cuda")
    assert torch.equal(nn_ops.module_embedding(m, idx), m(idx))

    class Scaled(torch.Tensor):                         # a weight with a lookup of its own
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            out = super().__torch_function__(func, types, args, kwargs or {})
            return out * 2 if func is torch.nn.functional.embedding else out

    e = torch.nn.Embedding(9, 4, device="cuda")
    del e._parameters["weight"]
    e.weight = torch.randn(9, 4, device="cuda").as_subclass(Scaled)
    assert torch.equal(nn_ops.module_embedding(e, idx).as_subclass(torch.Tensor), e(idx).as_subclass(torch.Tensor))


# ---- transforms, where a kernel stands for a library operator ------------------------------------------------------------------------------------

def test_transforms_are_seen():
    from torch.autograd import forward_ad
    from imagefolder_amd import ops_seq
    seen = []
    f = lambda t: (seen.append(ops_seq.transformed()), (t * t).sum())[1]  # noqa: E731
    x = torch.ones(3, requires_grad=True)
    f(x).backward()
    assert seen == [False]
    torch.func.grad(f)(torch.ones(3))
    torch.func.jvp(f, (torch.ones(3),), (torch.ones(3),))
    torch.vmap(f)(torch.ones(2, 3))
    with forward_ad.dual_level():
        f(torch.ones(3))
        assert not ops_seq.packed_attention_supported(packed(2, 50, 4, 32), 4)
    assert seen == [False] + [True] * 4 and not ops_seq.transformed()
    assert ops_seq.packed_attention_supported(packed(2, 50, 4, 32), 4)


@gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_level_table_under_transforms():
    from torch.autograd import forward_ad
    from imagefolder_amd import nn_ops
    m = torch.nn.Embedding(9, 16, device="cuda")
    idx = torch.randint(0, 9, (3, 5), device="cuda")
    w, d = torch.randn(9, 16, device="cuda"), torch.randn(9, 16, device="cuda")
    with forward_ad.dual_level():
        del m._parameters["weight"]
        m.weight = forward_ad.make_dual(w, d)
        y = forward_ad.unpack_dual(nn_ops.module_embedding(m, idx))
        assert torch.equal(y.primal, w[idx]) and torch.equal(y.tangent, d[idx])
    m = torch.nn.Embedding(9, 16, device="cuda")
    call = lambda p, i=idx: torch.func.functional_call(Lookup(m), {"m.weight": p}, (i,))  # noqa: E731
    got = torch.func.grad(lambda p: (call(p) ** 2).sum())(w)
    want = torch.zeros(9, 16, device="cuda").index_add_(0, idx.reshape(-1), 2 * w[idx].reshape(-1, 16))
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)
    assert torch.equal(torch.func.jvp(call, (w,), (d,))[1], d[idx])
    assert torch.equal(torch.vmap(call)(torch.stack((w, d))), torch.stack((w[idx], d[idx])))
    traced = torch.jit.trace(Lookup(m), (idx,), check_trace=False)
    assert "aten::embedding" in str(traced.inlined_graph)
    other = torch.randint(0, 9, (3, 5), device="cuda")
    assert torch.equal(traced(other), m(other))


class Lookup(torch.nn.Module):
    def __init__(self, m):
        super().__init__()
        self.m = m

    def forward(self, idx):
        from imagefolder_amd import nn_ops
        return nn_ops.module_embedding(self.m, idx)


@gpu
def test_packed_attention_under_a_transform():
    """the gradient of torch.func through the library's operator, against the kernels' own"""
    from torch.nn.attention import SDPBackend, sdpa_kernel
    from imagefolder_amd import nn_ops
    torch.manual_seed(2)
    x, g = torch.randn(2, 60, 3 * 4 * 32, device="cuda").to(BF), torch.randn(2, 60, 4 * 32, device="cuda").to(BF)
    leaf = x.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(nn_ops.attention_qkvpacked(leaf, 4), (leaf,), g)
    with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
        got = torch.func.grad(lambda t: (nn_ops.attention_qkvpacked(t, 4).float() * g.float()).sum())(x)
    # each side rounds P, dS, the rounded O in delta and the result to bf16: 4 * 2^-8 in norm, twice
    assert float((got.double() - want.double()).norm()) <= 8 * 2.0 ** -8 * float(want.double().norm())


@gpu
@pytest.mark.parametrize("pad", [None, 3])
def test_second_derivatives_of_a_level_table(pad):
    """as the module's: y = w[idx], L = sum c y^4, dL/dw, the gradient of its product with d, and of that once more (of fp32 sums of few terms: 2^-18 of their size)"""
    from imagefolder_amd import nn_ops
    torch.manual_seed(1)
    m = torch.nn.Embedding(9, 16, padding_idx=pad, device="cuda")
    idx = torch.randint(0, 9, (3, 20), device="cuda")
    c, d = torch.randn(3, 20, 16, device="cuda"), torch.randn(9, 16, device="cuda")

    def derivatives(look):
        (a,) = torch.autograd.grad((c * look(idx) ** 4).sum(), (m.weight,), create_graph=True)
        (b,) = torch.autograd.grad((a * d).sum(), (m.weight,), create_graph=True)
        (e,) = torch.autograd.grad((b * d).sum(), (m.weight,))
        return a.detach(), b.detach(), e

    nn_ops.IMPL.pop("embedding", None)
    got = derivatives(lambda i: nn_ops.module_embedding(m, i))
    assert nn_ops.IMPL["embedding"] == "hip"
    want = derivatives(m)
    for a, b in zip(got, want):
        assert float((a - b).abs().max()) <= 2.0 ** -18 * 24 * float(m.weight.detach().abs().max()) ** 3 * 60 * float(c.abs().max()) * max(1, float(d.abs().max())) ** 2
        assert float(b.abs().max()) > 1e-2 and (pad is None or not a[pad].any())


# ---- dropout in place --------------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("kind", [BF, F32])
@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("n", [1, 8, 4099, 3000001])
def test_dropout_in_place(n, first, kind):
    """xq_dropout with y = x (the C entry's promise), on aligned elements and from an odd one on, with and without a residual"""
    from imagefolder_amd import _lib
    key = torch.tensor([5, 7], device="cuda")
    base = torch.randn(n + first, device="cuda").to(kind)
    r = torch.randn(n + first, device="cuda").to(kind)[first:]
    stream = torch.cuda.current_stream().cuda_stream
    for res in (None, r.data_ptr()):
        apart, x = torch.zeros_like(base)[first:], base.clone()[first:]
        for y in (apart, x):
            assert _lib.lib().xq_dropout(x.data_ptr(), kind == BF, res, n, 0.3, key.data_ptr(), y.data_ptr(), kind == BF, stream) == 0
        assert torch.equal(apart, x)


# ---- offsets -----------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("H,Hk,Nq,taken", [(1 << 17, 1 << 17, 64, False), ((1 << 17) - 1, (1 << 17) - 1, 64, True), (1 << 17, 1, 2, False), ((1 << 17) - 2048, 1, 2, True), (1 << 23, 1, 1, True),
                                           ((1 << 23) + 1, 1, 1, False), (1 << 24, 1, 1, False)])
def test_rows_of_out_past_32_bits_of_bytes_are_refused(H, Hk, Nq, taken):
    """the C entry, on head-major q and dq (or broadcast ones): no launch either way, the workspace handed in is too small"""
    import ctypes
    from imagefolder_amd import _lib
    l, one, D, Nk = _lib.lib(), ctypes.c_void_p(16), 128, 300
    st = (ctypes.c_int64 * 9)(*[0, D, 0] + [64] * 6)
    grad = (ctypes.c_int64 * 9)(*[64, D, 8] + [64] * 6)
    rc = l.xq_xattn_backward(one, one, one, one, one, one, 1, Nq, Nk, H, Hk, D, st, None, 0, None, ctypes.c_float(0.1), one, one, one, grad, one, 0, None)
    assert (rc, "too small" if taken else "too wide") == (-2 if taken else -1, "too small" if taken else "too wide")
    assert ("too small" if taken else "too wide") in l.xq_last_error().decode()


def test_views_that_the_kernels_do_not_reach_over_are_copied():
    """head-major q of long sequences under many shared heads: 64 tokens and the group's heads span more than 2^30 elements (no memory behind meta tensors)"""
    from imagefolder_amd import ops_seq
    q = torch.empty(1, 512, 32768, 128, dtype=BF, device="meta").transpose(1, 2)           # heads 2^22 elements apart
    assert ops_seq._rows(q) is q and ops_seq._rows(q, 254) is q
    for group in (256, 512):
        copy = ops_seq._rows(q, group)
        assert copy.is_contiguous() and copy.shape == q.shape
    flat = torch.empty(1, 70, 512, 128, dtype=BF, device="meta")
    assert ops_seq._rows(flat, 512) is flat


# ---- on the CPU --------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("wt", [BF, torch.float16, F32, torch.float64])
@pytest.mark.parametrize("yt", [None, BF, F32, torch.float64])
def test_a_scaled_lookup_on_the_cpu_is_rounded_once(wt, yt):
    from imagefolder_amd import nn_ops
    torch.manual_seed(0)
    w, idx = torch.randn(50, 8).to(wt).requires_grad_(True), torch.randint(0, 50, (4, 30))
    y = nn_ops.embedding(idx, w, scale=1.7, dtype=yt)
    assert y.dtype == (yt or wt)
    want = w.detach().double()[idx] * 1.7
    # the product in 32 bits (64 for a 64-bit table), then the result's rounding
    product = 2.0 ** -52 if wt == torch.float64 else 2.0 ** -23
    assert bool(((y.detach().double() - want).abs() <= want.abs() * (torch.finfo(y.dtype).eps / 2 * (1 + 2.0 ** -7) + product)).all())
    (dw,) = torch.autograd.grad(y.sum(), (w,))
    assert dw.dtype == wt and dw[idx[0, 0], 0] > 0


def test_dropout_checks_its_arguments_on_every_path():
    """the CPU, evaluation and p = 0 refuse what a training step on the GPU refuses"""
    from imagefolder_amd import nn_ops
    from imagefolder_amd._lib import XqError
    x = torch.randn(6, 8)
    for training in (True, False):
        for kw, what in ((dict(p=1.5), r"\[0, 1\]"), (dict(p=float("nan")), r"\[0, 1\]"), (dict(p=-0.1), r"\[0, 1\]"), (dict(residual=torch.zeros(8)), "residual of shape"),
                         (dict(p=0.0, residual=torch.zeros(1, 8)), "residual of shape"), (dict(residual=x.to(BF)), "residual of type")):
            with pytest.raises(XqError, match=what):
                nn_ops.dropout(x, training=training, **{"p": 0.5, **kw})
        assert nn_ops.dropout(x, 0.5, training, residual=x).dtype == F32


@pytest.mark.parametrize("rt", [BF, F32])
def test_dropout_and_residual_on_the_cpu_are_rounded_once(rt):
    from imagefolder_amd import nn_ops
    x, r = torch.randn(5000).to(BF), torch.randn(5000).to(rt)
    y = nn_ops.dropout(x, 0.3, residual=r)
    assert y.dtype == rt
    kept, dropped = x.double() / 0.7 + r.double(), r.double()
    off = lambda want: (y.double() - want).abs() <= want.abs() * torch.finfo(rt).eps / 2 * (1 + 2.0 ** -7) + x.double().abs() * 2.0 ** -22  # noqa: E731
    assert bool((off(kept) | off(dropped)).all()) and 0.2 < float((y.double() == dropped).double().mean()) < 0.4


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("Nq,Nk", [(3, 5), (40, 40), (40, 300), (300, 700), (1, 3000)])
def test_rows_whose_scores_are_all_minus_infinity(device, Nq, Nk):
    """every second key has a score of -inf: as if it were masked; where those are the only valid ones a row is zero, on every path"""
    from imagefolder_amd import nn_ops
    torch.manual_seed(Nq)
    kind = BF if device == "cuda" else F32
    k, v = (torch.randn(2, Nk, 2, 16, device=device).to(kind) for _ in range(2))
    k[..., 0] = 0
    k[:, ::2] = 0
    k[:, ::2, :, 0] = float("-inf")
    q = torch.randn(2, Nq, 2, 16, device=device).to(kind)
    q[..., 0] = 1
    there = torch.ones(2, Nk, dtype=torch.bool, device=device)
    there[:, ::2] = False
    assert torch.equal(nn_ops.cross_attention(q, k, v), nn_ops.cross_attention(q, k, v, key_mask=there))
    assert not nn_ops.cross_attention(q, k, v, key_mask=~there).any()

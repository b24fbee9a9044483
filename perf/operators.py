"""Measured cases of the cross-attention, dropout and embedding operators (imagefolder_amd.nn_ops): what each one computes in plain
torch operations, the calls a user makes of it, and the work it cannot do without."""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one class / image query against one image's states: the latency of a serving call
        {"name": "attend_one_token", "op": "attend", "B": 1, "Nq": 1, "Nk": 257, "H": 12, "Hk": 12, "D": 64, "train": False, "ragged": False, "mask": False},
        # a batch of requests, one new token each, over long encoder states of different lengths, four query heads to a kv head
        {"name": "attend_one_token_long", "op": "attend", "B": 16, "Nq": 1, "Nk": 8111, "H": 32, "Hk": 8, "D": 128, "train": False, "ragged": True, "mask": False},
        # the tokenizer's geometry: 256 latent queries over 257 image tokens, twelve heads of 64, batch 128, a training step
        {"name": "attend_latents_train", "op": "attend", "B": 128, "Nq": 256, "Nk": 257, "H": 12, "Hk": 12, "D": 64, "train": True, "ragged": False, "mask": False},
        # a multi-scale token ladder (286 tokens) reading a padded condition: odd sizes, shared heads, holes in the mask, a sample with none left
        {"name": "attend_condition_train", "op": "attend", "B": 24, "Nq": 286, "Nk": 93, "H": 16, "Hk": 4, "D": 96, "train": True, "ragged": True, "mask": True},
        # long sequences on both sides: the largest training call
        {"name": "attend_long_train", "op": "attend", "B": 4, "Nq": 4096, "Nk": 4352, "H": 16, "Hk": 16, "D": 128, "train": True, "ragged": True, "mask": False},
        # the tokens of one image in a forward pass
        {"name": "drop_image", "op": "drop", "n": 256 * 768, "p": 0.1, "type": "bf16", "residual": "", "train": False},
        # a branch added to the fp32 residual stream of the tokenizer's blocks, batch 128, with its backward pass
        {"name": "drop_residual_train", "op": "drop", "n": 128 * 513 * 768, "p": 0.1, "type": "bf16", "residual": "fp32", "train": True},
        # an odd number of fp32 values
        {"name": "drop_odd_train", "op": "drop", "n": 1000003, "p": 0.37, "type": "fp32", "residual": "", "train": True},
        # sixteen requests' next codes
        {"name": "embed_next_codes", "op": "embed", "N": 16, "V": 16384, "D": 1024, "type": "fp32", "out": "bf16", "zipf": 0.0, "train": False},
        # the codes of 128 images into a ViT-B wide table, with the table's gradient
        {"name": "embed_codes_train", "op": "embed", "N": 128 * 256, "V": 8192, "D": 768, "type": "fp32", "out": "bf16", "zipf": 0.0, "train": True},
        # text-like ids: few rows take most of the tokens
        {"name": "embed_skewed_train", "op": "embed", "N": 99991, "V": 50021, "D": 512, "type": "bf16", "out": "bf16", "zipf": 1.1, "train": True},
        # the narrow rows of a codebook
        {"name": "embed_codebook_train", "op": "embed", "N": 128 * 680, "V": 16384, "D": 32, "type": "fp32", "out": "fp32", "zipf": 0.6, "train": True},
    ]


def _between(rng, lo, hi):
    """a whole number of [lo, hi], spread over its logarithm"""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "drop", "embed"])
    if op == "attend":
        D = rng.choice([32, 64, 80, 96, 128])
        Hk, G = rng.choice([1, 2, 4, 6, 8, 12]), rng.choice([1, 1, 2, 4])
        train = rng.random() < 0.6
        Nq = _between(rng, 8, 2048) if train else _between(rng, 1, 512)
        Nk = _between(rng, 8 if train else 1, 4096)       # (over a single key dq and dk are zero: nothing to compare)
        most = 4e8 if train else 1e8
        B = max(1, min(_between(rng, 1, 64), int(most / (Nq * Nk * Hk * G))))
        return {"op": "attend", "B": B, "Nq": Nq, "Nk": Nk, "H": Hk * G, "Hk": Hk, "D": D, "train": train, "ragged": rng.random() < 0.5,
                "mask": rng.random() < 0.3}
    if op == "drop":
        kind = rng.choice(["bf16", "fp32"])
        return {"op": "drop", "n": _between(rng, 1, 20_000_000), "p": round(rng.uniform(0.01, 0.9), 3), "type": kind,
                "residual": rng.choice(["", "fp32", kind]), "train": rng.random() < 0.6}
    D, V = rng.choice([8, 32, 64, 100, 384, 768, 1024]), _between(rng, 2, 60000)
    return {"op": "embed", "N": _between(rng, 1, 60000), "V": V, "D": D, "type": rng.choice(["bf16", "fp32"]), "out": rng.choice(["bf16", "fp32"]),
            "zipf": rng.choice([0.0, 0.6, 1.1]), "train": rng.random() < 0.6}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------

def _lens(case):
    """the samples' numbers of keys, before the seed's order: spread evenly from none to all where the case is ragged"""
    B, Nk = case["B"], case["Nk"]
    if not case["ragged"]:
        return [Nk] * B
    return [Nk - (Nk * b) // B if case["mask"] else Nk - (Nk * b) // (2 * B) for b in range(B - 1)] + [0 if case["mask"] and B > 1 else Nk // 2 + 1 if Nk > 1 else 1]


def _probabilities(case):
    r = np.arange(1, case["V"] + 1, dtype=np.float64) ** -case["zipf"]
    return r / r.sum()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape, type=torch.bfloat16):
        return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32).to(type)

    if case["op"] == "attend":
        B, Nq, Nk, H, Hk, D = (case[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
        s = {"case": case, "q": normal(B, Nq, H, D) * 1.5, "lens": None, "mask": None, "scale": D ** -0.5}
        kv = normal(B, Nk, 2, Hk, D)                       # the packed projection of the states: keys and values are views of it
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        if case["ragged"]:
            order = torch.randperm(B, generator=gen, device=DEV)
            s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)[order].contiguous()
        if case["mask"]:
            s["mask"] = torch.rand(B, Nk, generator=gen, device=DEV) < 0.9
        if case["train"]:
            s["g"] = normal(B, Nq, H, D)
            for n in ("q", "k", "v"):
                s[n] = s[n].detach().requires_grad_(True)
        return s
    if case["op"] == "drop":
        n, kind = case["n"], TYPES[case["type"]]
        s = {"case": case, "x": normal(n, type=kind), "residual": normal(n, type=TYPES[case["residual"]]) if case["residual"] else None,
             "key": torch.randint(0, 2 ** 62, (2,), generator=gen, device=DEV)}
        if case["train"]:
            s["g"] = normal(n, type=TYPES[case["residual"] or case["type"]])
            s["x"].requires_grad_(True)
            if s["residual"] is not None:
                s["residual"].requires_grad_(True)
        return s
    N, V, D = case["N"], case["V"], case["D"]
    s = {"case": case, "w": normal(V, D, type=TYPES[case["type"]]), "scale": D ** 0.5}
    if case["zipf"]:
        edges = torch.from_numpy(np.cumsum(_probabilities(case))).to(DEV)
        ranks = torch.searchsorted(edges, torch.rand(N, generator=gen, device=DEV, dtype=torch.float64)).clamp_(max=V - 1)
        s["idx"] = torch.randperm(V, generator=gen, device=DEV)[ranks]      # frequent rows lie anywhere in the table
    else:
        s["idx"] = torch.randint(0, V, (N,), generator=gen, device=DEV)
    if case["train"]:
        s["g"] = normal(N, D, type=TYPES[case["out"]])
        s["w"].requires_grad_(True)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------

def _plain_attend(s):
    with torch.no_grad():
        q, k, v = s["q"], s["k"], s["v"]
        B, Nq, H, D = q.shape
        Nk, Hk = k.shape[1], k.shape[2]
        G = H // Hk
        q4 = q.float().view(B, Nq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Nq, D)
        k4, v4 = (t.float().permute(0, 2, 1, 3).contiguous() for t in (k, v))
        valid = torch.ones(B, Nk, dtype=torch.bool, device=q.device)
        if s["lens"] is not None:
            valid = valid & (torch.arange(Nk, device=q.device)[None] < s["lens"][:, None])
        if s["mask"] is not None:
            valid = valid & s["mask"]
        P = (torch.matmul(q4, k4.transpose(2, 3).contiguous()) * s["scale"]).masked_fill_(~valid[:, None, None], float("-inf"))
        top = P.amax(-1, keepdim=True)
        P = (P - top.masked_fill(top == float("-inf"), 0.0)).exp_()
        total = P.sum(-1, keepdim=True)
        P = P / total.masked_fill(total == 0, 1.0)
        O = torch.matmul(P, v4)

        def heads(t):       # (B, Hk, G Nq, D) -> (B, Nq, H, D)
            return t.view(B, Hk, G, Nq, D).permute(0, 3, 1, 2, 4).reshape(B, Nq, H, D).to(q.dtype)

        if not s["case"]["train"]:
            return heads(O)
        g4 = s["g"].float().view(B, Nq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Nq, D)
        dv = torch.matmul(P.transpose(2, 3).contiguous(), g4)
        dS = torch.matmul(g4, v4.transpose(2, 3).contiguous())
        dS = dS.sub_((g4 * O).sum(-1, keepdim=True)).mul_(P).mul_(s["scale"])
        dq = torch.matmul(dS, k4)
        dk = torch.matmul(dS.transpose(2, 3).contiguous(), q4)
        return heads(O), heads(dq), dk.permute(0, 2, 1, 3).to(k.dtype).contiguous(), dv.permute(0, 2, 1, 3).to(v.dtype).contiguous()


def _words(n, key):
    """the ceil(n / 8) x 4 words of Philox4x32-10: counter (block, key[1]), key key[0]"""
    low = 0xFFFFFFFF
    at = torch.arange((n + 7) // 8, device=key.device, dtype=torch.int64)
    a, b = at & low, (at >> 32) & low
    c, d = (key[1] & low).expand_as(at), ((key[1] >> 32) & low).expand_as(at)
    k0, k1 = key[0] & low, (key[0] >> 32) & low
    for _ in range(10):
        p, r = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((r >> 32) & low) ^ b ^ k0, r & low, ((p >> 32) & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((a, b, c, d), 1)


def _plain_drop(s):
    with torch.no_grad():
        x, n = s["x"], s["case"]["n"]
        t = int(round(65536 * s["case"]["p"]))
        w = _words(n, s["key"])
        keep = torch.stack((w & 0xFFFF, w >> 16), 2).reshape(-1)[:n] >= t
        factor = keep.float() * (65536.0 / (65536 - t))
        y = x.float() * factor
        y = y.to(x.dtype) if s["residual"] is None else (y + s["residual"].float()).to(s["residual"].dtype)
        if not s["case"]["train"]:
            return y
        dx = (s["g"].float() * factor).to(x.dtype)
        return (y, dx) if s["residual"] is None else (y, dx, s["g"])


def _plain_embed(s):
    with torch.no_grad():
        w, idx, out = s["w"], s["idx"], TYPES[s["case"]["out"]]
        y = (w[idx].float() * s["scale"]).to(out)
        if not s["case"]["train"]:
            return y
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, idx, s["g"].float())
        return y, (dw * s["scale"]).to(w.dtype)


def run(s):
    case = s["case"]
    if not own:
        return _plain_attend(s) if case["op"] == "attend" else _plain_drop(s) if case["op"] == "drop" else _plain_embed(s)
    from imagefolder_amd import nn_ops
    if case["op"] == "attend":
        y = nn_ops.cross_attention(s["q"], s["k"], s["v"], kv_lens=s["lens"], key_mask=s["mask"], scale=s["scale"])
        return (y.detach(),) + torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["g"]) if case["train"] else y
    if case["op"] == "drop":
        y = nn_ops.dropout(s["x"], case["p"], key=s["key"], residual=s["residual"])
        leaves = (s["x"],) if s["residual"] is None else (s["x"], s["residual"])
        return (y.detach(),) + torch.autograd.grad(y, leaves, s["g"]) if case["train"] else y
    y = nn_ops.embedding(s["idx"], s["w"], scale=s["scale"], dtype=TYPES[case["out"]])
    return (y.detach(),) + torch.autograd.grad(y, (s["w"],), s["g"]) if case["train"] else y


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------------------------------------

def _exact_attend(s):
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    B, Nq, H, D = q.shape
    G = H // k.shape[2]
    g = s["g"] if s["case"]["train"] else None
    O, dQ = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dK, dV = torch.zeros(k.shape, dtype=torch.float64, device=q.device), torch.zeros(k.shape, dtype=torch.float64, device=q.device)
    for b in range(B):
        at = torch.arange(k.shape[1], device=q.device)
        if s["lens"] is not None:
            at = at[: int(s["lens"][b])]
        if s["mask"] is not None:
            at = at[s["mask"][b][at]]
        if not len(at):
            continue
        for h in range(H):
            Q, K, V = q[b, :, h].double(), k[b, at, h // G].double(), v[b, at, h // G].double()
            S = Q.mm(K.t()) * s["scale"]
            E = torch.exp(S - S.max(1, keepdim=True)[0])
            P = E / E.sum(1, keepdim=True)
            O[b, :, h] = P.mm(V)
            if g is not None:
                Y = g[b, :, h].double()
                dP = Y.mm(V.t())
                dS = P * (dP - (P * dP).sum(1, keepdim=True)) * s["scale"]
                dQ[b, :, h] = dS.mm(K)
                dK[b].index_put_((at, torch.tensor(h // G, device=q.device)), dS.t().mm(Q), accumulate=True)
                dV[b].index_put_((at, torch.tensor(h // G, device=q.device)), P.t().mm(Y), accumulate=True)
    return O if g is None else (O, dQ, dK, dV)


def _exact_drop(s):
    n, t = s["case"]["n"], int(round(65536 * s["case"]["p"]))
    seed, stream = (int(x) for x in s["key"].cpu())
    u32 = np.uint64(0xFFFFFFFF)
    block = np.arange(-(-n // 8), dtype=np.uint64)
    c = [block & u32, block >> np.uint64(32), np.full_like(block, stream & 0xFFFFFFFF), np.full_like(block, stream >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        x, y = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(y >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), y & u32, (x >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), x & u32]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    u16 = np.stack(c, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    factor = torch.from_numpy(np.where(u16 < t, 0.0, 65536.0 / (65536 - t))).to(DEV)
    y = s["x"].detach().double() * factor
    if s["residual"] is not None:
        y = y + s["residual"].detach().double()
    if not s["case"]["train"]:
        return y
    dx = s["g"].double() * factor
    return (y, dx) if s["residual"] is None else (y, dx, s["g"].double())


def _exact_embed(s):
    idx, w = s["idx"], s["w"].detach()
    y = w.index_select(0, idx).double() * s["scale"]
    if not s["case"]["train"]:
        return y
    V, D = w.shape
    at = torch.sort(idx, stable=True)
    run_ = torch.cat((torch.zeros(1, D, dtype=torch.float64, device=w.device), s["g"].double()[at.indices].cumsum(0)))
    edge = torch.searchsorted(at.values, torch.arange(V + 1, device=w.device))
    return y, (run_[edge[1:]] - run_[edge[:-1]]) * s["scale"]


def exact(case, seed):
    if case["op"] == "attend" and case["B"] * case["H"] > 20000:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_attend(s) if case["op"] == "attend" else _exact_drop(s) if case["op"] == "drop" else _exact_embed(s)


# ---- the work a pass cannot do without -----------------------------------------------------------------------------------------------------

def work(case):
    size = {"bf16": 2, "fp32": 4}
    if case["op"] == "attend":
        B, Nq, Nk, H, Hk, D = (case[n] for n in ("B", "Nq", "Nk", "H", "Hk", "D"))
        keys = sum(_lens(case)) * (0.9 if case["mask"] else 1.0)
        rows, kv = 2 * B * Nq * H * D, 2 * keys * Hk * D            # bytes of one query-sided and one key-sided tensor
        flops = 4.0 * Nq * H * D * keys
        if not case["train"]:
            return {"bytes": 2 * rows + 2 * kv, "flops": flops}
        return {"bytes": 4 * rows + 2 * kv + 2 * 2 * B * Nk * Hk * D, "flops": 3.5 * flops}      # q, g in; O, dq, dk, dv out; seven products
    if case["op"] == "drop":
        n, a, r = case["n"], size[case["type"]], size[case["residual"] or case["type"]]
        b = a + r + (r if case["residual"] else 0) + (r + a if case["train"] else 0)
        return {"bytes": float(n * b), "flops": n * (4.0 if case["train"] else 2.0)}
    N, V, D = case["N"], case["V"], case["D"]
    seen = float((1.0 - (1.0 - _probabilities(case)) ** N).sum())
    b = 8 * N + seen * D * size[case["type"]] + N * D * size[case["out"]]
    if case["train"]:
        b += 8 * N + N * D * size[case["out"]] + V * D * size[case["type"]]
    return {"bytes": b, "flops": float(N * D * (2 if case["train"] else 1))}

"""Cases of the GPT training operators around the matrix products: the token + position embedding
with its gradient by sorted tokens, the per-head RMS norm of queries and keys with the rotary
position encoding in the same pass, and the global gradient norm with clipping over many tensors.

``listed()`` are the measured cases, ``draw(rng)`` gives more of the same ranges. ``run(state)`` is
one pass: with ``own`` false the operators' plain form (elementary torch operations in fp32), with
``own`` true the framework's kernels. ``exact(case, seed)`` is the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one generated token for each of 8 sequences: latency of a lookup, positions given
        dict(name="embed forward 8 tokens", op="embed", train=False, b=8, s=1, v=50304, e=1280,
             pos="given", scale=1.0, dtype="bf16"),
        # forward of a GPT-2-medium micro-batch (the transformer benchmark's 32 x 1024 tokens)
        dict(name="embed forward 32x1024", op="embed", train=False, b=32, s=1024, v=50304, e=1024,
             pos="rows", scale=1.0, dtype="bf16"),
        # the "tiny" preset in fp32: a debugging run's embedding with all its gradients
        dict(name="embed train tiny fp32", op="embed", train=True, b=2, s=128, v=512, e=128,
             pos="rows", scale=1.0, dtype="fp32"),
        # GPT-2-medium training micro-batch: lookup, token gradient [V, E], position gradient
        dict(name="embed train 32x1024", op="embed", train=True, b=32, s=1024, v=50304, e=1024,
             pos="rows", scale=1.0, dtype="bf16"),
        # GPT-2-xl width, unpadded vocabulary, ragged length, scaled rows, no learned positions
        dict(name="embed train 31x2047 xl fp16", op="embed", train=True, b=31, s=2047, v=50257,
             e=1600, pos="none", scale=40.0, dtype="fp16"),
        # one generated token for each of 16 sequences at its own position
        dict(name="qk forward 16 tokens", op="qk", train=False, b=16, s=1, h=20, hk=20, d=64,
             rot=16, pos="given", dtype="bf16"),
        # a long prompt, grouped K/V heads, full rotation, a length that ends inside a tile
        dict(name="qk forward 1x8191 grouped", op="qk", train=False, b=1, s=8191, h=32, hk=8, d=128,
             rot=128, pos="rows", dtype="bf16"),
        # the "tiny" preset with a quarter of each head rotated
        dict(name="qk train tiny fp32", op="qk", train=True, b=2, s=128, h=2, hk=2, d=64, rot=16,
             pos="rows", dtype="fp32"),
        # GPT-2-large width, a training micro-batch of 32 x 1024 tokens
        dict(name="qk train 32x1024 large", op="qk", train=True, b=32, s=1024, h=20, hk=20, d=64,
             rot=16, pos="rows", dtype="bf16"),
        # the "tiny" preset's gradients, clipped: latency over 28 small tensors
        dict(name="clip tiny fp32", op="clip", clip=True, kind="gpt", layers=2, width=128, vocab=512,
             seq=128, dtype="fp32"),
        # norm alone (monitoring) over convolution-sized tensors, odd sizes and alignments
        dict(name="norm 161 odd tensors", op="clip", clip=False, kind="odd", tensors=161,
             numel=25557032, dtype="fp16"),
        # GPT-2-large: bf16 matrices with fp32 LayerNorm gradients, 774M elements, clipped
        dict(name="clip gpt2-large", op="clip", clip=True, kind="gpt", layers=36, width=1280,
             vocab=50304, seq=1024, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "qk", "qk", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embed":
        s = _log(rng, 1, 2048)
        b = max(1, min(64, _log(rng, 1, 65536) // s))
        e = rng.choice([rng.randrange(64, 1601), 8 * rng.randrange(8, 201), 64 * rng.randrange(1, 26)])
        return dict(op=op, train=rng.random() < 0.6, b=b, s=s, v=_log(rng, 300, 50304), e=e,
                    pos=rng.choice(["none", "rows", "given"]), scale=rng.choice([1.0, 1.0, math.sqrt(e)]),
                    dtype=dtype)
    if op == "qk":
        d = rng.choice([64, 64, 128, 128, 80, 96, 256])
        hk = rng.choice([1, 2, 3, 4, 8])
        h = hk * rng.choice([1, 1, 2, 4, 5])
        s = _log(rng, 1, 16384)
        b = max(1, min(64, _log(rng, 1, 65536) // s))
        rot = rng.choice([d, d, d // 2, d // 4, 0])
        pos = rng.choice(["rows", "given"]) if rot else "rows"
        return dict(op=op, train=rng.random() < 0.6, b=b, s=s, h=h, hk=hk, d=d, rot=rot, pos=pos,
                    dtype=dtype)
    if rng.random() < 0.4:
        return dict(op=op, clip=rng.random() < 0.7, kind="gpt", layers=rng.randrange(1, 25),
                    width=64 * rng.randrange(1, 21), vocab=_log(rng, 512, 50304), seq=_log(rng, 64, 2048),
                    dtype=dtype)
    tensors = _log(rng, 1, 700)
    return dict(op=op, clip=rng.random() < 0.7, kind="odd", tensors=tensors,
                numel=tensors * _log(rng, 1, 200000) + rng.randrange(1000), dtype=dtype)


# ------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _zipf(v):
    """Cumulative token probabilities of a language-like distribution, p ~ 1 / (rank + 2.7)."""
    p = 1.0 / (torch.arange(v, dtype=torch.float64) + 2.7)
    return (p / p.sum()).cumsum(0)


def _sizes(c):
    """[(shape, is it a matrix)] of a gradient list."""
    if c["kind"] == "gpt":
        w = c["width"]
        one = [((w,), 0), ((w,), 0), ((3 * w, w), 1), ((3 * w,), 1), ((w, w), 1), ((w,), 1),
               ((w,), 0), ((w,), 0), ((4 * w, w), 1), ((4 * w,), 1), ((w, 4 * w), 1), ((w,), 1)]
        return [((c["vocab"], w), 1), ((c["seq"], w), 1)] + one * c["layers"] + [((w,), 0), ((w,), 0)]
    # `tensors` sizes spread over four decades that sum to `numel`, the last one ragged
    n, total = c["tensors"], c["numel"]
    share = [10.0 ** (4.0 * ((i * 61) % n) / n) for i in range(n)]
    got = [max(1, int(total * x / sum(share))) | 1 for x in share[1:]]
    return [((x,), 1) for x in got + [max(1, total - sum(got))]]


def _flat(sizes, dtype, g):
    """Gradients as a backward pass leaves them, in one allocation, views of it, and its copy."""
    n = [math.prod(s) for s in sizes]
    kept = torch.randn(sum(n), generator=g, device=DEV, dtype=torch.float32).mul_(0.01).to(dtype)
    flat = kept.clone()
    views = [x.view(s) for x, s in zip(flat.split(n), sizes)]
    return kept, flat, views


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = DTYPES[c["dtype"]]
    if c["op"] == "embed":
        b, s, v, e = c["b"], c["s"], c["v"], c["e"]
        u = torch.rand(b * s, generator=g, device=DEV, dtype=torch.float64)
        idx = torch.searchsorted(_zipf(v).to(DEV), u).clamp_(max=v - 1).view(b, s)
        st = dict(c=c, idx=idx, w=(torch.randn(v, e, generator=g, device=DEV) * 0.02).to(dt), p=None, pos=None)
        if c["pos"] != "none":
            p = s if c["pos"] == "rows" else max(1024, s)
            st["p"] = (torch.randn(p, e, generator=g, device=DEV) * 0.02).to(dt)
            if c["pos"] == "given":
                st["pos"] = torch.randint(0, p, (b, s), generator=g, device=DEV)
        if c["train"]:
            st["dy"] = torch.randn(b, s, e, generator=g, device=DEV).to(dt)
            st["w"].requires_grad_(True)
            if st["p"] is not None:
                st["p"].requires_grad_(True)
        return st
    if c["op"] == "qk":
        b, s, h, hk, d = c["b"], c["s"], c["h"], c["hk"], c["d"]
        # the fused projection's output: queries, keys and values of a token side by side
        qkv = torch.randn(b, s, h + 2 * hk, d, generator=g, device=DEV).to(dt)
        st = dict(c=c, qkv=qkv, wq=1 + 0.1 * torch.randn(d, generator=g, device=DEV),
                  wk=1 + 0.1 * torch.randn(d, generator=g, device=DEV), cos=None, sin=None, pos=None)
        if c["rot"]:
            rows = s if c["pos"] == "rows" else max(4096, s)
            inv = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])
            ang = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv
            st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
            if c["pos"] == "given":
                st["pos"] = torch.randint(0, rows, (b, s), generator=g, device=DEV)
        if c["train"]:
            st["dq"] = torch.randn(b, s, h, d, generator=g, device=DEV).to(dt)
            st["dk"] = torch.randn(b, s, hk, d, generator=g, device=DEV).to(dt)
        return st
    sizes = _sizes(c)
    low = [s for s, m in sizes if m]
    norms = [s for s, m in sizes if not m]
    st = dict(c=c)
    st["kept"], st["flat"], views = _flat(low, dt, g)
    st["kept32"], st["flat32"], views32 = _flat(norms, torch.float32, g) if norms else (None, None, [])
    rest, rest32 = iter(views), iter(views32)
    st["params"] = []
    for _, matrix in sizes:
        grad = next(rest if matrix else rest32)
        st["params"].append(torch.nn.Parameter(torch.empty_like(grad)))
        st["params"][-1].grad = grad
    st["max_norm"] = 1.0
    return st


# ------------------------------------------------------------------------------------- one pass
def run(st):
    op = st["c"]["op"]
    if op == "embed":
        return _embed_own(st) if own else _embed_plain(st)
    if op == "qk":
        return _qk_own(st) if own else _qk_plain(st)
    return _clip(st)


def _embed_own(st):
    from determined_clone_amd.ops.embedding import embedding

    c = st["c"]
    out = embedding(st["idx"], st["w"], pos_weight=st["p"], positions=st["pos"], scale=c["scale"])
    if not c["train"]:
        return {"out": out}
    leaves = [st["w"]] + ([st["p"]] if st["p"] is not None else [])
    grads = torch.autograd.grad(out, leaves, st["dy"])
    return dict(zip(("out", "dw", "dp"), (out.detach(),) + grads))


@torch.no_grad()
def _embed_plain(st):
    c, idx, w, p = st["c"], st["idx"], st["w"], st["p"]
    out = w[idx].float() * c["scale"]
    if p is not None:
        out = out + (p[st["pos"]] if st["pos"] is not None else p[:idx.shape[1]]).float()
    r = {"out": out.to(w.dtype)}
    if not c["train"]:
        return r
    dy = st["dy"].float()
    rows = (dy * c["scale"]).view(-1, w.shape[1])
    r["dw"] = torch.zeros(w.shape, device=w.device).index_add_(0, idx.view(-1), rows).to(w.dtype)
    if p is not None:
        if st["pos"] is None:
            dp = dy.sum(0)
        else:
            dp = torch.zeros(p.shape, device=p.device).index_add_(0, st["pos"].view(-1), dy.view(-1, p.shape[1]))
        r["dp"] = dp.to(p.dtype)
    return r


def _qk_own(st):
    from determined_clone_amd.ops.qk_norm import qk_norm_rope

    c = st["c"]
    h, hk = c["h"], c["hk"]
    q, k = st["qkv"][:, :, :h], st["qkv"][:, :, h:h + hk]
    wq, wk = st["wq"], st["wk"]
    if not c["train"]:
        q, k = qk_norm_rope(q, k, wq, wk, st["cos"], st["sin"], rot_dim=c["rot"], positions=st["pos"], eps=EPS)
        return {"q": q, "k": k}
    x = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    q, k = qk_norm_rope(*x, st["cos"], st["sin"], rot_dim=c["rot"], positions=st["pos"], eps=EPS)
    grads = torch.autograd.grad((q, k), x, (st["dq"], st["dk"]))
    return dict(zip(("q", "k", "dq", "dk", "dwq", "dwk"), (q.detach(), k.detach()) + grads))


def _turn(x, cos, sin, rot):
    """Rotates the first `rot` features of each head in pairs (i, i + rot / 2)."""
    if not rot:
        return x
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rot:]), -1)


def _tables(st, dtype):
    if st["cos"] is None:
        return None, None
    at = st["pos"] if st["pos"] is not None else slice(0, st["c"]["s"])
    return tuple(t[at].to(dtype)[..., None, :] for t in (st["cos"], st["sin"]))


@torch.no_grad()
def _qk_plain(st):
    c = st["c"]
    rot, h, hk = c["rot"], c["h"], c["hk"]
    cos, sin = _tables(st, torch.float32)

    def forward(x, w):
        x = x.float()
        n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        return _turn(n * w, cos, sin, rot)

    def backward(x, w, dy):
        x, dy = x.float(), dy.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        g = _turn(dy, cos, -sin if rot else None, rot)
        n = x * r
        dw = (g * n).flatten(0, 2).sum(0)
        g = g * w
        return (r * (g - n * (g * n).mean(-1, keepdim=True))), dw

    dt = st["qkv"].dtype
    q, k = st["qkv"][:, :, :h], st["qkv"][:, :, h:h + hk]
    r = {"q": forward(q, st["wq"]).to(dt), "k": forward(k, st["wk"]).to(dt)}
    if c["train"]:
        dq, r["dwq"] = backward(q, st["wq"], st["dq"])
        dk, r["dwk"] = backward(k, st["wk"], st["dk"])
        r["dq"], r["dk"] = dq.to(dt), dk.to(dt)
    return r


@torch.no_grad()
def _clip(st):
    params = st["params"]
    if st["c"]["clip"]:
        # a training step's backward pass writes its gradients anew before each clipping
        st["flat"].copy_(st["kept"])
        if st["flat32"] is not None:
            st["flat32"].copy_(st["kept32"])
    if own:
        from determined_clone_amd.ops import optim

        if not st["c"]["clip"]:
            return {"norm": optim.grad_norm([p.grad for p in params])}
        norm = optim.clip_grad_norm_(params, st["max_norm"])
    else:
        grads = [p.grad for p in params]
        norm = torch.stack([(g.float() * g.float()).sum() for g in grads]).sum().sqrt()
        if not st["c"]["clip"]:
            return {"norm": norm}
        coef = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        [g.copy_(g.float() * coef) for g in grads]
    r = {"norm": norm, "grads": st["flat"]}
    if st["flat32"] is not None:
        r["grads32"] = st["flat32"]
    return r


# ------------------------------------------------------------------------------------- 64 bits
@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    c = case
    f8 = torch.float64
    if c["op"] == "embed":
        ids = st["idx"].flatten()
        out = st["w"].detach().to(f8).index_select(0, ids).mul_(c["scale"])
        where = None
        if st["p"] is not None:
            where = st["pos"].flatten() if st["pos"] is not None else \
                torch.arange(c["s"], device=DEV).repeat(c["b"])
            out += st["p"].detach().to(f8).index_select(0, where)
        r = {"out": out.view(c["b"], c["s"], c["e"])}
        if c["train"]:
            dy = st["dy"].to(f8).flatten(0, 1)
            for name, table, i, f in (("dw", st["w"], ids, c["scale"]), ("dp", st["p"], where, 1.0)):
                if table is not None:
                    # running sums of the rows in token order: a token's gradient is a difference
                    order = i.argsort()
                    sums = torch.cat((torch.zeros(1, c["e"], dtype=f8, device=DEV), (dy[order] * f).cumsum(0)))
                    end = torch.bincount(i, minlength=table.shape[0]).cumsum(0)
                    d = sums[end]
                    d[1:] -= sums[end[:-1]]
                    r[name] = d
        return r
    if c["op"] == "qk":
        rot, h, hk, d = c["rot"], c["h"], c["hk"], c["d"]
        half = rot // 2
        turn = None
        if rot:  # pairs as complex numbers
            at = st["pos"] if st["pos"] is not None else torch.arange(c["s"], device=DEV)
            turn = torch.complex(st["cos"].to(f8)[at], st["sin"].to(f8)[at]).unsqueeze(-2)

        def rotate(x, by):
            if by is None:
                return x
            z = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * by
            return torch.cat((z.real, z.imag, x[..., rot:]), -1)

        r = {}
        for name, lo, n in (("q", 0, h), ("k", h, hk)):
            x, w = st["qkv"][:, :, lo:lo + n].to(f8), st["w" + name].to(f8)
            inv = 1.0 / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()
            r[name] = rotate(x * inv * w, turn)
            if c["train"]:
                g = rotate(st["d" + name].to(f8), None if turn is None else turn.conj())
                r["dw" + name] = (g * x * inv).sum((0, 1, 2))
                gw = g * w
                r["d" + name] = inv * gw - x * inv.pow(3) * (gw * x).sum(-1, keepdim=True) / d
        return r
    kept = [t for t in (st["kept"], st["kept32"]) if t is not None]
    norm = sum(sum(torch.dot(x, x) for x in (y.to(f8) for y in t.split(1 << 26))) for t in kept).sqrt()
    if not c["clip"]:
        return {"norm": norm}
    scale = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    return dict(zip(("grads", "grads32"), [t.to(f8) * scale for t in kept]), norm=norm)


# ------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "embed":
        t, e = c["b"] * c["s"], c["e"]
        z = _zipf(c["v"])
        p = torch.diff(z, prepend=torch.zeros(1, dtype=z.dtype))
        used = float((1 - (1 - p) ** t).sum())  # rows of the table that are expected to be read
        rows = {"none": 0, "rows": c["s"], "given": max(1024, c["s"])}[c["pos"]]
        n = t * 8 * (2 if c["pos"] == "given" else 1) + (used + min(rows, t) + t) * e * size
        f = t * e * (2 if rows else 1)
        if c["train"]:
            n += (t + c["v"] + rows) * e * size
            f += t * e * (3 if rows else 2)
        return {"bytes": n, "flops": f}
    if c["op"] == "qk":
        heads = c["b"] * c["s"] * (c["h"] + c["hk"])
        table = c["s"] if c["pos"] == "rows" else min(c["b"] * c["s"], max(4096, c["s"]))
        n = heads * c["d"] * size * 2 + table * c["rot"] * 4 + 8 * c["d"] + \
            (8 * c["b"] * c["s"] if c["pos"] == "given" else 0)
        f = heads * (4 * c["d"] + 3 * c["rot"])
        if c["train"]:
            n += heads * c["d"] * size * 2 + 8 * c["d"]
            f += heads * (9 * c["d"] + 3 * c["rot"])
        return {"bytes": n, "flops": f}
    n = [(math.prod(s), size if m else 4) for s, m in _sizes(c)]
    elems, byte = sum(k for k, _ in n), sum(k * b for k, b in n)
    if not c["clip"]:
        return {"bytes": byte, "flops": 2 * elems}
    # gradients written by the backward pass (read the kept copy, write), then read, scaled, written
    return {"bytes": 4 * byte, "flops": 3 * elems}

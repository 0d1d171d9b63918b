"""Embedding HIP kernels against the formula in 64 bits (run on an MI355X).

Tolerances: a value is rounded once to its type (half a step, eps / 2 relative) after fp32
arithmetic, each operation of which is off by 2^-24 of the magnitudes that it adds."""
import pytest
import torch

from determined_clone_amd.ops import _ext, _grad
from determined_clone_amd.ops.embedding import embedding

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):  # half the spacing of the subnormal numbers
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _close(got, want, magnitude, steps, what=""):
    """|got - want| <= half a step of want + `steps` fp32 roundings of `magnitude`."""
    got64, wide = got.double(), steps * U * magnitude
    bound = (want.abs() + wide) * _half(got.dtype) + wide + _floor(got.dtype)
    off = (got64 - want).abs()
    assert torch.isfinite(got64).all(), what
    assert (off <= bound).all(), f"{what}: {(off / bound).max().item():.2f} times the bound"


def _inputs(b, s, v, e, dtype, seed=0, p=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.randint(0, v, (b, s), generator=g, device="cuda")
    w = torch.randn(v, e, generator=g, device="cuda").to(dtype)
    pw = None if p is None else torch.randn(p, e, generator=g, device="cuda").to(dtype)
    dy = torch.randn(b, s, e, generator=g, device="cuda").to(dtype)
    return idx, w, pw, dy


def _check_grad(dw, dy, idx, rows, scale=1.0, old=None, start=0):
    flat = idx.reshape(-1).long() - start
    ok = (flat >= 0) & (flat < rows)
    d = dy.reshape(-1, dy.shape[-1]).double()[ok]
    want = torch.zeros(rows, d.shape[1], dtype=torch.float64, device=dw.device).index_add_(0, flat[ok], d * scale)
    size = torch.zeros_like(want).index_add_(0, flat[ok], (d * scale).abs())
    n = int(torch.bincount(flat[ok], minlength=1).max()) if flat[ok].numel() else 0
    if old is not None:
        want, size = want + old.double(), size + old.double().abs()
    _close(dw, want, size, n + 2, "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,v,e", [(1, 1, 1, 1), (1, 1, 50304, 1024), (3, 7, 300, 65), (2, 129, 512, 128),
                                     (5, 33, 1000, 100), (1, 2047, 50257, 1600), (4, 512, 777, 2056)])
def test_forward_and_gradients(dtype, b, s, v, e):
    idx, w, p, dy = _inputs(b, s, v, e, dtype, p=s + 3)
    w.requires_grad_(True), p.requires_grad_(True)
    out = embedding(idx, w, p, scale=1.5)
    a, c = w.detach().double()[idx] * 1.5, p.detach().double()[:s]
    _close(out.detach(), a + c, a.abs() + c.abs(), 2, "forward")
    dw, dp = torch.autograd.grad(out, (w, p), dy)
    _check_grad(dw, dy, idx, v, 1.5)
    _check_grad(dp, dy, torch.arange(s, device="cuda").expand(b, s), s + 3)
    assert not dp[s:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("integer", [torch.int32, torch.int64])
def test_given_positions(dtype, integer):
    idx, w, p, dy = _inputs(4, 100, 300, 96, dtype, seed=1, p=50)
    pos = torch.randint(0, 50, (4, 100), device="cuda").to(integer)
    w.requires_grad_(True), p.requires_grad_(True)
    out = embedding(idx.to(integer), w, p, positions=pos)
    a, c = w.detach().double()[idx], p.detach().double()[pos.long()]
    _close(out.detach(), a + c, a.abs() + c.abs(), 2)
    dw, dp = torch.autograd.grad(out, (w, p), dy)
    _check_grad(dw, dy, idx, 300)
    _check_grad(dp, dy, pos, 50)
    row = embedding(idx, w, p, positions=pos[0])  # broadcast over the batch
    assert torch.equal(row[0], out[0])


# n around the borders of the single-launch form (128, 256), ranges and walks; below, table rows around
# the borders of the sort's owners (256) and counters (255, 1023 each)
@pytest.mark.parametrize("rows", [700, 5000])
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 128, 129, 256, 257, 1000, 4095, 4096, 4097, 8192, 12289, 16384, 65536, 65537, 70001])
def test_sorted_gradient_lengths(n, rows):
    idx, _, _, dy = _inputs(1, n, rows, 8, torch.float32, seed=n)
    dw = _ext.load().embed_grad(dy, idx, rows)
    _check_grad(dw, dy, idx, rows)


@pytest.mark.parametrize("e", [8, 1000])
@pytest.mark.parametrize("n", [200, 3000])
def test_few_ids_with_a_row(n, e):
    """Most ids belong to other shards, or to no table at all; the others are added to the old rows."""
    idx, _, _, dy = _inputs(1, n, 5000, e, torch.bfloat16, seed=n)
    idx[0, ::7] = -5
    acc = torch.randn(40, e, device="cuda").bfloat16()
    old = acc.clone()
    _ext.load().embed_grad(dy, idx, 40, 0.5, 100, acc)
    _check_grad(acc, dy, idx, 40, 0.5, old, start=100)
    idx.fill_(-1)
    assert not _ext.load().embed_grad(dy, idx, 40).any()


def test_a_wide_vocabulary():
    """More rows than 256 workgroups have counters for (1023 each)."""
    v = 400_000
    idx, _, _, dy = _inputs(1, 3000, v, 16, torch.float32, seed=11)
    idx[0, :200] = v - 1
    _check_grad(_ext.load().embed_grad(dy, idx, v), dy, idx, v)


@pytest.mark.parametrize("v", [1, 2, 255, 256, 257, 65279, 65280, 65281, 65537, 261888, 261889])
def test_sorted_gradient_table_sizes(v):
    idx, _, _, dy = _inputs(2, 5000, v, 8, torch.bfloat16, seed=v)
    idx[0, :3] = v - 1
    dw = _ext.load().embed_grad(dy, idx, v)
    _check_grad(dw, dy, idx, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e", [64, 333, 1600])
@pytest.mark.parametrize("kind", ["one", "two", "half", "zipf"])
def test_frequent_tokens(dtype, e, kind):
    """Tokens that cross many workgroups' ranges, next to ones that occur once."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n, v = 9001, 700
    idx = torch.randint(0, v, (1, n), generator=g, device="cuda")
    if kind == "one":
        idx.fill_(3)
    elif kind == "two":
        idx = idx % 2
    elif kind == "half":
        idx[:, ::2] = 350
    else:
        idx = (torch.rand(1, n, generator=g, device="cuda").pow(8) * v).long()
    dy = torch.randn(1, n, e, generator=g, device="cuda").to(dtype)
    dw = _ext.load().embed_grad(dy, idx, v, 0.5)
    _check_grad(dw, dy, idx, v, 0.5)
    assert torch.equal(dw, _ext.load().embed_grad(dy, idx, v, 0.5))  # the same to the bit


def test_mistaken_ids_give_nan_rows_and_no_gradient():
    idx, w, p, dy = _inputs(2, 6, 30, 16, torch.float32, p=8)
    pos = torch.arange(6, device="cuda").repeat(2, 1)
    idx[0, 1], idx[1, 5], idx[1, 0] = -1, 30, 2 ** 40
    pos[0, 3], pos[1, 3] = 8, -2 ** 35
    w.requires_grad_(True), p.requires_grad_(True)
    out = embedding(idx, w, p, positions=pos)
    bad = torch.zeros(2, 6, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 5] = bad[1, 0] = bad[0, 3] = bad[1, 3] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
    dw, dp = torch.autograd.grad(out, (w, p), dy)
    _check_grad(dw, dy, idx, 30)
    _check_grad(dp, dy, pos, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabulary_shards(dtype):
    idx, w, _, dy = _inputs(3, 500, 120, 40, dtype, seed=3)
    total = 0
    for s in range(0, 120, 30):
        shard = w[s:s + 30].clone().requires_grad_(True)
        out = embedding(idx, shard, vocab_start=s)
        mine = (idx >= s) & (idx < s + 30)
        assert torch.equal(out[mine], w[idx[mine]]) and not out[~mine].any()
        total = total + out
        dw, = torch.autograd.grad(out, shard, dy)
        _check_grad(dw, dy, idx, 30, start=s)
    assert torch.equal(total, w[idx])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_accumulates_into_persistent_grads(dtype):
    idx, w, p, dy = _inputs(2, 300, 90, 64, dtype, seed=4, p=400)
    idx[idx == 7] = 8  # token 7 does not occur
    params = [torch.nn.Parameter(w), torch.nn.Parameter(p)]
    for q in params:
        q._dca_direct_grad = True
        q.grad = torch.randn_like(q)
    old = [q.grad.clone() for q in params]
    out = embedding(idx, params[0], params[1], scale=2.0)
    out.backward(dy)
    _check_grad(params[0].grad, dy, idx, 90, 2.0, old[0])
    _check_grad(params[1].grad, dy, torch.arange(300, device="cuda").expand(2, 300), 400, 1.0, old[1])
    assert torch.equal(params[0].grad[7], old[0][7]) and torch.equal(params[1].grad[300:], old[1][300:])
    assert _grad.target(params[0]) is params[0].grad


def test_strided_tables_and_gradients():
    idx, w, p, dy = _inputs(2, 40, 50, 48, torch.bfloat16, seed=6, p=40)
    wide = torch.randn(50, 101, device="cuda").bfloat16()
    for table in (wide[:, 1:49], wide[:, 8:56], w.t().contiguous().t(), wide[::2, :48]):
        at = idx % table.shape[0]
        assert torch.equal(embedding(at, table), table[at])
    t = w.clone().requires_grad_(True)
    out = embedding(idx.t(), t)  # ids with strides
    assert torch.equal(out, w[idx.t()])
    dyt = torch.randn(40, 48, 2, device="cuda").bfloat16().transpose(1, 2)
    dw, = torch.autograd.grad(out, t, dyt)
    _check_grad(dw, dyt, idx.t(), 50)
    out = embedding(idx, t)
    dw, = torch.autograd.grad(out.sum(), t)  # a broadcast gradient
    _check_grad(dw, torch.ones_like(dy), idx, 50)


def test_far_offsets():
    """Rows whose offsets pass 32 bits: a table of 2.2 G elements, an output and a gradient row there."""
    v, e = 1_100_000, 2000
    w = torch.empty(v, e, device="cuda", dtype=torch.bfloat16)
    idx = torch.tensor([[v - 1, 0, v - 2, v - 1]], device="cuda")
    w[idx[0]] = torch.randn(4, e, device="cuda").bfloat16()
    assert torch.equal(embedding(idx, w), w[idx])
    dy = torch.randn(1, 4, e, device="cuda").bfloat16()
    dw = _ext.load().embed_grad(dy, idx, v)
    want = (dy[0, 0].double() + dy[0, 3].double())
    _close(dw[v - 1], want, dy[0, 0].double().abs() + dy[0, 3].double().abs(), 3)
    assert torch.equal(dw[v - 2], dy[0, 2]) and torch.equal(dw[0], dy[0, 1])


@pytest.mark.parametrize("n", [100, 1000])
@pytest.mark.parametrize("add", [False, True])
def test_a_table_of_many_rows(n, add):
    """More rows than one launch has waves for."""
    v, e = 2 ** 26 + 11, 8
    g = torch.Generator(device="cuda").manual_seed(n)
    idx = torch.randint(0, v, (1, n), generator=g, device="cuda")
    idx[0, :5] = torch.tensor([v - 1, 0, 2 ** 25, v - 1, v], device="cuda")  # the last one has no row
    dy = torch.randn(1, n, e, generator=g, device="cuda").bfloat16()
    acc = torch.zeros(v, e, device="cuda", dtype=torch.bfloat16) if add else None
    dw = _ext.load().embed_grad(dy, idx, v, acc=acc)
    rows, where = idx[idx < v].unique(return_inverse=True)
    _check_grad(dw[rows], dy[:, idx[0] < v], where[None], len(rows))
    assert int(dw.any(1).sum()) == int(dw[rows].any(1).sum())


def test_many_ids():
    """More workgroups than one launch takes (2^29 ids of a long axis)."""
    n, v = 2 ** 29 + 100, 1000
    g = torch.Generator(device="cuda").manual_seed(0)
    idx = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
    idx[-50:] = 7
    dw = _ext.load().embed_grad(torch.ones(n, 1, device="cuda", dtype=torch.bfloat16), idx, v)
    counts = torch.bincount(idx, minlength=v)
    assert int(counts.max()) < 2 ** 24  # so that the fp32 sums of ones are exact
    assert torch.equal(dw[:, 0], counts.float().bfloat16())


def test_captured_graph_replays():
    idx, w, p, dy = _inputs(4, 2500, 400, 64, torch.bfloat16, seed=8, p=2500)
    C = _ext.load()

    def step():
        return (C.embed_fwd(idx, w, p), C.embed_grad(dy, idx, 400), C.embed_pos_grad(dy, 2500))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        idx.copy_((idx + k) % 400)
        want = [t.clone() for t in step()]
        dy.mul_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), k


def test_on_a_side_stream_and_two_calls_at_once():
    idx, w, _, dy = _inputs(4, 3000, 400, 128, torch.bfloat16, seed=9)
    C = _ext.load()
    want = C.embed_grad(dy, idx, 400)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(C.embed_grad(dy, idx, 400))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got)


def test_float64_tables_take_plain_torch():
    idx, w, p, _ = _inputs(2, 6, 30, 16, torch.float32, p=8)
    torch.testing.assert_close(embedding(idx, w.double(), p.double(), scale=2.0), 2 * w.double()[idx] + p.double()[:6])


def test_transforms_and_forward_mode_take_plain_torch():
    idx, w, p, dy = _inputs(3, 6, 30, 16, torch.float32, p=8)
    t = torch.randn_like(w)
    want = w[idx] * 2.0 + p[:6]
    run = lambda i, a: embedding(i, a, p, scale=2.0)  # noqa: E731
    assert torch.equal(torch.vmap(run, (0, None))(idx, w), want)
    for out, tangent in (torch.func.jvp(lambda a: run(idx, a), (w,), (t,)), _dual(lambda a: run(idx, a), w, t)):
        assert torch.equal(out, want) and torch.equal(tangent, t[idx] * 2.0)
    torch.testing.assert_close(torch.func.grad(lambda a: (run(idx, a) * dy).sum())(w),
                               _ext.load().embed_grad(dy, idx, 30, 2.0), rtol=1e-5, atol=1e-5)
    shard = torch.vmap(lambda i: embedding(i, w[:10], vocab_start=0))(idx)
    assert torch.equal(shard, embedding(idx, w[:10], vocab_start=0))


def _dual(f, x, t):
    import torch.autograd.forward_ad as fw

    with fw.dual_level():
        return tuple(fw.unpack_dual(f(fw.make_dual(x, t))))


def test_refusals():
    w = torch.randn(5, 4, device="cuda")
    idx = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="idx on"):
        embedding(idx.cpu(), w)
    with pytest.raises(ValueError, match="positions on"):
        embedding(idx, w, w, positions=idx.cpu())
    with pytest.raises(RuntimeError, match="must be"):
        _ext.load().embed_grad(torch.zeros(2, 2, 4, device="cuda"), idx, 5)
    with pytest.raises(RuntimeError, match="accumulation target"):
        _ext.load().embed_grad(torch.zeros(2, 3, 4, device="cuda"), idx, 5, acc=torch.zeros(4, 4, device="cuda"))
    t = w.clone().requires_grad_(True)
    g, = torch.autograd.grad(embedding(idx, t).sum(), t, create_graph=True)
    assert g.shape == t.shape
    with pytest.raises(RuntimeError):
        g.sum().backward()  # no second derivatives
    dy = torch.randn(2, 3, 4, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(embedding(idx, t), t, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        (g.sum() + dy.sum()).backward()

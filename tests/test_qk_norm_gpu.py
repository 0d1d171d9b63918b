"""Query / key norm + rotary HIP kernels against the formula in 64 bits (run on an MI355X).

Tolerances: one rounding to the type (eps / 2 relative) after fp32 arithmetic. The sum of D squares
is off by at most D 2^-24 relative (all terms positive), its root by half of that; every other
operation by 2^-24 of the magnitudes that it combines."""
import pytest
import torch

from determined_clone_amd.ops import _ext
from determined_clone_amd.ops import transformer as T
from determined_clone_amd.ops.qk_norm import qk_norm_attention_qkvpacked, qk_norm_rope

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def _close(got, want, wide, what):
    """|got - want| <= `wide` + half a step of the result."""
    got64, info = got.double(), torch.finfo(got.dtype)
    bound = (want.abs() + wide) * info.eps / 2 + wide + info.smallest_normal * info.eps / 2
    assert torch.isfinite(got64).all(), what
    off = (got64 - want).abs()
    assert (off <= bound).all(), f"{what}: {(off / bound).max().item():.2f} times the bound"


def _turn(x, cos, sin, rot):
    h = rot // 2
    a, b = x[..., :h], x[..., h:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _turn_size(x, cos, sin, rot):
    h = rot // 2
    a, b, c, s = x[..., :h].abs(), x[..., h:rot].abs(), cos.abs(), sin.abs()
    return torch.cat([a * c + b * s, b * c + a * s, x[..., rot:].abs()], -1)


def _check(x, w, dy, cos, sin, rot, pos, eps, y, dx, dw):
    D = x.shape[-1]
    x, dy = x.detach().double(), dy.double()
    wd = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    c = s = None
    if rot:
        at = pos.long() if pos is not None else torch.arange(x.shape[1], device=x.device)
        c, s = cos.double()[at].unsqueeze(-2), sin.double()[at].unsqueeze(-2)
    else:
        c = s = torch.zeros(0, dtype=torch.float64, device=x.device)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * r
    steps = D + 16
    _close(y, _turn(n * wd, c, s, rot), steps * U * _turn_size(n * wd, c, s, rot), "forward")
    g, gs = _turn(dy, c, -s, rot), _turn_size(dy, c, s, rot)
    m = (g * wd * n).mean(-1, keepdim=True)
    ms = (gs * wd.abs() * n.abs()).mean(-1, keepdim=True)
    _close(dx, r * (g * wd - n * m), 2 * steps * U * r * (gs * wd.abs() + n.abs() * ms), "dx")
    if dw is not None:
        rows = x.numel() // D
        size = (gs * n.abs()).sum((0, 1, 2))
        _close(dw, (g * n).sum((0, 1, 2)), (rows + steps) * U * size, "dw")


def _case(b, s, h, hk, d, rot, dtype, pos="rows", weight=True, seed=0, packed=True, w_dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if packed:
        qkv = torch.randn(b, s, h + 2 * hk, d, generator=g, device="cuda").to(dtype)
        q, k = qkv[:, :, :h], qkv[:, :, h:h + hk]
    else:
        q = torch.randn(b, s, h, d, generator=g, device="cuda").to(dtype)
        k = torch.randn(b, s, hk, d, generator=g, device="cuda").to(dtype)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    ws = [(torch.randn(d, generator=g, device="cuda") + 1).to(w_dtype).requires_grad_(True) if weight else None
          for _ in range(2)]
    rows = max(s, 1) + 40
    cos, sin = T.rope_tables(rows, rot, device="cuda") if rot else (None, None)
    p = None
    if pos != "rows":
        p = torch.randint(0, rows, (s,) if pos == "shared" else (b, s), generator=g, device="cuda")
        p = p.int() if pos == "int32" else p
    dy = [torch.randn(b, s, n, d, generator=g, device="cuda").to(dtype) for n in (h, hk)]
    y = qk_norm_rope(q, k, *ws, cos, sin, rot_dim=rot, positions=p, eps=1e-5)
    leaves = [q, k] + [w for w in ws if w is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    for i in range(2):
        _check((q, k)[i], ws[i], dy[i], cos, sin, rot, p, 1e-5, y[i].detach(), grads[i],
               grads[2 + i] if weight else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot", [(64, 16), (64, 64), (128, 128), (128, 32), (80, 20), (80, 40), (80, 80), (96, 24),
                                   (96, 0), (256, 256), (40, 10), (33, 8), (7, 6), (2, 2), (1, 0), (320, 64),
                                   (1024, 512), (1000, 250), (513, 2)])
def test_head_dims(dtype, d, rot):
    _case(2, 19, 3, 1, d, rot, dtype, seed=d + rot)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,h,hk", [(1, 1, 1, 1), (16, 1, 20, 20), (1, 1, 32, 8), (3, 129, 25, 5), (2, 1000, 16, 1),
                                      (1, 4099, 4, 4), (64, 65, 12, 12), (1, 9, 1, 7)])
def test_shapes(dtype, b, s, h, hk):
    _case(b, s, h, hk, 64, 32, dtype, pos="given", seed=s)


@pytest.mark.parametrize("pos", ["rows", "given", "shared", "int32"])
@pytest.mark.parametrize("weight", [True, False])
def test_positions_and_weights(pos, weight):
    _case(3, 50, 6, 2, 128, 64, torch.bfloat16, pos=pos, weight=weight, packed=False)


@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float16])
def test_low_precision_weights(w_dtype):
    _case(2, 30, 4, 4, 64, 64, torch.bfloat16, w_dtype=w_dtype)


@pytest.mark.parametrize("rot", [0, 32])
@pytest.mark.parametrize("trained", ["q", "k"])
@pytest.mark.parametrize("other", ["absent", "frozen"])
@pytest.mark.parametrize("persistent", [False, True])
def test_one_trained_weight(rot, trained, other, persistent):
    """The gradient of one weight, the other one absent or frozen, returned or added to ``.grad``."""
    g = torch.Generator(device="cuda").manual_seed(rot)
    q = torch.randn(2, 21, 4, 64, generator=g, device="cuda")
    k = torch.randn(2, 21, 2, 64, generator=g, device="cuda")
    dy = [torch.randn(x.shape, generator=g, device="cuda") for x in (q, k)]
    w = torch.nn.Parameter(torch.rand(64, generator=g, device="cuda") + 0.5)
    frozen = torch.rand(64, generator=g, device="cuda") + 0.5 if other == "frozen" else None
    cos, sin = T.rope_tables(21, rot, device="cuda") if rot else (None, None)
    which = "qk".index(trained)
    ws = (w, frozen) if which == 0 else (frozen, w)
    old = torch.randn(64, generator=g, device="cuda")
    if persistent:
        w._dca_direct_grad = True
        w.grad = old.clone()
    leaves = [x.requires_grad_(True) for x in (q, k)]
    y = qk_norm_rope(*leaves, *ws, cos, sin, rot_dim=rot, eps=1e-5)
    torch.autograd.backward(y, dy)
    for i in range(2):
        _check(leaves[i], ws[i], dy[i], cos, sin, rot, None, 1e-5, y[i].detach(), leaves[i].grad,
               None if i != which or persistent else w.grad)
    if persistent:
        plain = w.grad.double() - old.double()
        w.grad, w._dca_direct_grad = None, False
        torch.autograd.backward(qk_norm_rope(q.detach(), k.detach(), *ws, cos, sin, rot_dim=rot, eps=1e-5)[which],
                                dy[which])
        # the same sum with one more fp32 addition
        assert ((plain - w.grad.double()).abs() <= U * (old.double().abs() + w.grad.double().abs()) * 1.001).all()


def test_no_tokens_and_no_key_heads():
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.randn(2, 0, 4, 64, device="cuda", requires_grad=True)
    y, z = qk_norm_rope(q, q, w, w)
    dw, = torch.autograd.grad((y.sum() + z.sum()), w)
    assert y.shape == q.shape and not dw.any()
    x = torch.randn(2, 3, 4, 64, device="cuda")
    y, z = qk_norm_rope(x, x[:, :, :0], w, None)
    assert torch.equal(y, qk_norm_rope(x, x, w, w)[0]) and z.shape == (2, 3, 0, 64)


def test_zero_rows_and_large_values():
    """Rows of zeros give zeros (eps keeps the root away from 0); rows whose squares leave bf16's and
    fp16's range do not overflow in fp32."""
    x = torch.zeros(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 1] = 1e15
    x[0, 2] = 1e-15
    x[0, 3, 0, 5] = 3.0
    y, _ = qk_norm_rope(x, x, eps=1e-6)
    assert not y[0, 0].any()
    torch.testing.assert_close(y[0, 1].float(), torch.ones(2, 64, device="cuda"), rtol=2 ** -8, atol=0)
    torch.testing.assert_close(y[0, 2].double(), x[0, 2].double() * 1e3, rtol=2 ** -7, atol=0)
    assert y[0, 3, 0, 5] == 8.0 and y[0, 3].float().abs().sum() == 8.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 33])
def test_tiny_rows_without_an_eps(dtype, d):
    """Mean squares below 2^-126. A square there is off by up to 2^-150, here 2^-23 of the mean square at
    most, its root by half of that: one of the steps that the bounds count."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = [(torch.rand(2, 9, 2, d, generator=g, device="cuda") * 0.2 + 0.9).mul(0.9e-19).to(dtype).requires_grad_(True)
         for _ in range(2)]
    w = [(torch.rand(d, generator=g, device="cuda") + 0.5).requires_grad_(True) for _ in range(2)]
    dy = [torch.randn(2, 9, 2, d, generator=g, device="cuda").to(dtype) for _ in range(2)]
    assert x[0].double().square().mean(-1).max() < 2.0 ** -126 and x[0].double().square().mean(-1).min() > 2.0 ** -127
    y = qk_norm_rope(*x, *w, eps=0.0)
    grads = torch.autograd.grad(y, x + w, dy)
    for i in range(2):
        _check(x[i], w[i], dy[i], None, None, 0, None, 0.0, y[i].detach(), grads[i], grads[2 + i])
    assert torch.isnan(qk_norm_rope(torch.zeros_like(x[0]), x[1], eps=0.0)[0]).all()  # 0 / 0


def test_strides():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 4, 30, 64, generator=g, device="cuda").bfloat16()  # [B, H, S, D]
    w = torch.rand(64, generator=g, device="cuda") + 0.5
    cos, sin = T.rope_tables(30, 64, device="cuda")
    t = x.transpose(1, 2)
    want = qk_norm_rope(t.contiguous(), t.contiguous(), w, w, cos, sin)
    got = qk_norm_rope(t, t, w, w, cos, sin)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.randn(2, 30, 4, 67, generator=g, device="cuda").bfloat16()[..., 1:65]  # unaligned rows
    want = qk_norm_rope(odd.contiguous(), odd.contiguous(), w, w, cos, sin)
    got = qk_norm_rope(odd, odd.contiguous(), w, w, cos, sin)
    # the two take different lane layouts: their fp32 results may differ by (64 + 16) roundings of
    # values up to 8, which can move the bf16 result by a step
    for a, b in zip(got, want):
        torch.testing.assert_close(a.float(), b.float(), rtol=2 ** -7, atol=80 * U * 8)
    last = torch.randn(2, 30, 64, 4, generator=g, device="cuda").bfloat16().transpose(2, 3)  # D not contiguous
    assert torch.equal(qk_norm_rope(last, last, w)[0], qk_norm_rope(last.contiguous(), last.contiguous(), w)[0])
    one = torch.randn(1, 30, 1, 64, generator=g, device="cuda").bfloat16().expand(3, 30, 4, 64)  # broadcast input
    one = one.detach().requires_grad_(True)
    dq, = torch.autograd.grad(qk_norm_rope(one, one, w)[0].sum(), one)
    assert dq.shape == one.shape and torch.equal(dq[0, :, 0], dq[2, :, 3])


def test_mistaken_positions_give_nan_in_the_rotated_part():
    q = torch.randn(1, 4, 2, 64, device="cuda")
    cos, sin = T.rope_tables(8, 16, device="cuda")
    pos = torch.tensor([0, 8, -1, 2 ** 40], device="cuda")
    y, _ = qk_norm_rope(q, q, None, None, cos, sin, rot_dim=16, positions=pos)
    assert torch.isfinite(y[0, 0]).all() and torch.isfinite(y[..., 16:]).all()
    assert torch.isnan(y[0, 1:, :, :16]).all()


def test_nan_and_infinity_stay_in_their_row():
    q = torch.randn(1, 3, 2, 64, device="cuda")
    want, _ = qk_norm_rope(q, q)
    q[0, 1, 0, 3], q[0, 2, 1, 0] = float("nan"), float("inf")
    y, _ = qk_norm_rope(q, q)
    good = torch.ones(3, 2, dtype=torch.bool)
    good[1, 0] = good[2, 1] = False
    assert torch.equal(y[0][good], want[0][good]) and torch.isnan(y[0, 1, 0]).all() and torch.isnan(y[0, 2, 1, 0])


def test_far_offsets():
    """Rows past 2^31 elements."""
    x = torch.empty(1, 40_000, 900, 64, device="cuda", dtype=torch.bfloat16)
    x[0, -1] = torch.randn(900, 64, device="cuda").bfloat16()
    y, _ = qk_norm_rope(x, x[:, :, :0])
    assert torch.equal(y[:, -1:], qk_norm_rope(x[:, -1:], x[:, -1:, :0])[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_accumulates_into_persistent_grads(dtype):
    x = torch.randn(2, 33, 4, 64, device="cuda").bfloat16()
    g = torch.randn_like(x)
    ws = [torch.nn.Parameter(torch.rand(64, device="cuda").to(dtype) + 0.5) for _ in range(2)]
    plain = torch.autograd.grad(qk_norm_rope(x, x, *ws), ws, (g, g))
    for w in ws:
        w._dca_direct_grad = True
        w.grad = torch.ones_like(w)
    torch.autograd.backward(qk_norm_rope(x, x, *ws), (g, g))
    for w, p in zip(ws, plain):
        torch.testing.assert_close(w.grad, p + 1, rtol=2 * torch.finfo(dtype).eps, atol=torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed", [False, True])
def test_one_weight_for_queries_and_keys(dtype, packed):
    """Both of its gradients arrive in the one persistent ``.grad``, each addition rounded once to it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(2, 70, 3, 4, 64, generator=g, device="cuda").bfloat16()
    dy = torch.randn(2, 70, 4, 64, generator=g, device="cuda").bfloat16()
    w = torch.nn.Parameter((torch.rand(64, generator=g, device="cuda") + 0.5).to(dtype))

    def backward(wq, wk):
        if packed:
            qk_norm_attention_qkvpacked(qkv, wq, wk).backward(dy)
        else:
            torch.autograd.backward(qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], wq, wk), (dy, dy))

    parts = [w.detach().float().requires_grad_(True) for _ in range(2)]  # the two gradients by themselves
    backward(*parts)
    a, b = (p.grad.double() for p in parts)
    w._dca_direct_grad = True
    w.grad = torch.randn(64, generator=g, device="cuda").to(dtype)
    old = w.grad.double()
    backward(w, w)
    # two additions in fp32 and their roundings to the type, half a step of each sum
    step = torch.finfo(dtype).eps / 2 + U
    first = old + a
    bound = step * (first.abs() + (first + b).abs()) * (1 + step) ** 2
    assert ((w.grad.double() - (first + b)).abs() <= bound).all()


@pytest.mark.parametrize("rot", [0, 16, 64])
def test_packed_attention(rot):
    """The fused function against its parts: the same kernels in the same order, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = torch.randn(2, 130, 3, 4, 64, generator=g, device="cuda").bfloat16().requires_grad_(True)
    ws = [(torch.rand(64, generator=g, device="cuda") + 0.5).requires_grad_(True) for _ in range(2)]
    cos, sin = T.rope_tables(130, rot, device="cuda") if rot else (None, None)
    lengths = torch.tensor([130, 77], device="cuda")
    do = torch.randn(2, 130, 4, 64, generator=g, device="cuda").bfloat16()
    o = qk_norm_attention_qkvpacked(qkv, *ws, cos, sin, rot_dim=rot, key_lengths=lengths)
    got = torch.autograd.grad(o, [qkv] + ws, do)
    q, k, v = qkv.unbind(2)
    q, k = qk_norm_rope(q, k, *ws, cos, sin, rot_dim=rot)
    p = T.flash_attention(q, k, v, key_lengths=lengths)
    want = torch.autograd.grad(p, [qkv] + ws, do)
    assert torch.equal(o, p)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("through", ["gradient", "input"])
def test_second_derivatives_are_refused(packed, through):
    """Gradients under ``create_graph`` have the right values; differentiating them raises, also when the
    incoming gradient is no part of a graph (a penalty on the gradients would lose its own)."""
    x = torch.randn(1, 30, 3, 2, 64, device="cuda").bfloat16().requires_grad_(True)
    w = (torch.rand(64, device="cuda") + 0.5).requires_grad_(True)
    dy = torch.randn(1, 30, 2, 64, device="cuda").bfloat16().requires_grad_(through == "gradient")

    def run():
        if packed:
            return qk_norm_attention_qkvpacked(x, w, None)
        return qk_norm_rope(x[:, :, 0], x[:, :, 1], w, None)[0]

    want = torch.autograd.grad(run(), (x, w), dy.detach())
    y = run()
    got = torch.autograd.grad(y, (x, w), dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="twice"):
        (y.float().sum() + got[0].float().square().sum()).backward()
    with pytest.raises(RuntimeError, match="twice"):
        got[1].sum().backward()


def test_captured_graph_replays():
    x = torch.randn(2, 65, 8, 64, device="cuda").bfloat16()
    g = torch.randn_like(x)
    w = torch.rand(64, device="cuda")
    cos, sin = T.rope_tables(65, 32, device="cuda")
    C = _ext.load()

    def step():
        y = C.qk_norm_rope(x, x, w, w, cos, sin, 32, None, 1e-6)
        return y + C.qk_norm_rope_bwd(g, g, x, x, w, w, cos, sin, 32, None, 1e-6, True, True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        x.copy_(x.roll(1, 0) * 1.5)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_refusals():
    q = torch.randn(1, 2, 2, 64, device="cuda")
    cos, sin = T.rope_tables(2, 64)
    with pytest.raises(ValueError, match="must be on"):
        qk_norm_rope(q, q, None, None, cos, sin)
    with pytest.raises(ValueError, match="weights"):
        qk_norm_rope(q, q, torch.ones(64))
    with pytest.raises(ValueError, match="GPU path"):
        qk_norm_rope(q.double(), q.double())
    with pytest.raises(ValueError, match="GPU path"):
        qk_norm_attention_qkvpacked(torch.randn(1, 2, 3, 2, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="table rows"):
        _ext.load().qk_norm_rope(q, q, None, None, cos.cuda()[:1], sin.cuda()[:1], 64, None, 1e-6)


def test_angle_tables_that_ask_for_gradients_are_refused():
    q = torch.randn(1, 2, 2, 64, device="cuda")
    cos, sin = T.rope_tables(2, 64, device="cuda")
    want = qk_norm_rope(q, q, None, None, cos, sin)[0]
    for i in range(2):
        tables = [t.clone().requires_grad_(i == j) for j, t in enumerate((cos, sin))]
        with pytest.raises(ValueError, match="no gradients for cos and sin"):
            qk_norm_rope(q, q, None, None, *tables)
        with pytest.raises(ValueError, match="no gradients for cos and sin"):
            qk_norm_attention_qkvpacked(torch.randn(1, 2, 3, 2, 64, device="cuda").bfloat16(), None, None, *tables)
        with torch.no_grad():
            assert torch.equal(qk_norm_rope(q, q, None, None, *tables)[0], want)


@pytest.mark.parametrize("b,s", [(0, 33), (2, 0)])
def test_packed_attention_without_tokens(b, s):
    """An empty output and zero weight gradients, and no failed launch left for the next call to report."""
    qkv = torch.randn(b, s, 3, 2, 64, device="cuda").bfloat16().requires_grad_(True)
    w = [torch.ones(64, device="cuda", requires_grad=True) for _ in range(2)]
    cos, sin = T.rope_tables(33, 64, device="cuda")
    out = qk_norm_attention_qkvpacked(qkv, *w, cos, sin, key_lengths=torch.ones(b, device="cuda", dtype=torch.long))
    assert out.shape == (b, s, 2, 64) and out.dtype == torch.bfloat16
    grads = torch.autograd.grad(out.float().sum(), [qkv] + w)
    assert grads[0].shape == qkv.shape and not any(g.any() for g in grads)
    assert torch.ones(5, device="cuda").sum() == 5


def test_gradients_with_mistaken_positions():
    """The mistake does not go unseen: NaN in its rows' gradients and in the weights' rotated features."""
    x = [torch.randn(1, 4, 2, 64, device="cuda", requires_grad=True) for _ in range(2)]
    w = [torch.ones(64, device="cuda", requires_grad=True) for _ in range(2)]
    cos, sin = T.rope_tables(8, 16, device="cuda")
    pos = torch.tensor([0, 8, 3, -1], device="cuda")
    y = qk_norm_rope(*x, *w, cos, sin, rot_dim=16, positions=pos)
    grads = torch.autograd.grad(y, x + w, [torch.randn(1, 4, 2, 64, device="cuda") for _ in range(2)])
    for dx, dw in zip(grads[:2], grads[2:]):
        assert torch.isnan(dx[0, [1, 3]]).all() and torch.isfinite(dx[0, [0, 2]]).all()
        assert torch.isnan(dw[:16]).all() and torch.isfinite(dw[16:]).all()

"""GPT with fused embeddings, query / key norms and clipping used together: against plain PyTorch on
the CPU, tensor parallel against dense, and on the GPU against the CPU model."""
import copy

import pytest
import torch
import torch.nn.functional as F
from test_tensor_parallel import _run

from determined_clone_amd.models import gpt2
from determined_clone_amd.models.gpt2_tp import TPGPT
from determined_clone_amd.ops import _grad
from determined_clone_amd.ops import optim as fopt
from determined_clone_amd.ops import transformer as T
from determined_clone_amd.parallel import tensor as tp


def _plain(model: gpt2.GPT, idx: torch.Tensor) -> torch.Tensor:
    """The network in plain PyTorch; query and key heads normed when the model norms them."""
    cfg = model.cfg
    B, S = idx.shape
    x = F.embedding(idx, model.wte.weight)
    if model.wpe is not None:
        x = x + model.wpe.weight[:S]
    for blk in model.blocks:
        h = F.layer_norm(x, (cfg.d_model,), blk.ln1.weight, blk.ln1.bias, cfg.ln_eps)
        q, k, v = F.linear(h, blk.attn.qkv.weight, blk.attn.qkv.bias).view(B, S, 3, cfg.n_head, cfg.head_dim).unbind(2)
        if cfg.qk_norm:
            q = F.rms_norm(q, (cfg.head_dim,), blk.attn.q_norm.weight, cfg.ln_eps)
            k = F.rms_norm(k, (cfg.head_dim,), blk.attn.k_norm.weight, cfg.ln_eps)
        if blk.attn.rot:
            q, k = (T.reference_rope(t, model.rope_cos, model.rope_sin, blk.attn.rot) for t in (q, k))
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
        x = x + F.linear(o.transpose(1, 2).reshape(B, S, -1), blk.attn.proj.weight, blk.attn.proj.bias)
        h = F.layer_norm(x, (cfg.d_model,), blk.ln2.weight, blk.ln2.bias, cfg.ln_eps)
        h = F.gelu(F.linear(h, blk.mlp.fc.weight, blk.mlp.fc.bias), approximate="tanh")
        x = x + F.linear(h, blk.mlp.proj.weight, blk.mlp.proj.bias)
    x = F.layer_norm(x, (cfg.d_model,), model.ln_f.weight, model.ln_f.bias, cfg.ln_eps)
    return F.linear(x, model.wte.weight)


def _model(pos, qk_norm=True, **kw):
    torch.manual_seed(0)
    m = gpt2.gpt2("tiny", pos_emb=pos, qk_norm=qk_norm, max_seq_len=160, **kw)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "_norm.weight" in n:
                p.uniform_(0.5, 1.5)
    return m


@pytest.mark.parametrize("pos", ["learned", "rotary"])
def test_qk_norm_model_and_gradients_match_plain(pos):
    m = _model(pos)
    assert {k for k in m.state_dict() if "_norm" in k} == {f"blocks.{i}.attn.{n}_norm.weight" for i in (0, 1) for n in "qk"}
    idx, tgt = torch.randint(0, 512, (2, 33)), torch.randint(0, 512, (2, 33))
    logits, loss = m(idx, tgt)
    want = _plain(m, idx)
    torch.testing.assert_close(logits, want, atol=1e-4, rtol=1e-4)
    got = torch.autograd.grad(loss, list(m.parameters()))
    ref = torch.autograd.grad(F.cross_entropy(want.flatten(0, 1), tgt.flatten()), list(m.parameters()))
    for (n, _), a, b in zip(m.named_parameters(), got, ref):
        torch.testing.assert_close(a, b, atol=1e-6, rtol=1e-3, msg=n)


def test_without_qk_norm_nothing_is_added():
    assert not any("_norm" in k for k in gpt2.gpt2("tiny").state_dict())
    m = gpt2.cast_for_mi355x(_model("rotary"))
    assert m.blocks[0].attn.q_norm.weight.dtype == torch.float32  # kept like LayerNorm's


def test_the_configs_earlier_fields_keep_their_places():
    from dataclasses import astuple, fields

    names = [f.name for f in fields(gpt2.GPTConfig)]
    old = [n for n in names if n != "qk_norm"]
    cfg = gpt2.GPTConfig(*astuple(gpt2.GPTConfig(extra={"a": 1}, pad_vocab_multiple=64))[:len(old)])
    assert old[-1] == "extra" and cfg.extra == {"a": 1} and cfg.pad_vocab_multiple == 64 and not cfg.qk_norm


def test_token_embedding_refuses_what_its_lookup_does_not_do():
    for kw in (dict(padding_idx=0), dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(ValueError, match="not supported"):
            gpt2.TokenEmbedding(4, 2, **kw)
        with pytest.raises(ValueError, match="not supported"):
            gpt2.TokenEmbedding.from_pretrained(torch.ones(4, 2), **kw)
    t = gpt2.TokenEmbedding(4, 2, device="cpu", dtype=torch.float64)
    assert t(torch.tensor([3])).dtype == torch.float64
    assert torch.equal(gpt2.TokenEmbedding.from_pretrained(torch.ones(4, 2))(torch.tensor([1])), torch.ones(1, 2))


@pytest.mark.parametrize("pos", ["learned", "rotary"])
def test_another_module_in_the_token_tables_place(pos):
    m = _model(pos, qk_norm=False)
    idx = torch.randint(0, 512, (2, 33))
    want, pipe = m(idx), gpt2.EmbeddingPipe(m.cfg)
    pipe.load_state_dict({k: v for k, v in m.state_dict().items() if k in pipe.state_dict()})
    first = pipe(idx)
    for module in (m, pipe):
        plain = torch.nn.Embedding(*module.wte.weight.shape)
        plain.load_state_dict(module.wte.state_dict())
        module.wte = plain
    torch.testing.assert_close(m(idx), want, rtol=0, atol=0)
    torch.testing.assert_close(pipe(idx), first, rtol=0, atol=0)


def test_tables_of_two_types_add_in_the_wider_one():
    pipe = gpt2.EmbeddingPipe(gpt2.config_for("tiny"))
    pipe.wte.bfloat16()
    idx = torch.randint(0, 512, (2, 33))
    want = pipe.wte.weight[idx].float() + pipe.wpe.weight[:33]
    torch.testing.assert_close(pipe(idx), want, rtol=0, atol=0)


def _tp_parity(rank, world, d, pos):
    torch.manual_seed(0)
    cfg = gpt2.config_for("tiny", n_layer=2, n_head=4, d_model=256, vocab_size=500, max_seq_len=32, pos_emb=pos,
                          qk_norm=True)
    full = gpt2.GPT(cfg)
    with torch.no_grad():
        for n, p in full.named_parameters():
            if "_norm.weight" in n:
                p.uniform_(0.5, 1.5)
    grid = tp.ModelParallelGrid(model_parallel_size=world)
    m = TPGPT(cfg, grid.get_model_parallel_group()).load_from(full)
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, cfg.vocab_size, (2, 32), generator=g)
    tgt = torch.randint(0, cfg.vocab_size, (2, 32), generator=g)
    _, ref = full(idx, tgt)
    ref.backward()
    _, loss = m(idx, tgt)
    loss.backward()
    torch.testing.assert_close(loss, ref, rtol=1e-5, atol=1e-5)
    for b, fb in zip(m.blocks, full.blocks):
        for n in ("q_norm", "k_norm"):
            torch.testing.assert_close(getattr(b.attn, n).weight.grad, getattr(fb.attn, n).weight.grad,
                                       rtol=1e-4, atol=1e-7)
    s, n = m.wte.start, m.wte.per
    torch.testing.assert_close(m.wte.weight.grad, full.wte.weight.grad[s:s + n], rtol=1e-4, atol=1e-6)
    sd = m.full_state_dict()
    for k, v in full.state_dict().items():
        torch.testing.assert_close(sd[k], v, msg=k)


@pytest.mark.parametrize("pos", ["learned", "rotary"])
def test_tensor_parallel_matches_dense(pos):
    _run(2, _tp_parity, pos)


@pytest.mark.gpu
@pytest.mark.parametrize("pos,qk_norm", [("learned", True), ("rotary", True), ("learned", False), ("rotary", False)])
def test_a_training_step_on_the_gpu(pos, qk_norm):
    """Lookup, norms, attention, loss, all gradients and clipping in bf16 against fp32 plain PyTorch
    (bf16 activations through two blocks: 5 % of a gradient's norm)."""
    m = _model(pos, qk_norm).cuda()
    idx, tgt = (torch.randint(0, 512, (3, 150), device="cuda") for _ in range(2))
    mb = gpt2.cast_for_mi355x(copy.deepcopy(m))
    m.load_state_dict({k: v.float() for k, v in mb.state_dict().items()}, strict=False)
    loss = F.cross_entropy(_plain(m, idx).flatten(0, 1), tgt.flatten())
    loss.backward()
    _, lb = mb(idx, tgt)
    lb.backward()
    assert abs(lb.item() - loss.item()) < 2e-2
    for (n, p), q in zip(m.named_parameters(), mb.parameters()):
        assert ((q.grad.float() - p.grad).norm() / p.grad.norm()).item() < 5e-2, n
    want = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.1)
    got = fopt.clip_grad_norm_(mb.parameters(), 0.1)
    assert abs(float(got) / float(want) - 1) < 2e-2
    # bf16 gradients are rounded to 2^-8 after scaling, which averages out in the norm
    assert abs(float(fopt.grad_norm(p.grad for p in mb.parameters())) - 0.1) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("pos", ["learned", "rotary"])
def test_gradients_added_in_place_are_the_returned_ones(pos):
    """With the fused optimizer's flat gradients the kernels add into ``.grad``: two backward passes
    give the sum of two plain ones, up to the rounding of the bf16 sums (two steps of 2^-8)."""
    m = gpt2.cast_for_mi355x(_model(pos)).cuda()
    flat = copy.deepcopy(m)
    opt = fopt.FusedAdamW(flat.parameters(), lr=1e-3)
    opt.space.ensure_views()
    opt.zero_grad()
    sums = None
    for seed in (1, 2):
        torch.manual_seed(seed)
        idx, tgt = (torch.randint(0, 512, (2, 100), device="cuda") for _ in range(2))
        got = torch.autograd.grad(m(idx, tgt)[1], list(m.parameters()))
        sums = [g.double() for g in got] if sums is None else [s + g.double() for s, g in zip(sums, got)]
        flat(idx, tgt)[1].backward()
    _grad.join()
    for (n, p), s in zip(flat.named_parameters(), sums):
        assert ((p.grad.double() - s).norm() / s.norm()).item() < 2 * 2 ** -8, n


@pytest.mark.gpu
def test_training_with_a_torch_optimizer_and_the_kernels_clipping():
    """Steps of a torch optimizer with clipping between: parameters follow torch's own clipping."""
    a = gpt2.cast_for_mi355x(_model("rotary")).cuda()
    b = copy.deepcopy(a)
    oa, ob = (torch.optim.SGD(m.parameters(), lr=0.1) for m in (a, b))
    for k in range(3):
        torch.manual_seed(k)
        idx = torch.randint(0, 512, (2, 64), device="cuda")
        for m, o, clip in ((a, oa, fopt.clip_grad_norm_), (b, ob, torch.nn.utils.clip_grad_norm_)):
            o.zero_grad()
            m(idx, idx)[1].backward()
            clip(m.parameters(), 0.5)
            o.step()
    for (n, p), q in zip(a.named_parameters(), b.named_parameters()):
        # torch rounds the coefficient to bf16, which moves an update by up to 2^-8 and a bf16
        # parameter by a step; fp32 parameters (norms, around 1) by updates of at most 0.05 * 2^-8
        torch.testing.assert_close(p, q[1], rtol=2 ** -7, atol=3e-4, msg=n)


@pytest.mark.gpu
def test_lookup_norm_and_clipping_in_one_captured_step():
    """Forward, backward and clipping captured once; replays on other inputs give the eager result."""
    from determined_clone_amd.ops.embedding import embedding
    from determined_clone_amd.ops.qk_norm import qk_norm_rope

    torch.manual_seed(0)
    B, S, H, D, V = 2, 700, 3, 64, 90
    cos, sin = T.rope_tables(S, 32, device="cuda")
    idx = torch.randint(0, V, (B, S), device="cuda")
    gq, gk = (torch.randn(B, S, H, D, device="cuda").bfloat16() for _ in range(2))
    shapes = [(V, 2 * H * D), (S, 2 * H * D), (D,), (D,)]
    init = [torch.randn(s, device="cuda").to(torch.bfloat16 if len(s) == 2 else torch.float32) for s in shapes]

    def step(params):
        for p in params:
            p.grad = None
        q, k = embedding(idx, params[0], params[1], scale=2.0).view(B, S, 2 * H, D).chunk(2, 2)
        q, k = qk_norm_rope(q, k, params[2], params[3], cos, sin, rot_dim=32)
        torch.autograd.backward((q, k), (gq, gk))
        return [fopt.clip_grad_norm_(params, 0.5)] + [p.grad for p in params]

    params = [torch.nn.Parameter(t.clone()) for t in init]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(params)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(params)
    eager = [torch.nn.Parameter(t.clone()) for t in init]  # leaves of their own for the eager steps
    for k in range(4):
        idx.copy_((idx * 7 + k) % V)
        gq.mul_(-0.5 if k % 2 else 3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(eager)):
            assert torch.equal(a, b), k


def test_the_gpt2_example_trains_with_qk_norm(tmp_path):
    from test_examples import _import_example

    from determined_clone_amd.common.storage import SharedFSStorageManager
    from determined_clone_amd.pytorch import Batch
    from determined_clone_amd.pytorch import deepspeed as det_ds

    m = _import_example("gpt2_deepspeed", "gpt2_trial")
    hp = {"model": "tiny", "seq_len": 32, "qk_norm": True,
          "overwrite_deepspeed_args": {"train_micro_batch_size_per_gpu": 2, "bf16": {"enabled": False},
                                       "scheduler": {"params": {"warmup_num_steps": 1, "total_num_steps": 10}}}}
    with det_ds.init(hparams=hp, exp_conf={}) as ctx:
        ctx._core.checkpoint._storage_manager = SharedFSStorageManager(str(tmp_path))
        t = m.GPT2Trial(ctx)
        det_ds.Trainer(t, ctx).fit(max_length=Batch(3), checkpoint_policy="none")
    norms = [p for n, p in t.engine.module.named_parameters() if n.endswith(("q_norm.weight", "k_norm.weight"))]
    assert len(norms) == 4 and all((p != 1).any() for p in norms)  # trained away from their start

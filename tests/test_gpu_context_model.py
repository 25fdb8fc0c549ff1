"""CloudContext and the pair model that calls it: the operators run together, in training (eager and as captured hipGraphs) and evaluation."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from tests.test_gpu_graphed_step import _assert_same, _batches, _state  # noqa: E402


@pytest.fixture(scope="module")
def pk():
    import se3_equi_graph_registration_amd as pkg
    pkg.lib()
    return pkg


def _plain_context(ctx, h, valid=None):
    """The same blocks as elementary fp64 operations."""
    _, b, n, c = h.shape
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in ctx.named_parameters()}

    def norm(v, w, bias):
        v = v - v.mean(-1, keepdim=True)
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * w + bias

    def attend(name, u, other, mask):
        heads = ctx.self_attention[0].num_heads
        split = lambda t: t.view(2 * b, -1, heads, c // heads).permute(0, 2, 1, 3)  # noqa: E731
        q, k, v = split(u @ p[name + ".to_q.weight"].mT), split(other @ p[name + ".to_k.weight"].mT), split(other @ p[name + ".to_v.weight"].mT)
        s = q @ k.mT * (c // heads) ** -0.5
        if mask is not None:
            s = s.masked_fill(~mask[:, None, None, :], float("-inf"))
        return (torch.softmax(s, -1) @ v).permute(0, 2, 1, 3).reshape(2 * b, n, c) @ p[name + ".to_out.weight"].mT

    def step(i, x, f):
        k = f"steps.{i}."
        y = x + p[k + "scale"] * norm(f, p[k + "post_weight"], p[k + "post_bias"])
        return y, norm(y, p[k + "pre_weight"], p[k + "pre_bias"]) if k + "pre_weight" in p else None

    leaf = h.detach().cpu().double().requires_grad_(True)
    x = leaf.reshape(2 * b, n, c)
    u = norm(x, p["first.pre_weight"], p["first.pre_bias"])
    mask = None if valid is None else valid.cpu().reshape(2 * b, n)
    for i in range(ctx.n_layers):
        x, u = step(3 * i, x, attend(f"self_attention.{i}", u, u, mask))
        x, u = step(3 * i + 1, x, attend(f"cross_attention.{i}", u, torch.cat([u[b:], u[:b]]), None if mask is None else torch.cat([mask[b:], mask[:b]])))
        z, g = u @ p[f"feed_forward.{i}.gate.weight"].mT, u @ p[f"feed_forward.{i}.up.weight"].mT
        x, u = step(3 * i + 2, x, (z * torch.sigmoid(z) * g) @ p[f"feed_forward.{i}.down.weight"].mT)
    return x.view(2, b, n, c), leaf, p


@pytest.mark.parametrize("width,heads,layers,masked", [(32, 4, 2, False), (33, 3, 1, True)])
def test_context_against_plain_operations(pk, width, heads, layers, masked):
    torch.manual_seed(3)
    ctx = pk.CloudContext(width, n_layers=layers, num_heads=heads, residual_scale=0.7, device="cuda")
    h = torch.randn(2, 2, 90, width)
    valid = torch.rand(2, 2, 90) < 0.8 if masked else None
    grad = torch.randn(2, 2, 90, width)
    hd = h.cuda().requires_grad_(True)
    out = ctx(hd, None if valid is None else valid.cuda())
    got = torch.autograd.grad(out, [hd] + list(ctx.parameters()), grad.cuda())
    ref, leaf, p = _plain_context(ctx, h, valid)
    want = torch.autograd.grad(ref, [leaf] + list(p.values()), grad.double())
    # fp32 end to end: a few hundred roundings deep, values of order one (norms between the blocks): 1e-5 of each tensor's largest value
    for name, g, w in zip(["out", "h"] + list(p), [out] + list(got), [ref] + list(want)):
        off, size = float((g.detach().cpu().double() - w.detach()).abs().max()), float(w.detach().abs().max())
        assert off <= 1e-5 * max(size, 1e-3), (name, off, size)


def _model(pk, feat=32, n=256, seed=0, variant="train"):
    torch.manual_seed(seed)
    egnn = pk.EGNN(feat, feat, feat, in_edge_nf=1, device="cuda", n_layers=2)
    ctx = pk.CloudContext(feat, num_heads=4, device="cuda")
    return pk.CrossAttentionPoseRegression(egnn, num_nodes=n, hidden_nf=feat, device="cuda", topk=64, variant=variant, context=ctx).cuda()


def test_training_with_a_context_graphed_equals_eager(pk):
    """The captured step (the blocks' parameters inside the flat bucket, off every 16-byte boundary) gives the eager loop's weights bit for
    bit, and every parameter of the blocks moves."""
    from se3_equi_graph_registration_amd import train
    batches = _batches(pk, 6)
    m_e, m_g = _model(pk), _model(pk)
    start = {k: v.detach().clone() for k, v in m_e.context.named_parameters()}
    o_e, o_g = train.make_optimizer(m_e, lr=1e-3), train.make_optimizer(m_g, lr=1e-3)
    train.train_one_epoch(m_e, batches, o_e, "cuda", 0, log_interval=0, k=8, graph=False)
    train.train_one_epoch(m_g, batches, o_g, "cuda", 0, log_interval=0, k=8)
    st = train.graphed_step_for(m_g, o_g, k=8)
    assert st.graph_mode == "one graph" and st.steps_replayed == 5
    _assert_same(_state(m_e, o_e), _state(m_g, o_g))
    for k, v in m_e.context.named_parameters():
        assert not torch.equal(v.detach(), start[k]), k


def test_evaluation_with_a_context(pk):
    m = _model(pk, variant="eval").eval()
    b = {k: (v[None] if torch.is_tensor(v) else v).cuda() for k, v in pk.synthetic_pair(5, n=256, feat=32).items()}
    graph = pk.build_pair_graph(b["src"], b["tgt"], 8)
    ones = torch.ones(1, 256 * 8, 1, device="cuda")
    with torch.no_grad():
        out = m(b["feat_src"], b["src"], graph, ones, b["feat_tgt"], b["tgt"], graph, ones, b["corr"], b["labels"], b["gt_pose"])
        h = m.egnn(torch.cat([b["feat_src"][0], b["feat_tgt"][0]]), torch.cat([b["src"][0], b["tgt"][0]]), graph, "ones")[0]
        want = m.context(h.view(2, 1, 256, 32))
    assert torch.equal(out[4], want[0]) and torch.equal(out[6], want[1])
    assert torch.isfinite(out[0]).all()


def test_without_a_context_the_model_is_unchanged(pk):
    egnn = pk.EGNN(32, 32, 32, in_edge_nf=1, device="cuda", n_layers=1)
    keys = pk.CrossAttentionPoseRegression(egnn, num_nodes=64, hidden_nf=32, device="cuda").state_dict()
    assert not [k for k in keys if k.startswith("context")]
    with pytest.raises(ValueError, match="context"):
        pk.CrossAttentionPoseRegression(egnn, num_nodes=64, hidden_nf=32, device="cuda", context=pk.CloudContext(16, num_heads=2, device="cuda"))


def test_refusals(pk):
    """What the operators do not take is refused on the host, before any launch."""
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    att, ff, rn = pk.cloud_attention, pk.gated_feed_forward, pk.residual_norm
    q, k = f(2, 5, 4, 16), f(2, 7, 2, 16)
    for bad in (lambda: att(q, k, f(2, 6, 2, 16)), lambda: att(q, f(2, 7, 3, 16), f(2, 7, 3, 16)), lambda: att(q, f(1, 7, 2, 16), f(1, 7, 2, 16)),
                lambda: att(q[0], k, k), lambda: att(q.double(), k.double(), k.double()), lambda: att(q, k.half(), k), lambda: att(q, k.cpu(), k),
                lambda: att(q, k, k, q_lens=torch.zeros(2, dtype=torch.int64, device="cuda")), lambda: att(q, k, k, kv_lens=f(3, dtype=torch.int32)),
                lambda: att(q, k, k, key_mask=f(2, 7)), lambda: att(q, k, k, key_mask=f(2, 5, dtype=torch.bool)),
                lambda: ff(f(3, 8), f(6, 8), f(6, 8), f(8, 5)), lambda: ff(f(3, 7), f(6, 8), f(6, 8), f(8, 6)), lambda: ff(f(3, 8), f(6, 8), f(5, 8), f(8, 6)),
                lambda: ff(f(3, 8), f(6, 8), f(6, 8), f(8, 6), b_up=f(8)), lambda: ff(f(3, 8), f(6, 8), f(6, 8), f(8, 6).half()),
                lambda: rn(f(3, 8), f(3, 9)), lambda: rn(f(3, 8), f(3, 8), gate=f(3)), lambda: rn(f(3, 8), f(3, 8), f(9)), lambda: rn(f(3, 8), f(3, 8).half()),
                lambda: rn(f(3, 8), f(3, 8), f(8), scale=f(1))):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: att(q, k, k, scale=0.0), lambda: att(q, k, k, scale=float("nan")), lambda: att(q, k, k, scale=-1.0),
                lambda: ff(f(3, 8), f(6, 8), f(6, 8), f(8, 6), activation="tanh"), lambda: rn(f(3, 8), f(3, 8), kind="group"), lambda: rn(f(3, 8), None),
                lambda: rn(f(3, 8), f(3, 8), None, f(8)), lambda: rn(f(3, 8), f(3, 8), eps=-1.0), lambda: rn(f(3, 8), None, f(8), scale=2.0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: att(f(1, 2, 1, 129), f(1, 2, 1, 129), f(1, 2, 1, 129)), lambda: rn(f(2, 8193), f(2, 8193)),
                lambda: pk.CloudAttention(512, 2), lambda: pk.ResidualNorm(9000)):
        with pytest.raises(NotImplementedError):
            bad()
    for bad in (lambda: att(q, k, None), lambda: att(q, k, k, q_lens=[1, 2]), lambda: ff(None, f(6, 8), f(6, 8), f(8, 6)), lambda: rn(None, None, f(8))):
        with pytest.raises(TypeError):
            bad()
    x = f(1, 4, 1, 8).requires_grad_(True)
    with pytest.raises(RuntimeError):                                      # differentiable once
        g, = torch.autograd.grad(att(x, x, x).sum(), x, create_graph=True)
        g.sum().backward()

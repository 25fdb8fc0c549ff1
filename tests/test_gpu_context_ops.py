"""The context operators (cloud_attention, gated_feed_forward, residual_norm) on the GPU against their fp64 definitions
(oracle/context_oracle.py), at the sizes and masks where they can go wrong.  The bounds come with the oracle: roundings of the documented
values, fp32 sums."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import context_oracle as orc  # noqa: E402

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def pkg():
    import se3_equi_graph_registration_amd as p
    return p


def normal(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def within(got, val, err, what):
    for n in val:
        if n not in got or got[n] is None:
            continue
        g = got[n].detach().cpu().double()
        assert g.shape == val[n].shape, (what, n, g.shape, val[n].shape)
        off = (g - val[n]).abs()
        bad = ~(off <= err[n])
        assert not bad.any(), f"{what} {n}: {int(bad.sum())} of {bad.numel()} values out of bounds, worst {float((off / err[n]).max()):.2f} x " \
                              f"at {bad.nonzero()[0].tolist()}"


def attention_case(seed, dtype, b, nq, nk, h, hk, d, causal=False, q_lens=None, kv_lens=None, mask=False, train=True, scale=None, size=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = normal(g, b, nq, h, d, dtype=dtype, scale=size), normal(g, b, nk, hk, d, dtype=dtype, scale=size), normal(g, b, nk, hk, d, dtype=dtype)
    m = None
    if mask:
        m = torch.rand(b, nk, generator=g) < 0.6
        m[0] = False                                                       # the first sample sees nothing
    ql = None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32)
    kl = None if kv_lens is None else torch.tensor(kv_lens, dtype=torch.int32)
    grad = normal(g, b, nq, h, d, dtype=dtype) if train else None
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    args = [t.cuda().requires_grad_(train) for t in (q, k, v)]
    out = pkg().cloud_attention(*args, q_lens=dev(ql), kv_lens=dev(kl), key_mask=dev(m), causal=causal, scale=scale)
    got = {"out": out}
    if train:
        got["grad_q"], got["grad_k"], got["grad_v"] = torch.autograd.grad(out, args, grad.cuda())
    val, err = orc.attention(q, k, v, grad, ql, kl, m, causal, scale)
    within(got, val, err, f"attention {dtype} {(b, nq, nk, h, hk, d)}")
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("b,nq,nk,h,hk,d", [
    (1, 1, 1, 1, 1, 1), (2, 5, 3, 2, 1, 8), (1, 33, 65, 3, 3, 11), (2, 64, 64, 4, 2, 32), (1, 129, 200, 2, 2, 33), (2, 130, 127, 4, 1, 64),
    (1, 70, 257, 6, 2, 80), (1, 257, 130, 2, 2, 128), (3, 31, 96, 1, 1, 127)])
def test_attention_shapes(dtype, b, nq, nk, h, hk, d):
    attention_case(1, dtype, b, nq, nk, h, hk, d)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("nq,nk,causal,q_lens,kv_lens,mask", [
    (100, 100, True, None, None, False), (40, 150, True, None, None, False), (150, 40, True, None, None, False),
    (70, 90, False, [70, 0, 1], [90, 40, 0], False), (70, 90, True, [33, 70, 7], [64, 65, 90], False), (66, 140, False, None, None, True),
    (66, 140, True, [66, 20, 64], [140, 1, 100], True), (50, 0, False, None, None, False), (50, 60, False, [99, -3, 50], [1000, 60, -1], False)])
def test_attention_masks(dtype, nq, nk, causal, q_lens, kv_lens, mask):
    attention_case(2, dtype, 3, nq, nk, 4, 2, 24, causal, q_lens, kv_lens, mask)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("nq,nk,h,hk,d,causal,kv_lens", [
    (1, 5000, 8, 2, 128, False, [5000, 3]), (3, 4097, 4, 4, 64, True, [4097, 2]), (1, 1, 4, 1, 32, False, [1, 0]), (8, 3001, 2, 1, 16, True, [3001, 1500])])
def test_attention_few_rows(dtype, nq, nk, h, hk, d, causal, kv_lens):
    """Single tokens against long caches: the key axis is split over workgroups and joined."""
    attention_case(3, dtype, 2, nq, nk, h, hk, d, causal, None, kv_lens, train=False)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_large_scores(dtype):
    """Scores far from zero (the running maximum moves, most probabilities vanish) and a scale of the caller's."""
    attention_case(4, dtype, 1, 96, 300, 2, 2, 48, size=4.0, scale=0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_hidden_values_are_never_used(dtype):
    """NaN, infinities and the type's lowest value in hidden keys and behind the lengths: same results, zero gradients there."""
    g = torch.Generator().manual_seed(5)
    b, nq, nk, h, d = 2, 40, 150, 2, 32
    q, k, v, go = (normal(g, b, n, h, d, dtype=dtype) for n in (nq, nk, nk, nq))
    m = torch.rand(b, nk, generator=g) < 0.5
    ql, kl = torch.tensor([40, 17], dtype=torch.int32), torch.tensor([150, 77], dtype=torch.int32)
    seen = m & (torch.arange(nk)[None] < kl[:, None])
    rows = torch.arange(nq)[None] < ql[:, None]

    def run(poison):
        t = [x.clone() for x in (q, k, v, go)]
        if poison:
            bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min], dtype=dtype)
            for x in t[1:3]:
                x[~seen] = bad[torch.arange(int((~seen).sum())) % 4][:, None, None]
            for x in (t[0], t[3]):
                x[~rows] = bad[torch.arange(int((~rows).sum())) % 4][:, None, None]
        a = [x.cuda().requires_grad_(True) for x in t[:3]]
        out = pkg().cloud_attention(*a, q_lens=ql.cuda(), kv_lens=kl.cuda(), key_mask=m.cuda())
        return [out] + list(torch.autograd.grad(out, a, t[3].cuda()))
    for clean, dirty, live in zip(run(False), run(True), (rows, rows, seen, seen)):
        assert torch.equal(clean, dirty)
        assert float(clean.detach()[~live.cuda()].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_attention_strides(dtype):
    """q, k, v as views of one projection, heads before points, broadcast keys, a strided last dimension, an offset that breaks alignment."""
    g = torch.Generator().manual_seed(6)
    b, n, h, d = 2, 70, 3, 16
    qkv = normal(g, b, n, 3, h, d, dtype=dtype)
    want = [qkv[:, :, i].contiguous() for i in range(3)]
    ref = pkg().cloud_attention(*(t.cuda() for t in want))
    dev = qkv.cuda()
    assert torch.equal(ref, pkg().cloud_attention(dev[:, :, 0], dev[:, :, 1], dev[:, :, 2]))
    hm = [t.cuda().transpose(1, 2).contiguous().transpose(1, 2) for t in want]
    assert torch.equal(ref, pkg().cloud_attention(*hm))
    last = [t.cuda().transpose(1, 3).contiguous().transpose(1, 3) for t in want]
    assert torch.equal(ref, pkg().cloud_attention(*last))
    off = []
    for t in want:
        buf = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        buf[1:].copy_(t.reshape(-1))
        off.append(buf[1:].view(t.shape))
    assert torch.equal(ref, pkg().cloud_attention(*off))
    one = want[1][:1].cuda()
    leaf = one.clone().requires_grad_(True)
    wide = pkg().cloud_attention(want[0].cuda(), leaf.expand(b, -1, -1, -1), want[2].cuda())
    full = one.expand(b, -1, -1, -1).contiguous().requires_grad_(True)
    same = pkg().cloud_attention(want[0].cuda(), full, want[2].cuda())
    assert torch.equal(wide, same)
    ga, = torch.autograd.grad(wide.sum(), leaf)                            # an expanded gradient, too
    gb, = torch.autograd.grad(same.sum(), full)
    torch.testing.assert_close(ga, gb.sum(0, keepdim=True), rtol=2 * torch.finfo(dtype).eps, atol=2 * torch.finfo(dtype).eps)


@pytest.mark.parametrize("layout", ["far samples", "far points"])
def test_attention_offsets_beyond_32_bits(layout):
    """Keys and values whose offsets pass 2^31 values: samples far apart, and a cache with points far apart; forward and backward."""
    g = torch.Generator().manual_seed(15)
    b, nk, stride = (2, 70, (2200000000, 64, 64, 1)) if layout == "far samples" else (1, 600, (1, 4000000, 64, 1))
    buf = torch.empty(2400100000, dtype=torch.bfloat16, device="cuda")
    k, v = normal(g, b, nk, 1, 64, dtype=torch.bfloat16), normal(g, b, nk, 1, 64, dtype=torch.bfloat16)
    q, go = normal(g, b, 40, 1, 64, dtype=torch.bfloat16).cuda(), normal(g, b, 40, 1, 64, dtype=torch.bfloat16).cuda()
    far = []
    for i, t in enumerate((k, v)):
        view = buf.as_strided((b, nk, 1, 64), stride, 10000 * i)
        view.copy_(t)
        far.append(view)

    def run(kk, vv):
        a = [t.detach().requires_grad_(True) for t in (q, kk, vv)]
        out = pkg().cloud_attention(*a)
        return [out.detach()] + list(torch.autograd.grad(out, a, go))
    assert all(torch.equal(x, y) for x, y in zip(run(k.cuda(), v.cuda()), run(*far)))


@pytest.mark.parametrize("dtype", [torch.float16], ids=["f16"])
@pytest.mark.parametrize("size", [1e-4, 1e3])
def test_attention_fp16_gradients_of_any_size(dtype, size):
    """Output gradients far below and above 1: the products' operands stay inside fp16's range."""
    g = torch.Generator().manual_seed(7)
    q, k, v = (normal(g, 1, 1500, 1, 32, dtype=dtype) for _ in range(3))
    go = normal(g, 1, 1500, 1, 32, dtype=dtype, scale=size)
    a = [x.cuda().requires_grad_(True) for x in (q, k, v)]
    out = pkg().cloud_attention(*a)
    got = dict(zip(("grad_q", "grad_k", "grad_v"), torch.autograd.grad(out, a, go.cuda())), out=out)
    val, err = orc.attention(q, k, v, go)
    within(got, val, err, f"attention fp16 gradient {size}")


def test_attention_is_reproducible_and_takes_partial_gradients():
    g = torch.Generator().manual_seed(8)
    q, k, v = (normal(g, 2, 300, 4, 64, dtype=torch.bfloat16).cuda().requires_grad_(True) for _ in range(3))
    go = normal(g, 2, 300, 4, 64, dtype=torch.bfloat16).cuda()
    f = lambda *w: torch.autograd.grad(pkg().cloud_attention(q, k, v, causal=True), w, go)  # noqa: E731
    first = f(q, k, v)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, f(q, k, v)))
    assert torch.equal(first[0], f(q)[0]) and torch.equal(first[1], f(k)[0]) and torch.equal(first[2], f(v)[0])


def test_attention_gradient_against_differences():
    """The directional derivative of sum(out * w) in fp32 against central differences of the fp64 definition."""
    g = torch.Generator().manual_seed(9)
    t = [normal(g, 1, 20, 2, 8, dtype=torch.float32) for _ in range(3)]
    w, dirs = normal(g, 1, 20, 2, 8, dtype=torch.float32), [normal(g, 1, 20, 2, 8, dtype=torch.float32) for _ in range(3)]
    a = [x.cuda().requires_grad_(True) for x in t]
    grads = torch.autograd.grad(pkg().cloud_attention(*a, causal=True), a, w.cuda())
    got = sum(float((x.cpu().double() * y.double()).sum()) for x, y in zip(grads, dirs))
    at = lambda e: float((_attention64(*(x.double() + e * y.double() for x, y in zip(t, dirs))) * w.double()).sum())  # noqa: E731
    want = (at(1e-4) - at(-1e-4)) / 2e-4
    assert abs(got - want) <= 1e-5 * (1 + abs(want)), (got, want)          # differences: 1e-8 x the third derivative; fp32 sums of 960 terms


def _attention64(q, k, v):
    s = torch.einsum("bihd,bjhd->bhij", q, k) * q.shape[-1] ** -0.5
    s = s.masked_fill(torch.ones(s.shape[-2:], dtype=torch.bool).triu(1), float("-inf"))
    return torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v)


# ------------------------------------------------------------------------------------------------ feed-forward
def feed_forward_case(seed, dtype, rows, width, hidden, out=None, activation="silu", biased=True, train=True):
    g = torch.Generator().manual_seed(seed)
    out = width if out is None else out
    t = {"x": normal(g, rows, width, dtype=dtype), "w_gate": normal(g, hidden, width, dtype=dtype, scale=width ** -0.5),
         "w_up": normal(g, hidden, width, dtype=dtype, scale=width ** -0.5), "w_down": normal(g, out, hidden, dtype=dtype, scale=hidden ** -0.5)}
    if biased:
        t.update(b_gate=normal(g, hidden, dtype=dtype, scale=0.2), b_up=normal(g, hidden, dtype=dtype, scale=0.2), b_down=normal(g, out, dtype=dtype))
    grad = normal(g, rows, out, dtype=dtype) if train else None
    dev = {n: v.cuda().requires_grad_(train) for n, v in t.items()}
    y = pkg().gated_feed_forward(**dev, activation=activation)
    got = {"y": y}
    if train:
        got.update(("grad_" + n, v) for n, v in zip(dev, torch.autograd.grad(y, list(dev.values()), grad.cuda())))
    val, err = orc.feed_forward(**t, grad=grad, activation=activation)
    within(got, val, err, f"feed_forward {dtype} {(rows, width, hidden, out)}")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,width,hidden,out", [(1, 1, 1, 1), (1, 32, 128, 32), (5, 33, 70, 33), (64, 32, 128, 48), (130, 129, 65, 20), (300, 64, 200, 64),
                                                   (1000, 40, 72, 40), (17, 512, 300, 256), (16, 640, 1280, 640), (33, 100, 1030, 7),
                                                   (2, 2100, 300, 33), (32, 130, 1500, 130), (9, 8, 17, 3)])
def test_feed_forward_shapes(dtype, rows, width, hidden, out):
    feed_forward_case(11, dtype, rows, width, hidden, out)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("rows,width,hidden", [(4100, 512, 1064), (2049, 1030, 1100)])
def test_feed_forward_large_tiles(dtype, rows, width, hidden):
    """Enough outputs for the large tile in every product, with tiles cut at every edge, and contractions cut into parts."""
    feed_forward_case(14, dtype, rows, width, hidden)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("activation", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("biased", [True, False])
def test_feed_forward_activations(dtype, activation, biased):
    feed_forward_case(12, dtype, 200, 48, 96, None, activation, biased)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_feed_forward_empty_partial_and_unaligned(dtype):
    g = torch.Generator().manual_seed(13)
    w = [normal(g, 40, 24, dtype=dtype).cuda(), normal(g, 40, 24, dtype=dtype).cuda(), normal(g, 24, 40, dtype=dtype).cuda()]
    x = normal(g, 3, 50, 24, dtype=dtype).cuda()
    ref = pkg().gated_feed_forward(x, *w)
    assert ref.shape == x.shape
    # weights inside one flat block, off every 16-byte boundary (what a flat optimizer bucket gives); x as a transposed view
    flat = torch.empty(1 + sum(t.numel() for t in w), dtype=dtype, device="cuda")
    off, views = 1, []
    for t in w:
        flat[off:off + t.numel()].copy_(t.reshape(-1))
        views.append(flat[off:off + t.numel()].view(t.shape))
        off += t.numel()
    assert torch.equal(ref, pkg().gated_feed_forward(x.transpose(0, 1).contiguous().transpose(0, 1), *views))
    # nothing in, nothing out; the weights' gradients are zeros
    leaf = [t.clone().requires_grad_(True) for t in w]
    none = pkg().gated_feed_forward(x[:0], *leaf)
    assert none.shape == (0, 50, 24)
    assert all(float(t.abs().max()) == 0.0 for t in torch.autograd.grad(none.sum(), leaf))
    # one gradient at a time gives what all at once give
    xs = x.clone().requires_grad_(True)
    go = normal(g, 3, 50, 24, dtype=dtype).cuda()
    both = torch.autograd.grad(pkg().gated_feed_forward(xs, *leaf), [xs] + leaf, go)
    for i, t in enumerate([xs] + leaf):
        assert torch.equal(both[i], torch.autograd.grad(pkg().gated_feed_forward(xs, *leaf), t, go)[0])


# ------------------------------------------------------------------------------------------------ residual norm
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("b,n,c", [(1, 1, 1), (2, 3, 7), (2, 100, 32), (3, 17, 33), (2, 9, 64), (1, 40, 65), (2, 30, 512), (2, 7, 1000), (1, 5, 2048), (1, 3, 3000), (2, 6, 1001), (1, 3, 4099),
                                   (1, 2, 8192)])
def test_residual_norm_shapes(dtype, kind, b, n, c):
    residual_norm_case(21, dtype, kind, b, n, c)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("post,pre,gate,scale", [(True, True, "sample", 0.3), (False, True, None, None), (True, False, "all", "tensor"), (False, False, "one", 2.0),
                                                 (False, True, "all", None), (True, True, None, "tensor"), (False, False, None, None)])
def test_residual_norm_parts(dtype, post, pre, gate, scale):
    residual_norm_case(22, dtype, "layer", 3, 50, 48, post, pre, gate, scale)
    residual_norm_case(23, dtype, "rms", 2, 300, 20, post, pre, gate, scale)


def residual_norm_case(seed, dtype, kind, b, n, c, post=True, pre=True, gate="sample", scale="tensor"):
    g = torch.Generator().manual_seed(seed)
    f32 = torch.float32
    t = {"x": normal(g, b, n, c, dtype=dtype), "f": normal(g, b, n, c, dtype=dtype, scale=3.0) + 1}
    if pre:
        t["pre_weight"] = 1 + normal(g, c, dtype=f32, scale=0.2)
    if post:
        t["post_weight"] = 1 + normal(g, c, dtype=f32, scale=0.2)
    if kind == "layer":
        for w in ("pre", "post"):
            if w + "_weight" in t:
                t[w + "_bias"] = normal(g, c, dtype=f32, scale=0.2)
    if gate:
        t["gate"] = normal(g, *{"sample": (b, c), "all": (b, n, c), "one": (c,)}[gate], dtype=dtype)
    if scale == "tensor":
        t["scale"] = normal(g, c, dtype=f32)
    eps = 1e-3                                                             # width 1: a spread of zero, 1 / sqrt(eps) bounds the amplification
    gy, gu = normal(g, b, n, c, dtype=dtype), normal(g, b, n, c, dtype=dtype) if pre else None
    dev = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    more = {} if scale in (None, "tensor") else {"scale": scale}
    x, f = dev["x"], dev["f"]
    rest = {k: v for k, v in dev.items() if k not in "xf"}
    y, u = pkg().residual_norm(x, f, **rest, **more, kind=kind, eps=eps)
    assert (u is None) == (not pre)
    outs = [(y, gy)] + ([(u, gu)] if pre else [])
    got = {"y": y, "u": u}
    got.update(("grad_" + k, v) for k, v in zip(dev, torch.autograd.grad([o for o, _ in outs], list(dev.values()), [w.cuda() for _, w in outs])))
    cpu = dict(t)
    if gate == "sample":
        cpu["gate"] = t["gate"][:, None, :]
    val, err = orc.residual_norm(**cpu, **more, kind=kind, eps=eps, grad_y=gy, grad_u=gu)
    for d in (val, err):
        if gate == "sample":
            d["grad_gate"] = d["grad_gate"][:, 0]
    within(got, val, err, f"residual_norm {dtype} {kind} {(b, n, c)}")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_residual_norm_without_f_and_with_one_gradient(dtype):
    g = torch.Generator().manual_seed(24)
    x, f, w = normal(g, 60, 40, dtype=dtype), normal(g, 60, 40, dtype=dtype), normal(g, 40, dtype=torch.float32)
    xs, fs, ws = x.cuda().requires_grad_(True), f.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y, u = pkg().residual_norm(xs, None, ws)
    assert y is xs
    gu = normal(g, 60, 40, dtype=dtype)
    gx, gw = torch.autograd.grad(u, [xs, ws], gu.cuda())
    val, err = orc.residual_norm(x, None, w, grad_u=gu)
    within({"u": u, "grad_x": gx, "grad_pre_weight": gw}, val, err, "residual_norm without f")
    for which in ("y", "u"):                                               # a loss that uses one of the two outputs
        y, u = pkg().residual_norm(xs, fs, ws)
        gx, gf = torch.autograd.grad(y if which == "y" else u, [xs, fs], gu.cuda())
        val, err = orc.residual_norm(x, f, w, **{"grad_" + which: gu})
        within({"grad_x": gx, "grad_f": gf}, val, err, f"residual_norm gradient of {which} only")
    none = pkg().residual_norm(xs[:0], fs[:0], ws)
    assert none[0].shape == (0, 40) and float(torch.autograd.grad(none[1].sum(), ws)[0].abs().max()) == 0.0


@pytest.mark.parametrize("rows,c", [(3, 8), (5, 300), (33, 16)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_residual_norm_without_eps(rows, c, kind):
    """eps = 0, with rows that do not fill a workgroup: the rows that are not there leave no trace in the parameters' gradients."""
    g = torch.Generator().manual_seed(25)
    x, f, gu = (normal(g, rows, c, dtype=torch.float32) for _ in range(3))
    w, v = normal(g, c, dtype=torch.float32), normal(g, c, dtype=torch.float32)
    dev = [t.cuda().requires_grad_(True) for t in (x, f, w, v)]
    bias = torch.zeros(c, device="cuda").requires_grad_(True) if kind == "layer" else None
    y, u = pkg().residual_norm(dev[0], dev[1], dev[2], bias, post_weight=dev[3], kind=kind, eps=0.0)
    got = dict(zip(("grad_x", "grad_f", "grad_pre_weight", "grad_post_weight"), torch.autograd.grad(u, dev, gu.cuda())), y=y, u=u)
    val, err = orc.residual_norm(x, f, w, None, v, kind=kind, eps=0.0, grad_u=gu)
    within(got, val, err, f"residual_norm eps 0 {kind} {(rows, c)}")


@pytest.mark.parametrize("gate", ["sample", "all", "one"])
def test_residual_norm_of_nothing(gate):
    """Clouds without points: empty outputs, parameter and gate gradients of zeros."""
    x = torch.zeros(2, 0, 16, device="cuda").requires_grad_(True)
    w = torch.ones(16, device="cuda").requires_grad_(True)
    gt = torch.ones({"sample": (2, 16), "all": (2, 0, 16), "one": (16,)}[gate], device="cuda").requires_grad_(True)
    y, u = pkg().residual_norm(x, x, w, gate=gt)
    assert y.shape == u.shape == (2, 0, 16)
    assert all(float(t.abs().sum()) == 0.0 for t in torch.autograd.grad(y.sum() + u.sum(), [x, w, gt]))


def test_concurrent_streams_share_nothing():
    """The same calls on two streams at once, each with its own workspace: what one stream alone gives."""
    g = torch.Generator().manual_seed(26)
    q = normal(g, 1, 1, 8, 64, dtype=torch.bfloat16).cuda()
    caches = [normal(g, 1, 20000, 2, 64, dtype=torch.bfloat16).cuda() for _ in range(2)]
    x, w = normal(g, 400, 64, dtype=torch.float32).cuda(), [normal(g, *s, dtype=torch.float32, scale=0.1).cuda() for s in ((3000, 64), (3000, 64), (64, 3000))]
    call = lambda i: (pkg().cloud_attention(q, caches[i], caches[i]), pkg().gated_feed_forward(x * (i + 1), *w))  # noqa: E731
    want = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_operators_on_another_stream_and_in_a_captured_graph():
    """A whole step of the three operators recorded once and replayed over new inputs, against the eager step; eager work in between."""
    g = torch.Generator().manual_seed(31)
    b, n, c, h = 2, 150, 64, 4
    new = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).cuda()  # noqa: E731
    params = [new(c, k=0.1) + 1, new(c, k=0.1), new(160, c, k=0.1), new(160, c, k=0.1), new(c, 160, k=0.1)]
    params = [p.requires_grad_(True) for p in params]
    x = new(b, n, c).requires_grad_(True)
    go = new(b, n, c)

    def step():
        w, bias, wg, wu, wd = params
        _, v = pkg().residual_norm(x, None, w, bias)
        a = pkg().cloud_attention(*(v.view(b, n, h, c // h),) * 3).view(b, n, c)
        y, v = pkg().residual_norm(x, a, w, bias, scale=0.5)
        y = y + pkg().gated_feed_forward(v, wg, wu, wd)
        return [y] + list(torch.autograd.grad(y, [x] + params, go))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            warm = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, t.detach()) for a, t in zip(warm, step()))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
        held = [t.detach() for t in held]
    for k in range(4):
        with torch.no_grad():
            x.copy_(new(b, n, c))
            go.copy_(new(b, n, c))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = [t.detach() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), k


def test_capture_beside_a_living_eager_graph_is_refused():
    """An eager graph of the same leaf that is still alive on another stream: recording a differentiable call raises before anything is
    recorded (the backward would synchronise with that stream); without it, or without gradients, it records."""
    x = torch.randn(2, 32, 2, 16, device="cuda").requires_grad_(True)
    alive = pkg().cloud_attention(x, x, x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="still alive"):
            pkg().cloud_attention(x, x, x)
        with torch.no_grad():
            out = pkg().cloud_attention(x, x, x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive.detach())
    del alive
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        out = pkg().cloud_attention(x, x, x)
        grad, = torch.autograd.grad(out, x, torch.ones_like(out))
    graph2.replay()
    torch.cuda.synchronize()
    want, = torch.autograd.grad(pkg().cloud_attention(x, x, x), x, torch.ones_like(out))
    assert torch.equal(grad, want)

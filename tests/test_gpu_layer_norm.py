"""Layer norm (functional.layer_norm, modules.LayerNorm) against its definition in 64 bits.

Tolerances.  A value of the result's type is off by half a step of that type (HALF_STEP, plus half a subnormal step).  Before
that rounding everything is fp32 with unit roundoff u = 2^-24: a sum over a row is formed by at most 8 * 2 additions per thread and
at most 10 levels of the team (walked rows: ceil(C / 8192) * 8 additions instead), so 64 u times the sum of magnitudes covers it
with the few operations on top; the mean's error reaches xh through (x - mu) * rstd, i.e. as 64 u * mean|x| * rstd.  The
parameters' gradients are sums over rows, whose additions per thread are counted in `additions`."""
import pytest
import torch

from oracle import train_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U32
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _make(shape, dt, seed, scale=1.5, shift=0.3):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dt)


def _within(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.2f} x the tolerance"


def _check(x, w, b, eps, r=None, gy=None, gs=None, place=lambda t: t.cuda(), dim=-1, need=(True, True, True, True)):
    """One forward (and backward) on the GPU against the oracle; `place` puts an operand into GPU memory."""
    from ayolov2_amd.functional import layer_norm
    dt, C = x.dtype, x.shape[dim]
    ops = [None if t is None else p(t) for t, p in ((x, place), (r, place), (w, lambda t: t.cuda()), (b, lambda t: t.cuda()))]
    if gy is not None:
        ops = [None if t is None else t.requires_grad_(n) for t, n in zip(ops, need)]
    xg, rg, wg, bg = ops
    out = layer_norm(xg, wg, bg, eps, residual=rg, dim=dim)
    y, s = out if r is not None else (out, None)
    last = lambda t: None if t is None else t.movedim(dim, -1)  # noqa: E731
    wy, ws = ref.layer_norm(last(x), w, b, eps, last(r))
    t = ws.double()
    n_add = 64 if C <= 8192 else 64 + -(-C // 8192) * 8
    mu = t.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((t - mu) ** 2).mean(-1, keepdim=True) + eps)
    m = 1.0 + t.abs().mean(-1, keepdim=True) * rstd                # how far the mean's error reaches
    xh = ((t - mu) * rstd).abs()
    aw = torch.ones(C, dtype=torch.float64) if w is None else w.double().abs()
    ab = 0.0 if b is None else b.double().abs()
    assert y.dtype == dt and y.shape == x.shape
    _within(last(y), wy, ref.HALF_STEP[dt] * wy.abs() * 1.001 + ref.TINY[dt] + n_add * U * ((m + xh) * (1.0 + xh) * aw + ab), "y")
    if s is not None:
        assert torch.equal(last(s).cpu(), ws), "the residual sum is x + r rounded once"
    if gy is None:
        return
    outs, gouts = [y], [place(gy)]
    if gs is not None:
        outs.append(s)
        gouts.append(place(gs))
    wanted = [v for v in ops if v is not None and v.requires_grad]
    grads = dict(zip([id(v) for v in wanted], torch.autograd.grad(outs, wanted, gouts)))
    dx, dw, db = ref.layer_norm_grads(ws, w, eps, last(gy), last(gs))
    gw = last(gy).double().abs() * aw
    inner = gw + gw.mean(-1, keepdim=True) + xh * (gw * xh).mean(-1, keepdim=True)
    rel = n_add * U * (m + xh) * rstd * inner * (1.0 + xh)
    for v in (xg, rg):
        if v is not None and id(v) in grads:
            got = grads[id(v)]
            assert got.dtype == dt and got.shape == x.shape
            _within(last(got), dx, ref.HALF_STEP[dt] * dx.abs() * 1.001 + ref.TINY[dt] + rel + 4 * U * dx.abs(), "dx")
    rows = x.numel() // C
    additions = rows // 64 + 128                                    # per thread (at least 64 groups of rows), teams, lines
    ga = last(gy).double().abs()
    flat = lambda v: v.reshape(-1, C).sum(0)  # noqa: E731
    if wg is not None and id(wg) in grads:
        got = grads[id(wg)]
        tol = additions * U * flat(ga * xh) + n_add * U * flat(ga * (m + xh) * (1 + xh)) + ref.HALF_STEP[w.dtype] * dw.abs() * 1.001 + ref.TINY[w.dtype]
        assert got.dtype == w.dtype
        _within(got, dw, tol, "dw")
    if bg is not None and id(bg) in grads:
        got = grads[id(bg)]
        _within(got, db, additions * U * flat(ga) + ref.HALF_STEP[b.dtype] * db.abs() * 1.001 + ref.TINY[b.dtype], "db")


def _params(C, dt, seed):
    return _make((C,), dt, seed, 0.2, 1.0), _make((C,), dt, seed + 1, 0.2, 0.0)


# every team size and its edges (16-bit vectors hold 8 elements, fp32 vectors 4), rows shorter than a vector, rows that are walked
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 257, 511, 513, 1000, 1024, 1025, 2049,
                               4096, 4097, 8191, 8193, 16384, 16385, 20011])
def test_widths(C, dt):
    rows = 5 if C > 2000 else 37
    x, gy = _make((rows, C), dt, C), _make((rows, C), dt, C + 1, 1.0, 0.0)
    r, gs = _make((rows, C), dt, C + 2, 1.0, 0.0), _make((rows, C), dt, C + 3, 0.5, 0.1)
    w, b = _params(C, torch.float32, C + 4)
    _check(x, w, b, 1e-5, gy=gy)
    _check(x, w.to(dt), b.to(dt), 1e-5, r=r, gy=gy, gs=gs)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 1000, 4099, 70001])
@pytest.mark.parametrize("C", [24, 96, 640])
def test_row_counts(rows, C):
    dt = torch.float16
    x, gy = _make((rows, C), dt, rows), _make((rows, C), dt, rows + 1, 1.0, 0.0)
    _check(x, *_params(C, torch.float32, 5), 1e-5, gy=gy)


@pytest.mark.parametrize("C", [16392, 33000])
def test_many_long_rows(C):
    """rows walked in pieces, more of them than the groups that sum the parameters' gradients"""
    x, gy = _make((150, C), torch.bfloat16, 1), _make((150, C), torch.bfloat16, 2, 1.0, 0.0)
    _check(x, *_params(C, torch.bfloat16, 3), 1e-5, r=_make((150, C), torch.bfloat16, 4), gy=gy, gs=_make((150, C), torch.bfloat16, 5))


def test_no_rows():
    from ayolov2_amd.functional import layer_norm
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w, b = torch.ones(16, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == (16,)


@pytest.mark.parametrize("which,need", [("none", "x"), ("w", "x"), ("b", "x"), ("w", "w"), ("b", "b"), ("w", "xw"), ("b", "xb")])
def test_optional_parameters_and_gradients(which, need):
    x, gy = _make((50, 72), torch.bfloat16, 1), _make((50, 72), torch.bfloat16, 2, 1.0, 0.0)
    w, b = _params(72, torch.float32, 3)
    w, b = (w if which == "w" else None), (b if which == "b" else None)
    _check(x, w, b, 1e-5, gy=gy, need=tuple(k in need for k in "xrwb"))


def test_parameters_of_other_types():
    """fp16 parameters beside fp32 activations, and a gain and a bias of different types."""
    x, gy = _make((40, 100), torch.float32, 1), _make((40, 100), torch.float32, 2, 1.0, 0.0)
    w, b = _params(100, torch.float32, 3)
    _check(x, w.half(), b.half(), 1e-5, gy=gy)
    _check(x.half(), w, b.half(), 1e-5, gy=gy.half())
    _check(x.half(), w.bfloat16(), None, 1e-5, gy=gy.half())


def _sliced(pad_c, off):
    def place(t):
        big = torch.full((*t.shape[:-1], t.shape[-1] + pad_c), float("nan"), dtype=t.dtype, device="cuda")
        v = big[..., off:off + t.shape[-1]]
        v.copy_(t)
        return v.detach()
    return place


def _window(t):
    """the middle of a batch of longer sequences: two levels of row strides"""
    big = torch.full((t.shape[0], t.shape[1] + 3, t.shape[2] + 5), float("nan"), dtype=t.dtype, device="cuda")
    v = big[:, 1:1 + t.shape[1], 2:2 + t.shape[2]]
    v.copy_(t)
    return v.detach()


def _turned(t):
    """rows in an order that two strides do not describe / the last dimension not innermost: copied"""
    return t.cuda().transpose(-1, -2).contiguous().transpose(-1, -2).detach()


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("place", [_sliced(1, 1), _sliced(64, 32), _sliced(7, 3), _window, _turned], ids=["odd", "half", "odd3", "window", "turned"])
def test_strides_and_alignment(dt, place):
    for C in (40, 129, 1000):
        x, gy = _make((3, 11, C), dt, C), _make((3, 11, C), dt, C + 1, 1.0, 0.0)
        r, gs = _make((3, 11, C), dt, C + 2, 1.0, 0.0), _make((3, 11, C), dt, C + 3, 0.5, 0.0)
        w, b = _params(C, torch.float32, C + 4)
        _check(x, w, b, 1e-5, r=r, gy=gy, gs=gs, place=place)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_maps(dt):
    """Channels of an NHWC activation, whole, as a channel slice of a wider buffer, and of an NCHW tensor (copied)."""
    def nhwc(t):
        return t.cuda().contiguous(memory_format=torch.channels_last)

    def slice_(t):
        big = torch.zeros(t.shape[0], t.shape[2], t.shape[3], t.shape[1] + 48, dtype=t.dtype, device="cuda")
        big[..., 16:16 + t.shape[1]] = t.cuda().permute(0, 2, 3, 1)
        return big[..., 16:16 + t.shape[1]].permute(0, 3, 1, 2).detach()

    for place in (nhwc, slice_, lambda t: t.cuda()):
        x, gy = _make((2, 48, 7, 5), dt, 1), _make((2, 48, 7, 5), dt, 2, 1.0, 0.0)
        r, gs = _make((2, 48, 7, 5), dt, 3, 1.0, 0.0), _make((2, 48, 7, 5), dt, 4, 0.5, 0.0)
        _check(x, *_params(48, torch.float32, 5), 1e-5, r=r, gy=gy, gs=gs, place=place, dim=1)


def test_expanded_inputs_and_gradients():
    """A residual and an output gradient that are broadcast views (row stride 0, or a scalar's expansion)."""
    from ayolov2_amd.functional import layer_norm
    x = _make((6, 9, 32), torch.float32, 1)
    r = _make((9, 32), torch.float32, 2)
    w, b = _params(32, torch.float32, 3)
    xg, rg, wg = x.cuda().requires_grad_(), r.cuda().requires_grad_(), w.cuda().requires_grad_()
    y, s = layer_norm(xg, wg, b.cuda(), residual=rg.expand_as(xg))
    (y.sum() * 0.5 + s.sum()).backward()                     # both gradients are expanded scalars
    t = [v.double().requires_grad_() for v in (x, r, w)]
    s64 = t[0] + t[1]
    y64 = torch.nn.functional.layer_norm(s64, (32,), t[2], b.double(), 1e-5)
    (y64.sum() * 0.5 + s64.sum()).backward()
    for got, want, terms in ((xg, t[0], 1), (rg, t[1], 6), (wg, t[2], 54)):
        # |ds| <= 1 + rstd * (gw + mean gw + xh mean(gw xh)) with gw = w / 2 about 0.5 .. 1, rstd < 1, |xh| < 4: below 8 per term
        assert float((got.grad.double().cpu() - want.grad).abs().max()) <= terms * 8 * 64 * U


def test_only_one_output_used():
    """A loss on the sum alone, or on the norm alone."""
    from ayolov2_amd.functional import layer_norm
    x, r = (_make((5, 24), torch.float32, k).cuda().requires_grad_() for k in (1, 2))
    w = torch.ones(24, device="cuda", requires_grad=True)
    y, s = layer_norm(x, w, None, residual=r)
    gx, gr, gw = torch.autograd.grad(s, (x, r, w), torch.ones_like(s), allow_unused=True, retain_graph=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, gx) and gw is None
    gy = _make((5, 24), torch.float32, 3, 1.0, 0.0)
    gx, gr = torch.autograd.grad(y, (x, r), gy.cuda())
    want = ref.layer_norm_grads(s.detach().cpu(), w.detach().cpu(), 1e-5, gy)[0]
    assert torch.equal(gx, gr)
    assert float((gx.double().cpu() - want).abs().max()) <= 64 * U * 64


def test_differentiable_once():
    """create_graph works as far as nobody asks for the derivative of a gradient; forward mode is refused; a weight changed in place
    between forward and backward is noticed"""
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.functional import layer_norm
    x = _make((5, 24), torch.float32, 1).cuda().requires_grad_()
    w = torch.ones(24, device="cuda", requires_grad=True)
    y, s = layer_norm(x, w, residual=x.detach())
    plain = torch.autograd.grad((y.sin().sum(), s.sum()), (x, w), retain_graph=True)
    kept = torch.autograd.grad((y.sin().sum(), s.sum()), (x, w), create_graph=True)
    for a, c in zip(plain, kept):
        assert torch.equal(a, c)
    with pytest.raises(RuntimeError, match="differentiable once"):
        kept[0].sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(AyoloError, match="forward-mode"):
            layer_norm(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)))
    y = layer_norm(x, w)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_in_place_use_of_the_outputs():
    """y may be changed in place (backward does not read it), the sum may not"""
    from ayolov2_amd.functional import layer_norm
    x = _make((2, 24, 3, 5), torch.float32, 1).cuda().requires_grad_()
    gy = _make((2, 24, 3, 5), torch.float32, 2).cuda()
    y = layer_norm(x, dim=1)
    want = torch.autograd.grad(y, x, 2 * gy)[0]
    y = layer_norm(x, dim=1)
    y.mul_(2.0)
    assert torch.equal(torch.autograd.grad(y, x, gy)[0], want)
    y, s = layer_norm(x, residual=x.detach(), dim=1)
    s.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (y + s).sum().backward()


def test_gradient_against_differences():
    """Directional derivative of sum(y * g) by central differences of the kernel's own fp32 forward: step h = 2^-6, error
    h^2 / 6 * |third derivative| (about 1e-4 of the value at unit scale) + 2 * 64 u * |y g| / h."""
    from ayolov2_amd.functional import layer_norm
    x = _make((4, 64), torch.float32, 1, 1.0, 0.0).cuda().requires_grad_()
    g, d = _make((4, 64), torch.float32, 2, 1.0, 0.0).cuda(), _make((4, 64), torch.float32, 3, 1.0, 0.0).cuda()
    w, b = (t.cuda() for t in _params(64, torch.float32, 4))
    f = lambda v: float((layer_norm(v, w, b).double() * g).sum())  # noqa: E731
    grad = torch.autograd.grad(layer_norm(x, w, b), x, g)[0]
    h = 2.0 ** -6
    with torch.no_grad():
        num = (f(x + h * d) - f(x - h * d)) / (2 * h)
    ana = float((grad.double() * d.double()).sum())
    scale = float(grad.double().norm() * d.double().norm())
    assert abs(num - ana) <= 10 * h * h / 6 * scale + 2 * 64 * U * float(g.abs().sum()) * 4 / h


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_large_offset_rows(dt):
    """Rows whose mean is far above their spread: the variance is formed from differences."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(64, 512, generator=g) + 1000.0).to(dt)
    _check(x, *_params(512, torch.float32, 2), 1e-5, gy=_make((64, 512), dt, 3, 1.0, 0.0))


def test_special_values_stay_in_their_row():
    from ayolov2_amd.functional import layer_norm
    x = _make((9, 130), torch.float16, 1).cuda()
    clean = layer_norm(x)
    x[2, 5], x[4, 129], x[6, 0] = float("nan"), float("inf"), float("-inf")
    y = layer_norm(x)
    for k in range(9):
        if k in (2, 4, 6):
            assert torch.isnan(y[k]).all()
        else:
            assert torch.equal(y[k], clean[k])


def test_constant_rows_and_zero_eps():
    from ayolov2_amd.functional import layer_norm
    x = torch.full((3, 40), 2.5, device="cuda")
    assert torch.equal(layer_norm(x), torch.zeros_like(x))                        # var 0: 0 * 1 / sqrt(eps)
    _check(_make((3, 40), torch.float32, 1), None, None, 0.0, gy=_make((3, 40), torch.float32, 2, 1.0, 0.0))


def test_same_bits_in_every_run_and_on_another_stream():
    from ayolov2_amd.functional import layer_norm
    x = _make((5000, 200), torch.bfloat16, 1).cuda().requires_grad_()
    w, b = (t.cuda().requires_grad_() for t in _params(200, torch.float32, 2))
    gy = _make((5000, 200), torch.bfloat16, 3, 1.0, 0.0).cuda()

    def run():
        y = layer_norm(x, w, b)
        return (y, *torch.autograd.grad(y, (x, w, b), gy))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_captured_forward_and_backward_replay():
    from ayolov2_amd.functional import layer_norm
    x = _make((300, 96), torch.float16, 1).cuda().requires_grad_()
    w, b = (t.cuda().requires_grad_() for t in _params(96, torch.float32, 2))
    gy = _make((300, 96), torch.float16, 3, 1.0, 0.0).cuda()

    def run():
        y, s = layer_norm(x, w, b, residual=x.detach())
        return (y, s, *torch.autograd.grad((y, s), (x, w, b), (gy, gy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    with torch.cuda.graph(graph2):
        outs2 = run()
    for k in range(4):
        with torch.no_grad():
            x.copy_(_make((300, 96), torch.float16, 10 + k))
            gy.copy_(_make((300, 96), torch.float16, 20 + k, 1.0, 0.0))
        want = run()
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        for a, a2, c in zip(outs, outs2, want):
            assert torch.equal(a, c) and torch.equal(a2, c)


def test_offsets_past_32_bits():
    """4.3e9 elements: the rows at both ends and around the 2^31st and 2^32nd element against the same rows on their own."""
    from ayolov2_amd.functional import layer_norm
    C, rows = 8192, (1 << 19) + 2
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    picks = [0, (1 << 18) - 1, 1 << 18, (1 << 19) - 1, 1 << 19, rows - 1]
    part = _make((len(picks), C), torch.bfloat16, 1).cuda()
    x[picks] = part
    x.requires_grad_()
    w = _params(C, torch.float32, 2)[0].cuda()
    y = layer_norm(x, w)
    assert torch.equal(y[picks], layer_norm(part, w))
    gy = torch.zeros_like(y)
    gpart = _make((len(picks), C), torch.bfloat16, 3, 1.0, 0.0).cuda()
    gy[picks] = gpart
    dx = torch.autograd.grad(y, x, gy)[0]
    part.requires_grad_()
    want = torch.autograd.grad(layer_norm(part, w), part, gpart)[0]
    assert torch.equal(dx[picks], want)


def test_module_and_yaml_row():
    """A LayerNorm row of the model yaml: forward and backward of the whole model against the same model with torch's layer norm."""
    import os

    import yaml

    import ayolov2_amd
    from ayolov2_amd import LayerNorm, YOLOModel
    cfg = yaml.safe_load(open(os.path.join(os.path.dirname(ayolov2_amd.__file__), "configs", "yolov5n.yaml")))
    cfg["backbone"].append([-1, 1, "LayerNorm", []])
    at = len(cfg["backbone"]) - 1                           # the head reads the normed map in the place of the last one
    cfg["head"][-1][0] = [at if f == at - 1 else f for f in cfg["head"][-1][0]]
    assert at in cfg["head"][-1][0]
    torch.manual_seed(0)
    m = YOLOModel(cfg).cuda().train()
    norms = [k for k in m.modules() if isinstance(k, LayerNorm)]
    assert len(norms) == 1 and norms[0].weight.shape[0] == m.model[at - 1].cv3.conv.out_channels
    x = torch.rand(2, 3, 64, 64, device="cuda")

    def run():
        m.zero_grad(set_to_none=True)
        raws = m(x)
        sum(r.square().mean() for r in raws).backward()
        return raws, norms[0].weight.grad.clone(), m.model[0].conv.weight.grad.clone()

    stats = {k: v.clone() for k, v in m.state_dict().items()}
    got = run()
    m.load_state_dict(stats)
    n = norms[0]
    n.forward = lambda t: torch.nn.functional.layer_norm(t.permute(0, 2, 3, 1), (n.weight.shape[0],), n.weight, n.bias, n.eps).permute(0, 3, 1, 2)
    want = run()
    # the model behind the norm is fp32 throughout: the oracle tests of these models allow 1e-4 of the logits, 2e-3 of gradients
    for a, c in zip(got[0], want[0]):
        assert float((a - c).abs().max()) <= 1e-4 * float(c.abs().max())
    for a, c in zip(got[1:], want[1:]):
        assert float((a - c).abs().max()) <= 2e-3 * float(c.abs().max())

"""Calls of the training operators on the GPU that their documentation allows or refuses and that a caller makes by the way."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rand(shape, seed, scale=1.0, dt=torch.float32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt).cuda()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1, 130, 2048, 5003])
def test_a_gradient_that_is_its_own_parameter(n, bits):
    """The gradient of a square's half: the step is the one with a copy of it, bit for bit; also where a moment serves as gradient."""
    from ayolov2_amd.optim import adamw_step, new_moment8

    def run(own, of):
        p, t = _rand(n, 1), torch.full((), 3.0, device="cuda")
        m, v = (new_moment8(p), new_moment8(p)) if bits == 8 else (_rand(n, 2, 0.1), _rand(n, 3, 0.1).square())
        g = {"p": p, "m": m, "v": v}[of]
        adamw_step([p], [g if own else g.clone()], [m], [v], [t], lr=1e-2, seed=5)
        return [p, t, *(m if bits == 8 else [m]), *(v if bits == 8 else [v])]

    for of in ("p",) if bits == 8 else ("p", "m", "v"):
        for x, y in zip(run(True, of), run(False, of)):
            assert torch.equal(x, y)


def test_what_shares_memory_is_refused():
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import adamw_step, clip_grads_, new_moment8, unpack_moments
    big, t = torch.zeros(900, device="cuda"), torch.zeros((), device="cuda")
    z = lambda: torch.zeros(300, device="cuda")  # noqa: E731
    with pytest.raises(AyoloError, match="share memory"):
        adamw_step([big[:300]], [big[1:301]], [z()], [z()], [t], lr=1e-3)
    with pytest.raises(AyoloError, match="share memory"):
        adamw_step([z()], [z()], [z()], [z()], [t], lr=t)
    with pytest.raises(AyoloError, match="share memory"):
        clip_grads_([big], 1.0, big[5])
    m = [new_moment8(z()), new_moment8(z())]
    with pytest.raises(AyoloError, match="share memory"):
        unpack_moments(m, True, [big[:300], big[200:500]])
    assert not big.any() and float(t) == 0.0
    # the same moment twice, the same gradient twice: only read
    a, b = unpack_moments([m[0], m[0]], True, [big[:300], big[300:600]])
    adamw_step([big[:300], big[300:600]], [big[600:900], big[600:900]], [z(), z()], [z(), z()], [t, torch.zeros((), device="cuda")], lr=1e-3)
    assert float(t) == 1.0 and not a.any() and not b.any()


def test_layer_norm_is_not_traced():
    """A trace would hold the call's buffers and not its kernel; whoever traces is told so."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.functional import layer_norm
    x = _rand((4, 24), 1)
    with pytest.raises(AyoloError, match="traced"):
        torch.jit.trace(lambda t: layer_norm(t) + 1.0, x, check_trace=False)
    for kw in ({}, {"tracing_mode": "fake"}):
        with pytest.raises(AyoloError, match="traced"):
            make_fx(lambda t: layer_norm(t) + 1.0, **kw)(x)
    y = layer_norm(x)                                      # and goes on afterwards
    assert torch.equal(y, layer_norm(x.clone()))


def test_modes_that_only_watch():
    """a dispatch mode that watches the calls (no tracer) leaves the operator as it is"""
    from torch.utils._python_dispatch import TorchDispatchMode

    from ayolov2_amd.functional import layer_norm

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x = _rand((4, 24), 1).requires_grad_()
    want = layer_norm(x)
    gw = torch.autograd.grad(want, x, x.detach())[0]
    with Watch():
        y = layer_norm(x)
        g = torch.autograd.grad(y, x, x.detach())[0]
    assert torch.equal(y, want) and torch.equal(g, gw)


def test_layer_norm_needs_tensors_with_memory():
    """Transforms' and wrapping tensors have no memory of their own: refused, a gain above all, which would count as none."""
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.functional import layer_norm

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError(str(func))

    x, w = _rand((4, 24), 1), _rand((24,), 2)
    for kw in (dict(weight=Wrapper(w)), dict(bias=Wrapper(w)), dict(residual=Wrapper(x))):
        with pytest.raises(AyoloError, match="memory of its own"):
            layer_norm(x, **kw)
    with pytest.raises(AyoloError, match="memory of its own"):
        layer_norm(Wrapper(x), w)
    with pytest.raises(AyoloError, match="memory of its own"):
        torch.func.vmap(layer_norm)(_rand((3, 4, 24), 2))
    with pytest.raises(AyoloError, match="memory of its own"):
        torch.func.grad(lambda t: layer_norm(t).sum())(x)
    e = torch.empty(0, 24, device="cuda")                  # nothing to hold is not missing memory
    assert layer_norm(e, w).shape == (0, 24)


def test_pending_negation():
    """A view that stands for its memory's negative (what .imag of a conjugate is): inputs and output gradients of layer norm are
    what they stand for; the lists' kernels, which read memory, refuse it."""
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.functional import layer_norm
    from ayolov2_amd.optim import clip_grads_, grad_norm
    x, r, gy, w, b = _rand((6, 40), 1), _rand((6, 40), 2), _rand((6, 40), 3), _rand((40,), 4), _rand((40,), 5)
    neg = torch._neg_view
    assert neg(x).is_neg()

    def run(x, r, w, b, gy, gs):
        ops = [t.detach().requires_grad_() for t in (x, r, w, b)]
        y, s = layer_norm(*[ops[k] for k in (0, 2, 3)], residual=ops[1])
        return [y, s, *torch.autograd.grad((y, s), ops, (gy, gs))]

    for a, c in zip(run(neg(x), neg(r), neg(w), neg(b), neg(gy), neg(x)), run(-x, -r, -w, -b, -gy, -x)):
        assert torch.equal(a, c)
    with torch.no_grad():
        assert torch.equal(layer_norm(neg(x)), layer_norm(-x))
    z = torch.complex(x, r).requires_grad_()               # and where autograd itself makes such gradients
    layer_norm(z.conj().imag).sum().backward()
    assert torch.isfinite(torch.view_as_real(z.grad)).all()
    with pytest.raises(AyoloError, match="strided tensor"):
        grad_norm([neg(x)])
    with pytest.raises(AyoloError, match="strided tensor"):
        clip_grads_([neg(x)], 1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_counts_what_it_writes(bits):
    """autograd notices that a moment or step count it has saved was changed, as with torch.optim.AdamW"""
    from ayolov2_amd.optim import adamw_step, new_moment8
    p = [_rand(300, 1), _rand(300, 2)]
    make = (lambda: [new_moment8(x) for x in p]) if bits == 8 else (lambda: [torch.zeros_like(x) for x in p])
    m, v, t = make(), make(), [torch.zeros((), device="cuda") for _ in p]
    parts = lambda s: list(s) if bits == 8 else [s]  # noqa: E731
    watched = [[p[k], *parts(m[k]), *parts(v[k]), t[k]] for k in range(2)]
    before = [[x._version for x in w] for w in watched]
    adamw_step(p, [_rand(300, 3), None], m, v, tuple(t), lr=1e-2)
    assert all(x._version > n for x, n in zip(watched[0], before[0])) and [x._version for x in watched[1]] == before[1]
    if bits == 32:
        w = torch.ones(300, device="cuda", requires_grad=True)
        loss = (w * m[0]).sum()
        adamw_step(p, [_rand(300, 3), None], m, v, t, lr=1e-2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_layer_norms_backward_is_not_traced():
    """a gradient taken inside a trace, of a norm computed before it"""
    from torch.fx.experimental.proxy_tensor import make_fx

    from ayolov2_amd.functional import layer_norm
    x = _rand((4, 24), 1).requires_grad_()
    y = layer_norm(x)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda g: torch.autograd.grad(y, x, g, retain_graph=True)[0] + 1.0)(_rand((4, 24), 2))
    assert torch.isfinite(torch.autograd.grad(y, x, x.detach())[0]).all()


@pytest.mark.parametrize("leaf", [True, False])
def test_the_residual_is_the_input_itself(leaf):
    """and gradients that the norm hands to two leaves are two tensors"""
    from ayolov2_amd.functional import layer_norm
    base, gy, gs = _rand((7, 96), 1), _rand((7, 96), 2), _rand((7, 96), 3)
    a = base.clone().requires_grad_()
    x = a if leaf else a * 1.0
    y, s = layer_norm(x, residual=x)
    assert torch.equal(s, base + base)
    torch.autograd.backward((y, s), (gy, gs))
    b = (base + base).requires_grad_()
    ds = torch.autograd.grad(layer_norm(b), b, gy)[0] + gs
    # 2 ds, ds rounded once more here than there: 2 u of its terms
    assert ((a.grad.double() - 2 * ds.double()).abs() <= 4 * 2.0 ** -24 * (2 * ds.abs() + 2 * gs.abs()).double()).all()
    p, q = base.clone().requires_grad_(), gs.clone().requires_grad_()
    y, s = layer_norm(p, residual=q)
    torch.autograd.backward((y, s), (gy, gs))
    assert torch.equal(p.grad, q.grad) and p.grad.data_ptr() != q.grad.data_ptr()
    kept = gs.clone()
    p, q = base.clone().requires_grad_(), base.clone().requires_grad_()
    layer_norm(p, residual=q)[1].backward(gs)              # only the sum: its gradient goes on as it is
    p.grad.zero_()
    assert torch.equal(q.grad, kept) and torch.equal(gs, kept)


def test_a_model_with_a_layer_norm_row_in_use():
    """evaluation, evaluation with augmentations, a 16-bit copy, the moving average and a clipped step, against the same model with
    the norm in torch operations"""
    import copy
    import os

    import yaml

    import ayolov2_amd
    from ayolov2_amd import LayerNorm, YOLOModel
    from ayolov2_amd.losses import ComputeLoss
    from ayolov2_amd.optim import AdamW
    from ayolov2_amd.trainer import ModelEMA, training_step
    from ayolov2_amd.tta import inference_with_tta
    cfg = yaml.safe_load(open(os.path.join(os.path.dirname(ayolov2_amd.__file__), "configs", "yolov5n.yaml")))
    cfg["backbone"].append([-1, 1, "LayerNorm", []])
    at = len(cfg["backbone"]) - 1
    cfg["head"][-1][0] = [at if f == at - 1 else f for f in cfg["head"][-1][0]]
    hyp = dict(box=0.05, cls=0.5, cls_pw=1.0, obj=1.0, obj_pw=1.0, anchor_t=4.0, fl_gamma=0.0, label_smoothing=0.0)
    torch.manual_seed(0)
    m = YOLOModel(cfg).cuda()
    m.hyp, m.gr = hyp, 1.0

    def torchs(model):
        other = copy.deepcopy(model)
        for n in other.modules():
            if isinstance(n, LayerNorm):
                n.forward = lambda t, n=n: torch.nn.functional.layer_norm(
                    t.permute(0, 2, 3, 1).float(), (n.weight.shape[0],), n.weight.float(), n.bias.float(), n.eps).permute(0, 3, 1, 2).to(t.dtype)
        return other

    x = torch.rand(2, 3, 64, 96, generator=torch.Generator().manual_seed(1)).cuda()
    m.eval()
    with torch.no_grad():
        for a, c in ((m(x)[0], torchs(m)(x)[0]), (inference_with_tta(m, x, (1.0, 0.83), (None, 3))[0], inference_with_tta(torchs(m), x, (1.0, 0.83), (None, 3))[0])):
            # as the fp32 model tests: 1e-4 of the largest value
            assert a.shape == c.shape and float((a - c).abs().max()) <= 1e-4 * float(c.abs().max())
        h = copy.deepcopy(m).half()
        a, c = h(x.half())[0].float(), torchs(h)(x.half())[0].float()
        # fp16 activations from the norm on: some 10 layers of half a step (2^-11) each
        assert torch.isfinite(a).all() and float((a - c).abs().max()) <= 10 * 2.0 ** -11 * float(c.abs().max())
    m.train()
    ema = ModelEMA(m)
    before = {k: v.clone() for k, v in m.state_dict().items()}
    o = AdamW(m.parameters(), lr=1e-3, state_bits=8)
    targets = torch.tensor([[0, 3, 0.5, 0.5, 0.4, 0.3], [1, 7, 0.3, 0.6, 0.2, 0.5]]).cuda()
    training_step(m, ComputeLoss(m), o, torch.amp.GradScaler("cuda", init_scale=64.0), x, targets, max_norm=0.5, ema=ema)
    name = next(k for k in before if k.startswith(f"model.{at}.") and k.endswith("weight"))
    after = m.state_dict()[name]
    assert not torch.equal(after, before[name]) and torch.isfinite(after).all()
    d = ema.decay(1)
    # one step of the average: two products and a sum
    assert torch.allclose(ema.ema.state_dict()[name], d * before[name] + (1 - d) * after, rtol=4 * 2.0 ** -24, atol=4 * 2.0 ** -24)

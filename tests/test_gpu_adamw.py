"""Gradient norm, clipping and the AdamW step over many tensors against their definitions in 64 bits; 8-bit moments bit for bit
against the numpy oracle.

Tolerances.  One AdamW element is a chain of at most 16 fp32 operations (unit roundoff u = 2^-24): 16 u of each term, plus half a
step of a 16-bit parameter.  The norm is summed in fp64 and rounded once: 2 u.  Clipping multiplies by a factor of at most three
more roundings."""
import copy

import numpy as np
import pytest
import torch

from oracle import train_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U32
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [1, 2, 3, 4, 5, 127, 128, 129, 1023, 4095, 4096, 4097, 8193, 100003]


def _rand(n, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, generator=g) * scale).to(dt)


def _apart(t, off=0):
    """a copy on the GPU that starts `off` elements behind an allocation's start, guarded on both sides"""
    n = t.numel()
    big = torch.full((n + off + 8,), 77, dtype=t.dtype, device="cuda")
    v = big[off:off + n].view(t.shape)
    v.copy_(t)
    return v, big


def _guarded(pairs):
    """nothing was written outside the tensors"""
    for v, big in pairs:
        off = v.storage_offset()
        assert (big[:off] == 77).all() and (big[off + v.numel():] == 77).all()


# ------------------------------------------------------------------------------------------------------ norm and clipping
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("off", [0, 1, 3])
def test_norm_and_clip(dt, off):
    from ayolov2_amd.optim import clip_grads_, grad_norm
    host = [_rand(n, dt, k, 0.1 * (1 + k % 3)) for k, n in enumerate(SIZES)]
    dev = [_apart(t, off) for t in host]
    grads = [v for v, _ in dev]
    want = torch.cat([t.double() for t in host]).norm()
    norm = grad_norm(grads)
    assert norm.dtype == torch.float32 and abs(float(norm) - float(want)) <= 2 * U * float(want)
    versions = [g._version for g in grads]
    got = clip_grads_([*grads[:3], None, *grads[3:]], 1.5)
    assert torch.equal(got, norm)
    f = min(1.0, 1.5 / (float(want) + 1e-6))
    for g, t, v in zip(grads, host, versions):
        w = t.double() * f
        assert ((g.double().cpu() - w).abs() <= (ref.HALF_STEP[dt] * 1.001 + 6 * U) * w.abs() + ref.TINY[dt]).all()
        assert g._version > v
    _guarded(dev)
    # nothing to clip: unchanged bits
    kept = [g.clone() for g in grads]
    clip_grads_(grads, 1e9)
    for g, k in zip(grads, kept):
        assert torch.equal(g, k)


def test_norm_over_many_tensors_of_mixed_types():
    from ayolov2_amd.optim import grad_norm
    host = [_rand(1 + 37 * k % 5000, TYPES[k % 3], k) for k in range(500)]
    want = float(torch.cat([t.double() for t in host]).norm())
    assert abs(float(grad_norm([t.cuda() for t in host])) - want) <= 2 * U * want
    scale = torch.tensor(1024.0, device="cuda")
    assert abs(float(grad_norm([t.cuda() for t in host], scale)) - want / 1024) <= 2 * U * want / 1024


@pytest.mark.parametrize("values,want", [([3e30, 4e30], 5e30), ([3e-30, 4e-30], 5e-30), ([0.0, 0.0], 0.0), ([float("inf"), 1.0], float("inf")),
                                         ([float("nan"), 1.0], float("nan"))])
def test_norm_range(values, want):
    """squares leave the range of fp32 and the norm does not"""
    from ayolov2_amd.optim import clip_grads_, grad_norm
    g = torch.tensor(values, device="cuda")
    n = float(grad_norm([g]))
    assert n == pytest.approx(want, rel=2 * U, nan_ok=True)
    clip_grads_([g], 1.0)
    t = torch.tensor(values)
    want_g = t * min(1.0, 1.0 / (want + 1e-6)) if want == want else t * float("nan")
    assert torch.allclose(g.cpu(), want_g, rtol=8 * U, atol=0, equal_nan=True)


def test_norm_of_empty_and_strided_gradients():
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import clip_grads_, grad_norm
    e = torch.empty(0, device="cuda")
    assert float(grad_norm([e])) == 0.0
    t = _rand(64, torch.float32, 1).view(8, 8).cuda()
    s = t[:, ::2]
    assert abs(float(grad_norm([s, e, None])) - float(s.double().norm())) <= 2 * U * 10
    with pytest.raises(AyoloError, match="dense"):
        clip_grads_([s], 1.0)
    with pytest.raises(AyoloError, match="share memory"):
        clip_grads_([t, t], 1.0)
    with pytest.raises(AyoloError, match="unsupported type"):
        grad_norm([t.double()])
    with pytest.raises(AyoloError, match="grad_scale"):
        grad_norm([t], torch.ones(2, device="cuda"))
    with pytest.raises(AyoloError, match="norm must"):
        clip_grads_([t], 1.0, torch.ones(()))


def test_clip_grad_norm_matches_torch():
    from ayolov2_amd.optim import clip_grad_norm_
    a = [torch.nn.Parameter(_rand((7, 5), torch.float32, 1).cuda()), torch.nn.Parameter(_rand((300,), torch.float32, 2).cuda())]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for k, (p, q) in enumerate(zip(a, b)):
        p.grad = _rand(p.shape, torch.float32, 5 + k).cuda()
        q.grad = p.grad.clone()
    n, m = clip_grad_norm_(a, 0.7), torch.nn.utils.clip_grad_norm_(b, 0.7)
    # torch sums in fp32 (at most log2-many levels of 335 terms: 16 u)
    assert abs(float(n) - float(m)) <= 16 * U * float(m)
    for p, q in zip(a, b):
        assert torch.allclose(p.grad, q.grad, rtol=32 * U, atol=0)
    a[0].grad[0, 0] = float("nan")
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(a, 0.7, error_if_nonfinite=True)


# ------------------------------------------------------------------------------------------------------------- 32 bits
def _check_p(got, want, p0, step, dt):
    tol = ref.HALF_STEP[dt] * 1.001 * want.abs() + ref.TINY[dt] + 16 * U * (p0.double().abs() + step.abs())
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("off", [0, 1, 2])
@pytest.mark.parametrize("b1,b2,eps,t0", [(0.9, 0.999, 1e-8, 0), (0.9, 0.95, 1e-6, 1000), (0.0, 0.99, 1e-3, 3), (0.5, 0.0, 1e-2, 0)])
def test_adamw_32(dt, off, b1, b2, eps, t0):
    from ayolov2_amd.optim import adamw_step
    lrs, wds = [1e-3 * (1 + k % 3) for k in range(len(SIZES))], [0.1 * (k % 2) for k in range(len(SIZES))]
    host = [[_rand(n, dt, 10 * k, 0.5), _rand(n, dt, 10 * k + 1, 0.01), _rand(n, torch.float32, 10 * k + 2, 0.003 if t0 else 0.0),
             _rand(n, torch.float32, 10 * k + 3, 0.01 if t0 else 0.0).square()] for k, n in enumerate(SIZES)]
    dev = [[_apart(t, off) for t in row] for row in host]
    steps = torch.full((len(SIZES),), float(t0), device="cuda")
    p, g, m, v = ([row[i][0] for row in dev] for i in range(4))
    adamw_step(p, g, m, v, list(steps.unbind()), lr=lrs, betas=(b1, b2), eps=eps, weight_decay=wds)
    assert (steps == t0 + 1).all()
    for k, (hp, hg, hm, hv) in enumerate(host):
        wp, wm, wv = ref.adamw(hp, hg, hm, hv, t0 + 1, lrs[k], b1, b2, eps, wds[k])
        g64 = hg.double()
        assert ((m[k].double().cpu() - wm).abs() <= 4 * U * (b1 * hm.double().abs() + (1 - b1) * g64.abs()) + 2.0 ** -149).all()
        assert ((v[k].double().cpu() - wv).abs() <= 6 * U * wv + 2.0 ** -148).all()
        # sqrt and 1 / (.) of a v that is 6 u off, m 4 u of its terms
        terms = lrs[k] * (b1 * hm.double().abs() + (1 - b1) * g64.abs()) / (1 - b1 ** (t0 + 1)) / ((wv / (1 - b2 ** (t0 + 1))).sqrt() + eps)
        _check_p(p[k], wp, hp, terms, dt)
        assert torch.equal(g[k].cpu(), hg)
    for row in dev:
        _guarded(row)


def test_adamw_many_tensors_and_skipped_ones():
    """more tensors than one launch (or one prepare launch) takes, some without a gradient, types mixed"""
    from ayolov2_amd.optim import adamw_step
    n = 700
    sizes = [1 + 61 * k % 900 for k in range(n)]
    host = [[_rand(s, TYPES[(k // 7) % 3], 4 * k), _rand(s, TYPES[(k // 7) % 3], 4 * k + 1), torch.zeros(s), torch.zeros(s)] for k, s in enumerate(sizes)]
    dev = [[t.cuda() for t in row] for row in host]
    on = [k % 5 != 2 for k in range(n)]
    steps = torch.zeros(n, device="cuda")
    adamw_step([r[0] for r in dev], [r[1] if o else None for r, o in zip(dev, on)], [r[2] if o else None for r, o in zip(dev, on)],
               [r[3] if o else None for r, o in zip(dev, on)], list(steps.unbind()), lr=1e-2)
    assert torch.equal(steps.cpu(), torch.tensor([float(o) for o in on]))
    for k in range(n):
        if not on[k]:
            assert torch.equal(dev[k][0].cpu(), host[k][0])
            continue
        wp, _, _ = ref.adamw(*host[k], 1, 1e-2, 0.9, 0.999, 1e-8, 1e-2)
        # the first step is lr * g / (|g| + eps) whatever g: the terms are lr
        _check_p(dev[k][0], wp, host[k][0], torch.full_like(wp, 1e-2), host[k][0].dtype)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_a_learning_rate_and_decay_per_tensor(bits):
    """more different pairs than one prepare launch holds"""
    from ayolov2_amd.optim import adamw_step, new_moment8
    n = 150
    host = [[_rand(100 + k, torch.float32, 2 * k), _rand(100 + k, torch.float32, 2 * k + 1)] for k in range(n)]
    p, g = [h[0].cuda() for h in host], [h[1].cuda() for h in host]
    state = (lambda: [new_moment8(x) for x in p]) if bits == 8 else (lambda: [torch.zeros_like(x) for x in p])
    steps, lrs, wds = torch.zeros(n, device="cuda"), [1e-3 * (k + 1) for k in range(n)], [0.01 * (k % 7) for k in range(n)]
    adamw_step(p, g, state(), state(), list(steps.unbind()), lr=lrs, weight_decay=wds)
    assert (steps == 1).all()
    for k, (hp, hg) in enumerate(host):
        wp, _, _ = ref.adamw(hp, hg, torch.zeros_like(hp), torch.zeros_like(hp), 1, lrs[k], 0.9, 0.999, 1e-8, wds[k])
        _check_p(p[k], wp, hp, torch.full_like(wp, lrs[k]), torch.float32)


def test_adamw_clipped_scaled_skipped_maximized():
    from ayolov2_amd.optim import adamw_step, grad_norm
    hp, hg = _rand(5000, torch.float32, 1), _rand(5000, torch.float32, 2)
    scale = torch.tensor(512.0, device="cuda")
    m0, v0 = _rand(5000, torch.float32, 3, 0.01), _rand(5000, torch.float32, 4, 0.1).square()

    def run(found, maximize=False, lr=1e-3):
        p, g, m, v, t = hp.cuda(), (hg * 512).cuda(), m0.cuda(), v0.cuda(), torch.full((), 9.0, device="cuda")
        norm = grad_norm([g], scale)
        adamw_step([p], [g], [m], [v], [t], lr=lr, total_norm=norm, max_norm=2.0, grad_scale=scale,
                   found_inf=torch.full((), found, device="cuda"), maximize=maximize)
        return p, m, v, t

    p, m, v, t = run(1.0)
    assert torch.equal(p.cpu(), hp) and torch.equal(m.cpu(), m0) and torch.equal(v.cpu(), v0) and float(t) == 9.0
    f = min(1.0, 2.0 / (float(hg.double().norm()) + 1e-6))
    for sign in (1.0, -1.0):
        p, m, v, t = run(0.0, sign < 0)
        wp, wm, wv = ref.adamw(hp, hg * sign, m0, v0, 10, 1e-3, 0.9, 0.999, 1e-8, 1e-2, f)
        assert float(t) == 10.0
        assert ((m.double().cpu() - wm).abs() <= 8 * U * (m0.double().abs() + hg.double().abs())).all()
        assert ((v.double().cpu() - wv).abs() <= 16 * U * wv).all()
        step = 1e-3 * (m0.double().abs() + hg.double().abs()) / (wv / (1 - 0.999 ** 10)).sqrt() / (1 - 0.9 ** 10)
        _check_p(p, wp, hp, step * 2, torch.float32)
    a = run(0.0, lr=torch.tensor(1e-3, device="cuda"))
    b = run(0.0, lr=1e-3)
    # the learning rate as a device scalar is fp32(1e-3), as an argument too
    assert torch.equal(a[0], b[0])


def test_adamw_special_gradients():
    """NaN and infinities reach their own element alone; zero gradients on zero states leave the parameter to its decay"""
    from ayolov2_amd.optim import adamw_step
    hp, hg = _rand(300, torch.float32, 1), _rand(300, torch.float32, 2)
    hg[5], hg[6], hg[299] = float("nan"), float("inf"), float("-inf")
    hg[10:20] = 0.0
    p, g, m, v, t = hp.cuda(), hg.cuda(), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros((), device="cuda")
    adamw_step([p], [g], [m], [v], [t], lr=1e-2, weight_decay=0.5)
    q = torch.nn.Parameter(hp.clone())
    q.grad = hg.clone()
    torch.optim.AdamW([q], lr=1e-2, weight_decay=0.5).step()
    assert torch.allclose(p.cpu(), q.detach(), rtol=1e-5, atol=1e-7, equal_nan=True)
    assert torch.isnan(p.cpu()).nonzero().flatten().tolist() == [5, 6, 299]
    assert torch.allclose(p.cpu()[10:20], hp[10:20] * (1 - 0.005), rtol=4 * U)


def test_adamw_refusals():
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import adamw_step, new_moment8
    mk = lambda n=8, dt=torch.float32: torch.zeros(n, dtype=dt, device="cuda")  # noqa: E731
    one = torch.zeros((), device="cuda")

    def refused(text, p=None, g=None, m=None, v=None, t=None, **kw):
        p, g, m, v, t = (d() if a is None else a for a, d in ((p, mk), (g, mk), (m, mk), (v, mk), (t, lambda: one)))
        with pytest.raises(AyoloError, match=text):
            adamw_step([p], [g], [m], [v], [t], **{"lr": 1e-3, **kw})

    refused("unsupported type", p=mk(dt=torch.float64))
    refused("type is not", g=mk(dt=torch.float16))
    refused("unsupported type", m=mk(dt=torch.float16))
    refused("sizes differ", v=mk(9))
    refused("sizes differ", g=mk(4))
    refused("not one number", t=mk(2))
    refused("unsupported type", t=one.double())
    refused("not on a GPU", t=torch.zeros(()))
    refused("not on a GPU", p=torch.zeros(8))
    refused("dense", p=mk(16)[::2])
    same = mk()
    refused("share memory", m=same, v=same)
    refused("share memory", p=same, m=same)
    refused("memory order", p=torch.zeros(2, 3, 4, 4, device="cuda").contiguous(memory_format=torch.channels_last),
            g=torch.zeros(2, 3, 4, 4, device="cuda"), m=torch.zeros(2, 3, 4, 4, device="cuda"), v=torch.zeros(2, 3, 4, 4, device="cuda"))
    refused("not a .codes, exponents. pair", m=new_moment8(mk()))
    refused("not a tensor", v=new_moment8(mk()))
    refused("exponents", m=tuple(new_moment8(mk(8))), v=(mk(8, torch.uint8), mk(2, torch.uint8)))
    refused("lr=", lr=-1.0)
    refused("lr=", lr=float("nan"))
    refused("2 values of lr", lr=[1.0, 2.0])
    refused("weight_decay", weight_decay=[-1.0])
    refused("lr", lr=[float("inf")])
    refused("betas", betas=(1.0, 0.9))
    refused("eps", eps=-1.0)
    refused("go together", max_norm=1.0)
    refused("max_norm", max_norm=-1.0, total_norm=one)
    refused("lr must", lr=torch.zeros(()))
    refused("found_inf", found_inf=one.half())
    with pytest.raises(AyoloError, match="share memory"):
        p = mk()
        adamw_step([p, p], [mk(), mk()], [mk(), mk()], [mk(), mk()], [one, one.clone()], lr=1e-3)
    with pytest.raises(AyoloError, match="share memory"):
        adamw_step([mk(), mk()], [mk(), mk()], [mk(), mk()], [mk(), mk()], [one, one], lr=1e-3)


# -------------------------------------------------------------------------------------------------------------- 8 bits
def _np8(p, g, mc, me, vc, ve, t, seed, position, b1=0.9, b2=0.999):
    """The moments after one step, one rounding per operation, and the codes they are kept as."""
    f = np.float32
    m, v, g = ref.decode(mc, me, True), ref.decode(vc, ve, False), g.float().numpy()
    with np.errstate(all="ignore"):
        m = m * f(b1) + g * f(1.0 - b1)
        v = v * f(b2) + g * g * f(1.0 - b2)
    rm, rv = ref.noise(seed, t, position, len(g))
    return m, v, ref.encode(m, rm, True), ref.encode(v, rv, False)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("off", [0, 1, 3])
def test_adamw_8_bit_for_bit(dt, off):
    from ayolov2_amd.optim import Moment8, adamw_step, unpack_moments
    host, dev, guards = [], [], []
    for k, n in enumerate(SIZES):
        p, g = _rand(n, dt, k), _rand(n, dt, 100 + k, 0.01) * torch.exp2(torch.randint(-12, 1, (n,), generator=torch.Generator().manual_seed(k)).float()).to(dt)
        if n >= 127:
            g[3], g[4], g[100] = float("nan"), float("inf"), float("-inf")
        host.append((p, g))
        nb = -(-n // 128)
        placed = [_apart(t, off) for t in (p, g, torch.zeros(n, dtype=torch.uint8), torch.zeros(n, dtype=torch.uint8),
                                           torch.zeros(nb, dtype=torch.uint8), torch.zeros(nb, dtype=torch.uint8))]
        guards += placed
        dev.append([v for v, _ in placed])
    steps = torch.zeros(len(SIZES), device="cuda")
    ms, vs = [Moment8(d[2], d[4]) for d in dev], [Moment8(d[3], d[5]) for d in dev]
    state = [(np.zeros(n, np.uint8), np.zeros(-(-n // 128), np.uint8)) * 2 for n in SIZES]
    for t in (1, 2, 3):
        before = [d[0].double().cpu() for d in dev]
        adamw_step([d[0] for d in dev], [d[1] for d in dev], ms, vs, list(steps.unbind()), lr=1e-3, seed=7)
        for k, (p, g) in enumerate(host):
            mc, me, vc, ve = state[k]
            m, v, (mc, me), (vc, ve) = _np8(p, g, mc, me, vc, ve, t, 7, k)
            state[k] = (mc, me, vc, ve)
            for got, want, what in ((dev[k][2], mc, "m"), (dev[k][4], me, "m's exponents"), (dev[k][3], vc, "v"), (dev[k][5], ve, "v's exponents")):
                assert np.array_equal(got.cpu().numpy(), want), (what, t, SIZES[k], np.flatnonzero(got.cpu().numpy() != want)[:5])
            ok = np.isfinite(m)
            with np.errstate(all="ignore"):
                step = 1e-3 * (m.astype(np.float64) / (1 - 0.9 ** t)) / (np.sqrt(v.astype(np.float64) / (1 - 0.999 ** t)) + 1e-8)
            want = before[k] - 1e-3 * 1e-2 * before[k] - torch.from_numpy(step)
            err = (dev[k][0].double().cpu() - want).abs()
            tol = ref.HALF_STEP[dt] * 1.001 * want.abs() + ref.TINY[dt] + 16 * U * (before[k].abs() + torch.from_numpy(np.abs(step)))
            assert (err <= tol)[torch.from_numpy(ok)].all()
            assert torch.isnan(dev[k][0].cpu())[torch.from_numpy(~ok)].all()
    for k in range(len(SIZES)):
        for mom, signed, (c, e) in ((ms[k], True, state[k][:2]), (vs[k], False, state[k][2:])):
            got = unpack_moments([mom], signed)[0].cpu().numpy()
            assert np.array_equal(got, ref.decode(c, e, signed), equal_nan=True)
    _guarded(guards)


def test_unpack_many_into_given_tensors():
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import Moment8, unpack_moments
    g = torch.Generator().manual_seed(0)
    ms, outs = [], []
    for k in range(300):
        n = 1 + 37 * k % 1000
        ms.append(Moment8(torch.randint(0, 256, (n,), generator=g).byte().cuda(), torch.randint(1, 255, (-(-n // 128),), generator=g).byte().cuda()))
        outs.append(_apart(torch.zeros(n), k % 4))
    for signed in (True, False):
        res = unpack_moments(ms, signed, [v for v, _ in outs])
        for m, o in zip(ms, res):
            assert np.array_equal(o.cpu().numpy(), ref.decode(m[0].cpu().numpy(), m[1].cpu().numpy(), signed), equal_nan=True)
    _guarded(outs)
    with pytest.raises(AyoloError, match="outputs"):
        unpack_moments(ms, True, outs[:2])
    with pytest.raises(AyoloError, match="sizes"):
        unpack_moments([Moment8(ms[0].codes, ms[200].exps)], True)


def test_8_bit_moments_follow_the_32_bit_ones():
    """Constant-variance gradients over 3000 steps: the second moment must neither stick nor drift.  With rounding to nearest a
    3-bit mantissa holds v where it was once 0.1 % of a step is below half a code; here E[v] is exact.  Standard deviation of v
    from the rounding alone: a step's variance is at most frac * code^2 with frac = 0.1 % / 12.5 %..6.25 %, code <= 12.5 %, i.e.
    <= 1.25e-4 v^2, summed by the average over 1 / (2 * 0.001) steps: below 0.25 v.  The mean over 4096 elements is then within
    5 * 0.25 / 64 = 2 % of the 32-bit mean."""
    from ayolov2_amd.optim import adamw_step, new_moment8, unpack_moments
    n = 4096
    p8 = torch.zeros(n, device="cuda")
    p32 = p8.clone()
    m8, v8 = new_moment8(p8), new_moment8(p8)
    m32, v32 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    t8, t32 = torch.zeros((), device="cuda"), torch.zeros((), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(3000):
        g = torch.randn(n, generator=gen, device="cuda") * 1e-3
        adamw_step([p8], [g], [m8], [v8], [t8], lr=1e-3)
        adamw_step([p32], [g], [m32], [v32], [t32], lr=1e-3)
    a, b = float(unpack_moments([v8], False)[0].mean()), float(v32.mean())
    assert abs(a / b - 1) <= 0.02
    a = unpack_moments([m8], True)[0]
    assert abs(float((a - m32).mean())) <= 5 * float(m32.std()) / 64      # unbiased as well


# ---------------------------------------------------------------------------------------------------------- optimiser class
def _params(seed, device="cuda", dt=torch.float32):
    shapes = [(32,), (64, 32, 3, 3), (255,), (16, 8, 1, 1), (7,), (128, 64, 1, 1), (3, 5)]
    ps = []
    for i, sh in enumerate(shapes):
        t = _rand(sh, dt, seed + i)
        if len(sh) == 4 and i % 2 == 1:
            t = t.contiguous(memory_format=torch.channels_last)
        ps.append(torch.nn.Parameter(t.to(device)))
    return ps


def _groups(ps):
    return [{"params": [ps[0], ps[4]], "weight_decay": 0.0}, {"params": [ps[1], ps[3], ps[5], ps[6]], "weight_decay": 0.1},
            {"params": [ps[2]], "lr": 3e-3, "betas": (0.8, 0.99)}]


def _train(opt, ps, steps, seed, skip=()):
    for k in range(steps):
        for i, p in enumerate(ps):
            g = _rand(p.shape, torch.float32, 1000 * seed + 10 * k + i, 0.1).to(p.dtype)
            # a gradient in a different memory order than the parameter must still be applied element by element
            p.grad = None if (k, i) in skip else g.to(p.device) if k % 2 else g.to(p.device).contiguous()
        opt.step()
        for gr in opt.param_groups:                        # schedulers rewrite the learning rate
            gr["lr"] *= 0.9


def test_class_matches_torch_and_shares_state_dicts():
    from ayolov2_amd.optim import AdamW
    a, b = _params(0), _params(0, "cpu")
    oa, ob = AdamW(_groups(a), lr=1e-2), torch.optim.AdamW(_groups(b), lr=1e-2)
    skip = {(0, 2), (1, 3)}
    _train(oa, a, 4, 1, skip)
    _train(ob, b, 4, 1, skip)
    # four steps of at most lr each, 16 u of the parameter and 32 u of the step per step on both sides
    close = lambda p, q: torch.allclose(p.detach().cpu(), q.detach().cpu(), rtol=8 * 16 * U, atol=8 * 64 * U * 1e-2 * 4 + 1e-8)  # noqa: E731
    for p, q in zip(a, b):
        assert close(p, q)
        assert float(oa.state[p]["step"]) == float(ob.state[q]["step"])
    # each loads the other's state dict and goes on
    c, d = _params(0), _params(0, "cpu")
    for src, dst in ((b, c), (a, d)):
        for p, q in zip(src, dst):
            q.data.copy_(p.detach())
    oc, od = AdamW(_groups(c), lr=1e-2), torch.optim.AdamW(_groups(d), lr=1e-2)
    oc.load_state_dict(ob.state_dict())
    od.load_state_dict({"state": {k: {n: t.cpu() for n, t in s.items()} for k, s in oa.state_dict()["state"].items()},
                        "param_groups": oa.state_dict()["param_groups"]})
    _train(oa, a, 2, 2)
    _train(oc, c, 2, 2)
    _train(od, d, 2, 2)
    for p, q, r in zip(a, c, d):
        assert close(p, q) and close(p, r)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_class_state_dict_round_trip(dt, tmp_path):
    """save, load, go on: the same bits as without; also through a deep copy, with 16-bit parameters and with 8-bit states"""
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import AdamW, unpack_moments
    for bits in (32, 8):
        a = _params(0, dt=dt)
        oa = AdamW(_groups(a), lr=1e-2, state_bits=bits, seed=3)
        _train(oa, a, 3, 1)
        torch.save(oa.state_dict(), tmp_path / "o.pt")
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        ob = AdamW(_groups(b), lr=1e-2, state_bits=bits, seed=3)
        ob.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
        for p, q in zip(a, b):
            for k, t in oa.state[p].items():
                u = ob.state[q][k]
                assert u.dtype == t.dtype and u.stride() == t.stride() and torch.equal(u, t) and u.data_ptr() != t.data_ptr()
        oc, c = copy.deepcopy((oa, a))
        for o, ps in ((oa, a), (ob, b), (oc, c)):
            _train(o, ps, 2, 2)
        for p, q, r in zip(a, b, c):
            assert torch.equal(p, q) and torch.equal(p, r)
    o32 = AdamW(_groups(b), lr=1e-2)
    o32.load_state_dict(oa.state_dict())                   # 8-bit states into 32-bit ones
    for p, q in zip(a, b):
        st = oa.state[p]
        assert torch.equal(o32.state[q]["exp_avg"], unpack_moments([(st["exp_avg"], st["exp_avg_exps"])], True)[0])
        assert set(o32.state[q]) == {"step", "exp_avg", "exp_avg_sq"}
    o8 = AdamW(_groups(a), lr=1e-2, state_bits=8)
    with pytest.raises(AyoloError, match="does not load"):
        o8.load_state_dict(o32.state_dict())


def test_class_with_gradscaler_and_clipping():
    from ayolov2_amd.optim import AdamW
    a, b = _params(0), _params(0, "cpu")
    oa, ob = AdamW(_groups(a), lr=1e-2, max_norm=0.5), torch.optim.AdamW(_groups(b), lr=1e-2)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    scaler.scale(torch.zeros(1, device="cuda"))
    for k in range(4):
        bad, scale = k in (0, 2), float(scaler.get_scale())
        for i, (p, q) in enumerate(zip(a, b)):
            q.grad = _rand(p.shape, torch.float32, 10 * k + i)
            p.grad = (q.grad * scale).to("cuda")
            if bad:
                p.grad.view(-1)[0] = float("inf")
        before = [p.detach().clone() for p in a]
        scaler.step(oa)
        scaler.update()
        if bad:
            assert all(torch.equal(p, q) for p, q in zip(a, before))
        else:
            torch.nn.utils.clip_grad_norm_(b, 0.5)
            ob.step()
            for p, q in zip(a, b):
                assert torch.allclose(p.detach().cpu(), q.detach(), rtol=8 * 16 * U, atol=8 * 64 * U * 1e-2 * 4 + 1e-8)
    assert {float(oa.state[p]["step"]) for p in a} == {2.0}


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay(bits):
    """A captured clipped step with a learning rate on the device, replayed with new gradients, against the same steps run eagerly;
    two graphs of two optimisers share nothing."""
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import AdamW
    make = lambda ps, lr: AdamW([{"params": ps[:3]}, {"params": ps[3:], "weight_decay": 0.0}], lr=lr, state_bits=bits, max_norm=0.3)  # noqa: E731
    sets = [_params(0) for _ in range(3)]
    lrs = [torch.tensor(1e-2, device="cuda") for _ in sets]
    opts = [make(ps, lr) for ps, lr in zip(sets, lrs)]
    for ps in sets:
        for p in ps:
            p.grad = torch.zeros_like(p)
    side = torch.cuda.Stream()
    with pytest.raises(AyoloError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opts[1].step()
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for o in opts:
            o.step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for o in opts[1:]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o.step()
        graphs.append(gr)
    for k in range(4):
        for ps, lr in zip(sets, lrs):
            for i, p in enumerate(ps):
                p.grad.copy_(_rand(p.shape, torch.float32, 100 * k + i))
            lr.fill_(1e-2 / (k + 1))
        opts[0].step()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(*sets):
            assert torch.equal(p, q) and torch.equal(p, r)
    assert float(opts[1].state[sets[1][0]]["step"]) == 5.0


def test_closure_and_no_gradients():
    from ayolov2_amd.optim import AdamW
    ps = _params(0)
    o = AdamW(ps, lr=1e-2)
    before = [p.detach().clone() for p in ps]
    o.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before))

    def closure():
        o.zero_grad()
        loss = sum(p.square().sum() for p in ps)
        loss.backward()
        return loss

    first = float(o.step(closure))
    assert first == pytest.approx(float(sum(p.double().square().sum() for p in before)), rel=1e-4)
    assert all(not torch.equal(p, q) for p, q in zip(ps, before))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_past_32_bits(bits):
    """A 16-bit tensor of 2^32 + 5 elements (several jobs): its ends and the places where 2^30, 2^31 and 2^32 are passed."""
    from ayolov2_amd.optim import adamw_step, clip_grads_, grad_norm, new_moment8, unpack_moments
    n = (1 << 32) + 5
    at = [0, 127, 128, (1 << 30) - 1, 1 << 30, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1]
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    p[at], g[at] = 1.0, torch.arange(1, len(at) + 1, dtype=torch.bfloat16, device="cuda")
    want = float(torch.arange(1, len(at) + 1).double().square().sum().sqrt())
    assert abs(float(grad_norm([g])) - want) <= 2 * U * want
    if bits == 8:
        m, v = new_moment8(p), new_moment8(p)
    else:
        m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    t = torch.zeros((), device="cuda")
    adamw_step([p], [g], [m], [v], [t], lr=0.25, weight_decay=0.0)
    assert (p[at] == 0.75).all() and int(torch.count_nonzero(p)) == len(at)     # the first step is lr * sign(g)
    if bits == 8:
        m = unpack_moments([m], True)[0]
    want_m = torch.arange(1, len(at) + 1, device="cuda") * 0.1
    assert ((m[at] - want_m).abs() <= want_m * (0.125 if bits == 8 else 4 * U)).all() and int(torch.count_nonzero(m)) == len(at)
    del m, v
    clip_grads_([g], want / 2)
    assert ((g[at].float() - torch.arange(1, len(at) + 1, device="cuda") / 2).abs() <= 2.0 ** -8 * 5).all()


def test_tensors_all_over_the_address_space():
    """Small tensors 5 GB apart, more such places than one launch's list can name."""
    from ayolov2_amd.optim import adamw_step, clip_grads_, grad_norm, new_moment8, unpack_moments
    n, blocks = 300, [torch.empty(5 << 30, dtype=torch.uint8, device="cuda") for _ in range(24)]
    used = [0] * len(blocks)

    def take(k, t):
        k %= len(blocks)
        v = blocks[k][used[k]:used[k] + t.numel() * t.element_size()].view(t.dtype)
        used[k] += 1 << 14
        v.copy_(t)
        return v

    host = [[_rand(n + k, torch.float32, 10 * k), _rand(n + k, torch.float32, 10 * k + 1, 0.1)] for k in range(60)]
    want = float(torch.cat([g for _, g in host]).double().norm())
    p, g = [take(k, h[0]) for k, h in enumerate(host)], [take(5 * k + 1, h[1]) for k, h in enumerate(host)]
    m, v, t = ([take(7 * k + j, torch.zeros(n + k)) for k in range(60)] for j in (2, 3, 4))
    t = [x[:1] for x in t]
    assert abs(float(grad_norm(g)) - want) <= 2 * U * want
    adamw_step(p, g, m, v, t, lr=1e-2)
    m8 = [new_moment8(x) for x in p]
    adamw_step([x.clone() for x in p], g, m8, [new_moment8(x) for x in p], [torch.zeros((), device="cuda") for _ in p], lr=1e-2)
    out = unpack_moments(m8, True, [take(11 * k + 3, torch.zeros(n + k)) for k in range(60)])
    clip_grads_(g, want / 2)
    for k, (hp, hg) in enumerate(host):
        wp, wm, wv = ref.adamw(hp, hg, torch.zeros(n + k), torch.zeros(n + k), 1, 1e-2, 0.9, 0.999, 1e-8, 1e-2)
        assert float(t[k]) == 1.0
        _check_p(p[k], wp, hp, torch.full_like(wp, 1e-2), torch.float32)
        assert ((m[k].double().cpu() - wm).abs() <= 4 * U * wm.abs()).all()
        assert ((out[k].double().cpu() - wm).abs() <= torch.maximum(wm.abs() / 8, wm.abs().max() * 2.0 ** -16)).all()
        assert ((g[k].double().cpu() - hg.double() / 2).abs() <= 8 * U * hg.double().abs()).all()


def test_two_threads_at_once():
    """Two host threads step two optimisers and run two norms, each on a stream of its own."""
    import threading

    from ayolov2_amd.functional import layer_norm
    from ayolov2_amd.optim import AdamW

    def work(seed):
        ps = _params(seed)
        x = _rand((500, 33), torch.float32, seed).cuda().requires_grad_()
        o = AdamW(_groups(ps), lr=1e-2, state_bits=8, max_norm=0.5)
        _train(o, ps, 8, seed)
        y = layer_norm(x)
        return [*ps, y, torch.autograd.grad(y, x, x.detach())[0]]

    want = [work(s) for s in (1, 2)]
    got, errors = [None, None], []

    def thread(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                got[k] = work(k + 1)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=thread, args=(k,)) for k in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_the_step_of_a_small_network():
    """Layer norm, its gradients, clipping and the step together, against float64; and the same steps captured once and replayed
    against eager ones (32- and 8-bit states)."""
    from ayolov2_amd.functional import layer_norm
    from ayolov2_amd.optim import AdamW
    x = _rand((64, 48), torch.float32, 1).cuda()
    init = [_rand((48, 48), torch.float32, 2, 0.15), torch.ones(48), torch.zeros(48)]

    def far(p, q):
        # an element whose gradient is near zero takes a step of its gradient's rounding's sign: at most 2 lr per step, and few of
        # them; the others agree to the gradients' rounding (48 terms: 64 u) over v's root
        d = (p.detach().double().cpu() - q.detach().double().cpu()).abs()
        return float(d.max()) > 3 * 2 * 1e-2 or float((d > 1e-5).double().mean()) > 0.01

    def step(ps, opt):
        y, s = layer_norm(x @ ps[0], ps[1], ps[2], residual=x)
        for p, g in zip(ps, torch.autograd.grad((y * y * y + s).mean(), ps)):
            p.grad = g
        opt.step()

    new = lambda: [torch.nn.Parameter(t.cuda()) for t in init]  # noqa: E731
    a, b = new(), [torch.nn.Parameter(t.double()) for t in init]
    oa, ob = AdamW(a, lr=1e-2, max_norm=1.0), torch.optim.AdamW(b, lr=1e-2)
    for _ in range(3):
        step(a, oa)
        x64 = x.double().cpu()
        s = x64 @ b[0] + x64
        y = torch.nn.functional.layer_norm(s, (48,), b[1], b[2], 1e-5)
        (y * y * y + s).mean().backward()
        torch.nn.utils.clip_grad_norm_(b, 1.0)
        ob.step()
        ob.zero_grad()
    assert not any(far(p, q) for p, q in zip(a, b))
    for bits in (32, 8):
        c, d = new(), new()
        oc, od = (AdamW(ps, lr=1e-2, max_norm=1.0, state_bits=bits) for ps in (c, d))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(c, oc)                                    # makes the states and warms the libraries up
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(c, oc)
        with torch.no_grad():
            for p, t in zip(c, init):
                p.copy_(t)
                for v in oc.state[p].values():
                    v.zero_()
        for _ in range(3):
            graph.replay()
            step(d, od)
            torch.cuda.synchronize()
            assert not any(far(p, q) for p, q in zip(c, d))
        assert float(oc.state[c[0]]["step"]) == 3.0


def test_training_step_clips():
    import os

    import ayolov2_amd
    from ayolov2_amd import YOLOModel
    from ayolov2_amd.losses import ComputeLoss
    from ayolov2_amd.optim import AdamW
    from ayolov2_amd.trainer import training_step
    cfg = os.path.join(os.path.dirname(ayolov2_amd.__file__), "configs", "yolov5n.yaml")
    hyp = dict(box=0.05, cls=0.5, cls_pw=1.0, obj=1.0, obj_pw=1.0, anchor_t=4.0, fl_gamma=0.0, label_smoothing=0.0)
    imgs = torch.rand(2, 3, 64, 64, generator=torch.Generator().manual_seed(0)).cuda()
    targets = torch.tensor([[0, 3, 0.5, 0.5, 0.4, 0.3], [1, 7, 0.3, 0.6, 0.2, 0.5]]).cuda()
    norms = []
    for how in ("own", "trainer", "scaler"):
        torch.manual_seed(0)
        m = YOLOModel(cfg).cuda().train()
        m.hyp, m.gr = hyp, 1.0
        o = AdamW(m.parameters(), lr=1e-3, betas=(0.0, 0.9), max_norm=0.1 if how == "own" else None)
        scaler = torch.amp.GradScaler("cuda", init_scale=256.0) if how == "scaler" else None
        training_step(m, ComputeLoss(m), o, scaler, imgs, targets, amp=False, max_norm=None if how == "own" else 0.1)
        # with beta1 = 0 the first moment IS the clipped gradient
        norms.append(float(torch.cat([o.state[p]["exp_avg"].reshape(-1).double() for p in m.parameters()]).norm()))
    # min(1, 0.1 / (n + 1e-6)) * n with n above 0.1, to the fp32 rounding of each element; the scaled run's gradients differ from
    # the unscaled ones' by their own roundings only
    for n in norms:
        assert abs(n - 0.1) <= 1e-5

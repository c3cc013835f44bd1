"""States of ``optim.AdamW`` that come from, or get into, another memory order than their parameter's.

An 8-bit moment's exponents belong to blocks of 128 codes in MEMORY order.  Taking it to another order means unpacking it in its
own order and forming new blocks: exact in 32 bits; in 8 bits each value is rounded once to nearest, i.e. by at most 1/16 of
itself, or below the normal codes by half a step (2^-17 of its new block's largest value for a first moment; for a second one
by a step, 2^-32, because a value above zero stays above zero)."""
import numpy as np
import pytest
import torch

from oracle import train_ref as ref

pytestmark = pytest.mark.gpu
SHAPES = [(64, 32, 3, 3), (40, 24, 3, 1), (7, 5, 3, 3), (130,), (16, 8, 1, 1)]
ORDERS = {"contiguous": torch.contiguous_format, "channels_last": torch.channels_last}


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def _in_order(t, order):
    return t.contiguous(memory_format=ORDERS[order]) if t.dim() == 4 else t


def _params(order, seed=0):
    return [torch.nn.Parameter(_in_order(_rand(s, seed + k, 0.1).cuda(), order)) for k, s in enumerate(SHAPES)]


def _copy_params(ps, order):
    return [torch.nn.Parameter(_in_order(p.detach().clone(memory_format=torch.contiguous_format), order)) for p in ps]


def _grads(ps, seed):
    """gradients whose size differs from input channel to input channel, so that blocks along them have other exponents"""
    for k, p in enumerate(ps):
        g = _rand(p.shape, 100 * seed + k, 0.01)
        if p.dim() == 4:
            g = g * torch.exp2(torch.arange(p.shape[1]) % 12 - 11.0).view(1, -1, 1, 1)
        p.grad = torch.empty_like(p).copy_(g)


def _steps(opt, ps, n, seed):
    for k in range(n):
        _grads(ps, seed + k)
        opt.step()


def _values(st, name):
    from ayolov2_amd.optim import unpack_moments
    return unpack_moments([(st[name], st[name + "_exps"])], name == "exp_avg")[0]


def _flat(t):
    """the elements in memory order"""
    return t.detach().as_strided((t.numel(),), (1,), t.storage_offset()).cpu().numpy()


def _repacked(values, codes, exps, signed):
    """`codes`, `exps` are what `values` (laid out as the codes are) round to, bit for bit, within the stated distance"""
    x = _flat(values)
    wc, we = ref.encode(x, np.full(x.size, 0x8000, np.uint32), signed)
    assert np.array_equal(_flat(codes), wc) and np.array_equal(_flat(exps), we)
    top = np.repeat(np.pad(np.abs(x), (0, -x.size % 128)).reshape(-1, 128).max(1), 128)[:x.size].astype(np.float64)
    err = np.abs(ref.decode(wc, we, signed).astype(np.float64) - x)
    assert (err <= np.maximum(np.abs(x) / 16.0, top * 2.0 ** (-17 if signed else -32))).all()


@pytest.mark.parametrize("where", ["cuda", "cpu"])
@pytest.mark.parametrize("src,dst", [("contiguous", "channels_last"), ("channels_last", "contiguous")])
def test_8_bit_states_load_into_another_memory_order(src, dst, where):
    from ayolov2_amd.optim import AdamW
    a = _params(src)
    oa = AdamW(a, lr=1e-3, state_bits=8, seed=3)
    _steps(oa, a, 5, 1)
    sd = oa.state_dict()
    if where == "cpu":
        sd = {"state": {i: {k: t.cpu() for k, t in s.items()} for i, s in sd["state"].items()}, "param_groups": sd["param_groups"]}
    b, c = _copy_params(a, dst), _copy_params(a, dst)
    o32, o8 = AdamW(b, lr=1e-3), AdamW(c, lr=1e-3, state_bits=8, seed=3)
    o32.load_state_dict(sd)
    o8.load_state_dict(sd)
    for p, q, r in zip(a, b, c):
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            want = _values(oa.state[p], name)
            got = o32.state[q][name]
            assert got.stride() == q.stride() and torch.equal(got, want)
            codes, exps = o8.state[r][name], o8.state[r][name + "_exps"]
            assert codes.stride() == r.stride()
            _repacked(got, codes, exps, signed)
            if p.stride() == r.stride():                   # nothing to re-lay: the same bytes
                assert torch.equal(codes, oa.state[p][name]) and torch.equal(exps, oa.state[p][name + "_exps"])
    # and they go on: the 32-bit optimiser from exactly the values that the 8-bit one held
    for o, ps in ((o32, b), (o8, c)):
        _steps(o, ps, 1, 77)
        assert all(float(o.state[p]["step"]) == 6.0 and torch.isfinite(p).all() for p in ps)


def _changed(sd, **state):
    """the state dict with entries of its first parameter's state replaced, or taken out (None)"""
    st = {k: v for k, v in {**sd["state"][0], **state}.items() if v is not None}
    return {"state": {**sd["state"], 0: st}, "param_groups": [{**g, "lr": 7.0} for g in sd["param_groups"]]}


@pytest.mark.parametrize("bits", [32, 8])
def test_refused_loads_change_nothing(bits):
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import AdamW
    ps = _params("channels_last")
    o = AdamW(ps, lr=1e-3, state_bits=bits)
    _steps(o, ps, 2, 1)
    other = AdamW(_copy_params(ps, "channels_last"), lr=1e-3, state_bits=40 - bits)
    _steps(other, other.param_groups[0]["params"], 1, 9)
    before = [{k: v.clone() for k, v in o.state[p].items()} for p in ps]
    sd, n = o.state_dict(), ps[0].numel()
    bad = [(_changed(sd, exp_avg=sd["state"][0]["exp_avg"][:1]), "shape"), (_changed(sd, exp_avg_sq=None), "no exp_avg_sq"),
           (_changed(sd, step=torch.zeros(2)), "one number")]
    if bits == 8:
        bytes_ = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")  # noqa: E731
        bad += [(other.state_dict(), "does not load"), (_changed(sd, exp_avg_exps=bytes_(n // 128 + 1)), "one byte"),
                (_changed(sd, exp_avg_exps=torch.zeros(n // 128, device="cuda")), "one byte"), (_changed(sd, exp_avg_sq_exps=None), "no exp_avg_sq_exps"),
                (_changed(sd, exp_avg=torch.zeros(ps[0].shape, device="cuda")), "codes"),
                (_changed(sd, exp_avg=bytes_(*ps[0].shape, 2)[..., 0]), "dense")]
    for d, text in bad:
        with pytest.raises(AyoloError, match=text):
            o.load_state_dict(d)
        assert all(g["lr"] == 1e-3 for g in o.param_groups)
        for p, st in zip(ps, before):
            assert set(o.state[p]) == set(st)
            for k, v in st.items():
                assert o.state[p][k].dtype == v.dtype and torch.equal(o.state[p][k], v)


@pytest.mark.parametrize("bits", [32, 8])
def test_load_hooks_are_heard(bits):
    from ayolov2_amd.optim import AdamW
    a, b = _params("contiguous"), _params("contiguous")
    oa, ob = AdamW(a, lr=1e-3, state_bits=bits), AdamW(b, lr=1e-3, state_bits=bits)
    _steps(oa, a, 3, 1)
    _steps(ob, b, 1, 5)
    given, seen = oa.state_dict(), []
    ob.register_load_state_dict_pre_hook(lambda _, sd: given)
    ob.register_load_state_dict_post_hook(lambda o: seen.extend(o.state[p]["exp_avg"].clone() for p in b))
    ob.load_state_dict(ob.state_dict())
    for p, q, s in zip(a, b, seen):
        for k, v in oa.state[p].items():
            assert ob.state[q][k].dtype == v.dtype and torch.equal(ob.state[q][k], v)
        assert torch.equal(s, oa.state[p]["exp_avg"])
    ob.register_load_state_dict_post_hook(lambda o: [o.state[p]["step"].fill_(40.0) for p in b])
    ob.load_state_dict(ob.state_dict())
    assert all(float(ob.state[q]["step"]) == 40.0 for q in b)


def _turn(ps, order):
    for p in ps:
        p.data = _in_order(p.data, order)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("src,dst", [("contiguous", "channels_last"), ("channels_last", "contiguous")])
def test_states_follow_their_parameters_memory_order(src, dst, bits):
    """Weights that change their memory order between two steps (the executors make weights channels-last at their first forward):
    as if the states had been saved before and loaded after; with 32-bit moments as if nothing had changed."""
    from ayolov2_amd.optim import AdamW
    a, b, c = _params(src), _params(src), _copy_params(_params(src), dst)
    oa, ob, oc = (AdamW(ps, lr=1e-3, state_bits=bits, seed=3, max_norm=0.5) for ps in (a, b, c))
    _steps(oa, a, 3, 1)
    _steps(ob, b, 3, 1)
    oc.load_state_dict(oa.state_dict())
    for p, r in zip(a, c):
        r.data.copy_(p.data)
    _turn(a, dst)
    for o, ps in ((oa, a), (ob, b), (oc, c)):
        _steps(o, ps, 2, 10)
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, r) and (bits == 8 or torch.equal(p, q))
        for k, v in oa.state[p].items():
            assert torch.equal(v, oc.state[r][k]) and (k not in ("exp_avg", "exp_avg_sq") or v.stride() == p.stride())


@pytest.mark.parametrize("bits", [32, 8])
def test_memory_order_changes_before_a_capture_not_inside(bits):
    from ayolov2_amd._lib import AyoloError
    from ayolov2_amd.optim import AdamW
    ps = _params("contiguous")
    o = AdamW(ps, lr=1e-3, state_bits=bits)
    _steps(o, ps, 1, 1)
    _turn(ps, "channels_last")
    _grads(ps, 2)
    torch.cuda.synchronize()
    with pytest.raises(AyoloError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            o.step()
    torch.cuda.synchronize()
    o.step()
    assert all(float(o.state[p]["step"]) == 2.0 for p in ps)


def test_gradients_in_another_memory_order():
    """are laid out like their parameters before the one call that is made; a type that does not fit is refused in any order"""
    from ayolov2_amd import _lib
    from ayolov2_amd.optim import adamw_step
    shape = (16, 8, 3, 3)
    p0, g0 = _rand(shape, 1), _rand(shape, 2)
    calls, call_on = [], _lib.call_on

    def counted(device, name, *args):
        calls.append(name)
        call_on(device, name, *args)

    res = []
    _lib.call_on = counted
    try:
        for turn in (lambda g: _in_order(g, "channels_last"), lambda g: g, lambda g: g.transpose(0, 3).contiguous().transpose(0, 3)):
            p, m, v, t = (_in_order(x.cuda(), "channels_last") for x in (p0, torch.zeros(shape), torch.zeros(shape), torch.zeros(())))
            g = turn(g0.cuda())
            adamw_step([p, p.clone()], [g, None], [m, None], [v, None], [t, None], lr=1e-2)
            res.append((p, m, v))
            with pytest.raises(_lib.AyoloError, match="type is not"):
                adamw_step([p], [g.half()], [m], [v], [t], lr=1e-2)
            with pytest.raises(_lib.AyoloError, match="not on a GPU|on device"):
                adamw_step([p.clone(), p], [_in_order(g, "channels_last"), g.cpu()], [m.clone(), m], [v.clone(), v], [t.clone(), t], lr=1e-2)
            with pytest.raises(_lib.AyoloError, match="memory order"):
                adamw_step([p], [g], [m.contiguous()], [v], [t], lr=1e-2)
    finally:
        _lib.call_on = call_on
    for r in res[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, res[0]))
    assert len(calls) == 4 * 3
    # an expanded gradient
    p, m, v, t = torch.zeros(5, 7, device="cuda"), torch.zeros(5, 7, device="cuda"), torch.zeros(5, 7, device="cuda"), torch.zeros((), device="cuda")
    adamw_step([p], [torch.full((), 2.0, device="cuda").expand(5, 7)], [m], [v], [t], lr=0.25, weight_decay=0.0)
    assert float(t) == 1.0 and ((p + 0.25).abs() <= 0.25 * 16 * ref.U32).all()

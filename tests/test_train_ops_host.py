"""The training operators without a GPU: refusals, the 8-bit moments' format (the oracle's own properties), CPU fall-backs."""
import copy

import numpy as np
import pytest
import torch

from ayolov2_amd import _lib, optim
from ayolov2_amd._lib import AyoloError
from ayolov2_amd.functional import layer_norm
from oracle import train_ref as ref


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(AyoloError, match="no CPU fallback"):
        layer_norm(x)
    with pytest.raises(AyoloError, match="no CPU fallback"):
        optim.grad_norm([x])
    with pytest.raises(AyoloError, match="no CPU fallback"):
        optim.clip_grads_([x], 1.0)
    with pytest.raises(AyoloError, match="no CPU fallback"):
        optim.adamw_step([x], [x], [x], [x], [torch.zeros(())], lr=1e-3)
    with pytest.raises(AyoloError, match="no CPU fallback"):
        optim.unpack_moments([optim.new_moment8(x)], True)


def test_empty_lists_do_nothing():
    assert float(optim.grad_norm([])) == 0.0 and float(optim.clip_grads_([None], 1.0)) == 0.0
    optim.adamw_step([], [], [], [], [], lr=1e-3)
    optim.adamw_step([torch.randn(3)], [None], [None], [None], [None], lr=1e-3)
    assert optim.unpack_moments([], True) == []


def test_argument_checks_before_the_gpu():
    x = torch.randn(4, 8)
    with pytest.raises(AyoloError, match="norm_type"):
        optim.clip_grad_norm_([x], 1.0, norm_type=1.0)
    with pytest.raises(AyoloError, match="max_norm"):
        optim.clip_grads_([x], -1.0)
    with pytest.raises(AyoloError, match="max_norm"):
        optim.clip_grads_([x], float("nan"))
    with pytest.raises(AyoloError, match="2 grads for 1 params"):
        optim.adamw_step([x], [x, x], [x], [x], [x], lr=1e-3)
    with pytest.raises(AyoloError, match="expected a tensor"):
        optim.grad_norm([1.0])
    with pytest.raises(AyoloError, match="state_bits"):
        optim.AdamW([torch.nn.Parameter(x)], state_bits=16)
    with pytest.raises(AyoloError, match="max_norm"):
        optim.AdamW([torch.nn.Parameter(x)], max_norm=-1.0)


def test_tensor_rows():
    t = torch.randn(3, 4, 5)
    u = torch.zeros(2, 3, 4, 5).contiguous(memory_format=torch.channels_last)
    rows = np.frombuffer(_lib.tensor_rows([t, None, t[:, ::2], u, u.contiguous(), t.half(), torch.zeros(0)], "x"), dtype=optim._TENSOR)
    assert rows["data"][0] == t.data_ptr() and rows["numel"].tolist() == [60, 0, 30, 120, 120, 60, 0]
    assert rows["present"].tolist() == [1, 0, 1, 1, 1, 1, 1] and (rows["device"] == -1).all()
    assert rows["layout"][2] == 0 and rows["layout"][3] != rows["layout"][4] and rows["layout"][0] == rows["layout"][5]
    assert rows["dtype"].tolist()[:1] + rows["dtype"].tolist()[5:6] == [_lib.F32, _lib.F16]
    # dimensions of one element have no order
    one = torch.zeros(4, 1, 3, 1)
    a, b = (np.frombuffer(_lib.tensor_rows([v], "x"), dtype=optim._TENSOR)["layout"][0]
            for v in (one, one.contiguous(memory_format=torch.channels_last)))
    assert (a == b) == (one.squeeze().stride() == one.contiguous(memory_format=torch.channels_last).squeeze().stride())
    for bad in ([1], ["x"], [torch.zeros(3).to_sparse()]):
        with pytest.raises(AyoloError):
            _lib.tensor_rows(bad, "x")
    with pytest.raises(AyoloError, match="pair"):
        _lib.tensor_rows([t], "x", 0)
    with pytest.raises(AyoloError, match="sequence"):
        _lib.tensor_rows(3, "x")


def test_c_abi_refuses_bad_lists():
    """The C entry points check their lists on the host before anything is launched."""
    lib = _lib.lib()
    t = torch.randn(8)
    rows = np.frombuffer(_lib.tensor_rows([t, t[:4]], "x"), dtype=optim._TENSOR).copy()
    rows["device"] = 0                                     # as if it lay on a GPU: nothing below reaches a launch
    ws = torch.zeros(64, dtype=torch.uint8)
    norm = torch.zeros(())

    def refused(rc, text):
        assert rc == -1 or rc == -3
        assert text in lib.ayolo_last_error().decode()

    refused(lib.ayolo_grad_clip(rows.tobytes(), 2, norm.data_ptr(), 1.0, None), "share memory")
    refused(lib.ayolo_grad_clip(rows.tobytes(), 2, norm.data_ptr(), -1.0, None), "max_norm")
    refused(lib.ayolo_grad_norm(rows.tobytes(), 2, None, norm.data_ptr(), ws.data_ptr(), 8, None), "workspace")
    for field, value, text in (("dtype", _lib.F32 + 10, "unsupported type"), ("layout", 0, "dense"), ("data", 0, "no memory"), ("data", 6, "aligned")):
        bad = rows[:1].copy()
        bad[field] = value
        refused(lib.ayolo_grad_norm(bad.tobytes(), 1, None, norm.data_ptr(), ws.data_ptr(), 64, None), text)
    mixed = rows.copy()
    mixed["device"][1] = 1
    refused(lib.ayolo_grad_norm(mixed.tobytes(), 2, None, norm.data_ptr(), ws.data_ptr(), 64, None), "device")

    store = [torch.randn(8) for _ in range(4)] + [torch.zeros(())]

    def adamw(change=None, **hyper):
        lists = [np.frombuffer(_lib.tensor_rows([v], "x"), dtype=optim._TENSOR).copy() for v in store]
        for l in lists:
            l["device"] = 0
        if change:
            change(lists)
        L, H = _lib.AdamWList(), _lib.AdamWHyper()
        L.p, L.g, L.m, L.v, L.step = (l.tobytes() for l in lists)
        L.n, H.beta1, H.beta2, H.eps = 1, 0.9, 0.999, 1e-8
        for k, v in hyper.items():
            setattr(H, k, v)
        return lib.ayolo_adamw_step(L, H, ws.data_ptr(), 4, None)

    refused(adamw(), "workspace")
    refused(adamw(beta1=1.0), "betas")
    refused(adamw(beta2=-0.1), "betas")
    refused(adamw(eps=-1.0), "eps")
    refused(adamw(eps=float("nan")), "eps")
    refused(adamw(lambda l: l[1].__setitem__("dtype", _lib.F16)), "type is not the parameter's")
    refused(adamw(lambda l: l[2].__setitem__("dtype", _lib.F16)), "unsupported type")
    refused(adamw(lambda l: l[2].__setitem__("numel", 4)), "sizes differ")
    refused(adamw(lambda l: l[3].__setitem__("layout", 77)), "memory order")
    refused(adamw(lambda l: l[4].__setitem__("numel", 2)), "not one number")
    refused(adamw(lambda l: l[0].__setitem__("present", 0)), "no parameter")
    refused(adamw(lambda l: l[3].__setitem__("data", l[2]["data"] + 4)), "share memory")


def test_layer_norm_c_abi_refuses():
    lib = _lib.lib()
    x = torch.zeros(4, 8)
    r = _lib.Rows(x.data_ptr(), 8, 0, 0)
    ok = (_lib.F32, r, None, 4, 8, None, None, _lib.F32, 1e-5, x.data_ptr(), None, None, None, None)

    def refused(at, value, text):
        args = list(ok)
        args[at] = value
        assert lib.ayolo_layer_norm_fwd(*args) == -1 and text in lib.ayolo_last_error().decode()

    refused(0, 7, "dtype")
    refused(7, _lib.F16, "gain")
    refused(3, -1, "rows")
    refused(3, 1 << 31, "rows")
    refused(4, 0, "C=0")
    refused(9, None, "null")
    refused(11, x.data_ptr(), "null")                      # mean without rstd
    refused(2, r, "null")                                  # residual without a place for the sum
    assert lib.ayolo_layer_norm_fwd(*[0 if k == 3 else v for k, v in enumerate(ok)]) == 0          # no rows: nothing to do
    assert lib.ayolo_layer_norm_bwd_workspace(_lib.F32, 0, 8) == 0
    need = lib.ayolo_layer_norm_bwd_workspace(_lib.F16, 1000, 64)
    assert need > 0 and need % (2 * 64 * 4) == 0
    assert lib.ayolo_layer_norm_bwd(_lib.F16, r, r, None, 1000, 64, None, _lib.F32, x.data_ptr(), x.data_ptr(), None, x.data_ptr(), None,
                                    x.data_ptr(), need - 1, None) == -3


def test_layer_norm_oracle_is_the_derivative():
    """The formula of the gradients against differences taken by autograd's checker in float64."""
    g = torch.Generator().manual_seed(0)
    x, w, b, gy, gs = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 7), (7,), (7,), (3, 7), (3, 7)))
    f = lambda x, w, b: (ref.layer_norm(x, w, b, 1e-3)[0] * gy).sum() + (x * gs).sum()  # noqa: E731
    leaves = [t.requires_grad_() for t in (x, w, b)]
    assert torch.autograd.gradcheck(f, leaves)
    auto = torch.autograd.grad(f(*leaves), leaves)
    for a, c in zip(auto, ref.layer_norm_grads(x.detach(), w.detach(), 1e-3, gy, gs)):
        assert torch.allclose(a, c, rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("signed", [True, False])
def test_moment_format(signed):
    rng = np.random.default_rng(0)
    n = 1000
    scale = np.exp2(rng.uniform(-12, 0, n)).astype(np.float32)
    x = (rng.standard_normal(n).astype(np.float32) * scale) if signed else (rng.random(n).astype(np.float32) * scale)
    r = rng.integers(0, 1 << 16, n).astype(np.uint32)
    codes, exps = ref.encode(x, r, signed)
    back = ref.decode(codes, exps, signed)
    # a value is moved by less than one step of its code: 2^-3 of itself, or the subnormals' spacing under its block's largest value
    top = np.repeat(np.pad(np.abs(x), (0, -n % 128)).reshape(-1, 128).max(1), 128)[:n]
    assert (np.abs(back - x) <= np.maximum(np.abs(x) / 8, top * 2.0 ** (-16 if signed else -32))).all()
    # what is stored is stored again unchanged, whatever the random bits
    again = ref.encode(back, np.full(n, 0xFFFF, np.uint32) * 0, signed)
    keep = exps == again[1]                                # (a carry into the next binade moves the block's exponent)
    assert (np.repeat(keep, 128)[:n] <= (ref.decode(*again, signed) == back)).all()
    # unbiased: the mean over all 2^16 random numbers is the value, to the half of the lowest random bit
    for v in (x[3], x[7], np.float32(top[0] * 2.0 ** -20)):
        v = abs(v)
        blk = np.full(128 * 512, v, np.float32)
        blk[::128] = top[0]                                # the block's exponent stays that of its largest value
        r = (np.arange(128 * 512) % 65536).astype(np.uint32)
        got = ref.decode(*ref.encode(blk, r, signed), signed).astype(np.float64)
        sel = np.arange(128 * 512) % 128 != 0
        step = max(v / 8, top[0] * 2.0 ** (-16 if signed else -32))
        if signed or v > top[0] * 2.0 ** -32:
            # 65024 of the 65536 random numbers, missing ones spread evenly: at most 1 / 128 of a step plus 2^-16
            assert abs(got[sel].mean() - v) <= step * (1 / 128 + 2.0 ** -16)


def test_moment_special_values():
    x = np.zeros(300, np.float32)
    x[[0, 1, 2]] = np.nan, np.inf, 3.0
    x[[130, 131]] = np.float32(1e-45), np.float32(2e-38)   # subnormal and smallest normal numbers
    x[299] = 1e-30
    r = np.zeros(300, np.uint32)
    for signed in (True, False):
        got = ref.decode(*ref.encode(x, r, signed), signed)
        assert np.isnan(got[0]) and np.isposinf(got[1]) and abs(got[2] - 3.0) <= 3 / 8
        assert (got[3:130] == 0).all() and abs(got[299] - 1e-30) <= 1e-30 / 8
    x[:3] = -np.inf, -2.0, 1.0
    got = ref.decode(*ref.encode(x, r, True), True)
    assert np.isneginf(got[0]) and got[1] == -2.0 and got[2] == 1.0
    # a second moment above zero stays above zero however small it is
    y = np.full(128, 1e-30, np.float32)
    y[0] = 1.0
    assert (ref.decode(*ref.encode(y, np.zeros(128, np.uint32), False), False) > 0).all()


def test_noise_is_even_and_differs():
    a, b = ref.noise(0, 1, 0, 1 << 16)
    for v in (a, b):
        hist = np.bincount(v >> 12, minlength=16)
        assert abs(hist - 4096).max() < 5 * 64              # five standard deviations of a uniform draw
    others = [ref.noise(*k, 1 << 16)[0] for k in ((1, 1, 0), (0, 2, 0), (0, 1, 1))]
    for o in others:
        assert abs(np.corrcoef(a.astype(float), o.astype(float))[0, 1]) < 5 / 256
    assert abs(np.corrcoef(a.astype(float), b.astype(float))[0, 1]) < 5 / 256
    assert abs(np.corrcoef(a[1:].astype(float), a[:-1].astype(float))[0, 1]) < 5 / 256


def test_adamw_on_the_cpu_is_torchs():
    g = torch.Generator().manual_seed(0)
    init = [torch.randn(5, 3, generator=g), torch.randn(7, generator=g)]
    a, b = ([torch.nn.Parameter(t.clone()) for t in init] for _ in range(2))
    oa = optim.AdamW(a, lr=0.01, weight_decay=0.1)
    ob = torch.optim.AdamW(b, lr=0.01, weight_decay=0.1)
    for _ in range(3):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=g)
            q.grad = p.grad.clone()
        oa.step()
        ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    with pytest.raises(AyoloError, match="GPU"):
        o = optim.AdamW(a, state_bits=8)
        o.step()
    # clipped: as torch's two calls
    oa, ob = optim.AdamW(a, lr=0.01, max_norm=0.5), torch.optim.AdamW(b, lr=0.01)
    torch.nn.utils.clip_grad_norm_(b, 0.5)
    oa.step()
    ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_8_bit_state_dicts_do_not_load_onto_the_cpu():
    p = torch.nn.Parameter(torch.randn(300))
    o = optim.AdamW([p])
    sd = o.state_dict()
    sd["state"] = {0: {"step": torch.tensor(1.0), "exp_avg": torch.zeros(300, dtype=torch.uint8), "exp_avg_exps": torch.zeros(3, dtype=torch.uint8),
                       "exp_avg_sq": torch.zeros(300, dtype=torch.uint8), "exp_avg_sq_exps": torch.zeros(3, dtype=torch.uint8)}}
    with pytest.raises(AyoloError, match="GPU"):
        o.load_state_dict(sd)


def test_adamw_copies_keep_their_settings():
    o = optim.AdamW([torch.nn.Parameter(torch.randn(3))], state_bits=8, max_norm=2.0, seed=5)
    c = copy.deepcopy(o)
    assert (c.state_bits, c.max_norm, c.seed) == (8, 2.0, 5)


def test_clip_grad_norm_on_the_cpu_is_torchs():
    p = torch.nn.Parameter(torch.randn(10))
    p.grad = torch.randn(10) * 5
    q = p.grad.clone()
    n = optim.clip_grad_norm_(p, 1.0)
    assert torch.allclose(n, q.norm()) and torch.allclose(p.grad, q / (q.norm() + 1e-6))
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.randn(2))], 1.0)) == 0.0


def test_yaml_row_builds_a_layer_norm():
    from ayolov2_amd import LayerNorm, YOLOModel
    cfg = {"input_channel": 3, "depth_multiple": 1.0, "width_multiple": 1.0,
           "backbone": [[-1, 1, "Conv", [16, 3, 2]], [-1, 1, "LayerNorm", [1e-6]], [-1, 1, "Conv", [8, 1, 1]]],
           "head": [[[-1], 1, "YOLOHead", [2, [[10, 13, 16, 30, 33, 23]]]]]}
    m = YOLOModel(cfg)
    assert isinstance(m.model[1], LayerNorm) and m.model[1].weight.shape == (16,) and m.model[1].eps == 1e-6 and m.model[1].dim == 1
    assert {"model.1.weight", "model.1.bias"} <= set(m.state_dict())

"""The states of ``optim.AdamW`` without a GPU: the conversion of fp32 values into 8-bit moments, against the oracle's format."""
import numpy as np
import pytest
import torch

from ayolov2_amd import optim
from ayolov2_amd._lib import AyoloError
from oracle import train_ref as ref


def _special(signed):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 37, 3, 3, generator=g) * torch.exp2(torch.randint(-60, 8, (5, 37, 1, 1), generator=g).float())
    x = x if signed else x.abs()
    v = x.view(-1)
    v[[3, 700]], v[[4, 701]], v[129:300], v[300:310] = float("nan"), float("inf"), 0.0, 1e-42
    v[310], v[311] = 3.0e38, 2.0 ** -126
    if signed:
        v[5], v[6], v[312] = float("-inf"), -0.0, -3.0e38
    return x


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("order", [torch.contiguous_format, torch.channels_last], ids=["contiguous", "channels_last"])
def test_packed_as_the_format_says(signed, order):
    """Bit for bit what the oracle makes of the values in memory order, rounding to nearest (the random number at its middle)."""
    x = _special(signed).contiguous(memory_format=order)
    m = optim._pack_moment(x, signed)
    assert m.codes.stride() == x.stride() and m.codes.dtype == m.exps.dtype == torch.uint8
    flat = lambda t: t.as_strided((t.numel(),), (1,)).numpy()  # noqa: E731
    codes, exps = ref.encode(flat(x), np.full(x.numel(), 0x8000, np.uint32), signed)
    assert np.array_equal(flat(m.codes), codes) and np.array_equal(m.exps.numpy(), exps)
    back = ref.decode(codes, exps, signed)
    assert np.array_equal(np.isnan(back), np.isnan(flat(x)))
    ok = np.isfinite(flat(x)) & (np.abs(flat(x)) < 3e38)
    top = np.where(np.isfinite(flat(x)), np.abs(flat(x)), 0)
    top = np.repeat(np.pad(top, (0, -top.size % 128)).reshape(-1, 128).max(1), 128)[:top.size].astype(np.float64)
    # half a step: 2^-4 of the value, 2^-17 of the block's largest below the normal codes (a second moment never becomes zero: a
    # step of 2^-32), and the spacing under the least exponents at the bottom of fp32's range
    tol = np.maximum(np.maximum(np.abs(flat(x).astype(np.float64)) / 16, top * 2.0 ** (-17 if signed else -32)), 2.0 ** -142)
    assert (np.abs(back[ok].astype(np.float64) - flat(x)[ok]) <= tol[ok]).all()
    if not signed:
        assert (back[ok & (flat(x) > 0)] > 0).all()


@pytest.mark.parametrize("n", [0, 1, 127, 128, 129])
def test_packed_sizes(n):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n))
    m = optim._pack_moment(x, True)
    assert m.codes.shape == (n,) and m.exps.shape == (-(-n // 128),)
    assert (np.abs(ref.decode(m.codes.numpy(), m.exps.numpy(), True) - x.numpy()) <= np.maximum(np.abs(x.numpy()) / 16, 5 * 2.0 ** -17)).all()


def _adamw(device="cpu"):
    p = torch.nn.Parameter(torch.ones(300, device=device))
    o = optim.AdamW([p], lr=0.5)
    p.grad = torch.ones_like(p)
    return o, p


def test_refused_loads_change_nothing():
    """8-bit states are refused on the CPU, and the optimiser is as it was: settings and states"""
    o, p = _adamw()
    o.step()
    before = {k: v.clone() for k, v in o.state[p].items()}
    sd = o.state_dict()
    sd = {"state": {0: {"step": torch.tensor(9.0), "exp_avg": torch.zeros(300, dtype=torch.uint8), "exp_avg_exps": torch.zeros(3, dtype=torch.uint8),
                        "exp_avg_sq": torch.zeros(300, dtype=torch.uint8), "exp_avg_sq_exps": torch.zeros(3, dtype=torch.uint8)}},
          "param_groups": [{**sd["param_groups"][0], "lr": 7.0}]}
    with pytest.raises(AyoloError, match="GPU"):
        o.load_state_dict(sd)
    assert o.param_groups[0]["lr"] == 0.5 and o.param_groups[0]["params"][0] is p
    assert set(o.state[p]) == set(before) and all(torch.equal(o.state[p][k], v) for k, v in before.items())
    # what the base class refuses is still the base class's error
    sd["param_groups"][0]["params"] = [0, 1]
    with pytest.raises(ValueError, match="parameter group"):
        o.load_state_dict(sd)


def test_load_hooks_are_heard():
    """a hook before the load hands on another state dict; a hook behind it sees the loaded states and changes them for good"""
    o, p = _adamw()
    o.step()
    seen = []

    def other(_, sd):
        return {"state": {0: {"step": torch.tensor(4.0), "exp_avg": torch.full((300,), 2.0), "exp_avg_sq": torch.full((300,), 3.0)}},
                "param_groups": sd["param_groups"]}

    def behind(opt):
        seen.append(float(opt.state[p]["exp_avg"][0]))
        opt.state[p]["exp_avg"] = torch.full((300,), 5.0)

    o.register_load_state_dict_pre_hook(other)
    o.register_load_state_dict_post_hook(behind)
    before = len(o._optimizer_load_state_dict_pre_hooks), len(o._optimizer_load_state_dict_post_hooks)
    o.load_state_dict(o.state_dict())
    assert seen == [2.0] and (o.state[p]["exp_avg"] == 5.0).all() and (o.state[p]["exp_avg_sq"] == 3.0).all()
    # what is handed on is checked too, and nothing stays registered
    o.register_load_state_dict_pre_hook(lambda _, sd: {"state": {0: {**sd["state"][0], "exp_avg_exps": torch.zeros(3)}}, "param_groups": sd["param_groups"]})
    with pytest.raises(AyoloError, match="GPU"):
        o.load_state_dict(o.state_dict())
    assert (len(o._optimizer_load_state_dict_pre_hooks), len(o._optimizer_load_state_dict_post_hooks)) == (before[0] + 1, before[1])


def test_places_in_another_memory_order():
    from ayolov2_amd import _lib
    host, rows = _lib.host(), lambda ts: _lib.tensor_rows(ts, "x")
    w = torch.zeros(4, 3, 5, 5)
    last = w.contiguous(memory_format=torch.channels_last)
    model = rows([w, last, w, None, w, w[:, :, ::2], torch.zeros(7)])
    assert host.unlike(rows([w, last, last, w, None, last, torch.zeros(7, dtype=torch.uint8)]), model) == [2]
    assert host.unlike(rows([w[:, ::2], w[:1].expand(4, 3, 5, 5), w.half(), None, w[:2], w, torch.zeros(8)]), model) == [0, 1, 4, 6]
    assert host.unlike(b"", b"") == []
    with pytest.raises(ValueError, match="lengths"):
        host.unlike(rows([w]), model)

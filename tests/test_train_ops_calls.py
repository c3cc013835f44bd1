"""Calls of the training operators that their documentation allows or refuses, without a GPU: what shares memory, what is traced, what
has no memory of its own."""
import numpy as np
import pytest
import torch

from ayolov2_amd import _lib, optim


def _rows(*tensors):
    """the list of these (CPU) tensors as if they lay on a GPU; every call below ends on the host"""
    rows = np.frombuffer(_lib.tensor_rows(list(tensors), "x"), dtype=optim._TENSOR).copy()
    rows["device"][rows["present"] != 0] = 0
    return rows.tobytes()


def _adamw(p, g, m, v, step, me=None, ve=None, **hyper):
    """(code, message) of an AdamW step whose workspace is too small, which is looked at last"""
    L, H = _lib.AdamWList(), _lib.AdamWHyper()
    L.p, L.g, L.m, L.v, L.step = _rows(*p), _rows(*g), _rows(*m), _rows(*v), _rows(*step)
    if me is not None:
        L.me, L.ve = _rows(*me), _rows(*ve)
    L.n, H.beta1, H.beta2, H.eps = len(p), 0.9, 0.999, 1e-8
    for k, t in hyper.items():
        setattr(H, k, t.data_ptr())
    ws = torch.zeros(64, dtype=torch.uint8)
    rc = _lib.lib().ayolo_adamw_step(L, H, ws.data_ptr(), 4, None)
    return rc, _lib.lib().ayolo_last_error().decode()


def _lists(n=2, size=300):
    make = lambda: [torch.zeros(size) for _ in range(n)]  # noqa: E731
    return dict(p=make(), g=make(), m=make(), v=make(), step=[torch.zeros(()) for _ in range(n)])


def _shares(res):
    assert res[0] == -1 and "share memory" in res[1], res


def _free(res):
    assert res[0] == -3 and "workspace" in res[1], res


def test_adamw_refuses_gradients_in_what_it_writes():
    big = torch.zeros(900)
    _free(_adamw(**_lists()))
    for name in ("p", "m", "v"):
        for lo in (-299, -4, 4, 299):                      # the gradient begins before or inside what is written
            l = _lists()
            l[name][0], l["g"][0] = big[300:600], big[300 + lo:600 + lo]
            _shares(_adamw(**l))
        l = _lists()
        l[name][0], l["g"][1] = big[:300], big[:300]       # another entry's gradient
        _shares(_adamw(**l))
        l = _lists()
        l[name][0], l["g"][0] = big[:300], big[300:600]    # side by side
        _free(_adamw(**l))
        l = _lists()
        l[name][0] = l["g"][0] = big[:300]                 # the gradient is the parameter or the moment itself
        _free(_adamw(**l))
    l = _lists()
    l["g"] = [big[:300], big[:300]]                        # gradients are only read
    _free(_adamw(**l))
    l["g"] = [big[:300], big[100:400]]
    _free(_adamw(**l))
    l["step"][1] = big[399]                                # ... and end where the longest of them ends
    _shares(_adamw(**l))
    l["step"][1] = big[400]
    _free(_adamw(**l))


def test_adamw_refuses_gradients_in_8_bit_moments():
    size = 300
    codes, exps = (lambda: [torch.zeros(size, dtype=torch.uint8) for _ in range(2)]), (lambda: [torch.zeros(3, dtype=torch.uint8) for _ in range(2)])
    base = lambda: {**_lists(), "m": codes(), "v": codes(), "me": exps(), "ve": exps()}  # noqa: E731
    _free(_adamw(**base()))
    for name in ("m", "v", "me", "ve"):
        l = base()
        n = l[name][0].numel()
        l[name][0] = l["g"][0].view(torch.uint8)[:n]
        _shares(_adamw(**l))
        l = base()
        l[name][1] = l["g"][0].view(torch.uint8)[-n:]
        _shares(_adamw(**l))


def test_adamw_refuses_scalars_in_what_it_writes():
    for name in ("lr_dev", "grad_scale", "found_inf", "norm"):
        for of in ("p", "m", "v", "step"):
            l = _lists()
            _shares(_adamw(**l, **{name: l[of][1].reshape(-1)[-1]}))
        l = _lists()
        _free(_adamw(**l, **{name: l["g"][0][3]}))         # read beside a gradient that is read
        one = torch.ones(())
        _free(_adamw(**l, lr_dev=one, grad_scale=one, found_inf=one, norm=one))


def test_clipping_refuses_a_norm_inside_the_gradients():
    g = torch.zeros(300)
    rc = _lib.lib().ayolo_grad_clip(_rows(g[:200]), 1, g[7].data_ptr(), 1.0, None)
    assert rc == -1 and "share memory" in _lib.lib().ayolo_last_error().decode()


def test_moment_values_refuses_shared_outputs():
    lib = _lib.lib()
    codes, exps = [torch.zeros(300, dtype=torch.uint8) for _ in range(2)], [torch.zeros(3, dtype=torch.uint8) for _ in range(2)]
    big = torch.zeros(900)

    def refused(codes, exps, out):
        rc = lib.ayolo_moment_values(_rows(*codes), _rows(*exps), _rows(*out), 2, 1, None)
        assert rc == -1 and "share memory" in lib.ayolo_last_error().decode()

    refused(codes, exps, [big[:300], big[:300]])           # twice the same
    refused(codes, exps, [big[:300], big[299:599]])
    inside = big.view(torch.uint8)
    refused([inside[1199:1499], codes[1]], exps, [big[:300], big[400:700]])
    refused(codes, [exps[0], inside[1600:1603]], [big[:300], big[400:700]])
    refused([codes[0]] * 2, [exps[0]] * 2, [big[:300], big[:300]])


def test_layer_norm_is_not_traced():
    from ayolov2_amd.functional import layer_norm
    with pytest.raises(_lib.AyoloError, match="traced"):
        torch.jit.trace(lambda t: layer_norm(t), torch.randn(2, 8), check_trace=False)
    with pytest.raises(_lib.AyoloError, match="no CPU fallback"):
        layer_norm(torch.randn(2, 8))


def test_lists_refuse_a_pending_negation():
    x = torch.randn(6)
    with pytest.raises(_lib.AyoloError, match="strided tensor"):
        _lib.tensor_rows([torch._neg_view(x)], "x")
    assert len(_lib.tensor_rows([-x, torch._neg_view(torch._neg_view(x))], "x")) == 2 * optim._TENSOR.itemsize


def test_versions_count_up():
    a, b, c, d = (torch.zeros(3) for _ in range(4))
    _lib.host().bump([a, (b, c), None, [d, b]], (a, a, a, None))
    assert [t._version for t in (a, b, c, d)] == [1, 1, 1, 0]
    with pytest.raises(TypeError):
        _lib.host().bump(3, [a])


@pytest.mark.parametrize("n", [1, 3, 60, 400])
@pytest.mark.parametrize("shuffled", [False, True])
def test_overlaps_among_many_ranges(n, shuffled):
    """Lists in any order, near and far apart (addresses are only compared here): found exactly where a pair of ranges, one of them
    written, shares a byte."""
    rng = np.random.default_rng(n + shuffled)
    lib, ws = _lib.lib(), torch.zeros(8, dtype=torch.uint8)
    slots = 4 * n                                          # slots of 4 KB, in 16 regions far apart; a tensor fills up to one
    for trial in range(24):
        base = np.sort(rng.integers(1 << 20, 1 << 35, 16)).astype(np.uint64) << np.uint64(12)
        place = rng.permutation(slots) if shuffled else np.arange(slots)
        addr = (base[place % 16] + (place // 16).astype(np.uint64) * np.uint64(1 << 12) * np.uint64(1 if trial % 2 else 1 << 9)).reshape(4, n)
        if not shuffled:
            addr = np.sort(addr, axis=1)
        lists = []
        numel = rng.integers(1, 1025, n)
        for k in range(4):
            l = np.zeros(n, dtype=optim._TENSOR)
            l["data"], l["numel"], l["layout"], l["dtype"], l["present"] = addr[k], numel, 77, _lib.F32, 1
            lists.append(l)
        step = np.zeros(n, dtype=optim._TENSOR)
        step["data"], step["numel"], step["layout"], step["dtype"], step["present"] = (1 << 62) + 4 * np.arange(n), 1, 1, _lib.F32, 1
        if trial % 3 == 0:                                 # one is moved to where another one ends, or a little before
            k, i, j, m = rng.integers(4), rng.integers(n), rng.integers(n), rng.integers(4)
            lists[k]["data"][i] = lists[m]["data"][j] + np.uint64(4 * (numel[j] - rng.integers(0, 2)))
        p, g, m, v = lists
        spans = [(int(a), int(a) + 4 * int(c), w, (k, i)) for k, (l, w) in enumerate(((p, 1), (g, 0), (m, 1), (v, 1)))
                 for i, (a, c) in enumerate(zip(l["data"], l["numel"]))]
        own = {i for i in range(n) if g["data"][i] in (p["data"][i], m["data"][i], v["data"][i])}
        spans = sorted(s for s in spans if not (s[3][0] == 1 and s[3][1] in own))
        want, written, any_ = False, 0, 0
        for a, b, w, _ in spans:
            want |= a < (any_ if w else written)
            any_, written = max(any_, b), max(written, b) if w else written
        L, H = _lib.AdamWList(), _lib.AdamWHyper()
        L.p, L.g, L.m, L.v, L.step = (l.tobytes() for l in (p, g, m, v, step))
        L.n, H.beta1, H.beta2, H.eps = n, 0.9, 0.999, 1e-8
        rc = lib.ayolo_adamw_step(L, H, ws.data_ptr(), 4, None)
        assert rc == (-1 if want else -3), (trial, lib.ayolo_last_error())


def test_rows_count_versions_where_a_gradient_is_given():
    a, b, c = (torch.zeros(3) for _ in range(3))
    _lib.tensor_rows([a, b, None], "x", -1, [a, None, a])
    _lib.tensor_rows([(a, b), (c, b)], "x", 1, [None, a])
    assert [t._version for t in (a, b, c)] == [1, 1, 0]
    _lib.tensor_rows([a, b], "x")
    assert [t._version for t in (a, b, c)] == [1, 1, 0]
    with pytest.raises(_lib.AyoloError, match="given"):
        _lib.tensor_rows([a], "x", -1, (a,))


def test_entries_without_a_gradient_share_what_they_like():
    """nothing of theirs is written"""
    l = _lists(3)
    l["g"][1] = l["g"][2] = None
    l["p"][2] = l["p"][1]
    l["step"][2] = l["step"][1]
    l["m"][1] = l["g"][0]
    _free(_adamw(**l))
    l["p"][2] = l["p"][0]
    _free(_adamw(**l))
    l["g"][2] = torch.zeros(300)
    _shares(_adamw(**l))

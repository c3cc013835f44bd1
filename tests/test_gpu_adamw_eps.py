"""AdamW with eps down to 0: where the root of a second moment is taken by the hardware's function, which takes subnormal numbers for
zero, and where by the exact one."""
import pytest
import torch

from oracle import train_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U32


@pytest.mark.parametrize("b2", [0.999, 0.99999])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-15, 0.99e-12, 1e-12, 1e-11, 1e-10, 1e-9, 1e-8])
@pytest.mark.parametrize("t0", [0, 500])
def test_adamw_with_the_smallest_eps(eps, b2, t0):
    """Second moments down to fp32's subnormal numbers, where their root is nothing beside an ordinary eps and all beside a small one.
    The parameters are zero, so that what is checked is the step itself, formed from the moments that the kernel leaves: 16 u."""
    from ayolov2_amd.optim import adamw_step
    n, b1, lr = 5000, 0.9, 1e-3
    gen = torch.Generator().manual_seed(1)
    size = torch.exp2(torch.rand(n, generator=gen) * -60 - 10)                      # 2^-10 .. 2^-70: squares 2^-20 .. 2^-140
    g = torch.randn(n, generator=gen) * size
    g = torch.where(g.abs() < 2.0 ** -70, torch.full_like(g, 2.0 ** -70), g)        # (a square of 0 has no step at eps = 0)
    m, v = (torch.randn(n, generator=gen) * size, (torch.randn(n, generator=gen) * size).square()) if t0 else (torch.zeros(n), torch.zeros(n))
    p, dm, dv, t = torch.zeros(n, device="cuda"), m.cuda(), v.cuda(), torch.full((), float(t0), device="cuda")
    adamw_step([p], [g.cuda()], [dm], [dv], [t], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0)
    g64 = g.double()
    wm, wv = b1 * m.double() + (1 - b1) * g64, b2 * v.double() + (1 - b2) * g64 * g64
    # the moments are those of the kernel, whose own rounding is tested elsewhere; a second moment of 0 stands for one below 2^-149
    assert ((dm.double().cpu() - wm).abs() <= 4 * U * (b1 * m.double().abs() + (1 - b1) * g64.abs()) + 2.0 ** -149).all()
    assert ((dv.double().cpu() - wv).abs() <= 6 * U * wv + 2.0 ** -148).all()
    km, kv = dm.double().cpu(), dv.double().cpu()
    kept = kv > 0
    want = -lr * (km / (1 - b1 ** (t0 + 1))) / (torch.sqrt(kv / (1 - b2 ** (t0 + 1))) + eps)
    assert int(kept.sum()) > n // 2 and ((p.double().cpu() - want).abs() <= 16 * U * want.abs() + 2.0 ** -149)[kept].all()

"""The gated activation at infinities and NaN when it has no clamp: its gradients are those of the formula, h = w g s u with s = 1 / (1 + exp(-g)).

Tolerances as in test_gpu_grouped: half a step of the type for the result, and (|g| + 8) 2^-23 of the magnitudes before the derivative's own
cancellation for the sigmoid by v_exp_f32 and v_rcp_f32 and the products around it, 2^-22 for those of w and dh."""
import pytest
import torch

from test_gpu_grouped import BF, HALF, HF, TINY

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("limit", [0.0, INF])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("save8", [False, True])
def test_without_a_clamp_nothing_is_cut(dev, dtype, limit, save8):
    from mi355moe import grouped
    gen = torch.Generator().manual_seed(21)
    I = 64
    gu, dh, w = torch.randn((9, 2 * I), generator=gen), torch.randn((9, I), generator=gen), torch.rand(9, generator=gen)
    # (row, column of g, column of u): a gate, an up, both
    for row, (g, u) in enumerate([(NAN, None), (None, NAN), (NAN, NAN), (INF, None), (-INF, None), (None, INF), (None, -INF), (INF, -INF)]):
        if g is not None:
            gu[row, 3] = g
        if u is not None:
            gu[row, I + 3] = u
    gu, dh = gu.to(dtype), dh.to(dtype)
    held = gu.double()
    if save8:                                             # 32 that hold an infinity or NaN come back as NaN; the others as they are held
        x = held.unflatten(1, (-1, 32))
        top = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / 127))
        e = torch.where(top > 127 * 2.0 ** e, e + 1, e)
        held = torch.where(top.isfinite(), torch.round(x / 2.0 ** e) * 2.0 ** e, NAN).flatten(1)
    g, u = held.chunk(2, 1)
    s, d = torch.sigmoid(g), w.double()[:, None] * dh.double()
    want = torch.cat([d * u * (s * (1 + g * (1 - s))), d * (g * s)], 1)
    err = torch.cat([(d * u * s).abs() * (1 + g.abs() * (1 - s)), (d * g * s).abs()], 1) * torch.cat([(g.abs() + 10) * 2.0 ** -23] * 2, 1)
    h, kept = grouped.swiglu_forward(gu.to(dev), weights=w.to(dev), limit=limit, save8=save8)
    dgu, dw, _ = grouped.swiglu_backward(dh.to(dev), kept, weights=w.to(dev), limit=limit)
    got = dgu.cpu().double()
    assert want[1, I + 3].isfinite() or save8            # an up of NaN: its own gradient is w dh silu(g), a number
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[got.isinf()].sign(), want[got.isinf()].sign())
    fine = want.isfinite()
    assert ((got - want).abs()[fine] <= (HALF[dtype] * want.abs() + err + TINY[dtype])[fine]).all()
    g, u = gu.double().chunk(2, 1)
    assert torch.equal(h.cpu().isnan(), (w.double()[:, None] * g * torch.sigmoid(g) * u).isnan())
    assert dw.cpu()[:8].isfinite().logical_not().all() and dw[8].isfinite()

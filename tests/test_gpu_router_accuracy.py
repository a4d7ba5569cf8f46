"""Router backward where products cancel, and where values are infinite, against float64.

Tolerances of dx: D and the gate are two fp16 parts each under a power of two per token (per hidden index). A part is off by half a
step, 2^-11 of its value, so two parts leave 2^-22 of the value, and the product of the two second parts, which is left out, is at most
2^-22: 3 x 2^-22 of a product. Values far below the largest of their row (scaled to at least 2^8) keep steps of 2^-24, half of which is
2^-33 of the largest. 3 E products are added in fp32 (3 E 2^-23 of the sum of magnitudes), and the result is rounded to bf16 (2^-8)."""
import pytest
import torch

from test_gpu_router_grad import close, router64, router_inputs

pytestmark = pytest.mark.gpu

PRODUCT = 3 * 2.0 ** -22


def backward_dx(dev, gate, D, H):
    from mi355moe import router
    T = D.shape[0]
    x = torch.zeros((T, H), dtype=torch.bfloat16, device=dev)
    ids, w = torch.zeros((T, 1), dtype=torch.int64, device=dev), torch.ones((T, 1), device=dev)
    dx, _ = router.topk_backward(x, gate.to(dev), ids, w, None, D.to(dev), need_gate=False)
    return dx


def check_dx(dx, gate, D):
    a, b = D.double(), gate.double()
    mag = a.abs() @ b.abs()
    far = a.abs().amax(1, keepdim=True) * b.abs().sum(0) + a.abs().sum(1, keepdim=True) * b.abs().amax(0)
    close(dx, a @ b, 2.0 ** -8 * (a @ b).abs() + (PRODUCT + 3 * len(b) * 2.0 ** -23) * mag + 2.0 ** -33 * far + 1e-37)


@pytest.mark.parametrize("T,H", [(1, 16), (70, 144)])
def test_dx_of_two_products_that_nearly_cancel(dev, T, H):
    """Factors just below 1 + 2^-7 and differences of 2^-20 of the products: what is left out of a product shows in the result."""
    g = torch.Generator().manual_seed(T)
    a0 = 1 + 2.0 ** -7 * 0.97
    a = a0 + torch.randint(-64, 65, (T,), generator=g) * 2.0 ** -20
    b = 1 + 2.0 ** -7 * (0.9 + 0.09 * torch.rand((H,), generator=g))
    D = torch.stack([a, -torch.ones(T)], 1)
    gate = torch.stack([b, b * a0])
    check_dx(backward_dx(dev, gate, D, H), gate, D)


@pytest.mark.parametrize("E", [16, 33])
def test_dx_of_a_component_common_to_all_experts(dev, E):
    """Rows of D that sum to zero (gradients of a softmax) cancel what the gate's rows share. By the roundings' random walk: the 3 E
    sums, and the parts' errors, over the root of the sum of the products' squares (eight times it), and the result's half step."""
    g = torch.Generator().manual_seed(E)
    T, H = 150, 256
    gate = 4000 * torch.randn((1, H), generator=g) + torch.randn((E, H), generator=g)
    p = torch.softmax(torch.randn((T, E), generator=g), 1).double()
    c = torch.randint(0, 9, (E,), generator=g).double()
    D = (p * (c - (p @ c)[:, None])).float()
    dx = backward_dx(dev, gate, D, H)
    check_dx(dx, gate, D)
    a, b = D.double(), gate.double()
    ref = a @ b
    rms = ((a ** 2) @ (b ** 2)).sum().sqrt()
    assert (dx.cpu().double() - ref).norm() <= 2.0 ** -8 * ref.norm() + (PRODUCT + 8 * (3 * E) ** 0.5 * 2.0 ** -24) * rms


def test_dx_of_rows_of_any_size(dev):
    """Tokens and hidden indices of magnitudes from 1e-18 to 1e18, values of 2^-30 of their row's largest, and rows of zeros."""
    g = torch.Generator().manual_seed(3)
    T, H, E = 90, 80, 70
    D = torch.randn((T, E), generator=g) * 10.0 ** torch.randint(-18, 19, (T, 1), generator=g).float()
    gate = torch.randn((E, H), generator=g) * 10.0 ** torch.randint(-18, 19, (1, H), generator=g).float()
    D[:, ::7] *= 2.0 ** -30
    gate[::5] *= 2.0 ** -30
    D[4], D[66], gate[:, 9] = 0.0, 0.0, 0.0
    check_dx(backward_dx(dev, gate, D, H), gate, D)


def test_dx_of_picks_that_cancel_the_logits_gradient(dev):
    """D is small where the two gradients cancel: its row is scaled by both, and what is left is what fp32 leaves."""
    from mi355moe import router
    x, gate, ids, w, dw, _ = router_inputs(100, 96, 40, 4, 12, dev)
    d = w * (dw - (w * dw).sum(1, keepdim=True))
    dl = torch.zeros((100, 40), device=dev).scatter_(1, ids, -d)
    dx, _ = router.topk_backward(x, gate, ids, w, dw, dl, need_gate=False)
    rx, _, mx, _, ex, _ = router64(x, gate, ids, w, dw, dl)
    one = router64(x, gate, ids, w, dw, torch.zeros_like(dl))
    # ex counts D's roundings from its own magnitudes; the gradient of the picks alone has the larger ones
    close(dx, rx, 2.0 ** -8 * rx.abs() + (PRODUCT + 3 * 40 * 2.0 ** -23) * mx + ex + one[4] + 2.0 ** -33 * 40 * one[2] + 1e-37)


@pytest.mark.parametrize("T,E", [(40, 20), (600, 33)])
@pytest.mark.parametrize("with_picks", [False, True])
def test_dgate_of_infinite_inputs_and_gradients(dev, T, E, with_picks):
    """dgate = D^T x with infinities as IEEE products and sums have them: +-inf by the signs, NaN for 0 x inf and inf - inf, whatever parts
    D is made of (values of few bits among them); the rest within the sums' roundings."""
    from mi355moe import router
    H = 48
    x, gate, ids, w, dw, dl = router_inputs(T, H, E, 3, T + E, dev)
    dl[3] = torch.tensor([1.0, -2.0, 0.375, 1 + 2.0 ** -7, -1 - 2.0 ** -8, 0.0])[torch.arange(E) % 6].to(dev)
    dl[7, ::2] = 0.0
    x[3, 5], x[7, 11], x[9, 13] = torch.inf, -torch.inf, torch.inf
    x[T - 1, 13] = torch.inf
    dl[12, 4], x[12, 20] = -torch.inf, 0.0
    x[15, 30] = torch.finfo(torch.bfloat16).max
    dl[15] = 2.0 ** -8
    dw = dw if with_picks else None
    _, dgate = router.topk_backward(x, gate, ids, w, dw, dl, need_x=False)
    _, ref, _, _, _, err = router64(x, gate, ids, w, dw, dl)
    if with_picks:                                             # (a pick may move D off zero, or leave it there)
        assert (torch.isinf(ref[:, 5]) | ref[:, 5].isnan()).all()
    got = dgate.cpu().double()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got == torch.inf, ref == torch.inf) and torch.equal(got == -torch.inf, ref == -torch.inf)
    assert (ref == torch.inf).any() and (ref == -torch.inf).any() and ref.isnan().any()
    ok = ref.isfinite()
    D, x64 = dl.cpu().double(), x.cpu().double()
    if with_picks:
        d = w * (dw - (w * dw).sum(1, keepdim=True))
        D = D.scatter_add(1, ids.cpu(), d.cpu().double())
    mag = torch.nan_to_num(D.abs(), posinf=0.0).t() @ torch.nan_to_num(x64.abs(), posinf=0.0)
    tol = (3 * T + 64) * 2.0 ** -23 * mag + torch.nan_to_num(err, nan=0.0, posinf=0.0) + 1e-37
    assert ((got - ref).abs()[ok] <= tol[ok]).all()


def test_balance_gradient_of_very_many_tokens(dev):
    """2^28 tokens: more than a launch has threads for at 16 tokens a workgroup of 256. Equal rows have equal gradients, known from the
    formula (scores of 1 / 2)."""
    from mi355moe import router
    T, E = (1 << 28) + 5, 2
    logits = torch.zeros((T, E), dtype=torch.float16, device=dev)
    counts = torch.tensor([3, 1], dtype=torch.int32, device=dev)
    dloss = torch.tensor(float(T) * T, device=dev)
    d = router.balance_loss_backward(dloss, logits, counts, torch.tensor(T, dtype=torch.int32, device=dev), 1)
    assert d.shape == logits.shape
    assert bool((d[:, 0] == d[0, 0]).all()) and bool((d[:, 1] == -d[0, 0]).all())
    assert abs(float(d[0, 0]) - E * 0.5 * (3 - 2)) <= 2.0 ** -10


@pytest.mark.parametrize("E", [20, 130])
def test_dx_where_picks_of_no_expert_have_the_large_gradients(dev, E):
    """They take part in the softmax's sum only; the row's scale is that of the picks of experts."""
    from mi355moe import router
    T, H = 70, 64
    x, gate, _, _, _, _ = router_inputs(T, H, E, 1, E, dev)
    ids = torch.tensor([3, -1, E]).repeat(T, 1).to(dev)
    ids[::2, 0] = E - 1
    w = torch.tensor([2.0 ** -30, 0.5, 0.5]).repeat(T, 1).to(dev)
    dw = torch.tensor([1.0, 2.0 ** 20, -2.0 ** 20]).repeat(T, 1).to(dev)
    dx, _ = router.topk_backward(x, gate, ids, w, dw, need_gate=False)
    want = gate[ids[:, 0]].cpu().double() * (2.0 ** -30 * (1 - 2.0 ** -30))
    close(dx, want, (2.0 ** -8 + 2.0 ** -19) * want.abs() + 2.0 ** -30 * 2.0 ** -33 * gate.abs().max().item())

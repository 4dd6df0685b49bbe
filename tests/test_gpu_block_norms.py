"""The norms between two sublayers (ops.add_normed_rmsnorm): what FP32 rows keep, and every form that rows and widths choose."""
import pytest
import torch

import plain_selective as plain
from test_gpu_selective import BF16, DEV, F32

pytestmark = pytest.mark.gpu


def _alike(rows, d, bits):
    """Rows of one number up to its sign, so small that the sums of its squares are exact: (y, the number)."""
    g = torch.Generator().manual_seed(d)
    whole = torch.randint(1 << (bits - 1), 1 << bits, (rows, 1), generator=g).float() * 2.0 ** torch.randint(-4, 4, (rows, 1), generator=g)
    return whole * (torch.randint(0, 2, (rows, d), generator=g) * 2 - 1), whole


@pytest.mark.parametrize("rows, d, bits", [(20000, 1, 11), (4000, 3, 11), (3000, 1001, 6), (200, 4096, 6), (700, 2048, 6), (40, 20001, 4), (3, 6001, 5)])
@pytest.mark.parametrize("out_type", [F32, BF16])
def test_float32_rows_keep_their_root_mean_square(rows, d, bits, out_type):
    """Exact sums leave, in half steps: one over the width and the mean with eps (1 each, half of it after the root), the root's inverse
    (its last rounding 1, half of the roundings in what the step of Newton's takes) and one product (1): 3.5.  In the second norm the
    squares and their sum as well: (d / 128 + 20) roundings one behind the other at most, half of them after the root."""
    from nanoinfer_b200.kernels import ops
    y, whole = _alike(rows, d, bits)
    eps, one = 0.0123, torch.ones(d, device=DEV)
    h, out = torch.zeros(rows, d, device=DEV), torch.empty(rows, d, dtype=out_type, device=DEV)
    ops.add_normed_rmsnorm(h, y.to(DEV), one, eps, one, eps, out)
    e = torch.tensor(eps).double()
    want = y.double() / torch.sqrt(whole.double() ** 2 + e)
    worst = ((h.double().cpu() - want) / want).abs().max().item() / plain.U
    assert worst <= 3.5, f"{worst:.2f} half steps"
    got = h.double().cpu()
    want = got / torch.sqrt((got * got).mean(1, keepdim=True) + e)
    bound = (3.5 + (d / 128 + 20) / 2) * plain.U + (plain.half_step(BF16) if out_type is BF16 else 0)
    worst = ((out.double().cpu() - want) / want).abs().max().item() / bound
    assert worst <= 1.001, f"{worst:.2f} times the bound"


@pytest.mark.parametrize("rows, d, bits", [(3000, 1001, 6), (3000, 4096, 6), (3000, 2999, 6), (400, 20001, 4)])
def test_float32_norms_are_as_exact_as_the_formula_in_32_bits(rows, d, bits):
    """The root mean square of the errors, where the sums are exact: below the formula's in 32 bits, step by step (a rounded mean, the
    library's root).  A twentieth below, as the kernel's root has one rounding behind its step of Newton's, the library's two units."""
    from nanoinfer_b200.kernels import ops
    y, whole = _alike(rows, d, bits)
    y = y.to(DEV)
    eps, one = 0.0123, torch.ones(d, device=DEV)
    h = torch.zeros(rows, d, device=DEV)
    ops.add_normed_rmsnorm(h, y, one, eps, None, 0.0, None)
    want = y.double() / torch.sqrt(whole.to(DEV).double() ** 2 + torch.tensor(eps).double().item())
    err, formula = (((t.double() - want) / want).square().mean().sqrt().item() / plain.U
                    for t in (h, y * torch.rsqrt(y.square().mean(1, keepdim=True) + eps)))
    assert err <= 0.95 * formula, f"{err:.3f} half steps, {formula:.3f} by the formula"


def test_rows_beyond_the_numbers():
    """Squares whose sum is infinite leave nothing (as the formula in 32 bits), a row of zeros without eps is no number."""
    from nanoinfer_b200.kernels import ops
    for kind in (F32, BF16):
        y = torch.ones(3, 96, dtype=kind, device=DEV)
        y[0], y[1] = 1e30, 0
        h, one = torch.zeros(3, 96, device=DEV), torch.ones(96, device=DEV)
        ops.add_normed_rmsnorm(h, y, one, 0.0, None, 0.0, None)
        assert (h[0] == 0).all() and h[1].isnan().all() and ((h[2] - 1).abs() <= 4 * plain.U).all()


# Rows beyond four per SM take eight numbers a thread and share an SM by threes; fewer rows few numbers a thread; widths that no
# 16-byte piece divides (or columns that begin off one) one number at a time, up to 8,192; wider ones are read twice.
@pytest.mark.parametrize("act", ["none", "silu", "sigmoid", "identity"])
@pytest.mark.parametrize("rows, d, left", [(700, 4096, 0), (700, 520, 0), (700, 2044, 0), (1201, 36, 0), (700, 2999, 0), (650, 1024, 1), (3, 6001, 0),
                                           (601, 8190, 0), (2, 4100, 0), (610, 16380, 0), (593, 5, 0)])
@pytest.mark.parametrize("y_type, out_type, in_place", [(BF16, BF16, False), (F32, F32, True), (BF16, F32, True)])
def test_every_form(act, rows, d, left, y_type, out_type, in_place):
    """Each form of the kernel with a last piece that is not whole, gated and not, against 64 bits; what lies around the columns stays."""
    from nanoinfer_b200.kernels import ops
    g = torch.Generator(device=DEV).manual_seed(rows + d)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def columns(t):
        whole = torch.full((t.shape[0], left + t.shape[1] + left), float("nan"), dtype=t.dtype, device=DEV)
        whole[:, left:left + t.shape[1]] = t
        return whole[:, left:left + t.shape[1]]

    h, y, w, gain = randn(rows, d) * 3, columns((randn(rows, d) * 2).to(y_type)), randn(d), randn(d)
    gate = None if act == "none" else columns(randn(rows, d).to(y_type))
    want, err, new, new_err = plain.norms(h, y, w, 1e-5, gain, 1e-6, 0.37, gate, act)
    stream, h_out = h.clone(), torch.full_like(h, 7.0)
    out = columns(torch.zeros(rows, d, dtype=out_type, device=DEV))
    ops.add_normed_rmsnorm(stream, y, w, 1e-5, gain, 1e-6, out, scale=0.37, gate=gate, gate_act=act, h_out=None if in_place else h_out)
    if not in_place:
        assert torch.equal(stream, h)
    for got, exact, bound, kind in ((stream if in_place else h_out, new, new_err, F32), (out, want, err, out_type)):
        worst = ((got.double() - exact).abs() / (bound + plain.half_step(kind) * (exact.abs() + bound) + 1e-37)).max().item()
        assert worst <= 1.0, f"{worst:.2f} times the bound"
    assert out._base is None or not left or (out._base[:, :left].isnan().all() and out._base[:, -left:].isnan().all())

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

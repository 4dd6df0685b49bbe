"""The operators of a selective state space layer where a call leaves the usual shape, against their formulas in 64 bits."""
import pytest
import torch

import plain_selective as plain
from test_gpu_selective import BF16, DEV, F32, _close, _conv_case, _cu, _i32, _scan, _scan_case

pytestmark = pytest.mark.gpu


def _behind(first, t, pad=5):
    """``t`` as the rows from ``first`` on of a matrix whose other rows hold NaN."""
    whole = torch.full((first + t.shape[0] + pad, t.shape[1]), float("nan"), dtype=t.dtype)
    whole[first:first + t.shape[0]] = t
    return whole.to(DEV)


BEHIND = {"two": [40, 56], "short": [2, 1, 3, 0, 1], "uneven": [40, 4, 0, 56, 1, 130], "many": [3, 0, 1, 17] * 10 + [90], "tokens": [1] * 9,
          "long": [700, 30]}


@pytest.mark.parametrize("first", [1, 7, 8, 16, 301])
@pytest.mark.parametrize("lens", BEHIND)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_first_row_above_zero(lens, first, dtype):
    """The later requests of a step, handed over with the whole step's rows: every request's state moves on once, in place and not, and
    rows that belong to no request stay.  In place several times (which of two blocks comes first is open)."""
    from nanoinfer_b200.kernels import ops
    lens = BEHIND[lens]
    n = sum(lens)
    rows = slice(first, first + n)
    cu = _cu([first] + lens)[1:]
    told = max(lens)
    for d in (40, 33):
        k, s = _conv_case(lens, d, 4, dtype, first + d), _scan_case(lens, d, 16, 1, dtype, first + d)
        x, u, dt, b, c, z = (_behind(first, t) for t in (k["x"], s["u"], s["dt"], s["b"], s["c"], s["z"]))
        for in_place in (True, False):
            to = k["slots"] if in_place else k["to"]
            want, err, new = plain.convolution(k["x"], k["w"], k["bias"], k["state"], lens, k["slots"], to, True)
            for turn in range(4 if in_place else 1):
                out, state = torch.full_like(x, 7.0), k["state"].to(DEV)
                ops.short_convolution(x, k["w"].to(DEV), k["bias"].to(DEV), state, cu, _i32(k["slots"]), len(lens), out,
                                      to_slots=None if in_place else _i32(to), max_q_len=told if turn % 2 else None)
                _close(out[rows], want, err, dtype, "convolution")
                assert torch.equal(state.double().cpu(), new), "the kept inputs"
                assert (out[:first] == 7).all() and (out[first + n:] == 7).all()
            to = s["slots"] if in_place else s["to"]
            want, err, new, new_err = plain.scan(s["u"], s["dt"], s["a"], s["b"], s["c"], s["state"], lens, s["slots"], to, s["skip"],
                                                 s["dt_bias"], s["z"])
            for max_q_len in (None, told):
                out, state = torch.full_like(u, 7.0), s["state"].to(DEV)
                ops.selective_scan(u, dt, s["a"].to(DEV), b, c, state, cu, _i32(s["slots"]), len(lens), out, skip=s["skip"].to(DEV),
                                   dt_bias=s["dt_bias"].to(DEV), z=z, to_slots=None if in_place else _i32(to), max_q_len=max_q_len)
                _close(out[rows], want, err, dtype, "scan")
                _close(state, new, new_err, F32, "state")
                assert (out[:first] == 7).all() and (out[first + n:] == 7).all()


def test_the_later_requests_of_a_step():
    """A step's rows, offsets and slots, first whole, then in two calls that take the lists from a request on: the same bits."""
    from nanoinfer_b200.kernels import ops
    lens = [50, 33, 1, 7, 64, 12]
    k = _conv_case(lens, 72, 4, F32, 3)
    x, w, cu, slots = k["x"].to(DEV), k["w"].to(DEV), _cu(lens), _i32(k["slots"])
    want, kept = torch.empty_like(x), k["state"].to(DEV)
    ops.short_convolution(x, w, None, kept, cu, slots, len(lens), want)
    for at in (1, 2, 4, 5):
        out, state = torch.empty_like(x), k["state"].to(DEV)
        ops.short_convolution(x, w, None, state, cu[at:], slots[at:], len(lens) - at, out)
        ops.short_convolution(x, w, None, state, cu, slots, at, out)
        assert torch.equal(out, want) and torch.equal(state, kept), at


@pytest.mark.parametrize("n, d", [(1, 40), (5, 33), (16, 40), (16, 33), (8, 64), (64, 16), (128, 24)])
@pytest.mark.parametrize("form", ["portion", "stepwise", "tokens", "parts"])
def test_steps_are_as_exact_far_below_zero(form, n, d):
    """delta alone, all over softplus' range: every other factor is one, nothing is left of the state before and one state is read.
    In half steps: 2^x is off by 4 (two units in the last place, its documented bound), what the argument's rounding is worth is
    multiplied in (1), with ln 2 rounded to 1.905e-9 (|v| log2(e) of that, 0.0461 |v|), the polynomial's ten steps leave 2.1 (each
    rounded at its size, times the powers of e <= 1 behind it, over the smallest value ln 2) and the last sum 1: 8.1 + 0.0461 |v|."""
    from nanoinfer_b200.kernels import ops
    g = torch.Generator().manual_seed(n + d)
    t = {"tokens": 90, "parts": 500}.get(form, 300)
    low = torch.tensor([-86.0, -20.0, -8.0, -1.0, -0.01, 1.0])
    high = torch.tensor([-20.0, -8.0, -1.0, 1.0, 0.01, 30.0])
    which = torch.randint(0, 6, (t, d), generator=g)
    v = low[which] + (high - low)[which] * torch.rand(t, d, generator=g)
    v[0, :3] = torch.tensor([0.0, -0.0, -86.0])
    want = torch.logaddexp(v.double(), torch.zeros((), dtype=torch.float64))
    one = torch.zeros(t, n)
    one[:, n // 2] = 1
    lens = [1] * t if form == "tokens" else [t]
    out, state = torch.empty(t, d, device=DEV), torch.zeros(t, d * n, device=DEV)
    ops.selective_scan(torch.ones(t, d, device=DEV), v.to(DEV), torch.full((d, n), -1e38, device=DEV), torch.ones(t, n, device=DEV), one.to(DEV),
                       state, _cu(lens), _i32(list(range(len(lens)))), len(lens), out, max_q_len=max(lens), stepwise=form == "stepwise")
    gone = want * 1e38 > 200           # (a decay below e^-200; the smallest steps keep some of the state before)
    worst = ((out.double().cpu() - want).abs() / (want * (8.1 + 0.0461 * v.double().abs()) * plain.U))[gone].max().item()
    assert gone.float().mean() > 0.9 and worst <= 1.0, f"{worst:.2f} times the bound"


@pytest.mark.parametrize("lens", [[3], [1, 1, 1], [70]])
def test_steps_that_are_not_finite(lens):
    """An infinite step where softplus' argument is one, none where it is minus infinity (the state before stays: 4 half steps of 2^x),
    NaN where it is NaN."""
    from nanoinfer_b200.kernels import ops
    t, d = sum(lens), 24
    v = torch.zeros(t, d)
    v[1, 4], v[1, 9], v[1, 14] = float("inf"), float("-inf"), float("nan")
    ones = torch.ones(t, 1, device=DEV)
    out, state = torch.empty(t, d, device=DEV), torch.zeros(t, d, device=DEV)
    ops.selective_scan(torch.ones(t, d, device=DEV), v.to(DEV), torch.full((d, 1), -1e38, device=DEV), ones, ones, state, _cu(lens),
                       _i32(list(range(len(lens)))), len(lens), out, max_q_len=max(lens))
    row = out[1].cpu()
    before = out[0, 9].item() if lens[0] > 1 else 0.0
    assert abs(row[9] - before) <= 4 * plain.U * before
    assert row[4] == float("inf") and row[14].isnan() and row[[0, 3, 5, 8, 10, 13, 15, 23]].isfinite().all()


@pytest.mark.parametrize("count, d, n, groups", [(61, 8192, 16, 1), (50, 8200, 16, 1), (40, 16384, 8, 1), (61, 4096, 32, 2), (61, 2048, 64, 4),
                                                 (61, 1024, 128, 1), (130, 40, 16, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_single_tokens_in_many_groups(count, d, n, groups, dtype):
    """So many requests of one token for their channels that a block walks several groups of them, past those whose states are on
    their way from the start; some have no tokens, some no row to come from or to go to."""
    from nanoinfer_b200.kernels import ops
    lens = [1] * count
    for i in (3, 10, count - 2):
        lens[i] = 0
    k = _scan_case(lens, d, n, groups, dtype, d + n)
    rows = len(k["state"])
    k["slots"] = [(-1 if i % 11 == 4 else rows + 3 if i % 11 == 9 else v) for i, v in enumerate(k["slots"])]
    k["to"] = [(-2 if i % 13 == 6 else rows if i % 13 == 12 else v) for i, v in enumerate(k["to"])]
    for in_place in (False, True):
        to = k["slots"] if in_place else k["to"]
        want, err, new, new_err = plain.scan(k["u"], k["dt"], k["a"], k["b"], k["c"], k["state"], lens, k["slots"], to, k["skip"], k["dt_bias"], k["z"])
        out, state = _scan(ops, k, lens, in_place)
        _close(out, want, err, dtype, "out")
        _close(state, new, new_err, F32, "state")


@pytest.mark.parametrize("lens", [[173], [40, 0, 205]])
@pytest.mark.parametrize("d, n", [(8192, 16), (8200, 16), (4096, 16), (1024, 64), (640, 128), (4096, 8), (2048, 32)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_tiles_of_many_channels(lens, d, n, dtype):
    """Enough tiles that each of a block's two buffers is filled several times, and a last one that is not whole, in blocks of every
    number of channels and lanes (64 channels of 16 states where there are many)."""
    from nanoinfer_b200.kernels import ops
    k = _scan_case(lens, d, n, 1, dtype, d + n)
    want, err, new, new_err = plain.scan(k["u"], k["dt"], k["a"], k["b"], k["c"], k["state"], lens, k["slots"], k["to"], k["skip"], k["dt_bias"], k["z"])
    for given in (dict(), dict(stepwise=True)) if dtype == F32 else (dict(),):
        out, state = _scan(ops, k, lens, **given)
        _close(out, want, err, dtype, "out")
        _close(state, new, new_err, F32, "state")

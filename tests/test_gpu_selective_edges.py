"""The operators of a selective state space layer where a call leaves the usual shape, against their formulas in 64 bits."""
import pytest
import torch

import plain_selective as plain
from test_gpu_selective import BF16, DEV, F32, _close, _conv_case, _cu, _i32, _scan_case

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

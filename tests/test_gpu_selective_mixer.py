"""What the selective state space mixer hands to the arrangement around it."""
from types import SimpleNamespace

import pytest
import torch

import plain_selective as plain
from test_gpu_selective import BF16, DEV, F32, _cu, _i32

pytestmark = pytest.mark.gpu
WIDTH, CHANNELS, STATES, TAPS = 64, 136, 16, 4
EXTRA = (("channels", CHANNELS), ("state_size", STATES), ("conv_taps", TAPS))


def _runtime(dtype):
    from nanoinfer_b200.engine.runtime import Runtime
    return Runtime(device=torch.device(DEV), dtype=dtype, page_size=8)


def _weights(cls, spec, seed):
    g = torch.Generator().manual_seed(seed)
    return {slot: torch.randn(tuple(int(n) for n in ws.shape), generator=g) * 0.2 for slot, ws in cls.weight_slots(spec, WIDTH).items()}


def _step(lens, rows):
    """A step's context and a cache of fresh states."""
    ctx = SimpleNamespace(cu_q=_cu(lens), slots=_i32(list(range(len(lens)))), n_seqs=len(lens), max_q_len=max(lens), positions=None)
    return ctx, SimpleNamespace(state=torch.zeros(rows, CHANNELS * (STATES + TAPS - 1), device=DEV))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens", [[40], [9, 30, 1], [1] * 20, [1] * 4])
def test_the_output_is_not_rounded(dtype, lens, monkeypatch):
    """The last product comes in FP32, whatever the rows: a sum of CHANNELS products, in FP32 each rounding at most half a step of the
    sum of their sizes."""
    from nanoinfer_b200.config import MixerSpec, part
    rt = _runtime(dtype)
    cls, spec = part("mixer", "selective_scan"), MixerSpec("selective_scan", extra=EXTRA)
    mixer = cls(spec, WIDTH, _weights(cls, spec, 5), rt)
    calls, linear = [], rt.linear

    def kept(x, w, *args, **kw):
        calls.append((x, w))
        return linear(x, w, *args, **kw)

    monkeypatch.setattr(rt, "linear", kept)
    ctx, cache = _step(lens, len(lens))
    out = mixer.forward(torch.randn(sum(lens), WIDTH, generator=torch.Generator().manual_seed(6)).to(DEV).to(dtype), ctx, cache)
    y, w = (t.double() for t in calls[-1])
    assert out.dtype == F32
    err = (out.double() - y @ w.t()).abs()
    assert (err <= (CHANNELS + 1) * plain.U * (y.abs() @ w.abs().t())).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("first", [True, False])
def test_beside_another_mixer(dtype, first):
    """One of two mixers that read the same input, on either side: the weighted sum of what both give alone."""
    from nanoinfer_b200.config import MixerSpec, part
    from nanoinfer_b200.config.registry import register_part
    from nanoinfer_b200.parts.base import Part, WeightSlot

    class Projection(Part):
        @staticmethod
        def weight_slots(spec, hidden_size):
            return {"w": WeightSlot((hidden_size, hidden_size))}

        def __init__(self, spec, hidden_size, weights, rt):
            Part.__init__(self, spec, hidden_size, weights, rt)
            self.w = rt.weight(weights["w"])

        def cache_need(self):
            return None

        def forward(self, x, ctx, cache):
            return self.rt.linear(x, self.w, out_dtype=F32)

    register_part("mixer", "projection_for_test", Projection, replace=True)
    rt = _runtime(dtype)
    sides = [MixerSpec("selective_scan", extra=EXTRA), MixerSpec("projection_for_test")]
    sides = sides if first else sides[::-1]
    spec = MixerSpec("parallel_mixers", extra=(("left", sides[0]), ("right", sides[1]), ("left_scale", 1.3), ("right_scale", 0.7)))
    cls = part("mixer", "parallel_mixers")
    weights = _weights(cls, spec, 8)
    both = cls(spec, WIDTH, weights, rt)
    x = torch.randn(33, WIDTH, generator=torch.Generator().manual_seed(9)).to(DEV).to(dtype)
    ctx, cache = _step([30, 3], 2)
    out = both.forward(x, ctx, cache)
    want, size = 0.0, 0.0
    for name, side, scale in (("left", sides[0], 1.3), ("right", sides[1], 0.7)):
        own = {slot[len(name) + 1:]: w for slot, w in weights.items() if slot.startswith(name + ".")}
        alone = part("mixer", side.kind)(side, WIDTH, own, rt).forward(x, *_step([30, 3], 2)).double() * scale
        want, size = want + alone, size + alone.abs()
    assert out.dtype == F32 and ((out.double() - want).abs() <= 4 * plain.U * size).all()       # scales, products and the sum

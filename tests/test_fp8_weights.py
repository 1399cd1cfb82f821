"""Weights in 8 bits, and who holds them (no GPU)."""
from __future__ import annotations

import pytest
import torch

from quanta_b200 import fp8
from quanta_b200.config import GuravikConfig, MiniMaxM3Config
from quanta_b200.config.registry import resolve
from quanta_b200.engine.model import Model
from quanta_b200.parts.dense import GatedDense
from tests.conftest import TINY


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (130, 300), (500, 64), (257, 129)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_weight(n, k, dtype):
    """Off by half a step of e4m3, 2^-4 of a normal number and 2^-10 of the scale below; the scales as defined; blocks do not see one another."""
    g = torch.Generator().manual_seed(n + k)
    w = (torch.randn(n, k, generator=g) * torch.exp(3 * torch.randn(n, 1, generator=g))).to(dtype)
    q = fp8.quantize_weight(w)
    assert q.q.dtype == torch.float8_e4m3fn and q.shape == (n, k) and q.scales.shape == (-(-n // 128), -(-k // 128))
    scales = q.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    assert torch.all((q.dequantized().double() - w.double()).abs() <= torch.maximum(2.0 ** -4 * w.double().abs(), 2.0 ** -10 * scales) * (1 + 1e-6))
    for r in range(q.scales.shape[0]):
        for c in range(q.scales.shape[1]):
            largest = w[128 * r: 128 * r + 128, 128 * c: 128 * c + 128].abs().max().float()
            assert torch.allclose(q.scales[r, c], largest / 448, rtol=1e-6)
    again = fp8.quantize_weight(w, rows_at_a_time=128)
    assert torch.equal(again.q.float(), q.q.float()) and torch.equal(again.scales, q.scales)


def test_quantize_weight_of_zeros_and_refusals():
    z = fp8.quantize_weight(torch.zeros(130, 20))
    assert torch.all(z.q.float() == 0) and torch.all(z.scales > 0) and torch.all(z.dequantized() == 0)
    for bad in (float("nan"), float("inf")):
        w = torch.ones(4, 4)
        w[1, 2] = bad
        with pytest.raises(ValueError, match="NaN"):
            fp8.quantize_weight(w)
    with pytest.raises(ValueError, match="128"):
        fp8.quantize_weight(torch.ones(4, 4), rows_at_a_time=100)


def _dense(hidden, inner):
    part = GatedDense(hidden, inner, {"gate": "g", "up": "u", "down": "d"})
    g = torch.Generator().manual_seed(1)
    w = {"g": torch.randn(inner, hidden, generator=g), "u": torch.randn(inner, hidden, generator=g), "d": torch.randn(hidden, inner, generator=g)}
    part.load(w.__getitem__)
    return part, w


def test_a_feed_forward_holds_its_matrices():
    part, w = _dense(64, 48)
    assert not part.reads_fp8
    part.hold_in_fp8()
    assert part.reads_fp8 and part.w_gate_up.shape == (96, 64) and part.w_down.shape == (64, 48)
    assert torch.all((part.w_gate_up.dequantized()[:48] - w["g"]).abs() <= 2.0 ** -4 * w["g"].abs() + 2.0 ** -10 * part.w_gate_up.scales.max())
    held = part.w_down
    part.hold_in_fp8()                    # once
    assert part.w_down is held
    for hidden, inner in ((64, 40), (72, 48)):
        with pytest.raises(ValueError, match="multiples of 16"):
            _dense(hidden, inner)[0].hold_in_fp8()


def test_models_that_hold_dense_weights():
    raw = {"architecture": "Guravik", "vocab": 50, "width": 32, "canon": {"taps": 2}, "loop": {"start": 0, "stop": 0, "times": 1}, "embedding": {"scale": 1.0},
           "norm": {"eps": 1e-5}, "layers": [{"type": "general_delta", "mixer": {"heads": 2, "dim": 8}, "mlp": {"kind": "dense", "ff": 48}}]}
    cfg = GuravikConfig.from_dict(raw)
    spec = resolve(raw).build_spec(cfg)
    assert Model(spec, device="cpu", dense_weights="fp8").dense_weights == "fp8"
    with pytest.raises(ValueError, match="fp8"):
        Model(spec, device="cpu", dense_weights="int4")
    m3 = MiniMaxM3Config.from_dict(TINY["A"])
    with pytest.raises(ValueError, match="no gated dense"):
        Model(resolve(TINY["A"]).build_spec(m3), device="cpu", dense_weights="fp8")


def test_a_text_of_one_token_has_no_perplexity():
    from quanta_b200.engine.score import TextScores
    assert TextScores([-1.0, -3.0], [1.0, 1.0]).perplexity == pytest.approx(7.38905609893065)
    assert TextScores().perplexity != TextScores().perplexity

"""The 8-bit feed-forward and the scoring as a model uses them.

Every operator of a run is held against float64 on the very numbers that it was given, with the bounds of ``test_fp8_gpu`` and
``test_token_logprobs_gpu``; whole models against themselves, run another way."""
from __future__ import annotations

import json
import math
import subprocess
import sys

import pytest
import torch

from tests import helpers as H
from tests.plain import guravik_plain as GP
from tests.test_fp8_gpu import U, _act, _product_within, _rows_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class _Ctx:
    def __init__(self, dtype):
        self.dtype, self.status = dtype, torch.zeros(4, dtype=torch.int32, device=DEV)


def _norm(width, gain, eps=1e-5):
    from quanta_b200.parts.norms import RMSNorm
    n = RMSNorm(width, eps, "n")
    n.weight = gain
    return n


def _dense(hidden, inner, activation, biases, dtype, seed):
    from quanta_b200.parts.dense import GatedDense
    g = torch.Generator(device=DEV).manual_seed(seed)
    part = GatedDense(hidden, inner, {k: k for k in ("gate", "up", "down", "gate_b", "up_b", "down_b")}, activation, biases, limit=3.0, alpha=1.702)
    shapes = {s.name: s for s in part.tensor_specs()}
    part.load(lambda name: (torch.randn(shapes[name].shape, device=DEV, generator=g) * (0.05 if shapes[name].kind == "matrix" else 0.3)
                            ).to(dtype if shapes[name].kind == "matrix" else torch.float32))
    part.hold_in_fp8()
    return part


@pytest.mark.parametrize("activation,biases", [("silu", False), ("clamped", True), ("gelu_tanh", False), ("silu", True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 7, 40, 150])
def test_norm_and_feed_forward(T, dtype, activation, biases, monkeypatch):
    """The norm into 8-bit rows, the two products and the activation, stage by stage on what the stage before left."""
    from quanta_b200 import kernels
    from quanta_b200.parts.base import Addends, NormedPending
    from quanta_b200.parts.norms import rows_for
    hidden, inner = 272, 400
    g = torch.Generator(device=DEV).manual_seed(T)
    part = _dense(hidden, inner, activation, biases, dtype, T)
    norm, post = _norm(hidden, 1 + 0.2 * torch.randn(hidden, device=DEV, generator=g)), _norm(hidden, torch.randn(hidden, device=DEV, generator=g), 1e-6)
    h, y = torch.randn(T, hidden, device=DEV, generator=g), torch.randn(T, hidden, device=DEV, generator=g)
    h0, seen = h.clone(), []
    for name in ("add_rmsnorm_fp8", "glu_act_fp8", "linear_fp8"):
        def spy(*a, _f=getattr(kernels, name), _n=name, **k):
            _f(*a, **k)
            seen.append((_n, a, k))
        monkeypatch.setattr(kernels, name, spy)
    rows = rows_for(part, norm, h, hidden, dtype)
    norm.forward(h, NormedPending(y, post), rows)
    ctx = _Ctx(dtype)
    out = part.forward(rows, ctx)
    assert [n for n, _, _ in seen] == ["add_rmsnorm_fp8", "linear_fp8", "glu_act_fp8", "linear_fp8"] and int(ctx.status[0]) == 0
    c = 2 * (hidden + 9) * U
    r = ((y.double() ** 2).mean(1, keepdim=True) + 1e-6).rsqrt()
    z = post.weight.double() * y.double() * r
    A = h0.double().abs() + 2 * z.abs()
    x = h0.double() + z
    assert torch.all((h.double() - x).abs() <= c * A)
    r = ((x * x).mean(1, keepdim=True) + 1e-5).rsqrt()
    off = c * norm.weight.double().abs() * r * (A + x.abs() * A.norm(dim=1, keepdim=True) / x.norm(dim=1, keepdim=True))
    _rows_within(rows.q, rows.scales, norm.weight.double() * x * r, off)
    for at in (1, 3):
        xq, xs, wq, ws, o = seen[at][1][:5]
        _product_within(o, xq, xs, wq, ws)
        assert o.dtype == (dtype if at == 1 else torch.float32)
    gate_up, q, s = seen[2][1][:3]
    both = gate_up.double() + (part.b_gate_up.double() if biases else 0.0)
    gate, up = both[:, :inner], both[:, inner:]
    v = _act(part.KINDS[activation], gate, up, 3.0, 1.702)
    arg = 2 * (gate.abs() + gate.abs() ** 3) if activation == "gelu_tanh" else 2 * gate.abs()
    size = gate_up.double().abs() + (part.b_gate_up.double().abs() if biases else 0.0)
    off = 32 * U * (1 + arg) * v.abs() + 2 * U * (size[:, :inner] * (up.abs() + 1) + size[:, inner:] * (gate.abs() + 1))
    _rows_within(q, s, v, off)
    assert isinstance(out, Addends) == biases
    # rows of the activation dtype are brought to 8 bits by the part itself
    plain = torch.randn(T, hidden, device=DEV, generator=g).to(dtype)
    seen.clear()
    part.forward(plain, ctx)
    xq, xs = seen[0][1][:2]
    _rows_within(xq, xs, plain.double(), torch.zeros_like(plain.double()))


def test_norms_that_write_8_bits_in_two_launches():
    """Addends that no single launch takes go through float32 rows: within the bound of e4m3 of the float32 norm."""
    from quanta_b200 import fp8
    from quanta_b200.parts.base import Addends, NormedPending, StreamCopy
    g = torch.Generator(device=DEV).manual_seed(5)
    norm, post = _norm(128, 1 + 0.2 * torch.randn(128, device=DEV, generator=g)), _norm(128, torch.randn(128, device=DEV, generator=g))
    y, e, b = (torch.randn(n, 128, device=DEV, generator=g) for n in (6, 6, 1))
    rows = torch.tensor([4, 0], dtype=torch.int32, device=DEV)
    for delta in (None, StreamCopy(y), y, y.bfloat16(), torch.stack([y, e], 1), Addends(y, bias=b[0]), Addends(y, extra=e), NormedPending(y, post),
                  NormedPending(Addends(y, extra=e, scale=0.5), post), NormedPending(torch.stack([y, e], 1), post)):
        for sel, store in ((None, True), (rows, False), (rows, True)):
            h = torch.randn(6, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6))
            h2 = h.clone()
            want = torch.empty(6 if sel is None else 2, 128, device=DEV)
            norm.forward(h, delta, want, rows=sel, store_h=store)
            out = fp8.empty_rows(want.shape[0], 128, DEV)
            norm.forward(h2, delta, out, rows=sel, store_h=store)
            assert torch.allclose(h2, h, rtol=1e-5, atol=1e-5)
            _rows_within(out.q, out.scales, want.double(), 1e-5 * (1 + want.double().abs()))


def _guravik(tmp_path, seed=3):
    from quanta_b200.weights.safetensors_io import write_safetensors
    cfg = {"architecture": "Guravik", "vocab": 97, "width": 64, "canon": {"taps": 3}, "loop": {"start": 0, "stop": 0, "times": 1}, "embedding": {"scale": 3.0},
           "norm": {"eps": 1e-5},
           "layers": [{"type": "general_delta", "mixer": {"heads": 2, "dim": 24}, "mlp": {"kind": "dense", "ff": 48}},
                      {"type": "latent_attention", "mlp": {"kind": "dense", "ff": 80},
                       "mixer": {"heads": 3, "dim": 16, "rot_dim": 8, "vdim": 24, "q_rank": 20, "kv_rank": 40, "scale": 1.0 / math.sqrt(24),
                                 "rot": {"base": 10000.0, "dims": 8}}}]}
    weights = GP.draw_weights(cfg, seed=seed, decay_rank=12)
    write_safetensors(tmp_path / "model.safetensors", weights)
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    return tmp_path, weights, cfg


def _spread(rows: dict, want: dict) -> float:
    return max(float((rows[k] - want[k] - (rows[k] - want[k]).mean()).pow(2).mean().sqrt() / want[k].std()) for k in want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_model_with_8_bit_feed_forwards(tmp_path, dtype):
    """Near the model it was made from (a feed-forward's output is off by some 4 % of itself: two roundings of e4m3, each 2^-4 / sqrt(3) at most and
    averaged over the columns; 0.25 of the logits' spread is several times what two layers make of that), the same in every cutting but for
    rounding, and its captured decode steps are those of the eager ones."""
    from quanta_b200.engine.model import load_model
    from quanta_b200.engine.step import Engine
    folder, weights, cfg = _guravik(tmp_path)
    reqs = {f"r{i}": H.random_tokens(n, 97, 20 + i) for i, n in enumerate((1, 37, 90))}
    want = {}
    for rid, toks in reqs.items():
        lg = GP.forward(weights, cfg, toks)
        want |= {(rid, i): lg[i] for i in range(len(toks))}
    got = {}
    for name, steps in (("whole", H.cut_whole(reqs)), ("decode", H.cut_tail_decode(reqs, tail=30)), ("mixed", H.cut_mixed(reqs, max_live=3, seed=5))):
        model, _ = load_model(folder, dtype=dtype, dense_weights="fp8")
        assert all(b.feed_forward.reads_fp8 for b in model.blocks)
        eng = Engine(model, num_pages=64, page_size=16, max_requests=4)
        got[name] = H.replay(eng, steps)
        assert len(got[name]) == len(want) and _spread(got[name], want) < 0.25
        if name == "decode":
            assert eng.graph_replays > 0
    for name in ("decode", "mixed"):
        assert _spread(got[name], got["whole"]) < 0.12


def test_generation_and_scores_with_8_bit_feed_forwards(tmp_path):
    from quanta_b200 import generate
    from quanta_b200.engine.generate import LLM
    folder, _, _ = _guravik(tmp_path)
    llm = LLM(folder, dtype="float32", dense_weights="fp8", num_pages=64, max_requests=4)
    prompts = [H.random_tokens(n, 97, n) for n in (5, 12)]
    outs = generate(llm, prompts, max_new_tokens=8, eos_id=[])
    assert all(len(o) == 8 for o in outs)
    scores = llm.score([p + o for p, o in zip(prompts, outs)], top=3)
    for p, o, s in zip(prompts, outs, scores):
        assert len(s.logprobs) == len(p) + 7 and s.perplexity > 1.0
        for i in range(8):
            at = len(p) - 1 + i
            # the greedy token is the most probable one, but where a step of another shape rounds a near tie the other way
            assert s.top_ids[at][0] == o[i] or s.top_logprobs[at][0] - s.logprobs[at] < 0.05
    with pytest.raises(ValueError, match="Model"):
        from quanta_b200.engine.model import load_model
        LLM(load_model(folder)[0], dense_weights="fp8")


@pytest.mark.parametrize("budget", [4096, 7])
def test_scores_are_the_plain_models(model_dirs, plain_models, budget):
    """float32: a logit is off by at most a few 1e-4 of the logits' spread (the engine's own tests), a log probability by twice that."""
    from quanta_b200.engine.generate import LLM
    from tests.plain import minimax_m3_plain as P
    weights, cfg = plain_models["A"]
    llm = LLM(str(model_dirs["A"]), dtype="float32", page_size=4, num_pages=24, max_requests=2, max_step_tokens=budget, prefill_chunk=16)
    texts = [H.random_tokens(n, 512, n) for n in (30, 1, 2, 17, 41, 5)]
    scores = llm.score(texts, top=4)
    for text, s in zip(texts, scores):
        n = len(text) - 1
        assert len(s.logprobs) == len(s.entropies) == len(s.top_ids) == len(s.top_logprobs) == n
        if not n:
            continue
        lp = torch.log_softmax(P.forward_logits(weights, cfg, text).double(), 1)[:-1]
        want = lp.gather(1, torch.tensor(text[1:])[:, None])[:, 0]
        tol = 1e-3 * float(lp.std())
        assert torch.all((torch.tensor(s.logprobs).double() - want).abs() <= tol)
        assert torch.all((torch.tensor(s.entropies).double() - torch.special.entr(lp.exp()).sum(1)).abs() <= 10 * tol)
        top = torch.tensor(s.top_ids)
        best = lp.topk(4, 1)
        assert torch.all((torch.tensor(s.top_logprobs).double() - best.values).abs() <= tol)
        assert torch.all((lp.gather(1, top) - best.values).abs() <= 2 * tol)
        assert s.perplexity == pytest.approx(math.exp(-float(want.mean())), rel=2 * tol)
    assert llm.engine.manager.stats()["live_requests"] == 0
    one = llm.score(texts[0])
    assert one.top_ids == [] and one.logprobs == pytest.approx(scores[0].logprobs, abs=1e-4)


def test_refusals_of_scoring(model_dirs):
    from quanta_b200.cache.manager import OutOfPages
    from quanta_b200.engine.generate import LLM
    llm = LLM(str(model_dirs["A"]), dtype="float32", page_size=4, num_pages=4, max_requests=2)
    for texts, top in (([[]], 0), ([[1, 2], [512, 3]], 0), ([[1, -1]], 0), ([[1, 2]], 65), ([[1, 2]], -1)):
        with pytest.raises(ValueError):
            llm.score(texts, top=top)
    with pytest.raises(OutOfPages):
        llm.score([[1, 2, 3], list(range(40))])
    assert llm.engine.manager.stats()["live_requests"] == 0
    assert len(llm.score([[1, 2, 3]])[0].logprobs) == 2


def test_score_command(model_dirs, tmp_path):
    file = tmp_path / "texts"
    file.write_text("5,17,3\n9 9\n")
    r = subprocess.run([sys.executable, "-m", "quanta_b200", "score", "--model", str(model_dirs["A"]), "--prompt-file", str(file), "--top", "2", "--dtype", "float32",
                        "--max-requests", "2", "--num-pages", "16"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    lines = [json.loads(line) for line in r.stdout.strip().splitlines()]
    assert [x["tokens"] for x in lines] == [3, 2] and [len(x["logprobs"]) for x in lines] == [2, 1] and len(lines[0]["top_ids"][0]) == 2

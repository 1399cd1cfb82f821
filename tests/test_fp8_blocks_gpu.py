"""8-bit feed-forwards in every kind of block that holds one: after a norm that writes 8-bit rows, beside a mixer on a second stream, behind norms in
groups with biases, and as the expert that every token passes; kernel by kernel and in captured steps.

Every kernel of a step is held against float64 on the very numbers it was given, with the bounds of ``test_fp8_gpu``, and each has to read what the one
before it left.  Captured steps repeat the eager ones' bits: the same kernels with the same launch sizes on the same numbers, no sum whose order varies."""
from __future__ import annotations

import importlib
import json

import pytest
import torch

from tests import helpers as H
from tests.test_fp8_gpu import U, _act, _product_within, _rows_within
from tests.test_fp8_model_gpu import _guravik

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WRITERS = ("add_rmsnorm_fp8", "rows_to_fp8")


def _watch(monkeypatch) -> list:
    """Every call of the 8-bit kernels from here on, in order: (name, arguments, options)."""
    from quanta_b200 import kernels
    seen: list = []
    for name in (*WRITERS, "glu_act_fp8", "linear_fp8"):
        def spy(*a, _f=getattr(kernels, name), _n=name, **k):
            _f(*a, **k)
            seen.append((_n, a, k))
        monkeypatch.setattr(kernels, name, spy)
    return seen


def _check_feed_forward(calls, dtype):
    """One feed-forward's four launches: rows, gate and up, activation, down."""
    (first, a, k), (_, gate_up, _), (_, act, opts), (_, down, _) = calls
    q, s = a[4:6] if first == "add_rmsnorm_fp8" else a[1:3]
    if first == "rows_to_fp8":
        _rows_within(q, s, a[0].double(), torch.zeros_like(a[0].double()))
    assert torch.all(torch.isfinite(q.float())) and torch.all(torch.isfinite(s))
    assert gate_up[0].data_ptr() == q.data_ptr() and gate_up[1].data_ptr() == s.data_ptr()
    assert act[0].data_ptr() == gate_up[4].data_ptr() and down[0].data_ptr() == act[1].data_ptr() and down[1].data_ptr() == act[2].data_ptr()
    assert gate_up[4].dtype == dtype and down[4].dtype == torch.float32
    for p in (gate_up, down):
        x, xs, w, ws, out = p[:5]
        _product_within(out, x, xs, w, ws)
    x, b, inner = act[0].double(), opts["bias"], act[1].shape[1]
    both = x if b is None else x + b.double()
    gate, up = both[:, :inner], both[:, inner:]
    v = _act(opts["kind"], gate, up, opts["limit"], opts["alpha"])
    arg = 2 * (gate.abs() + gate.abs() ** 3) if opts["kind"] == 2 else 2 * gate.abs()
    size = x.abs() if b is None else x.abs() + b.double().abs()
    _rows_within(act[1], act[2], v, 32 * U * (1 + arg) * v.abs() + 2 * U * (size[:, :inner] * (up.abs() + 1) + size[:, inner:] * (gate.abs() + 1)))


def _folder(tmp_path, name):
    if name == "guravik":
        return _guravik(tmp_path)[0]
    from quanta_b200.weights.safetensors_io import write_safetensors
    module = importlib.import_module(f"tests.test_{name}_gpu")
    cfg = module.CONFIGS["D"]
    write_safetensors(tmp_path / "model.safetensors", module.P.draw_weights(cfg, seed=11))
    (tmp_path / "config.json").write_text(json.dumps(getattr(module, "_file_config", lambda c: c)(cfg)))
    return tmp_path


# how many 8-bit feed-forwards the model has, and what writes the rows of the first
MODELS = {"guravik": (2, "add_rmsnorm_fp8"), "lotilix": (4, "rows_to_fp8"), "puvolix": (2, "rows_to_fp8"), "tarulix": (3, "rows_to_fp8"), "gedelorn": (2, None)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(MODELS))
def test_the_feed_forwards_of_a_model(tmp_path, name, dtype, monkeypatch):
    from quanta_b200.engine.model import load_model
    from quanta_b200.engine.step import Engine, StepEntry
    from quanta_b200.parts.dense import GatedDense
    model, cfg = load_model(_folder(tmp_path, name), dtype=dtype, dense_weights="fp8")
    parts = [p for p in model.parts() if isinstance(p, GatedDense)]
    n, first = MODELS[name]
    assert len(parts) == n and all(p.reads_fp8 for p in parts)
    eng = Engine(model, num_pages=64, page_size=16, max_requests=4, use_graphs=False)
    reqs = {f"r{i}": H.random_tokens(k, eng.vocab_size, 20 + i) for i, k in enumerate((1, 33, 70))}
    seen = _watch(monkeypatch)
    for step in H.cut_mixed(reqs, max_live=3, seed=5):
        seen.clear()
        logits = eng.step([StepEntry(e["id"], e["tokens"], tuple(e["want"])) for e in step["entries"]], end=step["end"])
        eng.check()
        assert logits is None or torch.all(torch.isfinite(logits))
        assert [c[0] for c in seen][1::4] == ["linear_fp8"] * n and [c[0] for c in seen][2::4] == ["glu_act_fp8"] * n
        assert [c[0] for c in seen][3::4] == ["linear_fp8"] * n and all(c[0] in WRITERS for c in seen[::4]) and first in (None, seen[0][0])
        for i in range(n):
            _check_feed_forward(seen[4 * i: 4 * i + 4], dtype)
            # these are the part's own weights
            assert any(seen[4 * i + 1][1][2] is p.w_gate_up.q and seen[4 * i + 3][1][2] is p.w_down.q for p in parts)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_captured_steps_of_a_model_are_the_eager_ones(tmp_path, dtype, monkeypatch):
    """Single tokens one by one, from captured steps and kernel by kernel.  A captured step sizes its launches for the longest context of its bucket; the
    eager steps are told that length too, so that both launch the same."""
    from quanta_b200.engine.model import load_model
    from quanta_b200.engine.step import Engine
    plain = Engine._context

    def context(self, dev, sizes, R, T, max_pages, info, max_len_after, *a, **k):
        return plain(self, dev, sizes, R, T, max_pages, info, self._bucket(max_len_after) if T == R else max_len_after, *a, **k)

    monkeypatch.setattr(Engine, "_context", context)
    folder, _, _ = _guravik(tmp_path)
    reqs = {f"r{i}": H.random_tokens(n, 97, 20 + i) for i, n in enumerate((37, 90))}
    got = {}
    for graphs in (False, True):
        model, _ = load_model(folder, dtype=dtype, dense_weights="fp8")
        eng = Engine(model, num_pages=64, page_size=16, max_requests=4, use_graphs=graphs)
        got[graphs] = H.replay(eng, H.cut_tail_decode(reqs, tail=30))
        assert (eng.graph_replays >= 50) == graphs
    assert got[True].keys() == got[False].keys() and all(torch.equal(got[True][k], got[False][k]) for k in got[True])


def _captured(run, outs):
    """``run``'s outputs from a captured graph, replayed over outputs that were wiped."""
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = outs(run())
    for _ in range(2):
        for t in held:
            t.fill_(float("nan"))
        graph.replay()
    torch.cuda.synchronize()
    return held


class _Ctx:
    def __init__(self, dtype, settled):
        from quanta_b200 import kernels
        self.dtype, self.settled, self.status = dtype, settled, kernels.new_status(DEV)


class _Doubles:
    """A mixer that shares nothing with the feed-forward but its input."""

    def forward(self, x, ctx, cache, state):
        return 2.0 * x.float()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 5, 24, 150])
def test_beside_a_mixer(T, dtype, monkeypatch):
    """The parallel block: the feed-forward on a second stream; rows of the activation dtype brought to 8 bits."""
    from quanta_b200.parts.block import ParallelBlock
    from tests.test_fp8_model_gpu import _dense, _norm
    g = torch.Generator(device=DEV).manual_seed(T)
    hidden, inner = 1024, 2064
    block = ParallelBlock.__new__(ParallelBlock)
    block.hidden, block.mixer, block.token_input = hidden, _Doubles(), None
    block.norm = _norm(hidden, 1 + 0.2 * torch.randn(hidden, device=DEV, generator=g))
    block.feed_forward = _dense(hidden, inner, "gelu_tanh", False, dtype, T)
    h = torch.randn(T, hidden, device=DEV, generator=g)
    seen = _watch(monkeypatch)
    total = block.forward(h, None, _Ctx(dtype, False), None, None)
    torch.cuda.synchronize()
    assert [c[0] for c in seen] == ["rows_to_fp8", "linear_fp8", "glu_act_fp8", "linear_fp8"]
    _check_feed_forward(seen, dtype)
    assert seen[0][1][0].dtype == dtype and total.extra.data_ptr() == seen[3][1][4].data_ptr()
    assert torch.equal(total.y, 2.0 * seen[0][1][0].float())
    ctx = _Ctx(dtype, True)
    held = _captured(lambda: block.forward(h, None, ctx, None, None), lambda t: (t.y, t.extra))
    assert int(ctx.status[0]) == 0 and torch.equal(held[0], total.y) and torch.equal(held[1], total.extra)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("kind", ["input_weighted_experts", "softmax_shared_experts"])
def test_the_expert_that_every_token_passes(kind, T, dtype, monkeypatch):
    """Beside the routed experts, which it leaves as they are."""
    from quanta_b200 import matmul
    from quanta_b200.parts.base import make
    matmul.configure()
    W, E, ff, shared = 128, 6, 32, 272
    g = torch.Generator(device=DEV).manual_seed(T)
    names = {"gate": "router", "bias": "bias", "w1": "e{e}.gate", "w3": "e{e}.up", "w2": "e{e}.down", "shared_gate": "s.gate", "shared_up": "s.up", "shared_down": "s.down"}
    more = dict(limit=0.9, alpha=1.702, shared_limit=1.1) if kind == "input_weighted_experts" else {}
    part = make("feed_forward", (kind, dict(hidden_size=W, expert_size=ff, n_experts=E, top_k=2, shared_size=shared, names=names, **more)))
    for p in (part, part.shared):
        specs = {s.name: s for s in p.tensor_specs()}
        p.load(lambda n: (torch.randn(specs[n].shape, device=DEV, generator=g) * 1.5 / (specs[n].shape[-1] ** 0.5)).to(torch.float32 if specs[n].kind == "f32" else dtype))
    x = torch.randn(T, W, device=DEV, generator=g).to(dtype)
    before = part.forward(x, _Ctx(dtype, False))
    part.shared.hold_in_fp8()
    seen = _watch(monkeypatch)
    after = part.forward(x, _Ctx(dtype, False))
    torch.cuda.synchronize()
    assert [c[0] for c in seen] == ["rows_to_fp8", "linear_fp8", "glu_act_fp8", "linear_fp8"]
    _check_feed_forward(seen, dtype)
    assert seen[0][1][0] is x and after.extra.data_ptr() == seen[3][1][4].data_ptr() and torch.equal(after.y, before.y)
    ctx = _Ctx(dtype, True)
    held = _captured(lambda: part.forward(x, ctx), lambda t: (t.y, t.extra))
    assert int(ctx.status[0]) == 0 and torch.equal(held[0], after.y) and torch.equal(held[1], after.extra)

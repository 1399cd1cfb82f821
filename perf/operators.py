"""Operators of the 8-bit feed-forward and of scoring, case by case, for measurements: inputs, one pass, what a pass cannot do without,
and what it should return (in 64 bits).

Four operators that are used together when a model's dense feed-forwards are held in 8 bits and its answers are scored:

* ``norm``: the residual stream takes a sublayer's output (as it is, as several slots, or normed first with a gain) and the RMS norm of
  the sum comes out in e4m3 with a float32 scale per row and 128 columns;
* ``glu``: the gated activation of a feed-forward, out in the same form;
* ``linear``: the product of two e4m3 matrices, the rows scaled per 128 columns, the weights per 128 x 128 block;
* ``scores``: from rows of logits, the log probability of a given token, the entropy and the most probable tokens.

The scales of rows are stored ``[blocks of 128 columns, rows]``.  A block that holds nothing but zeros has the scale 2^-100 / 448.
"""

from __future__ import annotations

import math
import random

import torch

own = False             # True: run() calls the framework's operators; False: their plain form

DEVICE = "cuda:0"
BLOCK = 128
E4M3 = torch.float8_e4m3fn
TOP = 448.0             # the largest e4m3
TINY = 2.0 ** -100      # a block's largest value counts as at least this
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
SIZE = {"bfloat16": 2, "float32": 4}
EPS = 1e-5
LIMIT, ALPHA = 7.0, 1.702       # of the clamped activation


# ---- the cases -----------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one user at a terminal: the norm between two sublayers of a decode step, width of the 2,048-wide decoders, output normed first
        dict(name="norm_token", op="norm", rows=1, width=2048, slots=1, delta="float32", gain=True),
        # a busy server's decode step at a width that ends inside a block of 128
        dict(name="norm_batch_odd", op="norm", rows=77, width=5000, slots=1, delta="bfloat16", gain=False),
        # prompts: the largest step, two partial results a token (routed and shared experts)
        dict(name="norm_prompt", op="norm", rows=8192, width=4096, slots=2, delta="float32", gain=False),
        # one token's activation, 5,632 wide
        dict(name="glu_token", op="glu", rows=1, width=5632, kind="silu", dtype="bfloat16", bias=False),
        # prompts: the clamped activation with biases, 11,008 wide
        dict(name="glu_prompt", op="glu", rows=8192, width=11008, kind="clamped", dtype="bfloat16", bias=True),
        # one token's gate and up product of a 4,096-wide decoder: bound by the weights' bytes
        dict(name="linear_token", op="linear", rows=1, inner=4096, outer=22016, dtype="bfloat16"),
        # a batch's down product, its sums kept in 32 bits for the residual stream
        dict(name="linear_batch_32", op="linear", rows=32, inner=11008, outer=4096, dtype="float32"),
        # a portion of a prompt of no round length, a matrix that ends inside a block both ways
        dict(name="linear_portion_odd", op="linear", rows=317, inner=5648, outer=2000, dtype="float32"),
        # prompts: the gate and up product of the largest step, bound by the tensor cores
        dict(name="linear_prompt", op="linear", rows=8192, inner=4096, outer=22016, dtype="bfloat16"),
        # the log probability of one chosen token over a vocabulary of 200,064, with its 20 best rivals
        dict(name="scores_token", op="scores", rows=1, vocab=200064, dtype="float32", top=20),
        # a decode step of a busy server, the vocabulary of the 2,048-wide decoders, the logits in bfloat16 (ties are common)
        dict(name="scores_batch", op="scores", rows=64, vocab=32000, dtype="bfloat16", top=5),
        # a document scored token by token
        dict(name="scores_prompt", op="scores", rows=2048, vocab=200064, dtype="float32", top=20),
    ]


def draw(rng: random.Random) -> dict:
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "glu", "linear", "linear", "scores"])
    if op == "norm":
        width, slots = spread(64, 8192), rng.choice([1, 1, 2, 8])
        rows = spread(1, min(8192, 8192 * 4096 * 2 // (width * slots)))
        return dict(op=op, rows=rows, width=width, slots=slots, delta=rng.choice(["float32", "bfloat16"]), gain=rng.random() < 0.5)
    if op == "glu":
        width = spread(64, 12288)
        return dict(op=op, rows=spread(1, min(8192, 8192 * 11008 // width)), width=width, kind=rng.choice(["silu", "gelu_tanh", "clamped"]),
                    dtype=rng.choice(["bfloat16", "float32"]), bias=rng.random() < 0.5)
    if op == "linear":
        rows, inner, outer = spread(1, 8192), 16 * spread(4, 768), spread(32, 22016)
        while rows * inner * outer > 8192 * 4096 * 22016:
            outer //= 2
        return dict(op=op, rows=rows, inner=inner, outer=outer, dtype=rng.choice(["bfloat16", "float32"]))
    vocab = spread(300, 200064)
    return dict(op=op, rows=spread(1, min(4096, 2048 * 200064 // vocab)), vocab=vocab, dtype=rng.choice(["float32", "bfloat16"]),
                top=rng.choice([0, 1, 5, 20]))


# ---- inputs --------------------------------------------------------------------------------------------
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEVICE)


def _blocks(x: torch.Tensor) -> torch.Tensor:
    """``[rows, columns]`` -> ``[rows, blocks, 128]``, zeros behind the last column."""
    pad = -x.shape[1] % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).view(x.shape[0], -1, BLOCK)


def _rows_to_8_bits(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows in e4m3 and their scales ``[blocks, rows]``."""
    b = _blocks(x)
    scale = b.abs().amax(2).clamp_min(TINY) / TOP
    q = (b / scale[:, :, None]).clamp(-TOP, TOP).view(x.shape[0], -1)[:, :x.shape[1]]
    return q.to(E4M3).contiguous(), scale.t().contiguous()


def _weight_to_8_bits(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = w.shape
    p = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    b = p.view(p.shape[0] // BLOCK, BLOCK, p.shape[1] // BLOCK, BLOCK)
    scale = b.abs().amax((1, 3)).clamp_min(TINY) / TOP
    q = (b / scale[:, None, :, None]).clamp(-TOP, TOP).reshape(p.shape)[:n, :k]
    return q.to(E4M3).contiguous(), scale.contiguous()


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    s, n = dict(case), case["rows"]
    if case["op"] == "norm":
        width, slots = case["width"], case["slots"]
        # the residual stream: a few coordinates far larger than the others, as in trained decoders
        s["h"] = _normal(g, n, width)
        s["h"][:, torch.randperm(width, generator=g, device=DEVICE)[: 1 + width // 500]] *= 30.0
        s["delta"] = (0.3 * _normal(g, n, *((slots,) if slots > 1 else ()), width)).to(DTYPES[case["delta"]])
        s["weight"] = 1.0 + 0.1 * _normal(g, width)
        s["delta_gain"] = 0.5 + 0.1 * _normal(g, width) if case["gain"] else None
    elif case["op"] == "glu":
        s["gate_up"] = (2.0 * _normal(g, n, 2 * case["width"])).to(DTYPES[case["dtype"]])
        s["bias"] = 0.2 * _normal(g, 2 * case["width"]) if case["bias"] else None
    elif case["op"] == "linear":
        s["x"], s["x_scales"] = _rows_to_8_bits(_normal(g, n, case["inner"]) * torch.exp(_normal(g, n, 1)))
        s["w"], s["w_scales"] = _weight_to_8_bits(0.02 * _normal(g, case["outer"], case["inner"]))
    else:
        vocab = case["vocab"]
        # logits of a model: most rows undecided, some sure of a token; a third of the rows may only choose among some of the tokens
        x = 2.5 * _normal(g, n, vocab)
        sure = torch.rand(n, generator=g, device=DEVICE) < 0.4
        best = torch.randint(0, vocab, (n,), generator=g, device=DEVICE)
        x[torch.arange(n, device=DEVICE), best] += 12.0 * sure
        bound = torch.rand(n, generator=g, device=DEVICE) < 0.33
        kept = torch.rand(vocab, generator=g, device=DEVICE) < 0.1
        x.masked_fill_(bound[:, None] & ~kept[None, :], -math.inf)
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["tokens"] = torch.where(torch.rand(n, generator=g, device=DEVICE) < 0.7, best,
                                  torch.randint(0, vocab, (n,), generator=g, device=DEVICE)).to(torch.int32)
        s["status"] = torch.zeros(4, dtype=torch.int32, device=DEVICE)
    return s


# ---- one pass ------------------------------------------------------------------------------------------
def run(s: dict) -> dict:
    return {"norm": _norm, "glu": _glu, "linear": _linear, "scores": _scores}[s["op"]](s)


def _norm(s: dict) -> dict:
    h, n, width = s["h"], s["rows"], s["width"]
    if own:
        from quanta_b200 import kernels
        q = torch.empty((n, width), dtype=E4M3, device=h.device)
        scales = torch.empty((-(-width // BLOCK), n), dtype=torch.float32, device=h.device)
        kernels.add_rmsnorm_fp8(h, s["delta"], s["weight"], EPS, q, scales, delta_gain=s["delta_gain"], delta_eps=EPS)
        return {"h": h, "q": q, "scales": scales}
    d = s["delta"].float()
    if d.dim() == 3:
        d = d.sum(1)
    if s["delta_gain"] is not None:
        d = s["delta_gain"] * (d * torch.rsqrt(d.square().mean(1, keepdim=True) + EPS))
    h += d
    q, scales = _rows_to_8_bits(s["weight"] * (h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)))
    return {"h": h, "q": q, "scales": scales}


def _glu(s: dict) -> dict:
    n, width, gate_up = s["rows"], s["width"], s["gate_up"]
    if own:
        from quanta_b200 import kernels
        kind = {"silu": kernels.GLU_SILU, "gelu_tanh": kernels.GLU_GELU_TANH, "clamped": kernels.GLU_CLAMPED}[s["kind"]]
        q = torch.empty((n, width), dtype=E4M3, device=gate_up.device)
        scales = torch.empty((-(-width // BLOCK), n), dtype=torch.float32, device=gate_up.device)
        kernels.glu_act_fp8(gate_up, q, scales, bias=s["bias"], kind=kind, limit=LIMIT, alpha=ALPHA)
        return {"q": q, "scales": scales}
    x = gate_up.float() if s["bias"] is None else gate_up.float() + s["bias"]
    gate, up = x[:, :width], x[:, width:]
    if s["kind"] == "silu":
        a = gate / (1.0 + torch.exp(-gate)) * up
    elif s["kind"] == "clamped":
        c = gate.clamp(max=LIMIT)
        a = c / (1.0 + torch.exp(-ALPHA * c)) * (up.clamp(-LIMIT, LIMIT) + 1.0)
    else:
        a = gate / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
    q, scales = _rows_to_8_bits(a)
    return {"q": q, "scales": scales}


def _linear(s: dict) -> torch.Tensor:
    x, w, inner = s["x"], s["w"], s["inner"]
    if own:
        from quanta_b200 import kernels
        out = torch.empty((s["rows"], s["outer"]), dtype=DTYPES[s["dtype"]], device=x.device)
        kernels.linear_fp8(x, s["x_scales"], w, s["w_scales"], out)
        return out
    xf = x.float() * s["x_scales"].t().repeat_interleave(BLOCK, 1)[:, :inner]
    wf = w.float() * s["w_scales"].repeat_interleave(BLOCK, 0)[: s["outer"]].repeat_interleave(BLOCK, 1)[:, :inner]
    return (xf @ wf.t()).to(DTYPES[s["dtype"]])


def _scores(s: dict) -> dict:
    logits, tokens, top = s["logits"], s["tokens"], s["top"]
    n, vocab = logits.shape
    if own:
        from quanta_b200 import kernels
        logprob, entropy = (torch.empty(n, dtype=torch.float32, device=logits.device) for _ in range(2))
        ids = torch.empty((n, top), dtype=torch.int32, device=logits.device)
        best = torch.empty((n, top), dtype=torch.float32, device=logits.device)
        kernels.token_logprobs(logits, tokens, logprob, entropy, ids, best, s["status"])
        return {"logprob": logprob, "entropy": entropy, "ids": ids, "best": best}
    x = logits.float()
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    entropy = -torch.where(lp == -math.inf, 0.0, torch.exp(lp) * lp).sum(1)
    logprob = lp.gather(1, tokens.long()[:, None])[:, 0]
    # whole numbers that are ordered as the logits are, equal ones by their place, the first first
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) + (vocab - 1 - torch.arange(vocab, device=x.device))
    ids = (vocab - 1 - key.topk(min(top, vocab), 1).values % (1 << 20)).to(torch.int32)
    return {"logprob": logprob, "entropy": entropy, "ids": ids, "best": lp.gather(1, ids.long())}


# ---- what a pass cannot do without ---------------------------------------------------------------------
def work(case: dict) -> dict:
    n = case["rows"]
    if case["op"] == "norm":
        width, slots = case["width"], case["slots"]
        gains = 2 if case["gain"] else 1
        return {"bytes": n * width * (4 + 4 + slots * SIZE[case["delta"]] + 1) + 4 * gains * width + 4 * n * -(-width // BLOCK),
                "flops": n * width * (slots + 6 + (4 if case["gain"] else 0))}
    if case["op"] == "glu":
        width = case["width"]
        return {"bytes": n * width * (2 * SIZE[case["dtype"]] + 1) + 4 * n * -(-width // BLOCK) + (8 * width if case["bias"] else 0),
                "flops": 12 * n * width}
    if case["op"] == "linear":
        k, m = case["inner"], case["outer"]
        blocks = -(-k // BLOCK)
        return {"bytes": n * k + m * k + 4 * n * blocks + 4 * blocks * -(-m // BLOCK) + n * m * SIZE[case["dtype"]], "flops": 2 * n * k * m}
    return {"bytes": n * case["vocab"] * SIZE[case["dtype"]] + 4 * n * (3 + 2 * case["top"]), "flops": 6 * n * case["vocab"]}


# ---- what it should return, in 64 bits -------------------------------------------------------------------
def _exact_rows(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The numbers that are to be rounded to e4m3, and the scales."""
    n, width = v.shape
    blocks = -(-width // BLOCK)
    wide = torch.zeros((n, blocks * BLOCK), dtype=torch.float64, device=v.device)
    wide[:, :width] = v
    largest = wide.reshape(n, blocks, BLOCK).abs().max(dim=2).values
    scale = torch.maximum(largest, torch.full_like(largest, TINY)) / TOP
    return (wide.reshape(n, blocks, BLOCK) / scale.unsqueeze(2)).reshape(n, -1)[:, :width], scale.T.contiguous()


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    n = case["rows"]
    if case["op"] == "norm":
        def normed(v):
            return v / ((v * v).sum(dim=1) / case["width"] + EPS).sqrt().unsqueeze(1)

        d = s["delta"].double().reshape(n, case["slots"], case["width"]).sum(dim=1)
        h = s["h"].double() + (normed(d) * s["delta_gain"].double() if case["gain"] else d)
        q, scales = _exact_rows(normed(h) * s["weight"].double())
        return {"h": h, "q": q, "scales": scales}
    if case["op"] == "glu":
        both = s["gate_up"].double()
        if case["bias"]:
            both = both + s["bias"].double()
        gate, up = both.split(case["width"], dim=1)
        if case["kind"] == "silu":
            v = gate * torch.sigmoid(gate) * up
        elif case["kind"] == "clamped":
            gate, up = torch.clamp_max(gate, LIMIT), torch.clamp(up, -LIMIT, LIMIT)
            v = gate * torch.sigmoid(ALPHA * gate) * (up + 1)
        else:
            v = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate))) * up
        q, scales = _exact_rows(v)
        return {"q": q, "scales": scales}
    if case["op"] == "linear":
        out = torch.zeros((n, case["outer"]), dtype=torch.float64, device=DEVICE)
        of_row = torch.arange(case["outer"], device=DEVICE) // BLOCK
        for b in range(-(-case["inner"] // BLOCK)):
            at = slice(b * BLOCK, min((b + 1) * BLOCK, case["inner"]))
            part = s["x"][:, at].double() @ s["w"][:, at].double().T
            out += part * s["x_scales"][b].double().unsqueeze(1) * s["w_scales"][:, b].double()[of_row].unsqueeze(0)
        return out
    parts = []
    for rows in range(0, n, 256):
        x, t = s["logits"][rows: rows + 256].double(), s["tokens"][rows: rows + 256].long()
        lp = torch.log_softmax(x, dim=1)
        p = lp.exp()
        order = torch.sort(lp, dim=1, descending=True, stable=True)
        k = min(case["top"], case["vocab"])
        parts.append((lp[torch.arange(len(t), device=x.device), t], torch.special.entr(p).sum(dim=1), order.indices[:, :k].to(torch.int32),
                      order.values[:, :k]))
    logprob, entropy, ids, best = (torch.cat(v) for v in zip(*parts))
    return {"logprob": logprob, "entropy": entropy, "ids": ids, "best": best}

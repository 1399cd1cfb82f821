"""What the kernels with e4m3 and the scores of tokens refuse before anything is launched (shapes, types, places), on tensors of the CPU."""
from __future__ import annotations

import pytest
import torch

from quanta_b200 import kernels

E4M3 = torch.float8_e4m3fn


def _rows(n, cols):
    return torch.zeros(n, cols).to(E4M3), torch.zeros(-(-cols // 128), n)


def test_norm():
    h, w = torch.zeros(3, 200), torch.ones(200)
    q, s = _rows(3, 200)
    rows = torch.zeros(3, dtype=torch.int32)
    for bad in (dict(h=h.bfloat16()), dict(h=h[0]), dict(weight=w[:100]), dict(weight=w.bfloat16()), dict(delta=torch.zeros(3, 100)),
                dict(delta=torch.zeros(2, 200)), dict(delta=torch.zeros(3, 0, 200)), dict(delta=torch.zeros(200)), dict(out=q[:2]), dict(out=q.float()),
                dict(scales=s.T.contiguous()), dict(scales=s.double()), dict(delta_gain=w), dict(delta=torch.zeros(3, 200), delta_gain=w[:5]),
                dict(rows=rows, delta=torch.zeros(3, 200)), dict(rows=rows.long(), store_h=False), dict(rows=rows[:2], store_h=False), dict()):
        a = dict(h=h, delta=None, weight=w, eps=1e-5, out=q, scales=s) | bad
        with pytest.raises(ValueError):
            kernels.add_rmsnorm_fp8(**a)


def test_activation_and_rows():
    x = torch.zeros(3, 400)
    q, s = _rows(3, 200)
    for bad in (dict(gate_up=x[:, :399]), dict(gate_up=x[0]), dict(bias=torch.zeros(200)), dict(bias=torch.zeros(400).bfloat16()), dict(kind=3), dict(kind=-1),
                dict(kind=kernels.GLU_CLAMPED), dict(out=q[:, :100]), dict(scales=s[:1]), dict(gate_up=x.half()), dict()):
        with pytest.raises(ValueError):
            kernels.glu_act_fp8(**(dict(gate_up=x, out=q, scales=s) | bad))
    for x in (torch.zeros(3), torch.zeros(3, 201), torch.zeros(3, 200)):
        with pytest.raises(ValueError):
            kernels.rows_to_fp8(x, q, s)


def test_product():
    x, xs = _rows(5, 256)
    w, ws, out = torch.zeros(300, 256).to(E4M3), torch.zeros(3, 2), torch.zeros(5, 300)
    for bad in (dict(x=x.view(torch.int8)), dict(x=x[:4]), dict(x=x[0]), dict(x_scales=xs[:1]), dict(x_scales=xs.T.contiguous()), dict(w=w[:, :128]),
                dict(w=w.to(torch.float8_e5m2)), dict(w_scales=ws[:2]), dict(w_scales=ws.bfloat16()), dict(out=out[:, :299]), dict(out=out.T.contiguous()),
                dict(status=torch.zeros(4)), dict(out=out.half()), dict()):
        with pytest.raises(ValueError):
            kernels.linear_fp8(**(dict(x=x, x_scales=xs, w=w, w_scales=ws, out=out) | bad))
    x, xs = _rows(5, 24)
    with pytest.raises(ValueError, match="multiple of 16"):
        kernels.linear_fp8(x, xs, torch.zeros(300, 24).to(E4M3), torch.zeros(3, 1), out)
    with pytest.raises(ValueError, match="multiple of 16"):
        kernels.linear_fp8(torch.zeros(5, 0).to(E4M3), torch.zeros(0, 5), torch.zeros(300, 0).to(E4M3), torch.zeros(3, 0), out)


def test_scores():
    x, t, f = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    ids, best = torch.zeros(4, 5, dtype=torch.int32), torch.zeros(4, 5)
    ok = dict(logits=x, tokens=t, logprob=f, entropy=f.clone(), ids=ids, best=best)
    for bad in (dict(logits=x[0]), dict(logits=x.half()), dict(logits=x.T), dict(logits=x[:, ::2]), dict(logits=x[:, :0]), dict(logits=x[:1].expand(4, 100)),
                dict(tokens=None), dict(logprob=None), dict(tokens=t.long()), dict(tokens=t[:3]), dict(entropy=f.double()), dict(entropy=f[:2]), dict(ids=None),
                dict(best=None), dict(ids=ids.long()), dict(best=best[:, :4]), dict(ids=ids[:3], best=best[:3]), dict(ids=ids[0], best=best[0]),
                dict(ids=torch.zeros(4, 65, dtype=torch.int32), best=torch.zeros(4, 65)), dict(status=torch.zeros(4)), dict()):
        with pytest.raises(ValueError):
            kernels.token_logprobs(**(ok | bad))
    with pytest.raises(ValueError, match="at most"):
        kernels.token_logprobs(torch.zeros(4, 3), None, None, None, ids[:, :4].contiguous(), best[:, :4].contiguous())


def test_sizes_that_32_bits_do_not_count():
    many = 2 ** 30 + 16
    meta = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="at most"):
        kernels.rows_to_fp8(meta(many, 16), meta(many, 16, dtype=E4M3), meta(1, many))
    with pytest.raises(ValueError, match="at most"):
        kernels.glu_act_fp8(meta(1, 2 * many), meta(1, many, dtype=E4M3), meta(many // 128 + 1, 1))
    with pytest.raises(ValueError, match="at most"):
        kernels.add_rmsnorm_fp8(meta(many, 16), None, meta(16), 1e-5, meta(many, 16, dtype=E4M3), meta(1, many))
    with pytest.raises(ValueError, match="at most"):
        kernels.add_rmsnorm_fp8(meta(2, 16), meta(2, many, 16), meta(16), 1e-5, meta(2, 16, dtype=E4M3), meta(1, 2))
    with pytest.raises(ValueError, match="at most"):
        kernels.linear_fp8(meta(1, 16, dtype=E4M3), meta(1, 1), meta(many, 16, dtype=E4M3), meta(many // 128 + 1, 1), meta(1, many))
    with pytest.raises(ValueError, match="at most"):
        kernels.linear_fp8(meta(many, 16, dtype=E4M3), meta(1, many), meta(16, 16, dtype=E4M3), meta(1, 1), meta(many, 16))
    for n, V in ((many, 1), (1, 2 ** 32 + 5)):
        with pytest.raises(ValueError, match="at most"):
            kernels.token_logprobs(meta(n, V), None, None, meta(n))

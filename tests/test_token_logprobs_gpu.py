"""Log probabilities, entropies and the most probable tokens against float64.

Tolerances (u = 2^-24).  With d = x - max, a weight e^d is off by 2^-21 + 4 u |d| of itself (the exponential's argument is rounded once as a
difference and once as a product, the exponential is good to 2 ulp), the sum s of the weights by the weighted mean of that and by one rounding an
addition: a thread adds at most V / 512 + 64 numbers one after the other, and some twenty joins follow, each good to a few u.  log s is off by the
relative error of s; the entropy, log s - sum e^d d / s, by that times one more than the mean of |d|, and by the error of the weights under the sum."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _scores(logits, tokens, top, status=None):
    from quanta_b200 import kernels
    n = logits.shape[0]
    lp, en = torch.full((n,), 5.0, device=DEV), torch.full((n,), 5.0, device=DEV)
    ids, best = torch.full((n, top), -7, dtype=torch.int32, device=DEV), torch.full((n, top), 5.0, device=DEV)
    kernels.token_logprobs(logits, tokens, lp, en, ids, best, status)
    return lp, en, ids, best


def _order(x, top):
    """The first ``top`` by value, equal ones by place, NaN as -inf, -0 as 0."""
    x = torch.where(torch.isnan(x), -torch.inf, x) + 0.0
    return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top].to(torch.int32)


def _check(logits, tokens, top):
    lp, en, ids, best = _scores(logits, tokens, top)
    x = logits.double()
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    p = torch.softmax(x, 1)
    d = torch.where(torch.isinf(x - m), 0.0, (x - m).abs())
    a, b = (p * d).sum(1), (p * d * d).sum(1)
    lse = torch.logsumexp(x, 1)
    tol = 2.0 ** -21 + 4 * U * a + (V / 512 + 100) * U
    want = x.gather(1, tokens.long()[:, None])[:, 0] - lse
    size = m[:, 0].abs() + (lse - m[:, 0]).abs()
    assert torch.equal(torch.isinf(lp), torch.isinf(want))
    fine = torch.isfinite(want)
    assert torch.all((lp.double() - want).abs()[fine] <= (tol + 4 * U * (size + want.abs()))[fine])
    ent = torch.special.entr(p).sum(1)
    assert torch.all((en.double() - ent).abs() <= tol * (1 + 2 * a) + 2.0 ** -20 * a + 8 * U * b + 4 * U * (size + ent))
    order = _order(x, top)
    assert torch.equal(ids, order)
    want = x.gather(1, order.long()) - lse[:, None]
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(best))
    assert torch.all(((best.double() - want).abs() <= (tol + 4 * U * size)[:, None] + 4 * U * want.abs())[fine])


CASES = [(1, 1, 1), (1, 2, 2), (2, 5, 5), (3, 64, 64), (1, 511, 20), (4, 3000, 20), (1, 32000, 5), (64, 32000, 20), (1, 200064, 20), (2, 200063, 64), (150, 20001, 20),
         (300, 777, 1), (5, 8191, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,top", CASES)
def test_scores(n, V, top, dtype):
    g = _gen(n + V)
    x = (3 * torch.randn(n, V, device=DEV, generator=g)).to(dtype)
    t = torch.randint(0, V, (n,), device=DEV, generator=g).to(torch.int32)
    x[0, int(t[0])] = 20.0
    _check(x, t, top)
    assert all(torch.equal(a, b) for a, b in zip(_scores(x, t, top), _scores(x, t, top)))


@pytest.mark.parametrize("n,V,dtype", [(1, 4300037, torch.float32), (1, 9000001, torch.bfloat16), (1190, 262150, torch.float32), (1190, 530001, torch.bfloat16), (700, 4097, torch.float32),
                                       (90, 33333, torch.bfloat16)])
def test_long_rows_and_many(n, V, dtype):
    """Rows longer than a block keeps a maximum of every 512 bytes for, and numbers of rows that are cut in three, five and more parts."""
    g = _gen(V)
    x = torch.randn(n, V, device=DEV, generator=g, dtype=dtype)
    t = torch.randint(0, V, (n,), device=DEV, generator=g).to(torch.int32)
    lp, en, ids, best = _scores(x, t, 20)
    for r in sorted({0, n // 2, n - 1}):
        _check(x[r: r + 1], t[r: r + 1].contiguous(), 20)
        lse = torch.logsumexp(x[r].double(), 0)
        order = _order(x[r: r + 1].double(), 20)[0]
        assert torch.equal(ids[r], order)
        assert torch.all((best[r].double() - (x[r].double()[order.long()] - lse)).abs() < 1e-4) and abs(float(lp[r]) - float(x[r, int(t[r])].double() - lse)) < 1e-4
    assert bool(torch.isfinite(lp).all()) and bool(torch.isfinite(en).all()) and bool((best[:, :-1] >= best[:, 1:]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_ties_masks_and_uneven_rows(n, dtype):
    """Rows of equal numbers, of few values, with few tokens left, and with the largest numbers where few threads read."""
    V = 20000
    g = _gen(n)
    x = torch.randn(n, V, device=DEV, generator=g)
    x[0] = 1.5
    if n > 1:
        x[1] = torch.randint(-2, 3, (V,), device=DEV, generator=g).float()
        x[2, 100:] = -torch.inf
        x[3] = -torch.inf
        x[3, 17777] = -2.0
        x[4] = torch.arange(V, device=DEV).flip(0) / 1000
        x[5] = torch.arange(V, device=DEV) / 1000
        x[6] = -torch.inf
        x[6, [3, 9999, 19999]] = torch.tensor([1.0, 1.0, 1.0], device=DEV)
        x[7], x[7, 5], x[7, 3] = -0.0, 0.0, 0.0
        x[8] = 30000.0
        x[9] = -30000.0
    if n > 100:
        # the pieces of 16 bytes that four neighbouring threads of 512 read
        per = 4 if dtype == torch.float32 else 8
        x[10].view(-1, 4)[torch.arange(V // 4, device=DEV) // (per // 4) % 512 < 4] += 50.0
    x = x.to(dtype)
    t = torch.randint(0, V, (n,), device=DEV, generator=g).to(torch.int32)
    if n > 1:
        t[3], t[2] = 17777, 150      # certain; masked
    _check(x, t, 20)
    _check(x, t, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_a_distribution(dtype):
    V = 9001
    g = _gen(3)
    for n in (8, 400):
        x = torch.randn(n, V, device=DEV, generator=g).to(dtype)
        x[1, 77], x[2], x[3, 5], x[4, 9000] = torch.nan, -torch.inf, torch.inf, torch.nan
        x[5], x[6, 3:] = torch.nan, -torch.inf
        x[6, 8000] = torch.nan
        t = torch.full((n,), 1, dtype=torch.int32, device=DEV)
        lp, en, ids, best = _scores(x, t, 20)
        bad = torch.zeros(n, dtype=torch.bool, device=DEV)
        bad[1:7] = True
        assert torch.equal(torch.isnan(lp), bad) and torch.equal(torch.isnan(en), bad)
        assert torch.all(torch.isnan(best[bad])) and torch.all(torch.isfinite(best[~bad]))
        assert torch.equal(ids, _order(x.double(), 20))
        _check(x[7:], t[7:], 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_places(dtype):
    g = _gen(4)
    big = torch.randn(7, 12345, device=DEV, generator=g).to(dtype)
    t = torch.randint(0, 9000, (7,), device=DEV, generator=g).to(torch.int32)
    for lo in (0, 1, 3, 8):
        _check(big[:, lo: lo + 9001], t, 10)
    _check(big[::3, 5: 9006], t[::3].contiguous(), 10)


def test_tokens_outside_the_vocabulary_and_parts_left_out():
    from quanta_b200 import kernels
    g = _gen(5)
    x = torch.randn(4, 5000, device=DEV, generator=g)
    status = kernels.new_status(DEV)
    t = torch.tensor([4999, 5000, -1, 0], dtype=torch.int32, device=DEV)
    lp, en, ids, best = _scores(x, t, 3, status)
    assert torch.equal(torch.isnan(lp), torch.tensor([False, True, True, False], device=DEV)) and torch.all(torch.isfinite(en))
    assert int(status[0]) == 1 and int(status[1]) in (5000, -1)
    with pytest.raises(kernels.KernelError, match="vocabulary"):
        kernels.raise_on_status(status.cpu())
    only = torch.empty(4, device=DEV)
    kernels.token_logprobs(x, None, None, only)
    assert torch.equal(only, en)
    i2, b2 = torch.empty_like(ids), torch.empty_like(best)
    kernels.token_logprobs(x, None, None, None, i2, b2)
    assert torch.equal(i2, ids) and torch.equal(b2, best)
    kernels.token_logprobs(x[:0], t[:0], lp[:0], en[:0], ids[:0], best[:0])
    kernels.token_logprobs(x, t, lp, en, torch.empty((4, 0), dtype=torch.int32, device=DEV), torch.empty((4, 0), device=DEV))


def test_in_a_graph_and_on_another_stream():
    g = _gen(6)
    x = torch.randn(2, 50000, device=DEV, generator=g)
    t = torch.tensor([4, 40000], dtype=torch.int32, device=DEV)
    want = _scores(x, t, 20)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = _scores(x, t, 20)
        graph.replay()
        graph.replay()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [8, 200])
def test_rows_of_the_lowest_numbers(n, dtype):
    """Masks of the type's lowest value, alone, beside -inf (which is less probable), and beside numbers some steps above it.

    Of the differences to the largest number only zeros have a weight, so the sum is exact: what is left are the logarithm (an ulp) and the roundings of
    the differences."""
    V, low = 20000, torch.finfo(dtype).min
    g = _gen(n)
    x = torch.randn(n, V, device=DEV, generator=g)
    x[0] = low
    x[1] = low
    x[1, [17, 19990]] = 0.0
    x[2] = -torch.inf
    x[2, 100:1100] = low
    x[3] = low
    x[3, ::2] = -3.35e38
    x[4, :19000] = low
    x[5] = -torch.inf
    x[5, :9000] = low
    x[5, 19000:] = -3.0e38
    x[6] = low
    x[6, 5000] = torch.nan
    x[7], x[7, 5:10] = low, -3.2965e38
    x = x.to(dtype)
    t = torch.full((n,), 4, dtype=torch.int32, device=DEV)
    t[2] = 1099
    lp, en, ids, best = _scores(x, t, 20)
    assert torch.equal(ids, _order(x.double(), 20))
    keep = torch.arange(n, device=DEV) != 6
    assert bool(torch.isnan(lp[6])) and bool(torch.isnan(en[6])) and bool(torch.isnan(best[6]).all())
    d = x[keep].double() - x[keep].double().amax(1, keepdim=True)
    log_s = d.exp().sum(1).log()
    tol = torch.full_like(log_s, 4 * U)
    tol[4] = tol[7:] = 2.0 ** -21 + (V / 512 + 100) * U      # rows with ordinary numbers, as above
    for got, want in ((lp[keep, None], d.gather(1, t[keep, None].long())), (best[keep], d.gather(1, ids[keep].long()))):
        want = want - log_s[:, None]
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        fine = torch.isfinite(want)
        assert torch.all(((got.double() - want).abs() <= tol[:, None] * (8 + log_s[:, None]) + 4 * U * want.abs())[fine])
    ent = torch.special.entr(torch.softmax(d, 1)).sum(1)
    assert torch.all((en[keep].double() - ent).abs() <= tol * 16 * (1 + ent))


def test_more_than_32_bits_of_numbers():
    g = _gen(8)
    n, V = 11000, 200064
    some = torch.randn(50, V, device=DEV, generator=g).bfloat16()
    pick = torch.randint(0, 50, (n,), device=DEV, generator=g)
    t = torch.randint(0, V, (50,), device=DEV, generator=g).to(torch.int32)
    want = _scores(some, t, 7)
    got = _scores(some[pick], t[pick].contiguous(), 7)
    # few rows are cut over several blocks, so the sums differ: by twice 2^-21 + (V / 512 + 100) u = 3e-5, the entropy by that times 1 + 2 a, a < 8
    assert torch.equal(got[2], want[2][pick])
    for k, tol in ((0, 6e-5), (1, 6e-5 * 17), (3, 6e-5)):
        assert torch.all((got[k] - want[k][pick]).abs() <= tol + 8 * U * want[k][pick].abs())
    _check(some, t, 7)

"""The kernels with e4m3 on either side against float64.

Tolerances (u = 2^-24).  A number v of a block whose scale is s comes out as q with |q - v / s| at most half a step of e4m3, 2^-4 of a normal
number and 2^-10 below 2^-6, and what the float32 arithmetic before it was off by.  That arithmetic: a sum of S slots and the stream is off by
at most (S + 1) u times the sum of the addends' sizes A; the sum of H squares by H u of itself, so a root mean square by half of that and by
what its addends were off by; products, quotients and rsqrt (2 ulp) by a few u.  Together at most 2 (H + S + 8) u (A + |x| |A| / |x|), norms over the
row, times the factors behind.  Activations: exp within 2 ulp of its value and u |argument| more, a handful of roundings, and the limit of the
sum 1 + e^-g: 32 u (1 + |g|) of |act|.  The product: a block's 128 products are exact in float32 and their sum is within 2 * 128 u of the sum of
their sizes (the tensor cores may truncate), the scaled blocks add one rounding each and the scales two."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
TINY = 2.0 ** -100


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _empty_rows(n, cols):
    return (torch.full((n, cols), 1.0, device=DEV).to(E4M3), torch.full((-(-cols // 128), n), float("nan"), device=DEV))


def _scales_of(v):
    n, cols = v.shape
    wide = torch.nn.functional.pad(v, (0, -cols % 128)).view(n, -1, 128)
    return (wide.abs().amax(2).clamp_min(TINY) / 448).T


def _spread(scales, cols):
    return scales.T.repeat_interleave(128, 1)[:, :cols]


def _rows_within(q, scales, v, off):
    """q, scales of the numbers v (float64), which the kernel had within ``off``."""
    want = _scales_of(v)
    worst = (torch.nn.functional.pad(off, (0, -v.shape[1] % 128)).view(v.shape[0], -1, 128).amax(2) / 448).T
    assert torch.all((scales.double() - want).abs() <= worst + 4 * U * want)
    s = _spread(scales.double(), v.shape[1])
    u = v / s
    assert torch.all((q.double() - u).abs() <= torch.maximum(2.0 ** -4 * u.abs(), torch.tensor(2.0 ** -10, device=DEV)) * (1 + 8 * U) + 2 * off / s + 8 * U * u.abs())


NORMS = [(1, 16, 1), (1, 2048, 1), (3, 1, 1), (2, 130, 2), (5, 1000, 8), (77, 5000, 1), (9, 8192, 2), (4, 8200, 1), (300, 640, 1), (2, 20000, 1)]


@pytest.mark.parametrize("gain", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,H,S", NORMS)
def test_norm(n, H, S, dtype, gain):
    from quanta_b200 import kernels
    g = _gen(n * H + S)
    h, w = _randn(g, n, H) * 3, 1 + 0.2 * _randn(g, H)
    d = (_randn(g, n, S, H) if S > 1 else _randn(g, n, H)).to(dtype)
    dg = _randn(g, H) if gain else None
    h0 = h.clone()
    q, scales = _empty_rows(n, H)
    kernels.add_rmsnorm_fp8(h, d, w, 1e-5, q, scales, delta_gain=dg, delta_eps=1e-6)

    def rms(v, eps):
        return ((v * v).mean(1, keepdim=True) + eps).rsqrt()

    slots = d.double().view(n, S, H)
    z, A = slots.sum(1), slots.abs().sum(1)
    c = 2 * (H + S + 8) * U
    if gain:
        r = rms(z, 1e-6)
        z, A = dg.double() * z * r, dg.double().abs() * r * (A + z.abs() * A.norm(dim=1, keepdim=True) / z.norm(dim=1, keepdim=True))
    x = h0.double() + z
    A = A + h0.double().abs()
    assert torch.all((h.double() - x).abs() <= c * A)
    r = rms(x, 1e-5)
    off = c * w.double().abs() * r * (A + x.abs() * A.norm(dim=1, keepdim=True) / x.norm(dim=1, keepdim=True))
    _rows_within(q, scales, w.double() * x * r, off)


def test_norm_of_selected_rows_and_without_a_delta():
    from quanta_b200 import kernels
    g = _gen(1)
    for H in (256, 300):
        h, w = _randn(g, 6, H), 1 + 0.1 * _randn(g, H)
        d = _randn(g, 6, H)
        rows = torch.tensor([5, 0, 0, 3], dtype=torch.int32, device=DEV)
        full, full_s = _empty_rows(6, H)
        h2 = h.clone()
        kernels.add_rmsnorm_fp8(h2, d, w, 1e-5, full, full_s)
        q, s = _empty_rows(4, H)
        before = h.clone()
        kernels.add_rmsnorm_fp8(h, d, w, 1e-5, q, s, rows=rows, store_h=False)
        assert torch.equal(h, before) and torch.equal(q.float(), full.float()[rows.long()]) and torch.equal(s, full_s[:, rows.long()])
        q2, s2 = _empty_rows(6, H)
        kernels.add_rmsnorm_fp8(h2, None, w, 1e-5, q2, s2)      # the sum is in h2
        assert torch.equal(q2.float(), full.float()) and torch.equal(s2, full_s)
        q3, s3 = _empty_rows(3, H)
        kernels.add_rmsnorm_fp8(h, d, w, 1e-5, q3, s3, rows=torch.tensor([-1, 2, 6], dtype=torch.int32, device=DEV), store_h=False)
        assert torch.all(torch.isnan(q3.float()[[0, 2]])) and torch.all(torch.isnan(s3[:, [0, 2]])) and torch.equal(q3.float()[1], full.float()[2])


def test_norm_with_rows_off_16_bytes():
    from quanta_b200 import kernels
    g = _gen(2)
    flat = _randn(g, 4 * 256 + 1)
    h, w, d = flat[1:].view(4, 256), 1 + 0.1 * _randn(g, 257)[1:], _randn(g, 4 * 256 + 2)[2:].view(4, 256)
    q, s = _empty_rows(4, 256)
    q1, s1 = _empty_rows(4, 256)
    h1 = h.clone()
    kernels.add_rmsnorm_fp8(h1, d.clone(), w.clone(), 1e-5, q1, s1)
    kernels.add_rmsnorm_fp8(h, d, w, 1e-5, q, s)
    assert torch.equal(h, h1)
    assert torch.all((s - s1).abs() <= 2 * 264 * U * s1) and float((q.float() != q1.float()).float().mean()) < 0.01


GLUS = [(1, 8), (1, 5632), (3, 1), (2, 100), (5, 130), (37, 1000), (300, 2056), (2, 12345)]


def _act(kind, g, up, limit, alpha):
    if kind == 0:
        return g * torch.sigmoid(g) * up
    if kind == 1:
        g, up = g.clamp(max=limit), up.clamp(-limit, limit)
        return g * torch.sigmoid(alpha * g) * (up + 1)
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * up


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", GLUS)
def test_activation(n, width, dtype, kind, bias):
    from quanta_b200 import kernels
    g = _gen(n * width + kind)
    x = (2 * _randn(g, n, 2 * width)).to(dtype)
    b = _randn(g, 2 * width) if bias else None
    q, s = _empty_rows(n, width)
    kernels.glu_act_fp8(x, q, s, bias=b, kind=kind, limit=3.0, alpha=1.702)
    both = x.double() + (b.double() if bias else 0.0)
    gate, up = both[:, :width], both[:, width:]
    v = _act(kind, gate, up, 3.0, 1.702)
    # the bias' sum is off by u of its size; an activation's slope is at most 1.2 (alpha 1.702: 1.1), the other factor at most |up| + 1
    size = x.double().abs() + (b.double().abs() if bias else 0.0)
    arg = 2 * (gate.abs() + gate.abs() ** 3) if kind == 2 else 2 * gate.abs()
    off = 32 * U * (1 + arg) * v.abs() + 2 * U * (size[:, :width] * (up.abs() + 1) + size[:, width:] * (gate.abs() + 1))
    _rows_within(q, s, v, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(1, 16), (2, 129), (7, 4096), (300, 264)])
def test_rows(n, width, dtype):
    from quanta_b200 import kernels
    g = _gen(n + width)
    x = (_randn(g, n, width) * torch.exp(3 * _randn(g, n, 1))).to(dtype)
    q, s = _empty_rows(n, width)
    kernels.rows_to_fp8(x, q, s)
    _rows_within(q, s, x.double(), torch.zeros_like(x.double()))


def test_blocks_of_zeros_of_tiny_numbers_and_with_nan_or_infinity():
    from quanta_b200 import kernels
    x = torch.zeros(6, 384, device=DEV)
    x[1] = 1e-38
    x[2, 5], x[2, 200] = float("nan"), 2.0
    x[3, 7], x[3, 300] = float("inf"), -448.0
    x[4] = 3e38
    x[5, :128] = -1.0
    q, s = _empty_rows(6, 384)
    kernels.rows_to_fp8(x, q, s)
    v = q.float() * _spread(s, 384)
    assert torch.all(v[0] == 0) and torch.all(v[1] == 0) and torch.all(torch.isfinite(s[:, [0, 1, 4, 5]]))
    assert torch.allclose(s[:, 0], torch.full((3,), TINY / 448, device=DEV), rtol=1e-6, atol=0.0)
    assert torch.isnan(v[2, 5]) and torch.isnan(s[0, 2]) and v[2, 200] == 2.0
    assert not torch.isfinite(v[3, 7]) and not torch.isfinite(s[0, 3]) and v[3, 300] == -448.0
    assert torch.all((v[4] - x[4]).abs() <= 1e-6 * x[4]) and torch.all((v[5, :128] + 1).abs() <= 1e-6) and torch.all(v[5, 128:] == 0)


def _operands(T, K, N, seed):
    g = _gen(seed)
    x = (_randn(g, T, K) * 100).clamp(-448, 448).to(E4M3)
    w = (_randn(g, N, K) * 100).clamp(-448, 448).to(E4M3)
    xs = torch.exp(_randn(g, -(-K // 128), T)) * 1e-2
    ws = torch.exp(_randn(g, -(-N // 128), -(-K // 128))) * 1e-3
    return x, xs, w, ws


def _product(x, xs, w, ws, size=False):
    K, N = x.shape[1], w.shape[0]
    a = x.double() * _spread(xs.double(), K)
    b = w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return a.abs() @ b.abs().T if size else a @ b.T


def _product_within(out, x, xs, w, ws):
    want, size = _product(x, xs, w, ws), _product(x, xs, w, ws, size=True)
    tol = (2 * 128 + xs.shape[0] + 8) * U * size + (2.0 ** -8 * want.abs() if out.dtype == torch.bfloat16 else 0.0)
    assert torch.all((out.double() - want).abs() <= tol)


PRODUCTS = [(1, 16, 1), (1, 128, 128), (1, 4096, 300), (2, 2048, 4096), (16, 144, 129), (17, 2048, 640), (32, 5632, 384), (33, 1040, 200), (64, 256, 77),
            (65, 11008, 256), (100, 272, 300), (128, 128, 128), (129, 4096, 257), (256, 640, 130), (300, 1040, 384), (513, 2048, 1000),
            (700, 5648, 2000), (1025, 512, 40), (2500, 384, 2304), (2500, 400, 4001), (2561, 1280, 4104), (20000, 256, 640)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N", PRODUCTS)
def test_product(T, K, N, dtype):
    from quanta_b200 import kernels
    ops = _operands(T, K, N, T + K + N)
    out = torch.full((T, N), float("nan"), device=DEV, dtype=dtype)
    status = kernels.new_status(DEV)
    kernels.linear_fp8(*ops, out, status)
    assert int(status[0]) == 0
    _product_within(out, *ops)
    again = torch.empty_like(out)
    kernels.linear_fp8(*ops, again)
    assert torch.equal(out, again)


def test_product_writes_its_rows_and_nothing_else():
    from quanta_b200 import kernels
    for T, K, N in ((3, 256, 130), (40, 2048, 100), (200, 256, 131), (300, 128, 257)):
        ops = _operands(T, K, N, T)
        big = torch.full((T * N + 512,), 7.0, device=DEV)
        out = big[256: 256 + T * N].view(T, N)
        kernels.linear_fp8(*ops, out)
        assert torch.all(big[:256] == 7) and torch.all(big[256 + T * N:] == 7)
        _product_within(out, *ops)


def test_nan_stays_in_its_row_and_column():
    from quanta_b200 import kernels
    for T in (5, 40, 300):
        x, xs, w, ws = _operands(T, 640, 300, T)
        xb = x.view(torch.uint8)
        xb[3, 130] = 0x7f
        w.view(torch.uint8)[77, 9] = 0xff
        xs[2, 1], ws[2, 1] = float("inf"), float("nan")
        out = torch.empty(T, 300, device=DEV)
        kernels.linear_fp8(x, xs, w, ws, out)
        bad = ~torch.isfinite(out)
        want = torch.zeros_like(bad)
        want[[1, 3]], want[:, 77], want[:, 256:] = True, True, True
        assert torch.equal(bad, want)


def test_on_another_stream_and_in_a_graph():
    from quanta_b200 import kernels
    g = _gen(5)
    h0, d, w = _randn(g, 9, 512), _randn(g, 9, 512), 1 + 0.1 * _randn(g, 512)
    _, _, wq, ws = _operands(1, 512, 384, 6)
    h = h0.clone()
    q, s = _empty_rows(9, 512)
    act, act_s = _empty_rows(9, 192)
    mid = torch.empty(9, 384, device=DEV, dtype=torch.bfloat16)

    def run():
        h.copy_(h0)
        kernels.add_rmsnorm_fp8(h, d, w, 1e-5, q, s)
        kernels.linear_fp8(q, s, wq, ws, mid)
        kernels.glu_act_fp8(mid, act, act_s)
        return [t.clone() for t in (h, q, s, mid, act, act_s)]

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = run()
    side.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    d.add_(0.0)
    for t in (mid, act_s):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held, want))


@pytest.mark.parametrize("T,K,N", [(3, 2048, 640), (24, 2048, 640), (50, 2048, 640), (200, 2048, 640), (700, 1024, 5000)])
def test_two_calls_at_once(T, K, N):
    """On two streams, neither waiting for the other: no call leaves anything that another could read."""
    from quanta_b200 import kernels
    a, b = _operands(T, K, N, 1), _operands(T, K, N, 2)
    want = []
    for ops in (a, b):
        want.append(torch.empty(T, N, device=DEV))
        kernels.linear_fp8(*ops, want[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty(T, N, device=DEV) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for k, ops in enumerate((a, b)):
            with torch.cuda.stream(streams[k]):
                kernels.linear_fp8(*ops, outs[k][i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[k]) for k in range(2) for o in outs[k])


def test_empty_calls():
    from quanta_b200 import kernels
    q, s = _empty_rows(0, 256)
    kernels.rows_to_fp8(torch.empty(0, 256, device=DEV), q, s)
    kernels.glu_act_fp8(torch.empty(0, 512, device=DEV), q, s)
    kernels.add_rmsnorm_fp8(torch.empty(0, 256, device=DEV), None, torch.ones(256, device=DEV), 1e-5, q, s)
    _, _, w, ws = _operands(1, 256, 100, 1)
    kernels.linear_fp8(q, s, w, ws, torch.empty(0, 100, device=DEV))
    x, xs, _, _ = _operands(5, 256, 100, 1)
    kernels.linear_fp8(x, xs, w[:0], ws[:0], torch.empty(5, 0, device=DEV))
    torch.cuda.synchronize()


# Products of few tokens whose matrix is too large for the kernel without tensor memory: one k block, k that ends inside one, k cut over the blocks
# of a cluster unevenly, weight rows that end inside a tile, as many tokens as a tile has and one more.
LARGE_PRODUCTS = [(9, 4112, 9001), (16, 8192, 5000), (17, 4112, 4104), (32, 11008, 4096), (33, 8208, 1003), (48, 2064, 8200), (64, 4240, 1000), (64, 16, 300001),
                  (50, 65552, 129), (65, 16, 260000), (100, 4112, 1001), (128, 16400, 257), (129, 2064, 2085), (200, 5648, 2000), (257, 16, 5), (257, 144, 200),
                  (300, 2064, 130), (260, 40016, 33), (1000, 144, 2600), (2049, 528, 1500), (33, 8208, 2003), (64, 4240, 2000), (50, 65552, 300), (40, 144, 20001),
                  (128, 16400, 520), (257, 16, 4100), (300, 2192, 640), (260, 40016, 130), (700, 2320, 384), (1000, 512, 64), (9000, 16, 16), (5, 16, 40001),
                  (400, 4112, 3000), (512, 5648, 4001), (1030, 4240, 2000), (1300, 4096, 4096), (200, 2064, 20008), (200, 2064, 20001),      # pairs with 128 weight rows
                  (100, 2064, 22016), (128, 528, 20001), (70, 144, 37888), (65, 1040, 19080),      # blocks alone with 256
                  (64, 4112, 8200), (33, 4112, 9480), (64, 528, 11264), (50, 4096, 22016)]      # up to 64 tokens, as rows or as columns


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N", LARGE_PRODUCTS)
def test_large_product(T, K, N, dtype):
    from quanta_b200 import kernels
    ops = _operands(T, K, N, T + K + N)
    out, again, ahead = (torch.full((T, N), float("nan"), device=DEV, dtype=dtype) for _ in range(3))
    status = kernels.new_status(DEV)
    kernels.linear_fp8(*ops, out, status)
    kernels.linear_fp8(*ops, again, status)
    kernels.linear_fp8(*ops, ahead, status, early=True)
    assert int(status[0]) == 0
    _product_within(out, *ops)
    assert torch.equal(out, again) and torch.equal(out, ahead)


@pytest.mark.parametrize("T", [40, 100])
@pytest.mark.parametrize("N", [1100, 2100])
def test_nan_stays_in_its_row_and_column_of_a_large_product(T, N):
    from quanta_b200 import kernels
    x, xs, w, ws = _operands(T, 6400, N, T)
    x.view(torch.uint8)[3, 130] = 0x7f
    w.view(torch.uint8)[77, 9] = 0xff
    xs[2, 1], ws[2, 1] = float("inf"), float("nan")
    out = torch.empty(T, N, device=DEV)
    kernels.linear_fp8(x, xs, w, ws, out)
    want = torch.zeros(T, N, dtype=torch.bool, device=DEV)
    want[[1, 3]], want[:, 77], want[:, 256:384] = True, True, True
    assert torch.equal(~torch.isfinite(out), want)


@pytest.mark.parametrize("T,K,N", [(1, 512, 2048), (7, 4096, 700), (20, 2048, 1024), (40, 512, 512), (20, 8192, 4000), (64, 2048, 4096), (64, 4096, 2100), (100, 4096, 1024), (100, 512, 20000), (300, 512, 640), (300, 2048, 640)])
def test_weights_read_ahead_of_the_rows(T, K, N):
    """Rows that the launch just before writes, in a chain, eagerly and in a graph: only the weights are read before it has ended."""
    from quanta_b200 import kernels
    g = _gen(T)
    _, _, w, ws = _operands(1, K, N, 3)
    xs = [_randn(g, T, K) * 4.0 ** i for i in range(6)]
    q, s = _empty_rows(T, K)

    def chain(outs, early):
        for x, out in zip(xs, outs):
            kernels.rows_to_fp8(x, q, s)
            kernels.linear_fp8(q, s, w, ws, out, early=early)

    want, got, held = (torch.empty(6, T, N, device=DEV) for _ in range(3))
    for x, out in zip(xs, want):
        kernels.rows_to_fp8(x, q, s)
        torch.cuda.synchronize()
        kernels.linear_fp8(q, s, w, ws, out)
        torch.cuda.synchronize()
    chain(got, True)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(held, True)
    for _ in range(3):
        held.zero_()
        graph.replay()
        assert torch.equal(held, want)


@pytest.mark.parametrize("T,K,N", [(30, 8192, 4000), (64, 4096, 2100), (100, 4096, 1024)])
def test_two_large_calls_at_once(T, K, N):
    test_two_calls_at_once(T, K, N)


@pytest.mark.parametrize("T,N", [(140000, 16400), (140000, 16401)])
def test_product_of_more_than_32_bits_of_numbers(T, N):
    from quanta_b200 import kernels
    K = 128
    g = _gen(T)
    _, _, w, ws = _operands(1, K, N, 1)
    some, scale = _operands(1000, K, 8, 2)[:2]
    pick = torch.randint(0, 1000, (T,), device=DEV, generator=g)
    x, xs = some.view(torch.uint8)[pick].view(E4M3), scale[:, pick].contiguous()
    out = torch.empty(T, N, device=DEV, dtype=torch.bfloat16)
    kernels.linear_fp8(x, xs, w, ws, out)
    few = torch.empty(1000, N, device=DEV, dtype=torch.bfloat16)
    kernels.linear_fp8(some, scale, w, ws, few)
    _product_within(few, some, scale, w, ws)
    for t0 in (0, 65536, 130900, T - 1000):
        assert torch.equal(out[t0: t0 + 1000], few[pick[t0: t0 + 1000]])


def test_rows_of_more_than_32_bits_of_numbers():
    from quanta_b200 import kernels
    g = _gen(9)
    n, width = 100000, 11008
    some = (2 * _randn(g, 500, 2 * width)).bfloat16()
    pick = torch.randint(0, 500, (n,), device=DEV, generator=g)
    q, s = _empty_rows(n, width)
    kernels.glu_act_fp8(some[pick], q, s)
    q0, s0 = _empty_rows(500, width)
    kernels.glu_act_fp8(some, q0, s0)
    ends = torch.cat([torch.arange(1000), torch.arange(n - 1000, n)]).to(DEV)
    assert torch.equal(q.view(torch.uint8)[ends], q0.view(torch.uint8)[pick[ends]]) and torch.equal(s[:, ends], s0[:, pick[ends]])
    n, H = 540000, 4096
    some, w = _randn(g, 500, H), 1 + 0.1 * _randn(g, H)
    pick = torch.randint(0, 500, (n,), device=DEV, generator=g)
    q, s = _empty_rows(n, H)
    kernels.add_rmsnorm_fp8(some[pick], None, w, 1e-5, q, s)
    q0, s0 = _empty_rows(500, H)
    kernels.add_rmsnorm_fp8(some, None, w, 1e-5, q0, s0)
    ends = torch.cat([torch.arange(1000), torch.arange(n - 1000, n)]).to(DEV)
    assert torch.equal(q.view(torch.uint8)[ends], q0.view(torch.uint8)[pick[ends]]) and torch.equal(s[:, ends], s0[:, pick[ends]])


def test_first_call_inside_a_capture():
    """Nothing that a kernel needs at its first launch keeps it from being captured: each in a process of its own kind of call."""
    import subprocess
    import sys
    code = """
import torch
from quanta_b200 import kernels, fp8
dev = "cuda:0"
kernels.lib().unit("fp8"); kernels.lib().unit("scores")
cases = [(1, 512, 640), (24, 512, 640), (30, 4224, 8000), (60, 4224, 8000), (100, 4224, 1000), (300, 2176, 640), (600, 4224, 4000), (2000, 512, 4000)]
held = []
x = [torch.randn(T, K, device=dev) for T, K, N in cases]
w = [fp8.quantize_weight(torch.randn(N, K, device=dev)) for T, K, N in cases]
logits = [torch.randn(n, 50000, device=dev) for n in (1, 200)]
torch.cuda.synchronize()
def run():
    outs = []
    for a, b in zip(x, w):
        r = fp8.quantize_rows(a)
        out = torch.empty(a.shape[0], b.shape[0], device=dev)
        kernels.linear_fp8(r.q, r.scales, b.q, b.scales, out)
        outs.append(out)
    for l in logits:
        en, ids, best = torch.empty(l.shape[0], device=dev), torch.empty(l.shape[0], 5, device=dev, dtype=torch.int32), torch.empty(l.shape[0], 5, device=dev)
        kernels.token_logprobs(l, None, None, en, ids, best)
        outs += [en, ids, best]
    return outs
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(held, run()))
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


ODD_NORMS = [(3, 2434, 1), (50, 1062, 8), (300, 789, 1), (4, 8191, 2), (2, 129, 1), (1000, 33, 3), (2, 8193, 1)]


@pytest.mark.parametrize("gain", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,H,S", ODD_NORMS)
def test_norm_of_rows_that_do_not_lie_on_16_bytes(n, H, S, dtype, gain):
    test_norm(n, H, S, dtype, gain)


def test_rows_of_any_place():
    """Rows that begin one number behind a 16-byte place, of a width that would be whole pieces: the same numbers as rows that do not."""
    from quanta_b200 import kernels
    g = _gen(12)
    n, H = 9, 1024
    h, d, w = _randn(g, n, H), _randn(g, n, H), 1 + 0.2 * _randn(g, H)
    q, s = _empty_rows(n, H)
    h0 = h.clone()
    kernels.add_rmsnorm_fp8(h0, d, w, 1e-5, q, s)
    behind = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    h1, q1, s1 = behind(h), behind(q.view(torch.uint8)).view(E4M3), torch.empty_like(s)
    kernels.add_rmsnorm_fp8(h1, behind(d), behind(w), 1e-5, q1, s1)
    assert torch.equal(h1, h0)
    # (the sums of squares are taken in another order)
    assert torch.all((q1.float() * _spread(s1, H) - q.float() * _spread(s, H)).abs() <= 2.0 ** -4 * (q.float() * _spread(s, H)).abs() + 2.0 ** -9 * _spread(s, H))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N", [(1054, 1280, 3207), (300, 144, 20003), (2000, 528, 1999), (128, 528, 20003), (100, 4112, 1003), (40, 8208, 2001), (130, 2064, 2086), (700, 4112, 4095)])
def test_product_whose_rows_do_not_lie_on_16_bytes(T, K, N, dtype):
    from quanta_b200 import kernels
    ops = _operands(T, K, N, T + K + N)
    big = torch.full((T * N + 512,), 7.0, device=DEV, dtype=dtype)
    out = big[256: 256 + T * N].view(T, N)
    kernels.linear_fp8(*ops, out)
    assert torch.all(big[:256] == 7) and torch.all(big[256 + T * N:] == 7)
    _product_within(out, *ops)

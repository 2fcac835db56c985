"""The 8-bit integer product and its quantisers against their definitions.

The integer sum is exact, so a product's output is off by the fp32 epilogue
and one rounding to its type: the conversion of the sum, two scales and the
residual are one half step of fp32 each (2^-24), SiLU adds its exponential and
division (2 ulp and the argument's error, together under 2^-20 of the value
for |g| <= 16: g * 2^-23 in the exponent), the rounding half a step of y."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def codes(rows, cols, seed, ld=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or -(-cols // 16) * 16
    return torch.randint(-127, 128, (rows, ld), dtype=torch.int8, device="cuda", generator=g)[:, :cols]


def want_y(xq, sx, wq, sw, planes, residual):
    n = wq.shape[0] // planes
    y = (xq.double() @ wq.double().T) * sx.double()[:, None] * sw.double()[None]
    if planes == 2:
        g, u = y[:, :n], y[:, n:]
        y = g * torch.sigmoid(g) * u
    return y if residual is None else y + residual.double()


def check_product(b2g, m, n, k, dtype="fp16", fuse=0, seed=3, ldx=None, op=None, ws=None):
    planes = 2 if fuse & b2g.FUSE_GATE_UP_SILU else 1
    xq, wq = codes(m, k, seed, ldx), codes(planes * n, k, seed + 1)
    g = torch.Generator(device="cuda").manual_seed(seed)
    sx = (0.5 + torch.rand(m, device="cuda", generator=g)) / 73
    sw = (0.5 + torch.rand(planes * n, device="cuda", generator=g)) / 73 / math.sqrt(k)
    t = TYPES[dtype]
    res = torch.randn(m, n, device="cuda", generator=g).to(t) if fuse & b2g.FUSE_RESIDUAL_ADD else None
    op = op or b2g.I8Op(k, n, max_m=m, fuse=fuse, dtype=dtype)
    ws = op.workspace() if ws is None else ws
    want = want_y(xq, sx, wq, sw, planes, res)
    for _ in range(2):  # the second call finds the workspace as the first one left it
        y = op.enqueue_codes(xq, sx, wq, sw, residual=res, workspace=ws)
        torch.cuda.synchronize()
        eps = torch.finfo(t).eps / 2
        parts = want.abs() if res is None else want.abs() + 2 * res.double().abs()
        bound = eps * want.abs() + (2.0 ** -19 if planes == 2 else 2.0 ** -21) * parts + 2.0 ** -25
        err = (y.double() - want).abs()
        assert bool((err <= bound).all()), (m, n, k, float((err / bound).max()))
    assert b2g.device_error() == 0
    return y


# (tokens, channels, k): one k block, k that is no multiple of the block or of
# 16, channels that end inside a tile, each way of cutting the work (whole
# tiles, clusters of 2, 4, 8, shared ranges, deep tiles), token tiles of 32 to
# 256.
SHAPES = [(1, 1, 1), (1, 128, 128), (2, 17, 40), (5, 100, 1000), (32, 128, 256), (33, 129, 129), (1, 4096, 2048),
          (8, 1024, 8192), (64, 2048, 512), (100, 8192, 256), (127, 300, 4096), (256, 19000, 128), (257, 513, 77),
          (300, 9600, 1024), (517, 1000, 640), (1, 20000, 64), (700, 5000, 300),
          (1000, 6000, 700), (1500, 5000, 333), (2049, 4100, 130),
          (30, 300, 8000), (34, 221, 7296), (512, 1024, 1500), (146, 272, 7184), (281, 1712, 1500), (2997, 1121, 136),
          (61, 6288, 448), (1026, 2241, 640)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_product(b2g, cuda, m, n, k, dtype):
    check_product(b2g, m, n, k, dtype)


@pytest.mark.parametrize("m,n,k", [s for s in SHAPES if s[1] < 10000])
def test_gate_up(b2g, cuda, m, n, k):
    check_product(b2g, m, n, k, "bf16", b2g.FUSE_GATE_UP_SILU)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_residual(b2g, cuda, m, n, k):
    check_product(b2g, m, n, k, "fp16", b2g.FUSE_RESIDUAL_ADD)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m", [3, 300])
def test_gates_far_from_zero(b2g, cuda, dtype, m):
    """Gates to +-200, past where exp overflows.  The gate is off by 3 half
    steps of fp32, its exponential by |g| times that, |g| 2^-24 for the argument
    and 2 ulp, the division by 2 ulp: (|g| + 8) 2^-22 of the value; where
    1 + exp(-g) passes 2^126 it may be 0, which is off by |g u| 2^-126."""
    n, k, t = 300, 128, TYPES[dtype]
    xq, wq = codes(m, k, 11), codes(2 * n, k, 12)
    sx = torch.full((m,), 1 / 73.0, device="cuda")
    sw = torch.cat([torch.full((n,), 60 / 73 / math.sqrt(k), device="cuda"),
                    torch.full((n,), 1 / 73 / math.sqrt(k), device="cuda")])
    op = b2g.I8Op(k, n, max_m=m, fuse=b2g.FUSE_GATE_UP_SILU, dtype=dtype)
    y = op.enqueue_codes(xq, sx, wq, sw, workspace=op.workspace())
    both = (xq.double() @ wq.double().T) * sx.double()[:, None] * sw.double()[None]
    g, u = both[:, :n], both[:, n:]
    assert float(g.min()) < -130 and float(g.max()) > 130
    want = g * torch.sigmoid(g) * u
    bound = (torch.finfo(t).eps / 2 + (g.abs() + 8) * 2.0 ** -22) * want.abs() + (g * u).abs() * 2.0 ** -126 + 2.0 ** -25
    assert bool(((y.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("m", [3, 300])
def test_gates_whose_exponential_is_large(b2g, cuda, m):
    """Gates of -60 to -100 under an up of 10^30: their SiLU is down to 10^-42, but
    the product is a plain bf16 number.  The bound is test_gates_far_from_zero's;
    below 2^-126 the exponential has steps of 2^-149."""
    n, k = 300, 128
    g = -60 - 40 * torch.arange(n, device="cuda").float() / n
    sw = torch.cat([-g / k, torch.full((n,), 1e30 / k, device="cuda")])
    xq, wq = torch.ones(m, k, dtype=torch.int8, device="cuda"), torch.ones(2 * n, k, dtype=torch.int8, device="cuda")
    wq[:n] = -1
    op = b2g.I8Op(k, n, max_m=m, fuse=b2g.FUSE_GATE_UP_SILU, dtype="bf16")
    y = op.enqueue_codes(xq, torch.ones(m, device="cuda"), wq, sw)
    gate, up = -k * sw[:n].double(), k * sw[n:].double()
    want = gate * torch.sigmoid(gate) * up
    bound = (2.0 ** -8 + (gate.abs() + 8) * 2.0 ** -22) * want.abs() + (gate * up).abs() * 2.0 ** -148
    assert bool(((y.double() - want).abs() <= bound).all())


def test_extreme_codes(b2g, cuda):
    """The largest sums: every product 127 * 127 or (-128) * (-128) at the
    largest k; one more k could reach 2^31 and is refused."""
    with pytest.raises(b2g.B2GError):
        b2g.I8Op(131072, 40, max_m=3)
    k = 131071
    op = b2g.I8Op(k, 40, max_m=3)
    x, w = (torch.full((rows, 131072), 127, dtype=torch.int8, device="cuda")[:, :k] for rows in (3, 40))
    w[1] = -128
    x[2] = -128
    one = torch.ones(40, device="cuda")
    y = op.enqueue_codes(x, one[:3] * 2.0 ** -20, w, one)
    want = (x.double() @ w.double().T) * 2.0 ** -20
    assert bool(((y.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -22) * want.abs()).all())


def test_rows_of_a_wider_matrix_and_y_in_place_of_the_residual(b2g, cuda):
    m, n, k = 70, 260, 300
    xq, wq = codes(m, k, 1, 512), codes(n, k, 2, 1024)
    sx, sw = torch.rand(m, device="cuda") / 100, torch.rand(n, device="cuda") / 100
    wide = torch.randn(m, 2 * n + 1, device="cuda").half()
    y = wide[:, 3:3 + n]
    res = y.clone()
    op = b2g.I8Op(k, n, max_m=128, fuse=b2g.FUSE_RESIDUAL_ADD)
    before = wide.clone()
    out = op.enqueue_codes(xq, sx, wq, sw, residual=y, y=y)
    assert out is y
    want = want_y(xq, sx, wq, sw, 1, res)
    assert bool(((y.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20 * (1 + want.abs())).all())
    before[:, 3:3 + n] = y
    assert torch.equal(before, wide)


def scales_right(s, v):
    """Each the fp32 number next to max(max|v|, fp32(1e-12)) / 127."""
    want = v.abs().amax(1).clamp(min=1e-12).double() / 127
    return bool(((s.double() - want).abs() <= 2.0 ** -24 * want).all())


def test_quantised_rows(b2g, cuda):
    """Codes are the rounded fp32 quotients, ties among them (x takes few
    values), the largest 127, scales rounded once."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for dtype in TYPES.values():
        for m, k in ((1, 1), (3, 8), (2, 13), (5, 1000), (7, 8192), (2, 16384), (2, 16385), (1, 100000), (300, 64)):
            x = torch.randn(m, k, device="cuda", generator=g).to(dtype)
            x[-1] = torch.round(x[-1] * 8) / 8
            wide = torch.zeros(m, -(-k // 8) * 8 + 8, device="cuda", dtype=dtype)
            wide[:, :k] = x
            for src in (x if k % 8 == 0 or m == 1 else wide[:, :k], wide[:, :k]):
                q, s = b2g.quantize_i8_rows(src)
                v = x.float()
                assert scales_right(s, v)
                assert torch.equal(q.float(), torch.round(v / s[:, None]))  # the fp32 quotient, ties to even
                assert bool((q.int().abs().amax(1) == 127).all())


def test_quantised_normalised_rows(b2g, cuda):
    g = torch.Generator(device="cuda").manual_seed(6)
    for dtype in TYPES.values():
        for m, k in ((1, 8), (5, 1000), (3, 8192), (2, 20000)):
            x = (torch.randn(m, k, device="cuda", generator=g) * 3).to(dtype)
            gamma = (1 + torch.randn(k, device="cuda", generator=g) / 8).to(dtype)
            for gm in (None, gamma):
                q, s = b2g.quantize_i8_rows(x, gamma=gm, rms_eps=1e-5)
                v = x.double() * torch.rsqrt(x.double().square().mean(1, keepdim=True) + 1e-5)
                v = v if gm is None else v * gm.double()
                want = v.abs().amax(1) / 127
                # a sum of k squares in fp32 (pairwise over at most 64 in a row), rsqrt, two products
                assert bool(((s.double() - want).abs() <= 2.0 ** -16 * want).all())
                assert bool(((v / want[:, None] - q.double()).abs() <= 0.5 + 127 * 2.0 ** -16).all())


def test_rows_that_are_zero_or_not_finite(b2g, cuda):
    k, n = 300, 40
    x = torch.randn(6, 304, device="cuda").half()[:, :k]
    x[1] = 0
    x[2, 7] = math.nan
    x[3, 299] = math.inf
    x[4, 0] = -math.inf
    q, s = b2g.quantize_i8_rows(x)
    assert scales_right(s[:2], x[:2].float()) and not bool(q[1].any())
    assert bool(s[2:5].isnan().all()) and not bool(q[2:5].any())
    w = torch.randn(n, k, device="cuda").half()
    wq, sw = b2g.quantize_i8_weights(w, layout="NK")
    for op, kw in ((b2g.I8Op(k, n, 6), {}), (b2g.I8Op(k, n, 6, fuse=b2g.FUSE_RMSNORM_INPUT), {})):
        y = op.enqueue(x, wq, sw, **kw)
        assert bool(y[2:5].isnan().all()) and bool(y[[0, 1, 5]].isfinite().all()) and not bool(y[1].any())


@pytest.mark.parametrize("layout", ["KN", "NK"])
def test_quantised_weights(b2g, cuda, layout):
    for K, N in ((1, 1), (33, 17), (200, 120), (1000, 64), (64, 1000)):
        w = torch.randn(K, N, device="cuda").bfloat16()
        q, s = b2g.quantize_i8_weights(w if layout == "KN" else w.T.contiguous(), layout)
        v = w.float().T
        assert scales_right(s, v)
        assert bool(((v.double() / s.double()[:, None] - q.double()).abs() <= 0.5 + 2.0 ** -15).all())


@pytest.mark.parametrize("m", [1, 3, 8, 130])
def test_rows_through_the_product_equal_codes_through_it(b2g, cuda, m):
    """enqueue is quantize_i8_rows and enqueue_codes, to the bit."""
    k, n = 1000, 700
    x = torch.randn(m, k, device="cuda").bfloat16()
    gamma = (1 + torch.randn(k, device="cuda") / 8).bfloat16()
    wq, sw = codes(2 * n, k, 4), torch.rand(2 * n, device="cuda") / 3000
    fuse = b2g.FUSE_GATE_UP_SILU
    a = b2g.I8Op(k, n, 130, fuse | b2g.FUSE_RMSNORM_INPUT, "bf16").enqueue(x, wq, sw, gamma=gamma, rms_eps=1e-6)
    xq, sx = b2g.quantize_i8_rows(x, gamma=gamma, rms_eps=1e-6)
    b = b2g.I8Op(k, n, 130, fuse, "bf16").enqueue_codes(xq, sx, wq, sw)
    assert torch.equal(a, b)


def test_captured_and_on_two_streams(b2g, cuda):
    m, n, k = 9, 1024, 4096
    op = b2g.I8Op(k, n, 16)
    x = torch.randn(m, k, device="cuda").half()
    wq, sw = codes(n, k, 4), torch.rand(n, device="cuda") / 3000
    want = op.enqueue(x, wq, sw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [op.enqueue(x, wq, sw, stream=streams[i % 2]) for i in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):  # a workspace each: replayed at the same time
        ws, y, g = op.workspace(), torch.empty(m, n, device="cuda", dtype=torch.float16), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            op.enqueue(x, wq, sw, y=y, workspace=ws)
        graphs.append((g, y, ws))
    for i in range(10):
        for s, (g, y, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, y, _ in graphs)
    x.copy_(torch.randn(m, k, device="cuda").half())
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], op.enqueue(x, wq, sw))


def test_sizes_in_turn_on_one_workspace(b2g, cuda):
    """One op, calls of every cut of the work one after the other."""
    op = b2g.I8Op(4096, 3000, max_m=300, fuse=b2g.FUSE_RMSNORM_INPUT)
    ws = op.workspace()
    wq, sw = codes(3000, 4096, 4), torch.rand(3000, device="cuda") / 3000
    for m in (300, 1, 200, 33, 300, 8):
        x = torch.randn(m, 4096, device="cuda").half()
        assert torch.equal(op.enqueue(x, wq, sw, workspace=ws), op.enqueue(x, wq, sw))


def test_refusals(b2g, cuda):
    op = b2g.I8Op(64, 32, 4)
    xq, sx, wq, sw = codes(4, 64, 1), torch.ones(4, device="cuda"), codes(32, 64, 2), torch.ones(32, device="cuda")
    ok = op.enqueue_codes(xq, sx, wq, sw)
    with pytest.raises(ValueError):
        op.enqueue_codes(xq, sx, wq[:31], sw)
    with pytest.raises(ValueError):
        op.enqueue_codes(xq, sx, wq.cpu(), sw)
    with pytest.raises(ValueError):
        op.enqueue_codes(xq, sx, wq, sw, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        op.enqueue(torch.randn(4, 64, device="cuda"), wq, sw)
    with pytest.raises(b2g.B2GError):  # more rows than max_m
        op.enqueue_codes(codes(5, 64, 1), torch.ones(5, device="cuda"), wq, sw)
    with pytest.raises(b2g.B2GError):  # a residual that the op does not take
        op.enqueue_codes(xq, sx, wq, sw, residual=ok)
    with pytest.raises(b2g.B2GError):  # rows that do not start 16-byte aligned
        op.enqueue_codes(codes(4, 65, 1, 65)[:, :64], sx, wq, sw)
    with pytest.raises(b2g.B2GError):  # codes cannot be normalised
        b2g.I8Op(64, 32, 4, b2g.FUSE_RMSNORM_INPUT).enqueue_codes(xq, sx, wq, sw)
    torch.cuda.synchronize()
    assert b2g.device_error() == 0

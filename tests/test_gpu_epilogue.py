"""The W8A8 product's epilogue: what comes before the activation is the product without one,
bit for bit; the activation and the residual are held to their formula in 64 bits on those
fp32 values.

Tolerances, with u = 2^-24 (half a step of fp32). A sigmoid form x / (1 + exp(-v)): v is
rounded three times, so exp(-v) is off by 3 |v| u and its own 2 u; through the quotient
that is at most u (3 max |v| s(v) s(-v) |x| + ...) <= u (0.7 |x| + 2 |y|), the sum and the
quotient add 2 u |y|: u (|x| + 4 |y|). The erfc form: its argument is off by 2 u, which
moves y by at most |x|/2 * 2/sqrt(pi) max(z exp(-z^2)) 2 u < u |x|; erfcf may be off by 16
units (32 u |y|), two products: u (|x| + 35 |y|). Adding the residual rounds once more:
u |y + r|. relu and no activation are exact."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24

# rows, in, out: the few-rows kernels (16 or 32 rows, 16 or 32 features a workgroup), then
# every tile that the library selects, with odd ends
SHAPES = [(1, 16, 1), (3, 64, 40), (16, 512, 4096), (29, 1040, 515), (10, 256, 5001),
          (100, 400, 1030), (70, 256, 6143), (300, 144, 3001), (1000, 96, 2051), (2050, 128, 1283),
          (4099, 64, 1280), (2000, 128, 6145), (4097, 48, 8190)]


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


def problem(rows, fin, fout, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + fout)
    xq = torch.randint(-127, 128, (rows, fin), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-127, 128, (fout, fin), generator=g, device="cuda").to(torch.int8)
    xs = 0.5 + torch.rand(rows, generator=g, device="cuda")
    # outputs of a few units either side of 0
    ws = (0.5 + torch.rand(fout, generator=g, device="cuda")) * (3.0 / (5376 * math.sqrt(fin)))
    bias = torch.randn(fout, generator=g, device="cuda")
    res = torch.randn((rows, fout), generator=g, device="cuda")
    return xq, xs, w, ws, bias, res


def activated(x, name):
    """The activation of fp32 values in float64, and its tolerance."""
    d = x.double()
    a = d.abs()
    if name == "relu":
        return d.clamp(min=0), 0 * a
    if name == "gelu_erf":
        y = 0.5 * d * torch.erfc(-d / math.sqrt(2))
        return y, U * (a + 35 * y.abs())
    if name == "none":
        return d, 0 * a
    v = d if name == "silu" else 2 * math.sqrt(2 / math.pi) * (d + 0.044715 * d ** 3)
    y = d / (1 + torch.exp(-v))
    return y, U * (a + 4 * y.abs())


def check(y, x, name, res=None):
    ref, tol = activated(x, name)
    if res is not None:
        ref = ref + res.double()
        tol = tol + U * ref.abs() * (1 + 1e-6)
    far = (y.double() - ref).abs() - tol
    assert float(far.max()) <= 0, (name, float(far.max()))


@pytest.mark.parametrize("rows,fin,fout", SHAPES)
def test_epilogue_matches_formula(reef, rows, fin, fout):
    xq, xs, w, ws, bias, res = problem(rows, fin, fout)
    print(f"\n[case] product {rows}x{fin}->{fout}", flush=True)
    plain = reef.gemm_w8a8(xq, xs, w, ws, bias)
    acc = (xq.cpu().double() @ w.cpu().double().t()).float() if rows * fin * fout < 1 << 28 else None
    if acc is not None:  # the engine's float steps, one rounding each
        assert torch.equal(plain.cpu(), acc * (xs.cpu()[:, None] * ws.cpu()[None]) + bias.cpu())
    for name in reef.ACTIVATIONS:
        y = reef.gemm_w8a8(xq, xs, w, ws, bias, activation=name, residual=res)
        check(y, plain, name, res)
    y = reef.gemm_w8a8(xq, xs, w, ws, bias, activation="gelu_tanh")
    check(y, plain, "gelu_tanh")
    nobias = reef.gemm_w8a8(xq, xs, w, ws)
    check(reef.gemm_w8a8(xq, xs, w, ws, residual=res), nobias, "none", res)
    assert torch.equal(reef.gemm_w8a8(xq, xs, w, ws, activation="none"), nobias)


@pytest.mark.parametrize("rows,fin,fout", [(5, 64, 33), (150, 128, 1030), (2050, 128, 1284)])
def test_epilogue_in_place_and_strided(reef, rows, fin, fout):
    """y over the residual; y and residual as columns of wider matrices, off 16 bytes."""
    xq, xs, w, ws, bias, res = problem(rows, fin, fout, 1)
    print(f"\n[case] product in place {rows}x{fin}->{fout}", flush=True)
    ref = reef.gemm_w8a8(xq, xs, w, ws, bias, activation="silu", residual=res)
    wide = torch.full((rows, fout + 9), 5.0, device="cuda")
    wide[:, 3:3 + fout] = res
    y = reef.gemm_w8a8(xq, xs, w, ws, bias, activation="silu", residual=wide[:, 3:3 + fout])
    assert torch.equal(y, ref)
    other = torch.full((rows, fout + 6), 7.0, device="cuda")
    reef.gemm_w8a8(xq, xs, w, ws, bias, activation="silu", residual=wide[:, 3:3 + fout],
                   out=other[:, 1:1 + fout])
    assert torch.equal(other[:, 1:1 + fout], ref)
    assert (other[:, :1] == 7).all() and (other[:, 1 + fout:] == 7).all()
    for view in (wide[:, 3:3 + fout], res):
        out = reef.gemm_w8a8(xq, xs, w, ws, bias, activation="silu", residual=view, out=view)
        assert out.data_ptr() == view.data_ptr() and torch.equal(view, ref)
    assert (wide[:, :3] == 5).all() and (wide[:, 3 + fout:] == 5).all()


def test_linear_with_epilogue(reef):
    print("\n[case] linear with epilogue", flush=True)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((77, 192), generator=g, device="cuda")
    _, _, w, ws, bias, res = problem(77, 192, 301)
    plain = reef.linear_w8a8(x, w, ws, bias)
    y = reef.linear_w8a8(x, w, ws, bias, activation="gelu_erf", residual=res)
    check(y, plain, "gelu_erf", res)
    q, s = reef.quantize_rows(x)
    assert torch.equal(y, reef.gemm_w8a8(q, s, w, ws, bias, activation="gelu_erf", residual=res))


def test_activations_over_their_range(reef):
    """One output per value: a product of 1 by codes, scaled. Far left of 0 the GELUs and
    SiLU go to 0 from below, far right to x."""
    print("\n[case] activations -300 .. 300", flush=True)
    n = 255
    w = torch.zeros((n, 16), dtype=torch.int8, device="cuda")
    w[:, 0] = torch.arange(-127, 128, device="cuda").to(torch.int8)
    xq = torch.zeros((6, 16), dtype=torch.int8, device="cuda")
    xq[:, 0] = 1
    xs = torch.tensor([1e-30, 1e-3, 0.01, 0.1, 2.4, 1e20], device="cuda")
    ws = torch.ones(n, device="cuda")
    plain = reef.gemm_w8a8(xq, xs, w, ws)
    for name in reef.ACTIVATIONS:
        check(reef.gemm_w8a8(xq, xs, w, ws, activation=name), plain, name)


def test_epilogue_flags_overflow(reef):
    print("\n[case] product overflow", flush=True)
    xq, xs, w, ws, bias, res = problem(20, 32, 50)
    res[3, 49] = float("inf")
    with pytest.raises(reef.Overflow):
        reef.gemm_w8a8(xq, xs, w, ws, bias, residual=res)
    bias[7] = -float("inf")  # relu would hide it
    with pytest.raises(reef.Overflow):
        reef.gemm_w8a8(xq, xs, w, ws, bias, activation="relu")
    bias[7] = float("nan")
    with pytest.raises(reef.Overflow):
        reef.gemm_w8a8(xq, xs, w, ws, bias, activation="relu")


def test_epilogue_in_a_graph(reef):
    """Norm, product with activation, quantize, product onto the residual: captured once,
    replayed between eager runs, every replay equal to the eager result."""
    print("\n[case] graph of a sublayer", flush=True)
    g = torch.Generator(device="cuda").manual_seed(21)
    x, r = (torch.randn((24, 256), generator=g, device="cuda") for _ in range(2))
    _, _, w1, s1, b1, _ = problem(24, 256, 640)
    _, _, w2, s2, b2, _ = problem(24, 640, 256)
    status = reef.StatusWord()

    def step():
        q, s, h = reef.rmsnorm_quantize(x, residual=r, status=status)
        up = reef.gemm_w8a8(q, s, w1, s1, b1, status, activation="gelu_tanh")
        return reef.linear_w8a8(up, w2, s2, b2, status, residual=h)

    eager = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(step(), eager)
    status.check("graph")

"""The root-mean-square norm with int8 rows against its formula in 64 bits: the residual
sum exact (one fp32 addition), each scale within half a step of fp32, each code equal
wherever the 64-bit quotient is not within 1e-9 of a half (the kernel's own 64-bit steps
are off by less than 1e-12 at 127). Each case prints its name before touching the GPU."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


def expected(h, w, eps):
    """Codes as float64 quotients, and scales, of fp32 rows h."""
    d = h.astype(np.float64)
    y = d if w is None else d * w.astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(y == 0, 0.0, y / np.sqrt((d * d).mean(1, keepdims=True) + eps))
    scale = (np.abs(y).max(1, keepdims=True) / 127).astype(np.float32)
    scale[scale == 0] = 1
    return y / scale.astype(np.float64), scale[:, 0]


def check(q, s, h, w, eps):
    quotient, scale = expected(h, w, eps)
    q, s = q.cpu().numpy().astype(np.float64), s.cpu().numpy()
    assert (np.abs(s.astype(np.float64) - scale) <= np.spacing(scale)).all()  # a tie of the rounding
    sure = np.abs(np.abs(quotient - np.floor(quotient)) - 0.5) > 1e-9
    rows = s == scale
    assert rows.mean() > 0.99
    assert (np.clip(np.rint(quotient), -127, 127) == q)[rows[:, None] & sure].all()
    assert (np.abs(quotient[rows] - q[rows]) <= 0.5 + 1e-4).all()


WIDTHS = [1, 3, 4, 63, 64, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2500, 4096, 4097,
          5003, 8192, 8193, 16384, 16385, 40001]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("residual,weight", [(True, True), (False, False)])
def test_norm_matches_formula(reef, width, residual, weight):
    rows = 9 if width > 5000 else 37
    print(f"\n[case] norm {rows}x{width} residual {residual} weight {weight}", flush=True)
    rng = np.random.default_rng(width)
    x = rng.standard_normal((rows, width)).astype(np.float32)
    r = (3 * rng.standard_normal((rows, width))).astype(np.float32) if residual else None
    w = rng.uniform(-2, 2, width).astype(np.float32) if weight else None
    t = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    out = reef.rmsnorm_quantize(t(x), t(w), residual=t(r), eps=1e-5)
    h = x if r is None else x + r
    if residual:
        assert np.array_equal(out[2].cpu().numpy().view(np.uint32), h.view(np.uint32))
    else:
        assert len(out) == 2
    check(out[0], out[1], h, w, 1e-5)


@pytest.mark.parametrize("rows,width", [(2050, 700), (2049, 2047), (3001, 1024), (9000, 8190)])
def test_norm_of_many_rows(reef, rows, width):
    """A wave per row, and streams beyond the last-level cache (9000 x 8190 with a residual)."""
    print(f"\n[case] norm of many rows {rows}x{width}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, r = (torch.randn((rows, width), generator=g, device="cuda") for _ in range(2))
    w = torch.rand(width, generator=g, device="cuda") + 0.5
    q, s, h = reef.rmsnorm_quantize(x, w, residual=r)
    assert torch.equal(h, x + r)
    some = torch.cat([torch.arange(40), torch.arange(rows - 40, rows)])
    check(q[some], s[some], h[some].cpu().numpy(), w.cpu().numpy(), 1e-6)
    d = h.double()  # the others on the GPU
    y = d * w.double() / (d.square().mean(1, keepdim=True) + 1e-6).sqrt()
    assert float((q.double() * s[:, None].double() - y).abs().max() / s.max()) < 0.5 + 1e-4


@pytest.mark.parametrize("width", [100, 2048, 6001, 20000])
@pytest.mark.parametrize("alias", ["x", "residual"])
def test_norm_in_place_and_strided(reef, width, alias):
    """The sum written over x or over the residual; rows a stride apart and off 16 bytes."""
    print(f"\n[case] norm in place over {alias}, width {width}", flush=True)
    rng = np.random.default_rng(width + 1)
    x = rng.standard_normal((2, 5, width)).astype(np.float32)
    r = rng.standard_normal((2, 5, width)).astype(np.float32)
    tx, tr = torch.from_numpy(x).cuda(), torch.from_numpy(r).cuda()
    q, s, h = reef.rmsnorm_quantize(tx, residual=tr, residual_out=tx if alias == "x" else tr)
    assert h is (tx if alias == "x" else tr) and q.shape == x.shape and s.shape == x.shape[:-1]
    assert np.array_equal(h.cpu().numpy(), x + r)
    other = tr.cpu().numpy() if alias == "x" else tx.cpu().numpy()
    assert np.array_equal(other, r if alias == "x" else x)
    check(q.view(10, -1), s.view(-1), (x + r).reshape(10, -1), None, 1e-6)
    wide = torch.zeros(7, width + 13, device="cuda")
    wide[:, 5:5 + width] = torch.from_numpy(x.reshape(10, -1)[:7]).cuda()
    q2, s2 = reef.rmsnorm_quantize(wide[:, 5:5 + width])
    check(q2, s2, x.reshape(10, -1)[:7], None, 1e-6)
    assert float(wide[:, :5].abs().sum() + wide[:, 5 + width:].abs().sum()) == 0


def test_norm_rows_of_zeros_and_extremes(reef):
    print("\n[case] norm zeros, tiny, huge, one value, ties", flush=True)
    x = np.zeros((8, 96), np.float32)
    x[1] = 1e-38                      # squares below fp32
    x[2] = 3e38                       # squares beyond fp32
    x[3, 17] = -2.5
    x[4, :] = np.arange(96) - 48
    x[5, 0] = 1e-45                   # the smallest subnormal
    x[6, ::2] = 1e30
    x[6, 1::2] = 1e-30
    x[7] = -1.0
    for eps in (0.0, 1e-6):
        q, s = reef.rmsnorm_quantize(torch.from_numpy(x).cuda(), eps=eps)
        check(q, s, x, None, eps)
        assert (q[0] == 0).all() and float(s[0]) == 1.0
    # a sum that cancels to 0 has the scale of a zero row
    t = torch.from_numpy(x[4:5].copy()).cuda()
    q, s, h = reef.rmsnorm_quantize(t, residual=-t)
    assert not q.any() and float(s) == 1.0 and not h.any()


def test_norm_rows_past_the_last_are_left(reef):
    """Narrow rows share a workgroup: the rows of the last one that do not exist write nothing."""
    for rows, width in ((1, 64), (5, 256), (6, 300)):
        print(f"\n[case] norm rows {rows} of {width}", flush=True)
        import ctypes as C
        x = torch.randn(rows, width, device="cuda")
        q = torch.full((rows + 4, width), 55, dtype=torch.int8, device="cuda")
        s = torch.full((rows + 4,), 7.0, device="cuda")
        st = reef.lib().reef_rmsnorm_quantize_int8(
            C.c_void_p(x.data_ptr()), rows, width, width, None, 0, None, 1e-6,
            C.c_void_p(q.data_ptr()), C.c_void_p(s.data_ptr()), None, 0, None,
            C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == reef.OK
        assert (q[rows:] == 55).all() and (s[rows:] == 7).all()
        check(q[:rows], s[:rows], x.cpu().numpy(), None, 1e-6)


def test_norm_flags_what_is_not_finite(reef):
    print("\n[case] norm non-finite", flush=True)
    for value in (float("inf"), float("nan"), -float("inf")):
        for width in (40, 3000, 20000):
            x = torch.randn(3, width, device="cuda")
            x[1, width - 1] = value
            with pytest.raises(reef.NonFiniteInput):
                reef.rmsnorm_quantize(x)
    x = torch.randn(3, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    w[3] = float("nan")
    with pytest.raises(reef.NonFiniteInput):
        reef.rmsnorm_quantize(x, w)
    big = torch.full((1, 64), 3e38, device="cuda")
    with pytest.raises(reef.NonFiniteInput):
        reef.rmsnorm_quantize(big, residual=big)
    # one value in a row of n has y = sqrt(n) weight: sqrt(65536) * 3.3e38 / 127 > 3.41e38
    one = torch.zeros(1, 65536, device="cuda")
    one[0, 5] = 1.0
    with pytest.raises(reef.Overflow):
        reef.rmsnorm_quantize(one, torch.full((65536,), 3.3e38, device="cuda"), eps=0.0)


def test_norm_feeds_the_product(reef):
    """rmsnorm_quantize's rows into gemm_w8a8: the same as the product of their values."""
    print("\n[case] norm -> product", flush=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(33, 512, generator=g, device="cuda") for _ in range(2))
    w = torch.randint(-127, 128, (96, 512), generator=g, device="cuda").to(torch.int8)
    ws = torch.rand(96, generator=g, device="cuda") / 1000
    q, s, h = reef.rmsnorm_quantize(x, residual=r)
    y = reef.gemm_w8a8(q, s, w, ws)
    acc = q.double() @ w.double().t()
    ref = acc.float() * (s[:, None] * ws[None, :])
    assert torch.equal(y, ref)


def test_more_rows_than_a_launch_has_threads(reef):
    """Rows past 2^32 / 64 and past the first row of workgroups: each is done."""
    rows = (1 << 26) + 5
    print(f"\n[case] norm of {rows} rows of 1", flush=True)
    x = torch.full((rows, 1), 3.0, device="cuda")
    x[::2] = -0.5
    q, s = reef.rmsnorm_quantize(x, eps=0.0)
    sign = torch.sign(x)
    assert torch.equal(q, (127 * sign).to(torch.int8))
    one = float(np.float32(1 / 127))
    assert bool((s == one).all())

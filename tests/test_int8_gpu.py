"""Products in 8-bit integers against the definition: codes and scales bit by bit, sums in 64 bits."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
U32, U16 = 2.0**-24, 2.0**-8  # half an ulp of float32 and of bfloat16


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def plain_quantise(x):
    """The definition in numpy: every step rounded once in float32."""
    x = x.float().cpu().numpy()
    s = np.abs(x).max(1).astype(np.float32) * np.float32(1 / 127)
    with np.errstate(all="ignore"):
        c = np.clip(np.rint(x / s[:, None]), -127, 127)
    c = np.where((s > 0)[:, None], c, 0)
    bad = ~np.isfinite(x).all(1)
    s[bad], c[bad] = np.nan, 0
    return torch.from_numpy(c.astype(np.int8)), torch.from_numpy(s)


def rows(m, k, dtype, seed=0, stride=None, offset=0):
    """Rows of numbers with a few large channels, inside a buffer of another row stride."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * (1 + 15 * (torch.rand(k, generator=g) < 0.02).float())
    flat = torch.full((m * (stride or k) + offset,), 7.0, dtype=dtype, device=DEV)
    view = torch.as_strided(flat, (m, k), (stride or k, 1), offset)
    view.copy_(x)
    return view


def codes(n, k, seed=1):
    from tokasaurus_b200.kernels import int8

    g = torch.Generator().manual_seed(seed)
    w = int8.lay_out_codes(torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(DEV))
    return w, (torch.rand(n, generator=g) * 0.01 + 1e-4).to(DEV)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k,stride,offset", [(1, 1, None, 0), (1, 2048, None, 0), (3, 7, 9, 1), (5, 1001, None, 0), (2, 1001, 1003, 3),
                                               (17, 8192, None, 0), (4, 8192, 8200, 8), (64, 4096, 6144, 0), (2, 33000, None, 0), (300, 64, None, 0)])
def test_rows_are_brought_to_codes_as_defined(dtype, m, k, stride, offset):
    from tokasaurus_b200.kernels import int8

    x = rows(m, k, dtype, seed=m + k, stride=stride, offset=offset)
    got, scale = int8.quantise_rows(x)
    want, want_scale = plain_quantise(x)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_halves_zeros_and_extremes(dtype):
    """Quotients that are exact halves go to the even code; zero rows, the smallest and the largest numbers, infinities and NaN."""
    from tokasaurus_b200.kernels import int8

    tiny = 2.0**-133 if dtype == BF else 2.0**-149
    x = torch.zeros(9, 40)
    x[0, :20] = torch.arange(20) * 0.5 + 0.5
    x[0, 20] = 127.0
    x[1, ::2], x[1, 1] = 1.5, 3.0           # halves of the largest
    x[3, :3] = torch.tensor([tiny, -tiny, 0])  # a scale that rounds to zero
    x[4, :3] = torch.tensor([2.0**-120, -(2.0**-126), 2.0**-127])
    x[5, :3] = torch.tensor([3.3e38, -3.3e38, 1.0])
    x[6, :2] = torch.tensor([float("inf"), 1.0])
    x[7, :2] = torch.tensor([float("nan"), 1.0])
    x[8, :4] = torch.tensor([190 * tiny, 100 * tiny, -190 * tiny, tiny])
    x = x.to(dtype).to(DEV)
    got, scale = int8.quantise_rows(x)
    want, want_scale = plain_quantise(x)
    assert torch.equal(got.cpu(), want)
    assert np.array_equal(scale.cpu().numpy(), want_scale.numpy(), equal_nan=True)


SIZES = [(1, 16, 16), (1, 2048, 16384), (2, 64, 509), (7, 1001, 130), (8, 8192, 2048), (16, 500, 96), (17, 130, 300), (33, 4096, 640),
         (64, 2048, 1000), (65, 256, 127), (100, 77, 33), (127, 640, 512), (128, 128, 128), (200, 1500, 257), (333, 1001, 509),
         (500, 2048, 2048), (1030, 511, 1040)]


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_product(m, k, n, out):
    from tokasaurus_b200.kernels import int8

    x = rows(m, k, BF if (m + k) % 2 else F32, seed=m)
    w, t = codes(n, k, seed=n)
    st = status()
    y = int8.linear_int8(x, w, t, st, out_dtype=out)
    c, s = plain_quantise(x)
    want = (c.to(DEV).double() @ w.double().t()) * s.to(DEV).double()[:, None] * t.double()
    # the sum is exact; its conversion, the scales' product and the product with it are rounded once each, then the result
    bound = want.abs() * (3.01 * U32 + (U16 if out == BF else 0)) + 2.0**-126
    assert y.dtype == out and ((y.double() - want).abs() <= bound).all() and int(st) == 0


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("m,k,n", [(1, 64, 16), (1, 2048, 16384), (5, 1001, 48), (8, 512, 1040), (16, 640, 2048), (40, 2048, 512), (64, 96, 272),
                                   (65, 130, 304), (200, 512, 1056), (513, 2048, 2064)])
def test_gated_product(m, k, n, out):
    from tokasaurus_b200.kernels import int8, ops

    x = rows(m, k, BF, seed=m + 1)
    gate, tg = codes(n // 2, k, seed=n)
    up, tu = codes(n // 2, k, seed=n + 1)
    tg, tu = tg / k**0.5, tu / k**0.5
    w = int8.lay_out_codes(ops.interleave_gate_up(gate, up))
    t = ops.interleave_gate_up(tg[:, None], tu[:, None])[:, 0].contiguous()
    st = status()
    y = int8.linear_int8(x, w, t, st, gated=True, out_dtype=out).double()
    c, s = plain_quantise(x)
    c, s = c.to(DEV).double(), s.to(DEV).double()[:, None]
    g, u = (c @ gate.double().t()) * s * tg.double(), (c @ up.double().t()) * s * tu.double()
    want = g * torch.sigmoid(g) * u
    # g and u are off by 3 roundings; e^-g by |g| times that of g's and of log2 e's, and 2 ulp; the quotient by 2 ulp
    bound = want.abs() * ((6 * g.abs() + 24) * U32 + (U16 if out == BF else 0)) + 2.0**-120
    live = g.abs() < 80  # beyond, e^-g leaves float32 on the one side, and g is the result on the other
    assert ((y - want).abs() <= torch.where(live, bound, 1e-30 + want.abs() * (U16 + 12 * U32))).all() and int(st) == 0


def test_longest_sums_and_full_range_weights():
    """The longest rows of the largest codes reach 2^31 less a few: no sum wraps."""
    from tokasaurus_b200.kernels import int8

    k = int8.MAX_K
    x = torch.ones(2, k, dtype=BF, device=DEV)
    x[1] = -1
    w = int8.lay_out_codes(torch.full((3, k), -128, dtype=torch.int8, device=DEV))
    t = torch.ones(3, device=DEV)
    y = int8.linear_int8(x, w, t, status(), out_dtype=F32).double().cpu()
    want = 127 * 128 * k * float(np.float32(1) * np.float32(1 / 127))
    assert ((y - torch.tensor([[-want] * 3, [want] * 3])).abs() <= want * 4 * U32).all()


@pytest.mark.parametrize("m", [3, 40, 200])
def test_a_row_that_is_no_number_stays_alone(m):
    from tokasaurus_b200.kernels import int8

    x = rows(m, 256, BF, seed=3).clone()
    w, t = codes(96, 256)
    clean = int8.linear_int8(x, w, t, status())
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    t2 = t.clone()
    t2[4] = float("nan")
    y = int8.linear_int8(x, w, t2, status())
    assert y[1:3].isnan().all() and y[:, 4].isnan().all()
    keep = torch.ones(96, dtype=torch.bool)
    keep[4] = False
    assert torch.equal(y[0, keep], clean[0, keep]) and torch.equal(y[3:][:, keep], clean[3:][:, keep])


def test_strided_rows_empty_steps_and_another_stream():
    from tokasaurus_b200.kernels import int8

    w, t = codes(512, 320)
    x = rows(70, 320, BF, stride=328)
    want = int8.linear_int8(x.contiguous(), w, t, status())
    assert torch.equal(int8.linear_int8(x, w, t, status()), want)
    wide = torch.zeros(512, 1024, dtype=torch.int8, device=DEV)
    wide[:, 64:384] = w
    assert torch.equal(int8.linear_int8(x, wide[:, 64:384], t, status()), want)
    assert torch.equal(int8.linear_int8(x[3:4].expand(70, 320), w, t, status()), want[3:4].expand(70, 512))
    assert int8.linear_int8(x[:0], w, t, status()).shape == (0, 512)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8.linear_int8(x, w, t, status())
    side.synchronize()
    assert torch.equal(got, want)


def test_same_result_however_many_rows_a_call_has():
    """Sums are exact, so a token's result has the same bits alone, among few and among many."""
    from tokasaurus_b200.kernels import int8

    x = rows(300, 2048, BF, seed=9)
    w, t = codes(528, 2048)
    whole = int8.linear_int8(x, w, t, status(), out_dtype=F32)
    for lo, hi in ((0, 1), (1, 9), (9, 26), (26, 90), (90, 300)):
        assert torch.equal(int8.linear_int8(x[lo:hi], w, t, status(), out_dtype=F32), whole[lo:hi])


def test_refusals():
    from tokasaurus_b200.kernels import int8
    from tokasaurus_b200.kernels.ops import KernelError

    x, (w, t), st = rows(4, 64, BF), codes(32, 64), status()
    for bad in (lambda: int8.linear_int8(x.half(), w, t, st), lambda: int8.linear_int8(x.cpu(), w, t, st),
                lambda: int8.linear_int8(x[:, :60], w, t, st), lambda: int8.linear_int8(x.t(), w[:, :4], t, st),
                lambda: int8.linear_int8(x, w.short(), t, st), lambda: int8.linear_int8(x, w, t[:31], st),
                lambda: int8.linear_int8(x, w, t.double(), st), lambda: int8.linear_int8(x, w, t, st, out_dtype=torch.float16),
                lambda: int8.linear_int8(x[:, :60], w[:, :60].contiguous(), t, st), lambda: int8.linear_int8(x[:, 1:], w[:, 1:], t, st),
                lambda: int8.linear_int8(x, w[:24], t[:24], st, gated=True), lambda: int8.linear_int8(x[:, :0], w[:, :0], t, st),
                lambda: int8.product_int8(torch.zeros(1, 132112, dtype=torch.int8, device=DEV), t[:1].contiguous(),
                                          torch.zeros(1, 132112, dtype=torch.int8, device=DEV), t[:1].contiguous(), st)):
        with pytest.raises(KernelError):
            bad()


@pytest.mark.parametrize("m,k,n,gated", [(3, 14336, 256, False), (20, 8192, 130, False), (40, 4096, 128, True), (100, 14336, 512, False), (129, 2048, 640, True),
                                         (130, 8192, 2048, False), (200, 4096, 1040, True), (256, 4096, 6144, False), (300, 8192, 96, False), (700, 1000, 272, True)])
def test_tiles_of_tokens_and_parts_of_k(m, k, n, gated):
    """Sizes at which tokens come in one tile or several and K in one part or up to eight: each result as its rows alone give it, and
    some of them against the definition."""
    from tokasaurus_b200.kernels import int8

    x = rows(m, k, BF, seed=m + n)
    w, t = codes(n, k, seed=k)
    t = t / k**0.5
    st = status()
    y = int8.linear_int8(x, w, t, st, gated=gated, out_dtype=F32)
    c, s = plain_quantise(x)
    z = (c.to(DEV).double() @ w.double().t()) * s.to(DEV).double()[:, None] * t.double()
    if gated:
        z = z.view(m, n // 16, 2, 8)
        g, u = z[:, :, 0].reshape(m, -1), z[:, :, 1].reshape(m, -1)
        want = g * torch.sigmoid(g) * u
        bound = want.abs() * (6 * g.abs() + 24) * U32 + 2.0**-120
        bound = torch.where(g.abs() < 80, bound, 1e-30 + want.abs() * 12 * U32)
    else:
        want = z
        bound = want.abs() * 3.01 * U32 + 2.0**-126
    assert ((y.double() - want).abs() <= bound).all() and int(st) == 0
    for lo, hi in ((0, 1), (m // 2, m // 2 + 9), (max(0, m - 70), m)):
        assert torch.equal(int8.linear_int8(x[lo:hi], w, t, st, gated=gated, out_dtype=F32), y[lo:hi])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_weights_made_right_before(m):
    """Nothing stands between the kernel that makes the weights' codes and the product that reads them."""
    from tokasaurus_b200.kernels import int8

    st = status()
    xs = [rows(m, 1024, BF, seed=i) for i in range(8)]
    ws = [rows(768, 1024, BF, seed=20 + i) for i in range(8)]
    made = [int8.quantise_rows(w) for w in ws]
    torch.cuda.synchronize()
    want = [int8.linear_int8(x, *cw, st) for x, cw in zip(xs, made)]
    torch.cuda.synchronize()
    got = []
    for x, w in zip(xs, ws):
        got.append((int8.linear_int8(x, *int8.quantise_rows(w), st), int8.product_int8(*int8.quantise_rows(x), *int8.quantise_rows(w), st)))
    for a, (b, c) in zip(want, got):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert int(st) == 0


def test_products_in_a_graph():
    """Replays of a captured step with other tokens in place."""
    from tokasaurus_b200.kernels import int8

    st = status()
    x, (w, t) = rows(9, 2048, BF), codes(512, 2048)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        int8.linear_int8(x, w, t, st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int8.linear_int8(x, w, t, st)
        z = int8.linear_int8(y, w[:, :512], t, st)
    for seed in range(3):
        x.copy_(rows(9, 2048, BF, seed=100 + seed))
        graph.replay()
        a = int8.linear_int8(x, w, t, st)
        assert torch.equal(y, a) and torch.equal(z, int8.linear_int8(a, w[:, :512], t, st))
    assert int(st) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_numbers_next_to_a_half_code(dtype):
    """Quotients within a few units of a half integer, on either side and on it, under scales of every size."""
    from tokasaurus_b200.kernels import int8

    g = np.random.default_rng(5)
    rows_ = []
    for i in range(300):
        top = np.float32(np.exp(g.uniform(-85, 85)))
        if dtype == BF:
            top = np.float32(torch.tensor(float(top)).to(BF).float())
        s = top * np.float32(1 / 127)
        x = ((g.integers(-126, 127, 512) + 0.5) * np.float64(s)).astype(np.float32)
        x = (x.view(np.int32) + g.integers(-2, 3, 512).astype(np.int32)).view(np.float32)
        x[7] = top
        rows_.append(x)
    x = torch.from_numpy(np.stack(rows_)).to(dtype).to(DEV)
    got, scale = int8.quantise_rows(x)
    want, want_scale = plain_quantise(x)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("m,k,n,gated", [(1, 2048, 49152, False), (2, 2048, 24576, True), (1, 4096, 16384, False), (3, 512, 2048, False), (8, 1024, 4096, False),
                                         (1, 8192, 8192, False), (1, 4096, 28672, True), (5, 16, 40, False), (4, 2064, 304, True), (1, 8176, 333, False)])
def test_few_tokens_past_matrices_of_many_shapes(m, k, n, gated):
    """Slices and rounds of the one-launch product, and the sizes from which on it is two: the codes' exact sums either way."""
    from tokasaurus_b200.kernels import int8

    x = rows(m, k, BF, seed=m + k)
    w, t = codes(n, k, seed=n)
    t = t / k**0.5
    st = status()
    y = int8.linear_int8(x, w, t, st, gated=gated, out_dtype=F32)
    c, s = int8.quantise_rows(x)
    assert torch.equal(int8.product_int8(c, s, w, t, st, gated=gated, out_dtype=F32), y) and int(st) == 0
    sums = torch.cat([(c.double() @ part.double().t()) for part in w.split(4096)], 1)
    z = sums * s.double()[:, None] * t.double()
    if not gated:
        assert ((y.double() - z).abs() <= z.abs() * 3.01 * U32 + 2.0**-126).all()

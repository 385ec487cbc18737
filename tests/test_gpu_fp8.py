"""The 8-bit operators on the GPU against their definition in 64 bits (tests/fp8_ref.py).

Tolerances, derived: quantising is exact (the same codes and exponents). In the linear layer the
products of two e4m3 values are exact in 32 bits, so an element is off by the additions alone. Each
of at most K + 2 additions is off by at most one step of a partial sum, 2^-23 of it, and a partial sum
is at most S = sum |x w| + |bias| + |residual|: |error| <= (K + 4) 2^-23 S for any order. Over a whole
result the rounded partial sums have the size of the result, and an accumulator takes 32 products at a
time: norm(error) <= 4 (K / 32 + 8) 2^-23 norm(sqrt(x^2 w^2 sums)). GELU has slope at most 1.13 and is
evaluated to 2^-20. A bf16 result adds half a step, 2^-8 |y| at most, an e4m3 one 2^-4 |y| or half of
its smallest step, 2^-10 of a scale that is at most amax / 224."""
import numpy as np
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def hard_rows(rng, rows, k):
    """Rows of very different sizes, with blocks of zeros, exact ties and values at the scale's border."""
    x = rng.standard_normal((rows, k)) * np.exp(rng.uniform(-30, 30, (rows, 1)))
    x[rows // 2] = 0.0
    x[rows // 3] = rng.integers(-64, 65, k) * 0.5  # ties of the 4-bit grid
    x[-1] = np.where(rng.random(k) < 0.5, 448.0, rng.integers(-448, 449, k))
    x[0, : k // 2] *= 1e-8
    return x.astype(np.float32)


def bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def check_store(q, code, E):
    got = bits(q.values)
    nan = (code & 127) == 127
    assert np.array_equal((got & 127) == 127, nan)
    assert np.array_equal(got[~nan], code[~nan])
    assert np.array_equal(q.exps.cpu().numpy(), E)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, k, pad, off", [(1, 1, 0, 0), (1, 768, 0, 0), (3, 127, 0, 0), (5, 128, 1, 0), (130, 129, 3, 1),
                                               (257, 514, 2, 0), (64, 2048, 8, 0), (128, 256, 0, 3), (9, 1000, 4, 2)])
def test_quantize_and_read_back(kk, block_rows, dtype, rows, k, pad, off):
    rng = np.random.default_rng(rows * 1000 + k)
    buf = torch.zeros(rows * (k + pad) + off + 4, device="cuda", dtype=dtype)
    x = buf[off:off + rows * (k + pad)].view(rows, k + pad)[:, :k]  # strided, at any offset of its elements
    x.copy_(torch.from_numpy(hard_rows(rng, rows, k)))
    x64 = x.double().cpu().numpy()
    code, E = ref.quantize(x64, block_rows)
    q = kk.fp8.quantize(x, block_rows=block_rows)
    check_store(q, code, E)
    assert np.array_equal(x.double().cpu().numpy(), x64)
    back = ref.dequantize(code, E, block_rows)
    got = kk.fp8.dequantize(q)
    assert got.dtype == torch.float32 and np.array_equal(got.double().cpu().numpy(), back.astype(np.float32).astype(np.float64))
    b16 = kk.fp8.dequantize(q, torch.bfloat16)
    assert torch.equal(b16, torch.from_numpy(back.astype(np.float32)).to(torch.bfloat16).cuda())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_infinities_and_nan(kk, block_rows):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((140, 300)).astype(np.float32)
    x[0, 3], x[1, 130], x[2, 299], x[139, 0] = np.inf, -np.inf, np.nan, np.nan
    x[4, :128] = np.nan  # nothing finite in the block
    x[5, 128:256] = np.inf
    code, E = ref.quantize(x.astype(np.float64), block_rows)
    q = kk.fp8.quantize(torch.from_numpy(x).cuda(), block_rows=block_rows)
    check_store(q, code, E)
    back = kk.fp8.dequantize(q).cpu().numpy()
    assert np.array_equal(np.isnan(back), ~np.isfinite(x))


def test_quantize_ends_of_the_range(kk):
    x = np.zeros((6, 128), np.float32)
    x[0, :4] = [3.4e38, -1e30, 1e25, 0]
    x[1, :4] = [1e-45, -1e-42, 0, 0]
    x[2, :2] = [2.0 ** -118, 2.0 ** -126]
    x[3, :3] = [448 * 2.0 ** -127, 2.0 ** -127, 2.0 ** -136]
    x[4, :2] = [-0.0, 0.0]
    x[5, :2] = [np.nextafter(np.float32(448), np.float32(500)), 1]
    code, E = ref.quantize(x.astype(np.float64))
    q = kk.fp8.quantize(torch.from_numpy(x).cuda())
    check_store(q, code, E)


def test_store_is_written_within_its_rows_and_columns(kk):
    fp8 = kk.fp8
    vals = torch.full((40, 320), 0x55, device="cuda", dtype=torch.uint8)
    exps = torch.full((40, 8), 0x66, device="cuda", dtype=torch.uint8)
    store = fp8.Fp8Tensor(vals.view(E4M3)[:, :300], exps[:, :3])
    x = torch.randn(7, 300, device="cuda")
    fp8.quantize(x, out=store[11:18])
    code, E = ref.quantize(x.double().cpu().numpy())
    check_store(store[11:18], code, E)
    v, e = vals.cpu().numpy(), exps.cpu().numpy()
    assert (v[:11] == 0x55).all() and (v[18:] == 0x55).all() and (v[:, 300:] == 0x55).all()
    assert (e[:11] == 0x66).all() and (e[18:] == 0x66).all() and (e[:, 3:] == 0x66).all()


def make(rng, m, n, k, fp8, wild=False):
    x = rng.standard_normal((m, k))
    if wild:
        x *= np.exp(rng.uniform(-8, 8, (m, 1)))
        x[:, : min(k, 128)] *= (rng.random((m, 1)) < 0.7)  # some rows' first block is all zeros
    w = rng.uniform(-1, 1, (n, k)) / np.sqrt(k)
    xq = fp8.quantize(torch.from_numpy(x.astype(np.float32)).cuda())
    wq = fp8.quantize(torch.from_numpy(w.astype(np.float32)).cuda(), block_rows=128)
    xd = ref.dequantize(bits(xq.values), xq.exps.cpu().numpy())
    wd = ref.dequantize(bits(wq.values), wq.exps.cpu().numpy(), 128)
    return xq, wq, xd, wd


def check_linear(got, y, S, rms, K, act, dtype):
    """got against y: element by element, and as a whole (32-bit results)."""
    tol = (K + 4) * 2.0 ** -23 * S * (1.13 if act else 1.0) + (2.0 ** -20 * np.abs(y) if act else 0.0)
    if dtype == E4M3:
        back = ref.dequantize(bits(got.values), got.exps.cpu().numpy())
        n = y.shape[1]
        amax = np.stack([np.abs(y[:, b:b + 128]).max(1) for b in range(0, n, 128)], 1)
        amax = np.repeat(amax, 128, 1)[:, :n]
        tol = tol * 1.07 + 2.0 ** -4 * np.abs(y) + 2.0 ** -10 * amax * (1 + 1e-3) / 224 + 1e-300
        err = np.abs(back - y)
    else:
        g = got.double().cpu().numpy()
        err = np.abs(g - y)
        if dtype == torch.bfloat16:
            tol = tol * 1.01 + 2.0 ** -8 * np.abs(y)
        else:
            tol = tol + 2.0 ** -24 * np.abs(y)
            whole = 4 * (K / 32 + 8) * 2.0 ** -23 * (1.13 if act else 1.0) + 2.0 ** -20 * (act is not None) + 2.0 ** -23
            assert np.linalg.norm(g - y) <= whole * np.linalg.norm(rms)
    bad = np.argwhere(~(err <= tol))
    assert len(bad) == 0, (len(bad), bad[:5].tolist(), err.max())


SIZES = [(1, 1, 1), (1, 16, 128), (1, 768, 768), (2, 130, 100), (7, 128, 129), (16, 2304, 768), (17, 50, 512), (33, 257, 300),
         (64, 512, 768), (65, 96, 640), (66, 2048, 768), (128, 768, 2048), (129, 255, 16), (200, 1090, 514), (300, 769, 1100),
         (512, 768, 2048), (700, 640, 520), (4800, 1000, 384), (9501, 513, 640), (2600, 2304, 768),
         (3, 20000, 4700), (140, 1000, 2500), (4800, 1000, 1700), (5003, 1157, 2100), (4900, 1024, 1030), (40000, 1, 130),
         (20000, 300, 33)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, E4M3])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_linear(kk, m, n, k, dtype):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    fp8 = kk.fp8
    xq, wq, xd, wd = make(rng, m, n, k, fp8, wild=True)
    bias = rng.standard_normal(n).astype(np.float32) * 0.1
    bias_d = torch.from_numpy(bias).cuda()
    res = None if dtype == E4M3 else torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32)).cuda().to(dtype)
    for act, r, b in ((None, None, bias_d), ("gelu", None, bias_d), (None, res, bias_d), ("gelu", res, None)):
        y, S = ref.linear(xd, wd, None if b is None else bias, act, None if r is None else r.double().cpu().numpy())
        got = fp8.linear(xq, wq, b, act=act, residual=r, out_dtype=dtype)
        rms = np.sqrt((xd ** 2) @ (wd ** 2).T + y ** 2)
        check_linear(got, y, S, rms, k, act, dtype)


def test_linear_nan_reaches_its_row_only(kk):
    rng = np.random.default_rng(3)
    for m in (5, 200):
        x = rng.standard_normal((m, 300)).astype(np.float32)
        x[3, 140] = np.inf
        w = torch.from_numpy(rng.standard_normal((150, 300)).astype(np.float32)).cuda()
        y = kk.fp8.linear(kk.fp8.quantize(torch.from_numpy(x).cuda()), kk.fp8.quantize(w, block_rows=128))
        assert y[3].isnan().all() and not y[:3].isnan().any() and not y[4:].isnan().any()


@pytest.mark.parametrize("m, n, k", [(5, 300, 256), (700, 640, 520), (4800, 1000, 300), (4800, 1000, 1700)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear_nan_column(kk, m, n, k, act):
    """A NaN or an infinity in one column's bias, or in a weight, stays in that column."""
    rng = np.random.default_rng(11)
    fp8 = kk.fp8
    x = fp8.quantize(torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).cuda())
    w = (rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    w[17, 3] = np.nan
    w = fp8.quantize(torch.from_numpy(w).cuda(), block_rows=128)
    bias = torch.zeros(n, device="cuda")
    bias[130], bias[131], bias[n - 1] = float("nan"), float("inf"), float("-inf")
    res = torch.ones(m, n, device="cuda")
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[[17, 130, 131, n - 1]] = False
    for dtype in (torch.float32, torch.bfloat16, E4M3):
        for r in (None, res) if dtype != E4M3 else (None,):
            y = fp8.linear(x, w, bias, act=act, out_dtype=dtype, residual=None if r is None else r.to(dtype))
            y = fp8.dequantize(y) if dtype == E4M3 else y.float()
            assert y[:, fine].isfinite().all()
            assert y[:, [17, 130]].isnan().all()
            assert (y[:, 131].isnan() if dtype == E4M3 else y[:, 131] == float("inf")).all()


@pytest.mark.parametrize("m, n", [(3, 128), (300, 256), (5000, 1024)])
def test_gelu_over_its_range(kk, m, n):
    """GELU of given values, through a layer whose product is zero: |error| <= 2^-20 |y| + 2^-27 (values below -5.6
    count as -5.6, 2.7e-9) in 32 bits."""
    rng = np.random.default_rng(m)
    bias = np.concatenate([np.linspace(-12, 12, n - 8), [0.0, 1e-30, -1e-30, 30.0, -30.0, 1e4, -1e4, 3e38]]).astype(np.float32)
    bias[:-8] = rng.permutation(bias[:-8])
    x = kk.fp8.quantize(torch.zeros(m, 128, device="cuda"))
    w = kk.fp8.quantize(torch.zeros(n, 128, device="cuda"), block_rows=128)
    got = kk.fp8.linear(x, w, torch.from_numpy(bias).cuda(), act="gelu").double().cpu().numpy()
    with np.errstate(over="ignore"):
        want = ref.gelu(bias.astype(np.float64))
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want) + 2.0 ** -27).all(), np.abs(got - want).max(0)


def test_linear_far_apart_scales(kk):
    """Rows of zeros, of 1e-30 and of 1e30 in one tile: each keeps its own relative accuracy."""
    rng = np.random.default_rng(4)
    for m in (6, 140):
        x = rng.standard_normal((m, 256))
        x[0], x[1], x[2] = 0.0, x[1] * 1e-30, x[2] * 1e30
        w = rng.standard_normal((200, 256)).astype(np.float32)
        w[:128] *= 1e-4
        xq = kk.fp8.quantize(torch.from_numpy(x.astype(np.float32)).cuda())
        wq = kk.fp8.quantize(torch.from_numpy(w).cuda(), block_rows=128)
        xd = ref.dequantize(bits(xq.values), xq.exps.cpu().numpy())
        wd = ref.dequantize(bits(wq.values), wq.exps.cpu().numpy(), 128)
        y, S = ref.linear(xd, wd)
        got = kk.fp8.linear(xq, wq).double().cpu().numpy()
        assert (np.abs(got - y) <= (256 + 4) * 2.0 ** -23 * S).all()


@pytest.mark.parametrize("m, n, k", [(1, 130, 200), (20, 300, 514), (150, 300, 514), (4900, 1010, 200), (4900, 1010, 1700)])
@pytest.mark.parametrize("ldy_pad, off", [(1, 0), (2, 1), (4, 4), (8, 0), (0, 3), (6, 0), (4, 0)])
def test_linear_any_strides_and_offsets(kk, m, n, k, ldy_pad, off):
    """Result and residual rows at strides and offsets of every alignment; nothing is written beside them."""
    rng = np.random.default_rng(m + n + ldy_pad)
    fp8 = kk.fp8
    xq, wq, xd, wd = make(rng, m, n, k, fp8)
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.full((off + (m + 2) * (n + ldy_pad),), 7.0, device="cuda", dtype=dtype)
        y = buf[off:off + m * (n + ldy_pad)].view(m, n + ldy_pad)[:, :n]
        rbuf = torch.randn(off + m * (n + ldy_pad + 1), device="cuda").to(dtype)
        r = rbuf[off:].view(m, n + ldy_pad + 1)[:, :n]
        got = fp8.linear(xq, wq, residual=r, out_dtype=dtype, out=y)
        assert got.data_ptr() == y.data_ptr()
        want, S = ref.linear(xd, wd, residual=r.double().cpu().numpy())
        check_linear(y, want, S, np.sqrt((xd ** 2) @ (wd ** 2).T + want ** 2), k, None, dtype)
        rest = buf.clone()
        rest[off:off + m * (n + ldy_pad)].view(m, n + ldy_pad)[:, :n] = 7.0
        assert (rest == 7.0).all()


def test_linear_onto_its_residual(kk):
    rng = np.random.default_rng(8)
    for m in (3, 300):
        xq, wq, xd, wd = make(rng, m, 768, 256, kk.fp8)
        y = torch.randn(m, 768, device="cuda")
        want = kk.fp8.linear(xq, wq, residual=y.clone())
        kk.fp8.linear(xq, wq, residual=y, out=y)
        assert torch.equal(y, want)


def test_linear_result_store_within_a_larger_one(kk):
    rng = np.random.default_rng(9)
    fp8 = kk.fp8
    for m in (5, 140):
        xq, wq, xd, wd = make(rng, m, 300, 256, fp8)
        vals = torch.full((m + 6, 336), 0x55, device="cuda", dtype=torch.uint8)
        exps = torch.full((m + 6, 4), 0x66, device="cuda", dtype=torch.uint8)
        store = fp8.Fp8Tensor(vals.view(E4M3)[:, :300], exps[:, :3])
        fp8.linear(xq, wq, out_dtype=E4M3, out=store[2:m + 2])
        want = fp8.linear(xq, wq, out_dtype=E4M3)
        assert np.array_equal(bits(store[2:m + 2].values), bits(want.values))
        assert torch.equal(store[2:m + 2].exps, want.exps)
        v, e = vals.cpu().numpy(), exps.cpu().numpy()
        assert (v[:2] == 0x55).all() and (v[m + 2:] == 0x55).all() and (v[:, 300:] == 0x55).all()
        assert (e[:2] == 0x66).all() and (e[m + 2:] == 0x66).all() and (e[:, 3:] == 0x66).all()


@pytest.mark.parametrize("m, n, k", [(3, 768, 2048), (700, 768, 2048), (5000, 1024, 768)])
def test_linear_twice_the_same(kk, m, n, k):
    """Same inputs, same bits (shares of K are added in their order)."""
    rng = np.random.default_rng(10)
    xq, wq, _, _ = make(rng, m, n, k, kk.fp8)
    r = torch.randn(m, n, device="cuda")
    for res in (None, r):
        a, b = kk.fp8.linear(xq, wq, residual=res), kk.fp8.linear(xq, wq, residual=res)
        assert torch.equal(a, b)


def feed_forward(fp8, x, w1, b1, w2, b2, residual):
    h = fp8.linear(fp8.quantize(x), w1, b1, act="gelu", out_dtype=E4M3)
    return fp8.linear(h, w2, b2, residual=residual)


@pytest.mark.parametrize("m", [1, 66, 513])
def test_feed_forward_block(kk, m):
    """The operators as they are used together; the middle store may round an element to the neighbouring
    code where 32 and 64 bits fall on two sides of a border: at most one step of 2^-3 for each such element."""
    rng = np.random.default_rng(m)
    fp8 = kk.fp8
    x = torch.from_numpy(rng.standard_normal((m, 768)).astype(np.float32)).cuda()
    W = [(rng.uniform(-1, 1, s) / np.sqrt(s[1])).astype(np.float32) for s in ((2048, 768), (768, 2048))]
    B = [(rng.uniform(-1, 1, s) * 0.03).astype(np.float32) for s in (2048, 768)]
    w1, w2 = (fp8.quantize(torch.from_numpy(w).cuda(), block_rows=128) for w in W)
    b1, b2 = (torch.from_numpy(b).cuda() for b in B)
    got = feed_forward(fp8, x, w1, b1, w2, b2, x).double().cpu().numpy()
    d1, d2 = (ref.dequantize(bits(w.values), w.exps.cpu().numpy(), 128) for w in (w1, w2))
    x64 = x.double().cpu().numpy()
    h, S = ref.linear(ref.dequantize(*ref.quantize(x64)), d1, B[0], "gelu")
    hd = ref.dequantize(*ref.quantize(h))
    y, S2 = ref.linear(hd, d2, B[1], None, x64)
    # elements whose 32-bit value may lie across a border: within the layer's tolerance of a border
    tol = (768 + 4) * 2.0 ** -23 * S * 1.13 + 2.0 ** -20 * np.abs(h)
    step = np.maximum(2.0 ** -3 * np.abs(hd), 2.0 ** -9 * np.abs(h).max() / 224)
    near = np.abs(np.abs(h - hd) - step / 2) <= tol + step / 4  # generous: a quarter of a step around each border
    slack = (near * step * 1.5) @ np.abs(d2).T
    assert (np.abs(got - y) <= (2048 + 4) * 2.0 ** -23 * S2 + slack + 2.0 ** -24 * np.abs(y)).all()
    assert np.linalg.norm(got - y) <= 2e-3 * np.linalg.norm(y - x64)


def test_streams_and_graphs(kk):
    fp8 = kk.fp8
    torch.manual_seed(0)
    x = torch.randn(300, 768, device="cuda")
    w1, w2 = (fp8.quantize(torch.randn(s, device="cuda") / 30, block_rows=128) for s in ((2048, 768), (768, 2048)))
    b1, b2 = torch.randn(2048, device="cuda"), torch.randn(768, device="cuda")
    want = feed_forward(fp8, x, w1, b1, w2, b2, x)
    want_small = feed_forward(fp8, x[:5], w1, b1, w2, b2, x[:5])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i, s in enumerate(streams * 3):  # calls at once on several streams
        with torch.cuda.stream(s):
            n = 5 if i % 2 else 300
            got.append((n, feed_forward(fp8, x[:n], w1, b1, w2, b2, x[:n])))
    torch.cuda.synchronize()
    for n, y in got:
        assert torch.equal(y, want if n == 300 else want_small)
    # two captured graphs of the same operators, replayed on new inputs, at once on two streams
    xs = [x.clone(), x.clone()]
    graphs, outs = [], []
    for xi in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(feed_forward(fp8, xi, w1, b1, w2, b2, xi))
        graphs.append(g)
    x2 = torch.randn(300, 768, device="cuda")
    xs[1].copy_(x2)
    want2 = feed_forward(fp8, x2, w1, b1, w2, b2, x2)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_gpu_refusals(kk):
    fp8 = kk.fp8
    x = fp8.quantize(torch.randn(4, 256, device="cuda"))
    w = fp8.quantize(torch.randn(130, 256, device="cuda"), block_rows=128)

    def refused(f, *a, **k):
        with pytest.raises(kk.KokoroError) as e:
            f(*a, **k)
        assert e.value.status == kk.engine.KK_ERR_INVALID_ARG
        return str(e.value)

    assert "block_rows 128" in refused(fp8.linear, x, x)
    assert "block_rows 1 " in refused(fp8.linear, w, w)
    w3 = fp8.quantize(torch.randn(130, 128, device="cuda"), block_rows=128)
    assert "columns" in refused(fp8.linear, x, w3)
    assert "act" in refused(fp8.linear, x, w, act="relu")
    assert "bias" in refused(fp8.linear, x, w, torch.zeros(131, device="cuda"))
    assert "bias" in refused(fp8.linear, x, w, torch.zeros(130, device="cuda", dtype=torch.bfloat16))
    assert "one device" in refused(fp8.linear, x, w, torch.zeros(130))
    assert "residual" in refused(fp8.linear, x, w, residual=torch.zeros(4, 129, device="cuda"))
    assert "residual" in refused(fp8.linear, x, w, residual=torch.zeros(4, 130, device="cuda", dtype=torch.bfloat16))
    assert "no residual" in refused(fp8.linear, x, w, residual=torch.zeros(4, 130, device="cuda"), out_dtype=E4M3)
    assert "out_dtype" in refused(fp8.linear, x, w, out_dtype=torch.float16)
    assert "out" in refused(fp8.linear, x, w, out=torch.zeros(4, 131, device="cuda"))
    assert "out" in refused(fp8.linear, x, w, out=torch.zeros(4, 130, device="cuda"), out_dtype=torch.bfloat16)
    assert "gradient" in refused(fp8.quantize, torch.zeros(4, 128, device="cuda", requires_grad=True))
    assert "dtype" in refused(fp8.dequantize, x, torch.float16)
    assert "block_rows" in refused(fp8.quantize, torch.zeros(4, 128, device="cuda"), block_rows=64)
    assert "slice" in refused(w.__getitem__, slice(0, 1))
    assert "exps" in refused(fp8.Fp8Tensor, x.values, x.exps[:3])
    v = torch.zeros(4, 100, device="cuda", dtype=torch.uint8).view(E4M3)  # rows 100 bytes apart
    assert "16 bytes" in refused(fp8.dequantize, fp8.Fp8Tensor(v, torch.zeros(4, 4, device="cuda", dtype=torch.uint8)[:, :1]))
    with torch.no_grad():
        fp8.quantize(torch.zeros(4, 128, device="cuda", requires_grad=True))


def test_no_rows(kk):
    fp8 = kk.fp8
    q = fp8.quantize(torch.empty(0, 256, device="cuda"))
    w = fp8.quantize(torch.randn(130, 256, device="cuda"), block_rows=128)
    assert fp8.linear(q, w).shape == (0, 130)
    assert fp8.linear(q, w, out_dtype=E4M3).shape == (0, 130)
    assert fp8.dequantize(q).shape == (0, 256)


def test_no_wait_has_expired(kk):
    kk.fp8.check()
    kk.fp8.check("cuda:0")


FIRST_CALL_IN_A_CAPTURE = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import conftest
fp8 = conftest.import_package().fp8
x, w = torch.randn(300, 768, device="cuda"), torch.randn(2048, 768, device="cuda") / 30
b = torch.randn(2048, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    wq = fp8.quantize(w, block_rows=128)
    y = fp8.dequantize(fp8.linear(fp8.quantize(x), wq, b, act="gelu", out_dtype=torch.float8_e4m3fn))
x.copy_(torch.randn(300, 768, device="cuda"))
g.replay()
want = fp8.dequantize(fp8.linear(fp8.quantize(x), fp8.quantize(w, 128), b, act="gelu", out_dtype=torch.float8_e4m3fn))
assert torch.equal(y, want)
fp8.check()
print("fine")
"""


def test_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE, os.path.dirname(os.path.abspath(__file__))],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_calls_of_several_host_threads_at_once(kk):
    import threading
    fp8 = kk.fp8
    torch.manual_seed(1)
    x = torch.randn(2000, 768, device="cuda")
    w1, w2 = (fp8.quantize(torch.randn(s, device="cuda") / 30, block_rows=128) for s in ((2048, 768), (768, 2048)))
    b1, b2 = torch.randn(2048, device="cuda"), torch.randn(768, device="cuda")
    sizes = (1, 40, 300, 2000)
    want = [feed_forward(fp8, x[:n], w1, b1, w2, b2, x[:n]) for n in sizes]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    n = sizes[i]
                    y = feed_forward(fp8, x[:n], w1, b1, w2, b2, x[:n])
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, want[i]):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    fp8.check()


@pytest.mark.parametrize("m, n, k", [(5, 130, 200), (700, 640, 520), (4800, 1000, 300)])
def test_what_lies_behind_a_row_is_not_read(kk, m, n, k):
    """Values behind column k that are NaN, and scales behind the last block that are NaN, change nothing."""
    rng = np.random.default_rng(13)
    fp8 = kk.fp8
    xq, wq, _, _ = make(rng, m, n, k, fp8)
    want = fp8.linear(xq, wq)

    def within(q):
        rows, kb = q.shape[0], q.exps.shape[1]
        ldv, lde = -(-k // 16) * 16 + 32, -(-kb // 4) * 4 + 4
        v = torch.full((rows + 3, ldv), 0x7F, device="cuda", dtype=torch.uint8)
        e = torch.full((q.exps.shape[0] + 3, lde), 0xFF, device="cuda", dtype=torch.uint8)
        v[:rows, :k] = q.values.view(torch.uint8)
        e[: q.exps.shape[0], :kb] = q.exps
        return fp8.Fp8Tensor(v.view(E4M3)[:rows, :k], e[: q.exps.shape[0], :kb], q.block_rows)

    x2, w2 = within(xq), within(wq)
    assert torch.equal(fp8.linear(x2, w2), want)
    assert torch.equal(fp8.linear(x2, w2, out_dtype=torch.bfloat16), fp8.linear(xq, wq, out_dtype=torch.bfloat16))
    a, b = fp8.linear(x2, w2, out_dtype=E4M3), fp8.linear(xq, wq, out_dtype=E4M3)
    assert np.array_equal(bits(a.values), bits(b.values)) and torch.equal(a.exps, b.exps)
    assert torch.equal(fp8.dequantize(x2), fp8.dequantize(xq)) and torch.equal(fp8.dequantize(w2), fp8.dequantize(wq))


@pytest.fixture
def much_memory():
    """For tests that hold tens of GB: what they leave cached goes back, for the engines of the tests after them."""
    yield
    torch.cuda.empty_cache()


def test_offsets_past_32_bits(kk, much_memory):
    """Rows that begin past 2^31 elements and 2^32 bytes: the last ones equal those of a small call."""
    fp8 = kk.fp8
    torch.manual_seed(14)
    # Two orders of adding 128 products, whose magnitudes add up to 130 at most here, differ by 2 * 128 * 2^-24 * 130.
    tol = 2.0 * 128 * 2.0 ** -24 * 130
    rows, k = 20000, 120000  # 2.4e9 elements
    x = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, k, device="cuda")
    q = fp8.quantize(x)
    small = fp8.quantize(x[-3:].clone())
    assert torch.equal(q[rows - 3:].values.view(torch.uint8), small.values.view(torch.uint8))
    assert torch.equal(q[rows - 3:].exps, small.exps)
    x.fill_(1.0)
    fp8.dequantize(q, torch.bfloat16, out=x)
    assert torch.equal(x[-3:], fp8.dequantize(small, torch.bfloat16)) and (x[:-3] == 0).all()
    del x, q
    m, n = 300000, 8192  # 2.5e9 results
    xq = fp8.quantize(torch.randn(m, 128, device="cuda"))
    wq = fp8.quantize(torch.randn(n, 128, device="cuda"), block_rows=128)
    res = torch.zeros(m, n, device="cuda")
    res[-5:] = 1.0
    want = fp8.linear(xq[m - 5:], wq)
    y = fp8.linear(xq, wq)
    assert torch.allclose(y[-5:], want, rtol=0, atol=tol)
    fp8.linear(xq, wq, residual=res, out=res)
    assert torch.allclose(res[-5:], want + 1.0, rtol=0, atol=tol) and torch.allclose(res[:1000], y[:1000], rtol=0, atol=tol)
    del res
    h = fp8.linear(xq, wq, out_dtype=E4M3)
    tail = fp8.dequantize(h[m - 5:])
    assert ((tail - want).abs() <= 2.0 ** -4 * want.abs() + want.abs().amax() * 2.0 ** -10 / 224 + tol).all()


def test_check_inside_a_capture_is_refused(kk):
    """...and leaves the capture as it was."""
    fp8 = kk.fp8
    rng = np.random.default_rng(15)
    xq, wq, _, _ = make(rng, 200, 256, 256, fp8)
    want = fp8.linear(xq, wq)
    y = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fp8.linear(xq, wq, out=y)
        with pytest.raises(kk.KokoroError):
            fp8.check()
        fp8.linear(xq, wq, out=y)
    g.replay()
    fp8.check()
    assert torch.equal(y, want)


@pytest.mark.parametrize("m, n, k", [(1, 1, (1 << 30) - 3), (3, 130, (1 << 28) + 200)])
def test_longest_rows(kk, much_memory, m, n, k):
    """The whole sum of the longest rows waits for one CTA's (or one cluster's) loads."""
    fp8 = kk.fp8
    rng = np.random.default_rng(16)
    at = np.unique(np.concatenate([rng.integers(0, k, 60), [0, k - 1]]))
    xv, wv = fp8.Fp8Tensor.empty(m, k), fp8.Fp8Tensor.empty(n, k, 128)
    for q in (xv, wv):
        q._buf.zero_()
        q.exps.fill_(127)
    # powers of two at some columns: sums of at most 62 products 2^-4 .. 2^4 are exact in 24 bits
    x = 2.0 ** rng.integers(-2, 3, (m, len(at))) * rng.choice((-1, 1), (m, len(at)))
    w = 2.0 ** rng.integers(-2, 3, (n, len(at))) * rng.choice((-1, 1), (n, len(at)))
    idx = torch.tensor(at, device="cuda")
    xv.values.view(torch.uint8)[:, idx] = torch.tensor(x, device="cuda", dtype=torch.float32).to(E4M3).view(torch.uint8)
    wv.values.view(torch.uint8)[:, idx] = torch.tensor(w, device="cuda", dtype=torch.float32).to(E4M3).view(torch.uint8)
    y = fp8.linear(xv, wv)
    fp8.check()
    assert np.array_equal(y.cpu().numpy(), (x @ w.T).astype(np.float32))


def test_most_rows(kk, much_memory):
    """2^31 - 1 rows, the most a call takes: the quantiser's, the read-back's and the layer's row indices."""
    fp8 = kk.fp8
    rows = (1 << 31) - 1
    at = torch.tensor([0, 1, (1 << 30) - 1, 1 << 30, rows - 2, rows - 1], device="cuda")
    vals = torch.tensor([1.0, -2.0, 3.0, 0.5, -7.0, 448.0], device="cuda")[:, None]
    x = torch.zeros(rows, 1, device="cuda")
    x[at] = vals
    q = fp8.quantize(x)
    x.fill_(5.0)
    fp8.dequantize(q, out=x)
    assert torch.equal(x[at], vals) and torch.count_nonzero(x).item() == len(at)
    w = fp8.quantize(torch.full((1, 1), 2.0, device="cuda"), block_rows=128)
    x.fill_(5.0)
    fp8.linear(q, w, out=x)
    fp8.check()
    assert torch.equal(x[at], 2.0 * vals) and torch.count_nonzero(x).item() == len(at)


@pytest.mark.parametrize("m, n, k", [(4900, 1010, 200), (4867, 1037, 300), (4900, 1024, 140)])
@pytest.mark.parametrize("ldy_pad, off", [(1, 0), (2, 1), (4, 4), (8, 0), (0, 3), (6, 0), (2, 0), (0, 0)])
def test_linear_any_strides_without_residual(kk, m, n, k, ldy_pad, off):
    """The same for the kernel without a residual, and a residual that is the result itself against one that is not."""
    rng = np.random.default_rng(m + n + ldy_pad + 1)
    fp8 = kk.fp8
    xq, wq, xd, wd = make(rng, m, n, k, fp8)
    want, S = ref.linear(xd, wd)
    rms = np.sqrt((xd ** 2) @ (wd ** 2).T + want ** 2)
    for dtype in (torch.float32, torch.bfloat16):
        def view(buf):
            return buf[off:off + m * (n + ldy_pad)].view(m, n + ldy_pad)[:, :n]

        buf = torch.full((off + (m + 2) * (n + ldy_pad),), 7.0, device="cuda", dtype=dtype)
        y = view(buf)
        fp8.linear(xq, wq, out_dtype=dtype, out=y)
        check_linear(y, want, S, rms, k, None, dtype)
        r = torch.randn(m, n, device="cuda").to(dtype)
        other = fp8.linear(xq, wq, residual=r, out_dtype=dtype)
        y.copy_(r)
        fp8.linear(xq, wq, residual=y, out_dtype=dtype, out=y)
        assert torch.equal(y, other)
        view(buf).fill_(7.0)
        assert (buf == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, k", [(1, 1), (3, 3), (5, 130), (40, 255), (9, 1027), (6000, 770), (300, 16301)])
def test_read_back_into_any_rows(kk, dtype, rows, k):
    """Rows at every offset and stride from a 16-byte boundary; nothing is written beside them."""
    rng = np.random.default_rng(rows + k)
    x = torch.from_numpy(rng.standard_normal((rows, k)).astype(np.float32)).cuda()
    for block_rows in (1, 128):
        q = kk.fp8.quantize(x, block_rows=block_rows)
        want = torch.from_numpy(ref.dequantize(bits(q.values), q.exps.cpu().numpy(), block_rows).astype(np.float32)).cuda().to(dtype)
        for pad, off in ((0, 0), (1, 0), (2, 1), (3, 3), (4, 5), (5, 2), (6, 7), (7, 4), (8, 6)):
            buf = torch.full((off + rows * (k + pad) + 9,), 7.0, device="cuda", dtype=dtype)
            y = buf[off:off + rows * (k + pad)].view(rows, k + pad)[:, :k]
            kk.fp8.dequantize(q, dtype, out=y)
            assert torch.equal(y, want)
            y.fill_(7.0)
            assert (buf == 7.0).all()


@pytest.mark.parametrize("rows, k, block_rows", [(1, 5, 1), (130, 300, 1), (130, 300, 128)])
def test_copies_of_a_store_have_memory_of_their_own(kk, rows, k, block_rows):
    import copy
    import io
    fp8 = kk.fp8
    x = torch.randn(rows, k, device="cuda")
    q = fp8.quantize(x, block_rows=block_rows)
    want = fp8.dequantize(q)
    file = io.BytesIO()
    torch.save(q, file)
    copies = [copy.deepcopy(q), copy.deepcopy(fp8.Fp8Tensor(q.values, q.exps, block_rows))]
    if block_rows == 1:
        copies.append(copy.deepcopy(q[0:rows]))
    file.seek(0)
    copies.append(torch.load(file, weights_only=False))
    fp8.quantize(torch.zeros_like(x), block_rows=block_rows, out=q)
    del q
    torch.cuda.empty_cache()
    for c in copies:
        assert c.shape == (rows, k) and c.block_rows == block_rows
        assert torch.equal(fp8.dequantize(c), want)
        fp8.quantize(2 * x, block_rows=block_rows, out=c)
        assert torch.equal(fp8.dequantize(c), 2 * want)


def test_a_store_keeps_the_memory_it_was_made_over(kk):
    fp8 = kk.fp8
    q = fp8.quantize(torch.randn(64, 256, device="cuda"))
    want = fp8.dequantize(q)
    v, e = q.values.clone(), torch.zeros(64, 4, device="cuda", dtype=torch.uint8)[:, :2]  # (rows 4 bytes apart)
    e.copy_(q.exps)
    s = fp8.Fp8Tensor(v, e)
    v.set_(torch.empty(0, 0, device="cuda", dtype=E4M3))
    e.set_(torch.empty(0, 0, device="cuda", dtype=torch.uint8))
    torch.cuda.empty_cache()
    assert torch.equal(fp8.dequantize(s), want)


@pytest.mark.parametrize("m, n, k", [(5, 300, 256), (700, 640, 520), (4800, 1000, 300), (4800, 1000, 1700)])
def test_gelu_of_minus_infinity(kk, m, n, k):
    """-inf (1 + tanh(-inf)) / 2 is NaN: in its columns only, the first and the last among them, in every result type and
    kernel, and without GELU it is minus infinity."""
    rng = np.random.default_rng(21)
    fp8 = kk.fp8
    xq, wq, xd, wd = make(rng, m, n, k, fp8)
    bias = torch.randn(n, device="cuda")
    cols = [0, 7, 8, 200, n - 1]
    bias[cols] = float("-inf")
    res = torch.ones(m, n, device="cuda")
    other = torch.ones(n, dtype=torch.bool, device="cuda")
    other[cols] = False
    for dtype in (torch.float32, torch.bfloat16, E4M3):
        for r in (None, res) if dtype != E4M3 else (None,):
            for act in ("gelu", None):
                y = fp8.linear(xq, wq, bias, act=act, out_dtype=dtype, residual=None if r is None else r.to(dtype))
                y = fp8.dequantize(y) if dtype == E4M3 else y.float()
                assert y[:, other].isfinite().all()
                assert (y[:, cols].isnan() if act or dtype == E4M3 else y[:, cols] == float("-inf")).all()


def test_forward_mode_tangents_are_refused(kk):
    """In every argument of a layer."""
    from torch.autograd import forward_ad
    fp8 = kk.fp8
    x = fp8.quantize(torch.randn(4, 256, device="cuda"))
    w = fp8.quantize(torch.randn(130, 256, device="cuda"), block_rows=128)
    b, y = torch.zeros(130, device="cuda"), torch.zeros(4, 130, device="cuda")
    want = fp8.linear(x, w, b, residual=y)
    with forward_ad.dual_level():
        db, dy = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (b, y))
        for kw in (dict(bias=db), dict(residual=dy), dict(out=dy)):
            with pytest.raises(kk.KokoroError, match="forward mode"):
                fp8.linear(x, w, **kw)
        with pytest.raises(kk.KokoroError, match="forward mode"):
            fp8.dequantize(fp8.quantize(y), out=dy)
        assert torch.equal(fp8.linear(x, w, b, residual=y), want)


def test_negation_still_to_be_done_is_refused(kk):
    """In every argument of a layer of one column, where the imaginary part of a conjugate has adjacent columns."""
    fp8 = kk.fp8
    x = fp8.quantize(torch.randn(4, 256, device="cuda"))
    w = fp8.quantize(torch.randn(1, 256, device="cuda"), block_rows=128)
    y = torch.randn(4, 1, dtype=torch.complex64, device="cuda").conj().imag
    b = torch.randn(1, dtype=torch.complex64, device="cuda").conj().imag
    assert y.is_neg() and b.is_neg()
    for kw in (dict(bias=b), dict(residual=y), dict(out=y)):
        with pytest.raises(kk.KokoroError, match="resolve_neg"):
            fp8.linear(x, w, **kw)
    for f in (lambda: fp8.quantize(y), lambda: fp8.dequantize(fp8.quantize(y.resolve_neg()), out=y)):
        with pytest.raises(kk.KokoroError, match="resolve_neg"):
            f()
    assert torch.equal(fp8.linear(x, w, b.resolve_neg(), residual=y.resolve_neg()),
                       fp8.linear(x, w, b.resolve_neg().clone(), residual=y.contiguous().resolve_neg().clone()))


def expired(kk):
    """Whether a check reports an expired wait."""
    try:
        kk.fp8.check()
        return False
    except kk.KokoroError as e:
        assert e.status == kk.engine.KK_ERR_TIMEOUT and "wait" in str(e)
        return True


@pytest.mark.parametrize("cluster", [False, True])
def test_an_expired_wait_is_reported_once(kk, cluster):
    """5 us on a barrier that nothing arrives on; the layers after it are as right as those before."""
    rng = np.random.default_rng(22)
    fp8 = kk.fp8
    layers = [make(rng, m, 256, 256, fp8)[:2] for m in (5, 6000)]
    want = [fp8.linear(*l) for l in layers]
    assert not expired(kk)
    fp8.wait_selftest(cluster=cluster)
    assert expired(kk)
    assert not expired(kk)
    for l, y in zip(layers, want):
        assert torch.equal(fp8.linear(*l), y)
    assert not expired(kk)


def test_no_check_takes_an_expired_wait_from_another(kk):
    """One of stream a is reported on stream b and to another thread, whoever checks first, once to each."""
    import threading
    fp8 = kk.fp8
    a, b = torch.cuda.Stream(), torch.cuda.Stream()

    def on(stream):
        with torch.cuda.stream(stream):
            return expired(kk)

    def elsewhere(f):
        got = []
        t = threading.Thread(target=lambda: got.append(f()))
        t.start()
        t.join()
        return got[0]

    for s in (a, b):
        on(s)  # (a stream's first check tells of what other tests left)
    assert not on(a) and not on(b)
    for first, second in ((a, b), (b, a)):
        with torch.cuda.stream(a):
            fp8.wait_selftest()
        a.synchronize()
        assert on(first) and on(second)
        assert not on(first) and not on(second)
        assert elsewhere(lambda: (on(a), on(a))) == (True, False)  # (this thread's first check)
        assert not on(a) and not on(b)
    # a failure between another stream's failure and its check
    with torch.cuda.stream(a):
        fp8.wait_selftest()
    with torch.cuda.stream(b):
        fp8.wait_selftest(cluster=True)
        b.synchronize()
    assert on(a) and on(b) and not on(a) and not on(b)
    expired(kk)  # (the current stream's own, for the tests after this one)
    assert not expired(kk)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_top_of_the_range_read_back(kk, block_rows):
    """From 248 * 2^120 on (a tie, to the even code) a value is held as 256 * 2^120 = 2^128: infinite where it is read
    back, a factor like any other in a layer."""
    fp8 = kk.fp8
    border = np.float32(248 * 2.0 ** 120)
    x = np.zeros((5, 128), np.float32)
    x[:, 0] = [border, np.nextafter(border, np.float32(0)), np.finfo(np.float32).max, -border, 232 * 2.0 ** 120]
    # (a tie of its own; -border, the maximum and the border share the block's scale when block_rows is 128)
    code, E = ref.quantize(x.astype(np.float64), block_rows)
    q = fp8.quantize(torch.from_numpy(x).cuda(), block_rows=block_rows)
    check_store(q, code, E)
    held = ref.dequantize(code, E, block_rows)
    assert held[0, 0] == 2.0 ** 128 and held[1, 0] == 240 * 2.0 ** 120 and held[4, 0] == 224 * 2.0 ** 120
    for dtype in (torch.float32, torch.bfloat16):
        got = fp8.dequantize(q, dtype).double().cpu().numpy()
        want = np.where(np.abs(held) >= 2.0 ** 128, np.copysign(np.inf, held), held)
        assert np.array_equal(got, want)
    w = torch.zeros(3, 128, device="cuda")
    w[:, 0] = torch.tensor([2.0 ** -3, -3 * 2.0 ** -20, 2.0 ** -100])
    if block_rows == 1:
        y = fp8.linear(q, fp8.quantize(w, block_rows=128)).double().cpu().numpy()
        # 2^-100 is below the smallest step at the scale of the block's 2^-3: it is held as 0
        assert np.array_equal(y, held[:, :1] * np.array([[2.0 ** -3, -3 * 2.0 ** -20, 0.0]]))


@pytest.mark.parametrize("m", [1, 66, 513, 5000])
def test_feed_forward_block_by_its_middle_store(kk, m):
    """The block's two layers each against the definition, the second on the codes that the first left: every element of
    both within its own layer's bound."""
    rng = np.random.default_rng(m + 1)
    fp8 = kk.fp8
    x = torch.from_numpy(rng.standard_normal((m, 768)).astype(np.float32)).cuda()
    W = [(rng.uniform(-1, 1, s) / np.sqrt(s[1])).astype(np.float32) for s in ((2048, 768), (768, 2048))]
    B = [(rng.uniform(-1, 1, s) * 0.03).astype(np.float32) for s in (2048, 768)]
    w1, w2 = (fp8.quantize(torch.from_numpy(w).cuda(), block_rows=128) for w in W)
    b1, b2 = (torch.from_numpy(b).cuda() for b in B)
    d1, d2 = (ref.dequantize(bits(w.values), w.exps.cpu().numpy(), 128) for w in (w1, w2))
    xq = fp8.quantize(x)
    xd = ref.dequantize(bits(xq.values), xq.exps.cpu().numpy())
    h = fp8.linear(xq, w1, b1, act="gelu", out_dtype=E4M3)
    want, S = ref.linear(xd, d1, B[0], "gelu")
    check_linear(h, want, S, None, 768, "gelu", E4M3)
    hd = ref.dequantize(bits(h.values), h.exps.cpu().numpy())
    for dtype in (torch.float32, torch.bfloat16):
        r = x.to(dtype)
        y, S2 = ref.linear(hd, d2, B[1], None, r.double().cpu().numpy())
        rms = np.sqrt((hd ** 2) @ (d2 ** 2).T + y ** 2)
        got = fp8.linear(h, w2, b2, residual=r, out_dtype=dtype)
        check_linear(got, y, S2, rms, 2048, None, dtype)
        if dtype == torch.float32:
            assert torch.equal(got, feed_forward(fp8, x, w1, b1, w2, b2, x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("m, n, k", [(66, 2048, 768), (700, 640, 520), (4800, 1000, 384), (5003, 1157, 2100), (2600, 2304, 768)])
def test_rounded_results_as_a_whole(kk, m, n, k, dtype):
    """The norm of what rounding leaves, beside check_linear's bound on each element. A value falls anywhere between two
    neighbours, so its rounding error has 1 / sqrt(3) of the most it can be (root mean square): 2^-8 |y| in bf16, 2^-4 |y| or
    half of the smallest step in e4m3, four standard deviations of the mean of N squares (each at most 1 where their mean
    is 1/3) above that; and the additions' part as for 32-bit results."""
    rng = np.random.default_rng(m + n + k)
    fp8 = kk.fp8
    xq, wq, xd, wd = make(rng, m, n, k, fp8)
    bias = rng.standard_normal(n).astype(np.float32) * 0.1
    res = torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32)).cuda().to(dtype) if dtype != E4M3 else None
    for act, r in ((None, None), ("gelu", None), (None, res), ("gelu", res)) if dtype != E4M3 else ((None, None), ("gelu", None)):
        y, S = ref.linear(xd, wd, bias, act, None if r is None else r.double().cpu().numpy())
        got = fp8.linear(xq, wq, torch.from_numpy(bias).cuda(), act=act, residual=r, out_dtype=dtype)
        if dtype == E4M3:
            g = ref.dequantize(bits(got.values), got.exps.cpu().numpy())
            amax = np.stack([np.abs(y[:, b:b + 128]).max(1) for b in range(0, n, 128)], 1)
            most = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 / 224 * np.repeat(amax, 128, 1)[:, :n])
        else:
            g, most = got.double().cpu().numpy(), 2.0 ** -8 * np.abs(y)
        rms = np.sqrt((xd ** 2) @ (wd ** 2).T + y ** 2)
        added = 4 * (k / 32 + 8) * 2.0 ** -23 * (1.13 if act else 1.0) + 2.0 ** -20 * (act is not None)
        rounded = np.sqrt((1 / 3 + 4 * 0.5 / np.sqrt(y.size)) * (most ** 2).sum())
        assert np.linalg.norm(g - y) <= added * np.linalg.norm(rms) + rounded


@pytest.mark.parametrize("dtype", [torch.float32, E4M3])
def test_short_kernels_of_pairs_in_a_row(kk, dtype):
    """One block of K and a tile or two a pair, hundreds of times in a row on two streams: blocks that begin in the shared
    memory of blocks that just ended."""
    rng = np.random.default_rng(23)
    fp8 = kk.fp8
    xq, wq, _, _ = make(rng, 25000, 300, 100, fp8)
    res = torch.randn(25000, 300, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(r):
        y = fp8.linear(xq, wq, residual=r if dtype != E4M3 else None, out_dtype=dtype)
        return y.values.view(torch.uint8) if dtype == E4M3 else y

    for r in (None, res):
        want = call(r)
        wrong = [torch.zeros((), device="cuda", dtype=torch.int64) for _ in streams]
        torch.cuda.synchronize()
        for _ in range(200):
            for s, bad in zip(streams, wrong):
                with torch.cuda.stream(s):
                    bad += (call(r) != want).sum()
        torch.cuda.synchronize()
        assert not any(bad.item() for bad in wrong)
    fp8.check()


def test_an_earlier_failure_is_not_this_calls(kk):
    """A call that the library refused with a CUDA error, on this thread, before each of the operators."""
    import ctypes
    fp8, lib = kk.fp8, kk.load_library()
    x = torch.randn(6000, 768, device="cuda")
    w = fp8.quantize(torch.randn(768, 768, device="cuda"), block_rows=128)
    n, buf = np.array([1], np.int32), np.zeros(2304, np.float32)

    def fail():
        assert lib.kk_attention_selftest(99, 1, n.ctypes.data_as(ctypes.c_void_p), buf.ctypes.data_as(ctypes.c_void_p),
                                         buf.ctypes.data_as(ctypes.c_void_p)) == kk.engine.KK_ERR_CUDA

    fail()
    q = fp8.quantize(x)
    fail()
    fp8.linear(q, w)
    fail()
    fp8.linear(q[:5], w, residual=x[:5])
    fail()
    assert torch.equal(fp8.dequantize(q), fp8.dequantize(q))
    fail()
    fp8.check()


def test_results_over_what_a_backward_pass_saved(kk):
    """A tensor that autograd keeps for its backward pass and that is then given as `out`: the backward pass says so."""
    fp8 = kk.fp8
    x = fp8.quantize(torch.randn(4, 256, device="cuda"))
    w = fp8.quantize(torch.randn(256, 256, device="cuda"), block_rows=128)
    for f in (lambda y: fp8.linear(x, w, out=y), lambda y: fp8.linear(x, w, residual=y, out=y), lambda y: fp8.dequantize(x, out=y)):
        a = torch.randn(4, 256, device="cuda", requires_grad=True)
        y = torch.randn(4, 256, device="cuda")
        z = (a * y).sum()
        f(y)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    with torch.inference_mode():
        y = torch.empty(4, 256, device="cuda")
        assert torch.equal(fp8.linear(x, w, out=y), fp8.linear(x, w))


FIRST_LARGE_CALLS_IN_A_CAPTURE = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import conftest
fp8 = conftest.import_package().fp8
E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16
m, n, k = 5000, 1040, 520
x, w = torch.randn(m, k, device="cuda"), torch.randn(n, k, device="cuda") / 25
b, r = torch.randn(n, device="cuda"), torch.randn(m, n, device="cuda")

def layers(y):
    xq, wq = fp8.quantize(x), fp8.quantize(w, 128)
    fp8.linear(xq, wq, b, residual=y, out=y)
    return [y, fp8.linear(xq, wq, b), fp8.linear(xq, wq, b, out_dtype=BF16),
            fp8.linear(xq, wq, b, residual=r.to(BF16), out_dtype=BF16),
            fp8.dequantize(fp8.linear(xq, wq, b, act="gelu", out_dtype=E4M3), BF16)]

y = r.clone()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = layers(y)
for seed in (1, 2):
    torch.manual_seed(seed)
    x.copy_(torch.randn(m, k, device="cuda"))
    y.copy_(r)
    g.replay()
    want = layers(r.clone())
    assert all(torch.equal(a, c) for a, c in zip(got, want))
fp8.check()
print("fine")
"""


def test_first_large_calls_of_a_process_may_be_captured():
    """The kernels of pairs, with and without a residual, in each result type: their first launches inside a capture, and
    replayed on new inputs."""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST_LARGE_CALLS_IN_A_CAPTURE, os.path.dirname(os.path.abspath(__file__))],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]

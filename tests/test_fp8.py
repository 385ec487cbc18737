"""The 8-bit operators on the CPU: the reference forms against each other, and every refusal of the C
entries and of the torch entries that needs no GPU."""
import ctypes

import numpy as np
import pytest
import torch

import fp8_ref as ref


def test_codes_against_torch_conversion():
    rng = np.random.default_rng(0)
    v = np.concatenate([rng.uniform(-448, 448, 4000), rng.standard_normal(4000), rng.standard_normal(4000) * 2.0 ** -8,
                        (ref._POS[1:] + ref._POS[:-1]) / 2, -(ref._POS[1:] + ref._POS[:-1]) / 2, ref._POS, -ref._POS])
    v = v.astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.e4m3_code(v.astype(np.float64)), want)
    assert np.array_equal(ref.TABLE[:127], torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())


def test_scale_is_the_smallest_that_holds_the_block():
    for a in (0.0, 1e-45, 2.0 ** -126, 1.0, 447.9, 448.0, 448.0001, 449.0, 896.0, 897.0, 3.4e38):
        e = ref.block_exp(a)
        assert a <= 448.0 * 2.0 ** (e - 127)
        assert e == 0 or a > 448.0 * 2.0 ** (e - 128)


def test_quantize_keeps_half_a_step():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((7, 300)) * np.exp(rng.uniform(-20, 20, (7, 1)))
    code, E = ref.quantize(x)
    back = ref.dequantize(code, E)
    amax = np.repeat([[np.abs(r[b * 128:(b + 1) * 128]).max() for b in range(3)] for r in x], 128, 1)[:, :300]
    # half a step of the value, or half of the smallest step (2^-9) at a scale below amax / 224
    assert (np.abs(back - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -10 * amax / 224).all()


# ---- refusals of the C entries (nothing is launched; the pointers are never followed)

P = 1 << 12  # an aligned address


def q_args(**kw):
    a = dict(dev=0, st=None, x=P, type=0, rows=4, k=256, ldx=256, br=1, v=P, ldv=256, e=P, lde=4)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, word", [
    (dict(rows=-1), "row count"), (dict(rows=1 << 31), "row count"), (dict(k=0), "column count"),
    (dict(k=1 << 31), "column count"), (dict(rows=1 << 30, k=1024, ldx=1024, ldv=1024, lde=8), "blocks"),
    (dict(br=2), "block_rows"), (dict(br=0), "block_rows"), (dict(x=None), "null"), (dict(type=2), "f32 or bf16"),
    (dict(type=-1), "f32 or bf16"), (dict(ldx=255), "row stride"), (dict(x=P + 2), "aligned"),
    (dict(v=None), "null"), (dict(e=None), "null"), (dict(ldv=255), "16 bytes"), (dict(ldv=240), "16 bytes"),
    (dict(ldv=264), "16 bytes"), (dict(lde=2), "4 bytes"), (dict(lde=5), "4 bytes"), (dict(v=P + 8), "16-byte"),
    (dict(e=P + 1), "4-byte"),
])
def test_quantize_refusals(kk, kw, word):
    lib = kk.load_library()
    assert lib.kk_fp8_quantize(*q_args(**kw)) == kk.engine.KK_ERR_INVALID_ARG
    assert word in lib.kk_fp8_error().decode()
    a = q_args(**kw)
    if "x" in kw or "ldx" in kw or "type" in kw:  # the same rows on the way back
        a = [a[0], a[1], a[8], a[9], a[10], a[11], a[7], a[4], a[5], a[2], a[3], a[6]]
        assert lib.kk_fp8_dequantize(*a) == kk.engine.KK_ERR_INVALID_ARG
        assert word in lib.kk_fp8_error().decode()


def l_args(**kw):
    a = dict(dev=0, st=None, m=4, n=256, k=128, x=P, ldx=128, xe=P, ldxe=4, w=P, ldw=128, we=P, ldwe=4, bias=None, act=0,
             res=None, ldr=256, yt=0, y=P, ldy=256, ye=None, ldye=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, word", [
    (dict(m=-1), "row count"), (dict(n=0), "column count"), (dict(k=0), "column count"), (dict(n=-5), "column count"),
    (dict(act=2), "activation"), (dict(yt=3), "output type"), (dict(x=None), "x: null"), (dict(w=None), "w: null"),
    (dict(x=P + 4), "x: values"), (dict(w=P + 4), "w: values"), (dict(ldx=100), "x: value rows"),
    (dict(ldxe=1), "x: exponent rows"), (dict(bias=P + 2), "bias"), (dict(y=None), "y: null"), (dict(ldy=255), "y: row stride"),
    (dict(res=P, ldr=200), "residual: row stride"), (dict(res=P + 1), "residual: rows"),
    (dict(yt=2, ldy=256, ye=P, ldye=4, res=P), "no residual"), (dict(yt=2, ldy=256, ye=None, ldye=4), "y: null"),
    (dict(yt=2, ldy=250, ye=P, ldye=4), "y: value rows"), (dict(yt=1, y=P + 1), "y: rows"),
])
def test_linear_refusals(kk, kw, word):
    lib = kk.load_library()
    assert lib.kk_fp8_linear(*l_args(**kw)) == kk.engine.KK_ERR_INVALID_ARG
    assert word in lib.kk_fp8_error().decode()


def test_packed_calls_are_the_same_calls(kk):
    """Each argument in its place: one is spoilt at a time, and the status and the message are those of the call itself."""
    import struct
    lib = kk.load_library()
    quant = q_args(x=1 << 30, v=1 << 31, e=1 << 32, dev=99)
    deq = [quant[0], quant[1], quant[8], quant[9], quant[10], quant[11], quant[7], quant[4], quant[5], quant[2], quant[3], quant[6]]
    lin = l_args(x=1 << 30, xe=1 << 31, w=1 << 32, we=1 << 33, y=1 << 34, res=1 << 35, bias=1 << 36, dev=99)
    lin8 = l_args(x=1 << 30, xe=1 << 31, w=1 << 32, we=1 << 33, y=1 << 34, yt=2, ye=1 << 35, ldye=4, bias=1 << 36, dev=99)
    seen = set()
    for op, f, good in ((0, lib.kk_fp8_quantize, quant), (1, lib.kk_fp8_dequantize, deq), (2, lib.kk_fp8_linear, lin),
                        (2, lib.kk_fp8_linear, lin8)):
        for i in [None, *range(len(good))]:
            for bad in (-1, 1, 7, 0):
                a = list(good)
                if i is not None:
                    if i < 2:
                        continue  # (the device and the stream: this machine may have none)
                    a[i] = bad
                st, msg = f(*a), lib.kk_fp8_error()
                packed = struct.pack(f"{len(a)}q", *(v or 0 for v in a))
                assert (lib.kk_fp8_call(op, packed, len(a)), lib.kk_fp8_error()) == (st, msg)
                seen.add(msg)
    assert len(seen) > 15
    packed = struct.pack("22q", *(v or 0 for v in lin))
    for op, p, n in ((2, packed, 21), (0, packed, 22), (3, packed, 12), (-1, packed, 22), (2, None, 22)):
        assert lib.kk_fp8_call(op, p, n) == kk.engine.KK_ERR_INVALID_ARG
    wide = list(quant)
    wide[3] = 1 << 32  # as an int it would be type 0
    assert lib.kk_fp8_call(0, struct.pack("12q", *(v or 0 for v in wide)), 12) == kk.engine.KK_ERR_INVALID_ARG
    assert "f32 or bf16" in lib.kk_fp8_error().decode()


def overlaps(a, b):
    """Whether two lists of (address, rows, bytes of a row, pitch) share a byte, byte by byte."""
    cells = lambda p, rows, width, pitch: {p + i * pitch + j for i in range(rows) for j in range(width)}
    return bool(cells(*a) & cells(*b))


def test_overlap_is_refused(kk):
    """Residual and result in one buffer, a row pitch apart or columns of it, against their bytes counted out."""
    lib, n, m, ld = kk.load_library(), 5, 3, 16
    base = 1 << 20
    far = dict(m=m, n=n, x=1 << 30, xe=1 << 31, w=1 << 32, we=1 << 33, y=base, ldy=ld, ldr=ld, dev=99)
    seen = set()
    for d in range(-70, 71):  # elements between the two
        for yt, es in ((0, 4), (1, 2)):
            want = d != 0 and overlaps((base, m, n * es, ld * es), (base + d * es, m, n * es, ld * es))
            assert lib.kk_fp8_linear(*l_args(**far, yt=yt, res=base + d * es)) != kk.engine.KK_OK
            assert ("residual must be" in lib.kk_fp8_error().decode()) == want, (d, yt)
            seen.add(want)
    assert seen == {True, False}
    # another pitch, and the same address at another pitch
    for kw in (dict(res=base, ldr=ld + 4), dict(res=base + 4 * n, ldr=8)):
        assert lib.kk_fp8_linear(*l_args(**{**far, **kw})) == kk.engine.KK_ERR_INVALID_ARG
        assert "residual must be" in lib.kk_fp8_error().decode()
    # one row: only its bytes count
    for d, want in ((0, False), (4 * n, False), (4, True)):
        lib.kk_fp8_linear(*l_args(**{**far, "m": 1, "res": base + d, "ldr": n}))
        assert ("residual must be" in lib.kk_fp8_error().decode()) == want


@pytest.mark.parametrize("kw, word", [
    (dict(y=1 << 30), "y must not"), (dict(y=1 << 31), "y must not"), (dict(y=(1 << 32) + 64), "y must not"),
    (dict(y=1 << 33), "y must not"), (dict(y=1 << 34, bias=(1 << 34) + 1020), "y must not"),
    (dict(yt=2, y=1 << 30, ldy=128, n=128, ye=1 << 35, ldye=4), "y must not"),
    (dict(yt=2, y=1 << 34, ye=1 << 31, ldye=4), "y must not"), (dict(yt=2, y=1 << 34, ye=(1 << 34) + 252, ldye=4), "y: the values"),
])
def test_result_over_its_inputs_is_refused(kk, kw, word):
    lib = kk.load_library()
    a = dict(x=1 << 30, xe=1 << 31, w=1 << 32, we=1 << 33)
    assert lib.kk_fp8_linear(*l_args(**{**a, **kw})) == kk.engine.KK_ERR_INVALID_ARG
    assert word in lib.kk_fp8_error().decode()


def test_quantize_over_its_input_is_refused(kk):
    lib = kk.load_library()
    x, v, e = 1 << 30, 1 << 31, 1 << 32
    for kw in (dict(v=x), dict(e=x), dict(e=v), dict(v=x + 1024 * 3 + 1008)):
        a = q_args(**{**dict(x=x, v=v, e=e), **kw})
        assert lib.kk_fp8_quantize(*a) == kk.engine.KK_ERR_INVALID_ARG and "overlap" in lib.kk_fp8_error().decode()
        if kw == dict(e=v):
            continue  # (a store that overlaps itself is not read back)
        a = [a[0], a[1], a[8], a[9], a[10], a[11], a[7], a[4], a[5], a[2], a[3], a[6]]
        assert lib.kk_fp8_dequantize(*a) == kk.engine.KK_ERR_INVALID_ARG and "overlap" in lib.kk_fp8_error().decode()


def test_no_rows_is_a_no_op(kk):
    lib = kk.load_library()
    assert lib.kk_fp8_quantize(*q_args(rows=0, x=None, v=None, e=None)) == kk.engine.KK_OK
    assert lib.kk_fp8_linear(*l_args(m=0, x=None, xe=None, y=None)) == kk.engine.KK_OK


def test_bad_ordinal_is_a_status(kk):
    lib = kk.load_library()
    assert lib.kk_fp8_quantize(*q_args(dev=99)) in (kk.engine.KK_ERR_INVALID_ARG, kk.engine.KK_ERR_CUDA)
    assert lib.kk_fp8_error()


# ---- refusals of the torch entries


def refused(kk, f, *a, **kw):
    with pytest.raises(kk.KokoroError) as e:
        f(*a, **kw)
    assert e.value.status == kk.engine.KK_ERR_INVALID_ARG
    return str(e.value)


def test_torch_refusals(kk):
    fp8 = kk.fp8
    assert "CUDA tensor" in refused(kk, fp8.quantize, torch.zeros(4, 128))
    assert "float32" in refused(kk, fp8.quantize, torch.zeros(4, 128, dtype=torch.float16))
    assert "rows are wanted" in refused(kk, fp8.quantize, torch.zeros(128))
    assert "adjacent" in refused(kk, fp8.quantize, torch.zeros(128, 4).t())
    assert "store is wanted" in refused(kk, fp8.dequantize, torch.zeros(4, 128))
    assert "block_rows 1" in refused(kk, fp8.linear, torch.zeros(4, 128), torch.zeros(4, 128))
    assert "CUDA device" in refused(kk, fp8.Fp8Tensor.empty, 4, 128, device="cpu")
    v = torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert "CUDA tensor" in refused(kk, fp8.Fp8Tensor, v, torch.zeros(4, 1, dtype=torch.uint8))
    assert "values" in refused(kk, fp8.Fp8Tensor, v.view(torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))


def test_fp8_error_is_per_thread(kk):
    import threading
    lib = kk.load_library()
    assert lib.kk_fp8_quantize(*q_args(k=0)) != 0
    got = []
    t = threading.Thread(target=lambda: got.append(ctypes.string_at(lib.kk_fp8_error())))
    t.start()
    t.join()
    assert lib.kk_fp8_error() and got == [b""]


def test_forward_mode_tangents_are_refused(kk):
    """As rows, and as the values of a store; outside of their level, or with forward mode off, there is none to lose."""
    from torch.autograd import forward_ad
    fp8 = kk.fp8
    x, v = torch.randn(4, 128), torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        assert "forward mode" in refused(kk, fp8.quantize, d)
        dv = forward_ad.make_dual(v, torch.zeros_like(v))
        assert "forward mode" in refused(kk, fp8.Fp8Tensor, dv, torch.zeros(4, 1, dtype=torch.uint8))
        with torch.no_grad():
            assert "forward mode" in refused(kk, fp8.quantize, d)
        with torch.inference_mode():  # (no tangents are kept here)
            assert "CUDA tensor" in refused(kk, fp8.quantize, d)
        assert "CUDA tensor" in refused(kk, fp8.quantize, x)
    assert "CUDA tensor" in refused(kk, fp8.quantize, d)
    with pytest.raises(kk.KokoroError, match="forward mode"):
        torch.func.jvp(fp8.quantize, (x,), (x,))
    assert "no gradient" in refused(kk, fp8.quantize, x.clone().requires_grad_())


def test_negation_still_to_be_done_is_refused(kk):
    """The imaginary part of a conjugate holds its numbers with the other sign."""
    c = torch.randn(5, 1, dtype=torch.complex64).conj().imag
    assert c.is_neg()
    assert "resolve_neg" in refused(kk, kk.fp8.quantize, c)
    assert "CUDA tensor" in refused(kk, kk.fp8.quantize, c.resolve_neg())


def test_check_of_another_kind_of_device_is_refused(kk):
    for device in ("cpu", torch.device("cpu"), "meta"):
        assert "CUDA device" in refused(kk, kk.fp8.check, device)


def test_wait_selftest_refusals(kk):
    lib = kk.load_library()
    for cluster, limit, word in ((2, 5000, "cluster"), (-1, 5000, "cluster"), (0, 999, "limit"), (1, 100000001, "limit"), (0, -1, "limit")):
        assert lib.kk_fp8_wait_selftest(0, None, cluster, limit) == kk.engine.KK_ERR_INVALID_ARG
        assert word in lib.kk_fp8_error().decode()
    assert "CUDA device" in refused(kk, kk.fp8.wait_selftest, "cpu")

"""The FP8 precision mode (the BF16 mode with ALBERT's layers in 8 bits) against
the CPU oracle with the same layers held in 8 bits, and against the plain oracle.

Bounds, derived: an e4m3 value is off by at most 2^-4, uniformly over its binade about 0.026 of it (rms),
so a layer's result by about 0.036 (two operands). What the engine does not share with the oracle's 8-bit
layers is the bf16 attention around them (2^-9): values that it moves across a rounding border, about two
in a hundred, change by a step of up to 2^-3, 0.013 of the result. The engine's rows are therefore expected
0.013 / 0.036 = 0.36 as far from the 8-bit oracle's as those are from the plain oracle's, in every layer
alike; the bound is 0.6. Over the 48 layers the plain distance stays below 0.25."""
import os
import tempfile

import numpy as np
import pytest
import torch

import fp8_ref as ref
from conftest import synth_item

pytestmark = pytest.mark.gpu

LAYER = "bert.encoder.albert_layer_groups.0.albert_layers.0"


def held(x, block_rows):
    """x as the stores hold it (torch, exact): the same rule as tests/fp8_ref.py, by torch's conversion."""
    r, k = x.shape
    p = torch.nn.functional.pad(x, (0, -k % 128, 0, -r % block_rows)).double()
    p = p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // 128, 128)
    amax = p.abs().amax(dim=(1, 3)).numpy()
    e = torch.tensor([[ref.block_exp(a) for a in row] for row in amax], dtype=torch.float64)[:, None, :, None]
    q = (p * 2.0 ** (127 - e)).float().to(torch.float8_e4m3fn).double() * 2.0 ** (e - 127)
    return q.view(p.shape[0] * block_rows, -1)[:r, :k].float()


@pytest.fixture(scope="module")
def oracle8(oracle_mod, state_dict):
    class Oracle8(oracle_mod.KokoroOracle):
        """The oracle with ALBERT's layers on operands held in 8 bits."""
        weights = {}

        def linear(self, x, prefix):
            if not prefix.startswith(LAYER):
                return super().linear(x, prefix)
            if prefix not in self.weights:
                self.weights[prefix] = held(self.t(prefix + ".weight"), 128)
            return held(x.float(), 1) @ self.weights[prefix].T + self.t(prefix + ".bias")

    return Oracle8(state_dict, threads=min(8, os.cpu_count() or 1))


@pytest.fixture(scope="module")
def eng8(kk, ckpt_path):
    e = kk.GpuKokoro(ckpt_path, 0, "fp8")
    yield e
    e.close()


@pytest.fixture(scope="module")
def cases(kk):
    rng = np.random.default_rng(31)
    items = []
    for i, n in enumerate((5, 60, 140, 300)):
        ids, ref_s = synth_item(rng, n)
        items.append(kk.BatchItem(ids, ref_s, 1.0, kk.ItemNoise(seed=200 + i)))
    return items


def test_fp8_encoder_rows(eng8, cases, oracle, oracle8):
    d = tempfile.mkdtemp()
    os.environ["KK_DEBUG_DUMP_DIR"] = d
    try:
        eng8.forward_batch(cases)
    finally:
        del os.environ["KK_DEBUG_DUMP_DIR"]
    bert = np.fromfile(os.path.join(d, "bert.f32"), np.float32).reshape(-1, 768)
    d_en = np.fromfile(os.path.join(d, "d_en.f32"), np.float32).reshape(-1, 640)[:, :512]
    at = 0
    for it in cases:
        ids = np.asarray(it.ids)
        T = len(ids)
        plain, eight = oracle.albert(ids), oracle8.albert(ids)
        for got, p8, p in ((bert[at:at + T], eight.numpy(), plain.numpy()),
                           (d_en[at:at + T], oracle8.linear(eight, "bert_encoder").numpy(),
                            oracle.linear(plain, "bert_encoder").numpy())):
            far = np.linalg.norm(p8 - p) / np.linalg.norm(p)
            off = np.linalg.norm(got - p8) / np.linalg.norm(p8)
            print(f"T {T}: 8-bit oracle {far:.3g} off the plain one, engine {off:.3g} off the 8-bit one")
            assert far <= 0.25 and off <= 0.6 * far
        at += T + 2


def test_fp8_durations(eng8, cases, oracle, oracle8):
    """Durations against the 8-bit oracle's (within a frame), and how many differ from the plain oracle's."""
    outs = eng8.forward_batch(cases)
    n = diff = most = 0
    for it, o in zip(cases, outs):
        r8 = oracle8.forward(it.ids, it.ref_s, 1.0, seed=it.noise.seed, want=("dur_q",))
        r = oracle.forward(it.ids, it.ref_s, 1.0, seed=it.noise.seed, want=("dur_q",))
        assert np.abs(o.pred_dur - r8["dur"]).max() <= 1
        assert o.audio.shape[0] == 600 * int(o.pred_dur.sum()) and np.isfinite(o.audio).all()
        n, diff = n + len(r["dur"]), diff + int((o.pred_dur != r["dur"]).sum())
        most = max(most, int(np.abs(o.pred_dur - r["dur"]).max()))
    print(f"{diff} of {n} durations differ from the plain oracle's, by at most {most}")


def test_fp8_twice_the_same_and_gap_rows_stay_out(kk, eng8, cases):
    """The same batch twice gives the same bits, also with every buffer NaN before it is written."""
    a = eng8.forward_batch(cases)
    b = eng8.forward_batch(cases)
    eng8.set_option(kk.engine.KK_OPT_GAP_CANARY, 1)
    try:
        c = eng8.forward_batch(cases)
    finally:
        eng8.set_option(kk.engine.KK_OPT_GAP_CANARY, 0)
    for x, y, z in zip(a, b, c):
        assert np.array_equal(x.pred_dur, y.pred_dur) and np.array_equal(x.audio, y.audio)
        assert np.array_equal(x.pred_dur, z.pred_dur) and np.isfinite(z.audio).all()


def test_fp8_mode_with_the_f32_attention(kk, eng8, cases):
    want = eng8.forward_batch(cases)
    eng8.set_option(kk.engine.KK_OPT_ATTENTION_F32, 1)
    try:
        got = eng8.forward_batch(cases)
    finally:
        eng8.set_option(kk.engine.KK_OPT_ATTENTION_F32, 0)
    for a, b in zip(want, got):
        assert np.abs(a.pred_dur - b.pred_dur).max() <= 1


def test_fp8_identity_and_vocoder(kk, ckpt_path, eng8):
    """The identity names the mode (resume keys differ); the vocoder is the BF16 mode's, bit for bit."""
    assert " fp8 " in eng8.identity
    rng = np.random.default_rng(5)
    asr = rng.standard_normal((20, 512)).astype(np.float32)
    f0 = np.exp(rng.uniform(np.log(80), np.log(400), 40)).astype(np.float32)
    nc = rng.standard_normal(40).astype(np.float32)
    s = (rng.standard_normal((1, 128)) * 0.1).astype(np.float32)
    e16 = kk.GpuKokoro(ckpt_path, 0, "bf16")
    try:
        assert np.array_equal(eng8.decode_batch([asr], [f0], [nc], s, seeds=[3])[0],
                              e16.decode_batch([asr], [f0], [nc], s, seeds=[3])[0])
    finally:
        e16.close()


def test_fp8_mode_holds_its_layers_in_8_bits_alone(kk, ckpt_path, cases):
    """The four layers' weights take a byte each and a scale for each 128 x 128, where the BF16 mode has 4 bytes (f32) and
    at least 2 (bf16 tiles); and a forward's buffers are no larger."""
    layers = ((2304, 768), (768, 768), (2048, 768), (768, 2048))
    values = sum(n * k for n, k in layers)
    scales = sum(-(-n // 128) * -(-k // 512) * 4 for n, k in layers)
    fresh, after = {}, {}
    for mode in ("bf16", "fp8"):
        e = kk.GpuKokoro(ckpt_path, 0, mode)
        try:
            fresh[mode] = e.device_bytes()
            e.forward_batch(cases)
            after[mode] = e.device_bytes()
        finally:
            e.close()
    assert fresh["bf16"] - fresh["fp8"] >= (4 + 2 - 1) * values - scales
    assert after["fp8"] - fresh["fp8"] <= after["bf16"] - fresh["bf16"]


def test_fp8_canary_audio_is_the_same(kk, eng8, cases):
    """With every buffer NaN before it is written, the audio too has the same bits."""
    want = eng8.forward_batch(cases)
    eng8.set_option(kk.engine.KK_OPT_GAP_CANARY, 1)
    try:
        got = eng8.forward_batch(cases)
    finally:
        eng8.set_option(kk.engine.KK_OPT_GAP_CANARY, 0)
    for a, b in zip(want, got):
        assert np.array_equal(a.audio, b.audio)


@pytest.fixture(scope="module")
def large(kk):
    """13 items of 511 tokens, 6,669 rows with their gaps: 53 tiles of 128 rows, at which every layer is past the small
    layers' kernel. That takes more than 2 x 148 tiles of 128 x 128 (QKV, 18 tiles wide; the output projection and the
    down projection, 6 wide: 318), more than 148 for the 8-bit result of the GELU layer (16 wide)."""
    rng = np.random.default_rng(33)
    items = []
    for i in range(13):
        ids, ref_s = synth_item(rng, 509)
        items.append(kk.BatchItem(ids, ref_s, 1.0, kk.ItemNoise(seed=300 + i)))
    return items


LOOKED_AT = (0, 6, 12)  # of the large batch, against the oracles


def test_fp8_encoder_rows_of_a_large_batch(eng8, large, oracle, oracle8):
    """The bounds of the small batches hold for the large layers' kernels and their rows for the attention."""
    d = tempfile.mkdtemp()
    os.environ["KK_DEBUG_DUMP_DIR"] = d
    try:
        eng8.forward_batch(large, forced_dur=[np.arange(511) < 4] * len(large))
    finally:
        del os.environ["KK_DEBUG_DUMP_DIR"]
    bert = np.fromfile(os.path.join(d, "bert.f32"), np.float32).reshape(-1, 768)
    for i in LOOKED_AT:
        ids = np.asarray(large[i].ids)
        p, p8 = oracle.albert(ids).numpy(), oracle8.albert(ids).numpy()
        got = bert[i * 513:i * 513 + 511]
        far = np.linalg.norm(p8 - p) / np.linalg.norm(p)
        off = np.linalg.norm(got - p8) / np.linalg.norm(p8)
        worst = (np.linalg.norm(got - p8, axis=1) / np.linalg.norm(p8, axis=1)).max()
        print(f"item {i}: 8-bit oracle {far:.3g} off the plain one, engine {off:.3g} off the 8-bit one, worst row {worst:.3g}")
        assert far <= 0.25 and off <= 0.6 * far
        # no row is lost among the others: a wrong one would be 1 or more off, the rounding errors of 768 columns average
        assert worst <= 3 * 0.6 * far


def test_fp8_durations_of_a_large_batch(kk, ckpt_path, eng8, large, oracle, oracle8):
    """What the mode says of its durations: some differ, by a frame, from the BF16 mode's and from the plain oracle's.

    How many: a duration is a rounded sum, so it changes with a probability that goes with how far the sum moves. The
    engine's rows are at most 0.6 as far from the 8-bit oracle's as those are from the plain ones, so at most 1.6 times as
    far from the plain ones, and 1.6 times as many durations may change as between the two oracles, give or take four
    standard deviations of a count."""
    outs = eng8.forward_batch(large, fetch=False)
    e16 = kk.GpuKokoro(ckpt_path, 0, "bf16")
    try:
        outs16 = e16.forward_batch(large, fetch=False)
    finally:
        e16.close()
    assert all(np.abs(a.pred_dur - b.pred_dur).max() <= 1 for a, b in zip(outs, outs16))
    n = moved = moved8 = 0
    for i in LOOKED_AT:
        it, got = large[i], outs[i].pred_dur
        plain, eight = (o.durations(it.ids, it.ref_s)[0] for o in (oracle, oracle8))
        assert np.abs(got - eight).max() <= 1 and np.abs(got - plain).max() <= 1
        n, moved, moved8 = n + len(got), moved + int((got != plain).sum()), moved8 + int((eight != plain).sum())
    print(f"{moved} of {n} durations differ from the plain oracle's, {moved8} between the oracles")
    assert 0 < moved <= 1.6 * moved8 + 4 * np.sqrt(1.6 * moved8) + 4


def test_an_earlier_failure_is_not_the_engines(kk, ckpt_path, eng8, cases):
    """A call that the library refused with a CUDA error, on this thread, before an engine is made (the FP8 mode launches
    kernels as it loads) and before a forward."""
    import ctypes
    lib = kk.load_library()
    n, buf = np.array([1], np.int32), np.zeros(2304, np.float32)
    want = eng8.forward_batch(cases[:1])[0]

    def fail():
        assert lib.kk_attention_selftest(99, 1, n.ctypes.data_as(ctypes.c_void_p), buf.ctypes.data_as(ctypes.c_void_p),
                                         buf.ctypes.data_as(ctypes.c_void_p)) == kk.engine.KK_ERR_CUDA

    fail()
    e = kk.GpuKokoro(ckpt_path, 0, "fp8")
    try:
        fail()
        got = e.forward_batch(cases[:1])[0]
    finally:
        e.close()
    assert np.array_equal(got.pred_dur, want.pred_dur) and np.array_equal(got.audio, want.audio)

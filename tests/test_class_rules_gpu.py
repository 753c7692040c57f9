"""Recognizers with rules on their classes and with the best classes of each
step, and the engine under rules, against the plain recognizer's probabilities:
the rules multiply a class's probability by exp(bias) or zero, and the rest is a
renormalisation."""

import numpy as np
import pytest

import ppocr_hip
import seeded
from helpers import argmax_last, ctc_greedy, model_path, quad_corners, synthetic_dictionary

pytestmark = pytest.mark.gpu

CLASSES = {"tiny": 6906, "medium": 18710}
# Both the ruled probabilities and the plain ones that the expected come from are
# fp32 softmaxes: an exponential's argument d = logit - largest, at least -88
# where the result is a normal number, takes up to three roundings of 2^-24
# relative to it, the exponential itself, the sum and the division a few more.
REL = 2 * (3 * 88 + 8) * 2.0 ** -24
# A plain probability below the normal range may have become 0.
TINY = 2.0 ** -126


@pytest.fixture(scope="module")
def gpu():
    g = ppocr_hip.Gpu(0)
    yield g
    g.close()


def lines(n, width, seed):
    return seeded.seeded_batch(n, 48, width, seed=seed, detector=False)


def rules_of(classes, seed):
    rng = np.random.default_rng(seed)
    allowed = rng.random(classes) < 0.3
    allowed[0] = True
    return allowed, rng.normal(size=classes).astype(np.float32)


def expected(probabilities, allowed, bias):
    """Ruled probabilities and their error: what the plain ones lost below the
    normal range counts for a class by itself and for all through the sum."""
    q = probabilities.astype(np.float64)
    lost = np.full(q.shape[-1], TINY)
    if bias is not None:
        q, lost = q * np.exp(bias.astype(np.float64)), lost * np.exp(bias.astype(np.float64))
    if allowed is not None:
        q, lost = q * allowed, lost * allowed
    whole = q.sum(-1, keepdims=True)
    want = q / whole
    return want, want * (REL + lost.sum() / whole) + 2 * lost / whole + TINY


@pytest.mark.parametrize("size,precision", [("tiny", "f32"), ("medium", "f32"), ("tiny", "bf16")])
@pytest.mark.parametrize("parts", ["mask", "bias", "both"])
def test_ruled_recognizers(gpu, size, precision, parts):
    path, shape = model_path("rec", size), (3, 3, 48, 200)
    x = lines(3, 200, 5)
    allowed, bias = rules_of(CLASSES[size], 6)
    kw = dict(allowed=allowed if parts != "bias" else None, bias=bias if parts != "mask" else None)
    plain = ppocr_hip.Recognizer.load(gpu, path, size, shape, precision)
    ruled = ppocr_hip.Recognizer.load(gpu, path, size, shape, precision, share_weights=plain, **kw)
    greedy = ppocr_hip.Recognizer.load(gpu, path, size, shape, precision, share_weights=ruled, greedy=True, **kw)
    top = ppocr_hip.Recognizer.load(gpu, path, size, shape, precision, share_weights=greedy, top_k=20, **kw)
    try:
        p = plain.forward(x).array()
        want, error = expected(p, **kw)
        got = ruled.forward(x).array()
        assert got.shape == p.shape
        wrong = np.abs(got - want) > error
        assert not wrong.any(), (got[wrong][:4], want[wrong][:4], error[wrong][:4])
        if kw["allowed"] is not None:
            assert (got[..., ~allowed] == 0).all()
        # The greedy step and the best classes of the same logits.
        g = greedy.forward(x).array()
        assert g.shape == p.shape[:2] + (2,)
        assert np.array_equal(g[..., 0], argmax_last(got))
        assert np.all(np.abs(g[..., 1] - got.max(-1)) <= REL * got.max(-1))
        t = top.forward(x).array()
        assert t.shape == p.shape[:2] + (20, 2)
        # Another k splits the sum between listed classes and the rest elsewhere:
        # the same class, its probability within the sums' roundings.
        assert np.array_equal(t[..., 0, 0], g[..., 0])
        assert np.all(np.abs(t[..., 0, 1] - g[..., 1]) <= REL * g[..., 1])
        assert (np.diff(t[..., 1], axis=-1) <= 0).all()
        classes = t[..., 0].astype(np.int64)
        assert np.all(np.abs(np.take_along_axis(got, classes, -1) - t[..., 1]) <= REL * t[..., 1] + TINY)
        best = -np.sort(-got, axis=-1)[..., :20]
        assert np.all(np.abs(best - t[..., 1]) <= REL * best + TINY)
        assert np.array_equal(plain.forward(x).array(), p)
    finally:
        for m in (top, greedy, ruled, plain):
            m.close()


def test_best_classes_without_rules_and_with_few_allowed(gpu):
    path, shape, x = model_path("rec", "tiny"), (2, 3, 48, 64), lines(2, 64, 7)
    plain = ppocr_hip.Recognizer.load(gpu, path, "tiny", shape)
    greedy = ppocr_hip.Recognizer.load(gpu, path, "tiny", shape, greedy=True)
    top = ppocr_hip.Recognizer.load(gpu, path, "tiny", shape, top_k=3)
    allowed = np.zeros(6906, bool)
    allowed[[0, 500]] = True
    few = ppocr_hip.Recognizer.load(gpu, path, "tiny", shape, top_k=4, allowed=allowed)
    try:
        p, t = plain.forward(x).array(), top.forward(x).array()
        assert np.array_equal(t[..., 0, 0], greedy.forward(x).array()[..., 0])
        assert np.all(np.abs(np.take_along_axis(p, t[..., 0].astype(np.int64), -1) - t[..., 1]) <= REL * t[..., 1] + TINY)
        f = few.forward(x).array()
        assert set(np.unique(f[..., :2, 0])) == {0.0, 500.0}
        assert np.all(np.abs(f[..., :2, 1].sum(-1) - 1) <= REL)
        assert (f[..., 2:, 0] == -1).all() and (f[..., 2:, 1] == 0).all()
    finally:
        for m in (few, top, greedy, plain):
            m.close()


def test_ruled_batches_in_chunks(gpu, monkeypatch):
    """A limit on buffers splits the batch; each chunk takes the same rules."""
    path, shape, x = model_path("rec", "tiny"), (5, 3, 48, 64), lines(5, 64, 8)
    allowed, bias = rules_of(6906, 9)
    whole = ppocr_hip.Recognizer.load(gpu, path, "tiny", shape, top_k=6, allowed=allowed, bias=bias)
    want = whole.forward(x).array()
    monkeypatch.setenv("PPOCR_HIP_MAX_BUFFER_BYTES", str(2 * 8 * 6906 * 4 + 4096))
    chunked = ppocr_hip.Recognizer.load(gpu, path, "tiny", shape, top_k=6, allowed=allowed, bias=bias)
    try:
        got = chunked.forward(x).array()
        assert np.array_equal(got[..., 0], want[..., 0])
        assert np.all(np.abs(got[..., 1] - want[..., 1]) <= 1e-4)
    finally:
        chunked.close()
        whole.close()


@pytest.mark.parametrize("greedy", [True, False])
def test_engine_under_rules(gpu, greedy):
    """Every line's tokens are allowed ones, equal to decoding the ruled
    probabilities of the line; without rules the engine answers as before."""
    img = seeded.seeded_rgb(540, 960, 23, pattern="blocks")
    dictionary = synthetic_dictionary(6906)
    engine = ppocr_hip.OcrEngine.load(gpu, model_path("det", "tiny"), model_path("rec", "tiny"), dictionary,
                                      greedy=greedy, binary_threshold=0.62, box_threshold=0.0)
    plain = ppocr_hip.Recognizer.load(gpu, model_path("rec", "tiny"), "tiny", (1, 3, 48, 320))
    allowed, bias = rules_of(6906, 10)
    bias[0] = -3.0
    image = gpu.upload_rgb(img)
    try:
        before = engine.recognize(img)
        engine.set_rules(allowed=allowed, bias=bias)
        ruled = engine.recognize(img)
        again = engine.recognize(img)
        engine.set_rules()
        after = engine.recognize(img)
        assert [ln.tokens for ln in after.lines] == [ln.tokens for ln in before.lines]
        assert [ln.recognition_score for ln in after.lines] == [ln.recognition_score for ln in before.lines]
        assert [ln.tokens for ln in again.lines] == [ln.tokens for ln in ruled.lines]
        assert len(ruled.lines) == len(before.lines) > 6
        used = {t for ln in ruled.lines for t in ln.tokens}
        assert used and all(allowed[t] for t in used)
        checked = 0
        for ln in ruled.lines:
            if ppocr_hip.recognizer_batch_width(ln.polygon[None]) != 320:
                continue
            content = ppocr_hip.recognition_input_plan(ln.polygon, 320)
            p, _ = expected(plain.forward_image(image, ln.polygon[None], [content]).array()[0], allowed, bias)
            s = np.sort(p, -1)
            if (s[:, -1] - s[:, -2]).min() <= 1e-4:
                continue  # a near-tied step may fall to either side
            text, score = ctc_greedy(p.astype(np.float32), dictionary, content, 320)
            # Lines of a batch share a canvas as wide as its widest line.
            if text == ln.text:
                assert abs(score - ln.recognition_score) <= 1e-3
                checked += 1
        assert checked > 0
    finally:
        image.close()
        plain.close()
        engine.close()


def test_engine_refuses_bad_rules_and_goes_on(gpu):
    engine = ppocr_hip.OcrEngine.load(gpu, model_path("det", "tiny"), model_path("rec", "tiny"),
                                      synthetic_dictionary(6906))
    try:
        with pytest.raises(ppocr_hip.GpuError, match="blank"):
            engine.set_rules(allowed=np.zeros(6906, bool))
        with pytest.raises(ppocr_hip.GpuError, match="non-finite"):
            engine.set_rules(bias=np.full(6906, np.nan))
        engine.recognize(seeded.seeded_rgb(240, 320, 3, pattern="blocks"))
    finally:
        engine.close()

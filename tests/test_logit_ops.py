"""Operators on rows of logits without a GPU: the refusals of the C entry
points, which come before any device work, the checks of the Python binding,
and the plain forms' gradient against differences."""

import ctypes

import numpy as np
import pytest
import torch

import logit_oracle as oracle
import ppocr_hip

BASE = 1 << 20  # an aligned address that is never followed


def logits(data=BASE, rows=4, classes=100, stride=100, kind=0):
    return ppocr_hip._Logits(data, rows, classes, stride, kind)


def rules(classes=100, **kw):
    return ppocr_hip._Rules(classes=classes, **kw)


def teacher(values=BASE, indices=BASE, rest=None, k=4):
    return ppocr_hip._Teacher(values, indices, rest, k)


def last():
    return ppocr_hip.lib().ppocr_hip_last_error().decode()


def refused(code, text):
    assert code == 10, (code, last())
    assert text in last(), last()


@pytest.mark.parametrize("kw,text", [
    (dict(rows=4, classes=0), "classes"),
    (dict(classes=262145, stride=262145), "classes"),
    (dict(stride=99), "stride"),
    (dict(stride=(1 << 40) + 1), "stride"),
    (dict(rows=(1 << 21) + 1), "rows"),
    (dict(data=None), "data is null"),
    (dict(data=BASE + 2), "aligned"),
    (dict(data=BASE + 1, kind=1), "aligned"),
    (dict(kind=2), "element type"),
])
def test_bad_rows_are_refused_by_every_operator(kw, text):
    L = ppocr_hip.lib()
    bad, r, t, out = logits(**kw), rules(), teacher(), 1 << 30
    refused(L.ppocr_hip_logit_rules(None, bad, r, out, 1 << 20, None), text)
    refused(L.ppocr_hip_top_logits(None, bad, None, 4, 1.0, out, out, None, None), text)
    refused(L.ppocr_hip_distill_loss(None, bad, t, 1.0, out, None, None), text)
    refused(L.ppocr_hip_distill_grad(None, bad, t, out, 1.0, None, out, 1 << 20, None), text)
    refused(L.ppocr_hip_distill(None, bad, t, 1.0, None, out, out, 1 << 20, None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(classes=99), "rules for 99 classes"),
    (dict(bias=BASE), "bias"),
    (dict(n_bias=1), "without the table"),
    (dict(row_bias=BASE), "without the table"),
    (dict(bias=BASE, n_bias=2), "need an index"),
    (dict(masks=BASE, n_masks=3), "need an index"),
    (dict(masks=BASE, n_masks=1 << 31, row_mask=BASE), "2^31"),
    (dict(masks=BASE + 2, n_masks=1), "aligned"),
    (dict(repetition=BASE), "offsets"),
    (dict(history=BASE, history_len=4), "offsets"),
    (dict(history_len=4, history_offsets=BASE), "history is null"),
    (dict(history=BASE, history_len=4, history_offsets=BASE + 4), "aligned"),
    (dict(history=BASE, history_len=(1 << 40) + 1, history_offsets=BASE), "2^40"),
])
def test_bad_rules_are_refused(kw, text):
    L = ppocr_hip.lib()
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(**{"classes": 100, **kw}), 1 << 30, 100, None), text)
    refused(L.ppocr_hip_top_logits(None, logits(), rules(**{"classes": 100, **kw}), 4, 1.0, BASE, BASE, None, None), text)


def test_bad_outputs_are_refused():
    L = ppocr_hip.lib()
    refused(L.ppocr_hip_logit_rules(None, logits(), None, 1 << 30, 100, None), "rules are null")
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(), None, 100, None), "out is null")
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(), 1 << 30, 99, None), "stride")
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(), (1 << 30) + 1, 100, None), "aligned")
    # Rows that lie in part on the logits: shifted, or at another stride.
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(), BASE + 4, 100, None), "overlaps")
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(), BASE, 104, None), "overlaps")
    refused(L.ppocr_hip_logit_rules(None, logits(), rules(), BASE - 4 * 399, 100, None), "overlaps")
    # Behind the last row, in place, or one row at any stride: only the context is missing.
    for out, stride, rows in ((BASE + 1600, 100, 4), (BASE, 100, 4), (BASE, 120, 1)):
        refused(L.ppocr_hip_logit_rules(None, logits(rows=rows), rules(), out, stride, None), "context is null")
    refused(L.ppocr_hip_distill(None, logits(), teacher(), 1.0, None, BASE, BASE + 4, 100, None), "overlaps")
    refused(L.ppocr_hip_distill(None, logits(), teacher(), 1.0, None, None, 1 << 30, 100, None), "loss is null")
    refused(L.ppocr_hip_distill_loss(None, logits(), teacher(), 1.0, None, None, None), "loss is null")
    refused(L.ppocr_hip_distill_grad(None, logits(), teacher(), None, 1.0, None, 1 << 30, 100, None), "state is null")
    refused(L.ppocr_hip_top_logits(None, logits(), None, 4, 1.0, None, BASE, None, None), "null")
    refused(L.ppocr_hip_top_logits(None, logits(), None, 4, 1.0, BASE, BASE, BASE + 2, None), "aligned")


@pytest.mark.parametrize("k", [0, 65])
def test_counts_outside_the_range_are_refused(k):
    L = ppocr_hip.lib()
    refused(L.ppocr_hip_top_logits(None, logits(), None, k, 1.0, BASE, BASE, None, None), "1 to 64")
    refused(L.ppocr_hip_distill_loss(None, logits(), teacher(k=k), 1.0, BASE, None, None), "1 to 64")


@pytest.mark.parametrize("tau", [0.0, -1.0, float("nan"), float("inf"), 5e-4, 2000.0])
def test_temperatures_outside_the_range_are_refused(tau):
    L = ppocr_hip.lib()
    refused(L.ppocr_hip_top_logits(None, logits(), None, 4, tau, BASE, BASE, None, None), "temperature")
    refused(L.ppocr_hip_distill_loss(None, logits(), teacher(), tau, BASE, None, None), "temperature")
    refused(L.ppocr_hip_distill_grad(None, logits(), teacher(), BASE, tau, None, 1 << 30, 100, None), "temperature")
    refused(L.ppocr_hip_distill(None, logits(), teacher(), tau, None, BASE, 1 << 30, 100, None), "temperature")


def test_null_structures_are_refused():
    L = ppocr_hip.lib()
    refused(L.ppocr_hip_logit_rules(None, None, rules(), BASE, 100, None), "logits is null")
    refused(L.ppocr_hip_top_logits(None, None, None, 4, 1.0, BASE, BASE, None, None), "logits is null")
    refused(L.ppocr_hip_distill_loss(None, logits(), None, 1.0, BASE, None, None), "teacher is null")
    refused(L.ppocr_hip_distill_loss(None, logits(), teacher(values=None), 1.0, BASE, None, None), "null")
    refused(L.ppocr_hip_distill_loss(None, logits(), teacher(), 1.0, BASE, None, None), "context is null")


def test_structure_layouts_match_the_header():
    assert ctypes.sizeof(ppocr_hip._Logits) == 5 * 8
    assert ppocr_hip._Logits.type.offset == 32
    assert ctypes.sizeof(ppocr_hip._Rules) == 13 * 8
    assert ppocr_hip._Rules.presence.offset == 96
    assert ctypes.sizeof(ppocr_hip._Teacher) == 4 * 8


# ------------------------------------------------------------------- binding

def test_the_binding_checks_tensors():
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ppocr_hip._rows(torch.zeros(2, 3, dtype=torch.float16), "logits")
    with pytest.raises(ValueError, match="adjacent"):
        ppocr_hip._rows(torch.zeros(3, 2).t(), "logits")
    with pytest.raises(ValueError, match="dimension"):
        ppocr_hip._rows(torch.zeros(()), "logits")
    with pytest.raises(RuntimeError):  # rows that are not one stride apart
        ppocr_hip._rows(torch.zeros(2, 3, 8)[:, :2, :5], "logits")
    with pytest.raises(ValueError, match="shape and type"):
        ppocr_hip._rows_like(torch.zeros(2, 4), torch.zeros(2, 3), "out")
    with pytest.raises(ValueError, match="needs 3"):
        ppocr_hip._packed(torch.zeros(4), "float32", 3, "grad_loss")
    with pytest.raises(ValueError, match="contiguous float32"):
        ppocr_hip._packed(torch.zeros(8)[::2], "float32", 4, "grad_loss")
    with pytest.raises(ValueError, match="one shape"):
        ppocr_hip._teacher(ppocr_hip.TopLogits(torch.zeros(2, 3), torch.zeros(2, 2, dtype=torch.int32)), 2)


def test_the_binding_reads_strides():
    r = ppocr_hip._rows(torch.zeros(5, 7, 13)[:, :, :9], "logits")
    assert (r.rows, r.classes, r.stride, r.type) == (35, 9, 13, 0)
    r = ppocr_hip._rows(torch.zeros(6, dtype=torch.bfloat16), "logits")
    assert (r.rows, r.classes, r.stride, r.type) == (1, 6, 6, 1)


def test_rules_check_their_rows():
    i32 = dict(dtype=torch.int32)
    r = ppocr_hip.LogitRules(40, masks=torch.zeros(2, 2, **i32), row_mask=torch.zeros(5, **i32))
    r.check(5)
    with pytest.raises(ValueError, match="row_mask is for 5 rows"):
        r.check(4)
    with pytest.raises(ValueError, match="words"):
        ppocr_hip.LogitRules(40, masks=torch.zeros(2, 1, **i32))
    with pytest.raises(ValueError, match="bias must be"):
        ppocr_hip.LogitRules(40, bias=torch.zeros(2, 41))
    r = ppocr_hip.LogitRules(40, history=torch.zeros(7, **i32), history_offsets=torch.zeros(4, dtype=torch.int64))
    r.check(3)
    with pytest.raises(ValueError, match="history_offsets"):
        r.check(4)


@pytest.mark.parametrize("classes", [1, 31, 32, 33, 100])
def test_class_masks_hold_one_bit_a_class(classes):
    allowed = torch.from_numpy(np.random.default_rng(classes).random((3, classes)) < 0.5)
    words = ppocr_hip.class_masks(allowed)
    assert words.dtype == torch.int32 and words.shape == (3, -(-classes // 32))
    assert np.array_equal(oracle.allowed_bits(words.numpy(), classes), allowed.numpy())


# ------------------------------------------------------------------- oracle

@pytest.mark.parametrize("with_rest", [True, False])
@pytest.mark.parametrize("tau", [0.7, 2.0])
def test_the_plain_gradient_agrees_with_differences(tau, with_rest):
    rng = np.random.default_rng(5)
    x = rng.normal(size=(3, 17)) * 2
    values, indices, rest, _ = oracle.top((x + rng.normal(size=x.shape)).astype(np.float32), 4, tau)
    indices[1, 2] = indices[1, 0]  # named twice
    indices[2, :3] = -1
    rest = rest if with_rest else None
    g = rng.uniform(0.5, 1.5, 3).astype(np.float32)
    _, _, grad, *_ = oracle.distill(x, values, indices, rest, tau, g)
    h = 1e-6
    for c in range(x.shape[1]):
        d = np.zeros_like(x)
        d[:, c] = h
        up, down = (oracle.distill(x + s * d, values, indices, rest, tau)[0] for s in (1, -1))
        # Truncation is h^2 times a third derivative of order 1, the losses' own
        # rounding 1e-15 / h.
        assert np.allclose(g * (up - down) / (2 * h), grad[:, c], atol=1e-8)

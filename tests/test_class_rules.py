"""Class rules of recognizers and of the engine: refusals, before any file is
read or device touched."""

import ctypes

import numpy as np
import pytest

import ppocr_hip


def load_with(options, size=2):
    L = ppocr_hip.lib()
    out = ctypes.c_void_p()
    shape = (ctypes.c_size_t * 4)(1, 3, 48, 320)
    code = L.ppocr_hip_recognizer_load_with(None, b"/nowhere", size, shape, 0,
                                            None if options is None else ctypes.byref(options), None, ctypes.byref(out))
    assert not out.value
    return code, L.ppocr_hip_last_error().decode()


def options(output=0, top_k=0, rules=None):
    return ppocr_hip._RecognizerOptions(output, top_k, None if rules is None else ctypes.pointer(rules))


@pytest.mark.parametrize("opts,text", [
    (None, "options are null"),
    (options(output=3), "unknown recognizer output"),
    (options(output=2), "top_k"),
    (options(output=2, top_k=65), "top_k"),
    (options(output=0, top_k=1), "top_k"),
    (options(output=1, top_k=5), "top_k"),
    (options(), "context is null"),
    (options(output=2, top_k=64), "context is null"),
])
def test_options_are_checked(opts, text):
    code, message = load_with(opts)
    assert code == 10 and text in message, message


def test_rules_are_checked():
    good = np.zeros(6906, np.float32)
    allowed = np.zeros(6906, bool)
    rules, kept = ppocr_hip._class_rules(6906, allowed, good)
    code, message = load_with(options(rules=rules))
    assert code == 10 and "blank" in message
    allowed[0] = True
    rules, kept = ppocr_hip._class_rules(6906, allowed, good)
    code, message = load_with(options(rules=rules))
    assert code == 10 and "context is null" in message
    code, message = load_with(options(rules=rules), size=0)  # medium: 18710 classes
    assert code == 10 and "18710" in message
    for bad in (np.nan, np.inf, -np.inf):
        good[77] = bad
        rules, kept = ppocr_hip._class_rules(6906, allowed, good)
        code, message = load_with(options(rules=rules))
        assert code == 10 and "non-finite" in message


def test_engine_refuses_without_a_handle():
    L = ppocr_hip._engine_lib()
    assert L.ppocr_hip_engine_set_rules(None, None) == 10


@pytest.mark.parametrize("kw", [dict(allowed=np.ones(5, bool), bias=None), dict(allowed=None, bias=np.ones(5))])
def test_the_binding_checks_lengths(kw):
    with pytest.raises(ValueError, match="needs 6906"):
        ppocr_hip._class_rules(6906, **kw)


def test_the_binding_packs_masks():
    allowed = np.zeros(6906, bool)
    allowed[[0, 31, 32, 6905]] = True
    rules, (_, words) = ppocr_hip._class_rules(6906, allowed, None)
    assert words.size == 216 and rules.bias is None
    assert words[0] == 0x80000001 and words[1] == 1 and words[215] == 1 << (6905 % 32)
    assert sum(bin(int(w)).count("1") for w in words) == 4

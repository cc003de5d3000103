"""CPU checks of the log probabilities: calls that do not hold are refused before any device work."""

import importlib

import pytest

FAKE = 1 << 20


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("hy_b200.logprobs")._library()


def _call(lib, logits=FAKE, rows=2, vocab=1000, stride=1000, dtype=0, device=0, tokens=FAKE, per_row=1, top=5, lp=FAKE,
          entropy=FAKE, ids=FAKE, alternatives=FAKE):
    return lib.hy_token_logprobs(logits, rows, vocab, stride, dtype, device, tokens, per_row, top, lp, entropy, ids,
                                 alternatives, None)


@pytest.mark.parametrize("over,message", [
    (dict(rows=-1), "rows"), (dict(dtype=2), "F32 or BF16"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1), "vocab"),
    (dict(per_row=-1), "negative"), (dict(top=-1), "top"), (dict(top=65), "top"), (dict(top=5, vocab=4), "top"),
    (dict(stride=-1), "negative"), (dict(device=-1), "device"), (dict(logits=None), "null"), (dict(tokens=None), "null"),
    (dict(lp=None), "null"), (dict(ids=None), "null"), (dict(alternatives=None), "null"), (dict(logits=FAKE + 2), "aligned"),
    (dict(dtype=1, logits=FAKE + 1), "aligned"), (dict(rows=1 << 28, top=64), "2^31"),
])
def test_refusals(lib, over, message):
    assert _call(lib, **over) in (1, 4)
    assert message in lib.hy_last_error().decode()


def test_empty_call(lib):
    assert _call(lib, rows=0, logits=None, tokens=None, lp=None, ids=None, alternatives=None) == 0


def test_the_context_form_needs_a_context(lib):
    assert lib.hy_lm_head_logprobs(None, FAKE, 1, None, 0, None, None, None, None) == 1
    assert b"null" in lib.hy_last_error()

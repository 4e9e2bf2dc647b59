"""The sticky device word has a bit per kind of error; reading one loses none of the others."""

import pytest
import torch

import prlstm_amd
from prlstm_amd import _lib

GAVE_UP, BEYOND = 1, 2


@pytest.mark.parametrize("word", [GAVE_UP, BEYOND, GAVE_UP | BEYOND, 8, 8 | BEYOND])
def test_check_errors_names_every_bit(monkeypatch, word):
    monkeypatch.setattr(_lib, "device_errors", lambda device=None, clear=True: word)
    with pytest.raises(RuntimeError, match=f"device error word {word:#x}") as e:
        prlstm_amd.check_errors()
    text = str(e.value)
    assert ("gave up a wait" in text) == bool(word & GAVE_UP), text
    assert ("beyond the vocabulary" in text) == bool(word & BEYOND), text
    assert ("unknown" in text) == bool(word & 8), text


def test_check_errors_of_a_clear_word(monkeypatch):
    monkeypatch.setattr(_lib, "device_errors", lambda device=None, clear=True: 0)
    prlstm_amd.check_errors()

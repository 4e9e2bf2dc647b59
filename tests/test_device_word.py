"""The sticky device word has a bit per kind of error; reading one loses none of the others."""

import pytest
import torch

import prlstm_amd
from prlstm_amd import _lib, functional

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


class FakeLibrary:
    """The error entry points over a word that is held here."""

    def __init__(self, word, flag=0):
        self.word, self.flag = word, flag

    def call(self, name, *args):
        if name == "hsl_poll_error":
            args[1]._obj.value = self.flag
        elif name == "hsl_device_errors":
            args[0]._obj.value = self.word
            self.word = 0 if args[1] else self.word
        elif name == "hsl_clear_device_errors":
            self.word &= ~args[0]
        else:
            raise AssertionError(name)


@pytest.mark.parametrize("others", [0, BEYOND])
def test_polling_a_call_clears_its_own_bit_alone(monkeypatch, others):
    """With checks after every recurrent call, a timed-out wait is raised there; an error of another
    kind stays for check_errors."""
    fake = FakeLibrary(GAVE_UP | others, flag=1)
    monkeypatch.setattr(_lib, "call", fake.call)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(functional, "_debug_checks", True)
    with pytest.raises(RuntimeError, match="timed out"):
        functional._poll(torch.zeros(1), "cuda:0")
    assert fake.word == others
    fake.flag = 0
    functional._poll(torch.zeros(1), "cuda:0")
    assert fake.word == others


@pytest.mark.gpu
def test_bits_are_cleared_one_by_one(dev):
    prlstm_amd.check_errors(dev)
    prlstm_amd.embedding(torch.tensor([9], device=dev), torch.zeros(4, 3, device=dev))
    assert _lib.device_errors(dev, clear=False) == BEYOND
    _lib.clear_device_errors(GAVE_UP, dev)
    assert _lib.device_errors(dev, clear=False) == BEYOND
    _lib.clear_device_errors(BEYOND, dev)
    assert _lib.device_errors(dev) == 0

"""core.check_device_status reads and clears the status of every kernel with bounded waits before it raises: a stand-in for
the library holds the words, no GPU is needed."""
import contextlib

import pytest
import torch


class _Words:
    """grws_spmm_check, grws_linear_ce_check: GRWS_ERR_DEVICE and a message if the word is set, which is cleared."""

    def __init__(self, spmm, ce):
        self.words, self.message = {"spmm": spmm, "ce": ce}, ""

    def _check(self, name):
        if not self.words[name]:
            return 0
        self.words[name], self.message = 0, f"a {name} launch gave up waiting"
        return -5

    def grws_spmm_check(self, stream):
        return self._check("spmm")

    def grws_linear_ce_check(self, stream):
        return self._check("ce")

    def grws_last_error(self):
        return self.message.encode()


@pytest.mark.parametrize("spmm,ce", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_every_word_is_read_and_cleared(monkeypatch, spmm, ce):
    from graph_rws_b200 import core
    from graph_rws_b200.core import _native
    words = _Words(spmm, ce)
    monkeypatch.setattr(_native, "lib", lambda: words)
    monkeypatch.setattr(core, "_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    if spmm or ce:
        with pytest.raises(RuntimeError) as e:
            core.check_device_status("cuda:0")
        assert ("spmm launch" in str(e.value)) == bool(spmm) and ("ce launch" in str(e.value)) == bool(ce) and "-5" in str(e.value)
    assert words.words == {"spmm": 0, "ce": 0}
    core.check_device_status("cuda:0")

"""Prompts that do not fit the cache are refused before any device work, whichever prefill there is."""
import numpy as np
import pytest


@pytest.mark.parametrize("prefill", ["steps", "batched"])
@pytest.mark.parametrize("ids", [[], [1] * 65, np.ones(65, np.int32)])
def test_logits_refuses_what_does_not_fit(prefill, ids):
    import limited
    import synth
    import w4format
    e = object.__new__(limited.Engine)                       # an engine without a device will do
    e.cfg, e.prefill_mode = w4format.Config(synth.tiny_arch()), prefill
    e.cfg.max_context = 64

    def device(*a):
        raise AssertionError("a token was stepped")
    e._prefill_token = e._prefill_buffers = e._empty_cache = device
    with pytest.raises(ValueError, match="prompt tokens for a 64-token context"):
        e.logits(ids)

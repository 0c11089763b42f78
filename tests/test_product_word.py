"""The error word of a product whose later launch is refused: the first one runs with it, so it is on record and not given out again."""

import pytest
import torch

from flashrnn_b200 import _lib, projection


def test_the_word_is_on_record_before_a_refusal_is_raised(monkeypatch):
    class Refuses:
        frnn_b200_product_forward = staticmethod(lambda *args: -2)

        def __getattr__(self, name):
            return getattr(lib, name)

    lib = _lib.load()
    events = []
    x, w = torch.zeros((300, 8192), dtype=torch.bfloat16), torch.zeros((256, 8192), dtype=torch.bfloat16)
    plan = _lib.product_plan(300, 256, 8192, -1)
    assert plan.forward_waits and plan.forward_work_bytes > 0       # tiles, then the pass that joins their parts
    monkeypatch.setattr(_lib, "load", Refuses)
    monkeypatch.setattr(projection, "poll_errors", lambda: None)
    monkeypatch.setattr(projection, "_stream", lambda device: 0)
    monkeypatch.setattr(projection, "_launch_word", lambda device: (128, "word"))
    monkeypatch.setattr(projection, "_launched", lambda word, what: events.append((word, what)))
    with pytest.raises(RuntimeError, match="frnn_b200_product_forward failed"):
        projection._product_forward(x, w, None, None, None, False)
    assert events == [("word", "frnn_b200_product_forward")]

"""The look for errors at the start of every call waits for nothing; poll_errors(block=True) does."""

import pytest
import torch

from flashrnn_b200 import functional as F


class Event:
    done, waited = False, 0

    def query(self):
        return self.done

    def synchronize(self):
        self.waited += 1
        self.done = True


class Block:
    """As F._ErrorBlock, one launch tracked, with an event of the test's"""

    def __init__(self, event):
        self.event, self.words, self.names, self.closed, self.given = event, torch.zeros((64, 32), dtype=torch.int32), ["launch"], 0, 1

    close = F._ErrorBlock.close


@pytest.fixture
def event(monkeypatch):
    monkeypatch.setattr(F, "_capturing", lambda: False)
    monkeypatch.setattr(F, "_last_poll", 0.0)
    monkeypatch.setattr(F, "_pending_errors", [])
    monkeypatch.setattr(F, "_captured_errors", [])
    monkeypatch.setattr(torch.cuda, "Event", Event)
    event = Event()
    monkeypatch.setattr(F, "_blocks", {"thread and stream": Block(event)})
    return event


def test_a_call_does_not_wait_for_the_launches_before_it(event, monkeypatch):
    asked = []
    word = torch.zeros(32, dtype=torch.int32)
    monkeypatch.setattr(F, "_captured_errors", [(word, "captured")])
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: asked.append(device))
    F.poll_errors()
    assert event.waited == 0 and not asked and [p[0] for p in F._pending_errors] == [event]
    F.poll_errors(block=True)
    assert event.waited == 1 and asked == [word.device] and not F._pending_errors


def test_it_waits_where_there_are_no_blocks_too(event, monkeypatch):
    monkeypatch.setattr(F, "_pending_errors", [(event, torch.zeros(32, dtype=torch.int32), "launch")])
    monkeypatch.setattr(F, "_blocks", {})
    F.poll_errors()
    assert event.waited == 0 and len(F._pending_errors) == 1
    F.poll_errors(block=True)
    assert event.waited == 1 and not F._pending_errors

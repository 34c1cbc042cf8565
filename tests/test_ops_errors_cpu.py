"""The plug-in's device error word on the host side, without a GPU: read back between calls, left alone under capture."""
import pytest
import torch

from psgd_pro_b200 import ops


class Event:
    def __init__(self, capturing):
        self.capturing, self.asked = capturing, 0

    def query(self):
        self.asked += 1
        if self.capturing:  # as CUDA does: asking an event invalidates the capture
            raise RuntimeError("operation not permitted when stream is capturing")
        return True


@pytest.mark.parametrize("capturing", [False, True])
@pytest.mark.parametrize("flags", [0, 1])
def test_an_earlier_error_is_raised_except_under_capture(monkeypatch, capturing, flags):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    words = ops._ErrorWords()
    dev = torch.device("cuda", 0)
    words.pending(dev)  # nothing has been launched
    words.word[0], words.host[0] = torch.zeros(1, dtype=torch.int32), torch.tensor([flags], dtype=torch.int32)
    words.event[0] = Event(capturing)
    if flags and not capturing:
        with pytest.raises(RuntimeError, match="0x1"):
            words.pending(dev)
    else:
        words.pending(dev)
    assert words.event[0].asked == (0 if capturing else 1)
    if capturing:
        words.after(dev)  # neither copied nor recorded
        assert words.event[0].asked == 0 and int(words.host[0]) == flags

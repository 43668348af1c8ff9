"""Calls of the attention over the hot rows as its documentation allows them, around the launch itself: where errCodes go,
which rows a slot may name, types, workspaces, and launches that give up."""
import pytest
import torch

from test_gpu_attend import Case

pytestmark = pytest.mark.gpu


class Spy:
    """A launch module that notes the error words of the attention's launches."""

    def __init__(self, k):
        self._k, self.words = k, []

    def __getattr__(self, name):
        return getattr(self._k, name)

    def attend_hot(self, *args, **named):
        self.words.append(named["err_word"])
        return self._k.attend_hot(*args, **named)


def test_a_tensor_as_error_word_is_the_one_that_the_launch_gets():
    c = Case(40)
    c.co._k = spy = Spy(c.co._k)
    device, pinned = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, pin_memory=True)
    for word in (device, pinned):
        c.check(*c.call(err_word=word))
    c.call()
    assert spy.words == [device.data_ptr(), pinned.data_ptr(), c.co._attend_err_at]
    assert device.item() == 0 and pinned.item() == 0
    with pytest.raises(ValueError, match="pinned"):
        c.call(err_word=torch.zeros(1, dtype=torch.int32))


def test_a_tensor_as_error_word_in_a_captured_call():
    c = Case(41)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.call(err_word=word)
    graph.replay()
    torch.cuda.synchronize()
    c.check(*out)
    assert word.item() == 0

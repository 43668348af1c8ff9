"""Arguments of XdsOffloadCoordinator.attend without a GPU: what reaches the launch, and what is refused."""
import pytest
import torch

from kv_offload_proto_b200.offload import XdsOffloadCoordinator

REQS, HEADS, ROWS = 2, 4, 16


class Launches:
    """In the place of the launch module: keeps what a call of attend passes on."""

    def __init__(self):
        self.calls = []

    def attend_workspace(self, *args):
        return 0

    def attend_hot(self, *args, **named):
        self.calls.append((args, named))


class HostCoordinator(XdsOffloadCoordinator):
    _require_cuda = False


def coordinator(k=8):
    co = HostCoordinator("cpu", 1, REQS, ROWS, k, REQS, 64)
    co._req_pool_indices = torch.arange(REQS)
    co._k = Launches()
    return co


def attend(co, **change):
    args = dict(q=torch.zeros((REQS, HEADS, 576), dtype=torch.float16),
                hot_row_base=torch.zeros((REQS * ROWS, 576), dtype=torch.float16), hot_req_stride_rows=ROWS, scale=0.07)
    args.update(change)
    return co.attend(args.pop("q"), args.pop("hot_row_base"), **args)


@pytest.mark.parametrize("value", [0, 0x103])
def test_an_error_word_is_passed_on_by_its_address(value):
    co, word = coordinator(), torch.full((1,), value, dtype=torch.int32)
    attend(co, err_word=word.data_ptr())
    assert co._k.calls[-1][1]["err_word"] == word.data_ptr()
    attend(co, err_word=word)
    assert [c[1]["err_word"] for c in co._k.calls] == [word.data_ptr()] * 2 and word.item() == value


@pytest.mark.parametrize("word", [torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32),
                                  torch.zeros(0, dtype=torch.int32), torch.zeros(1), None, "0"])
def test_error_words_of_other_kinds_are_refused(word):
    co = coordinator()
    with pytest.raises(ValueError, match="err_word"):
        attend(co, err_word=word)
    assert not co._k.calls


def shape_of(call):
    """(hot_req_stride_rows, hot_rows, report_slots) of a launch."""
    args, named = call
    return args[5], args[6], named["report_slots"]


@pytest.mark.parametrize("change, want", [
    (dict(), (ROWS, ROWS, True)),
    (dict(hot_rows=12), (ROWS, 12, False)),
    (dict(topk_device_slots=torch.zeros((REQS, 5), dtype=torch.int32)), (ROWS, ROWS, False)),
    (dict(hot_req_stride_rows=0), (0, REQS * ROWS, True)),         # shared: all that the tensor holds
    (dict(hot_req_stride_rows=0, hot_rows=20), (0, 20, False)),
    (dict(hot_req_stride_rows=0, hot_row_base=1 << 20), (0, ROWS, True)),  # an address tells no size
    (dict(hot_req_stride_rows=0, row_format="int8", hot_row_base=torch.zeros((30, 656), dtype=torch.uint8)), (0, 30, True)),
])
def test_which_rows_a_slot_may_name(change, want):
    co = coordinator()
    attend(co, **change)
    assert shape_of(co._k.calls[-1]) == want


def test_shared_rows_hold_the_buffer():
    with pytest.raises(ValueError, match="hot rows must"):
        attend(coordinator(), hot_req_stride_rows=0, hot_row_base=torch.zeros((ROWS - 1, 576), dtype=torch.float16))


RAW, STORED = (REQS * ROWS, 576), (REQS * ROWS, 656)


@pytest.mark.parametrize("hot, row_format", [
    (torch.zeros(RAW, dtype=torch.bfloat16), "raw"), (torch.zeros(RAW), "raw"), (torch.zeros(RAW, dtype=torch.float64), "raw"),
    (torch.zeros(RAW, dtype=torch.float16), "e4m3"), (torch.zeros(STORED), "int8"),
])
def test_hot_rows_of_another_type_are_refused(hot, row_format):
    co = coordinator()
    with pytest.raises(ValueError, match="hot rows of row_format"):
        attend(co, hot_row_base=hot, row_format=row_format)
    assert not co._k.calls


@pytest.mark.parametrize("hot, row_format", [
    (torch.zeros(RAW, dtype=torch.float16), "raw"), (torch.zeros(RAW, dtype=torch.int16), "raw"),
    (torch.zeros((REQS * ROWS, 1152), dtype=torch.uint8), "raw"), (torch.zeros((REQS * ROWS, 288), dtype=torch.int32), "raw"),
    (torch.zeros(STORED, dtype=torch.uint8), "int8"), (torch.zeros(STORED, dtype=torch.int8), "e4m3"),
    (torch.zeros((REQS * ROWS, 164), dtype=torch.int32), "e4m3"),
])
def test_hot_rows_as_bytes_and_integers(hot, row_format):
    co = coordinator()
    attend(co, hot_row_base=hot, row_format=row_format)
    assert co._k.calls[-1][0][4] == hot.data_ptr()


def test_bf16_rows_with_a_bf16_q():
    co = coordinator()
    attend(co, q=torch.zeros((REQS, HEADS, 576), dtype=torch.bfloat16), hot_row_base=torch.zeros(RAW, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="hot rows of row_format"):
        attend(co, q=torch.zeros((REQS, HEADS, 576), dtype=torch.bfloat16))
    assert len(co._k.calls) == 1


def test_the_scale_has_no_default():
    co = coordinator()
    with pytest.raises(ValueError, match="scale must be given"):
        attend(co, scale=None)
    assert not co._k.calls
    attend(co, scale=192 ** -0.5)
    assert co._k.calls[-1][0][28] == 192 ** -0.5


def test_a_workspace_is_contiguous_bytes():
    co, room = coordinator(), torch.zeros((64, 2), dtype=torch.uint8)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        attend(co, workspace=room[:, 0])  # what lies between its bytes is not its own
    assert not co._k.calls
    for ws in (room, torch.zeros(32, dtype=torch.float32)):
        attend(co, workspace=ws)
        assert co._k.calls[-1][0][19:21] == (ws.data_ptr(), 128)


def test_pool_indices_with_gaps_are_refused():
    co = coordinator()
    co._req_pool_indices = torch.arange(2 * REQS)[::2]
    with pytest.raises(ValueError, match="req_pool_indices must be contiguous"):
        attend(co)
    assert not co._k.calls


def test_pool_indices_elsewhere_are_refused():
    co = coordinator()
    co._req_pool_indices = torch.zeros(REQS, dtype=torch.int64, device="meta")
    with pytest.raises(ValueError, match="every tensor must be on"):
        attend(co)
    assert not co._k.calls

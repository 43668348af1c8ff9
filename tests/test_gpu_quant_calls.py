"""DevicePool calls over pools of 8-bit rows as their documentation allows them, around the launches: refused layer-steps,
the path that a step ran, and types."""
import pytest
import torch

from gpu_util import kv
from kv_offload_proto_b200.graph import StepGraph
from kv_offload_proto_b200.offload import XdsOffloadCoordinator
from kv_offload_proto_b200.pool import DevicePool

pytestmark = pytest.mark.gpu

R, CTX, K, DBS = 2, 128, 20, 64


class Step:
    """A pool with a coordinator whose next layer-step has misses."""

    def __init__(self, row_format="int8", layers=1, **kw):
        kv()
        self.pool = DevicePool(0, layers, R * CTX, 1152, 1, segment_devices=(0,), row_format=row_format, **kw)
        self.co = XdsOffloadCoordinator("cuda", layers, R, DBS, K, R, CTX)
        self.co.admit_all([CTX] * R, [r * CTX for r in range(R)])
        self.co.set_batch(torch.arange(R, device="cuda"), torch.full((R,), CTX, dtype=torch.int32, device="cuda"))
        g = torch.Generator().manual_seed(3)
        self.rows = torch.randn((layers, R * CTX, 576), generator=g).half().cuda()
        self.pool.wait(self.pool.batch_write_alllayers(0, R * CTX, self.rows, self.rows.stride(0) * 2))
        self.hot = torch.zeros((R * DBS + 1, 576), dtype=torch.float16, device="cuda")
        self.topk = (torch.arange(K, device="cuda", dtype=torch.int32) + DBS - 4).repeat(R, 1)

    def state(self):
        torch.cuda.synchronize()
        co = self.co
        return [x.clone() for x in (co.device_buffer_tokens, co.device_buffer_visited, co.device_buffer_ht, co.sieve_hand,
                                    co.top_k_device_slots, co.is_miss, self.hot)]


@pytest.mark.parametrize("change, message", [
    (dict(hot=2), "16-byte"), (dict(block_dim=9), "blockDim"), (dict(block_dim=0), "blockDim"), (dict(err_word=2), "err_word"),
    (dict(hot=None), "address is 0"),
])
def test_a_refused_layer_step_leaves_the_tables(change, message):
    s = Step()
    before = s.state()
    args = dict(hot_req_stride_rows=DBS)
    args.update(change)
    hot = args.pop("hot", 0)
    with pytest.raises(RuntimeError, match=message):
        s.pool.sieve_and_read(s.co, 0, s.topk, 0 if hot is None else s.hot.data_ptr() + hot, **args)
    for a, b in zip(before, s.state()):
        assert torch.equal(a, b)
    s.pool.wait(s.pool.sieve_and_read(s.co, 0, s.topk, s.hot, hot_req_stride_rows=DBS))
    assert int(s.co.miss_count()) == R * (K - 4)
    s.pool.destroy()


def test_the_path_of_a_step():
    raw, quant = Step("raw"), Step("int8")
    raw.pool.wait(raw.pool.sieve_and_read(raw.co, 0, raw.topk, raw.hot, hot_req_stride_rows=DBS, path="coop"))
    assert kv().last_step_path() == "coop"
    assert StepGraph(quant.pool, quant.co, [quant.hot], hot_req_stride_rows=DBS).path == "split"
    raw.pool.wait(raw.pool.sieve_and_read(raw.co, 0, raw.topk, raw.hot, hot_req_stride_rows=DBS, path="coop"))
    quant.pool.wait(quant.pool.sieve_and_read(quant.co, 0, quant.topk, quant.hot, hot_req_stride_rows=DBS, copy_wait_polls=5))
    assert kv().last_step_path() == "split"
    raw.pool.destroy()
    quant.pool.destroy()


def test_a_step_in_one_call_is_the_two_calls():
    one, two = Step("e4m3", layers=2), Step("e4m3", layers=2)
    for layer in (0, 1, 0):
        one.topk += 3
        two.topk += 3
        one.pool.wait(one.pool.sieve_and_read(one.co, layer, one.topk, one.hot, hot_req_stride_rows=DBS))
        two.co.sieve_update(layer, two.topk)
        two.pool.wait(two.pool.batch_read(layer, two.topk, two.co._req_pool_indices, two.co.req_host_base,
                                          two.co.top_k_device_slots, two.co.is_miss, two.co.num_real, two.hot, R, K,
                                          hot_req_stride_rows=DBS))
        for a, b in zip(one.state(), two.state()):
            assert torch.equal(a, b)
        assert int(one.co.miss_count()) > 0
    one.pool.destroy()
    two.pool.destroy()


@pytest.mark.parametrize("room", [0, 2])
def test_a_captured_attention_reports_to_its_step(room):
    """The step's error word is the attention's too: generated tokens without a place among the hot rows are in error()."""
    s = Step("raw")
    s.co.set_batch(torch.arange(R, device="cuda"), torch.full((R,), CTX + 2, dtype=torch.int32, device="cuda"))
    stride = s.co.padded_buffer_size + room
    hot = torch.zeros((R * stride, 576), dtype=torch.float16, device="cuda")
    q = torch.randn((R, 8, 576), device="cuda").half()
    word = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    graph = StepGraph(s.pool, s.co, [hot], hot_req_stride_rows=stride, err=word,
                      after_layer=lambda layer: s.co.attend(q, hot, hot_req_stride_rows=stride, scale=0.1, err_word=word))
    s.topk[:, -2:] = torch.tensor([CTX, CTX + 1], device="cuda")
    graph.topk[0].copy_(s.topk)
    assert graph.error() == 0
    for _ in range(2):
        graph.replay()
        assert graph.error() == (0 if room else 0x104)
    graph.clear_error()
    assert word.item() == 0 and s.co.attend_error() == 0
    for bad in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="err must be"):
            StepGraph(s.pool, s.co, [hot], hot_req_stride_rows=stride, err=bad)
    del graph
    s.pool.destroy()

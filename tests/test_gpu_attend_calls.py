"""Calls of the attention over the hot rows as its documentation allows them, around the launch itself: where errCodes go,
which rows a slot may name, types, workspaces, and launches that give up."""
import math

import pytest
import torch

import quant_model
from gpu_util import kv
from kv_offload_proto_b200.offload import XdsOffloadCoordinator
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


def with_generated_tokens(rows, shared):
    """A step in which SIEVE names tokens behind the prompt: a buffer of 20 slots (32 padded), a prompt of 40, three more."""
    kv()
    dbs, prefill, new, K, R, H = 20, 40, 3, 12, 2, 5
    co = XdsOffloadCoordinator("cuda", 1, R, dbs, K, R, 64)
    co.admit_all([prefill] * R, [0] * R)
    co.set_batch(torch.arange(R, device="cuda"), torch.full((R,), prefill + new, dtype=torch.int32, device="cuda"))
    co.sieve_update(0, torch.tensor([[0, 1, 2, 40, 41, 42, 3, 4, 5, 6, -1, 7], [40, 0, 9, 8, 7, 6, 5, 4, 3, 2, 1, 42]],
                                    dtype=torch.int32, device="cuda"))
    assert co.padded_buffer_size == 32 and int((co.top_k_device_slots >= 32).sum()) == 5
    c = Case.__new__(Case)
    c.B, c.T, c.H, c.K, c.D, c.rows, c.scale, c.co = R, 1, H, K, 0, rows, 0.07, co
    g = torch.Generator(device="cuda").manual_seed(1)
    c.q = torch.randn((R, 1, H, 576), generator=g, device="cuda").half()
    c.read = torch.randn((rows if shared else R * rows, 576), generator=g, device="cuda").half()
    c.draft = c.tree = None
    c.idx, c.stride, c.slots = co._req_pool_indices, 0 if shared else rows, co.top_k_device_slots
    return c


@pytest.mark.parametrize("shared", [False, True])
def test_tokens_generated_since_the_prompt_are_keys(shared):
    c = with_generated_tokens(35, shared)
    c.check(*c.co.attend(c.q, c.read, hot_req_stride_rows=c.stride, scale=c.scale))
    torch.cuda.synchronize()
    assert c.co.attend_error() == 0


@pytest.mark.parametrize("rows", [20, 34])
@pytest.mark.parametrize("shared", [False, True])
def test_generated_tokens_without_a_row_are_reported(shared, rows):
    """The last (or every) generated token has no row: the outputs are without it, and the next call raises."""
    c = with_generated_tokens(rows, shared)
    out = c.co.attend(c.q, c.read, hot_req_stride_rows=c.stride, scale=c.scale)
    torch.cuda.synchronize()
    c.check(*out)
    with pytest.raises(RuntimeError, match="padded_buffer_size.*0x104"):
        c.co.attend(c.q, c.read, hot_req_stride_rows=c.stride, scale=c.scale)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.co.attend(c.q, c.read, hot_req_stride_rows=c.stride, scale=c.scale, err_word=word)
    assert word.item() == 0x104 and c.co.attend_error() == 0


@pytest.mark.parametrize("change", [dict(hot_rows=20), dict(topk_device_slots="copy"), dict(num_real=0), dict(idx=7)])
def test_slots_left_out_on_purpose_are_not_reported(change):
    """hot_rows given, a list that is not SIEVE's own, batch rows behind num_real, and requests without hot rows."""
    c = with_generated_tokens(20, False)
    args = dict(hot_req_stride_rows=20, scale=c.scale)
    if "hot_rows" in change:
        args.update(change)
    if "topk_device_slots" in change:
        args["topk_device_slots"] = c.slots.clone()
    if "num_real" in change:
        c.co.num_real.fill_(0)
    if "idx" in change:
        c.idx.fill_(7)  # no such pool row
    out = c.co.attend(c.q, c.read, **args)
    torch.cuda.synchronize()
    assert c.co.attend_error() == 0
    if "num_real" not in change:
        c.check(*out)


@pytest.mark.parametrize("shape", [
    dict(B=64, T=1, H=128, K=2048, rows=2048, fmt="raw"),
    dict(B=40, T=1, H=128, K=2048, rows=2048, fmt="e4m3"),         # lists that are cut and joined
    dict(B=20, T=12, H=16, K=2048, rows=2048, D=12, fmt="int8", dtype="bf16"),
    dict(B=300, T=1, H=16, K=500, rows=512, fmt="raw", holes=0.3),  # several requests a run
], ids=lambda s: "-".join(map(str, s.values())))
def test_a_launch_whose_waits_run_out_says_so_and_leaves_nothing_behind(shape):
    """A limit shorter than a tile takes: the launch ends with errCode 0x103, and the launch behind it, which starts as it
    ends, is right. Limits near a tile's time give up in the middle of the work, or not at all."""
    c = Case(42, **shape)
    want = c.call()
    c.check(*want)
    for clocks in (1, 1, 200, 800, 1500, 2500, 3500, 5000, 8000, 20000):
        word = torch.zeros(1, dtype=torch.int32, device="cuda")
        cut = c.call(err_word=word, wait_clocks=clocks)
        behind = c.call()
        code = word.item()
        assert code == 0x103 if clocks == 1 else code in (0, 0x103)
        if code == 0:
            assert torch.equal(cut[0], want[0]) and torch.equal(cut[1], want[1])
        assert torch.equal(behind[0], want[0]) and torch.equal(behind[1], want[1])
    assert c.co.attend_error() == 0
    c.call(wait_clocks=1)  # by default the next call raises it
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="0x103"):
        c.call()
    c.check(*c.call())


@pytest.mark.parametrize("K", [2 ** 16 + 1, 100_000])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("first", [True, False])
def test_the_tail_of_a_long_list_counts(first, dtype, K):
    """One key whose value is 0 takes nearly all, and n = K - 1 keys of value 1 are e^-20.25 (2^-29.2) of it each: out is
    t = n e^-20.25 / (1 + n e^-20.25) in every dimension. Probabilities are rounded (u, and in fp16 by 2^-39 of the
    largest each: all the same way, n 2^-39), the output is (u t, and half an fp16 step below the normal numbers), the
    fp32 sums over K keys are off by K 2^-23 of t, and the exponent of 2 (29.2, an fp32 number) by 2^-20 of t at the most."""
    c = Case(43, B=148, H=4, K=K, rows=4, holes=0, dtype=dtype)  # a whole list to an SM
    c.q.zero_()
    c.q[..., 575] = 1
    c.hot.zero_()
    c.hot.view(148, 4, 576)[:, 0, :512] = 1
    c.hot.view(148, 4, 576)[:, 1, 575] = 20.25
    c.slots.zero_()
    c.slots[:, 0 if first else K - 1] = 1
    out, lse = c.call(scale=1.0)
    n = K - 1
    t = n * math.exp(-20.25) / (1 + n * math.exp(-20.25))
    u = torch.finfo(c.q.dtype).eps / 2
    tol = 2 * u * t + n * 2.0 ** -39 + K * 2.0 ** -23 * t + 2.0 ** -20 * t + (2.0 ** -25 if dtype == "fp16" else 0)
    assert (out.double() - t).abs().max() <= tol
    assert (lse.double() - (20.25 + math.log1p(n * math.exp(-20.25)))).abs().max() <= 2.0 ** -17


def test_probabilities_of_a_list_of_two_to_the_sixteen():
    """The longest list of the small lift: every tail key is off by 2^-29 of the largest at the most, 2^-13 in all."""
    K = 2 ** 16
    c = Case(44, B=148, H=2, K=K, rows=4, holes=0)
    c.q.zero_()
    c.q[..., 575] = 1
    c.hot.zero_()
    c.hot.view(148, 4, 576)[:, 0, :512] = 1
    c.hot.view(148, 4, 576)[:, 1, 575] = 20.25
    c.slots.zero_()
    c.slots[:, 0] = 1
    out, _ = c.call(scale=1.0)
    t = (K - 1) * math.exp(-20.25) / (1 + (K - 1) * math.exp(-20.25))
    assert (out.double() - t).abs().max() <= 2.0 ** -13 + 2.0 ** -10 * t


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("fmt", ["raw", "e4m3"])
@pytest.mark.parametrize("H, K", [(4, 70), (40, 3000)])  # a whole list, and one that is cut and joined
@pytest.mark.parametrize("dim", [3, 540])  # of a row's value, and of its rotary part, which only the score has
def test_a_listed_hot_row_that_is_not_finite(dim, H, K, fmt, bad):
    """It is NaN where the formula is (a score of NaN or +inf, or an infinite value times 0), and nowhere else."""
    c = Case(47, B=2, H=H, K=K, rows=200, fmt=fmt, dtype="bf16")
    c.slots[0, 1] = 17
    row = 17 + int(c.idx[0]) * 200
    c.read[row, dim] = bad
    if fmt == "raw":
        c.hot = c.read
    else:
        stored = quant_model.encode(c.read.cpu(), fmt, 512)
        c.hot, c.read = torch.from_numpy(stored).cuda(), quant_model.decode(stored, fmt, "bf16", 512).cuda()
    out, lse = c.call()
    for r in range(2):
        k = c.keys(r, 0)
        s = c.q[r, 0].double() @ k.T * c.scale
        want, log = (torch.softmax(s, 1) @ k[:, :512]).isnan(), torch.logsumexp(s, 1)
        assert torch.equal(out[r, 0].isnan(), want)
        assert torch.equal(lse[r, 0].isnan(), log.isnan() | (log == math.inf))
        assert want.any() == (r == 0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("H, K", [(4, 70), (40, 3000)])
def test_a_query_that_is_not_finite_harms_no_other(H, K, bad):
    c = Case(48, B=2, H=H, K=K, rows=200)
    want = c.call()
    c.q[1, 0, 2, 7] = bad
    out, lse = c.call()
    hit = torch.zeros_like(lse, dtype=torch.bool)
    hit[1, 0, 2] = True
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(out[~hit], want[0][~hit]) and torch.equal(lse[~hit], want[1][~hit])

"""GPU parity of the attention over the hot rows (attend_hot, XdsOffloadCoordinator.attend) with its
formula in 64 bits.

Tolerances count roundings. With u = eps / 2 of the rows' type, p the probabilities and v the values:
  * a score is a sum of 576 fp32 products: off by at most ds = 576 * 2^-23 * scale * max_k sum |q k|
    (2^-23: a matrix unit may cut instead of round), and its exponent, an fp32 number of magnitude up
    to max |s| / ln 2, by 2^-22 * max |s|; both move every p by that factor;
  * p is rounded to 16 bits for the second product (u), exp and the sums add some 2^-20, joining
    parts of a list adds two more fp32 factors, and the output is rounded once (u of the value, and
    half the smallest subnormal where fp16 has no normal number): with A = sum p |v|,
    |out - exact| <= u |exact| + tiny + (u + 2 (ds + 2^-22 max |s|) + 2^-19 + K 2^-23) A,
    K 2^-23 for the fp32 sum over K keys;
  * lse is off by ds + 2^-21 (max |s| + |lse| + 1) + K 2^-23.
"""
import math

import numpy as np
import pytest
import torch

import quant_model
from gpu_util import kv
from kv_offload_proto_b200.offload import XdsOffloadCoordinator, tree_masks
from quant_model import TORCH

pytestmark = pytest.mark.gpu


class Case:
    """One call's inputs and its exact outputs."""

    def __init__(self, seed, B=2, T=1, H=4, K=16, D=0, rows=64, own=False, fmt="raw", dtype="fp16", holes=0.1, pool=None,
                 shared=False, tree="random", spread=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        kv()
        self.B, self.T, self.H, self.K, self.D, self.rows, self.fmt, self.dtype = B, T, H, K, D, rows, fmt, dtype
        dt = TORCH[dtype]
        pool = B if pool is None else pool
        self.co = XdsOffloadCoordinator("cuda", 1, pool, rows, max(K, 1), B, 64)
        self.idx = torch.randperm(pool, generator=g, device="cuda")[:B]
        self.co.set_batch(self.idx, torch.full((B,), 64, dtype=torch.int32, device="cuda"))
        self.q = (torch.randn((B, T, H, 576), generator=g, device="cuda") * spread).to(dt)
        count = rows if shared else pool * rows
        x = torch.randn((count, 576), generator=g, device="cuda").to(dt)
        if fmt == "raw":
            self.hot = x
            self.read = x
        else:
            enc = quant_model.encode(x.cpu(), fmt, 512)
            self.hot = torch.from_numpy(enc).cuda()
            self.read = quant_model.decode(enc, fmt, dtype, 512).cuda()
        self.stride = 0 if shared else rows
        shape = (B, T, K) if own else (B, K)
        self.slots = torch.randint(0, rows, shape, generator=g, device="cuda", dtype=torch.int32)
        if K:
            self.slots[torch.rand(shape, generator=g, device="cuda") < holes] = -1
        self.draft = torch.randn((B, D, 576), generator=g, device="cuda").to(dt) if D else None
        self.tree = None
        if D and tree == "random":
            self.tree = torch.randint(-2 ** 62, 2 ** 62, (B, T), generator=g, device="cuda")
        self.scale = 0.07

    def call(self, **kw):
        args = dict(hot_req_stride_rows=self.stride, hot_rows=self.rows, row_format=self.fmt, scale=self.scale,
                    topk_device_slots=self.slots, draft_rows=self.draft, tree=self.tree)
        args.update(kw)
        q = args.pop("q", self.q)
        hot = args.pop("hot", self.hot)
        return self.co.attend(q, hot, **args)

    def keys(self, r, t):
        s = self.slots[r, t] if self.slots.dim() == 3 else self.slots[r]
        at = s[(s >= 0) & (s < self.rows)].long() + int(self.idx[r]) * self.stride
        parts = [self.read[at].double()] if 0 <= int(self.idx[r]) < self.co.pool_size else []
        if self.D:
            word = int(self.tree[r, t]) & (2 ** 64 - 1) if self.tree is not None else (2 << t) - 1
            parts.append(self.draft[r, [j for j in range(self.D) if word >> j & 1]].double())
        return torch.cat(parts) if parts else self.read[:0].double()

    def check(self, out, lse, num_real=None):
        u = torch.finfo(self.q.dtype).eps / 2
        tiny = torch.finfo(self.q.dtype).smallest_normal * u
        out = out.view(self.B, self.T, self.H, 512)
        lse = lse.view(self.B, self.T, self.H)
        for r in range(self.B if num_real is None else num_real):
            for t in range(self.T):
                k = self.keys(r, t)
                if not len(k):
                    assert (out[r, t] == 0).all() and (lse[r, t] == -math.inf).all(), (r, t)
                    continue
                q = self.q[r, t].double()
                s = q @ k.T * self.scale
                p = torch.softmax(s, 1)
                want = p @ k[:, :512]
                mass = p @ k[:, :512].abs()
                ds = 576 * 2.0 ** -23 * self.scale * (q.abs() @ k.abs().T).amax(1, keepdim=True)
                top = s.abs().amax(1, keepdim=True)
                n = len(k) * 2.0 ** -23
                tol = u * want.abs() + tiny + (u + 2 * (ds + 2.0 ** -22 * top) + 2.0 ** -19 + n) * mass
                off = (out[r, t].double() - want).abs()
                assert (off <= tol).all(), (r, t, float((off / tol).max()))
                le = torch.logsumexp(s, 1, keepdim=True)
                ltol = ds + 2.0 ** -21 * (top + le.abs() + 1) + n
                loff = (lse[r, t].double()[:, None] - le).abs()
                assert (loff <= ltol).all(), (r, t, float((loff / ltol).max()))


SHAPES = [
    dict(B=1, T=1, H=1, K=1, holes=0),
    dict(B=1, T=1, H=1, K=0, D=1),
    dict(B=2, T=1, H=16, K=127),
    dict(B=1, T=1, H=128, K=128, holes=0),
    dict(B=2, T=1, H=128, K=129, rows=300),
    dict(B=3, T=2, H=33, K=65, D=2),
    dict(B=2, T=5, H=24, K=333, D=5, own=True, rows=512, holes=0.3),
    dict(B=1, T=64, H=2, K=40, D=64),
    dict(B=1, T=64, H=3, K=7, D=63, own=True),
    dict(B=2, T=3, H=128, K=300, D=7, tree="chain"),
    dict(B=1, T=1, H=8, K=2048, rows=4096),
    dict(B=1, T=2, H=64, K=2500, rows=2600, D=2),
    dict(B=9, T=1, H=9, K=511, rows=520, shared=True),
    dict(B=40, T=1, H=16, K=256, rows=256, pool=50),
    dict(B=2, T=4, H=16, K=64, D=4, holes=1.0),
    dict(B=2, T=4, H=16, K=300, D=0, holes=0.99),
]


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join("{}{}".format(k, v) for k, v in s.items()))
def test_parity(shape, fmt, dtype):
    c = Case(sum(map(ord, str(shape))), fmt=fmt, dtype=dtype, **shape)
    c.check(*c.call())


@pytest.mark.parametrize("empty", ["first", "most", "all", "none"])
@pytest.mark.parametrize("fmt", ["raw", "int8"])
@pytest.mark.parametrize("B, H, K", [(400, 5, 40), (160, 130 // 2, 100), (90, 16, 700)])
def test_requests_without_any_key_among_others(B, H, K, fmt, empty):
    """A CTA's run has several requests (whole ones, or with ends that others share), and their queries are
    fetched ahead of the rows that none of them may have."""
    c = Case(31, B=B, H=H, K=K, rows=256, shared=True, fmt=fmt, holes=0.2)
    gone = {"first": torch.arange(B, device="cuda") % 5 < 2, "most": torch.arange(B, device="cuda") % 5 != 3,
            "all": torch.ones(B, device="cuda", dtype=torch.bool), "none": torch.zeros(B, device="cuda", dtype=torch.bool)}[empty]
    c.slots[gone] = -1
    c.check(*c.call())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K, B", [(2000, 1), (2000, 40), (64 * 150, 2)])
def test_scores_that_grow_along_the_list(K, B, dtype):
    """Later keys score higher and higher: the running references move again and again, in whole lists and in
    joined parts, and earlier probabilities become nothing."""
    c = Case(32, B=B, H=17, K=K, rows=K, shared=True, dtype=dtype, holes=0.0)
    c.slots[:] = torch.arange(K, dtype=torch.int32, device="cuda")
    c.read *= torch.linspace(0.1, 8.0, K, device="cuda", dtype=torch.float32).to(c.read.dtype)[:, None]
    c.check(*c.call())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_peaked_and_large_scores(dtype):
    """Scores up to hundreds: one key takes nearly all, and the running maximum moves late."""
    c = Case(5, B=2, T=2, H=32, K=700, rows=700, D=2, dtype=dtype, spread=20.0)
    c.read[c.slots[0, -1].clamp(min=0).long() + int(c.idx[0]) * c.rows] *= 3
    c.check(*c.call())


def test_three_dimensional_q_and_given_outputs():
    c = Case(6, B=3, H=20, K=100, D=1)
    out, lse = c.call(q=c.q[:, 0])
    assert out.shape == (3, 20, 512) and lse.shape == (3, 20)
    c.check(out, lse)
    o, s = torch.empty_like(out), torch.empty_like(lse)
    ws = torch.empty(max(16, kv().attend_workspace(3, 1, 20, 100, 1)), dtype=torch.uint8, device="cuda")
    got = c.call(q=c.q[:, 0], out=o, lse=s, workspace=ws)
    assert got[0] is o and got[1] is s
    assert torch.equal(o, out) and torch.equal(s, lse)


def test_rows_behind_num_real_are_left():
    c = Case(7, B=5, T=2, H=6, K=50, D=2)
    out = torch.full((5, 2, 6, 512), 3.0, dtype=c.q.dtype, device="cuda")
    lse = torch.full((5, 2, 6), 4.0, device="cuda")
    for n in (3, 0):
        c.co.num_real.fill_(n)
        before = out.clone(), lse.clone()
        c.call(out=out, lse=lse)
        assert torch.equal(out[n:], before[0][n:]) and torch.equal(lse[n:], before[1][n:])
        c.check(out, lse, n)
    c.co.num_real.fill_(99)  # more than the batch: every row of the batch
    c.check(*c.call())


def test_strides_of_every_input():
    c = Case(8, B=2, T=3, H=7, K=90, D=3, own=True)
    big = torch.randn((2, 5, 9, 600), device="cuda").to(c.q.dtype)
    big[:, :3, 1:8, 8:584] = c.q
    slots = torch.randint(0, 64, (2, 4, 101), device="cuda", dtype=torch.int32)
    slots[:, 1:, 5:95] = c.slots
    draft = torch.randn((2, 4, 1152), device="cuda").to(c.q.dtype)
    draft[:, :3, :576] = c.draft
    out, lse = c.call(q=big[:, :3, 1:8, 8:584], topk_device_slots=slots[:, 1:, 5:95], draft_rows=draft[:, :3, :576])
    want = c.call()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    c.check(out, lse)


@pytest.mark.parametrize("fmt", ["raw", "e4m3"])
def test_slots_and_pool_rows_out_of_range(fmt):
    c = Case(9, B=4, T=1, H=8, K=60, D=1, fmt=fmt, pool=4)
    c.slots[:, ::7] = 64          # one past the last row
    c.slots[:, 1::7] = 2 ** 31 - 1
    c.slots[:, 2::7] = -2 ** 31
    c.idx[1], c.idx[2] = -1, 4    # no such pool row
    c.check(*c.call())
    c.slots.fill_(-1)
    c.draft, c.D, c.tree = None, 0, None
    out, lse = c.call()
    assert (out == 0).all() and (lse == -math.inf).all()


def test_what_no_one_attends_to_may_be_nan():
    c = Case(10, B=2, T=4, H=8, K=70, D=4, rows=200)
    c.tree = tree_masks([[-1, 0, 0, 2], [-1, -1, 1, 0]]).cuda()
    want = c.call()
    named = torch.zeros(2, 200, dtype=torch.bool, device="cuda")
    for r in range(2):
        s = c.slots[r]
        named[int(c.idx[r]), s[s >= 0].long()] = True
    c.hot[~named.view(-1)] = float("nan")
    got = c.call()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for bad in (float("nan"), float("inf"), -float("inf")):
        c.draft[0, 3, 100] = bad     # seen by token 3 of request 0 only
        c.draft[1, 2, 575] = bad     # by token 2 of request 1
        got = c.call()
        seen = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
        seen[0, 3] = seen[1, 2] = True
        assert torch.equal(got[0][~seen], want[0][~seen]) and torch.equal(got[1][~seen], want[1][~seen])
        if bad != bad:
            assert got[0][seen].isnan().all() and got[1][seen].isnan().all()


def test_tree_words():
    """No words are a chain; bits from drafts on say nothing; a word of zero leaves the list alone."""
    c = Case(11, B=2, T=3, H=4, K=30, D=3, tree="chain")
    want = c.call()
    c.tree = tree_masks([[-1, 0, 1]] * 2).cuda()
    got = c.call()
    assert torch.equal(got[0], want[0])
    c.tree |= -8
    got = c.call()
    assert torch.equal(got[0], want[0])
    c.tree.zero_()
    c.check(*c.call())
    c.slots.fill_(-1)
    out, lse = c.call()
    assert (out == 0).all() and (lse == -math.inf).all()


def test_a_slot_named_twice_counts_twice():
    c = Case(12, B=1, H=3, K=2, rows=8, holes=0)
    c.slots[:] = torch.tensor([[5, 5]], dtype=torch.int32)
    out, lse = c.call()
    c.check(out, lse)
    c.slots = c.slots[:, :1].contiguous()
    one = c.call()
    assert (lse - one[1] - math.log(2)).abs().max() < 1e-5


def test_same_call_twice_is_the_same_bits():
    c = Case(13, B=3, T=2, H=128, K=1000, D=2, rows=1000, fmt="int8", dtype="bf16")
    a, b = c.call(), c.call()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_stored_rows_attend_as_what_they_read_back_as():
    for fmt in ("e4m3", "int8"):
        c = Case(14, B=2, T=2, H=40, K=400, D=2, rows=400, fmt=fmt, dtype="bf16")
        a = c.call()
        b = c.call(hot=c.read, row_format="raw")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_hot_rows_beyond_four_gigabytes():
    rows, pool = 1_000_000, 4
    c = Case(15, B=2, H=16, K=200, rows=64, pool=pool)
    hot = torch.zeros(pool * rows, 576, dtype=torch.float16, device="cuda")
    want = c.call()
    for p in range(pool):
        hot[(p + 1) * rows - 64:(p + 1) * rows] = c.hot[p * 64:(p + 1) * 64]
    moved = torch.where(c.slots >= 0, c.slots + rows - 64, c.slots)
    got = c.call(hot=hot, topk_device_slots=moved, hot_req_stride_rows=rows, hot_rows=rows)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams_at_once():
    a = Case(16, B=16, T=2, H=64, K=1500, D=2, rows=1500)
    b = Case(17, B=16, T=1, H=128, K=900, rows=1000, dtype="bf16")
    wa, wb = a.call(), b.call()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        with torch.cuda.stream(s1):
            x = a.call()
        y = b.call(stream=s2.cuda_stream)
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x[0], wa[0]) and torch.equal(y[0], wb[0])
        assert torch.equal(x[1], wa[1]) and torch.equal(y[1], wb[1])


def test_captured_and_replayed():
    c = Case(18, B=4, T=3, H=32, K=600, D=3, rows=700)
    c.call()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = c.call()
    with torch.cuda.graph(g2):
        o2 = c.call()
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(3):
        c.q.copy_(torch.randn(c.q.shape, generator=g, device="cuda"))
        c.slots.copy_(torch.randint(-1, 700, c.slots.shape, generator=g, device="cuda"))
        want = c.call()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for o in (o1, o2):
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_captured_first_behind_a_copy_and_behind_a_join_of_streams():
    """The launch is a programmatic dependent of the kernel before it: a graph whose node before is none, a copy, or two
    streams' ends has to order it all the same."""
    c = Case(33, B=3, T=2, H=64, K=900, D=2, rows=1000)
    new_q, new_slots = torch.randn_like(c.q), torch.randint(-1, 1000, c.slots.shape, device="cuda", dtype=torch.int32)
    c.call()
    first, copy, join = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        o1 = c.call()
    with torch.cuda.graph(copy):
        c.q.copy_(new_q)  # (a copy node)
        o2 = c.call()
        again = c.call()
    side = torch.cuda.Stream()
    with torch.cuda.graph(join):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            c.slots.copy_(new_slots)
        c.q.mul_(0.5)
        here.wait_stream(side)
        o3 = c.call()
    first.replay()
    torch.cuda.synchronize()
    c.check(*o1)
    copy.replay()
    torch.cuda.synchronize()
    c.check(*o2)
    assert torch.equal(again[0], o2[0]) and torch.equal(again[1], o2[1])
    join.replay()
    torch.cuda.synchronize()
    c.check(*o3)


def test_behind_an_event_of_another_stream_and_behind_kernels_that_write_its_inputs():
    c = Case(34, B=8, T=1, H=16, K=2000, rows=2000, dtype="bf16")  # (a list that is cut and joined)
    q0, hot0 = c.q.clone(), c.hot.clone()
    want = c.call()
    side = torch.cuda.Stream()
    for _ in range(20):
        c.q.zero_()
        c.hot.zero_()
        ready = torch.cuda.Event()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            torch.cuda._sleep(200_000)
            c.hot.copy_(hot0)
            ready.record()
        torch.mul(q0, 1.0, out=c.q)
        torch.cuda.current_stream().wait_event(ready)
        got = c.call()
        again = c.call(q=c.q, out=torch.empty_like(got[0]))
        c.q.zero_()  # after both
        assert torch.equal(got[0], want[0]) and torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_one_workspace_and_outputs_for_calls_in_a_row():
    c = Case(35, B=2, T=1, H=128, K=4000, rows=4000)
    need = kv().attend_workspace(2, 1, 128, 4000, 0)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty((2, 128, 512), dtype=torch.float16, device="cuda"), torch.empty((2, 128), device="cuda")
    qs = [torch.randn_like(c.q) for _ in range(6)]
    want = [c.call(q=q)[0].clone() for q in qs]
    got = [c.call(q=q, out=out, lse=lse, workspace=ws)[0].clone() for q in qs]
    for w, g in zip(want, got):
        assert torch.equal(w.view_as(g), g)
    assert c.co.attend_error() == 0


def test_an_earlier_launch_that_gave_up_is_raised_by_the_next_call():
    c = Case(36)
    c.call()
    torch.cuda.synchronize()
    c.co._attend_err[0] = 0x103  # as the kernel leaves it
    with pytest.raises(RuntimeError, match="0x103"):
        c.call()
    assert c.co.attend_error() == 0
    c.check(*c.call())


def test_hot_rows_elsewhere_are_refused():
    c = Case(37)
    with pytest.raises(ValueError, match="hot rows must be on"):
        c.call(hot=c.hot.cpu())
    with pytest.raises(ValueError, match="every tensor must be on"):
        c.call(topk_device_slots=c.slots.cpu())


def test_c_refusals():
    mod = kv()
    c = Case(19, B=2, T=1, H=4, K=16, D=1)
    out, lse = c.call()
    ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    good = dict(q=c.q.data_ptr(), q_stride_req=4 * 576, q_stride_token=576, q_stride_head=576,
                hot_row_base=c.hot.data_ptr(), hot_req_stride_rows=64, hot_rows=64,
                req_pool_indices=c.idx.data_ptr(), pool_size=2, topk_device_slots=c.slots.data_ptr(), slots_stride_req=16,
                slots_stride_token=0, num_real=c.co.num_real.data_ptr(), draft_rows=c.draft.data_ptr(),
                draft_stride_req=576, draft_stride_row=576, tree=c.tree.data_ptr(), out=out.data_ptr(),
                lse=lse.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(), max_num_reqs=2, tokens=1, heads=4,
                top_k=16, drafts=1, row_format="raw", row_dtype="fp16", scale=0.07)
    mod.attend_hot(**good)
    for change, message in [
        (dict(q=0), "address is 0"), (dict(hot_row_base=0), "address is 0"), (dict(out=0), "address is 0"),
        (dict(topk_device_slots=0), "address is 0"), (dict(req_pool_indices=0), "address is 0"),
        (dict(num_real=0), "address is 0"), (dict(draft_rows=0), "address is 0"),
        (dict(q=good["q"] + 2), "16-byte"), (dict(out=good["out"] + 8), "16-byte"),
        (dict(hot_row_base=good["hot_row_base"] + 4), "16-byte"), (dict(draft_rows=good["draft_rows"] + 2), "16-byte"),
        (dict(q_stride_head=580), "multiples of 8"), (dict(draft_stride_row=577), "multiples of 8"),
        (dict(lse=good["lse"] + 2), "alignment"), (dict(tree=good["tree"] + 4), "alignment"),
        (dict(tokens=0), "tokens"), (dict(tokens=65), "tokens"), (dict(heads=0), "heads"), (dict(heads=129), "heads"),
        (dict(drafts=65), "drafts"), (dict(top_k=(1 << 24) + 1), "out of range"),
        (dict(max_num_reqs=(1 << 16) + 1), "out of range"),
        # 2^16 requests x 64 lists of 2^18 tiles: more pairs than a 32-bit number counts
        (dict(max_num_reqs=1 << 16, tokens=64, slots_stride_token=16, top_k=1 << 24), "keys out of range"),
        (dict(max_num_reqs=1 << 16, top_k=(1 << 24) - 64 * 8), "the workspace|keys out of range"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            mod.attend_hot(**{**good, **change})
    with pytest.raises(ValueError, match="row_format"):
        mod.attend_hot(**{**good, "row_format": "fp8"})
    need = mod.attend_workspace(2, 1, 4, 100_000, 1)
    if need:
        with pytest.raises(RuntimeError, match="workspace"):
            mod.attend_hot(**{**good, "top_k": 100_000, "workspace_bytes": need - 1})
    mod.attend_hot(**{**good, "max_num_reqs": 0})  # nothing to do
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("hot_quantized", [False, True])
def test_decode_steps_over_a_quantised_pool(fmt, hot_quantized):
    """The operators as they are used together: a prompt quantised into the pool, decode steps that
    read their misses back and attend, captured as a graph; and both ways of keeping the hot rows."""
    from kv_offload_proto_b200.graph import StepGraph
    from kv_offload_proto_b200.pool import DevicePool
    from kv_offload_proto_b200.workload import sample_topk_device
    kv()
    R, ctx, K, dbs, L, T, H = 4, 1024, 200, 256, 2, 3, 16
    pool = DevicePool(0, L, R * ctx, 1152, 1, segment_devices=(0, 0), row_format=fmt, row_dtype="fp16",
                      hot_quantized=hot_quantized)
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = torch.randn((L, R * ctx, 576), generator=g, device="cuda").to(torch.float16)
    pool.wait(pool.batch_write_alllayers(0, R * ctx, rows, rows.stride(0) * 2))
    read = [quant_model.decode(quant_model.encode(rows[layer].cpu(), fmt, 512), fmt, "fp16", 512).cuda()
            for layer in range(L)]
    co = XdsOffloadCoordinator("cuda", L, R, dbs, K, R, ctx)
    co.admit_all([ctx] * R, [r * ctx for r in range(R)])
    co.set_batch(torch.arange(R, device="cuda"), torch.full((R,), ctx, dtype=torch.int32, device="cuda"))
    if hot_quantized:
        hot = torch.zeros((L, R * dbs, 656), dtype=torch.uint8, device="cuda")
    else:
        hot = torch.zeros((L, R * dbs, 576), dtype=torch.float16, device="cuda")
    # admission put tokens 0..dbs-1 in the slots: bring their rows (by an all-miss read)
    first = torch.arange(dbs, dtype=torch.int32, device="cuda").repeat(R, 1)
    for layer in range(L):
        pool.wait(pool.batch_read(layer, first, co._req_pool_indices, co.req_host_base, first,
                                  torch.ones((R, dbs), dtype=torch.int8, device="cuda"), co.num_real, hot[layer], R, dbs,
                                  hot_req_stride_rows=dbs))
    q = torch.randn((L, R, T, H, 576), generator=g, device="cuda").to(torch.float16)
    draft = torch.randn((L, R, T, 576), generator=g, device="cuda").to(torch.float16)
    tree = tree_masks([[-1, 0, 0]] * R).cuda()
    outs = {}
    kept = torch.empty((L, R, K), dtype=torch.int32, device="cuda")

    def after(layer):
        outs[layer] = co.attend(q[layer], hot[layer], hot_req_stride_rows=dbs, row_format=fmt if hot_quantized else "raw",
                                scale=0.07, draft_rows=draft[layer], tree=tree)
        kept[layer].copy_(co.top_k_device_slots)

    graph = StepGraph(pool, co, hot, path="auto", hot_req_stride_rows=dbs, after_layer=after)
    for _ in range(3):
        topk = torch.stack([sample_topk_device(co.device_buffer_tokens[layer, :R], ctx, dbs, K, 0.2, g)
                            for layer in range(L)])
        graph.topk.copy_(topk)
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert graph.error() == 0
        for layer in range(L):
            # The hand may pass a slot twice in a step of so small a buffer, and evict a row that an
            # earlier position of the same step names; where only one position names a slot, the slot
            # holds that position's row.
            named = torch.zeros((R, dbs), dtype=torch.int64, device="cuda")
            named.scatter_add_(1, kept[layer].long(), torch.ones_like(kept[layer], dtype=torch.int64))
            r, k = (named.gather(1, kept[layer].long()) == 1).nonzero(as_tuple=True)
            assert len(r) > R * K // 2
            if hot_quantized:
                held = quant_model.decode(hot[layer].cpu().numpy(), fmt, "fp16", 512).cuda()
            else:
                held = hot[layer]
            at = r * dbs + kept[layer][r, k].long()
            assert torch.equal(held[at], read[layer][r * ctx + topk[layer][r, k].long()])
            c = Case.__new__(Case)
            c.B, c.T, c.H, c.K, c.D, c.rows, c.scale, c.co = R, T, H, K, T, dbs, 0.07, co
            c.q, c.draft, c.tree, c.idx, c.stride = q[layer], draft[layer], tree, co._req_pool_indices, dbs
            c.slots, c.read = kept[layer], held
            c.check(*outs[layer])
    pool.destroy()

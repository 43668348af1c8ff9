"""GPU parity of the 8-bit row copies (export_quant_alllayer, export_quant, import_quant and the
DevicePool calls over them) with the codec model: every stored byte and every value read back."""
import numpy as np
import pytest
import torch

import quant_model
from gpu_util import dev, host, kv
from kv_offload_proto_b200.pool import DevicePool, device_view, per_layer_seg_rows_injective, seg_row_of
from quant_model import TORCH

pytestmark = pytest.mark.gpu


def make_rows(seed, shape, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape, generator=g))
    return x.clamp(-60000, 60000).to(TORCH[dtype])


def place(row, S, N, injective):
    return (0 if S == 0 else row // S % N), seg_row_of(row, S, N, injective)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("quant, plain, N, S, injective, lo, cnt, layers", [
    (512, 64, 1, 1, False, 0, 1, 1),
    (512, 64, 3, 2, True, 5, 301, 2),
    (512, 64, 2, 4, False, 3, 97, 3),   # the reference's map: the last row of a stripe stays
    (128, 0, 1, 0, False, 7, 33, 1),
    (1024, 72, 2, 1, False, 0, 65, 2),
    (640, 8, 1, 64, True, 63, 130, 1),
])
def test_export_alllayer_bytes(fmt, dtype, quant, plain, N, S, injective, lo, cnt, layers):
    mod = kv()
    rows = make_rows(quant + cnt, (layers, lo + cnt, quant + plain), dtype)
    rows[0, lo, :128] = 0
    if cnt > 40:
        rows[0, lo + 1, 3] = float("inf")
        rows[0, lo + 2, quant - 1] = float("nan")
        rows[0, lo + 3, :128] = 2.0 ** -24
    sb = quant_model.stored_bytes(quant, plain)
    total = lo + cnt
    plsr = per_layer_seg_rows_injective(total, S, N) if injective else (total if S == 0 else -(-total // N))
    rng = np.random.default_rng(0)
    want = [rng.integers(0, 256, (layers, plsr, sb), dtype=np.uint8) for _ in range(N)]
    segs = [dev(w) for w in want]
    src = rows.cuda()
    status = mod.alloc_status(8 * N)
    mod.export_quant_alllayer([s.data_ptr() for s in segs], plsr, fmt, dtype, quant, plain, lo, cnt, layers,
                              src.data_ptr(), src.stride(0) * 2, S, status, 0, 1, injective=injective)
    for n in range(N):
        assert mod.poll_status(status + 64 * n, 10_000_000) == 0
    torch.cuda.synchronize()
    for layer in range(layers):
        enc = quant_model.encode(rows[layer], fmt, quant)
        for r in range(lo, lo + cnt):
            n, at = place(r, S, N, injective)
            want[n][layer, at] = enc[r]
    for n in range(N):
        np.testing.assert_array_equal(host(segs[n]), want[n])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("quant, plain, N, S, R, K, num_real", [
    (512, 64, 1, 1, 1, 1, 1), (512, 64, 3, 2, 5, 131, 4), (256, 64, 2, 16, 3, 70, 9), (128, 0, 1, 1, 2, 300, 0)])
def test_single_rows_written_and_read_back(fmt, dtype, quant, plain, N, S, R, K, num_real):
    mod = kv()
    rng = np.random.default_rng(K)
    ctx, dbs = 512, 400
    sb, width = quant_model.stored_bytes(quant, plain), quant + plain
    plsr = per_layer_seg_rows_injective(R * ctx, S, N)
    segs_h = [rng.integers(0, 256, (2, plsr, sb), dtype=np.uint8) for _ in range(N)]
    segs = [dev(s) for s in segs_h]
    topk = np.stack([rng.choice(ctx, K, replace=False) for _ in range(R)]).astype(np.int32)
    slots = np.stack([rng.choice(dbs, K, replace=False) for _ in range(R)]).astype(np.int32)
    flags = (rng.random((R, K)) < 0.6).astype(np.int8)
    flags[0, 0] = 1
    if K > 1:
        topk[0, 1], slots[R - 1, K - 1] = -1, -1
    req = rng.permutation(R).astype(np.int64)
    if R > 2:
        req[1] = -1
    base = np.arange(R, dtype=np.int64) * ctx
    hot_h = make_rows(K, (R * dbs, width), dtype)
    hot = hot_h.cuda()
    back = torch.full((R * dbs, width), 7.0, dtype=TORCH[dtype], device="cuda")
    a = [dev(x) for x in (topk, req, base, slots, flags, np.array([num_real], np.int32))]
    ptrs = [x.data_ptr() for x in a]
    status = mod.alloc_status(8 * N)
    mod.export_quant([s.data_ptr() for s in segs], plsr, plsr, fmt, dtype, quant, plain, *ptrs, hot.data_ptr(), K, R, S,
                     status, 0, 1, hot_req_stride_rows=dbs, injective=True)
    for n in range(N):
        assert mod.poll_status(status + 64 * n, 10_000_000) == 0
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    mod.import_quant([s.data_ptr() for s in segs], plsr, plsr, fmt, dtype, quant, plain, *ptrs, back.data_ptr(), K, R,
                     S, status, 0, 2, hot_req_stride_rows=dbs, injective=True, err_word=err.data_ptr())
    for n in range(N):
        assert mod.poll_status(status + 64 * n, 10_000_000) == 0
        assert mod.poll_status(status + 64 * n + 8, 10_000_000) == 0
    torch.cuda.synchronize()
    assert err.item() == 0
    want = torch.full((R * dbs, width), 7.0, dtype=TORCH[dtype])
    enc = quant_model.encode(hot_h, fmt, quant)
    dec = quant_model.decode(enc, fmt, dtype, quant)
    for r in range(min(R, num_real)):
        for k in range(K):
            if flags[r, k] and topk[r, k] >= 0 and slots[r, k] >= 0 and req[r] >= 0:
                n, at = place(int(base[r] + topk[r, k]), S, N, True)
                i = int(req[r]) * dbs + int(slots[r, k])
                segs_h[n][1, at] = enc[i]
                want[i] = dec[i]
    for n in range(N):
        np.testing.assert_array_equal(host(segs[n]), segs_h[n])
    assert torch.equal(back.cpu().view(torch.int16), want.view(torch.int16))


def test_nonfinite_groups_read_back_as_nan():
    mod = kv()
    rows = make_rows(1, (3, 576), "fp16")
    rows[0, 130] = float("-inf")
    rows[1, 511] = float("nan")
    src, seg = rows.cuda(), torch.zeros(3 * 656, dtype=torch.uint8, device="cuda")
    status = mod.alloc_status(8)
    mod.export_quant_alllayer([seg.data_ptr()], 3, "int8", "fp16", 512, 64, 0, 3, 1, src.data_ptr(), 3 * 1152, 1, status)
    assert mod.poll_status(status, 10_000_000) == 0
    a = [dev(x) for x in (np.arange(3, dtype=np.int32)[None], np.zeros(1, np.int64), np.zeros(1, np.int64),
                          np.arange(3, dtype=np.int32)[None], np.ones((1, 3), np.int8), np.ones(1, np.int32))]
    back = torch.zeros((3, 576), dtype=torch.float16, device="cuda")
    mod.import_quant([seg.data_ptr()], 0, 3, "int8", "fp16", 512, 64, *[x.data_ptr() for x in a], back.data_ptr(), 3, 1,
                     1, status)
    assert mod.poll_status(status, 10_000_000) == 0
    back = back.cpu()
    assert back[0, 128:256].isnan().all() and back[1, 384:512].isnan().all()
    assert int(back.isnan().sum()) == 256
    assert torch.equal(back[:, 512:], rows[:, 512:])


def test_errcodes_and_refusals():
    mod = kv()
    a = [dev(x) for x in (np.arange(4, dtype=np.int32)[None], np.zeros(1, np.int64), np.zeros(1, np.int64),
                          np.arange(4, dtype=np.int32)[None], np.ones((1, 4), np.int8), np.ones(1, np.int32))]
    p = [x.data_ptr() for x in a]
    hot = torch.zeros(4 * 576, dtype=torch.float16, device="cuda")
    seg = torch.zeros(2 * 656, dtype=torch.uint8, device="cuda")
    codec = ("e4m3", "fp16", 512, 64)
    status = mod.alloc_status(8)
    mod.import_quant([0], 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, status)
    assert mod.poll_status(status, 10_000_000) == 0x101
    mod.import_quant([seg.data_ptr()], 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, status)
    assert mod.poll_status(status, 10_000_000) & 0xFF00 == 0x200
    mod.export_quant([seg.data_ptr()], 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, status)
    assert mod.poll_status(status, 10_000_000) & 0xFF00 == 0x200
    mod.export_quant_alllayer([0], 2, *codec, 0, 2, 1, hot.data_ptr(), 0, 1, status)
    assert mod.poll_status(status, 10_000_000) == 0x101
    mod.export_quant_alllayer([seg.data_ptr()], 2, *codec, 0, 4, 1, hot.data_ptr(), 0, 1, status)
    assert mod.poll_status(status, 10_000_000) & 0xFF00 == 0x200
    for call, message in [
        (lambda: mod.import_quant([seg.data_ptr() + 8], 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, 0), "16-byte"),
        (lambda: mod.import_quant([seg.data_ptr()], 0, 2, *codec, *p, hot.data_ptr() + 2, 4, 1, 1, 0), "16-byte"),
        (lambda: mod.import_quant([seg.data_ptr()], 0, 2, "int8", "fp16", 500, 64, *p, hot.data_ptr(), 4, 1, 1, 0),
         "quant_elems"),
        (lambda: mod.import_quant([], 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, 0), "node_num"),
        (lambda: mod.import_quant([seg.data_ptr()], 0, 2, *codec, 0, *p[1:], hot.data_ptr(), 4, 1, 1, 0), "address is 0"),
        (lambda: mod.export_quant([0] * 65, 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, 0), "node_num"),
        (lambda: mod.export_quant([seg.data_ptr()], 0, 2, *codec, *p, hot.data_ptr(), 4, 1, 1, 0, 0, 9), "blockDim"),
        (lambda: mod.export_quant_alllayer([], 2, *codec, 0, 2, 1, hot.data_ptr(), 0, 1, 0), "node_num"),
        (lambda: mod.export_quant_alllayer([seg.data_ptr()], 2, *codec, 0, 2, 1, hot.data_ptr(), 0, 1, 0, 0, 9), "blockDim"),
        (lambda: mod.export_quant_alllayer([seg.data_ptr()], 2, *codec, 0, 2, 1, hot.data_ptr() + 2, 0, 1, 0), "16-byte"),
        (lambda: mod.export_quant_alllayer([seg.data_ptr()], 2, *codec, 0, 2, 2, hot.data_ptr(), 1160, 1, 0), "16-byte"),
        (lambda: mod.export_quant_alllayer([seg.data_ptr()], 2, *codec, 0, 2, 1, 0, 0, 1, 0), "address is 0"),
        (lambda: mod.export_quant_alllayer([seg.data_ptr()], 2, *codec, 2 ** 32 - 1, 2, 1, hot.data_ptr(), 0, 1, 0), "32-bit"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
    # nothing to do is no error
    mod.import_quant([seg.data_ptr()], 0, 2, *codec, *p, hot.data_ptr(), 0, 1, 1, status)
    assert mod.poll_status(status, 10_000_000) == 0


@pytest.mark.parametrize("where", [0, -1])
def test_pool_round_trip(where):
    """A prompt written through a DevicePool and read back: device and pinned host segments."""
    kv()
    L, R, ctx, K, dbs = 2, 3, 64, 20, 32
    pool = DevicePool(0, L, R * ctx, 1152, 2, segment_devices=(where, where), injective=True, row_format="e4m3",
                      row_dtype=torch.float16)
    assert pool.seg_row_bytes == 656 and pool.segment_bytes == L * pool.per_layer_seg_rows * 656
    rows = make_rows(5, (L, R * ctx, 576), "fp16")
    src = rows.cuda()
    pool.wait(pool.batch_write_alllayers(0, R * ctx, src, src.stride(0) * 2))
    rng = np.random.default_rng(2)
    topk = np.stack([rng.choice(ctx, K, replace=False) for _ in range(R)]).astype(np.int32)
    slots = np.stack([rng.choice(dbs, K, replace=False) for _ in range(R)]).astype(np.int32)
    t = [dev(x) for x in (topk, np.arange(R, dtype=np.int64), np.arange(R, dtype=np.int64) * ctx, slots,
                          np.ones((R, K), np.int8), np.array([R], np.int32))]
    hot = torch.zeros((R * dbs, 576), dtype=torch.float16, device="cuda")
    for layer in range(L):
        for fused in (True, False):
            hot.zero_()
            pool.wait(pool.batch_read(layer, *t, hot, R, K, fused=fused, hot_req_stride_rows=dbs))
            got = hot.cpu()
            dec = quant_model.decode(quant_model.encode(rows[layer], "e4m3", 512), "e4m3", "fp16", 512)
            for r in range(R):
                assert torch.equal(got[r * dbs + slots[r].astype(np.int64)], dec[r * ctx + topk[r].astype(np.int64)])
    # one new row per request goes back in its place
    new = make_rows(9, (R, 576), "fp16")
    hot.view(R, dbs, 576)[:, 3] = new.cuda()
    one = [dev(np.full((R, 1), 7, np.int32)), t[1], t[2], dev(np.full((R, 1), 3, np.int32)), dev(np.ones((R, 1), np.int8)),
           t[5]]
    pool.wait(pool.batch_write(1, *one, hot, R, 1, hot_req_stride_rows=dbs))
    hot.zero_()
    pool.wait(pool.batch_read(1, *one, hot, R, 1, hot_req_stride_rows=dbs))
    dec = quant_model.decode(quant_model.encode(new, "e4m3", 512), "e4m3", "fp16", 512)
    assert torch.equal(hot.view(R, dbs, 576)[:, 3].cpu(), dec)
    pool.destroy()


def test_pool_refusals():
    kv()
    for kw, message in [(dict(row_format="fp8"), "row_format"), (dict(hot_quantized=True), "hot_quantized"),
                        (dict(row_format="int8", row_dtype=torch.float32), "float16 or bfloat16"),
                        (dict(row_format="int8", plain_elems=576), "plain_elems")]:
        with pytest.raises(ValueError, match=message):
            DevicePool(0, 1, 16, 1152, **kw)
    with pytest.raises(RuntimeError, match="quant_elems"):
        DevicePool(0, 1, 16, 1152, row_format="int8", plain_elems=56)
    pool = DevicePool(0, 1, 16, 1152, row_format="int8")
    with pytest.raises(ValueError, match="path"):
        pool.sieve_and_read(None, 0, torch.zeros(1, dtype=torch.int32), 0, path="coop")
    pool.destroy()


def test_rows_beyond_four_gigabytes():
    """Hot rows and segment rows whose byte offsets pass 2^32."""
    mod = kv()
    n = 4_000_000
    seg = torch.empty(n * 1100, dtype=torch.uint8, device="cuda")  # 4.4 GB: stored rows up to 6.7 million
    hot = torch.empty(n * 1152, dtype=torch.uint8, device="cuda")
    rows = make_rows(3, (2, 576), "bf16")
    src = rows.cuda().view(torch.uint8)
    at = [3_900_000, 3_999_999]
    seg_rows = [6_600_000, 6_700_000]
    for i in range(2):
        hot[at[i] * 1152:(at[i] + 1) * 1152] = src[i]
    a = [dev(x) for x in (np.array([[0], [100_000]], np.int32), np.array([0, 1], np.int64),
                          np.array([seg_rows[0], seg_rows[0]], np.int64), np.array([[at[0]], [at[1] - 1_000_000]], np.int32),
                          np.ones((2, 1), np.int8), np.array([2], np.int32))]
    p = [x.data_ptr() for x in a]
    status = mod.alloc_status(8)
    mod.export_quant([seg.data_ptr()], 0, 6_700_001, "e4m3", "bf16", 512, 64, *p, hot.data_ptr(), 1, 2, 1, status,
                     hot_req_stride_rows=1_000_000)
    assert mod.poll_status(status, 10_000_000) == 0
    enc = quant_model.encode(rows, "e4m3", 512)
    for i in range(2):
        got = host(device_view(seg.data_ptr() + seg_rows[i] * 656, 656, "cuda:0"))
        np.testing.assert_array_equal(got, enc[i])
        hot[at[i] * 1152:(at[i] + 1) * 1152] = 0
    mod.import_quant([seg.data_ptr()], 0, 6_700_001, "e4m3", "bf16", 512, 64, *p, hot.data_ptr(), 1, 2, 1, status,
                     hot_req_stride_rows=1_000_000)
    assert mod.poll_status(status, 10_000_000) == 0
    dec = quant_model.decode(enc, "e4m3", "bf16", 512)
    for i in range(2):
        got = hot[at[i] * 1152:(at[i] + 1) * 1152].view(torch.bfloat16).cpu()
        assert torch.equal(got, dec[i])


@pytest.mark.parametrize("fmt, dtype, quant, plain", [("e4m3", "fp16", 512, 64), ("int8", "bf16", 384, 8)])
def test_many_rows_in_tiles_and_rounds(fmt, dtype, quant, plain):
    """More rows than one round of the launch takes, written whole and by index and read back, over three segments."""
    mod = kv()
    layers, cnt, N, S, dbs = 3, 20_001, 3, 7, 1500
    rows = make_rows(12, (4000, quant + plain), dtype)
    src = rows.cuda()[torch.arange(layers * cnt, device="cuda") % 4000].view(layers, cnt, -1).contiguous()
    enc = quant_model.encode(rows, fmt, quant)
    dec = quant_model.decode(enc, fmt, dtype, quant).cuda()
    plsr = (cnt + S - 1) // S // N * S + S
    width = enc.shape[1]
    segs = [torch.zeros((layers, plsr, width), dtype=torch.uint8, device="cuda") for _ in range(N)]
    bases = [s.data_ptr() for s in segs]
    mod.export_quant_alllayer(bases, plsr, fmt, dtype, quant, plain, 0, cnt, layers, src.data_ptr(), src.stride(0) * 2, S, 0,
                              0, 1, injective=True)
    at = torch.arange(cnt, device="cuda")
    g = at // S
    place_of, seg_of = (g // N) * S + at % S, g % N
    want = torch.from_numpy(enc).cuda()
    for layer in range(layers):
        for n in range(N):
            mine = at[seg_of == n]
            assert torch.equal(segs[n][layer, place_of[mine]], want[(layer * cnt + mine) % 4000]), (layer, n)
    # every row of layer 1 is read back into hot rows of 16 requests, half of them flagged, then written to layer 2
    R, K = 16, 1250
    gen = torch.Generator(device="cuda").manual_seed(3)
    pos = torch.randperm(R * K, generator=gen, device="cuda").view(R, K).to(torch.int32)
    slots = torch.argsort(torch.rand((R, dbs), generator=gen, device="cuda"), 1)[:, :K].to(torch.int32).contiguous()
    flags = (torch.rand((R, K), generator=gen, device="cuda") < 0.5).to(torch.int8)
    idx, zero = torch.arange(R, device="cuda"), torch.zeros(R, dtype=torch.int64, device="cuda")
    real = torch.tensor([R], dtype=torch.int32, device="cuda")
    hot = torch.zeros((R, dbs, quant + plain), dtype=src.dtype, device="cuda")
    ptrs = [x.data_ptr() for x in (pos, idx, zero, slots, flags, real, hot)]
    mod.import_quant(bases, plsr, plsr, fmt, dtype, quant, plain, *ptrs, K, R, S, 0, 0, 1, hot_req_stride_rows=dbs,
                     injective=True)
    expect = torch.zeros_like(hot)
    r, k = flags.nonzero(as_tuple=True)
    expect[r, slots[r, k].long()] = dec[(cnt + pos[r, k].long()) % 4000]
    assert torch.equal(hot.view(torch.int16), expect.view(torch.int16))
    for s in segs:
        s[2].zero_()
    mod.export_quant(bases, 2 * plsr, plsr, fmt, dtype, quant, plain, *ptrs, K, R, S, 0, 0, 1, hot_req_stride_rows=dbs,
                     injective=True)
    p = pos[r, k].long()
    again = torch.from_numpy(quant_model.encode(dec.cpu(), fmt, quant)).cuda()
    for n in range(N):
        mine = p[seg_of[p] == n]
        assert torch.equal(segs[n][2, place_of[mine]], again[(cnt + mine) % 4000])
        rest = torch.ones(plsr, dtype=torch.bool, device="cuda")
        rest[place_of[mine]] = False
        assert (segs[n][2][rest] == 0).all()


def test_captured_and_on_two_streams():
    """The three launches in one graph, replayed with new rows, beside the same on another stream."""
    mod = kv()
    cnt, K = 600, 200
    one = torch.tensor([1], dtype=torch.int32, device="cuda")
    idx, zero = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")

    class Set:
        def __init__(self, seed):
            self.rows = make_rows(seed, (cnt, 576), "fp16").cuda()
            self.seg = torch.zeros((cnt, 656), dtype=torch.uint8, device="cuda")
            self.back = torch.zeros((1, cnt, 656), dtype=torch.uint8, device="cuda")
            self.hot = torch.zeros((K, 576), dtype=torch.float16, device="cuda")
            self.pos = torch.randperm(cnt, device="cuda")[:K].to(torch.int32)
            self.slots = torch.randperm(K, device="cuda").to(torch.int32)
            self.flags = torch.ones(K, dtype=torch.int8, device="cuda")

        def run(self):
            s = torch.cuda.current_stream().cuda_stream
            p = [x.data_ptr() for x in (self.pos, idx, zero, self.slots, self.flags, one, self.hot)]
            codec = ("e4m3", "fp16", 512, 64)
            mod.export_quant_alllayer([self.seg.data_ptr()], cnt, *codec, 0, cnt, 1, self.rows.data_ptr(), 0, 1, 0, s)
            mod.import_quant([self.seg.data_ptr()], 0, cnt, *codec, *p, K, 1, 1, 0, s)
            mod.export_quant([self.back.data_ptr()], 0, cnt, *codec, *p, K, 1, 1, 0, s)

        def check(self):
            enc = quant_model.encode(self.rows.cpu(), "e4m3", 512)
            dec = quant_model.decode(enc, "e4m3", "fp16", 512)
            pos = self.pos.cpu().long()
            assert torch.equal(self.seg.cpu(), torch.from_numpy(enc))
            assert torch.equal(self.hot.cpu()[self.slots.cpu().long()], dec[pos])
            assert torch.equal(self.back[0].cpu()[pos], torch.from_numpy(quant_model.encode(dec[pos], "e4m3", 512)))

    a, b = Set(21), Set(22)
    a.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run()
    side = torch.cuda.Stream()
    for seed in (23, 24):
        a.rows.copy_(make_rows(seed, (cnt, 576), "fp16"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(5):
                b.run()
        for _ in range(5):
            graph.replay()
        torch.cuda.synchronize()
        a.check()
        b.check()

"""SIEVE coordinator on CUDA: the B200 counterpart of the reference's caller
``xds.xds_offload.XdsOffloadCoordinator`` (xds/xds_offload.py:20-106).

Same constructor, attributes and methods, so code written against the reference's
coordinator runs unchanged with ``device="cuda:N"``. The per-layer SIEVE state lives in
HBM with the reference's tensor layout (xds/xds_offload.py:43-53) and every update goes
through the `_kvops` launch module (sieve_ht_init / sieve_update); nothing here runs the
SIEVE on the host.
"""
import contextlib

import torch

from . import kvops as _kvops_module
from .pool import dtype_name

__all__ = ["XdsOffloadCoordinator", "align", "compute_ht_size", "tree_masks"]

KEY_DIM, VALUE_DIM = 576, 512  # values of a row that attention scores use, and that it sums
ROW_BYTES = {"raw": 1152, "e4m3": 656, "int8": 656}
ATTEND_ERRORS = {0x103: "a wait inside an earlier call gave up",
                 0x104: "an earlier call's slots named rows that its hot rows have no place for (tokens generated since "
                        "the prompt have the slots from padded_buffer_size on; hot_rows given leaves them out)"}


def align(v, a):
    """Round v up to a multiple of a (xds/xds_ems_pool.py:50-51)."""
    return (v + a - 1) // a * a


def compute_ht_size(padded_buffer_size, top_k):
    """Power of two >= max(1024, 2*(padded+topK)): load factor <= 0.5
    (xds/xds_ems_pool.py:42-47; kvops_ext.cpp:297-300)."""
    p = 1024
    while p < 2 * (padded_buffer_size + top_k):
        p <<= 1
    return p


def tree_masks(parents):
    """The words that `XdsOffloadCoordinator.attend` takes as `tree`, from each drafted token's
    parent: parents[..., j] is the drafted token that token j continues (j's own index is larger),
    or -1 where it continues the context. Bit i of word j is set where i is j or an ancestor of j.
    Returns int64 of the same shape on the same device; up to 64 drafted tokens."""
    parents = torch.as_tensor(parents)
    n = parents.shape[-1]
    if n > 64:
        raise ValueError("at most 64 drafted tokens, got {}".format(n))
    index = torch.arange(n, device=parents.device)
    if parents.is_floating_point() or bool(((parents < -1) | (parents >= index)).any()):
        raise ValueError("parents[..., j] must be an integer in [-1, j)")
    parents = parents.to(torch.int64)
    masks = torch.zeros(parents.shape, dtype=torch.int64, device=parents.device)
    for j in range(n):
        up = masks.gather(-1, parents[..., j:j + 1].clamp(min=0))[..., 0]
        bit = 1 << j if j < 63 else -(1 << 63)
        masks[..., j] = torch.where(parents[..., j] >= 0, up, torch.zeros_like(up)) | bit
    return masks


def _word_address(word, device):
    """The address of an error word: an int as it is, or an int32 tensor of one element that kernels on `device` can
    write (there, or in pinned host memory). Only the address is looked at, never the word."""
    if isinstance(word, int):
        return word
    if not isinstance(word, torch.Tensor) or word.dtype != torch.int32 or word.numel() != 1:
        raise ValueError("err_word must be an address or an int32 tensor of one element")
    if word.device != device and not (word.device.type == "cpu" and word.is_pinned()):
        raise ValueError("err_word must be on {} or in pinned host memory".format(device))
    return word.data_ptr()


class XdsOffloadCoordinator:
    """Per-layer SIEVE state and decode-step driver for one device."""

    _require_cuda = True  # the kernels take device addresses (a host-only test subclass may lift this)

    def __init__(self, device, layer_num, pool_size, device_buffer_size, top_k, max_num_reqs, max_context_len):
        self._k = _kvops_module()
        self.device = torch.device(device)
        if self._require_cuda and self.device.type != "cuda":
            raise ValueError("XdsOffloadCoordinator needs a CUDA device, got {}".format(device))
        self.layer_num = layer_num
        self.pool_size = pool_size
        self.device_buffer_size = device_buffer_size
        self.top_k = top_k
        self.max_num_reqs = max_num_reqs
        self.max_context_len = max_context_len
        # Derived sizes (xds_offload.py:33-37).
        self.padded_buffer_size = align(device_buffer_size, 16)
        self.visited_stride_b = align((self.padded_buffer_size + 7) // 8, 64)
        self.ht_size = compute_ht_size(self.padded_buffer_size, top_k)
        L, p, padded, dev = layer_num, pool_size, self.padded_buffer_size, self.device
        self.device_buffer_tokens = torch.full((L, p, padded), -1, dtype=torch.int32, device=dev)
        self.device_buffer_visited = torch.zeros((L, p, self.visited_stride_b), dtype=torch.uint8, device=dev)
        # int16 storage, uint16 semantics (the kernel reinterprets the bits).
        self.device_buffer_ht = torch.zeros((L, p, self.ht_size), dtype=torch.int16, device=dev)
        self.sieve_hand = torch.zeros((L, p, 16), dtype=torch.int32, device=dev)
        self.prefill_lens = torch.zeros(p, dtype=torch.int32, device=dev)
        self.req_host_base = torch.zeros(max_num_reqs, dtype=torch.int64, device=dev)
        self.top_k_device_slots = torch.zeros((max_num_reqs, top_k), dtype=torch.int32, device=dev)
        self.is_miss = torch.zeros((max_num_reqs, top_k), dtype=torch.int8, device=dev)
        self.num_real = torch.zeros(1, dtype=torch.int32, device=dev)
        self._req_pool_indices = None
        self._seq_lens = None
        # pinned, where attend's launches leave their first errCode (made here, not in a call that may be captured)
        self._attend_err = torch.zeros(1, dtype=torch.int32, pin_memory=True).numpy() if dev.type == "cuda" else None
        self._attend_err_at = self._attend_err.ctypes.data if dev.type == "cuda" else 0

    def _stream(self):
        return torch.cuda.current_stream(self.device).cuda_stream if self.device.type == "cuda" else 0

    def _on_device(self):
        return torch.cuda.device(self.device) if self.device.type == "cuda" else contextlib.nullcontext()

    def admit_request(self, req_batch_idx, req_pool_idx, prefill_len, host_base_row):
        """Identity admission: slot s holds token s for s < min(prefill, dbs), then the
        tables of every layer are rebuilt on the device (xds_offload.py:56-77)."""
        if not 0 <= req_pool_idx < self.pool_size:
            raise ValueError("req_pool_idx out of range: {}".format(req_pool_idx))
        if not 0 <= req_batch_idx < self.max_num_reqs:
            raise ValueError("req_batch_idx out of range: {}".format(req_batch_idx))
        n = min(prefill_len, self.device_buffer_size)
        with self._on_device():
            self.device_buffer_tokens[:, req_pool_idx, :] = -1
            self.device_buffer_tokens[:, req_pool_idx, :n] = torch.arange(n, dtype=torch.int32, device=self.device)
            self.device_buffer_visited[:, req_pool_idx, :].zero_()
            self.sieve_hand[:, req_pool_idx, :].zero_()
            self.prefill_lens[req_pool_idx] = prefill_len
            self.req_host_base[req_batch_idx] = host_base_row
            self._k.sieve_ht_init(self.device_buffer_tokens.data_ptr(), self.device_buffer_ht.data_ptr(),
                                  self.prefill_lens.data_ptr(), req_pool_idx, 1, self.layer_num, self.pool_size,
                                  self.device_buffer_size, self.padded_buffer_size, self.ht_size, self._stream(),
                                  self.layer_num)

    def admit_all(self, prefill_lens, host_base_rows):
        """Admit pool rows 0..n-1 (batch row r = pool row r) with one table build."""
        n = len(prefill_lens)
        pre = torch.as_tensor(prefill_lens, dtype=torch.int32, device=self.device)
        with self._on_device():
            idx = torch.arange(self.padded_buffer_size, dtype=torch.int32, device=self.device)
            lim = torch.clamp(pre, max=self.device_buffer_size)[:, None]
            rows = torch.where(idx[None, :] < lim, idx[None, :], torch.full_like(idx[None, :], -1))
            self.device_buffer_tokens[:, :n, :] = rows[None]
            self.device_buffer_visited[:, :n, :].zero_()
            self.sieve_hand[:, :n, :].zero_()
            self.prefill_lens[:n] = pre
            self.req_host_base[:n] = torch.as_tensor(host_base_rows, dtype=torch.int64, device=self.device)
            self._k.sieve_ht_init(self.device_buffer_tokens.data_ptr(), self.device_buffer_ht.data_ptr(),
                                  self.prefill_lens.data_ptr(), 0, n, self.layer_num, self.pool_size,
                                  self.device_buffer_size, self.padded_buffer_size, self.ht_size, self._stream(), 0)

    def set_batch(self, req_pool_indices, seq_lens):
        """Batch context for the next decode steps (xds_offload.py:79-87)."""
        if req_pool_indices.dtype != torch.int64:
            raise ValueError("req_pool_indices must be int64")
        if seq_lens.dtype != torch.int32:
            seq_lens = seq_lens.to(torch.int32)
        self._req_pool_indices = req_pool_indices
        self._seq_lens = seq_lens
        self.num_real[0] = req_pool_indices.shape[0]

    def sieve_update(self, layer_id, topk_indices, block_dim=8, stream=None):
        """SIEVE miss detection for one layer (xds_offload.py:90-101)."""
        if topk_indices.dtype != torch.int32:
            raise ValueError("topk_indices must be int32")
        self._k.sieve_update(topk_indices.data_ptr(), self._req_pool_indices.data_ptr(), self._seq_lens.data_ptr(),
                             self.prefill_lens.data_ptr(), self.device_buffer_tokens[layer_id].data_ptr(),
                             self.device_buffer_visited[layer_id].data_ptr(),
                             self.device_buffer_ht[layer_id].data_ptr(), self.sieve_hand[layer_id].data_ptr(),
                             self.top_k_device_slots.data_ptr(), self.is_miss.data_ptr(), self.num_real.data_ptr(),
                             self.top_k, self.device_buffer_size, self.padded_buffer_size, self.visited_stride_b,
                             self.max_num_reqs, self.pool_size, self._stream() if stream is None else stream,
                             block_dim)

    def miss_count(self):
        """Device-side miss count tensor (xds_offload.py:103-106)."""
        return self.is_miss.sum()

    def attend_error(self):
        """The first errCode that a launch of attend() left since the last look (0: none), which clears it."""
        if self._attend_err is None:
            return 0
        code, self._attend_err[0] = int(self._attend_err[0]), 0
        return code

    def attend(self, q, hot_row_base, *, hot_req_stride_rows=0, hot_rows=None, row_format="raw", scale=None,
               topk_device_slots=None, draft_rows=None, tree=None, out=None, lse=None, workspace=None, stream=None,
               err_word=0, wait_clocks=0):
        """Attention of this step's tokens over one layer's hot rows (kvops_attend_hot).

        q: float16 or bfloat16 [B, heads, 576] (one token a request) or [B, tokens, heads, 576],
        B <= max_num_reqs; its batch rows are set_batch's. The keys of request r are the hot rows
        of its slots (the last sieve_update's top_k_device_slots, or `topk_device_slots`: int32
        [B, K], or [B, tokens, K] for a list per token), entries outside [0, hot_rows) left out,
        and of draft_rows [B, drafts, 576] those whose bit is set in tree[r, token] (int64
        [B, tokens], see tree_masks; None: a chain, token t seeing drafted rows 0..t). A row's
        first 512 values are its value. hot_row_base: the layer's hot rows (a tensor, or an
        address), hot_req_stride_rows from one pool row to the next (0: shared), of row_format
        "raw" (the type of q; a floating-point tensor of another type is refused, one of integers taken as it
        is) or stored in 8 bits. hot_rows: rows a slot may name (default: the
        stride; for shared rows those that the tensor holds, or device_buffer_size where an address is
        given). sieve_update gives a token generated since the prompt, position t >= prefill_len, the
        slot padded_buffer_size + t - prefill_len; its row belongs there, so the stride (or the shared
        rows) must reach that far. Where sieve_update's own slots do not fit the default, errCode 0x104
        says so; with hot_rows given they are left out. scale: of the scores. It has to be given: it is the
        model's, mostly the inverse square root of its heads' own width, which a row of 576 does not tell.

        Returns (out, lse): [.., heads, 512] in q's type and fp32 [.., heads], written for the
        batch rows below num_real only. A token without any key gets out 0 and lse -inf. out, lse
        and workspace (uint8, at least _kvops.attend_workspace(...) bytes, used by one call at a
        time) may be given; otherwise they are allocated for the call. err_word: address (or int32
        tensor of one element, on this device or pinned) of a word that receives errCode 0x103 if a wait
        inside the kernel gave up, which leaves outputs undefined, or 0x104 (above); by default a word of
        the coordinator's, whose code the next call raises (and `attend_error()` returns, once the launch
        has ended). wait_clocks: SM clocks that a tile of 64 keys may keep the next ones
        waiting (0: 2^30, half a second, as for every other wait inside the kernel)."""
        shape, strides = q.shape, q.stride()
        squeeze = len(shape) == 3
        if len(shape) not in (3, 4) or shape[-1] != KEY_DIM or strides[-1] != 1:
            raise ValueError("attend: q must be [B, heads, 576] or [B, tokens, heads, 576] with unit last stride")
        if squeeze:
            (B, H, _), T, strides = shape, 1, (strides[0], 0, strides[1])
        else:
            B, T, H, _ = shape
        dtype = dtype_name(q.dtype)
        if B > self.max_num_reqs:
            raise ValueError("attend: {} batch rows, max_num_reqs is {}".format(B, self.max_num_reqs))
        if self._req_pool_indices is None or self._req_pool_indices.shape[0] < B:
            raise RuntimeError("attend: call set_batch() with at least q's batch rows first")
        slots = self.top_k_device_slots if topk_device_slots is None else topk_device_slots
        s_shape, s_strides = slots.shape, slots.stride()
        if slots.dtype != torch.int32 or len(s_shape) not in (2, 3) or s_shape[0] < B or \
                (len(s_shape) == 3 and s_shape[1] != T) or (s_shape[-1] > 1 and s_strides[-1] != 1):
            raise ValueError("attend: topk_device_slots must be int32 [B, K] or [B, tokens, K] with unit last stride")
        K = s_shape[-1]
        if row_format not in ROW_BYTES:
            raise ValueError("attend: row_format must be 'raw', 'e4m3' or 'int8', got {!r}".format(row_format))
        report_slots = hot_rows is None and slots is self.top_k_device_slots
        if hot_rows is None:
            hot_rows = hot_req_stride_rows or self.device_buffer_size
            if hot_req_stride_rows == 0 and isinstance(hot_row_base, torch.Tensor):
                hot_rows = max(hot_rows, hot_row_base.numel() * hot_row_base.element_size() // ROW_BYTES[row_format])
        D, draft_at, draft_strides = 0, 0, (0, 0)
        if draft_rows is not None:
            if draft_rows.dim() != 3 or draft_rows.shape[0] < B or draft_rows.shape[2] != KEY_DIM or \
                    draft_rows.dtype != q.dtype or draft_rows.stride(2) != 1:
                raise ValueError("attend: draft_rows must be [B, drafts, 576] of q's type with unit last stride")
            D = draft_rows.shape[1]
            if D:
                draft_at = draft_rows.data_ptr()
                draft_strides = (draft_rows.stride(0) if draft_rows.shape[0] > 1 else 0, draft_rows.stride(1) if D > 1 else 0)
        if tree is not None and (tree.dtype != torch.int64 or tree.dim() != 2 or tree.shape[0] < B or
                                 tree.shape[1] != T or not tree.is_contiguous()):
            raise ValueError("attend: tree must be a contiguous int64 [B, tokens]")
        if isinstance(hot_row_base, torch.Tensor):
            need = ((self.pool_size - 1) * hot_req_stride_rows + hot_rows) * ROW_BYTES[row_format]
            if hot_row_base.numel() * hot_row_base.element_size() < need or not hot_row_base.is_contiguous():
                raise ValueError("attend: hot rows must be contiguous and hold {} bytes".format(need))
            if hot_row_base.is_floating_point() and (hot_row_base.dtype != q.dtype if row_format == "raw" else
                                                     hot_row_base.element_size() > 1):
                raise ValueError("attend: hot rows of row_format {!r} must be {}, got {}".format(
                    row_format, q.dtype if row_format == "raw" else "bytes", hot_row_base.dtype))
            if hot_row_base.device != self.top_k_device_slots.device:
                raise ValueError("attend: hot rows must be on {}".format(self.top_k_device_slots.device))
            hot = hot_row_base.data_ptr()
        else:
            hot = hot_row_base
        for name, x, want, each in (("out", out, q.dtype, VALUE_DIM), ("lse", lse, torch.float32, 1)):
            if x is not None and (x.dtype != want or not x.is_contiguous() or x.numel() != B * T * H * each):
                raise ValueError("attend: {} must be a contiguous {} of {} elements".format(name, want, B * T * H * each))
        dev = self.top_k_device_slots.device
        if workspace is not None and not workspace.is_contiguous():
            raise ValueError("attend: workspace must be contiguous")
        if not self._req_pool_indices.is_contiguous():
            raise ValueError("attend: set_batch()'s req_pool_indices must be contiguous")
        for x in (q, slots, draft_rows, tree, out, lse, workspace, self._req_pool_indices):
            if x is not None and x.device != dev:
                raise ValueError("attend: every tensor must be on {}".format(dev))
        err_word = _word_address(err_word, dev)
        if err_word == 0 and dev.type == "cuda":
            if self._attend_err[0] != 0:
                code = self.attend_error()
                raise RuntimeError("attend: {} (errCode 0x{:x})".format(ATTEND_ERRORS.get(code, "an earlier call failed"), code))
            err_word = self._attend_err_at
        args = (q, B, T, H, K, D, squeeze, strides, slots, hot, hot_req_stride_rows, hot_rows, row_format, dtype, scale,
                draft_at, draft_strides, tree, out, lse, workspace, stream, err_word, report_slots, wait_clocks)
        if dev.type == "cuda" and (stream is not None or torch.cuda.current_device() != dev.index):
            with torch.cuda.device(dev):
                if stream is None or (out is not None and lse is not None and workspace is not None):
                    return self._attend(*args)
                # what is allocated below belongs to the stream that uses it
                with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=dev)):
                    return self._attend(*args)
        return self._attend(*args)

    def _attend(self, q, B, T, H, K, D, squeeze, strides, slots, hot, hot_req_stride_rows, hot_rows, row_format, dtype, scale,
                draft_at, draft_strides, tree, out, lse, workspace, stream, err_word, report_slots,
                wait_clocks):
        """attend() on checked arguments and the current device."""
        if stream is None:  # (no Stream object: 4 us of a 20 us call)
            stream = torch._C._cuda_getCurrentRawStream(q.device.index) if q.is_cuda else 0
        s_shape, s_strides = slots.shape, slots.stride()
        if out is None:
            out = q.new_empty((B, H, VALUE_DIM) if squeeze else (B, T, H, VALUE_DIM))
        if lse is None:
            lse = q.new_empty((B, H) if squeeze else (B, T, H), dtype=torch.float32)
        room = workspace.numel() * workspace.element_size() if workspace is not None else 0
        if workspace is None:
            room = self._k.attend_workspace(B, T, H, K, D, row_format, dtype)
            if room:
                workspace = q.new_empty(room, dtype=torch.uint8)
        if scale is None:
            raise ValueError("attend: scale must be given (mostly the inverse square root of the heads' own width)")
        # (the stride of a dimension of one entry is never used)
        self._k.attend_hot(
            q.data_ptr(), strides[0] if B > 1 else 0, strides[1] if T > 1 else 0, strides[2] if H > 1 else 0, hot,
            hot_req_stride_rows, hot_rows, self._req_pool_indices.data_ptr(), self.pool_size, slots.data_ptr(),
            s_strides[0] if s_shape[0] > 1 else 0, s_strides[1] if len(s_shape) == 3 and T > 1 else 0,
            self.num_real.data_ptr(), draft_at, draft_strides[0], draft_strides[1],
            tree.data_ptr() if tree is not None else 0, out.data_ptr(), lse.data_ptr(),
            workspace.data_ptr() if room else 0, room, B, T, H, K, D, row_format, dtype,
            scale, stream, err_word=err_word, report_slots=report_slots,
            wait_clocks=wait_clocks)
        return out, lse

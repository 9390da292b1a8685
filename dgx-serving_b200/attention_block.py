"""A decoder layer's attention block: W4A8 projections around the 8-bit paged KV cache.

One step takes the new rows of any number of requests side by side (prompts, chunks of prompts and single tokens mixed):

    plan      block tables and slots of the step, from the lengths, on the GPU        w4a8_kv_plan
    qkv       the rows' queries, keys and values, one W4A8 product                    w4a8_linear
    rotate    the caller's, if there is one: rotary positions, norms                  -
    append    keys and values into their blocks as int8 codes                         w4a8_kv_append_q8
    attend    every row over all tokens that its request holds                        w4a8_attention_q8
    out       the output product                                                      w4a8_linear

The plan belongs to the step, not to the layer: PagedTables is shared by all layers, each of which has a cache of its own under the same
block ids.  Nothing here waits for the GPU; lengths, tables and the free list stay on it.  The graphs whose place this takes keep an fp32 or
fp16 cache, contiguous for each request (kernels/kv_store.cuh, models/qwen35_decode.cu:148-175).
"""
import importlib

import torch

w4a8 = importlib.import_module(__package__)


class PagedTables:
    """Which blocks the requests' tokens lie in: lengths, block tables and the free list of `num_blocks` blocks, on the GPU.  A step is step(),
    the layers' calls, done(), and release() of the requests that have ended."""

    def __init__(self, requests, width, num_blocks, block, device="cuda"):
        i32 = dict(dtype=torch.int32, device=device)
        self.R, self.width, self.num_blocks, self.block = requests, width, num_blocks, block
        self.kv_len = torch.zeros(requests, **i32)
        self.table = torch.full((requests, width), -1, **i32)
        self.free = torch.arange(num_blocks + 1, **i32)      # the last is no block: where release puts what is none
        self.seq_len = torch.zeros(requests, **i32)
        self.cu = torch.zeros(requests + 1, **i32)
        self.status = torch.zeros(4, **i32)                  # [0]: the first free block of the next step
        self.first = torch.zeros(1, **i32)
        self.slot = torch.empty(0, **i32)                    # of the step's rows, and their places in their requests
        self.position = torch.empty(0, **i32)

    def step(self, new_len, T):
        """Room for new_len[r] tokens of each request (int32, on the GPU), T rows in all; slots of the rows, -1 where there was none."""
        if new_len.dtype != torch.int32 or new_len.shape != (self.R,) or not new_len.is_contiguous() or new_len.device != self.table.device:
            raise ValueError("new_len: %d int32 numbers, contiguous, on %s" % (self.R, self.table.device))
        self.slot = torch.empty(T, dtype=torch.int32, device=new_len.device)
        self.position = torch.empty_like(self.slot)
        w4a8.kv_plan(self.kv_len, new_len, self.R, self.block, self.table, self.width, self.free, self.num_blocks, self.first, self.seq_len, self.cu,
                     self.slot, self.position, T, self.status)
        return self.slot

    def done(self):
        """After the step's last layer: the tokens placed are the requests'; those that got no room keep what they had."""
        torch.where(self.seq_len > 0, self.seq_len, self.kv_len, out=self.kv_len)
        self.first.copy_(self.status[:1])

    def release(self, ended):
        """Between done() and the next step: the requests that `ended` marks (bool, on the GPU) hold nothing any more, their blocks go back to the
        free list, in front of what is left of it."""
        held = (self.kv_len + self.block - 1) // self.block
        blocks = (torch.arange(self.width, device=held.device) < held[:, None]) & ended[:, None]
        at = self.first - torch.cumsum(blocks.flatten(), 0)
        self.free[torch.where(blocks.flatten(), at, self.num_blocks)] = self.table.flatten()
        self.first -= blocks.sum()
        self.table.masked_fill_(blocks, -1)
        self.kv_len.masked_fill_(ended, 0)


class AttentionBlock:
    """One layer.  wqkv: (Wq, scales) of [(heads_q + 2 * heads) * dim][hidden] (queries, keys, values), wo: of [hidden][heads_q * dim]; both
    packed int4 with fp32 scales of 32 elements.  rotate(q, k, position), if there is one, is called between the QKV product and the append with the rows'
    queries [T][heads_q][dim] and keys [T][heads][dim], to be changed in place (rotary positions, norms of queries and keys), and the rows' positions."""

    def __init__(self, wqkv, wo, hidden, heads_q, heads, dim, tables, max_rows, scale=None, window=0, softcap=0.0, rotate=None):
        self.wqkv, self.wo, self.hidden, self.heads_q, self.heads, self.dim, self.tables = wqkv, wo, hidden, heads_q, heads, dim, tables
        self.max_rows, self.rotate = max_rows, rotate
        self.scale, self.window, self.softcap = dim ** -0.5 if scale is None else scale, window, softcap
        dev = tables.table.device
        codes = (tables.num_blocks, heads, tables.block, dim)
        self.cache = w4a8.KVCache.of(torch.zeros(codes, dtype=torch.int8, device=dev), torch.zeros(codes, dtype=torch.int8, device=dev),
                                     torch.zeros(codes[:2], device=dev), torch.zeros(codes[:2], device=dev))
        self.cols = (heads_q + 2 * heads) * dim
        for (wq, sc), n, k, name in ((wqkv, self.cols, hidden, "wqkv"), (wo, hidden, heads_q * dim, "wo")):
            if wq.numel() * wq.element_size() != n * k // 2 or sc.dtype != torch.float32 or sc.numel() != n * k // 32 or not (wq.is_contiguous() and sc.is_contiguous()):
                raise ValueError("%s: %d rows of %d packed int4 and %d fp32 scales, contiguous" % (name, n, k, k // 32))
        self.qkv = torch.empty(max_rows, self.cols, device=dev)
        self.mix = torch.empty(max_rows, heads_q * dim, device=dev)
        widest = max(hidden, heads_q * dim)
        self.xq = torch.empty(max_rows * widest, dtype=torch.int8, device=dev)
        self.xs = torch.empty(max_rows * widest // 32, device=dev)
        self.xsum = torch.empty(max_rows * widest // 32, dtype=torch.int32, device=dev)
        self.workspace = torch.zeros(w4a8.attention_q8_workspace_bytes(heads_q, self.cache), dtype=torch.uint8, device=dev)

    def _check(self, X):
        """The launches below take pointers: what does not fit the buffers or the step's plan is refused here."""
        if X.dim() != 2 or X.shape[1] != self.hidden or X.dtype != torch.float32 or not X.is_contiguous():
            raise ValueError("X: contiguous fp32 rows of %d" % self.hidden)
        if X.shape[0] > self.max_rows:
            raise ValueError("%d rows: this block has room for %d" % (X.shape[0], self.max_rows))
        if X.shape[0] != self.tables.slot.numel():
            raise ValueError("%d rows: the step was planned for %d" % (X.shape[0], self.tables.slot.numel()))
        if not X.is_cuda or X.device != self.qkv.device:
            raise ValueError("X is on %s, the block on %s" % (X.device, self.qkv.device))

    def __call__(self, X, max_q=0):
        """X[T][hidden] fp32, the step's rows in the order of the requests -> the block's output [T][hidden], zeros in rows that no request
        owns (a padded step).  max_q: no request has more rows."""
        t, T = self.tables, X.shape[0]
        self._check(X)
        Y = torch.empty_like(X)
        q, k, v = self.qkv, self.qkv[:, self.heads_q * self.dim:], self.qkv[:, (self.heads_q + self.heads) * self.dim:]
        self.mix[:T].zero_()                                 # rows behind the last request's (a padded step) are left as they are by the attention
        w4a8.linear(X, self.xq, self.xs, self.xsum, *self.wqkv, self.qkv, T, self.cols, self.hidden)
        if self.rotate is not None:
            self.rotate(q[:T, : self.heads_q * self.dim].view(T, self.heads_q, self.dim), k[:T, : self.heads * self.dim].view(T, self.heads, self.dim), t.position)
        w4a8.launch_kv_append_q8(k, v, self.cols, t.slot, T, self.cache)
        w4a8.launch_attention_q8(q, self.cols, self.cache, t.table, t.width, t.cu, t.seq_len, t.R, T, self.heads_q, self.mix, self.heads_q * self.dim,
                                 self.scale, "fp32", self.workspace, window=self.window, softcap=self.softcap, max_q=max_q)
        w4a8.linear(self.mix, self.xq, self.xs, self.xsum, *self.wo, Y, T, self.hidden, self.heads_q * self.dim)
        return Y

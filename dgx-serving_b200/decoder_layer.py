"""A decoder layer of routed experts: the residual stream through the attention block and the expert block.

    add, norm     the block output that is still to be added, and the norm in front of the attention       w4a8_add_norm
    attention     attention_block.AttentionBlock
    add, norm     the attention's output, and the norm in front of the experts, in fp32 and as rows of 8 bits   w4a8_add_norm
    logits        the router's product, weights of 8 bits                                                  w4a8_gemm_w8a8
    route         the tokens' experts and their weights                                                    w4a8_moe_route
    experts       their products, added up                                                                 w4a8_moe_block

A layer leaves its expert output to be added by the next one's first norm (or the last one of the model), so that the stream is read and written
twice a layer.  Norms of a block's output before it is added, gates and residual scales are the Norms' (post_weight, gate, alpha).  Nothing here
waits for the GPU.  The graphs whose place this takes launch each step by itself (models/qwen35_decode.cu:140-229, models/moe_block.cuh:20-52).
"""
import importlib

import torch

w4a8 = importlib.import_module(__package__)
attention_block = importlib.import_module(__package__ + ".attention_block")


class DecoderLayer:
    """attention: an AttentionBlock.  norm_in, norm_mlp: Norms of its hidden size, fp32.  router: a Router; router_w: int8 [experts][hidden] and fp32 [experts].
    gate_up, down: (Wq, scales) of all experts as moe_block takes them, `inner` elements an expert."""

    def __init__(self, attention, norm_in, norm_mlp, router, router_w, gate_up, down, inner, scale_dtype=0, act=0):
        self.attention, self.norm_in, self.norm_mlp, self.router, self.router_w = attention, norm_in, norm_mlp, router, router_w
        self.gate_up, self.down, self.inner, self.scale_dtype, self.act = gate_up, down, inner, scale_dtype, act
        H, rows, dev = attention.hidden, attention.max_rows, attention.qkv.device
        self.H, E, k = H, router.experts, router.topk
        for n, name in ((norm_in, "norm_in"), (norm_mlp, "norm_mlp")):
            if n.K != H or n.dtype != w4a8.DTYPES["fp32"] or n.y_dtype != w4a8.DTYPES["fp32"] or n.gate_ld != 0:
                raise ValueError("%s: fp32 rows of %d, no gate of single tokens" % (name, H))
            w4a8.struct_on(n, dev, name)
            # what a launch in the middle of the layer would refuse
            if (n.variant in (0, 1) and not n.weight) or (n is norm_mlp and n.post_variant in (0, 1) and not n.post_weight):
                raise ValueError("%s: a norm without its weight" % name)
            if any((p or 0) % 16 for p in (n.weight, n.post_weight, n.gate)):
                raise ValueError("%s: weights and gate must be 16-byte aligned" % name)
            w4a8.check_norm(n)
        w4a8.struct_on(router, dev, "router")
        w4a8.check_router(router)
        if not attention_block.check_matrix(router_w, E, H, "router_w"):
            raise ValueError("router_w: int8")
        size = 2 if scale_dtype else 4
        for (wq, sc), n, kk, name in ((gate_up, 2 * inner, H, "gate_up"), (down, H, inner, "down")):
            if wq.device != dev or sc.device != dev or router_w[0].device != dev or router_w[1].device != dev:
                raise ValueError("%s, router_w: on %s, as the attention is" % (name, dev))
            if wq.numel() * wq.element_size() != E * n * kk // 2 or sc.numel() * sc.element_size() != E * n * kk // 32 * size or not (wq.is_contiguous() and sc.is_contiguous()):
                raise ValueError("%s: packed int4 of %d experts, [%d][%d], and scales of 32 elements, contiguous" % (name, E, n, kk))
            if wq.data_ptr() % 16 or sc.data_ptr() % 16:
                raise ValueError("%s: weights and scales must be 16-byte aligned" % name)
        w4a8.check_moe(k, H, inner, E, scale_dtype, act)
        self.normed = torch.empty(rows, H, device=dev)
        self.xq, self.xs = torch.empty(rows, H, dtype=torch.int8, device=dev), torch.empty(rows, device=dev)
        self.logits = torch.empty(rows, E, device=dev)
        self.idx, self.weight = torch.empty(rows, k, dtype=torch.int32, device=dev), torch.empty(rows, k, device=dev)
        self.workspace = torch.empty(w4a8.moe_layout_for(rows, k, H, inner, E).bytes, dtype=torch.uint8, device=dev)

    def __call__(self, h, y=None, max_q=0):
        """h[T][hidden] fp32, the residual stream, changed in place; y: what is still to be added to it, or None.  Returns the experts' output, to be added
        by what comes next."""
        T, H = h.shape[0], self.H
        for x, name in ((h, "h"), (y, "y")):
            if x is not None and (x.dim() != 2 or x.shape != (T, H) or x.dtype != torch.float32 or not x.is_contiguous() or x.device != self.normed.device):
                raise ValueError("%s: contiguous fp32 rows of %d on %s" % (name, H, self.normed.device))
        if T > self.normed.shape[0]:
            raise ValueError("%d rows: this layer has room for %d" % (T, self.normed.shape[0]))
        if not h.is_cuda or h.device.index != torch.cuda.current_device():
            raise ValueError("h is on %s, which is not the current GPU" % h.device)
        if max_q < 0 or T * self.router.topk > 1 << 24:
            raise ValueError("max_q=%d, %d rows of %d experts (at most 2^24)" % (max_q, T, self.router.topk))
        n = self.normed[:T]
        self.attention._check(n)                              # nothing is launched, and h not changed, for a call that is refused
        w4a8.launch_add_norm(self.norm_in, h, y, T, H_out=None if y is None else h, N=n)
        a = self.attention(n, max_q=max_q)
        w4a8.launch_add_norm(self.norm_mlp, h, a, T, H_out=h, N=n, xq=self.xq, xs=self.xs, group=0)
        w4a8.launch_gemm_w8a8(self.xq, self.xs, *self.router_w, self.logits, self.router.experts, T, self.router.experts, H)
        w4a8.launch_moe_route(self.router, self.logits, self.router.experts, T, self.idx, self.weight)
        out = torch.empty_like(h)
        w4a8.moe_block(n, *self.gate_up, *self.down, self.idx, self.weight, out, T, self.router.topk, H, self.inner, self.router.experts, self.workspace,
                       scale_dtype=self.scale_dtype, act=self.act)
        return out

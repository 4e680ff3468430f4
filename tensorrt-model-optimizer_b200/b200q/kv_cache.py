"""A paged KV cache held in NVFP4, in the arithmetic of the ``NVFP4_KV_CFG`` quantisers.

The KV configurations calibrate ``k_bmm_quantizer`` / ``v_bmm_quantizer`` of an attention module and fake-quantise keys
and values; this class holds what they stand for in 4.5 bits an element and attends over it.  Page tables, slots and
lengths live on the GPU (``ops.kv_step``), so that a step can be captured into a CUDA graph and replayed.

    cache = NVFP4KVCache.from_quantizers([(layer.k_bmm_quantizer, layer.v_bmm_quantizer) for layer in layers],
                                         num_pages=4096, kv_heads=8, head_dim=128, max_requests=64)
    step = cache.step(new_lens, tokens)                    # once a step
    for i, layer in enumerate(layers):                     # in every layer
        cache.append(i, k, v, step)
        out = cache.attend(i, q, step)
"""
from __future__ import annotations

import torch

from . import ops

__all__ = ["NVFP4KVCache"]


def _scale2(quantizer, what: str) -> torch.Tensor:
    from .export import get_scaling_factor

    bs = getattr(quantizer, "block_sizes", None) or {}
    if not (quantizer.is_enabled and quantizer.num_bits == (2, 1) and bs.get(-1) == 16 and bs.get("scale_bits") == (4, 3)):
        raise ValueError(f"b200q: the {what} quantiser is not an enabled NVFP4 quantiser with blocks of 16")
    if getattr(quantizer, "bias", None) or getattr(quantizer, "_bias_value", None) is not None:
        raise NotImplementedError(f"b200q: the {what} quantiser has an affine bias, which the cache does not hold")
    if getattr(quantizer, "_rotate", False):
        raise NotImplementedError(f"b200q: the {what} quantiser rotates its input; rotate queries and keys before the cache "
                                  "and use a quantiser without rotation")
    if getattr(quantizer, "pre_quant_scale", None) is not None:
        raise NotImplementedError(f"b200q: the {what} quantiser has a pre-quant scale, which the cache does not apply")
    s = get_scaling_factor(quantizer)
    if s is None or s.numel() != 1:
        raise ValueError(f"b200q: the {what} quantiser has no calibrated per-tensor amax")
    return s


class NVFP4KVCache:
    """``num_pages`` pages of ``page_size`` tokens shared by up to ``max_requests`` requests, for ``len(scales)`` layers.

    ``scales``: (k_scale2, v_scale2) per layer, amax / 2688 each.  Every layer has its own codes and block scales; the
    page table, the lengths and the free list are common to all.  Row r of ``lens`` and ``block_table`` is request r;
    a free row has length 0."""

    def __init__(self, scales, num_pages: int, kv_heads: int, head_dim: int, max_requests: int, page_size: int = 64,
                 max_pages_per_request: int | None = None, device="cuda"):
        if num_pages <= 0 or max_requests <= 0 or kv_heads <= 0 or page_size <= 0 or page_size % 16:
            raise ValueError("b200q: an NVFP4KVCache needs positive sizes and pages of a multiple of 16 tokens")
        if head_dim not in ops._KV_DIMS:
            raise ValueError(f"b200q: NVFP4KVCache covers heads of {ops._KV_DIMS}, got {head_dim}")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("b200q: NVFP4KVCache lives on a CUDA device (no CPU path exists)")
        self.page_size, self.kv_heads, self.head_dim = page_size, kv_heads, head_dim
        width = num_pages if max_pages_per_request is None else max_pages_per_request

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device=device)

        self.lens, self.taken, self.status = ints(max_requests), ints(1), ints(1)
        self.block_table = ints(max_requests, width, fill=-1)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.layers = []
        for k2, v2 in scales:
            def side():
                codes = torch.zeros(num_pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device)
                block = torch.zeros(num_pages, kv_heads, page_size, head_dim // 16, dtype=torch.uint8, device=device)
                return codes, block.view(torch.float8_e4m3fn)

            k2, v2 = (torch.as_tensor(s, dtype=torch.float32).reshape(()).to(device) for s in (k2, v2))
            self.layers.append((side(), side(), k2, v2))

    @classmethod
    def from_quantizers(cls, quantizers, **sizes) -> "NVFP4KVCache":
        """``quantizers``: (k_bmm_quantizer, v_bmm_quantizer) per layer, calibrated in an NVFP4 format."""
        return cls([(_scale2(k, "key"), _scale2(v, "value")) for k, v in quantizers], **sizes)

    def step(self, new_lens: torch.Tensor, tokens: int) -> ops.KvStep:
        """Room for ``new_lens[r]`` more tokens of every request r (int32 [max_requests], 0 for rows without any), in
        ``tokens`` rows of the step's tensors.  Lengths and tables advance; a request that does not fit keeps its length,
        gets no slots, and its rows see nothing (see ``check``)."""
        st = ops.kv_step(self.lens, new_lens, self.free_pages, self.taken, self.block_table, self.page_size, tokens)
        self.lens.copy_(st.lens)
        self.taken.copy_(st.taken)
        self.status.bitwise_or_(st.status)
        return st

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: ops.KvStep, return_values: bool = False):
        """Quantise the step's keys and values [tokens, kv_heads, head_dim] into ``layer`` (``ops.nvfp4_kv_append``)."""
        kc, vc, k2, v2 = self.layers[layer]
        return ops.nvfp4_kv_append(k, v, step.slots, kc, vc, k2, v2, return_values=return_values)

    def attend(self, layer: int, q: torch.Tensor, step: ops.KvStep, scale: float | None = None, out=None,
               return_lse: bool = False):
        """Causal attention of the step's queries [tokens, heads, head_dim] over ``layer`` (``ops.nvfp4_kv_attention``);
        rows of a request that the step refused are zero, and so are rows behind the last request's (a given ``out`` keeps
        what it holds there)."""
        kc, vc, k2, v2 = self.layers[layer]
        lens = step.lens if step.seen is None else step.seen
        return ops.nvfp4_kv_attention(q, kc, vc, k2, v2, self.block_table, lens, cu_q=step.cu_new, scale=scale, out=out,
                                      return_lse=return_lse)

    def release(self, request: int) -> None:
        """Give back the pages of a finished request and free its row.  Reads two lengths from the device (it
        synchronises); not for captured steps."""
        if not 0 <= request < self.lens.numel():
            raise IndexError(f"b200q: no request {request}")
        pages = -(-int(self.lens[request]) // self.page_size)
        taken = int(self.taken)
        self.free_pages[taken - pages:taken] = self.block_table[request, :pages]
        self.taken -= pages
        self.block_table[request] = -1
        self.lens[request] = 0

    def check(self) -> None:
        """Raise if a request was refused since the last check (reads the device: it synchronises)."""
        code = int(self.status)
        if code:
            self.status.zero_()
            why = [text for bit, text in ((1, "no free page was left"), (2, "its row of the block table is full"),
                                          (4, "a length was negative"), (8, "there were more new tokens than rows")) if code & bit]
            raise RuntimeError("b200q: a step refused a request: " + "; ".join(why))

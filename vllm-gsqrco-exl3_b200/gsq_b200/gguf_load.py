"""GGUF file -> GPU weights of this package's linear method, repacked on the GPU.

The reference copies each tensor from the host into the layer's parameter (plugin/vllm_gguf_plugin/quantization/
params.py:75-99, through vLLM's weight loaders) and repacks the IQ3 runs afterwards with torch ops
(quantization/linear.py:425-457). Here the file is memory-mapped (gguf.GGUFReader), each tensor goes to the device
through one reused pinned staging buffer in chunks (so the host never holds a second copy of a large tensor and the
host-side fill of chunk i + 1 overlaps the transfer of chunk i), is placed into the layer's padded multi-shard buffer
on the device, and the IQ3_S / Q6_K runs are repacked in place by the CUDA repack kernels
(process_weights_after_loading -> gsq_iq3s_repack / gsq_q6k_repack). `unpack` still returns GGUF bytes for a consumer
that needs them.

A mixture-of-experts layer's stacks ([experts, rows, row bytes] in the file) are read the same way into the two tensors that
quantization.fused_moe takes; they stay in GGUF order.

Only what these layers need is here: tensor enumeration and layer construction. Model architecture, tokenizer and config
handling of the reference's loader are not.
"""

from __future__ import annotations

import contextlib

import numpy as np
import torch

from . import ops
from .quantization import linear

_CHUNK = 64 << 20
_COPY_THREADS = 8
_pool = None


def _parallel_copy(dst: np.ndarray, src: np.ndarray) -> None:
    """dst[...] = src for row matrices, the rows split over a few threads: one thread copying out of the page cache
    reaches a fraction of what the staging buffer's transfer to the device can take (numpy's copy releases the GIL)."""
    global _pool
    rows = src.shape[0]
    if src.nbytes < (8 << 20) or rows < 2 * _COPY_THREADS:
        dst[...] = src
        return
    if _pool is None:
        from concurrent.futures import ThreadPoolExecutor

        _pool = ThreadPoolExecutor(max_workers=_COPY_THREADS, thread_name_prefix="gguf-stage")
    step = -(-rows // _COPY_THREADS)
    for f in [_pool.submit(np.copyto, dst[i:i + step], src[i:i + step]) for i in range(0, rows, step)]:
        f.result()


def tensors(path: str):
    """{name: (ggml type id, uint8 [rows, row_bytes] memory-mapped view)} of the quantised 2-D tensors of the file whose
    type this package serves, plus F32 / F16 / BF16 ones as (type id, array)."""
    import gguf

    out = {}
    for t in gguf.GGUFReader(path).tensors:
        tid = int(t.tensor_type)
        if tid in ops.LCPP_QUANT_TYPES:
            data = np.asarray(t.data)
            out[t.name] = (tid, data.reshape(data.shape[0], -1).view(np.uint8) if data.ndim == 2 else data.view(np.uint8))
        elif tid in ops.UNQUANTIZED_TYPES:
            out[t.name] = (tid, np.asarray(t.data))
    return out


class _Stager:
    """One pinned buffer, two halves used in turn: the copy of a chunk overlaps the placement of the one before."""

    def __init__(self, device):
        self.dev = torch.device(device)
        self.pin = torch.empty(2 * _CHUNK, dtype=torch.uint8).pin_memory()
        self.events = [torch.cuda.Event(), torch.cuda.Event()]
        self.turn = 0
        self.bytes = 0

    def to_device(self, src: np.ndarray, dst: torch.Tensor) -> None:
        """src: contiguous uint8 rows [r, row_bytes] on the host (memory-mapped); dst: [r, >= row_bytes] device view."""
        r, rb = src.shape
        per = max(1, _CHUNK // rb)
        for i in range(0, r, per):
            c = min(per, r - i)
            h = self.turn
            self.turn ^= 1
            self.events[h].synchronize()                       # the previous use of this half has been copied out
            stage = self.pin[h * _CHUNK: h * _CHUNK + c * rb].view(c, rb)
            _parallel_copy(stage.numpy(), src[i:i + c])
            dst[i:i + c, :rb].copy_(stage, non_blocking=True)
            self.events[h].record()
            self.bytes += c * rb


def load_linear(path_or_tensors, names: list[str], device="cuda:0", params_dtype=torch.bfloat16, stager: _Stager | None = None):
    """A fused linear layer from the named tensors of a GGUF file (one shard each, in this order: q/k/v, gate/up, or a
    single tensor): -> (layer, method) ready for method.apply(layer, x). All tensors must share K."""
    tens = tensors(path_or_tensors) if isinstance(path_or_tensors, str) else path_or_tensors
    metas = [tens[n] for n in names]
    bad = [n for n, (tid, _) in zip(names, metas) if tid not in ops.LCPP_QUANT_TYPES]
    if bad:
        raise ValueError(f"load_linear: {bad[0]} is not a quantised tensor of a served type")
    ks = {m[1].shape[1] // ops.GGML_QUANT_SIZES[m[0]][1] * ops.GGML_QUANT_SIZES[m[0]][0] for m in metas}
    if len(ks) != 1:
        raise ValueError(f"load_linear: tensors with different K: {sorted(ks)}")
    k = ks.pop()
    rows = [m[1].shape[0] for m in metas]
    stager = stager or _Stager(device)
    layer = torch.nn.Module()
    method = linear.GGUFLinearMethod(None)
    with torch.cuda.device(device):
        method.create_weights(layer, k, rows, k, sum(rows), params_dtype)
        fused = len(names) > 1
        for sid, (tid, data) in enumerate(metas):
            dev_rows = torch.empty(data.shape, dtype=torch.uint8, device=device)
            stager.to_device(data, dev_rows)
            layer.weight.load_shard(dev_rows, sid if fused else None)
            if fused:
                layer.weight_type.shard_weight_type[sid] = tid
        layer.weight_type.weight_type = metas[0][0]
        method.process_weights_after_loading(layer)          # pads, places, repacks IQ3_S / Q6_K runs on the GPU
        torch.cuda.synchronize()
    return layer, method


def load_experts(path_or_tensors, gate: str, up: str, down: str, device="cuda:0", experts: slice | None = None, stager: _Stager | None = None):
    """The experts of one layer from the named stacks of a GGUF file ([experts, inter, hidden] gate and up, [experts, hidden,
    inter] down): -> (w13, w2, w13_type, w2_type) for fused_moe.moe_layer_gguf / fused_moe_gguf. `experts` (step 1) takes a
    range of them: an expert-parallel rank's share, which fused_moe_gguf numbers from 0. Gate and up rows of an expert follow each other,
    so the two must have one type."""
    tens = tensors(path_or_tensors) if isinstance(path_or_tensors, str) else path_or_tensors
    names = (gate, up, down)
    for n in names:
        if tens[n][0] not in ops.LCPP_QUANT_TYPES or tens[n][1].ndim != 3:
            raise ValueError(f"load_experts: {n} is not a stack of quantised matrices of a served type")
    (t13, g), (tu, u), (t2, d) = (tens[n] for n in names)
    if t13 != tu or g.shape != u.shape:
        raise ValueError(f"load_experts: {gate} and {up} differ in type or shape: {t13} {g.shape}, {tu} {u.shape}")
    inter = d.shape[2] // ops.GGML_QUANT_SIZES[t2][1] * ops.GGML_QUANT_SIZES[t2][0]
    hidden = g.shape[2] // ops.GGML_QUANT_SIZES[t13][1] * ops.GGML_QUANT_SIZES[t13][0]
    if d.shape[:2] != (g.shape[0], hidden) or g.shape[1] != inter:
        raise ValueError(f"load_experts: {down} {d.shape} does not fit {gate} {g.shape}: {hidden} rows of {g.shape[1]} values expected")
    first, last, step = (experts or slice(None)).indices(g.shape[0])
    if step != 1 or last <= first:
        raise ValueError(f"load_experts: experts={experts} takes none of {g.shape[0]} or leaves gaps")
    n = last - first
    cuda = torch.device(device).type == "cuda"
    with torch.cuda.device(device) if cuda else contextlib.nullcontext():
        stager = stager or _Stager(device)
        w13 = torch.empty((n, 2 * inter, g.shape[2]), dtype=torch.uint8, device=device)
        w2 = torch.empty((n, *d.shape[1:]), dtype=torch.uint8, device=device)
        for src, dst in ((g, w13[:, :inter]), (u, w13[:, inter:]), (d, w2)):
            src, size = src[first:last], dst[0].numel()
            if size <= _CHUNK:                                 # several experts to a chunk: an expert is one row of the copy
                stager.to_device(src.reshape(n, size), dst.as_strided((n, size), (dst.stride(0), 1)))
            else:
                for e in range(n):
                    stager.to_device(src[e], dst[e])
        if cuda:
            torch.cuda.synchronize()
    return w13, w2, t13, t2

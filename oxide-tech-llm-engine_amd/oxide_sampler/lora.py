"""Low-rank adapters of many requests at once, beside the LM head.

`LoraAdapters` is a table of adapters on the GPU in the layout that the
kernels read (`oxs_lora_load`), and adds each row's own adapter to the output
of the projection that all rows share: y_b += B_a (s_a A_a x_b)
(`oxs_lora_add`). `LmHeadQ8_0.project(adapters=...)` calls it.
"""
from __future__ import annotations

import ctypes

from . import _abi
from ._abi import OxsLoraBatch, OxsLoraTable, check, load_library
from .logprobs import _ld, _on

NO_ADAPTER = -1  # OXS_LORA_NONE as int32


def _torch():
    import torch  # noqa: PLC0415 — torch is plumbing for device memory

    if not torch.cuda.is_available():
        raise RuntimeError("no HIP device visible to torch: adapters run on the GPU only")
    return torch


class LoraAdapters:
    """`max_adapters` slots for adapters of rank up to `max_rank` over a
    projection of `k` inputs and `m` outputs, and the workspace for batches of
    up to `max_batch` rows. `dtype` (float32, bfloat16 or float16) is that of
    the weights.

    Calls of one object share its workspace: use one object per stream, and
    one per captured graph that may replay beside another."""

    def __init__(self, m: int, k: int, max_adapters: int, max_rank: int, max_batch: int, dtype=None, device: int = 0):
        t = _torch()
        self.torch = t
        self.lib = load_library()
        self.device = t.device("cuda", device)
        self.dtype = t.bfloat16 if dtype is None else dtype
        kinds = {t.float32: _abi.OXS_DTYPE_F32, t.bfloat16: _abi.OXS_DTYPE_BF16, t.float16: _abi.OXS_DTYPE_F16}
        if self.dtype not in kinds:
            raise TypeError(f"adapter dtype {dtype} is not float32, bfloat16 or float16")
        if min(m, k, max_adapters, max_rank, max_batch) < 1:
            raise ValueError("m, k, max_adapters, max_rank and max_batch must be positive")
        self.m, self.k, self.max_adapters, self.max_rank = int(m), int(k), int(max_adapters), int(max_rank)
        self.max_batch = int(max_batch)
        self.table = OxsLoraTable(self.m, self.k, self.max_adapters, self.max_rank, kinds[self.dtype])
        a, b = ctypes.c_size_t(), ctypes.c_size_t()
        check(self.lib.oxs_lora_table_bytes(self.table, a, b), "oxs_lora_table_bytes")
        self._bytes = int(self.lib.oxs_lora_workspace_bytes(self.table, self.max_batch))
        if self._bytes == 0:
            raise ValueError(f"max_batch {max_batch} is above what one call takes")
        self._a = t.empty(a.value, dtype=t.uint8, device=self.device)
        self._b = t.empty(b.value, dtype=t.uint8, device=self.device)
        self.ranks = t.zeros(self.max_adapters, dtype=t.int32, device=self.device)
        self.scales = t.zeros(self.max_adapters, dtype=t.float32, device=self.device)
        self.workspace = t.empty(self._bytes, dtype=t.uint8, device=self.device)
        t.cuda.current_stream(self.device).synchronize()  # the slots are empty for every stream
        self.table.a, self.table.b = self._a.data_ptr(), self._b.data_ptr()
        self.table.ranks, self.table.scales = self.ranks.data_ptr(), self.scales.data_ptr()

    def _call(self, name, stream, *args):
        s = stream if stream is not None else self.torch.cuda.current_stream(self.device.index)
        call = getattr(self.lib, name)
        if self.torch.cuda.current_device() != self.device.index:
            with self.torch.cuda.device(self.device):
                check(call(self.table, *args, s.cuda_stream), name)
        else:
            check(call(self.table, *args, s.cuda_stream), name)

    def load(self, slot: int, a, b, scale: float = 1.0, stream=None) -> None:
        """Puts an adapter into `slot`: `a` is [rank, k] and `b` [m, rank]
        (device tensors of the table's dtype, any row stride). `scale` is what
        the product is multiplied by (lora_alpha / rank). In stream order:
        steps queued before still use what the slot held."""
        t = self.torch
        _on(a, "a", self.device, (self.dtype,), 2)
        _on(b, "b", self.device, (self.dtype,), 2)
        rank = int(a.shape[0])
        if not 0 <= slot < self.max_adapters:
            raise IndexError(f"slot {slot} outside 0..{self.max_adapters}")
        if not 1 <= rank <= self.max_rank:
            raise ValueError(f"rank {rank} outside 1..{self.max_rank}")
        if a.shape[1] != self.k or tuple(b.shape) != (self.m, rank):
            raise ValueError(f"a must be [rank, {self.k}] and b [{self.m}, rank]")
        if (rank > 1 and a.stride(0) < self.k) or (self.m > 1 and b.stride(0) < rank):
            raise ValueError("the rows of a and b must not overlap")
        self._call("oxs_lora_load", stream, slot, a.data_ptr(), _ld(a), b.data_ptr(), _ld(b), rank, float(scale))
        if stream is not None:
            a.record_stream(stream)
            b.record_stream(stream)

    def unload(self, slot: int, stream=None) -> None:
        """Empties `slot`: its rows become rows without an adapter."""
        if not 0 <= slot < self.max_adapters:
            raise IndexError(f"slot {slot} outside 0..{self.max_adapters}")
        self._call("oxs_lora_load", stream, slot, None, 0, None, 0, 0, 0.0)

    def descriptor(self, y, x, adapters) -> OxsLoraBatch:
        """Describes one call for `launch`: y [batch, m] and x [batch, k]
        (float32 or bfloat16, any row stride), `adapters` int32 [batch] with
        each row's slot (NO_ADAPTER for none). The tensors must outlive the
        launches."""
        t = self.torch
        kinds = {t.float32: _abi.OXS_DTYPE_F32, t.bfloat16: _abi.OXS_DTYPE_BF16}
        _on(y, "y", self.device, tuple(kinds), 2)
        _on(x, "x", self.device, tuple(kinds), 2)
        _on(adapters, "adapters", self.device, (t.int32,), 1)
        batch = int(y.shape[0])
        if y.shape[1] != self.m or tuple(x.shape) != (batch, self.k) or adapters.shape[0] != batch:
            raise ValueError(f"y must be [batch, {self.m}], x [batch, {self.k}] and adapters [batch]")
        if batch > self.max_batch:
            raise ValueError(f"batch {batch} above max_batch {self.max_batch}")
        if batch > 1 and (y.stride(0) < self.m or x.stride(0) < self.k):
            raise ValueError("the rows of y and x must not overlap")
        if batch and adapters.stride(0) != 1 and batch > 1:
            raise ValueError("adapters must be contiguous")
        return OxsLoraBatch(batch, kinds[x.dtype], kinds[y.dtype], x.data_ptr(), _ld(x), y.data_ptr(), _ld(y),
                            adapters.data_ptr(), self.workspace.data_ptr(), self._bytes)

    def launch(self, call: OxsLoraBatch, stream=None) -> None:
        """Launches a described call on `stream` (torch stream or None)."""
        self._call("oxs_lora_add", stream, call)

    def add(self, y, x, adapters, stream=None):
        """y_b += B_a (s_a A_a x_b) in place for every row with an adapter; returns y."""
        self.launch(self.descriptor(y, x, adapters), stream)
        return y

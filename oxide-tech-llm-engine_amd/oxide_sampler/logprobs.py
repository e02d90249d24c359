"""Log probabilities, ranks, entropy and alternatives of whole rows of logits.

`TokenLogprobs.compute` gives what a serving API returns beside a sampled
token, and what scoring a prompt or a set of choices needs, from the same
logits that the sampler reads (`oxs_token_logprobs`). A decode loop whose
buffers stay where they are describes the call once (`descriptor`) and
launches it every step (`launch`).
"""
from __future__ import annotations

import ctypes

from . import _abi
from ._abi import OxsLogprobs, check, load_library


def _torch():
    import torch  # noqa: PLC0415 — torch is plumbing for device memory

    if not torch.cuda.is_available():
        raise RuntimeError("no HIP device visible to torch: log probabilities are computed on the GPU only")
    return torch


def _on(t, what, device, dtypes, dim):
    if t.device != device or t.dtype not in dtypes or t.dim() != dim:
        raise ValueError(f"{what} must be a {dim}-D tensor of {' or '.join(str(d) for d in dtypes)} on {device}")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what} must have a last dimension of stride 1")
    return t


def _ld(t):
    """Elements between rows (a tensor of one row may carry any stride there)."""
    return int(t.stride(0)) if t.shape[0] > 1 else max(int(t.stride(0)), int(t.shape[1]))


class TokenLogprobs:
    """`oxs_token_logprobs` with its workspace on HIP device `device`.

    Calls of one object share its workspace: use one object per stream, and
    one per captured graph that may replay beside another."""

    def __init__(self, device: int = 0):
        t = _torch()
        self.torch = t
        self.lib = load_library()
        self.device = t.device("cuda", device)
        self._bytes = int(self.lib.oxs_logprobs_workspace_bytes())
        self.workspace = t.empty(self._bytes, dtype=t.uint8, device=self.device)

    def descriptor(self, logits, tokens=None, *, top: int = 0, mask=None, temperatures=None, softcap: float = 0.0,
                   out=None):
        """Describes one call: returns (OxsLogprobs, outputs) for `launch`.

        `logits` is [rows, V] float32 or bfloat16 with any row stride of at
        least V; `tokens` int32 [rows] or [rows, T] (T <= 64); `mask` packed
        int32 words [rows, ceil(V / 32)], or one row for all; `temperatures`
        float32 [rows]. The outputs are float32 `logsumexp`, `entropy` and
        int32 `status` [rows]; with tokens, float32 `logprobs` and int32
        `ranks` of the tokens' shape; with `top` (<= 32), int32 `top_ids` (-1
        past the last present token) and float32 `top_logprobs` [rows, top].
        `out` gives some or all of them. The tensors must outlive the launches.
        """
        t = self.torch
        _on(logits, "logits", self.device, (t.float32, t.bfloat16), 2)
        rows, vocab = int(logits.shape[0]), int(logits.shape[1])
        if rows > 1 and vocab and logits.stride(0) < vocab:
            raise ValueError("the rows of logits must not overlap")
        d = OxsLogprobs()
        d.rows, d.vocab = rows, vocab
        d.logits_dtype = _abi.OXS_DTYPE_F32 if logits.dtype == t.float32 else _abi.OXS_DTYPE_BF16
        d.logits, d.logits_ld = logits.data_ptr(), _ld(logits)
        shapes = {"logsumexp": ((rows,), t.float32), "entropy": ((rows,), t.float32), "status": ((rows,), t.int32)}
        if tokens is not None:
            _on(tokens, "tokens", self.device, (t.int32, t.uint32), tokens.dim() if tokens.dim() == 1 else 2)
            if tokens.shape[0] != rows:
                raise ValueError(f"tokens must have {rows} rows")
            two = tokens if tokens.dim() == 2 else tokens.unsqueeze(1)
            if rows > 1 and two.stride(0) < two.shape[1]:
                raise ValueError("the rows of tokens must not overlap")
            d.tokens_per_row = int(two.shape[1])
            if d.tokens_per_row > _abi.OXS_LOGPROBS_MAX_TOKENS:
                raise ValueError(f"at most {_abi.OXS_LOGPROBS_MAX_TOKENS} tokens per row")
            d.tokens, d.tokens_ld = tokens.data_ptr(), _ld(two)
            shapes["logprobs"] = (tuple(tokens.shape), t.float32)
            shapes["ranks"] = (tuple(tokens.shape), t.int32)
        if not 0 <= top <= _abi.OXS_LOGPROBS_MAX_TOP:
            raise ValueError(f"top {top} outside 0..{_abi.OXS_LOGPROBS_MAX_TOP}")
        d.top_n = top
        if top:
            shapes["top_ids"] = ((rows, top), t.int32)
            shapes["top_logprobs"] = ((rows, top), t.float32)
        if mask is not None:
            words = (vocab + 31) // 32
            _on(mask, "mask", self.device, (t.int32, t.uint32), mask.dim() if mask.dim() == 1 else 2)
            if mask.shape[-1] < words or (mask.dim() == 2 and mask.shape[0] != rows):
                raise ValueError(f"mask must be [{rows}, {words}] or [{words}] words")
            d.allowed_mask = mask.data_ptr()
            d.mask_ld = _ld(mask) if mask.dim() == 2 else 0
        if temperatures is not None:
            _on(temperatures, "temperatures", self.device, (t.float32,), 1)
            if temperatures.shape[0] != rows:
                raise ValueError(f"temperatures must be [{rows}]")
            d.temperatures = temperatures.data_ptr()
        d.logit_softcap = float(softcap)
        out = dict(out) if out is not None else {}
        for name, (shape, dtype) in shapes.items():
            o = out.get(name)
            if o is None:
                o = out[name] = t.empty(shape, dtype=dtype, device=self.device)
            elif tuple(o.shape) != shape or o.dtype != dtype or o.device != self.device or not o.is_contiguous():
                raise ValueError(f"out[{name!r}] must be a contiguous {dtype} tensor of shape {shape} on {self.device}")
            setattr(d, "out_" + name, o.data_ptr())
        d.workspace, d.workspace_bytes = self.workspace.data_ptr(), self._bytes
        return d, {name: out[name] for name in shapes}

    def launch(self, call: OxsLogprobs, stream=None) -> None:
        """Launches a described call on `stream` (torch stream or None)."""
        s = stream if stream is not None else self.torch.cuda.current_stream(self.device.index)
        if self.torch.cuda.current_device() != self.device.index:
            with self.torch.cuda.device(self.device):
                check(self.lib.oxs_token_logprobs(call, s.cuda_stream), "oxs_token_logprobs")
        else:
            check(self.lib.oxs_token_logprobs(call, s.cuda_stream), "oxs_token_logprobs")

    def compute(self, logits, tokens=None, *, top: int = 0, mask=None, temperatures=None, softcap: float = 0.0,
                out=None, stream=None):
        """`descriptor` and `launch` in one; returns the outputs. With `stream`,
        the outputs that the call allocates belong to that stream."""
        with self.torch.cuda.stream(stream):
            call, outs = self.descriptor(logits, tokens, top=top, mask=mask, temperatures=temperatures,
                                         softcap=softcap, out=out)
            self.launch(call, stream)
        return outs

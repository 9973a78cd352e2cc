"""Products whose weights every row picks for itself: expert layers (b200q_moe_*) with their routers (b200q_router_*), and low-rank
adapters (b200q_adapters_*).

A `Backend` makes the handles; they keep their weights and workspaces on its GPU until they are closed.  As everywhere
in this package PyTorch only holds device memory and streams.
"""
from __future__ import annotations

import ctypes
from ctypes import byref, c_void_p

import numpy as np

from . import _binding as B


def invalid(text: str) -> "B.B200QError":
    return B.B200QError(B.ERR_INVALID_CONFIG, text)


class Source:
    """Contiguous memory that a create or load call copies from: a NumPy array or a torch tensor, on the host or a GPU."""

    def __init__(self, data, what: str, dtype: str):
        if isinstance(data, np.ndarray):
            if data.dtype.name != dtype:
                raise invalid(f"{what} is {data.dtype}, not {dtype}")
            self.keep = np.ascontiguousarray(data)
            self.ptr, self.bytes, self.shape = self.keep.ctypes.data, self.keep.nbytes, self.keep.shape
            return
        if str(getattr(data, "dtype", "")) != "torch." + dtype:
            raise invalid(f"{what} is {getattr(data, 'dtype', type(data).__name__)}, not {dtype}")
        self.keep = data.detach().contiguous()
        if data.is_cuda:             # the copy runs on a stream of its own: what fills the tensor has to be done
            import torch

            torch.cuda.current_stream(data.device).synchronize()
        self.ptr, self.bytes, self.shape = self.keep.data_ptr(), self.keep.numel() * self.keep.element_size(), tuple(self.keep.shape)


def matrix(t, what: str, device: int, columns: int, dtypes: dict, rows: int | None = None):
    """(pointer, dtype id, leading dimension) of a CUDA tensor [rows, columns] whose rows are contiguous."""
    d, shape = dtypes.get(t.dtype), t.shape
    if d is None or t.get_device() != device or len(shape) != 2 or shape[1] != columns or (rows is not None and shape[0] != rows):
        if t.get_device() != device:
            raise invalid(f"{what} is on {t.device}, not on cuda:{device}")
        if d is None:
            raise invalid(f"{what} is {t.dtype}, not one of {', '.join(map(str, dtypes))}")
        raise invalid(f"{what} has shape {tuple(shape)}, not ({'rows' if rows is None else rows}, {columns})")
    ld, one = t.stride()
    if one != 1 and columns > 1:
        raise invalid(f"the rows of {what} are not contiguous")
    if shape[0] <= 1:
        ld = columns
    elif ld < columns:
        raise invalid(f"the rows of {what} overlap")
    return t.data_ptr(), d, ld


class Handle:
    """An object of the library that a Backend owns."""

    _destroy = ""

    def __init__(self, backend, handle: int):
        self.backend = backend
        self._h = c_void_p(handle)
        backend._children.add(self)

    def close(self) -> None:
        if self._h:
            getattr(B.lib(), self._destroy)(self._h)
            self._h = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class MoeLayer(Handle):
    """The experts of one layer, resident on the GPU (b200q_moe_create); `Backend.run_moe` runs them."""

    _destroy = "b200q_moe_destroy"

    def __init__(self, backend, gate, up, down, *, gate_up_type: int, down_type: int, top_k: int, n_embd: int, n_ff: int, max_rows: int,
                 activation: int, alpha: float, limit: float, gate_bias, up_bias, down_bias):
        parts = {n: Source(v, n, "uint8") for n, v in (("gate", gate), ("up", up), ("down", down))}
        per = B.lib().b200q_tensor_storage_bytes(gate_up_type, n_embd * n_ff)
        if per <= 0 or parts["gate"].bytes % per:
            raise invalid(f"gate: {parts['gate'].bytes} bytes are no whole number of experts of {n_ff} x {n_embd} weights of type {gate_up_type}")
        c = B.MoeConfig()
        c.n_experts, c.top_k, c.n_embd, c.n_ff, c.max_rows = parts["gate"].bytes // per, top_k, n_embd, n_ff, max_rows
        c.gate_up_type, c.down_type = gate_up_type, down_type
        for n, s in parts.items():
            setattr(c, n, s.ptr)
            setattr(c, n + "_bytes", s.bytes)
        for n, v, width in (("gate_bias", gate_bias, n_ff), ("up_bias", up_bias, n_ff), ("down_bias", down_bias, n_embd)):
            if v is not None:
                s = parts[n] = Source(v, n, "float32")
                if s.bytes != 4 * c.n_experts * width:
                    raise invalid(f"{n} has shape {s.shape}, not ({c.n_experts}, {width})")
                setattr(c, n, s.ptr)
        c.activation, c.alpha, c.limit = activation, alpha, limit
        out = c_void_p()
        backend._check(B.lib().b200q_moe_create(backend._h, byref(c), byref(out)))
        super().__init__(backend, out.value)
        self.n_experts, self.top_k, self.n_embd, self.n_ff, self.max_rows = c.n_experts, top_k, n_embd, n_ff, max_rows


class Router(Handle):
    """The router of an expert layer (b200q_router_create); `Backend.route` runs it."""

    _destroy = "b200q_router_destroy"

    def __init__(self, backend, weight, top_k: int, *, scoring: int, normalise: bool, scale: float, logit_bias, select_bias, max_rows: int):
        bf16 = str(getattr(weight, "dtype", "")) == "torch.bfloat16"
        w = Source(weight, "weight", "bfloat16" if bf16 else "float32")
        if len(w.shape) != 2:
            raise invalid(f"weight has shape {w.shape}, not (experts, n_embd)")
        c = B.RouterConfig()
        c.n_experts, c.n_embd = w.shape
        c.top_k, c.max_rows, c.w_dtype, c.scoring = top_k, max_rows, B.TYPE_BF16 if bf16 else B.TYPE_F32, scoring
        c.normalise, c.scale, c.w = bool(normalise), scale, w.ptr
        keep = []
        for n, v in (("logit_bias", logit_bias), ("select_bias", select_bias)):
            if v is not None:
                s = Source(v, n, "float32")
                if s.bytes != 4 * c.n_experts:
                    raise invalid(f"{n} has shape {s.shape}, not ({c.n_experts},)")
                keep.append(s)
                setattr(c, n, s.ptr)
        out = c_void_p()
        backend._check(B.lib().b200q_router_create(backend._h, byref(c), byref(out)))
        super().__init__(backend, out.value)
        self.n_experts, self.n_embd, self.top_k, self.max_rows = c.n_experts, c.n_embd, top_k, max_rows


class AdapterSet(Handle):
    """Numbered slots for the low-rank adapters of one projection (b200q_adapters_create); `Backend.apply_adapters` applies them."""

    _destroy = "b200q_adapters_destroy"

    def __init__(self, backend, n: int, k: int, dtype, max_adapters: int, max_rank: int):
        name = str(dtype).replace("torch.", "")
        kinds = {"float16": B.TYPE_F16, "bfloat16": B.TYPE_BF16}
        if name not in kinds:
            raise invalid(f"adapter dtype {dtype} is not float16 or bfloat16")
        out = c_void_p()
        backend._check(B.lib().b200q_adapters_create(backend._h, n, k, kinds[name], max_adapters, max_rank, byref(out)))
        super().__init__(backend, out.value)
        self.n, self.k, self.dtype, self.max_adapters, self.max_rank = n, k, name, max_adapters, max_rank

    def load(self, slot: int, a, b, scale: float = 1.0) -> None:
        """Puts an adapter into a slot: a [rank, k] and b [n, rank] of the set's dtype, on the host or the GPU."""
        pa, pb = Source(a, "a", self.dtype), Source(b, "b", self.dtype)
        rank = pa.shape[0] if len(pa.shape) == 2 else -1
        if pa.shape != (rank, self.k) or pb.shape != (self.n, rank):
            raise invalid(f"a has shape {pa.shape} and b {pb.shape}, not (rank, {self.k}) and ({self.n}, rank)")
        self.backend._check(B.lib().b200q_adapters_load(self.backend._h, self._h, slot, rank, scale, pa.ptr, pb.ptr))

    def unload(self, slot: int) -> None:
        self.backend._check(B.lib().b200q_adapters_load(self.backend._h, self._h, slot, 0, 0.0, None, None))

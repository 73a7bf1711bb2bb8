"""Query, key and value heads normed and rotated in one pass.

What a layer does to its heads between the projections and the cache::

    rotation = HeadRotation(128, inv_freq, q_weight=wq, k_weight=wk)      # once per layer
    q, k, _ = rotation.apply(q, k, positions=positions)                   # [n, heads, Q, 128]
    out = runtime.append_attend(layer, q, k, v, slots, scale)

The kernel is hand-written for gfx950 behind include/kvrt.h; there is no PyTorch
or CPU path. A call runs on the current torch stream of the rotation's device,
allocates its answers only, keeps nothing and can be captured; calls on several
streams may overlap. Replaces the norm and rotation launches of a listener's or
talker's layer (native/gemma4_listener_microbatch/gemma4_listener_kernels.cuh:
145-500, native/qwen_talker/qwen_talker_kernels.cu:13-205).
"""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from . import _lib as L
from .block8 import _on, _same
from .runtime import _check, calls, current_stream_handle, tensor_desc

_NORMS = {"none": 0, "qk": 3, "qkv": 7}

_calls_mod = None


def _calls():
    """The native call module with the entry point of this module connected."""
    global _calls_mod
    if _calls_mod is None:
        lib, mod = L.load(), calls()
        mod.connect_rotate(ctypes.cast(lib.kvrt_rotate_heads_async, ctypes.c_void_p).value)
        _calls_mod = mod
    return _calls_mod


class HeadRotation:
    """Norms and position rotation of one layer's heads.

    ``inv_freq``: angular frequencies (radians a position), a multiple of 8 of them and
    at most ``head_dim`` / 2 (none: nothing turns); a zero leaves its pair as it is, times
    ``scaling``.
    Pair f is dims (f, f + len(inv_freq)), with ``adjacent`` (2f, 2f + 1); dims past
    all pairs pass. ``axes``: for each frequency the axis (0 to 3) whose position turns
    it, in sections or alternating; default one axis. ``norm``: the kinds that are
    RMS-normed, "none", "qk" or "qkv", with ``eps`` in the root; ``q_weight``,
    ``k_weight`` [head_dim] multiply the normed heads (default ones; values have none).
    ``scaling`` multiplies cosines and sines. Dims that are neither normed nor turned leave
    bit for bit.

    Inference only: no gradient is recorded, of inputs that require one either. Tables and
    weights are copied to ``device``; the copies ``q_weight`` and ``k_weight`` (fp32, or
    None) may be written to in place.
    """

    def __init__(self, head_dim: int, inv_freq: Sequence[float] | torch.Tensor, *,
                 axes: Sequence[int] | None = None, adjacent: bool = False, norm: str = "qk",
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 scaling: float = 1.0, device: torch.device | str | None = None) -> None:
        lib = L.load()
        self.head_dim = int(head_dim)
        if self.head_dim not in (64, 128, 256, 512):
            raise ValueError(f"head_dim must be 64, 128, 256 or 512, got {head_dim}")
        if norm not in _NORMS:
            raise ValueError(f"norm must be one of {sorted(_NORMS)}, got {norm!r}")
        freq = inv_freq.detach() if isinstance(inv_freq, torch.Tensor) else torch.tensor(list(inv_freq), dtype=torch.float64)
        freq = freq.to("cpu", torch.float64).contiguous()
        if freq.dim() != 1 or freq.numel() % 8 != 0 or 2 * freq.numel() > self.head_dim:
            raise ValueError(f"inv_freq must hold a multiple of 8, at most head_dim / 2, frequencies; got {tuple(freq.shape)}")
        n = freq.numel()
        which = [0] * n if axes is None else [int(a) for a in axes]
        if len(which) != n or any(not 0 <= a < 4 for a in which):
            raise ValueError(f"axes must name an axis from 0 to 3 for each of the {n} frequencies")
        if not (0.0 <= float(eps) < float("inf")) or not abs(float(scaling)) < float("inf"):
            raise ValueError("eps must be finite and not negative, scaling finite")
        for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if w is not None and tuple(w.shape) != (self.head_dim,):
                raise ValueError(f"{name} must be [{self.head_dim}], got {tuple(w.shape)}")
            if w is not None and norm == "none":
                raise ValueError(f"{name} without a norm")
        turns = (ctypes.c_uint64 * max(1, n))()
        _check(lib.kvrt_rotation_turns((ctypes.c_double * max(1, n))(*freq.tolist()), n, turns), "kvrt_rotation_turns")
        dev = torch.device(device if device is not None else "cuda")
        if dev.type != "cuda" or not torch.cuda.is_available():
            raise RuntimeError("HeadRotation needs a ROCm GPU (torch.cuda); there is no CPU path")
        self.device = torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev
        self.n_axes = max(which, default=0) + 1
        self.norm = norm

        def copy(t):
            return None if t is None else t.detach().to(self.device, torch.float32, copy=True).contiguous()

        # (uint64 bit patterns as int64)
        self._turns = torch.tensor([ctypes.c_int64(t).value for t in turns], dtype=torch.int64, device=self.device)
        self._axis = torch.tensor(which or [0], dtype=torch.uint8, device=self.device)
        self.q_weight, self.k_weight = copy(q_weight), copy(k_weight)
        torch.cuda.current_stream(self.device).synchronize()  # (calls come on any stream)
        c = L.KvrtRotation()
        c.turns, c.axis = self._turns.data_ptr(), self._axis.data_ptr()
        c.q_weight, c.k_weight = (None if w is None else w.data_ptr() for w in (self.q_weight, self.k_weight))
        c.head_dim, c.n_freq, c.adjacent, c.norm, c.n_axes = self.head_dim, n, int(bool(adjacent)), _NORMS[norm], self.n_axes
        c.eps, c.scaling = float(eps), float(scaling)
        self._c, self._c_at = c, ctypes.addressof(c)
        # the weights that the struct points to (others that a caller assigns are not used)
        self._weights = (self.q_weight, self.k_weight)
        self._lib, self._call = lib, _calls()

    def apply(self, q: torch.Tensor | None, k: torch.Tensor | None = None, v: torch.Tensor | None = None, *,
              positions: torch.Tensor | None = None, out: tuple | None = None) -> tuple:
        """The heads of q, k, v (bf16 [n, heads, Q, head_dim], or packed rows [T, heads,
        head_dim]; each may be None and has its own number of heads) normed and rotated, as a
        tuple of three; None stays None. Views of a projection are read as they are (last dim
        contiguous, 16-byte aligned rows).

        ``positions``: int32 or int64 on the GPU, [n, Q] (packed: [T]) or [axes, n, Q]
        ([axes, T]), values within int32. ``out``: three destinations (None where the input
        is) instead of new contiguous tensors; one may be its input itself, and otherwise
        shares no memory with another tensor of the call."""
        oq, ok, ov = (None, None, None) if out is None else out
        got = self._call.rotate_heads(self._c_at, current_stream_handle(self.device), self.device.index, q, k, v,
                                      positions, oq, ok, ov)
        if type(got) is tuple:
            return got
        if got < 0:
            _check(got, "kvrt_rotate_heads_async")
        heads, descs, outs, packed = (q, k, v), [], [], None
        for t, o, name in zip(heads, (oq, ok, ov), "qkv"):
            if t is None:
                if o is not None:
                    raise ValueError(f"out for {name}, which is None")
                descs.append((None, None))
                outs.append(None)
                continue
            _same(t, name, self.device)
            if t.dim() not in (3, 4) or packed not in (None, t.dim() == 3):
                raise ValueError("q, k and v must be [n, heads, Q, head_dim], or packed rows [T, heads, head_dim]")
            packed = t.dim() == 3
            with _on(self.device):
                o = torch.empty(t.shape, dtype=t.dtype, device=self.device) if o is None else o
            _same(o, f"out of {name}", self.device)
            if o.shape != t.shape:
                raise ValueError(f"out of {name} must be {tuple(t.shape)}, got {tuple(o.shape)}")
            outs.append(o)
            descs.append(tuple(tensor_desc(x.unsqueeze(2) if packed else x) for x in (t, o)))
        if packed is None:
            raise ValueError("apply needs q, k or v")
        pd = None
        if self._c.n_freq:
            if positions is None:
                raise ValueError("apply needs positions")
            _same(positions, "positions", self.device)
            p = positions.unsqueeze(-1) if packed else positions
            p = p.unsqueeze(0) if p.dim() == 2 else p
            pd = ctypes.byref(tensor_desc(p))
        refs = [[None if d is None else ctypes.byref(d) for d in pair] for pair in descs]
        with _on(self.device):
            _check(self._lib.kvrt_rotate_heads_async(
                ctypes.byref(self._c), refs[0][0], refs[1][0], refs[2][0], pd, refs[0][1], refs[1][1], refs[2][1],
                ctypes.c_void_p(current_stream_handle(self.device))), "kvrt_rotate_heads_async")
        return tuple(outs)

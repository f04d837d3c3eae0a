"""Block-scaled 8-bit floating point: quantised rows, weights, expert slabs and the products on them.

Values are ``torch.float8_e4m3fn``.  Rows (activations) carry one power-of-two scale for each run of 128
values (``torch.float8_e8m0fnu``), weights one fp32 scale for each 128 x 128 block, as 8-bit checkpoints
store them: ``weight ~ values * scale``.  Inference only: nothing here has a backward.

    w = Weight.from_quantized(values, scales)      # once, at load time; Weight.quantize(w16) otherwise
    y = linear(x, w)                               # x is quantised inside the call
    rows = quantize(x); y = linear(rows, w)        # ... or once for several products

    slab = ExpertSlab.from_quantized(experts)      # or ExpertSlab.quantize(expert_weights16)
    parts, shared = moe_ffn(slab, x, topv, perm, shared=(gate, up, down), shared_gate=logits)
    ops.combine(parts, perm, shared, T, K, out)
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib, ops, weights
from ._lib import Fp8Matrix, SegList
from .ops import HALF_DTYPES, Permutation, _need, _need_half, _ptr, _same_device, call_on, dtype_code

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
TOP = 448.0


def blocks(n: int) -> int:
    return -(-int(n) // BLOCK)


def padded(n: int) -> int:
    return blocks(n) * BLOCK


# ------------------------------------------------------------------------------- rows
class Rows:
    """Quantised rows as ``quantize`` makes them: ``data [T, padded(K)]`` (zeros behind column K) and
    ``scales [T, blocks(K)]``; ``dtype`` is that of the rows they were made of."""

    __slots__ = ("data", "scales", "cols", "dtype")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, cols: int, dtype: torch.dtype) -> None:
        self.data, self.scales, self.cols, self.dtype = data, scales, cols, dtype

    @property
    def values(self) -> torch.Tensor:
        """The ``[T, K]`` values without the padding."""
        return self.data if self.data.shape[1] == self.cols else self.data[:, :self.cols]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        full = self.data.float().view(*self.scales.shape, BLOCK) * self.scales.float()[..., None]
        return full.reshape(self.data.shape)[:, :self.cols].to(dtype)


def quantize(x: torch.Tensor, out: Optional[Rows] = None) -> Rows:
    """Rows ``x [T, K]`` (bf16, fp16 or fp32) to 8 bits.  The scale of a run of 128 is the smallest
    ``2**s``, ``s >= -120``, with ``max|x| <= 448 * 2**s``; infinities and NaN become NaN and leave the rest
    of their run as it is."""
    _need(x, "x")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [T, K] with K >= 1, got {tuple(x.shape)}")
    T, K = x.shape
    code, index = dtype_code(x.dtype), x.get_device()
    if out is None:
        nb = -(-K // BLOCK)
        out = Rows(x.new_empty((T, nb * BLOCK), dtype=E4M3), x.new_empty((T, nb), dtype=E8M0), K, x.dtype)
    else:
        _need(out.data, "values", E4M3, (T, padded(K)))
        _need(out.scales, "scales", E8M0, (T, blocks(K)))
        out.cols, out.dtype = K, x.dtype
        _same_device(index, out.data, out.scales)
    rc = call_on(index, _lib.load().sparse_hip_fp8_quantize, x.data_ptr(), code, T, K, out.data.data_ptr(),
                 out.scales.data_ptr())
    _lib.check(rc, "sparse_hip_fp8_quantize")
    return out


# ----------------------------------------------------------------------------- weights
def tile_values(q: torch.Tensor) -> torch.Tensor:
    """8-bit values ``[N, K]`` in the kernels' order, flattened, zeros up to 16 rows and 128 columns:
    byte (row, k) goes to ``(row//16)*16*Kp + (k//128)*2048 + ((k//16)%2)*1024 + ((k//32)%4)*256 +
    (row%16)*16 + k%16``."""
    N, K = q.shape
    Np, Kp = -(-N // 16) * 16, padded(K)
    b = q.view(torch.uint8)
    if (Np, Kp) != (N, K):
        full = b.new_zeros((Np, Kp))
        full[:N, :K] = b
        b = full
    v = b.reshape(Np // 16, 16, Kp // 128, 4, 2, 16)       # [group, row, block, quarter, half, k16]
    return v.permute(0, 2, 4, 3, 1, 5).reshape(-1)          # [group, block, half, quarter, row, k16]


def untile_values(flat: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """Inverse of ``tile_values``."""
    Np, Kp = -(-rows // 16) * 16, padded(cols)
    v = flat.view(torch.uint8).reshape(Np // 16, Kp // 128, 2, 4, 16, 16)
    return v.permute(0, 4, 1, 3, 2, 5).reshape(Np, Kp)[:rows, :cols].contiguous().view(E4M3)


def quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(values [N, K] float8_e4m3fn, scales [blocks(N), blocks(K)] fp32)`` of a weight: the scale of a
    128 x 128 block is the smallest power of two ``2**s``, ``s >= -120``, with ``max|w| <= 448 * 2**s`` (the
    division is then exact and each value is rounded once).  Done once, at load time."""
    if w.dim() != 2:
        raise ValueError(f"a weight must be [N, K], got {tuple(w.shape)}")
    if not bool(torch.isfinite(w).all()):
        raise ValueError("a weight must be finite to be quantised")
    N, K = w.shape
    full = torch.zeros((padded(N), padded(K)), dtype=torch.float32, device=w.device)
    full[:N, :K] = w
    v = full.view(blocks(N), BLOCK, blocks(K), BLOCK)
    m, e = torch.frexp(v.abs().amax(dim=(1, 3)))
    s = torch.where(m <= 0.875, e - 9, e - 8)               # 448 = 0.875 * 2**9
    s = torch.where(m == 0, torch.full_like(s, -120), s).clamp_min(-120)
    q = torch.ldexp(v, -s[:, None, :, None]).reshape(full.shape)[:N, :K].to(E4M3).contiguous()
    return q, torch.ldexp(torch.ones_like(m), s)


def _check_quantized(values: torch.Tensor, scales: torch.Tensor, name: str = "weight") -> None:
    if values.dim() != 2 or values.dtype != E4M3 or values.numel() == 0:
        raise ValueError(f"{name} values must be [N, K] {E4M3}, got {tuple(values.shape)} {values.dtype}")
    want = (blocks(values.shape[0]), blocks(values.shape[1]))
    if tuple(scales.shape) != want or scales.dtype != torch.float32:
        raise ValueError(f"{name} scales must be {want} float32, got {tuple(scales.shape)} {scales.dtype}")
    if values.device != scales.device:
        raise ValueError(f"{name} values and scales are on different devices")


def are_pow2(scales: torch.Tensor) -> bool:
    """Whether every scale is a power of two in fp32's normal range.  (Products of many rows take such a scale as an
    exponent, which they find out by themselves.)"""
    m, _ = torch.frexp(scales)
    return bool(((m == 0.5) & (scales >= 2.0 ** -126)).all())


class Weight:
    """A matrix ``[rows, cols]`` laid out for the kernels (``data``, bytes in ``tile_values``' order), with its block
    ``scales``.  Both may be written into; they cannot be exchanged for other tensors, whose place the kernels would
    not know: make another ``Weight``, on another device too."""

    __slots__ = ("_data", "_scales", "rows", "cols", "desc", "ref")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, rows: int, cols: int) -> None:
        self._data, self._scales, self.rows, self.cols = data, scales, int(rows), int(cols)
        size = -(-self.rows // 16) * 16 * padded(self.cols)
        if data.dtype != torch.uint8 or data.numel() != size or not data.is_contiguous():
            raise ValueError(f"a [{rows}, {cols}] weight is {size} contiguous bytes, got {tuple(data.shape)} {data.dtype}")
        want = (blocks(self.rows), blocks(self.cols))
        if scales.dtype != torch.float32 or tuple(scales.shape) != want or not scales.is_contiguous():
            raise ValueError(f"weight scales must be {want} contiguous float32, got {tuple(scales.shape)} {scales.dtype}")
        if data.device != scales.device:
            raise ValueError("weight values and scales are on different devices")
        self.desc = Fp8Matrix(data.data_ptr(), scales.data_ptr(), self.rows, self.cols)
        self.ref = C.byref(self.desc)

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    @property
    def shape(self) -> Tuple[int, int]:
        return self.rows, self.cols

    @property
    def pow2(self) -> bool:
        """Whether every scale is a power of two, as they are now (reads them back)."""
        return are_pow2(self.scales)

    @classmethod
    def from_quantized(cls, values: torch.Tensor, scales: torch.Tensor) -> "Weight":
        """From a checkpoint's 8-bit values ``[N, K]`` and fp32 scales ``[blocks(N), blocks(K)]``."""
        _check_quantized(values, scales)
        return cls(tile_values(values.contiguous()).contiguous(), scales.contiguous().clone(), *values.shape)

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Weight":
        return cls.from_quantized(*quantize_weight(w))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        q = untile_values(self.data, self.rows, self.cols).to(wide)
        s = self.scales.to(wide).repeat_interleave(BLOCK, 0)[:self.rows].repeat_interleave(BLOCK, 1)[:, :self.cols]
        return (q * s).to(dtype)


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    p, q = a.data_ptr(), b.data_ptr()
    return p < q + b.numel() * b.element_size() and q < p + a.numel() * a.element_size()


def linear(x: Union[torch.Tensor, Rows], weight: Weight, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x W^T`` with ``x [T, K]`` (bf16 or fp16) quantised inside the call, or given as ``Rows`` of such an x:
    ``[T, N]`` in x's dtype, accumulated in fp32 and rounded once.  (From three rows on the matrix instruction forms
    sums of eight products with 13 bits below the largest: some ``2**-15`` of a usual result.)  ``out`` must not share
    memory with x."""
    dtype = x.dtype
    if dtype not in HALF_DTYPES:
        raise ValueError(f"x must be bfloat16 or float16, got {dtype}")
    rows = type(x) is Rows
    src = x.data if rows else x
    _need(src, "x")
    if src.dim() != 2:
        raise ValueError(f"x must be [T, K], got {tuple(src.shape)}")
    T, K = src.shape
    if rows:
        K = x.cols
        _need(src, "values", E4M3, (T, padded(K)))
        _need(x.scales, "scales", E8M0, (T, blocks(K)))
    if K != weight.cols:
        raise ValueError(f"x has {K} columns, the weight {weight.cols}")
    index = src.get_device()
    if out is None:
        out = src.new_empty((T, weight.rows), dtype=dtype)
    else:
        _need(out, "out", dtype, (T, weight.rows))
        _same_device(index, out)
        if overlap(out, src):
            raise ValueError("out overlaps x, which is read while out is written")
    _same_device(index, weight._data, x.scales if rows else None)
    lib = _lib.load()
    if rows:
        rc = call_on(index, lib.sparse_hip_fp8_linear, None, src.data_ptr(), x.scales.data_ptr(), dtype_code(dtype), T,
                     weight.ref, 1, out.data_ptr(), None)
    else:
        need = lib.sparse_hip_fp8_linear_ws_bytes(T, K)       # 0: the product quantises its rows itself
        ws = src.new_empty((need,), dtype=torch.uint8) if need else None
        rc = call_on(index, lib.sparse_hip_fp8_linear, src.data_ptr(), None, None, dtype_code(dtype), T, weight.ref, 1,
                     out.data_ptr(), _ptr(ws))
    _lib.check(rc, "sparse_hip_fp8_linear")
    return out


# ----------------------------------------------------------------------------- experts
Quantized = Tuple[torch.Tensor, torch.Tensor]


def slot_bytes(hidden: int, inter: int) -> int:
    """Bytes of one expert: gate, up and down values, then their scales, rounded up to 256."""
    return int(_lib.load().sparse_hip_fp8_slot_bytes(int(hidden), int(inter)))


def pack_expert_into(dst: torch.Tensor, expert: Tuple[Quantized, Quantized, Quantized], hidden: int, inter: int) -> None:
    """Lay one expert's (gate, up, down) (values, scales) pairs into one slot of bytes."""
    at = 0
    for (q, s), shape, name in zip(expert, ((inter, hidden), (inter, hidden), (hidden, inter)), ("gate", "up", "down")):
        _check_quantized(q, s, name)
        if tuple(q.shape) != shape:
            raise ValueError(f"{name} must be {shape}, got {tuple(q.shape)}")
        t = tile_values(q.contiguous())
        dst[at:at + t.numel()].copy_(t)
        at += t.numel()
    for _, s in expert:
        b = s.contiguous().view(torch.uint8).reshape(-1)
        dst[at:at + b.numel()].copy_(b)
        at += b.numel()
    dst[at:].zero_()


class ExpertSlab:
    """8-bit experts of one layer in HBM, one slot each.  Host segment lists name the slots of their experts;
    with a device list expert e is in slot e.  ``data`` may be written into, not exchanged for another tensor."""

    def __init__(self, num_slots: int, num_experts: int, hidden: int, inter: int, device) -> None:
        if hidden % 64 or inter % 64 or hidden <= 0 or inter <= 0:
            raise ValueError(f"hidden and inter must be positive multiples of 64, got {hidden}, {inter}")
        self.hidden, self.inter = int(hidden), int(inter)
        self.num_slots, self.num_experts = int(num_slots), int(num_experts)
        self.expert_bytes = slot_bytes(hidden, inter)
        self._data = torch.empty((self.num_slots, self.expert_bytes), dtype=torch.uint8, device=device)
        self._refs: dict = {}

    @classmethod
    def from_quantized(cls, experts: Sequence[Tuple[Quantized, Quantized, Quantized]], device=None) -> "ExpertSlab":
        """All experts resident, slot == expert id; ``experts[e]`` is (gate, up, down), each (values, scales)."""
        gate = experts[0][0][0]
        slab = cls(len(experts), len(experts), gate.shape[1], gate.shape[0], device if device is not None else gate.device)
        for e, expert in enumerate(experts):
            pack_expert_into(slab.data[e], expert, slab.hidden, slab.inter)
        return slab

    @classmethod
    def quantize(cls, experts: Sequence[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]], device=None) -> "ExpertSlab":
        """The same from 16- or 32-bit (gate, up, down) weights."""
        return cls.from_quantized([tuple(quantize_weight(w) for w in triple) for triple in experts], device)

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @property
    def pow2(self) -> bool:
        """Whether every scale of every slot is a power of two, as they are now (reads them back)."""
        at = 2 * self.inter * padded(self.hidden) + self.hidden * padded(self.inter)
        size = 4 * 3 * blocks(self.hidden) * blocks(self.inter)
        return are_pow2(self.data[:, at:at + size].contiguous().view(torch.float32))

    def slot_ptr(self, slot: int) -> int:
        return self.data.data_ptr() + int(slot) * self.expert_bytes

    def descriptor(self, dtype: torch.dtype):
        """The slab as the C entry takes it, for activations of ``dtype``; built once per dtype."""
        ref = self._refs.get(dtype)
        if ref is None:
            ref = C.byref(_lib.Experts(self.data.data_ptr(), self.expert_bytes, None, self.num_experts, self.hidden,
                                       self.inter, dtype_code(dtype)))
            self._refs[dtype] = ref
        return ref


class HostExpertArena(weights.HostExpertArena):
    """All routed experts of a layer as 8-bit slots in pinned host memory, one row per expert id: an upload is
    one copy of half the bytes of the 16-bit arena's."""

    def __init__(self, experts: Sequence[Tuple[Quantized, Quantized, Quantized]], hidden: int, inter: int,
                 pin: bool = True) -> None:
        self.hidden, self.inter, self.dtype = int(hidden), int(inter), torch.uint8
        self._allocate(len(experts), slot_bytes(hidden, inter), torch.uint8, pin)
        for e, expert in enumerate(experts):
            pack_expert_into(self.rows[e], expert, hidden, inter)


def module_weight(linear_mod, device=None) -> Quantized:
    """(values, scales) of a ``Linear``-like module: its own where it holds 8-bit weights with
    ``weight_scale_inv`` (the layout of 8-bit checkpoints, one scale per 128 x 128 block), else quantised."""
    w = linear_mod.weight.detach()
    if w.dtype == E4M3:
        s = getattr(linear_mod, "weight_scale_inv", None)
        if s is None:
            raise ValueError("an 8-bit weight needs weight_scale_inv")
        pair = w, s.detach().to(torch.float32)
        _check_quantized(*pair)
        return (pair[0].to(device), pair[1].to(device)) if device is not None else pair
    return quantize_weight(w if device is None else w.to(device))


def moe_ffn_ws_bytes(T: int, K: int, num_experts: int, num_segments: int, hidden: int, inter: int,
                     shared_inter: int = 0) -> int:
    return int(_lib.load().sparse_hip_fp8_moe_ffn_ws_bytes(int(T), int(K), int(num_experts), int(num_segments),
                                                           int(hidden), int(inter), int(shared_inter)))


def moe_ffn(experts: ExpertSlab, x: torch.Tensor, topv: torch.Tensor, perm: Permutation,
            shared: Optional[Tuple[Weight, Weight, Weight]] = None, shared_gate: Optional[torch.Tensor] = None,
            segs: Optional[SegList] = None, parts: Optional[torch.Tensor] = None,
            shared_out: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None
            ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Routed experts (over ``segs``, by default every active one) and the shared expert of one call of any
    size on 8-bit weights: returns ``(parts [T*K, H]`` in permuted order, each row times its route weight,
    ``shared [T, H]`` or None``)`` for ``ops.combine``.  ``x [T, H]`` bf16 or fp16, ``topv [T, K]`` of the same
    dtype; ``shared_gate [T]``: logits whose sigmoid multiplies the shared rows.  Gate and up, which are rounded to 8
    bits next, are products added in fp32 at every size; the down projection is summed as in ``linear``.  ``ws``: a byte tensor of
    ``moe_ffn_ws_bytes`` for callers that keep one."""
    _need_half(x, "x")
    if x.dim() != 2 or topv.dim() != 2:
        raise ValueError("x must be [T, H] and topv [T, K]")
    T, H = x.shape
    K = topv.shape[1]
    dtype, E, index = x.dtype, experts.num_experts, x.get_device()
    if H != experts.hidden:
        raise ValueError(f"x has hidden {H}, the expert slab has {experts.hidden}")
    _need(topv, "topv", dtype, (T, K))
    if perm.perm.numel() != T * K or perm.seg_offsets.numel() != E + 1:
        raise ValueError(f"the permutation does not belong to {T} tokens x {K} over {E} experts")
    if segs is None:
        segs = ops.seglist_device(perm, min(E, T * K))
    if segs.eids_dev:
        if experts.num_slots < E:
            raise ValueError(f"a device segment list needs a slot for each of the {E} experts, the slab has {experts.num_slots}")
    elif any(not 0 <= s < experts.num_slots for s in segs.slots[:segs.n]):
        raise ValueError(f"the segment list names slots outside the slab's {experts.num_slots}")
    if parts is None:
        parts = x.new_empty((T * K, H))
    else:
        _need(parts, "parts", dtype, (T * K, H))
    gate = up = down = None
    Is = 0
    if shared is not None:
        gate, up, down = shared
        Is = down.cols
        for m, want, name in ((gate, (Is, H), "gate_proj"), (up, (Is, H), "up_proj"), (down, (H, Is), "down_proj")):
            if (m.rows, m.cols) != want:
                raise ValueError(f"shared {name} must be {want}, got {m.shape}")
        _same_device(index, gate.data, up.data, down.data)
        gate, up, down = gate.ref, up.ref, down.ref
        if shared_gate is not None:
            _need(shared_gate, "shared gate logits", dtype)
            if shared_gate.numel() != T:
                raise ValueError("shared gate logits must hold T elements")
        if shared_out is None:
            shared_out = x.new_empty((T, H))
        else:
            _need(shared_out, "shared out", dtype, (T, H))
    else:
        shared_gate = shared_out = None
    if T == 0:
        return parts, shared_out
    lib = _lib.load()
    need = lib.sparse_hip_fp8_moe_ffn_ws_bytes(T, K, E, segs.n, H, experts.inter, Is)
    if ws is None:
        ws = x.new_empty((max(1, need),), dtype=torch.uint8)
    elif not ws.is_contiguous() or ws.numel() * ws.element_size() < need:
        raise ValueError(f"the workspace must hold {need} contiguous bytes")
    _same_device(index, topv, perm.perm, experts.data, parts, shared_gate, shared_out, ws)
    rc = call_on(index, lib.sparse_hip_fp8_moe_ffn, experts.descriptor(dtype), x.data_ptr(), topv.data_ptr(),
                 perm.perm.data_ptr(), perm.seg_offsets.data_ptr(), C.byref(segs), T, K, parts.data_ptr(), gate, up, down,
                 _ptr(shared_gate), 1, _ptr(shared_out), ws.data_ptr())
    _lib.check(rc, "sparse_hip_fp8_moe_ffn")
    return parts, shared_out
